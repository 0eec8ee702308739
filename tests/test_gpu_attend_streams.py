"""LayerCache.attend called on another stream than the bank's."""
import pytest

pytestmark = pytest.mark.gpu

H, D, TPF, FRAMES, TEXT = 2, 128, 40, 2, 8
L = FRAMES * TPF + TEXT


@pytest.mark.parametrize("history", [False, True])
def test_attend_waits_for_the_callers_stream(nkv, history):
    """Inputs still being written on the caller's stream, and the result read there, without a wait of the caller's."""
    import torch
    from nomas_kv import _abi
    g = torch.Generator(device="cuda").manual_seed(5)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()  # noqa: E731
    bank = nkv.KvBank(nkv.CacheConfig(storage=nkv.CacheStorage.int8(), sampling=nkv.HistorySampling.uniform(),
                                      past_frames=4), 1, 1, H, D, torch.bfloat16)
    try:
        if history:
            bank.commit_tensors(_abi.nkv_segment_desc(0, 0, FRAMES, FRAMES * TPF, TEXT, -1), [r(1, L, H, D)],
                                [r(1, L, H, D)])
        plan = nkv.AttendPlan([L], H, block=TPF)
        real = [r(L, H, D) for _ in range(3)]
        want, want_lse = (t.clone() for t in bank.layer(0).attend(plan, *real))
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            late = [torch.zeros_like(t) for t in real]
            torch.cuda._sleep(40_000_000)  # some 20 ms
            for t, x in zip(late, real):
                t.copy_(x)
            out, lse = bank.layer(0).attend(plan, *late)
            got, got_lse = out.clone(), lse.clone()
            del out, lse
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
        # memory given up by the caller while the bank's stream still reads it is not handed out again
        torch.cuda._sleep(40_000_000)  # the bank's stream (this one) is busy
        with torch.cuda.stream(side):
            again = [x.clone() for x in real]
            out, lse = bank.layer(0).attend(plan, *again)
            shapes = [t.shape for t in again]
            del again
            junk = [torch.full(s, 7.0, dtype=torch.bfloat16, device="cuda") for s in shapes]
            got, got_lse = out.clone(), lse.clone()
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
        del junk
        plan.check()
    finally:
        bank.close()


def test_attend_on_another_stream_in_a_graph(nkv):
    import torch
    bank = nkv.KvBank(nkv.CacheConfig(storage=nkv.CacheStorage.int8(), sampling=nkv.HistorySampling.uniform(),
                                      past_frames=4), 1, 1, H, D, torch.bfloat16, stream=torch.cuda.Stream())
    try:
        plan = nkv.AttendPlan([L], H, block=TPF)
        bufs = [torch.randn((L, H, D), device="cuda").bfloat16() for _ in range(3)]
        want, want_lse = (t.clone() for t in bank.layer(0).attend(plan, *bufs))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out, lse = bank.layer(0).attend(plan, *bufs)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
        g.reset()
    finally:
        bank.close()


def test_a_refused_call_leaves_the_streams_usable(nkv):
    import torch
    from nomas_kv import _abi
    bank = nkv.KvBank(nkv.CacheConfig(storage=nkv.CacheStorage.int8(), sampling=nkv.HistorySampling.uniform(),
                                      past_frames=4), 1, 1, H, D, torch.bfloat16)
    try:
        kv = [torch.randn((1, L, H, D), device="cuda").bfloat16() for _ in range(2)]
        bank.commit_tensors(_abi.nkv_segment_desc(0, 0, FRAMES, FRAMES * TPF, TEXT, -1), [kv[0]], [kv[1]])
        plan = nkv.AttendPlan([L], H, block=TPF)
        q = torch.randn((L, H, D), device="cuda").bfloat16()
        want, _ = bank.layer(0).attend(plan, q, q, q)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            with pytest.raises(nkv.GeometryError):
                bank.layer(0).attend(plan, q, q[:-1], q)
            got, _ = bank.layer(0).attend(plan, q, q, q)
            assert torch.equal(got, want)
    finally:
        bank.close()
