"""The operators of the attention block in a run, as a model's layer uses them
around the cache: residual_norm -> rope_tables -> kv_project -> rotary(q) ->
LayerCache.attend (history from the INT8 archive, merged with the current
segment) -> the staged commit -> residual_norm, over several segments, against
a float64 chain over the bank's own working set and the projected K / V.

Tolerances, before any run: the history part's output is within 2e-2 and its
log-sum-exp within 2e-3 (test_gpu_attend_history.py); the merge weights sum to
1, and a log-sum-exp error of 2e-3 moves them by as much of outputs whose
magnitude is below 4: 2e-2 + 8e-3; the current part adds half a step of bf16 of
P (2^-8 of at most 4) and the output's own rounding, 2^-8 each: 6e-2 in all.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

H, D, TPF, FRAMES, TEXT = 2, 128, 40, 2, 8
DIM, L = H * D, FRAMES * TPF + TEXT


def _positions(segment):
    import torch
    rows = [(segment * FRAMES + f, r, c) for f in range(FRAMES) for r in range(5) for c in range(8)]
    rows += [(segment * FRAMES + FRAMES - 1, 0, i) for i in range(TEXT)]
    return torch.tensor(rows, dtype=torch.int32, device="cuda")


def _attention64(q, ks, vs, seen):
    """softmax over the concatenated keys; seen: (queries, keys) of each part."""
    import torch
    k, v, m = torch.cat(ks).double(), torch.cat(vs).double(), torch.cat(seen, dim=1)
    s = torch.einsum("qhd,khd->hqk", q.double(), k) / math.sqrt(D)
    s = s.masked_fill(~m[None], -math.inf)
    return torch.einsum("hqk,khd->qhd", torch.softmax(s, dim=-1), v), torch.logsumexp(s, dim=-1)


def _seen(n_hist):
    """Every query sees the history and, of its segment, its frame and those before it."""
    import torch
    i = torch.arange(L, device="cuda")
    cur = i[None, :] < ((i // TPF + 1) * TPF).clamp(max=L)[:, None]
    return torch.ones((L, n_hist), dtype=torch.bool, device="cuda"), cur


def test_a_layer_over_several_segments(nkv):
    import torch
    from nomas_kv import _abi
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    w = {n: (r(DIM, DIM) / math.sqrt(DIM)).bfloat16() for n in ("wq", "wk", "wv")}
    gain = (1 + 0.1 * r(D)).bfloat16()
    norm_w, scale, shift, gate = 1 + 0.1 * r(DIM), 0.1 * r(3, DIM), 0.1 * r(3, DIM), 0.5 * r(3, DIM)
    frame = torch.tensor([0] * TPF + [1] * TPF + [2] * TEXT, dtype=torch.int32, device="cuda")
    axes = nkv.RotaryAxes((44, 42, 42))
    plan = nkv.AttendPlan([L], H, block=TPF)
    bank = nkv.KvBank(nkv.CacheConfig(storage=nkv.CacheStorage.int8(), sampling=nkv.HistorySampling.uniform(),
                                      past_frames=4), 1, 1, H, D, torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    try:
        for seg in range(4):
            x, pos = r(L, DIM).bfloat16(), _positions(seg)
            h0, y = nkv.residual_norm(x, weight=norm_w, scale=scale, shift=shift, mod_index=frame)
            assert h0 is x
            rope = nkv.rope_tables(pos, axes)
            k, v = torch.empty_like(y), torch.empty_like(y)
            nkv.kv_project(y, w["wk"], w["wv"], k_gain=gain, rope=rope, k_out=k, v_out=v, status=status)
            q0 = (y @ w["wq"].t()).view(L, H, D)
            q = nkv.rotary(pos, axes, q0, norm=True, q_weight=gain)
            # q has gone the way of kv_project's K: the same projection, norm, rotation (which rounds once more)
            kq = torch.empty_like(y)
            nkv.kv_project(y, w["wq"], w["wv"], k_gain=gain, rope=rope, k_out=kq, v_out=torch.empty_like(y),
                           status=status)
            assert float((kq.view(L, H, D).float() - q.float()).abs().max()) <= 3 * 2.0 ** -7 * float(q.abs().max())
            kc, vc = k.view(L, H, D), v.view(L, H, D)
            layer = bank.layer(0)
            kh, vh = (t[0] for t in layer.working_set())
            out, lse = layer.attend(plan, q, kc, vc)
            ref, ref_lse = _attention64(q, (kh, kc), (vh, vc), _seen(kh.shape[0]))
            assert float((out.double() - ref).abs().max()) <= 6e-2
            assert float((lse.double() - ref_lse).abs().max()) <= 4e-3
            # the same over the materialised working set, as storage without attend_history does it
            if kh.shape[0]:
                part = torch.empty((L, H, D), device="cuda")
                every = nkv.AttendPlan([L], H, k_lens=[kh.shape[0]], causal=False)
                hist = nkv.attend_packed(every, q, kh, vh, out=part)
                out2, lse2 = nkv.attend_packed(plan, q, kc, vc, history=hist)
                assert float((out2.double() - ref).abs().max()) <= 4 * 2.0 ** -7
                assert float((lse2.double() - ref_lse).abs().max()) <= 1e-3
                every.check()
            bank.commit_projected(_abi.nkv_segment_desc(seg, seg * FRAMES, FRAMES, FRAMES * TPF, TEXT, -1), [y],
                                  [dict(wk=w["wk"], wv=w["wv"], k_gain=gain)], rope=rope)
            h, y2 = nkv.residual_norm(x, out.view(L, DIM), gate=gate, post="rms", norm="layer", scale=scale, shift=shift,
                                      mod_index=frame)
            b = out.view(L, DIM).double()
            b = b / torch.sqrt((b * b).mean(1, keepdim=True) + 1e-6) * gate.double()[frame.long()]
            assert float((h.double() - (x.double() + b)).abs().max()) <= 2.0 ** -7 * float(h.abs().max())
            assert bool(y2.isfinite().all())
        assert bank.layer(0).n_segments() == 4 and int(status.item()) == 0
        plan.check()
    finally:
        bank.close()


@pytest.mark.parametrize("storage", ["floating", "qvg_"])
def test_other_storage_attends_over_the_working_set(nkv, storage):
    """The history part over a FLOAT or QVG bank's working set (its views in place), merged with the current segment."""
    import torch
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()  # noqa: E731
    bank = nkv.KvBank(nkv.CacheConfig(storage=getattr(nkv.CacheStorage, storage)(),
                                      sampling=nkv.HistorySampling.uniform(), past_frames=4), 2, 1, H, D, torch.bfloat16)
    try:
        from nomas_kv import _abi
        for seg in range(3):
            bank.commit_tensors(_abi.nkv_segment_desc(seg, seg * FRAMES, FRAMES, FRAMES * TPF, TEXT, -1),
                                [r(1, L, H, D) for _ in range(2)], [r(1, L, H, D) for _ in range(2)])
        q, kc, vc = r(L, H, D), r(L, H, D), r(L, H, D)
        plan = nkv.AttendPlan([L], H, block=TPF)
        for i in range(2):
            with pytest.raises(nkv.InvalidConfigError, match="INT8"):
                bank.layer(i).attend(plan, q, kc, vc)
            kh, vh = (t[0] for t in bank.layer(i).working_set())
            every = nkv.AttendPlan([L], H, k_lens=[kh.shape[0]], causal=False)
            hist = nkv.attend_packed(every, q, kh, vh, out=torch.empty((L, H, D), device="cuda"))
            out, lse = nkv.attend_packed(plan, q, kc, vc, history=hist)
            ref, ref_lse = _attention64(q, (kh, kc), (vh, vc), _seen(kh.shape[0]))
            assert float((out.double() - ref).abs().max()) <= 4 * 2.0 ** -7
            assert float((lse.double() - ref_lse).abs().max()) <= 1e-3
    finally:
        bank.close()


def test_attend_refuses_another_geometry_and_a_parked_bank(nkv):
    import torch
    bank = nkv.KvBank(nkv.CacheConfig(storage=nkv.CacheStorage.int8(), sampling=nkv.HistorySampling.uniform(),
                                      past_frames=4, phase_swap=True), 1, 1, H, D, torch.bfloat16)
    try:
        from nomas_kv import _abi
        t = [torch.randn((1, L, H, D), device="cuda").bfloat16() for _ in range(2)]
        q = t[0][0]
        with pytest.raises(nkv.GeometryError, match="heads"):
            bank.layer(0).attend(nkv.AttendPlan([L], 4), q, q, q)
        plan = nkv.AttendPlan([L], H, block=TPF)
        alone, _ = bank.layer(0).attend(plan, q, q, q)  # an empty history: the segment alone
        assert torch.equal(alone, nkv.attend_packed(plan, q, q, q)[0])
        bank.commit_tensors(_abi.nkv_segment_desc(0, 0, FRAMES, FRAMES * TPF, TEXT, -1), [t[0]], [t[1]])
        bank.park_all()
        with pytest.raises(nkv.CacheStateError, match="parked"):
            bank.layer(0).attend(plan, q, q, q)
        bank.unpark_all()
        bank.layer(0).attend(plan, q, q, q)
    finally:
        bank.close()
