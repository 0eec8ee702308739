"""The compiled binding of the block operators against block.py's own path: the
same results bit for bit, and None (so that block.py answers) for every call
that is not plain or not valid."""
import math

import pytest

pytestmark = pytest.mark.gpu


class _Off:
    def __getattr__(self, name):
        return lambda *a: None


@pytest.fixture
def both(nkv, monkeypatch):
    """Runs f through the binding, which has to take it, and without it."""
    from nomas_kv import block
    real, taken = block._block_binding, []

    class Watched:
        def __getattr__(self, name):
            def call(*a):
                taken.append(getattr(real, name)(*a))
                return taken[-1]
            return call

    def run(f):
        taken.clear()
        monkeypatch.setattr(block, "_block_binding", Watched())
        got = f()
        assert len(taken) == 1 and taken[0] is not None
        monkeypatch.setattr(block, "_block_binding", _Off())
        want = f()
        monkeypatch.setattr(block, "_block_binding", real)
        return got, want
    return run


def _equal(got, want):
    import torch
    if got is None or want is None:
        assert got is None and want is None
    elif isinstance(got, tuple):
        assert len(got) == len(want)
        for a, b in zip(got, want):
            _equal(a, b)
    else:
        assert got.shape == want.shape and got.dtype == want.dtype and got.device == want.device
        if got.numel():  # (an empty tensor's strides mean nothing)
            assert got.stride() == want.stride()
            assert torch.equal(got.view(torch.uint8).flatten(), want.view(torch.uint8).flatten())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("heads", [(3, 2), (4, None), (1, 1)])
def test_rotary_and_tables(nkv, both, dtype, heads):
    import torch
    dt, T, D = getattr(torch, dtype), 37, 64
    fused = torch.randn((T, 8, D), device="cuda").to(dt)
    q = fused[:, :heads[0]]
    k = None if heads[1] is None else fused[:, 5:5 + heads[1]]
    w = torch.randn(D, device="cuda").to(dt)
    for pt in (torch.int32, torch.int64, torch.float32):
        pos = torch.randint(0, 900, (T, 2), device="cuda").to(pt)
        for axes in (nkv.RotaryAxes((32, 32)), nkv.RotaryAxes((16, 14), interleaved=False)):
            _equal(*both(lambda: nkv.rope_tables(pos, axes)))
            _equal(*both(lambda: nkv.rotary(pos, axes, q, k=k)))
            _equal(*both(lambda: nkv.rotary(pos, axes, q, k=k, norm=True, q_weight=w, k_weight=None if k is None else w,
                                            eps=1e-5)))
    _equal(*both(lambda: nkv.rotary(pos[:0], axes, q[:0])))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("dim", [96, 95])
def test_residual_norm(nkv, both, dtype, dim):
    import torch
    dt, T = getattr(torch, dtype), 11
    x, b = (torch.randn((T, dim), device="cuda").to(dt) for _ in range(2))
    w = torch.randn(dim, device="cuda")
    m = torch.randn((3, dim), device="cuda")
    i = torch.randint(0, 3, (T,), dtype=torch.int32, device="cuda")
    for kw in (dict(), dict(norm="layer", weight=w), dict(branch=b, norm=None), dict(branch=b, post="rms", post_weight=w),
               dict(branch=b, post="layer", gate=m, scale=m, shift=m, mod_index=i, weight=w, eps=1e-3),
               dict(branch=b, gate=m[0], scale=m[1].to(dt) if dt == torch.float32 else m[1]),
               dict(scale=m[0].to(dt), weight=w.to(dt))):
        _equal(*both(lambda: nkv.residual_norm(x, **kw)))
    h, _ = nkv.residual_norm(x)
    assert h is x


@pytest.mark.parametrize("split", [False, True])
def test_attend_packed(nkv, both, split):
    import torch
    ql, kl = ([5, 0, 300], [70, 3, 300]) if not split else ([1], [9000])
    for dt in (torch.bfloat16, torch.float16):
        q = torch.randn((sum(ql), 6, 64), device="cuda").to(dt)
        kv = torch.randn((sum(kl) + 4, 4, 64), device="cuda").to(dt)
        plan = nkv.AttendPlan(ql, 6, kv_heads=2, head_dim=64, k_lens=kl)
        assert bool(plan.split_units) == split
        hist = (torch.randn(q.shape, device="cuda"), torch.randn((6, q.shape[0]), device="cuda"))
        for h in (None, hist):
            for scale in (None, 0.3, 1):
                _equal(*both(lambda: nkv.attend_packed(plan, q, kv[:, :2], kv[:, 2:], scale=scale, history=h)))
        plan.check()
        plan.close()
        with pytest.raises(nkv.ArgumentError, match="closed"):
            nkv.attend_packed(plan, q, kv[:, :2], kv[:, 2:])


def test_other_calls_are_left_to_the_other_path(nkv):
    import torch
    from nomas_kv import _block_binding as fast
    q = torch.randn((4, 2, 64), device="cuda")
    pos, ax = torch.zeros((4, 2), dtype=torch.int32, device="cuda"), nkv.RotaryAxes((32, 32))._packed
    w, e = torch.ones(64, device="cuda"), 1e-6
    assert fast.rotary(ax, pos, q, None, True, w, None, e, None, None) is not None
    leaf = q.clone().requires_grad_()
    for args in ((ax, pos, leaf, None, False, None, None, e), (ax, pos.cpu(), q, None, False, None, None, e),
                 (ax, pos, q.cpu(), None, False, None, None, e), (ax, pos[:3], q, None, False, None, None, e),
                 (ax, pos, q[..., ::2], None, False, None, None, e), (ax, pos, q, q.half(), False, None, None, e),
                 (ax, pos, q, None, False, w, None, e), (ax, pos, q, None, True, w[:32], None, e),
                 (ax, pos, q, None, True, w.half(), None, e), (ax, pos, q, None, True, w, w, e),
                 (ax, pos, q, None, True, w, None, -1.0), (ax, pos, q, None, True, w, None, math.nan),
                 (ax, pos, q, None, 1, w, None, e), (ax, pos, q.int(), None, False, None, None, e),
                 (ax[:-1], pos, q, None, False, None, None, e), (ax, pos, None, None, False, None, None, e),
                 (ax, pos, "q", None, False, None, None, e), (ax, pos, q), (),
                 (nkv.RotaryAxes((64, 64))._packed, pos, q, None, False, None, None, e)):
        assert fast.rotary(*args, None, None) is None
        assert fast.rotary(*args) is None
    with torch.no_grad():
        assert fast.rotary(ax, pos, leaf, None, False, None, None, e, None, None) is not None
    assert fast.rope_tables(ax, pos.double(), None, None) is None and fast.rope_tables(ax, pos[:, :1], None, None) is None
    x, m = torch.randn((4, 32), device="cuda"), torch.randn((2, 32), device="cuda")
    i = torch.zeros(4, dtype=torch.int32, device="cuda")
    full = dict(x=x, branch=x.clone(), gate=m, post=1, post_weight=m[0], norm=1, weight=m[0], scale=m, shift=m, mod_index=i,
                eps=e, h_out=None, y_out=None)
    assert fast.residual_norm(*full.values()) is not None
    for kw in (dict(branch=None), dict(branch=x[:3]), dict(gate=m[:, :31]), dict(gate=m[:1]), dict(mod_index=None),
               dict(mod_index=i.long()), dict(norm=0), dict(post=7), dict(norm=-1), dict(weight=m[0].half()),
               dict(scale=m.half()), dict(shift=m.t().contiguous().t()), dict(x=x.t()), dict(eps=None), dict(x=x[0]),
               dict(x=x.double()), dict(weight=m), dict(mod_index=i[:3])):
        assert fast.residual_norm(*{**full, **kw}.values()) is None
    assert fast.residual_norm(*{**full, **dict(gate=None, scale=None, shift=None)}.values()) is None  # an index of nothing
    b = torch.randn((4, 2, 64), device="cuda").bfloat16()
    plan = nkv.AttendPlan([4], 2, head_dim=64)
    key = plan._key
    assert fast.attend_packed(key, b, b, b, None, None, None, None, None) is not None
    big = torch.randn((5, 2, 64), device="cuda").bfloat16()
    ho, hl = torch.zeros((4, 2, 64), device="cuda"), torch.zeros((2, 4), device="cuda")
    assert fast.attend_packed(key, b, big, big, None, ho, hl, None, None) is not None
    off = torch.empty(4 * 2 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 2, 64)
    for args in ((key, big, b, b, None, None, None), (key, b, b[:3], b, None, None, None), (key, b, b, b.half(), None, None, None),
                 (key, b.float(), b, b, None, None, None), (key, b, b, b, 0.0, None, None), (key, b, b, b, math.nan, None, None),
                 (key, b, b, b, 3e38, None, None), (key, b, b, b, "s", None, None), (key, b, b, b, None, ho, None),
                 (key, b, b, b, None, ho[:, :1], hl), (key, b, b, b, None, ho, hl[:, :3]), (key, b, b, off, None, None, None),
                 (key, b, b, b, None, ho.bfloat16(), hl), (None, b, b, b, None, None, None), (key, b, b, b)):
        assert fast.attend_packed(*args, None, None) is None
    plan.check()


def test_given_outputs(nkv, both):
    """In place, into columns of a fused buffer, into outputs of the caller's: taken, and the same values."""
    import torch
    T, D = 9, 64
    buf = torch.randn((T, 5, D), device="cuda").bfloat16()
    pos, ax = torch.randint(0, 99, (T, 2), device="cuda"), nkv.RotaryAxes((32, 32))
    want = nkv.rotary(pos, ax, buf[:, :3], k=buf[:, 3:], norm=True)

    def in_place():
        b = buf.clone()
        q, k = b[:, :3], b[:, 3:]
        got = nkv.rotary(pos, ax, q, k=k, norm=True, q_out=q, k_out=k)
        assert got[0] is q and got[1] is k
        return b

    for b in both(in_place):
        assert torch.equal(b, torch.cat(want, dim=1))

    def tables():
        out = torch.empty((T, 32), device="cuda"), torch.empty((T, 32), device="cuda")
        got = nkv.rope_tables(pos, ax, cos=out[0], sin=out[1])
        assert got[0] is out[0] and got[1] is out[1]
        return got
    _equal(*both(tables))

    x0, b0 = (torch.randn((T, 96), device="cuda").bfloat16() for _ in range(2))
    h, y = nkv.residual_norm(x0, b0, post="rms")

    def stream():
        x, b = x0.clone(), b0.clone()
        got = nkv.residual_norm(x, b, post="rms", h_out=x, y_out=b)
        assert got[0] is x and got[1] is b
        return got
    for got in both(stream):
        _equal(got, (h, y))

    q = torch.randn((T, 2, D), device="cuda").bfloat16()
    plan = nkv.AttendPlan([T], 2, head_dim=D)
    for dt in (torch.bfloat16, torch.float32):
        def attend():
            out, lse = torch.empty((T, 2, D), dtype=dt, device="cuda"), torch.empty((2, T), device="cuda")
            got = nkv.attend_packed(plan, q, q, q, out=out, lse=lse)
            assert got[0] is out and got[1] is lse
            return got
        _equal(*both(attend))
    plan.check()


def test_outputs_that_do_not_fit_are_left_to_the_other_path(nkv):
    import torch
    from nomas_kv import _block_binding as fast
    e, T, D = 1e-6, 4, 64
    big = torch.randn((T + 1, 4, D), device="cuda")
    q, pos, ax = big[:T, :2], torch.zeros((T, 2), dtype=torch.int32, device="cuda"), nkv.RotaryAxes((32, 32))._packed
    k = big[:T, 2:]
    one = torch.empty((T, 2, D), device="cuda")
    for qo, ko, kk in ((q.half(), None, k), (one[:3], None, k), (one.expand(T, 2, D)[:, :1].expand(T, 2, D), None, k),
                       (big[1:, :2], None, k), (k, None, k), (None, q, k), (one, one, k), (q, None, q), (None, q, q),
                       (one.transpose(1, 2).contiguous().transpose(1, 2), None, k), (one, one, None),
                       (one.cpu(), None, k), ("x", None, k), (big[:T, 1:3], None, k)):
        assert fast.rotary(ax, pos, q, kk, False, None, None, e, qo, ko) is None
    assert fast.rotary(ax, pos, q, k, False, None, None, e, q, k) is not None
    t = torch.empty((T, 32), device="cuda")
    for c, s in ((t, t), (t.half(), None), (t[:3], None), (torch.empty((32, T), device="cuda").t(), None)):
        assert fast.rope_tables(ax, pos, c, s) is None
    m = torch.randn((T + 1, 32), device="cuda")
    x, b, w = m[:T], torch.randn((T, 32), device="cuda"), torch.randn(32, device="cuda")
    for ho, yo in ((m[1:], None), (None, m[1:]), (x, x), (b, b), (x.half(), None), (w.expand(T, 32), None),
                   (torch.empty((32, T), device="cuda").t(), None)):
        assert fast.residual_norm(x, b, None, 0, None, 1, w, None, None, None, e, ho, yo) is None
    assert fast.residual_norm(x, None, None, 0, None, 1, w, None, None, None, e, b, None) is None
    assert fast.residual_norm(x, b, None, 0, None, 0, None, None, None, None, e, None, b) is None
    a = torch.randn((T, 2, D), device="cuda").bfloat16()
    plan = nkv.AttendPlan([T], 2, head_dim=D)
    f = torch.empty((2, T), device="cuda")
    for out, lse in ((a, None), (a.half(), None), (torch.empty((T + 1, 2, D), device="cuda"), None), (None, f.half()),
                     (None, torch.empty((T, 2), device="cuda").t()), (torch.empty((2, T, D), device="cuda").transpose(0, 1), None)):
        assert fast.attend_packed(plan._key, a, a, a, None, None, None, out, lse) is None
    buf = torch.empty(T * 2 * D, device="cuda")
    assert fast.attend_packed(plan._key, a, a, a, None, None, None, buf.view(T, 2, D), buf[:2 * T].view(2, T)) is None


def test_plans_made_and_dropped_during_a_capture(nkv):
    import torch
    q = torch.randn((20, 2, 64), device="cuda").bfloat16()
    old, plan = nkv.AttendPlan([20], 2, head_dim=64), nkv.AttendPlan([20], 2, head_dim=64)
    want = nkv.attend_packed(plan, q, q, q)
    plans = []
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = nkv.attend_packed(plan, q, q, q)
        old.close()
        plans.append(nkv.AttendPlan([5, 15], 2, head_dim=64, causal=False))
        got2 = nkv.attend_packed(plans[0], q, q, q)
    g.replay()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    _equal(got2, nkv.attend_packed(plans[0], q, q, q))
    for p in (plan, *plans):
        p.check()


def test_a_captured_call(nkv):
    """The binding's calls in a graph: outputs from the graph's pool, on the capturing stream."""
    import torch
    pos, ax = torch.arange(40, dtype=torch.int32, device="cuda").view(20, 2), nkv.RotaryAxes((32, 32))
    q = torch.randn((20, 2, 64), device="cuda").bfloat16()
    plan = nkv.AttendPlan([20], 2, head_dim=64)
    want = nkv.attend_packed(plan, nkv.rotary(pos, ax, q), q, q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = nkv.attend_packed(plan, nkv.rotary(pos, ax, q), q, q)
    q2 = torch.randn_like(q)
    keep = q.clone()
    q.copy_(q2)
    g.replay()
    want2 = nkv.attend_packed(plan, nkv.rotary(pos, ax, q2), q2, q2)
    assert torch.equal(got[0], want2[0]) and torch.equal(got[1], want2[1])
    q.copy_(keep)
    g.replay()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
