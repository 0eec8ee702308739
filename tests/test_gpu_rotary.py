"""Rotary positions with several axes (nkv_rotary, nkv_rope_tables) against
their definition in float64.

Tolerances, before any run.  cos and sin: the f64 angle is exact to far below
f32, the reduced f32 argument is off by half a step (2^-25 of at most pi / 4),
the f32 functions by 2 ulp of values up to 1 (2^-23 each): 3 * 2^-24 * 2 <=
2^-21.  An output: u |y| for its rounding, and, with r the pair's length, 2^-21
r for the table, 3 * 2^-24 r for the products and the sum, and for the norm (D
/ 2 + 8) 2^-24 r for the sum of squares, the root and the products.
"""
import math
import types

import pytest

pytestmark = pytest.mark.gpu


def _angles(pos, dims, theta):
    import torch
    cols = []
    for a, d in enumerate(dims):
        f = torch.tensor([theta ** (-2.0 * i / d) for i in range(d // 2)], dtype=torch.float64, device=pos.device)
        cols.append(pos[:, a].double()[:, None] * f[None, :])
    return torch.cat(cols, dim=1)


def _reference(x, ang, inter, w=None, norm=False, eps=1e-6):
    import torch
    y = x.double()
    if norm:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if w is not None:
            y = y * w.double()
    n = ang.shape[1]
    a_, b_ = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if inter else (slice(0, n), slice(n, 2 * n))
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, b = y[..., a_].clone(), y[..., b_].clone()
    r = y.abs()
    r[..., a_] = r[..., b_] = torch.sqrt(a * a + b * b)
    out = y.clone()
    out[..., a_], out[..., b_] = a * c - b * s, b * c + a * s
    return out, r


def _check(got, x, ang, inter, w=None, norm=False, eps=1e-6):
    import torch
    ref, r = _reference(x, ang, inter, w, norm, eps)
    D = x.shape[-1]
    tol = torch.finfo(x.dtype).eps / 2 * ref.abs() + (2.0 ** -21 + 3 * 2.0 ** -24 + norm * (D / 2 + 8) * 2.0 ** -24) * r
    if x.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # below the normal range
    bad = (got.double() - ref).abs() > tol + 1e-37
    assert got.dtype == x.dtype and not bool(bad.any()), f"{int(bad.sum())} outside"


def _pos(T, n, kind, span=5000, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = torch.randint(-span, span, (T, n), generator=g, device="cuda")
    if kind == "float32":
        return (p + torch.rand((T, n), generator=g, device="cuda")).float()
    return p.to(getattr(torch, kind))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("inter", [True, False])
@pytest.mark.parametrize("T,H,KV,D,dims", [
    (1, 1, 1, 128, (44, 42, 42)), (5, 24, 24, 128, (128,)), (33, 6, 2, 128, (32, 24, 24)), (70, 3, 0, 64, (16, 16, 32)),
    (9, 1, 1, 16, (16,)), (9, 2, 1, 32, (2, 2, 2, 2)), (130, 2, 2, 256, (64, 64, 128)), (7, 5, 3, 96, (32, 32, 32)),
    (40, 2, 1, 80, (26, 26, 28)), (11, 1, 2, 10, (4, 2)), (3, 2, 2, 254, (250,)), (2, 1, 1, 2, (2,)),
    (65, 1, 1, 128, (30, 20)), (12, 7, 1, 232, (54, 52)),
])
def test_matches_float64(nkv, T, H, KV, D, dims, inter, dtype):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(T)
    q = torch.randn((T, H, D), generator=g, device="cuda").to(dt)
    k = torch.randn((T, KV, D), generator=g, device="cuda").to(dt) if KV else None
    qw = (1 + 0.2 * torch.randn((D,), generator=g, device="cuda")).to(dt)
    kw = (1 + 0.2 * torch.randn((D,), generator=g, device="cuda")).to(dt) if KV else None
    axes = nkv.RotaryAxes(dims, theta=10000.0, interleaved=inter)
    for kind in ("int32", "int64", "float32"):
        pos = _pos(T, len(dims), kind)
        ang = _angles(pos, dims, 10000.0)
        got = nkv.rotary(pos, axes, q, k=k)
        got = (got, None) if k is None else got
        _check(got[0], q, ang, inter)
        if k is not None:
            _check(got[1], k, ang, inter)
    got = nkv.rotary(pos, axes, q, k=k, norm=True, q_weight=qw, k_weight=kw, eps=1e-5)
    got = (got, None) if k is None else got
    _check(got[0], q, ang, inter, qw, True, 1e-5)
    if k is not None:
        _check(got[1], k, ang, inter, kw, True, 1e-5)
        only_q = nkv.rotary(pos, axes, q, k=k, norm=True, q_weight=qw)
        _check(only_q[1], k, ang, inter, None, True)


def test_zero_position_is_the_identity(nkv):  # rope.rs apply_rotary_identity_at_zero_position
    import torch
    q = torch.randn((6, 3, 128), device="cuda").to(torch.bfloat16)
    pos = torch.zeros((6, 3), dtype=torch.int32, device="cuda")
    assert torch.equal(nkv.rotary(pos, nkv.RotaryAxes((44, 42, 42)), q), q)


@pytest.mark.parametrize("span", [200_000, 2 ** 31 - 1])
def test_far_positions_keep_their_angles(nkv, span):
    import torch
    pos = _pos(501, 2, "int64", span=span, seed=3)
    axes = nkv.RotaryAxes((64, 64))
    cos, sin = nkv.rope_tables(pos, axes)
    ang = _angles(pos, (64, 64), 10000.0)
    # an f64 angle of up to 2^31 is itself uncertain by 2^-22
    tol = 2.0 ** -21 + span * 2.0 ** -52
    assert float((cos.double() - ang.cos()).abs().max()) <= tol and float((sin.double() - ang.sin()).abs().max()) <= tol


@pytest.mark.parametrize("T", [0, 1, 77, 6496])
def test_tables(nkv, T):
    import torch
    pos = _pos(T, 3, "int32", span=100)
    axes = nkv.RotaryAxes((44, 42, 42))
    cos, sin = nkv.rope_tables(pos, axes)
    assert cos.shape == sin.shape == (T, 64) and cos.dtype == torch.float32
    ang = _angles(pos, (44, 42, 42), 10000.0)
    if T:
        assert float((cos.double() - ang.cos()).abs().max()) <= 2.0 ** -21
        assert float((sin.double() - ang.sin()).abs().max()) <= 2.0 ** -21
    out = (torch.empty_like(cos), torch.empty_like(sin))
    got = nkv.rope_tables(pos, axes, cos=out[0], sin=out[1])
    assert got[0] is out[0] and torch.equal(cos, out[0]) and torch.equal(sin, out[1])


@pytest.mark.parametrize("D,inter", [(128, True), (128, False), (72, False), (72, True)])
def test_views_and_in_place(nkv, D, inter):
    """q and k as views of one fused projection, head-major tensors, outputs in place."""
    import torch
    T, H, KV = 37, 4, 2
    dt = torch.bfloat16
    x = torch.randn((T, H + 2 * KV, D), device="cuda").to(dt)
    x0 = x.clone()
    axes = nkv.RotaryAxes((16, 24, 32), interleaved=inter)
    pos = _pos(T, 3, "int32")
    w = (1 + 0.1 * torch.randn(D, device="cuda")).to(dt)
    kw = dict(norm=True, q_weight=w, k_weight=w)
    want = nkv.rotary(pos, axes, x[:, :H].contiguous(), k=x[:, H:H + KV].contiguous(), **kw)
    got = nkv.rotary(pos, axes, x[:, :H], k=x[:, H:H + KV], **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(x, x0)
    hm = x[:, :H].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(nkv.rotary(pos, axes, hm, norm=True, q_weight=w), want[0])
    odd = torch.zeros((T * H * D + 3,), dtype=dt, device="cuda")[3:].view(T, H, D)  # not 16-byte aligned
    odd.copy_(x[:, :H])
    assert float((nkv.rotary(pos, axes, odd, norm=True, q_weight=w).float() - want[0].float()).abs().max()) <= \
        2.0 ** -7 * float(want[0].float().abs().max())
    q, k = x[:, :H], x[:, H:H + KV]
    r = nkv.rotary(pos, axes, q, k=k, q_out=q, k_out=k, **kw)
    assert r[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    assert torch.equal(x[:, H + KV:], x0[:, H + KV:])  # v untouched


def test_nonfinite_values_stay_in_their_pairs(nkv):
    import torch
    q = torch.randn((4, 2, 128), device="cuda").to(torch.bfloat16)
    q[1, 0, 126] = math.inf     # passes through
    q[2, 1, 4] = math.nan       # pair 2
    pos = _pos(4, 1, "int32")
    out = nkv.rotary(pos, nkv.RotaryAxes((64,)), q)
    assert out[1, 0, 126].item() == math.inf and bool(out[1, 0, 127].isfinite())
    bad = ~out.isfinite()
    bad[1, 0, 126] = False
    assert bad.nonzero().tolist() == [[2, 1, 4], [2, 1, 5]]


def test_offsets_past_32_bits(nkv):
    import torch
    T, W = 9000, 1 << 18
    buf = torch.empty((T, 1, W), dtype=torch.bfloat16, device="cuda")  # 4.7 GB
    q, k = torch.randn((T, 1, 128), device="cuda").bfloat16(), torch.randn((T, 1, 128), device="cuda").bfloat16()
    qw, kw = buf[..., :128], buf[..., W - 128:]
    qw.copy_(q)
    kw.copy_(k)
    pos, axes = _pos(T, 3, "int32"), nkv.RotaryAxes((44, 42, 42))
    want = nkv.rotary(pos, axes, q, k=k, norm=True)
    got = nkv.rotary(pos, axes, qw, k=kw, norm=True, q_out=qw, k_out=kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = nkv.RotaryAxes((36, 2))
    want = nkv.rotary(pos[:, :2].contiguous(), odd, q[..., :44].contiguous())  # the path for any head_dim
    qw.copy_(q)
    assert torch.equal(nkv.rotary(pos[:, :2].contiguous(), odd, qw[..., :44]), want)


def test_graph_and_other_stream(nkv):
    import torch
    T = 300
    q = torch.randn((T, 4, 128), device="cuda").to(torch.bfloat16)
    pos = _pos(T, 3, "int32")
    axes = nkv.RotaryAxes((44, 42, 42))
    want, tabs = nkv.rotary(pos, axes, q), nkv.rope_tables(pos, axes)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out, t = nkv.rotary(pos, axes, q), nkv.rope_tables(pos, axes)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(t[0], tabs[0])
    q.mul_(2)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.float(), 2 * want.float())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    r = nkv.rotary(pos, axes, q, stream=s)
    s.synchronize()
    assert torch.equal(r, out)
    g.reset()


def test_refusals(nkv):
    import torch
    q = torch.zeros((4, 2, 64), dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros((4, 1), dtype=torch.int32, device="cuda")
    ax = nkv.RotaryAxes((64,))
    ge, ae = nkv.GeometryError, nkv.ArgumentError
    for err, kw in [
        (ge, dict(positions=pos[:3])), (ge, dict(positions=pos.double())), (ge, dict(positions=pos.expand(4, 2))),
        (ge, dict(axes=nkv.RotaryAxes((64, 2)))), (ge, dict(axes=nkv.RotaryAxes((66,)))), (ge, dict(q=q[..., ::2])),
        (ge, dict(q=q[..., :63])), (ge, dict(q=q.to(torch.int32))), (ge, dict(q=q[0])), (ge, dict(k=q[:3])),
        (ge, dict(k=q.float())), (ae, dict(q_weight=q[0, 0])), (ae, dict(k_weight=q[0, 0], norm=True)),
        (ge, dict(norm=True, q_weight=q[0, 0].float())), (ge, dict(norm=True, q_weight=q[0, 0, :32])),
        (ge, dict(q_out=q.float())), (ge, dict(q_out=q[:, :1].expand(4, 2, 64))),
        (ae, dict(q=q[:, :1], q_out=q[:, 1:].clone().as_strided((4, 1, 64), (64, 64, 1)), k=None,
                  positions=pos.cpu())),
        (ae, dict(q=q.clone().requires_grad_())), (ae, dict(norm=True, eps=-1.0)), (ae, dict(norm=True, eps=1e60)),
        (ae, dict(norm=True, eps=math.nan)),
    ]:
        a = dict(positions=pos, axes=ax, q=q)
        a.update(kw)
        with pytest.raises(err):
            nkv.rotary(**a)
    x = torch.zeros((5, 2, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ae, match="overlaps"):
        nkv.rotary(pos, ax, x[:4], q_out=x[1:])
    with pytest.raises(ae, match="overlaps"):
        nkv.rotary(pos, ax, q, k=x[:4], q_out=x[:4])
    for kw in (dict(q_out=q), dict(k_out=q), dict(q_out=q, k_out=q)):  # one tensor read as both
        with pytest.raises(ae, match="overlaps"):
            nkv.rotary(pos, ax, q, k=q, **kw)
    one, two = nkv.rotary(pos, ax, q, k=q)
    assert torch.equal(one, two)
    with pytest.raises(ae, match="stream"):
        nkv.rotary(pos, ax, q, stream=types.SimpleNamespace(device_index=1, cuda_stream=0))
    with pytest.raises(ae, match="overlaps"):
        t = torch.empty((4, 32), device="cuda")
        nkv.rope_tables(pos, ax, cos=t, sin=t)
    assert nkv.rotary(pos[:0], ax, q[:0]).shape == (0, 2, 64)
    assert nkv.rotary(pos, ax, q[:, :0]).shape == (4, 0, 64)
