"""The gated residual norm (nkv_residual_norm) against its definition in
float64.

Tolerances, before any run.  e = 64 * 2^-24 bounds the relative error of an f32
sum over a row (a tree over at most 2^5 values a thread, 2^5 lanes and 2^5
warps, plus the root and a few products); a centred value is off by e times
the row's mean magnitude.  With b_n, y_n the normalised values, m the mean
magnitude before the norm and i the factor 1 / sqrt(...):
  E(b_n) = e (|b_n| + m_b i_b),  E(h) = e |x| + |G| E(b_n) + e |G b_n|,
  E(y_n) = e (|y_n| + m_h i_h) + 2 i_h max_row E(h),
  E(y) = |W| E(y_n) + e (|W y_n| + |S|); each output adds u |output|.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

E = 64 * 2.0 ** -24


def _norm(v, kind, eps):
    """normalised values, mean magnitude, factor"""
    import torch
    m = v.abs().mean(1, keepdim=True)
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    i = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + eps)
    return v * i, m, i


def _check(x, b, got, gate=None, post=None, post_weight=None, norm="rms", weight=None, scale=None, shift=None,
           mod_index=None, eps=1e-6):
    import torch
    u = torch.finfo(x.dtype).eps / 2
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 1e-37

    def row(t):
        t = t.double().reshape(-1, x.shape[1])
        return t[mod_index.long()] if mod_index is not None else t

    h, Eh = x.double(), torch.zeros_like(x, dtype=torch.float64)
    if b is not None:
        bn, G = b.double(), torch.ones((1, 1), dtype=torch.float64, device=x.device)
        Eb = torch.zeros_like(bn)
        if post not in (None, "none"):
            bn, m, i = _norm(bn, post, eps)
            Eb = E * (bn.abs() + m * i)
        if post_weight is not None:
            G = G * post_weight.double()
        if gate is not None:
            G = G * row(gate)
        h = h + G * bn
        Eh = E * x.double().abs() + G.abs() * Eb + E * (G * bn).abs()
        bad = (got[0].double() - h).abs() > u * h.abs() + Eh + tiny
        assert got[0].dtype == x.dtype and not bool(bad.any()), f"h: {int(bad.sum())} outside"
    if norm in (None, "none"):
        assert got[1] is None
        return
    yn, m, i = _norm(h, norm, eps)
    En = E * (yn.abs() + m * i) + 2 * i * Eh.amax(1, keepdim=True)
    W = torch.ones((1, 1), dtype=torch.float64, device=x.device)
    if weight is not None:
        W = W * weight.double()
    if scale is not None:
        W = W * (1 + row(scale))
    S = row(shift) if shift is not None else torch.zeros((1, 1), dtype=torch.float64, device=x.device)
    y = yn * W + S
    Ey = W.abs() * En + E * ((W * yn).abs() + S.abs())
    bad = (got[1].double() - y).abs() > u * y.abs() + Ey + tiny
    assert got[1].dtype == x.dtype and not bool(bad.any()), f"y: {int(bad.sum())} outside"


def _make(T, dim, dt, groups, md, seed=0, branch=True):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    a = dict(x=(2 * r(T, dim) + 3).to(dt), b=r(T, dim).to(dt) if branch else None,
             gate=(0.5 * r(groups, dim)).to(md), scale=(0.3 * r(groups, dim)).to(md), shift=r(groups, dim).to(md),
             post_weight=(1 + 0.2 * r(dim)).to(md), weight=(1 + 0.2 * r(dim)).to(md))
    a["mod_index"] = torch.randint(0, groups, (T,), generator=g, device="cuda", dtype=torch.int32) if groups > 1 else None
    return a


@pytest.mark.parametrize("dtype,mod", [("bfloat16", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32"),
                                       ("float32", "float32")])
@pytest.mark.parametrize("T,dim", [(1, 1), (3, 7), (1, 8), (5, 64), (300, 96), (9, 1155), (2, 2048), (700, 1024),
                                   (64, 5120), (3, 8192), (5, 8200), (3, 16384), (2, 16392), (2, 32768), (3, 32767),
                                   (1, 10001)])
def test_matches_float64(nkv, T, dim, dtype, mod):
    import torch
    for groups in (1, 4):
        a = _make(T, dim, getattr(torch, dtype), groups, getattr(torch, mod), seed=dim)
        x, b = a.pop("x"), a.pop("b")
        for post in (None, "rms", "layer"):
            for norm in ("rms", "layer"):
                kw = dict(a, post=post, norm=norm)
                if post is None:
                    kw.pop("post_weight")
                _check(x, b, nkv.residual_norm(x, b, **kw), **kw)


@pytest.mark.parametrize("dim", [256, 333])
def test_every_part_is_optional(nkv, dim):
    import torch
    a = _make(20, dim, torch.bfloat16, 1, torch.float32)
    x, b = a["x"], a["b"]
    for kw in (dict(), dict(weight=a["weight"]), dict(scale=a["scale"]), dict(shift=a["shift"][0]),
               dict(weight=a["weight"], scale=a["scale"][0], shift=a["shift"], norm="layer")):
        h, y = nkv.residual_norm(x, **kw)
        assert h is x
        _check(x, None, (h, y), **kw)
        _check(x, b, nkv.residual_norm(x, b, **kw), **kw)
    for kw in (dict(norm=None), dict(norm=None, gate=a["gate"]), dict(norm="none", post="layer"),
               dict(norm=None, post_weight=a["post_weight"]), dict(norm="rms", gate=a["gate"][0], post="rms")):
        _check(x, b, nkv.residual_norm(x, b, **kw), **kw)


def test_constant_and_zero_rows(nkv):
    """A row of one value (variance 0), of zeros, and a large mean with a small spread."""
    import torch
    x = torch.zeros((3, 512), device="cuda")
    x[1] = 5.0
    x[2] = 1000.0 + torch.randn(512, device="cuda")
    for norm in ("rms", "layer"):
        h, y = nkv.residual_norm(x, norm=norm)
        assert bool(y.isfinite().all())
        _check(x, None, (h, y), norm=norm)
    assert bool((nkv.residual_norm(x, norm="layer")[1][:2].abs() < 1e-3).all())


@pytest.mark.parametrize("dim", [512, 513])
def test_index_out_of_range_gives_nan_rows(nkv, dim):
    import torch
    a = _make(12, dim, torch.bfloat16, 3, torch.float32)
    idx = torch.tensor([0, 1, 2, 3, -1, 0, 2 ** 31 - 1, -2 ** 31, 1, 2, 0, 1], dtype=torch.int32, device="cuda")
    kw = dict(gate=a["gate"], scale=a["scale"], shift=a["shift"])
    h, y = nkv.residual_norm(a["x"], a["b"], mod_index=idx, **kw)
    bad = torch.tensor([3, 4, 6, 7], device="cuda")
    good = torch.tensor([0, 1, 2, 5, 8, 9, 10, 11], device="cuda")
    assert bool(h[bad].isnan().all()) and bool(y[bad].isnan().all())
    _check(a["x"][good], a["b"][good], (h[good], y[good]), mod_index=idx[good], **kw)
    one = nkv.residual_norm(a["x"], scale=a["scale"][:1], mod_index=torch.ones(12, dtype=torch.int32, device="cuda"))
    assert bool(one[1].isnan().all())


@pytest.mark.parametrize("dim", [640, 641])
def test_strides_and_in_place(nkv, dim):
    import torch
    a = _make(50, dim, torch.bfloat16, 1, torch.float32)
    kw = dict(gate=a["gate"], post="rms", post_weight=a["post_weight"], weight=a["weight"], scale=a["scale"])
    want = nkv.residual_norm(a["x"], a["b"], **kw)
    wide = torch.zeros((50, 2 * dim + 16), dtype=torch.bfloat16, device="cuda")
    wide[:, :dim], wide[:, dim + 8:2 * dim + 8] = a["x"], a["b"]
    xs, bs = wide[:, :dim], wide[:, dim + 8:2 * dim + 8]
    keep = wide.clone()
    got = nkv.residual_norm(xs, bs, **kw)
    assert float((got[0].float() - want[0].float()).abs().max()) <= 2.0 ** -7 * float(want[0].abs().max())
    _check(a["x"], a["b"], got, **kw)
    assert torch.equal(wide, keep)
    got = nkv.residual_norm(xs, bs, h_out=xs, y_out=bs, **kw)  # both in place
    assert got[0] is xs and got[1] is bs
    _check(a["x"], a["b"], (xs, bs), **kw)
    assert torch.equal(wide[:, dim:dim + 8], keep[:, dim:dim + 8])
    rows = a["x"][:1].expand(50, dim)  # one broadcast row
    _check(rows, a["b"], nkv.residual_norm(rows, a["b"], **kw), **kw)


@pytest.mark.parametrize("dim", [256, 255])
def test_offsets_past_32_bits(nkv, dim):
    import torch
    T, W = 9000, 1 << 18
    a = _make(T, dim, torch.bfloat16, 4, torch.float32)
    buf = torch.empty((T, W), dtype=torch.bfloat16, device="cuda")  # 4.7 GB
    x, b = buf[:, :dim], buf[:, W - 256:W - 256 + dim]
    x.copy_(a["x"])
    b.copy_(a["b"])
    kw = dict(gate=a["gate"], scale=a["scale"], shift=a["shift"], mod_index=a["mod_index"], post="rms")
    want = nkv.residual_norm(a["x"], a["b"], **kw)
    got = nkv.residual_norm(x, b, h_out=x, y_out=b, **kw)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_graph_and_other_stream(nkv):
    import torch
    a = _make(100, 512, torch.bfloat16, 1, torch.float32)
    kw = dict(gate=a["gate"], weight=a["weight"], scale=a["scale"], shift=a["shift"])
    want = nkv.residual_norm(a["x"], a["b"], **kw)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        got = nkv.residual_norm(a["x"], a["b"], **kw)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = nkv.residual_norm(a["x"], a["b"], stream=s, **kw)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    g.reset()


def test_refusals(nkv):
    import torch
    x = torch.zeros((4, 64), dtype=torch.bfloat16, device="cuda")
    b = torch.zeros_like(x)
    v, m = torch.zeros(64, device="cuda"), torch.zeros((2, 64), device="cuda")
    idx = torch.zeros(4, dtype=torch.int32, device="cuda")
    ge, ae = nkv.GeometryError, nkv.ArgumentError
    for err, kw in [
        (ge, dict(x=x[0])), (ge, dict(x=x.t())), (ge, dict(x=x.to(torch.int32))), (ge, dict(branch=b[:3])),
        (ge, dict(branch=b.float())), (ae, dict(gate=v)), (ae, dict(post="rms")), (ae, dict(norm="batch")),
        (ae, dict(norm=None)), (ae, dict(branch=b, norm=None, scale=v)), (ge, dict(scale=m)),
        (ge, dict(scale=m, shift=v, mod_index=idx)), (ge, dict(scale=m, mod_index=idx[:3])),
        (ge, dict(scale=m, mod_index=idx.long())), (ae, dict(mod_index=idx)), (ge, dict(weight=v[:32])),
        (ge, dict(weight=v.half())), (ge, dict(branch=b, weight=v, post="rms", post_weight=v.bfloat16())),
        (ge, dict(y_out=x.float())), (ge, dict(h_out=x[:3], branch=b)), (ae, dict(h_out=x)),
        (ae, dict(branch=b, h_out=x, y_out=x)), (ae, dict(eps=-1.0)), (ae, dict(eps=math.nan)), (ae, dict(eps=1e60)),
        (ae, dict(x=x.float().requires_grad_())), (ae, dict(weight=v.cpu())),
    ]:
        a = dict(x=x)
        a.update(kw)
        with pytest.raises(err):
            nkv.residual_norm(**a)
    y = torch.zeros((5, 64), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ae, match="overlaps"):
        nkv.residual_norm(y[:4], y_out=y[1:])
    assert nkv.residual_norm(x[:0])[1].shape == (0, 64)
