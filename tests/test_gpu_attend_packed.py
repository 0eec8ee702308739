"""Packed attention (nkv_attend_packed) against float64 attention.

Tolerances, before any run.  With u the half step of the output's type, u_p
that of P's (the inputs' type) and A = sum_j p_j |v_j| per output:
 * scores are f32 sums of D exact products: |ds| <= E_s = (D + 8) 2^-23 scale
   max_j sum_d |q_d k_jd|, plus 2^-21 for ex2 and the scaling; a relative error
   of p of that size moves o by at most 2 E_s A;
 * P is rounded to the inputs' type: u_p A; below f16's normal range by at most
   2^-25 of a row whose sum is at least 2^-8: n 2^-17 2^-8 max|v|;
 * the rounding of the output: u |o|.  f32 sums of n terms: n 2^-24 A.
 * lse: E_s + 2^-21 + 2^-22 |lse|.
"""
import math

import pytest

pytestmark = pytest.mark.gpu


def _limits(ql, kl, causal, block):
    import torch
    if not causal:
        return torch.full((ql,), kl)
    p = torch.arange(ql) + kl - ql
    lim = (torch.div(p, block, rounding_mode="floor") + 1) * block
    return torch.where(p < 0, torch.zeros_like(p), lim.clamp(max=kl))


def _reference(q, k, v, q_lens, k_lens, causal, block, scale, history=None):
    """o, A, lse, E_s of the definition in f64; masked keys are left out, not multiplied by 0."""
    import torch
    H, KV, D = q.shape[1], k.shape[1], q.shape[2]
    qd, kd, vd = q.double(), k.double(), v.double()
    o = torch.zeros((sum(q_lens), H, D), dtype=torch.float64, device=q.device)
    A, lse, E = torch.zeros_like(o), torch.full((H, o.shape[0]), -math.inf, dtype=torch.float64, device=q.device), 0.0
    q0 = k0 = 0
    for ql, kl in zip(q_lens, k_lens):
        if ql and kl:
            lim = _limits(ql, kl, causal, block).to(q.device)
            hidden = torch.arange(kl, device=q.device)[None, :] >= lim[:, None]
            for h in range(H):
                kk, vv = kd[k0:k0 + kl, h * KV // H], vd[k0:k0 + kl, h * KV // H]
                qq = qd[q0:q0 + ql, h]
                s = (qq @ kk.t()) * scale
                s = torch.where(hidden, torch.full_like(s, -math.inf), s)
                fin = torch.where(kk.isfinite(), kk, torch.zeros_like(kk))
                E = max(E, float((qq.abs() @ fin.abs().t()).max()) * scale)
                z = torch.logsumexp(s, dim=1)
                p = torch.exp(s - torch.where(z == -math.inf, torch.zeros_like(z), z)[:, None])
                p = torch.where(hidden, torch.zeros_like(p), p)
                ok = vv.isfinite()
                v0 = torch.where(ok, vv, torch.zeros_like(vv))
                r = p @ v0
                if not bool(ok.all()):
                    for j in torch.nonzero(~ok.all(dim=1)).flatten().tolist():
                        add = torch.where(ok[j], torch.zeros_like(vv[j]), vv[j])
                        seen = (~hidden[:, j])[:, None]
                        r = torch.where(seen, r + add[None, :], r)
                o[q0:q0 + ql, h], A[q0:q0 + ql, h], lse[h, q0:q0 + ql] = r, p @ v0.abs(), z
        q0, k0 = q0 + ql, k0 + kl
    if history is not None:
        ho, hl = history[0].double()[:o.shape[0]], history[1].double()[:, :o.shape[0]]
        z = torch.logaddexp(lse, hl)
        zz = torch.where(z == -math.inf, torch.zeros_like(z), z)
        a, b = torch.exp(lse - zz).t()[..., None], torch.exp(hl - zz).t()[..., None]
        o = torch.where(a > 0, o * a, torch.zeros_like(o)) + torch.where(b > 0, ho * b, torch.zeros_like(o))
        A, lse = A * a + torch.where(b > 0, ho * b, torch.zeros_like(o)).abs(), z
    return o, A, lse, E


def _check(q, k, v, q_lens, k_lens, out, lse, causal=True, block=1, scale=None, history=None):
    import torch
    n, D = sum(q_lens), q.shape[2]
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    o, A, z, E = _reference(q, k, v, q_lens, k_lens, causal, block, scale, history)
    up, u = torch.finfo(q.dtype).eps / 2, torch.finfo(out.dtype).eps / 2
    Es = (D + 8) * 2.0 ** -23 * E + 2.0 ** -21
    longest = max(list(k_lens) + [1])
    tol = u * o.abs() + (up + 2 * Es + longest * 2.0 ** -24) * A + 1e-30
    if q.dtype == torch.float16:
        vmax = float(torch.where(v.isfinite(), v, torch.zeros_like(v)).abs().max()) if v.numel() else 0.0
        tol = tol + longest * 2.0 ** -25 * vmax + 2.0 ** -24 * (out.dtype == torch.float16)
    got, gl = out[:n].double(), lse[:, :n].double()
    fin = o.isfinite()
    assert torch.equal(got.isnan(), o.isnan()) and torch.equal(got[o.isinf()], o[o.isinf()]), "non-finite outputs differ"
    bad = (got[fin] - o[fin]).abs() > tol[fin]
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} outputs outside, worst " \
                                f"{float(((got[fin] - o[fin]).abs() / tol[fin]).max())} of the tolerance"
    empty = z == -math.inf
    assert torch.equal(gl == -math.inf, empty)
    ok = z.isfinite()
    assert bool(((gl[ok] - z[ok]).abs() <= Es + 2.0 ** -21 + 2.0 ** -22 * z[ok].abs()).all()), \
        f"lse off by {float((gl[ok] - z[ok]).abs().max())}, allowed {Es}"


def _inputs(q_lens, k_lens, H, KV, D, dtype, seed=0, qs=1.0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    return ((qs * r(sum(q_lens), H, D)).to(dtype), r(sum(k_lens), KV, D).to(dtype), r(sum(k_lens), KV, D).to(dtype))


CASES = [
    # q_lens, k_lens, H, KV, D, causal, block
    ([1], [1], 1, 1, 128, True, 1),
    ([1], [2], 2, 2, 64, True, 1),
    ([3], [3], 2, 1, 128, True, 1),
    ([127], [127], 2, 2, 128, True, 1),
    ([128], [128], 2, 2, 128, True, 1),
    ([129], [129], 2, 2, 128, True, 1),
    ([255, 256, 257], [255, 256, 257], 2, 2, 128, True, 1),
    ([300], [300], 3, 3, 128, False, 1),
    ([1, 0, 40, 2], [700, 5, 40, 0], 4, 2, 128, True, 1),       # idle, keyless
    ([50], [20], 2, 2, 128, True, 1),                            # 30 rows see nothing
    ([600], [130], 1, 1, 128, True, 1),                          # a whole item sees nothing
    ([200, 64], [331, 1000], 6, 2, 128, True, 1),                # groups of 3, chunks over a cache
    ([33], [33], 40, 8, 128, True, 1),                           # groups of 5
    ([100], [100], 8, 1, 128, True, 1),                          # one key/value head
    ([700], [700], 2, 2, 128, True, 100),                        # blocks
    ([700], [1100], 2, 2, 128, True, 333),
    ([1500], [1500], 1, 1, 128, True, 640),                      # a block of several tiles inside one item
    ([5, 260], [5, 260], 2, 2, 8, True, 1),
    ([5, 260], [5, 260], 2, 2, 40, True, 1),
    ([5, 260], [5, 260], 2, 2, 64, True, 1),
    ([5, 260], [5, 260], 2, 2, 72, True, 1),
    ([5, 260], [5, 260], 2, 2, 104, True, 1),
    ([1], [20000], 4, 2, 128, True, 1),                          # split keys
    ([1], [20001], 8, 1, 64, True, 1),
    ([7], [9000], 2, 2, 96, False, 1),
    ([2, 1, 300], [5000, 33, 12000], 4, 4, 128, True, 1),
    ([2100], [2100], 2, 2, 64, True, 1),
    ([0, 0], [0, 3], 2, 2, 64, True, 1),
    ([9], [300], 128, 1, 64, True, 1),                           # the largest group
    ([9], [300], 127, 1, 64, True, 1),                           # one token per half of an item
    ([70], [70], 48, 2, 128, True, 1),                           # groups of 24: 120 of 128 rows
    ([1] * 40, list(range(0, 400, 10)), 4, 2, 128, True, 1),     # many single tokens
    ([1, 2, 3] * 20, [500] * 60, 3, 3, 48, False, 1),            # several items of one half on a CTA
    ([1] * 400, [3] * 400, 2, 2, 64, True, 1),
    ([1] * 300, [0, 5, 0, 0, 200, 0] * 50, 4, 4, 128, True, 1),  # and items without keys among them
    ([130, 1, 0, 2] * 60, [130, 0, 4, 70] * 60, 3, 3, 64, True, 1),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "q{}_k{}_{}x{}x{}_{}{}".format(
    "-".join(map(str, c[0])), "-".join(map(str, c[1])), c[2], c[3], c[4], "c" if c[5] else "f", c[6]))
def test_matches_float64(nkv, case, dtype):
    import torch
    ql, kl, H, KV, D, causal, block = case
    q, k, v = _inputs(ql, kl, H, KV, D, getattr(torch, dtype))
    plan = nkv.AttendPlan(ql, H, kv_heads=KV, head_dim=D, k_lens=kl, causal=causal, block=block, device="cuda")
    out, lse = nkv.attend_packed(plan, q, k, v)
    plan.check()
    assert out.dtype == q.dtype and out.shape == q.shape and lse.shape == (H, q.shape[0])
    _check(q, k, v, ql, kl, out, lse, causal, block)


@pytest.mark.parametrize("seed", range(24))
def test_random_geometry(nkv, seed):
    """Lengths, groups, widths, masks, history and layouts drawn together."""
    import random

    import torch
    rng = random.Random(seed)
    n = rng.choice([1, 1, 2, 4, 7])
    pick = lambda hi: max(0, int(math.exp(rng.uniform(0, math.log(hi)))) - rng.choice([0, 0, 1]))  # noqa: E731
    ql = [pick(rng.choice([3, 60, 900])) for _ in range(n)]
    kl = [q if rng.random() < 0.4 else max(0, q + rng.choice([-5, 1, 64, 1000, 7000])) for q in ql]
    KV = rng.choice([1, 2, 3, 5])
    H = KV * rng.choice([1, 2, 3, 6, 8])
    D = rng.choice([64, 128, 8 * rng.randint(1, 16)])
    causal, block = rng.random() < 0.8, rng.choice([1, 1, 30, 400])
    dt = rng.choice([torch.bfloat16, torch.float16])
    q, k, v = _inputs(ql, kl, H, KV, D, dt, seed=seed, qs=rng.choice([0.5, 1.0, 4.0]))
    if rng.random() < 0.5:  # one projection's views
        kv = torch.cat((k, v), dim=1)
        k, v = kv[:, :KV], kv[:, KV:]
    history = None
    if rng.random() < 0.4:
        g = torch.Generator(device="cuda").manual_seed(seed)
        history = (torch.randn(q.shape, generator=g, device="cuda"),
                   6 * torch.rand((H, q.shape[0]), generator=g, device="cuda"))
    plan = nkv.AttendPlan(ql, H, kv_heads=KV, head_dim=D, k_lens=kl, causal=causal, block=block)
    out = torch.empty(q.shape, dtype=torch.float32, device="cuda") if rng.random() < 0.3 else None
    out, lse = nkv.attend_packed(plan, q, k, v, history=history, out=out)
    plan.check()
    _check(q, k, v, ql, kl, out, lse, causal, block, history=history)


@pytest.mark.parametrize("k_len", [70, 9000])
def test_nan_rows_stay_nan_in_the_merge(nkv, k_len):
    """A NaN of either part is not taken for "nothing seen" when the other part saw nothing."""
    import torch
    q, k, v = _inputs([70], [k_len], 1, 1, 64, torch.bfloat16)
    q[3] = math.nan
    ho, hl = torch.randn((70, 1, 64), device="cuda"), torch.full((1, 70), -math.inf, device="cuda")
    hl[0, 5] = math.nan
    plan = nkv.AttendPlan([70], 1, head_dim=64, k_lens=[k_len])
    out, lse = nkv.attend_packed(plan, q, k, v, history=(ho, hl))
    bad = torch.zeros(70, dtype=torch.bool, device="cuda")
    bad[3] = bad[5] = True
    assert torch.equal(out.isnan().all(-1)[:, 0], bad) and torch.equal(out.isnan().any(-1)[:, 0], bad)
    assert torch.equal(lse.isnan()[0], bad)
    none = nkv.AttendPlan([70], 1, head_dim=64, k_lens=[0])
    out, lse = nkv.attend_packed(none, q, k, v, history=(ho, hl))
    bad[3] = False
    assert torch.equal(out.isnan().all(-1)[:, 0], bad) and torch.equal(lse.isnan()[0], bad)
    assert bool((lse[0, ~bad] == -math.inf).all()) and bool((out[~bad] == 0).all())


def test_offsets_past_32_bits(nkv):
    """Keys, values and queries as columns of buffers whose rows lie half a megabyte apart."""
    import torch
    T, W = 9000, 1 << 18
    q, k, v = _inputs([T], [T], 1, 1, 64, torch.bfloat16, seed=11)
    buf = torch.empty((T, 1, W), dtype=torch.bfloat16, device="cuda")  # 4.7 GB
    wide = [buf[..., c:c + 64] for c in (0, W // 2, W - 64)]
    for w, t in zip(wide, (q, k, v)):
        w.copy_(t)
    last = slice(T - 300, T)
    plan = nkv.AttendPlan([T], 1, head_dim=64)
    out, lse = nkv.attend_packed(plan, *wide)
    near, near_lse = nkv.attend_packed(plan, q, k, v)
    assert torch.equal(out, near) and torch.equal(lse, near_lse)
    _check(q[last], k, v, [300], [T], out[last], lse[:, last])
    del buf


def test_f32_output_and_scale(nkv):
    import torch
    ql, kl = [130, 9], [130, 4000]
    q, k, v = _inputs(ql, kl, 4, 2, 128, torch.bfloat16, seed=1, qs=3.0)
    plan = nkv.AttendPlan(ql, 4, kv_heads=2, k_lens=kl)
    out = torch.empty(q.shape, dtype=torch.float32, device="cuda")
    o, lse = nkv.attend_packed(plan, q, k, v, scale=0.25, out=out)  # sharp rows: the running maximum moves
    assert o is out
    _check(q, k, v, ql, kl, out, lse, scale=0.25)


@pytest.mark.parametrize("out_dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("q_len,k_len", [(300, 300), (3, 9000), (50, 20), (4, 0)])
def test_history_merge(nkv, q_len, k_len, out_dtype):
    """Whole and split rows, rows that see nothing here, rows without a history (lse -inf, its o then unused)."""
    import torch
    q, k, v = _inputs([q_len], [k_len], 2, 2, 128, torch.bfloat16, seed=2)
    g = torch.Generator(device="cuda").manual_seed(9)
    ho = torch.randn((q_len, 2, 128), generator=g, device="cuda")
    hl = 5.0 + 3.0 * torch.randn((2, q_len), generator=g, device="cuda")
    hl[0, ::3] = -math.inf
    ho[::3, 0] = math.nan
    hl[1, 1::7] = 200.0   # the history outweighs everything
    hl[1, 2::7] = -200.0
    out = torch.empty((q_len, 2, 128), dtype=getattr(torch, out_dtype), device="cuda")
    plan = nkv.AttendPlan([q_len], 2, k_lens=[k_len])
    out, lse = nkv.attend_packed(plan, q, k, v, history=(ho, hl), out=out)
    clean = torch.where(ho.isnan(), torch.zeros_like(ho), ho)
    _check(q, k, v, [q_len], [k_len], out, lse, history=(clean, hl))


@pytest.mark.parametrize("layout", ["fused", "head_major", "every_other", "wide"])
@pytest.mark.parametrize("k_len", [257, 6000])
def test_strided_inputs(nkv, layout, k_len):
    import torch
    ql, H, KV, D = [k_len if k_len < 1000 else 3], 4, 2, 64
    q, k, v = _inputs(ql, [k_len], H, KV, D, torch.bfloat16, seed=3)
    if layout == "fused":  # k and v beside each other in one projection, q in a wider one
        kv = torch.cat((k, v), dim=1)
        qs, ks, vs = torch.cat((q, q.neg()), dim=1)[:, :H], kv[:, :KV], kv[:, KV:]
    elif layout == "head_major":
        qs, ks, vs = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v))
    elif layout == "every_other":
        qs, ks, vs = (torch.stack((t, t + 1), dim=1).flatten(0, 1)[::2] for t in (q, k, v))
    else:
        qs, ks, vs = (torch.cat((t, t + 1), dim=2)[..., :D] for t in (q, k, v))
    assert not (qs.is_contiguous() and ks.is_contiguous())
    plan = nkv.AttendPlan(ql, H, kv_heads=KV, head_dim=D, k_lens=[k_len])
    out, lse = nkv.attend_packed(plan, qs, ks, vs)
    _check(q, k, v, ql, [k_len], out, lse)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_nonfinite_values_of_masked_keys_have_no_effect(nkv, dtype):
    """Infinities and NaN in keys and values that a row does not see, behind a sequence and behind the last one; a row
    that does see one gets it."""
    import torch
    ql = kl = [70, 200, 5]
    q, k, v = _inputs([70, 200, 5], [70, 200, 50], 2, 2, 128, getattr(torch, dtype), seed=4)
    k[275:], v[275:] = math.nan, math.inf              # behind the last sequence
    v[70 + 150, 0, 3] = math.nan                       # seen by rows 150.. of the second sequence
    v[70 + 160, 1, 7] = math.inf
    v[70 + 170, 1, 7] = -math.inf                      # with the one above: NaN
    k[70 + 199, 1] = math.nan                          # seen by the last row only
    plan = nkv.AttendPlan(ql, 2)
    out, lse = nkv.attend_packed(plan, q, k, v)
    assert bool(out[:70].isfinite().all()) and bool(out[70:220].isfinite().all()) and bool(out[270:].isfinite().all())
    assert bool(out[220:269, 0, 3].isnan().all()) and bool(out[220:269, 0, :3].isfinite().all())
    assert bool((out[230:240, 1, 7] == math.inf).all()) and bool(out[240:269, 1, 7].isnan().all())
    assert bool(out[269, 1].isnan().all()) and bool(lse[1, 269].isnan()) and bool(lse[1, 268].isfinite())
    # everything else as without them
    kc, vc = k.clone(), v.clone()
    vc[~vc.isfinite()] = 0.0
    kc[~kc.isfinite()] = 0.0
    ref, rl = nkv.attend_packed(plan, q, kc, vc)
    same = out.isfinite()
    same[269, 1] = False
    # a NaN's key row changed for that one row and head; the rest must be bit-equal
    assert torch.equal(out[same], ref[same])
    assert torch.equal(lse[:, :269], rl[:, :269])


def test_nonfinite_values_in_split_keys(nkv):
    import torch
    q, k, v = _inputs([4], [9000], 2, 2, 64, torch.bfloat16, seed=5)
    v[8998, 0, 5] = math.inf      # seen by the last two tokens
    v[8999, 1, 6] = math.nan      # by the last
    plan = nkv.AttendPlan([4], 2, head_dim=64, k_lens=[9000])
    assert plan.split_units
    out, lse = nkv.attend_packed(plan, q, k, v)
    _check(q, k, v, [4], [9000], out, lse)


def test_infinite_scores(nkv):
    """A key of -inf scores is never chosen; a row with nothing else is empty."""
    import torch
    q = torch.ones((4, 1, 64), dtype=torch.bfloat16, device="cuda")
    k = torch.randn((4, 1, 64), device="cuda").to(torch.bfloat16)
    v = torch.randn((4, 1, 64), device="cuda").to(torch.bfloat16)
    k[0] = -math.inf
    plan = nkv.AttendPlan([4], 1, head_dim=64)
    out, lse = nkv.attend_packed(plan, q, k, v)
    assert bool((out[0] == 0).all()) and lse[0, 0].item() == -math.inf
    kk, vv = k[1:].double()[:, 0], v[1:].double()[:, 0]
    for i in range(1, 4):
        s = (kk[:i] @ q[0, 0].double()) / 8
        ref = torch.softmax(s, 0) @ vv[:i]
        assert float((out[i, 0].double() - ref).abs().max()) <= 2.0 ** -7 * float(vv.abs().max())


def test_rows_behind_the_last_sequence_stay(nkv):
    import torch
    ql, kl = [5, 60], [9, 400]
    q, k, v = _inputs([5, 60, 17], [9, 400, 30], 4, 2, 128, torch.bfloat16, seed=6)
    plan = nkv.AttendPlan(ql, 4, kv_heads=2, k_lens=kl)
    out = torch.full(q.shape, 7.0, dtype=q.dtype, device="cuda")
    lse = torch.full((4, 82), 9.0, device="cuda")
    ho, hl = torch.randn((82, 4, 128), device="cuda"), torch.randn((4, 82), device="cuda")
    nkv.attend_packed(plan, q, k, v, history=(ho, hl), out=out, lse=lse)
    assert bool((out[65:] == 7).all()) and bool((lse[:, 65:] == 9).all())
    _check(q[:65], k, v, ql, kl, out, lse, history=(ho, hl))
    out, lse = nkv.attend_packed(plan, q, k, v)
    assert bool((out[65:] == 0).all()) and bool((lse[:, 65:] == -math.inf).all())


@pytest.mark.parametrize("q_len,k_len", [(500, 500), (3, 12000)])
def test_graph_capture_and_replay(nkv, q_len, k_len):
    """Two graphs and eager calls of one plan: each has a workspace of its own; repeated runs are bit-equal."""
    import torch
    plan = nkv.AttendPlan([q_len], 4, kv_heads=2, k_lens=[k_len])
    sets = [_inputs([q_len], [k_len], 4, 2, 128, torch.bfloat16, seed=s) for s in (7, 8, 9)]
    want = [nkv.attend_packed(plan, *s) for s in sets]
    bufs, graphs, outs = [], [], []
    for i in range(2):
        buf = [t.clone() for t in sets[i]]
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            outs.append(nkv.attend_packed(plan, *buf))
        bufs.append(buf)
        graphs.append(g)
    for a, b in ((0, 1), (2, 0), (1, 2)):
        for buf, s in zip(bufs, (sets[a], sets[b])):
            for t, x in zip(buf, s):
                t.copy_(x)
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for st, g in zip(streams, graphs):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for (o, l), w in zip(outs, (want[a], want[b])):
            assert torch.equal(o, w[0]) and torch.equal(l, w[1])
    plan.check()
    for g in graphs:
        g.reset()


def test_other_stream_and_concurrent_calls(nkv):
    import torch
    plan = nkv.AttendPlan([2, 40], 4, kv_heads=4, k_lens=[15000, 4000])
    sets = [_inputs([2, 40], [15000, 4000], 4, 4, 128, torch.bfloat16, seed=s) for s in (1, 2)]
    want = [nkv.attend_packed(plan, *s) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for st, s in zip(streams, sets):
            got.append(nkv.attend_packed(plan, *s, stream=st))
    torch.cuda.synchronize()
    for i, (o, l) in enumerate(got):
        assert torch.equal(o, want[i % 2][0]) and torch.equal(l, want[i % 2][1])


def test_refusals(nkv):
    import torch
    plan = nkv.AttendPlan([4], 4, kv_heads=2, head_dim=64, k_lens=[8])
    q, k, v = _inputs([4], [8], 4, 2, 64, torch.bfloat16)
    ok = nkv.attend_packed(plan, q, k, v)
    ge, ae = nkv.GeometryError, nkv.ArgumentError
    bad = [
        (ge, dict(q=q[:3])), (ge, dict(q=q[:, :2])), (ge, dict(q=q.float())), (ge, dict(k=k[:7])),
        (ge, dict(k=k.half())), (ge, dict(v=v[:, :1])), (ge, dict(q=q.transpose(1, 2).contiguous().transpose(1, 2))),
        (ae, dict(scale=0.0)), (ae, dict(scale=-1.0)), (ae, dict(scale=1e60)), (ae, dict(scale=1e-60)), (ae, dict(scale=3e38)), (ae, dict(scale=math.inf)), (ae, dict(scale=math.nan)),
        (ae, dict(q=q.clone().requires_grad_())), (ae, dict(k=k.cpu())),
        (ge, dict(out=torch.empty((4, 4, 64), dtype=torch.float16, device="cuda"))),
        (ge, dict(out=torch.empty((3, 4, 64), dtype=torch.bfloat16, device="cuda"))),
        (ge, dict(lse=torch.empty((4, 5), device="cuda"))), (ae, dict(out=q)),
        (ge, dict(history=(torch.zeros((4, 4, 64), device="cuda"), torch.zeros((4, 3), device="cuda")))),
        (ge, dict(history=(torch.zeros((4, 4, 64), device="cuda").bfloat16(), torch.zeros((4, 4), device="cuda")))),
        (ae, dict(k=k[:, :1].expand(8, 2, 64))),
        (ae, dict(k=torch.zeros(8 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(8, 2, 64))),
        (ae, dict(v=torch.zeros((8, 2, 68), dtype=torch.bfloat16, device="cuda")[..., :64])),
    ]
    for err, change in bad:
        kw = dict(q=q, k=k, v=v)
        kw.update(change)
        with pytest.raises(err):
            nkv.attend_packed(plan, **kw)
    torch.cuda.synchronize()
    again = nkv.attend_packed(plan, q, k, v)
    assert torch.equal(ok[0], again[0])
    plan.close()
    with pytest.raises(ae, match="closed"):
        nkv.attend_packed(plan, q, k, v)
