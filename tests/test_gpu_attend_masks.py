"""Packed attention: values behind a mask, and probabilities far below a row's maximum.

A masked key's probability is 0, so whatever stands in its value row leaves the
rows that do not see it as they are, bit for bit.  In f16 a probability below
the type's normal range has an absolute error; the kernel holds them scaled so
that the error is at most 2^-32 of the row's largest one (half of the smallest
subnormal 2^-24, times 2^-7).
"""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("q_len,k_len,block,cut", [
    (200, 200, 1, 64),        # rows 0..63 do not see keys 64..
    (200, 200, 64, 64),       # the same by blocks
    (300, 300, 100, 200),     # both halves of an item
    (40, 9000, 1, 8961),      # split keys; the first row sees 8,961
    (50, 20, 1, 1),           # rows that see nothing at all
])
def test_large_finite_values_of_masked_keys_have_no_effect(nkv, q_len, k_len, block, cut, D, dtype):
    import torch
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn((n, 2, D), generator=g, device="cuda").to(dt) for n in (q_len, k_len, k_len))
    plan = nkv.AttendPlan([q_len], 2, head_dim=D, k_lens=[k_len], block=block)
    assert bool(plan.split_units) == (k_len == 9000)
    first = q_len - k_len  # row of the first key
    # rows whose limit is at most `cut`
    blind = [i for i in range(q_len) if i - first < 0 or ((i - first) // block + 1) * block <= cut]
    assert blind
    v[cut:] = 0.0
    out, lse = nkv.attend_packed(plan, q, k, v)
    for value in (torch.finfo(dt).max, torch.finfo(dt).min):
        v[cut:] = value
        got, got_lse = nkv.attend_packed(plan, q, k, v)
        assert torch.equal(got[blind], out[blind]) and torch.equal(got_lse, lse)
    plan.check()


def test_f16_keeps_the_mass_of_many_small_probabilities(nkv):
    """One key, and 131,072 that are 17.4 nats lower: 0.36 % of the mass in probabilities of 2^-25.1 each.
    Tolerance: n 2^-32 for P, n 2^-24 of the sum's magnitude, the output's half step twice over."""
    import torch
    n, rows = 131072, 148 * 256
    q = torch.zeros((rows, 1, 64), dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1.0
    k = torch.zeros((n + 1, 1, 64), dtype=torch.float16, device="cuda")
    k[1:, :, 0] = -17.40625
    v = torch.ones((n + 1, 1, 64), dtype=torch.float16, device="cuda")
    v[0] = 0.0
    plan = nkv.AttendPlan([rows], 1, head_dim=64, k_lens=[n + 1], causal=False)
    assert plan.split_units == 0  # one running maximum over all the keys
    out, lse = nkv.attend_packed(plan, q, k, v, scale=1.0, out=torch.empty(q.shape, device="cuda"))
    plan.check()
    mass = n * math.exp(-17.40625)
    want = mass / (1.0 + mass)
    tol = n * 2.0 ** -32 + n * 2.0 ** -24 * want + 2.0 ** -10 * want
    assert float((out.double() - want).abs().max()) <= tol
    # the running sum lies between 1 and 2 (times 2^7) and takes n / 64 steps' sums, each addition off by at most half
    # an ulp of it, 2^-24: 2^11 additions, 2^-13 in all (the sum of a step is 2^-19.1, 2^5 such half ulps)
    assert float((lse.double() - math.log1p(mass)).abs().max()) <= n / 64 * 2.0 ** -24 + 2.0 ** -20


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("k_len", [640, 20000])
def test_scores_that_rise_more_slowly_than_the_maximum_follows(nkv, dtype, k_len):
    """The running maximum may lag by 8 (base 2): the largest probabilities there are, with the largest values."""
    import torch
    from test_gpu_attend_packed import _check
    dt = getattr(torch, dtype)
    q = torch.zeros((3, 1, 64), dtype=dt, device="cuda")
    q[:, :, 0] = 1.0
    k = torch.zeros((k_len, 1, 64), dtype=dt, device="cuda")
    k[:, 0, 0] = -4.0
    k[64:, 0, 0] = 1.375   # 7.75 in base 2 above the first step's
    k[300:, 0, 0] = 6.5    # then it moves, and lags again
    v = torch.randn((k_len, 1, 64), device="cuda").clamp(-2, 2).to(dt)
    if dt == torch.float16:
        v *= 30000.0
    plan = nkv.AttendPlan([3], 1, head_dim=64, k_lens=[k_len], causal=False)
    out, lse = nkv.attend_packed(plan, q, k, v, scale=1.0)
    plan.check()
    assert bool(out.isfinite().all())
    _check(q, k, v, [3], [k_len], out, lse, causal=False, scale=1.0)
