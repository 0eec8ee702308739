"""Packed attention: values behind a mask.  A masked key's probability is 0, so
whatever stands in its value row leaves the rows that do not see it as they
are, bit for bit.
"""
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
