"""A plan whose status word is set (a bounded wait of one of its calls ran out)
gives NaN, so that stale memory does not pass for a result, until the failure
has been reported.  The word is set by the host here: no wait runs out."""
import math

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_dtype", ["same", "float32"])
@pytest.mark.parametrize("history", [False, True])
@pytest.mark.parametrize("q_lens,k_lens", [([70, 0, 300], [70, 4, 300]), ([3], [9000]), ([5, 600], [0, 9]),
                                           ([1] * 200, [300] * 200)])
def test_a_failed_plan_gives_nan_until_it_is_reported(nkv, q_lens, k_lens, history, out_dtype):
    import torch
    n, extra, H = sum(q_lens), 3, 6
    q = torch.randn((n + extra, H, 64), device="cuda").bfloat16()
    k, v = (torch.randn((sum(k_lens) + 1, 2, 64), device="cuda").bfloat16() for _ in range(2))
    hist = (torch.randn(q.shape, device="cuda"), torch.randn((H, n + extra), device="cuda")) if history else None
    plan = nkv.AttendPlan(q_lens, H, kv_heads=2, head_dim=64, k_lens=k_lens)
    assert bool(plan.split_units) == (k_lens == [9000])

    def call():
        out = torch.full(q.shape, 5.0, dtype=q.dtype if out_dtype == "same" else torch.float32, device="cuda")
        lse = torch.full((H, n + extra), 5.0, device="cuda")
        return nkv.attend_packed(plan, q, k, v, history=hist, out=out, lse=lse)

    want, want_lse = call()
    plan.check()
    nkv._check(nkv.lib().nkv_attend_plan_set_status(plan._h, 1))
    for _ in range(2):
        out, lse = call()
        assert bool(out[:n].isnan().all()) and bool(lse[:, :n].isnan().all())
        assert bool((out[n:] == 5).all()) and bool((lse[:, n:] == 5).all())
    with pytest.raises(nkv.CudaError, match="bounded wait"):
        plan.check()
    plan.check()  # reported: the plan works again
    out, lse = call()
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert math.isfinite(float(out[:n].float().sum()))
