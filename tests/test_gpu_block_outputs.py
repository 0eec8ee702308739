"""Outputs that a caller gives to the block operators, and values that they pass through."""
import pytest

pytestmark = pytest.mark.gpu


def _calls(nkv, stream):
    """(name, tensors that the call writes, call); fresh tensors each time."""
    import torch
    pos = torch.randint(0, 50, (6, 2), dtype=torch.int32, device="cuda")
    axes = nkv.RotaryAxes((32, 32))
    q, k = torch.randn((6, 3, 64), device="cuda"), torch.randn((6, 2, 64), device="cuda")
    yield "rotary", (q, k), lambda: nkv.rotary(pos, axes, q, k=k, q_out=q, k_out=k, stream=stream)
    cos, sin = torch.empty((6, 32), device="cuda"), torch.empty((6, 32), device="cuda")
    yield "tables", (cos, sin), lambda: nkv.rope_tables(pos, axes, cos=cos, sin=sin, stream=stream)
    x, b = torch.randn((6, 40), device="cuda"), torch.randn((6, 40), device="cuda")
    yield "norm", (x, b), lambda: nkv.residual_norm(x, b, h_out=x, y_out=b, stream=stream)
    plan = nkv.AttendPlan([6], 3, kv_heads=1, head_dim=64)
    t = torch.randn((6, 5, 64), device="cuda").bfloat16()
    out, lse = torch.empty((6, 3, 64), dtype=torch.bfloat16, device="cuda"), torch.empty((3, 6), device="cuda")
    yield "attend", (out, lse), lambda: nkv.attend_packed(plan, t[:, :3], t[:, 3:4], t[:, 4:], out=out, lse=lse,
                                                          stream=stream)


@pytest.mark.parametrize("path", ["binding", "python"])
def test_given_outputs_count_as_modified(nkv, path):
    """Autograd sees the write: a tensor saved for a backward pass is not silently another one."""
    import torch
    stream = None if path == "binding" else torch.cuda.Stream()
    torch.cuda.synchronize()
    for name, written, call in _calls(nkv, stream):
        before = [t._version for t in written]
        call()
        torch.cuda.synchronize()
        assert all(t._version > n for t, n in zip(written, before)), name
    for name, written, call in _calls(nkv, stream):
        w = [torch.ones_like(t, requires_grad=True) for t in written]
        loss = sum((a * t).sum() for a, t in zip(w, written))
        with torch.no_grad():
            call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


@pytest.mark.parametrize("path", ["binding", "python"])
def test_inference_tensors_are_taken(nkv, path):
    """They have no version to count; made and written in inference mode or out of it."""
    import torch
    stream = None if path == "binding" else torch.cuda.Stream()
    with torch.inference_mode():
        calls = list(_calls(nkv, stream))
        torch.cuda.synchronize()
        for _, _, call in calls:
            call()
        torch.cuda.synchronize()
    for _, written, call in calls:
        assert all(t.is_inference() for t in written)
        call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("layout", ["aligned", "odd"])
def test_values_past_the_rotated_ones_pass_through(nkv, dtype, interleaved, layout):
    """Bit for bit: zeros of either sign, infinities, subnormals."""
    import torch
    dt, T, H, D, R = getattr(torch, dtype), 9, 3, 64, 32
    x = torch.randn((T, H, D + 1), device="cuda").to(dt)
    x = x[..., 1:] if layout == "odd" else x[..., 1:].contiguous()
    x[..., R::4] = 0.0
    x[..., R + 1::4] = -0.0
    x[..., R + 2::8] = float("inf")
    x[..., R + 6::8] = torch.finfo(dt).smallest_normal / 4
    pos = torch.randint(1, 50, (T, 1), dtype=torch.int32, device="cuda")
    out = nkv.rotary(pos, nkv.RotaryAxes((R,), interleaved=interleaved), x)
    whole = {2: torch.int16, 4: torch.int32}[x.element_size()]
    assert torch.equal(out[..., R:].contiguous().view(whole), x[..., R:].contiguous().view(whole))
    assert bool(out[..., :R].isfinite().all())
