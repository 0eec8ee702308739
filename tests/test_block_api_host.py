"""CPU checks of the block operators' entry points."""
import contextlib
import os
import subprocess
import sys
from types import SimpleNamespace

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hy-nomas-rs_b200")


def test_plan_set_status_refuses_a_null_plan(nkv):
    assert nkv.lib().nkv_attend_plan_set_status(None, 0) == 6


def test_import_star_needs_no_torch():
    """The cache API alone: torch and the compiled binding are needed by the block operators, at their first use."""
    code = ("import sys; sys.modules['torch'] = None; sys.path.insert(0, sys.argv[1])\n"
            "from nomas_kv import *\n"
            "import nomas_kv\n"
            "assert KvBank is nomas_kv.KvBank and 'AttendPlan' in dir(nomas_kv)\n"
            "try:\n    nomas_kv.AttendPlan\nexcept ImportError: pass\nelse: raise SystemExit('no error')\n")
    subprocess.run([sys.executable, "-c", code, PKG], check=True)


def test_import_star_brings_the_block_operators_with_torch(nkv):
    code = ("import sys; sys.path.insert(0, sys.argv[1])\n"
            "from nomas_kv import *\n"
            "import nomas_kv\n"
            "assert AttendPlan is nomas_kv.AttendPlan and attend_packed and KvBank\n")
    subprocess.run([sys.executable, "-c", code, PKG], check=True)


def test_block_names_are_reached_through_the_package(nkv):
    for name in ("RotaryAxes", "rope_tables", "rotary", "residual_norm", "AttendPlan", "attend_packed"):
        assert getattr(nkv, name) is getattr(nkv.block, name) and name in dir(nkv)


@pytest.mark.parametrize("call", ["attend_history", "attend"])
def test_history_attention_refuses_tensors_elsewhere(nkv, monkeypatch, call):
    """An address of another device (or the host's) must not reach a kernel."""
    import torch
    reached = []

    class Lib:
        def __getattr__(self, name):
            def f(*a):
                reached.append(name)
                return 0
            return f

    monkeypatch.setattr(nkv, "lib", Lib)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda d=None: stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(nkv.LayerCache, "valid_len", lambda self: 4)
    stream = SimpleNamespace(device=torch.device("cuda", 0))
    layer = nkv.LayerCache(SimpleNamespace(heads=2, head_dim=128, stream=stream, _h=None), 0)
    q = torch.zeros((4, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(nkv.ArgumentError, match="cuda:0"):
        if call == "attend":
            layer.attend(SimpleNamespace(heads=2, head_dim=128), q, q, q)
        else:
            layer.attend_history(q)
    assert "nkv_bank_attend_history" not in reached


@pytest.mark.parametrize("change", [dict(q_lens=[2 ** 64 + 1]), dict(k_lens=[2 ** 64 + 5]), dict(block=2 ** 64 + 1),
                                    dict(heads=2 ** 32 + 4), dict(kv_heads=2 ** 32 + 4), dict(head_dim=2 ** 32 + 64),
                                    dict(heads=-2 ** 32 + 4)])
def test_plan_refuses_numbers_that_do_not_fit(nkv, monkeypatch, change):
    """2^64 + 1 must not be taken for 1: such a plan would be another one than was asked for."""
    made = []

    class Lib:
        def nkv_attend_plan_create(self, *a):
            made.append(a)
            raise nkv.CudaError("reached")

    from nomas_kv import block
    monkeypatch.setattr(block, "lib", Lib)
    with pytest.raises(nkv.CudaError, match="reached"):  # what fits gets there
        nkv.AttendPlan([1], 4, kv_heads=4, head_dim=64, k_lens=[5], device="cuda:0")
    made.clear()
    args = dict(dict(q_lens=[1], heads=4, kv_heads=4, head_dim=64, k_lens=[5], device="cuda:0"), **change)
    with pytest.raises((nkv.GeometryError, nkv.ArgumentError)):
        nkv.AttendPlan(args.pop("q_lens"), args.pop("heads"), **args)
    assert not made
