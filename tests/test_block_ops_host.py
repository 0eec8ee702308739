"""CPU checks of the attention block's operators: the schedule of packed
attention covers every (row, key tile) exactly once, arguments are refused
before any device call, and the ctypes structs match the header."""
import ctypes as C
import math
import os
import random
import shutil
import subprocess

import pytest


def _schedule(nk, q, k, heads, kv_heads, causal, block, sms):
    n = len(q)
    qa, ka, cnt = (C.c_uint64 * max(n, 1))(*q), (C.c_uint64 * max(n, 1))(*k), C.c_uint64()
    args = (qa, ka, n, heads, kv_heads, causal, block, sms)
    nk._check(nk.lib().nkv_attend_schedule(*args, None, 0, C.byref(cnt)))
    buf = (C.c_int64 * (8 * max(cnt.value, 1)))()
    nk._check(nk.lib().nkv_attend_schedule(*args, buf, cnt.value, C.byref(cnt)))
    return [tuple(buf[8 * i:8 * i + 8]) for i in range(cnt.value)]


def _limit(ql, kl, causal, block, i):
    if not causal:
        return kl
    p = i + kl - ql
    return 0 if p < 0 else min(kl, (p // block + 1) * block)


@pytest.mark.parametrize("seed", range(12))
def test_schedule_covers_every_row_and_tile_once(nkv, seed):
    rng = random.Random(seed)
    n = rng.randint(1, 6)
    q = [rng.choice([0, 1, rng.randint(1, 300), rng.randint(1, 3000)]) for _ in range(n)]
    k = [rng.choice([a, a + rng.randint(0, 20000), rng.randint(0, 500)]) for a in q]
    kv = rng.randint(1, 6)
    group = rng.choice([1, 2, 3, 8])
    causal, block, sms = rng.randint(0, 1), rng.choice([1, 7, 640]), rng.choice([1, 4, 148])
    items = _schedule(nkv, q, k, kv * group, kv, causal, block, sms)
    q0 = k0 = 0
    spans = {}
    parts = []
    for it in items:
        qs, ks, row0, rows, h, lo, hi, part = it
        assert 1 <= rows <= 256 and 0 <= h < kv and 0 <= lo <= hi
        spans.setdefault((qs, ks, h, row0, rows), []).append((lo, hi, part))
        if part >= 0:
            parts.append((part, part + rows))
    # partial rows do not overlap
    parts.sort()
    assert all(a[1] <= b[0] for a, b in zip(parts, parts[1:]))
    for ql, kl in zip(q, k):
        for h in range(kv):
            got = sorted((r0, n_) for (qs, ks, hh, r0, n_) in spans if (qs, ks, hh) == (q0, k0, h))
            if ql == 0:
                assert kl == 0 or not got  # without keys it shares its start with the next sequence
                continue
            assert sum(r for _, r in got) == ql * group
            at = 0
            for r0, rows in got:
                assert r0 == at
                at += rows
                lim = _limit(ql, kl, causal, block, (r0 + rows - 1) // group)
                ranges = sorted(spans[(q0, k0, h, r0, rows)])
                assert ranges[0][0] == 0 and ranges[-1][1] == -(-lim // 128)
                assert all(a[1] == b[0] for a, b in zip(ranges, ranges[1:]))
                assert (len(ranges) > 1) == (ranges[0][2] >= 0)
        q0 += ql
        k0 += kl


def test_schedule_fills_the_gpu_for_one_token(nkv):
    items = _schedule(nkv, [1], [29056], 24, 24, 1, 1, 148)
    assert 120 <= len(items) <= 148  # one round of CTAs, each a key range of its own
    assert max(i[6] - i[5] for i in items) <= 40


@pytest.mark.parametrize("q,k,heads,kv,block,code", [
    ([1], [1], 3, 2, 1, "GeometryError"), ([1], [1], 0, 1, 1, "GeometryError"), ([1], [1], 4, 0, 1, "GeometryError"),
    ([1], [1], 4, -4, 1, "GeometryError"), ([1], [1], 4, 4, 0, "ArgumentError"), ([2 ** 31], [1], 1, 1, 1, "GeometryError"),
    ([2 ** 63], [2 ** 63], 1, 1, 1, "GeometryError"), ([2 ** 30], [1], 4, 1, 1, "GeometryError"),
    ([1, 1], [2 ** 30, 2 ** 30], 1, 1, 1, "GeometryError"), ([1], [1], 4, 4, 2 ** 31, "ArgumentError"),
    ([1], [1], 129, 1, 1, "GeometryError"), ([2 ** 28], [1], 8, 8, 1, "GeometryError"),
    ([1] * 70, [1] * 70, 65535, 65535, 1, "GeometryError"),
])
def test_schedule_and_plan_refuse_bad_geometry(nkv, q, k, heads, kv, block, code):
    with pytest.raises(getattr(nkv, code)):
        _schedule(nkv, q, k, heads, kv, 1, block, 148)
    n = len(q)
    h = C.c_void_p()
    with pytest.raises(getattr(nkv, code)):
        nkv._check(nkv.lib().nkv_attend_plan_create((C.c_uint64 * n)(*q), (C.c_uint64 * n)(*k), n, heads, kv, 128, 1,
                                                    block, 0, C.byref(h)))
    assert not h.value


@pytest.mark.parametrize("head_dim", [0, 4, 12, 136, 256, -8])
def test_plan_refuses_head_dim(nkv, head_dim):
    h = C.c_void_p()
    one = (C.c_uint64 * 1)(1)
    with pytest.raises(nkv.GeometryError, match="head_dim"):
        nkv._check(nkv.lib().nkv_attend_plan_create(one, one, 1, 4, 4, head_dim, 1, 1, 0, C.byref(h)))


def test_plan_python_checks(nkv):
    with pytest.raises(nkv.GeometryError, match="negative"):
        nkv.AttendPlan([-1], 4)
    with pytest.raises(nkv.GeometryError, match="one entry per sequence"):
        nkv.AttendPlan([1, 2], 4, k_lens=[1])
    with pytest.raises(nkv.ArgumentError, match="block"):
        nkv.AttendPlan([1], 4, block=0)
    with pytest.raises(nkv.ArgumentError, match="CUDA device only"):
        nkv.AttendPlan([1], 4, device="cpu")


def test_plan_without_gpu_fails_loudly(nkv):
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(nkv.CudaError, match="no CUDA device"):
        nkv.AttendPlan([4], 4, device="cuda:0")


@pytest.mark.parametrize("dims,theta", [((), 1e4), ((2, 2, 2, 2, 2), 1e4), ((3,), 1e4), ((0,), 1e4), ((258,), 1e4),
                                        ((128, 130), 1e4), ((64,), 0.0), ((64,), -1.0), ((64,), math.nan),
                                        ((64,), math.inf)])
def test_axes_are_refused(nkv, dims, theta):
    with pytest.raises(nkv.InvalidConfigError):
        nkv.RotaryAxes(dims, theta=theta)
    from nomas_kv import _abi
    ax = _abi.nkv_rope_axes(len(dims), (C.c_int32 * 4)(*dims[:4]), 1, theta)
    with pytest.raises(nkv.InvalidConfigError):
        nkv._check(nkv.lib().nkv_rope_tables(C.byref(ax), None, 0, 0, None, None, None))


def _axes():
    from nomas_kv import _abi
    return _abi.nkv_rope_axes(1, (C.c_int32 * 4)(64, 0, 0, 0), 1, 1e4)


def test_null_arguments_are_refused(nkv):
    lib = nkv.lib()
    from nomas_kv import _abi
    assert lib.nkv_rope_tables(None, None, 0, 1, None, None, None) == 6
    assert lib.nkv_rotary(None, None) == 6
    assert lib.nkv_residual_norm(None, None) == 6
    assert lib.nkv_attend_packed(None, None, None) == 6
    assert lib.nkv_attend_plan_get_info(None, None) == 6
    assert lib.nkv_attend_plan_status(None, None) == 6
    assert lib.nkv_attend_plan_destroy(None) == 0
    assert lib.nkv_attend_schedule(None, None, 1, 1, 1, 1, 1, 148, None, 0, C.byref(C.c_uint64())) == 6
    ax = _axes()
    assert lib.nkv_rope_tables(C.byref(ax), None, 0, 4, None, None, None) == 6
    assert lib.nkv_rope_tables(C.byref(ax), None, 3, 0, None, None, None) == 6
    assert lib.nkv_rope_tables(C.byref(ax), None, 0, 2 ** 31, None, None, None) == 6
    assert lib.nkv_rope_tables(C.byref(ax), None, 0, 0, None, None, None) == 0  # no token: nothing to do
    a = _abi.nkv_rotary_args()
    a.axes, a.tokens, a.head_dim, a.dtype, a.eps = ax, 4, 64, 1, 1e-6
    a.q.heads = 2
    assert lib.nkv_rotary(C.byref(a), None) == 6  # null q


@pytest.mark.parametrize("change,code", [
    (dict(head_dim=62), 1), (dict(head_dim=65), 1), (dict(head_dim=258), 1), (dict(head_dim=0), 1),
    (dict(dtype=3), 6), (dict(norm=1, eps=-1.0), 6), (dict(norm=1, eps=math.nan), 6), (dict(tokens=2 ** 31), 6),
    (dict(position_type=9), 6),
])
def test_rotary_refuses_before_a_device_call(nkv, change, code):
    from nomas_kv import _abi
    a = _abi.nkv_rotary_args()
    a.axes, a.tokens, a.head_dim, a.dtype, a.eps = _axes(), 0, 64, 1, 1e-6
    assert nkv.lib().nkv_rotary(C.byref(a), None) == 0
    for f, v in change.items():
        setattr(a, f, v)
    assert nkv.lib().nkv_rotary(C.byref(a), None) == code


@pytest.mark.parametrize("change,code", [
    (dict(dim=0), 1), (dict(dim=32769), 1), (dict(dtype=5), 6), (dict(weight_dtype=2), 6), (dict(mod_dtype=2), 6),
    (dict(norm=3), 6), (dict(post=-1), 6), (dict(eps=-1.0), 6), (dict(eps=math.inf), 6),
    (dict(post=1), 6), (dict(gate=16), 6), (dict(post_weight=16), 6), (dict(norm=0), 6),
    (dict(norm=0, branch=16, weight=16), 6), (dict(scale=16, mod_rows=0), 1), (dict(scale=16, mod_rows=2), 1),
    (dict(tokens=2 ** 31), 6), (dict(tokens=1), 6),
])
def test_residual_norm_refuses_before_a_device_call(nkv, change, code):
    from nomas_kv import _abi
    a = _abi.nkv_residual_norm_args()
    a.dim, a.dtype, a.weight_dtype, a.mod_dtype, a.norm, a.eps = 64, 1, 0, 1, 1, 1e-6
    assert nkv.lib().nkv_residual_norm(C.byref(a), None) == 0
    for f, v in change.items():
        setattr(a, f, v)
    assert nkv.lib().nkv_residual_norm(C.byref(a), None) == code


def test_cpu_tensors_are_refused(nkv):
    import torch
    with pytest.raises(nkv.ArgumentError, match="CUDA device"):
        nkv.rotary(torch.zeros((2, 1), dtype=torch.int32), nkv.RotaryAxes((8,)), torch.zeros(2, 1, 8))
    with pytest.raises(nkv.ArgumentError, match="CUDA device"):
        nkv.rope_tables(torch.zeros((2, 1), dtype=torch.int32), nkv.RotaryAxes((8,)))
    with pytest.raises(nkv.ArgumentError, match="CUDA device"):
        nkv.residual_norm(torch.zeros(2, 8))


def test_overlap_rules(nkv):
    import torch
    from nomas_kv.block import _dense_order, _overlap
    x = torch.zeros(4, 6, 8)
    assert _overlap(x, x[:, :2]) and _overlap(x[:, 1:3], x[:, 2:4]) and _overlap(x[1:], x[:2])
    assert not _overlap(x[:, :2], x[:, 2:4]) and not _overlap(x[:2], x[2:]) and not _overlap(x[:, 4:], x[:, :4])
    assert not _overlap(x[:0], x) and not _overlap(x, torch.zeros(4, 6, 8))
    assert _overlap(x[:, 2:4], x[:1])  # other pitch classes: taken as overlapping
    assert _dense_order(x) and _dense_order(x.transpose(0, 1)) and not _dense_order(x[:, :1].expand(4, 6, 8))


def test_structs_match_the_header(nkv, tmp_path):
    from nomas_kv import _abi
    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    structs = {n: getattr(_abi, n) for n in ("nkv_rope_axes", "nkv_rotary_side", "nkv_rotary_args",
                                             "nkv_residual_norm_args", "nkv_attend_plan_info", "nkv_attend_args")}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "nomas_kv.h"', "int main(void) {"]
    for name, st in structs.items():
        lines.append(f'  printf("{name} %zu\\n", sizeof({name}));')
        for f, _ in st._fields_:
            lines.append(f'  printf("{name}.{f} %zu\\n", offsetof({name}, {f}));')
    lines += ["  return 0;", "}"]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines))
    inc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-std=c11", "-I", inc, str(src), "-o", str(exe)], check=True)
    out = dict(line.rsplit(" ", 1) for line in subprocess.run([str(exe)], capture_output=True, text=True,
                                                              check=True).stdout.splitlines())
    for name, st in structs.items():
        assert int(out[name]) == C.sizeof(st), name
        for f, _ in st._fields_:
            assert int(out[f"{name}.{f}"]) == getattr(st, f).offset, f"{name}.{f}"


def test_binding_leaves_cpu_tensors_to_the_checks(nkv):
    import torch
    from nomas_kv import _block_binding as fast
    q, pos = torch.zeros((2, 1, 8)), torch.zeros((2, 1), dtype=torch.int32)
    ax = nkv.RotaryAxes((8,))._packed
    assert fast.rotary(ax, pos, q, None, False, None, None, 1e-6, None, None) is None
    assert fast.rope_tables(ax, pos, None, None) is None
    assert fast.residual_norm(q[:, 0], None, None, 0, None, 1, None, None, None, None, 1e-6, None, None) is None
    assert fast.attend_packed(None, q, q, q, None, None, None, None, None) is None
    with pytest.raises(TypeError):
        fast.bind(1)
