"""The operators of the attention block beside the cache, on torch tensors.

``rope_tables`` and ``rotary`` (rotary positions with several axes),
``residual_norm`` (gated residual and the norms on both sides of a block) and
``attend_packed`` with its ``AttendPlan`` (softmax attention of packed
sequences with grouped heads, merged with the history part).  Every call runs
on the device of its tensors, on torch's current stream there or on
``stream``, synchronises nothing and may be captured into a CUDA graph.
Inference only: an input that requires a gradient is refused while gradients
are recorded.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import ArgumentError, CudaError, GeometryError, InvalidConfigError, _abi, _check, lib

try:
    from . import _block_binding
except ImportError as e:
    raise ImportError(f"{e}; build it with: python hy-nomas-rs_b200/build.py") from e

__all__ = ["RotaryAxes", "rope_tables", "rotary", "residual_norm", "AttendPlan", "attend_packed"]

_CODES = {torch.float32: _abi.NKV_F32, torch.bfloat16: _abi.NKV_BF16, torch.float16: _abi.NKV_F16}
_POSITIONS = {torch.int32: _abi.NKV_POS_I32, torch.int64: _abi.NKV_POS_I64, torch.float32: _abi.NKV_POS_F32}
_NORMS = {None: _abi.NKV_NORM_NONE, "none": _abi.NKV_NORM_NONE, "rms": _abi.NKV_NORM_RMS,
          "layer": _abi.NKV_NORM_LAYER}


# A call of a few microseconds of GPU work is bound by what happens here.  The
# plain calls (torch's current device and stream) go through the
# compiled binding, which returns None for whatever it does not take: the code
# below then serves the call or says what is wrong with it.  It packs the
# argument structs in one go (native layout, as the header's).
_block_binding.bind(*(C.cast(getattr(lib(), f), C.c_void_p).value
                      for f in ("nkv_rope_tables", "nkv_rotary", "nkv_residual_norm", "nkv_attend_packed")))
_AXES = struct.Struct("i4iid")
_ROTARY = struct.Struct("32sPiiQiif" + "PPqqqqPi0P" * 2)
_NORM = struct.Struct("QqiiiiifPPPPqqqqPPPPPPi0P")
_ATTEND = struct.Struct("iiQQPPPqqqqqqfPPPPPQ")
_PLAN = struct.Struct("QiiiiQQQ")
for _s, _t in ((_AXES, _abi.nkv_rope_axes), (_ROTARY, _abi.nkv_rotary_args), (_NORM, _abi.nkv_residual_norm_args),
               (_ATTEND, _abi.nkv_attend_args)):
    assert _s.size == C.sizeof(_t), _t.__name__

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


# ---------------------------------------------------------------- checks
def _device_of(first, *rest) -> int:
    """The index of the CUDA device all given tensors are on (None entries
    skipped)."""
    index = first.get_device()
    if index < 0:
        raise ArgumentError("the tensors must be on a CUDA device (no CPU fallback)")
    grad = torch.is_grad_enabled()
    if grad and first.requires_grad:
        raise ArgumentError(_NO_GRAD)
    for t in rest:
        if t is None:
            continue
        if t.get_device() != index:
            raise ArgumentError(f"all tensors must be on {first.device}, got one on {t.device}")
        if grad and t.requires_grad:
            raise ArgumentError(_NO_GRAD)
    return index


_NO_GRAD = "inference only: an input requires a gradient (use torch.no_grad() or detach())"


def _code(t, name: str) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise GeometryError(f"{name} must be f32, bf16 or f16, got {t.dtype}")
    return code


class _Elsewhere:
    """Makes a device current, and a stream other than its current one, whose
    work the tensors' memory is then tied to (the allocator keeps a tensor
    freed early until that work is done)."""

    def __init__(self, index, stream, tensors):
        self.device = torch.cuda.device(index)
        self.device.__enter__()
        self.stream = None
        if stream is not None and stream != torch.cuda.current_stream(index):
            self.stream = torch.cuda.stream(stream)
            self.stream.__enter__()
            for t in tensors:
                if t is not None:
                    t.record_stream(stream)

    def leave(self):
        if self.stream is not None:
            self.stream.__exit__(None, None, None)
        self.device.__exit__(None, None, None)


def _check_eps(eps) -> None:
    if not 0.0 <= eps <= 3.4e38:
        raise ArgumentError("eps must be finite and not negative")


def _fresh(like):
    """A contiguous tensor of like's shape and type (empty_like is the quicker
    call, but keeps the strides of a dense one)."""
    return torch.empty_like(like) if like.is_contiguous() else like.new_empty(like.shape)


def _enter(index, stream, tensors):
    """None where the call runs on the current device's current stream."""
    if stream is not None and stream.device_index != index:
        raise ArgumentError(f"the stream is on device {stream.device_index}, the tensors on {index}")
    if stream is None and torch.cuda.current_device() == index:
        return None
    return _Elsewhere(index, stream, tensors)


def _extent(t) -> int:
    """Bytes from the first element to the end of the last of a non-empty tensor."""
    es = t.element_size()
    if t.is_contiguous():
        return t.numel() * es
    n = 1
    for size, stride in zip(t.shape, t.stride()):
        n += (size - 1) * stride
    return n * es


def _overlap(a, b) -> bool:
    """Whether two tensors may share a byte: their ranges meet, and they are
    not column blocks of rows of one pitch that lie beside each other."""
    if a is None or b is None or a.numel() == 0 or b.numel() == 0:
        return False
    pa, pb = a.data_ptr(), b.data_ptr()
    if (pa + _extent(a) <= pb) if pa <= pb else (pb + _extent(b) <= pa):
        return False
    if a.dim() and b.dim():
        pitch = a.stride(0) * a.element_size()
        if pitch == b.stride(0) * b.element_size() and a.shape[0] > 1 and b.shape[0] > 1:
            ea, eb = _extent(a[0]), _extent(b[0])
            if ea <= pitch and eb <= pitch:
                d = (pb - pa) % pitch
                return d < ea or d + eb > pitch
    return True


def _same(a, b) -> bool:
    return b is not None and a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()


def _dense_order(t) -> bool:
    """No two elements of t share memory (the strides nest)."""
    if t.is_contiguous():
        return True
    need = 1
    for n, s in sorted(((n, s) for n, s in zip(t.shape, t.stride()) if n > 1), key=lambda p: p[1]):
        if s < need:
            return False
        need = s * (n - 1) + need
    return True


@dataclass
class _Like:
    shape: tuple
    dtype: object
    device: object

    def __post_init__(self):
        self.shape = torch.Size(self.shape)


def _check_out(out, like, ins, name: str, alias=(), others=()):
    """A caller's output: shape / dtype / device of `like`, memory apart from
    the inputs' (or exactly that of one in `alias`) and the other outputs'."""
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise GeometryError(f"{name} must be {tuple(like.shape)} {like.dtype} on {like.device}")
    if out.dim() and out.shape[-1] > 1 and out.stride(-1) != 1:
        raise GeometryError(f"the last dimension of {name} must be dense")
    if not _dense_order(out):
        raise GeometryError(f"elements of {name} overlap")
    for t in ins:
        if t is not None and not (_same(out, t) and any(t is x for x in alias)) and _overlap(out, t):
            raise ArgumentError(f"{name} overlaps an input")
    if any(_overlap(out, t) for t in others):
        raise ArgumentError(f"{name} overlaps another output")


def _written(*given) -> None:
    """Counts the write to the caller's outputs, as torch's in-place operations
    do: a backward pass that saved one of them raises."""
    for t in given:
        if t is not None and not t.is_inference():
            torch.autograd.graph.increment_version(t)


# ---------------------------------------------------------------- rotary
@dataclass(frozen=True)
class RotaryAxes:
    """The axes of the rotary positions: axis a owns dims[a] (even) of the
    sum(dims) rotated values of a head, in order, with the frequencies
    theta^(-2 i / dims[a]).  interleaved: pairs (2p, 2p + 1), the layout of
    kv_project and of the reference (rope.rs:257-306); else (p, p + half)."""

    dims: tuple
    theta: float = 10000.0
    interleaved: bool = True

    def __post_init__(self):
        dims = tuple(int(d) for d in self.dims)
        if not 1 <= len(dims) <= 4 or any(d < 2 or d % 2 for d in dims) or sum(dims) > 256:
            raise InvalidConfigError("rotary positions need 1 to 4 axes of even dims >= 2 with a sum of at most 256")
        if not (self.theta > 0 and math.isfinite(self.theta)):
            raise InvalidConfigError("theta must be finite and positive")
        object.__setattr__(self, "dims", dims)
        object.__setattr__(self, "_packed", _AXES.pack(len(dims), *(dims + (0,) * (4 - len(dims))),
                                                       int(bool(self.interleaved)), float(self.theta)))

    @property
    def pairs(self) -> int:
        return sum(self.dims) // 2

    def to_c(self) -> _abi.nkv_rope_axes:
        return _abi.nkv_rope_axes.from_buffer_copy(self._packed)


def _positions(positions, axes: RotaryAxes, tokens: Optional[int]) -> int:
    code = _POSITIONS.get(positions.dtype)
    if code is None:
        raise GeometryError(f"positions must be int32, int64 or f32, got {positions.dtype}")
    n = len(axes.dims)
    if positions.dim() != 2 or positions.shape[1] != n or (tokens is not None and positions.shape[0] != tokens):
        raise GeometryError(f"positions must be ({'tokens' if tokens is None else tokens}, {n})")
    if not positions.is_contiguous():
        raise GeometryError("positions must be contiguous")
    return code


def rope_tables(positions, axes: RotaryAxes, cos=None, sin=None, stream=None):
    """The (cos, sin) f32 tables (tokens, axes.pairs) of nkv_rope_tables: what
    kv_project takes as `rope` (64 pairs).  positions: (tokens, n_axes) int32,
    int64 or f32."""
    if stream is None:
        done = _block_binding.rope_tables(axes._packed, positions, cos, sin)
        if done is not None:
            return done
    index = _device_of(positions, cos, sin)
    code = _positions(positions, axes, None)
    shape = (positions.shape[0], axes.pairs)
    given = (cos, sin)
    away = _enter(index, stream, (positions, cos, sin))
    try:
        for name, t, other in (("cos", cos, sin), ("sin", sin, cos)):
            if t is not None:
                _check_out(t, _Like(shape, torch.float32, positions.device), (positions,), name, others=(other,))
                if not t.is_contiguous():
                    raise GeometryError(f"{name} must be contiguous")
        if cos is None:
            cos = positions.new_empty(shape, dtype=torch.float32)
        if sin is None:
            sin = positions.new_empty(shape, dtype=torch.float32)
        _check(lib().nkv_rope_tables(axes._packed, positions.data_ptr(), code, shape[0], cos.data_ptr(),
                                     sin.data_ptr(), _raw_stream(index)))
    finally:
        if away is not None:
            away.leave()
    _written(*given)
    return cos, sin


def rotary(positions, axes: RotaryAxes, q, k=None, norm: bool = False, q_weight=None, k_weight=None,
           eps: float = 1e-6, q_out=None, k_out=None, stream=None):
    """Rotate q (tokens, heads, D), and k (tokens, kv_heads, D) with the same
    D and dtype, by their tokens' positions (nkv_rotary); with `norm` an RMS
    norm per head with the (D) gains q_weight / k_weight comes first.  D even,
    up to 256; f32, bf16 or f16; any token and head strides with the last
    dimension dense, so q and k may be views of one fused projection.  q_out /
    k_out may be q / k themselves (in place, where k is not q).  Returns q_out, or (q_out,
    k_out) when k is given."""
    if stream is None:
        done = _block_binding.rotary(axes._packed, positions, q, k, norm, q_weight, k_weight, eps, q_out, k_out)
        if done is not None:
            return done
    index = _device_of(q, k, positions, q_weight, k_weight, q_out, k_out)
    code = _code(q, "q")
    if q.dim() != 3:
        raise GeometryError("q must be (tokens, heads, head_dim)")
    tokens, heads, D = q.shape
    if D < 2 or D % 2 or D > 256:
        raise GeometryError("head_dim must be even, 2 to 256")
    if 2 * axes.pairs > D:
        raise GeometryError(f"rotary axes {axes.dims} exceed head_dim {D}")
    if k is None:
        if k_weight is not None or k_out is not None:
            raise ArgumentError("k_weight and k_out need k")
    elif k.dim() != 3 or k.shape[0] != tokens or k.shape[2] != D or k.dtype != q.dtype:
        raise GeometryError(f"k must be ({tokens}, kv_heads, {D}) {q.dtype}")
    if not norm and (q_weight is not None or k_weight is not None):
        raise ArgumentError("q_weight and k_weight need norm=True")
    _check_eps(eps)
    pcode = _positions(positions, axes, tokens)
    q_st = q.stride()
    k_st = (0, 0, 1) if k is None else k.stride()
    if q_st[2] != 1 or k_st[2] != 1:
        raise GeometryError("the last dimension of q and k must be dense")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (D,) or w.dtype != q.dtype or not w.is_contiguous()):
            raise GeometryError(f"{name} must be a contiguous ({D},) {q.dtype} tensor")
    ins = (q, k, positions, q_weight, k_weight)
    apart = k is q  # read as both: neither may be rotated in place
    given = (q_out, k_out)
    away = _enter(index, stream, (*ins, q_out, k_out))
    try:
        if q_out is not None:
            _check_out(q_out, q, ins, "q_out", alias=() if apart else (q,), others=(k_out,))
            qo_st = q_out.stride()
        else:
            q_out = _fresh(q)
            qo_st = (heads * D, D)
        k_heads, k_p, ko_p, ko_st = 0, 0, 0, (0, 0)
        if k is not None:
            k_heads = k.shape[1]
            if k_out is not None:
                _check_out(k_out, k, ins, "k_out", alias=() if apart else (k,), others=(q_out,))
                ko_st = k_out.stride()
            else:
                k_out = _fresh(k)
                ko_st = (k_heads * D, D)
            k_p, ko_p = k.data_ptr(), k_out.data_ptr()
        _check(lib().nkv_rotary(
            _ROTARY.pack(axes._packed, positions.data_ptr(), pcode, code, tokens, D, 1 if norm else 0, eps,
                         q.data_ptr(), q_out.data_ptr(), q_st[0], q_st[1], qo_st[0], qo_st[1],
                         0 if q_weight is None else q_weight.data_ptr(), heads,
                         k_p, ko_p, k_st[0], k_st[1], ko_st[0], ko_st[1],
                         0 if k_weight is None else k_weight.data_ptr(), k_heads), _raw_stream(index)))
    finally:
        if away is not None:
            away.leave()
    _written(*given)
    return q_out if k is None else (q_out, k_out)


# ---------------------------------------------------- gated residual norm
def _vector(t, name: str, dim: int, dtype, seen):
    """A weight of `dim` values, f32 or the stream's dtype, like the others."""
    if t is None:
        return seen
    if t.shape != (dim,) or not t.is_contiguous():
        raise GeometryError(f"{name} must be a contiguous ({dim},) tensor")
    if t.dtype not in (torch.float32, dtype) or (seen is not None and t.dtype != seen):
        raise GeometryError(f"the weights must share one type, f32 or {dtype}")
    return t.dtype


def residual_norm(x, branch=None, *, gate=None, post=None, post_weight=None, norm="rms", weight=None, scale=None,
                  shift=None, mod_index=None, eps: float = 1e-6, h_out=None, y_out=None, stream=None):
    """The residual stream between two blocks (nkv_residual_norm):

        h = x + gate * (post(branch) * post_weight)
        y = norm(h) * weight * (1 + scale) + shift

    x, branch: (tokens, dim) f32, bf16 or f16 with dense rows; post / norm:
    None, "rms" or "layer"; weights (dim), gate / scale / shift (groups, dim)
    or (dim), f32 or x's type; mod_index: (tokens) int32, the row of gate /
    scale / shift of each token (needed when there are several; a token whose
    index is out of range gets NaN).  Without a branch h is x; with norm None
    y is None.  h_out / y_out may be x or branch.  Returns (h, y); y is what
    kv_project takes as x."""
    if stream is None and post in _NORMS and norm in _NORMS:
        done = _block_binding.residual_norm(x, branch, gate, _NORMS[post], post_weight, _NORMS[norm], weight, scale,
                                            shift, mod_index, eps, h_out, y_out)
        if done is not None:
            return done
    index = _device_of(x, branch, gate, post_weight, weight, scale, shift, mod_index, h_out, y_out)
    code = _code(x, "x")
    if x.dim() != 2 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise GeometryError("x must be (tokens, dim) with dense rows")
    tokens, dim = x.shape
    if not 1 <= dim <= 32768:
        raise GeometryError("dim must be 1 to 32768")
    if branch is not None and (branch.shape != x.shape or branch.dtype != x.dtype or
                               (dim > 1 and branch.stride(1) != 1)):
        raise GeometryError(f"branch must be ({tokens}, {dim}) {x.dtype} with dense rows")
    if post not in _NORMS or norm not in _NORMS:
        raise ArgumentError('post and norm must be None, "rms" or "layer"')
    post_c, norm_c = _NORMS[post], _NORMS[norm]
    if branch is None and (post_c or gate is not None or post_weight is not None or h_out is not None):
        raise ArgumentError("post, post_weight, gate and h_out need a branch")
    if not norm_c and (weight is not None or scale is not None or shift is not None or y_out is not None):
        raise ArgumentError("weight, scale, shift and y_out need a norm")
    if branch is None and not norm_c:
        raise ArgumentError("nothing to do: no branch and no norm")
    _check_eps(eps)
    wdt = _vector(post_weight, "post_weight", dim, x.dtype, None)
    wdt = _vector(weight, "weight", dim, x.dtype, wdt)
    mdt, groups = None, 0
    for name, t in (("gate", gate), ("scale", scale), ("shift", shift)):
        if t is None:
            continue
        g = 1 if t.dim() == 1 else t.shape[0]
        if t.dim() not in (1, 2) or t.shape[-1] != dim or not t.is_contiguous() or g < 1:
            raise GeometryError(f"{name} must be a contiguous (groups, {dim}) or ({dim},) tensor")
        if t.dtype not in (torch.float32, x.dtype) or (mdt is not None and t.dtype != mdt):
            raise GeometryError(f"gate, scale and shift must share one type, f32 or {x.dtype}")
        if groups and g != groups:
            raise GeometryError("gate, scale and shift must have the same number of rows")
        mdt, groups = t.dtype, g
    if mod_index is not None:
        if mod_index.shape != (tokens,) or mod_index.dtype != torch.int32 or not mod_index.is_contiguous():
            raise GeometryError(f"mod_index must be a contiguous ({tokens},) int32 tensor")
        if not groups:
            raise ArgumentError("mod_index needs gate, scale or shift")
    elif groups > 1:
        raise GeometryError("several modulation rows need mod_index")
    vectors = (gate, post_weight, weight, scale, shift, mod_index)
    away = _enter(index, stream, (x, branch, h_out, y_out, *vectors))
    try:
        h, y, h_p, y_p, h_st, y_st = x, None, 0, 0, 0, 0
        if branch is not None:
            if h_out is not None:
                _check_out(h_out, x, (x, branch, *vectors), "h_out", alias=(x, branch), others=(y_out,))
                h, h_st = h_out, h_out.stride(0)
            else:
                h, h_st = _fresh(x), dim
            h_p = h.data_ptr()
        if norm_c:
            if y_out is not None:
                _check_out(y_out, x, (x, branch, *vectors), "y_out", alias=(x, branch), others=(h_out,))
                y, y_st = y_out, y_out.stride(0)
            else:
                y, y_st = _fresh(x), dim
            y_p = y.data_ptr()
        p = [0 if t is None else t.data_ptr() for t in vectors]
        _check(lib().nkv_residual_norm(
            _NORM.pack(tokens, dim, code, code if wdt is None else _CODES[wdt], code if mdt is None else _CODES[mdt],
                       post_c, norm_c, eps, x.data_ptr(), 0 if branch is None else branch.data_ptr(), h_p, y_p,
                       x.stride(0), 0 if branch is None else branch.stride(0), h_st, y_st, p[1], p[2], p[0], p[3],
                       p[4], p[5], groups), _raw_stream(index)))
    finally:
        if away is not None:
            away.leave()
    _written(h_out, y_out)
    return h, y


# -------------------------------------------------------- packed attention
def _lens(v: Sequence[int], name: str):
    v = [int(n) for n in v]
    if any(n < 0 for n in v):
        raise GeometryError(f"{name} must not be negative")
    if any(n >= 2 ** 31 for n in v):  # (before ctypes takes them modulo 2^64)
        raise GeometryError("sequence too long")
    return v, (C.c_uint64 * max(len(v), 1))(*v)


class AttendPlan:
    """The work list of attend_packed for one set of sequence lengths
    (nkv_attend_plan_create): q_lens query tokens over k_lens keys each
    (default: the same), `heads` query heads in groups of at most 128 over
    kv_heads (default: heads) key/value heads, head_dim a multiple of 8 up to 128.  causal: token
    i sees the keys up to its own position, aligned to the sequence's last
    key; block > 1: up to the end of the block of `block` keys that holds it
    (tokens per frame: frame-causal).  causal False: every key.

    Made once per set of lengths (it uploads a table to `device`) and used for
    any number of layers, calls, streams and graphs; it must outlive them.
    Making one waits for the device's default stream and takes about half a
    millisecond, dropping one waits for the device (0.3 ms): cheap per segment,
    not per call.  Where a cache grows by a token at a time, share a step's
    plan among all layers."""

    def __init__(self, q_lens: Sequence[int], heads: int, kv_heads: Optional[int] = None, head_dim: int = 128,
                 k_lens: Optional[Sequence[int]] = None, causal: bool = True, block: int = 1, device=None):
        self._h = self._key = None
        q, qa = _lens(q_lens, "q_lens")
        k, ka = (q, qa) if k_lens is None else _lens(k_lens, "k_lens")
        if len(q) != len(k):
            raise GeometryError("q_lens and k_lens must have one entry per sequence")
        if not 1 <= int(block) < 2 ** 31:
            raise ArgumentError("block must be 1 to 2^31 - 1")
        self.heads, self.kv_heads = int(heads), int(heads if kv_heads is None else kv_heads)
        self.head_dim, self.causal, self.block = int(head_dim), bool(causal), int(block)
        if any(abs(n) >= 2 ** 31 for n in (self.heads, self.kv_heads, self.head_dim)):
            raise GeometryError("heads, kv_heads and head_dim must fit in 32 bits")
        if device is None:
            device = torch.device("cuda", torch.cuda.current_device() if torch.cuda.is_available() else 0)
        device = torch.device(device)
        if device.type != "cuda":
            raise ArgumentError("packed attention runs on a CUDA device only (no CPU fallback)")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        self.device = device
        h = C.c_void_p()
        _check(lib().nkv_attend_plan_create(qa, ka, len(q), self.heads, self.kv_heads, self.head_dim,
                                            int(self.causal), self.block, device.index, C.byref(h)))
        self._h = h
        info = _abi.nkv_attend_plan_info()
        _check(lib().nkv_attend_plan_get_info(h, C.byref(info)))
        self.q_tokens, self.k_tokens = int(info.q_tokens), int(info.k_tokens)
        self.items, self.split_units = int(info.items), int(info.split_units)
        self.workspace_bytes = int(info.workspace_bytes)
        self._key = _PLAN.pack(h.value, self.heads, self.kv_heads, self.head_dim, device.index, self.q_tokens,
                               self.k_tokens, self.workspace_bytes)

    def close(self):
        if getattr(self, "_h", None):
            self._key = None
            _check(lib().nkv_attend_plan_destroy(self._h))
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def check(self) -> None:
        """Wait for the device and raise CudaError if a call of this plan gave
        up on one of its bounded waits since the last check.  From such a call
        on the plan's results are NaN, until check has reported it."""
        w = C.c_uint32()
        _check(lib().nkv_attend_plan_status(self._h, C.byref(w)))
        if w.value:
            _check(lib().nkv_attend_plan_set_status(self._h, 0))
            raise CudaError("packed attention: a bounded wait ran out")


def attend_packed(plan: AttendPlan, q, k, v, scale: Optional[float] = None, history=None, out=None, lse=None,
                  stream=None):
    """Softmax attention of plan's packed sequences (nkv_attend_packed).  q
    (q_rows, heads, D), k / v (k_rows, kv_heads, D), bf16 or f16, any token and
    head strides that are multiples of 8 elements; rows behind the last
    sequence are neither read nor written.  history = (o, lse) of the same
    queries over other keys, as LayerCache.attend_history returns them: (q_rows,
    heads, D) and (heads, q_rows) f32; the result is then over both.  scale
    defaults to 1 / sqrt(D).  Returns out (q_rows, heads, D), of q's type unless
    a f32 `out` is given, and lse (heads, q_rows) f32; a row that sees no key is
    0 with lse -inf."""
    if plan._h is None:
        raise ArgumentError("the plan is closed")
    H, KV, D = plan.heads, plan.kv_heads, plan.head_dim
    ho, hl = (None, None) if history is None else history
    if stream is None:
        done = _block_binding.attend_packed(plan._key, q, k, v, scale, ho, hl, out, lse)
        if done is not None:
            return done
    index = _device_of(q, k, v, ho, hl, out, lse)
    if index != plan.device.index:
        raise ArgumentError(f"the plan is for {plan.device}, the tensors are on {q.device}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise GeometryError("packed attention needs bf16 or f16 queries, keys and values")
    if q.dim() != 3 or q.shape[1:] != (H, D) or q.shape[0] < plan.q_tokens:
        raise GeometryError(f"q must be (at least {plan.q_tokens}, {H}, {D})")
    rows = q.shape[0]
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    elif not 0.0 < scale <= 3.4e38:
        raise ArgumentError("scale must be finite and positive")
    for name, t in (("k", k), ("v", v)):
        if t.dim() != 3 or t.shape[1:] != (KV, D) or t.shape[0] < plan.k_tokens or t.dtype != q.dtype:
            raise GeometryError(f"{name} must be (at least {plan.k_tokens}, {KV}, {D}) {q.dtype}")
    k_rows = min(k.shape[0], v.shape[0])
    where = []  # address, token stride, head stride
    for name, t, heads in (("q", q, H), ("k", k, KV), ("v", v, KV)):
        p, (st, sh, sd) = t.data_ptr(), t.stride()
        if sd != 1:
            raise GeometryError(f"the last dimension of {name} must be dense")
        # a dimension of one has no stride that counts
        if t.shape[0] < 2:
            st = 0
        if heads < 2:
            sh = 0
        if (p | st * 2 | sh * 2) % 16:
            raise ArgumentError(f"{name} must be 16-byte aligned with strides of multiples of 8 elements")
        where.append((p, st, sh))
    ho_p = hl_p = 0
    if history is not None:
        for name, t, shape in (("o", ho, (rows, H, D)), ("lse", hl, (H, rows))):
            if t.shape != shape or t.dtype != torch.float32 or not t.is_contiguous():
                raise GeometryError(f"the history's {name} must be a contiguous f32 tensor of shape {shape}")
        ho_p, hl_p = ho.data_ptr(), hl.data_ptr()
    given = (out, lse)
    away = _enter(index, stream, (q, k, v, ho, hl, out, lse))
    try:
        padded = rows != plan.q_tokens
        if out is None:
            # a padded batch keeps rows that nothing writes: zeros, not stale memory
            out = q.new_zeros((rows, H, D)) if padded else _fresh(q)
        else:
            like = _Like((rows, H, D), torch.float32 if out.dtype == torch.float32 else q.dtype, q.device)
            _check_out(out, like, (q, k, v, ho, hl), "out", others=(lse,))
            if not out.is_contiguous():
                raise GeometryError("out must be contiguous")
        if lse is None:
            lse = q.new_full((H, rows), -math.inf, dtype=torch.float32) if padded else \
                q.new_empty((H, rows), dtype=torch.float32)
        else:
            _check_out(lse, _Like((H, rows), torch.float32, q.device), (q, k, v, ho, hl), "lse", others=(out,))
            if not lse.is_contiguous():
                raise GeometryError("lse must be contiguous")
        n = plan.workspace_bytes
        ws = q.new_empty(n, dtype=torch.uint8) if n else None
        (qp, qt, qh), (kp, kt, kh), (vp, vt, vh) = where
        _check(lib().nkv_attend_packed(
            plan._h, _ATTEND.pack(_CODES[q.dtype], _CODES[out.dtype], rows, k_rows, qp, kp, vp, qt, qh, kt, kh, vt, vh,
                                  scale, out.data_ptr(), lse.data_ptr(),
                                  ho_p, hl_p, ws.data_ptr() if n else 0, n), _raw_stream(index)))
    finally:
        if away is not None:
            away.leave()
    _written(*given)
    return out, lse
