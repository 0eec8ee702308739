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
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import ArgumentError, CudaError, GeometryError, InvalidConfigError, _abi, _check, lib

__all__ = ["RotaryAxes", "rope_tables", "rotary", "residual_norm", "AttendPlan", "attend_packed"]

_CODES = {torch.float32: _abi.NKV_F32, torch.bfloat16: _abi.NKV_BF16, torch.float16: _abi.NKV_F16}
_POSITIONS = {torch.int32: _abi.NKV_POS_I32, torch.int64: _abi.NKV_POS_I64, torch.float32: _abi.NKV_POS_F32}
_NORMS = {None: _abi.NKV_NORM_NONE, "none": _abi.NKV_NORM_NONE, "rms": _abi.NKV_NORM_RMS,
          "layer": _abi.NKV_NORM_LAYER}


# ---------------------------------------------------------------- checks
def _device_of(first, *rest):
    """The CUDA device all given tensors are on (None entries skipped)."""
    dev = first.device
    if dev.type != "cuda":
        raise ArgumentError("the tensors must be on a CUDA device (no CPU fallback)")
    grad = torch.is_grad_enabled()
    for t in (first, *rest):
        if t is None:
            continue
        if t.device != dev:
            raise ArgumentError(f"all tensors must be on {dev}, got one on {t.device}")
        if grad and t.requires_grad:
            raise ArgumentError("inference only: an input requires a gradient (use torch.no_grad() or detach())")
    return dev


def _code(t, name: str) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise GeometryError(f"{name} must be f32, bf16 or f16, got {t.dtype}")
    return code


class _On:
    """Device and stream of one call: makes the device current, gives the raw
    stream, and ties the tensors' memory to it when it is not the current one
    (the allocator then keeps a tensor freed early until the call's work is
    done)."""

    def __init__(self, dev, stream, tensors):
        self.guard = None if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)
        self.dev, self.stream, self.tensors = dev, stream, tensors

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        current = torch.cuda.current_stream(self.dev)
        self.switch = None
        if self.stream is None or self.stream == current:
            return C.c_void_p(current.cuda_stream)
        self.switch = torch.cuda.stream(self.stream)
        self.switch.__enter__()
        for t in self.tensors:
            if t is not None:
                t.record_stream(self.stream)
        return C.c_void_p(self.stream.cuda_stream)

    def __exit__(self, *exc):
        if self.switch is not None:
            self.switch.__exit__(*exc)
        if self.guard is not None:
            self.guard.__exit__(*exc)
        return False


def _extent(t) -> int:
    """Elements from the first to one past the last of a non-empty tensor."""
    return 1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))


def _overlap(a, b) -> bool:
    """Whether two tensors may share a byte: their ranges meet, and they are
    not column blocks of rows of one pitch that lie beside each other."""
    if a is None or b is None or a.numel() == 0 or b.numel() == 0:
        return False
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + _extent(a) * a.element_size() <= pb or pb + _extent(b) * b.element_size() <= pa:
        return False
    pitch = a.stride(0) * a.element_size()
    if pitch == b.stride(0) * b.element_size() and a.shape[0] > 1 and b.shape[0] > 1:
        ea, eb = _extent(a[0]) * a.element_size(), _extent(b[0]) * b.element_size()
        if ea <= pitch and eb <= pitch:
            d = (pb - pa) % pitch
            return d < ea or d + eb > pitch
    return True


def _same(a, b) -> bool:
    return b is not None and a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.stride() == b.stride()


def _dense_order(t) -> bool:
    """No two elements of t share memory (the strides nest)."""
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
        if _overlap(out, t) and not (any(t is a for a in alias) and _same(out, t)):
            raise ArgumentError(f"{name} overlaps an input")
    if any(_overlap(out, t) for t in others):
        raise ArgumentError(f"{name} overlaps another output")


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

    @property
    def pairs(self) -> int:
        return sum(self.dims) // 2

    def to_c(self) -> _abi.nkv_rope_axes:
        return _abi.nkv_rope_axes(len(self.dims), (C.c_int32 * 4)(*self.dims), int(self.interleaved),
                                  float(self.theta))


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
    dev = _device_of(positions, cos, sin)
    code = _positions(positions, axes, None)
    shape = (positions.shape[0], axes.pairs)
    with _On(dev, stream, (positions, cos, sin)) as s:
        for name, t, other in (("cos", cos, sin), ("sin", sin, cos)):
            if t is not None:
                _check_out(t, _Like(shape, torch.float32, dev), (positions,), name, others=(other,))
                if not t.is_contiguous():
                    raise GeometryError(f"{name} must be contiguous")
        if cos is None:
            cos = torch.empty(shape, dtype=torch.float32, device=dev)
        if sin is None:
            sin = torch.empty(shape, dtype=torch.float32, device=dev)
        c = axes.to_c()
        _check(lib().nkv_rope_tables(C.byref(c), positions.data_ptr(), code, shape[0], cos.data_ptr(),
                                     sin.data_ptr(), s))
    return cos, sin


def _rotary_side(t, out, weight) -> _abi.nkv_rotary_side:
    it, ih, _ = t.stride()
    ot, oh, _ = out.stride()
    return _abi.nkv_rotary_side(t.data_ptr(), out.data_ptr(), it, ih, ot, oh,
                                None if weight is None else weight.data_ptr(), t.shape[1])


def rotary(positions, axes: RotaryAxes, q, k=None, norm: bool = False, q_weight=None, k_weight=None,
           eps: float = 1e-6, q_out=None, k_out=None, stream=None):
    """Rotate q (tokens, heads, D), and k (tokens, kv_heads, D) with the same
    D and dtype, by their tokens' positions (nkv_rotary); with `norm` an RMS
    norm per head with the (D) gains q_weight / k_weight comes first.  D even,
    up to 256; f32, bf16 or f16; any token and head strides with the last
    dimension dense, so q and k may be views of one fused projection.  q_out /
    k_out may be q / k themselves (in place).  Returns q_out, or (q_out,
    k_out) when k is given."""
    dev = _device_of(q, k, positions, q_weight, k_weight, q_out, k_out)
    code = _code(q, "q")
    if q.dim() != 3:
        raise GeometryError("q must be (tokens, heads, head_dim)")
    tokens, _, D = q.shape
    if D < 2 or D % 2 or D > 256:
        raise GeometryError("head_dim must be even, 2 to 256")
    if 2 * axes.pairs > D:
        raise GeometryError(f"rotary axes {axes.dims} exceed head_dim {D}")
    if k is not None and (k.dim() != 3 or k.shape[0] != tokens or k.shape[2] != D or k.dtype != q.dtype):
        raise GeometryError(f"k must be ({tokens}, kv_heads, {D}) {q.dtype}")
    if k is None and (k_weight is not None or k_out is not None):
        raise ArgumentError("k_weight and k_out need k")
    if not norm and (q_weight is not None or k_weight is not None):
        raise ArgumentError("q_weight and k_weight need norm=True")
    pcode = _positions(positions, axes, tokens)
    for name, t in (("q", q), ("k", k)):
        if t is not None and t.stride(2) != 1:
            raise GeometryError(f"the last dimension of {name} must be dense")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (tuple(w.shape) != (D,) or w.dtype != q.dtype or not w.is_contiguous()):
            raise GeometryError(f"{name} must be a contiguous ({D},) {q.dtype} tensor")
    with _On(dev, stream, (q, k, positions, q_weight, k_weight, q_out, k_out)) as s:
        if q_out is not None:
            _check_out(q_out, q, (q, k, positions, q_weight, k_weight), "q_out", alias=(q,), others=(k_out,))
        else:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        if k is not None:
            if k_out is not None:
                _check_out(k_out, k, (k, q, positions, q_weight, k_weight), "k_out", alias=(k,), others=(q_out,))
            else:
                k_out = torch.empty(k.shape, dtype=k.dtype, device=dev)
        a = _abi.nkv_rotary_args()
        a.axes = axes.to_c()
        a.positions, a.position_type, a.dtype = positions.data_ptr(), pcode, code
        a.tokens, a.head_dim, a.norm, a.eps = tokens, D, int(bool(norm)), float(eps)
        a.q = _rotary_side(q, q_out, q_weight)
        if k is not None:
            a.k = _rotary_side(k, k_out, k_weight)
        _check(lib().nkv_rotary(C.byref(a), s))
    return q_out if k is None else (q_out, k_out)


# ---------------------------------------------------- gated residual norm
def _vector(t, name: str, dim: int, dtype, seen):
    """A weight of `dim` values, f32 or the stream's dtype, like the others."""
    if t is None:
        return seen
    if tuple(t.shape) != (dim,) or not t.is_contiguous():
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
    dev = _device_of(x, branch, gate, post_weight, weight, scale, shift, mod_index, h_out, y_out)
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
        if tuple(mod_index.shape) != (tokens,) or mod_index.dtype != torch.int32 or not mod_index.is_contiguous():
            raise GeometryError(f"mod_index must be a contiguous ({tokens},) int32 tensor")
        if not groups:
            raise ArgumentError("mod_index needs gate, scale or shift")
    elif groups > 1:
        raise GeometryError("several modulation rows need mod_index")
    vectors = (gate, post_weight, weight, scale, shift, mod_index)
    with _On(dev, stream, (x, branch, h_out, y_out, *vectors)) as s:
        h, y = x, None
        if branch is not None:
            if h_out is not None:
                _check_out(h_out, x, (x, branch, *vectors), "h_out", alias=(x, branch), others=(y_out,))
            h = torch.empty((tokens, dim), dtype=x.dtype, device=dev) if h_out is None else h_out
        if norm_c:
            if y_out is not None:
                _check_out(y_out, x, (x, branch, *vectors), "y_out", alias=(x, branch), others=(h_out,))
            y = torch.empty((tokens, dim), dtype=x.dtype, device=dev) if y_out is None else y_out
        p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
        a = _abi.nkv_residual_norm_args()
        a.tokens, a.dim, a.dtype = tokens, dim, code
        a.weight_dtype = code if wdt is None else _CODES[wdt]
        a.mod_dtype = code if mdt is None else _CODES[mdt]
        a.post, a.norm, a.eps = post_c, norm_c, float(eps)
        a.x, a.x_stride = x.data_ptr(), x.stride(0)
        if branch is not None:
            a.branch, a.branch_stride = branch.data_ptr(), branch.stride(0)
            a.h_out, a.h_stride = h.data_ptr(), h.stride(0)
        if norm_c:
            a.y_out, a.y_stride = y.data_ptr(), y.stride(0)
        a.post_weight, a.weight, a.gate, a.scale, a.shift = p(post_weight), p(weight), p(gate), p(scale), p(shift)
        a.mod_index, a.mod_rows = p(mod_index), groups
        _check(lib().nkv_residual_norm(C.byref(a), s))
    return h, y


# -------------------------------------------------------- packed attention
def _lens(v: Sequence[int], name: str):
    v = [int(n) for n in v]
    if any(n < 0 for n in v):
        raise GeometryError(f"{name} must not be negative")
    return v, (C.c_uint64 * max(len(v), 1))(*v)


class AttendPlan:
    """The work list of attend_packed for one set of sequence lengths
    (nkv_attend_plan_create): q_lens query tokens over k_lens keys each
    (default: the same), `heads` query heads in groups over kv_heads (default:
    heads) key/value heads, head_dim a multiple of 8 up to 128.  causal: token
    i sees the keys up to its own position, aligned to the sequence's last
    key; block > 1: up to the end of the block of `block` keys that holds it
    (tokens per frame: frame-causal).  causal False: every key.

    Made once per set of lengths (it uploads a table to `device`) and used for
    any number of layers, calls, streams and graphs; it must outlive them."""

    def __init__(self, q_lens: Sequence[int], heads: int, kv_heads: Optional[int] = None, head_dim: int = 128,
                 k_lens: Optional[Sequence[int]] = None, causal: bool = True, block: int = 1, device=None):
        self._h = None
        q, qa = _lens(q_lens, "q_lens")
        k, ka = (q, qa) if k_lens is None else _lens(k_lens, "k_lens")
        if len(q) != len(k):
            raise GeometryError("q_lens and k_lens must have one entry per sequence")
        if int(block) < 1:
            raise ArgumentError("block must be 1 to 2^31 - 1")
        self.heads, self.kv_heads = int(heads), int(heads if kv_heads is None else kv_heads)
        self.head_dim, self.causal, self.block = int(head_dim), bool(causal), int(block)
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

    def close(self):
        if getattr(self, "_h", None):
            _check(lib().nkv_attend_plan_destroy(self._h))
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def check(self) -> None:
        """Wait for the device and raise CudaError if a call of this plan gave
        up on one of its bounded waits."""
        w = C.c_uint32()
        _check(lib().nkv_attend_plan_status(self._h, C.byref(w)))
        if w.value:
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
    dev = _device_of(q, k, v, ho, hl, out, lse)
    if dev != plan.device:
        raise ArgumentError(f"the plan is for {plan.device}, the tensors are on {dev}")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise GeometryError("packed attention needs bf16 or f16 queries, keys and values")
    if q.dim() != 3 or q.shape[1:] != (H, D) or q.shape[0] < plan.q_tokens:
        raise GeometryError(f"q must be (at least {plan.q_tokens}, {H}, {D})")
    rows, k_rows = q.shape[0], k.shape[0] if k.dim() else 0
    for name, t in (("k", k), ("v", v)):
        if t.dim() != 3 or t.shape[1:] != (KV, D) or t.shape[0] < plan.k_tokens or t.dtype != q.dtype:
            raise GeometryError(f"{name} must be (at least {plan.k_tokens}, {KV}, {D}) {q.dtype}")
    k_rows = min(k_rows, v.shape[0])
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.stride(2) != 1:
            raise GeometryError(f"the last dimension of {name} must be dense")
        # a dimension of one has no stride that counts
        if t.numel() and (t.data_ptr() % 16 or (t.shape[0] > 1 and t.stride(0) % 8) or
                          (t.shape[1] > 1 and t.stride(1) % 8)):
            raise ArgumentError(f"{name} must be 16-byte aligned with strides of multiples of 8 elements")
    if history is not None:
        for name, t, shape in (("o", ho, (rows, H, D)), ("lse", hl, (H, rows))):
            if tuple(t.shape) != shape or t.dtype != torch.float32 or not t.is_contiguous():
                raise GeometryError(f"the history's {name} must be a contiguous f32 tensor of shape {shape}")
    with _On(dev, stream, (q, k, v, ho, hl, out, lse)) as s:
        if out is None:
            # a padded batch keeps rows that nothing writes: zeros, not stale memory
            new = torch.empty if rows == plan.q_tokens else torch.zeros
            out = new((rows, H, D), dtype=q.dtype, device=dev)
        else:
            like = _Like((rows, H, D), torch.float32 if out.dtype == torch.float32 else q.dtype, dev)
            _check_out(out, like, (q, k, v, ho, hl), "out", others=(lse,))
            if not out.is_contiguous():
                raise GeometryError("out must be contiguous")
        if lse is None:
            lse = torch.empty((H, rows), dtype=torch.float32, device=dev) if rows == plan.q_tokens else \
                torch.full((H, rows), -math.inf, dtype=torch.float32, device=dev)
        else:
            _check_out(lse, _Like((H, rows), torch.float32, dev), (q, k, v, ho, hl), "lse", others=(out,))
            if not lse.is_contiguous():
                raise GeometryError("lse must be contiguous")
        ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=dev) if plan.workspace_bytes else None
        a = _abi.nkv_attend_args()
        a.dtype, a.out_dtype = _CODES[q.dtype], _CODES[out.dtype]
        a.q_rows, a.k_rows = rows, k_rows
        one = lambda t, i: t.stride(i) if t.shape[i] > 1 else 0  # noqa: E731
        a.q, a.q_token_stride, a.q_head_stride = q.data_ptr(), one(q, 0), one(q, 1)
        a.k, a.k_token_stride, a.k_head_stride = k.data_ptr(), one(k, 0), one(k, 1)
        a.v, a.v_token_stride, a.v_head_stride = v.data_ptr(), one(v, 0), one(v, 1)
        a.scale = float(scale) if scale is not None else 1.0 / math.sqrt(D)
        a.out, a.lse = out.data_ptr(), lse.data_ptr()
        if ho is not None:
            a.hist_out, a.hist_lse = ho.data_ptr(), hl.data_ptr()
        if ws is not None:
            a.workspace, a.workspace_bytes = ws.data_ptr(), plan.workspace_bytes
        _check(lib().nkv_attend_packed(plan._h, C.byref(a), s))
    return out, lse
