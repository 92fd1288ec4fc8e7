"""Transformer-layer operators on torch tensors: the Python side of mibc_rms_norm, mibc_rope and mibc_attention
(include/mibc.h, which states the formulas).

Tensors live on one HIP device; the work goes to torch's current stream of that device and nothing is synchronised.  New
outputs and the workspace of a split attention come from torch's caching allocator, so a call can be captured into a graph.
There is no CPU form: a tensor elsewhere raises.  Forward only; no autograd graph is recorded, so inputs that require a
gradient are refused while gradients are being recorded, and so are forward-mode tangents, tracing (torch.jit.trace, make_fx) and
tensors without memory of their own (fake, functional, symbolic zeros): all of these would pass the work by.  A tensor given as
out= has its version raised, as by any operation in place."""
from __future__ import annotations

import ctypes as C
import struct

import torch
from torch.autograd import forward_ad

from .capi import MIBC_OK, MibcError, MibcNotSupported, lib

_TYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2, torch.int8: 3, torch.float8_e4m3fn: 4}
_FLOATS = (torch.float16, torch.bfloat16, torch.float32)
_QUANT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ATTN_END = -2147483648
SCALINGS = {"none": 0, "linear": 1, "base": 2, "by_parts": 3}

# the C structures, field by field (native sizes and alignment; checked against the library's by the tests)
_NORM_ARGS = struct.Struct("@6P6q5i2fi")
_ROPE_ARGS = struct.Struct("@2P2PPPq12q2q2i5if")
_ATTN_ARGS = struct.Struct("@4PP3PPPQ12q8i3i2fi")

_fns = None


# a number outside its field's range, or none at all
_BAD_FIELD = (struct.error, OverflowError)


def _entry():
    global _fns
    if _fns is None:
        L = lib()
        for f in (L.mibc_rms_norm, L.mibc_rope, L.mibc_attention):
            f.argtypes = [C.c_int, C.c_void_p, C.c_char_p]
            f.restype = C.c_int
        L.mibc_attention_workspace.argtypes = [C.c_char_p]
        L.mibc_attention_workspace.restype = C.c_uint64
        _fns = (L.mibc_rms_norm, L.mibc_rope, L.mibc_attention, L.mibc_attention_workspace)
    return _fns


def _check(rc: int, what: str) -> None:
    if rc != MIBC_OK:
        raise (MibcNotSupported if rc > 0 else MibcError)(f"{what}: {lib().mibc_last_error(None).decode()}")


_is_tracing, _modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack


def _infra(mode) -> bool:
    return getattr(mode, "_mode_key", None) is not None      # proxies, fake and functional tensors; counters and loggers have none


def _device(what: str, first: torch.Tensor, *others) -> int:
    """The device index all tensors share; refuses tensors elsewhere, gradients and transformations."""
    if _is_tracing() or (_modes() and any(map(_infra, torch.utils._python_dispatch._get_current_dispatch_mode_stack()))):
        raise MibcNotSupported(f"{what}: cannot be traced")
    if forward_ad._current_level >= 0:
        for t in (first, *others):
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise MibcNotSupported(f"{what}: forward only; tangents are not carried along")
    dev = first.device
    if dev.type != "cuda":
        raise MibcError(f"{what}: tensors must be on a HIP device (got {dev}); there is no CPU form")
    grad = first.requires_grad
    for t in others:
        if t is not None:
            if t.device != dev:
                raise MibcError(f"{what}: tensors on {dev} and {t.device}")
            grad = grad or t.requires_grad
    if grad and torch.is_grad_enabled():
        raise MibcNotSupported(f"{what}: forward only; call it under torch.no_grad() or on detached tensors")
    return dev.index


# the current stream's handle, without a Stream object around it where this torch offers that
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


def _ptr(what: str, t) -> int:
    """Address of an operand that may be left out (0)."""
    if t is None:
        return 0
    p = t.data_ptr()
    if p == 0 and t.numel():
        raise MibcNotSupported(f"{what}: a tensor without memory of its own")
    return p


def _written(t) -> None:
    """Raises the version of a tensor that the caller handed in to be written."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _row_stride(what: str, name: str, t: torch.Tensor, cols: int) -> int:
    """Elements from row to row of `t` seen as rows of `cols`."""
    st = t.stride()
    if st[-1] != 1 and cols > 1:
        raise MibcError(f"{what}: the last dimension of {name} must be contiguous")
    n = len(st)
    if n == 2:
        return st[0]
    if n == 1 or t.is_contiguous():
        return cols
    try:
        return t.view(-1, cols).stride(0)
    except RuntimeError:
        raise MibcError(f"{what}: the leading dimensions of {name} must be viewable as rows") from None


def _new(like: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(like) if like.is_contiguous() else like.new_empty(like.shape)


def _index32(what: str, name: str, t, n: int) -> int:
    """Pointer of a contiguous int32 tensor of n elements."""
    if t.dtype is not torch.int32 or t.shape != (n,) or not t.is_contiguous():
        raise MibcError(f"{what}: {name} must be a contiguous int32 tensor of {n} elements")
    return _ptr(what, t)


def rms_norm(x, weight=None, *, residual=None, alpha: float = 1.0, eps: float = 1e-5, quant=None, group: int = 0,
             return_sum: bool = False, out=None, sum_out=None):
    """h = x + alpha * residual; y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.

    x: f16, bf16 or f32, any shape with a contiguous last dimension; residual like x; weight [cols] f32 or of x's type.
    out and sum_out may be x or residual themselves; any other overlap of an output with an operand is refused, here and below.
    quant "int8" / "e4m3": the codes round(y / s) and the f32 scales s [..., groups], one per row (group 0) or per `group`
    (32, 64, 128) columns.  Returns y or (codes, scales), followed by h (x's type) if return_sum or sum_out is given."""
    dev = _device("rms_norm", x, weight, residual, out, sum_out)
    dtype, shape = x.dtype, x.shape
    if dtype not in _FLOATS:
        raise MibcNotSupported(f"rms_norm: type {dtype}")
    if not shape or shape[-1] == 0:
        raise MibcError("rms_norm: x needs a last dimension")
    cols = shape[-1]
    if cols == 1:      # the only width at which an imaginary part's view counts as contiguous
        for t in (x, residual, weight, out, sum_out):
            if t is not None and t.is_neg():
                raise MibcNotSupported("rms_norm: a tensor with its negation pending; resolve_neg() it")
    if weight is not None and (weight.shape != (cols,) or not (weight.dtype is torch.float32 or weight.dtype is dtype)
                               or not weight.is_contiguous()):
        raise MibcError(f"rms_norm: weight must be a contiguous [{cols}] tensor, f32 or {dtype}")
    if residual is not None and (residual.shape != shape or residual.dtype is not dtype):
        raise MibcError(f"rms_norm: residual must be {list(shape)} {dtype}")
    out_dtype, scale, groups = dtype, None, 0
    if quant is not None:
        if quant not in _QUANT:
            raise MibcError(f"rms_norm: quant must be None, 'int8' or 'e4m3', not {quant!r}")
        if group < 0 or (group and cols % group):
            raise MibcError("rms_norm: the columns must be a multiple of group")
        out_dtype, groups = _QUANT[quant], cols // group if group else 1
        scale = torch.empty(shape[:-1] + (groups,), dtype=torch.float32, device=x.device)
    xs = cols if x.is_contiguous() else _row_stride("rms_norm", "x", x, cols)
    rs = ss = os_ = cols
    out_given, sum_given = out is not None, sum_out is not None
    if residual is not None and not residual.is_contiguous():
        rs = _row_stride("rms_norm", "residual", residual, cols)
    if out is None:
        out = _new(x) if quant is None else torch.empty(shape, dtype=out_dtype, device=x.device)
    elif out.shape != shape or out.dtype is not out_dtype:
        raise MibcError(f"rms_norm: out must be {list(shape)} {out_dtype}")
    elif not out.is_contiguous():
        os_ = _row_stride("rms_norm", "out", out, cols)
    if sum_out is None:
        if return_sum:
            sum_out = _new(x)
    elif sum_out.shape != shape or sum_out.dtype is not dtype:
        raise MibcError(f"rms_norm: sum_out must be {list(shape)} {dtype}")
    elif not sum_out.is_contiguous():
        ss = _row_stride("rms_norm", "sum_out", sum_out, cols)
    try:
        args = _NORM_ARGS.pack(
            x.data_ptr(), 0 if residual is None else residual.data_ptr() or _ptr("rms_norm", residual),
            0 if weight is None else weight.data_ptr() or _ptr("rms_norm", weight),
            0 if sum_out is None else sum_out.data_ptr() or _ptr("rms_norm", sum_out), out.data_ptr(),
            0 if scale is None else scale.data_ptr(), x.numel() // cols,
            xs, rs, ss, os_, groups, cols, _TYPE[dtype], _TYPE[dtype if weight is None else weight.dtype], _TYPE[out_dtype], group, alpha, eps, 0)
    except _BAD_FIELD as e:
        raise MibcError(f"rms_norm: {e}") from None
    rc = (_fns or _entry())[0](dev, _stream(dev), args)
    if rc:
        _check(rc, "rms_norm")
    if out_given:
        _written(out)
    if sum_given:
        _written(sum_out)
    if scale is None:
        return out if sum_out is None else (out, sum_out)
    return (out, scale) if sum_out is None else (out, scale, sum_out)


def rope_frequencies(rot_dim: int, theta: float = 10000.0, *, scaling: str = "none", factor: float = 1.0,
                     original_length: float = 0.0, turns_low: float = 1.0, turns_high: float = 32.0, device="cuda"):
    """The f64 tensor [rot_dim / 2] of radians per position that `rope` takes (mibc_rope_frequencies).  scaling: "none",
    "linear" (positions squeezed by factor), "base" (a larger base: the slowest pair slows by factor), "by_parts" (pairs with
    at least turns_high turns over original_length stay, those with at most turns_low are squeezed, a ramp between)."""
    if scaling not in SCALINGS:
        raise MibcError(f"rope_frequencies: scaling must be one of {sorted(SCALINGS)}")
    f = torch.empty(max(rot_dim, 0) // 2, dtype=torch.float64)
    L = lib()
    L.mibc_rope_frequencies.argtypes = [C.c_int, C.c_int] + [C.c_double] * 5 + [C.c_void_p]
    _check(L.mibc_rope_frequencies(SCALINGS[scaling], rot_dim, theta, factor, original_length, turns_low, turns_high,
                                   f.data_ptr()), "rope_frequencies")
    return f.to(device)


def rope(q, k=None, *, freqs, positions=None, start: int = 0, interleaved: bool = False, amplitude: float = 1.0, out=None):
    """Rotary positions of q [batch, tokens, heads, head_dim] and, in the same launch, k (its own number of heads).

    freqs: f64 [rot_dim / 2] radians per position (rope_frequencies); columns behind rot_dim are copied.  positions: int32 or
    int64 [batch, tokens] or [tokens], or None for start, start + 1, ...; negated positions turn back.  out: None (new
    tensors), the tensors to write (one, or a pair), which may be q and k themselves.  Returns q, or (q, k)."""
    dev = _device("rope", q, k, freqs, positions)
    if q.dim() != 4:
        raise MibcError("rope: q must be [batch, tokens, heads, head_dim]")
    shape, dtype = q.shape, q.dtype
    b, t, h, d = shape
    if dtype not in _FLOATS:
        raise MibcNotSupported(f"rope: type {dtype}")
    if freqs.dtype is not torch.float64 or freqs.dim() != 1 or not freqs.is_contiguous():
        raise MibcError("rope: freqs must be a contiguous f64 tensor [rot_dim / 2]")
    where = 0
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise MibcError("rope: positions must be int32 or int64")
        if positions.shape != (b, t):
            if positions.shape != (t,):
                raise MibcError(f"rope: positions must be [{b}, {t}] or [{t}]")
            positions = positions.expand(b, t)
        positions = positions.contiguous()
        where = _ptr("rope", positions)
    if out is None:
        qo, ko = _new(q), None if k is None else _new(k)
    else:
        qo, ko = out if isinstance(out, (tuple, list)) else (out, None)
        if qo is None or (k is None) != (ko is None):
            raise MibcError("rope: out must be a tensor, or a pair where k is given")
        _device("rope", q, qo, ko)
        if qo.shape != shape or qo.dtype is not dtype:
            raise MibcError("rope: out must have the input's shape and type")
    qs, qos = q.stride(), qo.stride()
    plain = qs[3] == 1 and qos[3] == 1
    if k is None:
        kp, kop, kh, ks, kos = 0, 0, 0, (0, 0, 0, 1), (0, 0, 0, 1)
    else:
        kshape = k.shape
        if len(kshape) != 4 or kshape[0] != b or kshape[1] != t or kshape[3] != d or k.dtype is not dtype:
            raise MibcError("rope: k must be like q but for the number of heads")
        if out is not None and (ko.shape != kshape or ko.dtype is not dtype):
            raise MibcError("rope: out must have the input's shape and type")
        kp, kop, kh, ks, kos = k.data_ptr(), ko.data_ptr(), kshape[2], k.stride(), ko.stride()
        plain = plain and ks[3] == 1 and kos[3] == 1
    if not plain and d > 1:
        raise MibcError("rope: head_dim must be contiguous")
    try:
        args = _ROPE_ARGS.pack(q.data_ptr(), kp, qo.data_ptr(), kop, where, freqs.data_ptr(), start, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2],
                               qos[0], qos[1], qos[2], kos[0], kos[1], kos[2], b, t, h, kh, d, 2 * freqs.shape[0], _TYPE[dtype],
                               bool(interleaved), where != 0 and positions.dtype is torch.int64, amplitude)
    except _BAD_FIELD as e:
        raise MibcError(f"rope: {e}") from None
    rc = (_fns or _entry())[1](dev, _stream(dev), args)
    if rc:
        _check(rc, "rope")
    if out is not None:
        _written(qo)
        if k is not None:
            _written(ko)
    return qo if k is None else (qo, ko)


def attention(q, k, v, *, scale=None, causal: bool = False, window=(-1, -1), softcap: float = 0.0, slopes=None, k_len=None,
              prefix=None, doc_offsets=None, q_start=None, return_lse: bool = False, out=None):
    """softmax(scores) v over the keys a query sees; q [batch, q_tokens, heads, head_dim], k and v [batch, k_tokens, kv_heads,
    head_dim], f16 or bf16, heads a multiple of kv_heads.

    scores = scale * q.k (scale None: head_dim ** -0.5), softcap > 0: cap * tanh(scores / cap), slopes [heads] f32:
    - slope * |i - j|.  window (back, ahead): keys i - back .. i + ahead, negative = unlimited; causal = (-1, 0).  k_len
    [batch] int32: keys in use; query t stands at position k_len - q_tokens + t, or q_start + t.  prefix [batch] int32: that
    many first keys are seen by all.  doc_offsets [n + 1] int32 (batch 1, self attention): documents packed one after the
    other, each seeing itself only; prefix is then [n] and counts from the document's start.  A query that sees nothing gives
    zeros.  out: None or the tensor to write, which may be q itself.  f32 arithmetic; probabilities are rounded to the tensors' type
    before the product with v where a key head has more than 16 query rows.  Returns out like q, or (out, lse f32 [batch, heads, q_tokens])."""
    dev = _device("attention", q, k, v, slopes, k_len, prefix, doc_offsets, out)
    shape, kshape, dtype = q.shape, k.shape, q.dtype
    if len(shape) != 4 or len(kshape) != 4:
        raise MibcError("attention: q, k, v must be [batch, tokens, heads, head_dim]")
    b, n, h, d = shape
    if v.shape != kshape or kshape[0] != b or kshape[3] != d:
        raise MibcError("attention: k and v must be [batch, k_tokens, kv_heads, head_dim] like q")
    if k.dtype is not dtype or v.dtype is not dtype:
        raise MibcError("attention: q, k and v must be of one type")
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise MibcNotSupported(f"attention: type {dtype}")
    m, kh = kshape[1], kshape[2]
    back, ahead = window
    if causal:
        if back != -1 or ahead != -1:
            raise MibcError("attention: causal is window (-1, 0); give one of the two")
        ahead = 0
    back, ahead = max(-1, min(int(back), 0x7fffffff)), max(-1, min(int(ahead), 0x7fffffff))
    out_given = out is not None
    if out is None:
        out = _new(q)
    elif out.shape != shape or out.dtype is not dtype:
        raise MibcError("attention: out must have q's shape and type")
    qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), out.stride()
    if qs[3] != 1 or os_[3] != 1 or ((ks[3] != 1 or vs[3] != 1) and m and kh):
        raise MibcError("attention: head_dim must be contiguous")
    lens = pre = offs = slope = docs = 0
    if slopes is not None:
        if slopes.dtype is not torch.float32 or slopes.shape != (h,) or not slopes.is_contiguous():
            raise MibcError(f"attention: slopes must be a contiguous f32 tensor [{h}]")
        slope = _ptr("attention", slopes)
    if doc_offsets is not None:
        docs = doc_offsets.shape[0] - 1 if doc_offsets.dim() == 1 else -1
        if docs < 0:
            raise MibcError("attention: doc_offsets must be [n + 1]")
        offs = _index32("attention", "doc_offsets", doc_offsets, docs + 1)
    if k_len is not None:
        lens = _index32("attention", "k_len", k_len, b)
    if prefix is not None:
        pre = _index32("attention", "prefix", prefix, docs if doc_offsets is not None else b)
    if q_start is None:
        q_start = ATTN_END
    elif not -(1 << 28) <= q_start <= 1 << 28:
        raise MibcNotSupported("attention: q_start beyond 2^28")
    lse = torch.empty((b, h, n), dtype=torch.float32, device=q.device) if return_lse else None
    head = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), lens, pre, offs, slope)
    tail = (qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], os_[0], os_[1], os_[2], b, h, kh, n, m, d, docs, _TYPE[dtype],
            back, ahead, q_start, max(d, 1) ** -0.5 if scale is None else scale, softcap, 0)
    _, _, run, workspace = _fns or _entry()
    try:
        args = _ATTN_ARGS.pack(*head, 0, 0, *tail)
    except _BAD_FIELD as e:
        raise MibcError(f"attention: {e}") from None
    need = workspace(args) if m >= 512 else 0      # fewer keys are never split
    if need:
        room = torch.empty(need, dtype=torch.uint8, device=q.device)
        args = _ATTN_ARGS.pack(*head, room.data_ptr(), need, *tail)
    rc = run(dev, _stream(dev), args)
    if rc:
        _check(rc, "attention")
    if out_given:
        _written(out)
    return out if lse is None else (out, lse)
