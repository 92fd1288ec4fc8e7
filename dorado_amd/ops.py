"""Transformer-layer operators on torch tensors: the Python side of mibc_rms_norm, mibc_rope and mibc_attention
(include/mibc.h, which states the formulas).

Tensors live on one HIP device; the work goes to torch's current stream of that device and nothing is synchronised.  New
outputs and the workspace of a split attention come from torch's caching allocator, so a call can be captured into a graph.
There is no CPU form: a tensor elsewhere raises.  Forward only; no autograd graph is recorded, so inputs that require a
gradient are refused while gradients are being recorded."""
from __future__ import annotations

import ctypes as C
import struct

import torch

from .capi import MIBC_OK, MibcError, MibcNotSupported, lib

_TYPE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2, torch.int8: 3, torch.float8_e4m3fn: 4}
_QUANT = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
ATTN_END = -2147483648
SCALINGS = {"none": 0, "linear": 1, "base": 2, "by_parts": 3}

# the C structures, field by field (native sizes and alignment; checked against the library's by the tests)
_NORM_ARGS = struct.Struct("@6P6q5i2fi")
_ROPE_ARGS = struct.Struct("@2P2PPPq12q2q2i5if")
_ATTN_ARGS = struct.Struct("@4PP3PPPQ12q8i3i2fi")

_fns = None


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


def _device(what: str, first: torch.Tensor, *others) -> int:
    """The device index all tensors share; refuses tensors elsewhere and gradients."""
    dev = first.device
    if dev.type != "cuda":
        raise MibcError(f"{what}: tensors must be on a HIP device (got {dev}); there is no CPU form")
    grad = torch.is_grad_enabled()
    for t in (first,) + others:
        if t is None:
            continue
        if t.device != dev:
            raise MibcError(f"{what}: tensors on {dev} and {t.device}")
        if grad and t.requires_grad:
            raise MibcNotSupported(f"{what}: forward only; call it under torch.no_grad() or on detached tensors")
    return dev.index


def _stream(device: int) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _index32(what: str, name: str, t, n: int):
    """Pointer of a contiguous int32 tensor of n elements, 0 for None."""
    if t is None:
        return 0
    if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise MibcError(f"{what}: {name} must be a contiguous int32 tensor of {n} elements")
    return t.data_ptr()


def rms_norm(x, weight=None, *, residual=None, alpha: float = 1.0, eps: float = 1e-5, quant=None, group: int = 0,
             return_sum: bool = False, out=None, sum_out=None):
    """h = x + alpha * residual; y = h / sqrt(mean(h^2) + eps) * weight over the last dimension.

    x: f16, bf16 or f32, any shape with a contiguous last dimension; residual like x; weight [cols] f32 or of x's type.
    quant "int8" / "e4m3": the codes round(y / s) and the f32 scales s [..., groups], one per row (group 0) or per `group`
    (32, 64, 128) columns.  Returns y or (codes, scales), followed by h (x's type) if return_sum or sum_out is given."""
    dev = _device("rms_norm", x, weight, residual, out, sum_out)
    if x.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise MibcNotSupported(f"rms_norm: type {x.dtype}")
    if quant is not None and quant not in _QUANT:
        raise MibcError(f"rms_norm: quant must be None, 'int8' or 'e4m3', not {quant!r}")
    if x.dim() < 1 or x.shape[-1] == 0:
        raise MibcError("rms_norm: x needs a last dimension")
    shape, cols = x.shape, x.shape[-1]
    if weight is not None and (weight.dim() != 1 or weight.shape[0] != cols or weight.dtype not in (torch.float32, x.dtype)
                               or weight.stride(0) not in (1,) and cols > 1):
        raise MibcError(f"rms_norm: weight must be a contiguous [{cols}] tensor, f32 or {x.dtype}")

    def rows_of(t, name, dtype, width=cols):
        """(tensor, row stride) of `t` seen as rows."""
        if t.shape[:-1] != shape[:-1] or t.shape[-1] != width or t.dtype is not dtype:
            raise MibcError(f"rms_norm: {name} must be {list(shape[:-1]) + [width]} {dtype}")
        if width > 1 and t.stride(-1) != 1:
            raise MibcError(f"rms_norm: the last dimension of {name} must be contiguous")
        if t.dim() == 1:
            return t, width
        if t.dim() > 2:
            if t.is_contiguous():
                return t, width
            try:
                t = t.view(-1, width)
            except RuntimeError:
                raise MibcError(f"rms_norm: the leading dimensions of {name} must be viewable as rows") from None
        return t, t.stride(0)

    x2, xs = rows_of(x, "x", x.dtype)
    r2, rs = (None, 0) if residual is None else rows_of(residual, "residual", x.dtype)
    out_dtype = x.dtype if quant is None else _QUANT[quant]
    if out is None:
        out = torch.empty(shape, dtype=out_dtype, device=x.device)
    o2, os_ = rows_of(out, "out", out_dtype)
    if sum_out is None and return_sum:
        sum_out = torch.empty(shape, dtype=x.dtype, device=x.device)
    s2, ss = (None, 0) if sum_out is None else rows_of(sum_out, "sum_out", x.dtype)
    scale, groups = None, 0
    if quant is not None:
        if group and cols % group:
            raise MibcError("rms_norm: the columns must be a multiple of group")
        groups = cols // group if group else 1
        scale = torch.empty(shape[:-1] + (groups,), dtype=torch.float32, device=x.device)
    args = _NORM_ARGS.pack(x2.data_ptr(), 0 if r2 is None else r2.data_ptr(), 0 if weight is None else weight.data_ptr(),
                           0 if s2 is None else s2.data_ptr(), o2.data_ptr(), 0 if scale is None else scale.data_ptr(),
                           x.numel() // cols, xs, rs, ss, os_, groups, cols, _TYPE[x.dtype],
                           _TYPE[x.dtype if weight is None else weight.dtype], _TYPE[out_dtype], group, alpha, eps, 0)
    _check(_entry()[0](dev, _stream(dev), args), "rms_norm")
    if scale is None and sum_out is None:
        return out
    return (out,) + (() if scale is None else (scale,)) + (() if sum_out is None else (sum_out,))


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
    b, t, h, d = q.shape
    if q.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise MibcNotSupported(f"rope: type {q.dtype}")
    if k is not None and (k.dim() != 4 or k.shape[0] != b or k.shape[1] != t or k.shape[3] != d or k.dtype is not q.dtype):
        raise MibcError("rope: k must be like q but for the number of heads")
    if freqs.dtype is not torch.float64 or freqs.dim() != 1 or (freqs.shape[0] > 1 and freqs.stride(0) != 1):
        raise MibcError("rope: freqs must be a contiguous f64 tensor [rot_dim / 2]")
    rot = 2 * freqs.shape[0]
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise MibcError("rope: positions must be int32 or int64")
        if positions.shape == (t,) and b != 1:
            positions = positions.expand(b, t)
        elif positions.shape not in ((b, t), (t,)):
            raise MibcError(f"rope: positions must be [{b}, {t}] or [{t}]")
        positions = positions.contiguous()
    outs = out if isinstance(out, (tuple, list)) else (out, None)
    if out is not None and k is not None and (len(outs) != 2 or outs[1] is None):
        raise MibcError("rope: out must be a pair where k is given")
    if out is not None:
        _device("rope", q, *outs)
    qo = torch.empty((b, t, h, d), dtype=q.dtype, device=q.device) if out is None else outs[0]
    ko = None if k is None else torch.empty(k.shape, dtype=q.dtype, device=q.device) if out is None else outs[1]
    for x, o in ((q, qo), (k, ko)):
        if x is None:
            continue
        if o.shape != x.shape or o.dtype is not x.dtype:
            raise MibcError("rope: out must have the input's shape and type")
        if d > 1 and (x.stride(3) != 1 or o.stride(3) != 1):
            raise MibcError("rope: head_dim must be contiguous")
    ks, kos = (0, 0, 0) if k is None else k.stride()[:3], (0, 0, 0) if k is None else ko.stride()[:3]
    args = _ROPE_ARGS.pack(q.data_ptr(), 0 if k is None else k.data_ptr(), qo.data_ptr(), 0 if k is None else ko.data_ptr(),
                           0 if positions is None else positions.data_ptr(), freqs.data_ptr(), start, *q.stride()[:3], *ks,
                           *qo.stride()[:3], *kos, b, t, h, 0 if k is None else k.shape[2], d, rot, _TYPE[q.dtype],
                           int(interleaved), int(positions is not None and positions.dtype is torch.int64), amplitude)
    _check(_entry()[1](dev, _stream(dev), args), "rope")
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
    zeros.  Returns out like q, or (out, lse f32 [batch, heads, q_tokens])."""
    dev = _device("attention", q, k, v, slopes, k_len, prefix, doc_offsets, out)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise MibcError("attention: q, k, v must be [batch, tokens, heads, head_dim]")
    b, n, h, d = q.shape
    m, kh = k.shape[1], k.shape[2]
    if k.shape != v.shape or k.shape[0] != b or k.shape[3] != d:
        raise MibcError("attention: k and v must be [batch, k_tokens, kv_heads, head_dim] like q")
    if k.dtype is not q.dtype or v.dtype is not q.dtype:
        raise MibcError("attention: q, k and v must be of one type")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise MibcNotSupported(f"attention: type {q.dtype}")
    if causal:
        if tuple(window) != (-1, -1):
            raise MibcError("attention: causal is window (-1, 0); give one of the two")
        window = (-1, 0)
    if out is None:
        out = torch.empty((b, n, h, d), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype is not q.dtype:
        raise MibcError("attention: out must have q's shape and type")
    qs, ks, vs, os_ = q.stride(), k.stride(), v.stride(), out.stride()
    if qs[3] != 1 or os_[3] != 1 or (m and kh and (ks[3] != 1 or vs[3] != 1)):
        raise MibcError("attention: head_dim must be contiguous")
    if slopes is not None and (slopes.dtype is not torch.float32 or slopes.shape != (h,) or not slopes.is_contiguous()):
        raise MibcError(f"attention: slopes must be a contiguous f32 tensor [{h}]")
    docs = 0
    if doc_offsets is not None:
        docs = doc_offsets.shape[0] - 1 if doc_offsets.dim() == 1 else -1
        if docs < 0:
            raise MibcError("attention: doc_offsets must be [n + 1]")
    lens = _index32("attention", "k_len", k_len, b)
    pre = _index32("attention", "prefix", prefix, docs if doc_offsets is not None else b)
    offs = _index32("attention", "doc_offsets", doc_offsets, docs + 1)
    if q_start is None:
        q_start = ATTN_END
    elif not -(1 << 28) <= q_start <= 1 << 28:
        raise MibcNotSupported("attention: q_start beyond 2^28")
    limits = [max(-1, min(int(w), (1 << 31) - 1)) for w in window]
    lse = torch.empty((b, h, n), dtype=torch.float32, device=q.device) if return_lse else None

    def pack(ws, nbytes):
        return _ATTN_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(), lens,
                               pre, offs, 0 if slopes is None else slopes.data_ptr(), ws, nbytes, qs[0], qs[1], qs[2], ks[0], ks[1],
                               ks[2], vs[0], vs[1], vs[2], os_[0], os_[1], os_[2], b, h, kh, n, m, d, docs, _TYPE[q.dtype],
                               limits[0], limits[1], q_start, d ** -0.5 if scale is None else scale, softcap, 0)

    _, _, run, workspace = _entry()
    args = pack(0, 0)
    need = workspace(args)
    if need:
        room = torch.empty(need, dtype=torch.uint8, device=q.device)
        args = pack(room.data_ptr(), need)
    _check(run(dev, _stream(dev), args), "attention")
    return out if lse is None else (out, lse)
