"""Fused ops with the reference's signatures (``hydra.kernels``: hydra/kernels/__init__.py:13-38), running as
hand-written sm_100a CUDA kernels behind PyTorch-registered custom ops (``torch.ops.hydra_b200.*``).

    fused_rope(x, cos, sin)                         hydra/kernels/fused_ops.py:240-306
    fused_qk_norm(q, k, scale, temperature=1.0)     hydra/kernels/fused_ops.py:474-493
    fused_swiglu(gate, up)                          hydra/kernels/fused_ops.py:808-883
    fused_rms_norm(x, weight, eps=1e-6)             hydra/kernels/fused_ops.py:1114-1132
    fused_qk_norm_rope(q, k, cos, sin, ...)         the norm and the rotation in one pass (no counterpart)
    set_use_triton_kernels / get_kernel_status      hydra/kernels/fused_ops.py:123-166

Same argument meaning and result shapes/dtypes as the reference.  Differences, by design: tensors must live on
a CUDA device (a CPU tensor raises instead of silently taking a PyTorch path), the ops are forward-only
(inference), and arithmetic is fp32 inside the kernels whatever the storage dtype.
"""
from __future__ import annotations

from contextlib import nullcontext
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

Tensor = torch.Tensor

try:   # empty_strided on the current CUDA device by its shortest way: half the 1.5 us of torch.empty, several times a call
    _empty_strided = torch._C._dynamo.guards._empty_strided_cuda   # (size, stride: plain tuples; dtype)
except AttributeError:
    def _empty_strided(size, stride, dtype):
        return torch.empty_strided(size, stride, dtype=dtype, device="cuda")

# Flags the reference exports.  No Triton is involved here; the names are kept so callers that read them
# keep working, and they report whether the CUDA path is active.
TRITON_AVAILABLE = False
USE_TRITON_KERNELS = False
USE_FUSED_ROPE = True
USE_FUSED_QK_NORM = True
USE_FUSED_SWIGLU = True
USE_FUSED_RMS_NORM = True
# fused_qk_norm formula: "normalize" = x / max(||x||, 1e-12) (the reference's PyTorch path and what the
# attention module computes); "rsqrt" = x * rsqrt(sum x^2 + 1e-8) (the reference's device kernel).
QK_NORM_MODE = "rsqrt"

_DTYPES = {torch.float32: _lib.HB200_F32, torch.bfloat16: _lib.HB200_BF16, torch.float16: _lib.HB200_F16}


def _dtype_code(t: Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise TypeError(f"hydra_b200 kernels support float32, bfloat16 and float16, got {t.dtype}") from None


def _require_cuda(*ts: Tensor) -> torch.device:
    index = ts[0].get_device()                # -1 on the CPU
    for t in ts:
        if t.get_device() != index or index < 0:
            for u in ts:
                if not u.is_cuda:
                    raise RuntimeError("hydra_b200 kernels run on CUDA tensors only (there is no CPU fallback); "
                                       f"got a tensor on {u.device}")
            raise RuntimeError(f"hydra_b200: tensors on different devices ({ts[0].device} and {t.device})")
    return ts[0].device


_HERE = nullcontext()


def _on(dev: torch.device):
    """Context that makes `dev` the current CUDA device (kernels launch on the current device)."""
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream(dev: torch.device) -> int:
    """The device's current stream as the handle that the C entries take (its raw form: building the torch.cuda.Stream
    object around it costs 2 us a call)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


# ----------------------------------------------------------------------------- custom ops
@torch.library.custom_op("hydra_b200::fused_rms_norm", mutates_args=())
def _rms_norm_op(x: Tensor, weight: Tensor, eps: float) -> Tensor:
    dev = _require_cuda(x, weight)
    dim = x.shape[-1]
    if weight.numel() != dim:
        raise ValueError(f"fused_rms_norm: weight has {weight.numel()} elements, last dim is {dim}")
    xc = x.contiguous()
    w = weight.contiguous()
    if w.dtype != torch.float32 and w.dtype != x.dtype:
        w = w.float()
    y = torch.empty_like(xc)
    rows = xc.numel() // dim if dim else 0
    if rows == 0:
        return y
    with _on(dev):
        _lib.check(_lib.lib().hb200_rms_norm(xc.data_ptr(), w.data_ptr(), y.data_ptr(), rows, dim, float(eps),
                                             _dtype_code(xc), _dtype_code(w), _stream(dev)), "fused_rms_norm")
    return y


@_rms_norm_op.register_fake
def _(x, weight, eps):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


@torch.library.custom_op("hydra_b200::fused_rope", mutates_args=())
def _rope_op(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    dev = _require_cuda(x, cos, sin)
    if x.dim() != 4:
        raise ValueError(f"fused_rope: x must be [B, H, S, head_dim], got {tuple(x.shape)}")
    B, H, S, hd = x.shape
    if hd % 2:
        raise ValueError("fused_rope: head_dim must be even")
    if cos.dim() == 4:
        cos, sin = cos[0, 0], sin[0, 0]
    if cos.shape[0] < S or cos.shape[1] != hd // 2 or sin.shape != cos.shape:
        raise ValueError(f"fused_rope: tables {tuple(cos.shape)} do not cover S={S}, head_dim/2={hd // 2}")
    cos = cos.float().contiguous() if (cos.dtype != torch.float32 or cos.stride(1) != 1) else cos
    sin = sin.float().contiguous() if (sin.dtype != torch.float32 or sin.stride(1) != 1) else sin
    if x.stride(3) != 1 and x.numel() > 0:
        x = x.contiguous()
    y = torch.empty((B, H, S, hd), dtype=x.dtype, device=x.device)
    if y.numel() == 0:
        return y
    with _on(dev):
        _lib.check(_lib.lib().hb200_rope(x.data_ptr(), cos.data_ptr(), sin.data_ptr(), y.data_ptr(), B, H, S, hd,
                                         x.stride(0), x.stride(1), x.stride(2), cos.stride(0), _dtype_code(x),
                                         _stream(dev)), "fused_rope")
    return y


@_rope_op.register_fake
def _(x, cos, sin):
    return torch.empty(x.shape, dtype=x.dtype, device=x.device)


@torch.library.custom_op("hydra_b200::fused_qk_norm", mutates_args=())
def _qk_norm_op(q: Tensor, k: Tensor, scale: float, temperature: float, mode: int) -> Tuple[Tensor, Tensor]:
    dev = _require_cuda(q, k)
    if q.dtype != k.dtype or q.shape[-1] != k.shape[-1]:
        raise ValueError("fused_qk_norm: q and k must share dtype and head_dim")
    hd = q.shape[-1]
    qc, kc = q.contiguous(), k.contiguous()
    qo, ko = torch.empty_like(qc), torch.empty_like(kc)
    if qc.numel() + kc.numel() == 0:
        return qo, ko
    if qc.numel() == 0 or kc.numel() == 0:   # an empty tensor has a null data pointer: give the kernel a valid one
        dummy = torch.zeros(hd, dtype=q.dtype, device=q.device)
        qc = qc if qc.numel() else dummy
        kc = kc if kc.numel() else dummy
    with _on(dev):
        _lib.check(_lib.lib().hb200_qk_norm(qc.data_ptr(), kc.data_ptr(), qo.data_ptr(), ko.data_ptr(),
                                            qo.numel() // hd, ko.numel() // hd, hd, float(scale), float(temperature),
                                            int(mode), _dtype_code(qc), _stream(dev)), "fused_qk_norm")
    return qo, ko


@_qk_norm_op.register_fake
def _(q, k, scale, temperature, mode):
    return (torch.empty_like(q, memory_format=torch.contiguous_format),
            torch.empty_like(k, memory_format=torch.contiguous_format))


@torch.library.custom_op("hydra_b200::fused_swiglu", mutates_args=())
def _swiglu_op(gate: Tensor, up: Tensor) -> Tensor:
    dev = _require_cuda(gate, up)
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise ValueError("fused_swiglu: gate and up must have the same shape and dtype")
    cols = gate.shape[-1]
    out = torch.empty(gate.shape, dtype=gate.dtype, device=gate.device)
    if gate.numel() == 0:
        return out

    def rows_view(t: Tensor):
        """(tensor, leading dimension) if t is a [rows, cols] view with one row stride, else a copy."""
        if t.stride(-1) == 1:
            t2 = t.reshape(-1, cols) if t.dim() != 2 else t
            if t2.data_ptr() == t.data_ptr() and (t2.shape[0] == 1 or t2.stride(0) >= cols):
                return t2, (t2.stride(0) if t2.shape[0] > 1 else cols)
        c = t.contiguous().view(-1, cols)
        return c, cols

    g2, ldg = rows_view(gate)
    u2, ldu = rows_view(up)
    with _on(dev):
        _lib.check(_lib.lib().hb200_swiglu(g2.data_ptr(), u2.data_ptr(), out.data_ptr(), g2.shape[0], cols, ldg, ldu,
                                           _dtype_code(gate), _stream(dev)), "fused_swiglu")
    return out


@_swiglu_op.register_fake
def _(gate, up):
    return torch.empty(gate.shape, dtype=gate.dtype, device=gate.device)


# ----------------------------------------------------------------------------- reference-signature wrappers
def fused_rope(x: Tensor, cos: Tensor, sin: Tensor) -> Tensor:
    """Rotary embedding, interleaved pairs.  x [B, n_heads, S, head_dim] (may be a strided view);
    cos/sin [1, 1, max_seq, head_dim//2] or [S, head_dim//2].  Returns a contiguous tensor of x's dtype."""
    return _rope_op(x, cos, sin)


def fused_qk_norm(q: Tensor, k: Tensor, scale: float, temperature: float = 1.0) -> Tuple[Tensor, Tensor]:
    """L2-normalise q [B,Hq,S,hd] and k [B,Hkv,S,hd] over the last dim and scale (k also by temperature)."""
    return _qk_norm_op(q, k, float(scale), float(temperature), 0 if QK_NORM_MODE == "normalize" else 1)


def fused_swiglu(gate: Tensor, up: Tensor) -> Tensor:
    """silu(gate) * up; inputs may be the two chunk views of one gate_up projection."""
    return _swiglu_op(gate, up)


def fused_rms_norm(x: Tensor, weight: Tensor, eps: float = 1e-6) -> Tensor:
    """x * rsqrt(mean(x^2, -1) + eps) * weight."""
    return _rms_norm_op(x, weight, float(eps))


_INT32_MAX = 0x7fffffff


def _past_int32(what: str, *sizes: int) -> ValueError:
    """For sizes that the C entries take as 32 bits: ctypes would cut a larger one to its low 32."""
    return ValueError(f"{what}: a size of {max(sizes)} (up to 2^31 - 1)")


def _overlap(a: Tensor, b: Tensor) -> bool:
    """Whether the memory that one tensor reaches over, from its first byte to its last, meets the other's."""
    def reach(t):
        lo = t.data_ptr()
        return lo, lo + (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))) * t.element_size() if t.numel() else lo
    (a0, a1), (b0, b1) = reach(a), reach(b)
    return a0 < b1 and b0 < a1 and a0 < a1 and b0 < b1


def _refuse_autograd(what: str, *ts: Optional[Tensor]) -> None:
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what} is inference only: an input requires grad (wrap the call in torch.no_grad())")
    if forward_ad._current_level >= 0:
        _refuse_tangents(what, *ts)


def _refuse_tangents(what: str, *ts: Optional[Tensor]) -> None:
    """(Called within forward_ad.dual_level() only: a look at a tensor costs 0.3 us.)"""
    for t in ts:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} is inference only: an input carries a forward-mode tangent")


def _fp32(what: str, t: Tensor, n: int, dev: torch.device) -> Tensor:
    if t.get_device() != dev.index or t.numel() != n:
        raise ValueError(f"{what}: q_weight and k_weight must have {n} elements on {dev}, got {tuple(t.shape)} on {t.device}")
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


def _qk_norm_rope(what: str, dev: torch.device, q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Optional[Tensor],
                  q_weight: Optional[Tensor], k_weight: Optional[Tensor], norm: Optional[str], eps: float, q_scale: float,
                  k_scale: float, layout: str, v: Optional[Tensor] = None, slots: Optional[Tensor] = None, cache=None):
    """The call behind fused_qk_norm_rope and paged_append: q, k (v) [T, H, hd] or [B, H, S, hd]."""
    _refuse_autograd(what, q, k, v, cos, sin, q_weight, k_weight)
    try:
        norm_code, layout_code = _lib.QK_NORMS[norm], _lib.ROPE_LAYOUTS[layout]
    except KeyError:
        raise ValueError(f"{what}: norm must be 'rms', 'l2' or None and layout 'interleaved' or 'half', got {norm!r} and {layout!r}") from None
    dtype, torch_dtype, shape, k_shape = _dtype_code(q), q.dtype, q.shape, k.shape
    hd = shape[-1]
    if q.numel() > _INT32_MAX or k.numel() > _INT32_MAX:
        if max(*shape, *k_shape) > _INT32_MAX:
            raise _past_int32(what, *shape, *k_shape)
    if cos.dim() == 4 and cos.shape[:2] == (1, 1) and sin.shape == cos.shape:
        cos, sin = cos[0, 0], sin[0, 0]
    table = cos.shape
    if len(table) != 2 or sin.shape != table or 2 * table[1] > hd:
        raise ValueError(f"{what}: cos and sin must be [rows, rotated / 2] or [1, 1, rows, rotated / 2] with rotated <= {hd}, got {tuple(table)} and {tuple(sin.shape)}")
    table_rows, half = table
    table_ld, unit = cos.stride()
    if unit != 1 or table_ld < half or cos.dtype != torch.float32 or sin.dtype != torch.float32 or sin.stride() != (table_ld, 1):
        cos, sin = cos.float().contiguous(), sin.float().contiguous()
        table_ld = half
    qs, ks, vs = q.stride(), k.stride(), (0, 0, 1) if v is None else v.stride()
    if qs[-1] != 1 or ks[-1] != 1 or vs[-1] != 1:
        q, k, v = q.contiguous(), k.contiguous(), None if v is None else v.contiguous()
        qs, ks, vs = q.stride(), k.stride(), (0, 0, 1) if v is None else v.stride()
    # strides of batch, token and head; the results are contiguous
    if len(shape) == 3:
        S, Hq, _ = shape
        B, Hkv = 1, k_shape[1]
        new = (S, Hq, hd), (Hq * hd, hd, 1), (S, Hkv, hd), (Hkv * hd, hd, 1)
        strides = (0, qs[0], qs[1], 0, ks[0], ks[1], 0, vs[0], vs[1], 0, Hq * hd, hd, 0, Hkv * hd, hd)
    else:
        B, Hq, S, _ = shape
        Hkv = k_shape[1]
        new = (B, Hq, S, hd), (Hq * S * hd, S * hd, hd, 1), (B, Hkv, S, hd), (Hkv * S * hd, S * hd, hd, 1)
        strides = (qs[0], qs[2], qs[1], ks[0], ks[2], ks[1], 0, 0, 0, Hq * S * hd, hd, S * hd, Hkv * S * hd, hd, S * hd)
    where, where_64, where_stride = None, 0, 0
    if positions is not None:
        if positions.dtype == torch.int64:
            where_64 = 1
        elif positions.dtype != torch.int32:
            raise TypeError(f"{what}: positions must be int32 or int64, got {positions.dtype}")
        where_shape = positions.shape
        if where_shape != (S,) and where_shape != (B, S):
            raise ValueError(f"{what}: positions {tuple(where_shape)} for {B} x {S} tokens")
        where_strides = positions.stride()
        if where_strides[-1] != 1 and S > 1:
            positions = positions.contiguous()
            where_strides = positions.stride()
        where, where_stride = positions.data_ptr(), where_strides[0] if len(where_strides) == 2 else 0
    elif table_rows < S:
        raise ValueError(f"{what}: tables {tuple(table)} do not cover {S} positions")
    if q_weight is not None:
        q_weight = _fp32(what, q_weight, hd, dev)
    if k_weight is not None:
        k_weight = _fp32(what, k_weight, hd, dev)
    with _on(dev):
        q_out = _empty_strided(new[0], new[1], torch_dtype)
        k_out = _empty_strided(new[2], new[3], torch_dtype) if cache is None else None
        if (Hq + Hkv) * B * S * hd > 0:
            args = _lib.QkNormRopeArgs(        # in the order of the struct
                q.data_ptr(), k.data_ptr(), None if v is None else v.data_ptr(), q_out.data_ptr(), None if k_out is None else k_out.data_ptr(),
                None if slots is None else slots.data_ptr(), where, cos.data_ptr(), sin.data_ptr(),
                None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(), *strides, where_stride,
                table_rows, table_ld, where_64, B, S, Hq, Hkv, hd, 2 * half, layout_code, norm_code, dtype, eps, q_scale, k_scale)
            _lib.check(_lib.lib().hb200_qk_norm_rope(args, cache, _stream(dev)), what)
    return q_out, k_out


def fused_qk_norm_rope(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, positions: Optional[Tensor] = None, *,
                       q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None, norm: Optional[str] = "rms",
                       eps: float = 1e-6, q_scale: float = 1.0, k_scale: float = 1.0,
                       layout: str = "interleaved") -> Tuple[Tensor, Tensor]:
    """Norm of every query and key head and the position rotation, in one pass (``hb200_qk_norm_rope``; the reference norms
    and rotates in two, hydra/attention/backends/ccgqa/attention.py:257-266): 32 bits inside, rounded once.

    q [B, Hq, S, hd] and k [B, Hkv, S, hd], or packed tokens [T, Hq, hd] and [T, Hkv, hd]; strided views are read in place.
    ``norm``: "rms" (``x * rsqrt(mean(x^2) + eps)``), "l2" (``x * rsqrt(sum(x^2) + eps)``) or None; then times the weight [hd]
    of q or k (if given) and ``q_scale`` / ``k_scale`` (a softmax scale, CCGQA's key temperature).  cos, sin [rows, rot / 2] (or
    [1, 1, rows, rot / 2]) turn the first ``rot <= hd`` values of a head, whatever frequencies the tables were built with
    (scaled ones for long contexts); ``layout`` "interleaved" pairs values (2i, 2i + 1), "half" (i, i + rot / 2).  ``positions``
    int32 or int64 [S], [B, S] or [T] are table rows (default 0 .. S - 1): a negative one marks padding (zeros), one beyond
    the tables gives NaN.  hd up to 256.  Returns contiguous q and k."""
    dev = _require_cuda(q, k, cos, sin, *(() if positions is None else (positions,)))
    a, b = q.shape, k.shape
    if len(a) != len(b) or len(a) not in (3, 4) or a[-1] != b[-1] or a[0] != b[0] or (len(a) == 4 and a[2] != b[2]) or q.dtype != k.dtype:
        raise ValueError("fused_qk_norm_rope: q [B, Hq, S, hd] and k [B, Hkv, S, hd] (or [T, Hq, hd] and [T, Hkv, hd]) of one dtype "
                         f"are wanted, got {tuple(q.shape)} {q.dtype} and {tuple(k.shape)} {k.dtype}")
    return _qk_norm_rope("fused_qk_norm_rope", dev, q, k, cos, sin, positions, q_weight, k_weight, norm, eps, q_scale, k_scale, layout)


def set_use_triton_kernels(enabled: bool) -> None:
    """Kept for API compatibility (hydra/kernels/fused_ops.py:123-148).  There is exactly one implementation
    here and it has no Triton or PyTorch alternative, so the switch only records the request."""
    global USE_TRITON_KERNELS
    USE_TRITON_KERNELS = bool(enabled) and TRITON_AVAILABLE


def get_kernel_status() -> dict:
    """Same keys as the reference (hydra/kernels/fused_ops.py:151-166) plus a ``backend`` entry."""
    return {
        "triton_available": TRITON_AVAILABLE,
        "triton_version": "N/A",
        "use_triton_kernels": USE_TRITON_KERNELS,
        "fused_rope": USE_FUSED_ROPE,
        "fused_qk_norm": USE_FUSED_QK_NORM,
        "fused_qk_norm_backward": False,
        "fused_swiglu": USE_FUSED_SWIGLU,
        "fused_swiglu_backward": False,
        "fused_rms_norm": USE_FUSED_RMS_NORM,
        "fused_rms_norm_backward": False,
        "liger_ce_available": False,
        "use_liger_ce": False,
        "backend": "hydra_b200 sm_100a CUDA (C ABI v%d)" % _lib.lib().hb200_version(),
    }


__all__ = [
    "fused_rope", "fused_qk_norm", "fused_qk_norm_rope", "fused_swiglu", "fused_rms_norm", "set_use_triton_kernels",
    "get_kernel_status", "TRITON_AVAILABLE", "USE_TRITON_KERNELS", "USE_FUSED_ROPE", "USE_FUSED_QK_NORM",
    "USE_FUSED_SWIGLU", "USE_FUSED_RMS_NORM",
]
