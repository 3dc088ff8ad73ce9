"""Next-token sampling on the device (``hb200_sample_rows``): the sampler of the reference's generation helper
(diagnostics/eval_checkpoint.py:133-155: temperature, top-k, top-p, one draw) for bf16 logit rows.  The reference draws
with ``torch.multinomial``; here the draw is the inverse CDF at one uniform number per row, so a result is reproducible
from (logits, uniform)."""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch
from torch import Tensor

from . import _lib, kernels


def cross_entropy_rows(logits: Tensor, targets: Tensor, vocab: Optional[int] = None, ignore_index: int = -100) -> Tensor:
    """Per-row negative log-likelihood (``hb200_cross_entropy_rows``): logits bf16 [N, ld] on a CUDA device (row
    stride ``logits.stride(0)``, the first ``vocab`` columns count), targets int64 [N] -> fp32 [N], 0 where the target
    is ``ignore_index``.  Summed or averaged it is ``F.cross_entropy`` of the reference's evaluation helper
    (diagnostics/eval_checkpoint.py:168-193), computed in fp32 from the bf16 logits."""
    if not logits.is_cuda or targets.device != logits.device:
        raise RuntimeError("cross_entropy_rows needs CUDA tensors on one device (there is no CPU fallback)")
    if logits.dtype != torch.bfloat16 or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("cross_entropy_rows: logits must be bf16 [N, V] with unit column stride")
    N = logits.shape[0]
    V = int(vocab) if vocab is not None else logits.shape[1]
    targets = targets.to(torch.int64).contiguous().view(-1)
    if targets.numel() != N or not 1 <= V <= logits.shape[1]:
        raise ValueError("cross_entropy_rows: one target per row, vocab within the row length")
    bad = (targets != ignore_index) & ((targets < 0) | (targets >= V))
    if bool(bad.any()):
        raise ValueError("cross_entropy_rows: a target lies outside [0, vocab)")
    out = torch.empty(N, dtype=torch.float32, device=logits.device)
    with kernels._on(logits.device):
        _lib.check(_lib.lib().hb200_cross_entropy_rows(
            logits.data_ptr(), targets.data_ptr(), N, V, logits.stride(0) if N > 1 else max(logits.stride(0), V),
            int(ignore_index), out.data_ptr(), kernels._stream(logits.device)), "cross_entropy_rows")
    return out


class TokenLogprobs(NamedTuple):
    """What :func:`token_logprobs` returns for N rows."""
    logprobs: Tensor       # fp32 [N]
    entropy: Tensor        # fp32 [N], in nats
    top_logprobs: Tensor   # fp32 [N, top], most likely first
    top_ids: Tensor        # int64 [N, top]


def token_logprobs(logits: Tensor, tokens: Tensor, top: int = 0, temperature: float = 1.0, vocab: Optional[int] = None,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log probability of a given token, entropy and the ``top`` most likely tokens (up to 32) of each logit row
    (``hb200_token_logprobs``): one pass over the logits, 32 bits inside, nothing read on the host.

    logits [N, ld] bf16, f16 or fp32 on a CUDA device (any row stride, the first ``vocab`` columns count), tokens int64 [N].  The
    distribution is ``softmax(logits / temperature)``.  A row's log probability is 0 where its token is ``ignore_index`` and NaN
    where the token lies outside [0, vocab) otherwise (:func:`cross_entropy_rows` checks that on the host instead); entropy and
    alternatives do not depend on the token.  Of equal logits the lowest id comes first.  -inf logits (a grammar's mask) take
    no part and come last; a row without any other, or with NaN or +inf, gives NaN."""
    dev = kernels._require_cuda(logits, tokens)
    kernels._refuse_autograd("token_logprobs", logits)
    shape, strides = logits.shape, logits.stride()
    if len(shape) != 2 or (strides[1] != 1 and shape[1] > 1):
        raise ValueError("token_logprobs: logits must be [N, V] with unit column stride")
    dtype = kernels._dtype_code(logits)
    N, columns = shape
    V = int(vocab) if vocab is not None else columns
    top, temperature = int(top), float(temperature)
    if not 1 <= V <= columns:
        raise ValueError(f"token_logprobs: vocab {V} outside the row length {columns}")
    if V > kernels._INT32_MAX:
        raise kernels._past_int32("token_logprobs", V)
    if tokens.dtype != torch.int64 or tokens.numel() != N:
        raise ValueError(f"token_logprobs: one int64 token per row, got {tokens.dtype} {tuple(tokens.shape)} for {N} rows")
    if not 0 <= top <= min(32, V):
        raise ValueError(f"token_logprobs: top {top} (0 to 32, at most the vocabulary)")
    if not 1e-6 <= temperature <= 1e6:
        raise ValueError(f"token_logprobs: temperature {temperature} (1e-6 to 1e6)")
    ld = strides[0]
    if ld < V:
        if N > 1:
            logits = logits.contiguous()      # rows that overlap (an expanded row)
        ld = columns
    tokens = tokens if tokens.is_contiguous() else tokens.contiguous()
    with kernels._on(dev):
        new, f32 = kernels._empty_strided, torch.float32
        r = TokenLogprobs(new((N,), (1,), f32), new((N,), (1,), f32), new((N, top), (max(top, 1), 1), f32),
                          new((N, top), (max(top, 1), 1), torch.int64))
        if N > 0:
            _lib.check(_lib.lib().hb200_token_logprobs(
                logits.data_ptr(), tokens.data_ptr(), N, V, ld, ignore_index, temperature, top, r.logprobs.data_ptr(),
                r.entropy.data_ptr(), r.top_logprobs.data_ptr(), r.top_ids.data_ptr(), dtype, kernels._stream(dev)), "token_logprobs")
    return r


def sample_rows(logits: Tensor, temperature: float = 0.8, top_k: int = 50, top_p: float = 0.9,
                uniforms: Optional[Tensor] = None, generator: Optional[torch.Generator] = None,
                vocab: Optional[int] = None, out: Optional[Tensor] = None) -> Tensor:
    """logits bf16 [B, ld] on a CUDA device (row stride ``logits.stride(0)``; the first ``vocab`` columns count,
    default all) -> int64 [B] token ids.  ``uniforms`` fp32 [B] in [0, 1) are drawn from ``generator`` (a CUDA
    generator, or the device's default) when not given.  Defaults are the reference's (0.8 / 50 / 0.9);
    ``temperature <= 0`` or ``top_k == 1`` is the argmax."""
    if not logits.is_cuda:
        raise RuntimeError("sample_rows needs CUDA tensors (there is no CPU fallback)")
    if logits.dtype != torch.bfloat16 or logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("sample_rows: logits must be bf16 [B, V] with unit column stride")
    dev = logits.device
    B = logits.shape[0]
    V = int(vocab) if vocab is not None else logits.shape[1]
    if not 1 <= V <= logits.shape[1]:
        raise ValueError(f"sample_rows: vocab {V} outside the row length {logits.shape[1]}")
    greedy = not (temperature > 0.0) or top_k == 1
    if uniforms is None and not greedy:
        uniforms = torch.rand(B, dtype=torch.float32, device=dev, generator=generator)
    if uniforms is not None:
        if uniforms.device != dev or uniforms.dtype != torch.float32 or uniforms.numel() != B:
            raise ValueError("sample_rows: uniforms must be fp32 [B] on the logits' device")
        uniforms = uniforms.contiguous()
    if out is None:
        out = torch.empty(B, dtype=torch.int64, device=dev)
    elif out.device != dev or out.dtype != torch.int64 or out.numel() != B or not out.is_contiguous():
        raise ValueError("sample_rows: out must be a contiguous int64 [B] tensor on the logits' device")
    with kernels._on(dev):
        _lib.check(_lib.lib().hb200_sample_rows(
            logits.data_ptr(), B, V, logits.stride(0) if B > 1 else max(logits.stride(0), V), float(temperature),
            int(top_k), float(top_p), uniforms.data_ptr() if uniforms is not None else None, out.data_ptr(),
            kernels._stream(dev)), "sample_rows")
    return out
