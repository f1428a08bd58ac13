"""Log probabilities of given tokens under rows of logits, with entropy and the most probable tokens (nnq_token_logprobs).

The reference turns logits into probabilities on the host, in its samplers
(crates/nn-core/src/layers/generation/autoregressive_sampling.rs:14-21); here the logits stay on the device and are read once.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Any, Optional

from . import api


@dataclass
class TokenLogprobs:
    """logprob, entropy (nats) f32 [rows]; top_tokens int32 and top_logprobs f32 [rows, top], descending (None with top = 0)."""
    logprob: Any
    entropy: Any
    top_tokens: Any = None
    top_logprobs: Any = None


def token_logprobs(logits, tokens, top: int = 0, backend: Optional[api.Backend] = None) -> TokenLogprobs:
    """logits [rows, vocab] f32 or bf16 (rows may lie apart), tokens [rows] (a negative one has log probability 0); top 0 .. 32."""
    torch = api._torch()
    b = backend or api.gpu_backend()
    if logits.dim() != 2:
        raise api.RankMismatch(f"expected [rows, vocab], got rank {logits.dim()}")
    if not (logits.is_cuda and tokens.is_cuda and logits.get_device() == b.device and tokens.get_device() == b.device):
        raise api.InvalidArgument(f"expected tensors on cuda:{b.device}, got {logits.device} and {tokens.device}")
    rows, vocab = logits.shape
    if tokens.shape != (rows,):
        raise api.ShapeMismatch(f"tokens: expected ({rows},), got {tuple(tokens.shape)}")
    if logits.dtype != torch.float32 and logits.dtype != torch.bfloat16:
        logits = logits.float()
    if (vocab > 1 and logits.stride(1) != 1) or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    if tokens.dtype != torch.int32:
        tokens = tokens.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    if top < 0 or top > min(32, vocab):
        raise api.Unsupported(f"{top} alternatives: at most 32 and the vocabulary's size")
    dev = logits.device
    pair = torch.empty((2, rows), dtype=torch.float32, device=dev)
    at = pair.data_ptr()
    tt = tl = None
    if top:
        tt, tl = torch.empty((rows, top), dtype=torch.int32, device=dev), torch.empty((rows, top), dtype=torch.float32, device=dev)
    st = b._lib.nnq_token_logprobs(b._ctx, logits.data_ptr(), api._dtype_code(logits), rows, vocab, logits.stride(0) if rows > 1 else vocab, tokens.data_ptr(), top,
                                   at, at + 4 * rows, tt.data_ptr() if top else None, tl.data_ptr() if top else None, api._stream_ptr(None, b.device))
    if st:
        b.check(st)
    return TokenLogprobs(*pair.unbind(0), tt, tl)
