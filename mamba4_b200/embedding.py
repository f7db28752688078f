"""Embedding lookup with scaling, and its gradient by sorted tokens.

out[i] = round(scale weight[token_i]), rounded once to the residual stream's
dtype (no float32 copy of the rows), with the gradient
d_weight[v] = scale sum_{i: token_i = v} g_i in float32 sums of a fixed order
(those of ascending runs of places, joined in order): no atomics on floats, so a
step repeats bit for bit. Runs in the CUDA library
(`m4_embedding_fwd`, `m4_embedding_bwd`). No CPU path exists.
"""

from __future__ import annotations

import torch

from . import _lib

_DTYPES = (torch.float32, torch.bfloat16)
MAX_VOCAB, MAX_TOKENS = 1 << 21, 1 << 28  # of a lookup with a gradient


def _forward(tokens, weight, scale, dtype):
    rows, (vocab, dim) = tokens.numel(), weight.shape
    out = torch.empty(*tokens.shape, dim, dtype=dtype, device=weight.device)
    _lib.launch(weight, "m4_embedding_fwd", rows, vocab, dim, tokens.data_ptr(), weight.data_ptr(),
                weight.dtype == torch.bfloat16, scale, out.data_ptr(), dtype == torch.bfloat16)
    return out


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale, dtype):
        ctx.save_for_backward(tokens)
        ctx.cfg = (*weight.shape, weight.dtype, scale)
        return _forward(tokens, weight, scale, dtype)

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, grad):
        lib = _lib.load()
        tokens, = ctx.saved_tensors
        vocab, dim, dtype, scale = ctx.cfg
        grad = grad.contiguous()
        rows = tokens.numel()
        d_weight = torch.empty(vocab, dim, dtype=dtype, device=grad.device)
        nbytes = lib.m4_embedding_workspace_bytes(rows, vocab, dim)
        work = torch.empty(nbytes, dtype=torch.uint8, device=grad.device)
        _lib.launch(grad, "m4_embedding_bwd", rows, vocab, dim, tokens.data_ptr(), grad.data_ptr(),
                    grad.dtype == torch.bfloat16, scale, d_weight.data_ptr(), dtype == torch.bfloat16, work.data_ptr(),
                    nbytes)
        return None, d_weight, None, None


def embedding_lookup(tokens, weight, *, scale=1.0, dtype=None):
    """tokens [...] (integers) and weight [V, D] (float32 or bfloat16) ->
    scale * weight[tokens], [..., D] in `dtype` (the weight's by default).
    Ids outside [0, V) (padding) give zero rows and no gradient. With a
    gradient V is at most 2^21 and the number of tokens 2^28."""
    if not weight.is_cuda or not tokens.is_cuda:
        raise RuntimeError("embedding_lookup runs on CUDA tensors only (no CPU path)")
    dtype = weight.dtype if dtype is None else dtype
    if weight.ndim != 2 or weight.dtype not in _DTYPES or dtype not in _DTYPES:
        raise ValueError("embedding_lookup expects a [V, D] weight and an output of float32 or bfloat16")
    if tokens.dtype not in (torch.int64, torch.int32):
        raise ValueError("tokens must be int64 or int32")
    if tokens.device != weight.device:
        raise ValueError("tokens and weight must be on one device")
    if tokens.numel() == 0 or weight.numel() == 0:
        # (connected to the weight, so that its gradient is zero and not absent)
        return torch.zeros(*tokens.shape, weight.shape[1], dtype=dtype, device=weight.device) + 0 * weight.sum().to(dtype)
    run = _forward
    if _lib.autograd_sees(weight):
        if weight.shape[0] > MAX_VOCAB or tokens.numel() > MAX_TOKENS:
            raise ValueError(f"the gradient takes vocabularies up to {MAX_VOCAB} and up to {MAX_TOKENS} tokens")
        run = _EmbeddingLookup.apply
    if tokens.dtype != torch.int64:
        tokens = tokens.to(torch.int64)
    return run(tokens.contiguous(), weight.contiguous(), float(scale), dtype)
