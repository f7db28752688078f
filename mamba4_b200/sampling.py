"""Token sampling from logits: temperature, top-k, top-p and min-p, from given
uniform random numbers.

`sample_tokens` takes the logits of a decode step (`Mamba4LM.decode_step`,
`GraphedDecoder.step`) to token ids in one launch; it allocates only its
outputs and never synchronises, so it can be captured in a CUDA graph with the
step. Masses are integers, so a token depends on the logits, the settings and
the number alone, not on the order of summation. Runs in the CUDA library
(`m4_sample`). No CPU path exists.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib

MAX_VOCAB = 262144


class SampleResult(NamedTuple):
    tokens: torch.Tensor     # [...] int64 (-1 where every logit is -inf)
    log_prob: torch.Tensor   # [...] float32, among the kept tokens


def _setting(value, rows, device, dtype, name):
    """(per-row tensor or None, plain value)."""
    if not isinstance(value, torch.Tensor):
        return None, (max(0, min(int(value), MAX_VOCAB)) if dtype == torch.int32 else float(value))
    if value.device != device or value.numel() not in (1, rows):
        raise ValueError(f"{name} must be a number or one value per row on {device}")
    if dtype == torch.int32 and value.dtype == torch.int64:
        value = value.clamp(0, MAX_VOCAB)  # before it is narrowed to 32 bits
    value = value.detach().reshape(-1).to(dtype)
    return (value if value.numel() == rows else value.expand(rows)).contiguous(), 0


def sample_tokens(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """logits [..., V] (float32 or bfloat16) and uniform [...] float32 in
    [0, 1) -> SampleResult(tokens [...], log_prob [...]).

    Settings are numbers, or tensors with one value per row: temperature
    (<= 0: the largest logit, lowest index first), top_k (<= 0: off), top_p
    (>= 1: off: the smallest set of likeliest tokens that holds top_p of the
    mass top_k left), min_p (<= 0: off: tokens at least min_p times as likely
    as the likeliest). The token is the first in vocabulary order whose running
    kept probability exceeds the row's uniform number. log_prob is a value, not
    a function of the logits: it has no gradient.
    """
    if not logits.is_cuda:
        raise RuntimeError("sample_tokens runs on CUDA tensors only (no CPU path)")
    if logits.dtype not in (torch.float32, torch.bfloat16) or logits.ndim < 1:
        raise ValueError("logits must be float32 or bfloat16, [..., V]")
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"vocabulary size must be in 1..{MAX_VOCAB}")
    if uniform.shape != lead or uniform.device != logits.device or not uniform.is_floating_point():
        raise ValueError(f"uniform must be floating point of shape {tuple(lead)} on {logits.device}")
    if logits.ndim != 2:
        logits = logits.reshape(-1, vocab)
    if logits.stride(-1) != 1 or (logits.shape[0] > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    rows = logits.shape[0]
    tokens = torch.empty(lead, dtype=torch.int64, device=logits.device)
    log_prob = torch.empty(lead, dtype=torch.float32, device=logits.device)
    device = logits.device
    temperature, temperature_all = _setting(temperature, rows, device, torch.float32, "temperature")
    top_k, top_k_all = _setting(top_k, rows, device, torch.int32, "top_k")
    top_p, top_p_all = _setting(top_p, rows, device, torch.float32, "top_p")
    min_p, min_p_all = _setting(min_p, rows, device, torch.float32, "min_p")
    if rows:
        if uniform.dtype != torch.float32 or not uniform.is_contiguous():
            uniform = uniform.float().contiguous()
        ptr = _lib.ptr
        _lib.launch(logits, "m4_sample", rows, vocab, logits.stride(0) if rows > 1 else vocab, logits.data_ptr(),
                    logits.dtype == torch.bfloat16, uniform.data_ptr(), ptr(temperature), ptr(top_k), ptr(top_p),
                    ptr(min_p), temperature_all, top_k_all, top_p_all, min_p_all, tokens.data_ptr(), log_prob.data_ptr())
    return SampleResult(tokens, log_prob)
