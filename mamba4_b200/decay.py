"""Decay attention: linear attention with a decay for each head.

Per batch row and head the state follows S_t = e^(g_h) S_(t-1) + k_t v_t^T and
a token reads o_t = scale q_t S_t. It is the third linear-time mixer beside
the memory read (which solves against its evidence before it reads) and the
Mamba-3 scan (whose decay depends on the input); the decays here are
constants of each head.

  decay_attention       whole sequences (training and prompts): chunked form,
                        differentiable in q, k, v and the initial state
  decay_attention_step  one token per sequence against a carried state

The work runs in the CUDA library through the C ABI (`m4_decay_fwd`,
`m4_decay_bwd`, `m4_decay_step`). No CPU path exists.
"""

from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch
import torch.nn.functional as F

from . import _lib

MAX_DIM = 128  # largest key or value dim
_I3 = ctypes.c_int64 * 3


class DecayAttentionResult(NamedTuple):
    output: torch.Tensor   # [B, T, heads, value_dim] (step: [B, heads, value_dim])
    state: torch.Tensor    # [B, heads, key_dim, value_dim] float32, after the last token


def _dims(q, k, v, scale, strides):
    """M4DecayDims of operands [B, T, heads, dim]."""
    shape = q.shape
    head = (shape[0], shape[1] if strides else 1, shape[-2], k.shape[-2], shape[-1], v.shape[-1],
            q.dtype == torch.bfloat16, scale)
    if not strides:
        return _lib.DecayDims(*head)
    return _lib.DecayDims(*head, *(_I3(*t.stride()[:3]) for t in (q, k, v)))


def _rows16(t):
    """`t` with a contiguous last axis and rows that start on 16-byte
    boundaries (slices of a projection do, when their offsets are multiples of
    16 bytes); other layouts are copied."""
    unit = 16 // t.element_size()
    if t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % unit or not s for s, n in zip(t.stride(), t.shape[:-1]) if n > 1):
        return _dense16(t)
    return t


def _forward(q, k, v, initial, log_decay, lengths, scale):
    """m4_decay_fwd: (output, final state)."""
    lib = _lib.load()
    dims = _dims(q, k, v, scale, True)
    batch, time, heads, dk = q.shape
    output = torch.empty(batch, time, heads, v.shape[-1], dtype=q.dtype, device=q.device)
    final = torch.empty(batch, heads, dk, v.shape[-1], device=q.device)
    nbytes = lib.m4_decay_fwd_workspace_bytes(dims)
    work = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _lib.launch(q, "m4_decay_fwd", dims, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
                _lib.ptr(lengths), _lib.ptr(initial), output.data_ptr(), final.data_ptr(), work.data_ptr(), nbytes)
    return output, final


class _DecayAttention(torch.autograd.Function):
    """bfloat16: operands with dims that are multiples of 8."""

    @staticmethod
    def forward(ctx, q, k, v, initial, log_decay, lengths, scale):
        ctx.save_for_backward(q, k, v, initial, log_decay, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return _forward(q, k, v, initial, log_decay, lengths, scale)

    @staticmethod
    @_lib.once_differentiable
    def backward(ctx, d_output, d_final):
        lib = _lib.load()
        q, k, v, initial, log_decay, lengths = ctx.saved_tensors
        dims = _dims(q, k, v, ctx.scale, True)
        if d_output is None:
            d_output = torch.zeros(*q.shape[:3], v.shape[-1], dtype=q.dtype, device=q.device)
        d_output = _dense16(d_output.to(q.dtype))
        d_final = None if d_final is None else d_final.float().contiguous()
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        d_initial = None
        if initial is not None and ctx.needs_input_grad[3]:
            d_initial = torch.empty(initial.shape, device=q.device)
        nbytes = lib.m4_decay_bwd_workspace_bytes(dims)
        work = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
        _lib.launch(q, "m4_decay_bwd", dims, *map(_lib.ptr, (q, k, v, log_decay, lengths, initial, d_output, d_final, dq,
                                                             dk, dv, d_initial, work)), nbytes)
        return dq, dk, dv, d_initial, None, None, None


def _dense16(t):
    """Dense and on a 16-byte boundary (a fresh copy where a view is neither)."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def _check_operands(q, k, v, log_decay, what, ndim):
    if not q.is_cuda:
        raise RuntimeError(f"{what} runs on CUDA tensors only (no CPU path)")
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != ndim or len(ks) != ndim or len(vs) != ndim:
        raise ValueError(f"{what} expects q, k and v with {ndim} axes")
    if q.dtype not in (torch.float32, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v must share one dtype, float32 or bfloat16")
    device = q.device
    if k.device != device or v.device != device or log_decay.device != device:
        raise ValueError("operands must be on one device")
    heads, kv, dk, dv = qs[-2], ks[-2], qs[-1], vs[-1]
    if qs[:-2] != ks[:-2] or ks[:-1] != vs[:-1] or ks[-1] != dk:
        raise ValueError("q, k and v must agree in batch, time, key/value heads and key dim")
    if kv == 0 or heads % kv:
        raise ValueError(f"{heads} query heads must be a multiple of {kv} key/value heads")
    if not 1 <= dk <= MAX_DIM or not 1 <= dv <= MAX_DIM:
        raise ValueError(f"key and value dims must be in 1..{MAX_DIM}")
    if log_decay.shape != (heads,):
        raise ValueError(f"log_decay must have shape ({heads},)")
    if log_decay.requires_grad:
        raise ValueError("log_decay is a constant of each head and gets no gradient")


def _check_state(state, shape, device, name):
    if state.shape != shape or state.device != device or state.dtype != torch.float32:
        raise ValueError(f"{name} must be float32 of shape {tuple(shape)} on {device}")


def decay_attention(q, k, v, log_decay, *, scale=None, initial=None, lengths=None):
    """Whole sequences: q [B, T, heads, dk], k [B, T, kv_heads, dk], v
    [B, T, kv_heads, dv] (float32 or bfloat16; kv_heads divides heads and each
    key/value head serves heads / kv_heads neighbouring query heads; any
    strides: slices of one projection are read in place), log_decay [heads]
    float32 (<= 0, constant).

    scale: read scale, dk ** -0.5 by default. initial: state before the first
    token, [B, heads, dk, dv] float32. lengths: [B] int32, tokens of each
    sequence (values past T count as T); later tokens are not read, their
    outputs and gradients are zero, and the state is the one after the last
    token of the sequence.

    Returns DecayAttentionResult(output [B, T, heads, dv] in the operands'
    dtype, state float32); differentiable in q, k, v and initial. Sums and the
    state are float32; with bfloat16 operands the scores within 64 tokens, and
    the state where it is read, enter their products with 16 significant bits
    (2^-16 of the sum of absolute values, beside the result's own 2^-9). A NaN
    or an infinity reaches what depends on it in the recurrence and nothing
    else (with bfloat16 operands as NaN).
    """
    _check_operands(q, k, v, log_decay, "decay_attention", 4)
    batch, time, heads, dk = q.shape
    dv = v.shape[-1]
    scale = dk ** -0.5 if scale is None else float(scale)
    if initial is not None:
        _check_state(initial, (batch, heads, dk, dv), q.device, "initial")
    if lengths is not None:
        if lengths.shape != (batch,) or lengths.device != q.device or lengths.is_floating_point():
            raise ValueError(f"lengths must be integers of shape ({batch},) on {q.device}")
        if lengths.dtype != torch.int32:  # (clamped before it is narrowed)
            lengths = lengths.to(torch.int64).clamp(0, time).to(torch.int32)
        lengths = lengths.contiguous()
    if batch == 0 or time == 0:
        state = (torch.zeros(batch, heads, dk, dv, device=q.device) if initial is None
                 else initial.clone(memory_format=torch.contiguous_format))
        output = q.new_zeros(batch, time, heads, dv)
        if _lib.autograd_sees(q, k, v, initial):  # (connected, so that gradients are zero and not absent)
            nothing = 0 * (q.sum() + k.sum() + v.sum()).float()
            state = state + nothing
            output = output + (nothing if initial is None else nothing + 0 * initial.sum()).to(q.dtype)
        return DecayAttentionResult(output, state)
    # Zero coordinates never interact. The bfloat16 kernels take multiples of 8; the float32 ones take any
    # dim, with 16-byte copies of multiples of 4 (16 x 512 tokens of 8 heads, 63 x 127, trained: 872 us padded, 902 as it is).
    unit = 8 if q.dtype == torch.bfloat16 else 4
    pad_k, pad_v = -dk % unit, -dv % unit
    if pad_k or pad_v:
        q, k, v = F.pad(q, (0, pad_k)), F.pad(k, (0, pad_k)), F.pad(v, (0, pad_v))
        initial = None if initial is None else F.pad(initial, (0, pad_v, 0, pad_k))
    args = (_rows16(q), _rows16(k), _rows16(v), None if initial is None else initial.contiguous(),
            log_decay.float().contiguous(), lengths, scale)
    output, state = (_DecayAttention.apply if _lib.autograd_sees(*args[:4]) else _forward)(*args)
    if pad_k or pad_v:
        output, state = output[..., :dv], state[..., :dk, :dv].contiguous()  # (a step takes the state as it is)
    return DecayAttentionResult(output, state)


def decay_attention_step(state, q, k, v, log_decay, *, scale=None, inplace=False):
    """One token per sequence against a carried state: state [B, heads, dk, dv]
    float32, q [B, heads, dk], k [B, kv_heads, dk], v [B, kv_heads, dv].
    Returns DecayAttentionResult(output [B, heads, dv], state after the token),
    without a gradient (training runs whole sequences). inplace=True writes the new state over `state` (which must be contiguous).
    """
    _check_operands(q, k, v, log_decay, "decay_attention_step", 3)
    batch, heads, dk = q.shape
    dv = v.shape[-1]
    _check_state(state, (batch, heads, dk, dv), q.device, "state")
    if inplace and not state.is_contiguous():
        raise ValueError("inplace=True needs a contiguous state")
    scale = dk ** -0.5 if scale is None else float(scale)
    state = state.detach().contiguous()
    new = state if inplace else torch.empty_like(state)
    output = torch.empty(batch, heads, dv, dtype=q.dtype, device=q.device)
    if batch:
        q, k, v, decay = q.contiguous(), k.contiguous(), v.contiguous(), log_decay.float().contiguous()
        _lib.launch(q, "m4_decay_step", _dims(q, k, v, scale, False), state.data_ptr(), q.data_ptr(), k.data_ptr(),
                    v.data_ptr(), decay.data_ptr(), output.data_ptr(), new.data_ptr())
    if inplace and not state.is_inference():
        torch.autograd.graph.increment_version(state)  # (shared with the tensor that was given)
    return DecayAttentionResult(output, new)
