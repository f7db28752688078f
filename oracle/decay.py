"""Float64 restatement of decay attention: the recurrence token by token.

S_t = e^g S_(t-1) + k_t v_t^T, o_t = scale q_t S_t, and its gradients by the
reverse recurrence D_t = scale q_t do_t^T + e^g D_(t+1) (D past the last token:
the final state's cotangent, without a further decay).
"""

from __future__ import annotations

import torch


def attention(q, k, v, log_decay, scale, initial=None, lengths=None, d_output=None, d_final=None):
    """q [B,T,H,dk], k [B,T,Hk,dk], v [B,T,Hk,dv] (any dtype, computed in
    float64) -> dict of output, state and, given d_output, the gradients."""
    q, k, v, g = (t.detach().double().cpu() for t in (q, k, v, log_decay))
    batch, time, heads, dk = q.shape
    kv, dv = k.shape[2], v.shape[-1]
    head = torch.arange(heads) // (heads // kv)
    gamma = torch.exp(g)
    state = torch.zeros(batch, heads, dk, dv, dtype=torch.float64)
    if initial is not None:
        state = initial.detach().double().cpu().clone()
    ends = [time] * batch if lengths is None else [max(0, min(time, int(n))) for n in lengths.tolist()]
    out = torch.zeros(batch, time, heads, dv, dtype=torch.float64)
    result = dict(output=out, state=state)
    grads = d_output is not None
    if grads:
        do = d_output.detach().double().cpu()
        result.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v),
                      d_initial=torch.zeros_like(state))
    for b in range(batch):
        n = ends[b]
        states = torch.zeros(n + 1, heads, dk, dv, dtype=torch.float64)
        states[0] = state[b]
        for t in range(n):
            kt, vt = k[b, t, head], v[b, t, head]
            states[t + 1] = gamma[:, None, None] * states[t] + kt[:, :, None] * vt[:, None, :]
            out[b, t] = scale * torch.einsum("hx,hxy->hy", q[b, t], states[t + 1])
        state[b] = states[n]
        if grads:
            carry = torch.zeros(heads, dk, dv, dtype=torch.float64)
            if d_final is not None:
                carry = d_final[b].detach().double().cpu().clone()
            for t in reversed(range(n)):
                d = carry + scale * q[b, t][:, :, None] * do[b, t][:, None, :]
                result["dq"][b, t] = scale * torch.einsum("hxy,hy->hx", states[t + 1], do[b, t])
                result["dk"][b, t].index_add_(0, head, torch.einsum("hxy,hy->hx", d, v[b, t, head]))
                result["dv"][b, t].index_add_(0, head, torch.einsum("hxy,hx->hy", d, k[b, t, head]))
                carry = gamma[:, None, None] * d
            result["d_initial"][b] = carry
    return result
