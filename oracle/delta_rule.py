"""CPU statement of the gated delta rule (test infrastructure only): the token recurrence in
float64, differentiable through autograd.  Per value head, with state S [K, V]:

    S <- exp(g_t) S;  u_t = beta_t (v_t - S^T k_t);  S <- S + k_t u_t^T;  o_t = scale S^T q_t
"""
from __future__ import annotations

import torch


def gated_delta_rule_ref(q, k, v, g, beta, cu_seqlens, scale=None, initial_state=None):
    """(o [T, HV, V], final states [N, HV, K, V]) in float64; zeros for tokens of no sequence."""
    T, H, K = q.shape
    HV, V = v.shape[1:]
    scale = K ** -0.5 if scale is None else scale
    cu = [int(x) for x in cu_seqlens.tolist()]
    q, k, v, g, beta = (x.double() for x in (q, k, v, g, beta))
    q, k = (x.repeat_interleave(HV // H, 1) for x in (q, k))
    rows = [torch.zeros(HV, V, dtype=torch.float64)] * T
    finals = []
    for n in range(len(cu) - 1):
        S = torch.zeros(HV, K, V, dtype=torch.float64)
        if initial_state is not None:
            S = initial_state[n].double()
        for t in range(cu[n], cu[n + 1]):
            S = torch.exp(g[t])[:, None, None] * S
            u = beta[t][:, None] * (v[t] - torch.einsum("hkv,hk->hv", S, k[t]))
            S = S + torch.einsum("hk,hv->hkv", k[t], u)
            rows[t] = scale * torch.einsum("hkv,hk->hv", S, q[t])
        finals.append(S)
    o = torch.stack(rows) if T else torch.zeros(0, HV, V, dtype=torch.float64)
    return o, torch.stack(finals) if finals else torch.zeros(0, HV, K, V, dtype=torch.float64)
