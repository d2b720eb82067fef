"""Gated delta rule in float64, token by token, with its adjoint (numpy; what the CUDA kernels are compared with).

    S' = a_t S_{t-1},  y_t = v_t - S' k_t,  S_t = S' + beta_t y_t k_t^T,  o_t = scale S_t q_t,  a_t = exp(g_t)

q, k (b,Hk,T,N); v (b,H,T,P); g, beta (b,H,T); states (b,H,P,N).  Value head h reads key head h // (H // Hk).
"""

from __future__ import annotations

import numpy as np


def _wide(x, h):
    return np.repeat(x, h // x.shape[1], axis=1)


def forward(q, k, v, g, beta, scale, init=None):
    """-> (o, final, states): states[t] is the state before token t (T + 1 of them)."""
    q, k, v, g, beta = (np.asarray(x, np.float64) for x in (q, k, v, g, beta))
    b, h, T, P = v.shape
    q, k = _wide(q, h), _wide(k, h)
    S = np.zeros((b, h, P, q.shape[-1])) if init is None else np.asarray(init, np.float64)
    o, states = np.zeros_like(v), [S]
    for t in range(T):
        S = S * np.exp(g[:, :, t])[..., None, None]
        y = v[:, :, t] - np.einsum("bhpn,bhn->bhp", S, k[:, :, t])
        S = S + (beta[:, :, t, None] * y)[..., None] * k[:, :, t, None, :]
        o[:, :, t] = scale * np.einsum("bhpn,bhn->bhp", S, q[:, :, t])
        states.append(S)
    return o, S, states


def backward(q, k, v, g, beta, scale, init, d_o, d_final=None):
    """Gradients {q, k, v, g, beta, init} of sum(o * d_o) + sum(final * d_final)."""
    _, _, states = forward(q, k, v, g, beta, scale, init)
    hk = q.shape[1]
    q, k, v, g, beta, d_o = (np.asarray(x, np.float64) for x in (q, k, v, g, beta, d_o))
    b, h, T, P = v.shape
    q, k = _wide(q, h), _wide(k, h)
    R = np.zeros_like(states[0]) if d_final is None else np.asarray(d_final, np.float64)
    d = {n: np.zeros_like(x) for n, x in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta))}
    for t in reversed(range(T)):
        a = np.exp(g[:, :, t])[..., None, None]
        kt, S1, S0 = k[:, :, t], states[t + 1], states[t] * a
        y = v[:, :, t] - np.einsum("bhpn,bhn->bhp", S0, kt)
        d["q"][:, :, t] = scale * np.einsum("bhpn,bhp->bhn", S1, d_o[:, :, t])
        R = R + scale * d_o[:, :, t, :, None] * q[:, :, t, None, :]
        dd = np.einsum("bhpn,bhn->bhp", R, kt)
        d["beta"][:, :, t] = (dd * y).sum(-1)
        dy = beta[:, :, t, None] * dd
        d["v"][:, :, t] = dy
        d["k"][:, :, t] = (np.einsum("bhpn,bhp->bhn", R, beta[:, :, t, None] * y) - np.einsum("bhpn,bhp->bhn", S0, dy))
        R = R - dy[..., None] * kt[:, :, None, :]
        d["g"][:, :, t] = np.where(a[..., 0, 0] > 0, (R * S0).sum((-1, -2)), 0.0)
        R = R * a
    for n in ("q", "k"):
        d[n] = d[n].reshape(b, hk, h // hk, T, -1).sum(2)
    d["init"] = R
    return d
