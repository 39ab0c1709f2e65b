"""CPU restatement, in float64, of the operators over sequences: the gated
delta rule token by token (the recurrence of
prototype/gdn_replay_fp8_reference.py:137-163 on the raw rows of
prototype/gdn_replayssm_fp8_kernel.py:500-562), an attention layer's head norms
and rotation, and causal attention over a paged cache."""

from __future__ import annotations

import numpy as np


def _unit(x, eps=1e-6):
    return x / np.sqrt((x * x).sum(-1, keepdims=True) + eps)


def gdn_sequences(mixed, a, b, a_log, dt_bias, state, slots, starts, started=None, scale=None):
    """(out [T, HV, V], state [slots, HV, V, K]) after every sequence's tokens;
    rows of out outside the sequences are NaN. The arithmetic of non-finite
    inputs is the recurrence's own."""
    mixed, a, b, state = (np.asarray(x, np.float64) for x in (mixed, a, b, state))
    state = state.copy()
    (T, width), (_, HV, V, K) = mixed.shape, state.shape
    H = (width - HV * V) // (2 * K)
    G, scale = HV // H, K ** -0.5 if scale is None else scale
    q, k, v = np.split(mixed, [H * K, 2 * H * K], axis=1)
    q, k = (np.repeat(_unit(x.reshape(T, H, K)), G, axis=1) for x in (q, k))
    v = v.reshape(T, HV, V)
    z = a + np.asarray(dt_bias, np.float64)
    gamma = np.exp(-np.exp(np.asarray(a_log, np.float64)) * np.where(z > 20, z, np.log1p(np.exp(np.minimum(z, 20)))))
    beta = 1 / (1 + np.exp(-b))
    out = np.full((T, HV, V), np.nan)
    for n, slot in enumerate(slots):
        S = state[slot] if started is None or started[n] else np.zeros_like(state[slot])
        for t in range(int(starts[n]), int(starts[n + 1])):
            S = S * gamma[t][:, None, None]
            u = beta[t][:, None] * (v[t] - (S * k[t][:, None, :]).sum(-1))
            S = S + u[:, :, None] * k[t][:, None, :]
            out[t] = scale * (S * q[t][:, None, :]).sum(-1)
        state[slot] = S
    return out, state


def norm_rope(x, weight, table, positions, interleaved, eps=1e-6):
    """x [T, heads, D] normed (weight not None) and rotated by table[positions]."""
    x, table = np.asarray(x, np.float64), np.asarray(table, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    half = table.shape[1] // 2
    cos, sin = table[positions][:, None, :half], table[positions][:, None, half:]
    one = np.arange(half) * 2 if interleaved else np.arange(half)
    two = one + 1 if interleaved else one + half
    y = x.copy()
    y[..., one], y[..., two] = x[..., one] * cos - x[..., two] * sin, x[..., two] * cos + x[..., one] * sin
    return y


def paged_attention(q, k_cache, v_cache, table, starts, contexts, scale=None):
    """out [T, HQ, D]; rows outside the sequences are NaN, rows without keys 0."""
    q, k_cache, v_cache = (np.asarray(x, np.float64) for x in (q, k_cache, v_cache))
    T, HQ, D = q.shape
    page, HKV = k_cache.shape[1:3]
    scale, out = D ** -0.5 if scale is None else scale, np.full((T, HQ, D), np.nan)
    for n, C in enumerate(contexts):
        begin, end = int(starts[n]), int(starts[n + 1])
        at = np.arange(int(C))
        rows = np.asarray(table[n])[at // page], at % page
        for t in range(begin, end):
            seen = min(max(int(C) - end + t + 1, 0), int(C))
            for h in range(HQ):
                hk = h // (HQ // HKV)
                k, v = k_cache[rows[0][:seen], rows[1][:seen], hk], v_cache[rows[0][:seen], rows[1][:seen], hk]
                if seen == 0:
                    out[t, h] = 0
                    continue
                s = scale * (k @ q[t, h])
                p = np.exp(s - s.max())
                out[t, h] = (p[:, None] * v).sum(0) / p.sum()
    return out
