"""Definitions in 64 bits of the operators for trees of drafted tokens and of the cache copies around them.  TEST INFRASTRUCTURE ONLY.

The reference has no counterpart (its speculative mode verifies one chain); these restate the operators' own definitions, node by
node along each path, without the closed forms the kernels use.  No rounding anywhere (the chained operators of ``gdn_oracle`` keep the
reference's bf16 rounding points; the tree operators have none before their outputs).
"""
from __future__ import annotations

import numpy as np

HV, DK, KD, CD = 16, 128, 2048, 6144


def lines(parents):
    """For one tree (parents [N]): list of nodes root .. i for every node i, [] for unused (or malformed) nodes."""
    out = []
    for i, p in enumerate(np.asarray(parents).tolist()):
        if p == -1:
            out.append([i])
        elif 0 <= p < i and out[p]:
            out.append(out[p] + [i])
        else:
            out.append([])
    return out


def attn_tree(q, k_new, v_new, K, V, parents):
    """One sequence.  q [N, H, D], k_new, v_new [N, KV, D], K, V [KV, ctx, D].  Returns (o [N, H, D], a = the same sums with |V|: what an error
    relative to the weights is measured against)."""
    N, H, D = q.shape
    G = H // k_new.shape[1]
    o, a = np.zeros((N, H, D)), np.zeros((N, H, D))
    for i, line in enumerate(lines(parents)):
        if not line:
            continue
        for h in range(H):
            keys = np.concatenate([K[h // G], k_new[line, h // G]]).astype(np.float64)
            vals = np.concatenate([V[h // G], v_new[line, h // G]]).astype(np.float64)
            s = keys @ q[i, h].astype(np.float64) / 16
            w = np.exp(s - s.max())
            w /= w.sum()
            o[i, h], a[i, h] = w @ vals, w @ np.abs(vals)
    return o, a


def token(rows, conv_w, a, b, A_log, dt_bias):
    """Raw rows t-3 .. t [4, 6144] -> q, k, v [16, 128], decay and beta [16]."""
    x = (np.asarray(rows, np.float64) * np.asarray(conv_w, np.float64).reshape(CD, 4).T).sum(0)
    x = x / (1 + np.exp(-x))
    q, k, v = x.reshape(3, HV, DK)
    q = q / np.sqrt((q * q).sum(-1, keepdims=True) + 1e-6) / np.sqrt(DK)
    k = k / np.sqrt((k * k).sum(-1, keepdims=True) + 1e-6)
    rate = np.logaddexp(np.asarray(a, np.float64) + np.asarray(dt_bias, np.float64), 0)
    return q, k, v, np.exp(-np.exp(np.asarray(A_log, np.float64)) * rate), 1 / (1 + np.exp(-np.asarray(b, np.float64)))


def advance(S, window, row, conv_w, A_log, dt_bias):
    """One token: (y [16, 128], S, window)."""
    rows = np.concatenate([window, row[None, :CD]])
    q, k, v, g, beta = token(rows, conv_w, row[CD + KD + HV:CD + KD + 2 * HV], row[CD + KD:CD + KD + HV], A_log, dt_bias)
    S = S * g[:, None, None]
    d = (v - np.einsum("hvk,hk->hv", S, k)) * beta[:, None]
    S = S + d[:, :, None] * k[:, None, :]
    return np.einsum("hvk,hk->hv", S, q), S, rows[1:]


def deltanet_tree(proj, window, conv_w, A_log, dt_bias, S0, parents):
    """One sequence: proj [N, >= 8224], window [3, 6144], S0 [16, 128, 128].  Returns y [N, 2048] (zero rows for unused nodes)."""
    N = len(parents)
    y = np.zeros((N, KD))
    after = {-1: (np.asarray(S0, np.float64), np.asarray(window, np.float64))}
    for i, line in enumerate(lines(parents)):
        if line:
            S, win = after[line[-2] if len(line) > 1 else -1]
            out, S, win = advance(S, win, np.asarray(proj[i], np.float64), conv_w, A_log, dt_bias)
            y[i], after[i] = out.reshape(-1), (S, win)
    return y


def commit(proj, window, conv_w, A_log, dt_bias, S0, path):
    """State and window after the nodes ``path`` (in order)."""
    S, win = np.asarray(S0, np.float64), np.asarray(window, np.float64)
    for i in path:
        _, S, win = advance(S, win, np.asarray(proj[i], np.float64), conv_w, A_log, dt_bias)
    return S, win


def accept(parents, toks, ids):
    """The confirmed path of one tree."""
    alive = [bool(x) for x in lines(parents)]
    N, path, at = len(parents), [], -1
    while True:
        nxt = [i for i in range(N) if alive[i] and parents[i] == at and (at < 0 or toks[i] == ids[at])]
        if not nxt:
            return path
        at = nxt[0]
        path.append(at)
