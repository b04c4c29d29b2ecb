"""Definitions in 64 bits of the operators on a cache whose slots are not
positions, and the inputs their tests share (numpy, no GPU)."""
import numpy as np


def tree_mask(rng, tokens, branch=4):
    """(who sees whom, depth) of a random tree of drafts, parents first."""
    sees = np.zeros((tokens, tokens), dtype=bool)
    depth = np.zeros(tokens, dtype=np.int64)
    for i in range(tokens):
        if i:
            p = int(rng.integers(max(0, i - branch), i))
            sees[i] = sees[p]
            depth[i] = depth[p] + 1
        sees[i, i] = True
    return sees, depth


def mask_words(sees):
    t = sees.shape[-1]
    pad = np.zeros(sees.shape[:-1] + ((-t) % 32,), dtype=bool)
    return np.packbits(np.concatenate([sees, pad], -1), axis=-1, bitorder="little").view("<u4").astype(np.uint32)


def attend(q, k, v, n_ctx, n_tok, scale, sees=None, cap=0.0, window=0, slopes=None, q_pos=None, k_pos=None):
    """q [S][T][nqh][hd], k/v [S][H][slots][hd] (any float type), sees
    [S][T][T] bool or None (causal); k_pos [S][slots] or [S][H][slots].
    Returns (out float64, zeros for rows that see nothing or are not live;
    weights [S][H][slots])."""
    S, T, nqh, hd = q.shape
    H, N = k.shape[1], k.shape[2]
    G = nqh // H
    out = np.zeros(q.shape)
    wts = np.zeros((S, H, N))
    for b in range(S):
        n, t = int(n_ctx[b]), int(n_tok[b])
        end = n + t
        qp = np.asarray(q_pos[b][:t]) if q_pos is not None else n + np.arange(t)
        for h in range(H):
            if k_pos is not None:
                kp = (k_pos[b, h] if k_pos.ndim == 3 else k_pos[b])[:end].astype(np.int64)
                hole = kp < 0
            else:
                kp = np.concatenate([np.arange(n), qp])
                hole = np.zeros(end, dtype=bool)
            see = np.ones((t, end), dtype=bool)
            see[:, n:] = np.tril(np.ones((t, t), dtype=bool)) if sees is None else sees[b, :t, :t]
            see &= ~hole[None]
            dist = qp[:, None].astype(np.int64) - kp[None]
            if window:
                see &= dist < window
            for g in range(G):
                for i in range(t):
                    at = np.nonzero(see[i])[0]
                    if at.size == 0:
                        continue
                    x = k[b, h, at].astype(np.float64) @ q[b, i, h * G + g].astype(np.float64) * scale
                    if cap:
                        x = cap * np.tanh(x / cap)
                    if slopes is not None:
                        x = x - float(slopes[h * G + g]) * dist[i, at]
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[b, i, h * G + g] = p @ v[b, h, at].astype(np.float64)
                    wts[b, h, at] += p
    return out, wts


def rope(x, pos, axis, rot, theta, halves, factors=None):
    """x [n][heads][hd] turned to pos [n][axes] in 64 bits."""
    y = x.astype(np.float64).copy()
    f = np.float64(np.float32(theta)) ** (-np.arange(0, rot, 2) / rot)
    if factors is not None:
        f = f / np.asarray(factors, dtype=np.float32).astype(np.float64)
    ang = pos[:, axis].astype(np.float64) * f
    c, s = np.cos(ang)[:, None], np.sin(ang)[:, None]
    i0 = np.arange(rot // 2) if halves else np.arange(0, rot, 2)
    i1 = i0 + rot // 2 if halves else i0 + 1
    a, b = y[..., i0].copy(), y[..., i1].copy()
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    return y


def select(scores, n, keep, first, recent):
    """One list: ascending kept slots, -1 behind them."""
    out = np.full(keep, -1, dtype=np.int64)
    if n <= keep:
        out[:n] = np.arange(n)
        return out
    mid = scores[first:n - recent].astype(np.float64)
    mid = np.where(np.isnan(mid), -np.inf, mid)
    nan = np.isnan(scores[first:n - recent])
    order = np.lexsort((np.arange(mid.size), nan, -mid))[: keep - first - recent]   # ties: lower index; NaN below -inf
    out[:] = np.sort(np.concatenate([np.arange(first), order + first, np.arange(n - recent, n)]))
    return out
