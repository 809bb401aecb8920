"""Float64 numpy restatement of speculative decoding: attention of a draft tree over
a cache, verification of the drafts, and the cache rows kept (test infrastructure only)."""

from __future__ import annotations

import numpy as np


def line(parents, i):
    """Node i and its ancestors, or None where one of them is absent (a parent that is
    neither -1 nor an earlier node)."""
    out = []
    while True:
        out.append(i)
        p = int(parents[i])
        if p == -1:
            return out
        if not 0 <= p < i:
            return None
        i = p


def tree_attention(q, k, v, parents, lengths, scale=None):
    """(out, lse) in float64. q [B,H,T,D], k, v [B,H_kv,N,D], parents [B,T]. Each node's
    keys are picked out one by one, so that no other key can reach it."""
    B, H, T, D = q.shape
    Hkv = k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out = np.zeros((B, H, T, D))
    lse = np.full((B, H, T), -np.inf)
    for b in range(B):
        n = int(lengths[b])
        for i in range(T):
            up = line(parents[b], i)
            if up is None:
                continue
            keys = list(range(n)) + [n + j for j in sorted(up)]
            for h in range(H):
                hk = h // (H // Hkv)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k[b, hk, keys] @ q[b, h, i] * scale
                    m = s.max()
                    p = np.exp(s - m)
                    out[b, h, i] = p @ v[b, hk, keys] / p.sum()
                    lse[b, h, i] = m + np.log(p.sum())
    return out, lse


def _softmax(x, t):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x)
    if m == np.inf:
        e = (x == np.inf).astype(np.float64)
    else:
        e = np.exp((x - m) / t)
    return e / e.sum()


def _argmax(x):
    x = np.where(np.isnan(x), -np.inf, x)
    return -1 if x.max() == -np.inf else int(np.flatnonzero(x == x.max())[0])


def verify(logits, tokens, parents, uniforms, noise, temperature, drafts=None):
    """One sequence: (path, next token). logits, drafts [T,V]. Residuals are kept as
    normalised distributions and renormalised after each rejection. Also returns the
    least relative distance of any decision from its border, so that a caller can tell
    a wrong decision from one that rounding may turn."""
    T, V = logits.shape
    path, margin = [0], np.inf
    while True:
        node, nxt = path[-1], None
        children = [i for i in range(node + 1, T) if parents[i] == node]
        if temperature == 0:
            best = _argmax(logits[node].astype(np.float64))
            for i in children:
                if 0 <= tokens[i] < V and tokens[i] == best:
                    nxt = i
                    break
        else:
            p = w = _softmax(logits[node], temperature)
            q = None if drafts is None else _softmax(drafts[node], temperature)
            for i in children:
                x = int(tokens[i])
                if not 0 <= x < V:
                    continue
                if drafts is None:
                    if w[x] == 0 and p[x] > 0:
                        continue  # an earlier sibling's
                    lhs = float(uniforms[i])
                else:
                    lhs = float(uniforms[i]) * q[x]
                if max(lhs, w[x]) > 0:
                    margin = min(margin, abs(lhs - w[x]) / max(lhs, w[x]))
                if lhs < w[x]:
                    nxt = i
                    break
                w = w.copy()
                if drafts is None:
                    w[x] = 0
                else:
                    w = np.maximum(w - q, 0)
                w = w / w.sum() if w.sum() > 0 else w
        if nxt is None:
            break
        path.append(nxt)
    if temperature == 0:
        return path, best, margin
    for left in (w, p):
        with np.errstate(divide="ignore", invalid="ignore"):
            score = np.where(left > 0, left / noise.astype(np.float64), -np.inf)
        score = np.where(score >= 0, score, -np.inf)
        if score.max() > -np.inf:
            chosen = _argmax(score)
            others = np.sort(score)
            if V > 1 and np.isfinite(others[-1]) and others[-1] > 0 and others[-2] > 0:
                margin = min(margin, 1 - others[-2] / others[-1])
            return path, chosen, margin
    return path, -1, margin


def kept(path, count, nodes, length, rows):
    """The leading entries of a path that cab_kv_commit takes."""
    out = []
    for j in range(min(count, nodes) if length >= 0 else 0):
        f = int(path[j])
        if f <= (out[-1] if out else -1) or f >= nodes or length + f >= rows:
            break
        out.append(f)
    return out
