"""Float64 restatement of decoding over a paged cache: rotary positions, rows appended to pages,
attention over pages, adjusted logits. Written row by row, from the definitions (test
infrastructure)."""

import math

import numpy as np


def rotary_frequencies(dim, base=10000.0, scaling=None):
    """(radians a position of each pair, amplitude)."""
    s = scaling or {"type": "none"}
    kind, factor = s["type"], s.get("factor", 1.0)
    out, amplitude = [], 1.0
    if kind == "yarn":
        border = [dim * math.log(s["original_length"] / (n * 2 * math.pi)) / (2 * math.log(base))
                  for n in (s.get("beta_fast", 32), s.get("beta_slow", 1))]
        first, last = max(math.floor(border[0]), 0), min(math.ceil(border[1]), dim - 1)
        amplitude = s.get("amplitude", 0.1 * math.log(factor) + 1.0)
    for i in range(dim // 2):
        f = math.pow(base, -2 * i / dim)
        if kind == "linear":
            f /= factor
        elif kind == "ntk":
            f = math.pow(base * math.pow(factor, dim / (dim - 2)), -2 * i / dim)
        elif kind == "yarn":
            share = min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            f = share * f / factor + (1 - share) * f
        elif kind == "bands":
            turns, low, high = s["original_length"] * f / (2 * math.pi), s.get("low", 1), s.get("high", 4)
            if turns < low:
                f = f / factor
            elif turns <= high:
                w = (turns - low) / (high - low)
                f = (1 - w) * f / factor + w * f
        out.append(f)
    return np.array(out), amplitude


def rotary(x, positions, frequencies, amplitude=1.0, interleaved=False, inverse=False):
    """x ``[B, H, n, D]`` turned by positions ``[B, n]``."""
    y = np.array(x, dtype=np.float64)
    half = len(frequencies)
    angle = np.asarray(positions, dtype=np.float64)[:, None, :, None] * frequencies
    turn = amplitude * np.exp((-1j if inverse else 1j) * angle)
    at = ((slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved
          else (slice(0, half), slice(half, 2 * half)))
    z = (x[..., at[0]] + 1j * x[..., at[1]]) * turn
    y[..., at[0]], y[..., at[1]] = z.real, z.imag
    return y


def append(pages, new, table, lengths, counts=None):
    """Pages ``[P, H, S, D]`` with the new rows ``[B, H, n, D]`` in them."""
    pages = np.array(pages)
    P, _, S, _ = pages.shape
    B, _, n, _ = new.shape
    for b in range(B):
        for t in range(n if counts is None else min(n, max(0, int(counts[b])))):
            at = int(lengths[b]) + t
            if lengths[b] < 0 or at >= table.shape[1] * S:
                continue
            page = int(table[b, at // S])
            if 0 <= page < P:
                pages[page, :, at % S] = new[b, :, t]
    return pages


def attention(q, k_pages, v_pages, table, lengths, scale=None):
    """(out ``[B, H, 1, D]``, lse ``[B, H, 1]``)."""
    B, H, _, D = q.shape
    P, Hkv, S, _ = k_pages.shape
    scale = D ** -0.5 if scale is None else scale
    out, lse = np.zeros(q.shape), np.full((B, H, 1), -np.inf)
    for b in range(B):
        rows = [(int(table[b, s // S]), s % S) for s in range(min(int(lengths[b]), table.shape[1] * S))
                if 0 <= table[b, s // S] < P]
        if not rows:
            continue
        page, place = (np.array(x) for x in zip(*rows))
        for h in range(H):
            k, v = (x[page, h // (H // Hkv), place] for x in (k_pages, v_pages))
            with np.errstate(all="ignore"):
                z = (k @ q[b, h, 0]) * scale
                high = z.max()
                e = np.exp(z - high)
                if np.isnan(e.sum()) or e.sum() == 0:
                    out[b, h], lse[b, h] = np.nan, np.nan
                    continue
                out[b, h, 0], lse[b, h, 0] = (e / e.sum()) @ v, high + np.log(e.sum())
    return out, lse


def adjust(logits, history=None, lengths=None, prompts=None, repetition=1.0, presence=0.0,
           frequency=0.0, bias_tokens=None, bias=None, allowed=None, drafts=None, parents=None):
    """Adjusted logits ``[B, T, V]``; allowed: truth values ``[B, T, V]``."""
    x = np.array(logits, dtype=np.float64)
    B, T, V = x.shape
    of = lambda p, b: float(p[b]) if np.ndim(p) else float(p)
    for b in range(B):
        words = [] if history is None else [int(w) for w in history[b]]
        words = words if lengths is None else words[:max(0, int(lengths[b]))]
        given = 0 if prompts is None else max(0, int(prompts[b]))
        r, p, f = of(repetition, b), of(presence, b), of(frequency, b)
        for t in range(T):
            made, node = words[given:], t
            while drafts is not None:
                made = made + [int(drafts[b, node])]
                up = int(parents[b, node])
                if not 0 <= up < node:
                    break
                node = up
            for v in set(words[:given]) | set(made):
                if 0 <= v < V:
                    y = x[b, t, v]
                    x[b, t, v] = y / r if y > 0 else y * r
            for v in set(made):
                if 0 <= v < V:
                    x[b, t, v] -= f * made.count(v) + p
            if bias is not None:
                for v, y in {int(v): y for v, y in zip(bias_tokens[b], bias[b])}.items():
                    if 0 <= v < V:
                        x[b, t, v] += y
            if allowed is not None:
                x[b, t, ~allowed[b, t]] = -np.inf
    return x
