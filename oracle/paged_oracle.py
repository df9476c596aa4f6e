"""The paged key-value cache's operators in 64-bit numpy -- test infrastructure
only (what the CUDA path is compared with, never the product).

Pools are [n_pages, kv_heads, page_size, head_dim]; the cache index n of a row
is slot n % page_size of page tables[row, n // page_size].  Written from the
formulas, one row and head at a time.
"""
from __future__ import annotations

import numpy as np


def frequencies(rot, theta=150000.0, scaling="plain", factor=1.0, first=4096.0, alpha=1.0, beta=32.0):
    """Inverse frequencies of the rot / 2 pairs and the factor on cos and sin."""
    half = rot // 2
    base = float(np.float32(theta))
    i = np.arange(half, dtype=np.float64)
    if scaling == "ntk":
        base = base * factor ** (rot / (rot - 2.0))
    f = base ** (-2.0 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "yarn" and factor > 1:
        # the pair that turns t times within the first context has index half * ln(first / (2 pi t)) / ln(theta)
        low, high = (half * np.log(first / (2 * np.pi * t)) / np.log(base) for t in (beta, alpha))
        ramp = np.clip((i - low) / max(high - low, 1e-3), 0.0, 1.0)
        return f * (1 - ramp) + f / factor * ramp, 0.1 * np.log(factor) + 1
    if scaling == "streaming" and factor > 1:
        import attention_oracle as ao
        th, conc = ao.rope_theta({"theta": theta, "scaling_factor": factor, "initial_context": first,
                                  "ntk_alpha": alpha, "ntk_beta": beta}, rot)
        return np.asarray(th, np.float64), float(conc)
    return f, 1.0


def rotate(x, positions, inv, factor=1.0, interleaved=False, inverse=False):
    """x [tokens, heads, head_dim] -> the leading 2 len(inv) columns turned by position x frequency."""
    y = np.array(x, np.float64)
    half = len(inv)
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        angle = np.asarray(positions, np.float64)[:, None] * inv[i]
        c, s = factor * np.cos(angle), factor * np.sin(angle) * (-1 if inverse else 1)
        u, w = np.array(x[..., a], np.float64), np.array(x[..., b], np.float64)
        y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    return y


def place(tables, page_size, row, n):
    return tables[row, n // page_size], n % page_size


def decode(q, k, v, tables, lens, scale, window=0, sinks=None, quiet=False, bias=None, weight=None, k_scale=None,
           v_scale=None):
    """-> out, lse; adds the shares to `weight` in place where given."""
    rows, nH, hd = q.shape
    H, page = k.shape[1], k.shape[2]
    G = nH // H
    out, lse = np.zeros((rows, nH, hd)), np.full((rows, nH), -np.inf)
    for r in range(rows):
        n0 = max(0, lens[r] - window) if window else 0
        at = np.arange(n0, lens[r])
        pg, sl = place(tables, page, r, at)
        for h in range(nH):
            g = h // G
            kk = k[pg, g, sl].astype(np.float64) * (1.0 if k_scale is None else k_scale[g])
            vv = v[pg, g, sl].astype(np.float64) * (1.0 if v_scale is None else v_scale[g])
            s = kk @ q[r, h].astype(np.float64) * scale
            if bias is not None:
                b = bias[r if bias.shape[0] > 1 else 0, h if bias.shape[1] > 1 else 0].astype(np.float64)
                s = s + np.concatenate([b[n0:lens[r]], np.zeros(max(0, lens[r] - max(n0, len(b))))])
            more = ([sinks[h]] if sinks is not None else []) + ([0.0] if quiet else [])
            every = np.concatenate([s, np.asarray(more, np.float64)])
            m = every.max() if len(every) else -np.inf
            if m == -np.inf:
                continue
            p = np.exp(every - m)
            L = p.sum()
            p = p[:len(s)] / L
            lse[r, h] = m + np.log(L)
            seen = p != 0  # a masked key's value does not count, whatever it holds
            out[r, h] = p[seen] @ vv[seen]
            if weight is not None:
                weight[pg, g, sl] += p
    return out, lse


def evict(k, v, weight, position, tables, lens, seen, budget, sink, recent):
    """In place on the four pools -> new lengths."""
    H, page = weight.shape[1], weight.shape[2]
    for r, n in enumerate(lens):
        if n <= budget:
            continue
        pg, sl = place(tables, page, r, np.arange(n))
        for h in range(H):
            order = []
            for i in range(n):
                w, p = weight[pg[i], h, sl[i]], position[pg[i], h, sl[i]]
                if p < sink or p >= seen[r] - recent:
                    order.append((1, 0.0, i))
                else:
                    order.append((0, np.inf if np.isnan(w) else float(w), i))
            victims = set(sorted(range(n), key=lambda i: order[i])[: n - budget])
            holes = [i for i in range(budget) if i in victims]
            movers = [i for i in range(budget, n) if i not in victims]
            assert len(holes) == len(movers)
            for to, by in zip(holes, movers):
                for x in (k, v, weight, position):
                    x[pg[to], h, sl[to]] = x[pg[by], h, sl[by]]
    return np.minimum(lens, budget)
