"""The sparse-attention operators in 64 bits, from their definitions, on numpy
arrays: loops over sequences and heads, no code of the library.

A cache is `pool[block][layer][K|V][token][kv head][dim]`, its summaries
`summary[block][layer][kv head][min|max][dim]`, both float64 arrays of values
that the cache's element type holds exactly.
"""
from __future__ import annotations

import numpy as np


def rotate(x, pos, inv_freq, sections, interleaved):
    """x [..., D] turned by pos[axis] * inv_freq; len(inv_freq) pairs, the
    first sections[0] of them on axis 0 and so on."""
    half = len(inv_freq)
    axis = np.repeat(np.arange(len(sections)), sections)
    a = np.asarray(pos, dtype=np.float64)[axis] * np.asarray(inv_freq, dtype=np.float64)
    out = np.array(x, dtype=np.float64)
    i, j = (np.arange(0, 2 * half, 2), np.arange(1, 2 * half, 2)) if interleaved else \
        (np.arange(half), np.arange(half, 2 * half))
    u, w = np.array(out[..., i]), np.array(out[..., j])
    out[..., i] = u * np.cos(a) - w * np.sin(a)
    out[..., j] = w * np.cos(a) + u * np.sin(a)
    return out


def rope_append(pool, tables, ctx, new, layer, q, k, v, inv_freq, positions, sections, interleaved):
    """(query_out, [(block, slot, K rows, V rows)], {block: filled slots}).

    positions is [axes][batch][rows] or None (the cache position)."""
    T = pool.shape[3]
    out = np.zeros_like(q, dtype=np.float64)
    rows, filled = [], {}
    for b in range(len(ctx)):
        for t in range(int(new[b])):
            at = int(ctx[b]) - int(new[b]) + t
            pos = [at] * len(sections) if positions is None else positions[:, b, t]
            out[b, t] = rotate(q[b, t], pos, inv_freq, sections, interleaved)
            block = int(tables[b, at // T])
            rows.append((block, at % T, rotate(k[b, t], pos, inv_freq, sections, interleaved), v[b, t]))
            filled[block] = max(filled.get(block, 0), min(T, int(ctx[b]) - at // T * T))
    return out, rows, filled


def summary_of(pool, block, layer, filled):
    """[kv head][min|max][dim] of a block's first `filled` token slots."""
    k = pool[block, layer, 0, :filled]
    return np.stack((k.min(0), k.max(0)), axis=1)


def scores(q, summary, tables, b, blocks, layer, head, group):
    """The score of blocks 0 .. blocks - 1 of sequence b for one kv head."""
    x = q[b, head * group:(head + 1) * group].astype(np.float64)
    up, down = np.maximum(x, 0).sum(0), np.minimum(x, 0).sum(0)
    rows = summary[tables[b, :blocks], layer, head]
    with np.errstate(invalid="ignore", over="ignore"):
        s = (rows[:, 1] * up + rows[:, 0] * down).sum(-1)
    return np.where(np.isnan(s), np.inf, s)


def select(q, summary, tables, ctx, T, layer, hkv, keep, sink, recent):
    """selected [batch][hkv][keep]: ascending block numbers, then -1."""
    group = q.shape[1] // hkv
    out = np.full((len(ctx), hkv, keep), -1, dtype=np.int32)
    for b in range(len(ctx)):
        n = -(-int(ctx[b]) // T)
        for h in range(hkv):
            if n <= keep:
                chosen = list(range(n))
            else:
                s = scores(q, summary, tables, b, n, layer, h, group)
                always = [j for j in range(n) if j < sink or j >= n - recent]
                rest = sorted(range(sink, n - recent), key=lambda j: (-s[j], j))
                chosen = sorted(always + rest[:keep - sink - recent])
            out[b, h, :len(chosen)] = chosen
    return out


def attend(q, pool, tables, ctx, layer, scale, selected):
    """(out, size, reach): the attention over the listed blocks; per head
    sum_t p_t |v_t| (what errors of the weights scale with) and the largest
    scale * sum_d |q_d k_td| (what errors of the scores scale with)."""
    T, hkv, D = pool.shape[3], pool.shape[4], pool.shape[5]
    group = q.shape[1] // hkv
    out = np.zeros(q.shape, dtype=np.float64)
    size = np.zeros(q.shape, dtype=np.float64)
    reach = np.zeros(q.shape[:2], dtype=np.float64)
    for b in range(len(ctx)):
        for h in range(q.shape[1]):
            g = h // group
            keys, values = [], []
            for j in selected[b, g]:
                if 0 <= j and j * T < ctx[b]:
                    n = min(T, int(ctx[b]) - int(j) * T)
                    frame = int(tables[b, j])
                    keys.append(pool[frame, layer, 0, :n, g])
                    values.append(pool[frame, layer, 1, :n, g])
            if not keys:
                continue
            k, v = np.concatenate(keys), np.concatenate(values)
            s = scale * (k @ q[b, h].astype(np.float64))
            p = np.exp(s - s.max())
            p /= p.sum()
            out[b, h], size[b, h] = p @ v, p @ np.abs(v)
            reach[b, h] = abs(scale) * (np.abs(k) @ np.abs(q[b, h])).max()
    return out, size, reach
