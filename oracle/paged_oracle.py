"""CPU oracle of the paged block memory: the block tables request by request and
token by token, and the attention in float64, from the definitions."""
from __future__ import annotations

import numpy as np


def block_tables(lens, new_lens, tables, free_ring, free_state, block_len: int, n_tokens: int):
    """(tables, lens, cu_new, slot_map, free_state, n_short, free_ring) after the
    step, as int arrays; nothing given is changed."""
    lens, tables, ring = (np.array(x, dtype=np.int64) for x in (lens, tables, free_ring))
    head, count = (int(x) for x in free_state)
    B, W = tables.shape
    F, L = len(ring), block_len
    short, back, slots, cu = 0, [], [], [0]
    for b in range(B):
        held = min(-(-int(lens[b]) // L), W)
        new = int(new_lens[b])
        if new < 0:
            back += [int(x) for x in tables[b, :held]]
            tables[b], lens[b] = -1, 0
            cu.append(cu[-1])
            continue
        row = [int(x) for x in tables[b, :held]]
        for j in range(held, -(-(int(lens[b]) + new) // L)):
            if j < W and count > 0:
                row.append(int(ring[head]))
                head, count = (head + 1) % F, count - 1
            else:
                row.append(-1)
                short += 1
        for p in range(int(lens[b]), int(lens[b]) + new):
            slots.append(row[p // L] * L + p % L if row[p // L] >= 0 else -1)
        tables[b] = (row + [-1] * W)[:W]
        lens[b] += new
        cu.append(cu[-1] + new)
    for x in back:
        ring[(head + count) % F] = x
        count += 1
    slots = (slots + [-1] * n_tokens)[:n_tokens]
    return tables, lens, np.array(cu), np.array(slots, dtype=np.int64), np.array([head, count]), short, ring


def gather(pool, table, n: int):
    """Positions [0, n) of a block table: pool [blocks, H, L, d] -> [H, n, d] (float64)."""
    pool = np.asarray(pool)
    H, L, d = pool.shape[1:]
    k = -(-n // L)
    return np.asarray(pool[np.asarray(table)[:k]], dtype=np.float64).transpose(1, 0, 2, 3).reshape(H, k * L, d)[:, :n]


def prefix_attention(Q, pool_K, pool_V, tables, lens, cu_new, prefix_table, prefix_len: int, scale: float):
    """(out, lse, mean_abs, top) in float64; rows behind cu_new[-1] are zeros and -inf.
    mean_abs = sum p |v| / sum p and top = the largest scale * sum |q| |k| of a
    row, for error bounds."""
    Q = np.asarray(Q, dtype=np.float64)
    n, heads, _ = Q.shape
    H, dv = pool_K.shape[1], pool_V.shape[3]
    G = heads // H
    out, lse = np.zeros((n, heads, dv)), np.full((n, heads), -np.inf)
    mean_abs, top = np.zeros((n, heads, dv)), np.zeros((n, heads))
    pk, pv = gather(pool_K, prefix_table, prefix_len), gather(pool_V, prefix_table, prefix_len)
    for b in range(len(lens)):
        t0, t1, length = int(cu_new[b]), int(cu_new[b + 1]), int(lens[b])
        ok, ov = gather(pool_K, tables[b], length), gather(pool_V, tables[b], length)
        for t in range(t0, t1):
            sees = max(0, min(length, length - (t1 - t0) + (t - t0) + 1))
            for h in range(H):
                k = np.concatenate([pk[h], ok[h, :sees]])
                v = np.concatenate([pv[h], ov[h, :sees]])
                if len(k) == 0:
                    continue
                at = (t, slice(h * G, (h + 1) * G))
                s = (Q[at] @ k.T) * scale
                m = s.max(1, keepdims=True)
                p = np.exp(s - m)
                out[at] = (p @ v) / p.sum(1, keepdims=True)
                lse[at] = m[:, 0] + np.log(p.sum(1))
                mean_abs[at] = (p @ np.abs(v)) / p.sum(1, keepdims=True)
                top[at] = abs(scale) * (np.abs(Q[at]) @ np.abs(k).T).max(1)
    return out, lse, mean_abs, top
