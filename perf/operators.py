"""Cases of the paged block memory: the operators by which requests of ragged
lengths share one pool of L-token blocks.

``tables``  one step of the block tables: every request names how many tokens
            it appends (or that it ends); blocks are taken from the free ring,
            blocks of ended requests go back to it, and each new token gets its
            slot ``block * L + offset`` in the pool.
``append``  the new tokens' keys and values go to their slots.
``attend``  softmax attention of the new tokens over a prefix that all requests
            share (stored once) and over each request's own blocks, causal
            within the new tokens.

``run`` computes them in plain 32-bit torch operations where ``own`` is false
and calls the package's operators where it is true; ``exact`` computes the same
outputs in 64 bits from the definitions.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "f32": torch.float32}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _tables(name, requests, width, L, cached, new, ended):
    return {"name": name, "op": "tables", "requests": requests, "width": width, "L": L, "cached_lo": cached[0],
            "cached_hi": cached[1], "new_lo": new[0], "new_hi": new[1], "ended": ended}


def _append(name, dtype, heads, d, L, tokens, padded):
    return {"name": name, "op": "append", "dtype": dtype, "heads": heads, "d": d, "L": L, "tokens": tokens,
            "padded": padded}


def _attend(name, dtype, requests, heads, group, d, L, prefix, cached, new, lse):
    return {"name": name, "op": "attend", "dtype": dtype, "requests": requests, "heads": heads, "group": group, "d": d,
            "L": L, "prefix": prefix, "cached_lo": cached[0], "cached_hi": cached[1], "new_lo": new[0],
            "new_hi": new[1], "lse": lse}


def listed():
    return [
        # a handful of interactive requests, one token each: launch latency
        _tables("tables_small", 8, 32, 16, (1, 300), (1, 1), 0),
        # a full decode batch: one token each, one request in 32 ends
        _tables("tables_decode", 256, 512, 64, (1, 32000), (1, 1), 32),
        # a large pool of requests taking prompt pieces of odd lengths, many ending
        _tables("tables_prompts", 4096, 1024, 16, (0, 15000), (0, 400), 16),
        # the decode batch's keys and values of one layer
        _append("append_decode", "bf16", 8, 128, 64, 256, 0),
        # prompt pieces of one layer, the buffer padded behind the last request
        _append("append_prompts", "bf16", 8, 128, 64, 65000, 536),
        # two requests of the smallest streaming configuration: latency
        _attend("attend_small", "bf16", 2, 4, 2, 64, 16, 64, (0, 60), (1, 1), True),
        # the same in the 32-bit memory
        _attend("attend_small_f32", "f32", 2, 4, 1, 64, 16, 240, (3, 250), (1, 2), True),
        # an ordinary decode batch behind a system prompt
        _attend("attend_decode", "bf16", 64, 8, 4, 128, 64, 8192, (1, 1024), (1, 1), False),
        # few requests with long texts of their own (up to 512 blocks of 64)
        _attend("attend_decode_long", "bf16", 16, 8, 4, 128, 64, 2000, (4096, 32767), (1, 1), False),
        # many short requests over one long document
        _attend("attend_document", "bf16", 512, 4, 8, 128, 64, 32768, (0, 255), (1, 1), False),
        # checking drafted tokens: a few queries per request, odd group and prefix, small blocks
        _attend("attend_drafts", "fp16", 33, 4, 7, 128, 16, 5003, (0, 700), (3, 6), True),
        # prompt pieces of ragged lengths behind the shared prefix
        _attend("attend_prompts", "bf16", 12, 8, 4, 128, 128, 4096, (0, 500), (1, 1500), False),
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 0.999))))))


def _draw_once(rng):
    op = rng.choice(["tables", "append", "attend", "attend"])
    if op == "tables":
        requests, width, L = _log_int(rng, 1, 4096), _log_int(rng, 8, 1024), rng.choice([16, 32, 64, 128, 24])
        hi = _log_int(rng, 1, width * L - 1)
        return _tables(None, requests, width, L, (0, hi), (0, _log_int(rng, 1, 400)), rng.choice([0, 5, 16, 32]))
    if op == "append":
        return _append(None, rng.choice(list(DTYPES)), rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([64, 128, 256, 80]),
                       rng.choice([16, 32, 64, 128, 24]), _log_int(rng, 1, 32000), rng.choice([0, 1, 37]))
    dtype = rng.choice(["bf16", "bf16", "fp16", "bf16", "fp16", "f32"])
    new = rng.choice([(1, 1), (1, 1), (0, 3), (1, 8), (1, 900)])
    requests = _log_int(rng, 1, 512 if new[1] <= 8 else 12)
    prefix = rng.choice([0, _log_int(rng, 1, 32768)] + [_log_int(rng, 100, 32768) for _ in range(4)])
    hi = _log_int(rng, 1, 32000)
    group, heads = rng.choice([1, 2, 4, 5, 7, 8]), rng.choice([1, 2, 4, 8])
    return _attend(None, dtype, requests, heads, group, rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128]),
                   prefix, (rng.choice([0, 1, hi // 2]), hi), new, rng.choice([False, True]))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        b, f = most.get(c["op"], (0, 0))
        most[c["op"]] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        c = _draw_once(rng)
        del c["name"]
        w, (b, f) = work(c), most[c["op"]]
        # the 32-bit memory's products run on the FP32 units: an eighth of the work at most
        s = 8 if c["op"] == "attend" and c["dtype"] == "f32" else 1
        # padded keys of the plain form: requests x the longest text
        pad = c["op"] != "attend" or c["requests"] * (c["cached_hi"] + c["new_hi"]) * c["heads"] <= 16 * 32767 * 8
        wide = c["op"] != "attend" or \
            c["requests"] * c["new_hi"] * c["heads"] * c["group"] * (c["cached_hi"] + c["new_hi"]) <= 3 << 30
        if s * w["bytes"] <= b and s * w["flops"] <= f and pad and wide:
            return c


def _spread(i, lo, hi, step):
    """The i-th of evenly spread integers of [lo, hi] (multiples of an irrational step, modulo the range)."""
    return lo + int((hi - lo + 1) * ((0.37 + i * step) % 1.0))


def _lengths(case):
    """(cached, new) of each request; the seed only orders them.  new < 0: the request ends."""
    out = []
    for i in range(case["requests"]):
        # half of the requests short, half spread to the longest
        c = _spread(i, case["cached_lo"], case["cached_hi"], 0.6180339887498949)
        if i % 2 and case["cached_lo"] * 4 < case["cached_hi"]:
            c = case["cached_lo"] + (c - case["cached_lo"]) // 4
        n = _spread(i, case["new_lo"], case["new_hi"], 0.7548776662466927)
        if case.get("ended") and i % case["ended"] == case["ended"] - 1:
            n = -1
        out.append((c, n))
    if case["op"] == "attend" and all(n <= 0 for _, n in out):
        out[0] = (out[0][0], 1)
    return out


def _blocks(n, L):
    return (n + L - 1) // L


def work(case):
    L = case["L"]
    if case["op"] == "tables":
        B, W, lens = case["requests"], case["width"], _lengths(case)
        n = sum(max(x, 0) for _, x in lens)
        taken = sum(max(0, min(_blocks(c + x, L), W) - min(_blocks(c, L), W)) for c, x in lens if x >= 0)
        back = sum(min(_blocks(c, L), W) for c, x in lens if x < 0)
        held = sum(min(_blocks(c, L), W) for c, _ in lens)
        # lengths in and out, offsets out; the blocks held in; the tables and slots out; the ring's entries
        return {"bytes": 4 * (4 * B + 1 + held + B * W + n + taken + back + 5), "flops": 0}
    if case["op"] == "append":
        size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
        return {"bytes": case["tokens"] * (4 * case["heads"] * case["d"] * size + 4) + 4 * case["padded"], "flops": 0}
    size = torch.finfo(DTYPES[case["dtype"]]).bits // 8
    H, G, d, P = case["heads"], case["group"], case["d"], case["prefix"]
    lens = [(c, n) for c, n in _lengths(case) if n > 0]
    tokens = sum(n for _, n in lens)
    kv = P + sum(c + n for c, n in lens)
    pairs = sum(n * (P + c) + n * (n + 1) // 2 for c, n in lens)
    entries = _blocks(P, L) + sum(_blocks(c + n, L) for c, n in lens)
    return {"bytes": 2 * kv * H * d * size + 2 * tokens * H * G * d * size + 4 * entries + 8 * case["requests"]
            + (4 * tokens * H * G if case["lse"] else 0),
            "flops": 4 * pairs * H * G * d}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    host = np.random.default_rng(seed)
    state = {"case": dict(case)}
    L = case["L"]
    if case["op"] == "append":
        n, H, d, dt = case["tokens"] + case["padded"], case["heads"], case["d"], DTYPES[case["dtype"]]
        n_blocks = _blocks(case["tokens"], L) * 2 + 1
        slots = np.full(n, -1, dtype=np.int32)
        # requests write runs of tokens: blocks in any order, tokens within a block in order
        order = host.permutation(n_blocks)
        t = np.arange(case["tokens"])
        slots[:case["tokens"]] = order[t // L] * L + t % L
        state["slot_map"] = torch.from_numpy(slots).to(dev)
        state["K"] = torch.randn((n, H, d), generator=g, device=dev).to(dt)
        state["V"] = torch.randn((n, H, d), generator=g, device=dev).to(dt)
        state["pool_K"] = torch.zeros((n_blocks, H, L, d), dtype=dt, device=dev)
        state["pool_V"] = torch.zeros((n_blocks, H, L, d), dtype=dt, device=dev)
        return state

    lens = _lengths(case)
    order = host.permutation(len(lens))
    cached = np.array([lens[i][0] for i in order], dtype=np.int64)
    new = np.array([lens[i][1] for i in order], dtype=np.int64)
    B = len(lens)
    if case["op"] == "tables":
        W = case["width"]
        cached = np.minimum(cached, W * L)
        new = np.where(new > 0, np.minimum(new, W * L - cached), new)
        need = _blocks(cached, L)
        grow = int(np.maximum(_blocks(cached + np.maximum(new, 0), L) - need, 0).sum())
        n_blocks = int(need.sum()) + grow + 3 + B // 4
        blocks = host.permutation(n_blocks).astype(np.int32)
        table = np.full((B, W), -1, dtype=np.int32)
        at = 0
        for b in range(B):
            table[b, :need[b]] = blocks[at:at + need[b]]
            at += int(need[b])
        free = n_blocks - at
        head = int(host.integers(0, n_blocks))
        ring = np.full(n_blocks, -1, dtype=np.int32)
        ring[(head + np.arange(free)) % n_blocks] = blocks[at:]
        state.update(lens=torch.from_numpy(cached.astype(np.int32)).to(dev),
                     new_lens=torch.from_numpy(new.astype(np.int32)).to(dev),
                     tables=torch.from_numpy(table).to(dev), free_ring=torch.from_numpy(ring).to(dev),
                     free_state=torch.tensor([head, free], dtype=torch.int32, device=dev),
                     n_tokens=int(np.maximum(new, 0).sum()))
        return state

    H, G, d, P, dt = case["heads"], case["group"], case["d"], case["prefix"], DTYPES[case["dtype"]]
    new = np.maximum(new, 0)
    total = cached + new
    need = _blocks(total, L)
    W = max(1, int(need.max()))
    p_blocks = _blocks(P, L)
    n_blocks = p_blocks + int(need.sum()) + 2
    blocks = host.permutation(n_blocks).astype(np.int32)
    table = np.full((B, W), -1, dtype=np.int32)
    at = p_blocks
    for b in range(B):
        table[b, :need[b]] = blocks[at:at + need[b]]
        at += int(need[b])
    n = int(new.sum())
    state.update(
        Q=(1.5 * torch.randn((n, H * G, d), generator=g, device=dev)).to(dt),
        pool_K=_normal((n_blocks, H, L, d), g, dt), pool_V=_normal((n_blocks, H, L, d), g, dt),
        tables=torch.from_numpy(table).to(dev), lens=torch.from_numpy(total.astype(np.int32)).to(dev),
        cu_new=torch.from_numpy(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).to(dev),
        prefix_table=torch.from_numpy(blocks[:p_blocks].copy()).to(dev),
        prefix_len=torch.tensor([P], dtype=torch.int32, device=dev), scale=1.0 / math.sqrt(d),
        # sizes that a program knows on the host
        longest=int(total.max()), most_new=int(new.max()))
    return state


def _normal(shape, g, dt):
    """Normal values made in the memory's own type, some blocks at a time."""
    x = torch.empty(shape, dtype=dt, device="cuda")
    step = max(1, (1 << 27) // max(1, x[:1].numel()))
    for i in range(0, shape[0], step):
        x[i:i + step] = torch.randn(x[i:i + step].shape, generator=g, device="cuda").to(dt)
    return x


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        from gfst_hmb_public_b200 import paged
        if op == "tables":
            t = paged.block_tables(state["lens"], state["new_lens"], state["tables"], state["free_ring"],
                                   state["free_state"], block_len=state["case"]["L"], n_tokens=state["n_tokens"])
            return [t.tables, t.lens, t.cu_new, t.slot_map, t.free_state, t.n_short, state["free_ring"]]
        if op == "append":
            paged.paged_append(state["K"], state["V"], state["pool_K"], state["pool_V"], state["slot_map"])
            return [state["pool_K"], state["pool_V"]]
        out, lse = paged.prefix_attention(state["Q"], state["pool_K"], state["pool_V"], state["tables"],
                                          state["lens"], state["cu_new"], prefix_table=state["prefix_table"],
                                          prefix_len=state["prefix_len"], scale=state["scale"],
                                          return_lse=state["case"]["lse"])
        return [out, lse] if state["case"]["lse"] else [out]
    return {"tables": _plain_tables, "append": _plain_append, "attend": _plain_attend}[op](state)


def _plain_tables(s):
    L, F = s["case"]["L"], s["free_ring"].shape[0]
    lens, new, tables = s["lens"].long(), s["new_lens"].long(), s["tables"]
    B, W = tables.shape
    dev = tables.device
    head, count = s["free_state"][0].long(), s["free_state"][1].long()
    add, ends = new.clamp(min=0), new < 0
    held = ((lens + L - 1) // L).clamp(max=W)
    wanted = (lens + add + L - 1) // L
    need = torch.where(ends, torch.zeros_like(wanted), wanted.clamp(max=W))
    grow = (need - held).clamp(min=0)
    first = torch.cumsum(grow, 0) - grow                 # rank of the request's first new block
    back = torch.where(ends, held, torch.zeros_like(held))
    first_back = torch.cumsum(back, 0) - back
    w = torch.arange(W, device=dev)[None, :]
    rank = first[:, None] + w - held[:, None]
    fresh = s["free_ring"][(head + rank.clamp(min=0)) % F]
    fresh = torch.where(rank < count, fresh, torch.full_like(fresh, -1))
    out = torch.where(w < held[:, None], tables, torch.where(w < need[:, None], fresh, torch.full_like(tables, -1)))
    out = torch.where(ends[:, None], torch.full_like(tables, -1), out)
    # blocks of the ended requests, in order, behind the last free one
    given = ends[:, None] & (w < held[:, None])
    at = (head + count + first_back[:, None] + w) % F
    s["free_ring"][at[given]] = tables[given]
    cu = torch.cat([torch.zeros(1, dtype=torch.long, device=dev), torch.cumsum(add, 0)])
    i = torch.arange(s["n_tokens"], device=dev)
    b = torch.searchsorted(cu, i, right=True) - 1
    p = lens[b] + i - cu[b]
    block = out[b, (p // L).clamp(max=W - 1)].long()
    slot = torch.where((p // L < W) & (block >= 0), block * L + p % L, torch.full_like(p, -1))
    taken = torch.minimum(grow.sum(), count)
    short = grow.sum() - taken + (torch.where(ends, held, wanted) - W).clamp(min=0).sum()
    lens_out = torch.where(ends, torch.zeros_like(lens), lens + add)
    free = torch.stack([(head + taken) % F, count - taken + back.sum()])
    return [out, lens_out.int(), cu.int(), slot.int(), free.int(), short.int().reshape(1), s["free_ring"]]


def _plain_append(s):
    L = s["case"]["L"]
    keep = s["slot_map"] >= 0
    slot = s["slot_map"][keep].long()
    s["pool_K"][slot // L, :, slot % L] = s["K"][keep]
    s["pool_V"][slot // L, :, slot % L] = s["V"][keep]
    return [s["pool_K"], s["pool_V"]]


def _softmax_parts(scores, v, seen):
    """Largest score, sum of exponentials and weighted values over the last axis of ``scores``."""
    if seen is not None:
        scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(scores - base)
    return base + torch.log(e.sum(-1, keepdim=True)), e @ v / e.sum(-1, keepdim=True).clamp(min=1e-38)


def _plain_attend(s):
    c = s["case"]
    H, G, d, L, P = c["heads"], c["group"], c["d"], c["L"], c["prefix"]
    Q, cu = s["Q"], s["cu_new"].long()
    N, B, dev = Q.shape[0], s["lens"].shape[0], Q.device
    q = Q.float().reshape(N, H, G, d) * s["scale"]
    parts = []
    if P:
        t = s["prefix_table"].long()
        k = s["pool_K"][t].permute(1, 0, 2, 3).reshape(H, -1, d)[:, :P].float()
        v = s["pool_V"][t].permute(1, 0, 2, 3).reshape(H, -1, d)[:, :P].float()
        qh = q.permute(1, 0, 2, 3).reshape(H, N * G, d)
        step = max(1, (1 << 30) // (P * H))
        got = [_softmax_parts(qh[:, i:i + step] @ k.transpose(1, 2), v, None) for i in range(0, N * G, step)]
        parts.append([torch.cat(x, 1).reshape(H, N, G, -1).permute(1, 0, 2, 3) for x in zip(*got)])
    # the requests' own tokens, padded to the longest request
    S, M = s["longest"], s["most_new"]
    W = (S + L - 1) // L
    t = s["tables"][:, :W].long().clamp(min=0)
    k = s["pool_K"][t].permute(0, 2, 1, 3, 4).reshape(B, H, W * L, d).float()
    v = s["pool_V"][t].permute(0, 2, 1, 3, 4).reshape(B, H, W * L, d).float()
    pos = torch.arange(W * L, device=dev)
    v = v * (pos < s["lens"][:, None]).float()[:, None, :, None]
    n = cu[1:] - cu[:-1]
    j = torch.arange(M, device=dev)
    qi = (cu[:-1, None] + j).clamp(max=N - 1)             # [B, M] token of each padded query
    last = s["lens"].long()[:, None] - n[:, None] + j     # [B, M] last position it sees
    seen = (pos <= last[..., None])[:, None, :, None, :].expand(B, 1, M, G, W * L).reshape(B, 1, M * G, W * L)
    qb = q[qi].permute(0, 2, 1, 3, 4).reshape(B, H, M * G, d)
    lse, o = _softmax_parts(qb @ k.transpose(2, 3), v, seen)
    valid = j < n[:, None]
    parts.append([x.reshape(B, H, M, G, -1).permute(0, 2, 1, 3, 4)[valid] for x in (lse, o)])
    if len(parts) == 2:
        (la, oa), (lb, ob) = parts
        lse = torch.logaddexp(la, lb)
        o = torch.exp(la - lse) * oa + torch.exp(lb - lse) * ob
    else:
        lse, o = parts[0]
    out = o.reshape(N, H * G, d).to(Q.dtype)
    return [out, lse.reshape(N, H * G).contiguous()] if c["lse"] else [out]


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    L = case["L"]
    if case["op"] == "append":
        slots = s["slot_map"].cpu().numpy()
        rows = np.flatnonzero(slots >= 0)
        at = torch.from_numpy(slots[rows].astype(np.int64)).cuda()
        rows = torch.from_numpy(rows).cuda()
        outs = []
        for x, pool in ((s["K"], s["pool_K"]), (s["V"], s["pool_V"])):
            flat = pool.double().transpose(1, 2).reshape(-1, case["heads"], case["d"])
            flat[at] = x.double()[rows]
            outs.append(flat.reshape(pool.shape[0], L, case["heads"], case["d"]).transpose(1, 2).contiguous())
        return outs
    if case["op"] == "tables":
        return _exact_tables(s)
    return _exact_attend(s)


def _exact_tables(s):
    L = s["case"]["L"]
    lens, new = s["lens"].tolist(), s["new_lens"].tolist()
    table, ring = s["tables"].cpu().numpy().copy(), s["free_ring"].cpu().numpy().copy()
    head, count = s["free_state"].tolist()
    B, W = table.shape
    F, short, given, slots, cu = len(ring), 0, [], [], [0]
    for b in range(B):
        held = min((lens[b] + L - 1) // L, W)
        if new[b] < 0:
            given += table[b, :held].tolist()
            table[b] = -1
            lens[b] = 0
            cu.append(cu[-1])
            continue
        row = table[b, :held].tolist()
        want = (lens[b] + new[b] + L - 1) // L
        while len(row) < want:
            if count and len(row) < W:
                row.append(int(ring[head]))
                head, count = (head + 1) % F, count - 1
            else:
                row.append(-1)
                short += 1
        table[b, held:] = -1
        table[b, :min(want, W)] = row[:W]
        for p in range(lens[b], lens[b] + new[b]):
            k = row[p // L]
            slots.append(k * L + p % L if k >= 0 else -1)
        lens[b] += new[b]
        cu.append(cu[-1] + new[b])
    for k in given:
        ring[(head + count) % F] = k
        count += 1
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    return [torch.from_numpy(table).cuda(), as_int(lens), as_int(cu), as_int(slots), as_int([head, count]),
            as_int([short]), torch.from_numpy(ring).cuda()]


def _exact_attend(s):
    c = s["case"]
    if work(c)["flops"] > 2e13:
        return None
    H, G, d, L = c["heads"], c["group"], c["d"], c["L"]
    N = s["Q"].shape[0]
    out = torch.zeros((N, H * G, d), dtype=torch.float64, device="cuda")
    lse = torch.full((N, H * G), -math.inf, dtype=torch.float64, device="cuda")
    cu, lens, tables = s["cu_new"].tolist(), s["lens"].tolist(), s["tables"].cpu()
    kp, vp = (s[x][s["prefix_table"].long()].double() for x in ("pool_K", "pool_V"))   # [blocks, H, L, d]
    P = c["prefix"]
    for h in range(H):
        ka, va = kp[:, h].reshape(-1, d)[:P], vp[:, h].reshape(-1, d)[:P]
        for b in range(len(lens)):
            n, length = cu[b + 1] - cu[b], lens[b]
            if n == 0:
                continue
            t = tables[b, :_blocks(length, L)].long().cuda()
            k, v = (s[x][t, h].double().reshape(-1, d)[:length] for x in ("pool_K", "pool_V"))
            for i in range(0, n, 512):
                m = min(512, n - i)
                q = s["Q"][cu[b] + i:cu[b] + i + m, h * G:(h + 1) * G].double().reshape(m * G, d)
                a = torch.cat([q @ ka.T, q @ k.T], 1) * s["scale"]
                at = torch.arange(m, device="cuda").repeat_interleave(G) + (length - n + i)
                hide = torch.arange(length, device="cuda")[None, :] > at[:, None]
                a[:, P:][hide] = -math.inf
                z = torch.logsumexp(a, 1)
                w = torch.exp(a - z[:, None])
                o = w[:, :P] @ va + w[:, P:] @ v
                out[cu[b] + i:cu[b] + i + m, h * G:(h + 1) * G] = o.reshape(m, G, d)
                lse[cu[b] + i:cu[b] + i + m, h * G:(h + 1) * G] = z.reshape(m, G)
    return [out, lse] if c["lse"] else [out]
