"""Batches over a paged cache, and the plan, store, move and attention on them from their definitions (numpy, 64 bits)."""
import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def to64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def narrow(a, name):
    """A numpy array as a torch tensor of the named type, to nearest even."""
    return torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(TYPES[name])


def starts_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)


def parents_of(rng, lens, reach=6):
    return np.concatenate([[int(rng.integers(max(-1, t - reach), t)) if t else -1 for t in range(n)] for n in lens] + [[]]).astype(np.int32)


def sees(parents, lens):
    """One [n, n] truth table a request: which new tokens a new token sees."""
    tables, at = [], 0
    for n in lens:
        table = np.zeros((n, n), bool)
        for t in range(n):
            table[t, t] = True
            p = parents[at + t]
            if 0 <= p < t:
                table[t] |= table[p]
        tables.append(table)
        at += n
    return tables


def words_of(tables, words):
    rows = []
    for table in tables:
        bits = np.zeros((len(table), words * 64), bool)
        keep = min(table.shape[1], words * 64)
        bits[:, :keep] = table[:, :keep]
        rows.append(np.packbits(bits, axis=1, bitorder="little").view(np.uint64).reshape(len(table), words))
    return np.concatenate(rows) if rows else np.zeros((0, words), np.uint64)


def plan(context, lens, table, free, block, blocks, tokens, parents, words, with_masks):
    """(table, starts, slots, positions, masks, taken) as afhip_launch_batch_plan is to write them."""
    table, context, lens = table.copy(), np.maximum(context, 0), np.maximum(lens, 0)
    starts, slots, positions = starts_of(lens), np.full(tokens, -1, np.int32), np.full(tokens, -1, np.int32)
    masks, taken, walked = np.zeros((tokens, max(words, 1)), np.uint64), 0, words * 64 if with_masks else 1024
    for r, (c, n) in enumerate(zip(context, lens)):
        owned, needed = -(-int(c) // block), -(-(int(c) + int(n)) // block)
        for t in range(n):
            i, position = int(starts[r]) + t, int(c) + t
            if i >= tokens:
                continue
            column = position // block
            if column < table.shape[1]:
                if column >= owned and position % block == 0:
                    where = taken + column - owned
                    table[r, column] = free[where] if where < len(free) else -1
                b = int(table[r, column]) if column < owned else (int(free[taken + column - owned]) if taken + column - owned < len(free) else -1)
                if 0 <= b < blocks and b * block + position % block < 2 ** 31:
                    slots[i] = b * block + position % block
            depth = t
            if parents is not None:
                depth, line, at = 0, [], t
                if t < walked:
                    line = [t]
                    while 0 <= parents[starts[r] + at] < at:
                        at = int(parents[starts[r] + at])
                        line.append(at)
                    depth = len(line) - 1
            else:
                line = range(t + 1) if t < walked else []
            for p in line:
                if p < words * 64:
                    masks[i, p // 64] |= np.uint64(1 << (p % 64))
            positions[i] = c + depth
        taken += needed - owned
    return table, starts, slots, positions, masks, taken


def attend(q, keys, values, scale, starts, context, table, block, blocks, tables, max_query, max_keys, terms):
    """(out, the largest error that the kernel's arithmetic may have), f64 [tokens, heads, dim].  keys, values: f64 [blocks, block,
    kv heads, dim]; tables: what sees() gives, or None; terms: how the weights are kept: "f32" to 2^-17 at least, "bf16" and "f16" to half a unit of their 8 and 11 bits, 2^-8 and 2^-11.

    A score is off by its f32 sums (dim additions, 2^-23 each of the absolute products) and by the queries' terms (2^-22 of
    the row's largest value, f32 only); a weight by exp's argument, by exp2 (2^-22) and by its own terms; the sum over keys
    by one rounding of 2^-23 a tile of 32 keys and 32 inside it; the result by half a unit of its own type."""
    tokens, heads, dim = q.shape
    group = heads // keys.shape[2]
    out, off = np.full(q.shape, np.nan), np.zeros(q.shape)
    kept, last = {"f32": (2.0 ** -17, 2.0 ** -22), "bf16": (2.0 ** -8, 2.0 ** -8), "f16": (2.0 ** -11, 2.0 ** -11)}[terms]
    for r in range(len(context)):
        n = min(int(starts[r + 1] - starts[r]), max_query)
        c = max(int(context[r]), 0)
        total = min(c + n, table.shape[1] * block, max_keys)
        at = np.arange(total)
        page = table[r, at // block]
        there = (page >= 0) & (page < blocks)
        k, v = (x[np.where(there, page, 0), at % block] for x in (keys, values))
        for t in range(n):
            seen = there.copy()
            for j in range(c, total):
                p = j - c
                seen[j] &= (p <= t) if tables is None else bool(p < tables[r].shape[1] and tables[r][t, p])
            i = int(starts[r]) + t
            for h in range(heads):
                if not seen.any():
                    out[i, h] = 0
                    continue
                kk, vv, row = k[seen, h // group], v[seen, h // group], q[i, h]
                with np.errstate(all="ignore"):
                    s = scale * (kk @ row)
                    e = np.exp(s - s.max())
                    w = e / e.sum()
                    out[i, h] = w @ vv
                    wrong = abs(scale) * (dim * 2.0 ** -23 * (np.abs(kk) @ np.abs(row)) + (2.0 ** -22 * np.abs(row).max() * np.abs(kk).sum(1) if terms == "f32" else 0.0))
                    each = 2 * np.expm1(np.minimum(wrong.max(), 50)) + kept + 2.0 ** -21 + (len(w) / 32 + 40) * 2.0 ** -23
                    off[i, h] = each * (w @ np.abs(vv)) + last * np.abs(out[i, h]) + 1e-30
    return out, off
