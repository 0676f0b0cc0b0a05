"""8-bit caches, head rotation, attention over the cache and sampling from their definitions (numpy, 64 bits)."""
import numpy as np
import torch

LARGEST = {"i8": np.float32(127), "e4m3": np.float32(448)}
DTYPES = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# half a step of the last place, relative
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def quantize(x, stored):
    """(codes as f32 numbers, scales f32) of f32 [..., dim], in the f32 operations of the definition."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        most = np.maximum(np.abs(x).max(-1), np.float32(2.0 ** -100))
        scaled = x * (LARGEST[stored] / most)[..., None]
        scales = most / LARGEST[stored]
        codes = np.rint(scaled) if stored == "i8" else torch.from_numpy(scaled).to(torch.float8_e4m3fn).float().numpy()
    odd = ~np.isfinite(x).all(-1)
    codes[odd] = 0
    scales[odd] = np.nan
    return codes, scales


def numbers(codes):
    """Code tensors as f64 arrays."""
    return codes.detach().cpu().float().numpy().astype(np.float64)


def rotate(x, weight, positions, frequencies, interleaved, axes, eps=1e-6):
    """[tokens, heads, dim] f64 normed (weight) and rotated: positions [axes, tokens], axes: of every pair."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * np.asarray(weight, np.float64)
    y, pairs = x.copy(), len(frequencies)
    for p in range(pairs):
        angle = positions[axes[p]].astype(np.float64) * np.float64(frequencies[p])
        c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
        a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + pairs)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def rotation_error(x, weight, y, out, interleaved, pairs):
    """What f32 arithmetic may be off by: the mean square adds dim products one after the other in the worst order, half of its
    relative error enters the norm, and a dozen more roundings norm and turn; sine and cosine are good to 2^-22.  A pair's two
    values share their size."""
    dim = y.shape[-1]
    size = np.abs(y).copy()
    for p in range(pairs):
        a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + pairs)
        size[..., a] = size[..., b] = np.hypot(y[..., a], y[..., b])
    return size * ((dim / 2 if weight is not None else 0) + 12 + 8) * 2.0 ** -24 + np.abs(y) * HALF[out] + (2.0 ** -25 if out == "f16" else 1e-37)


def attend(q, keys, values, key_scales, value_scales, scale, starts, context, table, block, blocks, most_query, most_keys, kind, cap=0.0,
           window=0, slopes=None, digits=False):
    """(out, the largest error that the kernel's arithmetic may have), f64 [tokens, heads, dim].  keys, values: code numbers
    [blocks, block, kv heads, dim], scales beside them; kind: of query and out.

    `digits`: queries are whole numbers of 22 bits beside their row's largest value, at least 2^21: half a unit is 2^-22 of that.
    A score is off by its f32 sums (dim additions of exact products, 2^-23 each of the absolute ones), three roundings, and with a cap or
    slopes by tanh's 2^-20 of the cap and one rounding of the bias; a weight by exp's argument, exp2 (2^-22) and by its terms: half a
    step of 16 (f16, bf16) or 24 bits; the sum over keys by one rounding of 2^-23 a tile of 32 keys, 32 inside it and two a join; the
    result by half a step of its own type."""
    tokens, heads, dim = q.shape
    group = heads // keys.shape[2]
    out, off = np.full(q.shape, np.nan), np.zeros(q.shape)
    kept = {"f32": 2.0 ** -23, "f16": 2.0 ** -15, "bf16": 2.0 ** -15}[kind]
    for r in range(len(context)):
        n, c = min(int(starts[r + 1] - starts[r]), most_query), max(int(context[r]), 0)
        total = min(c + n, table.shape[1] * block, most_keys)
        at = np.arange(total)
        page = table[r, at // block]
        there = (page >= 0) & (page < blocks)
        where = (np.where(there, page, 0), at % block)
        k, v, ks, vs = keys[where], values[where], key_scales[where], value_scales[where]
        for t in range(n):
            i, position = int(starts[r]) + t, c + t
            seen = there & (at <= position) & ((window == 0) | (position - at < window))
            for h in range(heads):
                if not seen.any():
                    out[i, h] = 0
                    continue
                g = h // group
                kk, vv, row = k[seen, g] * ks[seen, g, None], v[seen, g] * vs[seen, g, None], q[i, h]
                with np.errstate(all="ignore"):
                    s = scale * (kk @ row)
                    wrong = abs(scale) * dim * 2.0 ** -23 * (np.abs(kk) @ np.abs(row)) + 2.0 ** -21 * np.abs(s)
                    if digits:
                        wrong = wrong + abs(scale) * 2.0 ** -22 * np.abs(row).max() * np.abs(kk).sum(1)
                    if cap:
                        s = cap * np.tanh(s / cap)
                        wrong = wrong + 2.0 ** -20 * cap
                    if slopes is not None:
                        s = s - slopes[h] * (position - at[seen])
                        wrong = wrong + 2.0 ** -22 * slopes[h] * (position - at[seen])
                    e = np.exp(s - s.max())
                    w = e / e.sum()
                    out[i, h] = w @ vv
                    worst = np.where(w > 1e-12, wrong, 0).max() if np.isfinite(wrong).any() else 0.0
                    each = 2 * np.expm1(np.minimum(worst, 50)) + kept + 2.0 ** -21 + (len(w) / 32 + 60) * 2.0 ** -23
                    off[i, h] = each * (w @ np.abs(vv)) + HALF[kind] * np.abs(out[i, h]) + (2.0 ** -25 if kind == "f16" else 1e-30)
    return out, off


def sample(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, its probability among the kept) of one row."""
    logits = np.where(np.isnan(logits), -np.inf, np.asarray(logits, np.float64))
    order = np.lexsort((np.arange(len(logits)), -logits))
    top = logits[order[0]]
    if top == -np.inf:
        return -1, 0.0
    if not t > 0:
        return int(order[0]), 1.0
    with np.errstate(all="ignore"):
        w = np.exp(np.where(logits[order] == top, 0.0, (logits[order] - top) / np.float64(t)))
    w = np.where(np.isnan(w), 0.0, w)
    n = min(k, len(w)) if k > 0 else len(w)
    w = w[:n]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int((before < np.float64(p) * w.sum()).sum()))
    if m > 0:
        n = max(1, min(n, int((w[:n] >= np.float64(m)).sum())))
    sums = np.cumsum(w[:n])
    u = 0.0 if not u > 0 else np.float64(u)
    at = int((sums <= u * sums[-1]).sum()) if u < 1 else int((sums < sums[-1]).sum())
    at = min(at, n - 1)
    return int(order[at]), float(w[at] / sums[-1])
