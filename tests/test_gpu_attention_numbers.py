"""Attention over a paged cache at the ends of its number types: weights far below a row's largest, queries of one large value,
scales near zero, infinities and no numbers.  Against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests import paged_ref as R  # noqa: E402
from tests.test_gpu_tree_attention import KINDS, Batch  # noqa: E402

# What a weight is off by: a part of itself, and a part of the row's largest weight; and half a unit of the result's type (and half of
# f16's smallest step, LEAST).
KEPT = {("f32", "f16"): (2.0 ** -21, 2.0 ** -44, 2.0 ** -22), ("f32", "bf16"): (2.0 ** -21, 0.0, 2.0 ** -22), ("f16", "f16"): (2.0 ** -11, 2.0 ** -32, 2.0 ** -11),
        ("bf16", "bf16"): (2.0 ** -8, 0.0, 2.0 ** -8)}
LEAST = {"f32": 1e-30, "f16": 2.0 ** -25, "bf16": 1e-30}


def want(b):
    """(out, the largest error that the kernel's arithmetic may have), f64 [tokens, heads, dim].

    A score is off by its f32 sums (dim additions, 2^-23 each of the absolute products) and, with f32 queries, by the terms of each
    query value (2^-22 of it, or 2^-39 of the row's largest); its exponent by four roundings of the score and the row's largest
    (log2 e, times the scale, the difference, 2^-24 each); a weight by exp2 (2^-22) and KEPT; sums by a rounding of 2^-23 a tile of 32 keys and
    some more.  An error e of a weight w moves the result by e (|v| + |out|)."""
    q, k, v = (R.to64(R.narrow(x, t)) for x, t in ((b.q, b.activations), (b.kv[0], b.stored), (b.kv[1], b.stored)))
    heads, dim = q.shape[1:]
    group = heads // k.shape[2]
    rel, floor, last = KEPT[b.activations, b.stored]
    out, off = np.full(q.shape, np.nan), np.zeros(q.shape)
    for r in range(len(b.context)):
        n, c = int(b.lens[r]), int(b.context[r])
        at = np.arange(c + n)
        kk, vv = (x[b.table[r, at // b.block], at % b.block] for x in (k, v))
        for t in range(n):
            seen = np.arange(c + n) <= c + t if b.tables is None else np.concatenate([np.ones(c, bool), b.tables[r][t]])
            i = int(b.starts[r]) + t
            for h in range(heads):
                if not seen.any():
                    out[i, h] = 0
                    continue
                keys, values, row = kk[seen, h // group], vv[seen, h // group], q[i, h]
                with np.errstate(all="ignore"):
                    s = b.scale * (keys @ row)
                    if (s > -np.inf).any() and not np.isnan(s).any():  # weights of zero add no error
                        keys, values, s = keys[s > -np.inf], values[s > -np.inf], s[s > -np.inf]
                    p = np.exp(s - s.max())
                    w = p / p.sum()
                    out[i, h] = w @ values
                    terms = np.maximum(2.0 ** -22 * np.abs(row), 2.0 ** -39 * np.abs(row).max()) if b.activations == "f32" else 0.0 * row
                    wrong = abs(b.scale) * (dim * 2.0 ** -23 * (np.abs(keys) @ np.abs(row)) + np.abs(keys) @ terms) + 2.0 ** -22 * (np.abs(s) + abs(s.max()))
                    each = np.expm1(wrong + wrong[s.argmax()]) + rel + 2.0 ** -22 + (len(w) / 32 + 40) * 2.0 ** -23
                    off[i, h] = (w * each + floor * w.max()) @ (np.abs(values) + np.abs(out[i, h])) + last * np.abs(out[i, h]) + LEAST[b.activations]
    return out, off


def check(b, **bounds):
    got, (expected, off) = b.run(**bounds), want(b)
    finite = np.isfinite(expected)
    assert np.array_equal(got[~finite], expected[~finite], equal_nan=True)
    assert np.isfinite(got[finite]).all()
    wrong, off = np.abs(got - expected)[finite], off[finite]
    assert (wrong <= off).all(), float((wrong / np.maximum(off, 1e-300)).max())
    return got


# One workgroup for all keys, with key groups that take tiles in turn; parts on several workgroups; many rows in one part and in several.
SHAPES = [([500], [2], 2, 1, 64), ([40000], [2], 2, 1, 64), ([3000, 150], [1, 3], 4, 2, 128), ([90, 400], [40, 64], 4, 2, 64), ([6000], [33], 8, 2, 128),
          ([2500], [5], 2, 1, 256)]


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("nats", [10.0, 14.0, 17.375, 18.0])
def test_many_small_weights_beside_a_large_one(activations, stored, shape, nats):
    """A key that leads by up to 18 nats and whose value is zero, or small: the result is the other keys'.  They score alike and have
    values of one, so what their weights lose adds up."""
    context, lens, heads, kv_heads, dim = SHAPES[shape]
    for first, size in ((True, 0.0), (False, 2.0 ** -10)):
        print(f"case: small weights {activations}/{stored} {SHAPES[shape]} {nats} nats, first={first}", flush=True)
        b = Batch(np.random.default_rng(shape), context, lens, heads, kv_heads, dim, 16, activations, stored, tree=False)
        b.scale = 0.125
        b.q[:] = 0
        b.q[..., 0] = 8
        for r, c in enumerate(context):
            at = np.arange(c + lens[r])
            b.kv[0][b.table[r, at // 16], at % 16] = 0
            b.kv[1][b.table[r, at // 16], at % 16] = 1
            p = 3 if first else c - 5
            b.kv[0][b.table[r, p // 16], p % 16, :, 0] = nats
            b.kv[1][b.table[r, p // 16], p % 16] = size
        check(b)


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_scores_of_all_sizes_beside_a_large_one(activations, stored, shape):
    """The same with scores and values that are spread out."""
    print(f"case: spread weights {activations}/{stored} {SHAPES[shape]}", flush=True)
    context, lens, heads, kv_heads, dim = SHAPES[shape]
    b = Batch(np.random.default_rng(shape), context, lens, heads, kv_heads, dim, 16, activations, stored, tree=False)
    b.kv[1][...] = np.abs(b.kv[1])
    b.q[..., 0] = 8
    b.scale = 0.125
    for r, c in enumerate(context):
        at = np.arange(c + lens[r])
        b.kv[0][b.table[r, at // 16], at % 16] *= 0.25
        b.kv[0][b.table[r, 2 // 16], 2 % 16] = 0
        b.kv[0][b.table[r, 2 // 16], 2 % 16, :, 0] = 16
        b.kv[1][b.table[r, 2 // 16], 2 % 16] = 0
    check(b)


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("shape", [([0, 40], [9, 40], 4, 2, 64), ([600], [2], 2, 1, 128), ([5000, 70], [3, 6], 4, 2, 128), ([300], [5], 2, 1, 256)])
def test_scores_that_vanish(activations, stored, shape):
    """Scales and queries so small that every seen key counts the same; keys that are not seen stay out."""
    sizes = [(1.0, 0.0), (1.0, -0.0), (1.0, 1e-42)] + ([(2.0 ** -60, 0.0), (2.0 ** -60, 1e-30), (2e-45, 0.125), (1e-38, 1e-38)] if activations != "f16" else [])
    for size, scale in sizes:
        print(f"case: vanishing scores {activations}/{stored} {shape} queries {size} scale {scale}", flush=True)
        b = Batch(np.random.default_rng(1), *shape, 16, activations, stored, spread=size)
        b.scale = scale
        b.tables[0][-1] = False
        check(b)


@pytest.mark.parametrize("activations,stored", [("f32", "f16"), ("f32", "bf16"), ("bf16", "bf16")])
def test_large_queries_under_a_small_scale(activations, stored):
    """Queries of 10^33 under a scale that brings the scores back."""
    print(f"case: small scale {activations}/{stored}", flush=True)
    b = Batch(np.random.default_rng(2), [90, 300], [7, 3], 4, 2, 128, 16, activations, stored, spread=1e33)
    b.scale = 2e-34
    check(b)


# ---- queries

@pytest.mark.parametrize("activations,stored", [("f32", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_queries_of_one_large_value(activations, stored, shape):
    """One value of a row 2^18 times the others', beside keys that have nothing there: the others keep their bits."""
    print(f"case: one large query value {activations}/{stored} {SHAPES[shape]}", flush=True)
    context, lens, heads, kv_heads, dim = SHAPES[shape]
    b = Batch(np.random.default_rng(shape), context, lens, heads, kv_heads, dim, 16, activations, stored, tree=False, spread=3.0)
    b.q[..., 5] = 2.0 ** 18
    b.kv[0][..., 5] = np.where(np.isnan(b.kv[0][..., 5]), np.nan, 0)
    check(b)


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("context", [20, 3000])
def test_a_scale_that_is_no_number(activations, stored, context):
    print(f"case: scale nan {activations}/{stored} context={context}", flush=True)
    b = Batch(np.random.default_rng(3), [context, 0], [7, 3], 4, 2, 64, 16, activations, stored)
    b.tables[1][1] = False
    b.scale = np.nan
    got = b.run()
    assert (got[8] == 0).all() and np.isnan(np.delete(got, 8, 0)).all()


# ---- infinities and no numbers that a row sees

PLACES = [([40], [9], 4, 2, 64), ([500, 30], [2, 5], 4, 2, 128), ([5000], [2], 4, 2, 128), ([3000, 200], [33, 64], 4, 2, 64), ([5000], [3], 2, 1, 256)]


@pytest.mark.parametrize("activations,stored", [("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("place", range(len(PLACES)))
@pytest.mark.parametrize("share", [0.3, 1.0])
def test_scores_of_minus_infinity(activations, stored, place, share):
    """A score of minus infinity is a weight of zero beside others, and no number where a row has no other."""
    scores_of_minus_infinity(activations, stored, place, share)


def scores_of_minus_infinity(activations, stored, place, share):
    context, lens, heads, kv_heads, dim = PLACES[place]
    print(f"case: minus infinity {activations}/{stored} {PLACES[place]} share={share}", flush=True)
    rng = np.random.default_rng(place)
    b = Batch(rng, context, lens, heads, kv_heads, dim, 16, activations, stored)
    b.q[..., 0] = 1 + np.abs(b.q[..., 0])
    for r, c in enumerate(context):
        p = np.arange(c + lens[r])
        p = p[(rng.random(len(p)) < share) | (p < c // 2)]  # all of some parts' keys
        b.kv[0][b.table[r, p // 16], p % 16, :, 0] = -np.inf
    b.tables[0][1] = False
    b.tables[0][1, 1] = True
    got = check(b)
    assert np.isnan(got).any() == (share == 1.0)


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("place", range(len(PLACES)))
def test_queries_and_keys_that_are_no_numbers(activations, stored, place):
    """A query that is none takes its own row, a key that is none the rows that see it."""
    context, lens, heads, kv_heads, dim = PLACES[place]
    print(f"case: no numbers {activations}/{stored} {PLACES[place]}", flush=True)
    b = Batch(np.random.default_rng(place), context, lens, heads, kv_heads, dim, 16, activations, stored)
    clean = b.run()
    b.q[1, heads - 1, 3] = np.nan
    got = b.run()
    assert np.isnan(got[1, heads - 1]).all()
    got[1, heads - 1] = clean[1, heads - 1]
    assert np.array_equal(got, clean)
    b.kv[0][b.table[0, 1], 5, 0, 7] = np.nan
    got = b.run()
    first, group = slice(0, lens[0]), heads // kv_heads
    assert np.isnan(got[first, :group]).all()
    got[first, :group] = clean[first, :group]
    got[1, heads - 1] = clean[1, heads - 1]
    assert np.array_equal(got, clean)


@pytest.mark.parametrize("stored", ["f16", "bf16"])
@pytest.mark.parametrize("place", range(len(PLACES)))
@pytest.mark.parametrize("share", [0.3, 1.0])
def test_f32_queries_on_scores_of_minus_infinity(stored, place, share):
    """A query value's terms agree about an infinite key, also where the value is its first term."""
    scores_of_minus_infinity("f32", stored, place, share)
    context, lens, heads, kv_heads, dim = PLACES[place]
    b = Batch(np.random.default_rng(place), context, lens, heads, kv_heads, dim, 16, "f32", stored)
    b.q[..., 3] = 2.0
    for r, c in enumerate(context):
        b.kv[0][b.table[r, 0], 1::3, :, 3] = -np.inf
    assert np.isfinite(check(b)).all()


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("place", range(len(PLACES)))
def test_infinite_values_of_the_context(activations, stored, place):
    """Values that every row sees: an infinity reaches its own dimensions with its sign, two signs make no number."""
    context, lens, heads, kv_heads, dim = PLACES[place]
    print(f"case: infinite values {activations}/{stored} {PLACES[place]}", flush=True)
    b = Batch(np.random.default_rng(place), context, lens, heads, kv_heads, dim, 16, activations, stored)
    for r in range(len(lens)):
        b.kv[1][b.table[r, 0], 3, :, 5] = np.inf
        b.kv[1][b.table[r, 1], 2, 0, 9:12] = -np.inf
        b.kv[1][b.table[r, 0], 7, :, 11] = np.inf
    got = check(b)
    assert np.isposinf(got[0, :, 5]).all() and np.isneginf(got[0, 0, 9:11]).all() and np.isnan(got[0, 0, 11])
