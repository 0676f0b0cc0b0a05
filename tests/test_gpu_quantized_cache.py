"""The 8-bit paged cache's store and load, and the norm and rotation of heads in front of it, through the C ABI."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from antfly_amd import paged  # noqa: E402
from tests import gpu_util as G  # noqa: E402
from tests import quantized_ref as R  # noqa: E402
from tests.paged_ref import narrow, to64  # noqa: E402

SHAPES = [(1, 16, 1, 16, False), (37, 16, 8, 128, False), (5, 24, 3, 80, True), (130, 1, 2, 256, True), (9, 64, 40, 64, False),
          (3, 16, 12, 192, False), (300, 8, 5, 112, False), (17, 16, 1, 96, False), (2, 16, 3, 48, True)]


def a_cache(rng, blocks, block, heads, dim, stored, outside):
    shape = (blocks, heads, block) if outside else (blocks, block, heads)
    codes = [torch.from_numpy(rng.integers(-100, 101, (*shape, dim)).astype(np.float32)).to(R.DTYPES[stored]).to(G.DEV) for _ in "kv"]
    scales = [torch.from_numpy(rng.uniform(0.001, 2, shape).astype(np.float32)).to(G.DEV) for _ in "kv"]
    return codes + scales


def by_slot(t, outside):
    """[blocks, block, ...] of a cache's tensor, as numbers."""
    a = R.numbers(t)
    return a.swapaxes(1, 2) if outside else a


def slots_of(rng, tokens, room):
    slots = rng.permutation(room)[:tokens].astype(np.int32)
    if tokens > 4:
        slots[1], slots[3], slots[4] = -1, room, 2 ** 31 - 1  # of padded tokens
    return slots


def awkward(rng, shape):
    """Normal values, heads of other sizes, of zeros, of tiny and huge values, and some that hold no numbers."""
    x = rng.standard_normal(shape).astype(np.float32) * 3
    flat = x.reshape(-1, shape[-1])
    flat[2::7] *= 1e-3
    flat[3::11] = 0
    flat[4::13] *= 1e-37
    flat[5::17, 3] = 60000
    flat[6::19, 1] = np.inf
    flat[7::23, 0] = np.nan
    flat[8::29] = -0.5  # every value the largest
    return x


def same_numbers(a, b):
    return np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.nan_to_num(a), np.nan_to_num(b))


@pytest.mark.parametrize("source", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stored", ["i8", "e4m3"])
@pytest.mark.parametrize("tokens,block,heads,dim,outside", SHAPES)
def test_store(source, stored, tokens, block, heads, dim, outside):
    """Codes and scales bit for bit; other slots stay."""
    print(f"case: store {source} to {stored} tokens={tokens} block={block} heads={heads} dim={dim} outside={outside}", flush=True)
    rng = np.random.default_rng(tokens + dim)
    blocks = tokens // block + 3
    cache = a_cache(rng, blocks, block, heads, dim, stored, outside)
    want = [by_slot(t, outside).copy() for t in cache]
    new = narrow(awkward(rng, (tokens, 2 * heads + 3, dim)), source).to(G.DEV)
    k, v = new[:, 1:1 + heads], new[:, 2 + heads:2 + 2 * heads]
    slots = slots_of(rng, tokens, blocks * block)
    paged.launchQuantizedStore(G.stream(), paged.quantizedCache(*cache, heads_outside=outside), k, v, G.to_dev(slots))
    torch.cuda.synchronize()
    for which, x in enumerate((k, v)):
        codes, scales = R.quantize(x.float().cpu().numpy(), stored)
        for i, s in enumerate(slots):
            if 0 <= s < blocks * block:
                want[which][s // block, s % block], want[2 + which][s // block, s % block] = codes[i], scales[i]
    for t, w in zip(cache, want):
        assert same_numbers(by_slot(t, outside), w)


@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stored", ["i8", "e4m3"])
@pytest.mark.parametrize("tokens,block,heads,dim,outside", SHAPES)
def test_load(out, stored, tokens, block, heads, dim, outside):
    """code * scale in f32, rounded once; slots more than once; tokens without one, and what lies around the arrays, stay."""
    print(f"case: load {stored} as {out} tokens={tokens} block={block} heads={heads} dim={dim} outside={outside}", flush=True)
    rng = np.random.default_rng(tokens + dim)
    blocks = tokens // block + 3
    cache = a_cache(rng, blocks, block, heads, dim, stored, outside)
    cache[2].view(-1)[::5] = float("nan")
    slots = slots_of(rng, tokens, blocks * block)
    if tokens > 8:
        slots[6] = slots[7]
    wide = torch.full((tokens + 2, 2 * heads + 1, dim), -7.0, dtype=R.DTYPES[out], device=G.DEV)
    k, v = wide[1:-1, :heads], wide[1:-1, heads + 1:]
    paged.launchQuantizedLoad(G.stream(), paged.quantizedCache(*cache, heads_outside=outside), k, v, G.to_dev(slots))
    torch.cuda.synchronize()
    want = torch.full(wide.shape, -7.0, dtype=R.DTYPES[out])
    for which, part in enumerate((want[1:-1, :heads], want[1:-1, heads + 1:])):
        codes, scales = (by_slot(cache[2 * n + which], outside).astype(np.float32) for n in (0, 1))
        for i, s in enumerate(slots):
            if 0 <= s < blocks * block:
                part[i] = torch.from_numpy(codes[s // block, s % block] * scales[s // block, s % block][:, None]).to(R.DTYPES[out])
    assert same_numbers(to64(wide), to64(want))


@pytest.mark.parametrize("out", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,heads,dim", [(18001, 8, 128), (60003, 8, 48), (9001, 9, 240)])
def test_load_many(out, tokens, heads, dim):
    rng = np.random.default_rng(tokens)
    cache = a_cache(rng, 20, 16, heads, dim, "i8", False)
    slots = rng.integers(-3, 330, tokens).astype(np.int32)
    k, v = (torch.full((tokens + 1, heads, dim), -7.0, dtype=R.DTYPES[out], device=G.DEV) for _ in "kv")
    paged.launchQuantizedLoad(G.stream(), paged.quantizedCache(*cache), k[:-1], v[:-1], G.to_dev(slots))
    torch.cuda.synchronize()
    there = np.append((slots >= 0) & (slots < 320), False)
    at = torch.from_numpy(np.where(there, np.append(slots, 0), 0)).long()
    for which, got in enumerate((k, v)):
        numbers = (cache[which].cpu().float() * cache[2 + which].cpu()[..., None]).view(320, heads, dim).to(R.DTYPES[out])
        want = torch.where(torch.from_numpy(there)[:, None, None], numbers[at], torch.tensor(-7.0, dtype=R.DTYPES[out]))
        assert torch.equal(got.cpu(), want)


ROTATIONS = [(1, 32, 8, 128, 128, False, 1), (37, 5, 1, 96, 48, True, 3), (130, 4, 4, 64, 64, True, 1), (7, 3, 3, 256, 256, False, 2), (3, 16, 2, 80, 40, False, 3),
             (600, 2, 1, 112, 56, False, 1), (5, 7, 1, 192, 96, True, 1), (11, 2, 2, 8, 8, False, 1), (4, 1, 1, 40, 0, False, 1), (2000, 28, 4, 128, 64, False, 2)]


def a_projection(rng, tokens, heads, kv_heads, dim, source):
    """Queries, keys and values side by side, as one product leaves them."""
    x = rng.standard_normal((tokens, heads + 2 * kv_heads, dim)) * rng.uniform(0.01, 30, (tokens, 1, 1))
    qkv = narrow(x, source).to(G.DEV)
    return qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]


def a_rotation(rng, tokens, dim, rotary, axes, norm):
    positions = rng.integers(0, 1 << 20, (axes, tokens)).astype(np.int32)
    positions[0, 0], positions[-1, -1] = 0, -1  # the last: of a padded batch
    frequencies = (10000.0 ** (-np.arange(rotary // 2) / max(1, rotary // 2))).astype(np.float32)
    weights = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) if norm else None for _ in "qk"]
    return positions, frequencies, [int(a) for a in rng.integers(0, axes, rotary // 2)], weights


def dev(a):
    return None if a is None else G.to_dev(a)


@pytest.mark.parametrize("source,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,interleaved,axes", ROTATIONS)
def test_rotation(source, out, norm, tokens, heads, kv_heads, dim, rotary, interleaved, axes):
    print(f"case: rotate {source} to {out} norm={norm} tokens={tokens} heads={heads}/{kv_heads} dim={dim} rotary={rotary} interleaved={interleaved} axes={axes}", flush=True)
    rng = np.random.default_rng(tokens + dim)
    q, k, _ = a_projection(rng, tokens, heads, kv_heads, dim, source)
    positions, frequencies, pair_axes, weights = a_rotation(rng, tokens, dim, rotary, axes, norm)
    wide = torch.full((tokens + 2, heads + kv_heads + 1, dim), -7.0, dtype=R.DTYPES[out], device=G.DEV)
    to = wide[1:-1, :heads], wide[1:-1, heads + 1:]
    paged.launchHeadRotation(G.stream(), paged.headRotation(q, k, *to, G.to_dev(positions), G.to_dev(frequencies), dev(weights[0]), dev(weights[1]),
                                                            interleaved=interleaved, pair_axes=pair_axes))
    torch.cuda.synchronize()
    assert (wide[0] == -7).all() and (wide[-1] == -7).all() and (wide[:, heads] == -7).all()
    for x, y, w in zip((q, k), to, weights):
        want = R.rotate(to64(x), w, positions, frequencies, interleaved, pair_axes)
        assert (np.abs(to64(y) - want) <= R.rotation_error(x, w, want, out, interleaved, rotary // 2)).all()


def test_rotation_in_place_and_of_keys_alone():
    rng = np.random.default_rng(1)
    q, k, _ = a_projection(rng, 9, 6, 2, 128, "bf16")
    positions, frequencies, _, weights = a_rotation(rng, 9, 128, 128, 1, True)
    fixed = [dev(positions[0]), dev(frequencies), dev(weights[0]), dev(weights[1])]
    apart = [torch.empty(9, n, 128, dtype=torch.bfloat16, device=G.DEV) for n in (6, 2)]
    paged.launchHeadRotation(G.stream(), paged.headRotation(q, k, *apart, *fixed))
    alone = torch.empty_like(apart[1])
    paged.launchHeadRotation(G.stream(), paged.headRotation(None, k, None, alone, *fixed))
    paged.launchHeadRotation(G.stream(), paged.headRotation(q, k, q, k, *fixed))
    torch.cuda.synchronize()
    assert torch.equal(q, apart[0]) and torch.equal(k, apart[1]) and torch.equal(alone, apart[1])


def test_heads_that_hold_no_numbers_stay_alone():
    rng = np.random.default_rng(2)
    q, k, _ = a_projection(rng, 6, 4, 2, 64, "f32")
    q[2, 1, 5], q[3, 0, 60], k[4, 1, 7] = float("nan"), float("inf"), -float("inf")
    positions, frequencies, _, weights = a_rotation(rng, 6, 64, 64, 1, True)
    to = [torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k)]
    paged.launchHeadRotation(G.stream(), paged.headRotation(q, k, *to, dev(positions), dev(frequencies), dev(weights[0]), dev(weights[1])))
    torch.cuda.synchronize()
    for x, y in zip((q, k), to):
        assert np.array_equal(np.isfinite(to64(x)).all(-1), np.isfinite(to64(y)).all(-1))


@pytest.mark.parametrize("source", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stored", ["f16", "bf16", "i8", "e4m3"])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,interleaved,axes", [r for r in ROTATIONS if r[3] % 16 == 0])
def test_rotated_store(source, stored, tokens, heads, kv_heads, dim, rotary, interleaved, axes):
    """Queries as by the rotation alone, values as by the stores, keys the nearest that the cache holds."""
    print(f"case: rotated store {source} to {stored} tokens={tokens} heads={heads}/{kv_heads} dim={dim} rotary={rotary}", flush=True)
    rng = np.random.default_rng(tokens + dim)
    q, k, v = a_projection(rng, tokens, heads, kv_heads, dim, source)
    positions, frequencies, pair_axes, weights = a_rotation(rng, tokens, dim, rotary, axes, True)
    block = 16
    blocks = tokens // block + 3
    coded = stored in R.LARGEST

    def make():
        if coded:
            tensors = a_cache(np.random.default_rng(5), blocks, block, kv_heads, dim, stored, False)
            return tensors, paged.quantizedCache(*tensors)
        tensors = [torch.full((blocks, block, kv_heads, dim), 3.0, dtype=R.DTYPES[stored], device=G.DEV) for _ in "kv"]
        return tensors, paged.cache(*tensors)

    slots = slots_of(rng, tokens, blocks * block)
    rest = [dev(positions), dev(frequencies), dev(weights[0]), dev(weights[1])]
    more = {"interleaved": interleaved, "pair_axes": pair_axes}
    q_out, q_alone = (torch.empty(tokens, heads, dim, dtype=R.DTYPES[source], device=G.DEV) for _ in range(2))
    k_alone = torch.empty(tokens, kv_heads, dim, dtype=R.DTYPES[source], device=G.DEV)
    tensors, cache = make()
    paged.launchRotatedStore(G.stream(), paged.headRotation(q, k, q_out, None, *rest, **more), cache, v, G.to_dev(slots))
    paged.launchHeadRotation(G.stream(), paged.headRotation(q, k, q_alone, k_alone, *rest, **more))
    apart, other = make()
    (paged.launchQuantizedStore if coded else paged.launchCacheStore)(G.stream(), other, v.contiguous(), v.contiguous(), G.to_dev(slots))
    torch.cuda.synchronize()
    assert torch.equal(q_out, q_alone)
    for n in ((1, 3) if coded else (1,)):
        assert same_numbers(R.numbers(tensors[n]), R.numbers(apart[n]))
    want = R.rotate(to64(k), weights[1], positions, frequencies, interleaved, pair_axes)
    near = R.rotation_error(k, weights[1], want, "f32", interleaved, rotary // 2)
    untouched = np.ones(blocks * block, bool)
    codes = R.numbers(tensors[0]).reshape(blocks * block, kv_heads, dim)
    scales = R.numbers(tensors[2]).reshape(blocks * block, kv_heads) if coded else None
    for i, s in enumerate(slots):
        if not 0 <= s < blocks * block:
            continue
        untouched[s] = False
        if not coded:
            assert (np.abs(codes[s] - want[i]) <= near[i] + np.abs(want[i]) * R.HALF[stored] + 2.0 ** -25).all()
            continue
        scale = np.abs(want[i]).max(-1) / float(R.LARGEST[stored])
        assert (np.abs(scales[s] - scale) <= scale * 2.0 ** -22 + near[i].max(-1) / float(R.LARGEST[stored])).all()
        # half a step: of whole numbers, or of four bits (2^-10 below the smallest normal number), and a code's own error
        step = 0.5 if stored == "i8" else np.maximum(np.abs(want[i] / scale[:, None]) * 2.0 ** -4, 2.0 ** -10)
        assert (np.abs(codes[s] * scales[s][:, None] - want[i]) <= (step * (1 + 2.0 ** -20)) * scale[:, None] + 2 * near[i] + np.abs(want[i]) * 2.0 ** -21).all()
    fresh = make()[0]
    for n, t in enumerate(tensors):
        assert np.array_equal(R.numbers(t).reshape(blocks * block, -1)[untouched], R.numbers(fresh[n]).reshape(blocks * block, -1)[untouched])


def test_far_positions():
    """Angles of positions near 2^31 keep f32's accuracy."""
    tokens = 8
    positions = np.array([0, 1, 2 ** 20 + 1, 2 ** 24 + 1, 2 ** 30 + 7, 2 ** 31 - 1, -5, -2 ** 31], np.int32)
    frequencies = np.array([1.0, 0.9999, 0.1, 3.0e-5], np.float32)
    k = torch.zeros(tokens, 1, 8, device=G.DEV)
    k[..., :4] = 1
    out = torch.empty_like(k)
    paged.launchHeadRotation(G.stream(), paged.headRotation(None, k, None, out, dev(positions), dev(frequencies)))
    torch.cuda.synchronize()
    angle = positions.astype(np.float64)[:, None] * frequencies.astype(np.float64)
    got = to64(out)[:, 0]
    # half a step of the angle's rest (at most an eighth of a turn), six roundings of the series
    assert np.abs(got[:, :4] - np.cos(angle)).max() <= 8 * 2.0 ** -24 and np.abs(got[:, 4:] - np.sin(angle)).max() <= 8 * 2.0 ** -24


def test_replayed():
    """A captured step of store and load over tokens that change, beside eager work."""
    rng = np.random.default_rng(4)
    tensors = a_cache(rng, 6, 16, 2, 64, "i8", False)
    cache = paged.quantizedCache(*tensors)
    q, k, v = (torch.empty(5, n, 64, device=G.DEV) for n in (4, 2, 2))
    positions, frequencies, _, weights = a_rotation(rng, 5, 64, 64, 1, True)
    positions, slots = dev(positions[0]), torch.empty(5, dtype=torch.int32, device=G.DEV)
    q_out, back = torch.empty_like(q), [torch.empty(5, 2, 64, dtype=torch.float16, device=G.DEV) for _ in "kv"]
    rotation = paged.headRotation(q, k, q_out, None, positions, dev(frequencies), dev(weights[0]), dev(weights[1]))

    def step():
        paged.launchRotatedStore(G.stream(), rotation, cache, v, slots)
        paged.launchQuantizedLoad(G.stream(), cache, *back, slots)

    slots.copy_(torch.arange(5))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for turn in range(4):
        for t in (q, k, v):
            t.copy_(torch.from_numpy(rng.standard_normal(tuple(t.shape)).astype(np.float32)))
        positions.copy_(torch.from_numpy(rng.integers(0, 9999, 5).astype(np.int32)))
        slots.copy_(torch.from_numpy(rng.permutation(96)[:5].astype(np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in (q_out, *back, *tensors)]
        for t in (q_out, *back):
            t.zero_()
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, (q_out, *back, *tensors))), turn
