"""The plan of a batch and the writes of a paged key / value cache through the C ABI, bit for bit."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from antfly_amd import paged  # noqa: E402
from tests import gpu_util as G  # noqa: E402
from tests import paged_ref as R  # noqa: E402


def run_plan(context, lens, table, free, block, tokens, parents=None, words=0, blocks=(1 << 31) - 1, twice=True):
    i32 = lambda a: G.to_dev(np.asarray(a, np.int32))  # noqa: E731
    d = {"c": i32(context), "q": i32(lens), "t": i32(table), "f": i32(free)}
    starts = torch.full((len(context) + 1 + 16,), -7, dtype=torch.int32, device=G.DEV)
    slots, positions = (torch.full((tokens + 16,), -7, dtype=torch.int32, device=G.DEV) for _ in range(2))
    taken = torch.full((3,), -7, dtype=torch.int32, device=G.DEV)
    masks = torch.full((tokens + 4, words), -7, dtype=torch.int64, device=G.DEV) if words else None
    p = None if parents is None else i32(np.concatenate([parents, np.full(tokens, -1)])[:tokens])
    for _ in range(2 if twice else 1):  # the same call again gives the same result
        paged.launchBatchPlan(G.stream(), d["c"], d["q"], d["t"], d["f"], block, starts[:len(context) + 1], slots[:tokens], positions[:tokens],
                              taken[:1], parents=p, masks=None if masks is None else masks[:tokens], blocks=blocks)
    torch.cuda.synchronize()
    assert (starts[len(context) + 1:] == -7).all() and (slots[tokens:] == -7).all() and (positions[tokens:] == -7).all() and (taken[1:] == -7).all()
    assert masks is None or (masks[tokens:] == -7).all()
    return (d["t"].cpu().numpy(), starts[:len(context) + 1].cpu().numpy(), slots[:tokens].cpu().numpy(), positions[:tokens].cpu().numpy(),
            None if masks is None else masks[:tokens].cpu().numpy().view(np.uint64), int(taken[0]))


def a_table(rng, context, lens, block, columns, spare=5):
    owned = -(-np.maximum(context, 0) // block)
    needed = -(-(np.maximum(context, 0) + np.maximum(lens, 0)) // block)
    order = rng.permutation(int(owned.sum() + (needed - owned).sum()) + spare).astype(np.int32)
    table, at = np.full((len(context), columns), -1, np.int32), 0
    for r, n in enumerate(owned):
        held = min(int(n), columns)
        table[r, :held] = order[at:at + held]
        at += int(n)
    return table, order[at:]


PLANS = [(1, 16, (0, 0), (1, 1), 1, 0), (3, 16, (0, 40), (1, 9), 1, 5), (8, 16, (90, 500), (9, 24), 1, 11), (5, 24, (1, 100), (60, 130), 3, 3),
         (2, 1, (0, 30), (1, 40), 1, 2), (40, 128, (0, 900), (0, 200), 0, 0), (700, 32, (0, 300), (0, 5), 1, 40), (3, 16, (0, 5), (900, 1100), 16, 7),
         (2, 7, (3, 9), (1000, 1500), 0, 3), (8192, 16, (0, 64), (0, 3), 0, 9)]


@pytest.mark.parametrize("requests,block,context,lens,words,spare", PLANS)
@pytest.mark.parametrize("tree", [False, True])
def test_plan(requests, block, context, lens, words, spare, tree):
    print(f"case: plan requests={requests} block={block} context={context} lens={lens} words={words} tree={tree}", flush=True)
    rng = np.random.default_rng(requests + block)
    c, q = rng.integers(context[0], context[1] + 1, requests), rng.integers(lens[0], lens[1] + 1, requests)
    columns = int((-(-(c + q) // block)).max()) + 2
    table, free = a_table(rng, c, q, block, columns)
    tokens = int(q.sum()) + spare
    parents = R.parents_of(rng, q) if tree else None
    want = R.plan(c, q, table, free, block, 2 ** 31 - 1, tokens, parents, words, words > 0)
    got = run_plan(c, q, table, free, block, tokens, parents, words)
    for name, g, w in zip(("table", "starts", "slots", "positions", "masks", "taken"), got, want):
        assert g is None or np.array_equal(g, w), name
    assert (want[2][:int(q.sum())] >= 0).all()


def test_plan_of_what_does_not_fit():
    """A free list, table or token arrays that are too short, blocks that the cache has not, lengths below zero, parents that
    are no earlier tokens."""
    rng = np.random.default_rng(3)
    c, q, block = np.array([30, -4, 0, 17]), np.array([20, 10, -3, 40]), 16
    table, free = a_table(rng, c, q, block, 3)
    parents = np.array([5, 0, 2, -9, 3, 4, 100] + [1] * 63, np.int32)
    for short in (0, 2, len(free)):
        for tokens in (75, 33, 0):
            for blocks in (2 ** 31 - 1, 4):
                want = R.plan(c, q, table, free[:short], block, blocks, tokens, parents, 1, True)
                got = run_plan(c, q, table, free[:short], block, tokens, parents, 1, blocks)
                for name, g, w in zip(("table", "starts", "slots", "positions", "masks", "taken"), got, want):
                    assert np.array_equal(g, w if name != "masks" else w[:tokens]), (name, short, tokens, blocks)
    got = run_plan(np.zeros(0), np.zeros(0), np.zeros((0, 3)), free, block, 5, None, 1)
    assert got[1].tolist() == [0] and (got[2] == -1).all() and (got[3] == -1).all() and (got[4] == 0).all() and got[5] == 0


def a_cache(rng, blocks, block, heads, dim, stored, outside):
    shape = (blocks, heads, block, dim) if outside else (blocks, block, heads, dim)
    return [torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(R.TYPES[stored]).to(G.DEV) for _ in "kv"]


def bits(t):
    return t.contiguous().view(torch.int16 if t.element_size() == 2 else torch.int32).cpu().numpy()


@pytest.mark.parametrize("source", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stored", ["f16", "bf16"])
@pytest.mark.parametrize("tokens,block,heads,dim,outside", [(1, 16, 1, 8, False), (37, 16, 8, 128, False), (5, 24, 3, 80, True), (130, 1, 2, 256, True),
                                                            (9, 64, 40, 64, False), (3, 16, 12, 192, False)])
def test_store(source, stored, tokens, block, heads, dim, outside):
    print(f"case: store {source} to {stored} tokens={tokens} block={block} heads={heads} dim={dim} outside={outside}", flush=True)
    rng = np.random.default_rng(tokens + dim)
    blocks = tokens // block + 3
    cache = a_cache(rng, blocks, block, heads, dim, stored, outside)
    want = [c.clone() for c in cache]
    # keys and values as parts of one wider projection; ties, overflow, and numbers that are none
    wide = rng.standard_normal((tokens, 2 * heads + 3, dim)).astype(np.float32) * np.float32(3)
    wide.reshape(-1)[::97] = 1 + 2.0 ** -9 * 1.5
    wide.reshape(-1)[5::211] = 70000
    wide.reshape(-1)[7::499] = np.nan
    wide.reshape(-1)[11::503] = 2.0 ** -26
    new = R.narrow(wide, source).to(G.DEV)
    k, v = new[:, 1:1 + heads], new[:, 2 + heads:2 + 2 * heads]
    slots = rng.permutation(blocks * block)[:tokens].astype(np.int32)
    if tokens > 4:
        slots[1], slots[3], slots[4] = -1, blocks * block, 2 ** 31 - 1  # of padded tokens: nothing is written
    paged.launchCacheStore(G.stream(), paged.cache(*cache, heads_outside=outside), k, v, G.to_dev(slots))
    torch.cuda.synchronize()
    for i, s in enumerate(slots):
        if 0 <= s < blocks * block:
            for w, n in zip(want, (k, v)):
                b, o = divmod(int(s), block)
                (w[b, :, o] if outside else w[b, o]).copy_(n[i].to(w.dtype))
    for c, w in zip(cache, want):
        ok = bits(c) == bits(w)
        nan = torch.isnan(w.float()).cpu().numpy()
        assert np.array_equal(torch.isnan(c.float()).cpu().numpy(), nan) and (ok | nan).all()


@pytest.mark.parametrize("stored", ["f16", "bf16"])
@pytest.mark.parametrize("requests,block,heads,dim,columns", [(1, 16, 1, 8, 1), (5, 16, 8, 128, 6), (3, 7, 2, 80, 21), (20, 1, 3, 64, 9)])
def test_move(stored, requests, block, heads, dim, columns):
    """Paths of any length in place: the steps in their order, whatever they overwrite."""
    print(f"case: move {stored} requests={requests} block={block} heads={heads} dim={dim} columns={columns}", flush=True)
    rng = np.random.default_rng(requests + dim)
    context, drafts = rng.integers(0, 50, requests), columns + rng.integers(0, 12, requests)
    table, _ = a_table(rng, context + drafts, np.zeros(requests, int), block, int((context + drafts).max()) // block + 1)
    blocks = int(table.max()) + 3
    cache = a_cache(rng, blocks, block, heads, dim, stored, False)
    lens = rng.integers(0, columns + 1, requests).astype(np.int32)
    lens[0] = columns + 3  # longer than the path's row: the row
    paths = np.stack([np.sort(rng.choice(n, columns, replace=False)) for n in drafts]).astype(np.int32)
    if columns > 5:
        paths[1, 2] = -1  # moves nothing
        table[requests - 1, -1] = blocks  # a block that the cache has not
    want = [c.cpu().clone() for c in cache]
    for r in range(requests):
        for i in range(min(int(lens[r]), columns)):
            places = [(int(table[r, p // block]), p % block) for p in (context[r] + paths[r, i], context[r] + i)] if paths[r, i] >= 0 else []
            if places and all(0 <= b < blocks for b, _ in places):
                for w in want:
                    w[places[1]] = w[places[0]]
    paged.launchCacheMove(G.stream(), paged.cache(*cache), G.to_dev(table), G.to_dev(context.astype(np.int32)), G.to_dev(paths), G.to_dev(lens))
    torch.cuda.synchronize()
    for c, w in zip(cache, want):
        assert np.array_equal(bits(c), bits(w))


def test_plan_and_store_in_a_replayed_graph():
    """A step of fixed capacity, captured once: every replay reads the lengths that are there then."""
    rng = np.random.default_rng(9)
    block, heads, dim, requests, tokens = 16, 2, 64, 6, 80
    batches = []
    for _ in range(3):
        c, q = rng.integers(0, 100, requests), rng.integers(0, 13, requests)
        table, free = a_table(rng, c, q, block, 8, spare=64)
        batches.append((c, q, table, free[:20], R.parents_of(rng, q)))
    state = [torch.zeros(n, dtype=torch.int32, device=G.DEV) for n in (requests, requests, requests * 8, 20, tokens)]
    table = state[2].view(requests, 8)
    out = [torch.empty(n, dtype=torch.int32, device=G.DEV) for n in (requests + 1, tokens, tokens, 1)]
    masks = torch.empty(tokens, 1, dtype=torch.int64, device=G.DEV)
    cache = [torch.zeros(80, block, heads, dim, dtype=torch.bfloat16, device=G.DEV) for _ in "kv"]
    new = [torch.randn(tokens, heads, dim, device=G.DEV) for _ in "kv"]

    def fill(batch):
        c, q, t, f, p = batch
        for d, a in zip(state, (c, q, t, f, np.concatenate([p, np.full(tokens - len(p), -1)]))):
            d.copy_(torch.from_numpy(np.ascontiguousarray(a, np.int32).reshape(-1)))

    def step():
        paged.launchBatchPlan(G.stream(), state[0], state[1], table, state[3], block, out[0], out[1], out[2], out[3], parents=state[4], masks=masks,
                              blocks=80)
        paged.launchCacheStore(G.stream(), paged.cache(*cache), new[0], new[1], out[1])

    fill(batches[0])
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in (1, 0, 2, 1):
        fill(batches[i])
        for c in cache:
            c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        c, q, t, f, p = batches[i]
        want = R.plan(c, q, t, f, block, 80, tokens, p, 1, True)
        for g, w in zip((table, out[0], out[1], out[2]), want[:4]):
            assert np.array_equal(g.cpu().numpy(), w)
        assert np.array_equal(masks.cpu().numpy().view(np.uint64), want[4]) and int(out[3]) == want[5]
        rows = torch.zeros(80 * block, heads, dim, dtype=torch.bfloat16)
        live = want[2] >= 0
        rows[torch.from_numpy(want[2][live]).long()] = new[0].cpu().to(torch.bfloat16)[torch.from_numpy(live)]
        assert np.array_equal(bits(cache[0]), bits(rows.view(80, block, heads, dim)))


def test_strides_of_one_token_do_not_count():
    """One token's keys and values as views with different strides of the token dimension."""
    wide = torch.arange(6 * 64, dtype=torch.float32, device=G.DEV).view(1, 6, 64)
    keys, values = wide[:, :2], wide[:, 2:4].clone(memory_format=torch.contiguous_format)
    assert keys.stride() != values.stride()
    k, v = (torch.zeros(3, 4, 2, 64, dtype=torch.bfloat16, device=G.DEV) for _ in range(2))
    paged.launchCacheStore(G.stream(), paged.cache(k, v), keys, values, torch.full((1,), 6, dtype=torch.int32, device=G.DEV))
    torch.cuda.synchronize()
    assert torch.equal(k[1, 2], keys[0].bfloat16()) and torch.equal(v[1, 2], values[0].bfloat16())
    k[1, 2], v[1, 2] = 0, 0
    assert not k.any() and not v.any()


@pytest.mark.parametrize("requests,most", [(8000, 9), (8000, 70), (700, 300)])
def test_plan_of_many_requests(requests, most):
    """Both sides of where a workgroup takes more tokens."""
    rng = np.random.default_rng(requests + most)
    context, lens = rng.integers(0, 300, requests), rng.integers(0, most, requests)
    columns = 24 + most // 16
    table, free = a_table(rng, context, lens, 16, columns)
    tokens = int(lens.sum()) + 77
    parents = R.parents_of(rng, lens)
    got = run_plan(context, lens, table, free, 16, tokens, parents)
    want = R.plan(context, lens, table, free, 16, (1 << 31) - 1, tokens, parents, 0, False)
    for g, w in zip(got, want):
        assert g is None or np.array_equal(g, w)
