"""Attention of drafted trees, chains and single tokens over a paged cache through the C ABI against 64 bits."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from antfly_amd import paged  # noqa: E402
from tests import gpu_util as G  # noqa: E402
from tests import paged_ref as R  # noqa: E402


class Batch:
    """Requests with `context` cached and `lens` new tokens; every slot that no token has holds NaN."""

    def __init__(self, rng, context, lens, heads, kv_heads, dim, block, activations, stored, tree=True, words=None, outside=False, strided=False,
                 spread=1.0, spare_tokens=0):
        self.context, self.lens, self.block, self.outside = np.array(context), np.array(lens), block, outside
        self.starts, requests = R.starts_of(lens), len(lens)
        total = self.context + self.lens
        columns = max(1, int((-(-total // block)).max()))
        held = -(-total // block)
        order = rng.permutation(int(held.sum()) + 2).astype(np.int32)
        self.blocks, self.table, at = len(order), np.full((requests, columns), -1, np.int32), 0
        for r in range(requests):
            self.table[r, :held[r]] = order[at:at + held[r]]
            at += held[r]
        self.kv = [np.full((self.blocks, block, kv_heads, dim), np.nan, np.float32) for _ in "kv"]
        for x in self.kv:
            for r in range(requests):
                p = np.arange(total[r])
                x[self.table[r, p // block], p % block] = rng.standard_normal((total[r], kv_heads, dim))
        self.stored, self.activations, self.tokens = stored, activations, int(self.starts[-1]) + spare_tokens
        self.q = (rng.standard_normal((self.tokens, heads, dim)) * spread).astype(np.float32)
        self.words = words if words is not None else max(1, -(-int(max(lens)) // 64))
        self.tables = R.sees(R.parents_of(rng, lens), lens) if tree else None
        self.strided, self.scale = strided, dim ** -0.5

    def run(self, max_query=None, max_keys=None, before=None):
        kv = [R.narrow(x.transpose(0, 2, 1, 3) if self.outside else x, self.stored).to(G.DEV) for x in self.kv]
        q = R.narrow(self.q, self.activations).to(G.DEV)
        tokens, heads, dim = q.shape
        if self.strided:  # a part of a fused projection, and a result with the tokens inside
            wide = torch.full((tokens, heads + 2, dim), float("nan"), dtype=q.dtype, device=G.DEV)
            wide[:, 1:-1] = q
            q = wide[:, 1:-1]
            whole = torch.full((heads, tokens + 2, dim), float("nan"), dtype=q.dtype, device=G.DEV)
            out = whole[:, 1:-1].transpose(0, 1)
        else:
            whole = torch.full((tokens + 2, heads, dim), float("nan"), dtype=q.dtype, device=G.DEV)
            out = whole[1:-1]
        masks = None
        if self.tables is not None:
            rows = np.zeros((tokens, self.words), np.uint64)
            rows[:int(self.starts[-1])] = R.words_of(self.tables, self.words)
            masks = G.to_dev(rows.view(np.int64))
        i32 = lambda a: G.to_dev(np.asarray(a, np.int32))  # noqa: E731
        call = paged.treeAttention(paged.cache(*kv, heads_outside=self.outside), out, q, i32(self.starts), i32(self.context), i32(self.table),
                                   max_query or int(self.lens.max()), max_keys or int((self.context + self.lens).max()), masks=masks, scale=self.scale)
        size = paged.treeAttentionWorkspaceBytes(call)
        ws = torch.full((size + 256,), 0xFF, dtype=torch.uint8, device=G.DEV)
        paged.launchTreeAttention(G.stream(), call, ws[:size] if size else paged.NO_BUFFER)
        torch.cuda.synchronize()
        assert bool((ws[size:] == 0xFF).all())
        got = R.to64(out)
        guard = torch.cat([whole[:, 0].reshape(-1), whole[:, -1].reshape(-1)]) if self.strided else torch.cat([whole[0].reshape(-1), whole[-1].reshape(-1)])
        assert bool(torch.isnan(guard).all())
        return got

    def want(self, max_query=None, max_keys=None):
        q, k, v = R.to64(R.narrow(self.q, self.activations)), R.to64(R.narrow(self.kv[0], self.stored)), R.to64(R.narrow(self.kv[1], self.stored))
        tables = self.tables
        if tables is not None:
            tables = [t[:, :self.words * 64] for t in tables]
        return R.attend(q, k, v, self.scale, self.starts, self.context, self.table, self.block, self.blocks, tables, max_query or int(self.lens.max()),
                        max_keys or int((self.context + self.lens).max()), self.activations if self.activations == "f32" else self.stored)

    def check(self, **bounds):
        got, (want, off) = self.run(**bounds), self.want(**bounds)
        real = ~np.isnan(want)
        assert np.array_equal(np.isnan(got), ~real)
        assert (np.abs(got - want)[real] <= off[real]).all(), float((np.abs(got - want)[real] / off[real]).max())
        norm = np.linalg.norm(want[real])
        most = {"f32": 1e-5, "bf16": 5e-3, "f16": 1e-3}[self.activations]
        assert np.linalg.norm((got - want)[real]) <= most * norm, float(np.linalg.norm((got - want)[real]) / norm)
        return got


KINDS = [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]
CASES = [  # context, lens, heads, kv heads, dim, block
    ([0], [1], 1, 1, 8, 16),
    ([701], [5], 8, 2, 128, 16),
    ([0, 3, 100, 31, 32], [1, 7, 13, 1, 33], 4, 2, 64, 16),
    ([300, 17, 0], [24, 1, 9], 14, 2, 128, 24),
    ([65, 0], [64, 61], 8, 1, 96, 5),
    ([511, 40], [3, 2], 12, 12, 80, 32),
    ([130, 5], [10, 19], 7, 1, 192, 7),
    ([257, 1], [6, 31], 10, 2, 256, 128),
    ([90], [130], 2, 1, 64, 16),
]


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("tree", [True, False])
def test_attention(activations, stored, case, tree):
    print(f"case: attention {activations}/{stored} {CASES[case]} tree={tree}", flush=True)
    rng = np.random.default_rng(case)
    Batch(rng, *CASES[case], activations, stored, tree=tree, outside=case % 2 == 1, strided=case % 3 == 2, spread=1.0 + case).check()


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("group", [1, 4, 7])
def test_long_contexts_are_shared_out(activations, stored, group):
    """Few rows on long contexts, one far shorter than the bound: parts on several workgroups and their join."""
    print(f"case: long {activations}/{stored} group={group}", flush=True)
    rng = np.random.default_rng(group)
    Batch(rng, [5000, 20, 1333], [3, 4, 1], group * 2, 2, 128, 16, activations, stored, spread=2.0).check(max_query=6, max_keys=9000)


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_as_many_parts_as_a_row_can_have(activations, stored, dim):
    """More than 32 of a row's parts hold keys: those of the joining wavefront's upper lanes count too."""
    print(f"case: many parts {activations}/{stored} dim={dim}", flush=True)
    Batch(np.random.default_rng(dim), [15900], [2], 2, 1, dim, 16, activations, stored).check()


@pytest.mark.parametrize("requests,context,tokens,heads,kv_heads", [(200, (0, 90), (1, 3), 16, 1), (130, (1200, 1500), (1, 2), 2, 1), (1100, (0, 60), (1, 2), 24, 1),
                                                                    (70, (900, 1030), (1, 1), 2, 2)])
def test_many_requests(requests, context, tokens, heads, kv_heads):
    """More requests than a wavefront has lanes, and more than are evened out; ragged, some without new tokens."""
    print(f"case: {requests} requests context={context} tokens={tokens} heads={heads}", flush=True)
    rng = np.random.default_rng(requests)
    lens = rng.integers(tokens[0], tokens[1] + 1, requests)
    lens[[3, requests // 2]] = 0
    lens[5] = tokens[1]
    Batch(rng, rng.integers(context[0], context[1] + 1, requests), lens, heads, kv_heads, 64, 16, "f32", "bf16").check(
        max_query=tokens[1] + 1, max_keys=context[1] + tokens[1])


@pytest.mark.parametrize("requests,context,tokens,heads,kv_heads,dim", [
    (100, (0, 1500), (17, 40), 4, 1, 64), (3, (900, 2600), (33, 64), 32, 8, 128), (16, (0, 900), (40, 64), 16, 4, 64), (70, (300, 700), (30, 33), 32, 4, 64),
    (12, (500, 1000), (1, 1), 32, 8, 128), (40, (0, 1900), (1, 4), 32, 8, 64)])
def test_ragged_batches_of_many_rows(requests, context, tokens, heads, kv_heads, dim):
    """Parts that fill one round of workgroups, batches that fill more, and single workgroups on a thousand keys and more."""
    print(f"case: {requests} requests context={context} tokens={tokens} heads={heads}/{kv_heads}", flush=True)
    rng = np.random.default_rng(requests + heads)
    lens = rng.integers(tokens[0], tokens[1] + 1, requests)
    lens[requests // 2] = 0
    lens[0] = tokens[1]
    Batch(rng, rng.integers(context[0], context[1] + 1, requests), lens, heads, kv_heads, dim, 16, "bf16", "bf16").check(
        max_query=tokens[1], max_keys=context[1] + tokens[1])


@pytest.mark.parametrize("activations,stored", KINDS)
def test_prompt_without_masks(activations, stored):
    """Hundreds of new tokens behind a short context: causal, many row tiles."""
    print(f"case: prompt {activations}/{stored}", flush=True)
    Batch(np.random.default_rng(1), [37, 0], [300, 129], 4, 2, 64, 16, activations, stored, tree=False).check()


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_that_see_nothing_and_holes(activations, stored, dim):
    """Empty masks, with and without a context; table entries that name no block inside a context; a request of nothing but
    holes; tokens past the batch (not written)."""
    print(f"case: holes {activations}/{stored} dim={dim}", flush=True)
    rng = np.random.default_rng(dim)
    b = Batch(rng, [0, 100, 64, 0], [9, 5, 4, 3], 4, 2, dim, 16, activations, stored, spare_tokens=3)
    b.tables[0][4], b.tables[0][8], b.tables[1][2] = False, False, False
    b.tables[0][5] = np.eye(9, dtype=bool)[1]  # not itself
    b.table[1, 2], b.table[1, 5] = -1, 10 ** 6
    b.table[2, :] = -1
    got = b.check()
    assert (got[4] == 0).all() and (got[8] == 0).all() and (got[14:18] == 0).all() and np.isnan(got[-3:]).all()


@pytest.mark.parametrize("activations,stored", KINDS)
@pytest.mark.parametrize("context", [0, 20, 64, 700])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_what_is_not_seen_does_not_count(activations, stored, context, what):
    """Keys and values of one draft branch are no finite numbers: rows outside it have the values that they would have had."""
    print(f"case: unseen {activations}/{stored} context={context} {what}", flush=True)
    rng = np.random.default_rng(context)
    b = Batch(rng, [context, 3], [40, 5], 8, 2, 128, 16, activations, stored)
    clean = b.run()
    bad = np.array([b.tables[0][t, [7, 30]].any() for t in range(40)] + [False] * 5)
    for draft in (7, 30):
        p = context + draft
        for x in b.kv:
            x[b.table[0, p // 16], p % 16, :, 5:90:3] = what
    got = b.run()
    assert bad.any() and not bad.all()
    assert np.array_equal(got[~bad], clean[~bad])
    assert not np.isfinite(got[bad]).all(axis=(1, 2)).any()
    # values alone: seen by a row, an infinity reaches exactly its own dimensions
    b.kv[0][np.isnan(b.kv[0]) | np.isinf(b.kv[0])] = 0.25
    got, (want, off) = b.run(), b.want()
    finite = np.isfinite(want)
    assert np.array_equal(np.isfinite(got), finite) and (np.abs(got - want)[finite] <= off[finite]).all()
    if np.isinf(what):
        assert (got[~finite] == what).all()


@pytest.mark.parametrize("activations,stored", [("f32", "f16"), ("f32", "bf16")])
@pytest.mark.parametrize("size", [2.0 ** -30, 1e-3, 300.0, 2.0 ** 40])
def test_f32_queries_of_any_size(activations, stored, size):
    """Queries far from one (2^40 is past what f16 can hold) under a scale that brings the scores back."""
    print(f"case: query size {stored} {size}", flush=True)
    b = Batch(np.random.default_rng(8), [90, 300], [7, 3], 4, 2, 128, 16, activations, stored, spread=size)
    b.scale = 0.2 / size
    b.check()


@pytest.mark.parametrize("activations,stored", KINDS)
def test_scores_far_apart_and_equal(activations, stored):
    """One key that outweighs all others, late in the context; scores that are all the same."""
    print(f"case: scores {activations}/{stored}", flush=True)
    rng = np.random.default_rng(4)
    b = Batch(rng, [600], [4], 2, 1, 128, 16, activations, stored, spread=3.0)
    b.kv[0][b.table[0, 555 // 16], 555 % 16, 0] = 3 * b.q[1, 0] / np.abs(b.q[1, 0]).max()
    b.check()
    b.q[:] = 0
    b.check()
    b.scale = -0.3
    b.q[:] = rng.standard_normal(b.q.shape)
    b.check()


def test_parts_of_a_bound_that_is_too_small():
    """Keys past max_key_len and tokens past max_query_len are left out; nothing else changes."""
    b = Batch(np.random.default_rng(6), [400, 50], [5, 3], 4, 2, 64, 16, "f32", "f16", tree=False)
    got, (want, off) = b.run(max_query=4, max_keys=300), b.want(max_query=4, max_keys=300)
    assert np.isnan(got[4]).all() and np.isnan(want[4]).all()
    rest = [0, 1, 2, 3, 5, 6, 7]
    assert (np.abs(got - want)[rest] <= off[rest]).all()


@pytest.mark.parametrize("context,words", [([100, 700], 1), ([4000, 10], 1)])
def test_other_stream_and_replayed_graph(context, words):
    """The launches follow the stream that they are given; a captured call reads the lengths, masks and queries of each replay."""
    rng = np.random.default_rng(2)
    batches = [Batch(rng, np.array(context) - 3 * i, [7 - i, 3 + i], 8, 2, 128, 16, "bf16", "bf16") for i in range(3)]
    expected = [b.run(max_query=8, max_keys=max(context) + 8) for b in batches]
    blocks = max(b.blocks for b in batches)
    kv = [torch.zeros(blocks, 16, 2, 128, dtype=torch.bfloat16, device=G.DEV) for _ in "kv"]
    q, out = (torch.zeros(10, 8, 128, dtype=torch.bfloat16, device=G.DEV) for _ in "qo")
    starts, lens = torch.zeros(3, dtype=torch.int32, device=G.DEV), torch.zeros(2, dtype=torch.int32, device=G.DEV)
    table = torch.full((2, max(b.table.shape[1] for b in batches)), -1, dtype=torch.int32, device=G.DEV)
    masks = torch.zeros(10, words, dtype=torch.int64, device=G.DEV)
    call = paged.treeAttention(paged.cache(*kv), out, q, starts, lens, table, 8, max(context) + 8, masks=masks)
    size = paged.treeAttentionWorkspaceBytes(call)
    ws = torch.empty(max(size, 256), dtype=torch.uint8, device=G.DEV)

    def fill(b):
        for d, s in zip(kv, b.kv):
            d[:b.blocks] = R.narrow(s, "bf16").to(G.DEV)
        q.copy_(R.narrow(b.q, "bf16"))
        starts.copy_(torch.from_numpy(b.starts))
        lens.copy_(torch.from_numpy(b.context.astype(np.int32)))
        table[:, :b.table.shape[1]] = G.to_dev(b.table)
        masks.copy_(torch.from_numpy(R.words_of(b.tables, words).view(np.int64)))
        out.fill_(float("nan"))

    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        fill(batches[1])
        paged.launchTreeAttention(G.stream(), call, ws)
        copied = out.clone()
    side.synchronize()
    assert np.array_equal(R.to64(copied), expected[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.launchTreeAttention(G.stream(), call, ws)
    for i in (0, 1, 2, 0):
        fill(batches[i])
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(R.to64(out), expected[i])


def test_offsets_past_32_bits():
    """A cache whose last blocks lie more than 2^32 bytes (and 2^31 elements) behind its first."""
    print("case: far blocks", flush=True)
    block, dim, blocks = 16, 64, 140000  # 16 heads: 32 KiB a block, 4.3 GiB a tensor
    kv = [torch.zeros(blocks, block, 16, dim, dtype=torch.float16, device=G.DEV) for _ in "kv"]
    rng = np.random.default_rng(7)
    table = np.array([[blocks - 1, 3, blocks - 2, 131073]], np.int32)
    content = [rng.standard_normal((4, block, 16, dim)).astype(np.float32) for _ in "kv"]
    for d, s in zip(kv, content):
        d[torch.from_numpy(table[0]).long().to(G.DEV)] = R.narrow(s, "f16").to(G.DEV)
    new = [rng.standard_normal((2, 16, dim)).astype(np.float32) for _ in "kv"]
    slots = np.array([(blocks - 2) * block + 5, 131073 * block + 9], np.int32)
    cache = paged.cache(*kv)
    paged.launchCacheStore(G.stream(), cache, G.to_dev(new[0]), G.to_dev(new[1]), G.to_dev(slots))
    for s, n in zip(content, new):
        s[2, 5], s[3, 9] = n[0], n[1]
    q = rng.standard_normal((1, 16, dim)).astype(np.float32)
    out = torch.empty(1, 16, dim, device=G.DEV)
    i32 = lambda a: G.to_dev(np.asarray(a, np.int32))  # noqa: E731
    call = paged.treeAttention(cache, out, G.to_dev(q), i32([0, 1]), i32([63]), i32(table), 1, 64)
    size = paged.treeAttentionWorkspaceBytes(call)
    ws = torch.empty(max(size, 256), dtype=torch.uint8, device=G.DEV)
    paged.launchTreeAttention(G.stream(), call, ws)
    torch.cuda.synchronize()
    k, v = (R.to64(R.narrow(s, "f16")) for s in content)
    want, off = R.attend(q.astype(np.float64), k, v, dim ** -0.5, [0, 1], [63], np.arange(4)[None, :], block, 4, None, 1, 64, "f32")
    assert (np.abs(R.to64(out) - want) <= off).all()
