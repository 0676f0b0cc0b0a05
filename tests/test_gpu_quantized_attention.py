"""Attention over the 8-bit paged cache against its definition in 64 bits, through the C ABI."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from antfly_amd import paged  # noqa: E402
from tests import gpu_util as G  # noqa: E402
from tests import quantized_ref as R  # noqa: E402
from tests.paged_ref import narrow, starts_of, to64  # noqa: E402
from tests.test_gpu_quantized_cache import a_cache, by_slot  # noqa: E402


def a_batch(rng, context, new, block, heads, kv_heads, dim, kind, stored, outside=False, garbage=True):
    context, new = np.asarray(context), np.asarray(new)
    held = -(-(context + new) // block)
    blocks = int(held.sum()) + 3
    tensors = a_cache(rng, blocks, block, kv_heads, dim, stored, outside)
    for t in tensors[2:]:
        t *= 0.02
    order = rng.permutation(blocks).astype(np.int32)
    table, at = np.full((len(context), int(held.max()) + 2), -1, np.int32), 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += int(n)
    if garbage:  # what no request holds: no numbers, in codes and scales
        for r, n in enumerate(context + new):
            end = table[r, (n - 1) // block] if n else 0
            spoil(tensors, [b for b in order[at:]], slice(None), outside, stored)
            if n and n % block:
                spoil(tensors, [end], slice(n % block, None), outside, stored)
    tokens = int(new.sum())
    q = narrow(rng.standard_normal((tokens, heads, dim)) * rng.uniform(0.3, 2.0, (tokens, heads, 1)), kind).to(G.DEV)
    return {"tensors": tensors, "table": table, "context": context.astype(np.int32), "starts": starts_of(new), "q": q, "block": block, "blocks": blocks,
            "outside": outside, "kind": kind, "most": (int(new.max()) if len(new) else 1, int((context + new).max()) if len(new) else 1)}


def spoil(tensors, blocks, slots, outside, stored):
    for n, t in enumerate(tensors):
        for b in blocks:
            part = (t[int(b)].transpose(0, 1) if outside else t[int(b)])[slots]
            if n >= 2:
                part.fill_(float("nan"))
            elif stored == "e4m3":
                part.view(torch.uint8).fill_(0x7F)


def attend(b, most=None, out=None, **how):
    cache = paged.quantizedCache(*b["tensors"], heads_outside=b["outside"])
    out = torch.full(b["q"].shape, -7.0, dtype=b["q"].dtype, device=G.DEV) if out is None else out
    arrays = [G.to_dev(b[n]) for n in ("starts", "context", "table")]
    slopes = how.pop("slopes", None)
    call = paged.quantizedAttention(cache, out, b["q"], *arrays, *(most or b["most"]), slopes=None if slopes is None else G.to_dev(slopes), **how)
    workspace = torch.full((paged.quantizedAttentionWorkspaceBytes(call),), 0xFF, dtype=torch.uint8, device=G.DEV)
    paged.launchQuantizedAttention(G.stream(), call, workspace)
    torch.cuda.synchronize()
    return out


def check(b, most=None, scale=None, cap=0.0, window=0, slopes=None):
    got = to64(attend(b, most, scale=scale, softcap=cap, window=window, slopes=slopes))
    keys, values, ks, vs = (by_slot(t, b["outside"]) for t in b["tensors"])
    want, off = R.attend(to64(b["q"]), keys, values, ks, vs, b["q"].shape[2] ** -0.5 if scale is None else scale, b["starts"], b["context"], b["table"], b["block"],
                         b["blocks"], *(most or b["most"]), b["kind"], cap, window, None if slopes is None else slopes.astype(np.float64),
                         b["tensors"][0].dtype == torch.int8)
    left = np.isnan(want) & (got == -7)  # tokens past max_query_len are left as they were
    assert np.array_equal(np.isnan(got), np.isnan(want) & ~left)
    wrong = np.where(np.isnan(want), 0, np.abs(got - want)) > off
    assert not wrong.any(), (np.argwhere(wrong)[:4], np.abs(got - want)[wrong][:4], off[wrong][:4])


CASES = [([0], [1], 16, 1, 1, 16), ([1], [1], 16, 4, 1, 64), ([31], [1], 16, 8, 2, 128), ([700], [1], 16, 32, 8, 128), ([63, 0, 5000, 301], [1, 1, 1, 1], 24, 6, 2, 96),
         ([100, 0, 33], [5, 17, 1], 1, 3, 3, 80), ([2000, 17], [3, 40], 8, 16, 2, 256), ([9000], [2], 64, 20, 4, 112), ([300] * 70, [1] * 70, 32, 2, 1, 64),
         ([129, 1, 640, 12], [0, 3, 0, 7], 7, 10, 2, 192), ([4], [300], 16, 4, 2, 48)]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stored", ["i8", "e4m3"])
@pytest.mark.parametrize("context,new,block,heads,kv_heads,dim", CASES)
def test_attention(kind, stored, context, new, block, heads, kv_heads, dim):
    print(f"case: attention {kind} on {stored} context={context[:4]} new={new[:4]} block={block} heads={heads}/{kv_heads} dim={dim}", flush=True)
    rng = np.random.default_rng(sum(context) + dim)
    check(a_batch(rng, context, new, block, heads, kv_heads, dim, kind, stored, outside=dim % 32 == 0))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stored", ["i8", "e4m3"])
@pytest.mark.parametrize("cap,window,bias", [(30.0, 0, False), (0.0, 1, False), (0.0, 37, False), (50.0, 700, True), (0.0, 4096, True), (5.0, 32, False), (0.0, 0, True)])
def test_capped_biased_windowed(kind, stored, cap, window, bias):
    print(f"case: attention {kind} on {stored} cap={cap} window={window} bias={bias}", flush=True)
    rng = np.random.default_rng(window + 3)
    slopes = (2.0 ** -np.arange(1, 11)).astype(np.float32) if bias else None
    for context, new in (([600, 0, 5000], [1, 1, 1]), ([40, 2500], [9, 6])):
        b = a_batch(rng, context, new, 24, 10, 2, 96, kind, stored)
        b["q"] *= 4  # scores that a cap bends
        check(b, cap=cap, window=window, slopes=slopes)


@pytest.mark.parametrize("kind,stored", [("f32", "e4m3"), ("bf16", "i8"), ("f16", "e4m3")])
@pytest.mark.parametrize("context,new,block,heads,kv_heads,dim", [([140000], [1], 64, 2, 1, 64), ([20000], [1], 16, 2, 1, 256), ([3000, 700, 2500], [1, 2, 1], 16, 8, 8, 256),
                                                                  ([1000 + 50 * r for r in range(16)], [3] * 16, 24, 20, 4, 96), ([3300] * 17, [1] * 17, 16, 8, 8, 32)])
def test_shared_out(kind, stored, context, new, block, heads, kv_heads, dim):
    """Keys over hundreds of workgroups, over tens, and wavefronts in pairs."""
    print(f"case: shared out {kind} on {stored} context={context[:4]} new={new[:4]} heads={heads}/{kv_heads} dim={dim}", flush=True)
    check(a_batch(np.random.default_rng(dim), context, new, block, heads, kv_heads, dim, kind, stored))


def test_bounds_of_the_launch():
    """New tokens past max_query_len and keys past max_key_len are left out; lengths below zero count as zero; a table that is
    too short, and blocks that there are not, are not seen."""
    rng = np.random.default_rng(9)
    b = a_batch(rng, [100, 50, 300], [6, 2, 4], 16, 8, 2, 64, "f32", "i8", garbage=False)
    check(b)
    check(b, most=(3, 304))
    check(b, most=(6, 120))
    b["table"][2, 3], b["table"][2, 5], b["table"][0, 0] = -1, b["blocks"], 2 ** 31 - 1
    check(b)
    b["table"] = np.ascontiguousarray(b["table"][:, :9])
    check(b)
    b["table"][:] = -1  # nothing is seen
    check(b)
    b["context"][1] = -5
    check(b)
    assert attend(b, most=(6, 0)).abs().max() == 0


def test_many_requests():
    """More requests than a wavefront has lanes, a few of them long, some without new tokens; and more than are shared out."""
    rng = np.random.default_rng(14)
    new = [int(n) for n in rng.integers(0, 3, 150)]
    check(a_batch(rng, [3000 if r % 41 == 7 else int(rng.integers(0, 60)) for r in range(150)], new, 16, 4, 2, 64, "f32", "e4m3"))
    check(a_batch(rng, [1100 if r == 1050 else r % 3 for r in range(1100)], [1] * 1100, 16, 2, 1, 64, "bf16", "i8", garbage=False))


def test_single_scores():
    """A scale of zero, a negative one, scores far apart, and a row whose scores all overflow to minus infinity."""
    rng = np.random.default_rng(10)
    for kind in ("f32", "bf16"):
        b = a_batch(rng, [333], [2], 16, 4, 2, 128, kind, "e4m3")
        check(b, scale=0.0)
        check(b, scale=-0.3)
        b["q"] *= 30
        check(b)
    b = a_batch(rng, [40], [1], 16, 1, 1, 16, "f32", "i8")
    for t in b["tensors"][:2]:
        t.fill_(-100)
    b["q"].fill_(1e37)
    assert torch.isnan(attend(b, scale=1e3)).all()


def test_no_numbers_where_nothing_looks():
    """A draft's key and value that are no numbers, and infinite scales, do not reach the tokens before it; nor a row's query the
    other rows."""
    for stored in ("i8", "e4m3"):
        for kind in ("f32", "f16", "bf16"):
            rng = np.random.default_rng(11)
            b = a_batch(rng, [45], [4], 16, 6, 2, 64, kind, stored)
            clean = attend(b)
            spoil(b["tensors"], [b["table"][0, 47 // 16]], slice(47 % 16, None), False, stored)  # new tokens 2 and 3
            got = attend(b)
            assert torch.equal(got[:2], clean[:2]) and torch.isnan(got[2:]).all()
            b["q"][0, 3, 5] = float("nan")
            got = attend(b)
            assert torch.isnan(got[0, 3]).all() and torch.equal(got[0, :3], clean[0, :3]) and torch.equal(got[1], clean[1])


def test_codes_that_are_no_numbers():
    """In one value of an e4m3 token: that value of the rows that see it, in tiles that all of them see and in others."""
    rng = np.random.default_rng(12)
    b = a_batch(rng, [100], [3], 16, 4, 2, 128, "bf16", "e4m3")
    clean = attend(b)
    for key, sees in ((7, 0), (101, 1)):
        where = b["tensors"][1].view(torch.uint8)[int(b["table"][0, key // 16]), key % 16, 1]
        held = int(where[77])
        where[77] = 0xFF
        got = attend(b)
        where[77] = held
        bad = torch.isnan(got)
        assert bad[sees:, 2:, 77].all() and int(bad.sum()) == 2 * (3 - sees) and torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("lens", [[1], [5000], [100, 2000, 7]])
def test_strides_streams_and_replays(lens):
    """Queries and results as parts of wider arrays, on a stream of its own, and replayed from a graph as the batch goes on."""
    rng = np.random.default_rng(13)
    b = a_batch(rng, lens, [1] * len(lens), 16, 8, 2, 128, "f32", "i8", garbage=False)
    plain = attend(b)
    wide, to = (torch.full((len(lens), 13, 128), 5.0, device=G.DEV) for _ in range(2))
    wide[:, 3:11] = b["q"]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attend(dict(b, q=wide[:, 3:11]), out=to[:, 2:10])
    assert torch.equal(to[:, 2:10], plain) and (to[:, :2] == 5).all() and (to[:, 10:] == 5).all()
    cache, out = paged.quantizedCache(*b["tensors"]), torch.empty_like(b["q"])
    context = G.to_dev(b["context"])
    call = paged.quantizedAttention(cache, out, b["q"], G.to_dev(b["starts"]), context, G.to_dev(b["table"]), *b["most"])
    workspace = torch.empty(paged.quantizedAttentionWorkspaceBytes(call), dtype=torch.uint8, device=G.DEV)
    paged.launchQuantizedAttention(G.stream(), call, workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.launchQuantizedAttention(G.stream(), call, workspace)
    for turn in range(4):
        context.copy_(torch.from_numpy((b["context"] * (turn + 1) // 4).astype(np.int32)))
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, attend(dict(b, context=context.cpu().numpy()))), turn
