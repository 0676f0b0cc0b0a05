"""Refusals of the 8-bit floating point product and of the paged cache's launchers: all of them before any launch (CPU only)."""
import copy

import pytest

from antfly_amd import _lib, kernels, paged
from antfly_amd._lib import Buffer

BIG = Buffer(0x1000, 1 << 40)
NONE = Buffer(0, 0)


def fp8(rows=4, in_dim=256, out_dim=130, dst=BIG, x=BIG, w=BIG, scales=BIG, workspace=BIG, **extra):
    kernels.launchLinearFp8F32(None, dst, x, w, scales, rows, in_dim, out_dim, workspace=workspace, **extra)


def fp8_codes(rows=4, in_dim=256, out_dim=130, q=BIG, q_scales=BIG, **extra):
    kernels.launchMatmulFp8F32(None, extra.pop("dst", BIG), q, q_scales, BIG, BIG, rows, in_dim, out_dim, **extra)


def test_fp8_product_refusals():
    for call in (fp8, fp8_codes):
        for in_dim in (0, 8, 130, 2 ** 31):
            with pytest.raises(_lib.InvalidHipState):
                call(in_dim=in_dim)
        with pytest.raises(_lib.InvalidHipState):
            call(rows=1 << 62)
        with pytest.raises(_lib.InvalidHipState):
            call(dst=Buffer(0x1000, 4 * 4 * 130 - 1))
        with pytest.raises(_lib.InvalidHipState):
            call(dst=Buffer(0x1002, 1 << 40))
        with pytest.raises(_lib.InvalidHipState):
            call(bias=Buffer(0x1000, 4 * 130 - 4))
        with pytest.raises(_lib.InvalidHipState):
            call(residual=Buffer(0x1000, 4 * 4 * 130 - 4))
        with pytest.raises(_lib.HipError) as e:
            call(activation=4)
        assert e.value.status == _lib.ERR_INVALID_ARGUMENT
        with pytest.raises(_lib.HipOpUnsupported):
            call(rows=1 << 20, out_dim=1)
        call(rows=0)  # nothing to do
        call(out_dim=0)
    for bad in (Buffer(0x1000, 4 * 4 * 256 - 1), Buffer(0x1008, 1 << 40), NONE):
        with pytest.raises(_lib.InvalidHipState):
            fp8(x=bad)
    for bad in (Buffer(0x1000, 256 * 130 - 1), Buffer(0x1008, 1 << 40), NONE):
        with pytest.raises(_lib.InvalidHipState):
            fp8(w=bad)
    for bad in (Buffer(0x1000, 4 * 2 * 2 - 1), Buffer(0x1002, 1 << 40), NONE):
        with pytest.raises(_lib.InvalidHipState):
            fp8(scales=bad)
    assert kernels.linearFp8WorkspaceBytes(4, 256, 130) == 0  # few values of X: quantized in the product's launch
    for bad in (Buffer(0x1000, kernels.linearFp8WorkspaceBytes(100, 256, 130) - 1), Buffer(0x1080, 1 << 40), NONE):
        with pytest.raises(_lib.InvalidHipState):
            fp8(rows=100, workspace=bad)
    for bad in (Buffer(0x1000, 4 * 256 - 1), Buffer(0x1008, 1 << 40), NONE):
        with pytest.raises(_lib.InvalidHipState):
            fp8_codes(q=bad)
    with pytest.raises(_lib.InvalidHipState):
        fp8_codes(q_scales=Buffer(0x1000, 4 * 4 * 2 - 1))
    for q, scales, x, in_dim in ((Buffer(0x1000, 1023), BIG, BIG, 256), (BIG, Buffer(0x1000, 31), BIG, 256), (BIG, BIG, Buffer(0x1000, 4095), 256),
                                 (BIG, BIG, BIG, 40)):
        with pytest.raises(_lib.InvalidHipState):
            kernels.launchQuantizeFp8(None, q, scales, x, 4, in_dim)
    kernels.launchQuantizeFp8(None, BIG, BIG, BIG, 0, 256)
    assert kernels.linearFp8WorkspaceBytes(0, 256, 4) == 0 and kernels.linearFp8WorkspaceBytes(3, 250, 4) == 0
    assert kernels.linearFp8WorkspaceBytes(5, 4096, 4096) >= 5 * 4096 + 5 * 32 * 4
    # a small grid on a long K: room for the sums of its shares behind the codes and scales
    assert kernels.linearFp8WorkspaceBytes(512, 14336, 1024) > 512 * 14336 + 512 * 112 * 4 + 2 * 512 * 1024 * 4


def a_cache(**change):
    fields = {"keys": BIG, "values": BIG, "type": _lib.TYPE_F16, "blocks": 10, "block_size": 16, "kv_heads": 2, "head_dim": 64,
              "block_stride": 2048, "slot_stride": 128, "head_stride": 64}
    return _lib.PagedCache(**dict(fields, **change))


BAD_CACHES = [{"blocks": 0}, {"block_size": 0}, {"kv_heads": 0}, {"head_dim": 0}, {"head_dim": 60}, {"block_stride": 2044}, {"slot_stride": 129},
              {"head_stride": 4}, {"blocks": 1 << 31}, {"keys": Buffer(0x1008, 1 << 40)}, {"values": NONE},
              {"keys": Buffer(0x1000, 10 * 2048 * 2 - 2)}, {"block_stride": 1 << 35}, {"head_stride": (1 << 64) - 8}]


def call_of(check, cache):
    if check == "store":
        _lib.check(_lib.lib().afhip_launch_cache_store(None, cache, 0, BIG, BIG, 128, 64, BIG, 3))
    elif check == "move":
        _lib.check(_lib.lib().afhip_launch_cache_move(None, cache, BIG, 5, BIG, BIG, BIG, 2, 4))
    else:
        _lib.check(_lib.lib().afhip_launch_tree_attention(None, attention(cache=cache), BIG))


@pytest.mark.parametrize("check", ["store", "move", "attention"])
def test_cache_refusals(check):
    for change in BAD_CACHES:
        with pytest.raises(_lib.InvalidHipState):
            call_of(check, a_cache(**change))
    with pytest.raises(_lib.UnsupportedTensorType):
        call_of(check, a_cache(type=_lib.TYPE_F32))


def attention(**change):
    fields = {"cache": a_cache(), "type": _lib.TYPE_F32, "scale": 0.125, "requests": 2, "tokens": 6, "heads": 4, "max_query_len": 4,
              "max_key_len": 100, "table_columns": 7, "mask_words": 1, "query_token_stride": 256, "query_head_stride": 64,
              "out_token_stride": 256, "out_head_stride": 64, "query": BIG, "out": BIG, "query_starts": BIG, "context_lens": BIG,
              "block_tables": BIG, "masks": BIG}
    return _lib.TreeAttention(**dict(fields, **change))


def test_attention_refusals():
    def refused(error, workspace=BIG, **change):
        with pytest.raises(error):
            _lib.check(_lib.lib().afhip_launch_tree_attention(None, attention(**change), workspace))

    for change in ({"heads": 0}, {"heads": 5}, {"query_token_stride": 255}, {"query_head_stride": 62}, {"out_token_stride": 258},
                   {"out_head_stride": 63}, {"query": Buffer(0x1000, 6 * 256 * 4 - 4)}, {"query": Buffer(0x1004, 1 << 40)},
                   {"out": Buffer(0x1000, 6 * 256 * 4 - 4)}, {"out": NONE}, {"query_starts": Buffer(0x1000, 11)}, {"query_starts": NONE},
                   {"context_lens": Buffer(0x1000, 7)}, {"block_tables": Buffer(0x1000, 55)}, {"block_tables": Buffer(0x1002, 1 << 40)},
                   {"masks": Buffer(0x1000, 47)}, {"masks": Buffer(0x1004, 1 << 40)}, {"tokens": 1 << 40},
                   {"type": _lib.TYPE_F16, "query_token_stride": 260}):
        refused(_lib.InvalidHipState, **change)
    refused(_lib.UnsupportedTensorType, type=_lib.TYPE_BF16)  # the cache is f16
    refused(_lib.UnsupportedTensorType, type=_lib.TYPE_Q8_0)
    for change in ({"mask_words": 17}, {"max_key_len": 1 << 28}, {"requests": 65536},
                   {"cache": a_cache(head_dim=264, head_stride=264, slot_stride=528, block_stride=8448)}):
        refused(_lib.HipOpUnsupported, **change)
    long = {"max_key_len": 100000, "table_columns": 6250}
    needed = _lib.lib().afhip_tree_attention_workspace_bytes(attention(**long))
    assert needed > 0
    refused(_lib.InvalidHipState, workspace=Buffer(0x1000, needed - 1), **long)
    refused(_lib.InvalidHipState, workspace=Buffer(0x1010, 1 << 40), **long)
    for change in ({"requests": 0}, {"tokens": 0}, {"max_query_len": 0}):  # nothing to do
        _lib.check(_lib.lib().afhip_launch_tree_attention(None, attention(**change), NONE))
    assert _lib.lib().afhip_tree_attention_workspace_bytes(attention(heads=5)) == 0
    assert _lib.lib().afhip_launch_tree_attention(None, None, BIG) == _lib.ERR_INVALID_ARGUMENT


def plan(**change):
    fields = {"requests": 2, "table_columns": 7, "block_size": 16, "blocks": 20, "tokens": 6, "mask_words": 1}
    fields.update({n: BIG for n in ("context_lens", "query_lens", "free_blocks", "parents", "block_tables", "query_starts", "slots",
                                    "positions", "masks", "blocks_taken")})
    return _lib.BatchPlan(**dict(fields, **change))


def test_plan_refusals():
    for change in ({"block_size": 0}, {"blocks": 1 << 31}, {"tokens": 1 << 31}, {"table_columns": 1 << 31}, {"context_lens": Buffer(0x1000, 7)},
                   {"query_lens": NONE}, {"free_blocks": Buffer(0x1001, 8)}, {"parents": Buffer(0x1000, 23)},
                   {"block_tables": Buffer(0x1000, 55)}, {"query_starts": Buffer(0x1000, 11)}, {"slots": Buffer(0x1000, 23)},
                   {"positions": Buffer(0x1002, 1 << 40)}, {"masks": Buffer(0x1000, 47)}, {"blocks_taken": NONE}):
        with pytest.raises(_lib.InvalidHipState):
            _lib.check(_lib.lib().afhip_launch_batch_plan(None, plan(**change)))
    for change in ({"requests": 8193}, {"mask_words": 17}):
        with pytest.raises(_lib.HipOpUnsupported):
            _lib.check(_lib.lib().afhip_launch_batch_plan(None, plan(**change)))
    assert _lib.lib().afhip_launch_batch_plan(None, None) == _lib.ERR_INVALID_ARGUMENT


def test_store_and_move_refusals():
    def store(type=0, keys=BIG, values=BIG, token_stride=128, head_stride=64, slots=BIG, tokens=3):
        _lib.check(_lib.lib().afhip_launch_cache_store(None, a_cache(), type, keys, values, token_stride, head_stride, slots, tokens))

    for change in ({"token_stride": 126}, {"head_stride": 62}, {"type": 1, "token_stride": 132}, {"keys": Buffer(0x1000, 3 * 128 * 4 - 4)},
                   {"values": Buffer(0x1008, 1 << 40)}, {"slots": Buffer(0x1000, 11)}, {"slots": NONE}, {"tokens": 1 << 31}):
        with pytest.raises(_lib.InvalidHipState):
            store(**change)
    with pytest.raises(_lib.UnsupportedTensorType):
        store(type=_lib.TYPE_Q8_0)
    store(tokens=0)
    assert _lib.lib().afhip_launch_cache_store(None, None, 0, BIG, BIG, 128, 64, BIG, 3) == _lib.ERR_INVALID_ARGUMENT

    def move(table=BIG, context=BIG, paths=BIG, lens=BIG, requests=2, columns=4):
        _lib.check(_lib.lib().afhip_launch_cache_move(None, a_cache(), table, 5, context, paths, lens, requests, columns))

    for change in ({"table": Buffer(0x1000, 39)}, {"context": Buffer(0x1000, 7)}, {"paths": Buffer(0x1000, 31)}, {"lens": NONE},
                   {"requests": 1 << 31}):
        with pytest.raises(_lib.InvalidHipState):
            move(**change)
    move(requests=0)
    move(columns=0)
    assert _lib.lib().afhip_launch_cache_move(None, None, BIG, 5, BIG, BIG, BIG, 2, 4) == _lib.ERR_INVALID_ARGUMENT


def test_array_checks():
    torch = pytest.importorskip("torch")
    k = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    c = paged.cache(k, k.clone())
    assert (c.blocks, c.block_size, c.kv_heads, c.head_dim, c.block_stride, c.slot_stride, c.head_stride) == (4, 16, 2, 64, 2048, 128, 64)
    c = paged.cache(k, k.clone(), heads_outside=True)
    assert (c.block_size, c.kv_heads, c.slot_stride, c.head_stride) == (2, 16, 64, 128)
    for keys, values in ((k, k[:3]), (k, k.float()), (k, k.transpose(1, 2)), (k[0], k[0]), (k.transpose(2, 3), k.transpose(2, 3))):
        with pytest.raises(_lib.InvalidShape):
            paged.cache(keys, values)
    q = torch.zeros(5, 4, 64)
    lens = torch.zeros(3, dtype=torch.int32)
    table = torch.zeros(2, 3, dtype=torch.int32)
    good = {"out": q, "query": q, "query_starts": lens, "context_lens": lens[:2], "block_tables": table, "max_query_len": 4, "max_key_len": 40}
    assert paged.treeAttention(paged.cache(k, k), **good).scale == 0.125
    for change in ({"out": q.half()}, {"out": q[:4]}, {"context_lens": lens[:2].long()}, {"block_tables": table.t().contiguous().t()},
                   {"query": q.transpose(0, 2)}, {"masks": torch.zeros(4, 1, dtype=torch.int64)}, {"masks": torch.zeros(5, dtype=torch.int64)}):
        with pytest.raises(_lib.InvalidShape):
            paged.treeAttention(paged.cache(k, k), **dict(good, **change))
    wide = torch.zeros(5, 6, 64)
    part = copy.copy(wide)[:, 1:5]
    b = paged.buffer(part)
    assert b.ptr == wide.data_ptr() + 256 and b.len == (4 * 384 + 3 * 64 + 64) * 4
    assert paged.buffer(None).ptr == 0
