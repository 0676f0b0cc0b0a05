"""Refusals of the 8-bit cache's launchers, the head rotation, the attention over that cache and sampling: all before any launch (CPU only)."""
import pytest

from antfly_amd import _lib, paged, sampling
from antfly_amd._lib import Buffer
from tests.test_operator_checks import a_cache as a_paged_cache

BIG = Buffer(0x1000, 1 << 40)
NONE = Buffer(0, 0)


def lib():
    return _lib.lib()


def refused(error, call, *args):
    with pytest.raises(error):
        _lib.check(call(*args))


def a_cache(**change):
    fields = {"keys": BIG, "values": BIG, "key_scales": BIG, "value_scales": BIG, "type": _lib.TYPE_I8, "blocks": 10, "block_size": 16, "kv_heads": 2,
              "head_dim": 64, "block_stride": 2048, "slot_stride": 128, "head_stride": 64, "scale_block_stride": 32, "scale_slot_stride": 2,
              "scale_head_stride": 1}
    return _lib.QuantizedCache(**dict(fields, **change))


BAD_CACHES = [{"blocks": 0}, {"block_size": 0}, {"kv_heads": 0}, {"head_dim": 0}, {"head_dim": 56}, {"block_stride": 2040}, {"slot_stride": 136}, {"head_stride": 8},
              {"blocks": 1 << 31}, {"keys": Buffer(0x1008, 1 << 40)}, {"values": NONE}, {"keys": Buffer(0x1000, 10 * 2048 - 1)}, {"block_stride": 1 << 35},
              {"head_stride": (1 << 64) - 16}, {"key_scales": Buffer(0x1002, 1 << 40)}, {"value_scales": NONE}, {"key_scales": Buffer(0x1000, 10 * 32 * 4 - 4)},
              {"scale_block_stride": 1 << 30}, {"scale_slot_stride": (1 << 64) - 1}]


def rotation(**change):
    fields = {"type": 0, "out_type": 0, "interleaved": 0, "epsilon": 1e-6, "tokens": 3, "heads": 4, "kv_heads": 2, "head_dim": 64, "rotary_dim": 32, "axes": 2,
              "query_token_stride": 512, "query_head_stride": 64, "key_token_stride": 512, "key_head_stride": 64, "out_query_token_stride": 256,
              "out_query_head_stride": 64, "out_key_token_stride": 128, "out_key_head_stride": 64}
    fields.update({n: BIG for n in ("query", "key", "out_query", "out_key", "positions", "frequencies", "query_weight", "key_weight")})
    made = _lib.HeadRotation(**dict(fields, **{n: v for n, v in change.items() if n != "pair_axes"}))
    for p, axis in enumerate(change.get("pair_axes", [0, 1] * 8)):
        made.pair_axes[p] = axis
    return made


def attention(**change):
    fields = {"cache": a_cache(), "type": _lib.TYPE_F32, "scale": 0.125, "softcap": 0.0, "window": 0, "requests": 2, "tokens": 6, "heads": 4, "max_query_len": 4,
              "max_key_len": 100, "table_columns": 7, "query_token_stride": 256, "query_head_stride": 64, "out_token_stride": 256, "out_head_stride": 64,
              "query": BIG, "out": BIG, "query_starts": BIG, "context_lens": BIG, "block_tables": BIG, "slopes": BIG}
    return _lib.QuantizedAttention(**dict(fields, **change))


def a_sample(**change):
    fields = {"type": _lib.TYPE_F32, "rows": 3, "vocab": 1000, "row_stride": 1000}
    fields.update({n: BIG for n in ("logits", "temperatures", "top_k", "top_p", "min_p", "uniforms", "tokens", "probabilities")})
    return _lib.Sample(**dict(fields, **change))


def stored(cache, type=0, keys=BIG, values=BIG, token_stride=128, head_stride=64, slots=BIG, tokens=3, call="store"):
    return getattr(lib(), "afhip_launch_quantized_" + call)(None, cache, type, keys, values, token_stride, head_stride, slots, tokens)


CALLS = {"store": lambda c: stored(c), "load": lambda c: stored(c, call="load"),
         "rotated": lambda c: lib().afhip_launch_rotated_store(None, rotation(), None, c, BIG, 512, 64, BIG),
         "attention": lambda c: lib().afhip_launch_quantized_attention(None, attention(cache=c), BIG)}


@pytest.mark.parametrize("name", list(CALLS))
def test_caches(name):
    for change in BAD_CACHES:
        refused(_lib.InvalidHipState, CALLS[name], a_cache(**change))
    for type in (_lib.TYPE_F16, _lib.TYPE_Q8_0, -1):
        refused(_lib.UnsupportedTensorType, CALLS[name], a_cache(type=type))
    refused(_lib.HipOpUnsupported, CALLS[name], a_cache(head_dim=272, head_stride=272, slot_stride=544, block_stride=16 * 544))


@pytest.mark.parametrize("call", ["store", "load"])
def test_store_and_load(call):
    for change in ({"token_stride": 126}, {"head_stride": 62}, {"type": 1, "token_stride": 132}, {"keys": Buffer(0x1000, 3 * 128 * 4 - 4)},
                   {"values": Buffer(0x1008, 1 << 40)}, {"slots": Buffer(0x1000, 11)}, {"slots": NONE}, {"tokens": 1 << 31}):
        refused(_lib.InvalidHipState, lambda: stored(a_cache(), call=call, **change))
    refused(_lib.UnsupportedTensorType, lambda: stored(a_cache(), call=call, type=_lib.TYPE_I8))
    refused(_lib.HipOpUnsupported, lambda: stored(a_cache(kv_heads=1 << 12, block_stride=1 << 22, slot_stride=1 << 18, scale_block_stride=1 << 16, scale_slot_stride=1 << 12),
                                                  call=call, tokens=1 << 24, token_stride=1 << 18, keys=Buffer(0x1000, 1 << 50), values=Buffer(0x1000, 1 << 50)))
    _lib.check(stored(a_cache(), call=call, tokens=0))
    assert stored(None, call=call) == _lib.ERR_INVALID_ARGUMENT


def test_rotation():
    def turn(r):
        return lib().afhip_launch_head_rotation(None, r)

    for change in ({"kv_heads": 0}, {"head_dim": 0}, {"head_dim": 60}, {"rotary_dim": 36}, {"rotary_dim": 72}, {"axes": 0}, {"axes": 17}, {"tokens": 1 << 31},
                   {"epsilon": -1.0}, {"epsilon": float("nan")}, {"pair_axes": [0, 2]}, {"query_token_stride": 511}, {"key_head_stride": 66}, {"out_query_head_stride": 2},
                   {"out_key_token_stride": 129}, {"query": Buffer(0x1008, 1 << 40)}, {"key": NONE}, {"out_query": Buffer(0x1000, 3 * 256 * 4 - 4)},
                   {"out_key": Buffer(0x1000, 3 * 128 * 4 - 4)}, {"positions": Buffer(0x1000, 23)}, {"frequencies": Buffer(0x1000, 63)}, {"frequencies": NONE},
                   {"query_weight": Buffer(0x1000, 255)}, {"key_weight": Buffer(0x1002, 1 << 40)}):
        refused(_lib.InvalidHipState, turn, rotation(**change))
    for change in ({"type": _lib.TYPE_Q8_0}, {"out_type": _lib.TYPE_I8}):
        refused(_lib.UnsupportedTensorType, turn, rotation(**change))
    refused(_lib.HipOpUnsupported, turn, rotation(head_dim=264, query_head_stride=264))
    refused(_lib.HipOpUnsupported, turn, rotation(heads=1 << 26, tokens=1, query_token_stride=0, out_query_token_stride=0))
    refused(_lib.HipOpUnsupported, turn, rotation(tokens=1 << 28, heads=0, positions=Buffer(0x1000, 1 << 44), key=Buffer(0x1000, 1 << 50), out_key=Buffer(0x1000, 1 << 50)))
    _lib.check(turn(rotation(tokens=0)))
    assert turn(None) == _lib.ERR_INVALID_ARGUMENT

    def store(r, cache=None, quantized=None, values=BIG, token_stride=512, head_stride=64, slots=BIG):
        return lib().afhip_launch_rotated_store(None, r, cache, quantized, values, token_stride, head_stride, slots)

    for change in ({"values": Buffer(0x1000, 3 * 512 * 4 - 4 * 385)}, {"values": NONE}, {"token_stride": 510}, {"head_stride": 2}, {"slots": Buffer(0x1000, 11)}):
        refused(_lib.InvalidHipState, lambda: store(rotation(), quantized=a_cache(), **change))
    for r in (rotation(kv_heads=1), rotation(head_dim=48)):
        refused(_lib.InvalidHipState, store, r, None, a_cache())
        refused(_lib.InvalidHipState, store, r, a_paged_cache())
    for pair in ((None, None), (a_paged_cache(), a_cache())):
        assert store(rotation(), *pair) == _lib.ERR_INVALID_ARGUMENT
    assert store(None, None, a_cache()) == _lib.ERR_INVALID_ARGUMENT
    _lib.check(store(rotation(tokens=0), None, a_cache()))


def test_attention():
    def attend(call, workspace=BIG):
        return lib().afhip_launch_quantized_attention(None, call, workspace)

    for change in ({"heads": 0}, {"heads": 5}, {"query_token_stride": 255}, {"query_head_stride": 62}, {"out_token_stride": 258}, {"out_head_stride": 63},
                   {"query": Buffer(0x1000, 6 * 256 * 4 - 4)}, {"query": Buffer(0x1004, 1 << 40)}, {"out": NONE}, {"query_starts": Buffer(0x1000, 11)},
                   {"context_lens": Buffer(0x1000, 7)}, {"block_tables": Buffer(0x1000, 55)}, {"slopes": Buffer(0x1000, 15)}, {"slopes": Buffer(0x1002, 1 << 40)},
                   {"tokens": 1 << 40}, {"window": 1 << 31}, {"softcap": -1.0}, {"softcap": float("nan")}, {"softcap": float("inf")},
                   {"type": _lib.TYPE_F16, "query_token_stride": 260}):
        refused(_lib.InvalidHipState, attend, attention(**change))
    refused(_lib.UnsupportedTensorType, attend, attention(type=_lib.TYPE_I8))
    for change in ({"max_key_len": 1 << 28}, {"max_key_len": (1 << 28) - 32}, {"requests": 65536}, {"max_query_len": 1 << 30}):
        refused(_lib.HipOpUnsupported, attend, attention(**change))
    huge = Buffer(0x1000, 1 << 46)
    refused(_lib.HipOpUnsupported, attend, attention(cache=a_cache(kv_heads=64, block_stride=1 << 16, slot_stride=1 << 12, scale_block_stride=1 << 10, scale_slot_stride=64),
                                                     heads=512, requests=65535, tokens=65535, max_query_len=512, query_token_stride=512 * 64, out_token_stride=512 * 64,
                                                     query=huge, out=huge))
    long = {"max_key_len": 100000, "table_columns": 6250}
    needed = lib().afhip_quantized_attention_workspace_bytes(attention(**long))
    assert needed > 0
    refused(_lib.InvalidHipState, attend, attention(**long), Buffer(0x1000, needed - 1))
    refused(_lib.InvalidHipState, attend, attention(**long), Buffer(0x1010, 1 << 40))
    for change in ({"requests": 0}, {"tokens": 0}, {"max_query_len": 0}):  # nothing to do
        _lib.check(attend(attention(**change), NONE))
    assert lib().afhip_quantized_attention_workspace_bytes(attention(heads=5)) == 0
    assert attend(None) == _lib.ERR_INVALID_ARGUMENT


def test_sample():
    def draw(call, workspace=BIG):
        return lib().afhip_launch_sample(None, call, workspace)

    for change in ({"vocab": 0}, {"logits": Buffer(0x1000, 3 * 4000 - 1)}, {"logits": Buffer(0x1002, 1 << 40)}, {"type": _lib.TYPE_BF16, "logits": Buffer(0x1001, 1 << 40)},
                   {"logits": NONE}, {"uniforms": NONE}, {"tokens": NONE}, {"uniforms": Buffer(0x1000, 11)}, {"tokens": Buffer(0x1002, 1 << 40)},
                   {"temperatures": Buffer(0x1000, 11)}, {"top_k": Buffer(0x1001, 1 << 40)}, {"top_p": Buffer(0x1000, 8)}, {"min_p": Buffer(0x1000, 4)},
                   {"probabilities": Buffer(0x1002, 1 << 40)}, {"row_stride": 1 << 62}):
        refused(_lib.InvalidHipState, draw, a_sample(**change))
    refused(_lib.UnsupportedTensorType, draw, a_sample(type=_lib.TYPE_I8))
    for change in ({"vocab": (1 << 24) + 1}, {"rows": 65536}):
        refused(_lib.HipOpUnsupported, draw, a_sample(**change))
    _lib.check(draw(a_sample(rows=0), NONE))
    assert draw(None) == _lib.ERR_INVALID_ARGUMENT and lib().afhip_sample_workspace_bytes(a_sample(vocab=0)) == 0


def test_arrays():
    torch = pytest.importorskip("torch")
    codes, scales = torch.zeros(4, 16, 2, 64, dtype=torch.int8), torch.zeros(4, 16, 2)
    made = paged.quantizedCache(codes, codes.clone(), scales, scales.clone())
    assert (made.type, made.blocks, made.block_size, made.kv_heads, made.head_dim, made.block_stride, made.slot_stride, made.head_stride) == (_lib.TYPE_I8, 4, 16, 2, 64, 2048, 128, 64)
    assert (made.scale_block_stride, made.scale_slot_stride, made.scale_head_stride) == (32, 2, 1)
    made = paged.quantizedCache(codes.to(torch.float8_e4m3fn), codes.to(torch.float8_e4m3fn), scales, scales, heads_outside=True)
    assert (made.type, made.block_size, made.kv_heads, made.slot_stride, made.head_stride, made.scale_slot_stride, made.scale_head_stride) == (_lib.TYPE_E4M3, 2, 16, 64, 128, 1, 2)
    for bad in ((codes, codes[:3], scales, scales), (codes, codes.to(torch.float8_e4m3fn), scales, scales), (codes, codes, scales[:3], scales), (codes, codes, scales, scales.half()),
                (codes, codes, scales, scales.transpose(0, 1).contiguous().transpose(0, 1)), (codes.transpose(2, 3), codes.transpose(2, 3), scales, scales)):
        with pytest.raises(_lib.InvalidShape):
            paged.quantizedCache(*bad)
    cache = paged.quantizedCache(codes, codes, scales, scales)
    k, slots = torch.zeros(5, 2, 64), torch.zeros(5, dtype=torch.int32)
    for call in (paged.launchQuantizedStore, paged.launchQuantizedLoad):
        for bad in ((k, k[:4], slots), (k, k.half(), slots), (k[:, :1], k[:, :1], slots), (k, k, slots[:4]), (k, k, slots.long()), (k.transpose(1, 2), k.transpose(1, 2), slots)):
            with pytest.raises(_lib.InvalidShape):
                call(None, cache, *bad)
    q, positions, frequencies = torch.zeros(5, 4, 64), torch.zeros(5, dtype=torch.int32), torch.zeros(16)
    good = {"query": q, "key": k, "out_query": q, "out_key": k, "positions": positions, "frequencies": frequencies}
    assert paged.headRotation(**good).rotary_dim == 32
    for change in ({"query": q[:4]}, {"query": q.half()}, {"out_key": k.half()}, {"positions": positions[:4]}, {"positions": positions.long()}, {"frequencies": frequencies.half()},
                   {"frequencies": torch.zeros(129)}, {"query_weight": torch.zeros(63)}, {"key_weight": torch.zeros(64).half()}, {"pair_axes": [0] * 15}):
        error = _lib.InvalidShape
        with pytest.raises(error):
            paged.headRotation(**dict(good, **change))
    with pytest.raises(_lib.InvalidHipState):
        paged.headRotation(**dict(good, pair_axes=[-1] * 16))
    rotated = paged.headRotation(**dict(good, out_key=None))
    for values, places in ((k.half(), slots), (k[:4], slots[:4]), (k, slots.long()), (k, slots[:4])):
        with pytest.raises(_lib.InvalidShape):
            paged.launchRotatedStore(None, rotated, cache, values, places)
    lens, table = torch.zeros(3, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    good = {"out": q, "query": q, "query_starts": lens, "context_lens": lens[:2], "block_tables": table, "max_query_len": 4, "max_key_len": 40}
    assert paged.quantizedAttention(cache, **good).scale == 0.125
    for change in ({"out": q.half()}, {"out": q[:4]}, {"context_lens": lens[:2].long()}, {"query": q.transpose(0, 2)}, {"slopes": torch.zeros(3)}, {"slopes": torch.zeros(4).half()}):
        with pytest.raises(_lib.InvalidShape):
            paged.quantizedAttention(cache, **dict(good, **change))
    for change in ({"window": -1}, {"max_query_len": -1}, {"max_key_len": 4.5}):
        with pytest.raises(_lib.InvalidHipState):
            paged.quantizedAttention(cache, **dict(good, **change))
    logits, numbers = torch.zeros(3, 50), torch.zeros(3)
    tokens = torch.zeros(3, dtype=torch.int32)
    assert sampling.sample(logits, tokens, numbers).vocab == 50
    for args, more in (((logits.t(), tokens, numbers), {}), ((logits, tokens.long(), numbers), {}), ((logits, tokens, numbers[:2]), {}), ((logits, None, numbers), {}),
                       ((logits, tokens, None), {}), ((logits, tokens, numbers), {"top_k": numbers}), ((logits, tokens, numbers), {"top_p": numbers.double()})):
        with pytest.raises(_lib.InvalidShape):
            sampling.sample(*args, **more)
