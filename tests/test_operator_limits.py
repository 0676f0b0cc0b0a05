"""Calls whose grids a launch cannot have (2^32 threads and more) are refused as such, before any launch (CPU only)."""
import pytest

from antfly_amd import _lib, kernels, paged
from antfly_amd._lib import Buffer
from tests.test_operator_checks import BIG, a_cache, attention, fp8, fp8_codes


def wide_cache():
    """Tokens of 136 parts of eight values: one a workgroup of the store."""
    return a_cache(kv_heads=17, block_stride=16 * 17 * 64, slot_stride=17 * 64)


def test_store_and_move():
    with pytest.raises(_lib.HipOpUnsupported):
        _lib.check(_lib.lib().afhip_launch_cache_store(None, wide_cache(), 0, BIG, BIG, 17 * 64, 64, BIG, 1 << 24))
    with pytest.raises(_lib.HipOpUnsupported):
        _lib.check(_lib.lib().afhip_launch_cache_move(None, a_cache(), BIG, 5, BIG, BIG, BIG, 1 << 24, 4))


def test_attention():
    """33 million workgroups of 256 threads."""
    big = Buffer(0x1000, 1 << 44)
    call = attention(cache=a_cache(kv_heads=64, block_stride=16 * 64 * 64, slot_stride=64 * 64), heads=512, requests=65535, tokens=65535, max_query_len=128,
                     query_token_stride=512 * 64, out_token_stride=512 * 64, query=big, out=big)
    with pytest.raises(_lib.HipOpUnsupported):
        _lib.check(_lib.lib().afhip_launch_tree_attention(None, call, big))


def test_fp8_products():
    with pytest.raises(_lib.HipOpUnsupported):
        kernels.launchQuantizeFp8(None, BIG, BIG, BIG, 1 << 29, 16)
    for call in (fp8, fp8_codes):
        for rows in (1, 16, 17, 40):
            with pytest.raises(_lib.HipOpUnsupported):
                call(rows=rows, in_dim=16, out_dim=1 << 28)
        with pytest.raises(_lib.HipOpUnsupported):
            call(rows=(1 << 20) - 16, in_dim=16, out_dim=1 << 18)
    with pytest.raises(_lib.HipOpUnsupported):  # the quantizer's
        fp8(rows=(1 << 20) - 16, in_dim=(1 << 16) + 16, out_dim=16, x=Buffer(0x1000, 1 << 44), workspace=Buffer(0x1000, 1 << 44))


def some_arrays():
    torch = pytest.importorskip("torch")
    k, q = torch.zeros(4, 16, 2, 64, dtype=torch.float16), torch.zeros(5, 4, 64)
    lens, table = torch.zeros(3, dtype=torch.int32), torch.zeros(2, 3, dtype=torch.int32)
    return torch, k, q, lens, table


def test_masks_of_no_words():
    """They have no address: the call would have read none as the causal mask."""
    torch, k, q, lens, table = some_arrays()
    with pytest.raises(_lib.InvalidShape):
        paged.treeAttention(paged.cache(k, k), q, q, lens, lens[:2], table, 4, 40, masks=torch.zeros(5, 0, dtype=torch.int64))


def test_numbers_below_zero():
    """Refused as they are by the launchers that pass them on."""
    torch, k, q, lens, table = some_arrays()
    for most in ((-1, 40), (4, -40), (4, 40.5)):
        with pytest.raises(_lib.InvalidHipState):
            paged.treeAttention(paged.cache(k, k), q, q, lens, lens[:2], table, *most)
    for change in ({"block_size": -16}, {"blocks": -1}):
        with pytest.raises(_lib.InvalidHipState):
            paged.launchBatchPlan(None, lens[:2], lens[:2], table, lens, query_starts=lens, slots=lens, positions=lens, blocks_taken=lens[:1],
                                  **dict({"block_size": 16}, **change))
