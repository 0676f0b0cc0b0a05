"""Values that are no numbers under weights that vanish, in attention over the 8-bit paged cache, through the C ABI."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_quantized_attention import a_batch, attend, check  # noqa: E402
from tests.paged_ref import to64  # noqa: E402


@pytest.mark.parametrize("kind,stored", [("f32", "i8"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("context", [500, 5000, 140000])  # by one workgroup, a few parts, hundreds of them
def test_seen_value_without_weight(kind, stored, context):
    """A seen value that is no number makes its rows none, however far its score lies below the others and whichever
    workgroup has its key: scores fall by one a key, so that the key's weight is zero in f32."""
    print(f"case: seen value without weight {kind} on {stored} context={context}", flush=True)
    rng = np.random.default_rng(context)
    b = a_batch(rng, [context], [2], 16, 4, 2, 64, kind, stored, garbage=False)
    slopes = np.ones(4, np.float32)
    check(b, slopes=slopes)
    clean = attend(b, slopes=slopes)
    values = b["tensors"][3]  # the scales of the values
    for key in (3, context // 2):
        place = (int(b["table"][0, key // 16]), key % 16, 1)
        held = float(values[place])
        values[place] = float("nan")
        check(b, slopes=slopes)
        got = attend(b, slopes=slopes)
        assert torch.isnan(got[:, 2:]).all() and torch.equal(got[:, :2], clean[:, :2])
        values[place] = held
    assert np.isfinite(to64(clean)).all()


@pytest.mark.parametrize("kind,stored", [("f32", "i8"), ("bf16", "e4m3")])
@pytest.mark.parametrize("context,new,heads,kv_heads,dim", [([0], [1200], 8, 8, 64), ([300, 0, 40], [5, 700, 33], 15, 5, 48), ([600], [1], 40, 40, 16),
                                                            ([5000], [90], 8, 1, 128), ([9, 0, 700], [400, 1, 9], 16, 8, 32)])
def test_prompts(kind, stored, context, new, heads, kv_heads, dim):
    """Long prompts beside short ones and alone, and single tokens of many key heads: shares go round the XCDs by heads and by tiles."""
    print(f"case: prompts {kind} on {stored} context={context} new={new} heads={heads}/{kv_heads} dim={dim}", flush=True)
    check(a_batch(np.random.default_rng(dim), context, new, 16, heads, kv_heads, dim, kind, stored))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("stored", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [48, 64, 96, 128, 256])
def test_keys_without_a_block(kind, stored, dim):
    """Keys that the table does not name, any of a tile's 32 and between others that are seen, and a bound of the keys at any place of a
    tile: of rows in sixteens and of more, under a window too."""
    print(f"case: keys without a block {kind} on {stored} dim={dim}", flush=True)
    rng = np.random.default_rng(dim)
    for heads, new, block in ((4, 2, 1), (16, 9, 1), (16, 5, 3)):
        b = a_batch(rng, [150, 40, 7], [new, 1, new], block, heads, 1, dim, kind, stored)
        b["table"][rng.random(b["table"].shape) < 0.3] = -1
        b["table"][2, :2] = b["blocks"]
        check(b)
        check(b, window=37)
    b = a_batch(rng, [70], [9], 16, 16, 1, dim, kind, stored)
    for most in range(60, 79):
        check(b, most=(9, most))
