"""Angles of the head rotation at far positions, against whole-number arithmetic of 200 bits, through the C ABI."""
import math
from fractions import Fraction

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from antfly_amd import paged  # noqa: E402
from tests import gpu_util as G  # noqa: E402
from tests.paged_ref import to64  # noqa: E402

BITS = 200


def turn_per_radian():
    """2^BITS / (2 pi): pi = 16 arctan(1/5) - 4 arctan(1/239)."""
    def arctan(n):
        power, total, k = (1 << (BITS + 40)) // n, 0, 1
        while power:
            total += power // k if k % 4 == 1 else -(power // k)
            power //= n * n
            k += 2
        return total
    pi = 16 * arctan(5) - 4 * arctan(239)
    return (1 << (2 * BITS + 40)) // (2 * pi)


def rests(positions, frequencies):
    """position * frequency less whole turns, in radians: [positions][frequencies]."""
    by = turn_per_radian()
    out = np.empty((len(positions), len(frequencies)))
    for j, f in enumerate(frequencies):
        exact = Fraction(float(f))
        for i, p in enumerate(positions):
            turns = int(p) * exact.numerator * by // exact.denominator  # times 2^BITS
            rest = turns % (1 << BITS)
            rest -= (1 << BITS) if rest >> (BITS - 1) else 0
            out[i, j] = float(Fraction(rest, 1 << BITS)) * 2 * math.pi
    return out


@pytest.mark.parametrize("most", [2 ** 17, 2 ** 24, 2 ** 28, 2 ** 31])
def test_angles(most):
    print(f"case: angles of positions up to {most}", flush=True)
    rng = np.random.default_rng(most % 1000)
    tokens, pairs = 1000, 32
    positions = rng.integers(most // 2, most, tokens).astype(np.int32)
    positions[1::2] *= -1
    positions[0] = most - 1
    frequencies = np.concatenate([rng.uniform(0.5, 1, 16), 10000.0 ** -rng.uniform(0, 1, 15), [np.float32(1) - np.float32(2.0 ** -24)]]).astype(np.float32)
    k = torch.zeros(tokens, 1, 2 * pairs, device=G.DEV)
    k[..., :pairs] = 1
    out = torch.empty_like(k)
    paged.launchHeadRotation(G.stream(), paged.headRotation(None, k, None, out, G.to_dev(positions), G.to_dev(frequencies)))
    torch.cuda.synchronize()
    got, rest = to64(out)[:, 0], rests(positions, frequencies)
    # An eighth of a turn in f32 is off by half a step, 0.4 * 2^-24 radians; the sine's series, its square and the product with the
    # angle by 2.5 half steps of a value of at most 0.71, 1.8 * 2^-24; the cosine's by 0.5 for the last sum and 1 for what is added.
    off = np.abs(np.concatenate([got[:, :pairs] - np.cos(rest), got[:, pairs:] - np.sin(rest)], 1)).max()
    assert off <= 3 * 2.0 ** -24, off * 2.0 ** 24
