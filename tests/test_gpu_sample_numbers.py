"""Tokens drawn from logits where one filter's place is searched right behind another's, and where sums are long, through the C ABI."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests import gpu_util as G  # noqa: E402
from tests.test_gpu_sample import check, draw, some_logits  # noqa: E402


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab", [(200, 32000), (9, 100003)])
def test_nucleus_of_many(kind, rows, vocab):
    """Top-k of too many tokens for a list, and top-p of these."""
    print(f"case: nucleus of many {kind} rows={rows} vocab={vocab}", flush=True)
    rng = np.random.default_rng(rows)
    logits = some_logits(rng, rows, vocab, kind, 1.5)
    k, p = rng.integers(vocab // 16, vocab // 4, rows), rng.choice([0.3, 0.9, 0.99], rows)
    check(logits, rng.random(rows), k=k, p=p)
    check(logits, rng.random(rows), t=rng.choice([0.7, 1.0, 2.0], rows), k=k, p=p, m=rng.choice([0.0, 0.01], rows))


@pytest.mark.parametrize("vocab", [65536, 100003])
def test_last_token_of_long_sums(vocab):
    """A number of 1 or more draws the last kept token that weighs anything, also where its weight is below the 53rd bit of the sum:
    behind tokens of one logit, some at e^-27 of them (2^-39; weights are whole multiples of 2^-46 or 2^-45)."""
    print(f"case: last token of long sums vocab={vocab}", flush=True)
    logits = torch.zeros(6, vocab, device=G.DEV)
    logits[:, 5] = -27.0
    logits[1, 7] = -40.0  # weighs nothing
    logits[2, 9] = -float("inf")
    logits[3, vocab - 1] = -27.125
    logits[4] = 1.0
    logits[5, vocab - 3:] = -26.0
    weights = np.exp(np.array([-27.0, -27.0, -27.0, -27.125, 0.0, -27.0]))
    share = weights / np.array([vocab - 1, vocab - 2, vocab - 2, vocab - 2, vocab, vocab - 4])  # (the others' weights are below 2^-50 of the sum)
    for u in (1.0, 2.0):
        tokens, probabilities = draw(logits, [u] * 6)
        assert tokens.tolist() == [5, 5, 5, vocab - 1, vocab - 1, 5]
        assert (np.abs(probabilities - share) <= share * 2.0 ** -23).all()
    assert draw(logits, [1.0] * 6, k=[vocab - 1] * 6)[0].tolist() == [vocab - 1, 5, 5, 5, vocab - 2, vocab - 1]


def test_zeros_beside_tiny_logits():
    """Too many logits in one bin for a list, among them zeros of both signs and some below zero by less than a normal number: where
    the bin is narrowed down to these, the zeros do not count among them."""
    rng = np.random.default_rng(6)
    x = np.concatenate([[np.nextafter(1.0, 0.0, dtype=np.float32)],  # (the narrower bins begin at this largest logit: one ends at the zeros)
                        np.zeros(700), np.full(800, -0.0), -rng.integers(1, 1 << 20, 1500) * 2.0 ** -149, rng.uniform(-1.0, -0.5, 7000)]).astype(np.float32)
    logits = G.to_dev(np.stack([x[rng.permutation(len(x))] for _ in range(6)]))
    t, u = [1000.0] * 6, np.array([0.05, 0.16, 0.2, 0.25, 0.29, 0.9])
    check(logits, u, t=t)
    check(logits, 4 * u / 3.7, t=t, p=[0.9, 0.9, 0.8, 0.9, 0.9, 0.22])
    check(logits, 2 * u, t=t, k=[5000] * 6)
