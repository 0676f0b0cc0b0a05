"""Tokens drawn from logits where one filter's place is searched right behind another's, through the C ABI."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests.test_gpu_sample import check, some_logits  # noqa: E402


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
