"""The example's decoder: drafts change the steps, not the tokens, and the tokens are the model's in 64 bits."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests import fp8_ref  # noqa: E402

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "speculative_decode.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("speculative_decode", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def prompts_of(model, lens):
    rng = np.random.default_rng(5)
    return [rng.integers(0, model.embedding.shape[0], n).tolist() for n in lens]


@pytest.mark.parametrize("drafts", [1, 6, 15])
def test_drafts_change_the_steps_only(example, drafts):
    model = example.Model()
    prompts = prompts_of(model, (3, 40, 17))
    plain, steps = example.generate(model, prompts, 48, 0)
    drafted, fewer = example.generate(model, prompts, 48, drafts)
    assert drafted == plain and steps == 47 and fewer <= steps


def test_tokens_are_the_models(example):
    model = example.Model(layers=1)
    prompt = prompts_of(model, (12,))[0]
    tokens = example.generate(model, [prompt], 24, 8)[0][0]
    logits = in_64_bits(example, model, prompt + tokens)[len(prompt) - 1:-1]
    # a code of an activation may round the other way: 2^-4 of one of hundreds of values that a sum adds, a few of them at most,
    # and as little of the logits' range
    chosen = logits[np.arange(len(tokens)), tokens]
    assert (logits.max(1) - chosen <= 0.02 * (logits.max(1) - logits.min(1))).all()


def linear(weight, x):
    codes, scales = fp8_ref.quantize(x.astype(np.float32))
    return fp8_ref.dense(codes, scales, 1) @ fp8_ref.dense(weight.codes.cpu().numpy(), weight.scales.cpu().numpy(), 128).T


def in_64_bits(example, model, tokens):
    """The logits of every token of one sequence, causal."""
    n, heads, kv, dim = len(tokens), model.heads, model.kv_heads, model.head_dim
    norm = lambda x: x / np.sqrt((x ** 2).mean(-1, keepdims=True) + 1e-6)  # noqa: E731
    rotate = lambda x: example.rotate(torch.from_numpy(x), torch.arange(n)).numpy()  # noqa: E731
    x = model.embedding.cpu().numpy()[tokens].astype(np.float64)
    for layer in model.layers:
        qkv = linear(layer["qkv"], norm(x)).reshape(n, heads + 2 * kv, dim)
        q, k, v = rotate(qkv[:, :heads]), rotate(qkv[:, heads:heads + kv]), qkv[:, heads + kv:]
        k, v = k.astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64)
        seen = np.zeros_like(q)
        for h in range(heads):
            score = q[:, h] @ k[:, h // (heads // kv)].T * dim ** -0.5
            score[np.triu_indices(n, 1)] = -np.inf
            p = np.exp(score - score.max(1, keepdims=True))
            seen[:, h] = p / p.sum(1, keepdims=True) @ v[:, h // (heads // kv)]
        x = x + linear(layer["out"], seen.reshape(n, -1))
        up = linear(layer["up"], norm(x))
        up = fp8_ref.activate(up, example.GELU)
        x = x + linear(layer["down"], up)
    return linear(model.head, norm(x))


@pytest.mark.parametrize("drafts", [6, 15])
def test_accepted_paths_move(example, drafts, monkeypatch):
    """Drafts are accepted, some of them not where their path's place is: the cache's tokens move, and the tokens stay the model's."""
    moved = []
    launch = example.paged.launchCacheMove

    def recorded(stream, cache, table, context, paths, lens):
        for path, n in zip(paths.tolist(), lens.tolist()):
            moved.extend(p - i for i, p in enumerate(path[:n]))
        launch(stream, cache, table, context, paths, lens)

    monkeypatch.setattr(example.paged, "launchCacheMove", recorded)
    model = example.Model()
    prompts = prompts_of(model, (3, 40, 17))
    plain, steps = example.generate(model, prompts, 48, 0)
    assert moved and not any(moved)  # one token a step: it lies where it belongs
    moved.clear()
    drafted, fewer = example.generate(model, prompts, 48, drafts)
    assert drafted == plain
    assert fewer < steps and any(moved) and min(moved) == 0
