"""Tokens drawn from logits against the definition in 64 bits, through the C ABI."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from antfly_amd import sampling  # noqa: E402
from tests import gpu_util as G  # noqa: E402
from tests import quantized_ref as R  # noqa: E402
from tests.paged_ref import narrow, to64  # noqa: E402


def draw(logits, u, t=None, k=None, p=None, m=None, with_probabilities=True):
    """logits: a device tensor [rows, vocab]; the others: numbers of every row, or None."""
    rows = logits.shape[0]
    f32 = lambda a: None if a is None else G.to_dev(np.asarray(a, np.float32))  # noqa: E731
    tokens = torch.full((rows + 2,), -7, dtype=torch.int32, device=G.DEV)
    probabilities = torch.full((rows + 2,), -7.0, device=G.DEV)
    call = sampling.sample(logits, tokens[1:-1], f32(u), temperatures=f32(t), top_k=None if k is None else G.to_dev(np.asarray(k, np.int32)),
                           top_p=f32(p), min_p=f32(m), probabilities=probabilities[1:-1] if with_probabilities else None)
    workspace = torch.full((sampling.sampleWorkspaceBytes(call),), 0xFF, dtype=torch.uint8, device=G.DEV)
    for _ in range(2):  # the same call again gives the same result
        sampling.launchSample(G.stream(), call, workspace)
    torch.cuda.synchronize()
    assert tokens[0] == -7 and tokens[-1] == -7 and probabilities[0] == -7 and probabilities[-1] == -7
    return tokens[1:-1].cpu().numpy(), probabilities[1:-1].cpu().numpy()


def check(logits, u, t=None, k=None, p=None, m=None):
    tokens, probabilities = draw(logits, u, t, k, p, m)
    rows = to64(logits)
    for r in range(len(rows)):
        one = lambda a, none, kind=np.float32: none if a is None else kind(a[r])  # noqa: E731
        token, probability = R.sample(rows[r], np.float32(u[r]), one(t, 1.0), one(k, 0, int), one(p, 1.0), one(m, 0.0))
        said = (r, one(t, 1.0), one(k, 0, int), one(p, 1.0), one(m, 0.0), u[r])
        assert tokens[r] == token, (said, int(tokens[r]), token)
        # sums of 64 bits, one rounding to f32
        assert abs(probabilities[r] - probability) <= probability * 2.0 ** -23 + 1e-30, (said, probabilities[r], probability)


def some_logits(rng, rows, vocab, kind, spread):
    x = rng.standard_normal((rows, vocab)) * spread
    x[rng.random((rows, vocab)) < 0.01] = -np.inf
    return narrow(x, kind).to(G.DEV)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,spread", [(1, 1.0), (2, 3.0), (7, 2.0), (63, 2.0), (1000, 1.0), (4099, 0.2), (32001, 2.5), (100003, 4.0), (151937, 0.01)])
def test_filters(kind, vocab, spread):
    print(f"case: sample {kind} vocab={vocab} spread={spread}", flush=True)
    rng = np.random.default_rng(vocab)
    rows = 48 if vocab < 50000 else 24
    logits = some_logits(rng, rows, vocab, kind, spread)
    u = rng.random(rows)
    u[:3] = 0.0, 1 - 2.0 ** -24, 0.5
    k = rng.choice([0, 1, 2, 40, 1024, 1025, 5000, vocab, vocab + 7, -3], rows)
    p = rng.choice([1.0, 0.9, 0.5, 0.999, 0.01, 0.0, 2.0], rows)
    m = rng.choice([0.0, 0.05, 0.3, 1.0, 1e-6], rows)
    t = rng.choice([1.0, 0.7, 0.1, 3.0, 50.0], rows)
    check(logits, u)
    check(logits, u, t)
    check(logits, u, k=k)
    check(logits, u, p=p)
    check(logits, u, m=m)
    check(logits, u, t, k, p, m)


@pytest.mark.parametrize("vocab", [5, 1023, 70001])
def test_ties(vocab):
    """Equal logits: their order is that of their indices, and all sums are exact."""
    rows = 16
    logits = torch.zeros(rows, vocab, device=G.DEV)
    u = np.arange(rows) / rows
    check(logits, u)
    check(logits, u, p=np.full(rows, 0.5))
    check(logits, u, k=np.full(rows, 3))
    check(logits, u, k=np.full(rows, min(vocab, 3000)), p=np.full(rows, 0.25))
    logits[:, vocab // 2:] = 1.0
    logits[:, ::3] = -0.0
    check(logits, u, p=np.full(rows, 0.9), k=np.full(rows, vocab - vocab // 5))
    few = torch.tensor([[1.0, 2.0, 2.0, 0.5, 2.0]], device=G.DEV).expand(4, 5)  # rows of one memory
    assert draw(few, [0.0, 0.3, 0.6, 0.9], k=[3] * 4)[0].tolist() == [1, 1, 2, 4]


def test_greedy():
    rng = np.random.default_rng(1)
    logits = some_logits(rng, 6, 40000, "bf16", 1.0)
    u = rng.random(6)
    tokens, probabilities = draw(logits, u, t=[0.0, -1.0, np.nan, 0.0, 0.0, 0.0])
    rows = to64(logits)
    assert tokens.tolist() == rows.argmax(1).tolist() and (probabilities == 1).all()
    assert draw(logits, u, t=[0.0] * 6, with_probabilities=False)[0].tolist() == tokens.tolist()
    assert draw(logits, u, k=[1] * 6)[0].tolist() == tokens.tolist() and draw(logits, u, p=[0.0] * 6)[0].tolist() == tokens.tolist()


@pytest.mark.parametrize("vocab", [300, 30000])
def test_far_temperatures(vocab):
    """Where all tokens weigh the same, whatever their logits, and where only the largest weighs."""
    rng = np.random.default_rng(7)
    logits = some_logits(rng, 8, vocab, "f32", 3.0)
    t = [np.inf, 1e30, 1e-30, 1e-45, 3e38, np.inf, 1e30, 1e6]
    check(logits, rng.random(8), t=t)
    check(logits, rng.random(8), t=t, k=[0, 100, 5, 0, 7000, 20, 1, 290])
    check(logits, rng.random(8), t=t, p=[0.9, 0.5, 0.9, 0.1, 0.99, 0.01, 0.9, 0.5], m=[0.0, 0.1, 0.5, 1.0, 0.2, 0.0, 1.0, 0.9])


@pytest.mark.parametrize("vocab", [300, 30000])
def test_numbers_that_are_none(vocab):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((8, vocab))
    x[0] = -np.inf
    x[1] = np.nan
    x[2, ::2] = np.nan
    x[3, [5, 77, 250]] = np.inf
    x[4, :] = -np.inf
    x[4, vocab - 1] = -3e38
    x[5] *= 1e38
    x[6] = -1e38
    logits = G.to_dev(x.astype(np.float32))
    u = np.array([0.5, 0.5, 0.7, 0.4, 0.9, 0.3, 0.999, 0.2], np.float32)
    check(logits, u)
    check(logits, u, t=[np.inf] * 8)
    check(logits, u, t=[1e-38] * 8, p=[0.9] * 8)
    check(logits, u, k=[2] * 8, m=[0.5] * 8)
    check(logits, u, p=[np.nan] * 8, m=[np.nan] * 8, k=[1500] * 8)
    check(logits, [-1.0, np.nan, -0.5, 1.0, 2.0, np.inf, 1.0, 1.5], p=[0.95] * 8)
    assert draw(logits, u)[0][:2].tolist() == [-1, -1]


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_rows_of_wider_arrays(kind):
    """Row strides and starts of any number of elements."""
    rng = np.random.default_rng(3)
    wide = some_logits(rng, 5, 4100, kind, 2.0)
    u = rng.random(5)
    for first, count in ((0, 4100), (1, 4099), (3, 4001), (7, 13)):
        check(wide[:, first:first + count], u, p=[0.9] * 5)
        check(wide[:, first:first + count], u, k=[20] * 5)


def test_draws_follow_the_probabilities():
    """Every token of a small row is drawn for exactly its share of evenly spread numbers (within one of them)."""
    logits = torch.tensor([0.3, -1.0, 2.0, 0.3, 1.1, -4.0], device=G.DEV)
    n = 4096
    tokens, _ = draw(logits[None].expand(n, 6), (np.arange(n) + 0.5) / n)
    shares = np.exp(to64(logits)) / np.exp(to64(logits)).sum()
    assert (np.abs(np.bincount(tokens, minlength=6) - shares * n) <= 1.0).all()


def test_replayed():
    rng = np.random.default_rng(4)
    rows, vocab = 3, 50001
    logits, u = some_logits(rng, rows, vocab, "f32", 1.0), torch.empty(rows, device=G.DEV)
    tokens, k = torch.empty(rows, dtype=torch.int32, device=G.DEV), torch.tensor([0, 30, 4000], dtype=torch.int32, device=G.DEV)
    p = torch.tensor([0.95, 0.9, 1.0], device=G.DEV)
    call = sampling.sample(logits, tokens, u, top_k=k, top_p=p)
    workspace = torch.empty(sampling.sampleWorkspaceBytes(call), dtype=torch.uint8, device=G.DEV)
    u.uniform_()
    sampling.launchSample(G.stream(), call, workspace)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sampling.launchSample(G.stream(), call, workspace)
    for turn in range(4):
        u.copy_(torch.from_numpy(rng.random(rows).astype(np.float32)))
        logits.copy_(some_logits(rng, rows, vocab, "f32", 1.0 + turn))
        graph.replay()
        torch.cuda.synchronize()
        want = draw(logits, u.cpu().numpy(), k=k.cpu().numpy(), p=p.cpu().numpy())[0]
        assert tokens.cpu().numpy().tolist() == want.tolist(), turn


def test_streams_and_shared_workspaces():
    """Two captured calls on one workspace, of other shapes, in turn with eager ones, on a stream that is not the first."""
    rng = np.random.default_rng(5)
    side, workspace = torch.cuda.Stream(), None
    calls = []
    for rows, vocab, kind in ((2, 32000, "f32"), (40, 7001, "bf16")):
        logits, u = some_logits(rng, rows, vocab, kind, 2.0), torch.rand(rows, device=G.DEV)
        p = torch.full((rows,), 0.9, device=G.DEV)
        calls.append((logits, u, p, sampling.sample(logits, torch.empty(rows, dtype=torch.int32, device=G.DEV), u, top_p=p)))
    workspace = torch.full((max(sampling.sampleWorkspaceBytes(c[3]) for c in calls),), 0xFF, dtype=torch.uint8, device=G.DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in calls:
            sampling.launchSample(G.stream(), c[3], workspace)
        side.synchronize()
        graphs = []
        for c in calls:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                sampling.launchSample(G.stream(), c[3], workspace)
            graphs.append(graph)
        for turn in range(4):
            for graph, (logits, u, p, call) in zip(graphs, calls):
                u.uniform_()
                graph.replay()
                got = call.arrays[1].clone()
                call.arrays[1].zero_()
                if turn % 2:
                    sampling.launchSample(G.stream(), call, workspace)
                    assert torch.equal(call.arrays[1], got)
                side.synchronize()
                assert got.cpu().numpy().tolist() == [R.sample(row, x, p=np.float32(0.9))[0] for row, x in zip(to64(logits), u.cpu().numpy())], turn
