"""The operators of a sampled serving step one after the other, as a program uses them."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from antfly_amd import paged, sampling  # noqa: E402
from tests import gpu_util as G  # noqa: E402
from tests import quantized_ref as R  # noqa: E402
from tests.paged_ref import narrow, starts_of, to64  # noqa: E402

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "sampled_decode.py")


class Step:
    """Requests over one cache; every array lives on, so that a captured step reads what is put there."""

    def __init__(self, rng, requests, longest, heads, kv_heads, dim, kind, stored, vocab, workspace):
        self.block, columns = 16, -(-longest // 16)
        self.blocks = (requests + 1) * columns
        self.heads, self.kv_heads, self.dim, self.kind, self.stored, self.requests, self.longest = heads, kv_heads, dim, kind, stored, requests, longest
        shape = self.blocks, self.block, kv_heads
        self.tensors = [torch.zeros(*shape, dim, device=G.DEV).to(R.DTYPES[stored]) for _ in "kv"] + [torch.full(shape, float("nan"), device=G.DEV) for _ in "kv"]
        self.cache = paged.quantizedCache(*self.tensors)
        order = rng.permutation(self.blocks).astype(np.int32)
        self.own, self.free = order[:columns], G.to_dev(order[columns:])  # a request's that begins with a context; the others, in the order they are taken
        self.turns = torch.arange(len(order) - columns, device=G.DEV)
        self.table = torch.full((requests, columns), -1, dtype=torch.int32, device=G.DEV)
        self.weights = [(1 + 0.3 * rng.standard_normal(dim)).astype(np.float32) for _ in "qk"]
        self.frequencies = (10000.0 ** (-np.arange(dim // 2) / (dim // 2))).astype(np.float32)
        self.slopes = (0.25 ** np.arange(1, heads + 1)).astype(np.float32)
        self.context = torch.zeros(requests, dtype=torch.int32, device=G.DEV)
        self.head = torch.from_numpy(rng.standard_normal((heads * dim, vocab)).astype(np.float32) * 4 / dim ** 0.5).to(G.DEV)
        self.drawn, self.probabilities, self.uniforms = (torch.zeros(requests, dtype=t, device=G.DEV) for t in (torch.int32, torch.float32, torch.float32))
        self.top_k, self.top_p = torch.arange(requests, dtype=torch.int32, device=G.DEV) * 20, torch.full((requests,), 0.9, device=G.DEV)
        self.fixed = [G.to_dev(a) for a in (self.frequencies, *self.weights, self.slopes)]
        self.workspace = workspace

    def batch(self, most_new):
        """Buffers of a batch of up to most_new tokens a request."""
        n = self.requests * most_new
        i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device=G.DEV)  # noqa: E731
        qkv = torch.zeros(n, self.heads + 2 * self.kv_heads, self.dim, dtype=R.DTYPES[self.kind], device=G.DEV)
        return {"qkv": qkv, "lens": i32(self.requests), "starts": i32(self.requests + 1), "slots": i32(n), "positions": i32(n), "taken": i32(1),
                "turned": torch.zeros(n, self.heads, self.dim, dtype=qkv.dtype, device=G.DEV), "seen": torch.zeros(n, self.heads, self.dim, dtype=qkv.dtype, device=G.DEV),
                "logits": torch.zeros(self.requests, self.head.shape[1], device=G.DEV), "most": most_new}

    def run(self, b):
        paged.launchBatchPlan(G.stream(), self.context, b["lens"], self.table, self.free, self.block, b["starts"], b["slots"], b["positions"], b["taken"], blocks=self.blocks)
        self.free.copy_(self.free[(self.turns + b["taken"]) % self.turns.shape[0]])
        q, k, v = b["qkv"].split((self.heads, self.kv_heads, self.kv_heads), 1)
        rotation = paged.headRotation(q, k, b["turned"], None, b["positions"], *self.fixed[:3])
        paged.launchRotatedStore(G.stream(), rotation, self.cache, v, b["slots"])
        call = paged.quantizedAttention(self.cache, b["seen"], b["turned"], b["starts"], self.context, self.table, b["most"], self.longest, softcap=20.0,
                                        window=200, slopes=self.fixed[3])
        assert paged.quantizedAttentionWorkspaceBytes(call) <= self.workspace.numel()
        paged.launchQuantizedAttention(G.stream(), call, self.workspace)
        last = (b["starts"][1:] - 1).clamp_min(0).long()
        torch.mm(b["seen"][last].float().view(self.requests, -1), self.head, out=b["logits"])
        call = sampling.sample(b["logits"], self.drawn, self.uniforms, top_k=self.top_k, top_p=self.top_p, probabilities=self.probabilities)
        assert sampling.sampleWorkspaceBytes(call) <= self.workspace.numel()
        sampling.launchSample(G.stream(), call, self.workspace)

    def check(self, b):
        """Every operator's results from what it read."""
        n, starts, context = int(b["lens"].sum()), b["starts"].cpu().numpy(), self.context.cpu().numpy()
        assert starts.tolist() == starts_of(b["lens"].cpu().numpy()).tolist()
        positions, slots = b["positions"].cpu().numpy()[None, :n], b["slots"].cpu().numpy()[:n]
        x = to64(b["qkv"])[:n]
        q, k, v = x[:, :self.heads], x[:, self.heads:-self.kv_heads], x[:, -self.kv_heads:]
        axes = [0] * (self.dim // 2)
        want = R.rotate(q, self.weights[0], positions, self.frequencies, False, axes)
        assert (np.abs(to64(b["turned"])[:n] - want) <= R.rotation_error(q, self.weights[0], want, self.kind, False, self.dim // 2)).all()
        k_codes, v_codes, k_scales, v_scales = (R.numbers(t) for t in self.tensors)
        at = slots // self.block, slots % self.block
        want = R.rotate(k, self.weights[1], positions, self.frequencies, False, axes)
        # a code is half a step off, and the scale of the head by as much as its largest value; the norm and rotation as for f32
        off = R.rotation_error(k, self.weights[1], want, "f32", False, self.dim // 2)
        most = np.abs(want).max(-1, keepdims=True)
        off = off + off.max(-1, keepdims=True) + 2.0 ** -20 * most
        step = most / 127 / 2 if self.stored == "i8" else np.maximum(2.0 ** -4 * np.abs(want), 2.0 ** -10 * most / 448)
        assert (np.abs(k_codes[at] * k_scales[at][..., None] - want) <= 1.07 * off + step).all()
        codes, scales = R.quantize(v, self.stored)
        assert np.array_equal(v_codes[at], codes) and np.array_equal(v_scales[at].astype(np.float32), scales)
        want, off = R.attend(to64(b["turned"])[:n], k_codes, v_codes, k_scales, v_scales, self.dim ** -0.5, starts, context, self.table.cpu().numpy(), self.block,
                             self.blocks, b["most"], self.longest, self.kind, 20.0, 200, self.slopes.astype(np.float64), self.stored == "i8")
        assert (np.abs(to64(b["seen"])[:n] - want) <= off).all()
        logits, u = to64(b["logits"]), self.uniforms.cpu().numpy()
        for r in range(self.requests):
            token, probability = R.sample(logits[r], u[r], k=int(self.top_k[r]), p=np.float32(0.9))
            assert int(self.drawn[r]) == token and abs(float(self.probabilities[r]) - probability) <= probability * 2.0 ** -23


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("stored", ["i8", "e4m3"])
def test_step_by_step(kind, stored):
    """Prompts, then single tokens replayed from a graph, two requests sets' graphs on one workspace in turn."""
    print(f"case: steps {kind} on {stored}", flush=True)
    rng = np.random.default_rng(21)
    workspace = torch.full((64 << 20,), 0xFF, dtype=torch.uint8, device=G.DEV)
    sets = [Step(rng, requests, longest, 6, 2, dim, kind, stored, vocab, workspace) for requests, longest, dim, vocab in ((3, 300, 64, 3001), (5, 2500, 128, 20011))]

    def put(s, b, lens):
        b["lens"].copy_(torch.tensor(lens))
        b["qkv"].copy_(narrow(rng.standard_normal(tuple(b["qkv"].shape)) * 2, kind))
        s.uniforms.copy_(torch.from_numpy(rng.random(s.requests).astype(np.float32)))

    graphs = []
    for s in sets:
        b = s.batch(90)
        put(s, b, [1, 90, 37, 64, 2][:s.requests])
        s.run(b)
        torch.cuda.synchronize()
        s.check(b)
        s.context += b["lens"]
        if s.longest > 2000:  # a long context of zeros
            for t in s.tensors[2:]:
                t.nan_to_num_(0.01)
            s.context[2] = 2300
            s.table[2].copy_(torch.from_numpy(s.own))
        b = s.batch(1)
        put(s, b, [1] * s.requests)
        s.run(b)  # (the first call of a shape belongs outside a capture)
        torch.cuda.synchronize()
        s.check(b)
        s.context += 1
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.run(b)
        graphs.append((graph, b))
    for turn in range(3):
        for s, (graph, b) in zip(sets, graphs):
            put(s, b, [1] * s.requests)
            graph.replay()
            torch.cuda.synchronize()
            s.check(b)
            s.context += 1


def test_far_blocks():
    """Codes past 4 GiB from the first give what the same ones do in a small cache."""
    rng = np.random.default_rng(22)
    block, heads, dim, far = 16, 4, 128, 560000  # 8 KiB a block
    tokens = 100
    new = [narrow(rng.standard_normal((tokens, heads, dim)), "f32").to(G.DEV) for _ in "kv"]
    q = narrow(rng.standard_normal((1, 8, dim)), "f32").to(G.DEV)
    got = []
    for blocks, ids in ((7, range(7)), (far, [far - 1, 3, far - 77, far // 2 + 5, far - 2, 1, far - 3])):
        shape = blocks, block, heads
        tensors = [torch.empty(*shape, dim, dtype=torch.int8, device=G.DEV) for _ in "kv"] + [torch.empty(shape, device=G.DEV) for _ in "kv"]
        cache = paged.quantizedCache(*tensors)
        table = np.array([list(ids)], np.int32)
        at = np.arange(tokens)
        slots = G.to_dev((table[0, at // block] * block + at % block).astype(np.int32))
        paged.launchQuantizedStore(G.stream(), cache, *new, slots)
        back = [torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device=G.DEV) for _ in "kv"]
        paged.launchQuantizedLoad(G.stream(), cache, *back, slots)
        out = torch.empty_like(q)
        arrays = [G.to_dev(np.array(a, np.int32)) for a in ([0, 1], [tokens - 1], table)]
        paged.launchQuantizedAttention(G.stream(), paged.quantizedAttention(cache, out, q, *arrays, 1, tokens))
        torch.cuda.synchronize()
        got.append([*back, out])
        del tensors, cache
    assert all(torch.equal(a, b) for a, b in zip(*got)) and torch.isfinite(got[0][2]).all()


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("sampled_decode", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("stored", ["int8", "float8_e4m3fn"])
def test_example(example, stored):
    """Replayed steps give the launched ones' tokens; other numbers give other tokens, no temperature gives the same whatever they are."""
    rng = np.random.default_rng(6)
    model = example.Model(stored=getattr(torch, stored))
    prompts = [rng.integers(0, model.embedding.shape[0], n).tolist() for n in (3, 40, 17)]
    uniforms = [torch.from_numpy(rng.random((24, 3)).astype(np.float32)).cuda() for _ in range(2)]
    sampled = example.Decoder(model, prompts, 24, temperature=0.9, top_k=40, top_p=0.95)
    launched = sampled.generate(uniforms[0], graph=False)
    assert torch.equal(sampled.generate(uniforms[0]), launched) and not torch.equal(sampled.generate(uniforms[1]), launched)
    assert launched.min() >= 0 and launched.max() < model.embedding.shape[0]
    greedy = example.Decoder(model, prompts, 24, temperature=0.0)
    assert torch.equal(greedy.generate(uniforms[0]), greedy.generate(uniforms[1], graph=False))
