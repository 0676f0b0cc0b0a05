"""Sampled decoding over an 8-bit paged cache with the library's operators: a small decoder of random weights, its projections in
8-bit floating point, goes on with several prompts at once.

A step:  plan the batch (slots, positions) -> per layer: project, norm and rotate queries and keys, keys and values into the cache,
attend, project back -> a token of every request from the logits.  No step waits for the host, so it is replayed from a graph.

    python examples/sampled_decode.py --requests 8 --new-tokens 128 --temperature 0.8 --top-k 50 --top-p 0.95
"""
import argparse
import os
import sys
import time

import torch

sys.path[:0] = [os.path.dirname(os.path.abspath(__file__)), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))]

from antfly_amd import paged, sampling  # noqa: E402
from speculative_decode import GELU, Linear, norm, stream  # noqa: E402


def scratch(nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device="cuda")


class Model:
    def __init__(self, vocab=2048, hidden=512, layers=2, heads=8, kv_heads=2, head_dim=64, blocks=512, block_size=16, stored=torch.float8_e4m3fn,
                 softcap=30.0, window=0, seed=1):
        g = torch.Generator().manual_seed(seed)

        def weight(out_dim, in_dim):
            return torch.randn(out_dim, in_dim, generator=g) * in_dim ** -0.5

        self.heads, self.kv_heads, self.head_dim, self.block_size, self.blocks = heads, kv_heads, head_dim, block_size, blocks
        self.softcap, self.window = softcap, window
        self.embedding = torch.randn(vocab, hidden, generator=g).cuda()
        self.frequencies = (10000.0 ** (-torch.arange(head_dim // 2) / (head_dim // 2))).cuda()
        self.layers = []
        for _ in range(layers):
            codes = [torch.zeros(blocks, block_size, kv_heads, head_dim, device="cuda").to(stored) for _ in "kv"]
            scales = [torch.zeros(blocks, block_size, kv_heads, device="cuda") for _ in "kv"]
            norms = [(1 + 0.1 * torch.randn(head_dim, generator=g)).cuda() for _ in "qk"]
            self.layers.append({"qkv": Linear(weight((heads + 2 * kv_heads) * head_dim, hidden)), "out": Linear(weight(hidden, heads * head_dim)),
                                "up": Linear(weight(4 * hidden, hidden)), "down": Linear(weight(hidden, 4 * hidden)), "norms": norms,
                                "cache": paged.quantizedCache(*codes, *scales)})
        self.head = Linear(weight(vocab, hidden))

    def __call__(self, tokens, positions, slots, starts, context, table, most_new, most_keys, rows=None):
        """The logits of a batch's new tokens (of `rows` alone); their keys and values are in the cache afterwards."""
        n, kv = tokens.shape[0], self.kv_heads
        x = self.embedding[tokens]
        for layer in self.layers:
            q, k, v = layer["qkv"](norm(x)).view(n, self.heads + 2 * kv, self.head_dim).split((self.heads, kv, kv), 1)
            turned = torch.empty(n, self.heads, self.head_dim, device="cuda")
            rotation = paged.headRotation(q, k, turned, None, positions, self.frequencies, *layer["norms"])
            paged.launchRotatedStore(stream(), rotation, layer["cache"], v, slots)
            seen = torch.empty_like(turned)
            attention = paged.quantizedAttention(layer["cache"], seen, turned, starts, context, table, most_new, most_keys, softcap=self.softcap,
                                                 window=self.window)
            paged.launchQuantizedAttention(stream(), attention, scratch(paged.quantizedAttentionWorkspaceBytes(attention)))
            x = layer["out"](seen.view(n, -1), residual=x)
            x = layer["down"](layer["up"](norm(x), activation=GELU), residual=x)
        return self.head(norm(x if rows is None else x[rows]))


class Decoder:
    """Requests over one cache, all they need to go on on the device."""

    def __init__(self, model, prompts, new_tokens, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        requests, i32 = len(prompts), lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
        self.model, self.longest = model, max(len(p) for p in prompts) + new_tokens
        columns = -(-self.longest // model.block_size)
        if requests * columns > model.blocks:
            raise RuntimeError("the cache is full")
        self.prompts, self.context, self.ones = prompts, i32([0] * requests), i32([1] * requests)
        self.table = torch.full((requests, columns), -1, dtype=torch.int32, device="cuda")
        self.free, self.turns = torch.arange(model.blocks, dtype=torch.int32, device="cuda"), torch.arange(model.blocks, device="cuda")
        fill = lambda x: torch.full((requests,), x, device="cuda")  # noqa: E731
        self.filters = {"temperatures": fill(float(temperature)), "top_k": fill(top_k).int(), "top_p": fill(float(top_p)), "min_p": fill(float(min_p))}
        self.drawn, self.uniforms, self.probabilities = i32([0] * requests), fill(0.0), fill(0.0)

    def run(self, tokens, lens, most_new, most_keys, rows=None):
        """The requests' new tokens through the model, and the next token of each into `drawn`."""
        n = tokens.shape[0]
        slots, positions = torch.empty(2, n, dtype=torch.int32, device="cuda")
        starts, taken = torch.empty(lens.shape[0] + 1, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
        paged.launchBatchPlan(stream(), self.context, lens, self.table, self.free, self.model.block_size, starts, slots, positions, taken,
                              blocks=self.model.blocks)
        self.free.copy_(self.free[(self.turns + taken) % self.model.blocks])  # the taken ones behind the others
        logits = self.model(tokens, positions, slots, starts, self.context, self.table, most_new, most_keys, rows)
        call = sampling.sample(logits, self.drawn, self.uniforms, probabilities=self.probabilities, **self.filters)
        sampling.launchSample(stream(), call, scratch(sampling.sampleWorkspaceBytes(call)))
        self.context += lens

    def generate(self, uniforms, graph=True):
        """The continuations [requests, new tokens] that the numbers uniforms [new tokens, requests] choose."""
        lens = [len(p) for p in self.prompts]
        self.context.zero_()
        self.uniforms.copy_(uniforms[0])
        last = torch.tensor(lens, device="cuda").cumsum(0) - 1
        self.run(torch.tensor(sum(self.prompts, []), device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda"), max(lens), max(lens), last)
        out = [self.drawn.clone()]

        def step():
            self.run(self.drawn, self.ones, 1, self.longest)

        captured = None
        for u in uniforms[1:]:
            self.uniforms.copy_(u)
            if captured is not None:
                captured.replay()
            else:
                step()
                if graph:  # the first step of its shape ran outside; a capture runs nothing
                    captured = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(captured):
                        step()
            out.append(self.drawn.clone())
        return torch.stack(out, 1)


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--requests", type=int, default=8)
    parser.add_argument("--new-tokens", type=int, default=128)
    parser.add_argument("--temperature", type=float, default=0.8)
    parser.add_argument("--top-k", type=int, default=50)
    parser.add_argument("--top-p", type=float, default=0.95)
    parser.add_argument("--min-p", type=float, default=0.0)
    args = parser.parse_args()
    model = Model()
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, model.embedding.shape[0], (20 + 7 * r,), generator=g).tolist() for r in range(args.requests)]
    uniforms = torch.rand(args.new_tokens, args.requests, generator=g).cuda()
    decoder = Decoder(model, prompts, args.new_tokens, args.temperature, args.top_k, args.top_p, args.min_p)
    for graph in (False, True):
        decoder.generate(uniforms[:3], graph)
        torch.cuda.synchronize()
        began = time.perf_counter()
        tokens = decoder.generate(uniforms, graph).tolist()
        print(f"{'replayed' if graph else 'launched'}: {args.new_tokens} tokens of {args.requests} requests in {time.perf_counter() - began:.3f} s; "
              f"request 0 ends in {tokens[0][-8:]}", flush=True)


if __name__ == "__main__":
    main()
