"""Speculative decoding over a paged cache with the library's operators: a small decoder of random weights, its projections in
8-bit floating point, verifies a tree of drafted tokens for every request at once.

A step:  plan the batch (slots, positions, ancestor masks) -> per layer: project, store keys and values, attend over context
and tree, project back -> the longest drafted path that the model agrees with -> its keys and values move behind the context.

    python examples/speculative_decode.py --requests 4 --new-tokens 96 --drafts 15
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from antfly_amd import _lib, kernels, paged  # noqa: E402

GELU = _lib.ACTIVATION_GELU
BLOCK = 128  # rows and columns of a weight that share a scale


def stream():
    return torch.cuda.current_stream().cuda_stream


class Linear:
    """A weight in e4m3 with a scale per 128 x 128; f32 in and out."""

    def __init__(self, weight):
        self.out_dim, self.in_dim = weight.shape
        rows, columns = -(-self.out_dim // BLOCK), -(-self.in_dim // BLOCK)
        padded = torch.zeros(rows * BLOCK, columns * BLOCK)
        padded[:self.out_dim, :self.in_dim] = weight
        blocks = padded.view(rows, BLOCK, columns, BLOCK)
        scales = blocks.abs().amax((1, 3)).clamp_min(1e-20) / 448.0
        codes = (blocks / scales[:, None, :, None]).view(padded.shape)[:self.out_dim, :self.in_dim].contiguous()
        self.codes = codes.to(torch.float8_e4m3fn).view(torch.uint8).cuda()
        self.scales = scales.contiguous().cuda()

    def __call__(self, x, residual=None, activation=0):
        rows = x.shape[0]
        y = torch.empty(rows, self.out_dim, device="cuda")
        workspace = torch.empty(kernels.linearFp8WorkspaceBytes(rows, self.in_dim, self.out_dim), dtype=torch.uint8, device="cuda")
        kernels.launchLinearFp8F32(stream(), paged.buffer(y), paged.buffer(x), paged.buffer(self.codes), paged.buffer(self.scales),
                                   rows, self.in_dim, self.out_dim, residual=paged.buffer(residual), activation=activation,
                                   workspace=paged.buffer(workspace))
        return y


def norm(x):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6)


def rotate(x, positions):
    """Rotary embedding of [tokens, heads, dim]."""
    half = x.shape[-1] // 2
    angle = positions.float()[:, None] * 10000.0 ** (-torch.arange(half, device=x.device) / half)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


class Model:
    def __init__(self, vocab=512, hidden=512, layers=2, heads=8, kv_heads=2, head_dim=64, blocks=256, block_size=16, seed=1):
        g = torch.Generator().manual_seed(seed)

        def weight(out_dim, in_dim):
            return torch.randn(out_dim, in_dim, generator=g) * in_dim ** -0.5

        self.heads, self.kv_heads, self.head_dim, self.block_size, self.blocks = heads, kv_heads, head_dim, block_size, blocks
        self.embedding = torch.randn(vocab, hidden, generator=g).cuda()
        self.layers = []
        for _ in range(layers):
            keys, values = (torch.zeros(blocks, block_size, kv_heads, head_dim, dtype=torch.float16, device="cuda") for _ in range(2))
            self.layers.append({"qkv": Linear(weight((heads + 2 * kv_heads) * head_dim, hidden)), "out": Linear(weight(hidden, heads * head_dim)),
                                "up": Linear(weight(4 * hidden, hidden)), "down": Linear(weight(hidden, 4 * hidden)),
                                "cache": paged.cache(keys, values)})
        self.head = Linear(weight(vocab, hidden))

    def __call__(self, tokens, positions, slots, starts, context, table, most_new, most_keys, masks):
        """The logits of a batch's new tokens [tokens, vocab]; their keys and values are in the cache afterwards."""
        n, kv = tokens.shape[0], self.kv_heads
        x = self.embedding[tokens]
        for layer in self.layers:
            qkv = layer["qkv"](norm(x)).view(n, self.heads + 2 * kv, self.head_dim)
            q, k = rotate(qkv[:, :self.heads], positions), rotate(qkv[:, self.heads:self.heads + kv], positions)
            v = qkv[:, self.heads + kv:].contiguous()
            paged.launchCacheStore(stream(), layer["cache"], k, v, slots)
            seen = torch.empty_like(q)
            attention = paged.treeAttention(layer["cache"], seen, q, starts, context, table, most_new, most_keys, masks=masks)
            workspace = torch.empty(paged.treeAttentionWorkspaceBytes(attention), dtype=torch.uint8, device="cuda")
            paged.launchTreeAttention(stream(), attention, workspace)
            x = layer["out"](seen.view(n, -1), residual=x)
            x = layer["down"](layer["up"](norm(x), activation=GELU), residual=x)
        return self.head(norm(x))


class Decoder:
    """Requests over one cache: their contexts, block tables and the blocks that nobody owns."""

    def __init__(self, model, requests, longest):
        self.model, self.context = model, [0] * requests
        self.table = torch.full((requests, -(-longest // model.block_size)), -1, dtype=torch.int32, device="cuda")

    def _free(self):
        table, taken = self.table.tolist(), set()
        for row, context in zip(table, self.context):
            taken.update(row[:-(-context // self.model.block_size)])
        return [b for b in range(self.model.blocks) if b not in taken]

    def run(self, tokens, parents=None):
        """tokens[r]: the new ones of request r, with parents[r] as a tree.  The model's choice after each of them."""
        lens = [len(t) for t in tokens]
        n, most = sum(lens), max(lens)
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        context, slots, positions = i32(self.context), *torch.empty(2, n, dtype=torch.int32, device="cuda")
        starts, taken = torch.empty(len(lens) + 1, dtype=torch.int32, device="cuda"), torch.empty(1, dtype=torch.int32, device="cuda")
        masks = torch.empty(n, -(-most // 64), dtype=torch.int64, device="cuda") if parents else None
        free = i32(self._free())
        paged.launchBatchPlan(stream(), context, i32(lens), self.table, free, self.model.block_size, starts, slots, positions, taken,
                              parents=i32(sum(parents, [])) if parents else None, masks=masks, blocks=self.model.blocks)
        if int(taken) > free.numel() or int(slots.min()) < 0:
            raise RuntimeError("the cache is full")
        logits = self.model(torch.tensor(sum(tokens, []), device="cuda"), positions, slots, starts, context, self.table, most,
                            most + max(self.context), masks)
        choice = logits.argmax(-1).tolist()
        return [choice[a:a + m] for a, m in zip(starts.tolist(), lens)]

    def accept(self, paths):
        """paths[r]: the tree's tokens that stay, from the root on; the others' places are free again."""
        lens, longest = [len(p) for p in paths], max(len(p) for p in paths)
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        context, table = i32(self.context), i32([p + [-1] * (longest - len(p)) for p in paths])
        for layer in self.model.layers:
            paged.launchCacheMove(stream(), layer["cache"], self.table, context, table, i32(lens))
        self.context = [c + m for c, m in zip(self.context, lens)]


def draft(history, drafts, width=2):
    """A tree behind the last token: its children are the latest successors that a token has had so far."""
    after = {}
    for a, b in zip(history, history[1:]):
        seen = after.setdefault(a, [])
        if b in seen:
            seen.remove(b)
        seen.insert(0, b)
    tokens, parents, at = [history[-1]], [-1], 0
    while at < len(tokens) and len(tokens) <= drafts:
        for t in after.get(tokens[at], [])[:width]:
            if len(tokens) <= drafts:
                tokens.append(t)
                parents.append(at)
        at += 1
    return tokens, parents


def agreed(tokens, parents, choice):
    """The path from the root along the model's choices, and its choice at the end."""
    path = [0]
    while True:
        wanted = choice[path[-1]]
        child = next((i for i in range(len(tokens)) if parents[i] == path[-1] and tokens[i] == wanted), None)
        if child is None:
            return path, wanted
        path.append(child)


def generate(model, prompts, new_tokens, drafts):
    """Greedy continuations of the prompts, and the number of steps that they took."""
    decoder = Decoder(model, len(prompts), max(len(p) for p in prompts) + new_tokens + 2 * drafts + 2)
    history = [list(p) for p in prompts]
    for h, choice in zip(history, decoder.run(history)):
        h.append(choice[-1])
    decoder.context = [len(p) for p in prompts]  # a chain's tokens lie where they belong
    steps = 0
    while min(len(h) - len(p) for h, p in zip(history, prompts)) < new_tokens:
        trees = [draft(h, drafts if len(h) - len(p) < new_tokens else 0) for h, p in zip(history, prompts)]
        found = [agreed(t, p, c) for (t, p), c in zip(trees, decoder.run([t for t, _ in trees], [p for _, p in trees]))]
        done = [len(h) - len(p) >= new_tokens for h, p in zip(history, prompts)]
        decoder.accept([[] if d else path for d, (path, _) in zip(done, found)])
        for h, d, (tokens, _), (path, last) in zip(history, done, trees, found):
            if not d:
                h.extend([tokens[i] for i in path[1:]] + [last])
        steps += 1
    return [h[len(p):len(p) + new_tokens] for h, p in zip(history, prompts)], steps


def main():
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--requests", type=int, default=4)
    parser.add_argument("--new-tokens", type=int, default=96)
    parser.add_argument("--drafts", type=int, default=15)
    args = parser.parse_args()
    model = Model()
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, model.embedding.shape[0], (20 + 7 * r,), generator=g).tolist() for r in range(args.requests)]
    for drafts in (0, args.drafts):
        generate(model, prompts, 4, drafts)
        torch.cuda.synchronize()
        began = time.perf_counter()
        tokens, steps = generate(model, prompts, args.new_tokens, drafts)
        print(f"{drafts} drafts a request: {steps} steps for {args.new_tokens} tokens, {time.perf_counter() - began:.3f} s; "
              f"request 0 ends in {tokens[0][-8:]}", flush=True)


if __name__ == "__main__":
    main()
