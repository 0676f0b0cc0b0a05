"""The operators of a speculative serving step that stand beside the quantized matmuls, as timed cases: a matrix product in
8-bit floating point, the plan of a batch over a paged key / value cache, the cache's writes, and attention of a tree of
drafted tokens over it.

A case is a dict of plain values:

  kind "linear"     y = act(x W^T + bias) + residual.  W is e4m3 with one f32 scale per 128 x 128 block; x is f32 and is
                    quantized to e4m3 with one scale per row and 128 columns within the call, or (`quantized`) comes as
                    codes and scales, as where several projections share one input
  kind "plan"       block tables, slots, positions and (`tree`) ancestor masks from the requests' lengths, their drafts'
                    parents and a list of free blocks
  kind "cache"      new keys and values into the slots of their tokens, then (`accept`) the accepted path of every
                    request's tree moved behind its context
  kind "attention"  every request's new tokens over its cached context and, where the mask has them, over each other

The lengths of a case's requests follow from the case alone, so that its work is known; everything else is made from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
BLOCK = 128  # values that share a scale of the 8-bit product
E4M3_MAX = 448.0
TINY = 2.0 ** -100  # smallest maximum that a block's scale is made from
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACTIVATIONS = {"none": 0, "relu": 1, "quick_gelu": 2, "gelu": 3}


def _linear(name, rows, in_dim, out_dim, quantized=False, bias=False, activation="none", residual=False):
    case = {"kind": "linear", "rows": rows, "in_dim": in_dim, "out_dim": out_dim, "quantized": quantized, "bias": bias,
            "activation": activation, "residual": residual}
    return dict(case, name=name) if name else case


def _plan(name, requests, context, drafts, tree, block, spare=0):
    """`context` and `drafts`: (least, most) cached and new tokens of a request; `spare`: token places past the batch's."""
    case = {"kind": "plan", "requests": requests, "context_least": context[0], "context_most": context[1],
            "drafts_least": drafts[0], "drafts_most": drafts[1], "tree": tree, "block": block, "spare": spare}
    return dict(case, name=name) if name else case


def _cache(name, requests, context, drafts, accept, block, kv_heads, dim, source, stored):
    case = {"kind": "cache", "requests": requests, "context_least": context[0], "context_most": context[1],
            "drafts_least": drafts[0], "drafts_most": drafts[1], "accept": accept, "block": block, "kv_heads": kv_heads,
            "dim": dim, "source": source, "stored": stored}
    return dict(case, name=name) if name else case


def _attention(name, requests, context, drafts, mask, block, heads, kv_heads, dim, activations, stored, paged="slots", empty=False):
    """`mask` "tree": ancestors; "chain": every earlier token.  `paged`: which of the slots and the heads of a block lie
    outside.  `empty`: the first request has no context, and the last token of every tree sees nothing."""
    case = {"kind": "attention", "requests": requests, "context_least": context[0], "context_most": context[1],
            "drafts_least": drafts[0], "drafts_most": drafts[1], "mask": mask, "block": block, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "activations": activations, "stored": stored, "paged": paged, "empty": empty}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token's attention output projection: the smallest product, where the call's latency counts
        _linear("linear_m1", 1, 4096, 4096),
        # a batch of verified drafts through the down projection, on codes that came from a fused gate
        _linear("linear_m48_quantized", 48, 14336, 4096, quantized=True),
        # an odd prompt on a small encoder's odd sizes, everything fused behind the product
        _linear("linear_m333_odd", 333, 2000, 1111, bias=True, activation="gelu", residual=True),
        # the largest prompt chunk through an up projection
        _linear("linear_m2048", 2048, 4096, 14336),
        # the plan of one verification step: eight requests with a tree of drafts each
        _plan("plan_tree_b8", 8, (100, 4000), (9, 24), True, 16, spare=11),
        # the plan of a large batch of prompt chunks
        _plan("plan_prompts_b512", 512, (0, 8000), (16, 1000), False, 16),
        # the drafts' keys and values of one verification step, and the accepted paths
        _cache("cache_tree_b8", 8, (100, 4000), (9, 24), 5, 16, 8, 128, "f32", "f16"),
        # a chunk of prompts into the cache
        _cache("cache_prompts_b16", 16, (0, 2000), (300, 700), 0, 32, 8, 128, "f32", "bf16"),
        # four drafts and one more token of one request: the smallest verification
        _attention("attention_chain_b1", 1, (701, 701), (5, 5), "chain", 16, 32, 8, 128, "f32", "f16"),
        # trees of up to 64 drafts, ragged requests
        _attention("attention_tree_b8", 8, (300, 4000), (33, 64), "tree", 16, 32, 8, 128, "bf16", "bf16", empty=True),
        # one token each of 64 requests
        _attention("attention_decode_b64", 64, (100, 4000), (1, 1), "chain", 32, 32, 8, 128, "f32", "bf16", paged="heads"),
        # small trees behind very long contexts, seven query heads to a key head
        _attention("attention_long_b2", 2, (99001, 131000), (7, 13), "tree", 64, 28, 4, 128, "bf16", "bf16"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over the logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["linear", "linear", "plan", "cache", "attention", "attention", "attention"])
    if kind == "linear":
        in_dim, out_dim = 16 * _spread(rng, 16, 896), _spread(rng, 128, 14336)
        # no more than the largest listed product
        rows = min(_spread(rng, 1, 2048), max(1, 2048 * 4096 * 14336 // (in_dim * out_dim)))
        activation = rng.choice(["none", "none", "relu", "quick_gelu", "gelu"])
        return _linear(None, rows, in_dim, out_dim, rng.random() < 0.3, rng.random() < 0.4, activation, rng.random() < 0.3)
    block = rng.choice([8, 16, 16, 24, 32, 64, 128])
    least = _spread(rng, 1, 2000)
    if kind == "plan":
        tree = rng.random() < 0.5
        drafts = _spread(rng, 1, 64 if tree else 1000)
        return _plan(None, _spread(rng, 1, 512), (least, 4 * least), (max(1, drafts // 2), drafts), tree, block, rng.randint(0, 40))
    dim, kv_heads = rng.choice([64, 80, 96, 128, 128, 192, 256]), rng.choice([1, 2, 4, 8, 8, 12])
    if kind == "cache":
        accept = rng.choice([0, 3, 6])
        drafts = _spread(rng, 1, 64 if accept else 500)
        return _cache(None, _spread(rng, 1, 32), (least, 2 * least), (max(1, drafts // 2), drafts), accept, block, kv_heads, dim,
                      rng.choice(["f32", "f32", "f16", "bf16"]), rng.choice(["f16", "bf16"]))
    stored, same = rng.choice(["f16", "bf16"]), rng.random() < 0.5
    group = rng.choice([1, 2, 4, 5, 7, 8])
    requests, drafts = _spread(rng, 1, 64), _spread(rng, 1, 64)
    # cached values no more than the longest listed contexts hold
    most = min(_spread(rng, 16, 131000), max(16, 2 * 131000 * 4 * 128 // (requests * kv_heads * dim)))
    # and no more products than the largest trees on them
    drafts = max(1, min(drafts, 8 * 64 * 32 * 128 * 4000 // (requests * kv_heads * group * dim * most)))
    return _attention(None, requests, (max(1, most // 5), most), (max(1, drafts // 2), drafts), rng.choice(["tree", "chain"]), block,
                      kv_heads * group, kv_heads, dim, stored if same else "f32", stored, rng.choice(["slots", "heads"]),
                      rng.random() < 0.3)


# ---- what follows from a case alone ----------------------------------------------------------------------------------

def _between(count, least, most, turn):
    """`count` whole numbers spread over [least, most] in an order that looks like none."""
    at = (np.arange(1, count + 1) * turn) % 1.0
    return np.minimum(most, least + np.floor(at * (most - least + 1)).astype(np.int64))


def _lengths(case):
    """Cached and new tokens of every request."""
    context = _between(case["requests"], case["context_least"], case["context_most"], 0.6180339887498949)
    drafts = _between(case["requests"], case["drafts_least"], case["drafts_most"], 0.7548776662466927)
    if case.get("empty"):
        context[0] = 0
    return context, drafts


def _blocks(tokens, block):
    return -(-tokens // block)


def work(case):
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["in_dim"], case["out_dim"]
        kb, nb = _blocks(k, BLOCK), _blocks(n, BLOCK)
        moved = n * k + 4 * kb * nb + (m * k + 4 * m * kb if case["quantized"] else 4 * m * k) + 4 * m * n
        moved += 4 * n * case["bias"] + 4 * m * n * case["residual"]
        return {"bytes": moved, "flops": 2 * m * k * n}
    context, drafts = _lengths(case)
    tokens = int(drafts.sum())
    if case["kind"] == "plan":
        owned, needed = _blocks(context, case["block"]), _blocks(context + drafts, case["block"])
        # lengths, new blocks read and written, the last owned block's entry; slot, position (parent, mask) of every token
        moved = case["requests"] * 16 + int((needed - owned).sum()) * 8 + (tokens + case["spare"]) * (20 if case["tree"] else 8)
        return {"bytes": moved, "flops": tokens}
    row = case["kv_heads"] * case["dim"]
    if case["kind"] == "cache":
        size = 4 if case["source"] == "f32" else 2
        moved = tokens * row * 2 * (size + 2) + 4 * tokens
        moved += int(np.minimum(drafts, case["accept"]).sum()) * (row * 8 + 4)
        return {"bytes": moved, "flops": 0}
    size = 4 if case["activations"] == "f32" else 2
    keys = context + drafts
    moved = int(keys.sum()) * row * 2 * 2 + 2 * tokens * case["heads"] * case["dim"] * size
    moved += 4 * int(_blocks(keys, case["block"]).sum()) + 8 * tokens * (case["mask"] == "tree")
    return {"bytes": moved, "flops": 4 * int((drafts * keys).sum()) * case["heads"] * case["dim"]}


# ---- inputs ----------------------------------------------------------------------------------------------------------

class _Source:
    def __init__(self, seed):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(seed)
        self.rng = np.random.default_rng(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=DEVICE)

    def hidden(self, rows, dim):
        """What enters a projection: normal values, some channels many times larger."""
        x = self.normal(rows, dim)
        return x * torch.where(torch.rand(dim, generator=self.gen, device=DEVICE) < 0.005, 20.0, 1.0)

    def shuffled(self, count):
        return torch.randperm(count, generator=self.gen, device=DEVICE).to(torch.int32)


def _int32(values):
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).to(DEVICE)


def _whole_blocks(rows, cols):
    return _blocks(rows, BLOCK) * BLOCK, _blocks(cols, BLOCK) * BLOCK


def _checkpoint_weight(src, out_dim, in_dim):
    """A matrix as a checkpoint has it: codes of the values over their block's scale, the largest of each block at the type's."""
    padded = torch.zeros(*_whole_blocks(out_dim, in_dim), device=DEVICE)
    padded[:out_dim, :in_dim] = src.normal(out_dim, in_dim) * (0.5 + torch.rand(out_dim, 1, generator=src.gen, device=DEVICE)) * in_dim ** -0.5
    blocks = padded.view(padded.shape[0] // BLOCK, BLOCK, padded.shape[1] // BLOCK, BLOCK)
    scales = blocks.abs().amax(dim=(1, 3)) / E4M3_MAX
    codes = (blocks / scales[:, None, :, None]).to(torch.float8_e4m3fn).view(padded.shape)
    return codes[:out_dim, :in_dim].contiguous(), scales


def _tree_parents(rng, drafts):
    """Parents within each request's tree, -1 behind the context; a token's parent comes before it."""
    parents = []
    for count in drafts:
        reach = rng.integers(1, 9)  # bushy and narrow trees
        parents += [int(rng.integers(max(-1, t - reach), t)) if t else -1 for t in range(count)]
    return np.array(parents, np.int32)


def _ancestor_masks(parents, drafts):
    """Bit p of a token's mask: token p of its request is the token itself or one of its ancestors."""
    masks, at = np.zeros(len(parents), np.uint64), 0
    for count in drafts:
        for t in range(count):
            parent = parents[at + t]
            masks[at + t] = np.uint64(1 << t) | (masks[at + parent] if parent >= 0 else np.uint64(0))
        at += count
    return masks


def _starts(drafts):
    return np.concatenate([[0], np.cumsum(drafts)])


def _tables(src, held, columns, spare_blocks):
    """A table [requests, columns] of blocks in no order, -1 past each request's; and the blocks that it leaves."""
    total = int(held.sum())
    blocks = src.shuffled(total + spare_blocks).cpu().numpy()
    table = np.full((len(held), columns), -1, np.int32)
    table[np.arange(columns)[None, :] < held[:, None]] = blocks[:total]
    return _int32(table), _int32(blocks[total:])


def _slots(table, context, drafts, block):
    """The slot of every new token."""
    table, request = table.cpu().numpy(), np.repeat(np.arange(len(drafts)), drafts)
    position = context[request] + np.arange(drafts.sum()) - _starts(drafts)[request]
    return _int32(table[request, position // block] * block + position % block)


def prepare(case, seed):
    src = _Source(seed)
    if case["kind"] == "linear":
        m, k, n = case["rows"], case["in_dim"], case["out_dim"]
        state = {"x": src.hidden(m, k)}
        if case["quantized"]:
            state["q"], state["q_scales"] = _quantize(state.pop("x"))
        state["weight"], state["scales"] = _checkpoint_weight(src, n, k)
        state["bias"] = src.normal(n) * 0.1 if case["bias"] else None
        state["residual"] = src.normal(m, n) if case["residual"] else None
        state["y"] = torch.empty(m, n, device=DEVICE)
        return dict(state, case=case)
    context, drafts = _lengths(case)
    tokens, block, requests = int(drafts.sum()), case["block"], case["requests"]
    columns = int(_blocks(context + drafts, block).max()) + 1
    state = {"case": case, "context": _int32(context), "drafts": _int32(drafts), "starts": _int32(_starts(drafts))}
    if case["kind"] == "plan":
        owned, needed = _blocks(context, block), int((_blocks(context + drafts, block) - _blocks(context, block)).sum())
        state["table"], state["free"] = _tables(src, owned, columns, needed + 17)
        state["places"] = places = tokens + case["spare"]
        state["parents"] = _int32(np.concatenate([_tree_parents(src.rng, drafts), np.full(case["spare"], -1)])) if case["tree"] else None
        state["out"] = {"starts": torch.empty(requests + 1, dtype=torch.int32, device=DEVICE),
                        "slots": torch.empty(places, dtype=torch.int32, device=DEVICE),
                        "positions": torch.empty(places, dtype=torch.int32, device=DEVICE),
                        "taken": torch.empty(1, dtype=torch.int32, device=DEVICE)}
        if case["tree"]:
            state["out"]["masks"] = torch.empty(places, 1, dtype=torch.int64, device=DEVICE)
        return state
    state["table"], _ = _tables(src, _blocks(context + drafts, block), columns, 9)
    blocks = int(_blocks(context + drafts, block).sum()) + 9
    kv_heads, dim, stored = case["kv_heads"], case["dim"], TYPES[case["stored"]]
    if case["kind"] == "cache":
        state["cache"] = [torch.empty(blocks, block, kv_heads, dim, dtype=stored, device=DEVICE).normal_(generator=src.gen) for _ in "kv"]
        state["new"] = [src.normal(tokens, kv_heads, dim).to(TYPES[case["source"]]) for _ in "kv"]
        state["slots"] = _slots(state["table"], context, drafts, block)
        if case["accept"]:
            count = np.minimum(drafts, case["accept"])
            paths = np.full((requests, case["accept"]), -1)
            for r in range(requests):
                paths[r, :count[r]] = np.sort(src.rng.choice(drafts[r], count[r], replace=False))
            state["paths"], state["accepted"] = _int32(paths), _int32(count)
        return state
    shape = (blocks, block, kv_heads, dim) if case["paged"] == "slots" else (blocks, kv_heads, block, dim)
    state["cache"] = [torch.empty(shape, dtype=stored, device=DEVICE).normal_(generator=src.gen) for _ in "kv"]
    # scores of a few units: some rows look at a handful of keys, others at many
    spread = 0.5 + 2.0 * torch.rand(tokens, case["heads"], 1, generator=src.gen, device=DEVICE)
    state["q"] = (src.normal(tokens, case["heads"], dim) * spread).to(TYPES[case["activations"]])
    state["out"] = torch.empty_like(state["q"])
    state["masks"] = None
    if case["mask"] == "tree":
        masks = _ancestor_masks(_tree_parents(src.rng, drafts), drafts)
        if case["empty"]:
            masks[_starts(drafts)[1:] - 1] = 0
        state["masks"] = torch.from_numpy(masks.view(np.int64)).to(DEVICE).view(tokens, 1)
    state["longest"] = {"keys": int((context + drafts).max()), "drafts": int(drafts.max())}
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"linear": _own_linear, "plan": _own_plan, "cache": _own_cache, "attention": _own_attention}[kind](state)
    return {"linear": _plain_linear, "plan": _plain_plan, "cache": _plain_cache, "attention": _plain_attention}[kind](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


_scratch = {}


def _workspace(count):
    """The scratch that a program lends to every call, as large as the largest has asked for."""
    held = _scratch.get("bytes")
    if held is None or held.numel() < count:
        held = _scratch["bytes"] = torch.empty(max(count, 1 << 20), dtype=torch.uint8, device=DEVICE)
    return held


def _own_linear(state):
    from antfly_amd import kernels
    from antfly_amd.paged import buffer
    case = state["case"]
    m, k, n = case["rows"], case["in_dim"], case["out_dim"]
    extra = {"bias": buffer(state["bias"]), "residual": buffer(state["residual"]), "activation": ACTIVATIONS[case["activation"]],
             "workspace": buffer(_workspace(kernels.linearFp8WorkspaceBytes(m, k, n)))}
    y, weight, scales = buffer(state["y"]), buffer(state["weight"]), buffer(state["scales"])
    if case["quantized"]:
        kernels.launchMatmulFp8F32(_stream(), y, buffer(state["q"]), buffer(state["q_scales"]), weight, scales, m, k, n, **extra)
    else:
        kernels.launchLinearFp8F32(_stream(), y, buffer(state["x"]), weight, scales, m, k, n, **extra)
    return state["y"]


def _own_plan(state):
    from antfly_amd import paged
    out = state["out"]
    paged.launchBatchPlan(_stream(), state["context"], state["drafts"], state["table"], state["free"], state["case"]["block"],
                          out["starts"], out["slots"], out["positions"], out["taken"], parents=state["parents"],
                          masks=out.get("masks"))
    return dict(out, table=state["table"])


def _own_cache(state):
    from antfly_amd import paged
    case, stream = state["case"], _stream()
    cache = paged.cache(state["cache"][0], state["cache"][1])
    paged.launchCacheStore(stream, cache, state["new"][0], state["new"][1], state["slots"])
    if case["accept"]:
        paged.launchCacheMove(stream, cache, state["table"], state["context"], state["paths"], state["accepted"])
    return state["cache"]


def _own_attention(state):
    from antfly_amd import paged
    cache = paged.cache(state["cache"][0], state["cache"][1], heads_outside=state["case"]["paged"] == "heads")
    call = paged.treeAttention(cache, state["out"], state["q"], state["starts"], state["context"], state["table"],
                               state["longest"]["drafts"], state["longest"]["keys"], masks=state["masks"])
    paged.launchTreeAttention(_stream(), call, _workspace(paged.treeAttentionWorkspaceBytes(call)))
    return state["out"]


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _quantize(x):
    """Codes e4m3 [rows, in_dim] and f32 scales [rows, blocks]: scale = max |x| / 448 over 128 values of a row, code = x (448 / max)."""
    rows, dim = x.shape
    count = _blocks(dim, BLOCK)
    padded = torch.nn.functional.pad(x, (0, count * BLOCK - dim)).view(rows, count, BLOCK)
    most = padded.abs().amax(dim=2).clamp_min(TINY)
    largest = torch.full_like(most, E4M3_MAX)
    codes = (padded * (largest / most)[:, :, None]).to(torch.float8_e4m3fn)
    return codes.view(rows, count * BLOCK)[:, :dim].contiguous(), most / largest


def _values(codes, scales, rows_to_scale):
    """What codes stand for: one scale per `rows_to_scale` rows and 128 columns."""
    wide = scales.repeat_interleave(rows_to_scale, 0)[:codes.shape[0]].repeat_interleave(BLOCK, 1)[:, :codes.shape[1]]
    return codes.float() * wide


def _activate(y, activation):
    if activation == "relu":
        return y.clamp_min(0.0)
    if activation == "quick_gelu":
        return y / (1.0 + torch.exp(-1.702 * y))
    if activation == "gelu":
        return 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    return y


def _plain_linear(state):
    q, q_scales = (state["q"], state["q_scales"]) if state["case"]["quantized"] else _quantize(state["x"])
    y = _values(q, q_scales, 1) @ _values(state["weight"], state["scales"], BLOCK).t()
    if state["bias"] is not None:
        y = y + state["bias"]
    y = _activate(y, state["case"]["activation"])
    return y if state["residual"] is None else y + state["residual"]


def _plain_plan(state):
    case, block, table = state["case"], state["case"]["block"], state["table"]
    context, drafts, free = state["context"].long(), state["drafts"].long(), state["free"].long()
    owned, needed = (context + block - 1) // block, (context + drafts + block - 1) // block
    ends = torch.cumsum(drafts, 0)
    starts = torch.nn.functional.pad(ends, (1, 0))
    taken_before = torch.nn.functional.pad(torch.cumsum(needed - owned, 0), (1, 0))
    at = torch.arange(table.shape[1], device=DEVICE)[None, :]
    fresh = (at >= owned[:, None]) & (at < needed[:, None])
    from_free = (taken_before[:-1, None] + at - owned[:, None]).clamp(0, free.numel() - 1)
    table = torch.where(fresh, free[from_free], table.long())
    token = torch.arange(state["places"], device=DEVICE)
    live = token < ends[-1]
    request = torch.searchsorted(ends, token, right=True).clamp_max(case["requests"] - 1)
    own_at = token - starts[request]
    position = context[request] + own_at
    slot = table[request, (position // block).clamp_max(table.shape[1] - 1)] * block + position % block
    out = {"starts": starts.int(), "slots": torch.where(live, slot, -1).int(), "taken": taken_before[-1:].int(), "table": table.int()}
    if case["tree"]:
        # a token reaches its ancestors in so many steps from child to parent
        parent, most = state["parents"].long(), case["drafts_most"]
        step = torch.zeros(case["requests"], most, most, device=DEVICE)
        has = live & (parent >= 0)
        step[request[has], own_at[has], parent[has]] = 1.0
        reach = (torch.matrix_power(step + torch.eye(most, device=DEVICE), most) > 0).long()
        masks = (reach << torch.arange(most, device=DEVICE)).sum(2)
        out["masks"] = torch.where(live, masks[request, own_at.clamp(0, most - 1)], 0)[:, None]
        position = context[request] + reach.sum(2)[request, own_at.clamp(0, most - 1)] - 1
    out["positions"] = torch.where(live, position, -1).int()
    return out


def _plain_cache(state):
    case, block = state["case"], state["case"]["block"]
    slots, moved = state["slots"].long(), []
    if case["accept"]:
        step = torch.arange(case["accept"], device=DEVICE)[None, :]
        live = step < state["accepted"][:, None]
        request = torch.arange(case["requests"], device=DEVICE)[:, None].expand_as(live)[live]
        start = state["context"].long()[request]
        source, target = start + state["paths"].long()[live], start + step.expand_as(live)[live]
        moved = [state["table"].long()[request, p // block] * block + p % block for p in (source, target)]
    return [_stored(cache, new, slots, moved) for cache, new in zip(state["cache"], state["new"])]


def _stored(cache, new, slots, moved):
    rows = cache.view(-1, *cache.shape[2:])
    rows[slots] = new.to(cache.dtype)
    if moved:
        rows[moved[1]] = rows[moved[0]]
    return cache


def _plain_attention(state):
    case, block = state["case"], state["case"]["block"]
    requests, heads, kv_heads, dim = case["requests"], case["heads"], case["kv_heads"], case["dim"]
    keys, drafts, group = state["longest"]["keys"], state["longest"]["drafts"], heads // kv_heads
    context, starts = state["context"].long(), state["starts"].long()
    count = starts[1:] - starts[:-1]
    tokens = state["q"].shape[0]
    at, t = torch.arange(keys, device=DEVICE), torch.arange(drafts, device=DEVICE)
    token = (starts[:-1, None] + t).clamp_max(tokens - 1)
    draft = at[None, :] - context[:, None]  # which draft a key is; below zero: of the context
    if state["masks"] is None:
        seen = draft[:, None, :] <= t[None, :, None]
    else:
        bits = state["masks"][:, 0][token][:, :, None] >> draft.clamp(0, 63)[:, None, :]
        seen = (draft < 0)[:, None, :] | ((bits & 1) == 1)
    held = draft < count[:, None]
    seen = seen & held[:, None, :]
    page = state["table"].long()[:, at // block].clamp_min(0)
    lined = [c if case["paged"] == "slots" else c.transpose(1, 2) for c in state["cache"]]
    # [requests, kv heads, keys, dim], nothing of what lies past a request's keys
    k, v = (torch.where(held[:, :, None, None], c[page, at % block].float(), 0.0).transpose(1, 2).contiguous() for c in lined)
    q = state["q"].float()[token].view(requests, drafts, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(requests, kv_heads, -1, dim)
    scores = (q @ k.transpose(2, 3)).view(requests, kv_heads, drafts, group, keys) * dim ** -0.5
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    most = scores.amax(-1, keepdim=True).clamp_min(-3e38)
    weights = torch.exp(scores - most)
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(requests, kv_heads, drafts * group, keys) @ v).view(requests, kv_heads, drafts, group, dim)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 2, 1, 3, 4).reshape(requests, drafts, heads, dim)
    request = torch.searchsorted(starts[1:], torch.arange(tokens, device=DEVICE), right=True)
    return out[request, torch.arange(tokens, device=DEVICE) - starts[request]].to(state["q"].dtype)


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"linear": _exact_linear, "plan": _exact_plan, "cache": _exact_cache, "attention": _exact_attention}[case["kind"]](state)


def _e4m3(x):
    """The nearest number of the type with 4 exponent and 3 mantissa bits, ties to the even one, in 64 bits."""
    exponent = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0)
    step = torch.exp2(exponent - 3.0)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_linear(state):
    weight, scales = state["weight"].double(), state["scales"].double()
    n, k = weight.shape
    y = torch.zeros(state["case"]["rows"], n, dtype=torch.float64, device=DEVICE)
    row_block = torch.arange(n, device=DEVICE) // BLOCK
    for b in range(_blocks(k, BLOCK)):
        part = slice(b * BLOCK, min(k, (b + 1) * BLOCK))
        if state["case"]["quantized"]:
            x = state["q"][:, part].double() * state["q_scales"][:, b, None].double()
        else:  # the codes are rounded from f32 products, and the scale is an f32: both are part of the definition
            most = state["x"][:, part].abs().amax(1, keepdim=True).clamp_min(TINY)
            ratio = (E4M3_MAX / most.double()).float()
            x = _e4m3((state["x"][:, part] * ratio).double()) * (most.double() / E4M3_MAX).float().double()
        y += x @ (weight[:, part] * scales[row_block, b, None]).t()
    if state["bias"] is not None:
        y += state["bias"].double()
    kind = state["case"]["activation"]
    if kind == "relu":
        y = torch.where(y < 0, 0.0, y)
    elif kind == "quick_gelu":
        y = y * torch.sigmoid(1.702 * y)
    elif kind == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
    return y if state["residual"] is None else y + state["residual"].double()


def _exact_plan(state):
    return None  # whole numbers


def _exact_cache(state):
    case, block = state["case"], state["case"]["block"]
    slots, table = state["slots"].cpu().numpy(), state["table"].cpu().numpy()
    caches = []
    for cache, new in zip(state["cache"], state["new"]):
        rows = cache.double().view(-1, *cache.shape[2:])
        rows[torch.from_numpy(slots).to(DEVICE).long()] = new.double()
        if case["accept"]:
            paths, context, count = (state[name].cpu().numpy() for name in ("paths", "context", "accepted"))
            for r in range(case["requests"]):
                for i in range(count[r]):  # in order: a place is read before a later step writes it
                    source, target = context[r] + paths[r, i], context[r] + i
                    rows[table[r, target // block] * block + target % block] = rows[table[r, source // block] * block + source % block]
        caches.append(rows.view(cache.shape))
    return caches


def _exact_attention(state):
    case, block = state["case"], state["case"]["block"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    starts, context, table = (state[name].cpu().numpy() for name in ("starts", "context", "table"))
    lined = [c if case["paged"] == "slots" else c.transpose(1, 2) for c in state["cache"]]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    for r in range(case["requests"]):
        first, last, cached = int(starts[r]), int(starts[r + 1]), int(context[r])
        total, t = cached + last - first, last - first
        pages = torch.from_numpy(table[r, :_blocks(total, block)]).to(DEVICE).long()
        k, v = (c[pages].flatten(0, 1)[:total].double() for c in lined)
        seen = torch.ones(t, total, dtype=torch.bool, device=DEVICE)
        if state["masks"] is None:
            seen[:, cached:] = torch.ones(t, t, dtype=torch.bool, device=DEVICE).tril()
        else:
            seen[:, cached:] = (state["masks"][first:last] >> torch.arange(t, device=DEVICE)) & 1 == 1
        rows = seen.any(1)
        for h in range(heads):
            g = h // (heads // kv_heads)
            scores = (state["q"][first:last, h].double() @ k[:, g].t().contiguous()) / math.sqrt(dim)
            weights = torch.softmax(scores.masked_fill(~seen, -math.inf)[rows], -1)
            out[first:last, h][rows] = weights @ v[:, g].contiguous()
    return out
