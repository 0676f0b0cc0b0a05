"""The operators of a sampled serving step on an 8-bit paged key / value cache, as timed cases.

A case is a dict of plain values:

  kind "rotate"     queries and keys of a projection, normed head by head and rotated by their tokens' positions; `store`: the keys
                    and the values go straight into an e4m3 or 16-bit paged cache, otherwise both come back as arrays
  kind "cache"      new keys and values quantized into the slots of their tokens, then `read` tokens of the request read back
  kind "attention"  every request's new tokens over its quantized cache: scores capped by a tanh, biased by distance, in a window
  kind "sample"     a token of every row of logits by temperature, top-k, top-p and min-p from a given random number, likely ones first

The lengths of a case's requests follow from the case alone, so that its work is known; everything else is made from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
TINY = 2.0 ** -100  # smallest maximum that a head's scale is made from
LARGEST = {"e4m3": 448.0, "i8": 127.0}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8}
SIZES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "i8": 1}


def _rotate(name, tokens, heads, kv_heads, dim, rotary, source, out, store="none", norm=True, interleaved=False, axes=1, reach=131000):
    """`rotary`: dimensions of a head that turn; `axes`: positions of a token; `reach`: the largest position."""
    case = {"kind": "rotate", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary, "source": source,
            "out": out, "store": store, "norm": norm, "interleaved": interleaved, "axes": axes, "reach": reach}
    return dict(case, name=name) if name else case


def _cache(name, tokens, read, block, kv_heads, dim, source, stored, out):
    """`read`: tokens that are read back behind the store of `tokens` new ones."""
    case = {"kind": "cache", "tokens": tokens, "read": read, "block": block, "kv_heads": kv_heads, "dim": dim, "source": source,
            "stored": stored, "out": out}
    return dict(case, name=name) if name else case


def _attention(name, requests, context, new, block, heads, kv_heads, dim, activations, stored, cap=0.0, window=0, bias=False,
               paged="slots"):
    """`context` and `new`: (least, most) cached and new tokens of a request.  `paged`: which of the slots and the heads of a
    block lie outside."""
    case = {"kind": "attention", "requests": requests, "context_least": context[0], "context_most": context[1], "new_least": new[0],
            "new_most": new[1], "block": block, "heads": heads, "kv_heads": kv_heads, "dim": dim, "activations": activations,
            "stored": stored, "cap": cap, "window": window, "bias": bias, "paged": paged}
    return dict(case, name=name) if name else case


def _sample(name, rows, vocab, source, filters="all", spread=2.5):
    """`filters`: which of k, p and m (top-k, top-p, min-p) rows use; "all": each row has its own set.  `spread`: of the logits."""
    case = {"kind": "sample", "rows": rows, "vocab": vocab, "source": source, "filters": filters, "spread": spread}
    return dict(case, name=name) if name else case


def listed():
    return [
        # between the projection and the attention of one token: the smallest call, where latency counts
        _rotate("rotate_b1", 1, 32, 8, 128, 128, "f32", "f32", "e4m3"),
        # image and text tokens with positions in time, height and width, keys and queries back as arrays
        _rotate("rotate_axes_t2111", 2111, 28, 4, 128, 96, "bf16", "bf16", axes=3, interleaved=True, reach=4000),
        # a chunk of prompts, 16 bits a query for the attention behind it
        _rotate("rotate_prompts_t7500", 7500, 32, 8, 128, 128, "f32", "bf16", "e4m3"),
        # one token each of 64 requests into the cache
        _cache("cache_b64", 64, 64, 16, 8, 128, "f32", "e4m3", "f16"),
        # a chunk of a prompt into the cache, the whole prompt back for a 16-bit attention
        _cache("cache_chunk_t4000", 4000, 30001, 32, 8, 128, "f32", "i8", "bf16"),
        # one token of one request: the smallest attention
        _attention("attention_b1", 1, (700, 700), (1, 1), 16, 32, 8, 128, "f32", "e4m3"),
        # one token each of 64 requests
        _attention("attention_b64", 64, (100, 4000), (1, 1), 32, 32, 8, 128, "f32", "i8", paged="heads"),
        # chains of drafts on a model with capped scores and a sliding window, odd sizes
        _attention("attention_chain_b16", 16, (300, 9000), (3, 7), 24, 20, 4, 96, "f16", "e4m3", cap=50.0, window=4095),
        # one token behind very long contexts, seven query heads to a key head, scores that fall with distance
        _attention("attention_long_b2", 2, (99001, 131000), (1, 1), 64, 28, 4, 128, "bf16", "e4m3", bias=True),
        # the next token of one request
        _sample("sample_b1", 1, 32000, "f32", "kp"),
        # verified drafts of a few requests, 16-bit logits full of ties
        _sample("sample_b24_bf16", 24, 100003, "bf16", "all"),
        # a large batch
        _sample("sample_b256", 256, 128000, "f32", "all"),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over the logarithm."""
    return min(high, max(low, round(low * (high / low) ** rng.random())))


def draw(rng):
    kind = rng.choice(["rotate", "rotate", "cache", "cache", "attention", "attention", "attention", "attention", "sample", "sample", "sample"])
    if kind == "sample":
        vocab = _spread(rng, 1000, 128000)
        rows = _spread(rng, 1, 256)
        return _sample(None, rows, vocab, rng.choice(["f32", "f32", "f16", "bf16"]), rng.choice(["none", "k", "p", "m", "kp", "pm", "all", "all"]),
                       rng.choice([0.5, 1.0, 2.5, 4.0]))
    dim, kv_heads = rng.choice([64, 80, 96, 112, 128, 128, 128, 192, 256]), rng.choice([1, 2, 4, 8, 8, 10])
    group = rng.choice([1, 2, 3, 4, 5, 7, 8])
    if kind == "rotate":
        tokens = _spread(rng, 1, max(16, 7500 * 48 * 128 // (kv_heads * (group + 2) * dim) * 2 // 3))
        rotary = rng.choice([dim, dim, dim // 2, dim // 4 * 2])
        store, source = rng.choice(["none", "e4m3", "e4m3", "f16", "bf16"]), rng.choice(["f32", "f32", "f16", "bf16"])
        axes = rng.choice([1, 1, 2, 3])
        return _rotate(None, tokens, kv_heads * group, kv_heads, dim, rotary, source, rng.choice([source, "f32", "bf16"]), store,
                       rng.random() < 0.7, rng.random() < 0.4, axes, rng.choice([2000, 131000, 1000000]))
    block = rng.choice([8, 16, 16, 24, 32, 64, 128])
    stored = rng.choice(["e4m3", "i8"])
    if kind == "cache":
        room = 30001 * 8 * 128 // (kv_heads * dim)
        tokens = _spread(rng, 1, min(4000, room))
        return _cache(None, tokens, rng.choice([tokens, _spread(rng, tokens, room)]), block, kv_heads, dim,
                      rng.choice(["f32", "f32", "f16", "bf16"]), stored, rng.choice(["f32", "f16", "bf16"]))
    requests, new = _spread(rng, 1, 64), rng.choice([1, 1, 1, _spread(rng, 2, 16)])
    # cached values no more than the longest listed contexts hold, and no more products
    most = min(_spread(rng, 16, 131000), max(16, 2 * 110000 * 4 * 128 // (requests * kv_heads * dim)))
    new = max(1, min(new, 2 * 131000 * 28 * 128 // (requests * kv_heads * group * dim * most)))
    cap, window = rng.choice([0.0, 0.0, 30.0, 50.0]), rng.choice([0, 0, 0, _spread(rng, 16, 8000)])
    return _attention(None, requests, (max(1, most // 5), most), (max(1, new // 2), new), block, kv_heads * group, kv_heads, dim,
                      rng.choice(["f32", "f32", "f16", "bf16"]), stored, cap, window, rng.random() < 0.25, rng.choice(["slots", "heads"]))


# ---- what follows from a case alone ----------------------------------------------------------------------------------

def _between(count, least, most, turn):
    """`count` whole numbers spread over [least, most] in an order that looks like none."""
    at = (np.arange(1, count + 1) * turn) % 1.0
    return np.minimum(most, least + np.floor(at * (most - least + 1)).astype(np.int64))


def _lengths(case):
    """Cached and new tokens of every request."""
    context = _between(case["requests"], case["context_least"], case["context_most"], 0.6180339887498949)
    return context, _between(case["requests"], case["new_least"], case["new_most"], 0.7548776662466927)


def _blocks(tokens, block):
    return -(-tokens // block)


def _sets(case):
    """The filters of every row: some of "k", "p" and "m"."""
    sets = ["", "k", "p", "m", "kp", "pm", "km", "kpm"] if case["filters"] == "all" else [case["filters"].replace("none", "")]
    return [sets[(3 * r + 5) % len(sets)] for r in range(case["rows"])]


def work(case):
    kind = case["kind"]
    if kind == "sample":
        values = case["rows"] * case["vocab"]
        return {"bytes": values * SIZES[case["source"]] + 28 * case["rows"], "flops": 20 * values}
    heads, dim = case["kv_heads"], case["dim"]
    if kind == "rotate":
        size, out = SIZES[case["source"]], SIZES[case["out"]]
        tokens, q, k = case["tokens"], case["heads"] * dim, heads * dim
        moved = tokens * (q * (size + out) + k * size + 4 * case["axes"]) + 2 * case["rotary"] + 8 * dim * case["norm"]
        if case["store"] == "none":
            moved += tokens * k * out
        else:  # the keys, and the values from one to the other
            moved += tokens * (k * (size + 2 * SIZES[case["store"]]) + 8 * heads * (case["store"] == "e4m3") + 4)
        return {"bytes": moved, "flops": tokens * (q + k) * (4 * case["norm"] + 3)}
    if kind == "cache":
        row = 2 * heads * dim
        moved = case["tokens"] * (row * (SIZES[case["source"]] + 1) + 8 * heads + 4)
        moved += case["read"] * (row * (SIZES[case["out"]] + 1) + 8 * heads + 4)
        return {"bytes": moved, "flops": 3 * case["tokens"] * row + case["read"] * row}
    context, new = _lengths(case)
    # keys that any of a request's new tokens sees, and pairs of a token and a key that it sees
    first = np.maximum(0, context - case["window"] + 1) if case["window"] else np.zeros_like(context)
    keys = context + new - first
    pairs = sum(sum(min(c + t + 1, case["window"] or c + t + 1) for t in range(n)) for c, n in zip(context.tolist(), new.tolist()))
    tokens = int(new.sum())
    moved = int(keys.sum()) * heads * (2 * dim + 8) + 2 * tokens * case["heads"] * dim * SIZES[case["activations"]]
    moved += 4 * int(_blocks(keys, case["block"]).sum()) + 8 * case["requests"] + 4 * case["heads"] * case["bias"]
    return {"bytes": moved, "flops": 4 * pairs * case["heads"] * dim}


# ---- inputs ----------------------------------------------------------------------------------------------------------

class _Source:
    def __init__(self, seed):
        self.gen = torch.Generator(device=DEVICE)
        self.gen.manual_seed(seed)
        self.rng = np.random.default_rng(seed)

    def normal(self, *shape):
        return torch.randn(*shape, generator=self.gen, device=DEVICE)

    def uniform(self, *shape):
        return torch.rand(*shape, generator=self.gen, device=DEVICE)

    def shuffled(self, count):
        return torch.randperm(count, generator=self.gen, device=DEVICE).to(torch.int32)

    def heads(self, tokens, heads, dim, dtype):
        """What comes out of a projection: normal values, some channels several times larger, tokens of different size."""
        x = self.normal(tokens, heads, dim) * torch.where(self.uniform(heads, dim) < 0.03, 6.0, 1.0)
        return (x * (0.5 + self.uniform(tokens, 1, 1))).to(dtype)

    def cache(self, blocks, block, kv_heads, dim, stored, paged="slots"):
        """Codes and scales of a cache that holds tokens already."""
        outer = (blocks, block, kv_heads) if paged == "slots" else (blocks, kv_heads, block)
        made = []
        for _ in "kv":
            if stored == "e4m3":
                codes = torch.empty(*outer, dim, device=DEVICE).normal_(generator=self.gen).mul_(150.0).clamp_(-448.0, 448.0)
            else:
                codes = torch.empty(*outer, dim, device=DEVICE).normal_(generator=self.gen).mul_(45.0).round_().clamp_(-127.0, 127.0)
            made.append(codes.to(TYPES[stored]))
        ones = 150.0 if stored == "e4m3" else 45.0
        scales = [(0.5 + self.uniform(*outer)) / ones for _ in "kv"]
        return {"keys": made[0], "values": made[1], "key_scales": scales[0], "value_scales": scales[1]}


def _int32(values):
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).to(DEVICE)


def prepare(case, seed):
    src = _Source(seed)
    return dict({"rotate": _prepare_rotate, "cache": _prepare_cache, "attention": _prepare_attention, "sample": _prepare_sample}[case["kind"]](case, src),
                case=case)


def _prepare_rotate(case, src):
    tokens, heads, kv_heads, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
    pairs = case["rotary"] // 2
    # one projection's output holds a token's queries, keys and values side by side
    qkv = src.heads(tokens, heads + 2 * kv_heads, dim, TYPES[case["source"]])
    state = {"q": qkv[:, :heads], "k": qkv[:, heads:heads + kv_heads], "v": qkv[:, heads + kv_heads:]}
    state["positions"] = torch.randint(0, case["reach"], (case["axes"], tokens), generator=src.gen, device=DEVICE).to(torch.int32)
    state["frequencies"] = (500000.0 ** (-torch.arange(pairs, dtype=torch.float64) / pairs)).float().to(DEVICE)
    # the first pairs turn with time, the others in turn with height and width
    axis = [0 if case["axes"] == 1 or p < pairs // 3 else 1 + p % (case["axes"] - 1) for p in range(pairs)]
    state["pair_axes"] = axis if case["axes"] > 1 else None
    state["q_weight"], state["k_weight"] = ((1.0 + 0.2 * src.normal(dim)) if case["norm"] else None for _ in "qk")
    state["q_out"] = torch.empty(tokens, heads, dim, dtype=TYPES[case["out"]], device=DEVICE)
    if case["store"] == "none":
        state["k_out"] = torch.empty(tokens, kv_heads, dim, dtype=TYPES[case["out"]], device=DEVICE)
        return state
    block = 16
    blocks = _blocks(tokens, block) + 5
    if case["store"] == "e4m3":
        state["cache"] = src.cache(blocks, block, kv_heads, dim, "e4m3")
    else:
        state["cache"] = {n: src.normal(blocks, block, kv_heads, dim).to(TYPES[case["store"]]) for n in ("keys", "values")}
    state["slots"] = src.shuffled(blocks * block)[:tokens].contiguous()
    return state


def _prepare_cache(case, src):
    tokens, kv_heads, dim, block = case["tokens"], case["kv_heads"], case["dim"], case["block"]
    held = max(tokens, case["read"])
    blocks = _blocks(held, block) + 3
    state = {"cache": src.cache(blocks, block, kv_heads, dim, case["stored"])}
    at = np.arange(held)
    slots = src.shuffled(blocks).cpu().numpy().astype(np.int64)[at // block] * block + at % block
    state["slots"] = _int32(slots[held - tokens:])  # the new tokens are a request's last
    state["new"] = [src.heads(tokens, kv_heads, dim, TYPES[case["source"]]) for _ in "kv"]
    state["read"] = _int32(slots[held - case["read"]:])
    state["out"] = [torch.empty(case["read"], kv_heads, dim, dtype=TYPES[case["out"]], device=DEVICE) for _ in "kv"]
    return state


def _prepare_attention(case, src):
    context, new = _lengths(case)
    block, kv_heads, heads, dim = case["block"], case["kv_heads"], case["heads"], case["dim"]
    held = _blocks(context + new, block)
    columns, total = int(held.max()) + 1, int(held.sum())
    blocks = src.shuffled(total + 9).cpu().numpy()
    table = np.full((case["requests"], columns), -1, np.int32)
    table[np.arange(columns)[None, :] < held[:, None]] = blocks[:total]
    tokens = int(new.sum())
    state = {"cache": src.cache(total + 9, block, kv_heads, dim, case["stored"], case["paged"]), "table": _int32(table),
             "context": _int32(context), "starts": _int32(np.concatenate([[0], np.cumsum(new)]))}
    # scores of a few units: some rows look at a handful of keys, others at many
    state["q"] = (src.normal(tokens, heads, dim) * (0.5 + 2.0 * src.uniform(tokens, heads, 1))).to(TYPES[case["activations"]])
    state["out"] = torch.empty_like(state["q"])
    # a head's bias reaches from some ten keys to some thousand
    state["slopes"] = torch.exp2(-2.0 - 8.0 * torch.arange(heads, device=DEVICE) / heads) if case["bias"] else None
    state["longest"] = {"keys": int((context + new).max()), "new": int(new.max())}
    return state


def _prepare_sample(case, src):
    rows, vocab = case["rows"], case["vocab"]
    logits = src.normal(rows, vocab) * case["spread"]
    # a few words stand out, as they do in a text; some are forbidden
    logits += torch.where(src.uniform(rows, vocab) < 20.0 / vocab, 4.0 * src.uniform(rows, vocab) * case["spread"], 0.0)
    logits = logits.masked_fill(src.uniform(rows, vocab) < 0.001, -math.inf)
    sets = _sets(case)
    has = {f: np.array([f in s for s in sets]) for f in "kpm"}
    k = np.where(has["k"], np.exp(src.rng.uniform(math.log(2), math.log(min(2000, vocab)), rows)).astype(np.int64), 0)
    p = np.where(has["p"], src.rng.uniform(0.5, 0.99, rows), 1.0).astype(np.float32)
    m = np.where(has["m"], np.exp(src.rng.uniform(math.log(0.005), math.log(0.2), rows)), 0.0).astype(np.float32)
    t = np.where(src.rng.random(rows) < 0.1, 0.0, src.rng.uniform(0.3, 1.5, rows)).astype(np.float32)  # zero: the largest
    if rows == 1:
        t[0] = 0.8
    return {"logits": logits.to(TYPES[case["source"]]), "k": _int32(k), "p": torch.from_numpy(p).to(DEVICE), "m": torch.from_numpy(m).to(DEVICE),
            "t": torch.from_numpy(t).to(DEVICE), "u": src.uniform(rows), "token": torch.empty(rows, dtype=torch.int32, device=DEVICE),
            "probability": torch.empty(rows, device=DEVICE)}


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"rotate": _own_rotate, "cache": _own_cache, "attention": _own_attention, "sample": _own_sample}[kind](state)
    return {"rotate": _plain_rotate, "cache": _plain_cache, "attention": _plain_attention, "sample": _plain_sample}[kind](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


_scratch = {}


def _workspace(count):
    """The scratch that a program lends to every call, as large as the largest has asked for."""
    held = _scratch.get("bytes")
    if held is None or held.numel() < count:
        held = _scratch["bytes"] = torch.empty(max(count, 1 << 20), dtype=torch.uint8, device=DEVICE)
    return held


def _own_quantized(held, paged_as="slots"):
    from antfly_amd import paged
    return paged.quantizedCache(held["keys"], held["values"], held["key_scales"], held["value_scales"], heads_outside=paged_as == "heads")


def _own_rotate(state):
    from antfly_amd import paged
    case = state["case"]
    rotation = paged.headRotation(state["q"], state["k"], state["q_out"], state.get("k_out"), state["positions"], state["frequencies"],
                                  query_weight=state["q_weight"], key_weight=state["k_weight"], interleaved=case["interleaved"],
                                  pair_axes=state["pair_axes"])
    if case["store"] == "none":
        paged.launchHeadRotation(_stream(), rotation)
        return [state["q_out"], state["k_out"]]
    cache = _own_quantized(state["cache"]) if case["store"] == "e4m3" else paged.cache(state["cache"]["keys"], state["cache"]["values"])
    paged.launchRotatedStore(_stream(), rotation, cache, state["v"], state["slots"])
    return [state["q_out"], state["cache"]]


def _own_cache(state):
    from antfly_amd import paged
    cache = _own_quantized(state["cache"])
    paged.launchQuantizedStore(_stream(), cache, state["new"][0], state["new"][1], state["slots"])
    paged.launchQuantizedLoad(_stream(), cache, state["out"][0], state["out"][1], state["read"])
    return state["out"]


def _own_attention(state):
    from antfly_amd import paged
    case = state["case"]
    call = paged.quantizedAttention(_own_quantized(state["cache"], case["paged"]), state["out"], state["q"], state["starts"], state["context"],
                                    state["table"], state["longest"]["new"], state["longest"]["keys"], softcap=case["cap"],
                                    window=case["window"], slopes=state["slopes"])
    paged.launchQuantizedAttention(_stream(), call, _workspace(paged.quantizedAttentionWorkspaceBytes(call)))
    return state["out"]


def _own_sample(state):
    from antfly_amd import sampling
    call = sampling.sample(state["logits"], state["token"], state["u"], temperatures=state["t"], top_k=state["k"], top_p=state["p"],
                           min_p=state["m"], probabilities=state["probability"])
    sampling.launchSample(_stream(), call, _workspace(sampling.sampleWorkspaceBytes(call)))
    return [state["token"], state["probability"]]


# ---- the plain forms -------------------------------------------------------------------------------------------------

def _normed(x, weight):
    x = x.float()
    return x if weight is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight


def _turned(x, state):
    """The first `rotary` dimensions of [tokens, heads, dim] by their tokens' angles: position times frequency, in 64 bits."""
    case, pairs = state["case"], state["case"]["rotary"] // 2
    axis = torch.zeros(pairs, dtype=torch.long, device=DEVICE) if state["pair_axes"] is None else torch.tensor(state["pair_axes"], device=DEVICE)
    angle = state["positions"].double()[axis].t() * state["frequencies"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    turning, rest = x[..., :2 * pairs], x[..., 2 * pairs:]
    if case["interleaved"]:
        a, b = turning[..., 0::2], turning[..., 1::2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = turning[..., :pairs], turning[..., pairs:]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, rest), -1)


def _quantized(x, stored):
    """Codes and f32 scales of [tokens, heads, dim]: scale = max |x| / largest, code = x (largest / max), to nearest."""
    most = x.abs().amax(-1).clamp_min(TINY)
    largest = torch.full_like(most, LARGEST[stored])
    scaled = x * (largest / most)[..., None]
    return (scaled if stored == "e4m3" else torch.round(scaled)).to(TYPES[stored]), most / largest


def _put(cache, keys, values, slots, stored):
    slots = slots.long()
    for name, x in (("keys", keys), ("values", values)):
        rows = cache[name].view(-1, *cache[name].shape[2:])
        if stored not in LARGEST:
            rows[slots] = x.to(rows.dtype)
            continue
        codes, scales = _quantized(x, stored)
        rows.view(torch.uint8)[slots] = codes.view(torch.uint8)
        cache[name[:-1] + "_scales"].view(-1, x.shape[1])[slots] = scales


def _plain_rotate(state):
    case = state["case"]
    q, k = _turned(_normed(state["q"], state["q_weight"]), state), _turned(_normed(state["k"], state["k_weight"]), state)
    if case["store"] == "none":
        return [q.to(TYPES[case["out"]]), k.to(TYPES[case["out"]])]
    _put(state["cache"], k, state["v"].float(), state["slots"], case["store"])
    return [q.to(TYPES[case["out"]]), state["cache"]]


def _plain_cache(state):
    case, cache = state["case"], state["cache"]
    _put(cache, state["new"][0].float(), state["new"][1].float(), state["slots"], case["stored"])
    slots, out = state["read"].long(), []
    for name in ("keys", "values"):
        codes = cache[name].view(torch.uint8).view(-1, *cache[name].shape[2:])[slots].view(cache[name].dtype)
        out.append((codes.float() * cache[name[:-1] + "_scales"].view(-1, case["kv_heads"])[slots][..., None]).to(TYPES[case["out"]]))
    return out


def _plain_attention(state):
    case, block = state["case"], state["case"]["block"]
    requests, heads, kv_heads, dim = case["requests"], case["heads"], case["kv_heads"], case["dim"]
    keys, new, group = state["longest"]["keys"], state["longest"]["new"], heads // kv_heads
    context, starts = state["context"].long(), state["starts"].long()
    count = starts[1:] - starts[:-1]
    tokens = state["q"].shape[0]
    at, t = torch.arange(keys, device=DEVICE), torch.arange(new, device=DEVICE)
    token = (starts[:-1, None] + t).clamp_max(tokens - 1)
    distance = (context[:, None] + t)[:, :, None] - at  # [requests, new, keys]
    seen = distance >= 0
    if case["window"]:
        seen = seen & (distance < case["window"])
    held = at < (context + count)[:, None]
    page = state["table"].long()[:, at // block].clamp_min(0)

    def values(name):
        codes, scales = state["cache"][name].view(torch.uint8), state["cache"][name[:-1] + "_scales"]
        if case["paged"] == "heads":
            codes, scales = codes.transpose(1, 2), scales.transpose(1, 2)
        x = codes[page, at % block].view(state["cache"][name].dtype).float() * scales[page, at % block][..., None]
        # [requests, kv heads, keys, dim], nothing of what lies past a request's keys
        return torch.where(held[:, :, None, None], x, 0.0).transpose(1, 2).contiguous()

    q = state["q"].float()[token].view(requests, new, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(requests, kv_heads, -1, dim)
    scores = (q @ values("keys").transpose(2, 3).contiguous()).view(requests, kv_heads, new, group, keys) * dim ** -0.5
    if case["cap"]:
        scores = case["cap"] * torch.tanh(scores / case["cap"])
    if case["bias"]:
        scores = scores - state["slopes"].view(1, kv_heads, 1, group, 1) * distance[:, None, :, None, :]
    scores = scores.masked_fill(~seen[:, None, :, None, :], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-3e38))
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(requests, kv_heads, new * group, keys) @ values("values")).view(requests, kv_heads, new, group, dim)
    out = torch.where(total > 0, out / total, 0.0).permute(0, 2, 1, 3, 4).reshape(requests, new, heads, dim)
    request = torch.searchsorted(starts[1:], torch.arange(tokens, device=DEVICE), right=True)
    return out[request, torch.arange(tokens, device=DEVICE) - starts[request]].to(state["q"].dtype)


def _plain_sample(state):
    logits, vocab = state["logits"].float(), state["case"]["vocab"]
    values, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    greedy = (state["t"] <= 0)[:, None]
    # which token it is hangs on sums next to a border: 64 bits
    weights = torch.exp((values.double() - values[:, :1].double()) / torch.where(greedy, 1.0, state["t"][:, None]).double())
    rank = torch.arange(vocab, device=DEVICE)
    most = torch.where((state["k"] <= 0) | greedy[:, 0], vocab, state["k"])[:, None]
    weights = torch.where(rank < torch.where(greedy, 1, most), weights, 0.0)
    before = torch.cumsum(weights, -1) - weights
    total = weights.sum(-1, keepdim=True)
    kept = (before < state["p"].double()[:, None] * total) | (state["p"] >= 1.0)[:, None]
    kept = kept & (weights >= state["m"].double()[:, None]) | (rank == 0)
    weights = torch.where(kept, weights, 0.0)
    sums = torch.cumsum(weights, -1)
    total = sums[:, -1:].contiguous()
    place = torch.searchsorted(sums, state["u"].double()[:, None] * total, right=True).clamp_max(vocab - 1)
    return [order.gather(1, place)[:, 0].int(), (weights.gather(1, place) / total)[:, 0].float()]


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    return {"rotate": _exact_rotate, "cache": _exact_cache, "attention": _exact_attention, "sample": _exact_sample}[case["kind"]](state)


def _rotated_heads(x, weight, state):
    case, pairs = state["case"], state["case"]["rotary"] // 2
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / case["dim"] + 1e-6) * weight.double()
    y = x.clone()
    for p in range(pairs):
        position = state["positions"][state["pair_axes"][p] if state["pair_axes"] else 0].double()
        angle = position * float(state["frequencies"][p])
        turn = torch.polar(torch.ones_like(angle), angle)
        a, b = (2 * p, 2 * p + 1) if case["interleaved"] else (p, p + pairs)
        z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn[:, None]
        y[..., a], y[..., b] = z.real, z.imag
    return y


def _eight_bits(x, stored):
    """The nearest codes, as numbers, and the scales, from 64 bits."""
    scale = x.abs().amax(-1, keepdim=True).clamp_min(TINY) / LARGEST[stored]
    y = x / scale
    if stored == "i8":
        return torch.round(y), scale[..., 0]
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0) - 3.0)
    return torch.round(y / step) * step, scale[..., 0]


def _exact_rotate(state):
    case = state["case"]
    q, k = _rotated_heads(state["q"], state["q_weight"], state), _rotated_heads(state["k"], state["k_weight"], state)
    if case["store"] == "none":
        return [q, k]
    cache, where = {}, state["slots"].long()
    for name, x in (("keys", k), ("values", state["v"].double())):
        codes = state["cache"][name].double()
        rows = codes.view(-1, *codes.shape[2:])
        if case["store"] != "e4m3":
            rows[where] = x
        else:
            scales = state["cache"][name[:-1] + "_scales"].double()
            rows[where], scales.view(-1, case["kv_heads"])[where] = _eight_bits(x, "e4m3")
            cache[name[:-1] + "_scales"] = scales
        cache[name] = codes
    return [q, cache]


def _exact_cache(state):
    case, made = state["case"], []
    for name, new in zip(("keys", "values"), state["new"]):
        codes, scales = state["cache"][name].double(), state["cache"][name[:-1] + "_scales"].double()
        rows, row_scales, where = codes.view(-1, *codes.shape[2:]), scales.view(-1, case["kv_heads"]), state["slots"].long()
        # codes are rounded from f32 products, and the scale is an f32: both are part of the definition
        x = new.float()
        most = x.abs().amax(-1).clamp_min(TINY)
        ratio = (LARGEST[case["stored"]] / most.double()).float()
        product = (x * ratio[..., None]).double()
        if case["stored"] == "i8":
            rows[where] = torch.round(product)
        else:
            step = torch.exp2(torch.floor(torch.log2(product.abs().clamp_min(2.0 ** -20))).clamp_min(-6.0) - 3.0)
            rows[where] = (torch.round(product / step) * step).clamp(-448.0, 448.0)
        row_scales[where] = (most.double() / LARGEST[case["stored"]]).float().double()
        read = state["read"].long()
        made.append(rows[read] * row_scales[read][..., None])
    return made


def _exact_attention(state):
    case, block = state["case"], state["case"]["block"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    starts, context, table = (state[name].cpu().numpy() for name in ("starts", "context", "table"))
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    for r in range(case["requests"]):
        first, last, cached = int(starts[r]), int(starts[r + 1]), int(context[r])
        total = cached + last - first
        pages = torch.from_numpy(table[r, :_blocks(total, block)]).to(DEVICE).long()
        lined = []
        for name in ("keys", "values"):
            codes, scales = state["cache"][name].view(torch.uint8)[pages].view(state["cache"][name].dtype).double(), state["cache"][name[:-1] + "_scales"][pages].double()
            if case["paged"] == "heads":
                codes, scales = codes.transpose(1, 2), scales.transpose(1, 2)
            lined.append((codes * scales[..., None]).flatten(0, 1)[:total])
        for t in range(last - first):
            position = cached + t
            low = max(0, position - case["window"] + 1) if case["window"] else 0
            k, v = (x[low:position + 1] for x in lined)
            for g in range(kv_heads):
                own_heads = slice(g * (heads // kv_heads), (g + 1) * (heads // kv_heads))
                scores = state["q"][first + t, own_heads].double() @ k[:, g].t().contiguous() / math.sqrt(dim)
                if case["cap"]:
                    scores = case["cap"] * torch.tanh(scores / case["cap"])
                if case["bias"]:
                    far = position - torch.arange(low, position + 1, device=DEVICE)
                    scores = scores - state["slopes"][own_heads, None].double() * far
                out[first + t, own_heads] = torch.softmax(scores, -1) @ v[:, g].contiguous()
    return out


def _exact_sample(state):
    """The probabilities; the tokens are whole numbers."""
    rows, made = state["case"]["rows"], []
    k, p, m, t, u = (state[name].cpu().numpy() for name in ("k", "p", "m", "t", "u"))
    for r in range(rows):
        logits = state["logits"][r].cpu().double().numpy()
        if t[r] <= 0:
            made.append(1.0)
            continue
        order = np.lexsort((np.arange(len(logits)), -logits))
        weights = np.exp((logits[order] - logits[order[0]]) / np.float64(t[r]))
        if k[r] > 0:
            order, weights = order[:k[r]], weights[:k[r]]
        count = len(order)
        if p[r] < 1:
            sums = np.cumsum(weights)
            count = 1 + int(np.sum(sums[:-1] < np.float64(p[r]) * sums[-1]))
        count = max(1, min(count, int(np.sum(weights >= np.float64(m[r])))))
        sums = np.cumsum(weights[:count])
        made.append(weights[min(count - 1, np.searchsorted(sums, np.float64(u[r]) * sums[-1], side="right"))] / sums[-1])
    return [None, torch.tensor(made, dtype=torch.float64)]
