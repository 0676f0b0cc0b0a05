"""A paged key / value cache and what a speculative decode step does with it: plan the batch, store the drafted tokens' keys
and values, attend over context and draft tree, move the accepted path behind the context.  And the same cache in 8 bits: heads of
a projection normed, rotated and stored, stored as they are, read back, attended.

The functions take device arrays: anything with torch's `data_ptr()`, `shape`, `stride()`, `dtype`, `numel()` and
`element_size()` (this package does not import torch).  Layouts, and what each launch reads and writes, are those of the C
ABI (include/antfly_hip_qmatmul.h); `stream` is a hipStream_t."""
from __future__ import annotations

import ctypes as C
import struct

from . import _lib
from ._lib import Buffer, check

NO_BUFFER = Buffer(0, 0)
_TYPES = {"torch.float32": _lib.TYPE_F32, "torch.float16": _lib.TYPE_F16, "torch.bfloat16": _lib.TYPE_BF16}
# A decode step makes these calls for every layer: arguments go into the C structs as one packed string of numbers, which
# takes a fifth of the time that filling their fields does.
_CACHE, _PLAN, _REST = struct.Struct("4Qi4x7Q"), struct.Struct("26Q"), struct.Struct("if23Q")  # _REST: TreeAttention behind its cache
_CODES, _ROTATION, _QUANTIZED_REST = struct.Struct("8Qi4x10Q"), struct.Struct("3if30Q128s"), struct.Struct("i2f4x23Q")
assert _CACHE.size == C.sizeof(_lib.PagedCache) and _PLAN.size == C.sizeof(_lib.BatchPlan)
assert _CACHE.size + _REST.size == C.sizeof(_lib.TreeAttention)
assert _CODES.size == C.sizeof(_lib.QuantizedCache) and _ROTATION.size == C.sizeof(_lib.HeadRotation)
assert _CODES.size + _QUANTIZED_REST.size == C.sizeof(_lib.QuantizedAttention)
_CODE_TYPES = {"torch.int8": _lib.TYPE_I8, "torch.float8_e4m3fn": _lib.TYPE_E4M3}


def _bad_shape():
    return _lib.InvalidShape(_lib.ERR_INVALID_SHAPE)


def _bad_number():
    """Of a number below zero, or none that is whole: what the C ABI answers to one that is too large."""
    return _lib.InvalidHipState(_lib.ERR_INVALID_STATE)


_names = {}  # of the types that have been seen


def _name(dtype) -> str:
    name = _names.get(dtype)
    if name is None:
        name = _names[dtype] = str(dtype)
    return name


def buffer(array) -> Buffer:
    """The memory that an array spans, from its first element to its last; None: no buffer."""
    if array is None:
        return NO_BUFFER
    return Buffer(array.data_ptr(), array.nbytes if array.is_contiguous() else _bytes(array))


def _bytes(array) -> int:
    if array.is_contiguous():
        return array.nbytes
    return (1 + sum((n - 1) * s for n, s in zip(array.shape, array.stride()))) * array.element_size() if array.numel() else 0


def _type(array) -> int:
    return _TYPES.get(_name(array.dtype), -1)


def _i32(array):
    """(address, bytes) of a contiguous array of int32."""
    if _name(array.dtype) != "torch.int32" or not array.is_contiguous():
        raise _bad_shape()
    return array.data_ptr(), array.nbytes


def _i32_buffer(array) -> Buffer:
    if _name(array.dtype) != "torch.int32" or not array.is_contiguous():
        raise _bad_shape()
    return Buffer(array.data_ptr(), array.nbytes)


def _optional(array, dtypes=("torch.int32",)):
    if array is None:
        return 0, 0
    if _name(array.dtype) not in dtypes or not array.is_contiguous():
        raise _bad_shape()
    return array.data_ptr(), array.nbytes


_U64 = ("torch.int64", "torch.uint64")


def _rows_of_heads(array, rows, heads, dim):
    """(token stride, head stride) of [rows, heads, dim] whose last dimension is contiguous."""
    strides = array.stride()
    if array.shape != (rows, heads, dim) or (dim > 1 and strides[2] != 1):
        raise _bad_shape()
    return strides[0], strides[1]


def _same_strides(a, b) -> bool:
    """Of arrays of one shape: those of dimensions of one element say nothing."""
    mine, theirs = a.stride(), b.stride()
    return mine == theirs or all(n <= 1 or s == t for n, s, t in zip(a.shape, mine, theirs))


def cache(keys, values, heads_outside: bool = False) -> _lib.PagedCache:
    """keys, values [blocks, block size, kv heads, head dim], or with heads_outside [blocks, kv heads, block size, head dim]."""
    shape, strides = keys.shape, keys.stride()
    if len(shape) != 4 or values.shape != shape or keys.dtype != values.dtype or not _same_strides(keys, values) or \
            (shape[3] > 1 and strides[3] != 1):
        raise _bad_shape()
    slot, head = (2, 1) if heads_outside else (1, 2)
    made = _lib.PagedCache.from_buffer_copy(_CACHE.pack(
        keys.data_ptr(), _bytes(keys), values.data_ptr(), _bytes(values), _type(keys), shape[0], shape[slot], shape[head],
        shape[3], strides[0], strides[slot], strides[head]))
    made.arrays = (keys, values)  # alive as long as the description of them is
    return made


def launchBatchPlan(stream, context_lens, query_lens, block_tables, free_blocks, block_size: int, query_starts, slots, positions,
                    blocks_taken, parents=None, masks=None, blocks: int = (1 << 31) - 1) -> None:
    """Writes block_tables (new entries), query_starts, slots, positions, masks and blocks_taken from the requests' lengths;
    `blocks`: how many the cache has (numbers outside name none)."""
    requests, columns = block_tables.shape
    tokens, words = slots.shape[0], 0
    if masks is not None:
        if len(masks.shape) != 2 or masks.shape[0] != tokens:
            raise _bad_shape()
        words = masks.shape[1]
    if positions.shape[0] != tokens or (parents is not None and parents.shape[0] != tokens):
        raise _bad_shape()
    try:
        plan = _lib.BatchPlan.from_buffer_copy(_PLAN.pack(
            requests, columns, block_size, blocks, tokens, words, *_i32(context_lens), *_i32(query_lens), *_i32(free_blocks),
            *_optional(parents), *_i32(block_tables), *_i32(query_starts), *_i32(slots), *_i32(positions), *_optional(masks, _U64),
            *_i32(blocks_taken)))
    except struct.error:
        raise _bad_number() from None
    check(_lib.lib().afhip_launch_batch_plan(stream, plan))


def launchCacheStore(stream, cache: _lib.PagedCache, keys, values, slots) -> None:
    """keys, values [tokens, kv heads, head dim] (f32, f16 or bf16) into the cache's slots."""
    shape, strides, dtype = keys.shape, keys.stride(), keys.dtype
    if values.shape != shape or values.dtype != dtype or (values.stride() != strides and not _same_strides(keys, values)) or \
            shape != (slots.shape[0], cache.kv_heads, cache.head_dim) or (shape[2] > 1 and strides[2] != 1):
        raise _bad_shape()
    check(_lib.lib().afhip_launch_cache_store(stream, cache, _TYPES.get(_name(dtype), -1), buffer(keys), buffer(values), strides[0],
                                              strides[1], _i32_buffer(slots), shape[0]))


def launchCacheMove(stream, cache: _lib.PagedCache, block_tables, context_lens, paths, path_lens) -> None:
    """The accepted path of every request's tree to the places behind its context."""
    requests, columns = block_tables.shape
    shape = paths.shape
    if len(shape) != 2 or shape[0] != requests:
        raise _bad_shape()
    check(_lib.lib().afhip_launch_cache_move(stream, cache, _i32_buffer(block_tables), columns, _i32_buffer(context_lens),
                                             _i32_buffer(paths), _i32_buffer(path_lens), requests, shape[1]))


def treeAttention(cache: _lib.PagedCache, out, query, query_starts, context_lens, block_tables, max_query_len: int,
                  max_key_len: int, masks=None, scale: float = None) -> _lib.TreeAttention:
    """The arguments of a call (of any number of calls while the arrays stay): query, out [tokens, heads, head dim]; scale:
    head_dim ** -0.5 unless given."""
    tokens, heads, dim = query.shape
    requests, columns = block_tables.shape
    q_token, q_head = _rows_of_heads(query, tokens, heads, cache.head_dim)
    o_token, o_head = _rows_of_heads(out, tokens, heads, cache.head_dim)
    words = 0
    if masks is not None:
        if len(masks.shape) != 2 or masks.shape[0] != tokens or masks.shape[1] == 0:  # (no words have no address, as no masks have)
            raise _bad_shape()
        words = masks.shape[1]
    if out.dtype != query.dtype:
        raise _bad_shape()
    try:
        made = _lib.TreeAttention.from_buffer_copy(bytes(cache) + _REST.pack(
            _type(query), dim ** -0.5 if scale is None else scale, requests, tokens, heads, max_query_len, max_key_len, columns, words,
            q_token, q_head, o_token, o_head, query.data_ptr(), _bytes(query), out.data_ptr(), _bytes(out), *_i32(query_starts),
            *_i32(context_lens), *_i32(block_tables), *_optional(masks, _U64)))
    except struct.error:
        raise _bad_number() from None
    made.arrays = (cache, out, query, query_starts, context_lens, block_tables, masks)
    return made


def treeAttentionWorkspaceBytes(attention: _lib.TreeAttention) -> int:
    return _lib.lib().afhip_tree_attention_workspace_bytes(attention)


def launchTreeAttention(stream, attention: _lib.TreeAttention, workspace: Buffer = NO_BUFFER) -> None:
    """`workspace`: a Buffer, or an array, of at least treeAttentionWorkspaceBytes(attention) bytes."""
    check(_lib.lib().afhip_launch_tree_attention(stream, attention,
                                                 workspace if isinstance(workspace, Buffer) else buffer(workspace)))


# ---- 8-bit caches -----------------------------------------------------------------------------------------------------

_kinds = {}  # of the types that have been seen: (type, bytes of an element)
_SIZES = {_lib.TYPE_F32: 4, _lib.TYPE_F16: 2, _lib.TYPE_BF16: 2, _lib.TYPE_I8: 1, _lib.TYPE_E4M3: 1, -1: 1}
_I32, _F32 = ("torch.int32", 4), ("torch.float32", 4)


def _kind(dtype):
    kind = _kinds.get(dtype)
    if kind is None:
        name = str(dtype)
        type = _TYPES.get(name, _CODE_TYPES.get(name, -1))
        kind = _kinds[dtype] = type, _SIZES[type]
    return kind


def _heads_of(array, size, rows, heads, dim):
    """(token stride, head stride, address, bytes) of [rows, heads, dim] whose last dimension is contiguous."""
    strides = array.stride()
    if array.shape != (rows, heads, dim) or (dim > 1 and strides[2] != 1):
        raise _bad_shape()
    token, head = strides[0], strides[1]
    return token, head, array.data_ptr(), ((rows - 1) * token + (heads - 1) * head + dim) * size if rows and heads else 0


def _line(array, dtype, count):
    """(address, bytes) of a contiguous array [count] of numbers of `dtype`, (name, bytes); None: none."""
    if array is None:
        return 0, 0
    if _name(array.dtype) != dtype[0] or array.shape != (count,) or not array.is_contiguous():
        raise _bad_shape()
    return array.data_ptr(), count * dtype[1]


def quantizedCache(keys, values, key_scales, value_scales, heads_outside: bool = False) -> _lib.QuantizedCache:
    """keys, values int8 or float8_e4m3fn [blocks, block size, kv heads, head dim] and their scales f32 [blocks, block size, kv
    heads]; with heads_outside [blocks, kv heads, block size(, head dim)]."""
    shape, strides, scale_strides, dtype = keys.shape, keys.stride(), key_scales.stride(), keys.dtype
    if len(shape) != 4 or values.shape != shape or values.dtype != dtype or (values.stride() != strides and not _same_strides(keys, values)) or \
            (shape[3] > 1 and strides[3] != 1) or key_scales.shape != shape[:3] or value_scales.shape != shape[:3] or \
            (value_scales.stride() != scale_strides and not _same_strides(key_scales, value_scales)) or \
            _name(key_scales.dtype) != "torch.float32" or _name(value_scales.dtype) != "torch.float32":
        raise _bad_shape()
    blocks, n1, n2, dim = shape
    s0, s1, s2, _ = strides
    t0, t1, t2 = scale_strides
    held = blocks and n1 and n2 and dim
    codes = (blocks - 1) * s0 + (n1 - 1) * s1 + (n2 - 1) * s2 + dim if held else 0
    scales = ((blocks - 1) * t0 + (n1 - 1) * t1 + (n2 - 1) * t2 + 1) * 4 if held else 0
    if heads_outside:
        n1, n2, s1, s2, t1, t2 = n2, n1, s2, s1, t2, t1
    type = _kind(dtype)[0]
    made = _lib.QuantizedCache.from_buffer_copy(_CODES.pack(
        keys.data_ptr(), codes, values.data_ptr(), codes, key_scales.data_ptr(), scales, value_scales.data_ptr(), scales, type, blocks, n1,
        n2, dim, s0, s1, s2, t0, t1, t2))
    made.arrays = (keys, values, key_scales, value_scales)  # alive as long as the description of them is
    return made


def _token_rows(cache, keys, values, slots):
    """What a store or a load of tokens [tokens, kv heads, head dim] passes on behind the cache."""
    tokens, heads, dim = keys.shape
    dtype = keys.dtype
    type, size = _kind(dtype)
    token, head, key_at, held = _heads_of(keys, size, tokens, cache.kv_heads, cache.head_dim)
    if values.dtype != dtype or values.shape != (tokens, heads, dim) or (values.stride() != keys.stride() and not _same_strides(keys, values)):
        raise _bad_shape()
    return type, Buffer(key_at, held), Buffer(values.data_ptr(), held), token, head, Buffer(*_line(slots, _I32, tokens)), tokens


def launchQuantizedStore(stream, cache: _lib.QuantizedCache, keys, values, slots) -> None:
    """keys, values [tokens, kv heads, head dim] (f32, f16 or bf16) quantized into the cache's slots."""
    check(_lib.lib().afhip_launch_quantized_store(stream, cache, *_token_rows(cache, keys, values, slots)))


def launchQuantizedLoad(stream, cache: _lib.QuantizedCache, keys, values, slots) -> None:
    """The slots' keys and values read back into keys, values [tokens, kv heads, head dim] (f32, f16 or bf16)."""
    check(_lib.lib().afhip_launch_quantized_load(stream, cache, *_token_rows(cache, keys, values, slots)))


_ONE_AXIS = bytes(128)
_NO_HEADS = (0, 0, 0, 0)


def headRotation(query, key, out_query, out_key, positions, frequencies, query_weight=None, key_weight=None, epsilon: float = 1e-6,
                 interleaved: bool = False, pair_axes=None) -> _lib.HeadRotation:
    """The norm and rotation of query [tokens, heads, head dim] (or None) and key [tokens, kv heads, head dim] into out_query and
    out_key (None for launchRotatedStore), which may be query and key themselves.  positions int32 [tokens] or [axes, tokens],
    frequencies f32 [pairs]: twice as many dimensions turn.  pair_axes: the axis of every pair (all 0 unless given)."""
    tokens, kv_heads, dim = key.shape
    dtype = key.dtype
    type, size = _kind(dtype)
    k_token, k_head, k_at, k_held = _heads_of(key, size, tokens, kv_heads, dim)
    heads, out_type = 0, type
    q_token, q_head, q_at, q_held = o_token, o_head, o_at, o_held = ok_token, ok_head, ok_at, ok_held = _NO_HEADS
    if query is not None:
        heads, out_dtype = query.shape[1], out_query.dtype
        out_type, out_size = _kind(out_dtype)
        if query.dtype != dtype or (out_key is not None and out_key.dtype != out_dtype):
            raise _bad_shape()
        q_token, q_head, q_at, q_held = _heads_of(query, size, tokens, heads, dim)
        o_token, o_head, o_at, o_held = _heads_of(out_query, out_size, tokens, heads, dim)
    if out_key is not None:
        out_type, out_size = _kind(out_key.dtype)
        ok_token, ok_head, ok_at, ok_held = _heads_of(out_key, out_size, tokens, kv_heads, dim)
    pairs, place = frequencies.shape[0], positions.shape
    axes = place[0] if len(place) == 2 else 1
    if pairs > 128 or place[-1] != tokens or len(place) > 2 or _name(positions.dtype) != "torch.int32" or not positions.is_contiguous():
        raise _bad_shape()
    if pair_axes is None:
        packed = _ONE_AXIS
    else:
        try:
            packed = bytes(list(pair_axes))  # (bytes of a number alone would be that many zeros)
        except (TypeError, ValueError):
            raise _bad_number() from None
        if len(packed) != pairs:
            raise _bad_shape()
    f_at, f_held = _line(frequencies, _F32, pairs)
    w_at, w_held = _line(query_weight, _F32, dim)
    kw_at, kw_held = _line(key_weight, _F32, dim)
    try:
        made = _lib.HeadRotation.from_buffer_copy(_ROTATION.pack(
            type, out_type, 1 if interleaved else 0, epsilon, tokens, heads, kv_heads, dim, 2 * pairs, axes, q_token, q_head, k_token, k_head,
            o_token, o_head, ok_token, ok_head, q_at, q_held, k_at, k_held, o_at, o_held, ok_at, ok_held, positions.data_ptr(),
            axes * tokens * 4, f_at, f_held, w_at, w_held, kw_at, kw_held, packed))
    except struct.error:
        raise _bad_number() from None
    made.arrays = (query, key, out_query, out_key, positions, frequencies, query_weight, key_weight)
    return made


def launchHeadRotation(stream, rotation: _lib.HeadRotation) -> None:
    check(_lib.lib().afhip_launch_head_rotation(stream, rotation))


def launchRotatedStore(stream, rotation: _lib.HeadRotation, cache, values, slots) -> None:
    """The rotation's queries into out_query, its keys and `values` [tokens, kv heads, head dim] into the slots of `cache` (a
    PagedCache or a QuantizedCache)."""
    tokens = rotation.tokens
    type, size = _kind(values.dtype)
    token, head, at, held = _heads_of(values, size, tokens, rotation.kv_heads, rotation.head_dim)
    if type != rotation.type:
        raise _bad_shape()
    quantized = isinstance(cache, _lib.QuantizedCache)
    check(_lib.lib().afhip_launch_rotated_store(stream, rotation, None if quantized else cache, cache if quantized else None, Buffer(at, held),
                                                token, head, Buffer(*_line(slots, _I32, tokens))))


def quantizedAttention(cache: _lib.QuantizedCache, out, query, query_starts, context_lens, block_tables, max_query_len: int, max_key_len: int,
                       scale: float = None, softcap: float = 0.0, window: int = 0, slopes=None) -> _lib.QuantizedAttention:
    """The arguments of a call (of any number of calls while the arrays stay): query, out [tokens, heads, head dim]; scale:
    head_dim ** -0.5 unless given; softcap 0: scores as they are; window 0: all earlier keys; slopes f32 [heads]."""
    tokens, heads, dim = query.shape
    requests, columns = block_tables.shape
    dtype = query.dtype
    type, size = _kind(dtype)
    if out.dtype != dtype or dim != cache.head_dim:
        raise _bad_shape()
    q_token, q_head, q_at, q_held = _heads_of(query, size, tokens, heads, dim)
    o_token, o_head, o_at, o_held = _heads_of(out, size, tokens, heads, dim)
    s_at, s_held = _line(slopes, _F32, heads)
    try:
        made = _lib.QuantizedAttention.from_buffer_copy(bytes(cache) + _QUANTIZED_REST.pack(
            type, dim ** -0.5 if scale is None else scale, softcap, window, requests, tokens, heads, max_query_len, max_key_len, columns,
            q_token, q_head, o_token, o_head, q_at, q_held, o_at, o_held, *_i32(query_starts), *_i32(context_lens), *_i32(block_tables),
            s_at, s_held))
    except struct.error:
        raise _bad_number() from None
    made.arrays = (cache, out, query, query_starts, context_lens, block_tables, slopes)
    return made


def quantizedAttentionWorkspaceBytes(attention: _lib.QuantizedAttention) -> int:
    return _lib.lib().afhip_quantized_attention_workspace_bytes(attention)


def launchQuantizedAttention(stream, attention: _lib.QuantizedAttention, workspace: Buffer = NO_BUFFER) -> None:
    """`workspace`: a Buffer, or an array, of at least quantizedAttentionWorkspaceBytes(attention) bytes."""
    check(_lib.lib().afhip_launch_quantized_attention(stream, attention,
                                                      workspace if isinstance(workspace, Buffer) else buffer(workspace)))
