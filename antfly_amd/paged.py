"""A paged key / value cache and what a speculative decode step does with it: plan the batch, store the drafted tokens' keys
and values, attend over context and draft tree, move the accepted path behind the context.

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
assert _CACHE.size == C.sizeof(_lib.PagedCache) and _PLAN.size == C.sizeof(_lib.BatchPlan)
assert _CACHE.size + _REST.size == C.sizeof(_lib.TreeAttention)


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
