"""A paged key / value cache and what a speculative decode step does with it: plan the batch, store the drafted tokens' keys
and values, attend over context and draft tree, move the accepted path behind the context.

The functions take device arrays: anything with torch's `data_ptr()`, `shape`, `stride()`, `dtype`, `numel()` and
`element_size()` (this package does not import torch).  Layouts, and what each launch reads and writes, are those of the C
ABI (include/antfly_hip_qmatmul.h); `stream` is a hipStream_t."""
from __future__ import annotations

import ctypes as C

from . import _lib
from ._lib import Buffer, check

NO_BUFFER = Buffer(0, 0)
_TYPES = {"torch.float32": _lib.TYPE_F32, "torch.float16": _lib.TYPE_F16, "torch.bfloat16": _lib.TYPE_BF16}


def buffer(array) -> Buffer:
    """The memory that an array spans, from its first element to its last; None: no buffer."""
    if array is None:
        return NO_BUFFER
    count = array.numel()
    if count and not array.is_contiguous():
        count = 1 + sum((n - 1) * s for n, s in zip(array.shape, array.stride()))
    return Buffer(array.data_ptr(), count * array.element_size())


def _type(array) -> int:
    return _TYPES.get(str(array.dtype), -1)


def _array(array, kind) -> Buffer:
    """A contiguous array of whole numbers of the given width."""
    if array is None:
        return NO_BUFFER
    if str(array.dtype) not in kind or not array.is_contiguous():
        raise _lib.InvalidShape(_lib.ERR_INVALID_SHAPE)
    return Buffer(array.data_ptr(), array.numel() * array.element_size())


_I32, _U64 = ("torch.int32",), ("torch.int64", "torch.uint64")


def _rows_of_heads(array, rows, heads, dim):
    """(token stride, head stride) of [rows, heads, dim] whose last dimension is contiguous."""
    if tuple(array.shape) != (rows, heads, dim) or (dim > 1 and array.stride(2) != 1):
        raise _lib.InvalidShape(_lib.ERR_INVALID_SHAPE)
    return array.stride(0), array.stride(1)


def cache(keys, values, heads_outside: bool = False) -> _lib.PagedCache:
    """keys, values [blocks, block size, kv heads, head dim], or with heads_outside [blocks, kv heads, block size, head dim]."""
    if len(keys.shape) != 4 or keys.shape != values.shape or keys.dtype != values.dtype or keys.stride() != values.stride() or \
            (keys.shape[3] > 1 and keys.stride(3) != 1):
        raise _lib.InvalidShape(_lib.ERR_INVALID_SHAPE)
    blocks, slots, heads, dim = keys.shape
    strides = keys.stride()
    slot_stride, head_stride = strides[1], strides[2]
    if heads_outside:
        slots, heads, slot_stride, head_stride = heads, slots, head_stride, slot_stride
    made = _lib.PagedCache(buffer(keys), buffer(values), _type(keys), blocks, slots, heads, dim, strides[0], slot_stride, head_stride)
    made.arrays = (keys, values)  # alive as long as the description of them is
    return made


def launchBatchPlan(stream, context_lens, query_lens, block_tables, free_blocks, block_size: int, query_starts, slots, positions,
                    blocks_taken, parents=None, masks=None, blocks: int = (1 << 31) - 1) -> None:
    """Writes block_tables (new entries), query_starts, slots, positions, masks and blocks_taken from the requests' lengths;
    `blocks`: how many the cache has (numbers outside name none)."""
    requests, columns = block_tables.shape
    tokens = slots.shape[0]
    if positions.shape[0] != tokens or (parents is not None and parents.shape[0] != tokens) or \
            (masks is not None and (len(masks.shape) != 2 or masks.shape[0] != tokens)):
        raise _lib.InvalidShape(_lib.ERR_INVALID_SHAPE)
    check(_lib.lib().afhip_launch_batch_plan(stream, C.byref(_lib.BatchPlan(
        requests, columns, block_size, blocks, tokens, 0 if masks is None else masks.shape[1],
        _array(context_lens, _I32), _array(query_lens, _I32), _array(free_blocks, _I32),
        _array(parents, _I32), _array(block_tables, _I32), _array(query_starts, _I32),
        _array(slots, _I32), _array(positions, _I32), _array(masks, _U64),
        _array(blocks_taken, _I32)))))


def launchCacheStore(stream, cache: _lib.PagedCache, keys, values, slots) -> None:
    """keys, values [tokens, kv heads, head dim] (f32, f16 or bf16) into the cache's slots."""
    tokens = slots.shape[0]
    strides = _rows_of_heads(keys, tokens, cache.kv_heads, cache.head_dim)
    if _rows_of_heads(values, tokens, cache.kv_heads, cache.head_dim) != strides or keys.dtype != values.dtype:
        raise _lib.InvalidShape(_lib.ERR_INVALID_SHAPE)
    check(_lib.lib().afhip_launch_cache_store(stream, C.byref(cache), _type(keys), buffer(keys), buffer(values), strides[0],
                                              strides[1], _array(slots, _I32), tokens))


def launchCacheMove(stream, cache: _lib.PagedCache, block_tables, context_lens, paths, path_lens) -> None:
    """The accepted path of every request's tree to the places behind its context."""
    requests, columns = block_tables.shape
    if len(paths.shape) != 2 or paths.shape[0] != requests:
        raise _lib.InvalidShape(_lib.ERR_INVALID_SHAPE)
    check(_lib.lib().afhip_launch_cache_move(stream, C.byref(cache), _array(block_tables, _I32), columns,
                                             _array(context_lens, _I32), _array(paths, _I32),
                                             _array(path_lens, _I32), requests, paths.shape[1]))


def treeAttention(cache: _lib.PagedCache, out, query, query_starts, context_lens, block_tables, max_query_len: int,
                  max_key_len: int, masks=None, scale: float = None) -> _lib.TreeAttention:
    """The arguments of a call (any number of calls while the arrays stay): query, out [tokens, heads, head dim]; scale: head_dim ** -0.5 unless given."""
    tokens, heads, dim = query.shape
    requests, columns = block_tables.shape
    q, o = _rows_of_heads(query, tokens, heads, cache.head_dim), _rows_of_heads(out, tokens, heads, cache.head_dim)
    if out.dtype != query.dtype or (masks is not None and (len(masks.shape) != 2 or masks.shape[0] != tokens)):
        raise _lib.InvalidShape(_lib.ERR_INVALID_SHAPE)
    made = _lib.TreeAttention(cache, _type(query), dim ** -0.5 if scale is None else scale, requests, tokens, heads, max_query_len,
                              max_key_len, columns, 0 if masks is None else masks.shape[1], q[0], q[1], o[0], o[1], buffer(query),
                              buffer(out), _array(query_starts, _I32), _array(context_lens, _I32),
                              _array(block_tables, _I32), _array(masks, _U64))
    made.arrays = (cache, out, query, query_starts, context_lens, block_tables, masks)
    return made


def treeAttentionWorkspaceBytes(attention: _lib.TreeAttention) -> int:
    return _lib.lib().afhip_tree_attention_workspace_bytes(C.byref(attention))


def launchTreeAttention(stream, attention: _lib.TreeAttention, workspace: Buffer = NO_BUFFER) -> None:
    """`workspace`: a Buffer, or an array, of at least treeAttentionWorkspaceBytes(attention) bytes."""
    check(_lib.lib().afhip_launch_tree_attention(stream, C.byref(attention),
                                                 workspace if isinstance(workspace, Buffer) else buffer(workspace)))
