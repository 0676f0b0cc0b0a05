"""A token of every row of logits, drawn by temperature, top-k, top-p and min-p from a given random number.

The functions take device arrays, as those of paged.py do; what is kept and drawn is said in the C ABI
(include/antfly_hip_qmatmul.h); `stream` is a hipStream_t."""
from __future__ import annotations

import ctypes as C
import struct

from . import _lib
from ._lib import Buffer, check
from .paged import NO_BUFFER, _bad_number, _bad_shape, _bytes, _name, _type, buffer

_SAMPLE = struct.Struct("i4x19Q")
assert _SAMPLE.size == C.sizeof(_lib.Sample)


def _a_row(array, rows, dtype="torch.float32"):
    """(address, bytes) of one number a row; None: none."""
    if array is None:
        return 0, 0
    if _name(array.dtype) != dtype or array.shape != (rows,) or not array.is_contiguous():
        raise _bad_shape()
    return array.data_ptr(), array.nbytes


def sample(logits, tokens, uniforms, temperatures=None, top_k=None, top_p=None, min_p=None, probabilities=None) -> _lib.Sample:
    """The arguments of a call (of any number of calls while the arrays stay): logits [rows, vocab] (f32, f16 or bf16) -> tokens int32
    [rows] and probabilities f32 [rows].  uniforms, temperatures, top_p, min_p f32 [rows], top_k int32 [rows]; what is None filters
    nothing, temperatures then are 1."""
    rows, vocab = logits.shape
    if (vocab > 1 and logits.stride(1) != 1) or tokens is None or uniforms is None:
        raise _bad_shape()
    try:
        made = _lib.Sample.from_buffer_copy(_SAMPLE.pack(
            _type(logits), rows, vocab, logits.stride(0), logits.data_ptr(), _bytes(logits), *_a_row(temperatures, rows),
            *_a_row(top_k, rows, "torch.int32"), *_a_row(top_p, rows), *_a_row(min_p, rows), *_a_row(uniforms, rows),
            *_a_row(tokens, rows, "torch.int32"), *_a_row(probabilities, rows)))
    except struct.error:
        raise _bad_number() from None
    made.arrays = (logits, tokens, uniforms, temperatures, top_k, top_p, min_p, probabilities)
    return made


def sampleWorkspaceBytes(sample: _lib.Sample) -> int:
    return _lib.lib().afhip_sample_workspace_bytes(sample)


def launchSample(stream, sample: _lib.Sample, workspace: Buffer = NO_BUFFER) -> None:
    """`workspace`: a Buffer, or an array, of at least sampleWorkspaceBytes(sample) bytes."""
    check(_lib.lib().afhip_launch_sample(stream, sample, workspace if isinstance(workspace, Buffer) else buffer(workspace)))
