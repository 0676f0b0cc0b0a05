"""A token of every row of logits, drawn by temperature, top-k, top-p and min-p from a given random number.

The functions take device arrays, as those of paged.py do; what is kept and drawn is said in the C ABI
(include/antfly_hip_qmatmul.h); `stream` is a hipStream_t."""
from __future__ import annotations

import ctypes as C
import struct

from . import _lib
from ._lib import Buffer, check
from .paged import _F32, _I32, NO_BUFFER, _bad_number, _bad_shape, _kind, _line, buffer

_SAMPLE = struct.Struct("i4x19Q")
assert _SAMPLE.size == C.sizeof(_lib.Sample)


def sample(logits, tokens, uniforms, temperatures=None, top_k=None, top_p=None, min_p=None, probabilities=None) -> _lib.Sample:
    """The arguments of a call (of any number of calls while the arrays stay): logits [rows, vocab] (f32, f16 or bf16) -> tokens int32
    [rows] and probabilities f32 [rows].  uniforms, temperatures, top_p, min_p f32 [rows], top_k int32 [rows]; what is None filters
    nothing, temperatures then are 1."""
    rows, vocab = logits.shape
    stride, step = logits.stride()
    if (vocab > 1 and step != 1) or tokens is None or uniforms is None:
        raise _bad_shape()
    type, size = _kind(logits.dtype)
    try:
        made = _lib.Sample.from_buffer_copy(_SAMPLE.pack(
            type, rows, vocab, stride, logits.data_ptr(), ((rows - 1) * stride + vocab) * size if rows else 0, *_line(temperatures, _F32, rows),
            *_line(top_k, _I32, rows), *_line(top_p, _F32, rows), *_line(min_p, _F32, rows), *_line(uniforms, _F32, rows),
            *_line(tokens, _I32, rows), *_line(probabilities, _F32, rows)))
    except struct.error:
        raise _bad_number() from None
    made.arrays = (logits, tokens, uniforms, temperatures, top_k, top_p, min_p, probabilities)
    return made


def sampleWorkspaceBytes(sample: _lib.Sample) -> int:
    return _lib.lib().afhip_sample_workspace_bytes(sample)


def launchSample(stream, sample: _lib.Sample, workspace: Buffer = NO_BUFFER) -> None:
    """`workspace`: a Buffer, or an array, of at least sampleWorkspaceBytes(sample) bytes."""
    check(_lib.lib().afhip_launch_sample(stream, sample, workspace if isinstance(workspace, Buffer) else buffer(workspace)))
