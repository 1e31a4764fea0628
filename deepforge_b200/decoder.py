"""ctypes view of the operators around the attention of a decoder's step (include/dfgpu_decoder.h): norms of query and key heads with
their rotary positions, products of 8-bit integers, beam search. Same conventions as `dfgpu` and `cache`: raw device addresses, an exception
for a non-zero status.

`pointers` of every call is the port list of the header, in order, None for an absent port; ports left off the end are absent.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Sequence

from . import dfgpu
from .dfgpu import DfgpuError, PlanInfo, Tensor, tensor  # noqa: F401  (tensor: what callers fill the descriptors with)

I8 = 12
HEAD_NORM_AUTO, HEAD_NORM_VECTOR, HEAD_NORM_SCALAR = range(3)
TOKEN_QUANTIZE_AUTO, TOKEN_QUANTIZE_VECTOR, TOKEN_QUANTIZE_SCALAR = range(3)
MATMUL_INT8_AUTO, MATMUL_INT8_CORES, MATMUL_INT8_UMMA, MATMUL_INT8_FEW = range(4)
MAX_STATES = 8


class _Scaled(C.Structure):
    """Whose scale is 1 where nothing else is said."""
    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if "scale" not in kwargs:
            self.scale = 1.0


class HeadNormParams(_Scaled):
    _fields_ = [("x", Tensor), ("y", Tensor), ("x2", Tensor), ("y2", Tensor), ("gain", Tensor), ("gain2", Tensor), ("positions", Tensor),
                ("frequencies", Tensor), ("interleaved", C.c_int32), ("scale", C.c_float), ("epsilon", C.c_float), ("gain_offset", C.c_float),
                ("kernel", C.c_int32), ("reserved", C.c_int32)]


class HeadNormGradParams(_Scaled):
    _fields_ = [("x", Tensor), ("dy", Tensor), ("dx", Tensor), ("x2", Tensor), ("dy2", Tensor), ("dx2", Tensor), ("gain", Tensor), ("dgain", Tensor),
                ("gain2", Tensor), ("dgain2", Tensor), ("positions", Tensor), ("frequencies", Tensor), ("interleaved", C.c_int32), ("scale", C.c_float),
                ("epsilon", C.c_float), ("gain_offset", C.c_float), ("kernel", C.c_int32), ("reserved", C.c_int32)]


class TokenQuantizeParams(C.Structure):
    _fields_ = [("x", Tensor), ("y", Tensor), ("scale", Tensor), ("kernel", C.c_int32), ("reserved", C.c_int32)]


class MatmulInt8Params(C.Structure):
    _fields_ = [("a", Tensor), ("b", Tensor), ("c", Tensor), ("a_scale", Tensor), ("b_scale", Tensor), ("bias", Tensor), ("kernel", C.c_int32),
                ("reserved", C.c_int32)]


class BeamSelectParams(C.Structure):
    _fields_ = [("logits", Tensor), ("scores", Tensor), ("finished", Tensor), ("lengths", Tensor), ("scores_out", Tensor), ("tokens", Tensor),
                ("parents", Tensor), ("finished_out", Tensor), ("lengths_out", Tensor), ("forks", Tensor), ("length_penalty", C.c_float),
                ("end", C.c_int32), ("pad", C.c_int32), ("source_base", C.c_int32), ("target_base", C.c_int32), ("reserved", C.c_int32)]

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if "end" not in kwargs:
            self.end = -1


class BeamReorderParams(C.Structure):
    _fields_ = [("parents", Tensor), ("source", Tensor * MAX_STATES), ("target", Tensor * MAX_STATES), ("count", C.c_int32), ("reserved", C.c_int32)]


# every symbol include/dfgpu_decoder.h declares
EXPORTS = ["dfgpu_decoder_abi_version", "dfgpu_query_head_norm", "dfgpu_head_norm", "dfgpu_query_head_norm_grad", "dfgpu_head_norm_grad",
           "dfgpu_query_token_quantize", "dfgpu_token_quantize", "dfgpu_query_matmul_int8", "dfgpu_matmul_int8", "dfgpu_query_beam_select",
           "dfgpu_beam_select", "dfgpu_query_beam_reorder", "dfgpu_beam_reorder"]

_PORTS = {"head_norm": 8, "head_norm_grad": 12, "token_quantize": 3, "matmul_int8": 6, "beam_select": 10, "beam_reorder": 1 + 2 * MAX_STATES}
_FUNCTIONS: dict = {}


def _call(name: str, params, pointers: Sequence[Optional[int]], scratch: Optional[int], stream: Optional[int]) -> None:
    """(A small kernel is over before its call is: the port list goes as packed bytes, a tenth of the time of an array of c_void_p.)"""
    found = _FUNCTIONS.get(name)
    if found is None:
        function = getattr(dfgpu.load(), "dfgpu_" + name)
        function.restype, function.argtypes = C.c_int, [C.c_void_p, C.c_char_p, C.c_void_p, C.c_void_p]
        found = _FUNCTIONS[name] = (function, struct.Struct(f"{_PORTS[name]}P"), _PORTS[name])
    function, ports, count = found
    if len(pointers) != count or None in pointers:
        if len(pointers) > count:
            raise ValueError(f"{name} has {count} ports, not {len(pointers)}")
        pointers = [p or 0 for p in pointers] + [0] * (count - len(pointers))
    code = function(C.addressof(params), ports.pack(*pointers), scratch, stream)
    if code != 0:
        raise DfgpuError(code, dfgpu.load().dfgpu_last_error().decode(errors="replace"))


def query(name: str, params) -> PlanInfo:
    """What the launcher `name` ("head_norm", "head_norm_grad", "token_quantize", "matmul_int8", "beam_select", "beam_reorder") will use for
    these params: kernel, launches, scratch bytes."""
    return dfgpu.query(name, params)


def head_norm(params: HeadNormParams, pointers: Sequence[Optional[int]], stream: Optional[int] = None) -> None:
    """pointers: X, Y[, gain[, positions, frequencies[, X2, Y2[, gain2]]]]."""
    _call("head_norm", params, pointers, None, stream)


def head_norm_grad(params: HeadNormGradParams, pointers: Sequence[Optional[int]], scratch: Optional[int] = None, stream: Optional[int] = None) -> None:
    """pointers: X, dY, dX[, gain, dgain[, positions, frequencies[, X2, dY2, dX2[, gain2, dgain2]]]]."""
    _call("head_norm_grad", params, pointers, scratch, stream)


def token_quantize(params: TokenQuantizeParams, pointers: Sequence[Optional[int]], stream: Optional[int] = None) -> None:
    """pointers: X, Y, scale."""
    _call("token_quantize", params, pointers, None, stream)


def matmul_int8(params: MatmulInt8Params, pointers: Sequence[Optional[int]], stream: Optional[int] = None) -> None:
    """pointers: A, B, C, a_scale, b_scale[, bias]."""
    _call("matmul_int8", params, pointers, None, stream)


def beam_select(params: BeamSelectParams, pointers: Sequence[Optional[int]], scratch: Optional[int] = None, stream: Optional[int] = None) -> None:
    """pointers: logits, scores, finished, lengths, scores_out, tokens, parents[, finished_out[, lengths_out[, forks]]]."""
    _call("beam_select", params, pointers, scratch, stream)


def beam_reorder(params: BeamReorderParams, pointers: Sequence[Optional[int]], stream: Optional[int] = None) -> None:
    """pointers: parents, source 0, target 0[, source 1, target 1, ...]."""
    _call("beam_reorder", params, pointers, None, stream)
