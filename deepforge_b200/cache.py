"""ctypes view of the operators around a paged key/value cache in 8 bits (include/dfgpu_cache.h): rotary positions, appending
tokens, attention and page bookkeeping. Same conventions as `dfgpu`: raw device addresses, an exception for a non-zero status.

`pointers` of every call is the port list of the header, in order, None for an absent port; ports left off the end are absent.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Sequence

from . import dfgpu
from .dfgpu import DfgpuError, PlanInfo, Tensor, tensor  # noqa: F401  (tensor: what callers fill the descriptors with)

ROPE_AUTO, ROPE_VECTOR, ROPE_SCALAR = range(3)
ROPE_SCALINGS = {name: code for code, name in enumerate(("none", "linear", "base", "ramp", "bands"))}
APPEND_AUTO, APPEND_VECTOR, APPEND_SCALAR = range(3)
SDPA_AUTO, SDPA_STREAM, SDPA_UMMA = range(3)
PAGE_OPS = {name: code for code, name in enumerate(("reserve", "fork", "free", "compact", "copy"))}
MAX_POOLS = 8


class RopeParams(C.Structure):
    _fields_ = [("x", Tensor), ("y", Tensor), ("x2", Tensor), ("y2", Tensor), ("positions", Tensor), ("frequencies", Tensor),
                ("interleaved", C.c_int32), ("inverse", C.c_int32), ("scale", C.c_float), ("kernel", C.c_int32)]

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if "scale" not in kwargs:
            self.scale = 1.0


class RopeScaling(C.Structure):
    _fields_ = [("kind", C.c_int32), ("rotary", C.c_int32), ("base", C.c_double), ("factor", C.c_double), ("original", C.c_double),
                ("low", C.c_double), ("high", C.c_double)]


class CacheAppendParams(C.Structure):
    _fields_ = [("k", Tensor), ("v", Tensor), ("k_cache", Tensor), ("v_cache", Tensor), ("k_scale", Tensor), ("v_scale", Tensor),
                ("page_table_k", Tensor), ("page_table_v", Tensor), ("lengths", Tensor), ("added", Tensor), ("lengths_out", Tensor),
                ("kernel", C.c_int32), ("reserved", C.c_int32)]


class CacheSdpaParams(C.Structure):
    _fields_ = [("q", Tensor), ("k", Tensor), ("v", Tensor), ("o", Tensor), ("stats", Tensor), ("k_scale", Tensor), ("v_scale", Tensor),
                ("seq_q", Tensor), ("seq_kv", Tensor), ("page_table_k", Tensor), ("page_table_v", Tensor), ("attn_scale", C.c_float),
                ("has_left_bound", C.c_int32), ("has_right_bound", C.c_int32), ("bottom_right", C.c_int32), ("left_bound", C.c_int64),
                ("right_bound", C.c_int64), ("s_kv", C.c_int64), ("kernel", C.c_int32), ("reserved", C.c_int32)]


class CachePagesParams(C.Structure):
    _fields_ = [("op", C.c_int32), ("pool_count", C.c_int32), ("block", C.c_int64), ("page_table", Tensor), ("lengths", Tensor),
                ("refs", Tensor), ("list", Tensor), ("pools", Tensor * MAX_POOLS)]


# every symbol include/dfgpu_cache.h declares
EXPORTS = ["dfgpu_cache_abi_version", "dfgpu_query_rope", "dfgpu_rope", "dfgpu_rope_frequencies", "dfgpu_query_cache_append", "dfgpu_cache_append",
           "dfgpu_query_cache_sdpa", "dfgpu_cache_sdpa", "dfgpu_query_cache_pages", "dfgpu_cache_pages"]

_PORTS = {"rope": 6, "cache_append": 11, "cache_sdpa": 11, "cache_pages": 8 + MAX_POOLS}
_FUNCTIONS: dict = {}


def _function(name: str):
    """The launcher and the array type of its ports. Its arguments keep their types here, so that a call converts no more than it must."""
    found = _FUNCTIONS.get(name)
    if found is None:
        function = getattr(dfgpu.load(), "dfgpu_" + name)
        function.restype, function.argtypes = C.c_int, [C.c_void_p] * 4
        found = _FUNCTIONS[name] = (function, C.c_void_p * _PORTS[name])
    return found


def _call(name: str, params, pointers: Sequence[Optional[int]], scratch: Optional[int], stream: Optional[int]) -> None:
    function, ports = _function(name)
    code = function(C.addressof(params), ports(*pointers), scratch, stream)
    if code != 0:
        raise DfgpuError(code, dfgpu.load().dfgpu_last_error().decode(errors="replace"))


def query(name: str, params) -> PlanInfo:
    """What the launcher `name` ("rope", "cache_append", "cache_sdpa", "cache_pages") will use for these params: kernel, launches, scratch bytes."""
    return dfgpu.query(name, params)


def rope(params: RopeParams, pointers: Sequence[Optional[int]], stream: Optional[int] = None) -> None:
    """pointers: X, Y, positions, frequencies[, X2, Y2]."""
    _call("rope", params, pointers, None, stream)


def rope_frequencies(rotary: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0, original: float = 0.0, low: float = 1.0,
                     high: float = 32.0) -> tuple[list[float], float]:
    """(frequencies of the rotary / 2 pairs, magnitude for RopeParams.scale); `scaling` is a key of ROPE_SCALINGS."""
    if scaling not in ROPE_SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r}: one of {', '.join(ROPE_SCALINGS)}")
    wanted = RopeScaling(ROPE_SCALINGS[scaling], rotary, base, factor, original, low, high)
    out, magnitude = (C.c_float * max(1, rotary // 2))(), C.c_float(math.nan)
    function = dfgpu.load().dfgpu_rope_frequencies
    function.restype = C.c_int
    code = function(C.byref(wanted), out, C.byref(magnitude))
    if code != 0:
        raise DfgpuError(code, dfgpu.load().dfgpu_last_error().decode(errors="replace"))
    return list(out), magnitude.value


def cache_append(params: CacheAppendParams, pointers: Sequence[Optional[int]], stream: Optional[int] = None) -> None:
    """pointers: K, V, K container, V container, K scale, V scale, page table of K, page table of V, lengths[, added[, lengths_out]]."""
    _call("cache_append", params, pointers, None, stream)


def cache_sdpa(params: CacheSdpaParams, pointers: Sequence[Optional[int]], scratch: Optional[int] = None, stream: Optional[int] = None) -> None:
    """pointers: Q, K container, V container, O, Stats, K scale, V scale, SEQ_LEN_Q, SEQ_LEN_KV, Page_table_K, Page_table_V."""
    _call("cache_sdpa", params, pointers, scratch, stream)


def cache_pages(params: CachePagesParams, pointers: Sequence[Optional[int]], scratch: Optional[int] = None, stream: Optional[int] = None) -> None:
    """pointers: page table, lengths, refs, list, table_out, lengths_out, refs_out, report[, pools...]."""
    _call("cache_pages", params, pointers, scratch, stream)
