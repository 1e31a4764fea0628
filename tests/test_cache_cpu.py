"""The cache operators' C ABI without a GPU: layouts, refusals before any CUDA call, frequencies, and the 64-bit restatement's own encoder."""
import ctypes as C
import math
import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import cache_reference as ref
from deepforge_b200 import cache, dfgpu
from deepforge_b200.dfgpu import BF16, E4M3, E8M0, F16, F32, I32, I64, U8, tensor

ROOT = Path(__file__).resolve().parent.parent


def test_exports_and_layouts(tmp_path):
    text = (ROOT / "include" / "dfgpu_cache.h").read_text()
    code = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"\b(dfgpu_[a-z0-9_]+)\s*\(", code)))
    assert sorted(cache.EXPORTS) == names
    lib = dfgpu.load()
    for name in names:
        assert hasattr(lib, name), name
    assert lib.dfgpu_cache_abi_version() == 1
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    structs = {"rope_params": cache.RopeParams, "rope_scaling": cache.RopeScaling, "cache_append_params": cache.CacheAppendParams,
               "cache_sdpa_params": cache.CacheSdpaParams, "cache_pages_params": cache.CachePagesParams}
    source = tmp_path / "sizes.c"
    source.write_text('#include <stdio.h>\n#include "dfgpu_cache.h"\nint main(void){' + "".join(f'printf("%zu\\n", sizeof(dfgpu_{n}));' for n in structs) + "return 0;}\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    sizes = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in sizes] == [C.sizeof(s) for s in structs.values()]


def refused(code, name, params, text=""):
    with pytest.raises(dfgpu.DfgpuError) as error:
        cache.query(name, params)
    assert error.value.code == code and text in str(error.value), error.value


def rope_params(**change):
    p = cache.RopeParams()
    p.x = p.y = tensor(BF16, [2, 4, 3, 64])
    p.positions, p.frequencies = tensor(I32, [2, 1, 3, 1]), tensor(F32, [1, 1, 1, 32])
    for key, value in change.items():
        setattr(p, key, value)
    return p


def test_rope_refusals():
    info = cache.query("rope", rope_params())
    assert (info.kernel, info.launches, info.scratch_bytes) == (cache.ROPE_VECTOR, 1, 0)
    assert cache.query("rope", rope_params(frequencies=tensor(F32, [1, 1, 1, 5]))).kernel == cache.ROPE_SCALAR
    refused(15, "rope", rope_params(frequencies=tensor(F32, [1, 1, 1, 33])))
    refused(20, "rope", rope_params(frequencies=tensor(F16, [1, 1, 1, 32])))
    refused(15, "rope", rope_params(positions=tensor(I32, [3, 1, 3, 1])))
    refused(20, "rope", rope_params(positions=tensor(F32, [1, 1, 3, 1])))
    refused(20, "rope", rope_params(y=tensor(F32, [2, 4, 3, 64])))
    refused(15, "rope", rope_params(y=tensor(BF16, [2, 4, 4, 64])))
    refused(14, "rope", rope_params(x=tensor(BF16, [2, 4, 3, 64], [1536, 384, 128, 2])))
    refused(15, "rope", rope_params(x2=tensor(BF16, [2, 1, 3, 64])))
    refused(15, "rope", rope_params(x2=tensor(BF16, [2, 1, 3, 32]), y2=tensor(BF16, [2, 1, 3, 32])))
    refused(20, "rope", rope_params(x=tensor(U8, [2, 4, 3, 64])))
    refused(1, "rope", rope_params(kernel=7))
    refused(20, "rope", rope_params(kernel=cache.ROPE_VECTOR, frequencies=tensor(F32, [1, 1, 1, 5])))
    assert cache.query("rope", rope_params(positions=tensor(I64, [1, 1, 3, 1]))).launches == 1
    for pointers in ([None, 16, 16, 16], [16, 16, 16, None], [17, 16, 16, 16], [16, 16, 18, 16]):
        with pytest.raises(dfgpu.DfgpuError) as error:
            cache.rope(rope_params(), pointers)
        assert error.value.code == 1
    with pytest.raises(dfgpu.DfgpuError) as error:   # in place with other strides
        cache.rope(rope_params(y=tensor(BF16, [2, 4, 3, 64], [768, 64, 256, 1])), [16, 16, 16, 16])
    assert error.value.code == 14


def append_params(**change):
    p = cache.CacheAppendParams()
    p.k = p.v = tensor(BF16, [2, 4, 3, 64])
    p.k_cache = p.v_cache = tensor(E4M3, [9, 4, 32, 64])
    p.k_scale = p.v_scale = tensor(E8M0, [9, 4, 2, 1])
    p.page_table_k = p.page_table_v = tensor(I32, [2, 1, 4, 1])
    p.lengths = tensor(I32, [2, 1, 1, 1])
    for key, value in change.items():
        setattr(p, key, value)
    return p


def test_append_refusals():
    assert cache.query("cache_append", append_params()).kernel == cache.APPEND_VECTOR
    assert cache.query("cache_append", append_params(k=tensor(BF16, [2, 4, 3, 64], [769, 192, 64, 1]))).kernel == cache.APPEND_SCALAR
    refused(15, "cache_append", append_params(v=tensor(BF16, [2, 4, 2, 64])))
    refused(20, "cache_append", append_params(v=tensor(F16, [2, 4, 3, 64])))
    refused(15, "cache_append", append_params(k_cache=tensor(BF16, [9, 4, 32, 64])))
    refused(15, "cache_append", append_params(k_cache=tensor(E4M3, [9, 4, 32, 128])))
    refused(15, "cache_append", append_params(v_cache=tensor(E4M3, [9, 4, 64, 64])))
    refused(14, "cache_append", append_params(k_cache=tensor(E4M3, [9, 4, 32, 64], [8192, 0, 64, 1])))
    refused(15, "cache_append", append_params(k_scale=tensor(E8M0, [9, 4, 3, 1])))
    refused(15, "cache_append", append_params(k_scale=tensor(E8M0, [9, 4, 4, 1])))
    refused(15, "cache_append", append_params(k_scale=tensor(F32, [9, 4, 2, 1])))
    refused(15, "cache_append", append_params(page_table_v=tensor(I64, [2, 1, 4, 1])))
    refused(15, "cache_append", append_params(lengths=tensor(I32, [3, 1, 1, 1])))
    refused(15, "cache_append", append_params(added=tensor(F32, [2, 1, 1, 1])))
    refused(1, "cache_append", append_params(kernel=9))
    good = [16] * 3 + [32] + [16, 32] + [16] * 3
    for i in range(9):
        with pytest.raises(dfgpu.DfgpuError) as error:
            cache.cache_append(append_params(), good[:i] + [None] + good[i + 1:])
        assert error.value.code == 1 and f"port {i}" in str(error.value)
    with pytest.raises(dfgpu.DfgpuError):   # one container for both
        cache.cache_append(append_params(), [16] * 9)
    with pytest.raises(dfgpu.DfgpuError):   # declared, not given
        cache.cache_append(append_params(added=tensor(I32, [2, 1, 1, 1])), good)


def sdpa_params(**change):
    p = cache.CacheSdpaParams(attn_scale=0.125, s_kv=100)
    p.q = p.o = tensor(BF16, [2, 8, 3, 64])
    p.k = p.v = tensor(E4M3, [9, 4, 32, 64])
    p.k_scale = p.v_scale = tensor(E8M0, [9, 4, 2, 1])
    p.page_table_k = p.page_table_v = tensor(I32, [2, 1, 4, 1])
    p.seq_kv = tensor(I32, [2, 1, 1, 1])
    for key, value in change.items():
        setattr(p, key, value)
    return p


def test_sdpa_refusals():
    assert cache.query("cache_sdpa", sdpa_params()).kernel == cache.SDPA_STREAM
    info = cache.query("cache_sdpa", sdpa_params(kernel=cache.SDPA_UMMA))
    assert (info.kernel, info.launches) == (cache.SDPA_UMMA, 3) and info.scratch_bytes > cache.query("cache_sdpa", sdpa_params()).scratch_bytes
    refused(20, "cache_sdpa", sdpa_params(q=tensor(F32, [2, 8, 3, 64])))
    refused(20, "cache_sdpa", sdpa_params(o=tensor(F16, [2, 8, 3, 64])))
    refused(15, "cache_sdpa", sdpa_params(o=tensor(BF16, [2, 8, 2, 64])))
    refused(14, "cache_sdpa", sdpa_params(o=tensor(BF16, [2, 8, 3, 64], [1536, 0, 64, 1])))
    refused(15, "cache_sdpa", sdpa_params(k=tensor(E4M3, [9, 4, 32, 128])))
    refused(15, "cache_sdpa", sdpa_params(v=tensor(E4M3, [9, 2, 32, 64])))
    refused(14, "cache_sdpa", sdpa_params(k=tensor(E4M3, [9, 4, 32, 64], [8200, 2050, 64, 1])))
    refused(20, "cache_sdpa", sdpa_params(k_scale=tensor(E8M0, [9, 4, 4, 1]), v_scale=tensor(E8M0, [9, 4, 4, 1])), "16 tokens")
    refused(15, "cache_sdpa", sdpa_params(v_scale=tensor(E8M0, [9, 4, 1, 1])))
    refused(15, "cache_sdpa", sdpa_params(s_kv=129), "capacity")
    refused(15, "cache_sdpa", sdpa_params(s_kv=0))
    refused(15, "cache_sdpa", sdpa_params(q=tensor(BF16, [2, 6, 3, 64]), o=tensor(BF16, [2, 6, 3, 64])))
    refused(15, "cache_sdpa", sdpa_params(seq_kv=tensor(I64, [2, 1, 1, 1])))
    refused(15, "cache_sdpa", sdpa_params(stats=tensor(F32, [2, 8, 1, 1])))
    refused(8, "cache_sdpa", sdpa_params(attn_scale=math.inf))
    refused(1, "cache_sdpa", sdpa_params(kernel=9))
    d = 96
    refused(20, "cache_sdpa", sdpa_params(q=tensor(BF16, [2, 8, 3, d]), o=tensor(BF16, [2, 8, 3, d]), k=tensor(E4M3, [9, 4, 32, d]), v=tensor(E4M3, [9, 4, 32, d])))
    d = 256
    wide = dict(q=tensor(BF16, [2, 8, 3, d]), o=tensor(BF16, [2, 8, 3, d]), k=tensor(E4M3, [9, 4, 32, d]), v=tensor(E4M3, [9, 4, 32, d]))
    assert cache.query("cache_sdpa", sdpa_params(**wide)).kernel == cache.SDPA_STREAM
    refused(20, "cache_sdpa", sdpa_params(kernel=cache.SDPA_UMMA, **wide))
    good = [16, 16, 16, 16, None, 16, 16, None, 16, 16, 16]
    for i in (0, 1, 2, 3, 5, 6, 8, 9, 10):
        with pytest.raises(dfgpu.DfgpuError) as error:
            cache.cache_sdpa(sdpa_params(), good[:i] + [None] + good[i + 1:], 256)
        assert error.value.code == 1 and f"port {i}" in str(error.value)
    with pytest.raises(dfgpu.DfgpuError):
        cache.cache_sdpa(sdpa_params(), [16, 24] + good[2:], 256)
    assert cache.query("cache_sdpa", sdpa_params()).scratch_bytes > 0
    with pytest.raises(dfgpu.DfgpuError) as error:
        cache.cache_sdpa(sdpa_params(), good, None)
    assert "scratch" in str(error.value)


def pages_params(op, **change):
    p = cache.CachePagesParams(op=cache.PAGE_OPS.get(op, 9), block=16)
    p.page_table, p.lengths, p.refs = tensor(I32, [3, 1, 4, 1]), tensor(I32, [3, 1, 1, 1]), tensor(I32, [20])
    if op != "compact":
        p.list = tensor(I32, [3, 2 if op in ("fork", "copy") else 1])
    pools = change.pop("pools", [])
    p.pool_count = len(pools)
    for i, pool in enumerate(pools):
        p.pools[i] = pool
    for key, value in change.items():
        setattr(p, key, value)
    return p


def test_pages_refusals():
    pool = tensor(U8, [2, 20, 64])
    for op in cache.PAGE_OPS:
        assert cache.query("cache_pages", pages_params(op)).launches == 1
    assert cache.query("cache_pages", pages_params("fork", pools=[pool])).launches == 2
    refused(1, "cache_pages", pages_params("nothing"))
    refused(1, "cache_pages", pages_params("free", pools=[pool]), "no pools")
    refused(1, "cache_pages", pages_params("reserve", pools=[pool]), "no pools")
    refused(15, "cache_pages", pages_params("fork", list=tensor(I32, [3, 1])))
    refused(15, "cache_pages", pages_params("reserve", list=tensor(I32, [4, 1])))
    refused(1, "cache_pages", pages_params("compact", list=tensor(I32, [4, 1])))
    refused(15, "cache_pages", pages_params("fork", block=0))
    refused(20, "cache_pages", pages_params("fork", block=1 << 30))
    refused(15, "cache_pages", pages_params("fork", page_table=tensor(I32, [3, 1, 4, 1], [5, 5, 1, 1])))
    refused(15, "cache_pages", pages_params("fork", refs=tensor(I64, [20])))
    refused(15, "cache_pages", pages_params("fork", pools=[tensor(U8, [2, 19, 64])]))
    refused(20, "cache_pages", pages_params("fork", pools=[tensor(dfgpu.FP4, [2, 20, 64])]))
    refused(14, "cache_pages", pages_params("fork", pools=[tensor(U8, [2, 20, 64], [1280, 63, 1])]), "overlap")
    refused(14, "cache_pages", pages_params("fork", pools=[tensor(U8, [2, 20, 64], [1279, 64, 1])]), "overlap")
    refused(14, "cache_pages", pages_params("fork", pools=[tensor(U8, [2, 20, 64], [0, 64, 1])]), "overlap")
    refused(14, "cache_pages", pages_params("fork", pools=[tensor(U8, [2, 20, 64], [64, 64, 1])]), "overlap")
    assert cache.query("cache_pages", pages_params("fork", pools=[tensor(U8, [2, 20, 64], [64, 128, 1])])).launches == 2   # pages outside, layers inside
    refused(1, "cache_pages", pages_params("fork", pool_count=9))
    good = [16] * 8
    for i in range(7):
        with pytest.raises(dfgpu.DfgpuError) as error:
            cache.cache_pages(pages_params("fork"), good[:i] + [None] + good[i + 1:], 256)
        assert error.value.code == 1
    with pytest.raises(dfgpu.DfgpuError) as error:
        cache.cache_pages(pages_params("fork"), good, None)
    assert "scratch" in str(error.value)
    with pytest.raises(dfgpu.DfgpuError) as error:
        cache.cache_pages(pages_params("fork", pools=[pool, pool]), good + [16, 16], 256)
    assert "the same" in str(error.value)


def python_frequencies(rotary, base, scaling, factor, original, low, high):
    """The same formulas, in Python floats."""
    if scaling == "base":
        base *= factor ** (rotary / (rotary - 2))
    f = [base ** (-2.0 * i / rotary) for i in range(rotary // 2)]
    if scaling == "linear":
        return [x / factor for x in f]
    if scaling == "ramp":
        at = [rotary * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (high, low)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary - 1)
        shares = [min(max((i - lo) / (hi - lo if hi > lo else 0.001), 0.0), 1.0) for i in range(rotary // 2)]
        return [x / factor * s + x * (1 - s) for x, s in zip(f, shares)]
    if scaling == "bands":
        shares = [min(max((original * x / (2 * math.pi) - low) / (high - low), 0.0), 1.0) for x in f]
        return [x / factor * (1 - s) + x * s for x, s in zip(f, shares)]
    return f


@pytest.mark.parametrize("scaling", list(cache.ROPE_SCALINGS))
@pytest.mark.parametrize("rotary,base,factor", [(128, 10000.0, 4.0), (64, 500000.0, 8.0), (4, 10000.0, 1.0), (250, 1e6, 32.0)])
def test_rope_frequencies(scaling, rotary, base, factor):
    got, magnitude = cache.rope_frequencies(rotary, base, scaling, factor, 8192.0, 1.0, 4.0 if scaling == "bands" else 32.0)
    want = python_frequencies(rotary, base, scaling, factor, 8192.0, 1.0, 4.0 if scaling == "bands" else 32.0)
    assert len(got) == rotary // 2
    assert np.allclose(got, want, rtol=2.0 ** -23, atol=0)   # one rounding to f32 (2^-24), and the last bits of pow and log
    assert magnitude == pytest.approx(0.1 * math.log(factor) + 1.0 if scaling == "ramp" else 1.0, rel=1e-6)
    if scaling == "base" and rotary > 2:
        assert got[0] == 1.0 and got[-1] == pytest.approx(base ** (-(rotary - 2) / rotary) / factor, rel=1e-6)


def test_rope_frequencies_refusals():
    for bad in (dict(rotary=7), dict(rotary=0), dict(rotary=8, base=1.0), dict(rotary=8, scaling="linear", factor=0.5), dict(rotary=8, scaling="ramp", factor=2.0),
                dict(rotary=8, scaling="bands", factor=2.0, original=100.0, low=4.0, high=4.0), dict(rotary=2, scaling="base", factor=2.0), dict(rotary=8, base=math.nan)):
        with pytest.raises(dfgpu.DfgpuError):
            cache.rope_frequencies(**bad)
    with pytest.raises(ValueError):
        cache.rope_frequencies(8, scaling="other")


def test_the_restatement_encodes_as_a_search_does():
    values = np.concatenate([np.linspace(-500, 500, 4001), 2.0 ** np.arange(-14, 10), ref.E4M3[np.isfinite(ref.E4M3)], [2.0 ** -10, -(2.0 ** -10), 3 * 2.0 ** -10, 0.0, -0.0, np.inf, -np.inf, np.nan]])
    codes = ref.encode_e4m3(values)
    finite = np.flatnonzero(np.isfinite(ref.E4M3))
    for value, code in zip(values, codes):
        if np.isnan(value):
            assert code == 0x7F
            continue
        distance = np.abs(ref.E4M3[finite] - np.clip(value, -448, 448))
        assert abs(ref.E4M3[code] - np.clip(value, -448, 448)) == distance.min()
        ties = finite[distance == distance.min()]
        assert len({abs(ref.E4M3[c]) for c in ties}) == 1 or code % 2 == 0
    assert ref.encode_e4m3(-0.0) == 0x80 and ref.encode_e4m3(-(2.0 ** -11)) == 0
    assert [ref.scale_code(x) for x in (0.0, 448.0, 448.0001, 896.0, 1.0, np.inf, np.nan)] == [0, 127, 128, 128, 119, 254, 255]


def test_outputs_that_overlap_are_refused():
    refused(14, "rope", rope_params(y=tensor(BF16, [2, 4, 3, 64], [768, 0, 64, 1])), "overlaps")
    assert cache.query("rope", rope_params(x=tensor(BF16, [2, 4, 3, 64], [768, 0, 64, 1]))).launches == 1   # (a broadcast input is none)
    both = rope_params(x2=tensor(BF16, [2, 4, 3, 64]), y2=tensor(BF16, [2, 4, 3, 64]))
    for pointers in ([16, 32, 16, 16, 64, 32], [16, 32, 16, 16, 64, 16], [16, 64, 16, 16, 64, 48]):
        with pytest.raises(dfgpu.DfgpuError) as error:
            cache.rope(both, pointers)
        assert error.value.code == 1 and "other" in str(error.value)
    refused(14, "cache_sdpa", sdpa_params(stats=tensor(F32, [2, 8, 3, 1], [24, 0, 1, 1])), "overlaps")


def test_containers_without_a_stride_are_refused():
    refused(14, "cache_sdpa", sdpa_params(k=tensor(E4M3, [9, 4, 32, 64], [2048, 0, 64, 1])), "positive")
    refused(14, "cache_sdpa", sdpa_params(v=tensor(E4M3, [9, 4, 32, 64], [8192, 2048, 0, 1])), "positive")


def test_pieces_of_long_sequences():
    """Few query blocks before many keys: pieces, a merge and scratch for their results; as many blocks as SMs: none."""
    long = dict(kernel=cache.SDPA_UMMA, page_table_k=tensor(I32, [2, 1, 400, 1]), page_table_v=tensor(I32, [2, 1, 400, 1]))
    short, cut = (cache.query("cache_sdpa", sdpa_params(**{**long, "s_kv": s_kv})) for s_kv in (500, 12800))
    assert (short.launches, cut.launches) == (3, 4) and cut.scratch_bytes > short.scratch_bytes
    rows = [2, 8, 2000, 64]
    many = cache.query("cache_sdpa", sdpa_params(**{**long, "s_kv": 12800, "q": tensor(BF16, rows), "o": tensor(BF16, rows)}))
    assert many.launches == 3


def test_reserve_refuses_tables_whose_demand_could_pass_32_bits():
    def table(b, slots):
        return dict(page_table=tensor(I32, [b, 1, slots, 1]), lengths=tensor(I32, [b, 1, 1, 1]), list=tensor(I32, [b, 1]))
    refused(20, "cache_pages", pages_params("reserve", **table(1 << 14, 1 << 17)), "2^31")
    refused(20, "cache_pages", pages_params("reserve", **table(1 << 27, 16)), "2^31")
    assert cache.query("cache_pages", pages_params("reserve", **table((1 << 14) - 1, 1 << 17))).launches == 1
    assert cache.query("cache_pages", pages_params("free", **table(1 << 14, 1 << 17))).launches == 1   # (counts pages, of which there are fewer than 2^28)


def test_attention_does_not_write_over_its_queries():
    for kernel in (cache.SDPA_AUTO, cache.SDPA_STREAM, cache.SDPA_UMMA):
        with pytest.raises(dfgpu.DfgpuError) as error:
            cache.cache_sdpa(sdpa_params(kernel=kernel), [4096, 16, 16, 4096, None, 16, 16, None, 16, 16, 16], 256)
        assert error.value.code == 1 and "O is Q" in str(error.value)


def test_append_does_not_write_lengths_over_the_counts_it_reads():
    vector = tensor(I32, [2, 1, 1, 1])
    with pytest.raises(dfgpu.DfgpuError) as error:
        cache.cache_append(append_params(added=vector, lengths_out=vector), [16, 16, 16, 32, 16, 32, 16, 16, 64, 128, 128])
    assert error.value.code == 1 and "lengths_out is added" in str(error.value)
