"""The C ABI of the operators of a decoder's step without a GPU: layouts, refusals before any CUDA call, and the restatement's own gradient."""
import ctypes as C
import re
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import decoder_reference as ref
from deepforge_b200 import decoder, dfgpu
from deepforge_b200.decoder import I8
from deepforge_b200.dfgpu import BF16, F16, F32, FP4, I32, I64, U8, tensor

ROOT = Path(__file__).resolve().parent.parent


def test_exports_and_layouts(tmp_path):
    text = (ROOT / "include" / "dfgpu_decoder.h").read_text()
    code = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = sorted(set(re.findall(r"\b(dfgpu_[a-z0-9_]+)\s*\(", code)))
    assert sorted(decoder.EXPORTS) == names
    lib = dfgpu.load()
    for name in names:
        assert hasattr(lib, name), name
    assert lib.dfgpu_decoder_abi_version() == 1
    if not shutil.which("gcc"):
        pytest.skip("no C compiler")
    structs = {"head_norm_params": decoder.HeadNormParams, "head_norm_grad_params": decoder.HeadNormGradParams, "token_quantize_params": decoder.TokenQuantizeParams,
               "matmul_int8_params": decoder.MatmulInt8Params, "beam_select_params": decoder.BeamSelectParams, "beam_reorder_params": decoder.BeamReorderParams}
    source = tmp_path / "sizes.c"
    source.write_text('#include <stdio.h>\n#include "dfgpu_decoder.h"\nint main(void){' + "".join(f'printf("%zu\\n", sizeof(dfgpu_{n}));' for n in structs) + "return 0;}\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(source), "-o", str(tmp_path / "sizes")], check=True)
    sizes = subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()
    assert [int(v) for v in sizes] == [C.sizeof(s) for s in structs.values()]


def refused(code, name, params, text=""):
    with pytest.raises(dfgpu.DfgpuError) as error:
        decoder.query(name, params)
    assert error.value.code == code and text in str(error.value), error.value


def call_refused(code, call, params, pointers, text="", **more):
    with pytest.raises(dfgpu.DfgpuError) as error:
        call(params, pointers, **more)
    assert error.value.code == code and text in str(error.value), error.value


def changed(p, change):
    for key, value in change.items():
        setattr(p, key, value)
    return p


# ---- head norms ------------------------------------------------------------------------------------

def norm_params(**change):
    p = decoder.HeadNormParams(epsilon=1e-6)
    p.x = p.y = tensor(BF16, [2, 4, 3, 64])
    p.gain = tensor(F32, [1, 1, 1, 64])
    p.positions, p.frequencies = tensor(I32, [2, 1, 3, 1]), tensor(F32, [1, 1, 1, 32])
    return changed(p, change)


def grad_params(**change):
    p = decoder.HeadNormGradParams(epsilon=1e-6)
    p.x = p.dy = p.dx = tensor(BF16, [2, 4, 3, 64])
    p.gain = p.dgain = tensor(F32, [1, 4, 1, 64])
    return changed(p, change)


def test_head_norm_refusals():
    info = decoder.query("head_norm", norm_params())
    assert (info.kernel, info.launches, info.scratch_bytes) == (decoder.HEAD_NORM_VECTOR, 1, 0)
    assert decoder.query("head_norm", norm_params(frequencies=tensor(F32, [1, 1, 1, 5]))).kernel == decoder.HEAD_NORM_SCALAR
    assert decoder.query("head_norm", norm_params(positions=dfgpu.ABSENT, frequencies=dfgpu.ABSENT, gain=dfgpu.ABSENT)).launches == 1
    refused(15, "head_norm", norm_params(frequencies=tensor(F32, [1, 1, 1, 33])))
    refused(20, "head_norm", norm_params(frequencies=tensor(F16, [1, 1, 1, 32])))
    refused(1, "head_norm", norm_params(positions=dfgpu.ABSENT), "together")
    refused(15, "head_norm", norm_params(positions=tensor(I32, [3, 1, 3, 1])))
    refused(20, "head_norm", norm_params(positions=tensor(F32, [1, 1, 3, 1])))
    refused(20, "head_norm", norm_params(y=tensor(F32, [2, 4, 3, 64])))
    refused(15, "head_norm", norm_params(y=tensor(BF16, [2, 4, 4, 64])))
    refused(14, "head_norm", norm_params(x=tensor(BF16, [2, 4, 3, 64], [1536, 384, 128, 2])))
    refused(14, "head_norm", norm_params(y=tensor(BF16, [2, 4, 3, 64], [0, 192, 64, 1])), "overlaps itself")
    refused(15, "head_norm", norm_params(gain=tensor(F32, [1, 3, 1, 64])))
    refused(15, "head_norm", norm_params(gain=tensor(F32, [1, 1, 1, 32])))
    refused(20, "head_norm", norm_params(gain=tensor(I32, [1, 1, 1, 64])))
    refused(1, "head_norm", norm_params(gain2=tensor(F32, [1, 1, 1, 64])), "X2")
    refused(15, "head_norm", norm_params(x2=tensor(BF16, [2, 1, 3, 64])))
    refused(15, "head_norm", norm_params(x2=tensor(BF16, [2, 1, 4, 64]), y2=tensor(BF16, [2, 1, 4, 64])))
    refused(20, "head_norm", norm_params(x2=tensor(F16, [2, 1, 3, 64]), y2=tensor(F16, [2, 1, 3, 64])))
    refused(20, "head_norm", norm_params(x=tensor(U8, [2, 4, 3, 64]), y=tensor(U8, [2, 4, 3, 64])))
    refused(8, "head_norm", norm_params(epsilon=-1.0))
    refused(8, "head_norm", norm_params(epsilon=float("nan")))
    refused(1, "head_norm", norm_params(kernel=7))
    refused(20, "head_norm", norm_params(kernel=decoder.HEAD_NORM_VECTOR, frequencies=tensor(F32, [1, 1, 1, 5])))
    wide = tensor(BF16, [1, 1, 1, 1032])
    refused(20, "head_norm", norm_params(x=wide, y=wide, gain=dfgpu.ABSENT, positions=dfgpu.ABSENT, frequencies=dfgpu.ABSENT))
    assert decoder.query("head_norm", norm_params(positions=tensor(I64, [1, 1, 3, 1]))).launches == 1
    for pointers in ([None, 16, 16, 16, 16], [16, 1 << 20, None, 16, 16], [16, 1 << 20, 16, 16, None], [17, 1 << 20, 16, 16, 16], [16, 1 << 20, 18, 16, 16], [16, 1 << 20, 16, 18, 16]):
        call_refused(1, decoder.head_norm, norm_params(), pointers)
    call_refused(14, decoder.head_norm, norm_params(y=tensor(BF16, [2, 4, 3, 64], [768, 64, 256, 1])), [16, 16, 1 << 20, 1 << 20, 1 << 20])   # in place with other strides
    call_refused(1, decoder.head_norm, norm_params(), [1024, 1040, 1 << 20, 1 << 20, 1 << 20], "overlaps")
    two = norm_params(x2=tensor(BF16, [2, 1, 3, 64]), y2=tensor(BF16, [2, 1, 3, 64]))
    call_refused(1, decoder.head_norm, two, [1024, 1024, 1 << 20, 1 << 20, 1 << 20, 1 << 22, 1024], "other")


def test_head_norm_gradient_refusals():
    info = decoder.query("head_norm_grad", grad_params())
    assert (info.kernel, info.launches) == (decoder.HEAD_NORM_VECTOR, 2) and info.scratch_bytes > 0 and info.scratch_bytes % (4 * 4 * 64) == 0
    assert decoder.query("head_norm_grad", grad_params(dgain=dfgpu.ABSENT)).scratch_bytes == 0
    assert decoder.query("head_norm_grad", grad_params(dgain=dfgpu.ABSENT)).launches == 1
    assert decoder.query("head_norm_grad", grad_params(gain=dfgpu.ABSENT)).launches == 2
    refused(15, "head_norm_grad", grad_params(dgain=tensor(F32, [1, 1, 1, 64])), "gradient")
    refused(14, "head_norm_grad", grad_params(dgain=tensor(F32, [1, 4, 1, 64], [256, 0, 64, 1])))
    refused(15, "head_norm_grad", grad_params(dy=tensor(BF16, [2, 4, 3, 32])))
    refused(20, "head_norm_grad", grad_params(dx=tensor(F32, [2, 4, 3, 64])))
    refused(14, "head_norm_grad", grad_params(dx=tensor(BF16, [2, 4, 3, 64], [768, 0, 64, 1])))
    far = [1 << 20, 2 << 20, 3 << 20, 4 << 20, 5 << 20]
    call_refused(1, decoder.head_norm_grad, grad_params(), far, "scratch")
    call_refused(1, decoder.head_norm_grad, grad_params(), far[:4] + [None], "null", scratch=16)
    call_refused(1, decoder.head_norm_grad, grad_params(), far[:4] + [far[3]], "overlaps", scratch=16)
    call_refused(1, decoder.head_norm_grad, grad_params(), far[:4] + [far[0] + 16], "overlaps", scratch=16)
    call_refused(1, decoder.head_norm_grad, grad_params(), [far[0], far[1], far[1] + 128, *far[3:]], "overlaps", scratch=16)


def test_the_restated_gradient_against_differences():
    rng = np.random.default_rng(1)
    x, dy = rng.standard_normal((2, 3, 5, 12)), rng.standard_normal((2, 3, 5, 12))
    positions, frequencies = rng.integers(0, 50, (2, 5)), 10.0 ** -np.arange(4)
    for heads in (1, 3):
        gain = 1 + 0.3 * rng.standard_normal((heads, 12))
        value = lambda x, gain: (ref.head_norm(x, gain, positions, frequencies, True, 1.25, 1e-3) * dy).sum()  # noqa: E731
        dx, dgain = ref.head_norm_grad(x, dy, gain, positions, frequencies, True, 1.25, 1e-3)
        ex, eg, h = rng.standard_normal(x.shape), rng.standard_normal(gain.shape), 1e-5
        assert abs((value(x + h * ex, gain) - value(x - h * ex, gain)) / (2 * h) - (dx * ex).sum()) < 1e-7 * np.abs(dx * ex).sum()
        assert abs((value(x, gain + h * eg) - value(x, gain - h * eg)) / (2 * h) - (dgain * eg).sum()) < 1e-7 * np.abs(dgain * eg).sum()


# ---- 8-bit integers ----------------------------------------------------------------------------------

def quantize_params(**change):
    p = decoder.TokenQuantizeParams()
    p.x, p.y, p.scale = tensor(BF16, [5, 64]), tensor(I8, [5, 64]), tensor(F32, [5, 1])
    return changed(p, change)


def test_token_quantize_refusals():
    info = decoder.query("token_quantize", quantize_params())
    assert (info.kernel, info.launches, info.scratch_bytes) == (decoder.TOKEN_QUANTIZE_VECTOR, 1, 0)
    assert decoder.query("token_quantize", quantize_params(x=tensor(BF16, [5, 64], [65, 1]))).kernel == decoder.TOKEN_QUANTIZE_SCALAR
    assert decoder.query("token_quantize", quantize_params(kernel=decoder.TOKEN_QUANTIZE_SCALAR)).kernel == decoder.TOKEN_QUANTIZE_SCALAR
    refused(20, "token_quantize", quantize_params(x=tensor(I32, [5, 64])))
    refused(20, "token_quantize", quantize_params(y=tensor(U8, [5, 64])))
    refused(20, "token_quantize", quantize_params(scale=tensor(F16, [5, 1])))
    refused(15, "token_quantize", quantize_params(y=tensor(I8, [5, 63])))
    refused(15, "token_quantize", quantize_params(scale=tensor(F32, [5, 2])))
    refused(15, "token_quantize", quantize_params(scale=tensor(F32, [5])))
    refused(14, "token_quantize", quantize_params(x=tensor(BF16, [5, 64], [128, 2])))
    refused(14, "token_quantize", quantize_params(y=tensor(I8, [5, 64], [0, 1])))
    refused(1, "token_quantize", quantize_params(kernel=3))
    refused(20, "token_quantize", quantize_params(kernel=decoder.TOKEN_QUANTIZE_VECTOR, x=tensor(BF16, [5, 64], [65, 1])))
    for pointers, text in (([None, 16, 16], "null"), ([17, 4096, 8192], "aligned"), ([16, 4096, 8193], "aligned"), ([4096, 4096, 16], "overlaps"), ([4096, 65536, 65600], "overlaps")):
        call_refused(1, decoder.token_quantize, quantize_params(), pointers, text)
    call_refused(1, decoder.token_quantize, quantize_params(kernel=decoder.TOKEN_QUANTIZE_VECTOR), [4098, 65536, 1 << 20], "boundary")


def int8_params(m=8, n=32, k=64, dtype=BF16, **change):
    p = decoder.MatmulInt8Params()
    p.a, p.b, p.c = tensor(I8, [m, k]), tensor(I8, [k, n], [1, k]), tensor(dtype, [m, n])
    p.a_scale, p.b_scale = tensor(F32, [m, 1]), tensor(F32, [1, n])
    return changed(p, change)


def test_matmul_int8_refusals():
    info = decoder.query("matmul_int8", int8_params(m=32))
    assert (info.kernel, info.launches, info.scratch_bytes) == (decoder.MATMUL_INT8_UMMA, 1, 0)
    few = decoder.MATMUL_INT8_FEW
    for m, n, k, kernel in ((1, 32000, 4096, few), (8, 4096, 16384, few), (9, 4096, 4096, decoder.MATMUL_INT8_UMMA), (16, 1024, 1024, few), (17, 64, 64, decoder.MATMUL_INT8_UMMA)):
        assert decoder.query("matmul_int8", int8_params(m=m, n=n, k=k)).kernel == kernel
    assert decoder.query("matmul_int8", int8_params(c=tensor(BF16, [8, 32], [1, 8]), bias=tensor(F32, [1, 32], [64, 2]))).kernel == few   # any C and bias
    for params in (int8_params(m=17, kernel=few), int8_params(k=65, kernel=few), int8_params(b=tensor(I8, [64, 32]), kernel=few)):
        refused(20, "matmul_int8", params, "few tokens")
    assert decoder.query("matmul_int8", int8_params(k=65)).kernel == decoder.MATMUL_INT8_CORES
    assert decoder.query("matmul_int8", int8_params(b=tensor(I8, [64, 32]))).kernel == decoder.MATMUL_INT8_UMMA
    assert decoder.query("matmul_int8", int8_params(a=tensor(I8, [8, 64], [1, 8]))).kernel == decoder.MATMUL_INT8_CORES
    assert decoder.query("matmul_int8", int8_params(m=32, a_scale=tensor(F32, [1, 1]), b_scale=tensor(F32, [1, 1]))).kernel == decoder.MATMUL_INT8_UMMA
    refused(20, "matmul_int8", int8_params(a=tensor(U8, [8, 64])))
    refused(20, "matmul_int8", int8_params(dtype=I32))
    refused(15, "matmul_int8", int8_params(b=tensor(I8, [63, 32])))
    refused(15, "matmul_int8", int8_params(a_scale=tensor(F32, [7, 1])))
    refused(15, "matmul_int8", int8_params(b_scale=tensor(F32, [8, 32])))
    refused(20, "matmul_int8", int8_params(b_scale=tensor(F16, [1, 32])))
    refused(15, "matmul_int8", int8_params(bias=tensor(F32, [1, 1])))
    refused(20, "matmul_int8", int8_params(bias=tensor(I32, [1, 32])))
    refused(14, "matmul_int8", int8_params(c=tensor(BF16, [8, 32], [0, 1])))
    refused(20, "matmul_int8", int8_params(k=131072), "32 bits")
    assert decoder.query("matmul_int8", int8_params(k=131071)).launches == 1
    refused(1, "matmul_int8", int8_params(kernel=4))
    refused(20, "matmul_int8", int8_params(kernel=decoder.MATMUL_INT8_UMMA, k=65))

    def batched(b_batch, strides=None, **change):
        p = decoder.MatmulInt8Params()
        p.a, p.b, p.c = tensor(I8, [3, 8, 64], strides), tensor(I8, [b_batch, 64, 32], [64 * 32, 1, 64]), tensor(BF16, [3, 8, 32])
        p.a_scale, p.b_scale = tensor(F32, [3, 8, 1]), tensor(F32, [1, 1, 32])
        return changed(p, change)
    assert decoder.query("matmul_int8", batched(1)).kernel == decoder.MATMUL_INT8_UMMA                               # rows lie evenly: one matrix
    assert decoder.query("matmul_int8", batched(1, [1024, 64, 1])).kernel == decoder.MATMUL_INT8_CORES
    assert decoder.query("matmul_int8", batched(3)).kernel == decoder.MATMUL_INT8_CORES
    assert decoder.query("matmul_int8", batched(1, a_scale=tensor(F32, [3, 1, 1]))).kernel == decoder.MATMUL_INT8_CORES
    refused(15, "matmul_int8", batched(2))
    many = decoder.MatmulInt8Params()                                                                                                   # a matrix for each of 65536
    many.a, many.b, many.c = tensor(I8, [65536, 1, 64]), tensor(I8, [65536, 64, 2]), tensor(BF16, [65536, 1, 2])
    many.a_scale, many.b_scale = tensor(F32, [65536, 1, 1]), tensor(F32, [1, 1, 2])
    refused(20, "matmul_int8", many, "65535")
    far = [(i + 1) << 20 for i in range(5)]
    call_refused(1, decoder.matmul_int8, int8_params(), [*far[:4], None], "null")
    call_refused(1, decoder.matmul_int8, int8_params(bias=tensor(F32, [1, 32])), far, "null")
    call_refused(1, decoder.matmul_int8, int8_params(), [far[0], far[1], far[2] + 1, *far[3:]], "aligned")
    call_refused(1, decoder.matmul_int8, int8_params(), [far[0], far[1], far[0] + 64, *far[3:]], "overlaps")
    call_refused(1, decoder.matmul_int8, int8_params(kernel=decoder.MATMUL_INT8_UMMA), [far[0] + 1, *far[1:]], "boundaries")
    call_refused(1, decoder.matmul_int8, int8_params(kernel=few), [far[0], far[1] + 8, *far[2:]], "boundaries")


# ---- beam search --------------------------------------------------------------------------------------

def select_params(b=2, w=4, v=100, dtype=BF16, **change):
    p = decoder.BeamSelectParams()
    p.logits = tensor(dtype, [b, w, v])
    p.scores = p.scores_out = tensor(F32, [b, w])
    p.tokens = p.parents = tensor(I32, [b, w])
    return changed(p, change)


def test_beam_select_refusals():
    info = decoder.query("beam_select", select_params())
    assert info.launches == 2 and info.scratch_bytes == 2 * 4 * 1 * (32 + 8 * 4)
    ints = tensor(I32, [2, 4])
    assert decoder.query("beam_select", select_params(finished=ints, lengths=ints, finished_out=ints, lengths_out=ints, forks=tensor(I32, [8, 2]))).launches == 2
    refused(15, "beam_select", select_params(logits=tensor(BF16, [2, 4])))
    refused(20, "beam_select", select_params(dtype=I32))
    refused(14, "beam_select", select_params(logits=tensor(BF16, [2, 4, 100], [800, 200, 2])))
    refused(20, "beam_select", select_params(w=33))
    refused(20, "beam_select", select_params(v=1 << 26))
    refused(15, "beam_select", select_params(scores=tensor(F32, [2, 3])))
    refused(20, "beam_select", select_params(scores=tensor(F16, [2, 4])))
    refused(20, "beam_select", select_params(tokens=tensor(I64, [2, 4])))
    refused(15, "beam_select", select_params(parents=dfgpu.ABSENT))
    refused(14, "beam_select", select_params(parents=tensor(I32, [2, 4], [0, 1])))
    refused(1, "beam_select", select_params(lengths_out=ints), "without lengths")
    refused(8, "beam_select", select_params(lengths=ints, length_penalty=float("inf")))
    refused(8, "beam_select", select_params(finished=ints, pad=100))
    refused(8, "beam_select", select_params(finished=ints, pad=-1))
    refused(15, "beam_select", select_params(forks=tensor(I32, [7, 2])))
    refused(14, "beam_select", select_params(forks=tensor(I32, [8, 2], [4, 1])))
    refused(8, "beam_select", select_params(forks=tensor(I32, [8, 2]), source_base=-1))
    refused(8, "beam_select", select_params(forks=tensor(I32, [8, 2]), target_base=0x7FFFFFFF))
    far = [(i + 1) << 20 for i in range(10)]
    pointers = [far[0], far[1], None, None, far[4], far[5], far[6]]
    call_refused(1, decoder.beam_select, select_params(), pointers, "scratch")
    call_refused(1, decoder.beam_select, select_params(), pointers, "16-byte", scratch=8)
    call_refused(1, decoder.beam_select, select_params(), pointers[:6] + [None], "null", scratch=16)
    call_refused(1, decoder.beam_select, select_params(), pointers[:6] + [far[5]], "overlaps", scratch=16)
    call_refused(1, decoder.beam_select, select_params(), pointers[:4] + [far[0] + 32, *pointers[5:]], "overlaps", scratch=16)
    call_refused(1, decoder.beam_select, select_params(), [far[0] + 1, *pointers[1:]], "aligned", scratch=16)
    call_refused(14, decoder.beam_select, select_params(scores_out=tensor(F32, [2, 4], [1, 2])), [*pointers[:4], far[1], *pointers[5:]], "in place", scratch=16)


def reorder_params(count=1, dims=(3, 2, 4, 10), dtype=BF16, **change):
    p = decoder.BeamReorderParams(count=count)
    p.parents = tensor(I32, [2, 4])
    for i in range(min(count, decoder.MAX_STATES)):
        p.source[i] = p.target[i] = tensor(dtype, list(dims))
    return changed(p, change)


def test_beam_reorder_refusals():
    info = decoder.query("beam_reorder", reorder_params())
    assert (info.launches, info.scratch_bytes) == (1, 0)
    refused(1, "beam_reorder", reorder_params(0))
    refused(1, "beam_reorder", reorder_params(9))
    refused(15, "beam_reorder", reorder_params(dims=(3, 4, 2, 10)))
    refused(15, "beam_reorder", reorder_params(dims=(3, 2, 4)))
    refused(20, "beam_reorder", reorder_params(dtype=FP4))
    refused(20, "beam_reorder", reorder_params(parents=tensor(F32, [2, 4])))
    p = reorder_params()
    p.target[0] = tensor(F16, [3, 2, 4, 10])
    refused(20, "beam_reorder", p, "type")
    p.target[0] = tensor(BF16, [3, 2, 4, 10], [80, 40, 0, 1])
    refused(14, "beam_reorder", p, "overlaps itself")
    p.target[0] = tensor(BF16, [3, 2, 4, 10], [160, 80, 20, 2])
    refused(14, "beam_reorder", p, "contiguous")
    refused(20, "beam_reorder", reorder_params(dims=(1 << 20, 2, 4, 1 << 20)))
    far = [(i + 1) << 20 for i in range(5)]
    call_refused(1, decoder.beam_reorder, reorder_params(), [None, *far[:2]])
    call_refused(1, decoder.beam_reorder, reorder_params(), [far[0], far[1], None], "null")
    call_refused(1, decoder.beam_reorder, reorder_params(), [far[0], far[1], far[1]], "overlaps")
    call_refused(1, decoder.beam_reorder, reorder_params(2), [far[0], far[1], far[2], far[3], far[1] + 32], "overlaps")
    call_refused(1, decoder.beam_reorder, reorder_params(2), [far[0], far[1], far[2], far[3], far[2]], "overlaps")
    call_refused(1, decoder.beam_reorder, reorder_params(), [far[0], far[1], far[0] - 16], "parents")


# ---- barriers of clusters ---------------------------------------------------------------------------------

def test_barriers_of_clusters_come_behind_a_converged_warp():
    """`aligned` wants all threads of a warp at the barrier together, which a branch or loop before it does not see to: where such code stands before it, the barrier is the helper's, which has a __syncwarp()."""
    sources = ROOT / "deepforge_b200" / "csrc"
    helper = re.search(r"void cluster_barrier\(\) \{(.*?)\n\}", (sources / "common.cuh").read_text(), re.S)
    assert helper and re.search(r"__syncwarp\(\);.*barrier\.cluster\.arrive\.release\.aligned.*barrier\.cluster\.wait\.acquire\.aligned", helper.group(1), re.S)
    head_norm, pages = ((sources / name).read_text() for name in ("head_norm.cu", "cache_pages.cu"))
    assert "barrier.cluster" not in head_norm and head_norm.count("cluster_barrier();") == 2
    matmul = (sources / "umma_matmul.cu").read_text()
    helpers = re.findall(r"void (\w+)\(\) \{\n    __syncwarp\(\);\n    asm volatile\(\"barrier\.cluster", matmul)
    assert helpers == ["cluster_arrive", "cluster_arrive_relaxed", "cluster_wait"] and matmul.count("barrier.cluster") == 3
    # (the pages' kernel: its first arrival and wait, before any branch, are its own)
    assert re.findall(r"void (\w+)\(\) \{[^}]*barrier\.cluster", pages) == ["cluster_arrive_first", "cluster_wait_first"] and pages.count("barrier.cluster") == 2


def test_beam_select_refuses_penalties_whose_powers_have_no_place():
    """Worths are scores over n^penalty in 64 bits, n up to 2^31 - 1: 2^(31 * 28) = 2^868 leaves room for f32 scores (2^-149 to 2^128) on either side of what 64 bits hold (2^-1022 to 2^1024)."""
    ints = tensor(I32, [2, 4])
    for penalty in (28.5, -28.5, 400.0, -400.0, 3e38, float("nan"), -float("inf")):
        refused(8, "beam_select", select_params(lengths=ints, length_penalty=penalty), "penalty")
        assert decoder.query("beam_select", select_params(length_penalty=penalty)).launches == 2   # (read only with lengths)
    for penalty in (28.0, -28.0, 0.0):
        assert decoder.query("beam_select", select_params(lengths=ints, length_penalty=penalty)).launches == 2
