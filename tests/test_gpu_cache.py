"""Rotary positions, the 8-bit paged cache and its pages on the GPU against the 64-bit restatement (cache_reference.py)."""
import numpy as np
import pytest

import cache_reference as ref
from deepforge_b200 import cache, dfgpu
from deepforge_b200.dfgpu import BF16, E4M3, E8M0, F16, F32, I32, I64, U8, contiguous_strides, tensor

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TORCH = {BF16: torch.bfloat16, F16: torch.float16, F32: torch.float32}


def half_step(dtype):
    return torch.finfo(TORCH[dtype]).eps / 2


def describe(t, code, dims=None):
    return tensor(code, list(dims or t.shape), list(t.stride()) if dims is None else contiguous_strides(dims))


def double(t):
    return t.double().cpu().numpy()


def randn(rng, shape, dtype, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape) * scale).to(TORCH[dtype]).cuda()


def ints(values, dtype=torch.int32):
    return torch.tensor(np.asarray(values), dtype=dtype, device="cuda")


# ---- rotary positions --------------------------------------------------------------------------

def run_rope(x, positions, frequencies, x2=None, interleaved=False, inverse=False, scale=1.0, in_place=False, kernel=0, dtype=BF16, stream=None, y=None):
    p = cache.RopeParams(interleaved=interleaved, inverse=inverse, scale=scale, kernel=kernel)
    y = x if in_place else torch.full_like(x, 7.0) if y is None else y
    p.x, p.y = describe(x, dtype), describe(y, dtype)
    y2 = None
    if x2 is not None:
        y2 = x2 if in_place else torch.full_like(x2, 7.0)
        p.x2, p.y2 = describe(x2, dtype), describe(y2, dtype)
    p.positions = tensor(I64 if positions.dtype == torch.int64 else I32, [positions.shape[0], 1, positions.shape[1], 1], [positions.stride(0), 1, positions.stride(1), 1])
    p.frequencies = tensor(F32, [1, 1, 1, len(frequencies)])
    cache.rope(p, [x.data_ptr(), y.data_ptr(), positions.data_ptr(), frequencies.data_ptr()] + ([x2.data_ptr(), y2.data_ptr()] if x2 is not None else []), stream=stream)
    return (y, y2) if x2 is not None else y


def check_rope(got, x, positions, frequencies, interleaved, inverse, scale, dtype):
    """The angle is off by pi 2^-25 after its reduction, sine and cosine by 2^-23 (two steps of f32 below one): 2.2e-7 of each of the two
    products, with three roundings of f32 (2^-24 each) 4e-7; 5e-7 of |x1| + |x2| bounds that. Then one rounding to the type, and for HALF its smallest step."""
    x64, at = double(x), positions.cpu().numpy()
    want = ref.rope(x64, np.broadcast_to(at, (x64.shape[0], at.shape[1])), frequencies.cpu().numpy(), interleaved, inverse, scale)
    size = ref.rope(np.abs(x64), np.zeros((x64.shape[0], at.shape[1])), frequencies.cpu().numpy(), interleaved, False, 1.0)
    half = len(frequencies)
    both = size.copy()
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    both[..., one] = both[..., two] = size[..., one] + size[..., two]
    bound = 5e-7 * both * abs(scale) + half_step(dtype) * np.abs(want) * 1.001 + (2.0 ** -25 if dtype == F16 else 0)
    bound[..., 2 * half:] = 0
    assert np.all(np.abs(double(got) - want) <= bound), np.max(np.abs(double(got) - want) - bound)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,h,h2,s,d,rotary", [(1, 1, 0, 1, 64, 64), (3, 5, 2, 17, 128, 128), (2, 4, 1, 9, 80, 40), (2, 3, 3, 33, 96, 96), (1, 2, 1, 5, 256, 64), (2, 1, 2, 7, 66, 10), (1, 1, 1, 3, 1024, 1024)])
def test_rope(interleaved, dtype, b, h, h2, s, d, rotary):
    rng = np.random.default_rng(b * 100 + d)
    x, x2 = randn(rng, (b, h, s, d), dtype), randn(rng, (b, h2, s, d), dtype) if h2 else None
    positions = ints(rng.integers(0, 2 ** 20, (b, s)))
    frequencies = torch.tensor(cache.rope_frequencies(rotary)[0], device="cuda")
    for inverse, scale in ((False, 1.0), (True, 1.25)):
        got = run_rope(x, positions, frequencies, x2, interleaved, inverse, scale, dtype=dtype)
        for y, source in zip(got if h2 else [got], (x, x2)):
            check_rope(y, source, positions, frequencies, interleaved, inverse, scale, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rope_strides_alignment_and_places(dtype):
    rng = np.random.default_rng(3)
    frequencies = torch.tensor(cache.rope_frequencies(32)[0], device="cuda")
    b, h, s, d = 2, 3, 21, 64
    positions = ints(np.arange(s)[None] * 1000 - 5000, torch.int64)    # one row for all sequences, INT64, negative too
    base = randn(rng, (b, s, h, d + 8), dtype)
    x = base[..., :d].transpose(1, 2)                                   # token-major, rows apart
    check_rope(run_rope(x, positions, frequencies, dtype=dtype), x, positions, frequencies, False, False, 1.0, dtype)
    flat = randn(rng, (b * h * s * d + 1,), dtype)
    odd = flat[1:].view(b, h, s, d)                                     # off every vector boundary
    check_rope(run_rope(odd, positions, frequencies, dtype=dtype), odd, positions, frequencies, False, False, 1.0, dtype)
    want = run_rope(x, positions, frequencies, dtype=dtype)
    around = base.clone()
    got = run_rope(x, positions, frequencies, in_place=True, dtype=dtype)   # nothing but the turned rows changes
    assert torch.equal(got, want) and torch.equal(base[..., d:], around[..., d:])
    contiguous = want.contiguous()
    assert torch.equal(run_rope(contiguous, positions, frequencies, kernel=cache.ROPE_SCALAR, dtype=dtype), run_rope(contiguous, positions, frequencies, dtype=dtype))
    one = x[:1].expand(b, h, s, d)                                      # a broadcast input
    check_rope(run_rope(one, positions, frequencies, dtype=dtype, y=torch.empty(b, h, s, d, device="cuda", dtype=TORCH[dtype])), one, positions, frequencies, False, False, 1.0, dtype)


def test_rope_gradient_is_the_transposed_map():
    """<rope(x), g> = <x, rope'(g)>, and against differences: the map is linear, so a step along e changes y by rope(e)."""
    rng = np.random.default_rng(8)
    x, g, e = (randn(rng, (2, 3, 19, 64), F32) for _ in range(3))
    positions, frequencies = ints(rng.integers(0, 10 ** 6, (2, 19))), torch.tensor(cache.rope_frequencies(48, scaling="bands", factor=4.0, original=8192, low=1, high=4)[0], device="cuda")
    for interleaved in (False, True):
        forward = lambda t: run_rope(t, positions, frequencies, interleaved=interleaved, scale=1.5, dtype=F32)  # noqa: E731
        back = run_rope(g, positions, frequencies, interleaved=interleaved, inverse=True, scale=1.5, dtype=F32)
        left, right = (forward(x).double() * g.double()).sum(), (x.double() * back.double()).sum()
        size = (x.double().abs() * g.double().abs()).sum() * 3
        assert abs(left - right) <= 1e-6 * size
        difference = ((forward(x + e).double() - forward(x - e).double()) * g.double()).sum() / 2
        along = (e.double() * back.double()).sum()
        assert abs(difference - along) <= 4e-6 * (g.double().abs() * (x.double().abs() + e.double().abs())).sum()


# ---- appending -----------------------------------------------------------------------------------

def cache_of(rng, pages, hk, page, t, d, layout="heads"):
    """Random codes (no NaN) and scales; layout "tokens": token-major memory under the same logical dims."""
    codes = rng.integers(0, 256, (pages, hk, page, d)).astype(np.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x38
    dev = torch.from_numpy(codes).cuda()
    if layout == "tokens":
        dev = dev.transpose(1, 2).contiguous().transpose(1, 2)
    scale = torch.from_numpy(rng.integers(117, 125, (pages, hk, page // t, 1)).astype(np.uint8)).cuda()
    return dev, scale


def table_of(rng, b, slots, pages):
    return rng.permutation(pages)[: b * slots].reshape(b, slots).astype(np.int32)


def run_append(k, v, caches, scales, tables, lengths, added=None, dtype=BF16, kernel=0, lengths_out=None, stream=None):
    p = cache.CacheAppendParams(kernel=kernel)
    b = k.shape[0]
    p.k, p.v = describe(k, dtype), describe(v, dtype)
    p.k_cache, p.v_cache = (describe(c, E4M3) for c in caches)
    p.k_scale, p.v_scale = (describe(s, E8M0) for s in scales)
    p.page_table_k, p.page_table_v = (tensor(I32, [b, 1, t.shape[1], 1]) for t in tables)
    p.lengths = tensor(I32, [b, 1, 1, 1])
    if added is not None:
        p.added = p.lengths
    if lengths_out is not None:
        p.lengths_out = p.lengths
    everything = [k, v, *caches, *scales, *tables, lengths, added, lengths_out]
    cache.cache_append(p, [None if x is None else x.data_ptr() for x in everything], stream=stream)


def check_append(rng, b, s, hk, d, page, t, lengths, added, dtype, layout="heads", spoil=None, strided=False, kernel=0, slots=None, bad_pages=False, in_place=False):
    slots = slots or (max(lengths) + s + page - 1) // page
    pages = b * slots + 3
    tables = [table_of(rng, b, slots, pages), table_of(rng, b, slots, pages)]
    if bad_pages:
        tables[0][0, 0], tables[1][-1, -1] = -1, pages
    k, v = (randn(rng, (b, s, hk, d) if strided else (b, hk, s, d), dtype) for _ in range(2))
    if strided:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    k *= 2.0 ** ints(rng.integers(-4, 5, (b, hk, s, 1)), torch.float32).to(k.dtype)
    if spoil:
        spoil(k, v)
    caches, scales = zip(*(cache_of(rng, pages, hk, page, t, d, layout) for _ in range(2)))
    expected = [(c.cpu().numpy().copy(), sc.cpu().numpy().copy()) for c, sc in zip(caches, scales)]
    dev_lengths, dev_added = ints(lengths), None if added is None else ints(added)
    out = dev_lengths if in_place else torch.full_like(dev_lengths, -7)
    run_append(k, v, caches, scales, [torch.from_numpy(x).cuda() for x in tables], dev_lengths, dev_added, dtype, kernel, out)
    torch.cuda.synchronize()
    n = [s] * b if added is None else added
    for x, (codes, scale), table, got, got_scale in zip((k, v), expected, tables, caches, scales):
        ref.append(double(x), codes, scale, table, lengths, n)
        assert np.array_equal(got_scale.cpu().numpy(), scale)
        wrong = np.argwhere(got.cpu().numpy() != codes)
        assert len(wrong) == 0, wrong[:5]
    assert out.tolist() == [min(max(x, 0) + min(max(y, 0), s), slots * page) for x, y in zip(lengths, n)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,s,hk,d,page,t,lengths,added", [
    (1, 1, 1, 64, 16, 16, [0], None),
    (4, 1, 3, 128, 64, 16, [0, 15, 16, 63], None),
    (3, 1, 2, 128, 64, 64, [1, 63, 130], [1, 0, 1]),
    (3, 37, 2, 64, 48, 16, [0, 5, 47], [37, 12, 0]),
    (2, 200, 2, 128, 64, 64, [17, 0], [200, 63]),
    (2, 130, 1, 256, 128, 128, [100, 0], None),
    (1, 300, 2, 256, 256, 256, [3], None),
    (2, 9, 2, 72, 10, 5, [3, 0], None),
    (2, 4, 1, 7, 6, 3, [1, 2], [4, 3]),
])
def test_append(dtype, b, s, hk, d, page, t, lengths, added):
    check_append(np.random.default_rng(s * 7 + d), b, s, hk, d, page, t, lengths, added, dtype)


def test_append_layouts_and_bounds():
    rng = np.random.default_rng(5)
    check_append(rng, 2, 21, 3, 64, 32, 16, [9, 30], None, BF16, layout="tokens", strided=True)
    check_append(rng, 2, 21, 3, 64, 32, 16, [9, 30], None, BF16, kernel=cache.APPEND_SCALAR)
    check_append(rng, 3, 40, 2, 64, 16, 16, [0, 20, 3], [40, 40, 10], BF16, slots=2)          # tokens past the table are not written
    check_append(rng, 2, 40, 2, 64, 16, 16, [0, 20], None, BF16, bad_pages=True)
    check_append(rng, 3, 5, 2, 64, 16, 16, [-4, 2, 31], [9, -3, 5], BF16, in_place=True)      # lengths and counts out of range
    check_append(rng, 300, 3, 1, 64, 16, 16, [i % 40 for i in range(300)], None, BF16, in_place=True)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_append_special_values(dtype):
    def spoil(k, v):
        k[0] = 0                       # blocks of zeros bound nothing
        k[1, :, 3] = float("nan")      # a NaN takes its whole block, what it held too
        v[0, 0, 2, 1] = float("inf")
        v[1] *= 1e-3
        if dtype == F32:
            v[2] = 1e-44               # amax / 448 rounds to zero
            k[2, :, 0] *= 1e30
    check_append(np.random.default_rng(1), 3, 20, 2, 64, 32, 16, [5, 9, 30], None, dtype, spoil=spoil)


# ---- attention --------------------------------------------------------------------------------------

def run_attend(q, caches, scales, tables, seq_kv, seq_q=None, s_kv=None, o_type=None, dtype=BF16, kernel=0, attn_scale=None, stream=None, o=None, left=None, right=None, bottom_right=False,
               stats=True, scratch=None):
    b, hq, sq, d = q.shape
    p = cache.CacheSdpaParams(attn_scale=d ** -0.5 if attn_scale is None else attn_scale, s_kv=s_kv or tables[0].shape[1] * caches[0].shape[2], kernel=kernel, bottom_right=bottom_right)
    if left is not None:
        p.has_left_bound, p.left_bound = 1, left
    if right is not None:
        p.has_right_bound, p.right_bound = 1, right
    o_type = dtype if o_type is None else o_type
    o = torch.full(q.shape, 77.0, device="cuda", dtype=TORCH[o_type]) if o is None else o
    p.q, p.o = describe(q, dtype), describe(o, o_type)
    p.k, p.v = (describe(c, E4M3) for c in caches)
    p.k_scale, p.v_scale = (describe(s, E8M0) for s in scales)
    p.page_table_k, p.page_table_v = (tensor(I32, [b, 1, t.shape[1], 1]) for t in tables)
    p.seq_kv = tensor(I32, [b, 1, 1, 1])
    if seq_q is not None:
        p.seq_q = p.seq_kv
    rows = torch.full((b, hq, sq, 1), 55.0, device="cuda") if stats else None
    if stats:
        p.stats = describe(rows, F32)
    info = cache.query("cache_sdpa", p)
    scratch = torch.full((info.scratch_bytes + 16,), 255, device="cuda", dtype=torch.uint8) if scratch is None else scratch   # (NaN patterns)
    everything = [q, *caches, o, rows, *scales, seq_q, seq_kv, *tables]
    cache.cache_sdpa(p, [None if x is None else x.data_ptr() for x in everything], scratch.data_ptr(), stream)
    return o, rows, info


def check_attend(got, rows, q, caches, scales, tables, seq_q, seq_kv, s_kv, o_type, attn_scale, weight_step=2.0 ** -11, **masks):
    """Weights are rounded by half a step of f16 (2^-11 of themselves; below 2^-14 * 2^-15 of the largest by 2^-40) or of bf16 in the tcgen05 form, scores by
    the f32 sum of D products (D 2^-24 of the sum of their magnitudes, once up and once down in a weight) and in their scaling and exponential (2^-21 of
    a score and 2^-21); O is rounded once more."""
    q64, d = double(q), q.shape[3]
    host = [c.cpu().numpy() for c in caches] + [s.cpu().numpy() for s in scales] + [t.cpu().numpy() for t in tables]
    with np.errstate(invalid="ignore"):
        o, stats, mean, products = ref.attend(q64, *host[:4], host[4], host[5], None if seq_q is None else seq_q.tolist(), seq_kv.tolist(), attn_scale, s_kv, **masks)
    score = d * 2.0 ** -24 * products + 2.0 ** -21 * (1 + products)
    bound = (weight_step * 1.01 + 2 * score)[..., None] * mean + half_step(o_type) * np.abs(o) * 1.01 + (2.0 ** -25 if o_type == F16 else 1e-30)
    actual = double(got)
    nan = np.isnan(o)
    assert np.array_equal(np.isnan(actual), nan)
    off = np.abs(np.where(nan, 0, actual - o)) - np.where(nan, 0, bound)
    assert np.all(off <= 0), (off.max(), np.unravel_index(off.argmax(), off.shape))
    if rows is not None:
        actual = double(rows)[..., 0]
        finite = np.isfinite(stats)
        assert np.array_equal(np.isnan(actual), np.isnan(stats)) and np.array_equal(actual[np.isinf(stats)], stats[np.isinf(stats)])
        assert np.all(np.abs(actual - stats)[finite] <= (2 * score + 1e-6 * (1 + np.abs(stats)))[finite])


def attend_case(seed, dtype, d, hk, g, sq, page, t, lengths, s_kv=None, seq_q=None, o_type=None, layout="heads", bad_pages=False, spoil=None, kernel=0, q_scale=1.0, slots=None, o=None, q=None,
                weight_step=2.0 ** -11, **masks):
    rng = np.random.default_rng(seed)
    b = len(lengths)
    slots = slots or max(1, (max(lengths) + page - 1) // page)
    pages = b * slots + 2
    tables = [table_of(rng, b, slots, pages), table_of(rng, b, slots, pages)]
    if bad_pages:
        tables[0][0, 0], tables[1][0, 1 % slots], tables[0][-1, slots // 2] = -5, pages, 2 ** 31 - 1
    tables = [torch.from_numpy(x).cuda() for x in tables]
    q = randn(rng, (b, hk * g, sq, d), dtype, q_scale) if q is None else q
    caches, scales = zip(*(cache_of(rng, pages, hk, page, t, d, layout) for _ in range(2)))
    if spoil:
        spoil(q, caches, scales, tables)
    seq_kv, dev_q = ints(lengths), None if seq_q is None else ints(seq_q)
    s_kv = s_kv or slots * page
    # (codes have magnitudes up to 448 and scales up to 2^-3 here: scores of a few hundred times q)
    got, rows, info = run_attend(q, caches, scales, tables, seq_kv, dev_q, s_kv, o_type, dtype, kernel, d ** -0.5 / 64, o=o, **masks)
    torch.cuda.synchronize()
    assert dfgpu.device_status() == 0
    names = {k: v for k, v in masks.items() if k in ("left", "right", "bottom_right")}
    check_attend(got, rows, q, caches, scales, tables, dev_q, seq_kv, s_kv, dtype if o_type is None else o_type, d ** -0.5 / 64, weight_step, **names)
    return got, rows, info


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,hk,g,sq,page,t,lengths", [
    (128, 1, 1, 1, 16, 16, [1]),
    (128, 2, 4, 1, 64, 16, [0, 1, 127, 128, 129, 500]),
    (64, 3, 8, 1, 48, 48, [0, 33, 700]),
    (256, 1, 3, 1, 32, 16, [5, 64, 65, 400]),
    (128, 1, 16, 1, 64, 64, [300]),
    (128, 1, 20, 1, 64, 64, [200, 40]),
    (64, 1, 70, 1, 256, 64, [300]),
])
def test_single_tokens(dtype, d, hk, g, sq, page, t, lengths):
    attend_case(d + g, dtype, d, hk, g, sq, page, t, lengths)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,hk,g,sq,page,t,lengths,left", [
    (128, 2, 4, 4, 64, 16, [0, 3, 4, 130, 600], None),
    (128, 2, 4, 7, 64, 16, [2, 130, 600], 100),
    (64, 1, 8, 5, 48, 16, [5, 300], 20),
    (256, 2, 2, 3, 64, 64, [100, 7], None),
    (128, 1, 2, 40, 16, 16, [40, 39, 170], 30),
    (64, 2, 3, 33, 32, 32, [33, 100], None),
    (256, 1, 1, 70, 64, 32, [70, 200], 64),
])
def test_several_tokens(dtype, d, hk, g, sq, page, t, lengths, left):
    attend_case(d + sq, dtype, d, hk, g, sq, page, t, lengths, right=0, left=left, bottom_right=True)


UMMA = cache.SDPA_UMMA


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,hk,g,sq,page,t,lengths,left", [
    (128, 1, 1, 128, 64, 16, [128], None),
    (128, 1, 4, 64, 64, 64, [300, 64], None),
    (64, 2, 2, 200, 48, 16, [200, 333], None),
    (128, 2, 5, 60, 32, 32, [500, 61, 60], None),
    (64, 1, 16, 30, 16, 16, [129, 31], 40),
    (128, 1, 3, 150, 256, 128, [1000], 200),
    (128, 1, 70, 3, 64, 64, [260, 2], None),
    (64, 1, 128, 2, 64, 16, [100], None),
    (128, 2, 8, 1, 64, 16, [700, 0, 1], None),
])
def test_chunks_of_prompts_on_tcgen05(dtype, d, hk, g, sq, page, t, lengths, left):
    _, _, info = attend_case(d + sq, dtype, d, hk, g, sq, page, t, lengths, right=0, left=left, bottom_right=True, kernel=UMMA)
    assert info.kernel == UMMA


def test_tcgen05_form_masks_and_types():
    attend_case(1, BF16, 128, 2, 2, 70, 64, 16, [200, 90, 5], seq_q=[70, 3, 0], right=0, bottom_right=True, kernel=UMMA)
    attend_case(2, BF16, 128, 1, 2, 70, 64, 16, [200, 90, 5], seq_q=[6, 90, -2], right=0, bottom_right=True, kernel=UMMA)
    attend_case(3, BF16, 64, 2, 2, 150, 32, 16, [100, 8], right=0, kernel=UMMA)                                  # aligned to the top left
    attend_case(4, F16, 64, 2, 2, 90, 32, 16, [100, 8], right=-2, left=50, bottom_right=True, kernel=UMMA)       # rows without keys
    attend_case(5, BF16, 64, 1, 2, 90, 32, 16, [400, 8], left=0, kernel=UMMA)                                   # no right bound
    attend_case(6, BF16, 128, 1, 4, 40, 64, 64, [700, 300], s_kv=450, kernel=UMMA)
    attend_case(7, BF16, 128, 1, 4, 40, 64, 64, [700, -3], slots=11, right=2 ** 62, left=2 ** 62, kernel=UMMA)
    attend_case(8, BF16, 128, 2, 4, 40, 64, 16, [300, 70], o_type=F32, right=0, bottom_right=True, kernel=UMMA)
    attend_case(10, F16, 128, 2, 4, 40, 48, 16, [300, 77], layout="tokens", bad_pages=True, right=0, bottom_right=True, kernel=UMMA)
    attend_case(13, BF16, 128, 1, 4, 40, 64, 16, [300, 70], q_scale=2.0 ** 70, kernel=UMMA)
    attend_case(14, BF16, 128, 1, 4, 40, 64, 16, [300, 70], q_scale=2.0 ** -90, stats=False, kernel=UMMA)
    attend_case(15, BF16, 128, 2, 2, 33, 64, 16, [40] * 130, right=0, bottom_right=True, kernel=UMMA)            # more sequences than are ranked


def test_masks_lengths_and_types():
    attend_case(1, BF16, 128, 2, 2, 6, 64, 16, [200, 90, 5], seq_q=[6, 3, 0], right=0, bottom_right=True)       # padded query rows
    attend_case(2, BF16, 128, 2, 2, 6, 64, 16, [200, 90, 5], seq_q=[6, 9, -2], right=0, bottom_right=True)      # and lengths out of range
    attend_case(3, BF16, 64, 2, 2, 9, 32, 16, [100, 8], right=0)                                               # aligned to the top left
    attend_case(4, BF16, 64, 2, 2, 9, 32, 16, [100, 8], right=-2, left=5, bottom_right=True)                    # rows without keys
    attend_case(5, BF16, 64, 2, 2, 2, 32, 16, [100, 8], left=0)                                                # nothing but what lies ahead
    attend_case(6, BF16, 128, 1, 4, 1, 64, 64, [700, 300], s_kv=450)                                           # lengths behind s_kv
    attend_case(7, BF16, 128, 1, 4, 1, 64, 64, [700, -3], slots=11, right=2 ** 62, left=2 ** 62)
    attend_case(8, BF16, 128, 2, 4, 3, 64, 16, [300, 70], o_type=F32, right=0, bottom_right=True)
    attend_case(9, F16, 256, 2, 1, 1, 64, 16, [300, 70], o_type=F32)
    attend_case(10, BF16, 128, 2, 4, 2, 48, 16, [300, 77], layout="tokens", bad_pages=True)
    attend_case(11, BF16, 64, 1, 4, 20, 64, 16, [300, 77], bad_pages=True, right=0, bottom_right=True)
    attend_case(12, BF16, 128, 2, 4, 1, 64, 16, [300, 70], stats=False)
    attend_case(13, BF16, 128, 2, 4, 1, 64, 16, [300, 70], q_scale=2.0 ** 70)                                  # far beyond f16: one key takes it all
    attend_case(14, BF16, 128, 2, 4, 1, 64, 16, [300, 70], q_scale=2.0 ** -90)


def test_strided_queries_and_outputs():
    rng = np.random.default_rng(4)
    q = randn(rng, (2, 3, 8, 128), BF16).transpose(1, 2)                       # [B, Sq, Hq, D] memory
    o = torch.full((2, 3, 8, 130), 9.0, device="cuda", dtype=torch.bfloat16)
    attend_case(4, BF16, 128, 2, 4, 3, 64, 16, [150, 64], q=q, o=o[..., 1:129].transpose(1, 2), right=0, bottom_right=True)   # O off a 16-byte boundary
    assert bool((o[..., 0] == 9).all()) and bool((o[..., 129] == 9).all())


@pytest.mark.parametrize("lengths,hk", [([9000], 1), ([5000, 12000], 2), ([300] * 40, 8)])
def test_long_contexts_and_many_chunks(lengths, hk):
    attend_case(len(lengths), BF16, 128, hk, 4, 1, 64, 64, lengths)
    attend_case(len(lengths), F16, 64, hk, 2, 3, 64, 16, lengths, right=0, bottom_right=True, left=3000)


@pytest.mark.parametrize("d,g,dtype", [(128, 2, BF16), (128, 12, BF16), (64, 4, F16), (256, 3, BF16), (256, 16, F16)])
def test_many_units_for_each_cta(d, g, dtype):
    """Every CTA's ring goes round several times, over the ends of lists of very different lengths."""
    attend_case(d + g, dtype, d, 8, g, 1, 64, 64, [9000, 100, 6000, 0, 12000, 33, 7000, 2000], right=0, bottom_right=True)


def test_scales_far_apart():
    """Neighbouring blocks of V 2^60 apart, one of zeros with a scale of 1 beside tiny ones: nothing is lost to the larger scale."""
    def spoil(q, caches, scales, tables):
        scales[1][..., 0] = 60
        scales[1][:, :, 1::2] = 127
        caches[1][:, :, 16:32] = 0
        caches[1][:, :, 48:] = 0
    attend_case(3, BF16, 128, 2, 4, 1, 64, 16, [300, 70], spoil=spoil)
    attend_case(3, BF16, 64, 2, 4, 5, 64, 16, [300, 70], spoil=spoil, right=0, bottom_right=True)
    attend_case(3, BF16, 128, 1, 4, 50, 64, 16, [300, 70], spoil=spoil, right=0, bottom_right=True, kernel=UMMA)   # (left to the streaming form)


def test_zeros_with_the_least_scale():
    """Blocks of zeros as an append writes them, among others and alone."""
    def spoil(q, caches, scales, tables):
        caches[1][:, :, :16] = 0
        scales[1][:, :, 0] = 0

    def all_zero(q, caches, scales, tables):
        caches[1].zero_()
        scales[1].zero_()
    for kernel, sq in ((0, 1), (0, 6), (UMMA, 40)):
        attend_case(6, BF16, 128, 1, 4, sq, 64, 16, [300, 70], spoil=spoil, right=0, bottom_right=True, kernel=kernel)
        attend_case(6, BF16, 64, 1, 4, sq, 64, 16, [300, 70], spoil=all_zero, right=0, bottom_right=True, kernel=kernel)


@pytest.mark.parametrize("kernel,sq", [(0, 1), (0, 9), (UMMA, 50)])
def test_nan_and_infinity_in_queries_and_seen_keys(kernel, sq):
    def spoil(q, caches, scales, tables):
        q[0, 1, 0, 5], q[1, 2, -1, 100] = float("inf"), float("nan")
        caches[0][tables[0][0, 1].item(), 0, 7, ::9] = 0xFF       # key 71: seen by every row of its sequence but the first
        caches[1][tables[1][1, 0].item(), 0, 9, 3] = 0x7F
    got, _, _ = attend_case(2, BF16, 128, 1, 4, sq, 64, 16, [60 + sq + 11, 150], spoil=spoil, right=0, bottom_right=True, kernel=kernel)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("sq", [1, 6, 30])
def test_nan_in_masked_places(d, sq):
    """NaN codes and scales behind a sequence's end, before its window and above the diagonal reach no row that does not see them; those of a key
    that is seen reach the rows that see it."""
    page, lengths = 32, [100, 61]

    def spoil(q, caches, scales, tables):
        for which, table in zip(range(2), tables):
            for b, n in enumerate(lengths):
                for key in (n, n + 1, n - 1, n - 3, n - 20):          # behind the end; the last keys, which only the last rows see
                    if key < table.shape[1] * page and (key >= n or sq > 1):
                        caches[which][table[b, key // page].item(), :, key % page, which::5] = 0x7F if key % 2 else 0xFF
                if n % 16:
                    pass
                else:
                    scales[which][table[b, n // page].item(), :, n % page // 16] = 255
            last = table.shape[1] * page - 1
            scales[which][table[1, last // page].item(), :, -1] = 255                 # a block that nobody reaches
    attend_case(d, BF16, d, 2, 2, sq, page, 16, lengths, spoil=spoil, right=0, bottom_right=True)
    attend_case(d, BF16, d, 2, 2, sq, page, 16, lengths, spoil=spoil, right=0, left=40, bottom_right=True)
    if d < 256:
        attend_case(d, BF16, d, 2, 2, sq, page, 16, lengths, spoil=spoil, right=0, bottom_right=True, kernel=UMMA)


def test_a_block_above_the_diagonal_has_no_scale():
    """The last block's scale is a NaN: rows that end before it are finite."""
    def spoil(q, caches, scales, tables):
        scales[1][tables[1][0, 1].item(), :, 1] = 255
        scales[0][tables[0][0, 1].item(), :, 1] = 255
    for kernel in (0, UMMA):
        got, rows, _ = attend_case(1, BF16, 128, 1, 2, 20, 32, 16, [64], spoil=spoil, right=0, bottom_right=True, kernel=kernel)
        assert bool(torch.isfinite(got[:, :, :4].float()).all()) and bool(torch.isnan(got[:, :, 4:].float()).all())


def test_offsets_past_32_bits():
    """A container of 5.4 GB whose last pages are read."""
    pages, hk, page, d = 41000, 8, 128, 128
    codes = torch.zeros(pages, hk, page, d, device="cuda", dtype=torch.uint8)
    scale = torch.full((pages, hk, 1, 1), 121, device="cuda", dtype=torch.uint8)
    table = torch.arange(pages - 3, pages, device="cuda", dtype=torch.int32)[None]
    rng = np.random.default_rng(0)
    k = randn(rng, (1, hk, 300, d), BF16)
    other, other_scale = torch.zeros(4, hk, page, d, device="cuda", dtype=torch.uint8), torch.zeros(4, hk, 1, 1, device="cuda", dtype=torch.uint8)
    near = ints([[0, 1, 2]])
    run_append(k, k, (codes, other), (scale, other_scale), (table, near), ints([0]))
    assert torch.equal(codes[pages - 3:], other[:3]) and torch.equal(scale[pages - 3:], other_scale[:3])
    q = randn(rng, (1, 16, 1, d), BF16)
    far_o, far_stats, _ = run_attend(q, (codes, codes), (scale, scale), (table, table), ints([300]))
    near_o, near_stats, _ = run_attend(q, (other, other), (other_scale, other_scale), (near, near), ints([300]))
    assert torch.equal(far_o, near_o) and torch.equal(far_stats, near_stats)
    p = cache.CachePagesParams(op=cache.PAGE_OPS["copy"], block=page, pool_count=1)
    p.refs, p.list, p.pools[0] = tensor(I32, [pages]), tensor(I32, [1, 2]), tensor(U8, [1, pages, hk * page * d])
    scratch = torch.empty(cache.query("cache_pages", p).scratch_bytes, device="cuda", dtype=torch.uint8)
    entries = ints([[pages - 1, pages - 40]])
    cache.cache_pages(p, [None, None, None, entries.data_ptr(), None, None, None, None, codes.data_ptr()], scratch.data_ptr())
    assert torch.equal(codes[pages - 1], codes[pages - 40])


# ---- pages ----------------------------------------------------------------------------------------------

POOLS = ([(1, 64, U8)], [(2, 96, BF16), (3, 20, U8), (1, 7, E8M0)], [(2, 12000, U8), (1, 8192, F32)])


def pages_state(rng, b, slots, pages, block, pools, empty=(), share=True):
    table = np.full((b, slots), -1, dtype=np.int32)
    refs = np.zeros(pages, dtype=np.int32)
    lengths = np.zeros(b, dtype=np.int32)
    ids = list(rng.permutation(pages))
    for i in range(b):
        if i in empty:
            continue
        lengths[i] = rng.integers(0, slots * block + 1)
        used = -(-int(lengths[i]) // block)
        while len(ids) < used + pages // 8:
            used -= 1
            lengths[i] = used * block
        used = max(used, 0)
        lengths[i] = max(lengths[i], 0)
        for s in range(used):
            table[i, s] = ids.pop()
            refs[table[i, s]] += 1
    if share:
        for i in range(1, b):
            if lengths[i] >= block and lengths[i - 1] >= block:   # the first page of two sequences
                refs[table[i, 0]] -= 1
                table[i, 0] = table[i - 1, 0]
                refs[table[i, 0]] += 1
    host = [rng.integers(0, 256, (layers, pages, n * dfgpu.DTYPE_BYTES[t])).astype(np.uint8) for layers, n, t in pools]
    return ref.Pages(table, lengths, refs, host, block)


def run_pages(op, state, entries, pool_types=(), in_place=False, stream=None, odd=0):
    b, slots = state.table.shape
    p = cache.CachePagesParams(op=cache.PAGE_OPS[op], block=state.block, pool_count=len(pool_types))
    p.page_table, p.lengths, p.refs = tensor(I32, [b, 1, slots, 1]), tensor(I32, [b, 1, 1, 1]), tensor(I32, [len(state.refs)])
    entries = None if entries is None else ints(entries)
    if entries is not None:
        p.list = tensor(I32, list(entries.shape))
    pools = []
    for i, (layers, n, t) in enumerate(pool_types):
        host = state.pools[i]
        buffer = torch.zeros(host.size + odd, device="cuda", dtype=torch.uint8)
        pools.append(buffer[odd:].view(host.shape))
        pools[-1].copy_(torch.from_numpy(host))
        p.pools[i] = tensor(t, [layers, host.shape[1], n])
    ins = [torch.from_numpy(x.copy()).cuda() for x in (state.table, state.lengths, state.refs)]
    outs = ins if in_place else [torch.full_like(x, -99) for x in ins]
    report = torch.full((4,), -1, device="cuda", dtype=torch.int32)
    scratch = torch.full((cache.query("cache_pages", p).scratch_bytes,), 255, device="cuda", dtype=torch.uint8)
    everything = [*ins, entries, *outs, report, *pools]
    cache.cache_pages(p, [None if x is None else x.data_ptr() for x in everything], scratch.data_ptr(), stream)
    torch.cuda.synchronize()
    return [x.cpu().numpy() for x in outs], report.tolist(), [x.cpu().numpy() for x in pools]


def check_pages(op, state, entries, pool_types=(), **how):
    want = ref.Pages(state.table, state.lengths, state.refs, state.pools, state.block)
    host = [] if entries is None else np.asarray(entries).tolist()
    report = {"reserve": lambda: want.reserve([e[0] for e in host]), "fork": lambda: want.fork([tuple(e) for e in host]), "free": lambda: want.free_sequences([e[0] for e in host]),
              "compact": want.compact, "copy": lambda: want.copy([tuple(e) for e in host])}[op]()
    (table, lengths, refs), got_report, pools = run_pages(op, state, entries, pool_types, **how)
    assert np.array_equal(table, want.table) and np.array_equal(refs, want.refs)
    assert np.array_equal(lengths, want.lengths)
    assert got_report == [int(x) for x in report]
    for got, expected in zip(pools, want.pools):
        assert np.array_equal(got, expected)
    return want


SIZES = [(1, 1, 2, 16), (3, 4, 20, 16), (17, 9, 200, 48), (64, 33, 3000, 64), (5, 3, 20000, 1)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("b,slots,pages,block", SIZES)
def test_reserve_and_free(b, slots, pages, block, in_place):
    rng = np.random.default_rng(b)
    state = pages_state(rng, b, slots, pages, block, [], empty=(0,))
    check_pages("reserve", state, rng.integers(-3, 2 * block, (b, 1)), in_place=in_place)
    check_pages("reserve", state, np.full((b, 1), slots * block), in_place=in_place)             # more than fits, or than there is
    check_pages("reserve", state, np.zeros((b, 1), dtype=int), in_place=in_place)
    check_pages("free", state, rng.permutation(b)[: b // 2 + 1, None], in_place=in_place)
    check_pages("free", state, [[0], [b], [0], [-1], [b - 1]], in_place=in_place)                # twice, out of range, skipped
    state.refs[:] = 1                                                                             # counts that do not add up stay at 0
    check_pages("free", state, np.arange(b)[:, None], in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pools", range(3))
@pytest.mark.parametrize("b,slots,pages,block", SIZES)
def test_fork(b, slots, pages, block, pools, in_place):
    if pages > 5000 and pools == 2:
        pytest.skip("1 GB of pools")
    rng = np.random.default_rng(b + 1)
    empty = tuple(range(b // 2, b))
    state = pages_state(rng, b, slots, pages, block, POOLS[pools], empty=empty)
    entries = [(int(rng.integers(0, max(1, b // 2))), t) for t in empty]
    check_pages("fork", state, entries, POOLS[pools], in_place=in_place)
    odd = [(-1, 0), (0, b), (b, 0), (0, 0), (0, empty[0]), (0, empty[-1]), (0, empty[0]), (empty[0], empty[-1]), (0, -3)]
    check_pages("fork", state, odd, POOLS[pools], in_place=in_place)
    state.refs[state.refs == 0] = 5                                                               # no free pages: whole ones can be shared
    check_pages("fork", state, entries, POOLS[pools], in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pools", range(3))
@pytest.mark.parametrize("b,slots,pages,block", SIZES)
def test_compact_and_copy(b, slots, pages, block, pools, in_place):
    if pages > 5000 and pools == 2:
        pytest.skip("1 GB of pools")
    rng = np.random.default_rng(b + 2)
    state = pages_state(rng, b, slots, pages, block, POOLS[pools])
    state.table[0, -1] = pages + 5                                                                # an id out of range stays
    check_pages("compact", state, None, POOLS[pools], in_place=in_place)
    check_pages("compact", check_pages("compact", state, None, POOLS[pools]), None, POOLS[pools], in_place=in_place)   # dense already
    n = min(pages // 2, 300)
    ids = rng.permutation(pages)
    check_pages("copy", state, np.stack([ids[:n], ids[pages - n:]], 1), POOLS[pools], in_place=in_place, odd=1)
    check_pages("copy", state, rng.integers(-1, pages + 1, (n + 3, 2)), POOLS[pools], in_place=in_place, odd=4)        # repeated, chained, out of range
    check_pages("copy", state, [[0, 1], [0, 1], [1, 0]] if pages > 1 else [[0, 0]], POOLS[pools], in_place=in_place)


def test_many_pages_and_entries():
    rng = np.random.default_rng(7)
    state = pages_state(rng, 9000, 3, 40000, 16, [(1, 16, U8)], empty=tuple(range(4000, 9000)))
    check_pages("reserve", state, rng.integers(0, 30, (9000, 1)))
    check_pages("fork", state, [(int(s), t) for s, t in zip(rng.integers(0, 4000, 5000), range(4000, 9000))], [(1, 16, U8)], in_place=True)
    check_pages("compact", state, None, [(1, 16, U8)], in_place=True)
    check_pages("copy", state, rng.integers(0, 40000, (9000, 2)), [(1, 16, U8)])


# ---- together ----------------------------------------------------------------------------------------------

class Program:
    """A small serving program: rotated keys and values of each step go into the pages, queries attend over them."""

    def __init__(self, b, hk, g, d, page, t, slots, pages, seed):
        rng = np.random.default_rng(seed)
        self.b, self.hk, self.g, self.d, self.page, self.t, self.slots, self.pages, self.rng = b, hk, g, d, page, t, slots, pages, rng
        self.caches = [torch.zeros(pages, hk, page, d, device="cuda", dtype=torch.uint8) for _ in range(2)]
        self.scales = [torch.zeros(pages, hk, page // t, 1, device="cuda", dtype=torch.uint8) for _ in range(2)]
        self.table, self.lengths, self.refs = torch.full((b, slots), -1, device="cuda", dtype=torch.int32), torch.zeros(b, device="cuda", dtype=torch.int32), torch.zeros(pages, device="cuda", dtype=torch.int32)
        self.frequencies = torch.tensor(cache.rope_frequencies(d)[0], device="cuda")
        self.report = torch.zeros(4, device="cuda", dtype=torch.int32)
        self.tokens = [[] for _ in range(b)]      # what each sequence holds: rotated (K, V) of every token, as written

    def manage(self, op, entries=None, stream=None):
        p = cache.CachePagesParams(op=cache.PAGE_OPS[op], block=self.page, pool_count=4 if op in ("fork", "compact", "copy") else 0)
        p.page_table, p.lengths, p.refs = tensor(I32, [self.b, 1, self.slots, 1]), tensor(I32, [self.b, 1, 1, 1]), tensor(I32, [self.pages])
        if entries is not None:
            p.list = tensor(I32, list(entries.shape))
        pools = [*self.caches, *self.scales] if p.pool_count else []
        for i, pool in enumerate(pools):
            p.pools[i] = tensor(U8, [1, self.pages, pool[0].numel()])
        scratch = torch.empty(cache.query("cache_pages", p).scratch_bytes, device="cuda", dtype=torch.uint8)
        own = [self.table, self.lengths, self.refs]
        cache.cache_pages(p, [x.data_ptr() for x in own] + [None if entries is None else entries.data_ptr()] + [x.data_ptr() for x in own] + [self.report.data_ptr()] +
                          [x.data_ptr() for x in pools], scratch.data_ptr(), stream)
        return scratch

    def step(self, s, added, stream=None):
        """One call of each operator for up to s new tokens a sequence; (q, O, Stats)."""
        q, k, v = (randn(self.rng, (self.b, h, s, self.d), BF16) for h in (self.hk * self.g, self.hk, self.hk))
        dev_added = ints(added)
        keep = [self.manage("reserve", dev_added[:, None].contiguous(), stream)]
        positions = (self.lengths[:, None] + torch.arange(s, device="cuda")).to(torch.int32)
        q, k = run_rope(q, positions, self.frequencies, k, stream=stream)
        run_append(k, v, self.caches, self.scales, (self.table, self.table), self.lengths, dev_added, lengths_out=self.lengths, stream=stream)
        o, rows, _ = run_attend(q, self.caches, self.scales, (self.table, self.table), self.lengths, dev_added, stream=stream, right=0, bottom_right=True)
        torch.cuda.synchronize()
        assert self.report[3].item() == 0 and dfgpu.device_status() == 0
        for i, n in enumerate(added):
            self.tokens[i] += [(double(k[i, :, j]), double(v[i, :, j])) for j in range(n)]
        return q, o, rows, dev_added, keep

    def check(self, q, o, rows, dev_added, keep):
        """Against the cache's own codes exactly, and against what was written within a step of its codes."""
        check_attend(o, rows, q, self.caches, self.scales, (self.table, self.table), dev_added, self.lengths, self.slots * self.page, BF16, self.d ** -0.5, right=0, bottom_right=True)
        assert self.lengths.tolist() == [len(x) for x in self.tokens]
        codes, scale, table = self.caches[0].cpu().numpy(), self.scales[0].cpu().numpy(), self.table.cpu().numpy()
        for i, tokens in enumerate(self.tokens):
            for at, (k, _) in enumerate(tokens):
                page, row = table[i, at // self.page], at % self.page
                step = ref.e8m0(scale[page, :, row // self.t, 0])[:, None]
                # each encoding is off by half a step of e4m3 (2^-4 of the value, 2^-10 of the scale at least); a code is encoded again when its block's scale
                # grows, at the most three times here, by a factor of two or more each: 2^-4 (1 + 1 + 1 + 1)
                assert np.all(np.abs(ref.E4M3[codes[page, :, row]] * step - k) <= 4 * 2.0 ** -4 * np.abs(k) + 4 * 2.0 ** -10 * step)


def test_a_serving_program():
    p = Program(b=6, hk=2, g=4, d=64, page=32, t=16, slots=8, pages=40, seed=1)
    p.check(*p.step(40, [40, 7, 33, 0, 0, 0]))                        # prompts
    p.check(*p.step(1, [1, 1, 1, 0, 0, 0]))                           # a token each
    p.manage("fork", ints([[0, 3], [2, 4], [0, 5]]))
    p.tokens[3], p.tokens[4], p.tokens[5] = list(p.tokens[0]), list(p.tokens[2]), list(p.tokens[0])
    for _ in range(3):
        p.check(*p.step(1, [1] * 6))                                  # branches go their own ways
    p.manage("free", ints([[0], [2]]))
    p.tokens[0], p.tokens[2] = [], []
    p.manage("compact")
    live = int((p.refs > 0).sum())
    assert bool((p.refs[:live] > 0).all()) and p.report.tolist()[0] == 40 - live
    p.check(*p.step(5, [5, 2, 0, 1, 5, 4]))                           # drafted tokens, an empty sequence
    assert sum(p.refs.tolist()) == sum(-(-n // 32) for n in p.lengths.tolist())


def test_captured_and_replayed_on_another_stream():
    """A decode step as a CUDA graph whose inputs change between replays, beside an eager call on a stream of its own."""
    rng = np.random.default_rng(11)
    b, hk, g, d, page, slots, pages = 3, 2, 4, 128, 64, 4, 16
    tables = torch.from_numpy(table_of(rng, b, slots, pages)).cuda()
    fresh = lambda: ([torch.zeros(pages, hk, page, d, device="cuda", dtype=torch.uint8) for _ in range(2)], [torch.zeros(pages, hk, page // 16, 1, device="cuda", dtype=torch.uint8) for _ in range(2)],  # noqa: E731
                     ints([0, 70, 129]))
    steps = [tuple(randn(rng, (b, h, 1, d), BF16) for h in (hk * g, hk, hk)) for _ in range(4)]
    prompt = tuple(randn(rng, (b, hk, 130, d), BF16) for _ in range(2))

    def fill(caches, scales):
        run_append(*prompt, caches, scales, (tables, tables), ints([0, 0, 0]), ints([0, 70, 129]))
        torch.cuda.synchronize()

    def eager():
        caches, scales, lengths = fresh()
        fill(caches, scales)
        results = []
        for q, k, v in steps:
            run_append(k, v, caches, scales, (tables, tables), lengths, lengths_out=lengths)
            results.append(run_attend(q, caches, scales, (tables, tables), lengths)[:2])
        torch.cuda.synchronize()
        return results
    want = eager()
    caches, scales, lengths = fresh()
    fill(caches, scales)
    q, k, v = (x.clone() for x in steps[0])
    o, rows_scratch = torch.empty_like(q), torch.full((1 << 20,), 255, device="cuda", dtype=torch.uint8)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        run_append(k, v, caches, scales, (tables, tables), lengths, lengths_out=lengths, stream=side.cuda_stream)
        _, rows, _ = run_attend(q, caches, scales, (tables, tables), lengths, stream=side.cuda_stream, o=o, scratch=rows_scratch)
    other = torch.cuda.Stream()
    for (new_q, new_k, new_v), (want_o, want_rows) in zip(steps, want):
        q.copy_(new_q), k.copy_(new_k), v.copy_(new_v)
        torch.cuda.synchronize()
        with torch.cuda.stream(other):   # a call of its own at the same time
            beside = run_rope(new_q, ints(np.full((b, 1), 77)), torch.tensor(cache.rope_frequencies(d)[0], device="cuda"), stream=other.cuda_stream)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want_o) and torch.equal(rows, want_rows)
        check_rope(beside, new_q, ints(np.full((b, 1), 77)), torch.tensor(cache.rope_frequencies(d)[0], device="cuda"), False, False, 1.0, BF16)
    assert lengths.tolist() == [4, 74, 133]


def test_results_do_not_depend_on_timing():
    rng = np.random.default_rng(2)
    q = randn(rng, (8, 16, 1, 128), BF16)
    caches, scales = zip(*(cache_of(rng, 400, 4, 64, 16, 128) for _ in range(2)))
    table = torch.from_numpy(table_of(rng, 8, 48, 400)).cuda()
    lengths = ints(rng.integers(100, 48 * 64, 8))
    first = run_attend(q, caches, scales, (table, table), lengths)[:2]
    for _ in range(5):
        again = run_attend(q, caches, scales, (table, table), lengths)[:2]
        assert all(torch.equal(x, y) for x, y in zip(first, again))


@pytest.mark.parametrize("dtype,d,hk,g,sq,page,t,lengths,left", [
    (BF16, 128, 1, 4, 64, 64, 64, [5000], None),                  # many pieces
    (F16, 64, 2, 2, 90, 48, 16, [2200, 130, 0, 91], None),        # short sequences: pieces without keys
    (BF16, 128, 1, 3, 130, 256, 128, [4097, 1025], 700),          # a window inside some of the pieces
    (F16, 128, 1, 128, 2, 64, 16, [3000], None),
])
def test_tcgen05_form_in_pieces(dtype, d, hk, g, sq, page, t, lengths, left):
    _, _, info = attend_case(d + sq, dtype, d, hk, g, sq, page, t, lengths, right=0, left=left, bottom_right=True, kernel=UMMA)
    assert info.kernel == UMMA and info.launches == 4


def test_tcgen05_form_in_pieces_without_a_bound():
    attend_case(7, BF16, 128, 1, 2, 150, 64, 64, [2500, 1200], seq_q=[150, 7], kernel=UMMA)


def test_tcgen05_form_in_pieces_over_special_values():
    def nan_code(q, caches, scales, tables):   # for the rows that see it alone: the streaming form has the call
        page = int(tables[1][0, 2400 // 64])
        caches[1].view(torch.uint8)[page, 0, 2400 % 64, 5] = 0x7f

    attend_case(8, BF16, 128, 1, 2, 150, 64, 64, [2500], right=0, bottom_right=True, kernel=UMMA, spoil=nan_code)


@pytest.mark.parametrize("dtype,d,hk,g,sq,left", [(F16, 64, 4, 8, 5, 300), (BF16, 128, 4, 16, 2, None)])
def test_drafted_tokens_of_large_groups_take_tcgen05(dtype, d, hk, g, sq, left):
    _, _, info = attend_case(d, dtype, d, hk, g, sq, 48, 16, [700, 5, 9, 1030, 100, 33, 64, 500], right=0, left=left, bottom_right=True)
    assert info.kernel == UMMA
    _, _, info = attend_case(d, dtype, d, hk, 7, 4, 48, 16, [700, 5, 9, 1030, 100, 33, 64, 500], right=0, left=left, bottom_right=True)
    assert info.kernel == cache.SDPA_STREAM
