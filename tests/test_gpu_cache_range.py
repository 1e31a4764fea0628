"""The edges of the 8-bit cache's operators: values and scales far apart, pages that are not there, lists that contradict themselves, many calls in a row."""
import numpy as np
import pytest

import cache_reference as ref
from deepforge_b200 import cache, dfgpu
from deepforge_b200.dfgpu import BF16, F16, F32, I32, U8, tensor
from test_gpu_cache import UMMA, attend_case, cache_of, ints, pages_state, randn, run_attend, run_pages, table_of

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


# ---- pages

@pytest.mark.parametrize("op", ["reserve", "compact"])
def test_page_operations_one_behind_the_other(op):
    """Nothing but chained launches on the stream: each CTA of a launch finds the others of its cluster running before it writes to them."""
    rng = np.random.default_rng(3)
    state = pages_state(rng, 64, 9, 3000, 16, [], empty=(0,))
    grow = rng.integers(0, 40, (64, 1))
    want = ref.Pages(state.table, state.lengths, state.refs, [], 16)
    report = want.reserve([int(x) for x in grow[:, 0]]) if op == "reserve" else want.compact()
    p = cache.CachePagesParams(op=cache.PAGE_OPS[op], block=16)
    p.page_table, p.lengths, p.refs = tensor(I32, [64, 1, 9, 1]), tensor(I32, [64, 1, 1, 1]), tensor(I32, [3000])
    if op == "reserve":
        p.list = tensor(I32, [64, 1])
    ins = [ints(x) for x in (state.table, state.lengths, state.refs)]
    entries, calls = ints(grow), 300
    outs = [torch.full((calls, *x.shape), -99, device="cuda", dtype=torch.int32) for x in (*ins, ints([0] * 4))]
    scratch = torch.full((cache.query("cache_pages", p).scratch_bytes,), 255, device="cuda", dtype=torch.uint8)
    for i in range(calls):
        cache.cache_pages(p, [x.data_ptr() for x in ins] + [entries.data_ptr() if op == "reserve" else None] + [x[i].data_ptr() for x in outs], scratch.data_ptr())
    torch.cuda.synchronize()
    for got, expected in zip(outs, (want.table, want.lengths, want.refs, report)):
        assert bool((got == ints(expected)).all())


# ---- attention: V scales and values far apart

def scales_in_turn(codes):
    """V scales of neighbouring runs of 16 tokens; under the least scale only zeros, as an append writes them."""
    def spoil(q, caches, scales, tables):
        for run in range(scales[1].shape[2]):
            code = codes[run % len(codes)]
            scales[1][:, :, run] = code
            if code == 0:
                caches[1][:, :, run * 16:run * 16 + 16] = 0
    return spoil


FALLING = [[118, 60, 0, 118], [127, 70, 20, 3], [120, 80, 0, 120], [200, 140, 80, 20], [127, 116, 105, 46]]


FALLING_FROM_FAR = [[240, 170, 100, 30], [241, 161, 81, 1]]      # (448 * 2^114 is below f32's largest)


def check_falling(d, codes):
    for sq, g in ((1, 4), (6, 2), (1, 20)):
        attend_case(d + sq, BF16, d, 2, g, sq, 64, 16, [300, 70, 1000], spoil=scales_in_turn(codes), right=0, bottom_right=True)
    attend_case(d, F16, d, 8, 4, 1, 64, 16, [9000, 100, 6000, 0, 12000, 33, 7000, 2000], spoil=scales_in_turn(codes), o_type=F32)      # all parts
    if d < 256:
        attend_case(d, BF16, d, 1, 4, 50, 64, 16, [300, 70], spoil=scales_in_turn(codes), right=0, bottom_right=True, kernel=UMMA)
        attend_case(d, BF16, d, 1, 4, 50, 64, 16, [3000], spoil=scales_in_turn(codes), right=0, bottom_right=True, kernel=UMMA)         # in pieces


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("codes", FALLING)
def test_scales_that_fall_in_steps(d, codes):
    """V scales that fall by less than 2^80 each and by more together: what was made of the larger ones stays finite."""
    check_falling(d, codes)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("codes", FALLING_FROM_FAR)
def test_scales_that_fall_in_steps_from_far_above_one(d, codes):
    check_falling(d, codes)


def large_values(code):
    def spoil(q, caches, scales, tables):
        caches[1][:] = 0x7E        # 448
        scales[1][:] = code
    return spoil


@pytest.mark.parametrize("code", [218, 228, 244])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_values_far_above_one(d, code):
    """V of 1e30, 2^110 and 2^126 under long sequences: the weights' scale and the number of keys do not reach the results."""
    for lengths, hk, sq in (([16000], 1, 1), ([5000, 16000, 700], 2, 3), ([60] * 512, 8, 1)):      # cut lists, and whole ones
        attend_case(d, BF16, d, hk, 2, sq, 64, 64, lengths, spoil=large_values(code), right=0, bottom_right=True)
    if d < 256:
        attend_case(d, BF16, d, 1, 4, 64, 64, 64, [5000], spoil=large_values(code), right=0, bottom_right=True, kernel=UMMA)
        attend_case(d, BF16, d, 2, 4, 64, 64, 64, [200, 130], spoil=large_values(code), right=0, bottom_right=True, kernel=UMMA)


@pytest.mark.parametrize("code", [1, 20])
def test_values_far_below_one(code):
    """V of 2^-117 and 2^-98, all alike: O is that, to the weights' rounding (2^-11) and, of the smallest, f32's last digits below its normal range (2^-18)."""
    rng = np.random.default_rng(code)
    for d, lengths, hk in ((128, [16000], 1), (64, [60] * 512, 8), (256, [3000, 700], 2)):
        slots = -(-max(lengths) // 64)
        caches, scales = zip(*(cache_of(rng, len(lengths) * slots, hk, 64, 64, d) for _ in range(2)))
        caches[1][:], scales[1][:] = 0x7E, code
        table = torch.from_numpy(table_of(rng, len(lengths), slots, len(lengths) * slots)).cuda()
        q = randn(rng, (len(lengths), hk * 2, 1, d), BF16)
        o, _, _ = run_attend(q, caches, scales, (table, table), ints(lengths), o_type=F32, attn_scale=d ** -0.5 / 64)
        off = (o.double() / (448.0 * 2.0 ** (code - 127)) - 1.0).abs().max().item()
        assert off <= 2.0 ** -11 * 1.01 + 2.0 ** -16, off


def test_absent_pages_beside_small_scales_on_tcgen05():
    """Keys whose V page is none count in the sum alone, however small the scales beside them."""
    def spoil(q, caches, scales, tables):
        scales[1][:] = torch.randint(85, 100, scales[1].shape, device="cuda").to(torch.uint8)
    for d in (64, 128):
        attend_case(d, BF16, d, 2, 4, 40, 64, 16, [300, 170], bad_pages=True, spoil=spoil, right=0, bottom_right=True, kernel=UMMA)
        attend_case(d, F16, d, 1, 4, 64, 64, 16, [3000], bad_pages=True, spoil=spoil, o_type=F32, right=0, bottom_right=True, kernel=UMMA)     # in pieces


@pytest.mark.parametrize("code", [140, 150, 180, 202, 245])
def test_zero_blocks_beside_large_values_on_tcgen05(code):
    """Blocks of zeros with the least scale, and pages that are none, beside V scales far above one: their weights stay in the sum."""
    def spoil(q, caches, scales, tables):
        scales[1][:] = code
        scales[1][:, :, ::2] = 0
        caches[1].view(*caches[1].shape[:2], -1, 2, 16, caches[1].shape[3])[:, :, :, 0] = 0
    for lengths in ([300, 170], [3000]):
        for bad_pages in (False, True):
            attend_case(code, BF16, 128, 1, 4, 64, 64, 16, lengths, bad_pages=bad_pages, spoil=spoil, right=0, bottom_right=True, kernel=UMMA)


@pytest.mark.parametrize("first,second", [(217, 52), (52, 217), (127, 52), (240, 90)])
def test_pieces_of_scales_far_apart_on_tcgen05(first, second):
    """One half of the keys under a V scale far above the other's, neighbours within each piece alike: the sum has the weights of both."""
    def spoil(q, caches, scales, tables):
        scales[1][tables[1][0, :40].long()] = first
        scales[1][tables[1][0, 40:].long()] = second
    for d in (64, 128):
        _, _, info = attend_case(d, BF16, d, 1, 4, 64, 64, 64, [5120], spoil=spoil, kernel=UMMA)
        assert info.launches == 4


@pytest.mark.parametrize("code", [47, 73, 92, 160, 200, 238])
@pytest.mark.parametrize("lengths", [[1, 1, 2, 1, 3, 1, 1, 2], [2100, 1900]])
def test_stats_under_v_scales_far_from_one_on_tcgen05(code, lengths):
    """Stats have nothing to do with V's scales, and no digit is lost to them."""
    def spoil(q, caches, scales, tables):
        scales[1][:] = code
    for seed in range(4):
        attend_case(seed, BF16, 64, 3, 4, 64, 64, 16, lengths, spoil=spoil, right=0, bottom_right=True, kernel=UMMA)


@pytest.mark.parametrize("near,far", [(66, 74), (200, 206), (50, 60)])
def test_stats_over_pieces_under_v_scales_that_differ_on_tcgen05(near, far):
    """Few keys, the last ones in a piece of their own: where the references of two pieces are far from zero, their difference is exact."""
    for behind in (4, 8, 14):
        def spoil(q, caches, scales, tables):
            scales[0][:] = 114
            scales[1][:] = far
            scales[1][tables[1][0, 5248 // 32:].long()] = near
        for seed in range(8):
            _, _, info = attend_case(seed, BF16, 128, 1, 4, 33, 32, 16, [5248 + behind], spoil=spoil, left=10, bottom_right=True, kernel=UMMA)
        assert info.launches == 4


# ---- lists and counts that contradict themselves

@pytest.mark.parametrize("in_place", [False, True])
def test_fork_into_pages_with_negative_counts(in_place):
    """A page whose count fell below 0 is free; a fork that takes it leaves it with a count of one."""
    table, lengths, refs = np.full((3, 4), -1, np.int32), np.array([20, 0, 0], np.int32), np.array([-3, -1, 0, 1, 0, 1], np.int32)
    table[0, :2] = 3, 5
    state = ref.Pages(table, lengths, refs, [np.arange(6 * 8, dtype=np.uint8).reshape(1, 6, 8)], 16)
    (got, got_lengths, got_refs), report, pools = run_pages("fork", state, [[0, 1], [0, 2]], [(1, 8, U8)], in_place=in_place)
    assert got.tolist() == [[3, 5, -1, -1], [3, 0, -1, -1], [3, 1, -1, -1]] and got_lengths.tolist() == [20, 20, 20]
    assert got_refs.tolist() == [1, 1, 0, 3, 0, 1] and report == [2, 2, 2, 0]
    assert np.array_equal(pools[0][0, 0], state.pools[0][0, 5]) and np.array_equal(pools[0][0, 1], state.pools[0][0, 5])


@pytest.mark.parametrize("entries,pairs,refused", [
    ([(0, 5), (1, 5), (2, 1)], [(2, 1)], 1),                # the last entry for 5 is refused, its source being a target: 5 receives nothing
    ([(1, 5), (2, 1), (0, 5)], [(2, 1), (0, 5)], 1),        # the last one stands
    ([(0, 5), (1, 5), (1, 5)], [(1, 5)], 0),                # the same twice
    ([(0, 5), (9, 5), (5, 5)], [(0, 5)], 2),                # ids out of range and equal ones name no target
    ([(0, 5), (5, 0), (1, 0)], [(1, 0)], 2),
    ([(-1, 5), (0, 5), (-2, 5)], [(0, 5)], 0),
])
def test_copy_takes_the_last_entry_of_a_target_alone(entries, pairs, refused):
    rng = np.random.default_rng(0)
    state = ref.Pages(np.full((1, 2), -1, np.int32), np.zeros(1, np.int32), np.array([1, 1, 1, 1, 1, 0, 0, 0], np.int32), [rng.integers(0, 256, (2, 8, 24)).astype(np.uint8)], 16)
    _, report, pools = run_pages("copy", state, entries, [(2, 24, U8)])
    want = state.pools[0].copy()
    for source, target in pairs:
        want[:, target] = state.pools[0][:, source]
    assert np.array_equal(pools[0], want) and report == [3, len(pairs), len(pairs), refused]


# ---- calls beside one another

@pytest.mark.parametrize("kernel,sq", [(cache.SDPA_STREAM, 1), (UMMA, 40)])
def test_two_streams_at_once(kernel, sq):
    """Each with scratch of its own; what one computes does not depend on the other."""
    rng = np.random.default_rng(5)
    calls = []
    for i in range(2):
        caches, scales = zip(*(cache_of(rng, 300, 4, 64, 16, 128) for _ in range(2)))
        table = torch.from_numpy(table_of(rng, 4, 48, 300)).cuda()
        calls.append((randn(rng, (4, 16, sq, 128), BF16), caches, scales, (table, table), ints(rng.integers(sq, 48 * 64, 4))))
    want = [run_attend(*call, kernel=kernel, attn_scale=2.0 ** -10, right=0, bottom_right=True) for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    scratch = [torch.empty(info.scratch_bytes, device="cuda", dtype=torch.uint8) for _, _, info in want]
    outs = [[torch.full_like(o, 77.0) for _ in range(30)] for o, _, _ in want]
    torch.cuda.synchronize()
    for turn in range(30):
        for i, call in enumerate(calls):
            run_attend(*call, kernel=kernel, attn_scale=2.0 ** -10, right=0, bottom_right=True, stream=streams[i].cuda_stream, o=outs[i][turn], stats=False, scratch=scratch[i])
    torch.cuda.synchronize()
    assert dfgpu.device_status() == 0
    for (o, _, _), made in zip(want, outs):
        assert bool(torch.isfinite(o).all()) and all(torch.equal(o, x) for x in made)
