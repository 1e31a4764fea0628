"""The operators of a decoder's step on the GPU against the 64-bit restatement (decoder_reference.py)."""
import numpy as np
import pytest

import decoder_reference as ref
from deepforge_b200 import cache, decoder, dfgpu
from deepforge_b200.decoder import I8
from deepforge_b200.dfgpu import BF16, E4M3, E8M0, F16, F32, I32, I64, U8, contiguous_strides, tensor

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
TORCH = {BF16: torch.bfloat16, F16: torch.float16, F32: torch.float32}
CODE = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.int32: I32, torch.int64: I64, torch.int8: I8, torch.uint8: U8}
U = 2.0 ** -24   # half a step of f32


def half_step(dtype):
    return torch.finfo(TORCH[dtype]).eps / 2


def describe(t):
    return tensor(CODE[t.dtype], list(t.shape), list(t.stride()))


def address(t):
    return None if t is None else t.data_ptr()


def double(t):
    return t.detach().double().cpu().numpy()


def randn(rng, shape, dtype, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape) * scale).to(TORCH[dtype]).cuda()


def ints(values, dtype=torch.int32):
    return torch.tensor(np.asarray(values), dtype=dtype, device="cuda")


# ---- head norms ------------------------------------------------------------------------------------------

class Heads:
    """Rows, gains and positions of one call, and the calls."""

    def __init__(self, seed, b, h, h2, s, d, rotary, dtype=BF16, gain=F32, per_head=False, interleaved=False, scale=1.0, epsilon=1e-6, offset=0.0, kernel=0):
        rng = np.random.default_rng(seed)
        self.dtype, self.interleaved, self.scale, self.epsilon, self.offset, self.kernel = dtype, interleaved, scale, epsilon, offset, kernel
        heads = [h, h2][: 1 + (h2 > 0)]
        self.x = [randn(rng, (b, n, s, d), dtype, 3.0) for n in heads]
        self.dy = [randn(rng, (b, n, s, d), dtype) for n in heads]
        self.gain = [None if gain is None else (1 - offset + randn(rng, (n if per_head else 1, d), F32, 0.3)).to(TORCH[gain]) for n in heads]
        self.positions = ints(rng.integers(0, 2 ** 20, (b, s))) if rotary else None
        self.frequencies = torch.tensor(cache.rope_frequencies(rotary)[0], device="cuda") if rotary else None

    def fill(self, p):
        p.interleaved, p.scale, p.epsilon, p.gain_offset, p.kernel = self.interleaved, self.scale, self.epsilon, self.offset, self.kernel
        if self.positions is not None:
            b, s = self.positions.shape
            p.positions = tensor(CODE[self.positions.dtype], [b, 1, s, 1], [self.positions.stride(0), 1, self.positions.stride(1), 1])
            p.frequencies = tensor(F32, [1, 1, 1, len(self.frequencies)])
        return p

    def gain_descriptor(self, gain):
        return tensor(CODE[gain.dtype], [1, gain.shape[0], 1, gain.shape[1]], [gain.numel(), gain.stride(0), gain.shape[1], 1])

    def forward(self, in_place=False, stream=None, out=None):
        p = self.fill(decoder.HeadNormParams())
        y = out or (self.x if in_place else [torch.full_like(x, 7.0) for x in self.x])
        for n, x, t, g in zip(("", "2"), self.x, y, self.gain):
            setattr(p, "x" + n, describe(x))
            setattr(p, "y" + n, describe(t))
            if g is not None:
                setattr(p, "gain" + n, self.gain_descriptor(g))
        pointers = [address(self.x[0]), address(y[0]), address(self.gain[0]), address(self.positions), address(self.frequencies)]
        if len(y) == 2:
            pointers += [address(self.x[1]), address(y[1]), address(self.gain[1])]
        decoder.head_norm(p, pointers, stream=stream)
        return y

    def gradient(self, out=None, dgain_type=torch.float32, wanted=True, stream=None, scratch=None):
        p = self.fill(decoder.HeadNormGradParams())
        dx = out or [torch.full_like(x, 7.0) for x in self.x]
        dgain = [None] * len(dx)
        for i, (n, x, dy, t, g) in enumerate(zip(("", "2"), self.x, self.dy, dx, self.gain)):
            for field, value in (("x", x), ("dy", dy), ("dx", t)):
                setattr(p, field + n, describe(value))
            if g is not None:
                setattr(p, "gain" + n, self.gain_descriptor(g))
            if wanted:
                dgain[i] = torch.full((1, x.shape[3]) if g is None else g.shape, 7.0, device="cuda", dtype=dgain_type)
                setattr(p, "dgain" + n, self.gain_descriptor(dgain[i]))
        info = decoder.query("head_norm_grad", p)
        room, behind = scratch, None
        if scratch is None:
            room = torch.full((info.scratch_bytes + (1 << 16),), 255, device="cuda", dtype=torch.uint8)
            scratch, behind = room, room[info.scratch_bytes:]
        pointers = [address(self.x[0]), address(self.dy[0]), address(dx[0]), address(self.gain[0]), address(dgain[0]), address(self.positions), address(self.frequencies)]
        if len(dx) == 2:
            pointers += [address(self.x[1]), address(self.dy[1]), address(dx[1]), address(self.gain[1]), address(dgain[1])]
        decoder.head_norm_grad(p, pointers, scratch.data_ptr(), stream=stream)
        if behind is not None:   # no more is written than the query said
            assert torch.all(behind == 255)
        return dx, dgain

    def parts(self, i):
        x, half = double(self.x[i]), 0 if self.frequencies is None else len(self.frequencies)
        gain = np.ones((1, x.shape[3])) if self.gain[i] is None else double(self.gain[i]) + self.offset
        at = np.zeros((x.shape[0], x.shape[2])) if self.positions is None else np.broadcast_to(self.positions.cpu().numpy(), (x.shape[0], x.shape[2]))
        frequencies = np.zeros(0) if self.frequencies is None else self.frequencies.cpu().numpy()
        return x, gain, at, frequencies, half

    def turn_error(self, half):
        return 0 if half == 0 else 5e-7 if self.dtype == F32 else 7.5e-7

    def check_forward(self, y):
        """r: the sum of squares goes through at most 64 additions of a lane and 5 across, rounded up to 70 half steps, half of which reach r; the mean and epsilon
        2, rsqrtf 4: 41 U of r. x r gain: 3 more, the gain with its offset 1. A turn: 5e-7 of |n1| + |n2| (sines of a reduced angle, three roundings) and 2 U
        for the scale; in 16 bits sines and cosines are off by 2^-21.4 = 3.6e-7 and the angle by 1.9e-7 (pi 2^-24), with three roundings 7.5e-7. Then one rounding to the type."""
        for i, got in enumerate(y):
            x, gain, at, frequencies, half = self.parts(i)
            want = ref.head_norm(x, gain, at, frequencies, self.interleaved, self.scale, self.epsilon)
            n = ref.head_norm(x, gain, at, np.zeros(0), epsilon=self.epsilon)
            both = ref.both_of_pair(n, half, self.interleaved) * max(1.0, abs(self.scale))
            bound = (47 * U + self.turn_error(half)) * both + half_step(self.dtype) * np.abs(want) * 1.001 + (2.0 ** -25 if self.dtype == F16 else 0)
            error = np.abs(double(got) - want)
            assert np.all(error <= bound), np.max(error - bound)

    def check_gradient(self, dx, dgain, dgain_type=torch.float32):
        """u: a turn of |dy1| + |dy2| and 2 U. mean(v x): its terms that of the pair's, 3 U, and a sum of 70 additions. r^2 twice 41 U, r once.
        dgain: a term has u's error and 43 U; a CTA's sum at most 128 additions a lane, 5 across, 4 warps, and one rounding, the rest in 64 bits."""
        for i, got in enumerate(dx):
            x, gain, at, frequencies, half = self.parts(i)
            dy = double(self.dy[i])
            want, sums = ref.head_norm_grad(x, dy, gain, at, frequencies, self.interleaved, self.scale, self.epsilon)
            r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + self.epsilon)
            u = ref.both_of_pair(dy, half, self.interleaved) * max(1.0, abs(self.scale))
            off = self.turn_error(half) + 2 * U
            v = u * np.abs(gain)[None, :, None]
            mean = (v * np.abs(x)).mean(-1, keepdims=True)
            bound = r * v * (off + 45 * U) + np.abs(x) * r ** 3 * mean * (off + (75 + 3 * 41 + 6) * U)
            bound += half_step(self.dtype) * np.abs(want) * 1.001 + (2.0 ** -25 if self.dtype == F16 else 0)
            error = np.abs(double(got) - want)
            assert np.all(error <= bound), np.max(error - bound)
            if dgain[i] is None:
                continue
            terms = (u * np.abs(x) * r).sum((0, 2))
            terms = terms if sums.shape[0] > 1 else terms.sum(0, keepdims=True)
            step = torch.finfo(dgain_type).eps / 2
            error = np.abs(double(dgain[i]) - sums)
            bound = terms * (off + (43 + 140) * U) + step * np.abs(sums) * 1.001
            assert np.all(error <= bound), np.max(error - bound)


SHAPES = [(1, 1, 0, 1, 64, 64), (3, 5, 2, 17, 128, 128), (2, 4, 1, 9, 80, 40), (2, 3, 3, 33, 96, 96), (1, 2, 1, 5, 256, 64), (2, 1, 2, 7, 66, 10), (1, 1, 1, 3, 1024, 1024),
          (1, 2, 0, 4, 8, 0), (2, 2, 1, 40, 128, 0), (1, 2, 1, 3, 1000, 0), (2, 1, 0, 3, 2, 2), (1, 3, 1, 2, 1, 0), (2, 17, 5, 35, 128, 64)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,h,h2,s,d,rotary", SHAPES)
def test_head_norm(interleaved, dtype, b, h, h2, s, d, rotary):
    heads = Heads(b * 100 + d, b, h, h2, s, d, rotary, dtype, interleaved=interleaved)
    heads.check_forward(heads.forward())
    heads = Heads(b * 100 + d, b, h, h2, s, d, rotary, dtype, gain=dtype, per_head=True, interleaved=interleaved, scale=1.25, epsilon=1e-3, offset=1.0)
    heads.check_forward(heads.forward())
    heads.kernel = decoder.HEAD_NORM_SCALAR
    heads.check_forward(heads.forward())


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,h,h2,s,d,rotary", SHAPES)
def test_head_norm_gradient(interleaved, dtype, b, h, h2, s, d, rotary):
    heads = Heads(b * 100 + d, b, h, h2, s, d, rotary, dtype, interleaved=interleaved)
    heads.check_gradient(*heads.gradient())
    heads = Heads(b * 100 + d, b, h, h2, s, d, rotary, dtype, gain=dtype, per_head=True, interleaved=interleaved, scale=1.25, epsilon=1e-3, offset=1.0)
    heads.check_gradient(*heads.gradient(dgain_type=TORCH[dtype]), TORCH[dtype])
    heads.kernel = decoder.HEAD_NORM_SCALAR
    heads.check_gradient(*heads.gradient(wanted=False))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_head_norm_strides_and_places(dtype):
    b, h, s, d = 2, 3, 21, 64
    heads = Heads(3, b, h, 2, s, d, 32, dtype)
    heads.positions = ints(np.arange(s)[None] * 1000 - 5000, torch.int64)                     # one row for all sequences, INT64, negative too
    # queries and keys as slices of one buffer, token by token
    both = randn(np.random.default_rng(4), (b, s, h + 2, d + 8), dtype)
    heads.x = [both[:, :, :h, :d].transpose(1, 2), both[:, :, h:, :d].transpose(1, 2)]
    want = heads.forward(out=[torch.empty(b, n, s, d, device="cuda", dtype=TORCH[dtype]) for n in (h, 2)])
    heads.check_forward(want)
    around = both.clone()
    got = heads.forward(in_place=True)
    assert all(torch.equal(g, w) for g, w in zip(got, want)) and torch.equal(both[..., d:], around[..., d:])
    # off every vector boundary, and a broadcast input
    heads = Heads(5, b, h, 0, s, d, 32, dtype)
    flat = randn(np.random.default_rng(6), (b * h * s * d + 1,), dtype)
    aligned = flat[1:].view(b, h, s, d).clone()
    heads.x = [aligned]
    want_y, (want_dx, want_dgain) = heads.forward(), heads.gradient()
    heads.x = [flat[1:].view(b, h, s, d)]
    heads.check_forward(heads.forward())
    heads.check_gradient(*heads.gradient())
    heads.x = [aligned[:1].expand(b, h, s, d)]
    heads.check_forward(heads.forward(out=[torch.empty(b, h, s, d, device="cuda", dtype=TORCH[dtype])]))
    heads.check_gradient(*heads.gradient(out=[torch.empty(b, h, s, d, device="cuda", dtype=TORCH[dtype])]))
    # dX on dY's place, and on X's: the same bits
    for name in ("dy", "x"):
        heads.x, held = [aligned.clone()], [heads.dy[0].clone()]
        heads.dy = held
        dx, dgain = heads.gradient(out=getattr(heads, name))
        assert torch.equal(dx[0], want_dx[0]) and torch.equal(dgain[0], want_dgain[0])
        heads.dy = Heads(5, b, h, 0, s, d, 32, dtype).dy
    assert want_y[0].shape == (b, h, s, d)


def test_head_norm_odd_values():
    """A row of zeros stays zeros (epsilon above 0), a NaN or an infinity stays in its row, and no other row changes."""
    heads = Heads(7, 2, 2, 0, 9, 128, 128, F32)
    want, (want_dx, _) = heads.forward(), heads.gradient()
    heads.x[0][0, 1, 3] = 0
    heads.x[0][1, 0, 4, 5] = float("nan")
    heads.x[0][1, 1, 8, 7] = float("inf")
    got, (dx, _) = heads.forward(), heads.gradient()
    assert torch.all(got[0][0, 1, 3] == 0)
    for y, w in ((got[0], want[0]), (dx[0], want_dx[0])):
        assert torch.isnan(y[1, 0, 4]).all() and torch.isnan(y[1, 1, 8]).any()
        for i, j, k in ((0, 1, 3), (1, 0, 4), (1, 1, 8)):
            y[i, j, k] = w[i, j, k]
        assert torch.equal(y, w)


def test_head_norm_gradient_against_differences():
    """The map is smooth: along e, (f(x + h e) - f(x - h e)) / 2h is <dx, e> up to h^2 and the f32 roundings of f over h."""
    heads = Heads(11, 2, 3, 0, 19, 64, 48, F32, per_head=True, interleaved=True, scale=1.5, epsilon=1e-2)
    (dx,), (dgain,) = heads.gradient()
    e, eg = randn(np.random.default_rng(12), heads.x[0].shape, F32), randn(np.random.default_rng(13), heads.gain[0].shape, F32)
    x, gain, dy, h = heads.x[0].clone(), heads.gain[0].clone(), double(heads.dy[0]), 2.0 ** -8
    values = []
    for sign in (1, -1):
        heads.x[0] = x + sign * h * e
        values.append((double(heads.forward()[0]) * dy))
    heads.x[0] = x
    size = np.abs(values[0]).sum()
    # third derivatives of a row are of the order of its values over |x|^3 (|x| about 3): h^2 / 6 of that, and 60 U of each value over h
    assert abs((values[0] - values[1]).sum() / (2 * h) - (double(dx) * double(e)).sum()) <= size * (h * h / 6 + 60 * U / h)
    values = []
    for sign in (1, -1):
        heads.gain[0] = gain + sign * h * eg
        values.append((double(heads.forward()[0]) * dy))
    assert abs((values[0] - values[1]).sum() / (2 * h) - (double(dgain) * double(eg)).sum()) <= np.abs(values[0]).sum() * 60 * U / h


def test_head_norm_gains_of_one_side_s_heads():
    """Queries with a gain for each head, keys with one for all, and the other way round; a side without any."""
    for order in (1, -1):
        heads = Heads(15, 2, 6, 3, 45, 64, 32, F32)
        whole = Heads(15, 2, 6, 3, 45, 64, 32, F32, per_head=True)
        heads.gain = [whole.gain[0], heads.gain[1]] if order == 1 else [heads.gain[0], whole.gain[1]]
        heads.check_forward(heads.forward())
        heads.check_gradient(*heads.gradient())
        heads.gain[0] = None
        heads.check_forward(heads.forward())
        heads.check_gradient(*heads.gradient())


def test_head_norm_of_many_tokens():
    """So many tokens that a CTA walks all heads of queries and keys, and runs that hold heads of both."""
    for h, h2, s in ((32, 8, 3300), (13, 5, 1700), (3, 9, 700)):
        heads = Heads(16, 3, h, h2, s, 64, 64, BF16)
        heads.check_forward(heads.forward())
        heads = Heads(17, 3, h, h2, s, 64, 32, F32, per_head=True)
        heads.check_forward(heads.forward())


@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_head_norm_gradient_behind_the_last_token(interleaved, per_head):
    """Tokens that do not fill the last CTA: what shared memory held before (here the NaN of a call with NaN frequencies on every SM) does not reach the sums."""
    heads = Heads(18, 3, 8, 2, 1581, 80, 80, F32, interleaved=interleaved, per_head=per_head)
    right = heads.frequencies
    for _ in range(3):
        heads.frequencies = torch.full_like(right, float("nan"))
        heads.gradient()
        heads.frequencies = right
        heads.check_gradient(*heads.gradient())


def test_head_norm_gradient_of_many_tokens():
    """Several runs of heads and tiles of tokens; the same call twice gives the same bits."""
    heads = Heads(14, 3, 40, 8, 500, 128, 128, BF16)
    dx, dgain = heads.gradient()
    heads.check_gradient(dx, dgain)
    again = heads.gradient()
    assert all(torch.equal(a, b) for a, b in zip(dx + dgain, again[0] + again[1]))


def rows_of(heads, i=0):
    """X and dY of one side, to be changed."""
    return heads.x[i], heads.dy[i]


KERNELS = [decoder.HEAD_NORM_VECTOR, decoder.HEAD_NORM_SCALAR]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_head_norm_of_rows_whose_squares_pass_the_range(kernel, per_head, interleaved, dtype):
    """Finite rows whose squares have no f32 sum give zeros, whatever the gain makes of their values before r; so do their gradients where the sum of v x is finite."""
    heads = Heads(23, 2, 3, 2, 5, 64, 32, dtype, per_head=per_head, interleaved=interleaved, kernel=kernel)
    for i in range(2):
        x, _ = rows_of(heads, i)
        heads.gain[i] = 2.0 + heads.gain[i]
        signs = torch.sign(x[0, 1, 2]) + (x[0, 1, 2] == 0)
        x[0, 1, 2], x[1, 0, 4] = 2e38 * signs, 1e20 * signs
    for y in heads.forward():
        assert torch.all(y[0, 1, 2] == 0) and torch.all(y[1, 0, 4] == 0) and torch.isfinite(y).all()
    for i in range(2):
        rows_of(heads, i)[0][0, 1, 2] = 1e20
    dx, dgain = heads.gradient()
    for i in range(2):
        assert torch.all(dx[i][0, 1, 2] == 0) and torch.all(dx[i][1, 0, 4] == 0) and torch.isfinite(dx[i]).all()
        rows_of(heads, i)[1][0, 1, 2] = rows_of(heads, i)[1][1, 0, 4] = 0
    without = heads.gradient()[1]
    assert all(torch.equal(a, b) for a, b in zip(dgain, without))   # (their terms are zeros)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [0, 32])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_head_norm_infinities_stay_in_channels_that_do_not_turn(kernel, per_head, interleaved, rotary, dtype):
    """A channel that no position turns has no partner: an infinity in it is its own NaN (inf * 0) in Y and dgain, and every other value is what the definition says."""
    def fresh():
        return Heads(24, 2, 3, 2, 5, 64, rotary, dtype, per_head=per_head, interleaved=interleaved, kernel=kernel)
    places = [(0, 1, 2, 41), (1, 2, 4, 62)]                          # rows of queries: of either half of a pair's place, head 1 and 2
    channels = torch.arange(64, device="cuda")
    heads, plain = fresh(), fresh()
    for b, h, s, c in places:
        heads.x[0][b, h, s, c] = float("inf")
    y, want = heads.forward(), plain.forward()
    (dx, dgain), still = heads.gradient(), fresh()
    for b, h, s, c in places:
        assert torch.equal(torch.isnan(y[0][b, h, s]), channels == c) and torch.all(y[0][b, h, s][channels != c] == 0)
        assert torch.isnan(dx[0][b, h, s]).all()                    # (r^3 of 0 times a mean of infinity)
        y[0][b, h, s] = want[0][b, h, s]
        still.dy[0][b, h, s] = 0
    assert torch.equal(y[0], want[0]) and torch.equal(y[1], want[1])
    rest = still.gradient()[1]                                       # the other channels' terms of these rows are u x 0 = 0
    hit = torch.zeros_like(dgain[0], dtype=torch.bool)
    for _, h, _, c in places:
        hit[h if per_head else 0, c] = True
    assert torch.equal(torch.isnan(dgain[0]), hit) and torch.equal(dgain[0][~hit], rest[0][~hit]) and torch.equal(dgain[1], rest[1])
    # an infinity in dY: the mean of v x is one, so dX of its row is -x times it, NaN in its own channel; dgain has it in its channel alone
    heads = fresh()
    for b, h, s, c in places:
        heads.dy[0][b, h, s, c] = float("inf")
    (dx, dgain), (want, _) = heads.gradient(), fresh().gradient()
    for b, h, s, c in places:
        x = heads.x[0][b, h, s].float()
        sign = torch.sign(x) * torch.sign(x[c])
        others = (channels != c) & (x != 0)
        assert torch.isnan(dx[0][b, h, s, c]) and torch.equal(dx[0][b, h, s][others].float(), -float("inf") * sign[others])
        dx[0][b, h, s] = want[0][b, h, s]
    assert torch.equal(dx[0], want[0]) and torch.equal(dx[1], want[1])
    assert torch.equal(torch.isinf(dgain[0]), hit) and torch.isfinite(dgain[0][~hit]).all() and torch.isfinite(dgain[1]).all()
    x, gain, at, frequencies, half = heads.parts(0)
    finite = np.where(np.isinf(double(heads.dy[0])), 0.0, double(heads.dy[0]))
    sums = ref.head_norm_grad(x, finite, gain, at, frequencies, interleaved)[1]
    terms = (ref.both_of_pair(finite, half, interleaved) * np.abs(x) / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6)).sum((0, 2))
    terms = terms if per_head else terms.sum(0, keepdims=True)
    keep = ~hit.cpu().numpy()
    assert np.all((np.abs(double(dgain[0]) - sums) <= terms * (heads.turn_error(half) + 185 * U))[keep])   # (as in check_gradient(), for f32 sums)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("per_head", [False, True])
@pytest.mark.parametrize("d,rotary", [(64, 32), (128, 128), (256, 0), (512, 256)])
def test_head_norm_on_8_byte_boundaries(dtype, interleaved, per_head, d, rotary):
    """Rows of 16-bit values that start 8 bytes behind a 16-byte boundary: the launch takes shorter vectors than the scratch was cut for."""
    def moved(t, places):
        flat = torch.full((t.numel() + 8,), 7.0, device="cuda", dtype=t.dtype)
        view = flat[places:places + t.numel()].view(t.shape)
        view.copy_(t)
        return view
    heads = Heads(25, 3, 5, 2, 37, d, rotary, dtype, per_head=per_head, interleaved=interleaved)
    want, (want_dx, want_dgain) = heads.forward(), heads.gradient()
    for tensors in ("x", "dy", "out"):
        again = Heads(25, 3, 5, 2, 37, d, rotary, dtype, per_head=per_head, interleaved=interleaved)
        out = [moved(torch.zeros_like(x), 4 if tensors == "out" else 0) for x in again.x]
        if tensors != "out":
            setattr(again, tensors, [moved(t, 4) for t in getattr(again, tensors)])
        again.kernel = decoder.HEAD_NORM_VECTOR
        again.check_forward(again.forward(out=out))
        again.check_gradient(*again.gradient(out=out))
    assert want[0].shape == want_dx[0].shape and want_dgain[0].shape[1] == d


# ---- 8-bit integers ------------------------------------------------------------------------------------------

def quantize(x, y=None, kernel=0, stream=None):
    p = decoder.TokenQuantizeParams(kernel=kernel)
    y = torch.full(x.shape, 99, device="cuda", dtype=torch.int8) if y is None else y
    scale = torch.full((*x.shape[:-1], 1), 7.0, device="cuda")
    p.x, p.y, p.scale = describe(x), describe(y), describe(scale)
    decoder.token_quantize(p, [x.data_ptr(), y.data_ptr(), scale.data_ptr()], stream=stream)
    return y, scale


def check_codes(x, y, scale):
    """The same f32 quotients: equal bits."""
    want, want_scale = ref.token_quantize(x.float().cpu().numpy())
    assert np.array_equal(scale.cpu().numpy(), want_scale, equal_nan=True)
    assert np.array_equal(y.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 64), (130, 256), (33, 1000), (4, 4096), (2, 8200), (3, 40000), (2, 5, 72), (2, 3, 4, 136), (1, 9, 33)])
def test_token_quantize(dtype, shape):
    x = randn(np.random.default_rng(sum(shape)), shape, dtype, 4.0)
    for kernel in (0, decoder.TOKEN_QUANTIZE_SCALAR):
        check_codes(x, *quantize(x, kernel=kernel))


def test_token_quantize_borders():
    """Halves, the largest magnitude with either sign, rows of zeros, of subnormals, with an infinity and a NaN, and far-apart magnitudes."""
    x = torch.zeros(12, 264, device="cuda")
    steps = torch.arange(-127, 128, device="cuda").float()
    x[0, :255], x[1, :255] = steps, steps - torch.sign(steps) * 0.5
    x[1, 255], x[2, 0], x[3, 0], x[4, 7] = 127.0, -3.0, 1e-44, 6e-42
    x[4, 8], x[5, 3], x[6, 5], x[7, 9], x[7, 10] = -3e-42, float("inf"), float("nan"), 3e38, -1e-38
    x[8] = torch.randn(264, device="cuda") * 1e-39
    x[9] = (torch.randn(264, device="cuda") * 2).exp2() * 1e30
    x[10, :255], x[10, 255] = (steps + 0.5) * 0.0371, 127 * 0.0371
    x[11, 1] = -0.0
    check_codes(x, *quantize(x))
    for dtype in (torch.bfloat16, torch.float16):
        check_codes(x.to(dtype), *quantize(x.to(dtype)))


def test_token_quantize_strides():
    rng = np.random.default_rng(2)
    base = randn(rng, (6, 5, 80), BF16)
    x = base[:, :, :64].transpose(0, 1)
    y = torch.full((5, 6, 80), 99, device="cuda", dtype=torch.int8)
    got, scale = quantize(x, y[:, :, :64])
    check_codes(x, got, scale)
    assert torch.all(y[:, :, 64:] == 99)
    flat = randn(rng, (3 * 128 + 1,), BF16)
    check_codes(flat[1:].view(3, 128), *quantize(flat[1:].view(3, 128)))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,k", [(3, 40001), (300, 4097), (301, 577), (400, 9), (2, 15), (310, 2305), (299, 1)])
def test_token_quantize_of_rows_anywhere(dtype, rows, k):
    """Rows that start on any element and end inside a vector, codes that start on any byte; what lies around them stays and is not looked at."""
    rng = np.random.default_rng(k)
    for shift, codes_shift, pitch in ((0, 0, k), (1, 0, (k + 15) // 16 * 16 + 16), (3, 5, k + 2), (2, 3, k)):
        base = torch.full((rows * pitch + 8,), float("nan"), device="cuda", dtype=TORCH[dtype])
        x = base[shift:].as_strided((rows, k), (pitch, 1))
        x.copy_(randn(rng, (rows, k), dtype, 3.0))
        around = torch.full((rows * (k + 3) + 8,), 99, device="cuda", dtype=torch.int8)
        y = around[codes_shift:].as_strided((rows, k), (k + 3, 1))
        got, scale = quantize(x, y)
        check_codes(x.contiguous(), got, scale)
        mask = torch.ones_like(around, dtype=torch.bool)
        mask[codes_shift:].as_strided((rows, k), (k + 3, 1)).fill_(False)
        assert torch.all(around[mask] == 99)


def int8s(rng, shape):
    return torch.from_numpy(rng.integers(-128, 128, shape).astype(np.int8)).cuda()


def product(a, b, a_scale, b_scale, dtype, bias=None, kernel=0, c=None, stream=None):
    p = decoder.MatmulInt8Params(kernel=kernel)
    c = torch.full((*a.shape[:-1], b.shape[-1]), 7.0, device="cuda", dtype=TORCH[dtype]) if c is None else c
    p.a, p.b, p.c, p.a_scale, p.b_scale = (describe(t) for t in (a, b, c, a_scale, b_scale))
    if bias is not None:
        p.bias = describe(bias)
    decoder.matmul_int8(p, [address(t) for t in (a, b, c, a_scale, b_scale, bias)], stream=stream)
    return c


def check_product(c, a, b, a_scale, b_scale, bias=None):
    """Integers are exact and the roundings in a given order: equal bits."""
    f32 = lambda t: t.float().cpu().numpy()  # noqa: E731
    want = ref.matmul_int8(a.cpu().numpy(), b.cpu().numpy(), f32(a_scale), f32(b_scale), None if bias is None else f32(bias))
    assert torch.equal(c.cpu(), torch.from_numpy(want).to(c.dtype)), (c.cpu().double() - torch.from_numpy(want).double()).abs().max()
    assert dfgpu.device_status() == 0


def scales(rng, shape):
    return torch.from_numpy(np.exp2(rng.uniform(-12, -4, shape)).astype(np.float32)).cuda()


def rows16(codes):
    """The same codes with rows on 16-byte boundaries."""
    wide = torch.full((*codes.shape[:-1], (codes.shape[-1] + 15) // 16 * 16), 99, device="cuda", dtype=torch.int8)
    wide[..., : codes.shape[-1]] = codes
    return wide[..., : codes.shape[-1]]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 64, 16), (3, 70, 33), (16, 128, 128), (17, 200, 1000), (64, 4096, 512), (128, 128, 4096), (129, 257, 300), (300, 192, 640), (256, 256, 128), (700, 1111, 250),
                                   (1000, 520, 1024), (2300, 2048, 200)])
def test_matmul_int8(dtype, m, n, k):
    rng = np.random.default_rng(m + n + k)
    a, b = rows16(int8s(rng, (m, k))), rows16(int8s(rng, (n, k))).T
    a_scale, b_scale = scales(rng, (m, 1)), scales(rng, (1, n))
    bias = randn(rng, (1, n), dtype)
    check_product(product(a, b, a_scale, b_scale, dtype, kernel=decoder.MATMUL_INT8_UMMA), a, b, a_scale, b_scale)
    check_product(product(a, b, a_scale, b_scale, dtype, bias, kernel=decoder.MATMUL_INT8_UMMA), a, b, a_scale, b_scale, bias)
    check_product(product(a, b, a_scale, b_scale, dtype, bias, kernel=decoder.MATMUL_INT8_CORES), a, b, a_scale, b_scale, bias)


@pytest.mark.parametrize("m,n,k", [(5, 96, 70), (130, 300, 384), (600, 1040, 1000)])
def test_matmul_int8_layouts(m, n, k):
    """B with N contiguous, one scale for all, C off the 16-byte boundaries, operands off theirs, A transposed."""
    rng = np.random.default_rng(m)
    a, b = rows16(int8s(rng, (m, k))), rows16(int8s(rng, (k, n)))
    a_scale, b_scale = scales(rng, (m, 1)), scales(rng, (1, n))
    check_product(product(a, b, a_scale, b_scale, BF16, kernel=decoder.MATMUL_INT8_UMMA), a, b, a_scale, b_scale)
    one = scales(rng, (1, 1))
    check_product(product(a, b, one, one, F32, kernel=decoder.MATMUL_INT8_UMMA), a, b, one, one)
    wide = torch.full((m, n + 3), 7.0, device="cuda", dtype=torch.float16)
    got = product(a, b, a_scale, b_scale, F16, c=wide[:, :n])
    check_product(got, a, b, a_scale, b_scale)
    assert torch.all(wide[:, n:] == 7.0)
    odd = torch.empty(m * k + 1, device="cuda", dtype=torch.int8)[1:].view(m, k)
    odd.copy_(a)
    check_product(product(odd, b, a_scale, b_scale, BF16), odd, b, a_scale, b_scale)
    turned = a.T.contiguous().T
    every = scales(rng, (2 * m, 3))[::2, :1]
    check_product(product(turned, b, every, b_scale, BF16), turned, b, every, b_scale)
    bias = randn(rng, (1, 2 * n), F32)[:, ::2]
    check_product(product(a, b, a_scale, b_scale, BF16, bias), a, b, a_scale, b_scale, bias)


def test_matmul_int8_batches_and_extremes():
    rng = np.random.default_rng(9)
    a, b = int8s(rng, (3, 5, 64)), int8s(rng, (1, 48, 64)).transpose(1, 2)
    a_scale, b_scale = scales(rng, (3, 5, 1)), scales(rng, (1, 1, 48))
    check_product(product(a, b, a_scale, b_scale, BF16), a, b, a_scale, b_scale)                      # folds into 15 rows
    each = int8s(rng, (3, 48, 64)).transpose(1, 2)
    check_product(product(a, each, a_scale, b_scale, BF16), a, each, a_scale, b_scale)                # a matrix for each
    group = scales(rng, (3, 1, 1))
    check_product(product(a, each, group, b_scale, F32), a, each, group, b_scale)
    step = int8s(rng, (4, 1, 64))
    one = scales(rng, (4, 1, 1))
    check_product(product(step, b, one, b_scale, F16), step, b, one, b_scale)                          # a token for each of four users
    # the largest sums of the greatest depth, on both kernels
    deep = torch.full((2, 131071), -128, device="cuda", dtype=torch.int8)
    deep[1] = 127
    wide = rows16(deep)
    unit = torch.ones(1, 1, device="cuda")
    for kernel in (decoder.MATMUL_INT8_UMMA, decoder.MATMUL_INT8_CORES):
        check_product(product(wide, wide.T, unit, unit, F32, kernel=kernel), wide, wide.T, unit, unit)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 17, 15), (2, 16, 16), (7, 33, 63), (8, 130, 64), (9, 64, 65), (16, 15, 100), (11, 200, 1000), (15, 96, 511), (16, 1111, 513), (16, 40, 4100), (3, 4099, 2048), (1, 16, 131071)])
def test_matmul_int8_of_few_tokens(dtype, m, n, k):
    rng = np.random.default_rng(m + n + k)
    a, b = rows16(int8s(rng, (m, k))), rows16(int8s(rng, (n, k))).T
    a_scale, b_scale = scales(rng, (m, 1)), scales(rng, (1, n))
    bias = randn(rng, (1, 2 * n), F32)[:, ::2]
    few = decoder.MATMUL_INT8_FEW
    wide = torch.full((m + 1, n + 3), 7.0, device="cuda", dtype=TORCH[dtype])
    check_product(product(a, b, a_scale, b_scale, dtype, c=wide[:m, :n], kernel=few), a, b, a_scale, b_scale)
    assert torch.all(wide[m] == 7.0) and torch.all(wide[:, n:] == 7.0)
    check_product(product(a, b, a_scale, b_scale, dtype, bias, kernel=few), a, b, a_scale, b_scale, bias)
    every, one = scales(rng, (2 * m, 3))[::2, :1], scales(rng, (1, 1))
    check_product(product(a, b, every, one, dtype, kernel=few), a, b, every, one)
    turned = torch.full((n, m), 7.0, device="cuda", dtype=TORCH[dtype]).T
    check_product(product(a, b, a_scale, b_scale, dtype, c=turned, kernel=few), a, b, a_scale, b_scale)
    # an infinite scale (a row with an infinity) and that of a NaN reach their own row alone
    a_scale[m - 1] = float("nan")
    got = product(a, b, a_scale, b_scale, dtype, kernel=few)
    assert torch.all(torch.isnan(got[m - 1]))
    if m > 1:
        check_product(got[: m - 1], a[: m - 1], b, a_scale[: m - 1], b_scale)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("m,n,k", [(20, 70, 100), (130, 300, 384), (64, 1111, 2048), (600, 1040, 200)])
def test_matmul_int8_scales_of_the_tensor_cores_anywhere(dtype, m, n, k):
    """tcgen05 with scales of rows and columns that lie apart, that start on any float, and one for all of either side; whole and split K."""
    rng = np.random.default_rng(m * n)
    a, b = rows16(int8s(rng, (m, k))), rows16(int8s(rng, (n, k))).T
    every_row, every_column = scales(rng, (3 * m, 2))[::3, 1:], scales(rng, (1, 2 * n + 1))[:, 1::2]
    row, column = scales(rng, (m + 1, 1))[1:], scales(rng, (1, n + 1))[:, 1:]
    one = scales(rng, (1, 1))
    bias = randn(rng, (1, n + 1), dtype)[:, 1:]
    for a_scale, b_scale in ((every_row, every_column), (row, column), (every_row, one), (one, every_column), (row, every_column), (every_row, column)):
        for more in (None, bias):
            check_product(product(a, b, a_scale, b_scale, dtype, more, kernel=decoder.MATMUL_INT8_UMMA), a, b, a_scale, b_scale, more)


# ---- beam search ---------------------------------------------------------------------------------------------

def select(logits, scores, finished=None, lengths=None, penalty=0.0, end=-1, pad=0, bases=None, in_place=False, stream=None, scratch=None):
    p = decoder.BeamSelectParams(length_penalty=penalty, end=end, pad=pad)
    b, w, _ = logits.shape
    whole = lambda: torch.full((b, w), 77, device="cuda", dtype=torch.int32)  # noqa: E731
    out = {"scores_out": scores if in_place else torch.full((b, w), 7.0, device="cuda"), "tokens": whole(), "parents": whole(),
           "finished_out": finished if in_place and finished is not None else whole(), "lengths_out": None if lengths is None else lengths if in_place else whole(),
           "forks": None if bases is None else torch.full((b * w, 2), 77, device="cuda", dtype=torch.int32)}
    given = {"logits": logits, "scores": scores, "finished": finished, "lengths": lengths, **out}
    for name, t in given.items():
        if t is not None:
            setattr(p, name, describe(t))
    if bases is not None:
        p.source_base, p.target_base = bases
    behind = None
    if scratch is None:
        size = decoder.query("beam_select", p).scratch_bytes
        scratch = torch.full((size + 4096,), 255, device="cuda", dtype=torch.uint8)
        behind = scratch[size:]
    decoder.beam_select(p, [address(given[n]) for n in ("logits", "scores", "finished", "lengths", "scores_out", "tokens", "parents", "finished_out", "lengths_out", "forks")],
                        scratch.data_ptr(), stream=stream)
    assert behind is None or torch.all(behind == 255)   # no more is written than the query said
    return out


def check_select(out, logits, scores, finished=None, lengths=None, penalty=0.0, end=-1, pad=0):
    """Choices are equal. Scores: a thread's sum of at most 32 additions, each term 4 U (exponential) and the two roundings of its argument and that of log2 e, which weigh
    at most |d| e^d and so no more than the entropy (below 13) in the sum, 3 U of each: 75 U together; then the rounding to f32."""
    numpy = lambda t: None if t is None else t.cpu().numpy()  # noqa: E731
    want = ref.beam_select(double(logits), double(scores), numpy(finished), numpy(lengths), penalty, end, pad)
    assert np.array_equal(out["tokens"].cpu().numpy(), want[1]) and np.array_equal(out["parents"].cpu().numpy(), want[2])
    got = double(out["scores_out"])
    infinite = np.isinf(want[0])
    assert np.array_equal(got[infinite], want[0][infinite])
    assert np.all(np.abs(got[~infinite] - want[0][~infinite]) <= 75 * U + 1.001 * U * np.abs(want[0][~infinite]))
    assert np.array_equal(out["finished_out"].cpu().numpy(), want[3])
    if lengths is not None:
        assert np.array_equal(out["lengths_out"].cpu().numpy(), want[4])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,w,v", [(1, 1, 1), (1, 4, 1), (2, 3, 2), (3, 4, 7), (1, 32, 40), (2, 5, 1001), (5, 8, 2048), (1, 4, 32000), (2, 32, 5000), (3, 2, 50001), (40, 8, 9000), (16, 12, 20001)])
def test_beam_select(dtype, b, w, v):
    rng = np.random.default_rng(b + w + v)
    logits, scores = randn(rng, (b, w, v), dtype, 3.0), randn(rng, (b, w), F32, 4.0) - 20
    check_select(select(logits, scores), logits, scores)
    finished, lengths = ints(rng.integers(0, 4, (b, w)) == 0), ints(rng.integers(0, 60, (b, w)))
    more = dict(finished=finished, lengths=lengths, penalty=0.7, end=v // 2, pad=v - 1)
    check_select(select(logits, scores, **more), logits, scores, **more)
    want = select(logits, scores, **more)
    held = {"finished": finished.clone(), "lengths": lengths.clone()}
    got = select(logits, scores.clone(), penalty=0.7, end=v // 2, pad=v - 1, in_place=True, **held)
    assert all(torch.equal(got[n], want[n]) for n in want if want[n] is not None)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_beam_select_equals_and_masks(dtype):
    rng = np.random.default_rng(5)
    b, w, v = 6, 4, 3001
    logits, scores = torch.zeros(b, w, v, device="cuda", dtype=TORCH[dtype]), torch.zeros(b, w, device="cuda") - 3
    logits[1] = randn(rng, (1, v), dtype).expand(w, v)                                       # four equal beams
    logits[2] = randn(rng, (w, v), dtype)
    scores[2, 1:] = -float("inf")                                                             # the first step: one beam lives
    logits[3] = -float("inf")
    logits[3, 2, 5], logits[3, 1, 2900], logits[3, 2, 1] = 1.0, 2.0, 0.5                      # all but three masked
    logits[4] = randn(rng, (w, v), dtype)
    logits[4, 0, 17], logits[4, 2, 9] = float("nan"), float("inf")                            # two beams without a sum
    logits[4, 3] = -float("inf")
    logits[5] = -1e4 + randn(rng, (w, v), dtype)                                              # far below zero, with a part that is masked
    logits[5, :, :2500] = -float("inf")
    check_select(select(logits, scores), logits, scores)
    steps = torch.round(4 * randn(rng, (b, w, v), F32)).to(TORCH[dtype])                      # many equals in every beam
    check_select(select(steps, scores), steps, scores)
    for value in (float("inf"), float("nan"), -float("inf")):
        scores[:, :] = value
        check_select(select(steps, scores), steps, scores)
    largest = torch.full((1, 2, 600), -3e38, device="cuda")
    largest[0, 0, 3], largest[0, 1, 500] = 3e38, 1.0                                          # the ends of f32
    check_select(select(largest, torch.zeros(1, 2, device="cuda")), largest, torch.zeros(1, 2, device="cuda"))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("b,w,v", [(9, 4, 40001), (2, 32, 40001), (45, 8, 20001), (9, 1, 3000), (300, 2, 9000)])
def test_beam_select_of_few_values_that_count(dtype, b, w, v):
    """Masks that leave next to nothing, equal rows, and large values in few lanes: the bound is reached by far more values than are wanted."""
    rng = np.random.default_rng(b * w)
    logits, scores = randn(rng, (b, w, v), dtype), randn(rng, (b, w), F32)
    token = torch.arange(v, device="cuda")
    for entry in range(b):
        x, kind = logits[entry], entry % 9 if b > 2 else 5 * entry
        keep = torch.from_numpy(rng.random((w, v)) < 5 / v).cuda()
        if kind == 0:
            x.masked_fill_(~keep, -float("inf"))
        elif kind == 1:
            x.masked_fill_(~keep, torch.finfo(x.dtype).min)
        elif kind == 2:
            x.fill_(1.0)
        elif kind == 3:
            x.fill_(-2.0)
            x[:, -10:] = 2.0
        elif kind == 4:
            x.copy_(torch.round(x))
        elif kind == 5:   # two lanes of a warp have all the large ones
            x[:, (token * x.element_size() // 16 % 32 == 3) | (token * x.element_size() // 16 % 32 == 17)] += 8.0
        elif kind == 6:
            x.masked_fill_(torch.from_numpy(rng.random((w, v)) < 0.5).cuda(), -float("inf"))
        elif kind == 7:
            x.copy_(torch.where(x > 0, 0.0, -0.0))
        else:
            x.masked_fill_(token != v - 1, -float("inf"))
    check_select(select(logits, scores), logits, scores)


def test_beam_select_strides_and_forks():
    rng = np.random.default_rng(6)
    b, w, v = 3, 5, 700
    base = randn(rng, (w, b, v + 3), BF16)
    logits = base[:, :, 1:v + 1].transpose(0, 1)                                               # beams apart, rows on odd places
    scores = randn(rng, (b, 2 * w), F32)[:, ::2]
    out = select(logits, scores, bases=(100, 7))
    check_select(out, logits, scores)
    forks = out["forks"].view(b, w, 2)
    at = torch.arange(b, device="cuda")[:, None] * w
    assert torch.equal(forks[..., 0], 100 + at + out["parents"]) and torch.equal(forks[..., 1], 7 + at + torch.arange(w, device="cuda"))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("b,w,v", [(2, 3, 7), (3, 4, 5001), (40, 8, 3001)])
def test_beam_select_lengths_and_finished_apart(dtype, b, w, v):
    """Lengths without flags of what is finished, and flags without lengths; in place too."""
    rng = np.random.default_rng(b * v)
    logits, scores = randn(rng, (b, w, v), dtype, 3.0), randn(rng, (b, w), F32, 4.0) - 20
    finished, lengths = ints(rng.integers(0, 3, (b, w)) == 0), ints(rng.integers(0, 60, (b, w)))
    for more in (dict(lengths=lengths, penalty=0.7, end=v // 2), dict(lengths=lengths), dict(finished=finished, end=v // 2, pad=v - 1)):
        want = select(logits, scores, **more)
        check_select(want, logits, scores, **more)
        held = {n: t.clone() if torch.is_tensor(t) else t for n, t in more.items()}
        got = select(logits, scores.clone(), in_place=True, **held)
        assert all(torch.equal(got[n], want[n]) for n in want if want[n] is not None)


@pytest.mark.parametrize("dtype", [torch.uint8, torch.bfloat16, torch.float32, torch.int64])
@pytest.mark.parametrize("layers,b,w,n", [(1, 1, 1, 1), (2, 3, 4, 7), (1, 16, 8, 1000), (3, 2, 5, 4096), (2, 1, 32, 33333), (5, 7, 3, 16)])
def test_beam_reorder(dtype, layers, b, w, n):
    rng = np.random.default_rng(n)
    parents = ints(rng.integers(0, w, (b, w)))
    states = [torch.from_numpy(rng.integers(0, 256, (layers, b, w, m, torch.empty(0, dtype=dtype).element_size())).astype(np.uint8)).cuda().view(dtype)[..., 0] for m in (n, 2 * n + 1)]
    states[1] = states[1][..., 1:]                                                             # rows off the boundaries, apart
    targets = [torch.zeros(t.shape, device="cuda", dtype=dtype) for t in states]
    wanted = [torch.gather(t, 2, parents.long()[None, :, :, None].expand(t.shape)) for t in states]
    p = decoder.BeamReorderParams(count=2)
    p.parents = describe(parents)
    for i in range(2):
        p.source[i], p.target[i] = describe(states[i]), describe(targets[i])
    decoder.beam_reorder(p, [parents.data_ptr(), states[0].data_ptr(), targets[0].data_ptr(), states[1].data_ptr(), targets[1].data_ptr()])
    for got, want in zip(targets, wanted):
        assert torch.equal(got.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


def test_beam_reorder_leaves_rows_of_bad_parents():
    parents = ints([[0, 3, -1], [2, 1, 1000000]])
    source = torch.arange(2 * 3 * 40, device="cuda", dtype=torch.int32).view(1, 2, 3, 40)
    target = torch.full_like(source, 5)
    p = decoder.BeamReorderParams(count=1)
    p.parents, p.source[0], p.target[0] = describe(parents), describe(source), describe(target)
    decoder.beam_reorder(p, [parents.data_ptr(), source.data_ptr(), target.data_ptr()])
    want = torch.full_like(source, 5)
    want[0, 0, 0], want[0, 1, 0], want[0, 1, 1] = source[0, 0, 0], source[0, 1, 2], source[0, 1, 1]
    assert torch.equal(target, want)


@pytest.mark.parametrize("penalty", [28.0, -28.0])
def test_beam_select_penalties_at_the_ends(penalty):
    """The largest penalties with the longest lengths: worths stay within 64 bits, and scores come out of them whole; finished beams of score 0 too."""
    rng = np.random.default_rng(8)
    logits, scores = randn(rng, (4, 3, 50), F32, 3.0), randn(rng, (4, 3), F32) - 5
    scores[0], scores[1, 0], scores[2] = 0.0, -3e38, -1e-38
    lengths, finished = ints([[0x7FFFFFFF, 0x7FFFFFFE, 1], [2, 3, 4], [0x7FFFFFFF] * 3, [-5, 0, 100]]), ints([[1, 0, 1], [0, 0, 1], [1, 1, 0], [0, 0, 0]])
    more = dict(finished=finished, lengths=lengths, penalty=penalty, end=7, pad=3)
    out = select(logits, scores, **more)
    assert torch.isfinite(out["scores_out"]).all()
    want = ref.beam_select(double(logits), double(scores), finished.cpu().numpy(), lengths.cpu().numpy(), penalty, 7, 3)
    assert np.array_equal(out["tokens"].cpu().numpy(), want[1]) and np.array_equal(out["parents"].cpu().numpy(), want[2])
    # (as in check_select(), with three roundings of 64 bits for quotient, power and product)
    assert np.all(np.abs(double(out["scores_out"]) - want[0]) <= 75 * U + 1.001 * U * np.abs(want[0]))


# ---- streams and graphs -------------------------------------------------------------------------------------------

def test_two_streams_and_graphs():
    """Every operator captured into graphs that run on two streams at once, each with its own buffers; replayed with new inputs."""
    rng = np.random.default_rng(20)

    class Work:
        def __init__(self, seed):
            self.heads = Heads(seed, 2, 8, 2, 70, 128, 128, BF16)
            self.x, self.weights = randn(rng, (70, 512), BF16), rows16(int8s(rng, (320, 512)))
            self.weight_scale = scales(rng, (1, 320))
            self.logits, self.scores = randn(rng, (4, 6, 9001), BF16, 3.0), randn(rng, (4, 6), F32)
            self.scratch = torch.empty(1 << 20, device="cuda", dtype=torch.uint8)
            self.more = torch.empty(1 << 20, device="cuda", dtype=torch.uint8)

        def run(self, stream):
            y = self.heads.forward(stream=stream)
            dx, dgain = self.heads.gradient(stream=stream, scratch=self.more)
            codes, scale = quantize(self.x, stream=stream)
            c = product(codes, self.weights.T, scale, self.weight_scale, BF16, stream=stream)
            out = select(self.logits, self.scores, stream=stream, scratch=self.scratch)
            return y + dx + dgain + [codes, scale, c, out["scores_out"], out["tokens"], out["parents"]]

    works = [Work(21), Work(22)]
    streams = [torch.cuda.Stream() for _ in works]
    graphs, results = [], []
    for work, stream in zip(works, streams):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            work.run(stream.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            results.append(work.run(stream.cuda_stream))
        graphs.append(graph)
    for seed in (31, 32):
        fresh = np.random.default_rng(seed)
        for work in works:
            for t in (*work.heads.x, *work.heads.dy, work.x, work.logits, work.scores):
                t.copy_(torch.from_numpy(fresh.standard_normal(t.shape)).to(t.dtype))
        torch.cuda.synchronize()
        for _ in range(3):
            for graph, stream in zip(graphs, streams):
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for work, got in zip(works, results):
            got = [t.clone() for t in got]
            torch.cuda.synchronize()
            want = work.run(torch.cuda.current_stream().cuda_stream)
            assert all(torch.equal(g, w) for g, w in zip(got, want))
            check_select({"scores_out": got[-3], "tokens": got[-2], "parents": got[-1], "finished_out": torch.zeros_like(got[-1])}, work.logits, work.scores)
    assert dfgpu.device_status() == 0


# ---- together ------------------------------------------------------------------------------------------------------

def linear(x, weights, weight_scale):
    codes, scale = quantize(x, torch.zeros(*x.shape, device="cuda", dtype=torch.int8))
    return product(codes, weights.T, scale, weight_scale, BF16)


def test_a_beam_search_over_the_paged_cache():
    """A decoder of one layer: projections in 8 bits, norms and positions, the cache's append and attention, logits, selection, FORK and FREE, and histories that
    follow their beams. After each step every beam's cache holds its parent's codes, attention is that of 64 bits over them, and the histories are the backward walk."""
    rng = np.random.default_rng(50)
    b, w, hk, group, d, vocabulary, page, slots, pages, steps = 2, 3, 2, 4, 64, 301, 16, 4, 64, 20
    rows, model, heads = b * w, 128, hk * group
    table_weights = randn(rng, (vocabulary, model), BF16)
    weights = {n: quantize(randn(rng, (m, model), BF16)) for n, m in (("qkv", (heads + 2 * hk) * d), ("logits", vocabulary))}
    out_codes, out_scale = quantize(randn(rng, (model, heads * d), BF16))
    gains = [1 + randn(rng, (1, d), F32, 0.2) for _ in range(2)]
    frequencies = torch.tensor(cache.rope_frequencies(d)[0], device="cuda")
    # two sets of sequences: the beams live in one, their continuations are forked into the other
    containers = [torch.zeros(pages, hk, page, d, device="cuda", dtype=torch.uint8) for _ in range(2)]
    block_scales = [torch.zeros(pages, hk, 1, 1, device="cuda", dtype=torch.uint8) for _ in range(2)]
    table, lengths, refs = ints(np.full((2 * rows, slots), -1)), ints(np.zeros(2 * rows)), ints(np.zeros(pages))
    report = ints(np.zeros(4))
    tokens, scores = ints(rng.integers(0, vocabulary, (b, w))), torch.tensor([[0.0] + [-float("inf")] * (w - 1)] * b, device="cuda")
    tokens[:, 1:] = tokens[:, :1]
    finished, counts = ints(np.zeros((b, w))), ints(np.zeros((b, w)))
    history = [torch.full((1, b, w, steps), -1, device="cuda", dtype=torch.int32) for _ in range(2)]
    walked, base = [], 0

    def pages_call(op, entries=None, pools=()):
        p = cache.CachePagesParams(op=cache.PAGE_OPS[op], block=page, pool_count=len(pools))
        p.page_table, p.lengths, p.refs = tensor(I32, [2 * rows, 1, slots, 1]), tensor(I32, [2 * rows, 1, 1, 1]), tensor(I32, [pages])
        p.list = tensor(I32, list(entries.shape))
        for i, pool in enumerate(pools):
            p.pools[i] = tensor(U8, [1, pages, pool.numel() // pages])
        scratch = torch.empty(max(16, cache.query("cache_pages", p).scratch_bytes), device="cuda", dtype=torch.uint8)
        cache.cache_pages(p, [address(t) for t in (table, lengths, refs, entries, table, lengths, refs, report, *pools)], scratch.data_ptr())
        assert report[3].item() == 0

    def held_codes(sequence):
        n = int(lengths[sequence])
        ids = table[sequence, torch.arange(n, device="cuda") // page].long()
        at = torch.arange(n, device="cuda") % page
        return [(c[ids, :, at].clone(), s[ids, :, 0, 0].clone()) for c, s in zip(containers, block_scales)]

    for step in range(steps):
        live = slice(base, base + rows)
        x = table_weights[tokens.view(-1).long()]
        qkv = linear(x, weights["qkv"][0], weights["qkv"][1].view(1, -1)).view(rows, 1, heads + 2 * hk, d)
        q, k, v = (qkv[:, :, s].transpose(1, 2) for s in (slice(0, heads), slice(heads, heads + hk), slice(heads + hk, None)))
        p = decoder.HeadNormParams(epsilon=1e-6)
        p.x = p.y = describe(q)
        p.x2 = p.y2 = describe(k)
        p.gain = p.gain2 = tensor(F32, [1, 1, 1, d])
        p.positions, p.frequencies = tensor(I32, [rows, 1, 1, 1]), tensor(F32, [1, 1, 1, d // 2])
        decoder.head_norm(p, [address(t) for t in (q, q, gains[0], lengths[live], frequencies, k, k, gains[1])])
        need = torch.zeros(2 * rows, 1, device="cuda", dtype=torch.int32)
        need[live] = 1
        pages_call("reserve", need)
        p = cache.CacheAppendParams()
        p.k, p.v = describe(k), describe(v)
        p.k_cache = p.v_cache = tensor(E4M3, list(containers[0].shape))
        p.k_scale = p.v_scale = tensor(E8M0, list(block_scales[0].shape))
        p.page_table_k = p.page_table_v = tensor(I32, [rows, 1, slots, 1])
        p.lengths = p.lengths_out = tensor(I32, [rows, 1, 1, 1])
        cache.cache_append(p, [address(t) for t in (k, v, *containers, *block_scales, table[live], table[live], lengths[live], None, lengths[live])])
        p = cache.CacheSdpaParams(attn_scale=d ** -0.5, s_kv=slots * page)
        o = torch.empty(rows, heads, 1, d, device="cuda", dtype=torch.bfloat16)
        p.q, p.o = describe(q), describe(o)
        p.k = p.v = tensor(E4M3, list(containers[0].shape))
        p.k_scale = p.v_scale = tensor(E8M0, list(block_scales[0].shape))
        p.page_table_k = p.page_table_v = tensor(I32, [rows, 1, slots, 1])
        p.seq_kv = tensor(I32, [rows, 1, 1, 1])
        scratch = torch.empty(max(16, cache.query("cache_sdpa", p).scratch_bytes), device="cuda", dtype=torch.uint8)
        cache.cache_sdpa(p, [address(q), *map(address, containers), address(o), None, *map(address, block_scales), None, address(lengths[live]), address(table[live]), address(table[live])], scratch.data_ptr())
        for row in range(rows):   # probabilities in f16 (2^-11), O in bf16 (2^-8), K and V exact: 2^-8 of the largest |v| and a little more
            (kc, ks), (vc, vs) = held_codes(base + row)
            keys, values = (c.view(torch.float8_e4m3fn).double() * torch.exp2(s.double() - 127)[:, :, None] for c, s in ((kc, ks), (vc, vs)))
            for h in range(heads):
                weight = torch.softmax(keys[:, h // group] @ q[row, h, 0].double() / d ** 0.5, 0)
                want = weight @ values[:, h // group]
                assert torch.all((o[row, h, 0].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9 * values[:, h // group].abs().amax())
        hidden = linear(o.view(rows, heads * d), out_codes, out_scale.view(1, -1))
        logits = linear(hidden, weights["logits"][0], weights["logits"][1].view(1, -1)).view(b, w, vocabulary)
        given = (scores.clone(), finished.clone(), counts.clone())
        target = rows - base
        out = select(logits, scores, finished=finished, lengths=counts, penalty=0.5, end=3, pad=0, bases=(base, target), in_place=True)
        check_select({**out, "scores_out": scores, "finished_out": finished, "lengths_out": counts}, logits, *given, 0.5, 3, 0)
        parents, tokens = out["parents"], out["tokens"]
        before = [held_codes(base + i) for i in range(rows)]
        pages_call("fork", out["forks"], [*containers, *block_scales])
        pages_call("free", ints(np.arange(base, base + rows)[:, None]))
        base = target
        p = decoder.BeamReorderParams(count=1)
        p.parents, p.source[0] = describe(parents), describe(history[0])
        p.target[0] = p.source[0]
        decoder.beam_reorder(p, [address(parents), address(history[0]), address(history[1])])
        history.reverse()
        history[0][0, :, :, step] = tokens
        walked.append((parents.cpu().numpy(), tokens.cpu().numpy()))
        for i in range(rows):
            parent = i // w * w + int(parents.view(-1)[i])
            for (c, s), (c0, s0) in zip(held_codes(base + i), before[parent]):
                assert torch.equal(c, c0) and torch.equal(s, s0)
    for i in range(b):
        for j in range(w):
            beam, line = j, []
            for parents, chosen in reversed(walked):
                line.append(chosen[i, beam])
                beam = parents[i, beam]
            assert history[0][0, i, j].tolist() == line[::-1]
    assert dfgpu.device_status() == 0
