"""The operators of a decoder's step (include/dfgpu_decoder.h) restated in 64 bits, in numpy."""
import numpy as np


def pairs_of(half, interleaved):
    return (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))


def turn(x, positions, frequencies, interleaved, scale, back=False):
    """x [B, H, S, D], positions [B, S], frequencies [R / 2]."""
    y, half = np.array(x, np.float64), len(frequencies)
    if half == 0:
        return y
    one, two = pairs_of(half, interleaved)
    angles = np.asarray(positions, np.float64)[:, None, :, None] * np.asarray(frequencies, np.float64)
    cosine, sine = scale * np.cos(angles), scale * np.sin(angles) * (-1.0 if back else 1.0)
    first, second = np.array(y[..., one]), np.array(y[..., two])
    y[..., one], y[..., two] = first * cosine - second * sine, second * cosine + first * sine
    return y


def both_of_pair(x, half, interleaved):
    """|x1| + |x2| in the place of each of a pair; |x| elsewhere."""
    y = np.abs(np.array(x, np.float64))
    if half:
        one, two = pairs_of(half, interleaved)
        y[..., one] = y[..., two] = y[..., one] + y[..., two]
    return y


def head_norm(x, gain, positions, frequencies, interleaved=False, scale=1.0, epsilon=1e-6):
    """gain [1 or H, D], its offset included."""
    x = np.asarray(x, np.float64)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon)
    return turn(x * r * np.asarray(gain, np.float64)[None, :, None], positions, frequencies, interleaved, scale)


def head_norm_grad(x, dy, gain, positions, frequencies, interleaved=False, scale=1.0, epsilon=1e-6):
    """(dX, dgain)."""
    x, gain = np.asarray(x, np.float64), np.asarray(gain, np.float64)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + epsilon)
    u = turn(dy, positions, frequencies, interleaved, scale, back=True)
    v = u * gain[None, :, None]
    dx = r * v - x * r ** 3 * (v * x).mean(-1, keepdims=True)
    dgain = (u * x * r).sum((0, 2))
    return dx, dgain if gain.shape[0] > 1 else dgain.sum(0, keepdims=True)


def token_quantize(x):
    """x f32 [..., K] -> (codes int8, scale f32 [..., 1]), by f32 quotients."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        largest = np.abs(x).max(-1, keepdims=True)   # (numpy's maximum keeps a NaN)
        scale = (largest / np.float32(127)).astype(np.float32)
        quotient = (x / scale).astype(np.float32)
        codes = np.where((scale > 0) & ~np.isnan(quotient), np.clip(np.rint(quotient), -127, 127), 0)
    return codes.astype(np.int8), scale


def matmul_int8(a, b, a_scale, b_scale, bias=None):
    """f32 values before the rounding to C's type: a [..., M, K], b [..., K, N] int8; scales and bias f32, broadcast."""
    total = np.matmul(a.astype(np.int64), b.astype(np.int64))
    value = (total.astype(np.float32) * a_scale.astype(np.float32)).astype(np.float32)   # (an integer below 2^53 rounds once)
    value = (value * b_scale.astype(np.float32)).astype(np.float32)
    return value if bias is None else (value + bias.astype(np.float32)).astype(np.float32)


def beam_select(logits, scores, finished=None, lengths=None, penalty=0.0, end=-1, pad=0):
    """logits [B, W, V] -> (scores [B, W] in 64 bits, tokens, parents, finished, lengths)."""
    logits, scores = np.asarray(logits, np.float64), np.asarray(scores, np.float64)
    batch, beams, vocabulary = logits.shape
    finished = np.zeros((batch, beams), np.int64) if finished is None else np.asarray(finished)
    count = np.zeros((batch, beams), np.int64) if lengths is None else np.asarray(lengths, np.int64)
    out = [np.zeros((batch, beams)), *(np.zeros((batch, beams), np.int64) for _ in range(4))]
    for b in range(batch):
        places, totals, worths = [], [], []
        for w in range(beams):
            n = max(1, count[b, w] + (0 if finished[b, w] else 1))
            if finished[b, w]:
                tokens, total = np.array([pad]), np.array([scores[b, w] if np.isfinite(scores[b, w]) else -np.inf])
            else:
                tokens, row = np.arange(vocabulary), logits[b, w]
                with np.errstate(all="ignore"):
                    top = row.max()
                    normaliser = top + np.log(np.exp(row - top).sum())
                    total = scores[b, w] + (row - normaliser)
                if not np.isfinite(scores[b, w]) or not np.isfinite(normaliser):
                    total = np.full(vocabulary, -np.inf)
            places.append(w * vocabulary + tokens)
            totals.append(total)
            worths.append(total / float(n) ** penalty if lengths is not None else total)
        places, totals, worths = (np.concatenate(v) for v in (places, totals, worths))
        chosen = np.lexsort((places, -worths))[:beams]
        out[0][b], out[1][b], out[2][b] = totals[chosen], places[chosen] % vocabulary, places[chosen] // vocabulary
        done = finished[b, out[2][b]] != 0
        out[3][b] = done | ((out[1][b] == end) if end >= 0 else False)
        out[4][b] = np.maximum(1, count[b, out[2][b]] + ~done)
    return out
