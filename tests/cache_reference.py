"""The operators of include/dfgpu_cache.h restated in 64 bits, one sequence, block and row at a time (numpy, host)."""
import numpy as np

E4M3 = np.array([np.nan if (c & 0x7F) == 0x7F else (-1.0 if c & 0x80 else 1.0) * ((c & 7) * 2.0 ** -9 if (c >> 3 & 15) == 0 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3 & 15) - 7)) for c in range(256)])


def e8m0(code):
    code = np.asarray(code, dtype=np.float64)
    return np.where(code == 255, np.nan, 2.0 ** (code - 127))


def encode_e4m3(x):
    """Nearest code, ties to even, saturating; NaN 0x7f; a negative that rounds to zero +0, an exact -0.0 keeps its sign."""
    x = np.asarray(x, dtype=np.float64)
    magnitude = np.minimum(np.abs(np.where(np.isnan(x), 0, x)), 448.0)
    exponent = np.maximum(np.floor(np.log2(np.where(magnitude > 0, magnitude, 1.0))), -6)
    steps = np.rint(magnitude / 2.0 ** (exponent - 3))           # 0..16 (16: the next binade)
    code = np.where(steps == 0, 0, np.where(magnitude < 2.0 ** -6, steps, (exponent + 7) * 8 + (steps - 8))).astype(np.int64)
    code = np.where(np.signbit(x) & ((code > 0) | (x == 0)), code | 0x80, code)
    return np.where(np.isnan(x), 0x7F, code).astype(np.uint8)


def scale_code(amax):
    if np.isnan(amax):
        return 255
    if amax == 0:
        return 0
    if np.isinf(amax):
        return 254
    return int(np.clip(np.ceil(np.log2(amax / 448.0)) + 127, 0, 254))


def append(x, cache, scale, table, lengths, added):
    """x [B,Hk,S,D] float64; cache [pages,Hk,T,D] and scale [pages,Hk,T/t,1] uint8 (changed in place)."""
    pages, heads, page, _ = cache.shape
    t = page // scale.shape[2]
    for b, (length, n) in enumerate(zip(lengths, added)):
        length, n = max(int(length), 0), min(max(int(n), 0), x.shape[2])
        at = length
        while at < length + n:
            begin = at // t * t
            end = min(begin + t, length + n)
            slot = begin // page
            p = table[b, slot] if slot < table.shape[1] else -1
            if 0 <= p < pages:
                row, block = begin % page, begin % page // t
                for h in range(heads):
                    new = x[b, h, at - length:end - length]
                    code = scale_code(np.max(np.abs(new)))     # (numpy's maximum keeps a NaN)
                    held = slice(row, row + at - begin)
                    if at > begin:
                        old = int(scale[p, h, block, 0])
                        code = max(code, old)
                        if code != old:
                            cache[p, h, held] = encode_e4m3(E4M3[cache[p, h, held]] * e8m0(old) / e8m0(code))
                    with np.errstate(invalid="ignore"):
                        cache[p, h, row + at - begin:row + end - begin] = encode_e4m3(new / e8m0(code))
                    scale[p, h, block, 0] = code
            at = end


def attend(q, k, v, ks, vs, table_k, table_v, seq_q, seq_kv, scale, s_kv, left=None, right=None, bottom_right=False):
    """q [B,Hq,Sq,D] float64, containers and scales uint8. In 64 bits; masked keys are never touched. (O, Stats, the weighted mean of |V|, the
    largest sum of |q k| times the scale): the latter two are what roundings of weights and scores are measured by."""
    b, hq, sq, d = q.shape
    mean, products = np.zeros((b, hq, sq, d)), np.zeros((b, hq, sq))
    pages, hk, page, _ = k.shape
    t = page // ks.shape[2]
    o, stats = np.zeros((b, hq, sq, d)), np.full((b, hq, sq), -np.inf)
    for i in range(b):
        length = int(seq_kv[i])
        rows = sq if seq_q is None else min(max(int(seq_q[i]), 0), sq)
        shift = length - (sq if seq_q is None else int(seq_q[i])) if bottom_right else 0
        keys = min(max(length, 0), s_kv)
        parts = []
        for codes, scales, table in ((k, ks, table_k), (v, vs, table_v)):
            full = np.zeros((keys, hk, d))
            for slot in range(min(-(-keys // page), table.shape[1])):
                p = table[i, slot]
                if 0 <= p < pages:
                    end = min(keys, (slot + 1) * page)
                    part = E4M3[codes[p]] * np.repeat(e8m0(scales[p, :, :, 0]), t, axis=1)[..., None]
                    full[slot * page:end] = part.transpose(1, 0, 2)[:end - slot * page]
            parts.append(full)
        for r in range(rows):
            lo, hi = 0, keys
            if right is not None:
                hi = min(hi, r + shift + right + 1)
            if left is not None:
                lo = max(lo, r + shift - left + 1)
            if lo >= hi:
                continue
            for h in range(hq):
                scores = parts[0][lo:hi, h // (hq // hk)] @ q[i, h, r] * scale
                top = scores.max()
                weights = np.exp(scores - top)
                o[i, h, r] = weights @ parts[1][lo:hi, h // (hq // hk)] / weights.sum()
                stats[i, h, r] = top + np.log(weights.sum())
                mean[i, h, r] = weights @ np.abs(parts[1][lo:hi, h // (hq // hk)]) / weights.sum()
                products[i, h, r] = (np.abs(parts[0][lo:hi, h // (hq // hk)]) @ np.abs(q[i, h, r])).max() * abs(scale)
    return o, stats, mean, products


def rope(x, positions, frequencies, interleaved, inverse, scale):
    """x [B,H,S,D] float64; positions [B,S]; frequencies f32."""
    half = len(frequencies)
    angle = positions.astype(np.float64)[:, None, :, None] * frequencies.astype(np.float64)
    c, s = np.cos(angle) * scale, np.sin(angle) * scale * (-1 if inverse else 1)
    one, two = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y = x.copy()
    y[..., one] = x[..., one] * c - x[..., two] * s
    y[..., two] = x[..., two] * c + x[..., one] * s
    return y


class Pages:
    """Page table, lengths, counts and pools, and what each operation makes of them (new objects)."""

    def __init__(self, table, lengths, refs, pools, block):
        self.table, self.lengths, self.refs, self.pools, self.block = table.copy(), lengths.copy(), refs.copy(), [p.copy() for p in pools], block

    def used(self, b):
        capacity = self.table.shape[1] * self.block
        return -(-min(max(int(self.lengths[b]), 0), capacity) // self.block)

    def length(self, b):
        return min(max(int(self.lengths[b]), 0), self.table.shape[1] * self.block)

    def fine(self, page):
        return 0 <= page < len(self.refs)

    def free(self):
        return [i for i, n in enumerate(self.refs) if n <= 0]

    def report(self, moved, copied, refused):
        return [len(self.free()), moved, copied, refused]

    def move(self, pairs):
        before = [p.copy() for p in self.pools]
        for s, t in pairs:
            for pool, old in zip(self.pools, before):
                pool[:, t] = old[:, s]

    def reserve(self, grow):
        free, asked, taken, refused = self.free(), 0, 0, 0
        for b, more in enumerate(grow):
            total = self.length(b) + max(int(more), 0)
            used = self.used(b)
            if total > self.table.shape[1] * self.block:
                refused += 1
                continue
            wanted = -(-total // self.block) - used
            asked += wanted
            if asked > len(free):
                refused += 1
                continue
            for k in range(wanted):
                page = free[asked - wanted + k]
                self.table[b, used + k] = page
                self.refs[page] = 1
            taken += wanted
        return self.report(taken, 0, refused)

    def fork(self, entries):
        free, asked, taken, refused, copied, named = self.free(), 0, 0, 0, [], set()
        table, lengths, refs = self.table.copy(), self.lengths.copy(), self.refs.copy()
        batch = range(len(lengths))
        for s, t in entries:
            if s < 0:
                continue
            if s not in batch or t not in batch or s == t or self.length(t) != 0 or t in named:
                refused += 1
                continue
            named.add(t)
            full, partial = self.length(s) // self.block, self.length(s) % self.block != 0
            asked += partial
            if asked > len(free):
                refused += 1
                continue
            row = [-1] * table.shape[1]
            row[:full] = self.table[s, :full]
            if partial:
                row[full] = free[asked - 1]
                taken += 1
                if self.fine(self.table[s, full]):
                    copied.append((self.table[s, full], row[full]))
            for page in row:
                if self.fine(page):
                    refs[page] += 1
            table[t], lengths[t] = row, self.length(s)
        self.table, self.lengths, self.refs = table, lengths, refs
        self.move(copied)
        return self.report(taken, len(copied), refused)

    def free_sequences(self, entries):
        refused = sum(e >= len(self.lengths) for e in entries)
        back = 0
        for b in sorted({e for e in entries if 0 <= e < len(self.lengths)}):
            for s in range(self.used(b)):
                page = self.table[b, s]
                if self.fine(page):
                    self.refs[page] -= 1
                    back += self.refs[page] == 0
            self.table[b] = -1
            self.lengths[b] = 0
        self.refs = np.maximum(self.refs, 0)
        return self.report(int(back), 0, refused)

    def compact(self):
        live = int((self.refs > 0).sum())
        movers = [i for i in range(live, len(self.refs)) if self.refs[i] > 0]
        holes = [i for i in range(live) if self.refs[i] <= 0]
        to = dict(zip(movers, holes))
        for b in range(len(self.lengths)):
            for s in range(self.used(b)):
                self.table[b, s] = to.get(int(self.table[b, s]), self.table[b, s])
        for m, h in to.items():
            self.refs[h], self.refs[m] = self.refs[m], 0
        self.refs[live:] = 0
        self.move(list(to.items()))
        return self.report(len(movers), len(movers), 0)

    def copy(self, entries):
        pages = range(len(self.refs))
        valid = [(i, s, t) for i, (s, t) in enumerate(entries) if s in pages and t in pages and s != t]
        last = {t: i for i, _, t in valid}
        refused = sum(s >= 0 for s, _ in entries) - len(valid) + sum(s in last for _, s, _ in valid)
        pairs = [(s, t) for i, s, t in valid if s not in last and last[t] == i]
        self.move(pairs)
        return self.report(len(pairs), len(pairs), refused)
