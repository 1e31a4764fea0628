"""Cases on which the operators around a paged KV cache in 8 bits are measured: rotary positions, writing new tokens into the cache
(E4M3 codes, an E8M0 scale for each block of tokens and head), attention over it, and the bookkeeping of its pages.

A case is a dict of plain values whose "op" names the operator:

  rope     rotary positions of queries and keys in one call, or their gradients (inverse)
  append   new keys and values quantised into the pages behind each sequence's length
  attend   attention of one or more new tokens a sequence over the cached codes
  pages    reserve, fork, free, compact or copy over page table, lengths, reference counts and pools

`run` computes the plain form in torch where `own` is false, and makes the framework's calls where it is true.
"""
import torch

own = False

TORCH = {"BFLOAT16": torch.bfloat16, "HALF": torch.float16, "FLOAT": torch.float32}


def listed():
    return [
        # one new token for each of 32 users: queries and keys of grouped heads, bound by launch latency
        {"name": "rope_token", "op": "rope", "b": 32, "s": 1, "h": 32, "h2": 8, "d": 128, "rotary": 128, "interleaved": False, "inverse": False, "io": "BFLOAT16", "far": 100000},
        # whole prompts, far positions
        {"name": "rope_prompts", "op": "rope", "b": 2, "s": 8192, "h": 32, "h2": 8, "d": 128, "rotary": 128, "interleaved": False, "inverse": False, "io": "BFLOAT16", "far": 1000000},
        # the gradient in training with f32 activations: pairs side by side, half of the head rotated, an odd length
        {"name": "rope_gradient", "op": "rope", "b": 3, "s": 1001, "h": 16, "h2": 16, "d": 128, "rotary": 64, "interleaved": True, "inverse": True, "io": "FLOAT", "far": 0},
        # a decode step's new token for each of 64 users, blocks partly filled
        {"name": "append_token", "op": "append", "b": 64, "s": 1, "hk": 8, "d": 128, "page": 64, "tokens": 16, "pages": 4096, "held": 2000, "io": "BFLOAT16"},
        # prompts of different lengths, padded to the longest
        {"name": "append_prompts", "op": "append", "b": 8, "s": 2048, "hk": 8, "d": 128, "page": 64, "tokens": 64, "pages": 320, "held": 100, "io": "BFLOAT16"},
        # a full decode batch over a 16384-page cache
        {"name": "attend_batch_64", "op": "attend", "b": 64, "sq": 1, "hk": 8, "g": 4, "d": 128, "page": 64, "tokens": 64, "pages": 16384, "least": 512, "most": 8192, "window": 0, "io": "BFLOAT16"},
        # two interactive users: few blocks in flight
        {"name": "attend_batch_2", "op": "attend", "b": 2, "sq": 1, "hk": 8, "g": 4, "d": 128, "page": 64, "tokens": 16, "pages": 320, "least": 512, "most": 8192, "window": 0, "io": "BFLOAT16"},
        # drafted tokens to be checked, a sliding window, pages that are no power of two
        {"name": "attend_draft", "op": "attend", "b": 16, "sq": 5, "hk": 4, "g": 8, "d": 64, "page": 48, "tokens": 16, "pages": 1500, "least": 200, "most": 4000, "window": 1024, "io": "HALF"},
        # the next 1000 tokens of long prompts, taken in chunks
        {"name": "attend_chunk", "op": "attend", "b": 2, "sq": 1000, "hk": 8, "g": 4, "d": 128, "page": 64, "tokens": 64, "pages": 512, "least": 3000, "most": 16000, "window": 0, "io": "BFLOAT16"},
        # a beam: every second sequence continues another one's pages
        {"name": "pages_fork", "op": "pages", "do": "fork", "b": 64, "slots": 64, "pages": 4096, "page": 64, "hk": 8, "d": 128, "fill": 50},
        # pages for the next step's tokens
        {"name": "pages_reserve", "op": "pages", "do": "reserve", "b": 256, "slots": 128, "pages": 40000, "page": 64, "hk": 8, "d": 128, "fill": 50},
        # a fragmented cache made dense again
        {"name": "pages_compact", "op": "pages", "do": "compact", "b": 64, "slots": 64, "pages": 8192, "page": 64, "hk": 8, "d": 128, "fill": 75},
    ]


MAX_BYTES, MAX_FLOPS = 5.0e8, 2.2e11


def draw(rng):
    def spread(low, high, step=1):
        """A multiple of step in [low, high], spread over the logarithm."""
        value = low * (high / low) ** rng.random()
        return max(low, min(high, int(value / step + 0.5) * step))

    while True:
        op = rng.choice(("rope", "append", "attend", "attend", "pages"))
        if op == "rope":
            d = rng.choice((64, 80, 96, 128, 128, 256))
            case = {"b": spread(1, 64), "s": spread(1, 8192), "h": spread(1, 64), "h2": rng.choice((0, 1, 2, 8, 8)), "d": d, "rotary": rng.choice((d, d, d // 2)),
                    "interleaved": rng.random() < 0.4, "inverse": rng.random() < 0.3, "io": rng.choice(("BFLOAT16", "BFLOAT16", "FLOAT", "HALF")), "far": rng.choice((0, 100000, 1000000))}
        elif op == "append":
            page = rng.choice((16, 32, 48, 64, 64, 128, 256))
            held, s = rng.choice((0, 100, 2000)), rng.choice((1, spread(1, 4096)))
            b = spread(1, 128)
            slots = -(-(held + s) // page) + 1
            case = {"b": b, "s": s, "hk": spread(1, 16), "d": rng.choice((64, 128, 128, 256)), "page": page, "tokens": rng.choice((16, page)), "pages": b * slots + rng.randrange(64),
                    "held": held, "io": rng.choice(("BFLOAT16", "BFLOAT16", "FLOAT", "HALF"))}
        elif op == "attend":
            page = rng.choice((16, 32, 48, 64, 64, 128, 256))
            kind = rng.choice(("token", "token", "draft", "chunk"))
            sq = 1 if kind == "token" else spread(2, 9) if kind == "draft" else spread(32, 2000)
            b = spread(1, 96) if kind == "token" else spread(1, 24) if kind == "draft" else spread(1, 4)
            most = spread(max(sq, 128), 16000)
            slots = -(-most // page)
            case = {"b": b, "sq": sq, "hk": rng.choice((1, 2, 4, 8, 8)), "g": rng.choice((1, 2, 4, 4, 5, 8, 16)), "d": rng.choice((64, 128, 128, 128, 256)), "page": page,
                    "tokens": rng.choice((16, page)), "pages": b * slots + rng.randrange(64), "least": rng.choice((0, sq, most // 8)), "most": most,
                    "window": rng.choice((0, 0, 0, 300, 4096)), "io": rng.choice(("BFLOAT16", "BFLOAT16", "HALF"))}
        else:
            b, slots = spread(2, 256), spread(4, 256)
            case = {"do": rng.choice(("reserve", "fork", "free", "compact", "copy")), "b": b, "slots": slots, "pages": 2 * b * slots + rng.randrange(100),
                    "page": rng.choice((16, 48, 64, 128)), "hk": spread(1, 8), "d": rng.choice((64, 128)), "fill": rng.choice((10, 50, 90))}
        case["op"] = op
        w = work(case)
        if op == "append" and 2 * case["pages"] * case["hk"] * case["page"] * case["d"] > 6e8:
            continue
        if op == "attend" and (2 * case["pages"] * case["hk"] * case["page"] * case["d"] > 2.2e9 or case["b"] * case["hk"] * case["g"] * case["sq"] * case["most"] > 1.1e9):
            continue
        if op == "attend" and case["b"] * case["hk"] * case["most"] * case["d"] > 6e8:
            continue
        if op == "pages" and case["do"] not in ("reserve", "free") and 2 * case["pages"] * case["hk"] * case["page"] * case["d"] > 1.2e9:
            continue
        if w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS:
            return case


# ---- shared pieces ---------------------------------------------------------------------

def lengths_of(b, least, most):
    """Spread evenly from least to most: the sum is the case's alone, the order the seed's."""
    return [most] if b == 1 else [least + round((most - least) * i / (b - 1)) for i in range(b)]


def added_of(case):
    """Tokens that an append writes for each sequence: ragged where there is more than one."""
    return [case["s"] if case["s"] == 1 else 1 + round((case["s"] - 1) * (i + 1) / case["b"]) for i in range(case["b"])]


def forks_of(case):
    return [(2 * i, 2 * i + 1) for i in range(case["b"] // 2)]


def used_of(case):
    """Tokens of each sequence of a pages case; every second sequence of a fork is empty."""
    capacity = case["slots"] * case["page"]
    used = [1 + (capacity * case["fill"] // 100 * (i + 1)) // case["b"] for i in range(case["b"])]
    return [n if i % 2 == 0 else 0 for i, n in enumerate(used)] if case["do"] == "fork" else used


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def tables(case, seed, slots, g):
    """Page ids of each sequence's slots, all different, anywhere in the pool."""
    ids = torch.randperm(case["pages"], device="cuda", generator=g, dtype=torch.int64)[: case["b"] * slots]
    return ids.to(torch.int32).view(case["b"], slots)


def e4m3(codes):
    return codes.view(torch.float8_e4m3fn)


def e8m0(codes):
    """2^(code - 127) in f32; 0xff is NaN."""
    power = torch.exp2(codes.to(torch.float32) - 127.0)
    return torch.where(codes == 255, torch.full_like(power, float("nan")), power)


def page_bytes(case):
    return 2 * case["hk"] * case["page"] * case["d"]


def copied_pages(case):
    """Pages whose contents a pages case moves."""
    used, t = used_of(case), case["page"]
    live = sum(-(-n // t) for n in used)
    if case["do"] == "fork":
        return sum(1 for s, _ in forks_of(case) if used[s] % t)
    if case["do"] == "copy":
        return min(live // 2, case["pages"] // 8)
    if case["do"] == "compact":   # live pages lie anywhere: that share of them behind the first `live` ids
        return live * (case["pages"] - live) // case["pages"]
    return 0


def work(case):
    """What one pass cannot do without: inputs read once, outputs written once."""
    op = case["op"]
    if op == "rope":
        size = 4 if case["io"] == "FLOAT" else 2
        rows = case["b"] * case["s"] * (case["h"] + case["h2"])
        return {"bytes": 2 * rows * case["d"] * size + 4 * case["b"] * case["s"], "flops": 3 * rows * case["rotary"]}
    if op == "append":
        size = 4 if case["io"] == "FLOAT" else 2
        values = 2 * sum(added_of(case)) * case["hk"] * case["d"]
        return {"bytes": values * (size + 1) + values // (case["d"] * case["tokens"]), "flops": 2 * values}
    if op == "attend":
        sq, d, heads = case["sq"], case["d"], case["hk"] * case["g"]
        lengths = lengths_of(case["b"], case["least"], case["most"])
        keys = sum(min(n, case["window"] + sq) if case["window"] else n for n in lengths)
        pairs = sum(max(0, min(n, (case["window"] or n)) * sq - (0 if case["window"] else sq * sq // 2)) for n in lengths)
        return {"bytes": 2 * keys * case["hk"] * d + 4 * case["b"] * heads * sq * d, "flops": 4 * pairs * heads * d}
    integers = 2 * (case["b"] * case["slots"] + case["pages"])
    return {"bytes": 4 * integers + 2 * copied_pages(case) * page_bytes(case), "flops": integers}


# ---- inputs ------------------------------------------------------------------------------

def prepare(case, seed):
    return {"rope": prepare_rope, "append": prepare_append, "attend": prepare_attend, "pages": prepare_pages}[case["op"]](case, seed)


def rope_frequencies(case):
    half = case["rotary"] // 2
    return (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).to(torch.float32).cuda()


def prepare_rope(case, seed):
    g = generator(seed)
    b, s, d, io = case["b"], case["s"], case["d"], TORCH[case["io"]]
    s_state = {"case": case, "frequencies": rope_frequencies(case)}
    s_state["x"] = torch.randn(b, case["h"], s, d, device="cuda", generator=g).to(io)
    if case["h2"]:
        s_state["x2"] = torch.randn(b, case["h2"], s, d, device="cuda", generator=g).to(io)
    start = torch.randint(0, case["far"] + 1, (b, 1), device="cuda", generator=g)
    s_state["positions"] = (start + torch.arange(s, device="cuda")).to(torch.int32)
    s_state["y"] = torch.empty_like(s_state["x"])
    if case["h2"]:
        s_state["y2"] = torch.empty_like(s_state["x2"])
    return s_state


def prepare_append(case, seed):
    g = generator(seed)
    b, s, hk, d, page, tokens, pages, io = (case[k] for k in ("b", "s", "hk", "d", "page", "tokens", "pages", "io"))
    slots = min(-(-(case["held"] + s) // page) + 1, pages // b)
    st = {"case": case}
    magnitude = torch.exp2(torch.randint(-3, 4, (b, hk, s, 1), device="cuda", generator=g).to(torch.float32))
    st["k"], st["v"] = ((torch.randn(b, hk, s, d, device="cuda", generator=g) * magnitude).to(TORCH[io]) for _ in range(2))
    for name in ("k", "v"):
        st[name + "_cache"] = (100.0 * torch.randn(pages, hk, page, d, device="cuda", generator=g)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        st[name + "_scale"] = torch.randint(118, 124, (pages, hk, page // tokens, 1), device="cuda", generator=g).to(torch.uint8)
    st["table"] = tables(case, seed, slots, g)
    st["lengths"] = torch.randint(0, case["held"] + 1, (b,), device="cuda", generator=g).clamp(max=slots * page - s).to(torch.int32)
    st["added"] = torch.tensor(added_of(case), device="cuda")[torch.randperm(b, device="cuda", generator=g)].to(torch.int32)
    st["lengths_out"] = torch.empty_like(st["lengths"])
    return st


def prepare_attend(case, seed):
    g = generator(seed)
    b, sq, hk, grp, d, page, tokens, pages = (case[k] for k in ("b", "sq", "hk", "g", "d", "page", "tokens", "pages"))
    slots = -(-case["most"] // page)
    st = {"case": case}
    st["q"] = torch.randn(b, hk * grp, sq, d, device="cuda", generator=g).to(TORCH[case["io"]])
    for name in ("k", "v"):
        st[name + "_cache"] = (110.0 * torch.randn(pages, hk, page, d, device="cuda", generator=g)).clamp_(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        st[name + "_scale"] = torch.randint(119, 122, (pages, hk, page // tokens, 1), device="cuda", generator=g).to(torch.uint8)
    st["table"] = tables(case, seed, slots, g) if b * slots <= pages else torch.stack([torch.randperm(pages, device="cuda", generator=g)[:slots] for _ in range(b)]).to(torch.int32)
    lengths = torch.tensor(lengths_of(b, case["least"], case["most"]), device="cuda", dtype=torch.int32)
    st["lengths"] = lengths[torch.randperm(b, device="cuda", generator=g)].contiguous()
    st["o"] = torch.empty_like(st["q"])
    st["stats"] = torch.empty(b, hk * grp, sq, device="cuda", dtype=torch.float32)
    st["seq_q"] = torch.full((b,), sq, device="cuda", dtype=torch.int32)
    return st


def prepare_pages(case, seed):
    g = generator(seed)
    b, slots, pages, page, hk, d = (case[k] for k in ("b", "slots", "pages", "page", "hk", "d"))
    st = {"case": case}
    used = torch.tensor(used_of(case), device="cuda")
    if case["do"] != "fork":
        used = used[torch.randperm(b, device="cuda", generator=g)]
    held = (used + page - 1) // page
    table = tables(case, seed, slots, g).to(torch.int64)
    inside = torch.arange(slots, device="cuda") < held[:, None]
    st["lengths"], st["table"] = used.to(torch.int32), torch.where(inside, table, -1).to(torch.int32)
    st["refs"] = torch.zeros(pages, device="cuda", dtype=torch.int32)
    st["refs"][table[inside]] = 1
    pools = 2 if case["do"] in ("fork", "compact", "copy") else 0   # (the other operations move no contents)
    st["pools"] = [torch.randint(0, 256, (1, pages, hk * page * d), device="cuda", generator=g, dtype=torch.uint8) for _ in range(pools)]
    if case["do"] == "reserve":
        entries = torch.randint(0, page + 1, (b, 1), device="cuda", generator=g)
    elif case["do"] == "fork":
        entries = torch.tensor(forks_of(case), device="cuda")[torch.randperm(b // 2, device="cuda", generator=g)]
    elif case["do"] == "free":
        entries = torch.randperm(b, device="cuda", generator=g)[: max(1, b // 2), None]
    elif case["do"] == "copy":
        live = table[inside]
        free = torch.nonzero(st["refs"] == 0)[:, 0]
        n = copied_pages(case)
        entries = torch.stack([live[torch.randperm(len(live), device="cuda", generator=g)[:n]], free[torch.randperm(len(free), device="cuda", generator=g)[:n]]], 1)
    else:
        entries = torch.zeros(0, 1, device="cuda")
    st["list"] = entries.to(torch.int32).contiguous()
    st["table_out"], st["lengths_out"], st["refs_out"] = (torch.empty_like(st[n]) for n in ("table", "lengths", "refs"))
    st["report"] = torch.zeros(4, device="cuda", dtype=torch.int32)
    return st


# ---- one pass --------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": own_rope, "append": own_append, "attend": own_attend, "pages": own_pages}[op](state)
    return {"rope": plain_rope, "append": plain_append, "attend": plain_attend, "pages": plain_pages}[op](state)


def plain_rotation(x, cosine, sine, rotary, interleaved):
    turned, rest = x[..., :rotary].float(), x[..., rotary:]
    if interleaved:
        first, second = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([first * cosine - second * sine, second * cosine + first * sine], -1).flatten(-2)
    else:
        first, second = turned[..., : rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat([first * cosine - second * sine, second * cosine + first * sine], -1)
    return torch.cat([turned.to(x.dtype), rest], -1)


def plain_rope(st):
    case = st["case"]
    angles = st["positions"].to(torch.float64)[:, None, :, None] * st["frequencies"].to(torch.float64)   # (far positions: f32 loses the angle)
    cosine, sine = torch.cos(angles).float(), torch.sin(angles).float()
    if case["inverse"]:
        sine = -sine
    return [plain_rotation(st[n], cosine, sine, case["rotary"], case["interleaved"]) for n in ("x", "x2") if n in st]


def plain_scale_codes(amax):
    """E8M0 code of 2^ceil(log2(amax / 448)); 0 for a block of zeros, 0xff for one with a NaN."""
    desired = amax / 448.0
    fraction, exponent = torch.frexp(desired)
    code = (exponent + torch.where(fraction > 0.5, 127, 126)).clamp(0, 254)
    code = torch.where(amax == 0, 0, torch.where(torch.isinf(amax), 254, code))
    return torch.where(torch.isnan(amax), 255, code)


def plain_append(st):
    case = st["case"]
    b, s, hk, d, page, tokens = (case[k] for k in ("b", "s", "hk", "d", "page", "tokens"))
    pages, per_page = st["k_cache"].shape[0], page // tokens
    index = torch.arange(s, device="cuda")
    heads = torch.arange(hk, device="cuda")
    lengths, table = st["lengths"].long(), st["table"].long()
    at = lengths[:, None] + index                                                     # [b, s] positions
    slot = (at // page).clamp(max=table.shape[1] - 1)
    where = torch.gather(table, 1, slot)
    fine = (index < st["added"].long()[:, None]) & (at < table.shape[1] * page) & (where >= 0) & (where < pages)
    where = torch.where(fine, where, 0)
    block = ((where * hk)[:, None, :] + heads[:, None]) * per_page + ((at % page) // tokens)[:, None, :]          # [b, hk, s] blocks
    ghost = pages * hk * per_page                                                      # one block more takes what is not written
    block = torch.where(fine[:, None, :], block, ghost)
    # the block that holds each sequence's last token already
    start = lengths // tokens * tokens
    slot0 = (start // page).clamp(max=table.shape[1] - 1)
    where0 = torch.gather(table, 1, slot0[:, None])[:, 0]
    held = (lengths % tokens != 0) & (where0 >= 0) & (where0 < pages) & (start < table.shape[1] * page)
    where0 = torch.where(held, where0, 0)
    block0 = torch.where(held[:, None], (where0[:, None] * hk + heads) * per_page + ((start % page) // tokens)[:, None], ghost)   # [b, hk]
    out = []
    for name in ("k", "v"):
        x, cache, scale = st[name].float(), st[name + "_cache"], st[name + "_scale"]
        amax = torch.zeros(ghost + 1, device="cuda", dtype=torch.int32)               # |x| as ordered bits: a NaN is above all
        bits = x.abs().amax(-1).view(torch.int32)
        nan = torch.isnan(x).any(-1)
        amax = amax.scatter_reduce(0, block.reshape(-1), torch.where(nan, 0x7fc00000, bits).reshape(-1), "amax")
        touched = torch.zeros(ghost + 1, device="cuda", dtype=torch.bool)
        touched[block.reshape(-1)] = True
        old = torch.cat([scale.reshape(-1).long(), torch.zeros(1, device="cuda", dtype=torch.long)])
        new = plain_scale_codes(amax.view(torch.float32)).long()
        bound = torch.zeros_like(new).scatter_reduce(0, block0.reshape(-1), old[block0.reshape(-1)], "amax")
        new = torch.where(touched, torch.maximum(new, bound), old)
        # what the block holds, in the new scale
        row = (start[:, None] % page + torch.arange(tokens, device="cuda"))            # [b, tokens]
        keep = (held[:, None] & (start[:, None] + torch.arange(tokens, device="cuda") < lengths[:, None]))[:, None, :] & (touched & (new != old))[block0][..., None]
        before = cache[where0[:, None, None], heads[:, None], row[:, None, :]]
        factor = e8m0(old[block0]) / e8m0(new[block0])
        after = (e4m3(before).float() * factor[..., None, None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        seq, head, token = torch.nonzero(keep, as_tuple=True)
        cache[where0[seq], head, row[seq, token]] = after[seq, head, token]
        # the new tokens
        codes = (x / e8m0(new[block])[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        seq, token = torch.nonzero(fine, as_tuple=True)
        cache[where[seq, token], :, (at % page)[seq, token]] = codes[seq, :, token]
        scale.copy_(new[:ghost].to(torch.uint8).view_as(scale))
        out += [e4m3(cache), scale]
    st["lengths_out"].copy_(lengths + st["added"].long())
    return out + [st["lengths_out"]]


def plain_attend(st):
    case = st["case"]
    b, sq, hk, grp, d, page = (case[k] for k in ("b", "sq", "hk", "g", "d", "page"))
    pages = st["k_cache"].shape[0]
    table = st["table"].long()
    fine = (table >= 0) & (table < pages)
    table = torch.where(fine, table, 0)
    keys = table.shape[1] * page

    def rows(name):
        x = e4m3(st[name + "_cache"][table]).float()                                   # [b, slots, hk, page, d]
        x = x.view(b, -1, hk, page // case["tokens"], case["tokens"], d) * e8m0(st[name + "_scale"][table])[..., None]
        x = torch.where(fine[:, :, None, None, None, None], x, 0.0)
        return x.view(b, -1, hk, page, d).transpose(1, 2).reshape(b, hk, keys, d)
    lengths = st["lengths"].long()
    key = torch.arange(keys, device="cuda")
    last = lengths[:, None] - sq + torch.arange(sq, device="cuda")                     # [b, sq]: the last key of each query
    allowed = (key <= last[..., None]) & (key < lengths[:, None, None])
    if case["window"]:
        allowed &= key > last[..., None] - case["window"]
    allowed = allowed[:, None, None]                                                   # [b, 1, 1, sq, keys]
    q = st["q"].float().view(b, hk, grp, sq, d)
    scores = (q.reshape(b, hk, grp * sq, d) @ rows("k").transpose(-1, -2)).view(b, hk, grp, sq, keys) * d ** -0.5
    scores = scores.masked_fill(~allowed, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(torch.isinf(top), 0.0, top))
    total = weights.sum(-1, keepdim=True)
    o = (weights.view(b, hk, grp * sq, keys) @ rows("v")).view(b, hk, grp, sq, d)
    o = torch.where(total > 0, o / torch.where(total > 0, total, 1.0), 0.0)
    stats = (torch.where(torch.isinf(top), 0.0, top) + torch.log(total))[..., 0]
    return [o.reshape(b, hk * grp, sq, d).to(st["q"].dtype), stats.reshape(b, hk * grp, sq)]


def plain_pages(st):
    case = st["case"]
    b, slots, pages, page = (case[k] for k in ("b", "slots", "pages", "page"))
    table, lengths, refs, entries = st["table"].long(), st["lengths"].long(), st["refs"].long(), st["list"].long()
    slot, free = torch.arange(slots, device="cuda"), torch.argsort((refs > 0).int(), stable=True)   # (free pages first, by id)
    available = (refs == 0).sum()
    used = ((lengths + page - 1) // page).clamp(0, slots)
    inside = (slot < used[:, None]) & (table >= 0) & (table < pages)
    zero = torch.zeros((), device="cuda", dtype=torch.long)
    moved = copied = refused = zero
    copies = torch.zeros(0, 2, device="cuda", dtype=torch.long)
    if case["do"] == "reserve":
        grow = entries[:, 0].clamp(min=0)
        wanted = (lengths + grow + page - 1) // page - used
        fits = lengths + grow <= slots * page
        wanted = torch.where(fits, wanted, 0)
        until = torch.cumsum(wanted, 0)
        served = fits & (until <= available)
        wanted_here = torch.where(served, wanted, 0)
        new = (slot >= used[:, None]) & (slot < (used + wanted_here)[:, None])
        ids = free[((until - wanted)[:, None] + slot - used[:, None]).clamp(0, pages - 1)]
        table = torch.where(new, ids, table)
        refs = refs.index_put((ids[new],), torch.ones((), device="cuda", dtype=torch.long))
        moved, refused = wanted_here.sum(), (~served).sum()
    elif case["do"] == "free":
        listed_too = torch.zeros(b, device="cuda", dtype=torch.bool)
        listed_too[entries[:, 0]] = True
        drop = inside & listed_too[:, None]
        fewer = (refs - torch.bincount(table[drop], minlength=pages)).clamp(min=0)
        moved = ((refs > 0) & (fewer == 0)).sum()
        refs, table, lengths = fewer, torch.where(listed_too[:, None], -1, table), torch.where(listed_too, 0, lengths)
    elif case["do"] == "fork":
        source, target = entries[:, 0], entries[:, 1]
        partial = (lengths[source] % page != 0).long()
        until = torch.cumsum(partial, 0)
        served = (lengths[target] == 0) & (until <= available)
        full = lengths[source] // page
        fresh = free[(until - 1).clamp(0)]
        row = torch.where(slot < full[:, None], table[source], -1)
        takes = served & (partial > 0)
        copies = torch.stack([table[source].gather(1, full[:, None].clamp(max=slots - 1))[:, 0], fresh], 1)[takes]
        row = torch.where((slot == full[:, None]) & (partial > 0)[:, None], fresh[:, None], row)
        refs = refs + torch.bincount(row[served][row[served] >= 0], minlength=pages)
        table, lengths = table.clone(), lengths.clone()
        table[target[served]], lengths[target[served]] = row[served], lengths[source[served]]
        moved, refused = takes.sum(), (~served).sum()
        copied = moved
    elif case["do"] == "compact":
        live = (refs > 0).sum()
        ids = torch.arange(pages, device="cuda")
        movers, holes = ids[(refs > 0) & (ids >= live)], ids[(refs == 0) & (ids < live)]
        to = ids.clone()
        to[movers] = holes
        copies = torch.stack([movers, holes], 1)
        table = torch.where(inside, to[table.clamp(0, pages - 1)], table)
        counts = refs.clone()
        counts[holes] = refs[movers]
        counts[movers] = 0
        refs = counts
        moved = copied = movers.numel() + zero
    else:
        copies, moved, copied = entries, entries.shape[0] + zero, entries.shape[0] + zero
    for pool in st["pools"]:
        pool[:, copies[:, 1]] = pool[:, copies[:, 0]]
    st["table_out"].copy_(table)
    st["lengths_out"].copy_(lengths)
    st["refs_out"].copy_(refs)
    st["report"].copy_(torch.stack([(refs == 0).sum(), moved, copied, refused]))
    return [st["table_out"], st["lengths_out"], st["refs_out"], st["report"]] + st["pools"]


# ---- the framework's calls ----------------------------------------------------------------------

DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}   # FLOAT, HALF, BFLOAT16 of the C ABI
E4M3, E8M0, I32, U8 = 3, 4, 5, 7


def own_rope(st):
    from deepforge_b200 import cache
    if "call" not in st:   # the descriptors that a program fills once
        case, tensor = st["case"], cache.tensor
        p = cache.RopeParams(interleaved=case["interleaved"], inverse=case["inverse"], scale=1.0)
        p.x = p.y = tensor(DTYPE[st["x"].dtype], st["x"].shape)
        if "x2" in st:
            p.x2 = p.y2 = tensor(DTYPE[st["x2"].dtype], st["x2"].shape)
        p.positions = tensor(I32, [case["b"], 1, case["s"], 1])
        p.frequencies = tensor(0, [1, 1, 1, case["rotary"] // 2])
        st["call"] = p
    names = ("x", "y", "positions", "frequencies") + (("x2", "y2") if "x2" in st else ())
    cache.rope(st["call"], [st[n].data_ptr() for n in names])
    return [st[n] for n in ("y", "y2") if n in st]


def own_append(st):
    from deepforge_b200 import cache
    if "call" not in st:
        case, tensor = st["case"], cache.tensor
        p = cache.CacheAppendParams()
        p.k = p.v = tensor(DTYPE[st["k"].dtype], st["k"].shape)
        p.k_cache = p.v_cache = tensor(E4M3, st["k_cache"].shape)
        p.k_scale = p.v_scale = tensor(E8M0, st["k_scale"].shape)
        p.page_table_k = p.page_table_v = tensor(I32, [case["b"], 1, st["table"].shape[1], 1])
        p.lengths = p.added = p.lengths_out = tensor(I32, [case["b"], 1, 1, 1])
        st["call"] = p
    names = ("k", "v", "k_cache", "v_cache", "k_scale", "v_scale", "table", "table", "lengths", "added", "lengths_out")
    cache.cache_append(st["call"], [st[n].data_ptr() for n in names])
    return [e4m3(st["k_cache"]), st["k_scale"], e4m3(st["v_cache"]), st["v_scale"], st["lengths_out"]]


def own_attend(st):
    from deepforge_b200 import cache
    if "call" not in st:
        case, tensor = st["case"], cache.tensor
        p = cache.CacheSdpaParams(attn_scale=case["d"] ** -0.5, has_right_bound=1, right_bound=0, bottom_right=1, s_kv=case["most"])
        if case["window"]:
            p.has_left_bound, p.left_bound = 1, case["window"]
        p.q = p.o = tensor(DTYPE[st["q"].dtype], st["q"].shape)
        p.stats = tensor(0, [case["b"], case["hk"] * case["g"], case["sq"], 1])
        p.k = p.v = tensor(E4M3, st["k_cache"].shape)
        p.k_scale = p.v_scale = tensor(E8M0, st["k_scale"].shape)
        p.page_table_k = p.page_table_v = tensor(I32, [case["b"], 1, st["table"].shape[1], 1])
        p.seq_q = p.seq_kv = tensor(I32, [case["b"], 1, 1, 1])
        st["scratch"] = torch.empty(max(1, cache.query("cache_sdpa", p).scratch_bytes), device="cuda", dtype=torch.uint8)
        st["call"] = p
    names = ("q", "k_cache", "v_cache", "o", "stats", "k_scale", "v_scale", "seq_q", "lengths", "table", "table")
    cache.cache_sdpa(st["call"], [st[n].data_ptr() for n in names], st["scratch"].data_ptr())
    return [st["o"], st["stats"]]


def own_pages(st):
    from deepforge_b200 import cache
    if "call" not in st:
        case, tensor = st["case"], cache.tensor
        p = cache.CachePagesParams(op=cache.PAGE_OPS[case["do"]], block=case["page"], pool_count=len(st["pools"]))
        p.page_table = tensor(I32, [case["b"], 1, case["slots"], 1])
        p.lengths = tensor(I32, [case["b"], 1, 1, 1])
        p.refs = tensor(I32, [case["pages"]])
        if case["do"] != "compact":
            p.list = tensor(I32, st["list"].shape)
        for i, pool in enumerate(st["pools"]):
            p.pools[i] = tensor(U8, pool.shape)
        st["scratch"] = torch.empty(cache.query("cache_pages", p).scratch_bytes, device="cuda", dtype=torch.uint8)
        st["call"] = p
    pointers = [st[n].data_ptr() for n in ("table", "lengths", "refs", "list", "table_out", "lengths_out", "refs_out", "report")]
    cache.cache_pages(st["call"], pointers + [pool.data_ptr() for pool in st["pools"]], st["scratch"].data_ptr())
    return [st["table_out"], st["lengths_out"], st["refs_out"], st["report"]] + st["pools"]


# ---- the definitions in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    return {"rope": exact_rope, "append": exact_append, "attend": exact_attend, "pages": lambda *_: None}[case["op"]](prepare(case, seed))


def exact_rope(st):
    """Each pair is a complex number, turned by the angle."""
    case = st["case"]
    sign = -1.0 if case["inverse"] else 1.0
    angles = sign * torch.einsum("bs,i->bsi", st["positions"].double(), st["frequencies"].double())
    turn = torch.polar(torch.ones_like(angles), angles)[:, None]
    results = []
    for name in ("x", "x2"):
        if name not in st:
            continue
        y, half = st[name].double(), case["rotary"] // 2
        if case["interleaved"]:
            at = (slice(0, 2 * half, 2), slice(1, 2 * half, 2))
        else:
            at = (slice(0, half), slice(half, 2 * half))
        turned = torch.complex(y[..., at[0]].contiguous(), y[..., at[1]].contiguous()) * turn
        y[..., at[0]], y[..., at[1]] = turned.real, turned.imag
        results.append(y)
    return results


def exact_e4m3(x):
    """The nearest value of four significant bits, exponents -6 to 8, ties to even, in 64 bits."""
    exponent = torch.frexp(x)[1].clamp(min=-5) - 4
    step = torch.ldexp(torch.ones_like(x), exponent)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def exact_append(st):
    """Sequence by sequence and block by block: the largest magnitude of the new tokens, the power of two, the codes."""
    case = st["case"]
    page, tokens = case["page"], case["tokens"]
    out = []
    lengths, added, table = st["lengths"].tolist(), st["added"].tolist(), st["table"].tolist()
    if sum(n // tokens + 2 for n in added) > 6000:
        return None
    for name in ("k", "v"):
        values, scale = e4m3(st[name + "_cache"]).double(), st[name + "_scale"]
        for i, (n, m) in enumerate(zip(lengths, added)):
            at = n
            while at < n + m:
                begin, end = at // tokens * tokens, min(n + m, at // tokens * tokens + tokens)
                p, row, block = table[i][at // page], begin % page, begin % page // tokens
                new = st[name][i, :, at - n:end - n].double()
                code = torch.ceil(torch.log2(new.abs().amax((1, 2)) / 448.0)) + 127
                code = torch.where(torch.isinf(code), 0.0, code)
                if at > begin:
                    old = scale[p, :, block, 0].double()
                    code = torch.maximum(code, old)
                    values[p, :, row:row + at - begin] = exact_e4m3(values[p, :, row:row + at - begin] * torch.exp2(old - code)[:, None, None])
                values[p, :, row + at - begin:row + end - begin] = exact_e4m3(new / torch.exp2(code - 127)[:, None, None])
                at = end
        out += [values, None]
    return out + [None]


def exact_attend(st):
    """Sequence by sequence, in 64 bits."""
    case = st["case"]
    sq, hk, grp, d, page = (case[k] for k in ("sq", "hk", "g", "d", "page"))
    o = torch.zeros(st["q"].shape, device="cuda", dtype=torch.float64)
    stats = torch.full(st["stats"].shape, float("-inf"), device="cuda", dtype=torch.float64)
    for i, n in enumerate(st["lengths"].tolist()):
        if n == 0:
            continue
        at = torch.arange(n, device="cuda")
        ids = st["table"][i].long()[at // page]
        parts = []
        for name in ("k", "v"):
            codes = e4m3(st[name + "_cache"][ids, :, at % page]).double()               # [n, hk, d]
            power = st[name + "_scale"][ids, :, at % page // case["tokens"], 0].double() - 127.0
            parts.append(codes * torch.exp2(power)[..., None])
        for t in range(0, sq, 128):
            query = torch.arange(t, min(sq, t + 128), device="cuda")
            limit = n - sq + query
            seen = at <= limit[:, None]
            if case["window"]:
                seen &= at > limit[:, None] - case["window"]
            for h in range(hk * grp):
                scores = st["q"][i, h, query].double() @ parts[0][:, h // grp].T / d ** 0.5
                scores[~seen] = float("-inf")
                some = seen.any(1)
                stats[i, h, query] = torch.logsumexp(scores, 1)
                o[i, h, query] = torch.where(some[:, None], torch.softmax(scores, 1) @ parts[1][:, h // grp], 0.0)
    return [o, stats]
