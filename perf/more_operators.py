"""Cases on which the operators of a decoder's step around the paged cache are measured: norms of query and key heads with the rotary
positions, products of 8-bit integers with a scale for each token and channel, and beam search.

A case is a dict of plain values whose "op" names the operator:

  norm     RMS norm of every head of queries and keys, its gains and the rotary positions in one call, or their gradients
  linear   activations quantised to 8 bits token by token, and their product with weights quantised channel by channel
  select   the best continuations of beams over beams and vocabulary
  reorder  the states of the beams that go on, gathered by parent

`run` computes the plain form in torch where `own` is false, and makes the framework's calls where it is true.
"""
import torch

own = False

TORCH = {"BFLOAT16": torch.bfloat16, "HALF": torch.float16, "FLOAT": torch.float32, "INT32": torch.int32}
SIZE = {"BFLOAT16": 2, "HALF": 2, "FLOAT": 4, "INT32": 4}
EPSILON = 1e-6


def listed():
    return [
        # one new token for each of 32 users: queries and keys of grouped heads, bound by launch latency
        {"name": "norm_token", "op": "norm", "b": 32, "s": 1, "h": 32, "h2": 8, "d": 128, "rotary": 128, "interleaved": False, "per_head": False, "gradient": False, "io": "BFLOAT16", "far": 100000},
        # whole prompts, far positions
        {"name": "norm_prompts", "op": "norm", "b": 2, "s": 8192, "h": 32, "h2": 8, "d": 128, "rotary": 128, "interleaved": False, "per_head": False, "gradient": False, "io": "BFLOAT16", "far": 1000000},
        # a training step's gradients of activations and gains
        {"name": "norm_gradient", "op": "norm", "b": 4, "s": 2048, "h": 32, "h2": 8, "d": 128, "rotary": 128, "interleaved": False, "per_head": False, "gradient": True, "io": "BFLOAT16", "far": 0},
        # f32 activations, gains of every head, pairs side by side, half of the head rotated, an odd length
        {"name": "norm_gradient_odd", "op": "norm", "b": 3, "s": 1001, "h": 16, "h2": 16, "d": 128, "rotary": 64, "interleaved": True, "per_head": True, "gradient": True, "io": "FLOAT", "far": 0},
        # a projection in a decode step of 32 users: the weights are what has to be read
        {"name": "linear_token", "op": "linear", "m": 32, "k": 4096, "n": 4096, "bias": False, "io": "BFLOAT16"},
        # the same projection over prompts: bound by the products
        {"name": "linear_prompts", "op": "linear", "m": 8192, "k": 4096, "n": 4096, "bias": False, "io": "BFLOAT16"},
        # extents that fill no tile, f16, a bias
        {"name": "linear_odd", "op": "linear", "m": 333, "k": 1000, "n": 1111, "bias": True, "io": "HALF"},
        # one user's beam
        {"name": "select_user", "op": "select", "b": 1, "w": 4, "v": 32000, "finished": 0, "alpha": 0.0, "io": "BFLOAT16"},
        # a batch of beams over a large vocabulary
        {"name": "select_batch", "op": "select", "b": 16, "w": 8, "v": 128000, "finished": 0, "alpha": 0.0, "io": "BFLOAT16"},
        # f32 logits of an odd vocabulary, some beams finished, scores weighed by length
        {"name": "select_odd", "op": "select", "b": 7, "w": 5, "v": 50001, "finished": 20, "alpha": 0.6, "io": "FLOAT"},
        # the token histories of a batch of beams
        {"name": "reorder_tokens", "op": "reorder", "layers": 1, "b": 16, "w": 8, "n": 1000, "states": 2, "io": "INT32"},
        # recurrent states or dense caches of several layers
        {"name": "reorder_layers", "op": "reorder", "layers": 8, "b": 8, "w": 4, "n": 131072, "states": 2, "io": "BFLOAT16"},
    ]


MAX_BYTES = {"norm": 3.4e8, "linear": 2.0e8, "select": 3.3e7, "reorder": 2.7e8}
MAX_FLOPS = 2.75e11


def draw(rng):
    def spread(low, high, step=1):
        """A multiple of step in [low, high], spread over the logarithm."""
        value = low * (high / low) ** rng.random()
        return max(low, min(high, int(value / step + 0.5) * step))

    while True:
        op = rng.choice(("norm", "norm", "linear", "linear", "select", "select", "reorder"))
        if op == "norm":
            d = rng.choice((64, 80, 96, 128, 128, 256))
            case = {"b": spread(1, 64), "s": rng.choice((1, spread(1, 8192), spread(1, 8192))), "h": spread(1, 64), "h2": rng.choice((0, 1, 2, 8, 8)), "d": d, "rotary": rng.choice((d, d, d // 2, 0)),
                    "interleaved": rng.random() < 0.4, "per_head": rng.random() < 0.3, "gradient": rng.random() < 0.5, "io": rng.choice(("BFLOAT16", "BFLOAT16", "FLOAT", "HALF")),
                    "far": rng.choice((0, 100000, 1000000))}
        elif op == "linear":
            case = {"m": rng.choice((spread(1, 64), spread(1, 8192))), "k": rng.choice((spread(64, 16384), spread(64, 16384, 64))), "n": rng.choice((spread(64, 32000), spread(64, 16384, 64))),
                    "bias": rng.random() < 0.5, "io": rng.choice(("BFLOAT16", "BFLOAT16", "FLOAT", "HALF"))}
        elif op == "select":
            case = {"b": spread(1, 64), "w": spread(1, 16), "v": spread(100, 256000), "finished": rng.choice((0, 0, 20)), "alpha": rng.choice((0.0, 0.0, 0.6, 1.0)),
                    "io": rng.choice(("BFLOAT16", "BFLOAT16", "FLOAT", "HALF"))}
        else:
            case = {"layers": spread(1, 32), "b": spread(1, 64), "w": spread(1, 16), "n": spread(1, 262144), "states": rng.choice((1, 2, 3)), "io": rng.choice(("BFLOAT16", "FLOAT", "INT32"))}
        case["op"] = op
        w = work(case)
        if w["bytes"] <= MAX_BYTES[op] and w["flops"] <= MAX_FLOPS:
            return case


def work(case):
    """What one pass cannot do without: inputs read once, outputs written once."""
    op, size = case["op"], SIZE[case["io"]]
    if op == "norm":
        heads = case["h"] + case["h2"]
        values = case["b"] * case["s"] * heads * case["d"]
        gains = 4 * case["d"] * (heads if case["per_head"] else 1 + (case["h2"] > 0))
        if case["gradient"]:
            return {"bytes": 3 * values * size + 4 * case["b"] * case["s"] + 2 * gains, "flops": 10 * values + 3 * values * case["rotary"] // case["d"]}
        return {"bytes": 2 * values * size + 4 * case["b"] * case["s"] + gains, "flops": 4 * values + 3 * values * case["rotary"] // case["d"]}
    if op == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k * (size + 1) + 4 * m + n * k + 4 * n + m * n * size + (n * size if case["bias"] else 0), "flops": 2 * m * k * n}
    if op == "select":
        rows = case["b"] * case["w"]
        live = rows - finished_of(case) * case["b"]
        return {"bytes": live * case["v"] * size + 40 * rows, "flops": 3 * live * case["v"]}
    values = case["layers"] * case["b"] * case["w"] * case["n"] * case["states"]
    return {"bytes": 2 * values * size + 4 * case["b"] * case["w"], "flops": values}


def finished_of(case):
    """Finished beams of each batch entry."""
    return case["w"] * case["finished"] // 100


# ---- inputs ------------------------------------------------------------------------------

def prepare(case, seed):
    return {"norm": prepare_norm, "linear": prepare_linear, "select": prepare_select, "reorder": prepare_reorder}[case["op"]](case, seed)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def prepare_norm(case, seed):
    g = generator(seed)
    b, s, d, io = case["b"], case["s"], case["d"], TORCH[case["io"]]
    st = {"case": case}
    if case["rotary"]:
        half = case["rotary"] // 2
        st["frequencies"] = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).to(torch.float32).cuda()
        start = torch.randint(0, case["far"] + 1, (b, 1), device="cuda", generator=g)
        st["positions"] = (start + torch.arange(s, device="cuda")).to(torch.int32)
    for suffix, heads in (("", case["h"]), ("2", case["h2"])):
        if not heads:
            continue
        magnitude = torch.exp2(torch.randint(-2, 3, (b, heads, 1, 1), device="cuda", generator=g).to(torch.float32))   # heads differ in size
        st["x" + suffix] = (torch.randn(b, heads, s, d, device="cuda", generator=g) * magnitude).to(io)
        st["gain" + suffix] = 1.0 + 0.3 * torch.randn(heads if case["per_head"] else 1, d, device="cuda", generator=g)
        if case["gradient"]:
            st["dy" + suffix] = torch.randn(b, heads, s, d, device="cuda", generator=g).to(io)
            st["dgain" + suffix] = torch.empty_like(st["gain" + suffix])
        st["out" + suffix] = torch.empty_like(st["x" + suffix])
    return st


def padded(columns):
    """Columns of a row that starts on a 16-byte boundary, as a program lays out 8-bit operands."""
    return (columns + 15) // 16 * 16


def prepare_linear(case, seed):
    g = generator(seed)
    m, k, n, io = case["m"], case["k"], case["n"], TORCH[case["io"]]
    loud = torch.where(torch.rand(k, device="cuda", generator=g) < 0.01, 16.0, 1.0)       # a few channels are far larger than the others
    st = {"case": case, "x": (torch.randn(m, k, device="cuda", generator=g) * loud).to(io)}
    st["weights"] = torch.zeros(n, padded(k), device="cuda", dtype=torch.int8)             # [N, K] with K contiguous, largest magnitude 127 in every row
    codes = torch.randn(n, k, device="cuda", generator=g)
    st["weights"][:, :k] = torch.round(codes * (127.0 / codes.abs().amax(1, keepdim=True))).to(torch.int8)
    st["weight_scale"] = (0.02 + 0.01 * torch.rand(n, device="cuda", generator=g)) / 127.0
    if case["bias"]:
        st["bias"] = torch.randn(n, device="cuda", generator=g).to(io)
    st["codes"] = torch.zeros(m, padded(k), device="cuda", dtype=torch.int8)
    st["scale"] = torch.empty(m, device="cuda")
    st["y"] = torch.empty(m, n, device="cuda", dtype=io)
    return st


def prepare_select(case, seed):
    g = generator(seed)
    b, w, v = case["b"], case["w"], case["v"]
    st = {"case": case, "logits": (3.0 * torch.randn(b, w, v, device="cuda", generator=g)).to(TORCH[case["io"]])}
    st["scores"] = -20.0 * torch.rand(b, w, device="cuda", generator=g) - 5.0
    order = torch.rand(b, w, device="cuda", generator=g).argsort(1)
    st["finished"] = (order < finished_of(case)).to(torch.int32)
    st["lengths"] = torch.randint(1, 200, (b, w), device="cuda", generator=g).to(torch.int32)
    st["scores_out"] = torch.empty(b, w, device="cuda")
    for name in ("tokens", "parents", "finished_out", "lengths_out"):
        st[name] = torch.empty(b, w, device="cuda", dtype=torch.int32)
    return st


END, PAD = 2, 0   # ids of the token that ends a sequence and of the one behind it


def prepare_reorder(case, seed):
    g = generator(seed)
    shape, io = (case["layers"], case["b"], case["w"], case["n"]), TORCH[case["io"]]
    st = {"case": case, "parents": torch.randint(0, case["w"], (case["b"], case["w"]), device="cuda", generator=g).to(torch.int32)}
    if io == torch.int32:
        st["states"] = [torch.randint(0, 128000, shape, device="cuda", generator=g, dtype=io) for _ in range(case["states"])]
    else:
        st["states"] = [torch.randn(shape, device="cuda", generator=g).to(io) for _ in range(case["states"])]
    st["moved"] = [torch.empty_like(t) for t in st["states"]]
    return st


# ---- one pass --------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": own_norm, "linear": own_linear, "select": own_select, "reorder": own_reorder}[op](state)
    return {"norm": plain_norm, "linear": plain_linear, "select": plain_select, "reorder": plain_reorder}[op](state)


def plain_turn(x, cosine, sine, rotary, interleaved):
    turned, rest = x[..., :rotary], x[..., rotary:]
    if interleaved:
        first, second = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([first * cosine - second * sine, second * cosine + first * sine], -1).flatten(-2)
    else:
        first, second = turned[..., : rotary // 2], turned[..., rotary // 2:]
        turned = torch.cat([first * cosine - second * sine, second * cosine + first * sine], -1)
    return torch.cat([turned, rest], -1)


def plain_norm(st):
    case = st["case"]
    rotary = case["rotary"]
    if rotary:
        angles = st["positions"].to(torch.float64)[:, None, :, None] * st["frequencies"].to(torch.float64)   # (far positions: f32 loses the angle)
        cosine, sine = torch.cos(angles).float(), torch.sin(angles).float()
    out = []
    for suffix in ("", "2"):
        if "x" + suffix not in st:
            continue
        x, gain = st["x" + suffix].float(), st["gain" + suffix][None, :, None]
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON)
        if not case["gradient"]:
            y = x * r * gain
            if rotary:
                y = plain_turn(y, cosine, sine, rotary, case["interleaved"])
            out.append(y.to(st["x" + suffix].dtype))
            continue
        u = st["dy" + suffix].float()
        if rotary:
            u = plain_turn(u, cosine, -sine, rotary, case["interleaved"])
        v = u * gain
        out.append((r * (v - x * (r * r * (v * x).mean(-1, keepdim=True)))).to(st["x" + suffix].dtype))
        dgain = (u * (x * r)).sum((0, 2), dtype=torch.float64)
        out.append((dgain if case["per_head"] else dgain.sum(0, keepdim=True)).float())
    return out


def plain_linear(st):
    case = st["case"]
    k = case["k"]
    x = st["x"].float()
    scale = x.abs().amax(1)
    scale = scale / torch.full_like(scale, 127.0)   # (by a tensor: a quotient rounded once)
    codes = torch.where(scale[:, None] > 0, torch.round(x / scale[:, None]), 0.0).clamp(-127.0, 127.0)
    weights = st["weights"][:, :k].float()
    total = 0.0
    for at in range(0, k, 1024):   # 1024 products of 8 bits are exact in 32-bit floats
        total = total + (codes[:, at:at + 1024] @ weights[:, at:at + 1024].T).double()
    y = total.float() * scale[:, None] * st["weight_scale"]
    if case["bias"]:
        y = y + st["bias"].float()
    return [codes.to(torch.int8), scale, y.to(st["x"].dtype)]


def plain_select(st):
    """Scores in 64 bits: two of them may be next to each other at the border of what is kept."""
    case = st["case"]
    b, w, v = case["b"], case["w"], case["v"]
    logits = st["logits"].double()
    top = logits.amax(2, keepdim=True)
    total = st["scores"].double()[..., None] + (logits - top - torch.log(torch.exp(logits - top).sum(2, keepdim=True)))
    done = st["finished"] > 0
    pad = torch.zeros(v, device="cuda", dtype=torch.bool)
    pad[PAD] = True
    total = torch.where(done[..., None], torch.where(pad, st["scores"].double()[..., None], -float("inf")), total)
    lengths = st["lengths"] + (~done).to(torch.int32)
    worth = total / lengths.double()[..., None] ** case["alpha"]
    worth, total = worth.view(b, w * v), total.view(b, w * v)
    index = torch.arange(w * v, device="cuda")
    chosen = []
    for _ in range(w):
        best = worth.amax(1, keepdim=True)
        at = torch.where(worth == best, index, w * v).amin(1, keepdim=True)   # (equals: the lowest index)
        chosen.append(at)
        worth.scatter_(1, at, -float("inf"))
    chosen = torch.cat(chosen, 1)
    parents, tokens = chosen // v, chosen % v
    ended = torch.gather(done, 1, parents) | (tokens == END)
    return [torch.gather(total, 1, chosen).float(), tokens.to(torch.int32), parents.to(torch.int32), ended.to(torch.int32), torch.gather(lengths, 1, parents)]


def plain_reorder(st):
    parents = st["parents"].long()
    rows = torch.arange(parents.shape[0], device="cuda")[:, None]
    return [t[:, rows, parents] for t in st["states"]]


# ---- the framework's calls ----------------------------------------------------------------------

DTYPE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2, torch.int32: 5}   # FLOAT, HALF, BFLOAT16, INT32 of the C ABI
F32, I32 = 0, 5


def own_norm(st):
    from deepforge_b200 import decoder
    case, tensor = st["case"], decoder.tensor
    names = [n for n in ("", "2") if "x" + n in st]
    if "call" not in st:   # the descriptors that a program fills once
        p = (decoder.HeadNormGradParams if case["gradient"] else decoder.HeadNormParams)(interleaved=case["interleaved"], scale=1.0, epsilon=EPSILON)
        for n in names:
            io = tensor(DTYPE[st["x" + n].dtype], st["x" + n].shape)
            gain = tensor(F32, [1, st["gain" + n].shape[0], 1, case["d"]])
            for field in ("x", "dy", "dx") if case["gradient"] else ("x", "y"):
                setattr(p, field + n, io)
            for field in ("gain", "dgain") if case["gradient"] else ("gain",):
                setattr(p, field + n, gain)
        if case["rotary"]:
            p.positions = tensor(I32, [case["b"], 1, case["s"], 1])
            p.frequencies = tensor(F32, [1, 1, 1, case["rotary"] // 2])
        st["call"] = p
        if case["gradient"]:
            st["scratch"] = torch.empty(max(1, decoder.query("head_norm_grad", p).scratch_bytes), device="cuda", dtype=torch.uint8)
    angles = [st[n].data_ptr() if n in st else None for n in ("positions", "frequencies")]
    fields = ("x", "dy", "out", "gain", "dgain") if case["gradient"] else ("x", "out", "gain")
    first, second = ([st[f + n].data_ptr() if f + n in st else None for f in fields] for n in ("", "2"))
    if case["gradient"]:
        decoder.head_norm_grad(st["call"], first + angles + second, st["scratch"].data_ptr())
        return [st[f + n] for n in names for f in ("out", "dgain")]
    decoder.head_norm(st["call"], first + angles + second)
    return [st["out" + n] for n in names]


def own_linear(st):
    from deepforge_b200 import decoder
    case, tensor = st["case"], decoder.tensor
    if "calls" not in st:
        m, k, n, wide = case["m"], case["k"], case["n"], padded(case["k"])
        io = DTYPE[st["x"].dtype]
        q = decoder.TokenQuantizeParams()
        q.x, q.y, q.scale = tensor(io, [m, k]), tensor(decoder.I8, [m, k], [wide, 1]), tensor(F32, [m, 1])
        p = decoder.MatmulInt8Params()
        p.a, p.b, p.c = q.y, tensor(decoder.I8, [k, n], [1, wide]), tensor(io, [m, n])
        p.a_scale, p.b_scale = q.scale, tensor(F32, [1, n])
        if case["bias"]:
            p.bias = tensor(io, [1, n])
        st["calls"] = q, p
    q, p = st["calls"]
    codes, scale = st["codes"].data_ptr(), st["scale"].data_ptr()
    decoder.token_quantize(q, [st["x"].data_ptr(), codes, scale])
    decoder.matmul_int8(p, [codes, st["weights"].data_ptr(), st["y"].data_ptr(), scale, st["weight_scale"].data_ptr(), st["bias"].data_ptr() if case["bias"] else None])
    return [st["codes"][:, : case["k"]], st["scale"], st["y"]]


def own_select(st):
    from deepforge_b200 import decoder
    case, tensor = st["case"], decoder.tensor
    if "call" not in st:
        b, w = case["b"], case["w"]
        p = decoder.BeamSelectParams(length_penalty=case["alpha"], end=END, pad=PAD)
        p.logits = tensor(DTYPE[st["logits"].dtype], st["logits"].shape)
        p.scores = p.scores_out = tensor(F32, [b, w])
        p.finished = p.lengths = p.tokens = p.parents = p.finished_out = p.lengths_out = tensor(I32, [b, w])
        st["call"] = p
        st["scratch"] = torch.empty(max(1, decoder.query("beam_select", p).scratch_bytes), device="cuda", dtype=torch.uint8)
    names = ("logits", "scores", "finished", "lengths", "scores_out", "tokens", "parents", "finished_out", "lengths_out")
    decoder.beam_select(st["call"], [st[n].data_ptr() for n in names], st["scratch"].data_ptr())
    return [st[n] for n in names[4:]]


def own_reorder(st):
    from deepforge_b200 import decoder
    case, tensor = st["case"], decoder.tensor
    if "call" not in st:
        p = decoder.BeamReorderParams(count=case["states"])
        p.parents = tensor(I32, [case["b"], case["w"]])
        for i, t in enumerate(st["states"]):
            p.source[i] = p.target[i] = tensor(DTYPE[t.dtype], t.shape)
        st["call"] = p
    pointers = [t.data_ptr() for pair in zip(st["states"], st["moved"]) for t in pair]
    decoder.beam_reorder(st["call"], [st["parents"].data_ptr()] + pointers)
    return st["moved"]


# ---- the definitions in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    return {"norm": exact_norm, "linear": exact_linear, "select": exact_select, "reorder": exact_reorder}[case["op"]](prepare(case, seed))


def exact_heads(st, x, gain):
    """The norm as a unit of length sqrt(D), each pair a complex number that the angle turns."""
    case = st["case"]
    half = case["rotary"] // 2
    y = x / torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / case["d"] + EPSILON) * gain[None, :, None]
    if not half:
        return y
    angles = torch.einsum("bs,i->bsi", st["positions"].double(), st["frequencies"].double())
    turn = torch.polar(torch.ones_like(angles), angles)[:, None]
    if case["interleaved"]:
        pairs = torch.view_as_complex(y[..., : 2 * half].unflatten(-1, (half, 2)).contiguous()) * turn
        turned = torch.view_as_real(pairs).flatten(-2)
    else:
        pairs = torch.complex(y[..., :half], y[..., half:2 * half]) * turn
        turned = torch.cat([pairs.real, pairs.imag], -1)
    return torch.cat([turned, y[..., 2 * half:]], -1)


def exact_norm(st):
    case, out = st["case"], []
    for suffix in ("", "2"):
        if "x" + suffix not in st:
            continue
        x, gain = st["x" + suffix].double(), st["gain" + suffix].double()
        if not case["gradient"]:
            out.append(exact_heads(st, x, gain))
            continue
        dx, dgain = torch.empty_like(x), torch.zeros_like(gain)
        for h in range(x.shape[1]):   # (head by head: the graph of a whole tensor in 64 bits takes much memory)
            leaf, row = x[:, h:h + 1].clone().requires_grad_(), gain[h if case["per_head"] else 0].clone().requires_grad_()
            y = exact_heads(st, leaf, row[None])
            dx[:, h:h + 1], more = torch.autograd.grad(y, (leaf, row), st["dy" + suffix][:, h:h + 1].double())
            dgain[h if case["per_head"] else 0] += more
        out += [dx, dgain]
    return out


def exact_linear(st):
    """The scale and its quotients are values of 32 bits (rounding those of 64 once more changes none); everything else is exact."""
    case = st["case"]
    x = st["x"].double()
    largest = x.abs().max(1).values
    scale = largest / torch.full_like(largest, 127.0)
    unit = scale.float().double()[:, None]
    quotients = torch.where(unit == 0, 0.0, x / unit).float()
    codes = torch.sign(quotients) * torch.minimum(torch.round(quotients.abs()), torch.full_like(quotients, 127.0))
    y = (codes.double() * unit) @ (st["weights"][:, : case["k"]].double() * st["weight_scale"].double()[:, None]).T
    return [codes.to(torch.int8), scale, y + st["bias"].double() if case["bias"] else y]


def exact_select(st):
    """Entry by entry: candidates of all beams in a list, sorted by worth, then by beam and token."""
    case = st["case"]
    w, scores_out, tokens_out, parents_out, finished_out, lengths_out = case["w"], [], [], [], [], []
    scores, finished, lengths = st["scores"].double(), st["finished"].tolist(), st["lengths"].tolist()
    for i in range(case["b"]):
        worth, score, parent, token = [], [], [], []
        for j in range(w):
            if finished[i][j]:
                s, t, n = scores[i, j:j + 1], torch.tensor([PAD], device="cuda"), lengths[i][j]
            else:
                row = torch.log_softmax(st["logits"][i, j].double(), 0)
                order = torch.sort(row, descending=True, stable=True).indices[:w]
                s, t, n = row[order] + scores[i, j], order, lengths[i][j] + 1
            worth += (s / float(n) ** case["alpha"]).tolist()
            score += s.tolist()
            token += t.tolist()
            parent += [j] * len(t)
        best = sorted(range(len(worth)), key=lambda c: (-worth[c], parent[c], token[c]))[:w]
        scores_out.append([score[c] for c in best])
        tokens_out.append([token[c] for c in best])
        parents_out.append([parent[c] for c in best])
        finished_out.append([int(finished[i][parent[c]] or token[c] == END) for c in best])
        lengths_out.append([lengths[i][parent[c]] + (0 if finished[i][parent[c]] else 1) for c in best])
    whole = [torch.tensor(values, device="cuda", dtype=torch.int32) for values in (tokens_out, parents_out, finished_out, lengths_out)]
    return [torch.tensor(scores_out, device="cuda", dtype=torch.float64)] + whole


def exact_reorder(st):
    rows = st["parents"].tolist()
    return [torch.stack([torch.stack([t[:, i, p] for p in row], 1) for i, row in enumerate(rows)], 1) for t in st["states"]]
