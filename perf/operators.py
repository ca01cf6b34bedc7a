"""Cases of the 8-bit weight operators: cast to blocks of 128 with a scale each, the product of two such matrices, and the
AdamW step over every key of an arena.

A block-scaled matrix is e4m3 codes [rows, cols] whose rows start 128 bytes apart or a multiple of it (zeros behind the last
column), and a scale for every 128 columns: of each row ("rows"), or of each 128 x 128 square ("tile").  value = code * scale.
Scales are float32 or powers of two (float8_e8m0fnu).

The optimizer's 8-bit states are e4m3 codes and a power-of-two scale for every 128 elements of the arena: the first moment, and
the ROOT of the second.  They are rounded up or down with probabilities given by a hash of the element's offset, the step's
number and a seed, so that a mean which moves by less than a code's distance still moves on average.
"""
import math

import torch

own = False

BLOCK = 128
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "e8m0": torch.float8_e8m0fnu}
SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
BETAS, EPS, LR = (0.9, 0.999), 1e-8, 1e-4


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the text encoder's 77 x 768 context, quantised by rows for one product: a call whose launch is most of its time
        dict(name="cast_context", op="cast", rows=77, cols=768, type="bf16", tile=False, sides="straight"),
        # a merged fp32 key of the feed-forward projection turned into 128 x 128 squares, for the product and for its gradient
        dict(name="cast_weight_both", op="cast", rows=10240, cols=1280, type="fp32", tile=True, sides="both"),
        # output gradients of an odd number of tokens by rows, along the channels (input gradient) and along the tokens (weight's)
        dict(name="cast_gradient_both", op="cast", rows=8269, cols=5120, type="bf16", tile=False, sides="both"),
        # an 8-bit key back to 16 bits, to be merged
        dict(name="uncast_weight", op="uncast", rows=5120, cols=2816, type="bf16", tile=True, scales="e8m0"),
        # the label embedding of one conditioned and one unconditioned sample: two rows, the weight's bytes are everything
        dict(name="product_two_rows", op="product", m=2, n=1280, k=2816, a="rows", b="tile", scales="e8m0", type="bf16", base=False),
        # keys of the cross attention for two contexts of 77 tokens, a stored checkpoint with float32 scales
        dict(name="product_context", op="product", m=154, n=640, k=2048, a="rows", b="tile", scales="fp32", type="fp16", base=False),
        # the feed-forward projection of 8192 tokens
        dict(name="product_forward", op="product", m=8192, n=10240, k=1280, a="rows", b="tile", scales="e8m0", type="bf16", base=False),
        # the same from float32 scales, an odd number of tokens, onto the residual
        dict(name="product_residual", op="product", m=8269, n=1280, k=5120, a="rows", b="tile", scales="fp32", type="bf16", base=True),
        # a weight's gradient over an odd number of tokens, added to what a float32 gradient holds already
        dict(name="product_weight_gradient", op="product", m=1280, n=5120, k=8269, a="rows", b="rows", scales="e8m0", type="fp32", base=True),
        # rank-8 factors of one narrow transformer block: twenty small keys, float32 throughout
        dict(name="adamw_factors", op="adamw", width=320, context=768, depth=1, rank=8, param="fp32", grad="fp32", copy="", bits=32, clip=False),
        # five wide blocks in full, float32 weights and a 16-bit copy of them for the next step, 16-bit gradients, clipped
        dict(name="adamw_blocks", op="adamw", width=1280, context=2048, depth=5, rank=0, param="fp32", grad="bf16", copy="bf16", bits=32, clip=True),
        # ten of them with 8-bit states and 16-bit weights
        dict(name="adamw_blocks_8bit", op="adamw", width=1280, context=2048, depth=10, rank=0, param="bf16", grad="bf16", copy="", bits=8, clip=False),
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["cast", "uncast", "product", "product", "adamw"])
    if op in ("cast", "uncast"):
        c = dict(op=op, rows=size(1, 16384), cols=size(32, 10240), type=rng.choice(["fp32", "fp16", "bf16"]), tile=rng.random() < 0.5)
        c["cols"] = min(c["cols"], 42_000_000 // c["rows"])
        c.update(dict(sides=rng.choice(["straight", "transposed", "both"])) if op == "cast" else dict(scales=rng.choice(["e8m0", "fp32"])))
        return c
    if op == "product":
        m, n, k = size(1, 16384), size(64, 10240), size(64, 8192)
        m = max(1, min(m, int(1.0e11 / (n * k))))
        return dict(op=op, m=m, n=n, k=k, a=rng.choice(["rows", "tile"]), b=rng.choice(["rows", "tile"]), scales=rng.choice(["e8m0", "fp32"]),
                    type=rng.choice(["fp32", "fp16", "bf16"]), base=rng.random() < 0.4)
    width = size(200, 1280)
    return dict(op=op, width=width, context=size(512, 2048), depth=rng.randint(1, 5), rank=rng.choice([0, 0, size(1, 128)]),
                param=rng.choice(["fp32", "fp32", "bf16"]), grad=rng.choice(["fp32", "bf16", "fp16"]), copy=rng.choice(["", "bf16", "fp16"]),
                bits=rng.choice([32, 8]), clip=rng.random() < 0.5)


def keys_of(case):
    """Element counts of the keys that are trained: the matrices, biases and norms of `depth` transformer blocks, or (rank > 0) the
    two factors of every matrix."""
    w, c, r = case["width"], case["context"], case["rank"]
    mats = [(w, w)] * 4 + [(w, w), (w, c), (w, c), (w, w)] + [(8 * w, w), (w, 4 * w)]
    if r:
        return [n for _ in range(case["depth"]) for o, i in mats for n in (o * r, r * i)]
    return [n for _ in range(case["depth"]) for n in [o * i for o, i in mats] + [w, w, 8 * w, w] + [w] * 6]


def arena_of(case):
    """(offsets, counts, length): each key starts at a multiple of 128 elements."""
    counts = keys_of(case)
    offsets, at = [], 0
    for n in counts:
        offsets.append(at)
        at += (n + BLOCK - 1) // BLOCK * BLOCK
    return offsets, counts, at


def blocks(n):
    return (n + BLOCK - 1) // BLOCK


# --------------------------------------------------------------------------------------------------------------- inputs
def matrix(g, rows, cols, form, scales):
    """A block-scaled matrix as a checkpoint or a cast leaves it: (codes [rows, cols], scales)."""
    codes = torch.zeros(rows, blocks(cols) * BLOCK, device="cuda", dtype=torch.float8_e4m3fn)
    codes[:, :cols] = (torch.randn(rows, cols, device="cuda", generator=g) * 120).clamp_(-448, 448).to(torch.float8_e4m3fn)
    shape = (rows if form == "rows" else blocks(rows), blocks(cols))
    if scales == "e8m0":
        s = torch.randint(113, 119, shape, device="cuda", generator=g, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    else:
        s = torch.rand(shape, device="cuda", generator=g) * 2.0 ** -9 + 2.0 ** -12
    return codes[:, :cols], s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case=case)
    if case["op"] == "cast":
        a = torch.randn(case["rows"], case["cols"], device="cuda", generator=g)
        a *= torch.exp(torch.randn(case["rows"], 1, device="cuda", generator=g))        # rows differ in size, and so do columns
        a *= torch.exp(torch.randn(1, case["cols"], device="cuda", generator=g)) * 0.02
        state["a"] = a.to(TYPES[case["type"]])
    elif case["op"] == "uncast":
        state["a"] = matrix(g, case["rows"], case["cols"], "tile" if case["tile"] else "rows", case["scales"])
    elif case["op"] == "product":
        state["a"] = matrix(g, case["m"], case["k"], case["a"], case["scales"])
        state["b"] = matrix(g, case["n"], case["k"], case["b"], case["scales"])
        if case["base"]:
            state["base"] = torch.randn(case["m"], case["n"], device="cuda", generator=g).to(TYPES[case["type"]])
    else:
        offsets, counts, total = arena_of(case)
        filled = torch.zeros(total, device="cuda")
        for o, n in zip(offsets, counts):
            filled[o:o + n] = 1.0

        def noise(size):
            return torch.randn(total, device="cuda", generator=g).mul_(size).mul_(filled)

        state["segments"] = torch.tensor([[o, n] for o, n in zip(offsets, counts)], dtype=torch.int64).cuda()
        state["decay"] = torch.tensor([0.01 if n > 8 * case["width"] or case["rank"] else 0.0 for n in counts]).cuda()
        state["step"] = 1 + seed % 1000
        state["params"] = noise(0.02).to(TYPES[case["param"]])
        state["grads"] = noise(1e-3).to(TYPES[case["grad"]])
        state["copy"] = torch.zeros(total, device="cuda", dtype=TYPES[case["copy"]]) if case["copy"] else None
        mean, root = noise(2e-4), noise(3e-4).abs_().add_(5e-4).mul_(filled)
        if case["bits"] == 32:
            state["mean"], state["square"] = mean, root.square_()
        else:
            state["mean"], state["mean_scale"] = to_blocks_flat(mean)
            state["square"], state["square_scale"] = to_blocks_flat(root)
    return state


# ----------------------------------------------------------------------------------------------------------- plain form
def exponent_of(largest):
    """The smallest e with largest <= 448 * 2^e, from the bits of a float32: 448 = 1.75 * 2^8."""
    bits = largest.view(torch.int32)
    return ((bits >> 23) - 135 + ((bits & 0x7FFFFF) > 0x600000).to(torch.int32)).clamp_(min=-127)


def power(e):
    """2^e, normal numbers only."""
    return ((e + 127) << 23).view(torch.float32)


def e8m0(e):
    return (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def to_blocks_flat(x):
    """Flat float32 [n], n a multiple of 128, to the nearest codes."""
    rows = x.view(-1, BLOCK)
    e = exponent_of(rows.abs().amax(dim=1))
    return (rows * power(-e)[:, None]).to(torch.float8_e4m3fn).view(-1), e8m0(e)


def spread(scales, rows, cols):
    """One scale an element."""
    s = scales.to(torch.float32)
    if s.shape[0] != rows:
        s = s.repeat_interleave(BLOCK, 0)[:rows]
    return s.repeat_interleave(BLOCK, 1)[:, :cols]


def plain_cast(a, tile):
    rows, cols = a.shape
    tall = blocks(rows) * BLOCK if tile else rows
    x = torch.zeros(tall, blocks(cols) * BLOCK, device=a.device)
    x[:rows, :cols] = a
    x4 = x.view(tall // BLOCK, BLOCK, -1, BLOCK) if tile else x.view(tall, 1, -1, BLOCK)
    e = exponent_of(x4.abs().amax(dim=(1, 3)))
    codes = (x4 * power(-e)[:, None, :, None]).to(torch.float8_e4m3fn)
    return codes.view(tall, -1)[:rows, :cols], e8m0(e)


def mix(n, step, seed, device):
    """32 bits for each offset: products by odd constants (the first 32 fractional bits of the golden ratio and of square roots) and
    shifts to the right, modulo 2^32."""
    low = 0xFFFFFFFF
    i = torch.arange(n, device=device)
    x = ((i & low) * 0x9E3779B9) & low
    x ^= x >> 16
    x = (x * 0x6A09E667) & low
    x = (x + step * 0x3C6EF373 + seed * 0x6A09E667 + (i >> 32) * 0xBB67AE85) & low
    x ^= x >> 15
    x = (x * 0xBB67AE85) & low
    return x ^ (x >> 16)


def dithered(x, u, least):
    """Codes and scales of the blocks of 128 of x; |x| goes down to a code with probability 1 - f and up with f, f its part of the
    codes' distance: floor(|x| / distance + u / 2^16).  `least`: what is not zero stays so."""
    rows = x.view(-1, BLOCK)
    e = exponent_of(rows.abs().amax(dim=1))
    y = rows * power(-e)[:, None]
    size = y.abs()
    small = size < 2.0 ** -6
    bits = torch.where(small, size + 2.0 ** -6, size).view(torch.int32)
    code = ((bits + (u.view(-1, BLOCK) << 4).to(torch.int32)) >> 20) - torch.where(small, 968, 960).to(torch.int32)
    if least:
        code = torch.where(size > 0, code.clamp(min=1), code)
    code = code | ((y.view(torch.int32) >> 24) & 0x80)
    return code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1), e8m0(e)


def plain_adamw(s):
    case, step = s["case"], s["step"]
    g = s["grads"].to(torch.float32)
    norm = None
    if case["clip"]:
        norm = g.double().square().sum().sqrt().float().view(1)
        g = g * (1.0 / (norm + 1e-6)).clamp(max=1.0)
    lengths = torch.cat([s["segments"][1:, 0], torch.full((1,), g.numel(), device=g.device)]) - s["segments"][:, 0]
    keep = torch.repeat_interleave(1.0 - LR * s["decay"], lengths, output_size=g.numel())
    size, root_size = LR / (1.0 - BETAS[0] ** step), 1.0 / math.sqrt(1.0 - BETAS[1] ** step)
    if case["bits"] == 32:
        m, v = s["mean"], s["square"]
    else:
        m = s["mean"].to(torch.float32) * spread(s["mean_scale"][None], 1, g.numel())[0]
        v = (s["square"].to(torch.float32) * spread(s["square_scale"][None], 1, g.numel())[0]).square()
    m = m * BETAS[0] + g * (1.0 - BETAS[0])
    v = v * BETAS[1] + g * g * (1.0 - BETAS[1])
    root = v.sqrt()
    p = s["params"].to(torch.float32) * keep - m / (root * root_size + EPS) * size
    s["params"].copy_(p)
    if s["copy"] is not None:
        s["copy"].copy_(p)
    if case["bits"] == 32:
        s["mean"].copy_(m)
        s["square"].copy_(v)
    else:
        u = mix(g.numel(), step, 7, g.device)
        mean, mean_scale = dithered(m, u & 0xFFFF, False)
        square, square_scale = dithered(root, u >> 16, True)
        s["mean"].copy_(mean)
        s["mean_scale"].copy_(mean_scale)
        s["square"].copy_(square)
        s["square_scale"].copy_(square_scale)
    return norm


def run(state):
    case = state["case"]
    if own:
        import sd_mecha_amd as amd
    if case["op"] == "cast":
        a, sides = state["a"], case["sides"]
        if own:
            got = amd.cast_blocks(a, tile=case["tile"], sides=sides, check_finite=False)
            got = [got] if sides != "both" else list(got)
            return [(q.values, q.scales) for q in got]
        got = [plain_cast(a, case["tile"])] if sides != "transposed" else []
        return got + ([plain_cast(a.t(), case["tile"])] if sides != "straight" else [])
    if case["op"] == "uncast":
        values, scales = state["a"]
        if own:
            return amd.uncast_blocks(amd.BlockScaled(values, scales), out_dtype=TYPES[case["type"]], check_finite=False)
        return (values.to(torch.float32) * spread(scales, *values.shape)).to(TYPES[case["type"]])
    if case["op"] == "product":
        (a, sa), (b, sb), base = state["a"], state["b"], state.get("base")
        if own:
            return amd.block_product(amd.BlockScaled(a, sa), amd.BlockScaled(b, sb), base=base, alpha=0.5, out_dtype=TYPES[case["type"]],
                                     check_finite=False)
        out = (a.to(torch.float32) * spread(sa, *a.shape)) @ (b.to(torch.float32) * spread(sb, *b.shape)).t()
        return (out * 0.5 if base is None else base.to(torch.float32) + out * 0.5).to(TYPES[case["type"]])
    if own:
        norm = amd.adamw_step(state["params"], state["grads"], state["mean"], state["square"], state["segments"], step=state["step"], lr=LR,
                              betas=BETAS, eps=EPS, weight_decay=state["decay"], max_norm=1.0 if case["clip"] else None, copy=state["copy"],
                              exp_avg_scales=state.get("mean_scale"), exp_avg_sq_scales=state.get("square_scale"), seed=7)
    else:
        norm = plain_adamw(state)
    return [state[k] for k in ("params", "mean", "square", "copy", "mean_scale", "square_scale") if state.get(k) is not None] + ([norm] if norm is not None else [])


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "cast":
        n = case["rows"] * case["cols"]
        sides = 2 if case["sides"] == "both" else 1
        scales = blocks(case["rows"]) * blocks(case["cols"]) if case["tile"] else n // BLOCK
        return {"bytes": n * SIZE[case["type"]] + sides * (n + scales), "flops": 2 * n}
    if case["op"] == "uncast":
        n = case["rows"] * case["cols"]
        scales = blocks(case["rows"]) * blocks(case["cols"]) if case["tile"] else n // BLOCK
        return {"bytes": n * (1 + SIZE[case["type"]]) + scales * (1 if case["scales"] == "e8m0" else 4), "flops": n}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        each = 1 if case["scales"] == "e8m0" else 4
        scales = sum((r if form == "rows" else blocks(r)) * blocks(k) for r, form in ((m, case["a"]), (n, case["b"])))
        return {"bytes": (m + n) * k + scales * each + m * n * SIZE[case["type"]] * (2 if case["base"] else 1), "flops": 2 * m * n * k}
    n = sum(keys_of(case))
    state = 16 if case["bits"] == 32 else 4 + 4 / BLOCK
    return {"bytes": n * (2 * SIZE[case["param"]] + SIZE[case["grad"]] + state + (SIZE[case["copy"]] if case["copy"] else 0)), "flops": 16 * n}


# ------------------------------------------------------------------------------------------------------- in 64 bits
def nearest_code(y):
    """The e4m3 number nearest to y (|y| <= 448), ties to the even code, in float64."""
    distance = torch.exp2(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1].double() - 4)
    return torch.round(y / distance) * distance


def exponent64(largest):
    mantissa, e = torch.frexp(largest / 448.0)
    return torch.where(largest > 0, e - (mantissa == 0.5).to(e.dtype), -127).clamp(min=-127).double()


def exact_cast(a, tile):
    rows, cols = a.shape
    high = BLOCK if tile else 1
    x = torch.nn.functional.pad(a.double(), (0, -cols % BLOCK, 0, -rows % high))
    x = x.unflatten(0, (-1, high)).unflatten(2, (-1, BLOCK))
    e = exponent64(x.abs().amax(dim=(1, 3)))
    codes = nearest_code(x / torch.exp2(e)[:, None, :, None])
    return codes.flatten(2).flatten(0, 1)[:rows, :cols], torch.exp2(e)


def values64(codes, scales):
    rows, cols = codes.shape
    r, c = torch.arange(rows, device="cuda"), torch.arange(cols, device="cuda") // BLOCK
    return codes.double() * scales.double()[r if scales.shape[0] == rows else r // BLOCK][:, c]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cast":
        return ([exact_cast(s["a"], case["tile"])] if case["sides"] != "transposed" else []) + \
               ([exact_cast(s["a"].t(), case["tile"])] if case["sides"] != "straight" else [])
    if case["op"] == "uncast":
        return values64(*s["a"])
    if case["op"] == "product":
        out = values64(*s["a"]) @ values64(*s["b"]).t() * 0.5
        return out + s["base"].double() if case["base"] else out
    n, t = s["params"].numel(), s["step"]
    g, norm = s["grads"].double(), None
    if case["clip"]:
        norm = torch.linalg.vector_norm(g).view(1)
        g *= min(1.0, 1.0 / (float(norm) + 1e-6))
    if case["bits"] == 32:
        m, v = s["mean"].double(), s["square"].double()
    else:
        m = (s["mean"].double().view(-1, BLOCK) * s["mean_scale"].double()[:, None]).view(-1)
        v = (s["square"].double().view(-1, BLOCK) * s["square_scale"].double()[:, None]).view(-1) ** 2
    m += (1 - BETAS[0]) * (g - m)
    v += (1 - BETAS[1]) * (g * g - v)
    del g
    p = s["params"].double()
    for (o, c), d in zip(s["segments"].tolist(), s["decay"].tolist()):
        p[o:o + c] *= 1 - LR * d
    p -= LR / (1 - BETAS[0] ** t) * m / (torch.sqrt(v / (1 - BETAS[1] ** t)) + EPS)
    copies = [p] if case["copy"] else []
    if case["bits"] == 32:
        states = [m, v] + copies
    else:
        i = torch.arange(n, device="cuda")
        x = (i * 0x9E3779B9) % 2 ** 32
        x = ((x ^ (x >> 16)) * 0x6A09E667 + t * 0x3C6EF373 + 7 * 0x6A09E667) % 2 ** 32
        x = ((x ^ (x >> 15)) * 0xBB67AE85) % 2 ** 32
        x = x ^ (x >> 16)

        def states_of(value, u, least):
            value = value.view(-1, BLOCK)
            e = exponent64(value.abs().amax(dim=1))
            y = value / torch.exp2(e)[:, None]
            distance = torch.exp2(torch.frexp(y.abs().clamp(min=2.0 ** -6))[1].double() - 4)
            code = torch.floor(y.abs() / distance + u.view(-1, BLOCK) / 65536.0) * distance
            if least:
                code = torch.where(y != 0, code.clamp(min=2.0 ** -9), code)
            return (code * torch.sign(y)).view(-1), torch.exp2(e)

        (mc, ms), (vc, vs) = states_of(m, x % 65536, False), states_of(v.sqrt(), x // 65536, True)
        states = [mc, vc] + copies + [ms, vs]
    return [p] + states + ([norm] if norm is not None else [])
