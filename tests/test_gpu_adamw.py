"""The AdamW step over an arena on the GPU against float64 (tests/blocks_reference.py: formulas and the bounds of float32 arithmetic)."""
import numpy as np
import pytest
import torch

import blocks_reference as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NUMELS = [320 * 320, 1, 7, 8, 129, 320, 2560 * 33 + 5, 0, 127, 128, 4096]
HYPER = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-8)


def arena(numels, align=128):
    from sd_mecha_amd.arena import plan_arena
    return plan_arena([(f"k{i}", n) for i, n in enumerate(numels)], align)


def inside(layout):
    m = np.zeros(layout.total_elems, dtype=bool)
    for o, n in zip(layout.offsets, layout.numels):
        m[o:o + n] = True
    return m


def make(layout, p_dt=torch.float32, g_dt=torch.float32, bits=32, seed=0, fill=5.0):
    """States some steps into a run; what lies between the keys is `fill`."""
    import sd_mecha_amd as amd
    g, n = torch.Generator().manual_seed(seed), layout.total_elems
    gap = torch.from_numpy(~inside(layout))

    def put(x, value=fill):
        x[gap] = value
        return x
    p, grad = put(torch.randn(n, generator=g) * 0.02), put(torch.randn(n, generator=g) * 1e-3)
    m, r = torch.randn(n, generator=g) * 2e-4, torch.rand(n, generator=g) * 1e-3 + 1e-5
    s = dict(params=p.to(p_dt).cuda(), grads=grad.to(g_dt).cuda(), segments=layout.device_segments("cuda"))
    if bits == 32:
        s.update(exp_avg=put(m).cuda(), exp_avg_sq=put(r * r).cuda())
    else:
        for name, x in (("exp_avg", m), ("exp_avg_sq", r)):
            q = amd.cast_blocks(put(x, 0.0).view(-1, 128).cuda())
            s[name], s[f"{name}_scales"] = q.values.reshape(-1).contiguous(), q.scales.reshape(-1)
    return s


def f64(t):
    return t.float().cpu().double().numpy() if t.dtype != torch.float64 else t.cpu().numpy()


def scaled(codes, scales):
    return (f64(codes).reshape(-1, 128) * f64(scales)[:, None]).reshape(-1)


def expected(s, layout, step, decay, coef=1.0, lr=1e-3, betas=(0.9, 0.99), eps=1e-8):
    """(p, m, v) in float64 and the bounds, from the states before the step; decay: per key"""
    d = np.zeros(layout.total_elems)
    for o, n, w in zip(layout.offsets, layout.numels, decay):
        d[o:o + n] = w
    if "exp_avg_scales" in s:
        m, v = scaled(s["exp_avg"], s["exp_avg_scales"]), scaled(s["exp_avg_sq"], s["exp_avg_sq_scales"]) ** 2
    else:
        m, v = f64(s["exp_avg"]), f64(s["exp_avg_sq"])
    # float32 of the decays, as the kernel holds them
    return R.adamw(f64(s["params"]), f64(s["grads"]), m, v, step, lr, *betas, eps, d.astype(np.float32).astype(np.float64), coef)


def near(got, want, bound, mask):
    b = bound + (np.abs(want) + bound) * R.HALF[got.dtype] + R.TINY[got.dtype]
    off = np.abs(f64(got) - want)[mask]
    assert (off <= b[mask]).all(), float((off / b[mask]).max())


def check_codes(codes, scales, want, rel, u, least, mask):
    """Codes of `want` (float64, flat) rounded with u: at most one code's distance off where float32's error moves an element over the
    border, |y| / distance <= 16 being off by rel * 16: in a share of that, plus 2^-16 for u's own grid, of the elements."""
    w = np.where(mask, want, 0.0)
    ref, e = R.dithered(w, u, least)
    assert np.array_equal(scales.view(torch.uint8).cpu().numpy().astype(np.float64) - 127, e)
    got = f64(codes)
    assert not got[~mask].any()
    assert (np.abs(got - ref)[mask] <= R.spacing(np.maximum(np.abs(got), np.abs(ref)))[mask]).all()
    share = (got != ref)[mask].mean()
    assert share <= 4 * (16 * rel + 2.0 ** -16) + 3.0 / mask.sum(), share


@pytest.mark.parametrize("p_dt", TYPES)
@pytest.mark.parametrize("g_dt", TYPES)
@pytest.mark.parametrize("step", [1, 1000])
def test_float32_states(p_dt, g_dt, step):
    import sd_mecha_amd as amd
    layout = arena(NUMELS)
    s = make(layout, p_dt, g_dt)
    decay = torch.tensor([0.0 if i % 2 else 0.1 for i in range(len(layout.keys))], device="cuda")
    copy = torch.full((layout.total_elems,), 5.0, dtype=torch.bfloat16, device="cuda")
    want = expected(s, layout, step, decay.cpu().numpy())
    flags = torch.zeros(len(layout.keys), dtype=torch.int32, device="cuda")
    assert amd.adamw_step(**s, step=step, weight_decay=decay, copy=copy, flags=flags, **HYPER) is None
    p, m, v, ep, em, ev = want
    mask = inside(layout)
    near(s["params"], p, ep, mask)
    near(copy, p, ep, mask)
    near(s["exp_avg"], m, em, mask)
    near(s["exp_avg_sq"], v, ev, mask)
    assert not flags.any()
    for t in (s["params"], s["exp_avg"], s["exp_avg_sq"], copy):                     # what lies between the keys
        assert (f64(t)[~mask] == 5.0).all()


@pytest.mark.parametrize("p_dt", TYPES)
@pytest.mark.parametrize("step", [1, 1000])
def test_8bit_states(p_dt, step):
    import sd_mecha_amd as amd
    layout = arena(NUMELS)
    s = make(layout, p_dt, torch.bfloat16, bits=8)
    p, m, v, ep, em, ev = expected(s, layout, step, [0.01] * len(layout.keys))
    amd.adamw_step(**s, step=step, weight_decay=0.01, seed=11, **HYPER)
    mask = inside(layout)
    near(s["params"], p, ep, mask)
    assert (f64(s["params"])[~mask] == 5.0).all()
    u = R.dither(layout.total_elems, step, 11)
    rel = float((em[mask] / np.maximum(np.abs(m[mask]), 1e-30)).mean())              # cancellation: the mean relative error of m
    check_codes(s["exp_avg"], s["exp_avg_scales"], m, rel, (u & np.uint64(0xFFFF)).astype(np.float64), False, mask)
    check_codes(s["exp_avg_sq"], s["exp_avg_sq_scales"], np.sqrt(v), 5 * R.U, (u >> np.uint64(16)).astype(np.float64), True, mask)


def test_8bit_roots_never_vanish_and_zeros_stay():
    """One large gradient in a block: the other roots are far under the smallest code, but not zero; blocks without gradients stay zero."""
    import sd_mecha_amd as amd
    layout = arena([384])
    st = amd.adamw_state(layout, "cuda", 8)
    p = torch.zeros(layout.total_elems, device="cuda")
    g = torch.zeros_like(p)
    g[0], g[1:100] = 1e6, 1e-6
    amd.adamw_step(p, g, segments=layout.device_segments("cuda"), step=1, weight_decay=0.0, **st, **HYPER)
    codes = f64(st["exp_avg_sq"])
    assert codes[0] > 200 and (codes[1:100] == 2.0 ** -9).all() and not codes[100:].any()
    assert (st["exp_avg_sq_scales"].view(torch.uint8)[1:] == 0).all()
    amd.adamw_step(p, torch.zeros_like(g), segments=layout.device_segments("cuda"), step=2, weight_decay=0.0, **st, **HYPER)
    assert bool(p.isfinite().all()) and float(p.abs().max()) < 1e-2 and not p[100:].any()


def test_8bit_codes_between_the_keys():
    """A key's last block of 128 is written whole, zeros behind its last element; blocks that no key reaches into stay as they were."""
    import sd_mecha_amd as amd
    offsets, numels, n = [0, 640, 1024], [130, 1, 384], 1536
    seg = torch.tensor([[o, c] for o, c in zip(offsets, numels)], device="cuda")
    st = amd.adamw_state(n, "cuda", 8)
    for t in st.values():
        t.view(torch.uint8).fill_(0x51)
    p, g = torch.full((n,), 5.0, device="cuda"), torch.ones(n, device="cuda")
    amd.adamw_step(p, g, segments=seg, step=1, **st)
    used, keys = torch.zeros(n, dtype=torch.bool), torch.zeros(n, dtype=torch.bool)
    for o, c in zip(offsets, numels):
        used[o:o + (c + 127) // 128 * 128] = True
        keys[o:o + c] = True
    for name in ("exp_avg", "exp_avg_sq"):
        codes, scales = st[name].view(torch.uint8).cpu(), st[f"{name}_scales"].view(torch.uint8).cpu()
        assert bool((codes[~used] == 0x51).all()) and bool((scales[~used[::128]] == 0x51).all())
        assert not codes[used & ~keys].any() and bool((codes[keys] != 0).all())
    assert bool((p.cpu()[~keys] == 5.0).all())


def test_8bit_second_moment_decays_like_float32():
    """Without gradients the root shrinks by sqrt(beta2) a step.  Rounded to nearest it would never move; here its mean over a key follows."""
    import sd_mecha_amd as amd
    layout = arena([1 << 16])
    st, seg = amd.adamw_state(layout, "cuda", 8), layout.device_segments("cuda")
    n, steps = layout.total_elems, 200
    st["exp_avg_sq"].view(torch.uint8).fill_(0x70)                                  # 2^(14 - 7) = 128
    st["exp_avg_sq_scales"].view(torch.uint8).fill_(127 - 10)
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    for t in range(1, steps + 1):
        amd.adamw_step(p, g, segments=seg, step=t, betas=(0.9, 0.999), **st)
    mean = scaled(st["exp_avg_sq"], st["exp_avg_sq_scales"]).mean() / 2.0 ** -3
    # each rounding is off by less than 1/8 of the value with mean zero: after 200 steps a standard deviation below
    # sqrt(200) / 8 = 1.77 of an element, 1.77 / 256 of the mean of 2^16; five of them
    assert abs(mean - 0.999 ** (steps / 2)) < 5 * 1.77 / 256


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("g_dt", TYPES)
def test_clipping(bits, g_dt):
    import sd_mecha_amd as amd
    layout = arena(NUMELS)
    for limit in (0.05, 1e9):
        s = make(layout, torch.float32, g_dt, bits, seed=3, fill=float("nan") if bits == 32 else 5.0)
        mask = inside(layout)
        g = f64(s["grads"])[mask]
        norm = float(np.sqrt((g * g).sum()))
        coef = min(1.0, limit / (norm + 1e-6))
        want = expected(s, layout, 5, [0.0] * len(layout.keys), coef)
        got = amd.adamw_step(**s, step=5, weight_decay=0.0, max_norm=limit, **HYPER)
        assert got.shape == (1,) and abs(float(got) - norm) <= norm * 2.0 ** -23
        p, m, v, ep, em, ev = want
        # the coefficient is off by three roundings, which count for the gradient's part of m and twice for v's
        extra = 4 * R.U * np.abs(0.1 * f64(s["grads"]) * coef)
        with np.errstate(invalid="ignore"):
            near(s["params"], p, ep + 1e-3 / (1 - 0.9 ** 5) * extra / (np.sqrt(v / (1 - 0.99 ** 5)) + 1e-8) + 8 * R.U * np.abs(p), mask)
        if bits == 32:
            near(s["exp_avg"], m, em + extra, mask)
            near(s["exp_avg_sq"], v, ev + 8 * R.U * v, mask)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_that_is_not_finite(bits):
    """With max_norm the step changes nothing and says so; without, the key's flag word is set and the other keys are as they should be."""
    import sd_mecha_amd as amd
    layout = arena([1000, 300, 5000])
    for value in (float("nan"), float("inf")):
        s = make(layout, bits=bits)
        before = {k: v.clone() for k, v in s.items()}
        s["grads"][layout.offsets[1] + 17] = value
        flags = torch.zeros(3, dtype=torch.int32, device="cuda")
        norm = amd.adamw_step(**s, step=3, max_norm=1.0, flags=flags)
        assert not bool(norm.isfinite()) and flags.tolist() == [0, 1, 0]
        for k in ("params", "exp_avg", "exp_avg_sq"):
            assert torch.equal(s[k].view(torch.uint8), before[k].view(torch.uint8)), k
        flags = torch.zeros(3, dtype=torch.int32, device="cuda")
        clean = {k: v.clone() for k, v in before.items()}
        amd.adamw_step(**s, step=3, flags=flags)
        amd.adamw_step(**clean, step=3)
        assert [int(f) & 1 for f in flags] == [0, 1, 0]
        far = torch.ones(layout.total_elems, dtype=torch.bool, device="cuda")
        far[layout.offsets[1]:layout.offsets[1] + 384] = False
        for k in ("params", "exp_avg", "exp_avg_sq"):
            assert torch.equal(s[k].view(torch.uint8).view(layout.total_elems, -1)[far], clean[k].view(torch.uint8).view(layout.total_elems, -1)[far])


def test_keys_at_multiples_of_8_and_unaligned_arenas():
    import sd_mecha_amd as amd
    layout = arena([5, 8, 13, 700, 1, 64], align=8)
    mask, one = inside(layout), [0.01] * 6
    s = make(layout, torch.bfloat16, torch.float16)
    want = expected(s, layout, 2, one)
    amd.adamw_step(**s, step=2, **HYPER)
    near(s["params"], want[0], want[3], mask)
    s = make(layout, torch.bfloat16, torch.float16)
    off = {}
    for k, t in s.items():                                                          # 2 or 4 bytes off
        if k != "segments":
            off[k] = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].copy_(t)
    amd.adamw_step(**off, segments=s["segments"], step=2, **HYPER)
    near(off["params"], want[0], want[3], mask)
    near(off["exp_avg"], want[1], want[4], mask)
    assert (f64(off["params"])[~mask] == 5.0).all()


def test_many_small_keys():
    """More keys than one look at the segment table (64 offsets) finds, several in one wave's 512 elements."""
    import sd_mecha_amd as amd
    layout = arena([1 + (i * 37) % 300 for i in range(5000)])
    s = make(layout)
    decay = torch.linspace(0, 5.0, 5000, device="cuda")
    p, m, v, ep, em, ev = expected(s, layout, 7, decay.cpu().numpy())
    amd.adamw_step(**s, step=7, weight_decay=decay, **HYPER)
    mask = inside(layout)
    near(s["params"], p, ep, mask)
    near(s["exp_avg_sq"], v, ev, mask)
    assert (f64(s["params"])[~mask] == 5.0).all()


def test_empty_and_zero_arenas():
    import sd_mecha_amd as amd
    z = torch.zeros(0, device="cuda")
    none = torch.zeros(0, 2, dtype=torch.int64, device="cuda")
    assert amd.adamw_step(z, z, z.clone(), z.clone(), none, step=1) is None
    assert float(amd.adamw_step(z, z, z.clone(), z.clone(), none, step=1, max_norm=1.0)) == 0.0
    layout = arena([1000])
    for bits in (32, 8):
        st = amd.adamw_state(layout, "cuda", bits)
        p = torch.zeros(layout.total_elems, device="cuda")
        amd.adamw_step(p, p.clone(), segments=layout.device_segments("cuda"), step=1, max_norm=1.0, **st)
        assert not p.any() and not st["exp_avg"].view(torch.uint8).any()


def test_offsets_past_two_to_the_32():
    """A key behind 2^32 elements of an arena of 8-bit states: offsets, hash and scales take 64 bits."""
    import sd_mecha_amd as amd
    n, at, count = (1 << 32) + 4096, (1 << 32) + 1024, 2000
    seg = torch.tensor([[0, 300], [at, count]], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    grad = torch.empty(n, dtype=torch.bfloat16, device="cuda")
    grad[at:at + count] = torch.randn(count, device="cuda", generator=g).to(torch.bfloat16)
    grad[:300] = 1.0
    st = amd.adamw_state(n, "cuda", 8)
    amd.adamw_step(p, grad, segments=seg, step=4, weight_decay=0.0, seed=5, **st, **HYPER)
    x = f64(grad[at:at + count])
    want = R.adamw(np.zeros(count), x, 0 * x, 0 * x, 4, 1e-3, 0.9, 0.99, 1e-8, 0.0)
    near(p[at:at + count], want[0], want[3], np.ones(count, dtype=bool))
    u = R.dither(2048, 4, 5, at)
    pad = lambda y: np.pad(y, (0, 48))                                              # noqa: E731
    sl, sc = slice(at, at + 2048), slice(at // 128, at // 128 + 16)
    check_codes(st["exp_avg"][sl], st["exp_avg_scales"][sc], pad(want[1]), 8 * R.U, (u & np.uint64(0xFFFF)).astype(np.float64), False, pad(np.ones(count)) > 0)
    assert float(p[0]) != 0.0 and not p[300:4096].any() and not p[at + count:].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_same_steps_in_a_graph_and_on_another_stream(bits):
    """Steps counted on the device: a captured step replayed with eager work in between equals eager steps by number, bit for bit."""
    import sd_mecha_amd as amd
    layout = arena(NUMELS)
    s, e = make(layout, torch.bfloat16, torch.bfloat16, bits), make(layout, torch.bfloat16, torch.bfloat16, bits)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    warm = {k: v.clone() for k, v in s.items()}
    amd.adamw_step(**warm, step=torch.ones(1, dtype=torch.int64, device="cuda"), max_norm=0.1, seed=2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.add_(1)
        norm = amd.adamw_step(**s, step=step, max_norm=0.1, seed=2)
    side = torch.cuda.Stream()
    for t in range(1, 6):
        fresh = torch.randn(layout.total_elems, device="cuda").to(torch.bfloat16) * 1e-3
        s["grads"].copy_(fresh)
        e["grads"].copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            want = amd.adamw_step(**e, step=t, max_norm=0.1, seed=2)
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        for k in s:
            assert torch.equal(s[k].view(torch.uint8), e[k].view(torch.uint8)), (t, k)


def test_cast_product_and_step_together():
    """One layer trained for three steps in 8 bits: the weight's gradient goes from the product into the gradient arena, the step updates the
    arena, the weight is cast again.  Every step against float64 from the state before it."""
    import sd_mecha_amd as amd
    out_f, in_f, tokens = 200, 320, 301
    layout = arena([out_f * in_f, out_f])
    n, seg = layout.total_elems, layout.device_segments("cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    p, grads = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    p[:out_f * in_f].normal_(0, 0.05, generator=g)
    st = amd.adamw_state(layout, "cuda", 8)
    x = torch.randn(tokens, in_f, device="cuda", generator=g).to(torch.bfloat16)
    target = torch.randn(tokens, out_f, device="cuda", generator=g)
    w, dw = p[:out_f * in_f].view(out_f, in_f), grads[:out_f * in_f].view(out_f, in_f)
    xq, xt = amd.cast_blocks(x, sides="both")
    for t in range(1, 4):
        wq = amd.cast_blocks(w, tile=True)
        y = amd.block_product(xq, wq)
        dy = (y - target).to(torch.bfloat16)
        gt = amd.cast_blocks(dy, sides="transposed")
        assert amd.block_product(gt, xt, out=dw) is dw
        want_dw = R.values(gt) @ R.values(xt).T
        assert (np.abs(f64(dw) - want_dw) <= (tokens + 8) * 2.0 ** -23 * (np.abs(R.values(gt)) @ np.abs(R.values(xt)).T)).all()
        grads[layout.offsets[1]:layout.offsets[1] + out_f] = dy.float().sum(0)
        state = dict(params=p.clone(), grads=grads, **{k: v.clone() for k, v in st.items()})
        want = expected(state, layout, t, [0.01, 0.01])
        amd.adamw_step(p, grads, segments=seg, step=t, seed=1, **st, **HYPER)
        near(p, want[0], want[3], inside(layout))
