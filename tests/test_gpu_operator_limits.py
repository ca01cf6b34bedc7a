"""The 8-bit operators and the AdamW step at the ends of the numbers' range: moments that overflow."""
import numpy as np
import pytest
import torch

import blocks_reference as R
from product_shapes import KERNELS

pytestmark = pytest.mark.gpu
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
H = float.fromhex


def raw(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int32 if t.element_size() == 4 else torch.int16)


# ----------------------------------------------------------------------------------------------------------------- AdamW
@pytest.mark.parametrize("value", [1e21, -1e21, float("inf"), float("nan")])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_gradient_without_a_square_stays_with_its_element(bits, value):
    """One gradient whose square is over float32's largest number, or that is no number: every other element of its block of 128 moves, bit for bit,
    as it does with a zero in that place, in this step and in the ones behind it.  A finite one leaves the weight finite, which only
    decays then."""
    import sd_mecha_amd as amd
    n, at, steps = 384, 128 + 17, 4
    seg = torch.tensor([[0, n]], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    p0, grads = torch.randn(n, device="cuda", generator=g) * 0.02, torch.randn(steps, n, device="cuda", generator=g) * 1e-3
    grads[:, at] = 0.0
    runs = []
    for bad in (False, True):
        st, p, flags = amd.adamw_state(n, "cuda", bits), p0.clone(), torch.zeros(1, dtype=torch.int32, device="cuda")
        trace = []
        for t in range(1, steps + 1):
            x = grads[t - 1].clone()
            if bad and t == 1:
                x[at] = value
            amd.adamw_step(p, x, segments=seg, step=t, lr=1e-2, weight_decay=0.1, seed=3, flags=flags, **st)
            trace.append([p.clone()] + [v.clone() for v in st.values()] + [int(flags)])
            flags.zero_()
        runs.append(trace)
    others = torch.arange(n, device="cuda") != at
    for t, (clean, bad) in enumerate(zip(*runs)):
        for x, y in zip(clean[:-1], bad[:-1]):
            same = raw(x) == raw(y)
            assert bool(same[others].all() if same.numel() == n else same.all()), t
        assert clean[-1] == 0
        if np.isfinite(value):
            assert float(bad[0][at]) == float(clean[0][at]) and bad[-1] == 2          # the gradient is finite, its square is not
        else:
            assert bool(bad[0][at].isnan()) and bad[-1] & 2 and bad[-1] & 1
        if bits == 8:
            assert bool(bad[2][at].float().isnan()) and bool(bad[1][at].float().isnan()) == (not np.isfinite(value))
    # and the others do move: weights in every step, roots over the steps
    assert bool((runs[1][0][0] != p0)[others].all()) and all(bool((runs[1][t][0] != runs[1][t - 1][0])[others].all()) for t in range(1, steps))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [256, 253])                              # whole vectors, and a key's last elements
def test_weights_that_their_type_stores_as_infinity_set_the_flag(n, bits):
    """The largest number plus a little less than half a step is stored as the largest number, plus half a step as infinity; in the arena or in the
    copy.  The gradient is zero and the decay, by 2^-12 of the weight, reaches the border from above."""
    import sd_mecha_amd as amd
    total = 256
    seg = torch.tensor([[0, n]], device="cuda")
    for p_dt, copy_dt, start, want in ((torch.float32, torch.float16, 65520.0, 0x7C00), (torch.float32, torch.float16, 65519.99, 0x7BFF), (torch.float32, torch.bfloat16, 3.3961775292304957e38, 0x7F80),
                                       (torch.float32, torch.bfloat16, 3.39617732e38, 0x7F7F), (torch.float32, None, 3.4e38, None), (torch.bfloat16, torch.float16, 65536.0, 0x7C00)):
        p = torch.zeros(total, dtype=p_dt, device="cuda")
        p[n - 1] = start
        copy = torch.zeros(total, dtype=copy_dt, device="cuda") if copy_dt else None
        flags = torch.zeros(1, dtype=torch.int32, device="cuda")
        amd.adamw_step(p, torch.zeros(total, device="cuda"), segments=seg, step=1, lr=1e-3, weight_decay=0.0, copy=copy, flags=flags, **amd.adamw_state(total, "cuda", bits))
        if copy is not None:
            assert (int(copy.view(torch.int16)[n - 1]) & 0xFFFF) == want, (p_dt, start)
        assert int(flags) == (2 if want in (0x7C00, 0x7F80) else 0), (p_dt, copy_dt, start)
    # a float16 arena whose weight a step carries over the border: p - lr * m / (sqrt(v) + eps) = p + lr in the first step
    for lr, over in ((15.0, False), (17.0, True)):
        p, grad = torch.zeros(total, dtype=torch.float16, device="cuda"), torch.zeros(total, device="cuda")
        p[n - 1], grad[n - 1] = 65504.0, -1.0
        flags = torch.zeros(1, dtype=torch.int32, device="cuda")
        amd.adamw_step(p, grad, segments=seg, step=1, lr=lr, weight_decay=0.0, flags=flags, **amd.adamw_state(total, "cuda", bits))
        assert bool(p[n - 1].isinf()) == over and int(flags) == (2 if over else 0), lr


@pytest.mark.parametrize("step", [1, 50])
def test_8bit_states_of_keys_that_share_blocks(step):
    """Keys at multiples of 8: several in a block of 128, one behind the block's first elements, one over three blocks, one of one element."""
    import sd_mecha_amd as amd
    from sd_mecha_amd.arena import ArenaLayout
    from test_gpu_adamw import HYPER, check_codes, expected, inside, make, near
    layout = ArenaLayout(list("abcdefg"), [40, 20, 200, 1, 9, 77, 30], [8, 64, 184, 512, 520, 568, 760], 1024)
    s, mask = make(layout, torch.bfloat16, torch.bfloat16, bits=8), inside(layout)
    s["grads"] *= 64                                                # so that every block's scales change
    decay = torch.linspace(0, 0.3, 7, device="cuda")
    p, m, v, ep, em, ev = expected(s, layout, step, decay.cpu().numpy())
    idle = s["exp_avg_scales"].view(torch.uint8)[7].clone()
    s["exp_avg_scales"].view(torch.uint8)[7] = 3                     # no key reaches into the last block
    amd.adamw_step(**s, step=step, weight_decay=decay, seed=11, **HYPER)
    assert int(s["exp_avg_scales"].view(torch.uint8)[7]) == 3
    s["exp_avg_scales"].view(torch.uint8)[7] = idle
    near(s["params"], p, ep, mask)
    assert bool((s["params"].float().cpu()[~torch.from_numpy(mask)] == 5.0).all())
    u = R.dither(layout.total_elems, step, 11)
    rel = float((em[mask] / np.maximum(np.abs(m[mask]), 1e-30)).mean())
    check_codes(s["exp_avg"], s["exp_avg_scales"], m, rel, (u & np.uint64(0xFFFF)).astype(np.float64), False, mask)
    check_codes(s["exp_avg_sq"], s["exp_avg_sq_scales"], np.sqrt(v), 5 * R.U, (u >> np.uint64(16)).astype(np.float64), True, mask)


# --------------------------------------------------------------------------------------------------------------- uncast
@pytest.mark.parametrize("cols", [128, 125])
def test_uncast_values_that_their_type_stores_as_infinity_set_the_flag(cols):
    import sd_mecha_amd as amd
    for dtype, code, scale, inf in ((torch.float16, 448.0, 146.25, True), (torch.float16, 448.0, 146.24, False), (torch.bfloat16, 256.0, H("0x1.ffp119"), True),
                                    (torch.bfloat16, 256.0, H("0x1.fefffep119"), False), (torch.float32, 256.0, H("0x1.ffp119"), False), (torch.float32, 256.0, 2.0 ** 120, True)):
        v = torch.zeros(3, cols, device="cuda")
        v[2, cols - 1] = code
        flags = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = amd.uncast_blocks(amd.BlockScaled(v.to(E4M3), torch.full((3, 1), scale, device="cuda")), out_dtype=dtype, flags=flags)
        assert bool(got[2, cols - 1].isinf()) == inf and int(flags) == (2 if inf else 0), (dtype, scale)
        assert not got[:2].any()


# -------------------------------------------------------------------------------------------------------------- product
# one shape for each kernel, for flags and scales
WAYS = [(3, 41, 200), (300, 301, 1000), (200, 1000, 2300), (700, 701, 2300), (2100, 2056, 300), (1035, 3665, 2300), (6492, 2312, 700), (7241, 2080, 700), (8097, 2873, 700),
        (1024, 1280, 5120), (900, 261, 8192)]


@pytest.mark.parametrize("based", [False, True])
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", WAYS)
def test_products_that_their_type_stores_as_infinity_set_the_flag(m, n, k, scales, based):
    """One result, in the last row and column: a product of one pair of codes, 1 x 1 x 2^15 (float16) or 2^127, and alpha up to the border."""
    import sd_mecha_amd as amd
    a, b = torch.zeros(m, k, device="cuda"), torch.zeros(n, k, device="cuda")
    a[m - 1, k - 1], b[n - 1, k - 1] = 1.0, 1.0
    kb = R.blocks(k)
    for dtype, e, alphas in ((torch.float16, 15, ((65520 / 32768, True), (65519.99 / 32768, False))), (torch.bfloat16, 120, ((H("0x1.ffp7"), True), (H("0x1.fefffep7"), False))),
                             (torch.float32, 120, ((H("0x1.ffp7"), False), (H("0x1.fffffep7"), False), (2.0 ** 8, True)))):
        s = torch.full((m, kb), 2.0 ** e, device="cuda")
        one = torch.ones(n, kb, device="cuda")
        if scales == "e8m0":
            s, one = s.to(E8M0), one.to(E8M0)
        qa, qb = amd.BlockScaled(a.to(E4M3), s), amd.BlockScaled(b.to(E4M3), one)
        for alpha, inf in alphas:
            flags = torch.zeros(1, dtype=torch.int32, device="cuda")
            base = torch.zeros(m, n, dtype=dtype, device="cuda") if based else None
            got = amd.block_product(qa, qb, base, alpha, out_dtype=dtype, flags=flags)
            assert bool(got[m - 1, n - 1].isinf()) == inf and int(flags) == (2 if inf else 0), (dtype, alpha)
            assert int((got != 0).sum()) == 1
    base = torch.zeros(m, n, dtype=torch.float16, device="cuda")              # a base that is not finite is the input's
    base[m - 1, n - 1] = float("-inf")
    flags.zero_()
    amd.block_product(qa, qb, base, 0.0, out_dtype=torch.float16, flags=flags)
    assert int(flags) == 3


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", WAYS)
def test_product_of_a_block_of_zeros_with_large_scales(m, n, k, scales, dtype):
    """A block whose codes are zeros on one side adds nothing, whatever its scales: 2^100 and 2^100 (their product is over float32's largest), in every
    row and in squares of b.  All the rest whole numbers: the results are those without that block, bit for bit."""
    import sd_mecha_amd as amd
    g = torch.Generator(device="cuda").manual_seed(m)
    va = torch.randint(-4, 5, (m, k), device="cuda", generator=g).float()
    vb = torch.randint(-4, 5, (n, k), device="cuda", generator=g).float()
    kb = R.blocks(k)
    lone = 1 if kb > 1 else 0                                        # a's codes are zeros in this block, b's in the last
    va[:, 128 * lone:128 * lone + 128] = 0
    vb[:, 128 * (kb - 1):] = 0
    want = (va.double() @ vb.double().t() * 2.0 ** -8).float().to(dtype)
    for tile in (False, True):
        sa = torch.ones(m, kb, device="cuda")
        sb = torch.ones(R.blocks(n) if tile else n, kb, device="cuda")
        for s in (sa, sb):
            s[:, lone] = 2.0 ** 100
            s[:, kb - 1] = 2.0 ** 100
        if scales == "e8m0":
            sa, sb = sa.to(E8M0), sb.to(E8M0)
        got = amd.block_product(amd.BlockScaled(va.to(E4M3), sa), amd.BlockScaled(vb.to(E4M3), sb), alpha=2.0 ** -8, out_dtype=dtype)
        assert torch.equal(got, want), tile


@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("m, n, k", WAYS)
def test_product_of_scales_whose_product_is_subnormal(m, n, k, tile):
    """2^-70 and 2^-70 (1 + 2^-10): 2^-140 (1 + 2^-10) is no float32, but every block's sum times the first, and that times the second, is.  A block's
    product and its addition are off by half a unit each of the sum so far, alpha by half of the result."""
    import sd_mecha_amd as amd
    kb = R.blocks(k)
    a = amd.BlockScaled(torch.full((m, k), 448.0, device="cuda").to(E4M3), torch.full((m, kb), 2.0 ** -70, device="cuda"))
    b = amd.BlockScaled(torch.full((n, k), 256.0, device="cuda").to(E4M3), torch.full((R.blocks(n) if tile else n, kb), 2.0 ** -70 * (1 + 2.0 ** -10), device="cuda"))
    want = k * 448.0 * 256.0 * 2.0 ** -140 * (1 + 2.0 ** -10) * 2.0 ** 110
    got = amd.block_product(a, b, alpha=2.0 ** 110).double()
    assert bool(((got - want).abs() <= (2 * kb + 1) * 2.0 ** -24 * want).all())


@pytest.mark.parametrize("m, n, k", WAYS)
def test_product_with_one_scale_of_b_at_the_ends(m, n, k):
    """Scales of b in squares, zero, subnormal and close to the largest, against ones of a that bring the results back to whole numbers."""
    import sd_mecha_amd as amd
    g = torch.Generator(device="cuda").manual_seed(n)
    kb = R.blocks(k)
    va, vb = (torch.randint(-4, 5, (x, k), device="cuda", generator=g).float() for x in (m, n))
    whole = va.double() @ vb.double().t()
    for sa, sb in ((2.0 ** 100, 2.0 ** -108), (2.0 ** -100, 2.0 ** 100), (1.0, 0.0), (2.0 ** 126, 0.0), (-3.0, 2.0 ** -60), (2.0 ** -140, 2.0 ** 100)):
        for dtype in (torch.float32, torch.bfloat16):
            a = amd.BlockScaled(va.to(E4M3), torch.full((m, kb), sa, device="cuda"))
            b = amd.BlockScaled(vb.to(E4M3), torch.full((R.blocks(n), kb), sb, device="cuda"))
            assert torch.equal(amd.block_product(a, b, out_dtype=dtype), (whole * (sa * sb)).float().to(dtype)), (sa, sb, dtype)


def test_product_of_copies_and_pickles():
    """Copies multiply what they hold, also when the original has changed since."""
    import copy
    import pickle
    import sd_mecha_amd as amd
    g = torch.Generator(device="cuda").manual_seed(0)
    for scales in (torch.float32, E8M0):
        a = amd.BlockScaled(torch.randn(40, 200, device="cuda", generator=g).to(E4M3), torch.full((40, 2), 0.5, device="cuda").to(scales))
        b = amd.cast_blocks(torch.randn(50, 200, device="cuda", generator=g), tile=True)
        want = amd.block_product(a, b)
        copies = [copy.deepcopy((a, b)), pickle.loads(pickle.dumps((a, b)))]
        a.values.view(torch.uint8).zero_()
        assert not amd.block_product(a, b).any()
        for x, y in copies:
            assert x.scales.dtype == scales and torch.equal(amd.block_product(x, y), want)


def test_product_over_no_columns_is_the_base():
    """k = 0: the base, checked, flagged and written like that of any other product."""
    import sd_mecha_amd as amd
    m, n = 6, 40
    a = amd.BlockScaled(torch.zeros(m, 0, device="cuda").to(E4M3), torch.ones(m, 0, device="cuda"))
    b = amd.BlockScaled(torch.zeros(n, 0, device="cuda").to(E4M3), torch.ones(n, 0, device="cuda"))
    base = torch.randn(m, n, device="cuda")
    for dtype in TYPES:
        assert torch.equal(amd.block_product(a, b, base, 3.0, out_dtype=dtype), base.to(dtype))
        out = torch.empty(m * n, dtype=dtype, device="cuda")                   # of another shape than the base's
        assert amd.block_product(a, b, base, out=out) is out and torch.equal(out.view(m, n), base.to(dtype))
        assert not amd.block_product(a, b, out_dtype=dtype).any()
    out = base.clone()
    assert amd.block_product(a, b, out, out=out) is out and torch.equal(out, base)
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    base[m - 1, n - 1] = 65520.0
    assert bool(amd.block_product(a, b, base, out_dtype=torch.float16, flags=flags)[m - 1, n - 1].isinf()) and int(flags) == 2
    base[0, 0] = float("inf")
    for out in (None, base, base.clone()):
        with pytest.raises(amd.NonFiniteStateDictKeyError):
            amd.block_product(a, b, base, out=out)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_between_forward_and_backward_is_noticed(bits):
    """What a backward pass saved is written in place: it raises, as behind torch's own in-place operations, and makes no gradient of other weights."""
    import sd_mecha_amd as amd
    n = 256
    seg, x = torch.tensor([[0, n]], device="cuda"), torch.randn(n, device="cuda", requires_grad=True)
    st = amd.adamw_state(n, "cuda", bits)
    p, copy = torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
    w = p[:128].view(8, 16)                                          # a key's view of the arena
    for saved in (p, copy, w):
        loss = (x[:saved.numel()].view_as(saved) * saved).sum()
        amd.adamw_step(p, torch.ones(n, device="cuda"), segments=seg, step=1, copy=copy, **st)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    before = [t._version for t in st.values()]
    amd.adamw_step(p, torch.ones(n, device="cuda"), segments=seg, step=2, **st)
    assert all(t._version > v for t, v in zip(st.values(), before))
    (x * p).sum().backward()
    assert torch.equal(x.grad, p)


def test_a_product_into_a_saved_tensor_is_noticed():
    import sd_mecha_amd as amd
    a, b = amd.cast_blocks(torch.randn(8, 128, device="cuda")), amd.cast_blocks(torch.randn(16, 128, device="cuda"))
    x, out = torch.randn(8, 16, device="cuda", requires_grad=True), torch.randn(8, 16, device="cuda")
    loss = (x * out).sum()
    amd.block_product(a, b, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        amd.block_product(a, b, out=torch.empty(8, 16, device="cuda"))


@pytest.mark.parametrize("tile", [False, True])
def test_cast_into_two_matrices_side_by_side(tile):
    """Straight and transposed codes in the rows of one buffer, through the C entry: the bytes of one lie between those of the other."""
    import sd_mecha_amd as amd
    from sd_mecha_amd import _lib
    n = 200
    a = torch.randn(n, n, device="cuda")
    want = amd.cast_blocks(a, tile=tile, sides="both")
    room, scales = torch.full((n, 512), 0x55, dtype=torch.uint8, device="cuda"), [torch.zeros_like(q.scales.view(torch.uint8)) for q in want]
    packed = [_lib.BLOCK_MATRIX.pack(room.data_ptr() + 256 * i, s.data_ptr(), n, n, 512, s.shape[1], tile, _lib.SCALE_E8M0) for i, s in enumerate(scales)]
    _lib.check(_lib.lib().mecha_cast_blocks(a.data_ptr(), n, _lib.F32, packed[0], packed[1], None, torch.cuda.current_stream().cuda_stream), "mecha_cast_blocks")
    for i, (q, s) in enumerate(zip(want, scales)):
        assert torch.equal(room[:, 256 * i:256 * i + n], q.values.view(torch.uint8)) and not room[:, 256 * i + n:256 * i + 256].any() and torch.equal(s, q.scales.view(torch.uint8))


def test_product_with_a_base_of_another_type_takes_no_room_for_parts():
    import sd_mecha_amd as amd
    m, n, k = 1024, 1280, 5120
    a, b = amd.cast_blocks(torch.randn(m, k, device="cuda")), amd.cast_blocks(torch.randn(n, k, device="cuda"), tile=True)
    assert amd.blocks._product_workspace(m, n, k, 1, True, 2) > 0
    base = torch.randn(m, n, device="cuda")

    def extra():
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        amd.block_product(a, b, base, out_dtype=torch.bfloat16, check_finite=False)
        return torch.cuda.max_memory_allocated() - before
    assert extra() == 2 * m * n


# ------------------------------------------------------------------------------------------ every kernel, bit for bit
def whole(rows, cols, form, scales, seed):
    """Codes -4 .. 4 and scales 2^-1 .. 2^1 or 1 .. 3, and what they stand for in float64, on the GPU."""
    import sd_mecha_amd as amd
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randint(-4, 5, (rows, cols), device="cuda", generator=g).float()
    shape = (rows if form == "rows" else R.blocks(rows), R.blocks(cols))
    s = torch.randint(1, 4, shape, device="cuda", generator=g).float()
    if scales == "e8m0":
        s = torch.exp2(s - 2).to(E8M0)
    r, c = torch.arange(rows, device="cuda"), torch.arange(cols, device="cuda") // 128
    return amd.BlockScaled(v.to(E4M3), s), v.double() * s.float().double()[r if form == "rows" else r // 128][:, c]


@pytest.mark.parametrize("fa, fb", [("rows", "tile"), ("rows", "rows"), ("tile", "rows"), ("tile", "tile")])
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", [shape for shape, _ in KERNELS])
def test_every_product_kernel_bit_for_bit(m, n, k, scales, fa, fb):
    """Sums are multiples of 2^-2 and at most 64 k < 2^20 (powers of two), or of 1 and at most 144 k < 2^21 (whole scales): every partial sum is a float32
    in any order, and so is 2^-7 of it with a whole base; products of codes up to 4 lie within 2^-13 of the largest.  So each result is the float64
    one, rounded once."""
    import sd_mecha_amd as amd
    (a, va), (b, vb) = whole(m, k, fa, scales, m), whole(n, k, fb, scales, n + 1)
    want = va @ vb.t() * 2.0 ** -7
    base = torch.randint(-64, 65, (m, n), device="cuda")
    onto = want + base.double()
    for dtype in TYPES:
        assert torch.equal(amd.block_product(a, b, alpha=2.0 ** -7, out_dtype=dtype), want.float().to(dtype)), dtype
        bd, w = base.to(dtype), onto.float().to(dtype)
        assert torch.equal(amd.block_product(a, b, bd, 2.0 ** -7, out_dtype=dtype), w), dtype
        room = torch.full((m * n + 9,), 7.0, dtype=dtype, device="cuda")            # one element off, between others
        assert torch.equal(amd.block_product(a, b, bd, 2.0 ** -7, out=room[1:m * n + 1]).view(m, n), w), dtype
        assert float(room[0]) == 7.0 and bool((room[m * n + 1:] == 7.0).all())
        assert torch.equal(amd.block_product(a, b, bd, 2.0 ** -7, out=bd), w), dtype
        other = base.to(torch.float32 if dtype != torch.float32 else torch.bfloat16)
        assert torch.equal(amd.block_product(a, b, other, 2.0 ** -7, out_dtype=dtype), w), dtype
    v = a.values.clone()                                                            # a NaN code in the last row's last column
    v.view(torch.uint8)[m - 1, k - 1] = 0x7F
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = amd.block_product(amd.BlockScaled(v, a.scales), b, alpha=2.0 ** -7, out_dtype=torch.bfloat16, flags=flags)
    assert int(flags) == 3 and bool(got[m - 1].isnan().all()) and torch.equal(got[:m - 1], want[:m - 1].float().to(torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", [(100, 300, 2300), (700, 701, 2300), (1035, 3672, 8500), (6492, 2312, 700), (8097, 2880, 700), (1024, 1280, 5120)])
def test_what_the_8bit_instructions_lose(m, n, k, scales, dtype):
    """1.5e-5 of a result (2-norm, normal codes) in front of the rounding to 16 bits: the first result as a base, negative, leaves what its rounding took off,
    which its own rounding (half a step of half a step) hides nothing of.  A third more would be another instruction."""
    import sd_mecha_amd as amd
    from test_gpu_blocks import matrix
    a, b = matrix(m, k, "rows", scales, 1), matrix(n, k, "tile", scales, 2)
    r, c = torch.arange(n, device="cuda") // 128, torch.arange(k, device="cuda") // 128
    want = (a.values.double() * a.scales.double()[:, c]) @ (b.values.double() * b.scales.double()[r][:, c]).t()
    alpha = float(2.0 ** -torch.log2(want.abs().max()).ceil())                    # (within float16's range)
    first = amd.block_product(a, b, alpha=alpha, out_dtype=dtype)
    rest = amd.block_product(a, b, -first, alpha, out_dtype=dtype)
    off = float((first.double() + rest.double() - want * alpha).norm() / (want * alpha).norm())
    assert off < 2e-5, off


# ------------------------------------------------------------------------------------------------------------------ cast
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_cast_16bit_magnitudes_at_the_ends(dtype, tile):
    """Every pattern of the type that is finite, subnormal ones among them: blocks of neighbours, blocks of the smallest, and each next to a large one."""
    import sd_mecha_amd as amd
    from test_gpu_blocks import same_cast
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    bits = bits[bits.isfinite()]
    least = 2.0 ** -24 if dtype == torch.float16 else 2.0 ** -133
    near = bits[:bits.numel() // 128 * 128].view(-1, 128)                           # neighbours in size
    mixed = near.t().contiguous().view(-1, 128)                                     # all sizes in a block
    small = (torch.arange(128 * 128).view(128, 128).double() * least).to(dtype)     # subnormal, and the first normal ones
    for a in (near, mixed, small, small[:1], small[:3, :5], -small):
        for x in (a.cuda(), a.cuda().t().contiguous()):
            for q, y in zip(amd.cast_blocks(x, tile=tile, sides="both"), (x, x.t())):
                same_cast(q, y, tile)


@pytest.mark.parametrize("form", ["tile", "rows"])
@pytest.mark.parametrize("m, n, k", WAYS)
def test_every_product_kernel_with_powers_of_two_at_the_ends(m, n, k, form):
    """2^-127 and 2^-124 of a against large ones of b, bit for bit; and a NaN scale on either side makes its rows or columns, and only those, NaN."""
    import sd_mecha_amd as amd
    g = torch.Generator(device="cuda").manual_seed(k)
    kb = R.blocks(k)
    va, vb = (torch.randint(-4, 5, (x, k), device="cuda", generator=g).float() for x in (m, n))
    exact = va.double() @ vb.double().t()

    def matrix(v, byte, rows):
        return amd.BlockScaled(v.to(E4M3), torch.full((rows, kb), byte, dtype=torch.uint8, device="cuda").view(E8M0))
    rows_b = n if form == "rows" else R.blocks(n)
    for ea, eb in ((0, 220), (3, 250), (240, 14), (127, 1)):
        for dtype in (torch.float32, torch.bfloat16):
            got = amd.block_product(matrix(va, ea, m), matrix(vb, eb, rows_b), out_dtype=dtype)
            assert torch.equal(got, (exact * 2.0 ** (ea + eb - 254)).float().to(dtype)), (ea, eb, dtype)
    a, b = matrix(va, 127, m), matrix(vb, 127, rows_b)
    a.scales.view(torch.uint8)[m // 2, kb - 1] = 255
    b.scales.view(torch.uint8)[rows_b - 1, 0] = 255
    last = slice(n - 1, n) if form == "rows" else slice((rows_b - 1) * 128, n)
    for scales in ("e8m0", "fp32"):
        if scales == "fp32":
            a, b = (amd.BlockScaled(q.values, q.scales.float()) for q in (a, b))
        for dtype in (torch.float32, torch.float16):
            want = exact.float().clone()
            want[m // 2], want[:, last] = float("nan"), float("nan")
            got = amd.block_product(a, b, alpha=2.0 ** -8, out_dtype=dtype, check_finite=False)
            assert torch.equal(got.nan_to_num(7.0), (want * 2.0 ** -8).to(dtype).nan_to_num(7.0)), (scales, dtype)


def test_a_layer_trained_as_the_readme_shows():
    """The calls of README.md: a layer, its gradients, the weight's straight into the gradient arena, and the step; captured and replayed as they stand."""
    import sd_mecha_amd as amd
    from sd_mecha_amd.arena import plan_arena
    out_f, in_f, tokens = 640, 320, 77
    layout = plan_arena([("w", out_f * in_f), ("b", out_f)])
    segments = layout.device_segments("cuda")
    gen = torch.Generator(device="cuda").manual_seed(1)
    x, g = torch.randn(tokens, in_f, device="cuda", generator=gen).bfloat16(), torch.randn(tokens, out_f, device="cuda", generator=gen).bfloat16()
    start = torch.randn(layout.total_elems, device="cuda", generator=gen) * 0.02

    def program():
        params, grads, t = start.clone(), torch.zeros_like(start), torch.zeros(1, dtype=torch.int64, device="cuda")
        w, w_grad = params[:out_f * in_f].view(out_f, in_f), grads[:out_f * in_f].view(out_f, in_f)
        state = amd.adamw_state(layout, "cuda", bits=8)

        def step():
            t.add_(1)
            w8, wt8 = amd.cast_blocks(w, tile=True, sides="both", check_finite=False)
            (x8, xt8), (g8, gt8) = amd.cast_blocks(x, sides="both", check_finite=False), amd.cast_blocks(g, sides="both", check_finite=False)
            y = amd.block_product(x8, w8, out_dtype=torch.bfloat16, check_finite=False)
            dx = amd.block_product(g8, wt8, out_dtype=torch.bfloat16, check_finite=False)
            amd.block_product(gt8, xt8, out=w_grad, check_finite=False)
            norm = amd.adamw_step(params, grads, **state, segments=segments, step=t, lr=1e-4, max_norm=1.0)
            return [y, dx, norm, params, grads, *state.values()]
        return step
    eager, captured = program(), program()
    captured()                                                     # (the first step warms up)
    graph, first = torch.cuda.CUDAGraph(), eager()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = captured()
    for _ in range(4):
        want = [v.clone() for v in eager()]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o.view(-1).view(torch.uint8), v.view(-1).view(torch.uint8)) for o, v in zip(outs, want))
    assert bool((first[3] != start)[:out_f * in_f].any())
