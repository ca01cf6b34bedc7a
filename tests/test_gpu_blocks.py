"""The 8-bit cast and product on the GPU against float64 (tests/blocks_reference.py).

cast and uncast have one rounding in the definition and are compared bit for bit.  The product: every product of codes is exact in
float32, so what a sum of k of them loses is at most (k + 8) roundings of 2^-23 (a float32 step) of the sum of magnitudes --
the 8 for scales, alpha and base -- and the result's own half step.  Results of 16 bits come from the 8-bit matrix instructions, which
align the products of 8 neighbouring k to the largest of them and cut off what lies under 2^-13 of it: the other 7 lose less than
2^-13 of the largest each, so all groups together less than 7 * 2^-13 of the sum of magnitudes."""
import numpy as np
import pytest
import torch

import blocks_reference as R

pytestmark = pytest.mark.gpu
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
OVER = {t: torch.finfo(t).max * (1 + torch.finfo(t).eps / 4) for t in TYPES}


def key(rows, cols, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a = torch.randn(rows, cols, device="cuda", generator=g) * torch.exp(2 * torch.randn(rows, 1, device="cuda", generator=g)) * 0.05
    return a.to(dtype)


def same_cast(q, a, tile):
    """q against the float64 cast of a, bit for bit, and zeros behind the last column"""
    want, e = R.cast(a.detach().double().cpu().numpy(), tile)
    assert np.array_equal(q.values.float().cpu().double().numpy(), want, equal_nan=True)
    assert np.array_equal(q.scales.view(torch.uint8).cpu().numpy().astype(np.float64) - 127, e)
    rows, cols = q.shape
    behind = torch.as_strided(q.values.view(torch.uint8), (rows, q.pitch), (q.pitch, 1))[:, cols:]
    assert not behind.any()


def matrix(rows, cols, form, scales, seed, ints=False):
    import sd_mecha_amd as amd
    g = torch.Generator(device="cuda").manual_seed(seed)
    v = torch.randint(-8, 9, (rows, cols), device="cuda", generator=g).float() if ints else (torch.randn(rows, cols, device="cuda", generator=g) * 120).clamp_(-448, 448)
    shape = (rows if form == "rows" else R.blocks(rows), R.blocks(cols))
    if scales == "e8m0":
        s = torch.randint(124 if ints else 110, 130 if ints else 140, shape, device="cuda", generator=g, dtype=torch.uint8).view(E8M0)
    else:
        s = torch.randint(1, 4, shape, device="cuda", generator=g).float() if ints else torch.rand(shape, device="cuda", generator=g) * 3 + 0.1
    return amd.BlockScaled(v.to(E4M3), s)


def check_product(got, a, b, base=None, alpha=1.0, extra=8):
    va, vb = torch.from_numpy(R.values(a)).cuda(), torch.from_numpy(R.values(b)).cuda()
    dtype, want, size = got.dtype, va @ vb.t() * alpha, va.abs() @ vb.abs().t() * abs(alpha)
    if base is not None:
        want, size = want + base.double().reshape(want.shape), size + base.double().abs().reshape(want.shape)
    bound = (a.shape[1] + extra) * 2.0 ** -23 * size + (0.0 if dtype == torch.float32 else 7 * 2.0 ** -13 * size)
    bound = bound + (want.abs() + bound) * R.HALF[got.dtype] + R.TINY[got.dtype]
    got = got.double().reshape(want.shape)
    # a magnitude from half a step over the type's largest number on rounds to infinity (float16: 65504 + 16)
    over = got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound >= OVER[dtype])
    off = torch.where(over, 0.0, (got - want).abs())
    assert bool((off <= bound).all()), float((off / bound.clamp(min=1e-300)).max())


# ------------------------------------------------------------------------------------------------------------------ cast
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 128), (3, 77), (77, 768), (128, 128), (129, 257), (200, 320), (5, 4096), (640, 136), (300, 127)])
def test_cast_all_sides(rows, cols, tile, dtype):
    import sd_mecha_amd as amd
    a = key(rows, cols, dtype)
    q = amd.cast_blocks(a, tile=tile)
    same_cast(q, a, tile)
    qt = amd.cast_blocks(a, tile=tile, sides="transposed")
    same_cast(qt, a.t(), tile)
    both = amd.cast_blocks(a, tile=tile, sides="both")
    for x, y in zip((q, qt), both):
        assert torch.equal(x.values.view(torch.uint8), y.values.view(torch.uint8)) and torch.equal(x.scales.view(torch.uint8), y.scales.view(torch.uint8))


@pytest.mark.parametrize("tile", [False, True])
def test_cast_extreme_magnitudes(tile):
    """Blocks of zeros, of subnormals, of the largest floats, exactly at and one step over 448 * 2^e, and ties between codes."""
    import sd_mecha_amd as amd
    rows = [np.zeros(128), np.full(128, 1e-45), np.linspace(-3.4028234663852886e38, 3.4028234663852886e38, 128), np.full(128, 448.0), np.full(128, 448.00003),
            np.concatenate([[448.0], np.arange(127) * 0.5 + 16.5]), np.concatenate([[448.0 * 2.0 ** -100], np.arange(127) * 2.0 ** -112]),
            np.concatenate([[448.0], (np.arange(127) + 0.5) * 2.0 ** -9]), np.full(128, 1.1754943508222875e-38), -np.arange(128.0)]
    a = torch.from_numpy(np.stack(rows)).float().cuda()
    for i in range(len(rows)):                                     # each by itself too: a tile has one scale
        for x in (a[i:i + 1], a[:i + 1]):
            for q, y in zip(amd.cast_blocks(x, tile=tile, sides="both"), (x, x.t())):
                same_cast(q, y, tile)


@pytest.mark.parametrize("tile", [False, True])
def test_cast_non_finite(tile):
    import sd_mecha_amd as amd
    a = key(150, 300, torch.bfloat16)
    a[3, 5], a[140, 290], a[0, 0] = float("inf"), float("nan"), float("-inf")
    with pytest.raises(amd.NonFiniteStateDictKeyError):
        amd.cast_blocks(a, tile=tile)
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, qt = amd.cast_blocks(a, tile=tile, sides="both", flags=flags)
    same_cast(q, a, tile)
    same_cast(qt, a.t(), tile)
    assert int(flags) & 1
    flags.zero_()
    amd.cast_blocks(a[10:100, :256], tile=tile, flags=flags)
    assert int(flags) == 0
    with pytest.raises(amd.NonFiniteStateDictKeyError):
        amd.uncast_blocks(q)
    back = amd.uncast_blocks(q, check_finite=False)
    assert torch.equal(back.isnan(), ~a.isfinite())


def test_cast_strides_and_shapes():
    """Rows apart, columns apart, an offset that is not 16-byte aligned, a broadcast row, convolutions, one-dimensional and empty keys."""
    import sd_mecha_amd as amd
    w = key(300, 400, torch.float16)
    for a in (w[::2], w[:, 3:203], w[7:, 8:264], w.t(), w[:1].expand(40, 400)):
        for tile in (False, True):
            for q, x in zip(amd.cast_blocks(a, tile=tile, sides="both"), (a, a.t())):
                same_cast(q, x, tile)
    conv = key(64, 9 * 32, torch.bfloat16).view(64, 32, 3, 3)
    same_cast(amd.cast_blocks(conv), conv.flatten(1), False)
    same_cast(amd.cast_blocks(w[0]), w[:1], False)
    assert amd.cast_blocks(w[:0]).shape == (0, 400) and amd.cast_blocks(w[:, :0], sides="transposed").shape == (0, 300)
    same_cast(amd.cast_blocks({"k": w}, key="k"), w, False)


# ---------------------------------------------------------------------------------------------------------------- uncast
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("form", ["rows", "tile"])
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 130), (257, 320), (64, 2816)])
def test_uncast(rows, cols, form, scales, dtype):
    import sd_mecha_amd as amd
    q = matrix(rows, cols, form, scales, 5)
    got = amd.uncast_blocks(q, out_dtype=dtype, check_finite=False)
    # a code has 4 significant bits and a scale 24: exact in float64, so float() is the one rounding of the float32 product
    assert torch.equal(got.cpu(), torch.from_numpy(R.values(q)).float().to(dtype))


def test_cast_there_and_back_keeps_codes():
    import sd_mecha_amd as amd
    a = key(500, 640, torch.bfloat16)
    q = amd.cast_blocks(a, tile=True)
    back = amd.uncast_blocks(q, out_dtype=torch.bfloat16)
    # half a step of 4 significant bits, or half of 2^-9 of the scale
    s = torch.from_numpy(np.repeat(np.repeat(q.scales.float().cpu().numpy(), 128, 0)[:500], 128, 1)[:, :640]).cuda()
    assert bool(((back.float() - a.float()).abs() <= torch.maximum(a.float().abs() * 2.0 ** -4, s * 2.0 ** -10)).all())
    again = amd.cast_blocks(back, tile=True)
    assert torch.equal(amd.uncast_blocks(again), back.float())


def test_uncast_extreme_scales():
    """Scale bytes 0 (2^-127, subnormal) and 254, and 255 = NaN."""
    import sd_mecha_amd as amd
    v = torch.tensor([[0.0, 1.0, -448.0, 2.0 ** -9]], device="cuda").to(E4M3).repeat(1, 32)
    for byte in (0, 1, 118, 254):
        s = torch.tensor([[byte]], dtype=torch.uint8, device="cuda").view(E8M0)
        got = amd.uncast_blocks(amd.BlockScaled(v, s), check_finite=False)
        with np.errstate(over="ignore"):
            want = (v.float().cpu().numpy().astype(np.float64) * 2.0 ** (byte - 127)).astype(np.float32)
        assert np.array_equal(got.cpu().numpy(), want)
    s = torch.tensor([[255]], dtype=torch.uint8, device="cuda").view(E8M0)
    with pytest.raises(amd.NonFiniteStateDictKeyError):
        amd.uncast_blocks(amd.BlockScaled(v, s))


# --------------------------------------------------------------------------------------------------------------- product
SIZES = [(1, 1, 1), (1, 640, 320), (2, 1280, 2816), (5, 17, 129), (16, 48, 128), (17, 1280, 1280), (77, 640, 2048), (33, 1000, 777), (128, 128, 128),
         (129, 130, 1), (154, 640, 2048), (200, 333, 1000), (256, 256, 256), (300, 2560, 640), (1000, 1000, 127), (520, 770, 9000), (2100, 300, 384)]


@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_product_whole_numbers_are_exact(m, n, k, scales):
    """Small whole codes with scales of small powers of two or small whole numbers: every partial sum is a float32."""
    import sd_mecha_amd as amd
    for fa, fb in (("rows", "tile"), ("rows", "rows"), ("tile", "rows"), ("tile", "tile")):
        a, b = matrix(m, k, fa, scales, m + 1, ints=True), matrix(n, k, fb, scales, n + 2, ints=True)
        got = amd.block_product(a, b)
        assert torch.equal(got.cpu().double(), torch.from_numpy(R.values(a) @ R.values(b).T)), (fa, fb)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_product(m, n, k, scales, dtype):
    import sd_mecha_amd as amd
    a, b = matrix(m, k, "rows", scales, m + 3), matrix(n, k, "tile", scales, n + 4)
    # magnitudes of a unit, so that float16 holds them
    a = amd.BlockScaled(a.values, (a.scales.float() / 2.0 ** 17).to(a.scales.dtype))
    got = amd.block_product(a, b, out_dtype=dtype)
    check_product(got, a, b)
    base = torch.randn(m, n, device="cuda").to(dtype)
    check_product(amd.block_product(a, b, base, 0.75, out_dtype=dtype), a, b, base, 0.75)
    out = base.clone()
    assert amd.block_product(a, b, out, -2.0, out=out) is out                       # onto itself
    check_product(out, a, b, base, -2.0)


LARGE = [(2100, 2056, 1100), (2049, 2048, 2300), (5000, 4200, 640), (300, 16392, 513), (16500, 264, 4097)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", LARGE)
def test_product_large(m, n, k, scales, dtype):
    """Many tiles, several to a workgroup, ragged in every direction, more blocks of k than scales are held at a time."""
    import sd_mecha_amd as amd
    for fa, fb in (("rows", "tile"), ("tile", "rows")):
        a, b = matrix(m, k, fa, scales, m + 1, ints=True), matrix(n, k, fb, scales, n + 2, ints=True)
        want = torch.from_numpy(R.values(a)).cuda() @ torch.from_numpy(R.values(b)).cuda().t()
        got = amd.block_product(a, b, alpha=2.0 ** -7, out_dtype=dtype)
        assert torch.equal(got, (want * 2.0 ** -7).float().to(dtype)), (fa, fb)
        base = torch.randint(-64, 64, (m, n), device="cuda").to(dtype)
        want = (want + base.double()).float().to(dtype)
        assert torch.equal(amd.block_product(a, b, base, out_dtype=dtype), want), (fa, fb)
        assert torch.equal(amd.block_product(a, b, base, out=base), want), (fa, fb)
    a, b = matrix(m, k, "rows", scales, m + 3), matrix(n, k, "tile", scales, n + 4)
    a = amd.BlockScaled(a.values, (a.scales.float() / 2.0 ** 17).to(a.scales.dtype))
    check_product(amd.block_product(a, b, out_dtype=dtype), a, b)
    v = a.values.clone()
    v.view(torch.uint8)[m - 1, k - 1] = 0x7F
    with pytest.raises(amd.NonFiniteStateDictKeyError):
        amd.block_product(amd.BlockScaled(v, a.scales), b, out_dtype=dtype)


@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", LARGE)
def test_product_large_float32(m, n, k, scales):
    """Partial sums are multiples of 2^-6 (powers of two: 2^-3 on each side; whole scales: of 1) and no larger than the sum S of the products'
    magnitudes: up to 2^24 of those units each is a float32 and the result exact.  Beyond (2049 x 2048: both sides are drawn alike, and the
    diagonal holds squares) each of k additions is off by half a unit of S at most."""
    import sd_mecha_amd as amd

    def same(got, va, vb, alpha=1.0, base=None):
        whole = va @ vb.t() * alpha
        size = va.abs() @ vb.abs().t()
        if base is not None:
            whole = whole + base.double()
        want, exact = whole.float(), size <= 2.0 ** (18 if scales == "e8m0" else 24)
        assert bool(exact.float().mean() > 0.9)
        return torch.equal(got[exact], want[exact]) and bool(((got.double() - whole).abs() <= (k + 2) * 2.0 ** -24 * abs(alpha) * (size + 64))[~exact].all())
    for fa, fb in (("rows", "tile"), ("rows", "rows")):
        a, b = matrix(m, k, fa, scales, m + 1, ints=True), matrix(n, k, fb, scales, n + 2, ints=True)
        va, vb = torch.from_numpy(R.values(a)).cuda(), torch.from_numpy(R.values(b)).cuda()
        assert same(amd.block_product(a, b), va, vb), (fa, fb)
        base = torch.randint(-64, 64, (m, n), device="cuda").float()
        assert same(amd.block_product(a, b, base, -2.0), va, vb, -2.0, base), (fa, fb)
        assert same(amd.block_product(a, b, base, -2.0, out=base.clone()), va, vb, -2.0, base), (fa, fb)
        out = base.clone()
        assert same(amd.block_product(a, b, out, -2.0, out=out), va, vb, -2.0, base), (fa, fb)
    a, b = matrix(m, k, "rows", scales, m + 3), matrix(n, k, "tile", scales, n + 4)
    check_product(amd.block_product(a, b), a, b)


# results of many tiles whose rows are not whole 16-byte pieces, with a base of another type, or of few k
MIDDLE = [(2100, 1003, 700), (2100, 1004, 700), (1300, 2570, 1300), (1500, 1501, 1700), (2100, 1000, 384), (1111, 2040, 200), (9000, 1100, 3), (70000, 200, 1), (5000, 3, 4100), (4000, 1, 8192)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", MIDDLE)
def test_product_middle(m, n, k, scales, dtype):
    import sd_mecha_amd as amd
    a, b = matrix(m, k, "rows", scales, m + 1, ints=True), matrix(n, k, "tile", scales, n + 2, ints=True)
    whole = torch.from_numpy(R.values(a)).cuda() @ torch.from_numpy(R.values(b)).cuda().t()
    assert torch.equal(amd.block_product(a, b, alpha=2.0 ** -7, out_dtype=dtype), (whole * 2.0 ** -7).float().to(dtype))
    base = torch.randint(-64, 64, (m, n), device="cuda")
    want = (whole * 2.0 ** -7 + base.double()).float().to(dtype)
    for base_dt in TYPES:
        assert torch.equal(amd.block_product(a, b, base.to(base_dt), 2.0 ** -7, out_dtype=dtype), want), base_dt
    room = torch.empty(m * n + 1, dtype=dtype, device="cuda")                       # 2 or 4 bytes off
    assert torch.equal(amd.block_product(a, b, base.to(dtype), 2.0 ** -7, out=room[1:]).view(m, n), want)


# few tiles and many blocks of k, whose parts are multiplied apart and joined
PARTS = [(640, 640, 8269), (1024, 1280, 5120), (300, 2560, 8192), (1281, 1288, 4100), (900, 264, 8192), (700, 643, 8269), (1024, 1282, 5120), (5100, 77, 6298)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", PARTS)
def test_product_in_parts(m, n, k, scales, dtype):
    import sd_mecha_amd as amd
    assert amd.blocks._product_workspace(m, n, k, int(scales == "e8m0"), True, 0 if dtype == torch.float32 else 1) >= 2 * 4 * m * n
    for fb in ("tile", "rows"):
        a, b = matrix(m, k, "rows", scales, m + 3), matrix(n, k, fb, scales, n + 4)
        a = amd.BlockScaled(a.values, (a.scales.float() / 2.0 ** 17).to(a.scales.dtype))
        check_product(amd.block_product(a, b, out_dtype=dtype), a, b)
        base = torch.randn(m, n, device="cuda").to(dtype)
        out = base.clone()
        assert amd.block_product(a, b, out, -2.0, out=out) is out
        check_product(out, a, b, base, -2.0)
        room = torch.empty(m * n + 1, dtype=dtype, device="cuda")                   # 2 or 4 bytes off
        check_product(amd.block_product(a, b, base, 0.5, out=room[1:]).view(m, n), a, b, base, 0.5)
    v = a.values.clone()
    v.view(torch.uint8)[m - 1, k - 1] = 0x7F
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = amd.block_product(amd.BlockScaled(v, a.scales), b, out_dtype=dtype, flags=flags, check_finite=False)
    # (float16: many results are over 65504 and infinite)
    assert int(flags) & 1 and bool(got[m - 1].isnan().all()) and not bool(got[:m - 1].isnan().any())
    base[0, n - 1] = float("inf")
    with pytest.raises(amd.NonFiniteStateDictKeyError):
        amd.block_product(a, b, base, out_dtype=dtype)


@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
def test_product_with_too_little_room_for_parts(scales):
    """The C entry with no, a short and the whole workspace: the same sums, in float32's rounding."""
    import sd_mecha_amd as amd
    L, (m, n, k) = amd._lib.lib(), PARTS[1]
    a, b = matrix(m, k, "rows", scales, 1, ints=True), matrix(n, k, "tile", scales, 2, ints=True)
    want = torch.from_numpy(R.values(a) @ R.values(b).T).float().cuda()
    size = L.mecha_block_product_workspace_bytes(m, n, k, a.scale_code, 1, 0)
    room = torch.empty(size, dtype=torch.uint8, device="cuda")
    for at, given in ((None, 0), (room.data_ptr(), size - 1), (room.data_ptr(), size), (room.data_ptr() + 4, size - 4)):
        out = torch.empty(m, n, device="cuda")
        amd._lib.check(L.mecha_block_product(a._packed, b._packed, None, 0, out.data_ptr(), 0, 1.0, None, at, given, torch.cuda.current_stream().cuda_stream), "product")
        assert torch.equal(out, want), given


def test_product_extreme_scales():
    """Powers of two from 2^-127 on one side against large ones on the other."""
    import sd_mecha_amd as amd
    for m, n, k in ((40, 50, 300), (2100, 2056, 1100)):
        for ea, eb in ((0, 220), (3, 250), (20, 235), (127, 1)):
            a, b = matrix(m, k, "rows", "e8m0", 1, ints=True), matrix(n, k, "tile", "e8m0", 2, ints=True)
            a = amd.BlockScaled(a.values, torch.full_like(a.scales.view(torch.uint8), ea).view(E8M0))
            b = amd.BlockScaled(b.values, torch.full_like(b.scales.view(torch.uint8), eb).view(E8M0))
            for dtype in (torch.float32, torch.bfloat16):
                va, vb = torch.from_numpy(a.values.float().cpu().double().numpy()).cuda(), torch.from_numpy(b.values.float().cpu().double().numpy()).cuda()
                want = va @ vb.t() * 2.0 ** (ea + eb - 254)
                assert torch.equal(amd.block_product(a, b, out_dtype=dtype), want.float().to(dtype)), (m, ea, eb, dtype)


def test_product_scales_that_are_not_a_number():
    """A NaN scale of either kind makes its row, and only that, NaN."""
    import sd_mecha_amd as amd
    for m, n, k in ((2, 64, 300), (40, 56, 300), (2100, 2056, 1100)):
        for scales in ("e8m0", "fp32"):
            a, b = matrix(m, k, "rows", scales, 1), matrix(n, k, "tile", scales, 2)
            a.scales.view(torch.uint8 if scales == "e8m0" else torch.int32)[1, -1] = 255 if scales == "e8m0" else 0x7FC00000
            for dtype in (torch.float32, torch.bfloat16):
                got = amd.block_product(a, b, out_dtype=dtype, check_finite=False)
                assert bool(got[1].isnan().all()) and int(got.isnan().sum()) == n, (m, scales, dtype)


def test_product_mixed_scales_base_types_and_shapes():
    import sd_mecha_amd as amd
    a, b = matrix(70, 200, "rows", "e8m0", 1), matrix(90, 200, "tile", "fp32", 2)
    for dt in TYPES:
        base = torch.randn(7, 10, 90, device="cuda").to(dt)
        got = amd.block_product(a, b, base, torch.tensor(0.5), out_dtype=torch.float32)
        assert got.shape == base.shape
        check_product(got, a, b, base, 0.5)
    base = torch.randn(90, 70, device="cuda").t()                                   # not contiguous
    check_product(amd.block_product(a, b, base), a, b, base)
    view = torch.zeros(70 * 90 + 1, device="cuda")[1:]                              # 4-byte aligned only
    check_product(amd.block_product(a, b, out=view), a, b)
    assert amd.block_product(amd.BlockScaled(a.values[:0], a.scales[:0]), b).shape == (0, 90)
    none = amd.BlockScaled(a.values[:, :0], a.scales[:, :0]), amd.BlockScaled(b.values[:, :0], b.scales[:, :0])
    assert not amd.block_product(*none).any()
    assert torch.equal(amd.block_product(*none, base), base)


@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
@pytest.mark.parametrize("m, n, k", [(3, 200, 300), (40, 64, 130), (300, 260, 1000), (700, 700, 129)])
def test_product_ignores_what_lies_behind_the_last_column(m, n, k, scales):
    """Columns cut out of wider matrices: the bytes behind column k are other numbers and NaN codes."""
    import sd_mecha_amd as amd
    a, b = matrix(m, k, "rows", scales, 1), matrix(n, k, "rows", scales, 2)
    want = amd.block_product(a, b)

    def wide(q):
        rows, cols = q.shape
        w = torch.full((rows, q.pitch + 256), 0x7F, dtype=torch.uint8, device="cuda").view(E4M3)
        w[:, 128:128 + cols] = q.values
        got = amd.BlockScaled(w[:, 128:128 + cols], q.scales)
        assert got.values.data_ptr() == w[:, 128:].data_ptr()
        return got
    assert torch.equal(amd.block_product(wide(a), wide(b)), want)


def test_product_flags():
    import sd_mecha_amd as amd
    a, b = matrix(40, 256, "rows", "e8m0", 1), matrix(50, 256, "tile", "e8m0", 2)
    amd.block_product(a, b)
    v = a.values.clone()
    v.view(torch.uint8)[7, 200] = 0x7F
    bad = amd.BlockScaled(v, a.scales)
    with pytest.raises(amd.NonFiniteStateDictKeyError):
        amd.block_product(bad, b)
    got = amd.block_product(bad, b, check_finite=False)
    assert bool(got[7].isnan().all()) and bool(got[torch.arange(40) != 7].isfinite().all())
    base = torch.zeros(40, 50, device="cuda")
    base[0, 0] = float("inf")
    with pytest.raises(amd.NonFiniteStateDictKeyError):
        amd.block_product(a, b, base)
    flags = torch.zeros(1, dtype=torch.int32, device="cuda")
    big = amd.BlockScaled(a.values, (a.scales.float() * 2.0 ** 14).to(E8M0))
    amd.block_product(big, b, out_dtype=torch.float16, flags=flags)                 # over float16's largest: an infinite output
    assert int(flags) in (0, 2)
    flags.zero_()
    amd.block_product(a, b, flags=flags)
    assert int(flags) == 0


def test_product_refusals_on_the_gpu():
    import sd_mecha_amd as amd
    a, b = matrix(40, 256, "rows", "e8m0", 1), matrix(50, 256, "tile", "e8m0", 2)
    with pytest.raises(ValueError):
        amd.block_product(a, matrix(50, 128, "tile", "e8m0", 2))
    with pytest.raises(ValueError):
        amd.block_product(a, b, torch.zeros(40, 51, device="cuda"))
    with pytest.raises(ValueError):
        amd.block_product(a, b, torch.zeros(40, 50))
    with pytest.raises(ValueError):
        amd.block_product(a, b, out=torch.zeros(50, 40, device="cuda").t())
    with pytest.raises(TypeError):
        amd.block_product(a, b, out_dtype=torch.float64)
    with pytest.raises(NotImplementedError):
        amd.block_product(a, b, alpha=torch.ones(2))
    x = torch.zeros(40 * 50, device="cuda")
    with pytest.raises(ValueError):
        amd.block_product(a, b, x.view(torch.bfloat16)[:2000], out=x)
    with pytest.raises(ValueError):
        amd.block_product(a, b, out=[0.0] * 2000)
    with pytest.raises(amd._lib.MechaError, match="shares memory"):
        amd.block_product(a, b, out=torch.as_strided(a.values.view(torch.uint8), (8000,), (1,)).view(torch.float32))


def test_product_flags_count_the_results_elements_only():
    """What the tiles hold behind the last row and column is made from the last ones without their base, and may be infinite where the
    result is not: 2^127 * 3 - 2^127 * 1.5."""
    import sd_mecha_amd as amd
    m, n, k = 2049, 2056, 700
    ones = torch.ones(m, k, device="cuda").to(E4M3), torch.ones(n, k, device="cuda").to(E4M3)
    a = amd.BlockScaled(ones[0], torch.full((m, 6), 2.0 ** 100, device="cuda"))
    b = amd.BlockScaled(ones[1], torch.ones(n, 6, device="cuda"))
    flags, alpha = torch.zeros(1, dtype=torch.int32, device="cuda"), 1.5 * 2.0 ** 28 / 700      # a @ b.T * alpha: 2^127 * 3, over the largest
    base = torch.full((m, n), -1.5 * 2.0 ** 127, device="cuda")
    got = amd.block_product(a, b, base, alpha, flags=flags, check_finite=False)
    assert bool(got.isfinite().all()) and int(flags) == 0


def test_product_outputs_past_two_to_the_31():
    import sd_mecha_amd as amd
    m, n, k = 33000, 66000, 130                                                     # 2.18e9 outputs
    a, b = matrix(m, k, "rows", "e8m0", 1, ints=True), matrix(n, k, "tile", "e8m0", 2, ints=True)
    got = amd.block_product(a, b, out_dtype=torch.bfloat16, check_finite=False)
    va, vb = R.values(a), R.values(b)
    for rows in (slice(0, 3), slice(16000, 16003), slice(m - 3, m)):
        want = torch.from_numpy(va[rows] @ vb.T).to(torch.bfloat16)
        assert torch.equal(got[rows].cpu(), want)


def test_linear_layer_forward_and_backward():
    """y = x w^T and its two gradients, all in 8 bits: against the same casts in float64, and the gradients against differences of the
    float64 product of what the casts stand for."""
    import sd_mecha_amd as amd
    x, w, g = key(301, 320, torch.bfloat16, 1), key(640, 320, torch.float32, 2), key(301, 640, torch.bfloat16, 3)
    (w8, wt8), (x8, xt8), (g8, gt8) = amd.cast_blocks(w, tile=True, sides="both"), amd.cast_blocks(x, sides="both"), amd.cast_blocks(g, sides="both")
    assert np.array_equal(R.values(w8), R.values(wt8).T)
    y, dx, dw = amd.block_product(x8, w8), amd.block_product(g8, wt8), amd.block_product(gt8, xt8)
    check_product(y, x8, w8)
    check_product(dx, g8, wt8)
    check_product(dw, gt8, xt8)
    # the loss sum(g y) is linear in x and in w: a difference of it is exact but for float64's own rounding
    xv, wv, gv, gtv, xtv = R.values(x8), R.values(w8), R.values(g8), R.values(gt8).T, R.values(xt8).T
    rng = np.random.default_rng(0)
    for _ in range(4):
        d = rng.normal(size=xv.shape)
        diff = (gv * ((xv + d) @ wv.T)).sum() - (gv * ((xv - d) @ wv.T)).sum()
        mine = 2 * (dx.double().cpu().numpy() * d).sum()
        assert abs(diff - mine) <= 648 * 2.0 ** -23 * 2 * (np.abs(gv) @ np.abs(wv) * np.abs(d)).sum()
        d = rng.normal(size=wv.shape)
        diff = (gtv * (xtv @ (wv + d).T)).sum() - (gtv * (xtv @ (wv - d).T)).sum()
        mine = 2 * (dw.double().cpu().numpy() * d).sum()
        assert abs(diff - mine) <= 310 * 2.0 ** -23 * 2 * ((np.abs(gtv).T @ np.abs(xtv)) * np.abs(d)).sum()


def test_same_result_every_time_on_any_stream_and_in_a_graph():
    """Cast and product: two streams at once, a captured graph replayed with eager work in between, all bit for bit."""
    import sd_mecha_amd as amd
    x, w = [key(m, 2048, torch.bfloat16, m) for m in (3, 154, 700)], amd.cast_blocks(key(640, 2048, torch.float32, 9), tile=True)

    def call(a):
        return amd.block_product(amd.cast_blocks(a, check_finite=False), w, out_dtype=torch.bfloat16, check_finite=False)
    want = [call(a) for a in x]
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, a in zip(streams, x):
            with torch.cuda.stream(s):
                got.append(call(a))
        torch.cuda.synchronize()
        assert all(torch.equal(g, v) for g, v in zip(got, want))
    static = [a.clone() for a in x]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [call(a) for a in static]
    for i in range(4):
        fresh = [key(a.shape[0], 2048, torch.bfloat16, 100 + i) for a in x]
        for s, f in zip(static, fresh):
            s.copy_(f)
        graph.replay()
        eager = [call(f) for f in fresh]
        torch.cuda.synchronize()
        assert all(torch.equal(o, e) for o, e in zip(outs, eager))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scales", ["e8m0", "fp32"])
def test_large_products_in_a_graph_and_side_by_side(scales, dtype):
    """Results of many tiles, of every kind of kernel, captured together and replayed next to the same products on another stream."""
    import sd_mecha_amd as amd
    pairs = [(matrix(m, k, "rows", scales, m), matrix(n, k, "tile", scales, n)) for m, n, k in ((2100, 2056, 1100), (2100, 1003, 700), (200, 640, 900), (640, 640, 4000))]
    pairs = [(amd.BlockScaled(a.values, (a.scales.float() / 2.0 ** 17).to(a.scales.dtype)), b) for a, b in pairs]

    def call():
        return [amd.block_product(a, b, out_dtype=dtype, check_finite=False) for a, b in pairs]
    want = call()
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        outs = call()
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            eager = call()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) and torch.equal(e, w) for o, e, w in zip(outs, eager, want))
