"""8-bit weights and the AdamW step without a GPU: layouts, refusals in Python and at the C entries."""
import numpy as np
import pytest
import torch

import blocks_reference as R

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def codes(rows, cols):
    return torch.zeros(rows, cols).to(E4M3)


def test_block_scaled_forms_and_layout():
    import sd_mecha_amd as amd
    q = amd.BlockScaled(codes(5, 100), torch.ones(5, 1))
    assert q.pitch == 128 and q.values.stride(0) == 128 and not q.tile and q.shape == (5, 100)
    q = amd.BlockScaled(codes(300, 256), torch.ones(3, 2).to(E8M0))
    assert q.pitch == 256 and q.tile and q.scale_pitch == 2
    whole = codes(4, 384)
    q = amd.BlockScaled(whole[:, 128:256], torch.ones(4, 1))                 # a view that can stay where it is
    assert q.values.data_ptr() == whole[:, 128:].data_ptr() and q.pitch == 384
    q = amd.BlockScaled(whole[:, 300:384], torch.ones(4, 1))                 # not 16-byte aligned
    assert q.pitch == 128 and q.values.data_ptr() != whole[:, 300:].data_ptr()
    short = torch.zeros(3 * 256 + 100, dtype=torch.uint8).view(E4M3).as_strided((4, 100), (256, 1))
    q = amd.BlockScaled(short, torch.ones(4, 1))                             # the last row's block of 128 ends behind the storage
    assert q.values.data_ptr() != short.data_ptr() and q.pitch == 128
    q = amd.BlockScaled(codes(256, 7).t(), torch.ones(7, 2))                 # columns next to each other in memory
    assert q.values.stride() == (256, 1)
    q = amd.BlockScaled(codes(1, 200), torch.ones(1, 2))
    assert not q.tile and q.pitch == 256
    s = torch.ones(2, 6)[:, ::3]
    q = amd.BlockScaled(codes(2, 256), s)
    assert q.scales.stride(1) == 1
    for rows, cols in ((0, 128), (4, 0)):
        assert amd.BlockScaled(codes(rows, cols), torch.ones(rows, R.blocks(cols))).shape == (rows, cols)


def test_laying_out_keeps_the_values():
    import sd_mecha_amd as amd
    g = torch.Generator().manual_seed(0)
    v = torch.randn(9, 131, generator=g).to(E4M3)
    q = amd.BlockScaled(v, torch.rand(9, 2, generator=g))
    assert torch.equal(q.values.view(torch.uint8), v.view(torch.uint8)) and q.pitch == 256


@pytest.mark.parametrize("values, scales, error", [
    (torch.zeros(4, 128), torch.ones(4, 1), TypeError),
    (codes(4, 128), torch.ones(4, 1, dtype=torch.float64), TypeError),
    (codes(4, 128), [1.0], TypeError),
    (codes(4, 128), torch.ones(4), ValueError),
    (codes(4, 128), torch.ones(4, 2), ValueError),
    (codes(300, 128), torch.ones(2, 1), ValueError),
    (codes(4, 128)[0], torch.ones(1, 1), ValueError),
])
def test_block_scaled_refusals(values, scales, error):
    import sd_mecha_amd as amd
    with pytest.raises(error):
        amd.BlockScaled(values, scales)


def test_calls_refuse_the_cpu_and_wrong_kinds():
    import sd_mecha_amd as amd
    q = amd.BlockScaled(codes(4, 128), torch.ones(4, 1))
    with pytest.raises(RuntimeError, match="no CPU path"):
        amd.cast_blocks(torch.zeros(4, 4))
    with pytest.raises(TypeError):
        amd.cast_blocks(torch.zeros(4, 4, dtype=torch.float64))
    with pytest.raises(ValueError):
        amd.cast_blocks(torch.zeros(4, 4), sides="left")
    with pytest.raises(amd.StateDictKeyError):
        amd.cast_blocks({}, key="absent")
    with pytest.raises(RuntimeError, match="no CPU path"):
        amd.uncast_blocks(q)
    with pytest.raises(RuntimeError, match="no CPU path"):
        amd.block_product(q, q)
    with pytest.raises(TypeError):
        amd.block_product(q.values, q)


ADAMW = dict(step=1)


def arenas(n=256, bits=32):
    import sd_mecha_amd as amd
    st = amd.adamw_state(n, "cpu", bits)
    return dict(params=torch.zeros(n), grads=torch.zeros(n), segments=torch.tensor([[0, n]]), step=1, **st)


@pytest.mark.parametrize("change, error", [
    (dict(), RuntimeError),                                                # all in order, but for the CPU
    (dict(params=torch.zeros(256, dtype=torch.float64)), TypeError),
    (dict(grads=torch.zeros(255)), ValueError),
    (dict(exp_avg=torch.zeros(256, dtype=torch.bfloat16)), TypeError),
    (dict(grads=torch.zeros(512)[::2]), ValueError),
    (dict(segments=torch.zeros(1, 2, dtype=torch.int32)), ValueError),
    (dict(segments=torch.zeros(2, dtype=torch.int64)), ValueError),
    (dict(step=0), ValueError),
    (dict(step=torch.tensor([1.0])), ValueError),
    (dict(betas=(0.9, 1.0)), ValueError),
    (dict(lr=-1.0), ValueError),
    (dict(lr=float("nan")), ValueError),
    (dict(weight_decay=torch.zeros(2)), ValueError),
    (dict(max_norm=-1.0), ValueError),
    (dict(max_norm=float("nan")), ValueError),
    (dict(flags=torch.zeros(2, dtype=torch.int32)), ValueError),
    (dict(copy=torch.zeros(255)), ValueError),
    (dict(exp_avg_scales=torch.zeros(2, dtype=torch.uint8).view(E8M0)), TypeError),     # float32 states with a scale
])
def test_adamw_refusals(change, error):
    import sd_mecha_amd as amd
    with pytest.raises(error):
        amd.adamw_step(**{**arenas(), **change})


def test_adamw_8bit_refusals_and_states():
    import sd_mecha_amd as amd
    a = arenas(bits=8)
    assert a["exp_avg"].dtype == E4M3 and a["exp_avg_sq_scales"].numel() == 2
    with pytest.raises(RuntimeError, match="no CPU path"):
        amd.adamw_step(**a)
    with pytest.raises(ValueError):
        amd.adamw_state(130, "cpu", 8)
    with pytest.raises(ValueError):
        amd.adamw_state(128, "cpu", 16)
    with pytest.raises(TypeError):
        amd.adamw_step(**{**a, "exp_avg_sq_scales": None})
    with pytest.raises(ValueError):
        amd.adamw_step(**{**a, "exp_avg_sq_scales": a["exp_avg_sq_scales"][:1]})


def test_c_entries_refuse_before_any_launch():
    """Every one of these returns an error code from the host's checks, with a message; nothing is launched."""
    from sd_mecha_amd import _lib
    L = _lib.lib()
    at = 4096                                                               # an address that is never read

    def packed(of, fields, change):
        return of.pack(*[change.get(n, d) for n, d in fields])

    def matrix(**k):
        return packed(_lib.BLOCK_MATRIX, (("codes", at), ("scales", at), ("rows", 4), ("cols", 100), ("pitch", 128), ("sp", 1), ("tile", 0), ("sdt", 1)), k)

    def cast(q=matrix(), qt=None, a=at, ld=100, dt=_lib.F32):
        return L.mecha_cast_blocks(a, ld, dt, q, qt, None, None)
    for bad in (dict(q=matrix(rows=-1)), dict(dt=7), dict(q=None), dict(ld=99), dict(q=matrix(pitch=100)), dict(q=matrix(pitch=0)), dict(q=matrix(sp=0)),
                dict(q=matrix(scales=0)), dict(q=matrix(codes=at + 8)), dict(a=None), dict(q=matrix(sdt=0)), dict(qt=matrix(rows=100, cols=4, pitch=100)),
                dict(qt=matrix(rows=100, cols=5)), dict(qt=matrix(rows=100, cols=4, tile=1)), dict(qt=matrix())):
        assert cast(**bad) < 0 and L.mecha_last_error(), bad

    def un(q=matrix(), out=at, dt=0):
        return L.mecha_uncast_blocks(q, out, dt, None, None)
    for bad in (dict(q=None), dict(q=matrix(codes=0)), dict(q=matrix(pitch=64)), dict(q=matrix(sdt=5)), dict(dt=9), dict(out=None), dict(q=matrix(cols=-1))):
        assert un(**bad) < 0, bad

    def prod(a=matrix(), b=matrix(), base=None, bdt=0, out=at, odt=0):
        return L.mecha_block_product(a, b, base, bdt, out, odt, 1.0, None, None, 0, None)
    for bad in (dict(a=matrix(rows=-1)), dict(a=matrix(cols=0), b=matrix(cols=0)), dict(a=matrix(cols=99)), dict(odt=3), dict(base=at, bdt=4), dict(a=matrix(sdt=2)),
                dict(a=matrix(sdt=0)), dict(out=None), dict(a=None), dict(b=None), dict(a=matrix(codes=0)), dict(b=matrix(pitch=127)), dict(a=matrix(sp=0)),
                dict(a=matrix(pitch=1 << 25)), dict(b=matrix(codes=at + 4)), dict(a=matrix(rows=1 << 20), b=matrix(rows=1 << 30)), dict(a=matrix(rows=1 << 31))):
        assert prod(**bad) < 0, bad

    room = L.mecha_block_product_workspace_bytes
    assert [room(*x) for x in ((0, 128, 4096, 1, 0, 0), (128, -1, 4096, 1, 0, 0), (1, 1280, 2816, 1, 1, 2), (8192, 10240, 1280, 1, 1, 2), (640, 640, 384, 1, 0, 0))] == [0] * 5
    for x in ((640, 640, 8192, 1, 1, 2), (1280, 1280, 8192, 0, 0, 0), (640, 641, 8192, 1, 0, 0)):
        part = 4 * x[0] * ((x[1] + 7) // 8 * 8)
        assert room(*x) % part == 0 and room(*x) >= 2 * part

    def ad(**k):
        return L.mecha_batched_adamw(packed(_lib.ADAMW, (
            ("p", at), ("g", at), ("m", at), ("v", at), ("ms", 0), ("vs", 0), ("copy", 0), ("segs", at), ("kwd", 0), ("sd", 0), ("clip", 0), ("flags", 0),
            ("total", 256), ("step", 1), ("lr", 1e-3), ("b1", 0.9), ("b2", 0.999), ("eps", 1e-8), ("wd", 0.0), ("n", 1), ("pd", 0), ("gd", 0), ("cd", 0),
            ("bits", 32), ("seed", 0)), k), None)
    for bad in (dict(n=0), dict(segs=0), dict(total=-1), dict(total=1 << 36), dict(pd=5), dict(copy=at, cd=9), dict(bits=16), dict(b1=1.0),
                dict(lr=-1.0), dict(eps=-1.0), dict(step=0), dict(p=0), dict(bits=8), dict(bits=8, ms=at, vs=at, total=130), dict(bits=8, ms=at, vs=at, m=at + 4)):
        assert ad(**bad) < 0, bad
    assert L.mecha_batched_adamw(None, None) < 0
    # results that share memory with what they are made from: the addresses lie apart but for one byte
    q, codes = dict(rows=4, cols=100, pitch=128), 4 * 128
    far = [at * 16 * i for i in range(1, 8)]
    one, two = matrix(**q, codes=far[0], scales=far[1]), matrix(**q, codes=far[2], scales=far[3])
    for out in (far[0] + codes - 1, far[1] + 3, far[2] - 63, far[3] - 63):
        assert prod(a=one, b=two, out=out) < 0 and b"shares memory" in L.mecha_last_error(), out
    for more in (dict(bdt=2), dict(base=far[4] + 4), dict(base=far[4] - 63)):
        assert prod(**{**dict(a=one, b=two, out=far[4], base=far[4]), **more}) < 0 and b"base itself" in L.mecha_last_error(), more
    apart = dict(zip(("p", "g", "m", "v", "copy"), far))
    for x in apart:
        for y in set(apart) - {x}:
            assert ad(**{**apart, x: apart[y] + 4 * 256 - 1}) < 0 and b"share memory" in L.mecha_last_error(), (x, y)
    assert ad(**apart, bits=8, ms=far[5], vs=far[5] + 1) < 0 and b"share memory" in L.mecha_last_error()
    norm = lambda **k: L.mecha_batched_grad_norm(*[k.get(n, d) for n, d in (                                   # noqa: E731
        ("g", at), ("segs", at), ("n", 1), ("total", 256), ("gd", 0), ("max", 1.0), ("out", at), ("ws", at), ("size", 1 << 20), ("stream", None))])
    for bad in (dict(g=None), dict(out=None), dict(max=-1.0), dict(ws=None), dict(size=8), dict(gd=4), dict(n=0)):
        assert norm(**bad) < 0, bad


def test_reference_cast_is_the_nearest_code():
    """The tests' own oracle: torch's conversion to e4m3 and the definition agree."""
    rng = np.random.default_rng(3)
    y = rng.uniform(-448, 448, 4096) * np.exp2(rng.integers(-18, 1, 4096))
    y32 = y.astype(np.float32).astype(np.float64)
    near = np.rint(y32 / R.spacing(y32)) * R.spacing(y32)
    assert np.array_equal(near, torch.from_numpy(y32).float().to(E4M3).double().numpy())


def test_reference_dither_moves_slow_means_on_average():
    """A mean that moves by 1/100 of its codes' distance a step moves in 1/100 of the elements, step after step."""
    n, hits = 1 << 16, []
    for step in range(1, 9):
        u = R.dither(n, step, 7)
        hits.append((np.floor(8.01 + (u & np.uint64(0xFFFF)).astype(np.float64) / 65536) == 9).mean())
        assert abs((u >> np.uint64(16)).astype(np.float64).mean() / 65536 - 0.5) < 5 * (1 / 12) ** 0.5 / n ** 0.5
    # a share of 0.01 of n: standard deviation sqrt(0.01 * 0.99 / n), five of them
    assert all(abs(h - 0.01) < 5 * (0.01 * 0.99 / n) ** 0.5 for h in hits)
