"""8-bit weights and the AdamW step without a GPU: copies, attributes and refusals."""
import copy
import io
import pickle

import pytest
import torch

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def block_scaled(rows, cols, scales=torch.float32, tile=False):
    import sd_mecha_amd as amd
    g = torch.Generator().manual_seed(rows)
    s = torch.rand((rows + 127) // 128 if tile else rows, (cols + 127) // 128, generator=g) + 0.5
    return amd.BlockScaled(torch.randn(rows, cols, generator=g).to(E4M3), s.to(scales))


def addresses(q):
    from sd_mecha_amd import _lib
    return _lib.BLOCK_MATRIX.unpack(q._packed)


@pytest.mark.parametrize("rows, cols, scales, tile", [(4, 128, torch.float32, False), (300, 200, E8M0, True), (5, 77, torch.float32, False), (1, 1, E8M0, False)])
def test_copies_of_a_block_scaled_matrix_have_addresses_of_their_own(rows, cols, scales, tile):
    import sd_mecha_amd as amd
    q = block_scaled(rows, cols, scales, tile)
    file = io.BytesIO()
    torch.save(q, file)
    file.seek(0)
    for c in (copy.deepcopy(q), pickle.loads(pickle.dumps(q)), torch.load(file, weights_only=False), copy.copy(q)):
        assert type(c) is amd.BlockScaled and c.shape == q.shape and c.tile == q.tile and c.scales.dtype == scales
        assert torch.equal(c.values.view(torch.uint8), q.values.view(torch.uint8)) and torch.equal(c.scales.view(torch.uint8), q.scales.view(torch.uint8))
        assert addresses(c) == (c.values.data_ptr(), c.scales.data_ptr(), rows, cols, c.pitch, c.scale_pitch, int(tile), c.scale_code)
        assert c.pitch % 128 == 0 and c.values.stride(0) in (c.pitch, cols)
    assert copy.deepcopy(q).values.data_ptr() != q.values.data_ptr()
    assert addresses(q)[:2] == (q.values.data_ptr(), q.scales.data_ptr())


def test_the_tensors_of_a_block_scaled_matrix_stay():
    """The kernels get the addresses of the tensors that it was made with: others in their place would not be read."""
    q = block_scaled(4, 256)
    for name, value in (("values", q.values.clone()), ("scales", q.scales * 2), ("rows", 8), ("cols", 128), ("tile", True), ("pitch", 512), ("scale_pitch", 1), ("scale_code", 1)):
        with pytest.raises(AttributeError):
            setattr(q, name, value)
    q.scales.mul_(2.0)                                                     # their elements may change
    assert addresses(q)[1] == q.scales.data_ptr()


@pytest.mark.parametrize("flags", [
    torch.zeros(1, dtype=torch.int32),                                     # in host memory, where a kernel's atomic would fault
    torch.zeros(1, dtype=torch.int32, device="meta"),
    torch.zeros(1, dtype=torch.uint8),
    torch.zeros(0, dtype=torch.int32),
    torch.zeros(1),
    [0],
])
def test_flag_words_that_a_kernel_could_not_write_are_refused(flags):
    from sd_mecha_amd.merge_methods import _Flags
    with pytest.raises(ValueError, match="flags must be"):
        _Flags(torch.device("cuda", 0), flags, True)


def test_flag_words_of_one_or_more_keys_are_taken():
    from sd_mecha_amd.merge_methods import _Flags
    for flags in (torch.zeros(1, dtype=torch.int32), torch.zeros(5, dtype=torch.int32)[2:], torch.zeros((), dtype=torch.int32), torch.zeros(3, dtype=torch.uint32)):
        assert _Flags(torch.device("cpu"), flags, True).ptr.value == flags.data_ptr()


def test_adamw_refuses_flags_that_are_no_tensor():
    import sd_mecha_amd as amd
    p = torch.zeros(128)
    with pytest.raises(ValueError, match="flags"):
        amd.adamw_step(p, p.clone(), segments=torch.tensor([[0, 128]]), step=1, flags=[0], **amd.adamw_state(128, "cpu"))


def test_c_entries_refuse_shared_memory_before_any_launch():
    """Host checks only: the addresses lie apart but for a byte or two, and nothing is launched."""
    from sd_mecha_amd import _lib
    L = _lib.lib()
    far = [1 << 32, 2 << 32, 3 << 32, 4 << 32, 5 << 32, 6 << 32, 7 << 32]

    def matrix(codes, scales, rows=100, cols=200, pitch=256, sp=2, tile=0, sdt=1):
        return _lib.BLOCK_MATRIX.pack(codes, scales, rows, cols, pitch, sp, tile, sdt)

    def cast(a=far[0], q=(far[1], far[2]), qt=(far[3], far[4]), ld=200, pitch=256):
        return L.mecha_cast_blocks(a, ld, _lib.F32, matrix(*q, pitch=pitch) if q else None, matrix(*qt, rows=200, cols=100, pitch=pitch, sp=1) if qt else None, None, None)
    codes, key = 99 * 256 + 256, 4 * (99 * 200 + 200)
    for bad in (dict(q=(far[0] + (key - 16), far[2])), dict(q=(far[0] - (codes - 16), far[2]), qt=None), dict(q=(far[1], far[0] + key - 1)), dict(q=(far[1], far[1] + codes - 1), qt=None),
                dict(qt=(far[0] - 16, far[4])), dict(q=None, qt=(far[3], far[3] + 5)), dict(q=None, qt=(far[3], far[0] - 199)),
                dict(qt=(far[1] + codes - 16, far[4])), dict(qt=(far[1] + 128, far[4])), dict(qt=(far[3], far[1])), dict(qt=(far[2] + 192, far[4])), dict(qt=(far[3], far[2] + 199)),
                dict(q=(far[1], far[2]), qt=(far[1] + 128, far[4]), pitch=384), dict(q=(far[1], far[2]), qt=(far[1] + 384, far[4]), pitch=384)):
        assert cast(**bad) < 0 and b"share memory" in L.mecha_last_error(), bad

    def un(out, rows=100, cols=200):
        return L.mecha_uncast_blocks(matrix(far[0], far[1]), out, _lib.F16, None, None)
    for out in (far[0], far[0] + codes - 1, far[0] - 2 * 100 * 200 + 1, far[1] + 199, far[1] - 1):
        assert un(out) < 0 and b"shares memory" in L.mecha_last_error(), out

    m, n, k = 1024, 1280, 5120
    size = L.mecha_block_product_workspace_bytes(m, n, k, 1, 0, _lib.BF16)
    assert size > 0
    a, b = matrix(far[0], far[1], m, k, k, 40), matrix(far[2], far[3], n, k, k, 40)
    for room in (far[0] - 16, far[1] - 16, far[2] + n * k - 16, far[3] + 16, far[4] + 2 * m * n - 16, far[4] - size + 16, far[5] + 2 * m * n - 16):
        assert L.mecha_block_product(a, b, far[5], _lib.BF16, far[4], _lib.BF16, 1.0, None, room, size, None) < 0 and b"workspace shares" in L.mecha_last_error(), room


def test_the_shapes_of_the_product_tests_take_every_kernel():
    """What the GPU tests rest on: if the choice of kernels changes, so do these shapes."""
    from product_shapes import KERNELS, MODES
    from sd_mecha_amd import _lib
    L = _lib.lib()

    def tile(m, n, k, scales, form, bits, other_base=0):
        v = L.mecha_block_product_tile(m, n, k, _lib.SCALE_E8M0 if scales == "e8m0" else _lib.SCALE_F32, int(form == "tile"), _lib.F32 if bits == 32 else _lib.BF16, other_base)
        return v >> 20, v >> 8 & 0xfff, v & 0xff
    seen = [set() for _ in MODES]
    for shape, tiles in KERNELS:
        for i, (mode, want) in enumerate(zip(MODES, tiles)):
            assert tile(*shape, *mode) == want, (shape, mode)
            seen[i].add(want[:2] + (want[2] > 1,))
            size = L.mecha_block_product_workspace_bytes(*shape, _lib.SCALE_E8M0 if mode[0] == "e8m0" else _lib.SCALE_F32, int(mode[1] == "tile"), _lib.F32 if mode[2] == 32 else _lib.BF16)
            assert (size > 0) == (want[2] > 1)
            assert tile(*shape, *mode, 1)[0] <= 128 and tile(*shape, *mode, 1)[2] == 1
    few = {(16, 16, False), (16, 32, False), (32, 32, False), (128, 128, False), (128, 256, False), (128, 256, True)}
    for got, more in zip(seen, ({(32, 64, False), (192, 256, False), (256, 256, False)}, {(32, 64, False), (192, 256, False), (256, 256, False)},
                                {(32, 64, False), (192, 256, False)}, {(32, 64, False)}, set())):
        assert got == few | more
    assert L.mecha_block_product_tile(0, 8, 8, 1, 0, 0, 0) == 0


def test_the_segment_table_of_a_layout_without_keys():
    """Every key frozen or empty: a table of no rows, which a step takes and does nothing with."""
    import sd_mecha_amd as amd
    from sd_mecha_amd.arena import plan_arena
    layout = plan_arena([("a", 0)])
    segments = layout.device_segments("cpu")
    assert segments.shape == (0, 2) and segments.dtype == torch.int64
    p = torch.zeros(layout.total_elems)
    with pytest.raises(RuntimeError, match="no CPU path"):                 # all else is in order
        amd.adamw_step(p, p.clone(), segments=segments, step=1, **amd.adamw_state(layout, "cpu"))
