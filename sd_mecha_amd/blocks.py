"""8-bit weights: e4m3 codes with a scale for each block of 128 (``BlockScaled``), made from and turned back into 16- and 32-bit
keys, and the product of two of them.  The kernels are in csrc/blocks.hip; like the merge methods, everything here takes tensors on
a ROCm device, works on the current stream and has no CPU path.  No counterpart in the reference, which holds keys in 16 and
32 bits (streaming.py:395-425)."""
from __future__ import annotations

from contextlib import nullcontext
from functools import lru_cache
from operator import attrgetter
from typing import Optional

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import SCALE_BLOCK, SCALE_E8M0, SCALE_F32
from .merge_methods import _DT, _Flags, _resolve

CODES = torch.float8_e4m3fn
_SCALE_DT = {torch.float32: SCALE_F32, torch.float8_e8m0fnu: SCALE_E8M0}
SIDES = ("straight", "transposed", "both")
_pack = _lib.BLOCK_MATRIX.pack


def _blocks(n: int) -> int:
    return (n + SCALE_BLOCK - 1) // SCALE_BLOCK


def _on(device: torch.device):
    """The device a call's tensors live on, made current for its launches."""
    return _HERE if device.index == torch.cuda.current_device() else torch.cuda.device(device)


_HERE = nullcontext()


def _stream(device: torch.device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


class BlockScaled:
    """A matrix in 8 bits: ``values`` float8_e4m3fn [rows, cols], ``scales`` float32 or float8_e8m0fnu (powers of two), either
    [rows, ceil(cols / 128)] -- one for 128 columns of a row -- or [ceil(rows / 128), ceil(cols / 128)] -- one for a 128 x 128
    square (``tile``).  What a value stands for is ``values.float() * its scale``.

    The kernels read rows in whole blocks of 128 bytes: ``cast_blocks`` lays rows a multiple of 128 bytes apart (``pitch``), with zeros
    behind the last column.  Values that lie otherwise (a stored tensor whose columns are no multiple of 128) are laid out so here, once.
    The tensors' elements may change; which tensors they are may not."""
    __slots__ = ("_values", "_scales", "_rows", "_cols", "_tile", "_pitch", "_scale_pitch", "_scale_code", "_packed")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        if not isinstance(values, torch.Tensor) or not isinstance(scales, torch.Tensor):
            raise TypeError("BlockScaled takes two tensors: values and scales")
        code = _SCALE_DT.get(scales.dtype)
        if values.dtype is not CODES or code is None:
            raise TypeError(f"BlockScaled: values of {values.dtype} (float8_e4m3fn) and scales of {scales.dtype} (float32, float8_e8m0fnu)")
        if values.dim() != 2 or scales.dim() != 2 or values.get_device() != scales.get_device():
            raise ValueError(f"BlockScaled: values {tuple(values.shape)} on {values.device} and scales {tuple(scales.shape)} on {scales.device} "
                             "must be matrices on one device")
        (rows, cols), (s_rows, s_cols) = values.shape, scales.shape
        if s_cols != (cols + 127) // 128 or (s_rows != rows and s_rows != (rows + 127) // 128):
            raise ValueError(f"BlockScaled: values {rows} x {cols} take scales {rows} x {_blocks(cols)} or {_blocks(rows)} x {_blocks(cols)}, "
                             f"got {tuple(scales.shape)}")
        s_pitch, s_step = scales.stride()
        if (s_step != 1 and s_cols > 1) or (s_pitch < s_cols and s_rows > 1):
            scales, s_pitch = scales.contiguous(), s_cols
        width = s_cols * SCALE_BLOCK
        pitch, step = values.stride()
        if rows == 1:
            pitch = width
        if rows and cols and ((step != 1 and cols > 1) or pitch % SCALE_BLOCK or pitch < width or values.data_ptr() % 16
                              # the last row's block of 128 has to lie inside the storage
                              or values.storage_offset() + (rows - 1) * pitch + width > values.untyped_storage().nbytes()):
            whole = torch.zeros((rows, width), dtype=torch.uint8, device=values.device).view(CODES)
            whole[:, :cols] = values
            values, pitch = whole[:, :cols], width
        self._set(values, scales, rows, cols, s_rows != rows, pitch, s_pitch if s_rows > 1 else s_cols, code)

    def _set(self, values, scales, rows, cols, tile, pitch, scale_pitch, scale_code):
        self._values, self._scales, self._rows, self._cols = values, scales, rows, cols
        self._tile, self._pitch, self._scale_pitch, self._scale_code = tile, pitch, scale_pitch, scale_code
        self._packed = _pack(values.data_ptr(), scales.data_ptr(), rows, cols, pitch, scale_pitch, tile, scale_code)

    # read-only: the addresses and sizes that the kernels get (_packed) are those of the tensors the matrix was made with
    values, scales = property(attrgetter("_values")), property(attrgetter("_scales"))
    rows, cols, tile = property(attrgetter("_rows")), property(attrgetter("_cols")), property(attrgetter("_tile"))
    pitch, scale_pitch, scale_code = property(attrgetter("_pitch")), property(attrgetter("_scale_pitch")), property(attrgetter("_scale_code"))

    @property
    def shape(self) -> torch.Size:
        return self._values.shape

    def __reduce__(self):                                  # copies and pickles hold the tensors, as bytes: they get addresses of their own
        scales = self._scales if self._scale_code == SCALE_F32 else self._scales.view(torch.uint8)
        return _from_bytes, (self._values.view(torch.uint8), scales)

    def __repr__(self):
        return f"BlockScaled({self._rows} x {self._cols}, {self._scales.dtype} scales {tuple(self._scales.shape)}, {self._values.device})"


def _from_bytes(values: torch.Tensor, scales: torch.Tensor) -> BlockScaled:
    return BlockScaled(values.view(CODES), scales if scales.dtype == torch.float32 else scales.view(torch.float8_e8m0fnu))


def _empty(rows: int, cols: int, tile: bool, device) -> BlockScaled:
    """Room for a cast's codes and scales."""
    s_cols = _blocks(cols)
    width = s_cols * SCALE_BLOCK
    codes = torch.empty((rows, width), dtype=CODES, device=device)
    s_rows = _blocks(rows) if tile else rows
    q = BlockScaled.__new__(BlockScaled)
    q._set(codes if cols == width else codes[:, :cols], torch.empty((s_rows, s_cols), dtype=torch.float8_e8m0fnu, device=device), rows, cols,
           tile, width, s_cols, SCALE_E8M0)
    return q


def _check_blocks(q, what: str) -> None:
    if not isinstance(q, BlockScaled):
        raise TypeError(f"{what} takes a BlockScaled, got {type(q).__name__}")
    if not q._values.is_cuda:
        raise RuntimeError(f"{what}: the matrix is on {q._values.device}; the MI355X backend has no CPU path")


def _flags(device, flags, check_finite: bool):
    """(pointer of the flag word or None, what raises for it)"""
    if flags is None and not check_finite:
        return None, None
    fl = _Flags(device, flags, check_finite)
    return fl.ptr, fl


def cast_blocks(a, *, tile: bool = False, sides: str = "straight", key=None, flags=None, check_finite: bool = True):
    """A float32, float16 or bfloat16 key (``flatten(start_dim=1)``; a 1-D key is one row) in 8 bits with power-of-two scales: the
    smallest 2^e with ``max|x| <= 448 * 2^e`` over the block, codes to nearest even.  ``tile``: a scale for a 128 x 128 square,
    else for 128 columns of a row.  ``sides``: ``"straight"`` the matrix, ``"transposed"`` its transpose (without ``tile`` that has scales of
    its own, for 128 original rows of a column), ``"both"`` the pair of them from one pass over the key.
    Non-finite elements raise ``NonFiniteStateDictKeyError`` (``check_finite``, which waits for the kernel: not in a captured graph) or set bit 0 of
    ``flags``, and become NaN codes."""
    a = _resolve(a, key)
    if sides not in SIDES:
        raise ValueError(f"cast_blocks: sides is one of {SIDES}, got {sides!r}")
    if not isinstance(a, torch.Tensor):
        raise TypeError(f"cast_blocks: got {type(a).__name__}, expected a torch.Tensor")
    if a.dtype not in _DT:
        raise TypeError(f"cast_blocks: unsupported dtype {a.dtype} (float32, float16, bfloat16)")
    if not a.is_cuda:
        raise RuntimeError(f"cast_blocks: the key is on {a.device}; the MI355X backend has no CPU path")
    if a.dim() == 0:
        raise ValueError("cast_blocks: a 0-d key has no block")
    if a.dim() != 2:
        a = a.unsqueeze(0) if a.dim() == 1 else a.flatten(start_dim=1)
    (rows, cols), (stride, step) = a.shape, a.stride()
    if (step != 1 and cols > 1) or stride < cols:
        if rows > 1 or step != 1:
            a = a.contiguous()
        stride = cols
    device, tile = a.device, bool(tile)
    q = _empty(rows, cols, tile, device) if sides != "transposed" else None
    qt = _empty(cols, rows, tile, device) if sides != "straight" else None
    if rows and cols:
        with _on(device):
            word, fl = _flags(device, flags, check_finite)
            _lib.check(_lib.lib().mecha_cast_blocks(a.data_ptr(), stride, _DT[a.dtype], q._packed if q is not None else None,
                                                    qt._packed if qt is not None else None, word, _stream(device)), "mecha_cast_blocks")
            if fl is not None:
                fl.finish(key)
    return q if qt is None else qt if q is None else (q, qt)


def uncast_blocks(q: BlockScaled, *, key=None, out_dtype=None, flags=None, check_finite: bool = True) -> torch.Tensor:
    """``values * scales`` in float32 as a contiguous matrix of ``out_dtype`` (default float32).  NaN codes and scales that are not finite raise
    ``NonFiniteStateDictKeyError`` (``check_finite``) or set bit 0 of ``flags``; a result that its type stores as infinity sets bit 1."""
    _check_blocks(q, "uncast_blocks")
    dtype = out_dtype or torch.float32
    if dtype not in _DT:
        raise TypeError(f"uncast_blocks: unsupported out_dtype {dtype} (float32, float16, bfloat16)")
    device, rows, cols = q._values.device, q._rows, q._cols
    out = torch.empty((rows, cols), dtype=dtype, device=device)
    if rows and cols:
        with _on(device):
            word, fl = _flags(device, flags, check_finite)
            _lib.check(_lib.lib().mecha_uncast_blocks(q._packed, out.data_ptr(), _DT[dtype], word, _stream(device)), "mecha_uncast_blocks")
            if fl is not None:
                fl.finish(key)
    return out


@lru_cache(maxsize=4096)
def _product_workspace(m: int, n: int, k: int, scale_code: int, b_tile: bool, out_code: int) -> int:
    return _lib.lib().mecha_block_product_workspace_bytes(m, n, k, scale_code, b_tile, out_code)


def block_product(a: BlockScaled, b: BlockScaled, base: Optional[torch.Tensor] = None, alpha: float = 1.0, *, out: Optional[torch.Tensor] = None,
                  key=None, out_dtype=None, flags=None, check_finite: bool = True) -> torch.Tensor:
    """``base + alpha * a @ b.T`` (``base=None``: ``alpha * a @ b.T``) of two 8-bit matrices a [m, k], b [n, k], summed in float32 and rounded once to
    ``out_dtype`` (default float32; for 16-bit results the 8-bit matrix instructions first cut the products of 8 neighbouring k off under
    2^-13 of the largest, 1.5e-5 of a typical result: about 1 % of bfloat16 results are the neighbour of the nearest number) -- add_difference(base, product, alpha).  ``base``: m * n elements; the result has its shape.  ``out``: where
    the result goes (contiguous, m * n elements, of the result's dtype); it may be ``base`` itself, and otherwise shares no memory with an input.

    A linear layer ``y = x @ w.T`` with w cast with ``tile=True, sides="both"`` to (w, wt), x and the output gradient g cast to (x, xt) and
    (g, gt): y = block_product(x, w), the input's gradient block_product(g, wt), the weight's block_product(gt, xt).
    A NaN result or a non-finite base raises ``NonFiniteStateDictKeyError`` (``check_finite``) or sets bit 0 of ``flags``; a result that its type
    stores as infinity sets bit 1.  The check waits for the kernel (18 us a call): ``check_finite=False`` in a step that is captured or repeated."""
    _check_blocks(a, "block_product")
    _check_blocks(b, "block_product")
    m, k, n, kb, device = a._rows, a._cols, b._rows, b._cols, a._values.device
    if k != kb or b._values.get_device() != device.index:
        raise ValueError(f"block_product: a {m} x {k} on {device} and b {n} x {kb} on {b._values.device} do not go together (a @ b.T)")
    if isinstance(alpha, torch.Tensor):
        if alpha.numel() != 1:
            raise NotImplementedError("block_product takes a scalar alpha")
        alpha = alpha.item()
    if base is not None:
        if not isinstance(base, torch.Tensor) or base.dtype not in _DT or base.device != device or base.numel() != m * n:
            raise ValueError(f"block_product: base must be a float32, float16 or bfloat16 tensor of {m} x {n} elements on {device}")
        shape = base.shape
        base = base if base.is_contiguous() else base.contiguous()
    else:
        shape = (m, n)
    given = out is not None
    if out is None:
        if out_dtype is not None and out_dtype not in _DT:
            raise TypeError(f"block_product: unsupported out_dtype {out_dtype} (float32, float16, bfloat16)")
        out = torch.empty(shape, dtype=out_dtype or torch.float32, device=device)
    elif not isinstance(out, torch.Tensor) or out.device != device or out.numel() != m * n or not out.is_contiguous() or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"block_product: out must be a contiguous tensor of {m} x {n} elements on {device}, of the out_dtype if that is given")
    if out.dtype not in _DT:
        raise TypeError(f"block_product: unsupported result dtype {out.dtype} (float32, float16, bfloat16)")
    if base is not None and (base.dtype != out.dtype or base.data_ptr() != out.data_ptr()):
        at, to = base.data_ptr(), out.data_ptr()
        if to < at + m * n * base.element_size() and at < to + m * n * out.element_size():
            raise ValueError("block_product: out may be base itself, of the same dtype, but not overlap it otherwise")
    if out.numel() == 0:
        return out
    if k == 0:                                             # an empty sum: one column of zeros
        a, b = (BlockScaled(torch.zeros((rows, 1), dtype=torch.uint8, device=device).view(CODES), torch.ones((rows, 1), device=device)) for rows in (m, n))
        k = 1
    if a._scale_code != b._scale_code:
        a, b = (q if q._scale_code == SCALE_F32 else BlockScaled(q._values, q._scales.to(torch.float32)) for q in (a, b))
    with _on(device):
        word, fl = _flags(device, flags, check_finite)
        # (a base of another type is added by kernels that do not share k out)
        size = _product_workspace(m, n, k, a._scale_code, b._tile, _DT[out.dtype]) if base is None or base.dtype == out.dtype else 0
        room = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        _lib.check(_lib.lib().mecha_block_product(
            a._packed, b._packed, base.data_ptr() if base is not None else None, _DT[base.dtype] if base is not None else _lib.F32, out.data_ptr(),
            _DT[out.dtype], alpha, word, room.data_ptr() if size else None, size, _stream(device)), "mecha_block_product")
        if given:                                         # written in place: a backward pass that saved it before raises
            increment_version(out)
        if fl is not None:
            fl.finish(key)
    return out
