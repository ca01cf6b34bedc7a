"""8-bit weights: e4m3 codes with a scale for each block of 128 (``BlockScaled``), made from and turned back into 16- and 32-bit
keys, and the product of two of them.  The kernels are in csrc/blocks.hip; like the merge methods, everything here takes tensors on
a ROCm device, works on the current stream and has no CPU path.  No counterpart in the reference, which holds keys in 16 and
32 bits (streaming.py:395-425)."""
from __future__ import annotations

import ctypes
from contextlib import nullcontext
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._lib import SCALE_BLOCK, SCALE_E8M0, SCALE_F32
from .merge_methods import _DT, _Flags, _resolve, cast

CODES = torch.float8_e4m3fn
_SCALE_DT = {torch.float32: SCALE_F32, torch.float8_e8m0fnu: SCALE_E8M0}
SIDES = ("straight", "transposed", "both")


def _blocks(n: int) -> int:
    return (n + SCALE_BLOCK - 1) // SCALE_BLOCK


def _on(device: torch.device):
    """The device a call's tensors live on, made current for its launches."""
    return nullcontext() if device.index == torch.cuda.current_device() else torch.cuda.device(device)


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


class BlockScaled(NamedTuple("BlockScaled", [("values", torch.Tensor), ("scales", torch.Tensor)])):
    """A matrix in 8 bits: ``values`` float8_e4m3fn [rows, cols], ``scales`` float32 or float8_e8m0fnu (powers of two), either
    [rows, ceil(cols / 128)] -- one for 128 columns of a row -- or [ceil(rows / 128), ceil(cols / 128)] -- one for a 128 x 128
    square.  What a value stands for is ``values.float() * its scale``.

    The kernels read rows in whole blocks of 128 bytes: ``cast_blocks`` lays rows a multiple of 128 bytes apart, with zeros behind the
    last column.  Values that lie otherwise (a stored tensor whose columns are no multiple of 128) are laid out so here, once."""
    __slots__ = ()

    def __new__(cls, values: torch.Tensor, scales: torch.Tensor):
        if not isinstance(values, torch.Tensor) or not isinstance(scales, torch.Tensor):
            raise TypeError("BlockScaled takes two tensors: values and scales")
        if values.dtype != CODES or scales.dtype not in _SCALE_DT:
            raise TypeError(f"BlockScaled: values of {values.dtype} (float8_e4m3fn) and scales of {scales.dtype} (float32, float8_e8m0fnu)")
        if values.dim() != 2 or scales.dim() != 2 or values.device != scales.device:
            raise ValueError(f"BlockScaled: values {tuple(values.shape)} on {values.device} and scales {tuple(scales.shape)} on {scales.device} "
                             "must be matrices on one device")
        rows, cols = values.shape
        if scales.shape[1] != _blocks(cols) or scales.shape[0] not in (rows, _blocks(rows)):
            raise ValueError(f"BlockScaled: values {rows} x {cols} take scales {rows} x {_blocks(cols)} or {_blocks(rows)} x {_blocks(cols)}, "
                             f"got {tuple(scales.shape)}")
        if scales.stride(1) != 1 and scales.shape[1] > 1 or scales.stride(0) < scales.shape[1] and scales.shape[0] > 1:
            scales = scales.contiguous()
        if rows and cols and not cls._laid_out(values):
            whole = torch.zeros((rows, _blocks(cols) * SCALE_BLOCK), dtype=torch.uint8, device=values.device).view(CODES)
            whole[:, :cols] = values
            values = whole[:, :cols]
        return super().__new__(cls, values, scales)

    @staticmethod
    def _laid_out(values: torch.Tensor) -> bool:
        """Rows in place for the kernels, and the last one's block of 128 inside the storage."""
        (rows, cols), (pitch, step) = values.shape, values.stride()
        width = _blocks(cols) * SCALE_BLOCK
        if (step != 1 and cols > 1) or (rows > 1 and (pitch % SCALE_BLOCK or pitch < width)) or values.data_ptr() % 16:
            return False
        return values.storage_offset() + (rows - 1) * pitch + width <= values.untyped_storage().nbytes()

    @property
    def tile(self) -> bool:
        """One scale for a 128 x 128 square (else for 128 columns of a row)."""
        return self.scales.shape[0] != self.values.shape[0]

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def pitch(self) -> int:
        """Bytes from row to row."""
        return self.values.stride(0) if self.values.shape[0] > 1 else _blocks(self.values.shape[1]) * SCALE_BLOCK

    @property
    def scale_pitch(self) -> int:
        return self.scales.stride(0) if self.scales.shape[0] > 1 else self.scales.shape[1]


def _empty(rows: int, cols: int, tile: bool, device) -> BlockScaled:
    codes = torch.empty((rows, _blocks(cols) * SCALE_BLOCK), dtype=CODES, device=device)
    return tuple.__new__(BlockScaled, (codes[:, :cols], torch.empty((_blocks(rows) if tile else rows, _blocks(cols)), dtype=torch.float8_e8m0fnu, device=device)))


def _check_blocks(q, what: str) -> None:
    if not isinstance(q, BlockScaled):
        raise TypeError(f"{what} takes a BlockScaled, got {type(q).__name__}")
    if not q.values.is_cuda:
        raise RuntimeError(f"{what}: the matrix is on {q.values.device}; the MI355X backend has no CPU path")


def cast_blocks(a, *, tile: bool = False, sides: str = "straight", key=None, flags=None, check_finite: bool = True):
    """A float32, float16 or bfloat16 key (``flatten(start_dim=1)``; a 1-D key is one row) in 8 bits with power-of-two scales: the
    smallest 2^e with ``max|x| <= 448 * 2^e`` over the block, codes to nearest even.  ``tile``: a scale for a 128 x 128 square,
    else for 128 columns of a row.  ``sides``: ``"straight"`` the matrix, ``"transposed"`` its transpose (without ``tile`` that has scales of
    its own, for 128 original rows of a column), ``"both"`` the pair of them from one pass over the key.
    Non-finite elements raise ``NonFiniteStateDictKeyError`` (``check_finite``) or set bit 0 of ``flags``, and become NaN codes."""
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
    a = a.unsqueeze(0) if a.dim() == 1 else a.flatten(start_dim=1)
    rows, cols = a.shape
    if (a.stride(1) != 1 and cols > 1) or (a.stride(0) < cols and rows > 1):
        a = a.contiguous()
    device, tile = a.device, bool(tile)
    q = _empty(rows, cols, tile, device) if sides != "transposed" else None
    qt = _empty(cols, rows, tile, device) if sides != "straight" else None
    if rows and cols:
        with _on(device):
            fl = _Flags(device, flags, check_finite)
            _lib.check(_lib.lib().mecha_cast_blocks(
                a.data_ptr(), rows, cols, a.stride(0) if rows > 1 else cols, _DT[a.dtype], tile,
                *((q.values.data_ptr(), q.pitch, q.scales.data_ptr(), q.scale_pitch) if q is not None else (None, 0, None, 0)),
                *((qt.values.data_ptr(), qt.pitch, qt.scales.data_ptr(), qt.scale_pitch) if qt is not None else (None, 0, None, 0)),
                fl.ptr, _stream(device)), "mecha_cast_blocks")
            fl.finish(key)
    return q if qt is None else qt if q is None else (q, qt)


def uncast_blocks(q: BlockScaled, *, key=None, out_dtype=None, flags=None, check_finite: bool = True) -> torch.Tensor:
    """``values * scales`` in float32 as a contiguous matrix of ``out_dtype`` (default float32)."""
    _check_blocks(q, "uncast_blocks")
    device, (rows, cols) = q.values.device, q.shape
    out = torch.empty((rows, cols), dtype=out_dtype or torch.float32, device=device)
    if out.dtype not in _DT:
        raise TypeError(f"uncast_blocks: unsupported out_dtype {out.dtype} (float32, float16, bfloat16)")
    if rows and cols:
        with _on(device):
            fl = _Flags(device, flags, check_finite)
            _lib.check(_lib.lib().mecha_uncast_blocks(q.values.data_ptr(), q.pitch, q.scales.data_ptr(), q.scale_pitch, _SCALE_DT[q.scales.dtype], q.tile,
                                                      rows, cols, out.data_ptr(), _DT[out.dtype], fl.ptr, _stream(device)), "mecha_uncast_blocks")
            fl.finish(key)
    return out


def block_product(a: BlockScaled, b: BlockScaled, base: Optional[torch.Tensor] = None, alpha: float = 1.0, *, out: Optional[torch.Tensor] = None,
                  key=None, out_dtype=None, flags=None, check_finite: bool = True) -> torch.Tensor:
    """``base + alpha * a @ b.T`` (``base=None``: ``alpha * a @ b.T``) of two 8-bit matrices a [m, k], b [n, k], summed in float32 and rounded once to
    ``out_dtype`` (default float32; for 16-bit results the 8-bit matrix instructions first cut the products of 8 neighbouring k off under
    2^-13 of the largest, 1.5e-5 of a typical result) -- add_difference(base, product, alpha).  ``base``: m * n elements; the result has its shape.  ``out``: where
    the result goes (contiguous, m * n elements, of the result's dtype); it may be ``base`` itself.

    A linear layer ``y = x @ w.T`` with w cast with ``tile=True, sides="both"`` to (w, wt), x and the output gradient g cast to (x, xt) and
    (g, gt): y = block_product(x, w), the input's gradient block_product(g, wt), the weight's block_product(gt, xt).
    A NaN result or a non-finite base raises ``NonFiniteStateDictKeyError`` (``check_finite``) or sets bit 0 of ``flags``."""
    _check_blocks(a, "block_product")
    _check_blocks(b, "block_product")
    (m, k), (n, kb), device = a.shape, b.shape, a.values.device
    if k != kb or b.values.device != device:
        raise ValueError(f"block_product: a {m} x {k} on {device} and b {n} x {kb} on {b.values.device} do not go together (a @ b.T)")
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
    if out is None:
        out = torch.empty(shape, dtype=out_dtype or torch.float32, device=device)
    elif out.device != device or out.numel() != m * n or not out.is_contiguous() or (out_dtype is not None and out.dtype != out_dtype):
        raise ValueError(f"block_product: out must be a contiguous tensor of {m} x {n} elements on {device}, of the out_dtype if that is given")
    if out.dtype not in _DT:
        raise TypeError(f"block_product: unsupported result dtype {out.dtype} (float32, float16, bfloat16)")
    if base is not None and out.numel() and out.dtype != base.dtype and out.untyped_storage().data_ptr() == base.untyped_storage().data_ptr():
        raise ValueError("block_product: out may be base only with base's dtype")
    if out.numel() == 0:
        return out
    if k == 0:
        return out.zero_() if base is None else out if out is base else out.copy_(cast(base, out.dtype, key=key, flags=flags, check_finite=check_finite))
    sa, sb = a.scales, b.scales
    if sa.dtype != sb.dtype:
        sa, sb = sa.to(torch.float32), sb.to(torch.float32)
    with _on(device):
        fl = _Flags(device, flags, check_finite)
        _lib.check(_lib.lib().mecha_block_product(
            a.values.data_ptr(), a.pitch, sa.data_ptr(), sa.stride(0) if sa.shape[0] > 1 else sa.shape[1], a.tile,
            b.values.data_ptr(), b.pitch, sb.data_ptr(), sb.stride(0) if sb.shape[0] > 1 else sb.shape[1], b.tile, _SCALE_DT[sa.dtype],
            base.data_ptr() if base is not None else None, out.data_ptr(), m, n, k, _DT[base.dtype] if base is not None else _lib.F32,
            _DT[out.dtype], ctypes.c_float(alpha), fl.ptr, _stream(device)), "mecha_block_product")
        fl.finish(key)
    return out
