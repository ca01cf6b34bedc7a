"""Training the keys of an arena: one AdamW step for all of them in one launch (csrc/adamw.hip), with optimizer states in 32 or in
8 bits.  Arenas and segment tables are those of arena.py: params, grads and states share one layout.  No counterpart in the
reference, which merges checkpoints and does not train them."""
from __future__ import annotations

from typing import Optional, Union

import torch
from torch.autograd.graph import increment_version

from . import _lib
from ._lib import SCALE_BLOCK
from .arena import ArenaLayout
from .blocks import CODES, _on, _stream
from .merge_methods import _DT


def adamw_state(total_elems: Union[int, ArenaLayout], device, bits: int = 32) -> dict:
    """The states of ``adamw_step`` before the first step, for an arena of ``total_elems`` elements, as its keyword arguments: float32 zeros, or
    (``bits=8``) zero codes and a scale for every 128 elements."""
    n = total_elems.total_elems if isinstance(total_elems, ArenaLayout) else int(total_elems)
    if bits == 32:
        return {name: torch.zeros(n, dtype=torch.float32, device=device) for name in ("exp_avg", "exp_avg_sq")}
    if bits != 8:
        raise ValueError(f"adamw_state: states are held in 32 or 8 bits, got {bits}")
    if n % SCALE_BLOCK:
        raise ValueError(f"adamw_state: an arena with 8-bit states holds a multiple of {SCALE_BLOCK} elements, got {n}")
    state = {name: torch.zeros(n, dtype=torch.uint8, device=device).view(CODES) for name in ("exp_avg", "exp_avg_sq")}
    state.update({f"{name}_scales": torch.zeros(n // SCALE_BLOCK, dtype=torch.uint8, device=device).view(torch.float8_e8m0fnu)
                  for name in ("exp_avg", "exp_avg_sq")})
    return state


def _arena(t, name: str, dtypes, n: int, device) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"adamw_step: {name} is {type(t).__name__}, expected a torch.Tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"adamw_step: {name} is of {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if t.shape != (n,) or t.device != device or not t.is_contiguous():
        raise ValueError(f"adamw_step: {name} must be a flat tensor of {n} elements on {device}, got {tuple(t.shape)} on {t.device}")


_F32_STATE, _CODES, _SCALES = (torch.float32,), (CODES,), (torch.float8_e8m0fnu,)


def adamw_step(params: torch.Tensor, grads: torch.Tensor, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, segments: torch.Tensor, *,
               step: Union[int, torch.Tensor], lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
               weight_decay: Union[float, torch.Tensor] = 0.01, max_norm: Optional[float] = None, copy: Optional[torch.Tensor] = None,
               exp_avg_scales: Optional[torch.Tensor] = None, exp_avg_sq_scales: Optional[torch.Tensor] = None, seed: int = 0,
               flags: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """One AdamW step for every key, in place::

        m = beta1 m + (1 - beta1) g        v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^step) * m / (sqrt(v) / sqrt(1 - beta2^step) + eps)

    in float32, whatever the arenas hold.  ``params``, ``grads``: arenas of float32, float16 or bfloat16; ``segments``: the layout's
    ``device_segments`` table (sorted, at multiples of 8 as every layout's; elements outside it stay as they are).  ``exp_avg``, ``exp_avg_sq``: m and v in float32, or, with
    their ``_scales``, e4m3 codes of m and of sqrt(v) with a power of two for every 128 elements.
    8-bit codes are rounded up or down by a hash of (offset, step, ``seed``), so that slow means move on average.

    ``step`` counts from 1: an int, or an int64 tensor on the device that the kernel reads (for captured graphs).  ``lr``, ``betas``, ``eps`` and ``max_norm``
    are numbers of the host: a captured step keeps the ones it was captured with, so a schedule captures again.  ``weight_decay``: a
    number, or float32 [keys] on the device, one per key.  ``copy``: an arena that receives the new weights in its own dtype.
    ``max_norm``: the gradients of all keys together are scaled down to this 2-norm first, and the norm is returned ([1], on the device);
    if it is not finite, the step sets flags and changes nothing else.  The arenas share no memory.  ``flags``: int32 [keys], per-key flag words (bit 0: a gradient or weight is
    inf / NaN, bit 1: a new weight, as stored, or second moment is: a gradient over 1.8e19 has no square in float32, and its weight only decays from then
    on)."""
    for t, name in ((params, "params"), (segments, "segments")):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"adamw_step: {name} is {type(t).__name__}, expected a torch.Tensor")
    device, n = params.device, params.numel()
    bits8 = exp_avg_scales is not None or exp_avg_sq_scales is not None
    states = _CODES if bits8 else _F32_STATE
    for t, name, dtypes in ((params, "params", _DT), (grads, "grads", _DT), (exp_avg, "exp_avg", states), (exp_avg_sq, "exp_avg_sq", states)):
        _arena(t, name, dtypes, n, device)
    if bits8:
        if n % SCALE_BLOCK:
            raise ValueError(f"adamw_step: an arena with 8-bit states holds a multiple of {SCALE_BLOCK} elements, got {n}")
        for t, name in ((exp_avg_scales, "exp_avg_scales"), (exp_avg_sq_scales, "exp_avg_sq_scales")):
            _arena(t, name, _SCALES, n // SCALE_BLOCK, device)
    if copy is not None:
        _arena(copy, "copy", _DT, n, device)
    if segments.dtype != torch.int64 or segments.dim() != 2 or segments.shape[1] != 2 or segments.device != device or not segments.is_contiguous():
        raise ValueError(f"adamw_step: segments must be the layout's device_segments: contiguous int64 [keys, 2] on {device}")
    keys = segments.shape[0]
    if not (0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0) or not lr >= 0.0 or not eps >= 0.0:
        raise ValueError(f"adamw_step: betas {tuple(betas)} must be in [0, 1), lr {lr} and eps {eps} must not be negative")
    if isinstance(step, torch.Tensor):
        if step.dtype != torch.int64 or step.numel() != 1 or step.device != device:
            raise ValueError(f"adamw_step: step is an int or an int64 tensor of one element on {device}")
    elif step < 1:
        raise ValueError(f"adamw_step: steps count from 1, got {step}")
    per_key = isinstance(weight_decay, torch.Tensor)
    if per_key and (weight_decay.dtype != torch.float32 or tuple(weight_decay.shape) != (keys,) or weight_decay.device != device
                    or not weight_decay.is_contiguous()):
        raise ValueError(f"adamw_step: weight_decay is a number or float32 [{keys}] on {device}")
    if max_norm is not None and not max_norm >= 0.0:
        raise ValueError(f"adamw_step: max_norm must not be negative, got {max_norm}")
    if flags is not None and (not isinstance(flags, torch.Tensor) or flags.dtype != torch.int32 or flags.numel() != keys or flags.device != device or not flags.is_contiguous()):
        raise ValueError(f"adamw_step: flags must be int32 [{keys}] on {device}")
    if not params.is_cuda:
        raise RuntimeError(f"adamw_step: the arenas are on {device}; the MI355X backend has no CPU path")
    if keys == 0 or n == 0:
        return torch.zeros(1, dtype=torch.float32, device=device) if max_norm is not None else None
    L = _lib.lib()
    with _on(device):
        stream, norm = _stream(device), None
        if max_norm is not None:
            size = L.mecha_batched_grad_norm_workspace_bytes(n)
            ws = torch.empty(size, dtype=torch.uint8, device=device)
            norm = torch.empty(2, dtype=torch.float32, device=device)
            _lib.check(L.mecha_batched_grad_norm(grads.data_ptr(), segments.data_ptr(), keys, n, _DT[grads.dtype], float(max_norm), norm.data_ptr(),
                                                 ws.data_ptr(), size, stream), "mecha_batched_grad_norm")
        on_device = isinstance(step, torch.Tensor)
        _lib.check(L.mecha_batched_adamw(_lib.ADAMW.pack(
            params.data_ptr(), grads.data_ptr(), exp_avg.data_ptr(), exp_avg_sq.data_ptr(), exp_avg_scales.data_ptr() if bits8 else 0,
            exp_avg_sq_scales.data_ptr() if bits8 else 0, copy.data_ptr() if copy is not None else 0, segments.data_ptr(),
            weight_decay.data_ptr() if per_key else 0, step.data_ptr() if on_device else 0, norm.data_ptr() if norm is not None else 0,
            flags.data_ptr() if flags is not None else 0, n, 0 if on_device else int(step), lr, betas[0], betas[1], eps,
            0.0 if per_key else weight_decay, keys, _DT[params.dtype], _DT[grads.dtype], _DT[copy.dtype] if copy is not None else _lib.F32,
            8 if bits8 else 32, int(seed) & 0xFFFFFFFF), stream), "mecha_batched_adamw")
    # written in place: a backward pass that saved one of them before raises, as behind torch's own steps
    increment_version([t for t in (params, exp_avg, exp_avg_sq, exp_avg_scales, exp_avg_sq_scales, copy, flags) if t is not None])
    return norm[:1] if norm is not None else None
