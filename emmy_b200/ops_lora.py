"""Low-rank adapters of many requests beside a shared projection, on torch CUDA tensors."""

from __future__ import annotations

import ctypes as C

import torch

from . import lib as L
from .ops import _DTYPE, _need_here, _scratch, _stream

_widths: dict = {}


def _section_array(sections, n):
    """The HOST array of section widths; one per tuple of widths (it holds nothing else)."""
    key = tuple(sections) if sections is not None else (n,)
    array = _widths.get(key)
    if array is None:
        array = _widths[key] = (C.c_int64 * len(key))(*key)
    return array


def lora_workspace(t: int, adapters: int, sections: int, rank: int, device) -> torch.Tensor:
    """Zeroed scratch for calls of up to t rows over `adapters` slots of `sections` x `rank`."""
    return torch.zeros(max(L.load().eq_lora_workspace_bytes(t, adapters, sections, rank), 256), dtype=torch.uint8, device=device)


def lora_status(workspace: torch.Tensor) -> None:
    """Synchronizes the stream; raises EmmyqError(EQ_ERR_TIMEOUT) if a bounded wait of the last call of more than 256 rows on this workspace ran out."""
    _need_here(workspace)
    L.check(L.load().eq_lora_status(workspace.data_ptr(), _stream()))


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, scaling: torch.Tensor, adapter_ids: torch.Tensor, sections=None,
             workspace: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = y[t] + scaling[l] * b[l] @ (a[l] @ x[t]) with l = adapter_ids[t]; rows whose id lies outside [0, L) keep y[t].

    y [T, N] is a linear's output for x [T, K]; a [L, R, K] (or [L, S, R, K] for a projection of S linears side by side whose widths are
    `sections`), b [L, N, R], scaling f32 [L], adapter_ids int32 [T].  `out` may be y (and is refused where it overlaps
    anything else: x, with y = x too).  Above 256 rows the kernels wait for one another, with a limit: `out` holds the result only if
    lora_status(workspace) raises nothing (a loop asks once for many calls, with a workspace of its own for each that it asks about)."""
    _need_here(y, x, a, b, scaling, adapter_ids, out, workspace)
    (t, k), n = x.shape, y.shape[1]
    if a.dim() == 4:
        adapters, s, r, ka = a.shape
    else:
        (adapters, r, ka), s = a.shape, 1
    if ka != k or b.shape != (adapters, n, r) or y.shape != (t, n):
        raise ValueError(f"lora_add: y {tuple(y.shape)}, x {tuple(x.shape)}, a {tuple(a.shape)}, b {tuple(b.shape)} do not fit")
    if scaling.shape != (adapters,) or adapter_ids.shape != (t,) or scaling.dtype is not torch.float32 or adapter_ids.dtype is not torch.int32:
        raise ValueError("lora_add: scaling is f32 with one value per adapter, adapter_ids int32 with one per row")
    dtype = x.dtype
    if not (dtype is y.dtype is a.dtype is b.dtype) or (dtype is not torch.bfloat16 and dtype is not torch.float16):
        raise ValueError(f"lora_add: y, x, a and b share one 16-bit dtype, got {y.dtype}, {x.dtype}, {a.dtype}, {b.dtype}")
    widths = _section_array(sections, n)
    if len(widths) != s:
        raise ValueError(f"lora_add: a holds {s} sections, sections are {sections}")
    if out is None:
        out = torch.empty_like(y)
    elif out.shape != y.shape or out.dtype is not dtype:
        raise ValueError(f"lora_add: out {tuple(out.shape)} {out.dtype} does not fit y {tuple(y.shape)} {dtype}")
    lib = L.load()
    if workspace is None and t > 256:
        workspace = _scratch(lib.eq_lora_workspace_bytes(t, adapters, s, r), x.device)
    status = lib.eq_lora_add(
        y.data_ptr(), x.data_ptr(), a.data_ptr(), b.data_ptr(), scaling.data_ptr(), adapter_ids.data_ptr(), t, k, n, r, adapters, s, widths, _DTYPE[dtype],
        out.data_ptr(), workspace.data_ptr() if workspace is not None else None, workspace.numel() if workspace is not None else 0, _stream(),
    )
    if status:
        L.check(status)
    return out
