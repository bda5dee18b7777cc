"""8-bit (E4M3) matrix products with FP32 scales for blocks of 128, and the quantisers that make
their operands.

* :func:`quantize_rows`: activations, one scale for 128 consecutive values of a row;
* :func:`quantize_tiles`: weights, one scale for a 128 x 128 tile (of one matrix, or of each of a
  stack);
* :func:`matmul_blockscaled`: ``y = (a * a_scales) @ (b * b_scales).T`` on the tensor cores' 8-bit path,
  every block's sum scaled and added in FP32; with ``group_ends``, over rows grouped by expert as
  :func:`heliostune_b200.grouped.grouped_matmul`.

A block's scale is ``amax / 448`` and its values are ``e4m3(x * (448 / amax))`` with
``amax = max(max |x|, 2**-100)``, quotients and product rounded to FP32, values to nearest even. An
infinity or a NaN makes its block's scale infinite or NaN, and with it every sum it enters.

The heliostune reference has no counterpart (its products are FP16). None of these has a gradient.
"""

from __future__ import annotations

import torch

from heliostune_b200 import _native
from heliostune_b200.grouped import _DTYPES, MAX_GROUPS, _check_ends, _readable, _row_stride, _workspace
from heliostune_b200.kernel import _device_guard, _stream

#: Values that share a scale along a row (and, for tiles, along a column).
BLOCK = 128


def _blocks(extent: int) -> int:
    return -(-extent // BLOCK)


def _refuse_gradient(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradient; detach its inputs or run it under torch.no_grad()")


def _quantize(x: torch.Tensor, tiles: bool) -> tuple[torch.Tensor, torch.Tensor]:
    what = "quantize_tiles" if tiles else "quantize_rows"
    if x.device.type != "cuda":
        raise ValueError(f"{what} expects a CUDA tensor")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what} serves torch.float16 or torch.bfloat16, got {x.dtype}")
    _refuse_gradient(what, x)
    batch = x.shape[:-2]
    rows, cols = int(x.shape[-2]), int(x.shape[-1])
    # Rows of q start on 16 bytes, so that the products read them in place.
    width = -(-cols // 16) * 16
    q = torch.empty((*batch, rows, width), device=x.device, dtype=torch.float8_e4m3fn)[..., :cols]
    if tiles:
        scales = torch.empty((*batch, _blocks(rows), _blocks(cols)), device=x.device, dtype=torch.float32)
    else:
        # Stored [blocks, rows]: the products read one block's scales of neighbouring rows together.
        scales = torch.empty((_blocks(cols), rows), device=x.device, dtype=torch.float32).T
    count = int(batch[0]) if batch else 1
    lead = (x.stride(0), q.stride(0), scales.stride(0)) if batch else (0, 0, 0)
    with _device_guard(x.device):
        _native.check(
            _native.library().hst_quantize_e4m3(
                _DTYPES[x.dtype], int(tiles), x.data_ptr(), lead[0], x.stride(-2), x.stride(-1), q.data_ptr(), lead[1],
                q.stride(-2), scales.data_ptr(), lead[2], scales.stride(-2), scales.stride(-1), count, rows, cols,
                _stream(x.device),
            )
        )  # fmt: skip
    return q, scales


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scales)`` of ``x [T, K]`` (FP16 or BF16, any strides): ``q [T, K]`` in ``torch.float8_e4m3fn``
    and FP32 ``scales [T, ceil(K / 128)]``, one for each 128 consecutive values of a row. The scales are
    the transposed view of ``[blocks, T]`` storage."""
    if x.ndim != 2:
        raise ValueError("quantize_rows expects x [T, K]")
    return _quantize(x, False)


def quantize_tiles(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scales)`` of ``weight [N, K]`` or ``[E, N, K]`` (FP16 or BF16, any strides): ``q`` of its shape
    in ``torch.float8_e4m3fn`` and FP32 ``scales [..., ceil(N / 128), ceil(K / 128)]``, one for each
    128 x 128 tile."""
    if weight.ndim not in (2, 3):
        raise ValueError("quantize_tiles expects weight [N, K] or [E, N, K]")
    return _quantize(weight, True)


def _check_scales(name: str, scales: torch.Tensor, shape: tuple[int, ...], device: torch.device) -> None:
    if tuple(scales.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(scales.shape)}")
    if scales.dtype != torch.float32:
        raise ValueError(f"{name} must have dtype torch.float32")
    if scales.device != device:
        raise ValueError(f"{name} must be on the device of the operands")


def matmul_blockscaled(
    a: torch.Tensor,
    a_scales: torch.Tensor,
    b: torch.Tensor,
    b_scales: torch.Tensor,
    group_ends: torch.Tensor | None = None,
    *,
    out_dtype: torch.dtype = torch.bfloat16,
) -> torch.Tensor:
    """``y[t, n] = sum_c a_scales[t, c] * b_scales[n // 128, c] * sum_{k in block c} a[t, k] * b[n, k]``.

    ``a [T, K]`` and ``b [N, K]`` are ``torch.float8_e4m3fn``, ``a_scales [T, ceil(K / 128)]`` and
    ``b_scales [ceil(N / 128), ceil(K / 128)]`` FP32 with any strides; ``y [T, N]`` is ``out_dtype`` (FP16 or
    BF16). With ``group_ends [E]``, ``b`` is ``[E, N, K]``, ``b_scales [E, ...]``, and each row of ``a`` meets
    its expert's weight; rows past the last end are zero."""
    if a.ndim != 2 or b.ndim != (2 if group_ends is None else 3):
        raise ValueError("matmul_blockscaled expects a [T, K] and b [N, K], or b [E, N, K] with group_ends [E]")
    if a.shape[1] != b.shape[-1]:
        raise ValueError(f"incompatible shapes: a {tuple(a.shape)} and b {tuple(b.shape)}")
    if a.device.type != "cuda" or b.device != a.device:
        raise ValueError("a and b must be on the same CUDA device")
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn:
        raise ValueError("a and b must have dtype torch.float8_e4m3fn")
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype must be torch.float16 or torch.bfloat16, got {out_dtype}")
    rows, k, n = int(a.shape[0]), int(a.shape[1]), int(b.shape[-2])
    groups = 1
    lead: tuple[int, ...] = ()
    if group_ends is not None:
        groups = int(b.shape[0])
        lead = (groups,)
        if not 1 <= groups <= MAX_GROUPS:
            raise ValueError(f"matmul_blockscaled serves 1 to {MAX_GROUPS} experts, got {groups}")
        _check_ends(group_ends, groups, a.device)
    _check_scales("a_scales", a_scales, (rows, _blocks(k)), a.device)
    _check_scales("b_scales", b_scales, (*lead, _blocks(n), _blocks(k)), a.device)
    _refuse_gradient("matmul_blockscaled", a, a_scales, b, b_scales)
    y = torch.empty((rows, n), device=a.device, dtype=out_dtype)
    a, b = _readable(a), _readable(b)
    workspace = _workspace(_native.GROUPED_SCALED, rows, groups, n, k, a.device)
    with _device_guard(a.device):
        _native.check(
            _native.library().hst_matmul_blockscaled(
                _DTYPES[out_dtype], a.data_ptr(), _row_stride(a), a_scales.data_ptr(), a_scales.stride(0),
                a_scales.stride(1), b.data_ptr(), b.stride(0), _row_stride(b), b_scales.data_ptr(),
                b_scales.stride(0), b_scales.stride(-2), b_scales.stride(-1),
                None if group_ends is None else group_ends.data_ptr(), groups, y.data_ptr(), rows, n, k,
                workspace.data_ptr(), workspace.numel(), _stream(a.device),
            )
        )  # fmt: skip
    return y
