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
from heliostune_b200.grouped import (
    _DTYPES, MAX_GROUPS, _check_ends, _operator, _refuse_gradient, _workspace,
)  # fmt: skip
from heliostune_b200.kernel import _device_guard, _stream

#: Values that share a scale along a row (and, for tiles, along a column).
BLOCK = 128


def _blocks(extent: int) -> int:
    return -(-extent // BLOCK)


def _check_quantize(what: str, x: torch.Tensor) -> None:
    _refuse_gradient(what, x)
    if not x.is_cuda:
        raise ValueError(f"{what} expects a CUDA tensor")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what} serves torch.float16 or torch.bfloat16, got {x.dtype}")


def _check_rows(x: torch.Tensor) -> None:
    if x.ndim != 2:
        raise ValueError("quantize_rows expects x [T, K]")
    _check_quantize("quantize_rows", x)


def _check_tiles(weight: torch.Tensor) -> None:
    if weight.ndim not in (2, 3):
        raise ValueError("quantize_tiles expects weight [N, K] or [E, N, K]")
    _check_quantize("quantize_tiles", weight)


def _outputs(x: torch.Tensor, tiles: bool) -> tuple[torch.Tensor, torch.Tensor]:
    *batch, rows, cols = x.shape
    # Rows of q start on 16 bytes, so that the products read them in place.
    width = -(-cols // 16) * 16
    q = x.new_empty((*batch, rows, width), dtype=torch.float8_e4m3fn)
    if width != cols:
        q = q[..., :cols]
    if tiles:
        return q, x.new_empty((*batch, _blocks(rows), _blocks(cols)), dtype=torch.float32)
    # Stored [blocks, rows]: the products read one block's scales of neighbouring rows together.
    return q, x.new_empty_strided((rows, _blocks(cols)), (1, rows), dtype=torch.float32)


def _quantize(x: torch.Tensor, tiles: bool) -> tuple[torch.Tensor, torch.Tensor]:
    q, scales = _outputs(x, tiles)
    *batch, rows, cols = x.shape
    device = x.device
    width = -(-cols // 16) * 16
    blocks = _blocks(cols)
    s_batch, s_row, s_col = (_blocks(rows) * blocks, blocks, 1) if tiles else (0, 1, rows)
    *x_batch, x_row, x_col = x.stride()
    count, lead = (batch[0], (x_batch[0], rows * width, s_batch)) if batch else (1, (0, 0, 0))
    with _device_guard(device):
        _native.check(
            _native.library().hst_quantize_e4m3(
                _DTYPES[x.dtype], tiles, x.data_ptr(), lead[0], x_row, x_col, q.data_ptr(), lead[1], width,
                scales.data_ptr(), lead[2], s_row, s_col, count, rows, cols, _stream(device),
            )
        )  # fmt: skip
    return q, scales


_quantize_rows, *_ = _operator(
    "quantize_rows(Tensor x) -> (Tensor, Tensor)", _check_rows, lambda x: _quantize(x, False), lambda x: _outputs(x, False)
)
_quantize_tiles, *_ = _operator(
    "quantize_tiles(Tensor weight) -> (Tensor, Tensor)",
    _check_tiles,
    lambda weight: _quantize(weight, True),
    lambda weight: _outputs(weight, True),
)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scales)`` of ``x [T, K]`` (FP16 or BF16, any strides): ``q [T, K]`` in ``torch.float8_e4m3fn``
    and FP32 ``scales [T, ceil(K / 128)]``, one for each 128 consecutive values of a row. The scales are
    the transposed view of ``[blocks, T]`` storage."""
    return _quantize_rows(x)


def quantize_tiles(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scales)`` of ``weight [N, K]`` or ``[E, N, K]`` (FP16 or BF16, any strides): ``q`` of its shape
    in ``torch.float8_e4m3fn`` and FP32 ``scales [..., ceil(N / 128), ceil(K / 128)]``, one for each
    128 x 128 tile. Contiguous rows are read at the rate of HBM, those of a transposed view a value at a time
    (18944 x 3584: 37 us and 531)."""
    return _quantize_tiles(weight)


def _check_scales(name: str, scales: torch.Tensor, shape: tuple[int, ...], device: int) -> None:
    if scales.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(scales.shape)}")
    if scales.dtype != torch.float32:
        raise ValueError(f"{name} must have dtype torch.float32")
    if scales.get_device() != device:
        raise ValueError(f"{name} must be on the device of the operands")


def _check_product(
    a: torch.Tensor,
    a_scales: torch.Tensor,
    b: torch.Tensor,
    b_scales: torch.Tensor,
    group_ends: torch.Tensor | None,
    out_dtype: torch.dtype,
) -> None:
    _refuse_gradient("matmul_blockscaled", a, a_scales, b, b_scales)
    if a.ndim != 2 or b.ndim != (2 if group_ends is None else 3):
        raise ValueError("matmul_blockscaled expects a [T, K] and b [N, K], or b [E, N, K] with group_ends [E]")
    if a.shape[1] != b.shape[-1]:
        raise ValueError(f"incompatible shapes: a {tuple(a.shape)} and b {tuple(b.shape)}")
    index = a.get_device()
    if not a.is_cuda or not b.is_cuda or b.get_device() != index:
        raise ValueError("a and b must be on the same CUDA device")
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn:
        raise ValueError("a and b must have dtype torch.float8_e4m3fn")
    if out_dtype not in _DTYPES:
        raise ValueError(f"out_dtype must be torch.float16 or torch.bfloat16, got {out_dtype}")
    (rows, k), n = a.shape, b.shape[-2]
    lead: tuple[int, ...] = ()
    if group_ends is not None:
        lead = (b.shape[0],)
        if not 1 <= b.shape[0] <= MAX_GROUPS:
            raise ValueError(f"matmul_blockscaled serves 1 to {MAX_GROUPS} experts, got {b.shape[0]}")
        _check_ends(group_ends, b.shape[0], index)
    _check_scales("a_scales", a_scales, (rows, _blocks(k)), index)
    _check_scales("b_scales", b_scales, (*lead, _blocks(n), _blocks(k)), index)


def _launch_product(
    a: torch.Tensor,
    a_scales: torch.Tensor,
    b: torch.Tensor,
    b_scales: torch.Tensor,
    group_ends: torch.Tensor | None,
    out_dtype: torch.dtype,
) -> torch.Tensor:
    (rows, k), n, device = a.shape, b.shape[-2], a.device
    y = a.new_empty((rows, n), dtype=out_dtype)
    a_pointer, a_strides, b_pointer, b_strides, sb_strides = a.data_ptr(), a.stride(), b.data_ptr(), b.stride(), b_scales.stride()
    if group_ends is None:
        groups, ends, b_strides, sb_strides = 1, None, (0, *b_strides), (0, *sb_strides)
    else:
        groups, ends = b.shape[0], group_ends.data_ptr()
    workspace, ws_pointer, ws_bytes = _workspace(
        "hst_matmul_blockscaled",
        device,
        (a_pointer & 15, *a_strides, b_pointer & 15, *b_strides, groups, rows, n, k),
    )
    with _device_guard(device):
        _native.check(
            _native.library().hst_matmul_blockscaled(
                _DTYPES[out_dtype], a_pointer, *a_strides, a_scales.data_ptr(), *a_scales.stride(), b_pointer, *b_strides,
                b_scales.data_ptr(), *sb_strides, ends, groups, y.data_ptr(), rows, n, k, ws_pointer, ws_bytes,
                _stream(device),
            )
        )  # fmt: skip
    del workspace  # stream-ordered reuse by the caching allocator is safe on this stream
    return y


def _empty_product(
    a: torch.Tensor,
    a_scales: torch.Tensor,
    b: torch.Tensor,
    b_scales: torch.Tensor,
    group_ends: torch.Tensor | None,
    out_dtype: torch.dtype,
) -> torch.Tensor:
    return a.new_empty((a.shape[0], b.shape[-2]), dtype=out_dtype)


_product, *_ = _operator(
    "matmul_blockscaled(Tensor a, Tensor a_scales, Tensor b, Tensor b_scales, Tensor? group_ends, ScalarType out_dtype) -> Tensor",
    _check_product,
    _launch_product,
    _empty_product,
)


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
    return _product(a, a_scales, b, b_scales, group_ends, out_dtype)
