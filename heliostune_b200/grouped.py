"""Matrix products over rows grouped by expert, with their gradients (mixture-of-experts layers).

The rows of ``x [T, K]`` are sorted by expert; ``group_ends [E]`` (int32, on the GPU) holds each
expert's end, so expert ``e`` owns rows ``group_ends[e - 1]`` to ``group_ends[e]``::

    y = grouped_matmul(x, weight, group_ends)      # y[t] = x[t] @ weight[e(t)], weight [E, K, N]

``weight`` may also be the transposed view of ``[E, N, K]`` storage (``nn.Linear``'s): both are read
in place. The result is differentiable in ``x`` and ``weight``: ``dx[t] = dy[t] @ weight[e(t)].T`` is
the same kernel on the transposed view, ``dweight[e] = x[e].T @ dy[e]`` its own
(:func:`grouped_weight_grad`).

Nothing is read back from the GPU: the sizes stay there, and a call can be captured into a CUDA
graph and replayed with other ends. (A backward pass is captured, as with any torch operator, while no
eager graph of the same leaves is alive: their gradient nodes would tie the capture to the eager
stream.) Rows past the last end belong to no expert: their outputs and input gradients are zero, and
they enter no weight gradient. An expert without rows gets a zero weight gradient. Each end is taken
clamped to ``[previous end, T]``.

The products are ``torch.library`` operators (``heliostune_b200::grouped_matmul`` and
``::grouped_weight_grad``), so that what traces a program (``torch.jit.trace``, ``make_fx``,
``torch.compile``) records them. ``torch.func``'s transforms are refused.

The heliostune reference has no counterpart (its products have one weight).
"""

from __future__ import annotations

import ctypes
import functools
from collections.abc import Callable
from typing import Any

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from heliostune_b200 import _native
from heliostune_b200.kernel import _device_guard, _stream

#: Most experts one call serves.
MAX_GROUPS = 1024

_DTYPES = {torch.float16: _native.HST_F16, torch.bfloat16: _native.HST_BF16}

_LIBRARY = torch.library.Library("heliostune_b200", "DEF")
#: What a thread adds to every call's dispatch keys by default, and in inference mode.
_PLAIN_THREAD = (
    torch._C.DispatchKeySet(torch._C.DispatchKey.BackendSelect).add(torch._C.DispatchKey.ADInplaceOrView).raw_repr(),
    torch._C.DispatchKeySet(torch._C.DispatchKey.BackendSelect).raw_repr(),
)
_thread_keys = torch._C._dispatch_tls_local_include_set
_PLAIN_TENSORS = (torch.Tensor, torch.nn.Parameter)


def _operator(
    schema: str, check: Callable[..., None], launch: Callable[..., Any], empty: Callable[..., Any]
) -> tuple[Callable[..., Any], Callable[..., Any], Callable[..., Any]]:
    """The operator of ``schema``: ``check`` refuses arguments, ``launch`` runs the kernel, ``empty`` gives the outputs'
    layout. Without it a tracer would see the outputs' allocation alone, and what it makes of a program would
    return uninitialised memory. Returns the function to call and what
    it calls, the kernel or the operator (:func:`_plain`)."""
    name = schema.split("(")[0]

    def kernel(*args: Any) -> Any:
        check(*args)
        return launch(*args)

    def fake(*args: Any) -> Any:
        check(*args)
        return empty(*args)

    _LIBRARY.define(schema)
    # On every device: the kernels refuse those that are not CUDA, as they refuse other types.
    _LIBRARY.impl(name, kernel, "CompositeExplicitAutograd")
    torch.library.register_fake(f"heliostune_b200::{name}", fake, lib=_LIBRARY)
    operator = getattr(torch.ops.heliostune_b200, name).default

    def call(*args: Any) -> Any:
        return kernel(*args) if _plain(args) else operator(*args)

    return call, kernel, operator


def _plain(args: tuple[Any, ...]) -> bool:
    """Whether the dispatcher would lead a call of these arguments straight to the kernel: no tracer, mode or transform
    is on in this thread, and the operands are plain tensors as they stand in memory. The kernel is then called
    at once, which saves 3 us; torch.func's transforms are refused."""
    if torch.compiler.is_compiling():
        return False
    if _thread_keys().raw_repr() not in _PLAIN_THREAD:
        _refuse_transforms()
        return False
    for arg in args:
        if type(arg) in _PLAIN_TENSORS:
            if arg.is_neg():
                return False
        elif arg is not None and type(arg) is not torch.dtype:
            return False
    return True


def _refuse_transforms() -> None:
    """Refuses torch.func's transforms: at their levels the operators have no derivatives."""
    if torch._C._are_functorch_transforms_active():
        raise ValueError("the grouped, quantising and block-scaled operators are not available under torch.func's transforms")


def _refuse_gradient(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise ValueError(f"{what} has no gradient; detach its inputs or run it under torch.no_grad()")
    if forward_ad._current_level >= 0:
        _refuse_tangents(what, *tensors)


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(product: str, device: int, operands: tuple[int, ...]) -> int:
    """Bytes of workspace, by everything the native planner reads: alignments, strides, extents, device."""
    size = ctypes.c_size_t(0)
    _native.check(getattr(_native.library(), f"{product}_workspace")(*operands, device, ctypes.byref(size)))
    return size.value


def _workspace(
    product: str, device: torch.device, operands: tuple[int, ...]
) -> tuple[torch.Tensor | None, int | None, int]:
    """The workspace of one call -- FP32 pieces of tiles shared between CTA pairs, copies of operands a tensor
    map cannot describe -- as a tensor (None if there is none), its address and its bytes."""
    index = device.index if device.index is not None else torch.cuda.current_device()
    nbytes = _workspace_bytes(product, index, operands)
    if nbytes == 0:
        return None, None, 0
    buffer = torch.empty(nbytes, device=device, dtype=torch.uint8)
    return buffer, buffer.data_ptr(), nbytes


def _refuse_tangents(what: str, *tensors: torch.Tensor) -> None:
    """Refuses operands with a forward-mode gradient: the result would come without one, and without an error."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{what} has no forward-mode gradient; take its operands' primals")


def _check_ends(group_ends: torch.Tensor, groups: int, device: int) -> None:
    if group_ends.ndim != 1 or group_ends.shape[0] != groups:
        raise ValueError(f"group_ends must have one entry for each of {groups} weights, got {tuple(group_ends.shape)}")
    if group_ends.dtype != torch.int32:
        raise ValueError("group_ends must have dtype torch.int32")
    if group_ends.get_device() != device:
        raise ValueError("group_ends must be on the device of the operands")
    if not group_ends.is_contiguous():
        raise ValueError("group_ends must be contiguous")


def _check_operands(what: str, x: torch.Tensor, other: torch.Tensor, names: tuple[str, str]) -> None:
    if not x.is_cuda or not other.is_cuda or other.get_device() != x.get_device():
        raise ValueError(f"{names[0]} and {names[1]} must be on the same CUDA device")
    if x.dtype not in _DTYPES or other.dtype != x.dtype:
        raise ValueError(f"{what} serves torch.float16 or torch.bfloat16, the same for {names[0]} and {names[1]}")


def _check_matmul(x: torch.Tensor, weight: torch.Tensor, group_ends: torch.Tensor) -> None:
    # A recorded program calls the operator itself, which has no gradient.
    _refuse_gradient("grouped_matmul", x, weight)
    if x.ndim != 2 or weight.ndim != 3:
        raise ValueError("grouped_matmul expects x [T, K] and weight [E, K, N]")
    if x.shape[1] != weight.shape[1]:
        raise ValueError(f"incompatible shapes: x {tuple(x.shape)} and weight {tuple(weight.shape)}")
    _check_operands("grouped_matmul", x, weight, ("x", "weight"))
    if not 1 <= weight.shape[0] <= MAX_GROUPS:
        raise ValueError(f"grouped_matmul serves 1 to {MAX_GROUPS} experts, got {weight.shape[0]}")
    _check_ends(group_ends, weight.shape[0], x.get_device())


def _launch_matmul(x: torch.Tensor, weight: torch.Tensor, group_ends: torch.Tensor) -> torch.Tensor:
    groups, k, n = weight.shape
    rows, device = x.shape[0], x.device
    y = x.new_empty((rows, n))
    x_pointer, x_strides, w_pointer, w_strides = x.data_ptr(), x.stride(), weight.data_ptr(), weight.stride()
    workspace, ws_pointer, ws_bytes = _workspace(
        "hst_grouped_matmul", device, (x_pointer & 15, *x_strides, w_pointer & 15, *w_strides, groups, rows, n, k)
    )
    with _device_guard(device):
        _native.check(
            _native.library().hst_grouped_matmul(
                _DTYPES[x.dtype], x_pointer, *x_strides, w_pointer, *w_strides, group_ends.data_ptr(), groups,
                y.data_ptr(), rows, n, k, ws_pointer, ws_bytes, _stream(device),
            )
        )  # fmt: skip
    del workspace  # stream-ordered reuse by the caching allocator is safe on this stream
    return y


def _empty_matmul(x: torch.Tensor, weight: torch.Tensor, group_ends: torch.Tensor) -> torch.Tensor:
    return x.new_empty((x.shape[0], weight.shape[2]))


def _check_weight_grad(x: torch.Tensor, dy: torch.Tensor, group_ends: torch.Tensor) -> None:
    _refuse_gradient("grouped_weight_grad", x, dy)
    if x.ndim != 2 or dy.ndim != 2 or x.shape[0] != dy.shape[0]:
        raise ValueError(f"grouped_weight_grad expects x [T, K] and dy [T, N], got {tuple(x.shape)} and {tuple(dy.shape)}")
    _check_operands("grouped_weight_grad", x, dy, ("x", "dy"))
    groups = int(group_ends.shape[0]) if group_ends.ndim == 1 else 0
    if not 1 <= groups <= MAX_GROUPS:
        raise ValueError(f"grouped_weight_grad serves 1 to {MAX_GROUPS} experts, got {groups}")
    _check_ends(group_ends, groups, x.get_device())


def _launch_weight_grad(left: torch.Tensor, right: torch.Tensor, group_ends: torch.Tensor) -> torch.Tensor:
    groups = group_ends.shape[0]
    (rows, lcols), rcols, device = left.shape, right.shape[1], left.device
    out = left.new_empty((groups, lcols, rcols))
    l_pointer, l_strides, r_pointer, r_strides = left.data_ptr(), left.stride(), right.data_ptr(), right.stride()
    workspace, ws_pointer, ws_bytes = _workspace(
        "hst_grouped_weight_grad",
        device,
        (l_pointer & 15, *l_strides, r_pointer & 15, *r_strides, groups, rows, lcols, rcols),
    )
    with _device_guard(device):
        _native.check(
            _native.library().hst_grouped_weight_grad(
                _DTYPES[left.dtype], l_pointer, *l_strides, r_pointer, *r_strides, group_ends.data_ptr(), groups,
                out.data_ptr(), rows, lcols, rcols, ws_pointer, ws_bytes, _stream(device),
            )
        )  # fmt: skip
    del workspace
    return out


def _empty_weight_grad(left: torch.Tensor, right: torch.Tensor, group_ends: torch.Tensor) -> torch.Tensor:
    return left.new_empty((group_ends.shape[0], left.shape[1], right.shape[1]))


_matmul, _matmul_kernel, _matmul_operator = _operator(
    "grouped_matmul(Tensor x, Tensor weight, Tensor group_ends) -> Tensor", _check_matmul, _launch_matmul, _empty_matmul
)
_weight_grad, _weight_grad_kernel, _weight_grad_operator = _operator(
    "grouped_weight_grad(Tensor x, Tensor dy, Tensor group_ends) -> Tensor",
    _check_weight_grad,
    _launch_weight_grad,
    _empty_weight_grad,
)


def grouped_weight_grad(x: torch.Tensor, dy: torch.Tensor, group_ends: torch.Tensor) -> torch.Tensor:
    """``out[e] = x[rows of e].T @ dy[rows of e]``, ``[E, K, N]``: the weight gradient of
    :func:`grouped_matmul`, with FP32 sums over the rows and one rounding. ``x [T, K]`` and ``dy [T, N]``
    are FP16 or BF16 with any strides (copied in every call where their rows are
    not 16-byte aligned)."""
    return _weight_grad(x, dy, group_ends)


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, group_ends):  # type: ignore[no-untyped-def]
        y = _matmul(x, weight, group_ends)
        # Each gradient reads the other operand: what is frozen keeps nothing alive.
        need_x, need_weight, _ = ctx.needs_input_grad
        ctx.save_for_backward(x if need_weight else None, weight if need_x else None, group_ends)
        # [E, N, K] storage: its gradient gets the same layout, so that it adds up in place.
        ctx.weight_by_n = weight.stride(1) == 1 and weight.stride(2) != 1
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):  # type: ignore[no-untyped-def]
        x, weight, group_ends = ctx.saved_tensors
        # The saved tensors are checked again: a hook may have packed and unpacked them.
        plain = _plain((dy, x, weight, group_ends))
        matmul, weight_grad = (_matmul_kernel, _weight_grad_kernel) if plain else (_matmul_operator, _weight_grad_operator)
        dx = dweight = None
        if ctx.needs_input_grad[0]:
            dx = matmul(dy, weight.transpose(1, 2), group_ends)
        if ctx.needs_input_grad[1]:
            if ctx.weight_by_n:
                dweight = weight_grad(dy, x, group_ends).transpose(1, 2)
            else:
                dweight = weight_grad(x, dy, group_ends)
        return dx, dweight, None


def grouped_matmul(x: torch.Tensor, weight: torch.Tensor, group_ends: torch.Tensor) -> torch.Tensor:
    """``y[t] = x[t] @ weight[e(t)]`` with FP32 accumulation: ``x [T, K]``, ``weight [E, K, N]`` (either of
    its last two dimensions contiguous), both FP16 or both BF16, ``y [T, N]`` of their type; 1 to
    :data:`MAX_GROUPS` experts. Any strides are served; operands whose rows are not 16-byte aligned
    are copied in every call, the weights of experts that have rows (4096 rows over 32 experts, N 1408, FP16: K 2048
    53 us, 2047 with rows along N 59, along K 130). Differentiable in ``x`` and ``weight`` (once, in reverse mode)."""
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        if not torch.compiler.is_compiling():
            _refuse_transforms()
        _refuse_tangents("grouped_matmul", x, weight)
        return _GroupedMatmul.apply(x, weight, group_ends)
    return _matmul(x, weight, group_ends)
