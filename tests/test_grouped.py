"""The products over rows grouped by expert (``grouped.grouped_matmul``, ``grouped_weight_grad``) against
the same sums in 64 bits.

Tolerance: one rounding to the output type, at most ``eps / 2`` of the value, and the FP32 sum of ``K``
exact products, each step of which is off by at most one unit in the last place (2^-23) of the sum of
magnitudes so far: ``K * 2^-23 * sum |a||b|``. FP16 results below 2^-14 are off by up to half a
subnormal step, 2^-25.
"""

from __future__ import annotations

import ctypes
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from heliostune_b200 import _native, grouped

gpu = pytest.mark.gpu
DTYPES = (torch.float16, torch.bfloat16)


@pytest.fixture(autouse=True)
def _status(request: pytest.FixtureRequest):  # type: ignore[no-untyped-def]
    yield
    if request.node.get_closest_marker("gpu") and torch.cuda.is_available():
        assert _native.status(torch.cuda.current_device()) == 0


def _bounds(ends: list[int], rows: int) -> list[tuple[int, int]]:
    """The rows of each group as the operators take them: every end clamped to [previous end, rows]."""
    out, start = [], 0
    for end in ends:
        end = max(start, min(max(end, 0), rows))
        out.append((start, end))
        start = end
    return out


def _assert_close(out: torch.Tensor, exact: torch.Tensor, magnitude: torch.Tensor, terms: int) -> None:
    assert out.shape == exact.shape
    half_step = torch.finfo(out.dtype).eps / 2
    slack = (terms + 1) * 2.0**-23 * magnitude
    bound = half_step * exact.abs() + (1 + half_step) * slack + 2.0**-25
    error = (out.double() - exact).abs()
    assert bool((error <= bound).all()), ((error - bound).max().item(), error.max().item())


def _check_forward(y: torch.Tensor, x: torch.Tensor, w: torch.Tensor, ends: list[int]) -> None:
    covered = 0
    for e, (start, end) in enumerate(_bounds(ends, x.shape[0])):
        a, b = x[start:end].double(), w[e].double()
        _assert_close(y[start:end], a @ b, a.abs() @ b.abs(), x.shape[1])
        covered = end
    assert bool((y[covered:] == 0).all())


def _check_weight_grad(dw: torch.Tensor, x: torch.Tensor, dy: torch.Tensor, ends: list[int]) -> None:
    for e, (start, end) in enumerate(_bounds(ends, x.shape[0])):
        a, b = x[start:end].double().T, dy[start:end].double()
        _assert_close(dw[e], a @ b, a.abs() @ b.abs(), end - start)
        if start == end:
            assert bool((dw[e] == 0).all())


def _operands(rows: int, groups: int, k: int, n: int, dtype: torch.dtype, layout: str, seed: int):  # type: ignore[no-untyped-def]
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, k), generator=g, device="cuda").to(dtype)
    shape = (groups, k, n) if layout == "kn" else (groups, n, k)
    w = (torch.randn(shape, generator=g, device="cuda") / max(k, 1) ** 0.5).to(dtype)
    dy = torch.randn((rows, n), generator=g, device="cuda").to(dtype)
    return x, w if layout == "kn" else w.transpose(1, 2), dy


def _ends(values: list[int]) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------
# Refusals, before any CUDA work
# ------------------------------------------------------------------------------------------


def test_inputs_are_checked_before_any_cuda_work() -> None:
    x = torch.zeros((4, 16), dtype=torch.float16)
    w = torch.zeros((2, 16, 8), dtype=torch.float16)
    ends = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match=r"x \[T, K\]"):
        grouped.grouped_matmul(x[0], w, ends)
    with pytest.raises(ValueError, match="incompatible shapes"):
        grouped.grouped_matmul(x[:, :8], w, ends)
    with pytest.raises(ValueError, match="same CUDA device"):
        grouped.grouped_matmul(x, w, ends)
    with pytest.raises(ValueError, match=r"x \[T, K\] and dy"):
        grouped.grouped_weight_grad(x, x[:3], ends)
    with pytest.raises(ValueError, match="same CUDA device"):
        grouped.grouped_weight_grad(x, x, ends)


def test_operands_with_a_forward_gradient_are_refused() -> None:
    """A dual tensor does not require grad: its tangent would be lost without an error."""
    x = torch.zeros((4, 16), dtype=torch.float16)
    w = torch.zeros((2, 16, 8), dtype=torch.float16)
    ends = torch.zeros(2, dtype=torch.int32)
    with forward_ad.dual_level():
        for args in ((forward_ad.make_dual(x, x), w), (x, forward_ad.make_dual(w, w))):
            with pytest.raises(ValueError, match="grouped_matmul has no forward-mode gradient"):
                grouped.grouped_matmul(*args, ends)
        with pytest.raises(ValueError, match="grouped_weight_grad has no forward-mode gradient"):
            grouped.grouped_weight_grad(x, forward_ad.make_dual(x, x), ends)
        with pytest.raises(ValueError, match="same CUDA device"):  # as before
            grouped.grouped_matmul(x, w, ends)


@gpu
def test_a_forward_gradient_is_refused_on_the_gpu_and_its_primal_taken() -> None:
    x, w, dy = _operands(9, 2, 32, 16, torch.float16, "kn", seed=31)
    ends = _ends([4, 9])
    expected = grouped.grouped_matmul(x, w, ends)
    with forward_ad.dual_level():
        for grad in (torch.no_grad(), torch.enable_grad()):
            with grad:
                for args in ((forward_ad.make_dual(x, x), w), (x, forward_ad.make_dual(w, w))):
                    with pytest.raises(ValueError, match="forward-mode"):
                        grouped.grouped_matmul(*args, ends)
        assert torch.equal(grouped.grouped_matmul(forward_ad.unpack_dual(forward_ad.make_dual(x, x)).primal, w, ends), expected)
        with pytest.raises(ValueError, match="forward-mode"):
            grouped.grouped_weight_grad(forward_ad.make_dual(x, x), dy, ends)
        leaf = x.clone().requires_grad_()
        with pytest.raises(ValueError, match="forward-mode"):
            torch.autograd.grad(grouped.grouped_matmul(leaf, w, ends), (leaf,), forward_ad.make_dual(dy, dy))


def test_the_library_refuses_bad_calls_before_any_cuda_work() -> None:
    # In a thread of its own: the library keeps the last error of each.
    with ThreadPoolExecutor(1) as thread:
        thread.submit(_refused_calls).result()


def _refused_calls() -> None:
    _native.build_library()
    lib = _native.library()

    def matmul(dtype=0, groups=2, rows=4, n=8, k=16, x=16, w=16, ends=16, y=16):  # type: ignore[no-untyped-def]
        return lib.hst_grouped_matmul(dtype, x, k, 1, w, k * n, n, 1, ends, groups, y, rows, n, k, None, 0, None)

    for kwargs, message in (
        ({"dtype": 7}, b"data type"),
        ({"groups": 0}, b"1 to 1024"),
        ({"groups": 1025}, b"1 to 1024"),
        ({"ends": None}, b"ends are null"),
        ({"rows": -1}, b"row count"),
        ({"n": -1}, b"extents"),
        ({"k": 2**31}, b"extents"),
        ({"y": None}, b"y is null"),
        ({"x": None}, b"x or w is null"),
        ({"w": None}, b"x or w is null"),
        ({"x": 17}, b"x must be aligned to 2"),
        ({"w": 17}, b"w must be aligned to 2"),
        ({"y": 17}, b"y must be aligned to 2"),
        ({"ends": 18}, b"ends must be aligned to 4"),
    ):
        assert matmul(**kwargs) == _native.HST_ERR_INVALID, kwargs
        assert message in lib.hst_last_error(), kwargs
    assert matmul(rows=0) == _native.HST_OK
    assert lib.hst_grouped_weight_grad(0, None, 8, 1, 16, 8, 1, 16, 2, 16, 4, 8, 8, None, 0, None) == _native.HST_ERR_INVALID
    assert b"left or right is null" in lib.hst_last_error()
    assert lib.hst_grouped_weight_grad(0, 17, 8, 1, 16, 8, 1, 16, 2, 16, 4, 8, 8, None, 0, None) == _native.HST_ERR_INVALID
    assert b"left must be aligned" in lib.hst_last_error()
    assert lib.hst_grouped_weight_grad(3, 16, 8, 1, 16, 8, 1, 16, 2, 16, 4, 8, 8, None, 0, None) == _native.HST_ERR_INVALID


def test_broadcast_operands_too_large_to_copy_are_refused_before_any_cuda_work() -> None:
    """1024 weights of 7 * 2^27 rows and columns that share one row: the bytes of their copy, 49 * 2^65, are 0 in 64 bits."""
    with ThreadPoolExecutor(1) as thread:
        thread.submit(_refused_copies).result()


def _refused_copies() -> None:
    _native.build_library()
    lib = _native.library()
    size = ctypes.c_size_t(0)
    k = n = 7 * 2**27
    calls = (
        lambda: lib.hst_grouped_matmul_workspace(16, k, 1, 16, 0, 0, 1, 1024, 1, n, k, 0, ctypes.byref(size)),
        lambda: lib.hst_grouped_matmul(0, 16, k, 1, 16, 0, 0, 1, 16, 1024, 16, 1, n, k, None, 0, None),
        lambda: lib.hst_grouped_weight_grad_workspace(16, 0, 1, 16, 0, 1, 1, n, k, 8, 0, ctypes.byref(size)),
        lambda: lib.hst_grouped_weight_grad(0, 16, 0, 1, 16, 8, 1, 16, 1, 16, n, k, 8, None, 0, None),
        lambda: lib.hst_matmul_blockscaled_workspace(16, k, 1, 16, 0, 0, 1, 1024, 1, n, k, 0, ctypes.byref(size)),
        lambda: lib.hst_matmul_blockscaled(0, 16, k, 1, 16, 1, 1, 16, 0, 0, 1, 16, 1, 1, 1, 16, 1024, 16, 1, n, k, None, 0, None),
    )
    for call in calls:
        assert call() == _native.HST_ERR_UNSUPPORTED
        assert b"too large" in lib.hst_last_error()


# ------------------------------------------------------------------------------------------
# Tracing and transforms
# ------------------------------------------------------------------------------------------


def test_tracing_records_the_operators() -> None:
    """On fake CUDA tensors: what is recorded are the operators, not the allocation of their outputs."""
    with FakeTensorMode():
        x = torch.empty((9, 32), device="cuda", dtype=torch.float16)
        w = torch.empty((2, 32, 16), device="cuda", dtype=torch.float16)
        dy = torch.empty((9, 16), device="cuda", dtype=torch.float16)
        ends = torch.empty(2, device="cuda", dtype=torch.int32)

        def step(x, w, dy, ends):  # type: ignore[no-untyped-def]
            return grouped.grouped_matmul(x, w, ends), grouped.grouped_weight_grad(x, dy, ends)

        traced = make_fx(step)(x, w, dy, ends)
        called = [node.target for node in traced.graph.nodes if node.op == "call_function"]
        ops = torch.ops.heliostune_b200
        assert called == [ops.grouped_matmul.default, ops.grouped_weight_grad.default]
        y, dw = step(x, w, dy, ends)
        assert y.shape == (9, 16) and dw.shape == (2, 32, 16) and y.dtype == dw.dtype == torch.float16
        with pytest.raises(ValueError, match="incompatible shapes"):
            grouped.grouped_matmul(x[:, :8], w, ends)


def test_transforms_are_refused() -> None:
    x = torch.zeros((4, 16), dtype=torch.float16)
    w = torch.zeros((2, 16, 8), dtype=torch.float16)
    ends = torch.zeros(2, dtype=torch.int32)
    one = torch.ones_like(x)

    def product(x: torch.Tensor) -> torch.Tensor:
        return grouped.grouped_matmul(x, w, ends)

    for transformed in (
        lambda: torch.func.jvp(product, (x,), (one,)),
        lambda: torch.func.grad(lambda x: product(x).sum())(x),
        lambda: torch.vmap(product)(x[None]),
        lambda: torch.func.grad(lambda x: torch.vmap(product)(x[None]).sum())(x),
        lambda: torch.func.jvp(lambda x: grouped.grouped_weight_grad(x, x, ends), (x,), (one,)),
    ):
        with pytest.raises(ValueError, match="torch.func's transforms"):
            transformed()


@gpu
def test_traced_programs_compute_what_they_recorded() -> None:
    x, w, dy = _operands(90, 3, 96, 56, torch.float16, "nk", seed=32)
    ends = _ends([19, 19, 83])

    def step(x, w, dy, ends):  # type: ignore[no-untyped-def]
        return grouped.grouped_matmul(x, w, ends), grouped.grouped_weight_grad(x, dy, ends)

    others = _operands(90, 3, 96, 56, torch.float16, "nk", seed=33)
    expected = step(*others, _ends([40, 41, 90]))
    for program in (
        torch.jit.trace(step, (x, w, dy, ends)),
        make_fx(step)(x, w, dy, ends),
        make_fx(step, tracing_mode="fake")(x, w, dy, ends),
        torch.compile(step, fullgraph=True, backend="aot_eager"),
    ):
        for got, want in zip(program(*others, _ends([40, 41, 90])), expected, strict=True):
            assert torch.equal(got, want) and got.stride() == want.stride()
    # A recorded operator has no gradient of its own; what the public call does with one stays as it is.
    with pytest.raises(ValueError, match="no gradient"):
        make_fx(step)(x, w, dy, ends)(x.clone().requires_grad_(), w, dy, ends)


@gpu
def test_views_that_stand_for_the_negative_of_their_memory() -> None:
    """The imaginary part of a conjugate is a view with the negative bit set: its values are not those in memory."""
    x, w, _ = _operands(60, 2, 64, 48, torch.float16, "kn", seed=35)
    ends = _ends([23, 60])
    x = torch.view_as_complex(x.view(60, 32, 2)).conj().imag
    dy = torch.view_as_complex(torch.randn((60, 48, 2), device="cuda").half()).conj().imag
    w = w[:, :32]
    assert x.is_neg() and dy.is_neg()
    assert torch.equal(grouped.grouped_matmul(x, w, ends), grouped.grouped_matmul(x.resolve_neg(), w, ends))
    expected = grouped.grouped_weight_grad(x.resolve_neg(), dy.resolve_neg(), ends)
    assert torch.equal(grouped.grouped_weight_grad(x, dy, ends), expected)
    leaf = w.detach().clone().requires_grad_()
    grouped.grouped_matmul(x, leaf, ends).backward(dy)
    assert torch.equal(leaf.grad, expected)


@gpu
def test_a_compiled_step_has_the_eager_gradients() -> None:
    x, w, dy = _operands(90, 3, 96, 56, torch.bfloat16, "kn", seed=34)
    ends = _ends([19, 19, 83])
    x.requires_grad_()
    w = w.detach().requires_grad_()
    eager = torch.autograd.grad(grouped.grouped_matmul(x, w, ends), (x, w), dy)
    compiled = torch.compile(grouped.grouped_matmul, backend="aot_eager")
    for got, want in zip(torch.autograd.grad(compiled(x, w, ends), (x, w), dy), eager, strict=True):
        assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------
# Values
# ------------------------------------------------------------------------------------------

#: (rows, ends): one row; tile edges of 32, 256 and their neighbours; empty groups first, last and between;
#: rows past the last end; all groups empty.
ROWS = (
    (1, [1]),
    (1, [0, 1, 1]),
    (7, [3, 3, 7]),
    (96, [32, 63, 96]),
    (300, [0, 255, 255, 300]),
    (700, [256, 513, 700]),
    (530, [1, 2, 259, 500]),
    (40, [0, 0, 0]),
    (1111, [600, 600, 1100]),
)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ("kn", "nk"))
@pytest.mark.parametrize("rows,ends", ROWS)
@pytest.mark.parametrize("k,n", ((64, 256), (200, 264), (1000, 72), (1096, 264)))
def test_forward_and_gradients(dtype: torch.dtype, layout: str, rows: int, ends: list[int], k: int, n: int) -> None:
    x, w, dy = _operands(rows, len(ends), k, n, dtype, layout, seed=rows + k)
    x.requires_grad_()
    w = w.detach().requires_grad_()
    y = grouped.grouped_matmul(x, w, _ends(ends))
    assert y.dtype == dtype
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    x, w = x.detach(), w.detach()
    _check_forward(y.detach(), x, w, ends)
    _check_forward(dx, dy, w.transpose(1, 2), ends)
    _check_weight_grad(dw, x, dy, ends)
    assert dw.stride() == w.stride()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ("kn", "nk"))
@pytest.mark.parametrize("k,n", ((1, 1), (13, 17), (65, 7), (8, 1001)))
def test_extents_that_tma_cannot_read(dtype: torch.dtype, layout: str, k: int, n: int) -> None:
    ends = [5, 5, 40, 70]
    x, w, dy = _operands(75, 4, k, n, dtype, layout, seed=k * n)
    _check_forward(grouped.grouped_matmul(x, w, _ends(ends)), x, w, ends)
    _check_forward(grouped.grouped_matmul(dy, w.transpose(1, 2), _ends(ends)), dy, w.transpose(1, 2), ends)
    _check_weight_grad(grouped.grouped_weight_grad(x, dy, _ends(ends)), x, dy, ends)


@gpu
def test_long_sums_and_many_tiles_are_joined_across_pairs() -> None:
    ends = [40, 41, 300]
    x, w, dy = _operands(300, 3, 4104, 520, torch.bfloat16, "kn", seed=3)
    _check_forward(grouped.grouped_matmul(x, w, _ends(ends)), x, w, ends)
    ends = [5000, 5003, 9000]
    x, w, dy = _operands(9001, 3, 136, 520, torch.float16, "nk", seed=4)
    _check_weight_grad(grouped.grouped_weight_grad(x, dy, _ends(ends)), x, dy, ends)
    _check_forward(grouped.grouped_matmul(x, w, _ends(ends)), x, w, ends)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ("kn", "nk"))
@pytest.mark.parametrize("rows,ends", ((1, [0, 1]), (70, [33, 33, 70]), (300, [0, 255, 255, 290]), (700, [256, 513, 700]), (40, [0, 0])))
@pytest.mark.parametrize("n", (264, 72, 1001))
def test_deep_tiles_are_cut_and_joined(dtype: torch.dtype, layout: str, rows: int, ends: list[int], n: int) -> None:
    x, w, _ = _operands(rows, len(ends), 4176, n, dtype, layout, seed=rows + n)
    _check_forward(grouped.grouped_matmul(x, w, _ends(ends)), x, w, ends)


@gpu
@pytest.mark.parametrize("ends", ([4600, 4600, 4650], [0, 3100, 6100, 6101], [6200]))
@pytest.mark.parametrize("k,n", ((200, 264), (301, 77), (72, 1000)))
def test_deep_weight_gradients_are_cut_and_joined(ends: list[int], k: int, n: int) -> None:
    x, _, dy = _operands(6200, 1, k, n, torch.bfloat16, "kn", seed=k)
    _check_weight_grad(grouped.grouped_weight_grad(x, dy, _ends(ends)), x, dy, ends)


@gpu
def test_a_replay_cuts_tiles_where_its_ends_ask_for_it() -> None:
    # 66 K blocks, 19 column tiles: of two groups 38 tiles (whole), of one 19 (cut: a pair would idle for 49 blocks).
    x, w, _ = _operands(300, 3, 4168, 4736, torch.bfloat16, "kn", seed=23)
    ends = _ends([0, 0, 0])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        grouped.grouped_matmul(x, w, ends)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = grouped.grouped_matmul(x, w, ends)
    for values in ([200, 200, 300], [0, 1, 1], [100, 200, 300], [0, 0, 0], [0, 256, 256]):
        ends.copy_(_ends(values))
        graph.replay()
        torch.cuda.synchronize()
        _check_forward(y, x, w, values)
        assert torch.equal(y, grouped.grouped_matmul(x, w, ends))


@gpu
@pytest.mark.parametrize("k,n", ((2312, 2056), (2304, 2048)))  # 90 and 72 tiles a group: more and fewer than the pairs of SMs
@pytest.mark.parametrize("ends", ([300, 300, 1700], [0, 1100, 1101], [1500, 1500, 1500]))
def test_weight_gradients_of_many_tiles(k: int, n: int, ends: list[int]) -> None:
    x, _, dy = _operands(1703, 1, k, n, torch.float16, "kn", seed=20)
    _check_weight_grad(grouped.grouped_weight_grad(x, dy, _ends(ends)), x, dy, ends)


def _pairs() -> int:
    count = ctypes.c_int(0)
    _native.check(_native.library().hst_device_sm_count(torch.cuda.current_device(), ctypes.byref(count)))
    return count.value // 2


def _cut_weight_grad(x: torch.Tensor, dy: torch.Tensor, ends: list[int]) -> tuple[torch.Tensor, int]:
    """The weight gradient over the C ABI, and into how many FP32 pieces its cut tiles were written: those of
    the workspace (one of 128 x 256 values for each CTA of a pair, contiguous operands) that hold anything."""
    lib, (rows, k), n, groups = _native.library(), x.shape, dy.shape[1], len(ends)
    size = ctypes.c_size_t(0)
    operands = x.data_ptr(), k, 1, dy.data_ptr(), n, 1
    _native.check(lib.hst_grouped_weight_grad_workspace(*operands, groups, rows, k, n, x.get_device(), ctypes.byref(size)))
    workspace = torch.full((size.value // 4,), -1, device="cuda", dtype=torch.int32)
    out, group_ends = torch.empty((groups, k, n), device="cuda", dtype=x.dtype), _ends(ends)
    _native.check(
        lib.hst_grouped_weight_grad(
            grouped._DTYPES[x.dtype], *operands, group_ends.data_ptr(), groups, out.data_ptr(), rows, k, n,
            workspace.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream,
        )
    )  # fmt: skip
    return out, _pieces(workspace, 256)


def _pieces(workspace: torch.Tensor, width: int) -> int:
    """Pieces of a workspace, filled with ones before the call, that hold anything: 128 x width values for each of
    the two CTAs of a pair."""
    return int((workspace.view(-1, 2 * 128 * width) != -1).any(dim=1).sum())


def _cut_forward(x: torch.Tensor, w: torch.Tensor, ends: list[int]) -> tuple[torch.Tensor, int]:
    """The same for the forward product (no operand of which needs a copy)."""
    lib, (rows, k), (groups, _, n) = _native.library(), x.shape, w.shape
    size = ctypes.c_size_t(0)
    operands = x.data_ptr(), *x.stride(), w.data_ptr(), *w.stride()
    _native.check(lib.hst_grouped_matmul_workspace(*operands, groups, rows, n, k, x.get_device(), ctypes.byref(size)))
    workspace = torch.full((size.value // 4,), -1, device="cuda", dtype=torch.int32)
    y, group_ends = torch.empty((rows, n), device="cuda", dtype=x.dtype), _ends(ends)
    _native.check(
        lib.hst_grouped_matmul(
            grouped._DTYPES[x.dtype], *operands, group_ends.data_ptr(), groups, y.data_ptr(), rows, n, k,
            workspace.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream,
        )
    )  # fmt: skip
    return y, _pieces(workspace, min(256, -(-rows // 32) * 32))


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ("kn", "nk"))
@pytest.mark.parametrize(
    "rows,ends,tiles",  # tiles of 224 and 256 rows, of 160 twice, of 32 twice
    ((456, [200, 200, 456], 2), (300, [0, 300], 2), (20, [3, 3, 20], 2)),
)
def test_more_tiles_than_pairs_are_cut(dtype: torch.dtype, layout: str, rows: int, ends: list[int], tiles: int) -> None:
    """Six tiles more than there are pairs, 66 K blocks deep: a pair takes a whole tile and parts of others."""
    cols = (_pairs() + 6) // tiles
    x, w, _ = _operands(rows, len(ends), 4168, 256 * cols - 8, dtype, layout, seed=rows)
    y, pieces = _cut_forward(x, w, ends)
    assert tiles * cols > _pairs() and pieces >= 2
    _check_forward(y, x, w, ends)
    assert torch.equal(y, grouped.grouped_matmul(x, w, _ends(ends)))


@gpu
@pytest.mark.parametrize("ends", ([300, 300, 4900], [4096], [700, 3600, 3601]))
def test_weight_gradients_cut_what_whole_tiles_leave(ends: list[int]) -> None:
    """Each pair takes whole tiles of every group first; the line of what remains is cut (over 40 K blocks deep)."""
    pairs = _pairs()
    k, n = 256 * (pairs + 16) // 9 // 256 * 256 + 8, 2056  # 11 x 9 tiles of a group with 74 pairs: one for each pair, 25 over
    assert pairs < -(-k // 256) * 9 < 2 * pairs
    x, _, dy = _operands(5000, 1, k, n, torch.bfloat16, "kn", seed=43)
    dw, pieces = _cut_weight_grad(x, dy, ends)
    assert pieces >= 2
    _check_weight_grad(dw, x, dy, ends)
    assert torch.equal(dw, grouped.grouped_weight_grad(x, dy, _ends(ends)))


def _rounding_excess(out: torch.Tensor, exact: torch.Tensor) -> float:
    """The RMS error of ``out`` over that of the exact values rounded once."""
    once = exact.to(out.dtype).double() - exact
    return ((out.double() - exact).square().mean() / once.square().mean()).sqrt().item()


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_pieces_are_joined_in_32_bits(dtype: torch.dtype) -> None:
    """The error of cut tiles is that of one rounding. FP32 sums of up to 6200 products, 16 at a time, are off by at most
    388 * 2^-23 = 2^-14.4 of the sum's size; one rounding of FP16 by 2^-11 / sqrt(3) or so (2^-12.3 on the average of
    the mantissas): the two together are at most 3% more, and less in BF16. Pieces rounded to 16 bits have as much error
    as the result's rounding, 41% more."""
    ends = [33, 33, 70]
    x, w, _ = _operands(70, 3, 4168, 520, dtype, "kn", seed=44)
    y, pieces = _cut_forward(x, w, ends)
    exact = torch.cat([x[s:e].double() @ w[i].double() for i, (s, e) in enumerate(_bounds(ends, 70))])
    assert pieces >= 2 and _rounding_excess(y, exact) <= 1.05
    ends = [0, 3100, 6200]
    x, _, dy = _operands(6200, 1, 264, 136, dtype, "kn", seed=45)
    dw, pieces = _cut_weight_grad(x, dy, ends)
    exact = torch.stack([x[s:e].double().T @ dy[s:e].double() for s, e in _bounds(ends, 6200)])
    assert pieces >= 2 and _rounding_excess(dw, exact) <= 1.05
    # The test tells the two apart: the same sums from pieces of 256 rows rounded to 16 bits.
    parts = [(x[s : s + 256].double().T @ dy[s : s + 256].double()).to(dtype) for s in range(0, 3100, 256)]
    rough = torch.stack(parts).double().sum(0).to(dtype)
    assert _rounding_excess(rough, x[:3100].double().T @ dy[:3100].double()) > 1.2


@gpu
def test_a_tile_left_over_by_the_pairs_is_cut_into_shares_worth_a_join() -> None:
    """A tile more than there are pairs, 64 K blocks deep: the one left over is cut into shares of four blocks, the
    least a share has, and not into one for each pair."""
    x, _, dy = _operands(4096, 1, 256 * (_pairs() + 1), 256, torch.bfloat16, "kn", seed=41)
    dw, pieces = _cut_weight_grad(x, dy, [4096])
    _check_weight_grad(dw, x, dy, [4096])
    assert pieces == 16


@gpu
def test_many_groups() -> None:
    groups = grouped.MAX_GROUPS
    counts = torch.randint(0, 4, (groups,), generator=torch.Generator().manual_seed(1))
    ends = torch.cumsum(counts, 0).tolist()
    x, w, dy = _operands(ends[-1] + 2, groups, 64, 40, torch.float16, "kn", seed=5)
    _check_forward(grouped.grouped_matmul(x, w, _ends(ends)), x, w, ends)
    _check_weight_grad(grouped.grouped_weight_grad(x, dy, _ends(ends)), x, dy, ends)


@gpu
@pytest.mark.parametrize("ends", ([50, 20, 90], [-5, 30, 1000], [2**31 - 1, 0, 10], [-1, -2, -3], [20, -(2**31), 60]))
def test_ends_out_of_order_or_range_are_clamped(ends: list[int]) -> None:
    x, w, dy = _operands(80, 3, 72, 48, torch.float16, "kn", seed=6)
    _check_forward(grouped.grouped_matmul(x, w, _ends(ends)), x, w, ends)
    _check_weight_grad(grouped.grouped_weight_grad(x, dy, _ends(ends)), x, dy, ends)


@gpu
@pytest.mark.parametrize("poison", (float("nan"), float("inf")))
def test_what_stands_in_other_rows_stays_out(poison: float) -> None:
    """Groups end inside 16-row steps and 64-row blocks; the rows of group 1 and past the last group hold
    NaN or infinity in both operands."""
    ends = [37, 37 + 75, 37 + 75 + 130]
    rows = ends[-1] + 9
    x, w, dy = _operands(rows, 3, 264, 136, torch.bfloat16, "kn", seed=7)
    bad = slice(ends[0], ends[1])
    clean = x.clone(), dy.clone()
    for t in (x, dy):
        t[bad] = poison
        t[ends[2] :] = poison
    y = grouped.grouped_matmul(x, w, _ends(ends))
    dw = grouped.grouped_weight_grad(x, dy, _ends(ends))
    assert not bool(torch.isfinite(y[bad]).any()) and not bool(torch.isfinite(dw[1]).any())
    y[bad] = 0
    assert bool(torch.isfinite(y).all()) and bool((y[ends[2] :] == 0).all())
    expected = grouped.grouped_weight_grad(*clean, _ends(ends))
    assert torch.equal(dw[0], expected[0]) and torch.equal(dw[2], expected[2])


@gpu
def test_strides_views_and_broadcasts() -> None:
    ends = [33, 70, 100]
    g = torch.Generator(device="cuda").manual_seed(8)
    wide = torch.randn((100, 3 * 80), generator=g, device="cuda").half()
    w = (torch.randn((3, 64, 80), generator=g, device="cuda") / 8).half()
    for x in (wide[:, 80:144], wide[:, 3:67], wide.T.contiguous().T[:, 8:72], wide[:, ::3][:, :64], wide[0, :64].expand(100, 64)):
        _check_forward(grouped.grouped_matmul(x, w, _ends(ends)), x, w, ends)
        _check_weight_grad(grouped.grouped_weight_grad(x, wide[:, :24], _ends(ends)), x, wide[:, :24], ends)
    x = wide[:, :64]
    for v in (w[1].expand(3, 64, 80), w[:, :, ::2], w.flip(0)[:, :, 8:40], w[:, :, 1:9], w.permute(1, 0, 2).contiguous().permute(1, 0, 2)):
        _check_forward(grouped.grouped_matmul(x, v, _ends(ends)), x, v, ends)
    # One weight broadcast to every expert and a loss that sums: both gradients are sums of shared entries.
    one = w[:1].detach().requires_grad_()
    leaf = x.detach().clone().requires_grad_()
    grouped.grouped_matmul(leaf, one.expand(3, 64, 80), _ends(ends)).sum().backward()
    exact = x.double().sum(0)[:, None].expand(64, 80)
    # Three rounded gradients of the experts, then their rounded sum: at most four half steps of the magnitudes.
    bound = 4 * 2.0**-11 * x.double().abs().sum(0)[:, None]
    assert bool(((one.grad[0].double() - exact).abs() <= bound).all())
    exact = w[0].double().sum(1)
    _assert_close(leaf.grad, exact.expand(100, 64), w[0].double().abs().sum(1).expand(100, 64), 80)


@gpu
def test_empty_extents() -> None:
    ends = _ends([2, 4])
    x, w, dy = _operands(4, 2, 16, 24, torch.float16, "kn", seed=9)
    assert grouped.grouped_matmul(x[:0], w, ends).shape == (0, 24)
    assert grouped.grouped_matmul(x, w[:, :, :0], ends).shape == (4, 0)
    assert bool((grouped.grouped_matmul(x[:, :0], w[:, :0], ends) == 0).all())
    assert bool((grouped.grouped_weight_grad(x[:0], dy[:0], ends) == 0).all())
    assert grouped.grouped_weight_grad(x[:, :0], dy, ends).shape == (2, 0, 24)


@gpu
@pytest.mark.parametrize("rows,k,n", ((0, 16, 24), (4, 0, 24), (4, 16, 0)))
def test_gradients_of_empty_extents(rows: int, k: int, n: int) -> None:
    x, w, dy = _operands(rows, 2, k, n, torch.float16, "kn", seed=46)
    x.requires_grad_()
    w.requires_grad_()
    y = grouped.grouped_matmul(x, w, _ends([2, 4]))
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert y.shape == (rows, n) and dx.shape == x.shape and dw.shape == w.shape
    for t in (y, dx, dw):
        assert bool((t == 0).all())


@gpu
def test_gradients_match_differences() -> None:
    """y is linear in x and in w, so (Y(x + d) - Y(x - d)) / 2 is the derivative along d exactly; Y in 64 bits."""
    ends = [19, 19, 83]
    x, w, dy = _operands(90, 3, 96, 56, torch.float16, "nk", seed=10)
    x.requires_grad_()
    w = w.detach().requires_grad_()
    dx, dw = torch.autograd.grad(grouped.grouped_matmul(x, w, _ends(ends)), (x, w), dy)

    def loss(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
        parts = [(a[s:e] @ b[i] * dy[s:e].double()).sum() for i, (s, e) in enumerate(_bounds(ends, 90))]
        return torch.stack(parts).sum()

    xd, wd = x.detach().double(), w.detach().double()
    g = torch.Generator(device="cuda").manual_seed(11)
    for grad, size, along in (
        (dx, xd, lambda d: (loss(xd + d, wd) - loss(xd - d, wd)) / 2),
        (dw, wd, lambda d: (loss(xd, wd + d) - loss(xd, wd - d)) / 2),
    ):
        d = torch.randn(size.shape, generator=g, device="cuda", dtype=torch.float64)
        # Every entry of the gradient is off by its rounding, 2^-11, and FP32 sums well below that.
        slack = (2.0**-10 * grad.double().abs() * d.abs()).sum() + 1e-3
        assert abs((grad.double() * d).sum() - along(d)) <= slack


@gpu
def test_only_the_gradients_asked_for_and_no_second_derivative() -> None:
    ends = _ends([4, 9])
    x, w, dy = _operands(9, 2, 32, 16, torch.float16, "kn", seed=12)
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(grouped.grouped_matmul(leaf, w, ends), (leaf,), dy)
    _check_forward(dx, dy, w.transpose(1, 2), [4, 9])
    leaf = w.clone().requires_grad_()
    grouped.grouped_matmul(x, leaf, ends).backward(dy)
    _check_weight_grad(leaf.grad, x, dy, [4, 9])
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(grouped.grouped_matmul(leaf, w, ends), (leaf,), dy, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
    with pytest.raises(ValueError, match="no gradient"):
        grouped.grouped_weight_grad(leaf, dy, ends)


@gpu
def test_a_frozen_operand_keeps_the_other_out_of_the_graph() -> None:
    ends = _ends([4, 9])
    x, w, _ = _operands(9, 2, 32, 16, torch.float16, "kn", seed=13)

    def saved(x: torch.Tensor, w: torch.Tensor) -> set[int]:
        kept: set[int] = set()

        def keep(t: torch.Tensor) -> torch.Tensor:
            kept.add(t.data_ptr())
            return t

        with torch.autograd.graph.saved_tensors_hooks(keep, lambda t: t):
            grouped.grouped_matmul(x, w, ends)
        return kept

    leaf_x, leaf_w = x.clone().requires_grad_(), w.clone().requires_grad_()
    assert saved(leaf_x, w) == {w.data_ptr(), ends.data_ptr()}
    assert saved(x, leaf_w) == {x.data_ptr(), ends.data_ptr()}
    assert saved(leaf_x, leaf_w) == {leaf_x.data_ptr(), leaf_w.data_ptr(), ends.data_ptr()}


@gpu
@pytest.mark.parametrize("moved", (lambda t: t.cpu(), lambda t: t.float()))
def test_what_a_saved_tensors_hook_gives_back_is_checked(moved) -> None:  # type: ignore[no-untyped-def]
    x, w, dy = _operands(9, 2, 32, 16, torch.float16, "kn", seed=47)
    for frozen_x in (False, True):
        leaf_x, leaf_w = x.clone().requires_grad_(not frozen_x), w.clone().requires_grad_(frozen_x)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, moved):
            y = grouped.grouped_matmul(leaf_x, leaf_w, _ends([4, 9]))
        with pytest.raises(ValueError):
            y.backward(dy)


@gpu
def test_bad_arguments_are_rejected() -> None:
    x, w, dy = _operands(9, 2, 32, 16, torch.float16, "kn", seed=13)
    ends = _ends([4, 9])
    for args, message in (
        ((x.float(), w.float(), ends), "float16 or torch.bfloat16"),
        ((x, w.bfloat16(), ends), "float16 or torch.bfloat16"),
        ((x, w, ends[:1]), "one entry"),
        ((x, w, ends.long()), "int32"),
        ((x, w, ends.cpu()), "on the device"),
        ((x, w, _ends([4, 0, 9, 0])[::2]), "contiguous"),
        ((x, w[:0], ends[:0]), "1 to 1024"),
    ):
        with pytest.raises(ValueError, match=message):
            grouped.grouped_matmul(*args)
    with pytest.raises(ValueError, match="1 to 1024"):
        grouped.grouped_weight_grad(x, dy, ends[:0])


# ------------------------------------------------------------------------------------------
# Streams, graphs, repeats
# ------------------------------------------------------------------------------------------


@gpu
def test_repeats_are_bitwise_identical() -> None:
    ends = _ends([130, 130, 391, 900])
    x, w, dy = _operands(900, 4, 520, 392, torch.bfloat16, "kn", seed=14)
    y, dw = grouped.grouped_matmul(x, w, ends), grouped.grouped_weight_grad(x, dy, ends)
    for _ in range(3):
        assert torch.equal(y, grouped.grouped_matmul(x, w, ends))
        assert torch.equal(dw, grouped.grouped_weight_grad(x, dy, ends))


@gpu
def test_two_streams_at_once() -> None:
    ends = [100, 300, 640]
    x, w, dy = _operands(640, 3, 2056, 520, torch.float16, "kn", seed=15)
    e = _ends(ends)
    expected = grouped.grouped_matmul(x, w, e), grouped.grouped_weight_grad(x, dy, e)
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    results = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            results.append((grouped.grouped_matmul(x, w, e), grouped.grouped_weight_grad(x, dy, e)))
    torch.cuda.synchronize()
    for y, dw in results:
        assert torch.equal(y, expected[0]) and torch.equal(dw, expected[1])


@gpu
@pytest.mark.parametrize("k", (264, 4168))
def test_captured_steps_follow_new_ends_and_inputs(k: int) -> None:
    """Two graphs of a training step, replayed in turn with other ends and inputs than they were captured with."""
    x, w, dy = _operands(300, 3, k, 200, torch.float16, "kn", seed=16)
    ends = _ends([100, 200, 300])
    x.requires_grad_()
    w.requires_grad_()

    def step():  # type: ignore[no-untyped-def]
        y = grouped.grouped_matmul(x, w, ends)
        return (y.detach(), *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outputs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outputs.append(step())
        graphs.append(graph)
    for i, values in enumerate(([0, 300, 300], [17, 18, 290], [300, 300, 300], [5, 5, 5])):
        with torch.no_grad():
            ends.copy_(_ends(values))
            x.mul_(-1)
        graphs[i % 2].replay()
        y, dx, dw = outputs[i % 2]
        _check_forward(y, x.detach(), w.detach(), values)
        _check_forward(dx, dy, w.detach().transpose(1, 2), values)
        _check_weight_grad(dw, x.detach(), dy, values)


@gpu
def test_outputs_past_32_bit_offsets() -> None:
    """70000 x 32776 outputs, 2.3e9 values: the last rows of the last group."""
    rows, n, k = 70_000, 32_776, 64
    x, w, _ = _operands(rows, 2, k, n, torch.float16, "nk", seed=19)
    y = grouped.grouped_matmul(x, w, _ends([33, rows - 3]))
    last = slice(rows - 40, rows - 3)
    _assert_close(y[last], x[last].double() @ w[1].double(), x[last].double().abs() @ w[1].double().abs(), k)
    assert bool((y[rows - 3 :] == 0).all())


@gpu
def test_the_workspace_is_checked_and_its_contents_do_not_matter() -> None:
    x, w, dy = _operands(120, 2, 4104, 264, torch.float16, "kn", seed=17)
    ends = _ends([50, 120])
    lib = _native.library()
    y = torch.empty((120, 264), device="cuda", dtype=torch.float16)

    def needed(k: int) -> int:
        size = ctypes.c_size_t(1)
        assert lib.hst_grouped_matmul_workspace(16, 4104, 1, 16, 4104 * 264, 264, 1, 2, 120, 264, k, 0, ctypes.byref(size)) == 0
        return size.value

    def call(workspace: torch.Tensor) -> int:
        return lib.hst_grouped_matmul(
            0, x.data_ptr(), 4104, 1, w.data_ptr(), 4104 * 264, 264, 1, ends.data_ptr(), 2, y.data_ptr(), 120, 264, 4104,
            workspace.data_ptr(), workspace.numel(), torch.cuda.current_stream().cuda_stream,
        )  # fmt: skip

    assert needed(520) == 0
    size = needed(4104)
    assert call(torch.empty(size - 1, device="cuda", dtype=torch.uint8)) == _native.HST_ERR_WORKSPACE
    for fill in (0, 255):
        assert call(torch.full((size,), fill, device="cuda", dtype=torch.uint8)) == _native.HST_OK
        _check_forward(y, x, w, [50, 120])
