"""The E4M3 quantisers and the block-scaled products (``blockscale``) against their formulas.

Quantisers: bit for bit against the same FP32 formula on the CPU. Products: against 64-bit sums of the
same 8-bit operands. A product of two E4M3 values has 8 significant bits, exact in FP32; a block's sum of 128
of them and the scaled sum over the blocks are off by at most one unit (2^-23) of the sum of magnitudes at
each step, the scale's own product by half of one: ``(128 + blocks + 2) * 2^-23 * sum |a||b| sa sb``, and the
output by ``eps / 2``.
"""

from __future__ import annotations

import ctypes
from concurrent.futures import ThreadPoolExecutor

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from heliostune_b200 import _native, blockscale, grouped
from tests.test_grouped import _bounds, _ends, _pairs, _pieces, _rounding_excess

gpu = pytest.mark.gpu
DTYPES = (torch.float16, torch.bfloat16)


@pytest.fixture(autouse=True)
def _status(request: pytest.FixtureRequest):  # type: ignore[no-untyped-def]
    yield
    if request.node.get_closest_marker("gpu") and torch.cuda.is_available():
        assert _native.status(torch.cuda.current_device()) == 0


def _quantize_cpu(x: torch.Tensor, tiles: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """The formula on the CPU, block by block."""
    x = x.detach().cpu().float()
    rows, cols = x.shape
    high = 128 if tiles else 1
    q = torch.empty((rows, cols), dtype=torch.float8_e4m3fn)
    scales = torch.empty((-(-rows // high), -(-cols // 128)))
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            at = (slice(i * high, (i + 1) * high), slice(j * 128, (j + 1) * 128))
            amax = x[at].abs().max().clamp(min=2.0**-100)
            most = torch.tensor(448.0)  # a tensor: torch takes 448.0 / amax as 448.0 * (1 / amax)
            scales[i, j] = amax / most
            q[at] = (x[at] * (most / amax)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q, scales


def _same_bits(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Equal values, NaN where the other has NaN."""
    a, b = a.detach().float().cpu(), b.detach().float().cpu()
    return a.shape == b.shape and bool(((a == b) | (a.isnan() & b.isnan())).all())


def _dequantize(q: torch.Tensor, s: torch.Tensor, tiles: bool) -> torch.Tensor:
    s = s.double().repeat_interleave(128, -1)[..., : q.shape[-1]]
    if tiles:
        s = s.repeat_interleave(128, -2)[..., : q.shape[-2], :]
    return q.double() * s


def _assert_product(y: torch.Tensor, a: torch.Tensor, b: torch.Tensor) -> None:
    """``y`` against ``a @ b.T`` for the dequantised operands in 64 bits."""
    exact, magnitude = a @ b.T, a.abs() @ b.abs().T
    half_step = torch.finfo(y.dtype).eps / 2
    slack = (128 + -(-a.shape[1] // 128) + 2) * 2.0**-23 * magnitude
    bound = half_step * exact.abs() + (1 + half_step) * slack + 2.0**-25
    error = (y.double() - exact).abs()
    assert y.shape == exact.shape
    assert bool((error <= bound).all()), ((error - bound).max().item(), error.max().item())


def _operands(rows: int, n: int, k: int, seed: int, groups: int = 0):  # type: ignore[no-untyped-def]
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, k), generator=g, device="cuda") * torch.exp(torch.randn((rows, 1), generator=g, device="cuda"))
    shape = (groups, n, k) if groups else (n, k)
    w = torch.randn(shape, generator=g, device="cuda") / k**0.5
    a, sa = blockscale.quantize_rows(x.bfloat16())
    b, sb = blockscale.quantize_tiles(w.bfloat16())
    return a, sa, b, sb


# ------------------------------------------------------------------------------------------
# Refusals, before any CUDA work
# ------------------------------------------------------------------------------------------


def test_inputs_are_checked_before_any_cuda_work() -> None:
    a = torch.zeros((4, 128), dtype=torch.float8_e4m3fn)
    s = torch.zeros((4, 1))
    with pytest.raises(ValueError, match=r"a \[T, K\]"):
        blockscale.matmul_blockscaled(a[0], s, a, s[:1])
    with pytest.raises(ValueError, match=r"a \[T, K\]"):
        blockscale.matmul_blockscaled(a, s, a, s[:1], torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="incompatible shapes"):
        blockscale.matmul_blockscaled(a, s, a[:, :64], s[:1])
    with pytest.raises(ValueError, match="same CUDA device"):
        blockscale.matmul_blockscaled(a, s, a, s[:1])
    with pytest.raises(ValueError, match=r"x \[T, K\]"):
        blockscale.quantize_rows(s[0])
    with pytest.raises(ValueError, match="CUDA tensor"):
        blockscale.quantize_rows(s)
    with pytest.raises(ValueError, match=r"weight \[N, K\]"):
        blockscale.quantize_tiles(s[0])


def test_operands_with_a_forward_gradient_are_refused() -> None:
    a = torch.zeros((4, 128), dtype=torch.float8_e4m3fn)
    s = torch.zeros((4, 1))
    x = torch.zeros((4, 128), dtype=torch.float16)
    with forward_ad.dual_level():
        for quantize in (blockscale.quantize_rows, blockscale.quantize_tiles):
            with torch.no_grad(), pytest.raises(ValueError, match="no forward-mode gradient"):
                quantize(forward_ad.make_dual(x, x))
        for args in ((a, forward_ad.make_dual(s, s), a, s[:1]), (a, s, a, forward_ad.make_dual(s, s)[:1])):
            with pytest.raises(ValueError, match="no forward-mode gradient"):
                blockscale.matmul_blockscaled(*args)


def test_the_library_refuses_bad_calls_before_any_cuda_work() -> None:
    # In a thread of its own: the library keeps the last error of each.
    with ThreadPoolExecutor(1) as thread:
        thread.submit(_refused_calls).result()


def _refused_calls() -> None:
    _native.build_library()
    lib = _native.library()

    def scaled(out=0, a=16, sa=16, b=16, sb=16, ends=16, groups=2, y=16, rows=4, n=8, k=128):  # type: ignore[no-untyped-def]
        return lib.hst_matmul_blockscaled(
            out, a, k, 1, sa, 1, 1, b, n * k, k, 1, sb, 1, 1, 1, ends, groups, y, rows, n, k, None, 0, None
        )

    for kwargs, message in (
        ({"out": 3}, b"data type"),
        ({"groups": 0}, b"1 to 1024"),
        ({"ends": None}, b"ends are null"),
        ({"k": -1}, b"extents"),
        ({"a": None}, b"a or b is null"),
        ({"b": None}, b"a or b is null"),
        ({"sa": None}, b"scales"),
        ({"y": None}, b"y is null"),
        ({"sa": 18}, b"a_scales must be aligned to 4"),
        ({"sb": 18}, b"b_scales must be aligned to 4"),
        ({"ends": 18}, b"ends must be aligned to 4"),
        ({"y": 17}, b"y must be aligned to 2"),
    ):
        assert scaled(**kwargs) == _native.HST_ERR_INVALID, kwargs
        assert message in lib.hst_last_error(), kwargs

    def quantize(dtype=0, tiles=0, x=16, q=16, q_row=128, s=16, batch=1, rows=4, cols=128):  # type: ignore[no-untyped-def]
        return lib.hst_quantize_e4m3(dtype, tiles, x, 0, 128, 1, q, 0, q_row, s, 0, 1, 1, batch, rows, cols, None)

    for kwargs, message in (
        ({"dtype": 2}, b"data type"),
        ({"rows": -1}, b"extents"),
        ({"batch": 2}, b"one matrix"),
        ({"tiles": 1, "batch": 65536}, b"65535"),
        ({"x": None}, b"null"),
        ({"q_row": 127}, b"shorter"),
        ({"x": 17}, b"x must be aligned to 2"),
        ({"s": 18}, b"scales must be aligned to 4"),
    ):
        assert quantize(**kwargs) == _native.HST_ERR_INVALID, kwargs
        assert message in lib.hst_last_error(), kwargs
    assert quantize(rows=0) == _native.HST_OK


# ------------------------------------------------------------------------------------------
# Tracing
# ------------------------------------------------------------------------------------------


def _served(x: torch.Tensor, w: torch.Tensor, ends: torch.Tensor) -> torch.Tensor:
    return blockscale.matmul_blockscaled(*blockscale.quantize_rows(x), *blockscale.quantize_tiles(w), ends, out_dtype=torch.float16)


def test_tracing_records_the_operators() -> None:
    """On fake CUDA tensors: the operators are recorded, and their outputs' layouts are the kernels'."""
    with FakeTensorMode():
        x = torch.empty((9, 130), device="cuda", dtype=torch.float16)
        w = torch.empty((2, 200, 130), device="cuda", dtype=torch.float16)
        ends = torch.empty(2, device="cuda", dtype=torch.int32)
        traced = make_fx(_served)(x, w, ends)
        called = [node.target for node in traced.graph.nodes if node.op == "call_function"]
        ops = torch.ops.heliostune_b200
        assert [t for t in called if t in (ops.quantize_rows.default, ops.quantize_tiles.default, ops.matmul_blockscaled.default)] == [
            ops.quantize_rows.default, ops.quantize_tiles.default, ops.matmul_blockscaled.default,
        ]  # fmt: skip
        assert not any("empty" in str(t) for t in called)
        q, s = blockscale.quantize_rows(x)
        assert q.shape == (9, 130) and q.stride() == (144, 1) and s.shape == (9, 2) and s.stride() == (1, 9)
        q, s = blockscale.quantize_tiles(w)
        assert q.shape == (2, 200, 130) and q.stride() == (28800, 144, 1) and s.shape == (2, 2, 2) and s.is_contiguous()
        assert _served(x, w, ends).shape == (9, 200)


def test_transforms_are_refused() -> None:
    x = torch.zeros((4, 128), dtype=torch.float16)
    for quantize in (blockscale.quantize_rows, blockscale.quantize_tiles):
        for transformed in (lambda q=quantize: torch.func.jvp(q, (x,), (x,)), lambda q=quantize: torch.vmap(q)(x[None])):
            with pytest.raises(ValueError, match="torch.func's transforms"):
                transformed()


@gpu
def test_traced_programs_compute_what_they_recorded() -> None:
    g = torch.Generator(device="cuda").manual_seed(31)
    x, other = (torch.randn((90, 264), generator=g, device="cuda").half() for _ in range(2))
    w = torch.randn((3, 136, 264), generator=g, device="cuda").half()
    ends = _ends([19, 19, 83])
    expected = _served(other, w, ends)
    for program in (
        torch.jit.trace(_served, (x, w, ends)),
        make_fx(_served)(x, w, ends),
        make_fx(_served, tracing_mode="fake")(x, w, ends),
        torch.compile(_served, fullgraph=True, backend="aot_eager"),
    ):
        assert torch.equal(program(other, w, ends), expected)


# ------------------------------------------------------------------------------------------
# Quantisers
# ------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tiles", (False, True))
@pytest.mark.parametrize("rows,cols", ((1, 1), (1, 128), (3, 129), (128, 128), (130, 264), (257, 1000), (5, 4096), (129, 77)))
def test_quantisers_match_the_formula(dtype: torch.dtype, tiles: bool, rows: int, cols: int) -> None:
    g = torch.Generator(device="cuda").manual_seed(rows * cols)
    x = (torch.randn((rows, cols), generator=g, device="cuda") * torch.exp(2 * torch.randn((rows, 1), generator=g, device="cuda"))).to(dtype)
    q, s = (blockscale.quantize_tiles if tiles else blockscale.quantize_rows)(x)
    expected_q, expected_s = _quantize_cpu(x, tiles)
    assert q.dtype == torch.float8_e4m3fn and s.dtype == torch.float32
    assert _same_bits(s, expected_s) and _same_bits(q, expected_q)
    # And what they stand for: half a step of E4M3 (2^-4 of the value, or half of the least step, 2^-10, of the scale).
    exact = x.double()
    off = (_dequantize(q, s, tiles) - exact).abs()
    scale = _dequantize(torch.ones_like(exact), s, tiles)
    assert bool((off <= exact.abs() * 2.0**-4 * (1 + 1e-6) + scale * 2.0**-10 * (1 + 1e-6)).all())


@gpu
@pytest.mark.parametrize("tiles", (False, True))
@pytest.mark.parametrize("cols", (256, 250))  # vector and general loads
def test_quantisers_at_the_ends_of_the_range(tiles: bool, cols: int) -> None:
    quantize = blockscale.quantize_tiles if tiles else blockscale.quantize_rows
    for dtype in DTYPES:
        least = torch.finfo(dtype).smallest_normal
        for values in (
            [0.0], [-0.0], [least], [least / 4, 0.0], [torch.finfo(dtype).max], [1.0, -3.0, 448.0], [17.0, 0.0, 448.0, 18.0],
            [float("inf"), 1.0], [float("-inf"), float("nan")], [float("nan")], [1e-6, 5.0],
        ):  # fmt: skip
            x = torch.zeros((2, cols), device="cuda", dtype=dtype)
            x[0, : len(values)] = torch.tensor(values, dtype=dtype)
            x[1, 130 : 130 + len(values)] = torch.tensor(values, dtype=dtype)
            q, s = quantize(x)
            expected_q, expected_s = _quantize_cpu(x, tiles)
            # A maximum over a block with NaN is NaN in both.
            assert _same_bits(s, expected_s), (dtype, values)
            assert _same_bits(q, expected_q), (dtype, values)


@gpu
def test_quantisers_take_any_strides_and_stacks() -> None:
    g = torch.Generator(device="cuda").manual_seed(1)
    base = torch.randn((3, 200, 320), generator=g, device="cuda").half()
    for x in (base[0].T, base[1, ::2], base[1, :, ::3], base[0, :, 1:130], base[2, 5:6].expand(9, 320), base[:, 7, :]):
        for tiles, quantize in ((False, blockscale.quantize_rows), (True, blockscale.quantize_tiles)):
            q, s = quantize(x)
            expected_q, expected_s = _quantize_cpu(x, tiles)
            assert _same_bits(s, expected_s) and _same_bits(q, expected_q)
    for stack in (base, base.transpose(1, 2), base[:, ::2], base[:, :, 3:141]):
        q, s = blockscale.quantize_tiles(stack)
        for i in range(3):
            expected_q, expected_s = _quantize_cpu(stack[i], True)
            assert _same_bits(s[i], expected_s) and _same_bits(q[i], expected_q)
    for empty in (base[0, :0], base[0, :, :0]):
        for quantize in (blockscale.quantize_rows, blockscale.quantize_tiles):
            q, s = quantize(empty)
            assert q.shape == empty.shape and s.numel() == 0


# ------------------------------------------------------------------------------------------
# Products
# ------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("out_dtype", DTYPES)
@pytest.mark.parametrize("rows", (1, 2, 31, 33, 64, 65, 127, 128, 200, 256, 257, 600))
@pytest.mark.parametrize("n,k", ((128, 128), (136, 264), (520, 1040), (72, 4096), (1000, 16), (201, 4368)))
def test_dense(out_dtype: torch.dtype, rows: int, n: int, k: int) -> None:
    a, sa, b, sb = _operands(rows, n, k, seed=rows + n + k)
    y = blockscale.matmul_blockscaled(a, sa, b, sb, out_dtype=out_dtype)
    assert y.dtype == out_dtype
    _assert_product(y, _dequantize(a, sa, False), _dequantize(b, sb, True))


@gpu
@pytest.mark.parametrize("rows", (1, 40, 300))
@pytest.mark.parametrize("n,k", ((1, 1), (17, 13), (129, 129), (130, 1001)))
def test_extents_and_strides_that_tma_cannot_read(rows: int, n: int, k: int) -> None:
    a, sa, b, sb = _operands(rows, n, k, seed=rows + n + k)
    expected = _dequantize(a, sa, False), _dequantize(b, sb, True)
    forms = [(a, sa, b, sb), (a.contiguous(), sa.contiguous(), b.contiguous(), sb.T.contiguous().T)]
    wide = torch.zeros((rows, k + 7), device="cuda", dtype=torch.uint8)
    wide[:, 3 : 3 + k] = a.view(torch.uint8) if a.is_contiguous() else a.contiguous().view(torch.uint8)
    forms.append((wide.view(torch.float8_e4m3fn)[:, 3 : 3 + k], sa, b.T.contiguous().T, sb))
    spread = torch.zeros((rows * 2, sa.shape[1] * 3), device="cuda")
    spread[::2, ::3] = sa
    forms.append((a, spread[::2, ::3], b, sb))
    for form in forms:
        _assert_product(blockscale.matmul_blockscaled(*form), *expected)


@gpu
@pytest.mark.parametrize(
    "rows,ends",
    ((1, [0, 1]), (9, [3, 3, 8]), (96, [40, 41, 96]), (300, [0, 255, 255, 300]), (700, [256, 513, 700]), (40, [0, 0, 0]), (1111, [600, 600, 1100])),
)
@pytest.mark.parametrize("n,k", ((136, 264), (520, 1040), (264, 2192), (264, 4368)))  # the last: tiles are cut
def test_grouped(rows: int, ends: list[int], n: int, k: int) -> None:
    a, sa, b, sb = _operands(rows, n, k, seed=rows + n, groups=len(ends))
    y = blockscale.matmul_blockscaled(a, sa, b, sb, _ends(ends), out_dtype=torch.float16)
    last = 0
    da, db = _dequantize(a, sa, False), _dequantize(b, sb, True)
    for e, (start, end) in enumerate(_bounds(ends, rows)):
        _assert_product(y[start:end], da[start:end], db[e])
        last = end
    assert bool((y[last:] == 0).all())


def _cut_product(a, sa, b, sb, ends: list[int] | None, out_dtype: torch.dtype) -> tuple[torch.Tensor, int]:  # type: ignore[no-untyped-def]
    """The product over the C ABI, and into how many FP32 pieces its cut tiles were written."""
    lib, (rows, k), n, groups = _native.library(), a.shape, b.shape[-2], 1 if ends is None else len(ends)
    lead = (0,) if ends is None else ()
    operands = b.data_ptr(), *lead, *b.stride()
    size = ctypes.c_size_t(0)
    _native.check(lib.hst_matmul_blockscaled_workspace(a.data_ptr(), *a.stride(), *operands, groups, rows, n, k, 0, ctypes.byref(size)))
    workspace = torch.full((size.value // 4,), -1, device="cuda", dtype=torch.int32)
    y, group_ends = torch.empty((rows, n), device="cuda", dtype=out_dtype), None if ends is None else _ends(ends)
    _native.check(
        lib.hst_matmul_blockscaled(
            grouped._DTYPES[out_dtype], a.data_ptr(), *a.stride(), sa.data_ptr(), *sa.stride(), *operands, sb.data_ptr(), *lead,
            *sb.stride(), None if ends is None else group_ends.data_ptr(), groups, y.data_ptr(), rows, n, k,
            workspace.data_ptr(), size.value, torch.cuda.current_stream().cuda_stream,
        )
    )  # fmt: skip
    width = min(64, -(-rows // 32) * 32) if rows <= max(64, 8 * groups) else 256
    return y, _pieces(workspace, width)


@gpu
@pytest.mark.parametrize("rows", (20, 40, 300))  # widths of 32 and 64 with few rows, and the wide form
@pytest.mark.parametrize("blocks,cut", ((40, True), (5, False)))
def test_more_tiles_than_pairs(rows: int, blocks: int, cut: bool) -> None:
    """Six tiles more than there are pairs, cut where they are deep; shallow ones stay whole, two for some pairs."""
    cols = (_pairs() + 6) // (2 if rows == 300 else 1)
    a, sa, b, sb = _operands(rows, 256 * cols - 16, 128 * blocks - 16, seed=rows + blocks)
    y, pieces = _cut_product(a, sa, b, sb, None, torch.float16)
    assert pieces >= 2 if cut else pieces == 0
    _assert_product(y, _dequantize(a, sa, False), _dequantize(b, sb, True))
    assert torch.equal(y, blockscale.matmul_blockscaled(a, sa, b, sb, out_dtype=torch.float16))


@gpu
@pytest.mark.parametrize("n,k", ((136, 264), (1032, 4368)))
@pytest.mark.parametrize(
    "rows,ends",
    (
        (340, [0, 200, 200, 200, 330, 331, 331, 331]),
        (500, [1, 66, 130, 386, 500, 500, 500, 500]),  # 1, 65, 64, 256 and 114 rows
        (2000, [1, 65, 130, 386, 643, 963, 1284, 2000]),  # 1, 64, 65, 256, 257, 320, 321 and 716 rows
    ),
)
def test_groups_of_many_rows(rows: int, ends: list[int], n: int, k: int) -> None:
    a, sa, b, sb = _operands(rows, n, k, seed=rows + n, groups=len(ends))
    y = blockscale.matmul_blockscaled(a, sa, b, sb, _ends(ends))
    da, db = _dequantize(a, sa, False), _dequantize(b, sb, True)
    for e, (start, end) in enumerate(_bounds(ends, rows)):
        _assert_product(y[start:end], da[start:end], db[e])
    assert bool((y[ends[-1] :] == 0).all())


@gpu
@pytest.mark.parametrize("n,k", ((136, 264), (1032, 4368)))
def test_groups_of_many_rows_among_few(n: int, k: int) -> None:
    """270 rows over 40 groups, so in the few-rows form: groups of 200 (tiles of 64, 64, 64 and 32), 65 and 1 rows."""
    ends = [1] * 5 + [201] * 20 + [266] * 10 + [267] * 5
    a, sa, b, sb = _operands(270, n, k, seed=n, groups=40)
    y = blockscale.matmul_blockscaled(a, sa, b, sb, _ends(ends))
    da, db = _dequantize(a, sa, False), _dequantize(b, sb, True)
    for e, (start, end) in enumerate(_bounds(ends, 270)):
        _assert_product(y[start:end], da[start:end], db[e])
    assert bool((y[267:] == 0).all())


@gpu
@pytest.mark.parametrize(
    "rows,groups,width", ((64, 1, 64), (65, 1, 256), (64, 8, 64), (65, 8, 256), (256, 32, 64), (257, 32, 256), (2000, 32, 256))
)
def test_the_form_goes_by_the_rows_of_all_groups(rows: int, groups: int, width: int) -> None:
    """2000 rows over 32 groups may be 2000 of one: 64 rows a tile would read its weight 32 times."""
    size = ctypes.c_size_t(0)
    n, k = 25600, 6400  # deep, and tiles enough for every pair
    status = _native.library().hst_matmul_blockscaled_workspace(16, k, 1, 16, n * k, k, 1, groups, rows, n, k, 0, ctypes.byref(size))
    assert status == _native.HST_OK and size.value == _pairs() * 4 * 128 * width * 4


@gpu
def test_hundreds_of_groups() -> None:
    groups = 300
    counts = torch.randint(0, 4, (groups,), generator=torch.Generator().manual_seed(7))
    counts[123] = 200
    ends = torch.cumsum(counts, 0).tolist()
    a, sa, b, sb = _operands(ends[-1] + 3, 136, 264, seed=8, groups=groups)
    y = blockscale.matmul_blockscaled(a, sa, b, sb, _ends(ends))
    da, db = _dequantize(a, sa, False), _dequantize(b, sb, True)
    for e, (start, end) in enumerate(_bounds(ends, a.shape[0])):
        _assert_product(y[start:end], da[start:end], db[e])
    assert bool((y[ends[-1] :] == 0).all())


@gpu
@pytest.mark.parametrize("rows", (3, 300))
def test_pieces_are_joined_in_32_bits(rows: int) -> None:
    """As for the 16-bit products: the error of cut tiles is that of one rounding."""
    a, sa, b, sb = _operands(rows, 520, 5120, seed=rows)
    y, pieces = _cut_product(a, sa, b, sb, None, torch.float16)
    assert pieces >= 2
    assert _rounding_excess(y, _dequantize(a, sa, False) @ _dequantize(b, sb, True).T) <= 1.05


@gpu
@pytest.mark.parametrize("rows", (40, 400))
def test_nan_and_infinity_stay_in_their_rows_and_columns(rows: int) -> None:
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn((rows, 300), generator=g, device="cuda").bfloat16()
    w = (torch.randn((200, 300), generator=g, device="cuda") / 17).bfloat16()
    x[3, 140] = float("inf")
    x[rows - 1, 299] = float("nan")
    w[150, 7] = float("nan")
    a, sa = blockscale.quantize_rows(x)
    b, sb = blockscale.quantize_tiles(w)
    y = blockscale.matmul_blockscaled(a, sa, b, sb)
    bad = torch.zeros((rows, 200), dtype=torch.bool, device="cuda")
    bad[3] = bad[rows - 1] = True
    bad[:, 128:] = True  # the scale of the tile that holds the NaN
    assert torch.equal(~torch.isfinite(y), bad)


@gpu
@pytest.mark.parametrize("rows", (20, 40, 400))
@pytest.mark.parametrize("size", (130, -142))
def test_scales_whose_product_leaves_the_range_of_fp32(rows: int, size: int) -> None:
    """Scales of about 2^(size / 2) each: their product is no normal FP32 value, what they scale is. Where it is too
    large, the last block, of zeros in ``a``, has the largest scales there are. One row's scales are zero."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    n, k = 200, 384

    def values(*shape: int) -> torch.Tensor:
        if size > 0:  # multiples of E4M3's least value: block sums of a few 2^-18
            v = torch.randint(-1, 2, shape, generator=g, device="cuda") * 2.0**-9
        else:
            v = (torch.randn(shape, generator=g, device="cuda") * 200).clamp(-448, 448)
        return v.to(torch.float8_e4m3fn)

    def scales(*shape: int) -> torch.Tensor:
        return (1 + torch.rand(shape, generator=g, device="cuda")) * 2.0 ** (size / 2)

    a, b, sa, sb = values(rows, k), values(n, k), scales(rows, 3), scales(2, 3)
    if size > 0:
        a[:, 256:] = 0
        sa[:, 2] = sb[:, 2] = torch.finfo(torch.float32).max
    sa[7] = 0
    y = blockscale.matmul_blockscaled(a, sa, b, sb)
    assert bool(torch.isfinite(y).all()) and bool((y[7] == 0).all())
    da, db = _dequantize(a, sa, False), _dequantize(b, sb, True)
    exact, magnitude = da @ db.T, da.abs() @ db.abs().T
    # As above, with one more rounding of each block's sum, and half a subnormal step of BF16 (2^-133).
    bound = 2.0**-8 * exact.abs() + (1 + 2.0**-8) * (128 + 3 + 3) * 2.0**-23 * magnitude + 2.0**-134
    assert bool(((y.double() - exact).abs() <= bound).all())


@gpu
def test_groups_keep_to_their_rows_next_to_nan() -> None:
    ends = [37, 120, 250]
    a, sa, b, sb = _operands(260, 136, 264, seed=3, groups=3)
    clean = blockscale.matmul_blockscaled(a, sa, b, sb, _ends(ends))
    sa = sa.clone()
    sa[37:120] = float("nan")
    sa[250:] = float("nan")
    y = blockscale.matmul_blockscaled(a, sa, b, sb, _ends(ends))
    assert bool(torch.isnan(y[37:120]).all())
    y[37:120] = clean[37:120]
    assert torch.equal(y, clean)


@gpu
def test_empty_extents_and_refusals() -> None:
    a, sa, b, sb = _operands(8, 136, 256, seed=4)
    assert blockscale.matmul_blockscaled(a[:0], sa[:0], b, sb).shape == (0, 136)
    assert blockscale.matmul_blockscaled(a, sa, b[:0], sb[:0]).shape == (8, 0)
    assert bool((blockscale.matmul_blockscaled(a[:, :0], sa[:, :0], b[:, :0], sb[:, :0]) == 0).all())
    for args, message in (
        ((a.float(), sa, b, sb), "float8_e4m3fn"),
        ((a, sa[:, :1], b, sb), "a_scales must have shape"),
        ((a, sa, b, sb[:1]), "b_scales must have shape"),
        ((a, sa.double(), b, sb), "float32"),
        ((a, sa.cpu(), b, sb), "on the device"),
        ((a, sa.clone().requires_grad_(), b, sb), "no gradient"),
    ):
        with pytest.raises(ValueError, match=message):
            blockscale.matmul_blockscaled(*args)
    with pytest.raises(ValueError, match="out_dtype"):
        blockscale.matmul_blockscaled(a, sa, b, sb, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="no gradient"):
        blockscale.quantize_rows(torch.zeros((2, 128), device="cuda", dtype=torch.float16, requires_grad=True))
    with pytest.raises(ValueError, match="float16 or torch.bfloat16"):
        blockscale.quantize_tiles(torch.zeros((2, 128), device="cuda"))


@gpu
@pytest.mark.parametrize("rows", (3, 700))
@pytest.mark.parametrize("k", (1040, 2320))
def test_captured_and_concurrent_calls(rows: int, k: int) -> None:
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((rows, k), generator=g, device="cuda").bfloat16()
    w = (torch.randn((520, k), generator=g, device="cuda") / 32).bfloat16()
    b, sb = blockscale.quantize_tiles(w)

    def step() -> torch.Tensor:
        return blockscale.matmul_blockscaled(*blockscale.quantize_rows(x), b, sb)

    expected = step()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    results = []
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            results.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(expected, y) for y in results)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step()
    for _ in range(3):
        x.mul_(-1.5)
        graph.replay()
        assert torch.equal(y, step())


# ------------------------------------------------------------------------------------------
# Together
# ------------------------------------------------------------------------------------------


@gpu
def test_an_expert_layer_trained_in_16_bits_and_served_in_8() -> None:
    """Tokens routed to two of four experts: the layer in 16 bits with its gradients, then the same weights
    quantised. Against the 64-bit layer; the 8-bit one against the 64-bit layer of its own operands."""
    g = torch.Generator(device="cuda").manual_seed(6)
    tokens, experts, hidden, inner = 70, 4, 264, 392
    x = torch.randn((tokens, hidden), generator=g, device="cuda").bfloat16().requires_grad_()
    up = (torch.randn((experts, inner, hidden), generator=g, device="cuda") / hidden**0.5).bfloat16().requires_grad_()
    down = (torch.randn((experts, hidden, inner), generator=g, device="cuda") / inner**0.5).bfloat16().requires_grad_()
    choice = torch.randn((tokens, experts), generator=g, device="cuda").topk(2).indices.reshape(-1)
    order = torch.argsort(choice, stable=True)
    ends = torch.cumsum(torch.bincount(choice, minlength=experts), 0).to(torch.int32)
    source = order // 2
    bounds = _bounds(ends.tolist(), 2 * tokens)

    def layer(rows, first, second, product):  # type: ignore[no-untyped-def]
        h = torch.relu(product(rows, first))
        return torch.zeros((tokens, hidden), device="cuda", dtype=h.dtype).index_add(0, source, product(h, second))

    y = layer(x[source], up, down, lambda a, w: grouped.grouped_matmul(a, w.transpose(1, 2), ends))
    y.sum().backward()
    leaves = [t.detach().double().requires_grad_() for t in (x, up, down)]
    exact = layer(leaves[0][source], leaves[1], leaves[2], lambda a, w: torch.cat([a[s:e] @ w[i].T for i, (s, e) in enumerate(bounds)]))
    exact.sum().backward()
    # Norms: each of the layer's BF16 roundings is off by at most 2^-8 of its value; a value passes at most
    # three of them forward (h, product, sum) and five on the way back, and where a rounding moves h across zero, relu's
    # share follows continuously.
    for got, want, steps in ((y, exact, 3), *((a.grad, b.grad, 8) for a, b in zip((x, up, down), leaves, strict=True))):
        assert (got.double() - want).norm() <= steps * 2.0**-8 * want.norm()

    w8 = [blockscale.quantize_tiles(w.detach()) for w in (up, down)]
    with torch.no_grad():
        rows = x.detach()[source]
        a, sa = blockscale.quantize_rows(rows)
        h = blockscale.matmul_blockscaled(a, sa, *w8[0], ends)
        for i, (s, e) in enumerate(bounds):
            _assert_product(h[s:e], _dequantize(a, sa, False)[s:e], _dequantize(*w8[0], True)[i])
        a, sa = blockscale.quantize_rows(torch.relu(h))
        out = blockscale.matmul_blockscaled(a, sa, *w8[1], ends)
        for i, (s, e) in enumerate(bounds):
            _assert_product(out[s:e], _dequantize(a, sa, False)[s:e], _dequantize(*w8[1], True)[i])
        served = torch.zeros((tokens, hidden), device="cuda").index_add(0, source, out.float())
    # Four operands rounded to E4M3 (2^-4 of the value each at most, independent signs).
    assert (served.double() - exact).norm() <= 4 * 2.0**-4 * exact.norm()
