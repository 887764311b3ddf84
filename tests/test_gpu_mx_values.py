"""Values of the microscaled operators where they are easily lost: sums that cancel, results of every type out of every kernel, the activations' tails,
values next to a border between two codes, row scales, and what lies beside a result.

Tolerances, u = 2^-24, half(t) = torch.finfo(t).eps / 2.
  sums          products of e2m1 / e4m3 values and powers of two are exact in fp32; a K step of 128 adds at most 128 roundings and each further step
                one, none larger than u times the products' magnitudes, in whatever order and for whatever type of result; then two fp32 roundings
                (bias, residual) and one to the result's type
                (test_gpu_mx_ops.py allows e4m3 rows with 16-bit results, and the norm's codes, more than they now need)
  activations   of an exact argument, relative.  16-bit results: their own half step and 2^-14 (a fit good to 2^-15.1, and exp2's argument,
                at most 128 with two roundings of u: 256 u ln 2 < 2^-16).  fp32: 16 u (exp2 and rcp 2 u each, the fit and its
                eight steps 6 u, four products and sums 4 u; the exponential's argument is carried in two floats).  Results below 2^-120 may be
                lost to subnormal numbers on the way
"""
import numpy as np
import pytest
import torch

from clip_assisted_data_labeling_amd import _lib, mx_ops as mx
from oracle import mx_oracle as ora

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
DTYPES = [BF16, F16, F32]


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _lay_out(codes, scale, fmt, cols, gpu):
    return mx.MXTensor(torch.from_numpy(ora.pack(codes, fmt)).to(gpu), torch.from_numpy(scale).to(gpu), fmt, cols)


def _coded(rows, cols, fmt, seed, gpu, low, high):
    """Any codes, scales 2^low .. 2^high, zero behind the columns; and the values on the GPU in 64 bits."""
    r = np.random.RandomState(seed)
    kp = ora.padded(cols)
    codes = r.randint(0, 16 if fmt == "e2m1" else 256, (rows, kp)).astype(np.uint8)
    if fmt == "e4m3":
        codes[(codes & 127) == 127] = 0                          # its NaN codes
    codes[:, cols:] = 0
    scale = r.randint(127 + low, 128 + high, (rows, kp // 32)).astype(np.uint8)
    return _lay_out(codes, scale, fmt, cols, gpu), torch.from_numpy(ora.values(codes, scale, fmt, cols)).to(gpu)


def _operands(m, n, k, fmt, gpu):
    """Rows and weights whose sums are a few units wide."""
    a, av = _coded(m, k, fmt, m + k, gpu, *((-10, -7) if fmt == "e4m3" else (-3, 0)))
    w, wv = _coded(n, k, "e2m1", n + k, gpu, -6, -3)
    return a, av, w, wv


def _activate(u, act):
    if act == "gelu":
        return u * torch.special.erfc(-u / 2 ** 0.5) / 2
    return u / (1 + torch.exp(-1.702 * u)) if act == "quick_gelu" else u


def _act_error(want, dtype):
    return (16 * U if dtype == F32 else 2.0 ** -14) * want.abs() + 2.0 ** -120


def _check(y, u, pre, act, residual, dtype, what):
    """u: the sums with their bias in 64 bits, good to `pre`."""
    want = _activate(u, act)
    tol = pre if act is None else 1.13 * pre + _act_error(want, dtype)
    if residual is not None:
        want = want + residual.double()
    tol = tol + 2 * U * want.abs()
    tol = tol + _half(dtype) * (want.abs() + tol) + float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    off = (y.double() - want).abs() - tol
    assert y.dtype == dtype and y.shape == want.shape and not torch.isnan(y).any()
    assert not (off > 0).any(), (what, off.max().item(), np.unravel_index(int(off.argmax()), tuple(off.shape)))


# One shape or two -- whole tiles, ragged ones -- for each kernel of a product: the few-row kernel (up to 16 rows, or one or two workgroups a CU of 64 rows x 16
# columns), 64 x 64 tiles (a few hundred), 128 x 128 in four stages (up to 256 of them), 128 x 128 in two, 256 x 256 (from 256 of them on; rows that
# would leave a last round nearly empty go to a smaller kernel), and those of a long K
KERNELS = {"few-1": (1, 1000, 700), "few-16": (16, 1664, 1281), "few-64": (61, 500, 1000), "few-columns": (300, 17, 600),
           "tiles-64": (320, 1024, 384), "tiles-64-ragged": (301, 1101, 200),
           "tiles-128-deep": (2048, 1664, 640), "tiles-128-deep-ragged": (2885, 1003, 601),
           "tiles-128": (2816, 2944, 384), "tiles-128-ragged": (2900, 3001, 200),
           "tiles-256": (4096, 4096, 256), "tiles-256-ragged": (5300, 4090, 300), "tiles-256-and-few": (4100, 4090, 300), "tiles-256-and-128": (11000, 1664, 130),
           "tiles-256-long": (4096, 4096, 1664), "tiles-256-long-ragged": (5300, 4104, 1801)}


# ------------------------------------------------------------------------------------------ sums
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kernel", KERNELS)
def test_sums_of_e4m3_rows_whose_large_products_cancel(gpu, kernel, dtype):
    """Two of eight neighbouring columns hold +-448 against the same weight 6, the six others make the result."""
    m, n, k = KERNELS[kernel]
    k = ora.padded(k)
    r = np.random.RandomState(m)
    codes = (0x10 + r.randint(0, 8, (m, k))).astype(np.uint8)                     # 2^-5 .. 2^-4, positive
    codes[:, 2::8], codes[:, 5::8] = 0x7E, 0xFE                                   # +-448
    wcodes = r.randint(2, 4, (n, k)).astype(np.uint8)                             # 1, 1.5
    wcodes[:, 2::8] = wcodes[:, 5::8] = 7                                         # 6
    ones = lambda rows: np.full((rows, k // 32), 127, np.uint8)                   # noqa: E731
    a, w = _lay_out(codes, ones(m), "e4m3", k, gpu), _lay_out(wcodes, ones(n), "e2m1", k, gpu)
    av, wv = (torch.from_numpy(ora.values(c, s, f, k)).to(gpu) for c, s, f in ((codes, ones(m), "e4m3"), (wcodes, ones(n), "e2m1")))
    u, size = av @ wv.t().contiguous(), av.abs() @ wv.abs().t().contiguous()
    y = mx.linear(a, w, out_dtype=dtype)
    _check(y, u, (128 + k // 128) * U * size, None, None, dtype, kernel)
    if m <= 16:                                                                   # and from values, which are these codes
        x = av.to(F32)
        assert torch.equal(mx.dequantize(mx.quantize(x, "e4m3"), F32), x)
        _check(mx.linear(x, w, out_dtype=dtype), u, (128 + k // 128) * U * size, None, None, dtype, kernel)


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_sums_whose_large_products_cancel_far_apart(gpu, kernel, fmt):
    """Blocks 2^12 times the others cancel against another block of the same or of another K step."""
    m, n, k = KERNELS[kernel]
    k = max(256, ora.padded(k))
    r = np.random.RandomState(n)
    top, sign = (8, 8) if fmt == "e2m1" else (128, 128)
    codes = r.randint(0, top // 2, (m, k)).astype(np.uint8)
    scale, wscale = np.full((m, k // 32), 127, np.uint8), np.full((n, k // 32), 127, np.uint8)
    wcodes = r.randint(0, 16, (n, k)).astype(np.uint8)
    for at, to in ((0, 2), (1, 5)):                                               # of one step, of two
        codes[:, to * 32:to * 32 + 32] = codes[:, at * 32:at * 32 + 32] | sign
        wcodes[:, to * 32:to * 32 + 32] = wcodes[:, at * 32:at * 32 + 32]
        scale[:, [at, to]] += 12
    a, w = _lay_out(codes, scale, fmt, k, gpu), _lay_out(wcodes, wscale, "e2m1", k, gpu)
    av, wv = (torch.from_numpy(ora.values(c, s, f, k)).to(gpu) for c, s, f in ((codes, scale, fmt), (wcodes, wscale, "e2m1")))
    u, size = av @ wv.t().contiguous(), av.abs() @ wv.abs().t().contiguous()
    for dtype in DTYPES:
        _check(mx.linear(a, w, out_dtype=dtype), u, (128 + k // 128) * U * size, None, None, dtype, kernel)


@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_codes_of_e4m3_rows_are_in_their_own_row_only(gpu, kernel):
    m, n, k = KERNELS[kernel]
    a, _, w, _ = _operands(m, n, k, "e4m3", gpu)
    a.data[m // 2, k - 1] = 0x7F
    a.data[m - 1, 3] = 0xFF
    want = torch.zeros(m, n, dtype=torch.bool, device=gpu)
    want[m // 2] = want[m - 1] = True
    for dtype in DTYPES:
        assert torch.equal(torch.isnan(mx.linear(a, w, out_dtype=dtype)), want)


# ------------------------------------------------------------------------------------------ every kernel, every type of result
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_every_kernel_every_type_and_epilogue(gpu, kernel, fmt):
    m, n, k = KERNELS[kernel]
    a, av, w, wv = _operands(m, n, k, fmt, gpu)
    g = torch.Generator().manual_seed(k)
    bias = (3 * torch.randn(n, generator=g)).to(gpu)
    res = (50 * torch.randn(m, n, generator=g)).to(gpu)
    u, size = av @ wv.t().contiguous(), av.abs() @ wv.abs().t().contiguous()
    with_bias, count = u + bias.double(), 128 + ora.padded(k) // 128 + 2
    pre = count * U * (size + bias.double().abs())
    for dtype in DTYPES:
        _check(mx.linear(a, w, out_dtype=dtype), u, count * U * size, None, None, dtype, dtype)
        for act in (None, "gelu", "quick_gelu"):
            _check(mx.linear(a, w, bias=bias, act=act, out_dtype=dtype), with_bias, pre, act, None, dtype, (dtype, act))
        r = res.to(dtype)
        _check(mx.linear(a, w, bias=bias, residual=r, out_dtype=dtype), with_bias, pre, None, r, dtype, (dtype, "residual"))


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(301, 1101, 200), (2885, 1003, 601), (4100, 4090, 300)])
def test_values_through_tiles_are_quantize_and_linear(gpu, m, n, k, dtype, fmt):
    _, _, w, wv = _operands(1, n, k, fmt, gpu)
    x = (0.5 * torch.randn(m, k, generator=torch.Generator().manual_seed(m))).to(dtype).to(gpu)
    q = mx.quantize(x, fmt)
    av = torch.from_numpy(ora.values(ora.unpack(q.data.cpu().numpy(), fmt), q.scale.cpu().numpy(), fmt, k)).to(gpu)
    u, size = av @ wv.t().contiguous(), av.abs() @ wv.abs().t().contiguous()
    y = mx.linear(x, w, x_fmt=fmt)
    _check(y, u, (128 + ora.padded(k) // 128) * U * size, None, None, dtype, "values")
    assert torch.equal(y, mx.linear(q, w, out_dtype=dtype))


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_residual_in_place_and_nothing_behind_the_last_row(gpu, kernel, fmt):
    lib, s = _lib.load(), _lib.current_stream_ptr(gpu)
    m, n, k = KERNELS[kernel]
    a, _, w, _ = _operands(m, n, k, fmt, gpu)
    for code, dtype in enumerate(DTYPES):
        res = (50 * torch.randn(m, n, generator=torch.Generator().manual_seed(n))).to(dtype).to(gpu)
        want = mx.linear(a, w, residual=res, out_dtype=dtype)
        out = torch.full((m + 2, n), 7.0, device=gpu, dtype=dtype)
        out[:m] = res
        _lib.check(lib.clipenc_op_gemm_mx(a.data.data_ptr(), a.scale.data_ptr(), mx.FORMATS[fmt], w.data.data_ptr(), w.scale.data_ptr(), m, n, k, None, -1, out.data_ptr(),
                                          out.data_ptr(), code, s), "gemm")
        assert torch.equal(out[:m], want) and (out[m:] == 7.0).all()


@pytest.mark.parametrize("fmt", ["e2m1", "e4m3"])
@pytest.mark.parametrize("kernel", KERNELS)
def test_a_block_that_is_not_finite_is_in_its_own_row_or_column_only(gpu, kernel, fmt):
    m, n, k = KERNELS[kernel]
    a, _, w, _ = _operands(m, n, k, fmt, gpu)
    a.scale[m // 2, 1] = 255
    w.scale[n // 3, 0] = 255
    want = torch.zeros(m, n, dtype=torch.bool, device=gpu)
    want[m // 2] = True
    want[:, n // 3] = True
    for dtype in (BF16, F32):
        for act in (None, "gelu", "quick_gelu"):
            assert torch.equal(torch.isnan(mx.linear(a, w, act=act, out_dtype=dtype)), want)


# ------------------------------------------------------------------------------------------ activations
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["gelu", "quick_gelu"])
@pytest.mark.parametrize("m,n", [(1, 4000), (300, 4000), (1, 30000), (4096, 4096), (4100, 4000)])
def test_activations_of_exact_arguments(gpu, m, n, act, dtype):
    """Products of zero rows: the argument is the bias."""
    w, _ = _coded(n, 128, "e2m1", n, gpu, -3, 0)
    x = mx.MXTensor(torch.zeros(m, 128, dtype=torch.uint8, device=gpu), torch.full((m, 4), 127, dtype=torch.uint8, device=gpu), "e4m3", 128)
    g = torch.Generator().manual_seed(n)
    bias = 26 * torch.rand(n, generator=g) - 13
    bias[::7] *= 2.0 ** -6
    bias[5:20] = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 13.5, -40.0, 40.0, 1e4, -1e4, 1e30, -1e30, 3e38, -3e38, float("inf"), float("nan")])
    u = bias.to(gpu).double()
    y = mx.linear(x, w, bias=bias.to(gpu), act=act, out_dtype=dtype)
    want = _activate(u, act)
    assert torch.isnan(y[:, 19]).all() and torch.isinf(y[:, 18]).all()
    far = want.abs() > torch.finfo(dtype).max
    assert (y[:, far].double() == want[far].sign() * float("inf")).all()
    fine = ~far & ~torch.isnan(want)
    want, got = want[fine], y[:, fine].double()
    tol = _act_error(want, dtype)
    tol = tol + _half(dtype) * (want.abs() + tol) + float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    off = (got - want).abs() - tol
    assert not (off > 0).any(), (off.max().item(), u[fine][int(off.max(0).values.argmax())].item())


# ------------------------------------------------------------------------------------------ norm
@pytest.mark.parametrize("fmt", ["e2m1", "e4m3", "e4m3_row"])
@pytest.mark.parametrize("rows,cols", [(1, 64), (3, 1000), (5, 1280), (3000, 1280), (4, 2400), (2, 9000)])
def test_norm_of_values_beside_a_tie_has_the_codes_of_64_bits(gpu, rows, cols, fmt):
    """Rows of +-1, whose root mean square is 1: y = +-gamma + beta with gamma a tie of the format and beta +-2^-30 of it, which fp32 does not hold."""
    r = np.random.RandomState(cols)
    kind = "e2m1" if fmt == "e2m1" else "e4m3"
    grid = ora.grid(kind)
    ties = (grid[1:] + grid[:-1]) / 2
    gamma = ties[r.randint(1, len(ties), cols)]
    gamma[::32] = grid[-1]                                                        # every block's and the row's largest: scales of 1
    beta = gamma * 2.0 ** -30 * r.choice([-1.0, 1.0], cols)
    beta[::32] = 0.0
    sign = r.choice([-1.0, 1.0], (rows, cols))
    y = sign * gamma + beta
    dev = lambda v, t: torch.from_numpy(v).to(t).to(gpu)                          # noqa: E731
    _, q = mx.norm_quantize(dev(sign, BF16), dev(gamma, F32), bias=dev(beta, F32), eps=0.0, fmt=fmt)
    codes = ora.unpack(q.data.cpu().numpy(), fmt)[:, :cols]
    assert (q.scale == 1.0).all() if fmt == "e4m3_row" else (q.scale[:, :cols // 32] == 127).all()
    want = ora.nearest_code(np.abs(y), kind) | np.where(np.signbit(y), 8 if fmt == "e2m1" else 128, 0)
    assert np.array_equal(codes, want)
    assert (want != (ora.nearest_code(np.float32(np.abs(y)).astype(np.float64), kind) | np.where(np.signbit(y), 8 if fmt == "e2m1" else 128, 0))).any()


# ------------------------------------------------------------------------------------------ reading back
def _rounded(v, dtype):
    """float64 values, each the product of two numbers of at most 24 and 4 bits, to the nearest of the type, ties to even, in one rounding."""
    bits, low = {BF16: (8, -133), F16: (11, -24), F32: (24, -149)}[dtype]
    _, e = np.frexp(v)
    unit = np.ldexp(1.0, np.maximum(e - bits, low))
    v = np.rint(v / unit) * unit
    return np.where(np.abs(v) > torch.finfo(dtype).max, np.copysign(np.inf, v), v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [9, 128, 1001])
def test_rows_with_one_scale_are_read_back_in_one_rounding(gpu, cols, dtype):
    """Scales of any bits, and such that a product lies just beside a tie between two values of the type."""
    r = np.random.RandomState(cols)
    rows = 600
    codes = r.randint(0, 256, (rows, ora.padded(cols))).astype(np.uint8)
    codes[(codes & 127) == 127] = 0
    codes[:, :8] = np.arange(0x38, 0x40)                                          # 1 .. 1.875
    codes[:, cols:] = 0
    scale = np.exp(r.uniform(-8, 4, rows)).astype(np.float32)
    bits = {BF16: 8, F16: 11, F32: 23}[dtype]
    tie = (2 * r.randint(2 ** (bits - 1), 2 ** bits, rows - 100) + 1) * 2.0 ** -bits
    scale[100:] = (tie / (1 + r.randint(0, 8, rows - 100) / 8)).astype(np.float32)
    q = mx.MXTensor(torch.from_numpy(codes).to(gpu), torch.from_numpy(scale).to(gpu), "e4m3_row", cols)
    want = _rounded(ora.values(codes, scale, "e4m3_row", cols), dtype)
    got = mx.dequantize(q, dtype).cpu().double().numpy()
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]


def test_rows_with_scales_at_the_ends_of_their_range(gpu):
    scale = np.array([0.0, -0.0, 1.0, np.float32(2.0 ** -149), np.float32(2.0 ** -130), np.float32(3e38), np.inf, np.nan], np.float32)
    codes = np.tile(np.arange(128, dtype=np.uint8), (8, 1))
    codes[:, 64:] |= 0x80
    q = mx.MXTensor(torch.from_numpy(codes).to(gpu), torch.from_numpy(scale).to(gpu), "e4m3_row", 128)
    with np.errstate(invalid="ignore"):
        want = ora.values(codes, scale, "e4m3_row", 128)
    for dtype in DTYPES:
        got = mx.dequantize(q, dtype).cpu().double().numpy()
        with np.errstate(invalid="ignore"):
            assert np.array_equal(got, np.where(np.isfinite(want), _rounded(np.where(np.isfinite(want), want, 0.0), dtype), want), equal_nan=True)


# ------------------------------------------------------------------------------------------ sizes
@pytest.mark.parametrize("m", [1, 17])
def test_more_columns_than_a_launch_has_work_items_for(gpu, m):
    """2^27 and some weight rows of 1000 columns: 64 GiB, eight waves a workgroup."""
    n, k = (1 << 27) + 77, 1000
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info(gpu)[0] < 90 << 30:
        pytest.skip("needs 90 GiB of device memory")
    at = torch.tensor([0, 1, 15, 16, n // 2, (1 << 27) - 1, 1 << 27, n - 70, n - 17, n - 1])
    a, av, some, wv = _operands(m, len(at), k, "e2m1", gpu)
    data, scale = torch.zeros(n, 512, dtype=torch.uint8, device=gpu), torch.full((n, 32), 127, dtype=torch.uint8, device=gpu)
    data[at.to(gpu)], scale[at.to(gpu)] = some.data, some.scale
    y = mx.linear(a, mx.MXTensor(data, scale, "e2m1", k))
    u, size = av @ wv.t().contiguous(), av.abs() @ wv.abs().t().contiguous()
    _check(y[:, at.to(gpu)], u, (128 + 8) * U * size, None, None, BF16, "columns")
    y[:, at.to(gpu)] = 0
    assert not y.any()
    del data, scale, y
    torch.cuda.empty_cache()
