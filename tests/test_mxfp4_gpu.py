"""MXFP4 quantization, its inverse and the products, against plain 64-bit forms."""
import pytest
import torch

from mpserve_amd.mxfp4 import mxfp4_dequantize, mxfp4_linear, mxfp4_matmul, mxfp4_quantize
from tests import mx_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = (torch.bfloat16, torch.float16, torch.float32)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def check_quantize(x):
    codes, scales = mxfp4_quantize(x)
    want_codes, want_scales = plain.quantize(x.reshape(-1, x.shape[-1]))
    nb = plain.blocks_of(x.shape[-1])
    assert codes.shape == (*x.shape[:-1], 16 * nb) and scales.shape == (*x.shape[:-1], nb)
    assert torch.equal(scales.cpu().reshape(want_scales.shape), want_scales)
    assert torch.equal(codes.cpu().reshape(want_codes.shape), want_codes)
    return codes, scales


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 31), (1, 32), (3, 33), (2, 64), (5, 100), (17, 257), (64, 1024), (1, 4096),
                                    (1000, 72), (300, 5001)])
def test_quantize_matches_definition(dtype, rows, k):
    x = torch.randn(rows, k, generator=gen(k), device=DEV) * torch.exp2(torch.randint(-12, 5, (rows, k), generator=gen(1), device=DEV).float())
    codes, scales = check_quantize(x.to(dtype))
    for out in TYPES:
        got = mxfp4_dequantize(codes, scales, k, out)
        assert got.dtype == out and torch.equal(got, plain.dequantize(codes, scales, k).to(out))


def test_quantize_every_bf16_value():
    every = torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(torch.bfloat16).to(DEV)
    finite = every[torch.isfinite(every)]
    check_quantize(finite.view(-1, 1))  # each alone: the scale
    for seed in (0, 1):  # against a larger one, 2^0 to 2^9 times: the rounding, its ties, and what falls to zero
        g = gen(seed)
        x = finite.view(-1, 1).expand(-1, 32).clone()
        top = torch.exp2(torch.randint(0, 10, (x.shape[0],), generator=g, device=DEV).float())
        x[:, 5] = (x[:, 5].float() * top).clamp(-3e38, 3e38).to(torch.bfloat16)
        check_quantize(x)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_ties_and_range(dtype):
    """Halfway points between codes, both signs, and what a block's largest element rounds to."""
    v = torch.tensor([4.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.5, 1.5, 3.0, 6.0, 7.0, 7.96875, 0.0, 0.125], device=DEV)
    x = torch.cat([v, -v]).repeat(40, 1) * torch.exp2(torch.arange(-10, 30, device=DEV).clamp(max=12).float()).unsqueeze(1)
    check_quantize(x.to(dtype))


def test_quantize_smallest_and_largest():
    tiny = torch.tensor([2.0 ** -149, 2.0 ** -128, 2.0 ** -127, 2.0 ** -126, 3 * 2.0 ** -126, 2.0 ** -125, 2.0 ** -124, 0.0], device=DEV)
    big = torch.tensor([3.4028234e38, 2.0 ** 127, 2.0 ** 126, 2.0 ** 125, 2.0 ** 124, -3.4028234e38, 1.0, 0.0], device=DEV)
    x = torch.stack([tiny, -tiny, big, -big, torch.zeros_like(big), -torch.zeros_like(big)])
    for dtype in (torch.float32, torch.bfloat16):
        codes, scales = check_quantize(torch.where(torch.isfinite(x.to(dtype).float()), x, torch.zeros_like(x)).to(dtype))
        for out in (torch.float32, torch.bfloat16):
            assert torch.equal(mxfp4_dequantize(codes, scales, 8, out), plain.dequantize(codes, scales, 8).float().to(out))


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_not_finite_block_is_nan(dtype):
    x = torch.randn(4, 100, generator=gen(3), device=DEV).to(dtype)
    x[0, 3], x[1, 40], x[2, 99], x[3, 64] = float("inf"), float("nan"), -float("inf"), float("nan")
    codes, scales = check_quantize(x)
    y = mxfp4_dequantize(codes, scales, 100, dtype)
    nan = torch.zeros(4, 100, dtype=torch.bool, device=DEV)
    nan[0, :32] = nan[1, 32:64] = nan[2, 96:] = nan[3, 64:96] = True
    assert torch.equal(torch.isnan(y), nan)


def test_dequantize_every_scale_and_code():
    codes = torch.arange(256, dtype=torch.uint8, device=DEV).view(16, 16).repeat(256, 1)
    scales = torch.arange(256, dtype=torch.uint8, device=DEV).repeat_interleave(16).view(-1, 1).contiguous()
    want = plain.dequantize(codes, scales, 32).float()
    for dtype in TYPES:
        got = mxfp4_dequantize(codes, scales, 32, dtype)
        assert torch.equal(got.nan_to_num(7.0, 1e9, -1e9), want.to(dtype).nan_to_num(7.0, 1e9, -1e9))


def test_quantize_views():
    base = torch.randn(40, 3, 200, generator=gen(5), device=DEV).to(torch.bfloat16)
    check_quantize(base)
    check_quantize(base[:, 1, 64:192])       # rows apart, 16-byte aligned
    check_quantize(base[:, 1, 3:131])        # rows apart, not aligned
    check_quantize(base[:, 1].t()[:, ::2])   # elements apart
    check_quantize(base[:1, 0].expand(7, 200))  # one row many times
    check_quantize(base[0, 0])               # one dimension


def test_quantize_empty():
    for shape in ((0, 64), (3, 0), (0,)):
        codes, scales = mxfp4_quantize(torch.empty(shape, device=DEV))
        nb = plain.blocks_of(shape[-1])
        assert codes.shape == (*shape[:-1], 16 * nb) and scales.shape == (*shape[:-1], nb)
        assert mxfp4_dequantize(codes, scales, shape[-1]).shape == shape


# --------------------------------------------------------------------------- products
def whole_numbers(g, t, k, dtype):
    return torch.randint(-8, 9, (t, k), generator=g, device=DEV).to(dtype)


SHAPES = [  # t, k, n
    (1, 1, 1), (1, 32, 16), (1, 4096, 512), (2, 31, 17), (3, 33, 15), (5, 96, 100), (8, 160, 33), (15, 256, 64),
    (16, 1000, 48), (17, 288, 257), (31, 64, 128), (33, 544, 31), (48, 2080, 300), (64, 128, 512), (65, 512, 130),
    (100, 5000, 77), (127, 736, 255), (128, 1024, 256), (130, 96, 1), (200, 1056, 513), (256, 256, 1024),
    (257, 320, 769), (300, 1500, 260), (512, 2048, 520), (1030, 672, 384),
    # sizes at which each shape of a workgroup for few rows is the one that is taken
    (1, 1030, 16), (130, 1030, 1030), (130, 2056, 520), (500, 1030, 520), (50, 2056, 2100), (500, 1030, 1030),
    (130, 500, 1030), (500, 500, 520), (70, 500, 20000), (1, 500, 20000), (60, 320, 100),
    # enough tiles for each of the larger ones, ends of rows and columns inside them, one block to several periods of k
    (700, 96, 4300), (1100, 64, 8300), (2100, 32, 8300), (2300, 704, 8500), (4500, 160, 5000), (9000, 544, 2100),
    (200, 608, 5000), (250, 1030, 4101), (1000, 1030, 8195), (2000, 1030, 4101), (130, 4100, 5000),
]


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("t,k,n", SHAPES)
def test_linear_whole_numbers_are_exact(dtype, t, k, n):
    """Products and sums that FP32 holds exactly (below 2^24 halves): any wrong, lost or doubled term shows."""
    g = gen(t * 7 + k)
    x = whole_numbers(g, t, k, dtype)
    codes, scales = plain.random_weight(g, (n,), k, DEV, 126, 129)
    want = x.double() @ plain.dequantize(codes, scales, k).T
    assert torch.equal(mxfp4_linear(x, codes, scales, out_dtype=torch.float32).double(), want)
    bias = torch.randint(-64, 65, (n,), generator=g, device=DEV).to(dtype)
    assert torch.equal(mxfp4_linear(x, codes, scales, bias), (want + bias.double()).float().to(dtype))


@pytest.mark.parametrize("t,k,n", SHAPES)
def test_matmul_whole_numbers_are_exact(t, k, n):
    g = gen(t * 5 + k)
    xc, xs = plain.random_weight(g, (t,), k, DEV, 126, 129)
    codes, scales = plain.random_weight(g, (n,), k, DEV, 126, 129)
    want = plain.dequantize(xc, xs, k) @ plain.dequantize(codes, scales, k).T
    assert torch.equal(mxfp4_matmul(xc, xs, codes, scales, out_dtype=torch.float32).double(), want)
    bias = torch.randint(-64, 65, (n,), generator=g, device=DEV).float()
    for dtype in (torch.bfloat16, torch.float16):
        assert torch.equal(mxfp4_matmul(xc, xs, codes, scales, bias, out_dtype=dtype), (want + bias.double()).float().to(dtype))


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("t,k,n", [(1, 4096, 1000), (7, 1001, 130), (40, 2048, 512), (300, 4096, 384), (1000, 736, 600)])
def test_linear_is_close(dtype, out, t, k, n):
    g = gen(t + k)
    x = (torch.randn(t, k, generator=g, device=DEV) * torch.exp(torch.randn(k, generator=g, device=DEV))).to(dtype)
    codes, scales = plain.random_weight(g, (n,), k, DEV)
    w = plain.dequantize(codes, scales, k)
    bias = torch.randn(n, generator=g, device=DEV)
    want, size = x.double() @ w.T + bias.double(), x.double().abs() @ w.abs().T + bias.double().abs()
    plain.close(mxfp4_linear(x, codes, scales, bias, out_dtype=out), want, size, k + 1)


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("t,k,n", [(1, 4096, 1000), (7, 1001, 130), (40, 2048, 512), (300, 4096, 384), (1000, 736, 600)])
def test_matmul_is_close(out, t, k, n):
    g = gen(t + k)
    xc, xs = plain.random_weight(g, (t,), k, DEV, 100, 135)
    codes, scales = plain.random_weight(g, (n,), k, DEV, 100, 130)
    x, w = plain.dequantize(xc, xs, k), plain.dequantize(codes, scales, k)
    plain.close(mxfp4_matmul(xc, xs, codes, scales, out_dtype=out), x @ w.T, x.abs() @ w.abs().T, k)


@pytest.mark.parametrize("t", (1, 20, 300))
def test_linear_views_and_out(t):
    g = gen(t)
    base = whole_numbers(g, t, 1200, torch.bfloat16)
    codes, scales = plain.random_weight(g, (100,), 320, DEV, 126, 129)
    w = plain.dequantize(codes, scales, 320).T
    for x in (base[:, 64:384], base[:, 3:323], base[:, :640:2], base[:1, :320].expand(t, 320)):
        assert torch.equal(mxfp4_linear(x, codes, scales, out_dtype=torch.float32).double(), x.double() @ w)
    x3 = base[:, :960].reshape(t, 3, 320)
    out = torch.empty(t, 3, 100, dtype=torch.bfloat16, device=DEV)
    assert mxfp4_linear(x3, codes, scales, out=out) is out
    assert torch.equal(out, (x3.double() @ w).float().to(torch.bfloat16))
    assert mxfp4_linear(x3[0, 0], codes, scales).shape == (100,)
    part = codes[40:], scales[40:]  # a slice of the weight's rows
    assert torch.equal(mxfp4_linear(base[:, :320], *part, out_dtype=torch.float32).double(), base[:, :320].double() @ w[:, 40:])


@pytest.mark.parametrize("t", (2, 300))
def test_products_keep_nan_and_infinity_where_they_belong(t):
    g = gen(9)
    x = torch.randn(t, 320, generator=g, device=DEV).to(torch.bfloat16)
    codes, scales = plain.random_weight(g, (300,), 320, DEV)
    scales[37, 4] = 255                # NaN weights: output column 37
    x[1, 319] = float("inf")           # row 1
    y = mxfp4_linear(x, codes, scales)
    bad = ~torch.isfinite(y)
    assert bool(bad[:, 37].all()) and bool(bad[1].all())
    bad[:, 37] = bad[1] = False
    assert not bool(bad.any())
    xc, xs = mxfp4_quantize(x)
    bad = ~torch.isfinite(mxfp4_matmul(xc, xs, codes, scales))
    assert bool(bad[:, 37].all()) and bool(bad[1].all())
    bad[:, 37] = bad[1] = False
    assert not bool(bad.any())


def test_products_smallest_and_largest_scales():
    g = gen(11)
    for lo, hi in ((0, 4), (240, 252)):
        codes, scales = plain.random_weight(g, (64,), 256, DEV, lo, hi)
        w = plain.dequantize(codes, scales, 256)
        x = (torch.randn(20, 256, generator=g, device=DEV) * (2.0 ** 40 if lo == 0 else 2.0 ** -40)).to(torch.bfloat16)
        plain.close(mxfp4_linear(x, codes, scales, out_dtype=torch.float32), x.double() @ w.T, x.double().abs() @ w.abs().T, 256)
        xc, xs = mxfp4_quantize(x)
        xv = plain.dequantize(xc, xs, 256)
        plain.close(mxfp4_matmul(xc, xs, codes, scales, out_dtype=torch.float32), xv @ w.T, xv.abs() @ w.abs().T, 256)


LARGEST = [(1, 1030, 16), (1, 4096, 512), (8, 160, 33), (16, 1000, 48), (50, 2056, 2100), (64, 128, 512), (130, 1030, 1030), (130, 2056, 520),
           (500, 1030, 520), (70, 500, 20000), (60, 320, 100), (250, 1030, 4101), (700, 96, 4300), (1100, 64, 8300), (2300, 704, 8500)]


@pytest.mark.parametrize("kind", (torch.bfloat16, torch.float16, "mxfp4"))
@pytest.mark.parametrize("t,k,n", LARGEST)
def test_products_with_the_largest_scales_are_exact(kind, t, k, n):
    """Weights of 2^128 and more in every second column, ordinary ones beside them, and small x, zeros among them:
    whole numbers times powers of two, so that FP32 holds all products and sums (in quarters of halves, below 2^24)."""
    g = gen(t + k + n)
    codes, scales = plain.random_weight(g, (n,), k, DEV, 126, 129)
    scales[::2] = torch.randint(252, 255, scales[::2].shape, generator=g, device=DEV, dtype=torch.uint8)
    if kind == "mxfp4":
        xc, xs = plain.random_weight(g, (t,), k, DEV, 66, 69)
        x, got = plain.dequantize(xc, xs, k), mxfp4_matmul(xc, xs, codes, scales, out_dtype=torch.float32)
    else:
        x = (whole_numbers(g, t, k, torch.float32) * (2.0 ** -60 if kind is torch.bfloat16 else 2.0 ** -20)).to(kind)
        got = mxfp4_linear(x, codes, scales, out_dtype=torch.float32)
    want = x.double() @ plain.dequantize(codes, scales, k).T
    assert torch.equal(got.double(), want)


@pytest.mark.parametrize("t", (3, 300))
def test_linear_bf16_largest_scales_beside_others(t):
    """NaN scales, the smallest ones, and infinite x, in tiles with the largest scales. Two terms a sum, of powers of two."""
    g = gen(t)
    codes, scales = plain.random_weight(g, (300,), 320, DEV, 250, 255)
    tiny = torch.zeros(300, dtype=torch.bool, device=DEV)
    tiny[1::3] = True
    scales[tiny] = torch.randint(0, 4, scales[tiny].shape, generator=g, device=DEV, dtype=torch.uint8)
    scales[36, 4] = 255
    x = torch.zeros(t, 320, dtype=torch.bfloat16, device=DEV)
    x[0, 7], x[0, 300], x[1, 319], x[2, 7], x[2, 300] = 2.0 ** -10, -2.0 ** -9, float("inf"), 2.0 ** 30, 2.0 ** 31
    y = mxfp4_linear(x, codes, scales, out_dtype=torch.float32)
    assert bool(torch.isnan(y[:, 36]).all()) and not bool(torch.isfinite(y[1]).any())
    want = x.double() @ plain.dequantize(codes, scales, 320).T
    large = ~tiny
    large[36] = False
    assert torch.equal(y[0, large].double(), want[0, large])
    assert torch.equal(y[2, tiny].double(), want[2, tiny])
    assert bool((y[3:, tiny | large] == 0).all())


@pytest.mark.parametrize("t", (3, 40, 200))
def test_linear_f16_with_scales_outside_f16(t):
    """Weights far below and far above what FP16 holds, and blocks of both in one row."""
    g = gen(t)
    codes, scales = plain.random_weight(g, (70,), 256, DEV, 0, 3)
    scales[::2, 1::2] = torch.randint(60, 100, (35, 4), generator=g, device=DEV, dtype=torch.uint8)
    scales[3] = torch.randint(150, 160, (8,), generator=g, device=DEV, dtype=torch.uint8)
    w = plain.dequantize(codes, scales, 256)
    x = torch.randn(t, 256, generator=g, device=DEV).to(torch.float16)
    want, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    normal = size > 2.0 ** -100  # FP32 sums of the other columns are below its normal numbers
    y = mxfp4_linear(x, codes, scales, out_dtype=torch.float32)
    plain.close(torch.where(normal, y, torch.zeros_like(y)), torch.where(normal, want, torch.zeros_like(want)), size, 256)
    assert float((y.double() - want).abs()[~normal].max()) <= 256 * 2.0 ** -149
    scales[9, 0] = 255
    assert bool(torch.isnan(mxfp4_linear(x, codes, scales)[:, 9]).all())


def test_products_without_rows_columns_or_terms():
    codes, scales = torch.zeros(5, 0, dtype=torch.uint8, device=DEV), torch.zeros(5, 0, dtype=torch.uint8, device=DEV)
    bias = torch.arange(5, device=DEV).to(torch.bfloat16)
    y = mxfp4_linear(torch.empty(3, 0, dtype=torch.bfloat16, device=DEV), codes, scales, bias)
    assert torch.equal(y, bias.expand(3, 5))
    y = mxfp4_matmul(torch.empty(3, 0, dtype=torch.uint8, device=DEV), torch.empty(3, 0, dtype=torch.uint8, device=DEV), codes, scales)
    assert torch.equal(y, torch.zeros(3, 5, dtype=torch.bfloat16, device=DEV))
    codes, scales = plain.random_weight(gen(0), (5,), 64, DEV)
    assert mxfp4_linear(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), codes, scales).shape == (0, 5)
    assert mxfp4_linear(torch.empty(2, 64, dtype=torch.bfloat16, device=DEV), codes[:0], scales[:0]).shape == (2, 0)


def test_linear_output_past_32_bits():
    """Over 2^31 output elements (and over 2^32 bytes of x): the last rows are as right as the first."""
    t, k, n = 70000, 32, 32000
    g = gen(2)
    x = whole_numbers(g, t, 40000, torch.bfloat16)[:, 39968:]  # rows 80000 bytes apart: 5.6 GB
    codes, scales = plain.random_weight(g, (n,), k, DEV, 126, 129)
    y = mxfp4_linear(x, codes, scales)
    w = plain.dequantize(codes, scales, k).T
    for rows in (slice(0, 3), slice(t // 2, t // 2 + 3), slice(67107, 67112), slice(t - 3, t)):
        assert torch.equal(y[rows], (x[rows].double() @ w).float().to(torch.bfloat16))


def test_quantize_past_32_bits():
    """Over 2^32 work-items and 2^35 elements: the last rows are as right as the first."""
    rows, k = (1 << 20) + 40, 32800
    if torch.cuda.mem_get_info()[0] < 110 << 30:
        pytest.skip("needs 110 GB of free memory")
    x = torch.empty(rows, k, dtype=torch.bfloat16, device=DEV)
    ends = (slice(0, 2), slice(rows // 2, rows // 2 + 2), slice((1 << 20) - 2, (1 << 20) + 2), slice(rows - 2, rows))
    for i, part in enumerate(ends):
        x[part] = torch.randn(x[part].shape, generator=gen(i), device=DEV).to(torch.bfloat16)
    codes, scales = mxfp4_quantize(x)
    for part in ends:
        want_codes, want_scales = plain.quantize(x[part])
        assert torch.equal(codes[part].cpu(), want_codes) and torch.equal(scales[part].cpu(), want_scales)
    back = x  # decoded over the input, which is not needed any more
    mxfp4_dequantize(codes, scales, k, out=back)
    for part in ends:
        assert torch.equal(back[part], plain.dequantize(codes[part], scales[part], k).to(torch.bfloat16))
    del x, back, codes, scales
    torch.cuda.empty_cache()


def test_products_repeat_bit_for_bit():
    g = gen(21)
    for t in (1, 40, 600):
        x = torch.randn(t, 4096, generator=g, device=DEV).to(torch.bfloat16)
        codes, scales = plain.random_weight(g, (700,), 4096, DEV)
        xc, xs = mxfp4_quantize(x)
        first = mxfp4_linear(x, codes, scales), mxfp4_matmul(xc, xs, codes, scales)
        for _ in range(3):
            assert torch.equal(mxfp4_linear(x, codes, scales), first[0])
            assert torch.equal(mxfp4_matmul(xc, xs, codes, scales), first[1])


def test_products_on_another_stream():
    g = gen(31)
    x = whole_numbers(g, 200, 512, torch.float16)
    codes, scales = plain.random_weight(g, (300,), 512, DEV, 126, 129)
    want = x.double() @ plain.dequantize(codes, scales, 512).T
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = mxfp4_linear(x, codes, scales, out_dtype=torch.float32)
        xc, xs = mxfp4_quantize(x)
        back = mxfp4_dequantize(xc, xs, 512, torch.float32)
    side.synchronize()
    assert torch.equal(y.double(), want)
    assert torch.equal(back.double(), plain.dequantize(*(t.to(DEV) for t in plain.quantize(x)), 512))


# --------------------------------------------------------------------------- refusals
def test_refusals():
    x = torch.randn(4, 64, device=DEV).to(torch.bfloat16)
    codes, scales = plain.random_weight(gen(0), (8,), 64, DEV)
    for call, message in (
            (lambda: mxfp4_quantize(x.int()), "x must be torch.bfloat16"),
            (lambda: mxfp4_quantize(torch.tensor(1.0, device=DEV)), "at least one dimension"),
            (lambda: mxfp4_dequantize(codes.int(), scales, 64), "codes must be torch.uint8"),
            (lambda: mxfp4_dequantize(codes, scales[:, :1], 64), "scales must be contiguous"),
            (lambda: mxfp4_dequantize(codes, scales[:, :1].contiguous(), 64), "must agree"),
            (lambda: mxfp4_dequantize(codes, scales, 65), "does not fit"),
            (lambda: mxfp4_dequantize(codes, scales, 32), "does not fit"),
            (lambda: mxfp4_dequantize(codes, scales, 64, torch.float64), "dtype must be"),
            (lambda: mxfp4_dequantize(codes, scales, 64, out=torch.empty(8, 64, device=DEV)), "out must be"),
            (lambda: mxfp4_linear(x.float(), codes, scales), "x must be torch.bfloat16 or torch.float16"),
            (lambda: mxfp4_linear(x[:, :32], codes, scales), "do not fit"),
            (lambda: mxfp4_linear(x, codes[0], scales[0]), "dimension"),
            (lambda: mxfp4_linear(x, codes.cpu(), scales), "must be a CUDA tensor"),
            (lambda: mxfp4_linear(x, codes, scales, torch.zeros(7, device=DEV)), "bias must have shape"),
            (lambda: mxfp4_linear(x, codes, scales, torch.zeros(8, dtype=torch.int32, device=DEV)), "bias must be"),
            (lambda: mxfp4_linear(x, codes, scales, out_dtype=torch.int32), "out_dtype must be"),
            (lambda: mxfp4_linear(x, codes, scales, out=torch.empty(4, 9, dtype=torch.bfloat16, device=DEV)), "out must be"),
            (lambda: mxfp4_linear(x, torch.zeros(8 * 32 + 1, dtype=torch.uint8, device=DEV)[1:].view(8, 32), scales), "16-byte aligned"),
            (lambda: mxfp4_matmul(codes, scales, *plain.random_weight(gen(0), (8,), 96, DEV)), "blocks a row")):
        with pytest.raises(ValueError, match=message):
            call()
    for call in (lambda: mxfp4_quantize(x.float().requires_grad_()), lambda: mxfp4_linear(x.detach().requires_grad_(), codes, scales),
                 lambda: mxfp4_matmul(codes, scales, codes, scales, torch.zeros(8, device=DEV, requires_grad=True))):
        with pytest.raises(RuntimeError, match="has no gradient"):
            call()
    with torch.no_grad():
        assert mxfp4_linear(x.detach().requires_grad_(), codes, scales).shape == (4, 8)


def test_out_and_autograd():
    """A tensor that autograd follows is not written behind its back."""
    from mpserve_amd.experts import expert_sort, mxfp4_expert_linear

    x = torch.randn(4, 64, device=DEV).to(torch.bfloat16)
    codes, scales = plain.random_weight(gen(0), (8,), 64, DEV)
    sort = expert_sort(torch.zeros(4, 1, dtype=torch.int32, device=DEV), 1)
    calls = (lambda out: mxfp4_linear(x, codes, scales, out=out), lambda out: mxfp4_matmul(*mxfp4_quantize(x), codes, scales, out=out),
             lambda out: mxfp4_expert_linear(x, codes[None], scales[None], sort, out=out))
    for call in calls + (lambda out: mxfp4_dequantize(codes[:4, :16].contiguous(), scales[:4, :1].contiguous(), 8, torch.bfloat16, out=out),):
        out = torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV)
        with pytest.raises(RuntimeError, match="out must not require a gradient"):
            call(out.requires_grad_())
        with torch.no_grad():
            assert call(out) is out
        out, factor = torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV), torch.ones(4, 8, dtype=torch.bfloat16, device=DEV, requires_grad=True)
        product = out * factor  # autograd keeps `out`
        call(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            product.sum().backward()
        with torch.inference_mode():
            out = torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV)
            assert call(out) is out
