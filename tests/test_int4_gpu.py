"""Products with int4 weights, of one weight and of experts', against plain 64-bit forms."""
import pytest
import torch

from mpserve_amd.experts import ExpertSort, expert_combine, expert_gather, expert_sort, int4_expert_linear
from mpserve_amd.int4 import int4_from_awq, int4_linear, int4_pack
from tests import int4_plain as plain
from tests import mx_plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALVES = (torch.bfloat16, torch.float16)
TYPES = (*HALVES, torch.float32)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def whole_numbers(g, t, k, dtype):
    return torch.randint(-8, 9, (t, k), generator=g, device=DEV).to(dtype)


def close(y, x, values, scales, zeros, group, bias=None):
    """Sums of k products, with x times q and x times z apart or together: at most 2 k + 3 (a group's scale and zero, the
    bias) additions a term of either; corrections by zero from sums in two or three pieces add 2^-22 of theirs."""
    w, far = plain.weight(values, scales, zeros, group), plain.reach(values, scales, zeros, group)
    want, size = x.double() @ w.T, x.double().abs() @ far.T
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    mx_plain.close(y, want, size, 2 * x.shape[1] + 5)


SHAPES = [  # t, k, n, group
    (1, 1, 1, 32), (1, 32, 16, 32), (1, 4096, 512, 128), (2, 31, 17, 64), (3, 33, 15, 32), (5, 96, 100, 64), (8, 160, 33, 128),
    (15, 256, 64, 256), (16, 1000, 48, 128), (17, 288, 257, 32), (31, 64, 128, 64), (33, 544, 31, 512), (48, 2080, 300, 128),
    (64, 128, 512, 128), (65, 512, 130, 64), (100, 5000, 77, 128), (127, 736, 255, 1024), (128, 1024, 256, 32), (130, 96, 1, 64),
    (200, 1056, 513, 128), (256, 256, 1024, 64), (257, 320, 769, 32), (300, 1500, 260, 128), (512, 2048, 520, 128),
    (1030, 672, 384, 256), (1, 1030, 16, 64), (130, 2056, 520, 32), (50, 2056, 2100, 128), (500, 1030, 1030, 64),
    (130, 500, 1030, 128), (70, 500, 20000, 128), (1, 500, 20000, 32), (700, 96, 4300, 128), (1100, 64, 8300, 64),
    (2100, 32, 8300, 32), (2300, 704, 8500, 128), (4500, 160, 5000, 32), (250, 1030, 4101, 64), (2000, 1030, 4101, 256),
    (4, 14336, 300, 128), (20, 8192, 700, 2048), (16, 4090, 13000, 128), (13, 4096, 14000, 32),
]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,k,n,group", SHAPES)
def test_linear_whole_numbers_are_exact(dtype, t, k, n, group):
    """Products and sums that FP32 holds exactly (halves, below 2^23): any wrong, lost or doubled term shows."""
    g = gen(t * 7 + k)
    x = whole_numbers(g, t, k, dtype)
    for zeros in (True, False):
        values, scales, z = plain.random_weight(g, (n,), k, group, dtype, zeros, DEV, whole=True)
        want = x.double() @ plain.weight(values, scales, z, group).T
        codes = int4_pack(values)
        assert torch.equal(int4_linear(x, codes, scales, z, group=group, out_dtype=torch.float32).double(), want)
        bias = torch.randint(-64, 65, (n,), generator=g, device=DEV).to(dtype)
        assert torch.equal(int4_linear(x, codes, scales, z, bias, group=group), (want + bias.double()).float().to(dtype))


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("stype", HALVES)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,k,n,group", [(1, 4096, 1000, 128), (7, 1001, 130, 32), (40, 2048, 512, 64), (300, 4096, 384, 128), (1000, 736, 600, 32),
                                         (3000, 1024, 2100, 128)])
def test_linear_is_close(dtype, stype, out, t, k, n, group):
    g = gen(t + k)
    x = (torch.randn(t, k, generator=g, device=DEV) * torch.exp(torch.randn(k, generator=g, device=DEV))).to(dtype)
    values, scales, z = plain.random_weight(g, (n,), k, group, stype, t % 2 == 1, DEV)
    bias = torch.randn(n, generator=g, device=DEV)
    close(int4_linear(x, int4_pack(values), scales, z, bias, group=group, out_dtype=out), x, values, scales, z, group, bias)


@pytest.mark.parametrize("t", (1, 20, 300, 2000))
def test_linear_views_and_out(t):
    g = gen(t)
    base = whole_numbers(g, t, 1200, torch.bfloat16)
    values, scales, z = plain.random_weight(g, (100,), 320, 64, torch.float16, True, DEV, whole=True)
    codes, w = int4_pack(values), plain.weight(values, scales, z, 64).T
    for x in (base[:, 64:384], base[:, 3:323], base[:, :640:2], base[:1, :320].expand(t, 320)):
        assert torch.equal(int4_linear(x, codes, scales, z, group=64, out_dtype=torch.float32).double(), x.double() @ w)
    x3 = base[:, :960].reshape(t, 3, 320)
    out = torch.empty(t, 3, 100, dtype=torch.bfloat16, device=DEV)
    assert int4_linear(x3, codes, scales, z, group=64, out=out) is out
    assert torch.equal(out, (x3.double() @ w).float().to(torch.bfloat16))
    assert int4_linear(x3[0, 0], codes, scales, z, group=64).shape == (100,)
    part = codes[41:], scales[41:], z[41:]  # a slice of the weight's rows, whose scales and zeros are not aligned
    assert torch.equal(int4_linear(base[:, :320], *part, group=64, out_dtype=torch.float32).double(), base[:, :320].double() @ w[:, 41:])


def test_zeros_count_by_their_low_five_bits():
    g = gen(3)
    x = whole_numbers(g, 9, 256, torch.float16)
    values, scales, z = plain.random_weight(g, (40,), 256, 64, torch.float16, True, DEV, whole=True)
    want = int4_linear(x, int4_pack(values), scales, z, group=64)
    assert torch.equal(int4_linear(x, int4_pack(values), scales, z | 0xe0, group=64), want)


@pytest.mark.parametrize("t", (3, 40, 300, 1500))
@pytest.mark.parametrize("dtype", HALVES)
def test_what_lies_past_the_last_column_does_not_count(dtype, t):
    """Codes of the last block past column k, x behind its rows, and rows behind x."""
    g = gen(t)
    for k in (1, 30, 33, 100, 500):
        whole = torch.full((t + 3, k + 40), float("nan"), dtype=dtype, device=DEV)
        whole[:t, :k] = whole_numbers(g, t, k, dtype)
        x = whole[:t, :k]
        values, scales, z = plain.random_weight(g, (300,), k, 32, dtype, True, DEV, whole=True)
        codes = int4_pack(torch.nn.functional.pad(values, (0, -k % 32), value=13))
        want = x.double() @ plain.weight(values, scales, z, 32).T
        assert torch.equal(int4_linear(x, codes, scales, z, group=32, out_dtype=torch.float32).double(), want)
        assert torch.equal(int4_linear(x.contiguous(), codes, scales, z, group=32, out_dtype=torch.float32).double(), want)


@pytest.mark.parametrize("t", (2, 40, 300, 1500))
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("group", (32, 128))
def test_infinities_and_nan_stay_in_their_rows_and_columns(dtype, t, group):
    """An infinity in x gives what it gives in the plain form: infinite of the weight's sign, NaN where the weight is zero."""
    g = gen(t)
    k, n = 544, 300
    x = whole_numbers(g, t, k, dtype)
    x[1, 37], x[t - 1, 500] = float("inf"), -float("inf")
    if t > 2:
        x[2, 0] = float("nan")
        x[5, 3], x[5, 400] = float("inf"), float("inf")
    values, scales, z = plain.random_weight(g, (n,), k, group, dtype, True, DEV, whole=True)
    scales[17, 0] = float("nan")
    y = int4_linear(x, int4_pack(values), scales, z, group=group, out_dtype=torch.float32).double()
    want = x.cpu().double() @ plain.weight(values, scales, z, group).cpu().T
    assert torch.equal(y.cpu().nan_to_num(7.5, 1e300, -1e300), want.nan_to_num(7.5, 1e300, -1e300))


def test_linear_without_rows_columns_or_terms():
    empty = torch.zeros(5, 0, dtype=torch.uint8, device=DEV)
    bias = torch.arange(5, device=DEV).to(torch.bfloat16)
    y = int4_linear(torch.empty(3, 0, dtype=torch.bfloat16, device=DEV), empty, empty.to(torch.bfloat16), None, bias)
    assert torch.equal(y, bias.expand(3, 5))
    values, scales, z = plain.random_weight(gen(0), (5,), 64, 32, torch.bfloat16, True, DEV)
    codes = int4_pack(values)
    assert int4_linear(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), codes, scales, z, group=32).shape == (0, 5)
    assert int4_linear(torch.empty(2, 64, dtype=torch.bfloat16, device=DEV), codes[:0], scales[:0], z[:0], group=32).shape == (2, 0)


def test_linear_output_past_32_bits():
    """Over 2^31 output elements (and over 2^32 bytes of x): the last rows are as right as the first."""
    t, k, n = 70000, 32, 32000
    g = gen(2)
    x = whole_numbers(g, t, 40000, torch.bfloat16)[:, 39968:]  # rows 80000 bytes apart: 5.6 GB
    values, scales, z = plain.random_weight(g, (n,), k, 32, torch.bfloat16, True, DEV, whole=True)
    y = int4_linear(x, int4_pack(values), scales, z, group=32)
    w = plain.weight(values, scales, z, 32).T
    for rows in (slice(0, 3), slice(t // 2, t // 2 + 3), slice(67107, 67112), slice(t - 3, t)):
        assert torch.equal(y[rows], (x[rows].double() @ w).float().to(torch.bfloat16))


def test_codes_and_x_past_32_bits():
    """Codes of over 2^32 bytes (the last expert's lie behind them), and x of over 2^31 elements."""
    g = gen(3)
    experts, n, k, group = 33, 16384, 16384, 512
    codes = torch.randint(0, 256, (experts, n, k // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.exp2(torch.randint(-1, 2, (experts, n, k // group), generator=g, device=DEV).float()).to(torch.bfloat16)
    z = torch.randint(0, 17, scales.shape, generator=g, device=DEV, dtype=torch.uint8)
    for t in (2, 600):  # few rows an expert, and tiles of them
        x = whole_numbers(g, t, k, torch.bfloat16)
        ids = torch.full((t, 1), experts - 1, dtype=torch.int32, device=DEV)
        ids[0] = 0
        y = int4_expert_linear(x, codes, scales, expert_sort(ids, experts), z, group=group, gather=True, out_dtype=torch.float32)
        for rows, e in ((slice(0, 1), 0), (slice(1, t), experts - 1)):
            want = int4_linear(x[rows], codes[e], scales[e], z[e], group=group, out_dtype=torch.float32)
            assert torch.equal(y[rows], want)  # whole numbers, whose sums are exact in any order
    t = 2 ** 31 // k + 70
    x = torch.zeros(t, k, dtype=torch.bfloat16, device=DEV)
    x[-70:] = whole_numbers(g, 70, k, torch.bfloat16)
    y = int4_linear(x, codes[1, :100], scales[1, :100], z[1, :100], group=group, out_dtype=torch.float32)
    assert not bool(y[:-70].any())
    assert torch.equal(y[-70:], int4_linear(x[-70:], codes[1, :100], scales[1, :100], z[1, :100], group=group, out_dtype=torch.float32))


def test_awq_checkpoint():
    """A layer as an AWQ checkpoint stores it: column 8 c + (0, 2, 4, 6, 1, 3, 5, 7)[i] in bits 4 i of word c."""
    g = gen(6)
    k, n, group = 384, 72, 128
    values, scales, z = plain.random_weight(g, (n,), k, group, torch.float16, True, DEV, whole=True)
    z = z.clamp(max=15)

    def words(m):  # [rows, n] -> int32 [rows, n / 8]
        out = torch.zeros(m.shape[0], m.shape[1] // 8, dtype=torch.int64, device=DEV)
        for i, col in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
            out += m[:, col::8].long() << (4 * i)
        return torch.where(out >= 2 ** 31, out - 2 ** 32, out).int()

    w = int4_from_awq(words(values.t()), words(z.t()), scales.t())
    assert torch.equal(w.codes, plain.pack(values)) and torch.equal(w.scales, scales) and torch.equal(w.zeros, z)
    x = whole_numbers(g, 5, k, torch.float16)
    assert torch.equal(int4_linear(x, *w, group=group, out_dtype=torch.float32).double(), x.double() @ plain.weight(values, scales, z, group).T)


def test_products_repeat_bit_for_bit():
    g = gen(21)
    for t in (1, 40, 600, 2000):
        for dtype in HALVES:
            x = torch.randn(t, 4096, generator=g, device=DEV).to(dtype)
            values, scales, z = plain.random_weight(g, (700,), 4096, 128, dtype, True, DEV)
            codes = int4_pack(values)
            first = int4_linear(x, codes, scales, z)
            for _ in range(3):
                assert torch.equal(int4_linear(x, codes, scales, z), first)


def test_on_another_stream():
    g = gen(31)
    x = whole_numbers(g, 200, 512, torch.float16)
    values, scales, z = plain.random_weight(g, (300,), 512, 128, torch.float16, True, DEV, whole=True)
    codes, want = int4_pack(values), x.double() @ plain.weight(values, scales, z, 128).T
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = int4_linear(x, codes, scales, z, out_dtype=torch.float32)
    side.synchronize()
    assert torch.equal(y.double(), want)


EXPERT_CASES = [  # t, top, experts, k, n, group, dropped
    (1, 1, 1, 32, 16, 32, 0.0), (1, 4, 64, 512, 100, 128, 0.0), (4, 4, 64, 1024, 256, 128, 0.2), (7, 2, 8, 100, 33, 64, 0.3),
    (16, 2, 4, 160, 130, 32, 0.0), (50, 4, 16, 1000, 77, 128, 0.1), (64, 8, 128, 256, 64, 256, 0.5), (300, 2, 4, 320, 257, 64, 0.1),
    (500, 4, 8, 512, 384, 32, 0.0), (1500, 6, 60, 288, 200, 128, 0.05), (2000, 2, 3, 1056, 300, 128, 0.0), (40, 1, 5, 64, 48, 64, 1.0),
    (3000, 4, 8, 96, 2100, 32, 0.05), (9000, 2, 16, 544, 1500, 128, 0.0),
]


def routing(seed, t, top, experts, dropped):
    g = gen(seed)
    liked = torch.randn(t, experts, generator=g, device=DEV) + torch.randn(experts, generator=g, device=DEV)
    ids = liked.topk(min(top, experts), dim=1).indices.int()
    none = torch.rand(ids.shape, generator=g, device=DEV)
    ids = torch.where(none < dropped / 2, torch.full_like(ids, -1), ids)
    return torch.where(none > 1 - dropped / 2, torch.full_like(ids, experts + 3), ids).contiguous()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,top,experts,k,n,group,dropped", EXPERT_CASES)
def test_expert_linear_whole_numbers_are_exact(dtype, t, top, experts, k, n, group, dropped):
    g = gen(t + k)
    ids = routing(t + n, t, top, experts, 2.0 * dropped)
    top = ids.shape[1]
    sort = expert_sort(ids, experts)
    x = whole_numbers(g, t, k, dtype)
    values, scales, z = plain.random_weight(g, (experts, n), k, group, dtype, t % 2 == 0, DEV, whole=True)
    codes = int4_pack(values)
    bias = torch.randint(-64, 65, (experts, n), generator=g, device=DEV).to(dtype)
    rows = expert_gather(x, sort)
    order, _, offsets = mx_plain.sort(ids, experts)
    want = torch.zeros(t * top, n, dtype=torch.float64, device=DEV)
    biased = want.clone()
    for e in range(experts):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if b > a:
            want[a:b] = x.double()[(order[a:b] // top).to(DEV)] @ plain.weight(values[e], scales[e], z[e] if z is not None else None, group).T
            biased[a:b] = want[a:b] + bias[e].double()
    how = dict(group=group)
    assert torch.equal(int4_expert_linear(x, codes, scales, sort, z, gather=True, out_dtype=torch.float32, **how).double(), want)
    assert torch.equal(int4_expert_linear(rows, codes, scales, sort, z, out_dtype=torch.float32, **how).double(), want)
    assert torch.equal(int4_expert_linear(x, codes, scales, sort, z, bias, gather=True, **how), biased.float().to(dtype))
    wide = torch.full((t, k + 37), float("nan"), dtype=dtype, device=DEV)
    wide[:, 5:5 + k] = x
    out = torch.full((t * top, n), float("nan"), dtype=torch.float32, device=DEV)
    assert int4_expert_linear(wide[:, 5:5 + k], codes, scales, sort, z, gather=True, out=out, **how) is out
    assert torch.equal(out.double(), want)


def test_expert_linear_without_rows_or_terms():
    sort = expert_sort(torch.empty(0, 2, dtype=torch.int32, device=DEV), 4)
    values, scales, _ = plain.random_weight(gen(0), (4, 8), 64, 128, torch.bfloat16, False, DEV)
    assert int4_expert_linear(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), int4_pack(values), scales, sort).shape == (0, 8)
    sort = expert_sort(torch.tensor([[0, 3], [-1, 1]], dtype=torch.int32, device=DEV), 4)
    bias = torch.randn(4, 8, device=DEV)
    empty = torch.zeros(4, 8, 0, dtype=torch.uint8, device=DEV)
    y = int4_expert_linear(torch.empty(2, 0, dtype=torch.bfloat16, device=DEV), empty, empty.to(torch.bfloat16), sort, None, bias, gather=True,
                           out_dtype=torch.float32)
    assert torch.equal(y, torch.cat([bias[[0, 1, 3]], torch.zeros(1, 8, device=DEV)]))


@pytest.mark.parametrize("t", (20, 3000))
def test_bad_orders_and_offsets_stay_in_bounds(t):
    """A sort that expert_sort did not make gives wrong sums, never a bad address."""
    top, experts, k, n = 2, 4, 64, 400
    x = torch.randn(t, k, device=DEV).to(torch.bfloat16)
    values, scales, z = plain.random_weight(gen(0), (experts, n), k, 32, torch.bfloat16, True, DEV)
    for fill in (-2 ** 31, -7, 10 ** 6, 2 ** 31 - 1):
        bad = ExpertSort(*(torch.full(s, fill, dtype=torch.int32, device=DEV) for s in ((t * top,), (t, top), (experts + 1,))))
        assert int4_expert_linear(x, int4_pack(values), scales, bad, z, group=32, gather=True).shape == (t * top, n)
    torch.cuda.synchronize()


@pytest.mark.parametrize("t", (6, 700))
def test_in_a_graph(t):
    """One weight's product and experts', captured once and replayed on new tokens, with other work between."""
    g = gen(4)
    k, n, experts, top = 250, 136, 8, 2
    values, scales, z = plain.random_weight(g, (experts, n), k, 64, torch.bfloat16, True, DEV)
    codes = int4_pack(values)
    x = torch.empty(t, k, dtype=torch.bfloat16, device=DEV)
    ids, weights = torch.empty(t, top, dtype=torch.int32, device=DEV), torch.empty(t, top, device=DEV)

    def path():
        sort = expert_sort(ids, experts)
        y = int4_expert_linear(x, codes, scales, sort, z, group=64, gather=True)
        return int4_linear(x, codes[0], scales[0], z[0], group=64), expert_combine(y, weights, sort)

    def fill(seed):
        h = gen(seed)
        x.copy_(torch.randn(t, k, generator=h, device=DEV))
        ids.copy_(torch.randint(-1, experts, (t, top), generator=h, device=DEV))
        weights.copy_(torch.rand(t, top, generator=h, device=DEV))

    fill(0)
    path()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = path()
    for seed in range(1, 5):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        kept = [v.clone() for v in got]
        for a, b in zip(kept, path()):
            assert torch.equal(a, b)


# --------------------------------------------------------------------------- refusals
def test_refusals():
    x = torch.randn(4, 64, device=DEV).to(torch.bfloat16)
    values, scales, z = plain.random_weight(gen(0), (8,), 64, 32, torch.bfloat16, True, DEV)
    codes = int4_pack(values)
    sort = expert_sort(torch.zeros(4, 1, dtype=torch.int32, device=DEV), 1)
    call = lambda **change: int4_linear(**{**dict(x=x, codes=codes, scales=scales, zeros=z, group=32), **change})  # noqa: E731
    for change, message in (
            (dict(x=x.float()), "x must be torch.bfloat16 or torch.float16"), (dict(x=x[0, 0]), "at least one dimension"),
            (dict(codes=None), "codes must be defined"), (dict(scales=None), "scales must be defined"), (dict(codes=codes.cpu()), "must be a CUDA"),
            (dict(x=x[:, :32]), "do not fit"), (dict(codes=codes[0]), "dimension"), (dict(codes=codes.int()), "must be torch.uint8"),
            (dict(zeros=z.int()), "must be torch.uint8"), (dict(scales=scales.float()), "scales must be torch.bfloat16 or"),
            (dict(group=48), "power of two"), (dict(group=16), "power of two"), (dict(group=0), "power of two"), (dict(group=-32), "power of two"),
            (dict(group=64), "scales must have shape"), (dict(zeros=z[:, :1].contiguous()), "zeros must have shape"),
            (dict(scales=scales[:, :1]), "must be contiguous"), (dict(bias=torch.zeros(7, device=DEV)), "bias must have shape"),
            (dict(bias=torch.zeros(8, dtype=torch.int32, device=DEV)), "bias must be"), (dict(out_dtype=torch.int32), "out_dtype must be"),
            (dict(out=torch.empty(4, 9, dtype=torch.bfloat16, device=DEV)), "out must be"),
            (dict(codes=torch.zeros(8 * 32 + 1, dtype=torch.uint8, device=DEV)[1:].view(8, 32)), "16-byte aligned")):
        with pytest.raises(ValueError, match=message):
            call(**change)
    with pytest.raises(ValueError, match="sort has 1 experts"):
        int4_expert_linear(x, codes.repeat(2, 1, 1), scales.repeat(2, 1, 1), sort, z.repeat(2, 1, 1), group=32)
    for bad in (dict(x=x.detach().requires_grad_()), dict(scales=scales.detach().requires_grad_()),
                dict(bias=torch.zeros(8, device=DEV, requires_grad=True))):
        with pytest.raises(RuntimeError, match="has no gradient"):
            call(**bad)
    with pytest.raises(RuntimeError, match="has no gradient"):
        int4_expert_linear(x.detach().requires_grad_(), codes[None], scales[None], sort, z[None], group=32)
    with pytest.raises(RuntimeError, match="out must not require a gradient"):
        call(out=torch.zeros(4, 8, dtype=torch.bfloat16, device=DEV, requires_grad=True))
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            call(x=forward_ad.make_dual(x, torch.ones_like(x)))
