"""Tokens to their experts and back, and the experts' products, against plain forms."""
import pytest
import torch

from mpserve_amd.experts import ExpertSort, expert_combine, expert_gather, expert_sort, mxfp4_expert_linear
from tests import mx_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = (torch.bfloat16, torch.float16, torch.float32)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def routing(seed, t, top, experts, dropped=0.1, dtype=torch.int32):
    """Different experts a token, some of them liked more, some pairs of none (ids below 0 and from `experts` on)."""
    g = gen(seed)
    liked = torch.randn(t, experts, generator=g, device=DEV) + torch.randn(experts, generator=g, device=DEV)
    ids = liked.topk(min(top, experts), dim=1).indices
    none = torch.rand(ids.shape, generator=g, device=DEV)
    ids = torch.where(none < dropped / 2, torch.full_like(ids, -1), ids)
    ids = torch.where(none > 1 - dropped / 2, torch.full_like(ids, experts + 3), ids)
    return ids.to(dtype).contiguous()


def check_sort(ids, experts):
    got = expert_sort(ids, experts)
    order, positions, offsets = plain.sort(ids, experts)
    assert torch.equal(got.offsets.cpu().long(), offsets)
    assert torch.equal(got.positions.cpu().long(), positions)
    assert torch.equal(got.order.cpu().long(), order)
    return got


@pytest.mark.parametrize("dtype", (torch.int32, torch.int64))
@pytest.mark.parametrize("t,top,experts", [(0, 2, 4), (1, 1, 1), (1, 8, 1024), (3, 2, 8), (37, 2, 8), (64, 1, 60), (100, 4, 64), (513, 6, 60),
                                           (1000, 8, 128), (4096, 4, 64), (5000, 3, 1000), (8192, 8, 128), (40000, 8, 256)])
def test_sort(dtype, t, top, experts):
    check_sort(routing(t + top, t, top, experts, 0.1, dtype), experts)


@pytest.mark.parametrize("pairs", (1, 63, 64, 65, 1023, 1024, 1025, 20000, 300001))
def test_sort_uneven(pairs):
    """All pairs of one expert, of none, of the last one, and experts that nothing goes to."""
    for e in (0, 5, 7, -1, 8, 2 ** 31 - 1, -2 ** 31):
        check_sort(torch.full((pairs, 1), e, dtype=torch.int32, device=DEV), 8)
    check_sort((torch.arange(pairs, device=DEV) % 3 * 3).view(-1, 1), 8)
    check_sort(torch.arange(pairs, device=DEV).flip(0).view(-1, 1), 1024)
    far = torch.randint(0, 4, (pairs, 1), generator=gen(1), device=DEV) + 2 ** 32  # in 64 bits none of these is an expert
    check_sort(far, 8)
    check_sort(far - 2 ** 33, 8)


def plain_combine(y, weights, ids, sort):
    """In 64 bits, with the sum of the terms' magnitudes."""
    positions = sort.positions.long()
    there = (positions >= 0).unsqueeze(-1)
    rows = torch.where(there, y.double()[positions.clamp(min=0)], torch.zeros((), dtype=torch.float64, device=DEV))
    terms = rows * torch.where(there, weights.double().unsqueeze(-1), torch.zeros((), dtype=torch.float64, device=DEV))
    return terms.sum(1), terms.abs().sum(1)


CASES = [(1, 1, 1, 1), (3, 2, 4, 8), (5, 2, 8, 33), (37, 2, 8, 1001), (64, 4, 64, 256), (200, 8, 128, 136), (33, 6, 60, 4100), (700, 1, 16, 512)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,top,experts,width", CASES)
def test_gather_and_combine(dtype, t, top, experts, width):
    g = gen(t)
    ids = routing(t, t, top, experts)
    sort = expert_sort(ids, experts)
    top = ids.shape[1]
    x = torch.randn(t, width, generator=g, device=DEV).to(dtype)
    kept = int(sort.offsets[-1])
    want = torch.zeros(t * top, width, dtype=dtype, device=DEV)
    want[:kept] = x[(sort.order[:kept] // top).long()]
    assert torch.equal(expert_gather(x, sort), want)
    assert torch.equal(expert_gather(x.t().contiguous().t(), sort), want)
    y = torch.randn(t * top, width, generator=g, device=DEV).to(dtype)
    y[kept:] = float("nan")  # never read
    for wtype in (torch.float32, dtype):
        weights = torch.rand(t, top, generator=g, device=DEV).to(wtype)
        exact, size = plain_combine(y, weights, ids, sort)
        plain.close(expert_combine(y, weights, sort), exact, size, 2 * top)


@pytest.mark.parametrize("dtype", TYPES[:2])
def test_gather_copies_bits(dtype):
    """Every value of 16 bits, signalling NaN too, in a row's whole pieces and in the part at its end."""
    x = torch.arange(65536, dtype=torch.int32, device=DEV).to(torch.uint16).view(-1, 1).repeat(1, 11).view(dtype)
    sort = expert_sort(torch.zeros(65536, 1, dtype=torch.int32, device=DEV), 1)
    assert torch.equal(expert_gather(x, sort).view(torch.int16), x.view(torch.int16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,top,experts,width", CASES)
def test_gradients_match_formulas(dtype, t, top, experts, width):
    g = gen(t + 1)
    ids = routing(t, t, top, experts)
    sort = expert_sort(ids, experts)
    top = ids.shape[1]
    kept, token = int(sort.offsets[-1]), None
    token = (sort.order[:kept] // top).long()
    x, dout = (torch.randn(t, width, generator=g, device=DEV).to(dtype) for _ in range(2))
    y, drows = (torch.randn(t * top, width, generator=g, device=DEV).to(dtype) for _ in range(2))
    y[kept:], drows[kept:] = float("nan"), float("inf")  # in places of pairs of no expert: never read
    for wtype in {torch.float32, dtype}:
        weights = torch.rand(t, top, generator=g, device=DEV).to(wtype)
        leaves = [v.clone().requires_grad_() for v in (x, y, weights)]
        rows, out = expert_gather(leaves[0], sort), expert_combine(leaves[1], leaves[2], sort)
        dx, dy, dw = torch.autograd.grad((rows, out), leaves, (drows, dout))
        assert dx.dtype == dtype and dy.dtype == dtype and dw.dtype == wtype
        ones = torch.ones(t, top, device=DEV)
        plain.close(dx, *plain_combine(drows, ones, ids, sort), top)
        want = torch.zeros(t * top, width, dtype=torch.float64, device=DEV)
        want[:kept] = weights.double().view(-1)[sort.order[:kept].long()].unsqueeze(1) * dout.double()[token]
        plain.close(dy, want, want.abs(), 1)
        terms = torch.zeros(t * top, width, dtype=torch.float64, device=DEV)
        terms[sort.order[:kept].long()] = y.double()[:kept] * dout.double()[token]
        plain.close(dw, terms.sum(1).view(t, top), terms.abs().sum(1).view(t, top), width + 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,top,experts,width", CASES + [(300, 4, 16, 4096)])
def test_one_gradient_alone(dtype, t, top, experts, width):
    """The gradient of y or of the weights alone is what it is beside the other one; the weights' makes no rows
    for y, and that of y keeps no y."""
    g = gen(t + 2)
    sort = expert_sort(routing(t, t, top, experts), experts)
    top = sort.positions.shape[1]
    y, dout = torch.randn(t * top, width, generator=g, device=DEV).to(dtype), torch.randn(t, width, generator=g, device=DEV).to(dtype)
    weights = torch.rand(t, top, generator=g, device=DEV)
    both = [v.clone().requires_grad_() for v in (y, weights)]
    dy, dw = torch.autograd.grad(expert_combine(*both, sort), both, dout)
    w = weights.clone().requires_grad_()
    out = expert_combine(y, w, sort)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    (alone,) = torch.autograd.grad(out, w, dout)
    assert torch.equal(alone, dw)
    if y.numel() * y.element_size() >= 1 << 20:
        assert torch.cuda.max_memory_allocated() - before < y.numel() * y.element_size()
    leaf = y.clone().requires_grad_()
    other = leaf * 1
    out = expert_combine(other, weights, sort)
    other.zero_()  # not kept for this gradient
    (alone,) = torch.autograd.grad(out, leaf, dout)
    assert torch.equal(alone, dy)


def test_gradients_match_differences():
    """The combine is linear in y and in the weights, so a difference is exact but for rounding: with whole
    numbers it is exact."""
    t, top, experts, width = 20, 3, 6, 40
    g = gen(8)
    ids = routing(8, t, top, experts)
    sort = expert_sort(ids, experts)
    whole = lambda *s: torch.randint(-4, 5, s, generator=g, device=DEV).float()  # noqa: E731
    x, y, weights, dout, drows = whole(t, width), whole(t * top, width), whole(t, top), whole(t, width), whole(t * top, width)

    def loss(x, y, weights):
        return (expert_combine(y, weights, sort) * dout).sum() + (expert_gather(x, sort) * drows).sum()

    leaves = [v.clone().requires_grad_() for v in (x, y, weights)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i in range(3):
        for _ in range(4):
            step = whole(*leaves[i].shape)
            moved = [x, y, weights]
            moved[i] = moved[i] + step
            assert float(loss(*moved) - loss(x, y, weights)) == float((grads[i] * step).sum())


EXPERT_CASES = [  # t, top, experts, k, n, dropped
    (1, 1, 1, 32, 16, 0.0), (1, 4, 64, 512, 100, 0.0), (4, 4, 64, 1024, 256, 0.2), (7, 2, 8, 100, 33, 0.3), (16, 2, 4, 160, 130, 0.0),
    (50, 4, 16, 1000, 77, 0.1), (64, 8, 128, 256, 64, 0.5), (300, 2, 4, 320, 257, 0.1), (500, 4, 8, 512, 384, 0.0),
    (1500, 6, 60, 288, 200, 0.05), (2000, 2, 3, 1056, 300, 0.0), (40, 1, 5, 64, 48, 1.0),
    (3000, 4, 8, 96, 2100, 0.05), (9000, 2, 16, 544, 1500, 0.0),
]


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
@pytest.mark.parametrize("t,top,experts,k,n,dropped", EXPERT_CASES)
def test_expert_linear_whole_numbers_are_exact(dtype, t, top, experts, k, n, dropped):
    g = gen(t + k)
    ids = routing(t + n, t, top, experts, 2.0 * dropped)
    top = ids.shape[1]
    sort = expert_sort(ids, experts)
    x = torch.randint(-8, 9, (t, k), generator=g, device=DEV).to(dtype)
    codes, scales = plain.random_weight(g, (experts, n), k, DEV, 126, 129)
    bias = torch.randint(-64, 65, (experts, n), generator=g, device=DEV).to(dtype)
    rows = expert_gather(x, sort)
    order, _, offsets = plain.sort(ids, experts)
    want = torch.zeros(t * top, n, dtype=torch.float64, device=DEV)
    biased = want.clone()
    for e in range(experts):
        a, b = int(offsets[e]), int(offsets[e + 1])
        if b > a:
            want[a:b] = x.double()[(order[a:b] // top).to(DEV)] @ plain.dequantize(codes[e], scales[e], k).T
            biased[a:b] = want[a:b] + bias[e].double()
    assert torch.equal(mxfp4_expert_linear(x, codes, scales, sort, gather=True, out_dtype=torch.float32).double(), want)
    assert torch.equal(mxfp4_expert_linear(rows, codes, scales, sort, out_dtype=torch.float32).double(), want)
    assert torch.equal(mxfp4_expert_linear(x, codes, scales, sort, bias, gather=True), biased.float().to(dtype))
    wide = torch.randint(-8, 9, (t, k + 37), generator=g, device=DEV).to(dtype)
    wide[:, 5:5 + k] = x
    out = torch.full((t * top, n), float("nan"), dtype=torch.float32, device=DEV)
    assert mxfp4_expert_linear(wide[:, 5:5 + k], codes, scales, sort, gather=True, out=out) is out
    assert torch.equal(out.double(), want)


@pytest.mark.parametrize("t,top,experts,k,n,dropped", EXPERT_CASES)
def test_mxfp4_rows_of_experts_are_exact(t, top, experts, k, n, dropped):
    """MXFP4 x in the sorted order, which the C entry takes: the same products with whole numbers, through
    the kernels of few and of many rows, uneven loads and pairs of no expert."""
    import ctypes

    from mpserve_amd import _native

    g = gen(t + k)
    ids = routing(t + n, t, top, experts, 2.0 * dropped)
    rows = ids.numel()
    sort = expert_sort(ids, experts)
    xc, xs = plain.random_weight(g, (rows,), k, DEV, 126, 129)
    codes, scales = plain.random_weight(g, (experts, n), k, DEV, 126, 129)
    bias = torch.randint(-64, 65, (experts, n), generator=g, device=DEV).float()
    x = plain.dequantize(xc, xs, k)
    offsets = plain.sort(ids, experts)[2].tolist()
    want = torch.zeros(rows, n, dtype=torch.float64, device=DEV)
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        if b > a:
            want[a:b] = x[a:b] @ plain.dequantize(codes[e], scales[e], k).T + bias[e].double()
    out = torch.full((rows, n), float("nan"), device=DEV)
    p = _native.MpsMxfp4Product(x=xc.data_ptr(), x_scales=xs.data_ptr(), w=codes.data_ptr(), w_scales=scales.data_ptr(), bias=bias.data_ptr(),
                                out=out.data_ptr(), offsets=sort.offsets.data_ptr(), rows=rows, n=n, k=k, experts=experts, top=ids.shape[1],
                                x_type=_native.MPS_TYPE_MXFP4, bias_type=_native.MPS_TYPE_F32, out_type=_native.MPS_TYPE_F32)
    _native.check(_native.lib().mps_mxfp4_multiply(p, None, 0, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)))
    assert torch.equal(out.double(), want)


def test_expert_linear_without_rows_or_terms():
    sort = expert_sort(torch.empty(0, 2, dtype=torch.int32, device=DEV), 4)
    codes, scales = plain.random_weight(gen(0), (4, 8), 64, DEV)
    assert mxfp4_expert_linear(torch.empty(0, 64, dtype=torch.bfloat16, device=DEV), codes, scales, sort).shape == (0, 8)
    ids = torch.tensor([[0, 3], [-1, 1]], dtype=torch.int32, device=DEV)
    sort = expert_sort(ids, 4)
    bias = torch.randn(4, 8, device=DEV)
    y = mxfp4_expert_linear(torch.empty(2, 0, dtype=torch.bfloat16, device=DEV), codes[:, :, :0].contiguous(), scales[:, :, :0].contiguous(),
                            sort, bias, gather=True, out_dtype=torch.float32)
    assert torch.equal(y, torch.cat([bias[[0, 1, 3]], torch.zeros(1, 8, device=DEV)]))


def test_bad_orders_and_offsets_stay_in_bounds():
    """A sort that expert_sort did not make gives wrong sums, never a bad address."""
    t, top, experts, k, n = 20, 2, 4, 64, 40
    x = torch.randn(t, k, device=DEV).to(torch.bfloat16)
    codes, scales = plain.random_weight(gen(0), (experts, n), k, DEV)
    weights = torch.rand(t, top, device=DEV, requires_grad=True)
    for fill in (-2 ** 31, -7, 10 ** 6, 2 ** 31 - 1):
        bad = ExpertSort(*(torch.full(s, fill, dtype=torch.int32, device=DEV) for s in ((t * top,), (t, top), (experts + 1,))))
        y = mxfp4_expert_linear(x, codes, scales, bad, gather=True)
        rows = expert_gather(x, bad).requires_grad_()
        out = expert_combine(rows, weights, bad)
        torch.autograd.grad(out.sum(), (rows, weights))
        assert y.shape == (t * top, n) and out.shape == (t, k)
    torch.cuda.synchronize()


def test_bad_offsets_of_many_rows_stay_in_bounds():
    """Every second expert has all of 4e8 rows, so that the counts of tiles pass 2^31: no tile may come out of
    what is left of them."""
    rows, experts = 400_000_000, 1024
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB of free memory")
    offsets = torch.tensor([0, 2 ** 31 - 1], dtype=torch.int32, device=DEV).repeat(experts // 2 + 1)[:experts + 1].contiguous()
    order = torch.zeros(rows, dtype=torch.int32, device=DEV)
    codes, scales = plain.random_weight(gen(0), (experts, 1), 32, DEV)
    x = torch.zeros(1, 32, dtype=torch.bfloat16, device=DEV).expand(rows, 32)
    y = mxfp4_expert_linear(x, codes, scales, ExpertSort(order, order.view(rows, 1), offsets))
    torch.cuda.synchronize()
    assert y.shape == (rows, 1)


def test_no_second_gradient():
    """A graph of the gradients may be asked for; a gradient through it is refused."""
    sort = expert_sort(torch.tensor([[0, 1], [2, -1]], dtype=torch.int32, device=DEV), 3)
    x = torch.randn(2, 8, device=DEV, requires_grad=True)
    weights = torch.rand(2, 2, device=DEV, requires_grad=True)
    out = expert_combine(expert_gather(x, sort), weights, sort)
    once = torch.autograd.grad(out.square().sum(), (x, weights), retain_graph=True)
    again = torch.autograd.grad(out.square().sum(), (x, weights), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, again))
    with pytest.raises(RuntimeError, match="once_differentiable"):
        again[0].sum().backward()


def test_no_forward_mode():
    """A dual tensor requires no gradient, but a result without its tangent would be wrong."""
    from torch.autograd import forward_ad

    from mpserve_amd.mxfp4 import mxfp4_linear, mxfp4_matmul, mxfp4_quantize

    sort = expert_sort(torch.tensor([[0, 1], [2, -1]], dtype=torch.int32, device=DEV), 3)
    x, y, w, bias = torch.randn(2, 32, device=DEV), torch.randn(4, 32, device=DEV), torch.rand(2, 2, device=DEV), torch.randn(8, device=DEV)
    half = x.to(torch.bfloat16)
    codes, scales = plain.random_weight(gen(0), (8,), 32, DEV)
    codes3, scales3 = plain.random_weight(gen(0), (3, 8), 32, DEV)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: expert_gather(dual(x), sort), lambda: expert_combine(dual(y), w, sort), lambda: expert_combine(y, dual(w), sort),
                     lambda: mxfp4_quantize(dual(x)), lambda: mxfp4_linear(dual(half), codes, scales),
                     lambda: mxfp4_linear(half, codes, scales, dual(bias)), lambda: mxfp4_matmul(codes, scales, codes, scales, dual(bias)),
                     lambda: mxfp4_expert_linear(dual(half), codes3, scales3, sort, gather=True)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
        assert expert_combine(expert_gather(x, sort), w, sort).shape == (2, 32)


def test_whole_path_in_a_graph():
    """Sort, product, weighted sum and gradients, captured once and replayed on new routings and tokens."""
    t, top, experts, k, n = 50, 4, 16, 256, 136
    g = gen(4)
    codes, scales = plain.random_weight(g, (experts, n), k, DEV)
    x = torch.empty(t, k, dtype=torch.bfloat16, device=DEV)
    ids, weights = torch.empty(t, top, dtype=torch.int32, device=DEV), torch.empty(t, top, device=DEV)

    def path():
        w = weights.detach().requires_grad_()
        sort = expert_sort(ids, experts)
        y = mxfp4_expert_linear(x, codes, scales, sort, gather=True)
        rows = expert_gather(x, sort)
        out = expert_combine(y, w, sort)
        (dw,) = torch.autograd.grad(out, w, out.detach())
        return [out.detach(), dw, rows, sort.positions]

    def fill(seed):
        x.copy_(torch.randn(t, k, generator=gen(seed), device=DEV))
        ids.copy_(routing(seed, t, top, experts))
        weights.copy_(torch.rand(t, top, generator=gen(seed), device=DEV))

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        path()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = path()
    for seed in (1, 2, 3, 4):
        fill(seed)
        want = [v.clone() for v in path()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_block_of_experts(dtype):
    """The block that serves MXFP4 experts, against 64-bit arithmetic on the same MXFP4 weights. Every step
    rounds to 16 bits: products, silu, its product with up, the weighted sum and the shared expert's
    part, and MXFP4 activations are the quantized ones exactly. Each is off by its roundoff, amplified by
    less than the two products' condition, which the sum of magnitudes of the last one covers."""
    from mpserve_amd.mxfp4 import mxfp4_quantize
    from mpserve_amd.mxfp4_experts import Mxfp4Experts, decoded_weight

    t, hidden, ffn, experts, top = 45, 256, 160, 8, 3
    g = gen(6)
    device = torch.device(DEV, torch.cuda.current_device())
    gu, dn = decoded_weight((experts, 2 * ffn, hidden), 1, device), decoded_weight((experts, hidden, ffn), 2, device)
    sgu, sdn = decoded_weight((2 * ffn, hidden), 3, device), decoded_weight((hidden, ffn), 4, device)
    block = Mxfp4Experts(gu, dn, top, shared=(sgu, sdn))
    x = torch.randn(t, hidden, generator=g, device=DEV).to(dtype)
    logits = torch.randn(t, experts, generator=g, device=DEV)
    out = block(x, logits)
    value = lambda pair, k: plain.dequantize(*pair, k)  # noqa: E731

    def gated(h):
        a, b = h.chunk(2, -1)
        return a * torch.sigmoid(a) * b

    best, ids = logits.topk(top, dim=1)
    w = torch.softmax(best, 1).double()
    wgu, wdn = value(block.gate_up, hidden), value(block.down, ffn)
    want, size = torch.zeros(t, hidden, dtype=torch.float64, device=DEV), torch.zeros(t, hidden, dtype=torch.float64, device=DEV)
    for e in range(experts):
        token, slot = torch.where(ids == e)
        h = gated(x[token].double() @ wgu[e].T)
        want[token] += w[token, slot].unsqueeze(1) * (h @ wdn[e].T)
        size[token] += w[token, slot].unsqueeze(1) * (h.abs() @ wdn[e].abs().T)
    h = gated(value(mxfp4_quantize(x), hidden) @ value(block.shared[0], hidden).T)
    want, size = want + h @ value(block.shared[1], ffn).T, size + h.abs() @ value(block.shared[1], ffn).abs().T
    # gate, up, silu and their product: each rounded, silu's slope is below 1.1, so 4.1 roundoffs of h at most
    # relative to |gate * up| (which silu's factor shrinks: twice that is taken); the products, sums and the
    # last addition round four times more.
    u = plain.ROUNDOFF[dtype]
    off = (out.double() - want).abs()
    assert bool((off <= 16 * u * size + 4 * u * want.abs() + 2.0 ** -24).all()), float((off / size).max() / u)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float16))
def test_block_of_experts_that_rounds_less(dtype):
    """With ``rounded=False`` the only roundings to 16 bits are those of gate and up, of silu (whose slope is below
    1.1) and of its product with up, 4.1 roundoffs of |gate * up|, and that of the answer. FP32 sums of n terms are
    off by n * 2^-23 of their terms' magnitudes. The default, which rounds the shared expert's activations to
    4 bits, is far outside."""
    from mpserve_amd.mxfp4_experts import Mxfp4Experts

    t, hidden, ffn, experts, top = 45, 256, 160, 8, 3
    g = gen(16)
    weights = [0.05 * torch.randn(s, generator=g, device=DEV) for s in ((experts, 2 * ffn, hidden), (experts, hidden, ffn), (2 * ffn, hidden), (hidden, ffn))]
    block = Mxfp4Experts(weights[0], weights[1], top, shared=(weights[2], weights[3]), rounded=False)
    x = torch.randn(t, hidden, generator=g, device=DEV).to(dtype)
    logits = torch.randn(t, experts, generator=g, device=DEV)
    best, ids = logits.topk(top, dim=1)
    w = torch.softmax(best, 1).double()
    u, step = plain.ROUNDOFF[dtype], 2.0 ** -23

    def expert(rows, gate_up, down):
        """(answer, bound of its error before it is rounded)"""
        (a, b), (big_a, big_b) = (rows @ gate_up.T).chunk(2, -1), (rows.abs() @ gate_up.abs().T).chunk(2, -1)
        h = a * torch.sigmoid(a) * b
        off = 4.2 * u * (a * b).abs() + 1.2 * hidden * step * (big_a * b.abs() + big_b * a.abs() + hidden * step * big_a * big_b)
        return h @ down.T, (off + (ffn + top + 2) * step * (h.abs() + off)) @ down.abs().T

    gu, dn = plain.dequantize(*block.gate_up, hidden), plain.dequantize(*block.down, ffn)
    want, bound = expert(x.double(), plain.dequantize(*block.shared[0], hidden), plain.dequantize(*block.shared[1], ffn))
    for e in range(experts):
        token, slot = torch.where(ids == e)
        y, off = expert(x[token].double(), gu[e], dn[e])
        want[token] += w[token, slot].unsqueeze(1) * y
        bound[token] += w[token, slot].unsqueeze(1) * off
    bound = bound + u * (want.abs() + bound) + 2.0 ** -25
    out = block(x, logits)
    assert out.dtype == dtype and bool(((out.double() - want).abs() <= bound).all())
    block.rounded = True
    assert not bool(((block(x, logits).double() - want).abs() <= bound).all())


def test_refusals():
    ids = routing(0, 6, 2, 4)
    sort = expert_sort(ids, 4)
    x = torch.randn(6, 64, device=DEV).to(torch.bfloat16)
    codes, scales = plain.random_weight(gen(0), (4, 8), 64, DEV)
    w = torch.rand(6, 2, device=DEV)
    for call, message in (
            (lambda: expert_sort(ids.cpu(), 4), "ids must be a CUDA tensor"),
            (lambda: expert_sort(ids.float(), 4), "ids must be torch.int32 or torch.int64"),
            (lambda: expert_sort(ids.view(-1), 4), "ids must have 2 dimensions"),
            (lambda: expert_sort(ids.t(), 4), "ids must be contiguous"),
            (lambda: expert_sort(ids, 0), "num_experts must be in"),
            (lambda: expert_sort(ids, 1025), "num_experts must be in"),
            (lambda: expert_gather(x[:5], sort), "x must have shape"),
            (lambda: expert_gather(x.int(), sort), "x must be torch.bfloat16"),
            (lambda: expert_gather(x, ExpertSort(sort.order[:4], sort.positions, sort.offsets)), "sort must be what expert_sort returns"),
            (lambda: expert_gather(x, ExpertSort(sort.order.long(), sort.positions, sort.offsets)), "sort.order must be torch.int32"),
            (lambda: expert_combine(x, w, sort), "y must have shape"),
            (lambda: expert_combine(x.repeat(2, 1), w[:, :1], sort), "weights must have shape"),
            (lambda: expert_combine(x.repeat(2, 1), w.int(), sort), "weights must be torch.bfloat16"),
            (lambda: mxfp4_expert_linear(x, codes, scales, sort), "x must have shape"),
            (lambda: mxfp4_expert_linear(x.float(), codes, scales, sort, gather=True), "x must be torch.bfloat16 or torch.float16"),
            (lambda: mxfp4_expert_linear(x, codes[:3], scales[:3], sort, gather=True), "sort has 4 experts and codes 3"),
            (lambda: mxfp4_expert_linear(x[:, :32], codes, scales, sort, gather=True), "do not fit"),
            (lambda: mxfp4_expert_linear(x, codes, scales, sort, torch.zeros(8, device=DEV), gather=True), "bias must have shape"),
            (lambda: mxfp4_expert_linear(x, codes[0], scales[0], sort, gather=True), "dimension")):
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(RuntimeError, match="has no gradient"):
        mxfp4_expert_linear(x.detach().requires_grad_(), codes, scales, sort, gather=True)
