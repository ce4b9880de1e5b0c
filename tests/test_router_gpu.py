"""The experts' router and the balance loss, with their gradients, against plain 64-bit forms."""
import pytest
import torch

from mpserve_amd.experts import expert_balance, expert_combine, expert_gather, expert_route, expert_sort, int4_expert_linear
from mpserve_amd.int4 import int4_pack
from tests import int4_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = (torch.bfloat16, torch.float16, torch.float32)
#: Half a step of each type, relative, and half the smallest step of FP16.
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}
NONE = float("-inf")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def logits_of(seed, t, experts, dtype, masked=0.0, padded=0.0, spread=1.0):
    g = gen(seed)
    logits = spread * (torch.randn(t, experts, generator=g, device=DEV) + torch.randn(experts, generator=g, device=DEV))
    if masked:
        logits = torch.where(torch.rand(t, experts, generator=g, device=DEV) < masked, torch.full_like(logits, NONE), logits)
    if padded:
        logits = torch.where(torch.rand(t, 1, generator=g, device=DEV) < padded, torch.full_like(logits, NONE), logits)
    return logits.to(dtype)


def share_error(experts):
    """Relative: exp to 2 steps of FP32 in numerator and denominator (and its argument, a difference rounded at a size of
    at most 32: 2^-19 of 1), sums of up to `experts` terms, a quotient and a factor."""
    return 2.0 ** -18 + (experts + 8) * 2.0 ** -24


CASES = [(1, 1, 1), (1, 2, 2), (3, 8, 2), (37, 8, 8), (5, 16, 3), (64, 17, 4), (20, 32, 8), (33, 60, 6), (100, 64, 4), (7, 65, 65), (50, 128, 8),
         (41, 129, 5), (30, 256, 8), (9, 300, 20), (6, 512, 10), (5, 700, 70), (3, 1024, 8), (2, 1024, 1024), (3000, 64, 4), (9, 4, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores", ("softmax", "sigmoid"))
@pytest.mark.parametrize("t,experts,top", CASES)
def test_route(dtype, scores, t, experts, top):
    for masked, padded in ((0.0, 0.0), (0.4, 0.2)):
        logits = logits_of(t + experts, t, experts, dtype, masked, padded)
        bias = torch.randn(experts, generator=gen(5), device=DEV)
        for b in (None, bias):
            for normalize, scale in ((True, 1.0), (False, 2.5)):
                ids, weights = expert_route(logits, top, scores=scores, bias=b, normalize=normalize, scale=scale)
                assert ids.shape == weights.shape == (t, top) and ids.dtype == torch.int32 and weights.dtype == torch.float32
                want_ids, want = plain.route(logits, top, scores, b, normalize, scale)
                assert torch.equal(ids, want_ids)
                off = (weights.double() - want).abs()
                assert bool((off <= share_error(experts) * want.abs() + 2.0 ** -126).all()), float(off.max())


def test_route_ties_go_to_the_lowest_expert():
    for experts, top in ((8, 3), (64, 8), (128, 8), (200, 9), (600, 4), (1000, 40)):
        for dtype in TYPES:
            logits = torch.randint(-2, 3, (50, experts), generator=gen(experts), device=DEV).to(dtype)
            logits[0], logits[1] = 0.0, NONE
            logits[2, ::2], logits[2, 1::2] = -0.0, 0.0  # the two zeros are equal
            for bias in (None, torch.zeros(experts, device=DEV)):
                ids, _ = expert_route(logits, top, bias=bias)
                assert torch.equal(ids, plain.route(logits, top, "softmax", bias)[0])


def test_route_with_few_experts_left():
    """Masks that leave fewer experts than are wanted, or none, by logits and by the bias."""
    logits = torch.full((5, 60), NONE, device=DEV)
    logits[1, 59], logits[2, 3], logits[2, 40], logits[3] = 2.0, -1e30, 5.0, torch.finfo(torch.float32).min
    logits[4] = torch.arange(60, device=DEV)
    ids, weights = expert_route(logits, 4)
    assert ids.tolist() == [[-1] * 4, [59, -1, -1, -1], [40, 3, -1, -1], [0, 1, 2, 3], [59, 58, 57, 56]]
    assert weights[0].tolist() == [0] * 4 and weights[1].tolist() == [1, 0, 0, 0] and weights[2].tolist() == [1, 0, 0, 0]
    assert weights[3].tolist() == [0.25] * 4
    bias = torch.full((60,), NONE, device=DEV)
    bias[7] = 1.0
    ids, weights = expert_route(logits, 2, scores="sigmoid", bias=bias)
    assert ids.tolist() == [[-1, -1], [-1, -1], [-1, -1], [7, -1], [7, -1]]
    assert weights[3:, 0].tolist() == [1, 1]  # of the lowest logits too, whose sigmoids are all 0 in FP32


def test_route_near_the_border():
    """Scores that FP32 cannot tell apart, but 64 bits can."""
    logits = torch.full((2, 128), -5.0, device=DEV)
    logits[:, 100], logits[:, 7] = 12.0, 12.0 - 2.0 ** -19
    logits[1, 100], logits[1, 7] = logits[0, 7], logits[0, 100]
    zero = torch.zeros(128, device=DEV)
    assert expert_route(logits, 1, scores="sigmoid", bias=zero).ids.view(-1).tolist() == [100, 7]
    assert expert_route(logits, 1, scores="softmax", bias=zero).ids.view(-1).tolist() == [100, 7]


def test_route_keeps_nan_in_its_row():
    logits = logits_of(1, 6, 64, torch.float32)
    clean = expert_route(logits, 4)
    logits[2, 10], logits[4, 11] = float("nan"), float("inf")
    for normalize in (True, False):
        ids, weights = expert_route(logits, 4, normalize=normalize)
        assert bool((ids[2] != 10).all()) and int(ids[4, 0]) == 11
        assert bool(torch.isnan(weights[2]).all()) and bool(torch.isnan(weights[4]).any())
        rest = [0, 1, 3, 5]
        assert torch.equal(ids[rest], clean.ids[rest]) and bool(torch.isfinite(weights[rest]).all())
    ids, weights = expert_route(logits, 4, scores="sigmoid", normalize=False)
    assert bool(torch.isfinite(weights).all()) and float(weights[4, 0]) == 1.0  # a NaN of an expert that is not taken


@pytest.mark.parametrize("experts", (64, 256, 1000))
def test_route_with_a_bias_keeps_nan_in_its_row(experts):
    """Softmax scores that are all NaN still choose, by the bias, and give NaN for weights."""
    logits = logits_of(1, 6, experts, torch.float32)
    bias = torch.randn(experts, generator=gen(5), device=DEV)
    bias[20:40] = bias[3]  # ties, for which keys are made again in 64 bits
    clean = expert_route(logits, 30, bias=bias)
    logits[2, 10], logits[4, 11], logits[2, 12] = float("nan"), float("inf"), NONE
    for normalize in (True, False):
        ids, weights = expert_route(logits, 30, bias=bias, normalize=normalize)
        for row, without in ((2, (10, 12)), (4, ())):
            order = sorted((e for e in range(experts) if e not in without), key=lambda e: (-float(bias[e]), e))
            assert ids[row].tolist() == order[:30]
            assert bool(torch.isnan(weights[row]).all())
        rest = [0, 1, 3, 5]
        assert torch.equal(ids[rest], clean.ids[rest]) and bool(torch.isfinite(weights[rest]).all())
    ids, weights = expert_route(logits, 4, scores="sigmoid", bias=bias)
    assert bool((ids[2] != 10).all()) and bool(torch.isfinite(weights).all())


@pytest.mark.parametrize("scores", ("softmax", "sigmoid"))
@pytest.mark.parametrize("experts,top", ((20, 6), (128, 8), (256, 8), (1000, 100)))
def test_route_with_keys_that_are_near_one_another(scores, experts, top):
    """Rows beside one another, of keys that lie within FP32's errors in groups, that are all alike, that are masked but for a few, and
    that are far apart; the order is that of 64 bits."""
    g = gen(experts)
    base = torch.randint(-3, 4, (40, experts), generator=g, device=DEV).float()
    logits = base + 2.0 ** -18 * torch.randint(0, 5, (40, experts), generator=g, device=DEV)
    logits[5], logits[6] = 0.0, NONE
    logits[7, 2:] = NONE
    logits[8] = torch.randn(experts, generator=g, device=DEV)
    for bias in (torch.zeros(experts, device=DEV), 0.25 * torch.randint(-1, 2, (experts,), generator=g, device=DEV).float()):
        ids, weights = expert_route(logits, top, scores=scores, bias=bias)
        want_ids, want = plain.route(logits, top, scores, bias)
        # FP64 of both sides agrees to some 2^-50 of 1; keys nearer than that have no order to check
        key = plain.scores_of(logits, scores) + bias.double()
        at = [torch.gather(torch.where(logits > NONE, key, torch.full_like(key, -9.0)), 1, i.clamp(min=0).long()) for i in (ids, want_ids)]
        assert torch.equal(ids < 0, want_ids < 0)
        assert bool((((at[0] - at[1]).abs() <= 2.0 ** -45) | (ids < 0)).all())
        for row in range(40):
            assert len(set(i for i in ids[row].tolist() if i >= 0)) == int((ids[row] >= 0).sum())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores", ("softmax", "sigmoid"))
@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("t,experts,top", CASES)
def test_route_gradient_matches_formula(dtype, scores, normalize, t, experts, top):
    """Errors of shares and of the sum that is subtracted, relative to the terms' magnitudes."""
    for masked, padded, scale in ((0.0, 0.0, 1.0), (0.4, 0.2, 2.5)):
        logits = logits_of(t + experts + 1, t, experts, dtype, masked, padded).requires_grad_()
        ids, weights = expert_route(logits, top, scores=scores, normalize=normalize, scale=scale)
        assert not ids.requires_grad and weights.requires_grad
        dweights = torch.randn(t, top, generator=gen(3), device=DEV)
        (got,) = torch.autograd.grad(weights, logits, dweights)
        assert got.dtype == dtype and got.shape == logits.shape
        live = torch.where((logits > NONE).any(dim=1))[0]
        want = torch.zeros(t, experts, dtype=torch.float64, device=DEV)
        size = want.clone()
        if live.numel() and top:
            leaf = logits.detach()[live].double().requires_grad_()
            share = plain.shares_of(leaf, ids[live], scores, normalize)
            (want[live],) = torch.autograd.grad(share * scale, leaf, dweights[live].double())
            most = dweights.abs().amax(dim=1, keepdim=True).double()[live] * scale
            p = plain.scores_of(logits.detach()[live], scores)
            chosen = torch.zeros_like(p).scatter_add_(1, ids[live].clamp(min=0).long(), torch.where(ids[live] >= 0, share.detach(), torch.zeros_like(share)))
            size[live] = 2 * most * (chosen if normalize or scores == "sigmoid" else p + chosen)
        bound = want.abs() * U[dtype] + size * 3 * share_error(experts) + TINY[dtype] + 2.0 ** -126
        off = (got.double() - want).abs()
        assert bool((off <= bound).all()), float((off - bound).max())
        assert bool((got[logits == NONE] == 0).all())


def test_route_gradient_matches_differences():
    """Central differences in 64 bits around FP32 logits: with h = 2^-8 their own error is h^2 / 6 of a third derivative of at most 4
    (scores' derivatives are below 1), and the kernel's is share_error of terms below 2."""
    logits = logits_of(4, 6, 16, torch.float32)
    dweights = torch.randn(6, 3, generator=gen(1), device=DEV)
    for scores in ("softmax", "sigmoid"):
        for normalize in (True, False):
            leaf = logits.clone().requires_grad_()
            ids, weights = expert_route(leaf, 3, scores=scores, normalize=normalize)
            (got,) = torch.autograd.grad(weights, leaf, dweights)
            h = 2.0 ** -8
            for e in range(16):
                step = torch.zeros(16, dtype=torch.float64, device=DEV)
                step[e] = h
                up, down = (plain.shares_of(logits.double() + s * step, ids, scores, normalize) for s in (1, -1))
                want = ((up - down) * dweights.double()).sum(dim=1) / (2 * h)
                most = dweights.abs().sum(dim=1).double()
                assert bool(((got[:, e].double() - want).abs() <= most * (h * h + 6 * share_error(16))).all())


def test_logits_of_any_layout():
    wide = logits_of(7, 40, 200, torch.float32)
    for view in (wide[:, 3:67], wide[:, :128:2], wide.t()[:40, :].contiguous().t()[:, :40], wide[:1, :64].expand(9, 64), wide[::3, 5:70]):
        for dtype in TYPES:
            v = view.to(dtype) if dtype != torch.float32 else view
            leaf, flat = v.detach().requires_grad_(), v.contiguous().clone().requires_grad_()
            a, b = expert_route(leaf, 4), expert_route(flat, 4)
            assert torch.equal(a.ids, b.ids) and torch.equal(a.weights, b.weights)
            la, lb = expert_balance(leaf, a.ids), expert_balance(flat, b.ids)
            assert torch.equal(la.loss, lb.loss) and torch.equal(la.counts, lb.counts)
            ga, gb = (torch.autograd.grad(w.sum() * 3 + (w * w).sum() + l, x) for w, l, x in ((a.weights, la.loss, leaf), (b.weights, lb.loss, flat)))
            assert torch.equal(ga[0], gb[0])


def test_logits_past_32_bits():
    """Over 2^31 logits: the last rows are as right as by themselves."""
    experts, more = 256, 1000
    t = 2 ** 31 // experts + more
    logits = torch.full((t, experts), NONE, dtype=torch.bfloat16, device=DEV)
    logits[-more:] = logits_of(1, more, experts, torch.bfloat16)
    last = logits[-more:].clone().requires_grad_()
    logits.requires_grad_()
    a, b = expert_route(logits, 2), expert_route(last, 2)
    assert torch.equal(a.ids[-more:], b.ids) and torch.equal(a.weights[-more:], b.weights) and not bool((a.ids[:-more] >= 0).any())
    la, lb = expert_balance(logits, a.ids), expert_balance(last, b.ids)
    assert torch.equal(la.counts, lb.counts) and abs(float(la.loss.detach()) - float(lb.loss.detach())) <= 2.0 ** -12
    (ga,), (gb,) = (torch.autograd.grad((w * w).sum() + loss, x) for w, loss, x in ((a.weights, la.loss, logits), (b.weights, lb.loss, last)))
    assert torch.equal(ga[-more:], gb) and not bool(ga[:1000].any()) and not bool(ga[t // 2:t // 2 + 1000].any())


BALANCE = [(1, 1, 1), (1, 8, 2), (37, 60, 2), (100, 16, 4), (64, 33, 3), (500, 64, 4), (1000, 128, 8), (300, 256, 8), (50, 500, 6), (70, 1000, 8),
           (40000, 8, 2), (20000, 60, 6), (9000, 128, 8), (5000, 1024, 4)]


@pytest.mark.parametrize("id_type", (torch.int32, torch.int64))
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scores", ("softmax", "sigmoid"))
@pytest.mark.parametrize("t,experts,top", BALANCE)
def test_balance(dtype, scores, id_type, t, experts, top):
    for masked, padded in ((0.0, 0.0), (0.3, 0.2)):
        logits = logits_of(t + experts, t, experts, dtype, masked, padded).requires_grad_()
        best, ids = logits.detach().float().topk(top, dim=1)
        ids = torch.where(best == NONE, torch.full_like(ids, -1), ids)
        ids[::7, 0] = experts + 5  # on another rank
        ids = ids.to(id_type).contiguous()
        loss, counts = expert_balance(logits, ids, scores=scores)
        assert loss.shape == () and loss.dtype == torch.float32 and counts.dtype == torch.int32 and not counts.requires_grad
        leaf = logits.detach().double().requires_grad_()
        want, want_counts = plain.balance(leaf, ids, scores)
        assert torch.equal(counts, want_counts)
        # p to share_error, its sums over tokens in FP32 by lane and wave (at most t of them), the rest in FP64
        assert abs(float(loss) - float(want)) <= float(want) * (share_error(experts) + (t + 4) * 2.0 ** -24 + 2.0 ** -24)
        factor = float(t)
        (got,) = torch.autograd.grad(loss, logits, torch.tensor(factor, device=DEV))
        assert got.dtype == dtype
        (d,) = torch.autograd.grad(want, leaf, torch.tensor(factor, dtype=torch.float64, device=DEV))
        live = (logits > NONE).any(dim=1, keepdim=True)
        p = plain.scores_of(logits.detach(), scores)
        p = p / torch.where(live, p.sum(dim=1, keepdim=True), torch.ones_like(p[:, :1]))
        n, tokens = max(int(counts.sum()), 1), max(int(live.sum()), 1)
        c = counts.double()
        size = factor * experts / (n * tokens) * p * (c + (c * p).sum(dim=1, keepdim=True))
        bound = d.abs() * U[dtype] + size * 3 * share_error(experts) + TINY[dtype] + 2.0 ** -126
        off = (got.double() - d).abs()
        assert bool((off <= bound).all()), float((off - bound).max())
        assert bool((got[logits == NONE] == 0).all())


def test_balance_gradient_matches_differences():
    """As for the route: the loss's third derivative by one logit is at most 4 experts times a token's share."""
    t, experts = 5, 12
    logits = logits_of(8, t, experts, torch.float32)
    ids = torch.randint(0, experts, (t, 2), generator=gen(2), device=DEV)
    for scores in ("softmax", "sigmoid"):
        leaf = logits.clone().requires_grad_()
        (got,) = torch.autograd.grad(expert_balance(leaf, ids, scores=scores).loss, leaf)
        h = 2.0 ** -8
        for i in range(t):
            for e in range(experts):
                step = torch.zeros(t, experts, dtype=torch.float64, device=DEV)
                step[i, e] = h
                want = float(plain.balance(logits.double() + step, ids, scores)[0] - plain.balance(logits.double() - step, ids, scores)[0]) / (2 * h)
                assert abs(float(got[i, e]) - want) <= experts / t * (h * h + 6 * share_error(experts))


def test_balance_of_nothing():
    for t, experts, top in ((0, 8, 2), (5, 8, 0), (5, 8, 2)):
        logits = torch.zeros(t, experts, device=DEV, requires_grad=True)
        loss, counts = expert_balance(logits, torch.full((t, top), -1, dtype=torch.int32, device=DEV))
        assert float(loss) == 0 and counts.tolist() == [0] * experts
        assert not torch.autograd.grad(loss, logits)[0].any()
    logits = torch.full((30, 8), NONE, device=DEV, requires_grad=True)
    loss, counts = expert_balance(logits, torch.zeros(30, 1, dtype=torch.int32, device=DEV))
    assert float(loss) == 0 and counts.tolist() == [30] + [0] * 7
    assert not torch.autograd.grad(loss, logits)[0].any()
    for t in (0, 3):
        ids, weights = expert_route(torch.zeros(t, 8, device=DEV, requires_grad=True), 2 if t == 0 else 0)
        assert ids.numel() == 0 and weights.numel() == 0


def test_balance_is_one_where_loads_are_alike():
    for experts in (4, 64, 512):
        logits = logits_of(1, 300, experts, torch.float32)
        ids = torch.arange(experts, dtype=torch.int32, device=DEV).repeat(300, 1)
        loss, counts = expert_balance(logits, ids)
        assert counts.tolist() == [300] * experts and abs(float(loss) - 1) < 300 * 2.0 ** -24 + share_error(experts)


def test_counts_may_be_changed_in_place():
    """A program adds up its ranks' counts; the gradient keeps its own."""
    logits = logits_of(2, 50, 16, torch.float32).requires_grad_()
    ids = torch.randint(0, 16, (50, 2), generator=gen(2), device=DEV)
    want = torch.autograd.grad(expert_balance(logits, ids).loss, logits)[0]
    loss, counts = expert_balance(logits, ids)
    counts.zero_()
    assert torch.equal(torch.autograd.grad(loss, logits)[0], want)


def test_repeats_bit_for_bit_and_on_another_stream():
    logits = logits_of(3, 30000, 128, torch.bfloat16).requires_grad_()

    def step():
        route = expert_route(logits, 8, scores="sigmoid", scale=2.5)
        loss, counts = expert_balance(logits, route.ids, scores="sigmoid")
        return (*route, loss, counts, *torch.autograd.grad((route.weights * route.weights).sum() + loss, logits))

    first = [v.detach().clone() for v in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for stream in (torch.cuda.current_stream(), side, side):
        with torch.cuda.stream(stream):
            again = step()
        stream.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_no_second_gradient_and_no_forward_mode():
    from torch.autograd import forward_ad

    logits = logits_of(3, 4, 8, torch.float32).requires_grad_()
    ids, weights = expert_route(logits, 2)
    loss = expert_balance(logits, ids).loss
    for out in ((weights * weights).sum(), loss):
        (once,) = torch.autograd.grad(out, logits, retain_graph=True)
        (again,) = torch.autograd.grad(out, logits, create_graph=True)
        assert torch.equal(once, again)
        with pytest.raises(RuntimeError, match="has no gradient"):
            again.sum().backward()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(logits.detach(), torch.ones_like(logits))
        for call in (lambda: expert_route(dual, 2), lambda: expert_balance(dual, ids)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()


def test_a_training_step_in_a_graph():
    """Route, balance, the experts' products and the gradients, captured once and replayed on new tokens, with the
    program's own work between; eagerly the same bits."""
    t, top, experts, k, n = 60, 4, 16, 256, 136
    g = gen(4)
    values, scales, z = plain.random_weight(g, (experts, n), k, 64, torch.bfloat16, True, DEV)
    codes = int4_pack(values)
    x = torch.empty(t, k, dtype=torch.bfloat16, device=DEV)
    logits = torch.empty(t, experts, device=DEV)

    def path():
        leaf = logits.detach().requires_grad_()
        route = expert_route(leaf, top, normalize=False)
        loss, counts = expert_balance(leaf, route.ids)
        sort = expert_sort(route.ids, experts)
        y = int4_expert_linear(x, codes, scales, sort, z, group=64, gather=True)
        out = expert_combine(y, route.weights, sort)
        (d,) = torch.autograd.grad((out, loss), leaf, (torch.ones_like(out), torch.ones_like(loss)))
        return out.detach(), loss.detach(), counts, d

    def fill(seed):
        h = gen(seed)
        x.copy_(torch.randn(t, k, generator=h, device=DEV))
        logits.copy_(torch.randn(t, experts, generator=h, device=DEV))
        logits[:seed] = NONE

    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        path()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = path()
    for seed in range(1, 5):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        kept = [v.clone() for v in got]
        assert all(torch.equal(a, b) for a, b in zip(kept, path()))


def test_a_layer_of_experts_against_a_plain_one():
    """Route, sort, product and weighted sum as they are used together, and the router's gradient through them."""
    t, top, experts, k, n = 90, 3, 8, 160, 70
    g = gen(12)
    x = torch.randn(t, k, generator=g, device=DEV).to(torch.bfloat16)
    logits = logits_of(12, t, experts, torch.float32, 0.2, 0.1).requires_grad_()
    values, scales, z = plain.random_weight(g, (experts, n), k, 32, torch.bfloat16, True, DEV)
    route = expert_route(logits, top, scores="sigmoid", scale=2.0)
    loss, counts = expert_balance(logits, route.ids, scores="sigmoid")
    sort = expert_sort(route.ids, experts)
    assert torch.equal(counts.cumsum(0).int(), sort.offsets[1:])
    y = int4_expert_linear(x, int4_pack(values), scales, sort, z, group=32, gather=True, out_dtype=torch.float32)
    out = expert_combine(y, route.weights, sort)
    dout = torch.randn(t, n, generator=g, device=DEV)
    (got,) = torch.autograd.grad((out, loss), logits, (dout, torch.tensor(3.0, device=DEV)))

    leaf = logits.detach().double().requires_grad_()
    live = torch.where((logits > NONE).any(dim=1))[0]
    every = torch.stack([x.double() @ plain.weight(values[e], scales[e], z[e], 32).T for e in range(experts)], dim=1)  # [t, experts, n]
    ids = plain.route(logits.detach(), top, "sigmoid")[0]
    assert torch.equal(ids, route.ids)
    share = plain.shares_of(leaf, ids, "sigmoid", True) * 2.0
    rows = every.gather(1, ids.clamp(min=0).long().unsqueeze(-1).expand(-1, -1, n)) * (ids >= 0).unsqueeze(-1)
    want = (rows * share.unsqueeze(-1)).sum(dim=1)
    size = float((rows.abs() * share.detach().unsqueeze(-1)).sum(dim=1).max())
    assert float((out.double() - want).abs().max()) <= size * (share_error(experts) + 2 * k * 2.0 ** -23 * 8)
    (d,) = torch.autograd.grad((want, plain.balance(leaf, ids, "sigmoid")[0]), leaf, (dout.double(), torch.tensor(3.0, dtype=torch.float64, device=DEV)))
    d = torch.where(torch.isnan(d), torch.zeros_like(d), d)  # of rows without a score
    most = float((rows.abs() * dout.double().abs().unsqueeze(1)).sum(dim=-1).max()) * 4 + 3.0 * experts
    assert float((got.double() - d).abs()[live].max()) <= most * (share_error(experts) * 4 + (n + 2 * k * 8) * 2.0 ** -23)
    assert expert_gather(x, sort).shape == (t * top, k)


def test_refusals():
    logits = torch.zeros(4, 8, device=DEV)
    ids = torch.zeros(4, 2, dtype=torch.int32, device=DEV)
    for call, message in (
            (lambda: expert_route(logits.int(), 2), "logits must be torch.bfloat16"), (lambda: expert_route(logits[0], 2), "2 dimensions"),
            (lambda: expert_route(logits, 9), "top must be in"), (lambda: expert_route(logits, -1), "top must be in"),
            (lambda: expert_route(logits, 2, scores="tanh"), "scores must be"), (lambda: expert_route(torch.zeros(2, 1025, device=DEV), 2), "1 to 1024"),
            (lambda: expert_route(torch.zeros(2, 0, device=DEV), 0), "1 to 1024"),
            (lambda: expert_route(logits, 2, bias=torch.zeros(7, device=DEV)), "bias must be"),
            (lambda: expert_route(logits, 2, bias=torch.zeros(8, dtype=torch.float64, device=DEV)), "bias must be"),
            (lambda: expert_route(logits, 2, bias=torch.zeros(8)), "bias must be a CUDA"),
            (lambda: expert_balance(logits, ids.float()), "ids must be torch.int32"), (lambda: expert_balance(logits, ids[:3].contiguous()), "ids must have shape"),
            (lambda: expert_balance(logits, ids.cpu()), "must be a CUDA"), (lambda: expert_balance(logits, ids, scores=None), "scores must be")):
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(RuntimeError, match="bias of expert_route has no gradient"):
        expert_route(logits, 2, bias=torch.zeros(8, device=DEV, requires_grad=True))
