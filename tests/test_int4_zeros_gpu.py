"""What the zeros of int4 weights take away: how exact it is, and that all of its pieces count.

y = sum over groups of s (sum x q - z sum x). The second term may be larger than the result by far, where x has a mean. It is taken away
by spans of a group or, of a larger one, 128 columns: one at a time for few rows, four at a time for tiles of many rows."""
import ctypes

import pytest
import torch

from mpserve_amd import _native
from mpserve_amd.experts import expert_gather, expert_sort, int4_expert_linear
from mpserve_amd.int4 import _int4_product, int4_linear, int4_pack
from tests import int4_plain as plain
from tests.test_int4_gpu import close, routing

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALVES = (torch.bfloat16, torch.float16)
MANY = 128  # columns whose sum of x is taken at once, at most


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def takes_tiles(x, codes, scales, zeros, group):
    """Whether the product goes to the tiles of many rows: these need sums of x in a workspace, which rows that need no packing do not."""
    assert x.shape[1] % 32 == 0 and x.is_contiguous()
    p = _int4_product(x, codes, scales, zeros, None, group, x.shape[1], codes.shape[0])
    p.rows, p.out = x.shape[0], x.data_ptr()
    need = ctypes.c_int64(0)
    _native.check(_native.lib().mps_int4_product_workspace(p, need))
    return need.value > 0


def near_their_zeros(g, shape, k, group):
    """Whole numbers that are their group's zero, one more or one less: (values, scales of 1, zeros)."""
    groups = (k + group - 1) // group
    zeros = torch.randint(9, 15, (*shape, groups), generator=g, device=DEV, dtype=torch.uint8)
    off = torch.randint(-1, 2, (*shape, k), generator=g, device=DEV, dtype=torch.int8)
    values = (zeros.repeat_interleave(group, dim=-1)[..., :k].to(torch.int8) + off).to(torch.uint8)
    return values, torch.ones(*shape, groups, device=DEV), zeros


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("group", (32, 64, 128, 256, 32768))
@pytest.mark.parametrize("t,n", ((1, 64), (6, 100), (40, 96), (300, 4100), (600, 2060), (2000, 4100)))
def test_sums_are_no_larger_than_they_need_be(t, n, group, dtype):
    """x is 200 to 255 in all of 28672 columns: what the zeros take away adds up to 28672 * 228 * 9 and more, past 2^25, of which FP32 loses
    the last bits. The result (below 28672 * 255) and four spans' part (below 512 * 255 * 15) together stay below 2^24, as do a span's sums of
    x q: sums made in that order are exact."""
    k, g = 28672, gen(t + group)
    x = torch.randint(200, 256, (t, k), generator=g, device=DEV).to(dtype)
    values, scales, zeros = near_their_zeros(g, (n,), k, group)
    codes, scales = int4_pack(values), scales.to(dtype)
    assert takes_tiles(x, codes, scales, zeros, group) == (t >= 300)
    want = x.double() @ plain.weight(values, scales, zeros, group).T
    assert float(want.abs().max()) < 2 ** 24 - 512 * 255 * 15
    assert torch.equal(int4_linear(x, codes, scales, zeros, group=group, out_dtype=torch.float32).double(), want)


@pytest.mark.parametrize("gather", (True, False))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("t", (8, 900))
def test_sums_of_experts_are_no_larger_than_they_need_be(t, group, gather):
    k, n, experts, top, g = 28672, 1030, 3, 2, gen(t + group)
    x = torch.randint(200, 256, (t, k), generator=g, device=DEV).to(torch.bfloat16)
    values, scales, zeros = near_their_zeros(g, (experts, n), k, group)
    scales, ids = scales.to(torch.float16), routing(t, t, top, experts, 0.1)
    sort = expert_sort(ids, experts)
    y = int4_expert_linear(x if gather else expert_gather(x, sort), int4_pack(values), scales, sort, zeros, group=group, gather=gather,
                           out_dtype=torch.float32)
    offsets, order = sort.offsets.tolist(), sort.order.long()
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        want = x[order[a:b] // top].double() @ plain.weight(values[e], scales[e], zeros[e], group).T
        assert torch.equal(y[a:b].double(), want)
    assert not bool(y[offsets[-1]:].any())


def spans_in_three_pieces(g, t, k, span, dtype):
    """x [t, k] whose sums over spans are 2^a (1.5 + 2^-8 + 2^-17): in eight bits each, none of a sum's first, second and third piece is zero.
    1/64 once, and whole numbers from 64 to 127, which any of the types hold."""
    spans, total = k // span, 3080 * span // 32
    v = torch.full((t * spans, span - 1), total // (span - 1), device=DEV)
    v[:, :total - int(v[0].sum())] += 1
    for col in range(0, span - 2, 2):  # neighbours apart by chance, their sum kept
        by = torch.randint(0, 24, (t * spans,), generator=g, device=DEV)
        v[:, col] += by
        v[:, col + 1] -= by
    assert bool((v.sum(dim=1) == total).all()) and int(v.min()) > 0 and int(v.max()) < 256
    first = torch.full((t * spans, 1), span / 32 / 64, device=DEV)
    return torch.cat([first, v.float()], dim=1).view(t, k).to(dtype)


def weight_in_two_pieces(g, shape, spans, span, stype):
    """Whole numbers, scales and zeros [*shape, spans] of which s z has more than eight bits."""
    values = torch.randint(0, 16, (*shape, spans * span), generator=g, device=DEV, dtype=torch.uint8)
    zeros = torch.tensor([5, 8, 13, 15], device=DEV, dtype=torch.uint8)[torch.randint(0, 4, (*shape, spans), generator=g, device=DEV)]
    scales = (257 / 256 if stype == torch.float16 else 129 / 128) * torch.exp2(torch.randint(-1, 2, (*shape, 1), generator=g, device=DEV).float())
    return values, scales.expand(*shape, spans).to(stype).contiguous(), zeros


def all_pieces_count(got, x, values, scales, zeros, span):
    """A sum's third piece is 2^-17.6 of it, the product of its second and of what eight bits leave of s z up to 2^-17. Each span adds at most
    six numbers that are not zero to a result (five of what the zeros take away, and s sum x q, which is exact), each off by a step of the
    largest sum on the way, of all spans before and four spans' part: the bound is 6 2^-23 of that, a span, below the 2^-17.6 of a
    span's part that a lost piece is, for one span and for four."""
    spans = scales.shape[-1]
    w = plain.weight(values, scales, zeros, span)
    prefix = torch.zeros_like(got, dtype=torch.float64)
    most = prefix.clone()
    part = (scales.double() * zeros.double()) * float(x[0, :span].double().sum())  # [n, spans]: the same in all rows
    for at in range(spans):
        prefix += x[:, at * span:(at + 1) * span].double() @ w[:, at * span:(at + 1) * span].T
        most = torch.maximum(most, prefix.abs())
    four = torch.stack([part[:, at:at + 4].sum(dim=1) for at in range(0, spans, 4)]).amax(dim=0)
    off = (got.double() - prefix).abs()
    bound = 6 * spans * 2.0 ** -23 * (most + four)
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("stype", HALVES)
@pytest.mark.parametrize("span", (32, 64, 128))
@pytest.mark.parametrize("spans", (1, 4, 21))
def test_every_piece_of_the_sums_and_of_scales_and_zeros_counts(spans, span, stype, dtype):
    t, n, g = 2500, 2060, gen(spans + span)
    x = spans_in_three_pieces(g, t, spans * span, span, dtype)
    values, scales, zeros = weight_in_two_pieces(g, (n,), spans, span, stype)
    codes = int4_pack(values)
    assert takes_tiles(x, codes, scales, zeros, span)
    all_pieces_count(int4_linear(x, codes, scales, zeros, group=span, out_dtype=torch.float32), x, values, scales, zeros, span)


@pytest.mark.parametrize("gather", (True, False))
@pytest.mark.parametrize("span", (32, 64, 128))
@pytest.mark.parametrize("spans", (1, 4))
def test_every_piece_counts_for_experts(spans, span, gather):
    t, n, experts, top, g = 2500, 2060, 3, 2, gen(spans + span)
    x = spans_in_three_pieces(g, t, spans * span, span, torch.float16)
    values, scales, zeros = weight_in_two_pieces(g, (experts, n), spans, span, torch.float16)
    sort = expert_sort(routing(t, t, top, experts, 0.1), experts)
    y = int4_expert_linear(x if gather else expert_gather(x, sort), int4_pack(values), scales, sort, zeros, group=span, gather=gather,
                           out_dtype=torch.float32)
    offsets, order = sort.offsets.tolist(), sort.order.long()
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        all_pieces_count(y[a:b], x[order[a:b] // top], values[e], scales[e], zeros[e], span)


@pytest.mark.parametrize("group", (32, 64, 128, 1024))
@pytest.mark.parametrize("t", (24, 512))
def test_a_mean_of_x_costs_no_digits(t, group):
    """x of mean 1 and sigma 1, results in FP32. A span adds six numbers to a sum that is as large as the result and four spans' part
    (one, for few rows); roundings, each up to half a step of it, add up as their squares do. Twice that is allowed."""
    k, n, g = 28672, 4096, gen(t + group)
    x = (1 + torch.randn(t, k, generator=g, device=DEV)).to(torch.float16)
    values, scales, _ = plain.random_weight(g, (n,), k, group, torch.float16, False, DEV)
    codes, w = int4_pack(values), plain.weight(values, scales, None, group)
    assert takes_tiles(x, codes, scales, None, group) == (t == 512)
    want = x.double() @ w.T
    off = int4_linear(x, codes, scales, group=group, out_dtype=torch.float32).double() - want
    span = min(group, MANY)
    part = (8 * scales.double()).repeat_interleave(max(1, group // span), dim=1)[:, :k // span] * span  # [n, spans], for a mean of 1
    four = part.view(n, -1, 4).sum(dim=2).square().mean().sqrt()
    size = want.square().mean().sqrt() + four
    assert float(off.square().mean().sqrt()) <= 2 * 2.0 ** -24 * (6 * k / span) ** 0.5 * float(size)


@pytest.mark.parametrize("zeros", (True, False))
@pytest.mark.parametrize("stype", HALVES)
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("t,k,n,group", [(40, 2048, 512, 64), (300, 4096, 384, 128), (1000, 736, 600, 32), (900, 736, 700, 64), (3000, 1024, 2100, 128),
                                         (700, 1000, 1030, 256)])
def test_linear_is_close_with_and_without_zeros(dtype, stype, zeros, t, k, n, group):
    g = gen(t + k)
    x = (0.5 + torch.randn(t, k, generator=g, device=DEV) * torch.exp(torch.randn(k, generator=g, device=DEV))).to(dtype)
    values, scales, z = plain.random_weight(g, (n,), k, group, stype, zeros, DEV)
    bias = torch.randn(n, generator=g, device=DEV)
    close(int4_linear(x, int4_pack(values), scales, z, bias, group=group, out_dtype=torch.float32), x, values, scales, z, group, bias)
