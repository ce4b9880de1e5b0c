"""The balance loss where its ordinary tests' tolerances are wide: rows that are lost or count twice, and loads that are nearly alike."""
import pytest
import torch

from mpserve_amd.experts import expert_balance
from tests import int4_plain as plain
from tests.test_router_gpu import NONE, U, gen, logits_of, share_error

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("scores", ("softmax", "sigmoid"))
@pytest.mark.parametrize("t,experts", ((4096, 64), (65536, 64), (30000, 250), (3000, 1000)))
def test_gradient_of_loads_that_are_nearly_alike(t, experts, scores):
    """Errors are those of the loads' differences from their mean, not of the loads: relative ones of shares and of a sum of `experts` terms.
    The 64-bit form has errors of the loads themselves, which show where all that are left in a row are alike and the gradient is zero: a
    product, a sum of `experts` terms and the sigmoid's or softmax's own, of a few steps of 2^-53 each."""
    top = 4
    pairs = t * top // experts * experts
    ids = torch.full((t * top,), -1, dtype=torch.int32, device=DEV)
    ids[:pairs] = torch.arange(pairs, device=DEV, dtype=torch.int32) % experts
    ids[0], ids[5] = 7, 9  # two loads are one more, two one less
    ids = ids.view(t, top)
    logits = logits_of(t, t, experts, torch.float32, 0.2, 0.1).requires_grad_()
    dloss = torch.tensor(float(t), device=DEV)
    loss, counts = expert_balance(logits, ids, scores=scores)
    (got,) = torch.autograd.grad(loss, logits, dloss)
    leaf = logits.detach().double().requires_grad_()
    want, want_counts = plain.balance(leaf, ids, scores)
    assert torch.equal(counts, want_counts) and int(counts.max() - counts.min()) == 2
    (d,) = torch.autograd.grad(want, leaf, dloss.double())
    live = (logits > NONE).any(dim=1, keepdim=True)
    p = plain.scores_of(logits.detach(), scores)
    p = p / torch.where(live, p.sum(dim=1, keepdim=True), torch.ones_like(p[:, :1]))
    away = (counts.double() - counts.double().mean()).abs()
    size = float(t) * experts / (int(counts.sum()) * int(live.sum())) * p * (away + (away * p).sum(dim=1, keepdim=True))
    form = float(t) * experts / (int(counts.sum()) * int(live.sum())) * p * 2 * float(counts.max()) * (experts + 64) * 2.0 ** -53
    off = (got.double() - d).abs()
    bound = d.abs() * U[torch.float32] + size * 3 * share_error(experts) + form + 2.0 ** -126
    assert bool((off <= bound).all()), float((off - bound).max())


def test_gradient_of_loads_that_are_alike_is_zero():
    for experts in (4, 60, 1000):
        logits = logits_of(1, 300, experts, torch.float32).requires_grad_()
        loss, _ = expert_balance(logits, torch.arange(experts, dtype=torch.int32, device=DEV).repeat(300, 1))
        assert not bool(torch.autograd.grad(loss, logits)[0].any())


@pytest.mark.parametrize("scores", ("softmax", "sigmoid"))
@pytest.mark.parametrize("t,experts,dtype", (
    (1, 8, torch.float32), (37, 60, torch.float32), (255, 64, torch.bfloat16), (2047, 8, torch.float32), (2049, 8, torch.float16), (16385, 3, torch.float32),
    (9000, 128, torch.bfloat16), (20000, 60, torch.float32), (40000, 8, torch.float16), (65537, 128, torch.float32), (65536, 256, torch.bfloat16),
    (5000, 1024, torch.float32), (70001, 17, torch.bfloat16)))
def test_every_row_counts_once(t, experts, dtype, scores):
    """Each row has one expert that is not masked, whose share is 1: the sums over tokens are whole numbers, and the loss is the nearest FP32
    number to a quotient of whole numbers but for FP64's errors. Rows differ in what they add, the least of them 2^-20 of the whole and more
    (a seventh of the mean of up to 70001 rows), so that one that is lost, or counts for another, shows."""
    g = gen(t + experts)
    mine = torch.randint(0, experts, (t,), generator=g, device=DEV)
    logits = torch.full((t, experts), NONE, device=DEV)
    logits[torch.arange(t, device=DEV), mine] = 4 * torch.randn(t, generator=g, device=DEV)
    padded = torch.rand(t, generator=g, device=DEV) < (0.1 if t > 30 else 0.0)
    logits[padded] = NONE
    load = torch.randint(1, 8, (experts,), generator=g, device=DEV)  # pairs of an expert
    ids = torch.repeat_interleave(torch.arange(experts, device=DEV), load)
    ids = torch.nn.functional.pad(ids, (0, -ids.numel() % t), value=-1).view(-1, t).t().contiguous().int()
    loss, counts = expert_balance(logits.to(dtype), ids, scores=scores)
    assert torch.equal(counts.long(), load)
    want = experts * float(load[mine[~padded]].sum()) / (float(load.sum()) * float((~padded).sum()))
    assert abs(float(loss) - want) <= want * 2.0 ** -23
