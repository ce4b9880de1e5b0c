"""Backward passes of the experts' operators under saved-tensor hooks, which may give back what was saved in other memory and another
layout. Without a GPU: the calls into the library are recorded in place of being made."""
import contextlib

import pytest
import torch

from mpserve_amd import experts


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(experts, "_call", lambda device, entry, *args: made.append((entry.__name__, args)))
    return made


class Hooks(torch.autograd.graph.saved_tensors_hooks):
    """Every tensor comes back as ``change`` of it; ``given`` holds these."""

    def __init__(self, change=lambda t: t.clone(memory_format=torch.contiguous_format)):
        self.given = []

        def unpack(t):
            self.given.append(change(t))
            return self.given[-1]

        super().__init__(lambda t: t, unpack)

    def __enter__(self):
        super().__enter__()
        return self

    def at(self, pointer):
        return next(t for t in self.given if t.data_ptr() == pointer)


def route(logits):
    return experts._Route.apply(logits, 2, experts._SCORES["sigmoid"], None, True, 1.0)[1]


def balance(logits):
    return experts._Balance.apply(logits, torch.zeros(logits.shape[0], 2, dtype=torch.int32), experts._SCORES["softmax"])[0]


@pytest.mark.parametrize("call", (route, balance))
def test_rows_are_as_far_apart_as_in_the_tensor_that_a_hook_gives(calls, call):
    wide = torch.randn(6, 200)
    leaf = wide[:, 3:67].requires_grad_()
    with Hooks() as hooks:
        out = call(leaf)
    torch.autograd.grad(out, leaf, torch.ones_like(out))
    name, args = calls[-1]
    assert name.endswith("_grad")
    logits = hooks.at(args[0])
    assert logits.stride() == (64, 1) and args[2:5] == (6, 64, 64)


@pytest.mark.parametrize("call", (route, balance))
def test_columns_that_a_hook_puts_apart_are_put_together(calls, call):
    leaf = torch.randn(6, 64).requires_grad_()
    with Hooks(lambda t: t.t().contiguous().t() if t.dim() == 2 else t.repeat(2, 1).t().contiguous().t()[0] if t.dim() == 1 else t) as hooks:
        out = call(leaf)
    torch.autograd.grad(out, leaf, torch.ones_like(out))
    given = {t.data_ptr() for t in hooks.given if not t.is_contiguous()}
    assert given and not given & set(a for a in calls[-1][1] if isinstance(a, int) and a > 2 ** 20)


@pytest.mark.parametrize("call", (route, balance))
@pytest.mark.parametrize("change", (lambda t: t.to(torch.float16) if t.is_floating_point() else t, lambda t: t[:-1], lambda t: t.to("meta"),
                                    lambda t: t.long() if not t.is_floating_point() else t))
def test_what_is_not_the_saved_tensor_is_refused(calls, call, change):
    leaf = torch.randn(6, 64).requires_grad_()
    with Hooks(change):
        out = call(leaf)
    before = len(calls)
    with pytest.raises(RuntimeError, match="saved-tensor hook"):
        torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert len(calls) == before


def test_combine_and_gather_take_what_hooks_give(calls):
    t, top, width, num = 5, 2, 16, 4
    order, positions, offsets = torch.zeros(t * top, dtype=torch.int32), torch.zeros(t, top, dtype=torch.int32), torch.zeros(num + 1, dtype=torch.int32)
    apart = lambda v: v.t().contiguous().t() if v.dim() == 2 else v.repeat(2, 1).t().contiguous().t()[0]  # noqa: E731
    y, weights, x = torch.randn(t * top, width).requires_grad_(), torch.rand(t, top).requires_grad_(), torch.randn(t, width).requires_grad_()
    for change, fine in ((apart, True), (lambda v: v[:-1], False), (lambda v: v.to("meta"), False), (lambda v: v.half(), False)):
        for call, leaves in ((lambda: experts._Combine.apply(y, weights, order, positions, offsets), (y, weights)),
                             (lambda: experts._Gather.apply(x, order, positions, offsets), (x,))):
            with Hooks(change) as hooks:
                out = call()
            before = len(calls)
            if fine:
                torch.autograd.grad(out, leaves, torch.ones_like(out))
                given = {v.data_ptr() for v in hooks.given if not v.is_contiguous()}
                assert given and not given & set(a for a in calls[-1][1] if isinstance(a, int) and a > 2 ** 20)
            else:
                with pytest.raises(RuntimeError, match="saved-tensor hook"):
                    torch.autograd.grad(out, leaves, torch.ones_like(out))
                assert len(calls) == before


@pytest.mark.gpu
@pytest.mark.parametrize("scores,normalize", (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)))
def test_gradients_of_a_slice_that_is_kept_on_the_host(scores, normalize):
    """``save_on_cpu`` gives back a dense copy of a slice of columns: the gradients are the contiguous call's."""
    wide = torch.randn(300, 200, generator=torch.Generator().manual_seed(3)).cuda()
    leaf, flat = wide[:, 3:67].requires_grad_(), wide[:, 3:67].contiguous().requires_grad_()
    assert leaf.stride() == (200, 1)
    got = []
    for x, hooks in ((leaf, torch.autograd.graph.save_on_cpu()), (flat, contextlib.nullcontext())):
        with hooks:
            chosen = experts.expert_route(x, 4, scores=scores, normalize=normalize, scale=2.5)
            loss = experts.expert_balance(x, chosen.ids, scores=scores).loss
        got.append([torch.autograd.grad(out, x, dout)[0] for out, dout in ((chosen.weights, chosen.weights.detach() + 1), (loss, loss.detach()))])
    assert all(torch.equal(a, b) and bool(a.any()) for a, b in zip(*got))


@pytest.mark.gpu
def test_experts_of_rows_that_are_kept_on_the_host():
    t, top, width, num = 70, 3, 40, 8
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(-1, num, (t, top), generator=g).cuda()
    x, weights = torch.randn(t, width, generator=g).cuda().requires_grad_(), torch.rand(t, top, generator=g).cuda().requires_grad_()
    sort, dout = experts.expert_sort(ids, num), torch.randn(t, width, generator=g).cuda()
    got = []
    for hooks in (torch.autograd.graph.save_on_cpu(), contextlib.nullcontext()):
        with hooks:
            out = experts.expert_combine(experts.expert_gather(x, sort) * 2, weights, sort)
        got.append(torch.autograd.grad(out, (x, weights), dout))
    assert all(torch.equal(a, b) and bool(a.any()) for a, b in zip(*got))
