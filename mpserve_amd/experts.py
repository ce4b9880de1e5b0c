"""Mixtures of experts: the router, tokens to their experts and back, and products with MXFP4 and int4 experts.

A router gives each of ``t`` tokens ``top`` experts; an expert id outside ``[0, experts)`` (say
-1) means none here: the pair was dropped, or its expert is on another rank.

* :func:`expert_route` — from a router's logits to experts and weights (differentiable);
* :func:`expert_balance` — the loss that keeps experts' loads alike, and their counts (differentiable);
* :func:`expert_sort` — the pairs of tokens and experts ordered by expert;
* :func:`expert_gather` — the tokens' rows in that order (differentiable);
* :func:`mxfp4_expert_linear` — each row times its expert's MXFP4 weight;
* :func:`int4_expert_linear` — each row times its expert's int4 weight;
* :func:`expert_combine` — the weighted sum of each token's rows (differentiable).

Shapes do not depend on the routing, so nothing synchronises and all of it can be captured
into a graph. The calls run on the current stream of their tensors' device; results do not
depend on the order in which the GPU ran anything. Gradients are those of backward mode; tensors
that carry a tangent are refused.

Experts' rows are rounded to the type of ``x`` between the product and the weighted sum, and the sum once more:
a relative error of 0.0023 in BF16 where one rounding has 0.0017. Rows of ``out_dtype=torch.float32``, whose
sum is FP32 too and is rounded by the caller's ``.to``, spare the first: 8192 tokens, four of 64 experts each, 4096 ->
2048, then take 612 us in place of 548, four tokens 32 in place of 28.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad

from . import _native
from ._common import _check_cuda_contig
from .int4 import _check_int4, _HALVES, _int4_multiply, _int4_product
from .mxfp4 import BLOCK, _TYPES, _call, _check_bias, _check_cuda, _check_mx, _check_out, _multiply, _no_grad, _no_tangent, _set_x, _type


class ExpertRoute(NamedTuple):
    """Each token's experts, by falling score."""
    ids: torch.Tensor      # int32 [t, top]: -1 where no expert was left
    weights: torch.Tensor  # FP32 [t, top]: 0 there


class ExpertBalance(NamedTuple):
    """A batch's balance loss and loads."""
    loss: torch.Tensor    # FP32, no dimensions
    counts: torch.Tensor  # int32 [experts]: pairs of each expert


class ExpertSort(NamedTuple):
    """Where each pair (token, slot) stands once pairs are ordered by expert."""
    order: torch.Tensor      # int32 [t * top]: the pair (token * top + slot) at each place
    positions: torch.Tensor  # int32 [t, top]: each pair's place, -1 where it has no expert
    offsets: torch.Tensor    # int32 [experts + 1]: each expert's first place; the last: pairs that have an expert


def expert_sort(ids: torch.Tensor, num_experts: int) -> ExpertSort:
    """Order the pairs of ``ids [t, top]`` (int32 or int64) by expert, an expert's pairs as they come and
    the pairs of no expert last."""
    _check_cuda_contig(ids, "ids", None)
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be torch.int32 or torch.int64, got {ids.dtype}")
    if ids.dim() != 2:
        raise ValueError("ids must have 2 dimensions")
    num_experts = int(num_experts)
    if not 1 <= num_experts <= _native.MPS_MAX_EXPERTS:
        raise ValueError(f"num_experts must be in [1, {_native.MPS_MAX_EXPERTS}]")
    device, (t, top) = ids.device, ids.shape
    lib = _native.lib()
    need = ctypes.c_int64(0)
    rc = lib.mps_expert_sort_workspace(t, top, num_experts, need)
    if rc:
        _native.check(rc)
    order = torch.empty(t * top, dtype=torch.int32, device=device)
    positions = torch.empty((t, top), dtype=torch.int32, device=device)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=device)
    work = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
    _call(device, lib.mps_expert_sort, ids.data_ptr(), ids.dtype == torch.int64, t, top, num_experts, order.data_ptr(),
          positions.data_ptr(), offsets.data_ptr(), work.data_ptr() if need.value else None, need.value)
    return ExpertSort(order, positions, offsets)


def _check_sort(sort: ExpertSort, device: torch.device) -> None:
    order, positions, offsets = sort
    i32 = torch.int32
    if isinstance(order, torch.Tensor) and isinstance(positions, torch.Tensor) and isinstance(offsets, torch.Tensor) \
            and order.device == positions.device == offsets.device == device \
            and order.dtype == positions.dtype == offsets.dtype == i32 \
            and order.is_contiguous() and positions.is_contiguous() and offsets.is_contiguous():
        if positions.dim() != 2 or order.dim() != 1 or offsets.dim() != 1 or order.numel() != positions.numel() \
                or offsets.numel() < 2:
            raise ValueError("sort must be what expert_sort returns")
        return
    for t, name in ((order, "sort.order"), (positions, "sort.positions"), (offsets, "sort.offsets")):
        _check_cuda_contig(t, name, device)
        if t.dtype != i32:
            raise ValueError(f"{name} must be torch.int32")


def _check_rows(t: torch.Tensor, name: str, rows: int, device: Optional[torch.device] = None) -> None:
    _check_cuda(t, name, device)
    _type(t, name)
    if t.dim() != 2 or t.shape[0] != rows:
        raise ValueError(f"{name} must have shape [{rows}, width], got {tuple(t.shape)}")


def _sum_rows(y: torch.Tensor, weights: Optional[torch.Tensor], positions: torch.Tensor) -> torch.Tensor:
    t, top = positions.shape
    out = torch.empty((t, y.shape[1]), dtype=y.dtype, device=y.device)
    _call(y.device, _native.lib().mps_expert_combine, y.data_ptr(), _TYPES[y.dtype],
          weights.data_ptr() if weights is not None else None, _TYPES[weights.dtype] if weights is not None else 0, t,
          top, y.shape[1], positions.data_ptr(), out.data_ptr())
    return out


def _gather_rows(x: torch.Tensor, order: torch.Tensor, positions: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    t, top = positions.shape
    rows = torch.empty((t * top, x.shape[1]), dtype=x.dtype, device=x.device)
    _call(x.device, _native.lib().mps_expert_gather, x.data_ptr(), _TYPES[x.dtype], t, top, offsets.numel() - 1,
          x.shape[1], order.data_ptr(), positions.data_ptr(), offsets.data_ptr(), rows.data_ptr())
    return rows


def _first_gradient(backward):
    """``once_differentiable``, whose wrapper costs 5 us of a small backward's 45, only where a graph of the
    gradients is being made."""
    once = torch.autograd.function.once_differentiable(backward)

    def run(ctx, grad):
        return once(ctx, grad) if torch.is_grad_enabled() else backward(ctx, grad)

    return run


def _kept(t: torch.Tensor, shape, dtype: torch.dtype, device: torch.device, rows: bool = False) -> torch.Tensor:
    """A tensor that a forward pass saved, contiguous, or with ``rows`` as rows that may lie apart. Autograd's saved-tensor hooks may give
    back other memory, laid out in another way (an offload's copy of a slice of columns has its rows side by side); what has
    another size, type or device is refused: kernels would read past its end."""
    if t.shape != shape or t.dtype is not dtype or t.device != device:
        raise RuntimeError(f"a saved-tensor hook gave back {tuple(t.shape)} {t.dtype} on {t.device} for what was saved as "
                           f"{tuple(shape)} {dtype} on {device}")
    return t if t.is_contiguous() or (rows and (t.stride(1) == 1 or t.shape[1] == 1)) else t.contiguous()


class _Gather(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order, positions, offsets):
        ctx.save_for_backward(positions)
        ctx.how = positions.shape
        return _gather_rows(x, order, positions, offsets)

    @staticmethod
    @_first_gradient
    def backward(ctx, drows):
        (positions,) = ctx.saved_tensors
        positions = _kept(positions, ctx.how, torch.int32, drows.device)
        return _sum_rows(drows.contiguous(), None, positions), None, None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, order, positions, offsets):
        # y is needed for the weights' gradient only
        ctx.save_for_backward(y if ctx.needs_input_grad[1] else None, weights, order, positions, offsets)
        ctx.how = weights.dtype, weights.shape, offsets.shape
        return _sum_rows(y, weights, positions)

    @staticmethod
    @_first_gradient
    def backward(ctx, dout):
        y, weights, order, positions, offsets = ctx.saved_tensors
        weights_type, shape, ends = ctx.how
        (t, top), device, i32 = shape, dout.device, torch.int32
        dout = dout.contiguous()
        width, dy, dweights = dout.shape[1], None, None
        if y is not None:
            y = _kept(y, (t * top, width), dout.dtype, device)
        weights = _kept(weights, shape, weights_type, device)
        order, positions = _kept(order, (t * top,), i32, device), _kept(positions, shape, i32, device)
        offsets = _kept(offsets, ends, i32, device)
        if ctx.needs_input_grad[0]:
            dy = torch.empty((t * top, width), dtype=dout.dtype, device=dout.device)
        if ctx.needs_input_grad[1]:
            dweights = torch.empty_like(weights)
        _call(dout.device, _native.lib().mps_expert_combine_grad, y.data_ptr() if y is not None else None, dout.data_ptr(), _TYPES[dout.dtype],
              weights.data_ptr(), _TYPES[weights.dtype], t, top, offsets.numel() - 1, width, order.data_ptr(),
              positions.data_ptr(), offsets.data_ptr(), dy.data_ptr() if dy is not None else None,
              dweights.data_ptr() if dweights is not None else None)
        return dy, dweights, None, None, None


def expert_gather(x: torch.Tensor, sort: ExpertSort) -> torch.Tensor:
    """``rows [t * top, width]`` of ``x [t, width]`` (BF16, FP16 or FP32) in the sorted order; the places
    of pairs of no expert, the last ones, are zero. Its gradient is the sum of a token's rows' gradients."""
    _check_cuda(x, "x")
    _check_sort(sort, x.device)
    _check_rows(x, "x", sort.positions.shape[0])
    if forward_ad._current_level >= 0:
        _no_tangent("expert_gather", x)
    if not (x.requires_grad and torch.is_grad_enabled()):
        return _gather_rows(x.contiguous(), *sort)
    return _Gather.apply(x.contiguous(), *sort)


def expert_combine(y: torch.Tensor, weights: torch.Tensor, sort: ExpertSort) -> torch.Tensor:
    """``out[token] = sum over slots of weights[token, slot] * y[place of the pair]``, without the pairs of no
    expert: zero for a token that has none. ``y [t * top, width]`` is BF16, FP16 or FP32, ``weights [t, top]``
    any of these; the sum is FP32 and is rounded once to the type of ``y``. The gradients are those of ``y``
    (zero in the places of pairs of no expert) and of ``weights`` (zero for these pairs)."""
    _check_cuda(y, "y")
    _check_sort(sort, y.device)
    _check_rows(y, "y", sort.order.numel())
    _check_cuda(weights, "weights", y.device)
    _type(weights, "weights")
    if weights.shape != sort.positions.shape:
        raise ValueError(f"weights must have shape {tuple(sort.positions.shape)}, got {tuple(weights.shape)}")
    if forward_ad._current_level >= 0:
        _no_tangent("expert_combine", y, weights)
    y, weights = y.contiguous(), weights.contiguous()
    if not ((y.requires_grad or weights.requires_grad) and torch.is_grad_enabled()):
        return _sum_rows(y, weights, sort.positions)
    return _Combine.apply(y, weights, *sort)


def mxfp4_expert_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, sort: ExpertSort,
                        bias: Optional[torch.Tensor] = None, *, gather: bool = False,
                        out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[j] = x[j] @ w[e].T + bias[e]`` for the rows ``j`` of expert ``e`` in the sorted order.

    ``x`` is BF16 or FP16: the sorted rows ``[t * top, k]``, or with ``gather`` the tokens ``[t, k]``, whose
    rows are read where they are, without a gathered copy. ``codes [experts, n, 16 * ceil(k / 32)]`` and
    ``scales [experts, n, ceil(k / 32)]`` are the experts' weights in MXFP4, ``bias [experts, n]`` is
    BF16, FP16 or FP32. Returns ``y [t * top, n]``; the places of pairs of no expert are zero. Exact products,
    FP32 sums, one rounding to ``out_dtype`` (default: the type of ``x``)."""
    _check_cuda(x, "x")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"x must be torch.bfloat16 or torch.float16, got {x.dtype}")
    _no_grad("mxfp4_expert_linear", x, bias)
    device = x.device
    _check_sort(sort, device)
    _check_rows(x, "x", sort.positions.shape[0] if gather else sort.order.numel())
    _check_mx(codes, scales, "", 3, device)
    experts, n, k = codes.shape[0], codes.shape[1], x.shape[1]
    if sort.offsets.numel() != experts + 1:
        raise ValueError(f"sort has {sort.offsets.numel() - 1} experts and codes {experts}")
    if scales.shape[2] != (k + BLOCK - 1) // BLOCK:
        raise ValueError(f"x has {k} columns, which do not fit the weights' {scales.shape[2]} blocks of {BLOCK}")
    dtype = out_dtype if out_dtype is not None else (out.dtype if out is not None else x.dtype)
    p = _native.MpsMxfp4Product()
    p.out_type, p.bias_type = _type(dtype, "out_dtype"), _check_bias(bias, (experts, n), device)
    rows = sort.order.numel()
    out = _check_out(out, (rows, n), dtype, device)
    if x.stride(1) != 1:
        x = x.contiguous()
    whole = _set_x(p, x, k)
    p.rows = rows
    p.w, p.w_scales, p.out, p.n, p.k = codes.data_ptr(), scales.data_ptr(), out.data_ptr(), n, k
    if bias is not None:
        p.bias = bias.data_ptr()
    p.experts, p.offsets, p.order = experts, sort.offsets.data_ptr(), sort.order.data_ptr()
    p.top, p.gather = max(1, sort.positions.shape[1]), bool(gather)
    _multiply(p, whole, device)
    return out


def int4_expert_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, sort: ExpertSort,
                       zeros: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, *, group: int = 128,
                       gather: bool = False, out_dtype: Optional[torch.dtype] = None,
                       out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``y[j] = x[j] @ w[e].T + bias[e]`` for the rows ``j`` of expert ``e`` in the sorted order.

    As :func:`mxfp4_expert_linear`, with the experts' weights in int4: ``codes [experts, n, 16 * ceil(k / 32)]``,
    ``scales [experts, n, ceil(k / group)]`` and ``zeros`` of that shape or None, as ``int4_linear`` takes
    them. Returns ``y [t * top, n]``; the places of pairs of no expert are zero."""
    _check_cuda(x, "x")
    if x.dtype not in _HALVES:
        raise ValueError(f"x must be torch.bfloat16 or torch.float16, got {x.dtype}")
    _no_grad("int4_expert_linear", x, scales, bias)
    device, group = x.device, int(group)
    _check_sort(sort, device)
    _check_rows(x, "x", sort.positions.shape[0] if gather else sort.order.numel())
    k = x.shape[1]
    _check_int4(codes, scales, zeros, k, group, 3, device)
    experts, n = codes.shape[0], codes.shape[1]
    if sort.offsets.numel() != experts + 1:
        raise ValueError(f"sort has {sort.offsets.numel() - 1} experts and codes {experts}")
    dtype = out_dtype if out_dtype is not None else (out.dtype if out is not None else x.dtype)
    out_type, bias_type, rows = _type(dtype, "out_dtype"), _check_bias(bias, (experts, n), device), sort.order.numel()
    out = _check_out(out, (rows, n), dtype, device)
    if x.stride(1) != 1:
        x = x.contiguous()
    p = _int4_product(x, codes, scales, zeros, bias, group, k, n)
    p.rows, p.out, p.out_type, p.bias_type = rows, out.data_ptr(), out_type, bias_type
    p.experts, p.offsets, p.order = experts, sort.offsets.data_ptr(), sort.order.data_ptr()
    p.top, p.gather = max(1, sort.positions.shape[1]), bool(gather)
    _int4_multiply(p, device)
    return out


_SCORES = {"softmax": _native.MPS_SCORES_SOFTMAX, "sigmoid": _native.MPS_SCORES_SIGMOID}


def _check_logits(logits: torch.Tensor, scores: str) -> int:
    _check_cuda(logits, "logits")
    _type(logits, "logits")
    if logits.dim() != 2:
        raise ValueError("logits must have 2 dimensions")
    if not 1 <= logits.shape[1] <= _native.MPS_MAX_EXPERTS:
        raise ValueError(f"logits must have 1 to {_native.MPS_MAX_EXPERTS} columns, got {logits.shape[1]}")
    code = _SCORES.get(scores)
    if code is None:
        raise ValueError(f"scores must be 'softmax' or 'sigmoid', got {scores!r}")
    return code


def _adjacent(logits: torch.Tensor) -> torch.Tensor:
    return logits if logits.stride(1) == 1 or logits.shape[1] == 1 else logits.contiguous()


def _route(logits, top, code, bias, normalize, scale, shares):
    (t, experts), device = logits.shape, logits.device
    ids = torch.empty((t, top), dtype=torch.int32, device=device)
    weights = torch.empty((t, top), dtype=torch.float32, device=device)
    kept = torch.empty_like(weights) if shares else None
    _call(device, _native.lib().mps_expert_route, logits.data_ptr(), _TYPES[logits.dtype], t, experts, logits.stride(0), top, code,
          bias.data_ptr() if bias is not None else None, normalize, scale, ids.data_ptr(), weights.data_ptr(),
          kept.data_ptr() if shares else None)
    return ids, weights, kept


class _NoSecond(torch.autograd.Function):
    """A gradient that has none itself: of a tensor that hangs on ``sources``, so that one is refused, not left out."""

    @staticmethod
    def forward(ctx, gradient, name, *sources):
        ctx.name = name
        return gradient

    @staticmethod
    def backward(ctx, _):
        raise RuntimeError(f"the gradient of {ctx.name} has no gradient")


def _only_gradient(gradient, name, ctx, grad):
    if torch.is_grad_enabled():
        with torch.no_grad():
            d = gradient(ctx, grad)
        return _NoSecond.apply(d, name, grad, ctx.saved_tensors[0])
    return gradient(ctx, grad)


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top, code, bias, normalize, scale):
        ids, weights, shares = _route(logits, top, code, bias, normalize, scale, scale != 1.0)
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, ids, weights if shares is None else shares)
        # what the backward pass would ask for again, on the engine's thread; not the stride, which a hook may change
        ctx.how = _native.lib().mps_expert_route_grad, logits.dtype, logits.shape, top, code, normalize, scale
        return ids, weights

    @staticmethod
    def backward(ctx, _, dweights):
        return None if dweights is None else _only_gradient(_route_grad, "expert_route", ctx, dweights), None, None, None, None, None


def _route_grad(ctx, dweights):
    logits, ids, shares = ctx.saved_tensors
    entry, dtype, shape, top, code, normalize, scale = ctx.how
    (t, experts), device, chosen = shape, dweights.device, dweights.shape
    logits = _kept(logits, shape, dtype, device, True)
    ids = _kept(ids, chosen, torch.int32, device)
    shares = _kept(shares, chosen, torch.float32, device)
    if not dweights.is_contiguous():
        dweights = dweights.contiguous()
    dlogits = logits.new_empty((t, experts))
    _call(device, entry, logits.data_ptr(), _TYPES[dtype], t, experts, logits.stride(0), top, code, normalize, scale, ids.data_ptr(),
          shares.data_ptr(), dweights.data_ptr(), dlogits.data_ptr())
    return dlogits


def expert_route(logits: torch.Tensor, top: int, *, scores: str = "softmax", bias: Optional[torch.Tensor] = None,
                 normalize: bool = True, scale: float = 1.0) -> ExpertRoute:
    """The ``top`` experts of each token, by falling score, and their weights.

    ``logits [t, experts]`` are BF16, FP16 or FP32; ``scores`` is ``"softmax"`` (over a token's logits) or
    ``"sigmoid"``. The experts of the largest logits are taken, or with ``bias [experts]`` (FP32) those of the largest
    ``score + bias``, compared in FP64; ties go to the lower expert. The bias counts for the choice only. A weight is the expert's score,
    with ``normalize`` divided by the sum of the token's chosen scores, times ``scale``. An expert whose logit or
    bias is -inf or NaN is not taken (a token's softmax weights are NaN where it has a logit that is NaN or +inf, and the
    bias alone chooses there): where fewer than ``top`` are left, as in a row of padding, ids are
    -1 and weights 0, which :func:`expert_sort` and :func:`expert_combine` take for no expert. The gradient is that of the
    weights; the choice has none."""
    code = _check_logits(logits, scores)
    top = int(top)
    (t, experts), device = logits.shape, logits.device
    if not 0 <= top <= experts:
        raise ValueError(f"top must be in [0, {experts}], got {top}")
    if bias is not None:
        _check_cuda_contig(bias, "bias", device)
        if bias.dtype != torch.float32 or tuple(bias.shape) != (experts,):
            raise ValueError(f"bias must be torch.float32 of shape {(experts,)}, got {bias.dtype} {tuple(bias.shape)}")
        _no_grad("the bias of expert_route", bias)
    if forward_ad._current_level >= 0:
        _no_tangent("expert_route", logits)
    logits, normalize, scale = _adjacent(logits), bool(normalize), float(scale)
    if logits.requires_grad and torch.is_grad_enabled():
        return ExpertRoute(*_Route.apply(logits, top, code, bias, normalize, scale))
    return ExpertRoute(*_route(logits, top, code, bias, normalize, scale, False)[:2])


def _balance(logits, ids, code, keep):
    (t, experts), device = logits.shape, logits.device
    lib = _native.lib()
    need = ctypes.c_int64(0)
    rc = lib.mps_expert_balance_workspace(t, experts, ids.shape[1], need)
    if rc:
        _native.check(rc)
    loss = torch.empty((), dtype=torch.float32, device=device)
    counts = torch.empty(experts, dtype=torch.int32, device=device)
    kept = torch.empty(experts + 1, dtype=torch.int32, device=device) if keep else None
    work = torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None
    _call(device, lib.mps_expert_balance, logits.data_ptr(), _TYPES[logits.dtype], t, experts, logits.stride(0), code, ids.data_ptr(),
          ids.dtype == torch.int64, ids.shape[1], loss.data_ptr(), counts.data_ptr(), kept.data_ptr() if keep else None,
          work.data_ptr() if need.value else None, need.value)
    return loss, counts, kept


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, code):
        loss, counts, kept = _balance(logits, ids, code, True)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, kept)  # not the counts: a program may add up its ranks' in place
        ctx.how = _native.lib().mps_expert_balance_grad, logits.dtype, logits.shape, code  # as in _Route
        return loss, counts

    @staticmethod
    def backward(ctx, dloss, _):
        return None if dloss is None else _only_gradient(_balance_grad, "expert_balance", ctx, dloss), None, None


def _balance_grad(ctx, dloss):
    logits, kept = ctx.saved_tensors
    entry, dtype, shape, code = ctx.how
    (t, experts), device = shape, dloss.device
    logits = _kept(logits, shape, dtype, device, True)
    kept = _kept(kept, (experts + 1,), torch.int32, device)
    dlogits = logits.new_empty((t, experts))
    _call(device, entry, logits.data_ptr(), _TYPES[dtype], t, experts, logits.stride(0), code, kept.data_ptr(), dloss.data_ptr(),
          dlogits.data_ptr())
    return dlogits


def expert_balance(logits: torch.Tensor, ids: torch.Tensor, *, scores: str = "softmax") -> ExpertBalance:
    """The balance loss of a batch, ``experts * sum over e of f[e] * P[e]``, and each expert's count of pairs.

    ``f[e]`` is the share of the pairs of ``ids [t, top]`` (int32 or int64; an id outside ``[0, experts)`` is no expert's)
    that are expert ``e``'s, ``P[e]`` the mean over the tokens of ``p[t, e]``, the softmax of ``logits [t, experts]``
    (BF16, FP16 or FP32) or, for ``"sigmoid"``, their sigmoids divided by the token's sum of them. The loss is 1 where either is alike for
    all experts. Tokens whose logits are all -inf, as padding's are, count for nothing; without pairs or tokens the loss is
    0. Sums are in a fixed order. The gradient is that of ``P``: the counts have none."""
    code = _check_logits(logits, scores)
    _check_cuda_contig(ids, "ids", logits.device)
    if ids.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"ids must be torch.int32 or torch.int64, got {ids.dtype}")
    if ids.dim() != 2 or ids.shape[0] != logits.shape[0]:
        raise ValueError(f"ids must have shape [{logits.shape[0]}, top], got {tuple(ids.shape)}")
    if forward_ad._current_level >= 0:
        _no_tangent("expert_balance", logits)
    logits = _adjacent(logits)
    if logits.requires_grad and torch.is_grad_enabled():
        return ExpertBalance(*_Balance.apply(logits, ids, code))
    return ExpertBalance(*_balance(logits, ids, code, False)[:2])
