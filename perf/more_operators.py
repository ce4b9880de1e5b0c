"""The performance cases of the int4 products and of the router of a mixture of experts.

An AWQ checkpoint holds a weight [n, k] as whole numbers q of 4 bits, and for each group of
neighbouring columns of a row a scale s and a zero z: w = s * (q - z). Its user multiplies by
such weights as they are, sends tokens through experts of such weights, and has a router
choose the experts, in training with a loss that keeps their loads alike.

Codes lie in blocks of 32 elements, 16 bytes each: byte b of each 4 bytes holds element b of
eight in its low half and element b + 4 in its high half. A row's last block is filled up.

A case is a dict of plain values:

``kind``      what one pass is:
              ``linear``      x [t, k] in 16 bits times an int4 weight [n, k];
              ``experts``     tokens sorted by expert, each row times its expert's int4 weight
                              [n, k], and the weighted sum of a token's rows;
              ``route``       from scores to experts: the ids and weights of t tokens;
              ``route_train`` the same, and the gradient of the logits from the weights';
              ``balance``     the balance loss, the counts, and the gradient of the logits.
``t``, ``k``, ``n``  tokens (rows), inputs, outputs.
``dtype``     the type of x and of the scales, or of the logits.
``group``     columns a scale.
``zeros``     whether there are zeros (else z = 8).
``bias``      whether a bias is added (linear, experts), or one to the scores before the choice (route).
``experts``, ``top``  experts, and experts a token.
``dropped``   share of the pairs that are routed to no expert here.
``scores``    softmax or sigmoid.
``normalize`` whether a token's weights are divided by their sum.
``padded``    share of the tokens that only fill up a batch: all their logits are -inf.
"""
from __future__ import annotations

import torch

own = False

DEVICE = "cuda"
BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
LARGEST_FLOPS = 2 * 4096 * 4096 * 14336
LARGEST_SCORES = 65536 * 128
SCALE = 2.5  # what weights of a sigmoid router are multiplied by


def _linear(t, k, n, dtype, group, zeros=True, bias=False):
    return {"kind": "linear", "t": t, "k": k, "n": n, "dtype": dtype, "group": group, "zeros": zeros, "bias": bias}


def _experts(t, k, n, experts, top, dtype, group, zeros=True, bias=False, dropped=0.0):
    return {"kind": "experts", "t": t, "k": k, "n": n, "experts": experts, "top": top, "dtype": dtype, "group": group,
            "zeros": zeros, "bias": bias, "dropped": dropped}


def _route(kind, t, experts, top, dtype, scores, normalize=True, bias=False, padded=0.0):
    return {"kind": kind, "t": t, "experts": experts, "top": top, "dtype": dtype, "scores": scores, "normalize": normalize,
            "bias": bias, "padded": padded}


def _balance(t, experts, top, dtype, scores, padded=0.0):
    return {"kind": "balance", "t": t, "experts": experts, "top": top, "dtype": dtype, "scores": scores, "padded": padded}


def listed():
    return [
        # Decoding one token: the gate projection of an 8B layer, bound by the weight's bytes.
        dict(_linear(1, 4096, 14336, "bf16", 128), name="linear_token"),
        # A few tokens of several requests in FP16, and a weight of odd widths whose last group is cut.
        dict(_linear(37, 5000, 3001, "f16", 64, bias=True), name="linear_ragged"),
        # A decoding batch through an attention projection of a 70B layer, without zeros.
        dict(_linear(64, 8192, 8192, "bf16", 128, zeros=False), name="linear_batch"),
        # A prompt through the gate projection of an 8B layer.
        dict(_linear(4096, 4096, 14336, "bf16", 128), name="linear_prompt"),
        # A shorter prompt through the gate projection of a 70B layer, in FP16 and with the finest groups.
        dict(_linear(1024, 8192, 28672, "f16", 32), name="linear_fine"),
        # Decoding a few tokens through 64 experts: each is met by hardly any row, some by none.
        dict(_experts(4, 4096, 2048, 64, 4, "bf16", 128, bias=True), name="experts_token"),
        # A prompt through 64 experts of uneven load, some pairs on another rank.
        dict(_experts(8192, 4096, 2048, 64, 4, "bf16", 128, dropped=0.05), name="experts_prompt"),
        # The router of that block for a few tokens: the call's own latency counts.
        dict(_route("route", 4, 64, 4, "f32", "softmax"), name="route_token"),
        # A prompt through a router of sigmoid scores whose loads a bias keeps alike.
        dict(_route("route", 8192, 256, 8, "f32", "sigmoid", bias=True), name="route_prompt"),
        # A training step's router, some of the batch being padding.
        dict(_route("route_train", 65536, 128, 8, "f32", "softmax", padded=0.05), name="route_train"),
        # A small training step of odd sizes.
        dict(_balance(37, 60, 2, "f32", "softmax"), name="balance_small"),
        # A training step's balance loss, its logits in 16 bits.
        dict(_balance(65536, 128, 8, "bf16", "softmax", padded=0.05), name="balance_train"),
    ]


def _between(rng, lo, hi):
    """A whole number whose logarithm is spread evenly."""
    return max(lo, min(hi, int(lo * (hi / lo) ** rng.random() + 0.5)))


def _width(rng, lo, hi):
    """A width: a multiple of 128, of 32, or any number."""
    w = _between(rng, lo, hi)
    step = rng.choice([128, 128, 32, 1])
    return max(step, w // step * step)


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "experts", "experts", "route", "route_train", "balance"])
    experts = rng.choice([4, 8, 16, 60, 64, 128, 256])
    top = min(experts, rng.choice([1, 2, 4, 6, 8]))
    t = _between(rng, 1, 8192)
    dtype, group = rng.choice(["bf16", "bf16", "f16"]), rng.choice([32, 64, 128, 128, 256])
    zeros, bias = rng.random() < 0.6, rng.random() < 0.3
    if kind == "linear":
        k, n = _width(rng, 64, 28672), _width(rng, 64, 28672)
        while 2 * t * k * n > LARGEST_FLOPS:
            t = (t + 1) // 2
        return _linear(t, k, n, dtype, group, zeros, bias)
    if kind == "experts":
        k, n = _width(rng, 64, 8192), _width(rng, 64, 8192)
        while experts * k * n > 64 * 4096 * 2048:
            n = (n + 1) // 2
        while 2 * t * top * k * n > LARGEST_FLOPS:
            t = (t + 1) // 2
        return _experts(t, k, n, experts, top, dtype, group, zeros, bias, rng.choice([0.0, 0.0, 0.05, 0.5]))
    t, dtype = min(_between(rng, 1, 65536), LARGEST_SCORES // experts), rng.choice(["f32", "f32", "bf16", "f16"])
    scores, padded = rng.choice(["softmax", "softmax", "sigmoid"]), rng.choice([0.0, 0.05, 0.5])
    padded = padded if t >= 32 else 0.0
    if kind == "balance":  # tokens that go to all experts have a gradient of zero
        return _balance(t, experts, min(top, experts // 2), dtype, scores, padded)
    normalize = rng.random() < 0.7 and top > 1  # and so has a weight that is always 1
    return _route(kind, t, experts, top, dtype, scores, normalize, bias, padded)


# --------------------------------------------------------------------------- plain forms
def _pack(q):
    """q [rows, k] of whole numbers below 16 as codes [rows, 16 * blocks] u8."""
    q = torch.nn.functional.pad(q, (0, -q.shape[1] % BLOCK)).reshape(q.shape[0], -1, 2, 4)
    return (q[:, :, 0] + 16 * q[:, :, 1]).reshape(q.shape[0], -1)


def _values(codes, k):
    """The whole numbers [..., k] of codes, in 32 bits."""
    c = codes.reshape(*codes.shape[:-1], -1, 1, 4)
    return torch.cat([c & 15, c >> 4], dim=-2).reshape(*codes.shape[:-1], -1)[..., :k].float()


def plain_weight(codes, scales, zeros, k, group):
    """w [..., k] in 32 bits."""
    z = torch.full_like(scales, 8.0).float() if zeros is None else zeros.float()
    wide = lambda v: v.repeat_interleave(group, dim=-1)[..., :k]  # noqa: E731
    return (_values(codes, k) - wide(z)) * wide(scales.float())


def _plain_sort(ids, experts):
    """(where each pair [t, top] stands among the sorted ones or -1, offsets [experts + 1])."""
    flat = ids.reshape(-1, 1)
    hit = (flat == torch.arange(experts, device=ids.device)).int()
    seen = hit.cumsum(0, dtype=torch.int32)
    offsets = torch.nn.functional.pad(seen[-1].cumsum(0, dtype=torch.int32), (1, 0))
    at = ((seen - 1 + offsets[:-1]) * hit).sum(dim=1, dtype=torch.int32)
    return torch.where(hit.sum(dim=1) > 0, at, torch.full_like(at, -1)).reshape(ids.shape), offsets


def _plain_experts(s):
    x, ids, k = s["x"], s["ids"], s["x"].shape[1]
    experts = s["codes"].shape[0]
    at, offsets = _plain_sort(ids, experts)
    most = int((offsets[1:] - offsets[:-1]).max().clamp(min=1))
    there = (at >= 0).reshape(-1)
    e = ids.reshape(-1).clamp(min=0).long()
    row = torch.where(there, at.reshape(-1) - offsets[e], torch.zeros_like(e)).long()
    e = torch.where(there, e, torch.full_like(e, experts))  # pairs of no expert go to one more, which is cut off
    rows = torch.zeros(experts + 1, most, k, device=x.device)
    rows[e, row] = x.float().repeat_interleave(ids.shape[1], dim=0)
    w = plain_weight(s["codes"], s["scales"], s["zeros"], k, s["group"])
    y = torch.bmm(w, rows[:experts].transpose(1, 2).contiguous())  # [experts, n, most]
    if s["bias"] is not None:
        y = y + s["bias"].float().unsqueeze(-1)
    mine = y[e.clamp(max=experts - 1), :, row] * (there * s["weights"].reshape(-1)).unsqueeze(1)
    return mine.reshape(*ids.shape, -1).sum(dim=1).to(x.dtype)


def _plain_scores(logits, scores):
    """(softmax or sigmoid of logits [t, experts], zero in rows that are -inf throughout; those rows)."""
    empty = (logits == float("-inf")).all(dim=1, keepdim=True)
    if scores == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-logits)), empty
    top = torch.where(empty, torch.zeros_like(logits[:, :1]), logits.amax(dim=1, keepdim=True))
    e = torch.exp(logits - top)
    return e / torch.where(empty, torch.ones_like(top), e.sum(dim=1, keepdim=True)), empty


def _plain_route(s):
    logits, top = s["logits"], s["top"]
    score, _ = _plain_scores(logits.float(), s["scores"])
    # The choice falls by the logits themselves or, with a bias, by scores in 64 bits: neighbours are near.
    key = logits.float() if s["bias"] is None else _plain_scores(logits.double(), s["scores"])[0] + s["bias"].double()
    key = torch.where(logits == float("-inf"), torch.full_like(key, float("-inf")), key)
    best, order = torch.sort(key, dim=1, descending=True, stable=True)
    none = best[:, :top] == float("-inf")
    at = order[:, :top]
    mine = torch.where(none, torch.zeros((), device=key.device), score.gather(1, at))
    total = mine.sum(dim=1, keepdim=True) if s["normalize"] else torch.ones_like(mine[:, :1])
    share = mine / torch.where(total > 0, total, torch.ones_like(total))
    out = {"ids": torch.where(none, torch.full_like(at, -1), at).int(), "weights": share * s["scale"]}
    if s["kind"] == "route_train":
        dw = s["dweights"] * s["scale"]
        if s["normalize"]:
            dw = dw - (share * dw).sum(dim=1, keepdim=True)
        dw = torch.where(none, torch.zeros_like(dw), dw)
        ds = torch.zeros_like(score).scatter_add_(1, at, dw / torch.where(total > 0, total, torch.ones_like(total)))
        if s["scores"] == "sigmoid":
            d = ds * score * (1 - score)
        else:
            d = score * (ds - (ds * score).sum(dim=1, keepdim=True))
        out["dlogits"] = d.to(logits.dtype)
    return out


def _plain_balance(s):
    logits, ids = s["logits"], s["ids"]
    experts = logits.shape[1]
    counts = (ids.reshape(-1, 1) == torch.arange(experts, device=ids.device)).sum(dim=0)
    score, empty = _plain_scores(logits.float(), s["scores"])
    p = score
    if s["scores"] == "sigmoid":
        total = score.sum(dim=1, keepdim=True)
        p = score / torch.where(total > 0, total, torch.ones_like(total))
    tokens, pairs = (~empty).sum().clamp(min=1), counts.sum().clamp(min=1)
    mean = p.sum(dim=0, dtype=torch.float64) / tokens
    loss = (experts * (counts * mean).sum() / pairs).float()
    c = counts.float()
    d = p * (c - (c * p).sum(dim=1, keepdim=True)) * (s["dloss"] * experts / (pairs * tokens).float())
    if s["scores"] == "sigmoid":
        d = d * (1 - score)
    return {"loss": loss, "counts": counts.int(), "dlogits": d.to(logits.dtype)}


# --------------------------------------------------------------------------- the calls
def _own(s):
    from mpserve_amd.experts import expert_balance, expert_combine, expert_route, expert_sort, int4_expert_linear
    from mpserve_amd.int4 import int4_linear

    kind = s["kind"]
    if kind == "linear":
        return int4_linear(s["x"], s["codes"], s["scales"], s["zeros"], s["bias"], group=s["group"])
    if kind == "experts":
        sort = expert_sort(s["ids"], s["codes"].shape[0])
        # rows in 32 bits until they are added up: the plain form rounds once, too
        y = int4_expert_linear(s["x"], s["codes"], s["scales"], sort, s["zeros"], s["bias"], group=s["group"], gather=True,
                               out_dtype=torch.float32)
        return expert_combine(y, s["weights"], sort).to(s["x"].dtype)
    if kind == "route":
        ids, weights = expert_route(s["logits"], s["top"], scores=s["scores"], bias=s["bias"], normalize=s["normalize"],
                                    scale=s["scale"])
        return {"ids": ids, "weights": weights}
    logits = s["logits"].detach().requires_grad_()
    if kind == "route_train":
        ids, weights = expert_route(logits, s["top"], scores=s["scores"], bias=s["bias"], normalize=s["normalize"],
                                    scale=s["scale"])
        (dlogits,) = torch.autograd.grad(weights, logits, s["dweights"])
        return {"ids": ids, "weights": weights.detach(), "dlogits": dlogits}
    loss, counts = expert_balance(logits, s["ids"], scores=s["scores"])
    (dlogits,) = torch.autograd.grad(loss, logits, s["dloss"])
    return {"loss": loss.detach(), "counts": counts, "dlogits": dlogits}


def run(state):
    if own:
        return _own(state)
    kind = state["kind"]
    if kind == "linear":
        x = state["x"]
        y = x.float() @ plain_weight(state["codes"], state["scales"], state["zeros"], x.shape[1], state["group"]).t()
        return (y if state["bias"] is None else y + state["bias"].float()).to(x.dtype)
    if kind == "experts":
        return _plain_experts(state)
    return _plain_balance(state) if kind == "balance" else _plain_route(state)


# --------------------------------------------------------------------------- inputs
def _activations(g, t, k, dtype):
    """Rows whose channels differ in size, a few of them by far, as before a layer's products."""
    size = torch.exp(0.5 * torch.randn(k, generator=g, device=DEVICE))
    size = torch.where(torch.rand(k, generator=g, device=DEVICE) < 0.002, 8.0 * size, size)
    return (torch.randn(t, k, generator=g, device=DEVICE) * size).to(dtype)


def _weight(g, rows, k, dtype, group, zeros):
    """int4 of a weight with sigma 0.02 whose rows differ in size, rounded within each group's range (or, without
    zeros, its largest magnitude); rows in chunks, which bounds the memory."""
    groups = (k + group - 1) // group
    codes = torch.empty(rows, (k + BLOCK - 1) // BLOCK * 16, dtype=torch.uint8, device=DEVICE)
    scales = torch.empty(rows, groups, dtype=dtype, device=DEVICE)
    z = torch.empty(rows, groups, dtype=torch.uint8, device=DEVICE) if zeros else None
    step = max(1, (1 << 27) // k)
    for r in range(0, rows, step):
        m = min(step, rows - r)
        size = 0.02 * torch.exp(0.3 * torch.randn(m, 1, generator=g, device=DEVICE))
        w = torch.nn.functional.pad(torch.randn(m, k, generator=g, device=DEVICE) * size, (0, groups * group - k)).view(m, groups, group)
        if zeros:
            lo, hi = w.amin(dim=2).clamp(max=0), w.amax(dim=2).clamp(min=0)
            s = ((hi - lo) / 15).to(dtype)
            z[r:r + m] = torch.round(-lo / s.float()).clamp(0, 15).to(torch.uint8)
            zero = z[r:r + m].float()
        else:
            s = (w.abs().amax(dim=2) / 7).to(dtype)
            zero = torch.full_like(s, 8.0).float()
        scales[r:r + m] = s
        q = (torch.round(w / s.float().unsqueeze(2)) + zero.unsqueeze(2)).clamp(0, 15).to(torch.uint8)
        codes[r:r + m] = _pack(q.view(m, -1)[:, :k])
    return codes, scales, z


def _logits(g, t, experts, dtype, padded):
    """A router's logits, whose experts are not equally liked; padding is -inf."""
    logits = torch.randn(t, experts, generator=g, device=DEVICE) + 0.5 * torch.randn(experts, generator=g, device=DEVICE)
    if padded:
        logits = torch.where(torch.rand(t, 1, generator=g, device=DEVICE) < padded, torch.full_like(logits, float("-inf")), logits)
    return logits.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    kind, dtype, t = case["kind"], DTYPES[case["dtype"]], case["t"]
    s = {"kind": kind}
    if kind in ("linear", "experts"):
        e, n, k = case.get("experts", 1), case["n"], case["k"]
        s["x"], s["group"] = _activations(g, t, k, dtype), case["group"]
        s["codes"], s["scales"], s["zeros"] = _weight(g, e * n, k, dtype, case["group"], case["zeros"])
        s["bias"] = (0.1 * torch.randn(e, n, generator=g, device=DEVICE)).to(dtype) if case["bias"] else None
        if kind == "linear":
            s["bias"] = s["bias"][0] if case["bias"] else None
            return s
        for name in ("codes", "scales", "zeros"):
            s[name] = s[name].view(e, n, -1) if s[name] is not None else None
        best, ids = _logits(g, t, e, torch.float32, 0.0).topk(case["top"], dim=1)
        s["weights"], ids = torch.softmax(best, dim=1), ids.int()
        if case["dropped"]:
            ids = torch.where(torch.rand(*ids.shape, generator=g, device=DEVICE) < case["dropped"], torch.full_like(ids, -1), ids)
        s["ids"] = ids
        return s
    s["logits"], s["scores"] = _logits(g, t, case["experts"], dtype, case["padded"]), case["scores"]
    if kind == "balance":
        best, ids = s["logits"].float().topk(case["top"], dim=1)
        s["ids"] = torch.where(best == float("-inf"), torch.full_like(ids, -1), ids).int()
        # The loss's share in a step's loss; FP16's is scaled up, which keeps its gradients in range.
        s["dloss"] = torch.tensor(float(t) if case["dtype"] == "f16" else 0.01, device=DEVICE)
        return s
    s["top"], s["normalize"], s["scale"] = case["top"], case["normalize"], SCALE if case["scores"] == "sigmoid" else 1.0
    s["bias"] = 0.05 * torch.randn(case["experts"], generator=g, device=DEVICE) if case["bias"] else None
    if kind == "route_train":
        s["dweights"] = torch.randn(t, case["top"], generator=g, device=DEVICE)
    return s


def work(case):
    kind, t, size = case["kind"], case["t"], SIZE[case["dtype"]]
    if kind in ("linear", "experts"):
        k, n, e = case["k"], case["n"], case.get("experts", 1)
        pairs = t * case.get("top", 1) * (1.0 - case.get("dropped", 0.0))
        met = e if kind == "linear" else e * (1.0 - (1.0 - 1.0 / e) ** pairs)  # experts that get a row, if all were alike
        groups = (k + case["group"] - 1) // case["group"]
        weight = n * ((k + BLOCK - 1) // BLOCK * 16 + groups * (size + (1 if case["zeros"] else 0)) + (size if case["bias"] else 0))
        routing = t * case["top"] * 8 if kind == "experts" else 0
        return {"bytes": t * k * size + met * weight + t * n * size + routing, "flops": 2 * pairs * k * n}
    scores, pairs = t * case["experts"], t * case["top"]
    if kind == "route":  # logits in; ids and weights out
        return {"bytes": scores * size + pairs * 8, "flops": 4 * scores}
    if kind == "route_train":  # the weights' gradient in and the logits' out too
        return {"bytes": 2 * scores * size + pairs * 12, "flops": 8 * scores}
    return {"bytes": 2 * scores * size + pairs * 4 + case["experts"] * 4, "flops": 8 * scores}


# --------------------------------------------------------------------------- 64 bits
def _exact_weight(codes, scales, zeros, k, group):
    """w of rows [rows, k], element by element from the layout's definition, in 64 bits."""
    col = torch.arange(k, device=codes.device)
    byte = codes[:, col // 8 * 4 + col % 4].long()
    q = torch.where(col % 8 < 4, byte % 16, byte // 16)
    z = zeros.long()[:, col // group] if zeros is not None else 8
    return (q - z).double() * scales.double()[:, col // group]


def _exact_scores(logits, scores):
    """Scores of rows of which none is -inf throughout."""
    return torch.sigmoid(logits) if scores == "sigmoid" else torch.softmax(logits, dim=1)


def _exact_route(case, s):
    t, experts, top = case["t"], case["experts"], case["top"]
    ids = torch.full((t, top), -1, dtype=torch.int32, device=DEVICE)
    weights = torch.zeros(t, top, dtype=torch.float64, device=DEVICE)
    dlogits = torch.zeros(t, experts, dtype=torch.float64, device=DEVICE)
    live = torch.where((s["logits"] != float("-inf")).any(dim=1))[0]
    lower = torch.arange(experts, device=DEVICE)
    lower = lower.unsqueeze(0) < lower.unsqueeze(1)  # [e, j]: j stands before e
    for rows in live.split(max(1, (1 << 26) // (experts * experts))):
        logits = s["logits"][rows].double().requires_grad_()
        score = _exact_scores(logits, s["scores"])
        key = logits.detach() if s["bias"] is None else score.detach() + s["bias"].double()
        # an expert's rank: how many have a larger key, or the same and a lower number
        rank = ((key.unsqueeze(1) > key.unsqueeze(2)) | ((key.unsqueeze(1) == key.unsqueeze(2)) & lower)).sum(dim=2)
        at = torch.argsort(rank, dim=1)[:, :top]
        mine = score.gather(1, at)
        w = s["scale"] * (mine / mine.sum(dim=1, keepdim=True) if s["normalize"] else mine)
        ids[rows], weights[rows] = at.int(), w.detach()
        if case["kind"] == "route_train":
            dlogits[rows] = torch.autograd.grad(w, logits, s["dweights"][rows].double())[0]
    out = {"ids": ids, "weights": weights}
    if case["kind"] == "route_train":
        out["dlogits"] = dlogits
    return out


def _exact_balance(case, s):
    counts = torch.bincount(s["ids"].reshape(-1).long() + 1, minlength=case["experts"] + 1)[1:]
    dlogits = torch.zeros(case["t"], case["experts"], dtype=torch.float64, device=DEVICE)
    live = torch.where((s["logits"] != float("-inf")).any(dim=1))[0]
    if live.numel() == 0:
        return {"loss": torch.zeros((), dtype=torch.float64, device=DEVICE), "counts": counts.int(), "dlogits": dlogits}
    logits = s["logits"][live].double().requires_grad_()
    p = _exact_scores(logits, s["scores"])
    p = p / p.sum(dim=1, keepdim=True)
    loss = case["experts"] * (counts.double() / counts.sum() * p.mean(dim=0)).sum()
    dlogits[live] = torch.autograd.grad(loss, logits, s["dloss"].double())[0]
    return {"loss": loss.detach(), "counts": counts.int(), "dlogits": dlogits}


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "balance":
        return _exact_balance(case, s)
    if kind in ("route", "route_train"):
        return _exact_route(case, s)
    k, group = case["k"], case["group"]
    if kind == "linear":
        y = s["x"].double() @ _exact_weight(s["codes"], s["scales"], s["zeros"], k, group).T
        return y + s["bias"].double() if s["bias"] is not None else y
    ids, w = s["ids"].long(), s["weights"].double()
    out = torch.zeros(case["t"], case["n"], dtype=torch.float64, device=DEVICE)
    for e in range(case["experts"]):
        token, slot = torch.where(ids == e)
        if token.numel():
            zeros = s["zeros"][e] if s["zeros"] is not None else None
            y = s["x"][token].double() @ _exact_weight(s["codes"][e], s["scales"][e], zeros, k, group).T
            if s["bias"] is not None:
                y = y + s["bias"][e].double()
            out[token] += w[token, slot].unsqueeze(1) * y  # a token meets an expert once
    return out
