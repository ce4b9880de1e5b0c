"""The performance cases of the MXFP4 operators and of the experts they serve.

A user of this framework turns BF16 weights (decoded from a checkpoint's sidecar) and
activations into microscaled 4-bit floating point, multiplies by such weights, and sends
the tokens of a mixture of experts to their experts and back. MXFP4 holds a row in blocks
of 32 elements: a scale 2^(s - 127) in a byte ``s`` and 32 codes of 4 bits (a sign and
one of 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte, the first in the low half. A row's last
block is filled up with zero codes.

A case is a dict of plain values:

``kind``     what one pass is:
             ``quantize``  a tensor [t, k] to MXFP4 and back to its own type;
             ``linear``    x [t, k] in 16 bits times a weight [n, k] in MXFP4;
             ``matmul``    x [t, k] quantized to MXFP4, times a weight [n, k] in MXFP4;
             ``experts``   tokens sorted by expert, each row times its expert's weight
                           [n, k] in MXFP4, and the weighted sum of a token's rows;
             ``dispatch``  a training step's way to the experts and back: sort, gather, the
                           weighted sum of the experts' rows, and the gradients of the
                           tokens, of the experts' rows and of the weights.
``t``, ``k``, ``n``  tokens (rows), inputs, outputs.
``dtype``    the type of x.
``bias``     whether a bias is added.
``experts``, ``top``  experts, and experts a token.
``dropped``  share of the (token, expert) pairs that are routed to no expert here.
"""
from __future__ import annotations

import torch

own = False

DEVICE = "cuda"
BLOCK = 32
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
LARGEST_FLOPS = 2 * 8192 * 8192 * 28672


def _quantize(t, k, dtype):
    return {"kind": "quantize", "t": t, "k": k, "dtype": dtype}


def _linear(kind, t, k, n, dtype, bias=False):
    return {"kind": kind, "t": t, "k": k, "n": n, "dtype": dtype, "bias": bias}


def _experts(t, k, n, experts, top, dtype, bias=False, dropped=0.0):
    return {"kind": "experts", "t": t, "k": k, "n": n, "experts": experts, "top": top, "dtype": dtype, "bias": bias,
            "dropped": dropped}


def _dispatch(t, k, experts, top, dtype, dropped=0.0):
    return {"kind": "dispatch", "t": t, "k": k, "experts": experts, "top": top, "dtype": dtype, "dropped": dropped}


def listed():
    return [
        # One token's activations before a product: the calls' own latency counts.
        dict(_quantize(1, 4096, "bf16"), name="quantize_token"),
        # An odd width in 32 bits (a state or a gradient that is kept in 4 bits).
        dict(_quantize(1000, 5001, "f32"), name="quantize_ragged"),
        # A gate projection of an 8B layer, quantized offline or right after its decode.
        dict(_quantize(14336, 4096, "bf16"), name="quantize_gate"),
        # Decoding one token: the gate projection of an 8B layer, bound by the weight's bytes.
        dict(_linear("linear", 1, 4096, 14336, "bf16"), name="linear_token"),
        # A few tokens of several requests in FP16, and a weight of odd widths with a bias.
        dict(_linear("linear", 37, 5000, 3001, "f16", bias=True), name="linear_ragged"),
        # A prompt through the gate projection of an 8B layer.
        dict(_linear("linear", 4096, 4096, 14336, "bf16"), name="linear_prompt"),
        # A decoding batch through an attention projection of a 70B layer, activations in 4 bits too.
        dict(_linear("matmul", 64, 8192, 8192, "bf16"), name="matmul_batch"),
        # Prompts through the gate projection of a 70B layer, activations in 4 bits too: the largest.
        dict(_linear("matmul", 8192, 8192, 28672, "bf16"), name="matmul_prompt"),
        # Decoding a few tokens through 64 experts: each is met by hardly any row, some by none.
        dict(_experts(4, 4096, 2048, 64, 4, "bf16", bias=True), name="experts_token"),
        # A prompt through 64 experts of uneven load, some pairs on another rank.
        dict(_experts(8192, 4096, 2048, 64, 4, "bf16", dropped=0.05), name="experts_prompt"),
        # A small training step of odd sizes in 32 bits.
        dict(_dispatch(37, 1001, 8, 2, "f32", dropped=0.05), name="dispatch_small"),
        # A training step over 128 experts, eight a token.
        dict(_dispatch(8192, 4096, 128, 8, "bf16"), name="dispatch_train"),
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
    case = _drawn(rng)
    return {name: 3104 if value == 3072 else value for name, value in case.items()}


def _drawn(rng):
    kind = rng.choice(["quantize", "linear", "linear", "matmul", "matmul", "experts", "experts", "dispatch"])
    if kind == "quantize":
        k = _width(rng, 32, 28672)
        return _quantize(min(_between(rng, 1, 32768), 14336 * 4096 // k), k, rng.choice(["bf16", "bf16", "f16", "f32"]))
    if kind in ("linear", "matmul"):
        t, k, n = _between(rng, 1, 8192), _width(rng, 64, 28672), _width(rng, 64, 28672)
        most = LARGEST_FLOPS // (1 if kind == "matmul" else 4)
        while 2 * t * k * n > most:
            t = (t + 1) // 2
        return _linear(kind, t, k, n, rng.choice(["bf16", "bf16", "f16"]), rng.random() < 0.3)
    experts = rng.choice([4, 8, 16, 60, 64, 128])
    top = min(experts, rng.choice([1, 2, 4, 6, 8]))
    t, dropped = _between(rng, 1, 8192), rng.choice([0.0, 0.0, 0.05, 0.5])
    if kind == "dispatch":
        k = _width(rng, 64, 8192)
        while t * top * k > 8192 * 8 * 4096:
            t = (t + 1) // 2
        return _dispatch(t, k, experts, top, rng.choice(["bf16", "bf16", "f16", "f32"]), dropped)
    k, n = _width(rng, 64, 8192), _width(rng, 64, 8192)
    while experts * k * n > 64 * 4096 * 2048:
        n = (n + 1) // 2
    while 2 * t * top * k * n > LARGEST_FLOPS // 4:
        t = (t + 1) // 2
    return _experts(t, k, n, experts, top, rng.choice(["bf16", "bf16", "f16"]), rng.random() < 0.3, dropped)


# --------------------------------------------------------------------------- plain forms
def _blocks(x, k):
    """x [..., k] as [..., blocks, 32], the last block filled up with zeros."""
    return torch.nn.functional.pad(x, (0, -k % BLOCK)).reshape(*x.shape[:-1], -1, BLOCK)


def plain_quantize(x):
    """(codes [..., 16 * blocks] u8, scales [..., blocks] u8) of x [..., k]."""
    b = _blocks(x.float(), x.shape[-1])
    top = b.abs().amax(dim=-1, keepdim=True)
    e = torch.frexp(top).exponent - 3  # floor(log2(top)) - 2: top is in [2^(e + 2), 2^(e + 3))
    e = torch.where(top > 0, e, torch.full_like(e, -127)).clamp(min=-127)
    half = (e / 2).floor().to(e.dtype)
    v = torch.ldexp(torch.ldexp(b, -half), half - e).abs()
    code = ((v > 0.25).to(torch.uint8) + (v >= 0.75) + (v > 1.25) + (v >= 1.75) + (v > 2.5) + (v >= 3.5) + (v > 5.0)).to(torch.uint8)
    code = code + 8 * torch.signbit(b).to(torch.uint8)
    finite = torch.isfinite(top)
    code = torch.where(finite, code, torch.zeros_like(code))
    scale = torch.where(finite, e + 127, torch.full_like(e, 255)).to(torch.uint8).squeeze(-1)
    code = code.reshape(*x.shape[:-1], -1)
    return code[..., 0::2] + 16 * code[..., 1::2], scale


def plain_dequantize(codes, scales, k):
    """The values [..., k] in 32 bits."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    code = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(*scales.shape, BLOCK).int()
    scale = torch.exp2(scales.float() - 127.0)
    scale = torch.where(scales == 255, torch.full_like(scale, float("nan")), scale)
    return (table[code] * scale.unsqueeze(-1)).reshape(*scales.shape[:-1], -1)[..., :k]


def _plain_sort(ids, experts):
    """(where each pair [t, top] stands among the sorted ones or -1, offsets [experts + 1])."""
    flat = ids.reshape(-1, 1)
    hit = (flat == torch.arange(experts, device=ids.device)).int()
    seen = hit.cumsum(0, dtype=torch.int32)
    counts = seen[-1]
    offsets = torch.nn.functional.pad(counts.cumsum(0, dtype=torch.int32), (1, 0))
    at = ((seen - 1 + offsets[:-1]) * hit).sum(dim=1, dtype=torch.int32)
    there = hit.sum(dim=1) > 0
    return torch.where(there, at, torch.full_like(at, -1)).reshape(ids.shape), offsets


def _plain_linear(x, codes, scales, bias):
    y = x.float() @ plain_dequantize(codes, scales, x.shape[-1]).t()
    return y if bias is None else y + bias.float()


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
    w = plain_dequantize(s["codes"], s["scales"], k)
    y = torch.bmm(w, rows[:experts].transpose(1, 2).contiguous())  # [experts, n, most]
    if s["bias"] is not None:
        y = y + s["bias"].float().unsqueeze(-1)
    inside = e.clamp(max=experts - 1)
    mine = y[inside, :, row] * (there * s["weights"].reshape(-1)).unsqueeze(1)
    return mine.reshape(*ids.shape, -1).sum(dim=1).to(x.dtype)


def _plain_dispatch(s):
    x, y, ids, w = s["x"].float(), s["y"].float(), s["ids"], s["weights"]
    dout, drows, dtype = s["dout"].float(), s["drows"].float(), s["x"].dtype
    at, offsets = _plain_sort(ids, s["experts"])
    pairs, k = ids.numel(), x.shape[1]
    there = (at >= 0).unsqueeze(-1)
    where = torch.where(at >= 0, at, torch.full_like(at, pairs)).reshape(-1).long()  # one more row for pairs of no expert
    read = where.clamp(max=pairs - 1)
    rows = torch.zeros(pairs + 1, k, device=x.device)
    rows[where] = x.repeat_interleave(ids.shape[1], dim=0)
    rows[pairs] = 0
    mine = torch.where(there, y[read].reshape(*ids.shape, k), torch.zeros((), device=x.device))
    out = (mine * w.unsqueeze(-1)).sum(dim=1)
    dw = (mine * dout.unsqueeze(1)).sum(dim=-1)
    dy = torch.zeros(pairs + 1, k, device=x.device)
    dy[where] = (dout.unsqueeze(1) * w.unsqueeze(-1)).reshape(-1, k)
    dx = torch.where(there, drows[read].reshape(*ids.shape, k), torch.zeros((), device=x.device)).sum(dim=1)
    return {"rows": rows[:pairs].to(dtype), "out": out.to(dtype), "dx": dx.to(dtype), "dy": dy[:pairs].to(dtype), "dw": dw,
            "positions": at, "offsets": offsets}


# --------------------------------------------------------------------------- the calls
def _own(case_kind, s):
    from mpserve_amd.experts import expert_combine, expert_gather, expert_sort, mxfp4_expert_linear
    from mpserve_amd.mxfp4 import mxfp4_dequantize, mxfp4_linear, mxfp4_matmul, mxfp4_quantize

    x = s["x"]
    if case_kind == "quantize":
        codes, scales = mxfp4_quantize(x)
        return mxfp4_dequantize(codes, scales, x.shape[1], x.dtype)
    if case_kind == "linear":
        return mxfp4_linear(x, s["codes"], s["scales"], s["bias"])
    if case_kind == "matmul":
        codes, scales = mxfp4_quantize(x)
        return mxfp4_matmul(codes, scales, s["codes"], s["scales"], s["bias"], out_dtype=x.dtype)
    if case_kind == "experts":
        sort = expert_sort(s["ids"], s["codes"].shape[0])
        y = mxfp4_expert_linear(x, s["codes"], s["scales"], sort, s["bias"], gather=True)
        return expert_combine(y, s["weights"], sort)
    x, y, weights = (s[name].detach().requires_grad_() for name in ("x", "y", "weights"))
    sort = expert_sort(s["ids"], s["experts"])
    rows = expert_gather(x, sort)
    out = expert_combine(y, weights, sort)
    dy, dw, dx = torch.autograd.grad((out, rows), (y, weights, x), (s["dout"], s["drows"]))
    return {"rows": rows.detach(), "out": out.detach(), "dx": dx, "dy": dy, "dw": dw, "positions": sort.positions,
            "offsets": sort.offsets}


def run(state):
    kind = state["kind"]
    if own:
        return _own(kind, state)
    x = state["x"]
    if kind == "quantize":
        return plain_dequantize(*plain_quantize(x), x.shape[1]).to(x.dtype)
    if kind == "linear":
        return _plain_linear(x, state["codes"], state["scales"], state["bias"]).to(x.dtype)
    if kind == "matmul":
        rounded = plain_dequantize(*plain_quantize(x), x.shape[1])
        return _plain_linear(rounded, state["codes"], state["scales"], state["bias"]).to(x.dtype)
    return _plain_experts(state) if kind == "experts" else _plain_dispatch(state)


# --------------------------------------------------------------------------- inputs
def _activations(g, t, k, dtype):
    """Rows whose channels differ in size, a few of them by far, as before a layer's products."""
    size = torch.exp(0.5 * torch.randn(k, generator=g, device=DEVICE))
    size = torch.where(torch.rand(k, generator=g, device=DEVICE) < 0.002, 8.0 * size, size)
    return (torch.randn(t, k, generator=g, device=DEVICE) * size).to(dtype)


def _weight(g, rows, k):
    """MXFP4 of a weight with sigma 0.02 whose rows differ in size; rows in chunks, which bounds the memory."""
    codes = torch.empty(rows, (k + BLOCK - 1) // BLOCK * 16, dtype=torch.uint8, device=DEVICE)
    scales = torch.empty(rows, (k + BLOCK - 1) // BLOCK, dtype=torch.uint8, device=DEVICE)
    step = max(1, (1 << 28) // k)
    for r in range(0, rows, step):
        m = min(step, rows - r)
        size = 0.02 * torch.exp(0.3 * torch.randn(m, 1, generator=g, device=DEVICE))
        codes[r:r + m], scales[r:r + m] = plain_quantize(torch.randn(m, k, generator=g, device=DEVICE) * size)
    return codes, scales


def _routing(g, t, experts, top, dropped):
    """(ids [t, top] int32, weights [t, top]) of a router whose experts are not equally liked."""
    logits = torch.randn(t, experts, generator=g, device=DEVICE) + 0.5 * torch.randn(experts, generator=g, device=DEVICE)
    best, ids = logits.topk(top, dim=1)
    ids = ids.int()
    if dropped:
        ids = torch.where(torch.rand(t, top, generator=g, device=DEVICE) < dropped, torch.full_like(ids, -1), ids)
    return ids, torch.softmax(best, dim=1)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    s = {"kind": kind, "x": _activations(g, case["t"], case["k"], dtype)}
    if kind in ("experts", "dispatch"):
        s["ids"], s["weights"] = _routing(g, case["t"], case["experts"], case["top"], case["dropped"])
    if kind == "dispatch":
        s["experts"], pairs = case["experts"], case["t"] * case["top"]
        s["y"] = _activations(g, pairs, case["k"], dtype)  # the experts' answers, and the gradients of both ways
        s["dout"], s["drows"] = (torch.randn(r, case["k"], generator=g, device=DEVICE).to(dtype) for r in (case["t"], pairs))
    if kind in ("linear", "matmul", "experts"):
        e, n = case.get("experts", 1), case["n"]
        s["codes"], s["scales"] = _weight(g, e * n, case["k"])
        s["bias"] = (0.1 * torch.randn(e, n, generator=g, device=DEVICE)).to(dtype) if case["bias"] else None
        if kind == "experts":
            s["codes"], s["scales"] = s["codes"].view(e, n, -1), s["scales"].view(e, n, -1)
        elif case["bias"]:
            s["bias"] = s["bias"][0]
    return s


def work(case):
    kind, t, k, size = case["kind"], case["t"], case["k"], SIZE[case["dtype"]]
    blocks = (k + BLOCK - 1) // BLOCK
    if kind == "quantize":  # x in, codes and scales, the values
        return {"bytes": t * k * size * 2 + t * blocks * 17, "flops": 2 * t * k}
    pairs = t * case.get("top", 1) * (1.0 - case.get("dropped", 0.0))
    routing = t * case.get("top", 1) * 8
    if kind == "dispatch":  # x, y and the gradients dout, drows in; rows, out, dx, dy, dw out
        return {"bytes": (4 * t + 4 * t * case["top"]) * k * size + 2 * routing, "flops": 6 * pairs * k}
    n, e = case["n"], case.get("experts", 1)
    met = e if kind != "experts" else e * (1.0 - (1.0 - 1.0 / e) ** pairs)  # experts that get a row, if all were alike
    bias = met * n * size if case["bias"] else 0
    return {"bytes": t * k * size + met * n * blocks * 17 + t * n * size + bias + (routing if kind == "experts" else 0),
            "flops": 2 * pairs * k * n}


# --------------------------------------------------------------------------- 64 bits
def _exact_quantize(x):
    """The values that MXFP4 holds of x [t, k], from the format's definition, in 64 bits."""
    t, k = x.shape
    v = torch.zeros(t, (k + BLOCK - 1) // BLOCK * BLOCK, dtype=torch.float64, device=x.device)
    v[:, :k] = x.double()
    v = v.view(t, -1, BLOCK)
    top = v.abs().amax(dim=-1, keepdim=True)
    # whole logarithms in 64 bits, put right where log2 has rounded over a power of two
    e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top))))
    e = torch.where(torch.exp2(e) > top, e - 1, e)
    e = torch.where(torch.exp2(e + 1) <= top, e + 1, e)
    scale = torch.exp2(torch.where(top > 0, e - 2, torch.full_like(e, -127.0)).clamp(min=-127.0))
    a = (v / scale).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()  # the spacing of the codes
    a = (torch.round(a / step) * step).clamp(max=6.0)  # ties to the even code
    return (torch.copysign(a, v) * scale).view(t, -1)[:, :k]


def _exact_weight(codes, scales, k):
    """The values of MXFP4 codes from their bits (sign, two of exponent, one of mantissa) in 64 bits."""
    rows = codes.shape[0]
    nibble = torch.empty(rows, codes.shape[1] * 2, dtype=torch.int64, device=codes.device)
    nibble[:, 0::2], nibble[:, 1::2] = (codes % 16).long(), (codes // 16).long()
    ex, m = nibble // 2 % 4, (nibble % 2).double()
    a = torch.where(ex > 0, torch.exp2((ex - 1).double()) * (1 + 0.5 * m), 0.5 * m)
    a = torch.where(nibble >= 8, -a, a).view(rows, -1, BLOCK)
    return (a * torch.exp2(scales.double() - 127.0).unsqueeze(-1)).view(rows, -1)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    kind, x, k = s["kind"], s["x"], case["k"]
    if kind == "quantize":
        return _exact_quantize(x)
    if kind in ("linear", "matmul"):
        xe = x.double() if kind == "linear" else _exact_quantize(x)
        y = xe @ _exact_weight(s["codes"], s["scales"], k).T
        return y + s["bias"].double() if s["bias"] is not None else y
    ids, w = s["ids"].long(), s["weights"].double()
    if kind == "experts":
        out = torch.zeros(case["t"], case["n"], dtype=torch.float64, device=x.device)
        for e in range(case["experts"]):
            token, slot = torch.where(ids == e)
            if token.numel():
                y = x[token].double() @ _exact_weight(s["codes"][e], s["scales"][e], k).T
                if s["bias"] is not None:
                    y = y + s["bias"][e].double()
                out[token] += w[token, slot].unsqueeze(1) * y  # a token meets an expert once
        return out
    xd, yd, dout, drows, pairs = x.double(), s["y"].double(), s["dout"].double(), s["drows"].double(), ids.numel()
    key = torch.where(ids >= 0, ids, torch.full_like(ids, case["experts"])).reshape(-1)
    order = torch.sort(key, stable=True).indices
    kept = int((key < case["experts"]).sum())
    order, token = order[:kept], order[:kept] // case["top"]
    positions = torch.full((pairs,), -1, dtype=torch.int32, device=x.device)
    positions[order] = torch.arange(kept, dtype=torch.int32, device=x.device)
    offsets = torch.searchsorted(torch.sort(key).values, torch.arange(case["experts"] + 1, device=x.device)).int()
    rows, dy = torch.zeros_like(yd), torch.zeros_like(yd)
    out, dx, dw = torch.zeros_like(xd), torch.zeros_like(xd), torch.zeros(pairs, dtype=torch.float64, device=x.device)
    share = w.reshape(-1)[order].unsqueeze(1)
    rows[:kept], dy[:kept] = xd[token], dout[token] * share
    out.index_add_(0, token, yd[:kept] * share)
    dx.index_add_(0, token, drows[:kept])
    dw[order] = (yd[:kept] * dout[token]).sum(1)
    return {"rows": rows, "out": out, "dx": dx, "dy": dy, "dw": dw.view(ids.shape), "positions": positions.view(ids.shape),
            "offsets": offsets}
