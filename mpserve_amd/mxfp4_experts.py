"""A mixture-of-experts block over MXFP4 weights: the MXFP4 and expert operators as a serving program uses them.

``Mxfp4Experts`` holds the experts' gate/up and down projections in MXFP4, and optionally a
shared expert's, whose gate/up product takes its activations in MXFP4 too. It rounds to the type of ``x``
after each step, or with ``rounded=False`` as little as it can. The weights may come
from anywhere in BF16, for instance from a checkpoint's FP8 bytes and sidecars through
``DecodePlan``, which is what the command does with small synthetic ones:

    python -m mpserve_amd.mxfp4_experts --tokens 64 --experts 16 --top 4
"""
from __future__ import annotations

import argparse
from typing import Optional, Tuple

import torch

from .experts import expert_combine, expert_sort, mxfp4_expert_linear
from .mxfp4 import mxfp4_linear, mxfp4_matmul, mxfp4_quantize


def _gated(h: torch.Tensor) -> torch.Tensor:
    gate, up = h.chunk(2, dim=-1)
    return torch.nn.functional.silu(gate) * up


class Mxfp4Experts:
    """``gate_up [experts, 2 * ffn, hidden]`` and ``down [experts, hidden, ffn]`` in BF16, FP16 or FP32;
    ``shared``: the same pair of a shared expert, ``[2 * ffn, hidden]`` and ``[hidden, ffn]``.
    ``rounded=False``: the down products stay FP32 until they are added up, and the shared expert takes its
    activations as they are, not in MXFP4."""

    def __init__(self, gate_up: torch.Tensor, down: torch.Tensor, top: int,
                 shared: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, rounded: bool = True):
        self.experts, self.top, self.rounded = gate_up.shape[0], int(top), bool(rounded)
        self.gate_up, self.down = mxfp4_quantize(gate_up), mxfp4_quantize(down)
        self.shared = None if shared is None else tuple(mxfp4_quantize(w) for w in shared)

    @torch.no_grad()
    def __call__(self, x: torch.Tensor, router_logits: torch.Tensor) -> torch.Tensor:
        """``x [tokens, hidden]`` in BF16 or FP16, ``router_logits [tokens, experts]``."""
        best, ids = router_logits.float().topk(self.top, dim=-1)
        weights = torch.softmax(best, dim=-1)
        sort = expert_sort(ids, self.experts)
        h = _gated(mxfp4_expert_linear(x, *self.gate_up, sort, gather=True))
        rows = x.dtype if self.rounded else torch.float32
        out = expert_combine(mxfp4_expert_linear(h, *self.down, sort, out_dtype=rows), weights, sort)
        if self.shared is not None:
            gate_up, down = self.shared
            h = mxfp4_matmul(*mxfp4_quantize(x), *gate_up, out_dtype=x.dtype) if self.rounded else mxfp4_linear(x, *gate_up)
            out = out + mxfp4_linear(_gated(h), *down, out_dtype=rows)
        return out.to(x.dtype)


def decoded_weight(shape, seed: int, device: torch.device) -> torch.Tensor:
    """A synthetic weight, as a loader gets it: FP8 bytes and a sidecar, decoded to BF16 by one plan."""
    import MPServe_cuda

    from .decode import DecodePlan
    from .synthetic import make_weight

    n, m = shape[0] * shape[1] if len(shape) == 3 else shape[0], shape[-1]
    w = make_weight(n, m, sigma=0.02, seed=seed, device=device)
    sidecar = MPServe_cuda.huffman_build_fp8_decode_tables(w.bf16, w.fp8_u8, w.scale_u16, max_len=7, threads_per_block=1024)
    out = torch.empty((n, m), dtype=torch.bfloat16, device=device)
    DecodePlan([(w.fp8_u8, sidecar, out)]).decode()
    torch.cuda.current_stream(device).synchronize()  # the plan and the sidecar go with this call
    return out.view(shape)


def main(argv=None) -> int:
    p = argparse.ArgumentParser(description="run a block of MXFP4 experts on synthetic weights")
    p.add_argument("--tokens", type=int, default=64)
    p.add_argument("--hidden", type=int, default=1024)
    p.add_argument("--ffn", type=int, default=512)
    p.add_argument("--experts", type=int, default=16)
    p.add_argument("--top", type=int, default=4)
    a = p.parse_args(argv)
    device = torch.device("cuda", torch.cuda.current_device())
    shapes = [(a.experts, 2 * a.ffn, a.hidden), (a.experts, a.hidden, a.ffn), (2 * a.ffn, a.hidden), (a.hidden, a.ffn)]
    weights = [decoded_weight(s, i, device) for i, s in enumerate(shapes)]
    block = Mxfp4Experts(weights[0], weights[1], a.top, shared=(weights[2], weights[3]))
    g = torch.Generator(device=device).manual_seed(7)
    x = torch.randn(a.tokens, a.hidden, generator=g, device=device).to(torch.bfloat16)
    logits = torch.randn(a.tokens, a.experts, generator=g, device=device)
    out = block(x, logits)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    for _ in range(10):
        block(x, logits)
    end.record()
    end.synchronize()
    held = sum(t.numel() for pair in (block.gate_up, block.down, *block.shared) for t in pair)
    print(f"{a.tokens} tokens, {a.experts} experts ({a.top} a token) and a shared one: {start.elapsed_time(end) * 100:.1f} us a pass; "
          f"weights {held} bytes in MXFP4, {sum(w.numel() for w in weights) * 2} in BF16; output rms {float(out.float().square().mean().sqrt()):.4f}")
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
