"""Microscaled 4-bit floating point (MXFP4): quantization, its inverse and products.

A row of ``k`` elements is held in ``ceil(k / 32)`` blocks of 32: a byte ``s`` a block, its
scale ``2 ** (s - 127)`` (255: the block is NaN), and a code of 4 bits an element (a sign
and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6), two to a byte, the earlier element in the low half.
A row's last block is filled up with zero codes.

* :func:`mxfp4_quantize` — BF16, FP16 or FP32 to codes and scales;
* :func:`mxfp4_dequantize` — back to any of these;
* :func:`mxfp4_linear` — ``x @ w.T + bias`` with 16-bit ``x`` and an MXFP4 weight;
* :func:`mxfp4_matmul` — the same with both operands in MXFP4.

The weights that the decode ops rebuild (``huffman_decode_fp8``, ``DecodePlan``) go straight
into ``mxfp4_quantize``; a weight's codes and scales are kept as they are. All calls run on
the current stream of their tensors' device, do not synchronise, and can be captured into a
graph. They have no gradients, and refuse tensors that ask for one or carry a tangent. The work is done by the
HIP kernels of libmpserve_amd.so; there is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _native
from ._common import _check_cuda_contig

BLOCK = 32

_TYPES = {torch.bfloat16: _native.MPS_TYPE_BF16, torch.float16: _native.MPS_TYPE_F16,
          torch.float32: _native.MPS_TYPE_F32}


def _type(t: torch.Tensor | torch.dtype, name: str) -> int:
    dtype = t if isinstance(t, torch.dtype) else t.dtype
    code = _TYPES.get(dtype)
    if code is None:
        raise ValueError(f"{name} must be torch.bfloat16, torch.float16 or torch.float32, got {dtype}")
    return code


def _no_tangent(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses dual tensors, which need not require a gradient: their tangents would be lost."""
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled():
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative: call it with the primal tensors")


def _no_grad(name: str, *tensors: Optional[torch.Tensor]) -> None:
    if forward_ad._current_level >= 0:
        _no_tangent(name, *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{name} has no gradient: call it under torch.no_grad() or with detached tensors")


def _check_cuda(t: torch.Tensor, name: str, device: Optional[torch.device] = None) -> None:
    if t is None:
        raise ValueError(f"{name} must be defined")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} must be on {device}, got {t.device}")


def _call(device: torch.device, entry, *args) -> None:
    """``entry(*args, stream)`` on the current stream of ``device``. (The raw handle costs 0.1 us, a Stream
    object 1.9 of the 10 that a small call took; the raw device 0.1, torch.cuda.current_device() 0.26.)"""
    index = device.index
    stream = torch._C._cuda_getCurrentRawStream(index)
    if torch._C._cuda_getDevice() == index:
        rc = entry(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = entry(*args, stream)
    if rc:
        _native.check(rc)


def _rows(x: torch.Tensor, k: int) -> torch.Tensor:
    """x [..., k] as rows [r, k] whose elements are adjacent; rows may lie apart (a slice of columns)."""
    if x.dim() != 2:
        x = x.reshape(x.numel() // k if k else 0, k)
    return x if x.stride(1) == 1 or k <= 1 else x.contiguous()


def _check_mx(codes: torch.Tensor, scales: torch.Tensor, name: str, dims: Optional[int] = None,
              device: Optional[torch.device] = None) -> None:
    if codes is not None and scales is not None:  # all is well in one go; what is not is named below
        c, s = codes.shape, scales.shape
        n, at = len(c), codes.device
        if codes.dtype is torch.uint8 and scales.dtype is torch.uint8 and codes.is_cuda and at == scales.device \
                and (device is None or at == device) and codes.is_contiguous() and scales.is_contiguous() \
                and n == len(s) and n >= 1 and (dims is None or n == dims) and c[-1] == 16 * s[-1] \
                and (c[0] == s[0] if n == 2 else c[:-1] == s[:-1]) and not codes.data_ptr() & 15:
            return
    for t, part in ((codes, "codes"), (scales, "scales")):
        full = f"{name}{part}"
        _check_cuda_contig(t, full, device if device is not None or codes is None else codes.device)
        if t.dtype != torch.uint8:
            raise ValueError(f"{full} must be torch.uint8")
        if t.dim() < 1 or (dims is not None and t.dim() != dims):
            raise ValueError(f"{full} must have {dims if dims is not None else 'at least one'} dimension(s)")
    if codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != 16 * scales.shape[-1]:
        raise ValueError(f"{name}codes {tuple(codes.shape)} and {name}scales {tuple(scales.shape)} must agree: "
                         "16 bytes of codes a scale")
    raise ValueError(f"{name}codes must be 16-byte aligned")


def _check_out(out: Optional[torch.Tensor], shape, dtype: torch.dtype, device: torch.device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if out.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("out must not require a gradient: the calls have none for it")
    if forward_ad._current_level >= 0:
        _no_tangent("a call with out", out)
    if out.dtype != dtype or out.device != device or not out.is_contiguous() or tuple(out.shape) != tuple(shape):
        raise ValueError(f"out must be a contiguous {dtype} tensor of shape {tuple(shape)} on {device}")
    torch.autograd.graph.increment_version(out)  # so that autograd knows if it had saved what is there now
    return out


def mxfp4_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(codes [..., 16 * ceil(k / 32)], scales [..., ceil(k / 32)])``, both uint8, of ``x [..., k]``.

    A block's scale is ``2 ** (floor(log2(max|x|)) - 2)``, at least ``2 ** -127``; a code is the
    nearest value, ties to the even code, magnitudes above 6 to 6 (the largest element of a block
    is below 8 times the scale). A block with an infinity or a NaN becomes NaN as a whole."""
    _check_cuda(x, "x")
    t = _type(x, "x")
    _no_grad("mxfp4_quantize", x)
    shape, device = x.shape, x.device
    if len(shape) < 1:
        raise ValueError("x must have at least one dimension")
    k = shape[-1]
    blocks = (k + BLOCK - 1) // BLOCK
    if len(shape) == 2:
        n = shape[0]
        rows = x if x.stride(1) == 1 or k <= 1 else x.contiguous()
        codes = torch.empty((n, 16 * blocks), dtype=torch.uint8, device=device)
        scales = torch.empty((n, blocks), dtype=torch.uint8, device=device)
    else:
        rows = _rows(x, k)
        n = rows.shape[0]
        codes = torch.empty((*shape[:-1], 16 * blocks), dtype=torch.uint8, device=device)
        scales = torch.empty((*shape[:-1], blocks), dtype=torch.uint8, device=device)
    _call(device, _native.lib().mps_mxfp4_quantize, rows.data_ptr(), t, n, k, rows.stride(0), codes.data_ptr(), scales.data_ptr())
    return codes, scales


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor, k: int, dtype: torch.dtype = torch.bfloat16, *,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values ``[..., k]`` of MXFP4 codes and scales, in ``dtype`` (exact in BF16 and FP32; FP16 rounds)."""
    _check_mx(codes, scales, "")
    t = _type(dtype, "dtype")
    k = int(k)
    if (k + BLOCK - 1) // BLOCK != scales.shape[-1] or k < 0:
        raise ValueError(f"k ({k}) does not fit {scales.shape[-1]} blocks of {BLOCK}")
    out = _check_out(out, (*codes.shape[:-1], k), dtype, codes.device)
    rows = scales.numel() // scales.shape[-1] if scales.shape[-1] else 0
    _call(codes.device, _native.lib().mps_mxfp4_dequantize, codes.data_ptr(), scales.data_ptr(), rows, k,
          out.data_ptr(), t)
    return out


def _multiply(p: "_native.MpsMxfp4Product", x_whole: bool, device: torch.device) -> None:
    """``x_whole``: x is MXFP4, or its rows are whole blocks at 16-byte addresses, and needs no workspace."""
    lib = _native.lib()
    if x_whole:
        return _call(device, lib.mps_mxfp4_multiply, p, None, 0)
    need = ctypes.c_int64(0)
    _native.check(lib.mps_mxfp4_product_workspace(p, need))
    work = torch.empty(need.value, dtype=torch.uint8, device=device)
    _call(device, lib.mps_mxfp4_multiply, p, work.data_ptr(), need.value)


def _set_x(p: "_native.MpsMxfp4Product", x: torch.Tensor, k: int) -> bool:
    """Rows ``x [r, k]`` of adjacent 16-bit elements; whether they need no workspace."""
    at, stride = x.data_ptr(), x.stride(0)
    p.x, p.x_type, p.x_stride = at, _TYPES[x.dtype], stride
    return not (k & 31 or at & 15 or stride & 7)


def _check_bias(bias: Optional[torch.Tensor], shape, device: torch.device) -> int:
    if bias is None:
        return 0
    _check_cuda_contig(bias, "bias", device)
    if tuple(bias.shape) != tuple(shape):
        raise ValueError(f"bias must have shape {tuple(shape)}, got {tuple(bias.shape)}")
    return _type(bias, "bias")


def mxfp4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor] = None, *,
                 out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w.T + bias`` for ``x [..., k]`` in BF16 or FP16 and ``w [n, k]`` in MXFP4.

    Exact products, FP32 sums, one rounding to ``out_dtype`` (default: the type of ``x``). ``bias [n]``
    is BF16, FP16 or FP32."""
    _check_cuda(x, "x")
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"x must be torch.bfloat16 or torch.float16, got {x.dtype}")
    _no_grad("mxfp4_linear", x, bias)
    shape, device = x.shape, x.device
    if len(shape) < 1:
        raise ValueError("x must have at least one dimension")
    k = shape[-1]
    _check_mx(codes, scales, "", 2, device)
    n, blocks = scales.shape
    if blocks != (k + BLOCK - 1) // BLOCK:
        raise ValueError(f"x has {k} columns, which do not fit the weight's {blocks} blocks of {BLOCK}")
    dtype = out_dtype if out_dtype is not None else (out.dtype if out is not None else x.dtype)
    p = _native.MpsMxfp4Product()
    p.out_type, p.bias_type = _type(dtype, "out_dtype"), _check_bias(bias, (n,), device)
    out = _check_out(out, (shape[0], n) if len(shape) == 2 else (*shape[:-1], n), dtype, device)
    rows = _rows(x, k)
    whole = _set_x(p, rows, k)
    p.rows = rows.shape[0] if k else (out.numel() // n if n else 0)
    p.w, p.w_scales, p.out, p.n, p.k = codes.data_ptr(), scales.data_ptr(), out.data_ptr(), n, k
    if bias is not None:
        p.bias = bias.data_ptr()
    _multiply(p, whole, device)
    return out


def mxfp4_matmul(x_codes: torch.Tensor, x_scales: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor,
                 bias: Optional[torch.Tensor] = None, *, out_dtype: Optional[torch.dtype] = None,
                 out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w.T + bias`` for ``x [..., k]`` and ``w [n, k]``, both in MXFP4 (as mxfp4_quantize returns them).

    Exact products, FP32 sums, one rounding to ``out_dtype`` (default: BF16)."""
    _check_mx(x_codes, x_scales, "x_")
    device = x_codes.device
    _check_mx(codes, scales, "", 2, device)
    _no_grad("mxfp4_matmul", bias)
    if scales.shape[1] != x_scales.shape[-1]:
        raise ValueError(f"x has {x_scales.shape[-1]} blocks a row and the weight {scales.shape[1]}")
    n = codes.shape[0]
    dtype = out_dtype if out_dtype is not None else (out.dtype if out is not None else torch.bfloat16)
    p = _native.MpsMxfp4Product()
    p.out_type, p.bias_type = _type(dtype, "out_dtype"), _check_bias(bias, (n,), device)
    out = _check_out(out, (*x_codes.shape[:-1], n), dtype, device)
    p.x, p.x_scales, p.x_type, p.rows = x_codes.data_ptr(), x_scales.data_ptr(), _native.MPS_TYPE_MXFP4, out.numel() // n if n else 0
    p.w, p.w_scales, p.out, p.n, p.k = codes.data_ptr(), scales.data_ptr(), out.data_ptr(), n, BLOCK * scales.shape[1]
    if bias is not None:
        p.bias = bias.data_ptr()
    _multiply(p, True, device)
    return out
