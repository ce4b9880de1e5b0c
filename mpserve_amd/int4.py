"""Products with int4 weights: whole numbers of 4 bits with a scale and a zero for each group of columns.

A weight ``[n, k]`` is ``scales * (q - zeros)``: ``q`` whole numbers from 0 to 15, ``scales [n,
ceil(k / group)]`` in BF16 or FP16, ``zeros`` of the same shape from 0 to 16 in uint8 (their low
five bits count), or None where all are 8. ``group`` is a power of two, at least 32; one that is not below
``k`` means a scale a row. This is what an AWQ checkpoint holds. The AWQ builders and decode ops
(``huffman_decode_awq_int4_bucket`` and its kin) take such whole numbers and scales too, but what they give back is the BF16
weight that was quantised, bit by bit. The products here are with the quantised weight itself, about half a scale or less
away from that: results are those of an AWQ model, not of the model that it was made of.

* :func:`int4_pack` — whole numbers ``[..., k]`` to codes, once a weight;
* :func:`int4_from_awq` — an AWQ checkpoint's tensors to codes, scales and zeros;
* :func:`int4_linear` — ``x @ w.T + bias`` with 16-bit ``x``.

Codes lie in blocks of 32 elements, 16 bytes each, a row's last block filled up; byte ``b`` of
each 4 bytes holds element ``b`` of eight in its low half and element ``b + 4`` in its high half.
``int4_linear`` runs on the current stream of its tensors' device, does not synchronise, and can be captured
into a graph. It has no gradient, and refuses tensors that ask for one or carry a tangent. The work is
done by the HIP kernels of libmpserve_amd.so; there is no CPU path.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _native
from ._common import _check_cuda_contig
from .mxfp4 import BLOCK, _TYPES, _call, _check_bias, _check_cuda, _check_out, _no_grad, _rows, _type

_HALVES = (torch.bfloat16, torch.float16)


class Int4Weight(NamedTuple):
    """An int4 weight, in the order in which the products take it."""
    codes: torch.Tensor   # uint8 [..., n, 16 * ceil(k / 32)]
    scales: torch.Tensor  # BF16 or FP16 [..., n, ceil(k / group)]
    zeros: Optional[torch.Tensor]  # uint8, of the shape of the scales


def int4_pack(values: torch.Tensor) -> torch.Tensor:
    """Codes ``[..., 16 * ceil(k / 32)]`` of whole numbers ``values [..., k]`` from 0 to 15 (uint8; the low four
    bits count), such as the ``int4_values_u8`` that the AWQ ops take. Works on any device."""
    if values is None:
        raise ValueError("values must be defined")
    if values.dtype != torch.uint8:
        raise ValueError(f"values must be torch.uint8, got {values.dtype}")
    if values.dim() < 1:
        raise ValueError("values must have at least one dimension")
    k = values.shape[-1]
    blocks = (k + BLOCK - 1) // BLOCK
    v = torch.nn.functional.pad(values & 15, (0, blocks * BLOCK - k)).reshape(*values.shape[:-1], blocks * 4, 2, 4)
    return (v[..., 0, :] | v[..., 1, :] << 4).reshape(*values.shape[:-1], blocks * 16)


#: column of eight that each half byte of an AWQ checkpoint's word holds, from the lowest on
_AWQ_ORDER = (0, 2, 4, 6, 1, 3, 5, 7)


def _awq_unpack(words: torch.Tensor) -> torch.Tensor:
    out = torch.empty((*words.shape, 8), dtype=torch.uint8, device=words.device)
    for i, col in enumerate(_AWQ_ORDER):
        out[..., col] = (words >> (4 * i) & 15).to(torch.uint8)
    return out.reshape(*words.shape[:-1], words.shape[-1] * 8)


def int4_from_awq(qweight: torch.Tensor, qzeros: torch.Tensor, scales: torch.Tensor) -> Int4Weight:
    """An AWQ checkpoint's linear layer, ``qweight [k, n / 8]`` and ``qzeros [k / group, n / 8]`` in int32 and
    ``scales [k / group, n]`` in FP16 or BF16, as :func:`int4_linear` takes it. Works on any device."""
    for t, name in ((qweight, "qweight"), (qzeros, "qzeros"), (scales, "scales")):
        if t is None:
            raise ValueError(f"{name} must be defined")
        if t.dim() != 2:
            raise ValueError(f"{name} must have 2 dimensions")
    if qweight.dtype != torch.int32 or qzeros.dtype != torch.int32:
        raise ValueError("qweight and qzeros must be torch.int32")
    if scales.dtype not in _HALVES:
        raise ValueError(f"scales must be torch.float16 or torch.bfloat16, got {scales.dtype}")
    n = 8 * qweight.shape[1]
    if qzeros.shape[1] != qweight.shape[1] or scales.shape[1] != n or qzeros.shape[0] != scales.shape[0]:
        raise ValueError(f"qweight {tuple(qweight.shape)}, qzeros {tuple(qzeros.shape)} and scales {tuple(scales.shape)} do not agree")
    return Int4Weight(int4_pack(_awq_unpack(qweight).t().contiguous()), scales.t().contiguous(), _awq_unpack(qzeros).t().contiguous())


def _check_int4(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor], k: int, group: int, dims: int,
                device: torch.device) -> None:
    if codes is not None and scales is not None:  # all is well in one go; what is not is named below
        c, s = codes.shape, scales.shape
        if codes.dtype is torch.uint8 and (scales.dtype is torch.bfloat16 or scales.dtype is torch.float16) \
                and codes.device == device == scales.device and codes.is_contiguous() and scales.is_contiguous() \
                and len(c) == dims == len(s) and c[:-1] == s[:-1] and c[-1] == (k + BLOCK - 1) // BLOCK * 16 \
                and group >= 32 and not group & (group - 1) and s[-1] == (k + group - 1) // group and not codes.data_ptr() & 15 \
                and (zeros is None or (zeros.dtype is torch.uint8 and zeros.shape == s and zeros.device == device
                                       and zeros.is_contiguous())):
            return
    for t, name in ((codes, "codes"), (scales, "scales"), (zeros, "zeros")):
        if name == "zeros" and t is None:
            continue
        _check_cuda_contig(t, name, device)
        if t.dim() != dims:
            raise ValueError(f"{name} must have {dims} dimension(s)")
    if codes.dtype != torch.uint8 or (zeros is not None and zeros.dtype != torch.uint8):
        raise ValueError("codes and zeros must be torch.uint8")
    if scales.dtype not in _HALVES:
        raise ValueError(f"scales must be torch.bfloat16 or torch.float16, got {scales.dtype}")
    if group < 32 or group & (group - 1):
        raise ValueError(f"group must be a power of two, at least 32, got {group}")
    want = (*codes.shape[:-1], (k + group - 1) // group)
    if codes.shape[-1] != (k + BLOCK - 1) // BLOCK * 16:
        raise ValueError(f"x has {k} columns, which do not fit the weight's {codes.shape[-1]} bytes of codes a row")
    for t, name in ((scales, "scales"), (zeros, "zeros")):
        if t is not None and tuple(t.shape) != want:
            raise ValueError(f"{name} must have shape {want} for groups of {group}, got {tuple(t.shape)}")
    raise ValueError("codes must be 16-byte aligned")


def _int4_product(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor],
                  bias: Optional[torch.Tensor], group: int, k: int, n: int) -> "_native.MpsInt4Product":
    """The operands that any product has; ``x [r, k]`` has adjacent elements."""
    p = _native.MpsInt4Product()
    p.x, p.x_stride, p.x_type = x.data_ptr(), x.stride(0), _TYPES[x.dtype]
    p.w, p.scales, p.scale_type, p.group, p.n, p.k = codes.data_ptr(), scales.data_ptr(), _TYPES[scales.dtype], group, n, k
    if zeros is not None:
        p.zeros = zeros.data_ptr()
    if bias is not None:
        p.bias = bias.data_ptr()
    return p


def _int4_multiply(p: "_native.MpsInt4Product", device: torch.device) -> None:
    if torch._C._cuda_getDevice() != device.index:  # the choice of a kernel goes by the device's compute units
        with torch.cuda.device(device):
            return _int4_multiply(p, device)
    lib = _native.lib()
    need = ctypes.c_int64(0)
    rc = lib.mps_int4_product_workspace(p, need)
    if rc:
        _native.check(rc)
    if need.value:
        work = torch.empty(need.value, dtype=torch.uint8, device=device)
        _call(device, lib.mps_int4_multiply, p, work.data_ptr(), need.value)
    else:
        _call(device, lib.mps_int4_multiply, p, None, 0)


def int4_linear(x: torch.Tensor, codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None,
                bias: Optional[torch.Tensor] = None, *, group: int = 128, out_dtype: Optional[torch.dtype] = None,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w.T + bias`` for ``x [..., k]`` in BF16 or FP16 and ``w [n, k]`` in int4.

    Whole numbers are multiplied exactly; each group's FP32 sum gets its scale in FP32, and the sum of all is
    rounded once, to ``out_dtype`` (default: the type of ``x``). ``bias [n]`` is BF16, FP16 or FP32. Sums are ``x`` times
    ``q`` less ``x`` times the zeros, taken apart for up to 512 columns at a time: FP32's errors are of these columns' sums of ``|x| (q + zeros)``,
    and of the result."""
    _check_cuda(x, "x")
    if x.dtype not in _HALVES:
        raise ValueError(f"x must be torch.bfloat16 or torch.float16, got {x.dtype}")
    _no_grad("int4_linear", x, scales, bias)
    shape, device, group = x.shape, x.device, int(group)
    if len(shape) < 1:
        raise ValueError("x must have at least one dimension")
    k = shape[-1]
    _check_int4(codes, scales, zeros, k, group, 2, device)
    n = codes.shape[0]
    dtype = out_dtype if out_dtype is not None else (out.dtype if out is not None else x.dtype)
    out_type, bias_type = _type(dtype, "out_dtype"), _check_bias(bias, (n,), device)
    out = _check_out(out, (shape[0], n) if len(shape) == 2 else (*shape[:-1], n), dtype, device)
    rows = _rows(x, k)
    p = _int4_product(rows, codes, scales, zeros, bias, group, k, n)
    p.rows = rows.shape[0] if k else (out.numel() // n if n else 0)
    p.out, p.out_type, p.bias_type = out.data_ptr(), out_type, bias_type
    _int4_multiply(p, device)
    return out
