"""The MXFP4 and expert operators refuse host tensors, and their C entries bad sizes and types, without a GPU."""
import ctypes

import pytest
import torch

from mpserve_amd import _native
from mpserve_amd.experts import ExpertSort, expert_combine, expert_gather, expert_sort, mxfp4_expert_linear
from mpserve_amd.mxfp4 import mxfp4_dequantize, mxfp4_linear, mxfp4_matmul, mxfp4_quantize
from tests import mx_plain as plain


def test_host_tensors_are_refused():
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    codes, scales = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    ids = torch.zeros(2, 1, dtype=torch.int32)
    sort = ExpertSort(torch.zeros(2, dtype=torch.int32), ids, torch.zeros(2, dtype=torch.int32))
    for call in (lambda: mxfp4_quantize(x), lambda: mxfp4_dequantize(codes, scales, 32), lambda: mxfp4_linear(x, codes, scales),
                 lambda: mxfp4_matmul(codes, scales, codes, scales), lambda: expert_sort(ids, 1), lambda: expert_gather(x, sort),
                 lambda: expert_combine(x, torch.zeros(2, 1), sort), lambda: mxfp4_expert_linear(x, codes[None], scales[None], sort)):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call()


def test_missing_tensors_are_refused():
    codes, scales = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8)
    for call, name in ((lambda: mxfp4_quantize(None), "x"), (lambda: mxfp4_dequantize(None, scales, 32), "codes"),
                       (lambda: mxfp4_matmul(None, scales, codes, scales), "x_codes"), (lambda: mxfp4_linear(None, codes, scales), "x"),
                       (lambda: expert_sort(None, 1), "ids")):
        with pytest.raises(ValueError, match=f"^{name} must be defined"):
            call()


def test_c_entries_refuse_bad_arguments():
    lib = _native.lib()
    p = ctypes.c_void_p(4096)  # never read: each call is refused before any work
    odd = ctypes.c_void_p(4098)
    for rc in (lib.mps_mxfp4_quantize(p, 7, 1, 32, 32, p, p, None), lib.mps_mxfp4_quantize(p, 0, -1, 32, 32, p, p, None),
               lib.mps_mxfp4_quantize(None, 0, 1, 32, 32, p, p, None), lib.mps_mxfp4_quantize(p, 0, 1, 32, -1, p, p, None),
               lib.mps_mxfp4_quantize(p, 0, 2 ** 32, 32, 32, p, p, None), lib.mps_mxfp4_quantize(p, 0, 1, 32, 32, odd, p, None),
               lib.mps_mxfp4_dequantize(p, None, 1, 32, p, 0, None), lib.mps_mxfp4_dequantize(p, p, 1, -32, p, 0, None),
               lib.mps_mxfp4_multiply(None, None, 0, None), lib.mps_expert_sort(p, 0, 2 ** 30, 4, 8, p, p, p, None, 0, None),
               lib.mps_expert_sort(p, 0, 4, 4, 0, p, p, p, None, 0, None), lib.mps_expert_sort(p, 0, 4, 4, 1025, p, p, p, None, 0, None),
               lib.mps_expert_sort(None, 0, 4, 4, 8, p, p, p, None, 0, None), lib.mps_expert_gather(p, 3, 4, 4, 8, 32, p, p, p, p, None),
               lib.mps_expert_gather(p, 0, 4, 4, 8, -1, p, p, p, p, None), lib.mps_expert_combine(p, 0, p, 9, 4, 4, 32, p, p, None),
               lib.mps_expert_combine_grad(p, p, 0, None, 0, 4, 4, 8, 32, p, p, p, p, p, None)):
        assert rc == _native.MPS_ERR_INVALID_ARGUMENT and lib.mps_last_error()
    good = dict(x=p, x_stride=32, w=p, w_scales=p, out=p, rows=4, n=8, k=32, x_type=0, out_type=0)
    for change in (dict(x_type=2), dict(out_type=3), dict(bias=p, bias_type=5), dict(rows=-1), dict(rows=2 ** 31), dict(n=2 ** 33),
                   dict(experts=2000), dict(out=None), dict(w=odd), dict(x=None), dict(x_type=3), dict(experts=2), dict(gather=1),
                   dict(experts=2, offsets=p, gather=1), dict(x_stride=-1)):
        args = _native.MpsMxfp4Product(**{**good, **change})
        assert lib.mps_mxfp4_multiply(args, None, 0, None) == _native.MPS_ERR_INVALID_ARGUMENT, change


def test_gather_of_mxfp4_rows_is_refused():
    """MXFP4 x has rows / top rows where it is gathered, but is read by sorted place: none of it may be launched."""
    lib = _native.lib()
    p = ctypes.c_void_p(4096)  # never read
    args = _native.MpsMxfp4Product(x=p, x_scales=p, w=p, w_scales=p, out=p, offsets=p, order=p, rows=8, n=8, k=32, experts=2, top=2,
                                   gather=1, x_type=_native.MPS_TYPE_MXFP4)
    need = ctypes.c_int64(0)
    for rc in (lib.mps_mxfp4_multiply(args, None, 0, None), lib.mps_mxfp4_product_workspace(args, need)):
        assert rc == _native.MPS_ERR_INVALID_ARGUMENT and b"16-bit" in lib.mps_last_error()


@pytest.mark.parametrize("rows,top", [(3, 4), (1, 2 ** 31 + 1), (9, 2)])
def test_gather_of_parts_of_tokens_is_refused(rows, top):
    """x has rows / top rows: with fewer rows than top there would be none to keep bad orders within."""
    lib = _native.lib()
    p = ctypes.c_void_p(4096)  # never read
    args = _native.MpsMxfp4Product(x=p, x_stride=32, w=p, w_scales=p, out=p, offsets=p, order=p, rows=rows, n=8, k=32, experts=2, top=top, gather=1)
    assert lib.mps_mxfp4_multiply(args, None, 0, None) == _native.MPS_ERR_INVALID_ARGUMENT and b"multiple of top" in lib.mps_last_error()


@pytest.mark.parametrize("pairs", (4097, 65536, 2113929216, 2113930241, 2 ** 31 - 1025))
def test_sort_asks_for_its_workspace(pairs):
    """Up to the most pairs there may be, both entries want the same: chunks of 2^25 pairs, counted in 64 bits."""
    lib = _native.lib()
    p = ctypes.c_void_p(4096)  # never read
    need = ctypes.c_int64(0)
    assert lib.mps_expert_sort_workspace(pairs, 1, 8, need) == 0 and need.value > 0 and need.value <= 64 * 9 * 4
    for work, size in ((None, 0), (p, need.value - 1)):
        rc = lib.mps_expert_sort(p, 0, pairs, 1, 8, p, p, p, work, size, None)
        assert rc == _native.MPS_ERR_INVALID_ARGUMENT and b"%d bytes of workspace" % need.value in lib.mps_last_error()


def test_dual_tensors_are_told():
    from torch.autograd import forward_ad

    from mpserve_amd.mxfp4 import _no_grad, _no_tangent

    x = torch.zeros(2, 32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        assert not dual.requires_grad
        for call in (lambda: _no_tangent("op", None, x, dual), lambda: _no_grad("op", dual)):
            with pytest.raises(RuntimeError, match="op has no forward-mode derivative"):
                call()
        _no_tangent("op", None, x, forward_ad.unpack_dual(dual).primal)
        with torch.inference_mode():  # no derivative is being taken
            _no_tangent("op", dual)
    _no_tangent("op", x)


def test_combine_grad_wants_something_to_write():
    lib = _native.lib()
    p = ctypes.c_void_p(4096)  # never read
    for y, dy, dw in ((p, None, None), (None, p, p), (None, None, p)):
        rc = lib.mps_expert_combine_grad(y, p, 0, p, 0, 4, 4, 8, 32, p, p, p, dy, dw, None)
        assert rc == _native.MPS_ERR_INVALID_ARGUMENT and b"null pointer" in lib.mps_last_error()


def test_plain_quantization_known_answers():
    """The oracle of these tests against a block worked out by hand: the largest element 5 has floor(log2) 2, so the
    scale is 2^0; 5 is halfway between 4 (code 6, even) and 6, 0.75 between 0.5 and 1 (code 2, even)."""
    x = torch.zeros(1, 34, dtype=torch.float64)
    x[0, :6] = torch.tensor([5.0, 0.75, -0.25, -3.0, 2.5, 0.26])
    x[0, 32:] = torch.tensor([7.0, -0.0])
    codes, scales = plain.quantize(x)
    assert scales.tolist() == [[127, 127]]
    assert codes[0, :3].tolist() == [6 + 16 * 2, 8 + 16 * 13, 4 + 16 * 1]
    assert codes[0, 3:16].tolist() == [0] * 13 and codes[0, 16].item() == 7 + 16 * 8
    assert plain.dequantize(codes, scales, 34)[0, :6].tolist() == [4.0, 1.0, -0.0, -3.0, 2.0, 0.5]
