"""The int4 products and the router refuse host tensors, and their C entries bad sizes and types, without a GPU."""
import ctypes

import pytest
import torch

from mpserve_amd import _native
from mpserve_amd.experts import ExpertSort, expert_balance, expert_route, int4_expert_linear
from mpserve_amd.int4 import int4_from_awq, int4_linear, int4_pack
from tests import int4_plain as plain


@pytest.mark.parametrize("k", (1, 4, 5, 8, 31, 32, 33, 100, 128))
def test_pack_matches_definition(k):
    values = torch.randint(0, 16, (7, k), generator=torch.Generator().manual_seed(k), dtype=torch.uint8)
    codes = int4_pack(values)
    assert codes.shape == (7, 16 * ((k + 31) // 32)) and codes.is_contiguous() and torch.equal(codes, plain.pack(values))
    assert torch.equal(int4_pack(values | 0xf0), codes)
    assert torch.equal(int4_pack(values.t().contiguous().t()), codes)
    assert torch.equal(int4_pack(values.view(7, 1, k)), codes.view(7, 1, -1))


def test_pack_and_awq_refusals():
    v = torch.zeros(4, 8, dtype=torch.uint8)
    q, z, s = torch.zeros(64, 2, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, 16, dtype=torch.float16)
    for call, message in ((lambda: int4_pack(v.int()), "values must be torch.uint8"), (lambda: int4_pack(None), "values must be defined"),
                          (lambda: int4_pack(torch.tensor(1, dtype=torch.uint8)), "at least one dimension"),
                          (lambda: int4_from_awq(q.long(), z, s), "must be torch.int32"), (lambda: int4_from_awq(q, z, s.float()), "scales must be"),
                          (lambda: int4_from_awq(q, z, s[:, :8]), "do not agree"), (lambda: int4_from_awq(q, z[:, :1], s), "do not agree"),
                          (lambda: int4_from_awq(q, None, s), "qzeros must be defined"), (lambda: int4_from_awq(q[0], z, s), "2 dimensions")):
        with pytest.raises(ValueError, match=message):
            call()


def test_host_and_missing_tensors_are_refused():
    x = torch.zeros(2, 32, dtype=torch.bfloat16)
    codes, scales = torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.bfloat16)
    ids = torch.zeros(2, 1, dtype=torch.int32)
    sort = ExpertSort(torch.zeros(2, dtype=torch.int32), ids, torch.zeros(2, dtype=torch.int32))
    for call in (lambda: int4_linear(x, codes, scales), lambda: int4_expert_linear(x, codes[None], scales[None], sort),
                 lambda: expert_route(x, 1), lambda: expert_balance(x, ids)):
        with pytest.raises(ValueError, match="must be a CUDA tensor"):
            call()
    for call, name in ((lambda: int4_linear(None, codes, scales), "x"), (lambda: expert_route(None, 1), "logits"), (lambda: expert_balance(None, ids), "logits")):
        with pytest.raises(ValueError, match=f"^{name} must be defined"):
            call()


def test_product_entry_refuses_bad_arguments():
    lib = _native.lib()
    p, odd = ctypes.c_void_p(4096), ctypes.c_void_p(4098)  # never read: each call is refused before any work
    good = dict(x=p, x_stride=32, w=p, scales=p, out=p, rows=4, n=8, k=32, group=32, x_type=0, scale_type=0, out_type=0)
    need = ctypes.c_int64(0)
    for change in (dict(x_type=2), dict(x_type=3), dict(scale_type=2), dict(out_type=3), dict(bias=p, bias_type=5), dict(rows=-1),
                   dict(rows=2 ** 31), dict(n=2 ** 33), dict(k=-1), dict(k=2 ** 25), dict(group=0), dict(group=16), dict(group=48),
                   dict(group=-32), dict(group=2 ** 31), dict(group=2 ** 62), dict(experts=2000), dict(out=None), dict(w=odd), dict(x=None),
                   dict(scales=None), dict(experts=2), dict(gather=1), dict(experts=2, offsets=p, gather=1), dict(x_stride=-1),
                   dict(experts=2, offsets=p, order=p, gather=1, top=3), dict(experts=2, offsets=p, order=p, gather=1, top=0)):
        args = _native.MpsInt4Product(**{**good, **change})
        assert lib.mps_int4_multiply(args, None, 0, None) == _native.MPS_ERR_INVALID_ARGUMENT and lib.mps_last_error(), change
        assert lib.mps_int4_product_workspace(args, need) == _native.MPS_ERR_INVALID_ARGUMENT, change
    assert lib.mps_int4_multiply(None, None, 0, None) == _native.MPS_ERR_INVALID_ARGUMENT
    assert lib.mps_int4_product_workspace(_native.MpsInt4Product(**good), None) == _native.MPS_ERR_INVALID_ARGUMENT


def test_router_entries_refuse_bad_arguments():
    lib = _native.lib()
    p = ctypes.c_void_p(4096)  # never read
    need = ctypes.c_int64(0)
    route = dict(logits=p, type=2, tokens=4, experts=8, stride=8, top=2, scores=0, bias=None, normalize=1, scale=1.0, ids=p, weights=p, shares=None, stream=None)
    grad = dict(logits=p, type=2, tokens=4, experts=8, stride=8, top=2, scores=0, normalize=1, scale=1.0, ids=p, shares=p, dweights=p, dlogits=p, stream=None)
    balance = dict(logits=p, type=2, tokens=4, experts=8, stride=8, scores=0, ids=p, ids_64=0, top=2, loss=p, counts=p, kept=p, work=None, size=0, stream=None)
    balance_grad = dict(logits=p, type=2, tokens=4, experts=8, stride=8, scores=0, kept=p, dloss=p, dlogits=p, stream=None)
    sizes = (dict(type=3), dict(type=-1), dict(scores=2), dict(scores=-1), dict(experts=0), dict(experts=1025), dict(tokens=-1), dict(tokens=2 ** 31), dict(stride=-1), dict(logits=None))
    for entry, good, more in (
            (lib.mps_expert_route, route, (dict(top=9), dict(top=-1), dict(ids=None), dict(weights=None), dict(tokens=2 ** 30, top=4))),
            (lib.mps_expert_route_grad, grad, (dict(top=9), dict(ids=None), dict(shares=None), dict(dweights=None), dict(dlogits=None))),
            (lib.mps_expert_balance, balance, (dict(top=-1), dict(ids=None), dict(loss=None), dict(tokens=2 ** 30, top=4), dict(tokens=100000))),
            (lib.mps_expert_balance_grad, balance_grad, (dict(kept=None), dict(dloss=None), dict(dlogits=None)))):
        for change in (*sizes, *more):
            assert entry(*{**good, **change}.values()) == _native.MPS_ERR_INVALID_ARGUMENT and lib.mps_last_error(), (entry, change)
    assert lib.mps_expert_balance_workspace(-1, 8, 2, need) == _native.MPS_ERR_INVALID_ARGUMENT
    assert lib.mps_expert_balance_workspace(4, 8, 2, None) == _native.MPS_ERR_INVALID_ARGUMENT
    for tokens, experts in ((1, 8), (2 ** 31 - 1025, 1), (2 ** 31 - 1025, 1024), (100000, 1000)):
        assert lib.mps_expert_balance_workspace(tokens, experts, 1, need) == 0 and 0 <= need.value <= 256 * 2049 * 4
