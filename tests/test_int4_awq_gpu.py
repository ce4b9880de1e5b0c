"""From the AWQ ops' own tensors to the int4 product: whole numbers and scales are the same, the weight is another."""
import pytest
import torch

from mpserve_amd import awq
from mpserve_amd.int4 import int4_linear, int4_pack
from mpserve_amd.synthetic import make_awq_weight
from tests import int4_plain as plain
from tests import mx_plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("t", (1, 20, 700))
def test_product_of_the_awq_ops_tensors_is_that_of_the_quantised_weight(t):
    """s (q - 8), of the whole numbers and scales that the sidecar's builder takes. Its decoder gives back the weight that was quantised, which is
    up to half a step of s away (and 7 2^-8 more, where s, rounded to BF16, is below a seventh of the largest element)."""
    n, m, group = 200, 640, 128
    a = make_awq_weight(n, m, group, seed=3, device=DEV)
    values, scales = a.int4_u8, a.scale_u16.view(torch.bfloat16)
    x = torch.randn(t, m, generator=torch.Generator(device=DEV).manual_seed(t), device=DEV).to(torch.bfloat16)
    y = int4_linear(x, int4_pack(values), scales, group=group, out_dtype=torch.float32)
    w = plain.weight(values, scales, None, group)
    mx_plain.close(y, x.double() @ w.T, x.double().abs() @ plain.reach(values, scales, None, group).T, 2 * m + 5)

    side = awq.huffman_build_awq_int4_bucket_decode_tables_by_scale(a.bf16, values, a.scale_u16, 11, 1024, 64)
    back = awq.huffman_decode_awq_int4_bucket_by_scale(
        values, side["bitstream_u64"], side["decode_syms_u16"], side["decode_lens_u8"], side["bucket_table_i32"], side["bucket_group_offsets_i32"],
        side["group_rows_i32"], side["group_col_start_i32"], side["bucket_thread_startbit_u32"], side["bucket_bit_base_i64"], n, m, 11, group)
    assert torch.equal(back.view(torch.uint16), a.bf16.view(torch.uint16))
    step = scales.double().repeat_interleave(group, dim=1)
    off = (back.double() - w).abs() / step
    assert float(off.max()) <= 0.5 + 7 * 2.0 ** -8 + 2.0 ** -20 and float(off.mean()) > 0.2  # another weight, not this one rounded once more
