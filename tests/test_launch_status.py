"""A call that fails says so, and the calls after it are judged by themselves."""
import pytest

import rocm_sgemm_b200 as pkg

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu


@gpu
def test_a_failed_allocation_does_not_fail_later_calls(sgemm):
    """The 3xTF32 product of col-major matrices asks for a transposed copy of A, here 1 TB, before it touches them."""
    f32, a = pkg.m_type.f32, torch.randn(64, 64, device="cuda")
    status = sgemm.lib().b200_sgemm_3xtf32(1, 1, 1, a.data_ptr(), a.data_ptr(), a.data_ptr(), 1 << 20, 64, 1 << 18, None)
    assert status > 0
    codes, scales = (torch.empty(n, dtype=torch.uint8, device="cuda") for n in sgemm.mx4_sizes(0, 64, 64))
    out, ids = torch.empty_like(a), torch.zeros(64, 1, dtype=torch.int32, device="cuda")
    weights = torch.ones(64, 1, device="cuda")
    for layout in (0, 1):
        sgemm.mx4_quantize(0, layout, f32, a, 64, 64, codes, scales)
    sgemm.mx4_dequantize(0, f32, codes, scales, 64, 64, out)
    for m in (1, 2, 64):
        sgemm.gemm_mx4(0, 0, f32, out, codes, scales, codes, scales, m, 64, 64)
    offsets, counts, slot_row, row_slot = (torch.empty(n, dtype=torch.int32, device="cuda") for n in (2, 1, 64, 64))
    sgemm.route_sort(ids, 64, 1, 1, 1, offsets, counts, slot_row, row_slot, 64)
    sgemm.route_dispatch(f32, a, 64, 64, slot_row, 1, out, 64)
    assert torch.equal(out, a)
    sgemm.route_combine(f32, a, 64, 64, slot_row, 64, 1, out)
    assert torch.equal(out, a)
    sgemm.route_combine_backward(f32, a, a, 64, 64, slot_row, 64, 1, weights, out, weights)
    assert torch.equal(out, a)


@gpu
def test_a_failed_allocation_does_not_fail_later_fp32_products(sgemm):
    """The same refusal, then products whose launches are checked by the thread's last error."""
    a, b, c = (torch.randn(96, 96, device="cuda") for _ in range(3))
    assert sgemm.lib().b200_sgemm_3xtf32(1, 1, 1, a.data_ptr(), a.data_ptr(), a.data_ptr(), 1 << 20, 64, 1 << 18, None) > 0
    want = (a.double() @ b.double()).float()
    at = a.T.contiguous()  # col-major A, row-major B: both are copied
    sgemm.gemm_3xtf32(0, 1, 0, c, at, b, 96, 96, 96)
    assert torch.allclose(c, want, atol=1e-3)
    c.zero_()
    sgemm.gemm(0, 0, 0, c, a, b, 96, 96, 96)
    assert torch.allclose(c, want, atol=1e-3)
