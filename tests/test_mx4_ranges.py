"""4-bit quantisation and products at the ends of their ranges: values, scales, lengths of K."""
import numpy as np
import pytest

import mx4_reference as ref
import rocm_sgemm_b200 as pkg

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FORMATS = [ref.NVFP4, ref.MXFP4]
fmt_ids = lambda f: ("nvfp4", "mxfp4")[f]  # noqa: E731


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def quantize(sgemm, fmt, x, rows, K, dtype, layout=0, g=None):
    nc, ns = sgemm.mx4_sizes(fmt, rows, K)
    codes, scales = (torch.full((n,), 0xA5, dtype=torch.uint8, device="cuda") for n in (nc, ns))
    sgemm.mx4_quantize(fmt, layout, pkg.m_type[dtype], x, rows, K, codes, scales, global_scale=g)
    return codes, scales


@gpu
@pytest.mark.parametrize("g", [1.0, 2.0 ** -10, 2.0 ** -20, 1.5 * 2.0 ** -30, 2.0 ** -90, 0.7 * 2.0 ** -40])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("layout", [0, 1])
def test_quantize_saturates_with_the_sign(sgemm, g, dtype, layout):
    """Values far above what a matrix scale can hold, whose quotient leaves FP32, beside values of every size."""
    rows, K = 40, 96
    r = np.random.default_rng(1)
    x = r.standard_normal((rows, K)) * np.exp2(r.integers(-10, 10, (rows, K))) * g * 448
    far = r.random((rows, K)) < 0.3
    x[far] = r.choice([1e36, 3e38, 2.0 ** 127, 2.0 ** 60], far.sum()) * r.choice([-1, 1], far.sum())
    x = torch.from_numpy(x).to(TYPES[dtype])
    want = ref.pack(ref.NVFP4, *ref.quantize(ref.NVFP4, x.double().numpy(), np.float32(g)))
    gt = torch.tensor([g], dtype=torch.float32, device="cuda")
    codes, scales = quantize(sgemm, ref.NVFP4, (x if layout == 0 else x.T).contiguous().cuda(), rows, K, dtype, layout, gt)
    assert np.array_equal(scales.cpu().numpy(), want[1])
    assert np.array_equal(codes.cpu().numpy(), want[0])
