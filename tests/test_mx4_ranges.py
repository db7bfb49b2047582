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


@gpu
@pytest.mark.parametrize("M,N", [(1, 300), (2, 129), (300, 1), (40, 130), (300, 200)])
def test_product_of_scales_that_exceed_fp32_together(sgemm, M, N):
    """mxfp4 blocks whose scales make 2^128 or 2^129 and whose codes make 1/4: 2^126 and 2^127, which FP32 holds, and every
    sum of which it holds."""
    K = 1056
    sides = []
    for side, rows in enumerate((M, N)):
        code = np.zeros((rows, K), np.uint8)
        code[:, ::32] = 1  # 0.5 once in each block
        code[:, 32::64] |= 8 * side  # and a product of -1/4 in every other one
        code[:, 128:] *= side  # four blocks count
        byte = np.full((rows, K // 32), 127 + 64, np.uint8)
        byte[:, 2] += 1 - side  # 2^126 - 2^126 + 2^127 - 2^126
        sides.append((*(dev(v) for v in ref.pack(ref.MXFP4, code, byte)), ref.values(ref.MXFP4, code, byte)))
    a, b = sides
    want = a[2] @ b[2].T
    assert (want == 2.0 ** 126).all()
    c = torch.empty(M, N, device="cuda")
    sgemm.gemm_mx4(ref.MXFP4, 0, pkg.m_type.f32, c, a[0], a[1], b[0], b[1], M, N, K)
    assert np.array_equal(c.cpu().numpy(), want.astype(np.float32))
    assert sgemm.mx4_device_status() == 0


def repeated(fmt, rows, period, repeats, seed):
    """A quantised matrix of positive values whose K is one period over and over, and the float64 values of a period."""
    r = np.random.default_rng(seed)
    code = r.integers(1, 8, (rows, period)).astype(np.uint8)
    blocks = period // ref.BLOCK[fmt]
    byte = (r.integers(0x30, 0x40, (rows, blocks)) if fmt == ref.NVFP4 else r.integers(124, 128, (rows, blocks))).astype(np.uint8)
    codes, scales = ref.pack(fmt, code, byte)
    codes = dev(codes).view(rows, -1).repeat(1, repeats)
    bands = -(-rows // 128)
    scales = dev(scales).view(bands, -1).repeat(1, repeats)
    return codes.view(-1), scales.view(-1), ref.values(fmt, code, byte)


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("dtype,K", [("f16", 1 << 24), ("bf16", 1 << 27)])
def test_long_sums_of_one_sign(sgemm, fmt, dtype, K):
    """The tensor core cuts off where it adds (2^-22 of the sum for each of its 64 k): 16-bit results too have to leave it
    before that shows.  One accumulator holds 2^15 k for FP16 and 2^18 for BF16, 2^9 and 2^12 of its steps; the parts, and
    the sums of up to eight CTAs, are added with 2^-24 each."""
    M, N, period = 3, 5, 4096
    a, b = repeated(fmt, M, period, K // period, 1), repeated(fmt, N, period, K // period, 2)
    want = a[2] @ b[2].T * (K // period)
    alpha = 2.0 ** -np.floor(np.log2(want.max()))
    c = torch.empty(M, N, dtype=TYPES[dtype], device="cuda")
    sgemm.gemm_mx4(fmt, 0, pkg.m_type[dtype], c, a[0], a[1], b[0], b[1], M, N, K, alpha=float(alpha))
    want = want * alpha
    held = 15 if dtype == "f16" else 18
    bound = 2.0 ** (held - 6 - 22) + (K / 2.0 ** held + 8) * 2.0 ** -24 + ref.TYPE_EPS[dtype] / 2 + 4 * 2.0 ** -24
    off = np.abs(c.double().cpu().numpy() - want) / want
    assert off.max() <= bound, f"{off.max() / bound:.3g} times the bound"
    assert sgemm.mx4_device_status() == 0


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("layout_c", [0, 1])
def test_long_sums_in_wide_tiles(sgemm, fmt, dtype, layout_c):
    """K beyond what one accumulator may hold of FP16, in tiles of 256 columns."""
    M, N, period, repeats = 2304, 2560, 1024, 33
    K = period * repeats
    assert sgemm.mx4_sizes(fmt, M, K)[0] == M * K // 2
    a, b = repeated(fmt, M, period, repeats, 3), repeated(fmt, N, period, repeats, 4)
    va, vb = torch.from_numpy(a[2]).cuda(), torch.from_numpy(b[2]).cuda()
    want = (va @ vb.T * repeats).cpu().numpy()
    alpha = float(2.0 ** -np.floor(np.log2(want.max())))
    ld = (N if layout_c == 0 else M) + 8
    c = torch.full((M if layout_c == 0 else N, ld), 9.0, dtype=TYPES[dtype], device="cuda")
    sgemm.gemm_mx4(fmt, layout_c, pkg.m_type[dtype], c, a[0], a[1], b[0], b[1], M, N, K, ldc=ld, alpha=alpha)
    assert (c[:, ld - 8:] == 9).all()
    got = c[:, :ld - 8].double().cpu().numpy()
    got = got if layout_c == 0 else got.T
    held = {"f32": 11, "f16": 15, "bf16": 18}[dtype]
    steps = min(2.0 ** held, K) / 64
    bound = steps * 2.0 ** -22 + (K / 2.0 ** held + 8) * 2.0 ** -24 + ref.TYPE_EPS[dtype] / 2 + 4 * 2.0 ** -24
    off = np.abs(got - want * alpha) / (want * alpha)
    assert off.max() <= bound, f"{off.max() / bound:.3g} times the bound"
    assert sgemm.mx4_device_status() == 0


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("g", [0.0, 2.0 ** -120, 2.0 ** 100])
def test_zeros_stay_zero_whatever_the_matrix_scale(sgemm, dtype, layout, g):
    """A matrix of zeros has amax / 2688 = 0 for a scale: its values are zero, not NaN, and so are its products."""
    M, N, K = 70, 130, 100
    gt = torch.tensor([g], dtype=torch.float32, device="cuda")
    x = torch.zeros(M, K, dtype=TYPES[dtype], device="cuda")
    x[3, 5] = -0.0
    a = quantize(sgemm, ref.NVFP4, x if layout == 0 else x.T.contiguous(), M, K, dtype, layout, gt)
    assert not a[0].any() and not a[1].any()
    out = torch.full((M, K), 7.0, device="cuda")
    sgemm.mx4_dequantize(ref.NVFP4, pkg.m_type.f32, *a, M, K, out, global_scale=gt)
    assert not out.any()
    b = quantize(sgemm, ref.NVFP4, torch.randn(N, K, device="cuda"), N, K, "f32")
    for rows in (1, 2, M):
        c = torch.full((rows, N), 7.0, device="cuda")
        sgemm.gemm_mx4(ref.NVFP4, 0, pkg.m_type.f32, c, *a, *b, rows, N, K, global_a=gt)
        assert not c.any()
    # a value in it that is not zero makes its own block NaN and no other
    x[7, 20] = 1.0
    a = quantize(sgemm, ref.NVFP4, x if layout == 0 else x.T.contiguous(), M, K, dtype, layout, gt)
    _, byte = ref.unpack(ref.NVFP4, a[0].cpu().numpy(), a[1].cpu().numpy(), M, K)
    want = np.zeros_like(byte)
    want[7, 1] = 0x7F
    assert np.array_equal(byte, want) and not a[0].any()


@gpu
@pytest.mark.parametrize("g", [-1.0, float("nan"), float("inf"), -float("inf")])
def test_zeros_with_a_matrix_scale_that_is_no_scale(sgemm, g):
    a = quantize(sgemm, ref.NVFP4, torch.zeros(5, 40, device="cuda"), 5, 40, "f32", g=torch.tensor([g], device="cuda"))
    _, byte = ref.unpack(ref.NVFP4, a[0].cpu().numpy(), a[1].cpu().numpy(), 5, 40)
    assert (byte == 0x7F).all()
