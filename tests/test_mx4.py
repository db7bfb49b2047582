"""4-bit quantisation and products (b200_sgemm_mx4_*) against 64-bit numpy."""
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


def source(rows, K, seed, dtype="f32"):
    """Blocks of very different sizes, with zeros, ties between codes, subnormals of the scale and an all-zero block."""
    r = np.random.default_rng(seed)
    x = r.standard_normal((rows, K)) * np.exp2(r.integers(-12, 8, (rows, 1)))
    x[r.random((rows, K)) < 0.05] = 0
    tie = r.random((rows, K)) < 0.2
    x[tie] = r.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, -0.25, -5, -6], tie.sum())
    if rows > 2:
        x[1] = 0
        x[2] *= 1e-6
    t = torch.from_numpy(x).to(TYPES[dtype])
    return t, t.double().numpy()


def quantize(sgemm, fmt, x, rows, K, dtype, layout=0, g=None, **kw):
    nc, ns = sgemm.mx4_sizes(fmt, rows, K)
    codes = torch.full((nc,), 0xA5, dtype=torch.uint8, device="cuda")
    scales = torch.full((ns,), 0xA5, dtype=torch.uint8, device="cuda")
    sgemm.mx4_quantize(fmt, layout, pkg.m_type[dtype], x, rows, K, codes, scales, global_scale=g, **kw)
    return codes, scales


# ---- without a device ------------------------------------------------------------------------------------------------

def test_sizes(sgemm):
    assert sgemm.mx4_sizes(ref.NVFP4, 129, 33) == (129 * 32, 2 * 512)
    assert sgemm.mx4_sizes(ref.NVFP4, 1, 65) == (48, 2 * 512)
    assert sgemm.mx4_sizes(ref.MXFP4, 128, 128) == (128 * 64, 512)
    assert sgemm.mx4_sizes(ref.MXFP4, 256, 129) == (256 * 80, 2 * 2 * 512)
    assert sgemm.mx4_sizes(2, 128, 128) == (0, 0)
    big = 1 << 30
    assert sgemm.mx4_sizes(ref.NVFP4, big, big) == (big * big // 2, big // 128 * (big // 64) * 512)


def test_reference_packing_is_its_inverse():
    r = np.random.default_rng(0)
    for fmt in FORMATS:
        code = r.integers(0, 16, (131, 70)).astype(np.uint8)
        byte = r.integers(0, 127, (131, -(-70 // ref.BLOCK[fmt]))).astype(np.uint8)
        c, b = ref.unpack(fmt, *ref.pack(fmt, code, byte), 131, 70)
        assert np.array_equal(c, code) and np.array_equal(b, byte)


def test_quantize_refuses(sgemm):
    l = sgemm.lib()
    ok = dict(format=0, layout=0, type=0, X=256, rows=4, K=32, ldx=0, index=None, source=0, div=1, g=None, codes=256, scales=256)

    def call(**kw):
        return l.b200_sgemm_mx4_quantize(*{**ok, **kw}.values(), None)

    bad = [dict(format=2), dict(format=-1), dict(layout=2), dict(type=3), dict(X=None), dict(rows=0), dict(K=0), dict(codes=None),
           dict(scales=None), dict(ldx=31), dict(layout=1, ldx=3), dict(X=258), dict(type=2, X=257), dict(codes=264), dict(scales=260),
           dict(g=258), dict(format=1, g=256), dict(source=4), dict(index=256), dict(index=256, source=4, div=0),
           dict(index=258, source=4), dict(index=256, source=4, layout=1)]
    for kw in bad:
        assert call(**kw) == pkg.INVALID_ARGUMENT, kw
    for kw in (dict(rows=(1 << 30) + 1), dict(K=(1 << 30) + 1), dict(ldx=1 << 41), dict(rows=1 << 30, K=1 << 30)):
        assert call(**kw) == pkg.UNSUPPORTED_SIZE, kw


def test_dequantize_refuses(sgemm):
    l = sgemm.lib()
    ok = dict(format=0, type=0, codes=256, scales=256, rows=4, K=32, g=None, X=256, ldx=0)

    def call(**kw):
        return l.b200_sgemm_mx4_dequantize(*{**ok, **kw}.values(), None)

    for kw in (dict(format=2), dict(type=3), dict(codes=None), dict(scales=None), dict(X=None), dict(rows=0), dict(K=0), dict(ldx=31),
               dict(codes=8), dict(scales=8), dict(X=257), dict(g=1), dict(format=1, g=256)):
        assert call(**kw) == pkg.INVALID_ARGUMENT, kw
    assert call(rows=1 << 31) == pkg.UNSUPPORTED_SIZE


def test_product_refuses(sgemm):
    l = sgemm.lib()
    ok = dict(format=0, lc=0, type=0, C=256, ac=256, as_=256, bc=256, bs=256, M=4, N=8, K=32, ldc=0, alpha=1.0, ga=None, gb=None)

    def call(**kw):
        return l.b200_sgemm_mx4(*{**ok, **kw}.values(), None)

    for kw in (dict(format=2), dict(lc=2), dict(type=-1), dict(C=None), dict(ac=None), dict(as_=None), dict(bc=None), dict(bs=None),
               dict(M=0), dict(N=0), dict(K=0), dict(ldc=7), dict(lc=1, ldc=3), dict(C=258), dict(type=2, C=257), dict(ac=8),
               dict(as_=8), dict(bc=8), dict(bs=8), dict(ga=2), dict(gb=2), dict(format=1, ga=256), dict(format=1, gb=256)):
        assert call(**kw) == pkg.INVALID_ARGUMENT, kw
    for kw in (dict(M=1 << 31), dict(N=1 << 31), dict(K=1 << 31), dict(ldc=1 << 41)):
        assert call(**kw) == pkg.UNSUPPORTED_SIZE, kw


def test_grouped_refuses(sgemm):
    l = sgemm.lib()
    ok = dict(format=0, type=0, C=256, ac=256, as_=256, bc=256, bs=256, rows=256, N=8, K=32, ldc=0, groups=2, off=256, cnt=256,
              used=0, alpha=1.0, ga=None, gb=None)

    def call(**kw):
        return l.b200_sgemm_mx4_grouped(*{**ok, **kw}.values(), None)

    for kw in (dict(format=2), dict(type=3), dict(C=None), dict(ac=None), dict(as_=None), dict(bc=None), dict(bs=None), dict(off=None),
               dict(cnt=None), dict(rows=0), dict(N=0), dict(K=0), dict(groups=0), dict(ldc=7), dict(C=258), dict(ac=8), dict(as_=8),
               dict(bc=8), dict(bs=8), dict(off=2), dict(cnt=2), dict(ga=2), dict(gb=2), dict(format=1, ga=256)):
        assert call(**kw) == pkg.INVALID_ARGUMENT, kw
    for kw in (dict(rows=1 << 31), dict(groups=1025), dict(N=1 << 22, groups=1024), dict(ldc=1 << 41)):
        assert call(**kw) == pkg.UNSUPPORTED_SIZE, kw
    assert l.b200_sgemm_mx4_device_status(None) == pkg.INVALID_ARGUMENT


# ---- quantisation ----------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("fmt,g", [(ref.MXFP4, None), (ref.NVFP4, None), (ref.NVFP4, 0.125), (ref.NVFP4, 0.0123)],
                         ids=lambda v: ("nvfp4", "mxfp4")[v] if isinstance(v, int) else str(v))
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("shape", [(1, 1), (1, 16), (3, 33), (129, 70), (128, 512), (40, 1030), (300, 600)],
                         ids=lambda s: "x".join(map(str, s)))
def test_quantize_is_exact(sgemm, fmt, dtype, layout, shape, g):
    rows, K = shape
    x, x64 = source(rows, K, rows * 1000 + K, dtype)
    gt = None if g is None else torch.tensor([g], dtype=torch.float32, device="cuda")
    x = (x if layout == 0 else x.T).contiguous().cuda()
    codes, scales = quantize(sgemm, fmt, x, rows, K, dtype, layout, gt)
    want = ref.pack(fmt, *ref.quantize(fmt, x64, 1.0 if g is None else np.float32(g)))
    assert np.array_equal(scales.cpu().numpy(), want[1])
    assert np.array_equal(codes.cpu().numpy(), want[0])
    # and back
    code, byte = ref.unpack(fmt, *want, rows, K)
    for out_type in TYPES:
        out = torch.full((rows, K), 7.0, dtype=TYPES[out_type], device="cuda")
        sgemm.mx4_dequantize(fmt, pkg.m_type[out_type], codes, scales, rows, K, out, global_scale=gt)
        exact = ref.values(fmt, code, byte)  # fits FP32; times g one rounding, to the type another
        v = torch.from_numpy(exact.astype(np.float32)) * (1.0 if g is None else torch.tensor(np.float32(g)))
        assert torch.equal(out.cpu(), v.to(TYPES[out_type]))


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
def test_quantize_leading_dimension_and_alignment(sgemm, fmt):
    rows, K, ld = 70, 100, 109
    for dtype in TYPES:
        for layout in (0, 1):
            n, m = (rows, K) if layout == 0 else (K, rows)
            full = torch.randn(n, ld, dtype=torch.float64).to(TYPES[dtype])
            for shift in (0, 1):  # a base that is not on 16 bytes
                view = full.cuda().reshape(-1)[shift:]
                part = full.reshape(-1)[shift:][:(n - 1) * ld + m]
                x = torch.as_strided(part, (n, m), (ld, 1)).double().numpy()
                codes, scales = quantize(sgemm, fmt, view, rows, K, dtype, layout, ldx=ld)
                want = ref.pack(fmt, *ref.quantize(fmt, x if layout == 0 else x.T))
                assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
def test_quantize_special_values(sgemm, fmt):
    tiny, big = 2.0 ** -149, 3.4028234663852886e38
    x = np.zeros((8, 64), np.float32)
    x[0, 3], x[1, 40], x[2, 17] = np.nan, np.inf, -np.inf
    x[0, 35], x[2, 50] = 5.0, 1.0
    x[3, :32], x[3, 32:] = tiny, big
    x[4] = np.linspace(-1, 1, 64) * 2.0 ** -130
    x[5, 0], x[5, 1], x[5, 2] = 1.0, 2.0 ** -30, -(2.0 ** -30)
    x[6] = -0.0
    x[7] = np.linspace(-448 * 6 * 4, 448 * 6 * 4, 64)  # above what nvfp4 holds with g = 1
    codes, scales = quantize(sgemm, fmt, dev(x), 8, 64, "f32")
    code, byte = ref.quantize(fmt, x.astype(np.float64))
    want = ref.pack(fmt, code, byte)
    got = ref.unpack(fmt, codes.cpu().numpy(), scales.cpu().numpy(), 8, 64)
    assert np.array_equal(got[1], byte)
    assert np.array_equal(got[0], code)
    assert np.array_equal(codes.cpu().numpy(), want[0])
    out = torch.empty(8, 64, device="cuda")
    sgemm.mx4_dequantize(fmt, pkg.m_type.f32, codes, scales, 8, 64, out)
    nan = np.isnan(out.cpu().numpy())
    b = ref.BLOCK[fmt]
    for row, k in ((0, 3), (1, 40), (2, 17)):
        assert nan[row, k // b * b:(k // b + 1) * b].all()
    assert nan.sum() == 3 * b


@gpu
@pytest.mark.parametrize("g", [0.0, -1.0, float("nan"), float("inf"), 2.0 ** -91, 2.0 ** 91])
def test_quantize_bad_matrix_scale_gives_nan(sgemm, g):
    x = torch.randn(5, 40, device="cuda")
    codes, scales = quantize(sgemm, ref.NVFP4, x, 5, 40, "f32", g=torch.tensor([g], device="cuda"))
    code, byte = ref.unpack(ref.NVFP4, codes.cpu().numpy(), scales.cpu().numpy(), 5, 40)
    assert (byte == 0x7F).all() and (code == 0).all()


@gpu
def test_quantize_borders_of_an_awkward_matrix_scale(sgemm):
    """Values next to the border between two codes, where the quotient in FP32 cannot tell the side."""
    r = np.random.default_rng(3)
    for trial in range(30):
        g = np.float32(r.uniform(0.5, 2.0) * 2.0 ** float(r.integers(-30, 10)))
        if trial >= 20:  # few bits, and as close below a power of two as 12 or 13 of them come
            g = np.float32([1.0, 0.75, 2 - 2.0 ** -11, 2 - 2.0 ** -12, 1 + 2.0 ** -11][trial % 5])
        s = ref.E4M3[r.integers(8, 0x7E, (64, 8))]
        mid = r.choice([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], (64, 8, 16))
        x = (mid * s[..., None] * float(g)).astype(np.float32)
        step = r.integers(-1, 2, x.shape)
        x = np.where(step < 0, np.nextafter(x, np.float32(0)), np.where(step > 0, np.nextafter(x, np.float32(np.inf)), x))
        x[..., 0] = (6 * s * float(g)).astype(np.float32)
        x = (x * r.choice([-1, 1], x.shape)).astype(np.float32).reshape(64, 128)
        codes, scales = quantize(sgemm, ref.NVFP4, dev(x), 64, 128, "f32", g=torch.tensor([g], device="cuda"))
        want = ref.pack(ref.NVFP4, *ref.quantize(ref.NVFP4, x.astype(np.float64), g))
        assert np.array_equal(scales.cpu().numpy(), want[1])
        assert np.array_equal(codes.cpu().numpy(), want[0])


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
def test_quantize_gathers_rows(sgemm, fmt):
    rows, K, n = 400, 96, 50
    x, x64 = source(n, K, 9)
    r = np.random.default_rng(4)
    index = r.integers(0, n * 3, rows).astype(np.int32)  # slot numbers, three per row of X
    index[r.random(rows) < 0.3] = -1
    index[128:256] = -1         # a band without any
    index[300] = n * 3          # behind X
    codes, scales = quantize(sgemm, fmt, x.cuda(), rows, K, "f32", row_index=dev(index), source_rows=n, index_div=3)
    code, byte = ref.quantize(fmt, x64)
    used = (index >= 0) & (index < n * 3)
    got_code, got_byte = ref.unpack(fmt, codes.cpu().numpy(), scales.cpu().numpy(), rows, K)
    assert np.array_equal(got_code[used], code[index[used] // 3])
    assert np.array_equal(got_byte[used], byte[index[used] // 3])
    assert (codes.cpu().numpy().reshape(rows, -1)[~used] == 0xA5).all()
    assert (got_byte[128:256] == 0xA5).all() and (got_byte[~used][: (~used)[:128].sum()] == 0).all()


# ---- products --------------------------------------------------------------------------------------------------------

def operand(fmt, rows, K, seed, spread=3):
    """A quantised matrix made of its own parts: all codes, scales over a few powers of two."""
    r = np.random.default_rng(seed)
    code = r.integers(0, 16, (rows, K)).astype(np.uint8)
    blocks = -(-K // ref.BLOCK[fmt])
    byte = (r.integers(40 - 8 * spread, 40 + 8 * spread, (rows, blocks)) if fmt == ref.NVFP4
            else r.integers(127 - spread, 127 + spread, (rows, blocks))).astype(np.uint8)
    codes, scales = ref.pack(fmt, code, byte)
    return dev(codes), dev(scales), ref.values(fmt, code, byte)


def check(got, want, bound):
    got = got.double().cpu().numpy()
    off = np.abs(got - want) / bound
    assert np.isfinite(got).all() and off.max() <= 1, f"{off.max():.3g} times the bound at {np.unravel_index(off.argmax(), off.shape)}"


SHAPES = [(1, 1, 1), (1, 128, 64), (3, 5, 7), (128, 128, 256), (17, 130, 100), (33, 257, 515), (65, 64, 320), (129, 300, 1000),
          (200, 520, 2048), (1, 700, 4096), (20, 256, 8192), (300, 2, 777), (4, 129, 2048), (3, 1000, 5000), (2100, 1, 96), (2, 4, 33), (4, 4, 640), (5, 300, 4096), (40, 50, 1), (200, 100, 31), (1, 3, 9000), (1000, 16, 200), (512, 640, 130)]


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("layout_c", [0, 1])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_product(sgemm, fmt, layout_c, dtype, shape):
    M, N, K = shape
    a, b = operand(fmt, M, K, M + K), operand(fmt, N, K, 7 * N + K)
    alpha, ga, gb = 0.75, 0.01, 0.3
    g = None if fmt == ref.MXFP4 else torch.tensor([ga, gb], device="cuda")
    factor = alpha * (1.0 if g is None else float(np.float32(ga)) * float(np.float32(gb)))
    ld = (N if layout_c == 0 else M) + 3
    n = M if layout_c == 0 else N
    c = torch.full((n, ld), 11.0, dtype=TYPES[dtype], device="cuda")
    sgemm.gemm_mx4(fmt, layout_c, pkg.m_type[dtype], c, a[0], a[1], b[0], b[1], M, N, K, ldc=ld, alpha=alpha,
                   global_a=None if g is None else g[:1], global_b=None if g is None else g[1:])
    assert sgemm.mx4_device_status() == 0
    assert (c[:, ld - 3:] == 11).all()
    want = a[2] @ b[2].T * factor
    bound = ref.product_bound(a[2], b[2] * factor, want, dtype)
    got = c[:, :ld - 3]
    check(got if layout_c == 0 else got.T, want, bound)


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("M,N", [(1, 300), (2, 129), (40, 130), (200, 1), (300, 200), (2100, 2300)])
def test_product_over_the_whole_range_of_scales(sgemm, fmt, dtype, M, N):
    """The smallest and the largest scales of both formats, zero scales among them; products stay in FP32's range."""
    K = 1100
    r = np.random.default_rng(M)
    sides = []
    for rows, sign in ((M, 1), (N, -1)):
        code = r.integers(0, 16, (rows, K)).astype(np.uint8)
        blocks = -(-K // ref.BLOCK[fmt])
        if fmt == ref.NVFP4:
            byte = r.choice([0, 1, 7, 8, 0x38, 0x70, 0x7D, 0x7E], (rows, blocks))
        else:  # 2^+-100 on one side against 2^-+100 on the other, and 2^-127
            byte = np.where(r.random((rows, blocks)) < 0.1, 0, 127 + sign * 100 + r.integers(-12, 12, (rows, blocks)))
        byte = byte.astype(np.uint8)
        sides.append((*(dev(v) for v in ref.pack(fmt, code, byte)), ref.values(fmt, code, byte)))
    a, b = sides
    c = torch.empty(M, N, dtype=TYPES[dtype], device="cuda")
    sgemm.gemm_mx4(fmt, 0, pkg.m_type[dtype], c, a[0], a[1], b[0], b[1], M, N, K)
    want = a[2] @ b[2].T
    check(c, want, ref.product_bound(a[2], b[2], want, dtype))
    assert sgemm.mx4_device_status() == 0


@gpu
@pytest.mark.parametrize("M,N", [(1, 300), (300, 2), (40, 130), (300, 200)])
def test_product_of_huge_scales_where_the_codes_are_zero(sgemm, M, N):
    """mxfp4 scales of 2^100 and more on both sides, where one side's codes are all zero; the other blocks' sums are exact."""
    K, r = 1088, np.random.default_rng(M)
    sides = []
    for side, rows in enumerate((M, N)):
        code = r.integers(0, 16, (rows, K)).astype(np.uint8)
        byte = r.choice([227, 240, 252], (rows, K // 32)).astype(np.uint8)
        block = np.arange(K // 32) % 4
        code[:, np.repeat(block == side, 32)] = 0  # block % 4: 0 and 1 zero on one side, 2 on both, 3 on neither
        code[:, np.repeat(block == 2, 32)] = 0
        byte[:, block == 3] = 127
        sides.append((*(dev(v) for v in ref.pack(ref.MXFP4, code, byte)), ref.values(ref.MXFP4, code, byte)))
    a, b = sides
    c = torch.empty(M, N, device="cuda")
    sgemm.gemm_mx4(ref.MXFP4, 0, pkg.m_type.f32, c, a[0], a[1], b[0], b[1], M, N, K)
    assert np.array_equal(c.cpu().numpy(), (a[2] @ b[2].T).astype(np.float32))
    assert sgemm.mx4_device_status() == 0


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_product_many_tiles(sgemm, fmt, dtype):
    """More tiles than SMs, packed C, and the same bits on every call."""
    M, N, K = 1500, 2200, 1100
    a, b = operand(fmt, M, K, 1), operand(fmt, N, K, 2)
    for layout_c in (0, 1):
        c = [torch.full((M, N) if layout_c == 0 else (N, M), float("nan"), dtype=TYPES[dtype], device="cuda") for _ in range(2)]
        for out in c:
            sgemm.gemm_mx4(fmt, layout_c, pkg.m_type[dtype], out, a[0], a[1], b[0], b[1], M, N, K)
        assert sgemm.mx4_device_status() == 0
        assert torch.equal(c[0], c[1])
        want = a[2] @ b[2].T
        check(c[0] if layout_c == 0 else c[0].T, want, ref.product_bound(a[2], b[2], want, dtype))


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("layout_c", [0, 1])
@pytest.mark.parametrize("shape", [(2100, 2300, 700), (2304, 2560, 64), (1025, 5000, 2049)], ids=lambda s: "x".join(map(str, s)))
def test_product_by_pairs_of_ctas(sgemm, fmt, dtype, layout_c, shape):
    M, N, K = shape
    a, b = operand(fmt, M, K, 3), operand(fmt, N, K, 4)
    n, m = (M, N) if layout_c == 0 else (N, M)
    for ld in (m, m + 5):
        c = torch.full((n, ld), 9.0, dtype=TYPES[dtype], device="cuda")
        sgemm.gemm_mx4(fmt, layout_c, pkg.m_type[dtype], c, a[0], a[1], b[0], b[1], M, N, K, ldc=ld, alpha=0.5)
        assert sgemm.mx4_device_status() == 0
        assert (c[:, m:] == 9).all()
        want = a[2] @ b[2].T * 0.5
        check(c[:, :m] if layout_c == 0 else c[:, :m].T, want, ref.product_bound(a[2], b[2] * 0.5, want, dtype))


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
def test_product_exact_sums(sgemm, fmt):
    """Integers that the accumulator holds exactly come out exactly: one value per row and column, all of K."""
    M, N, K = 130, 140, 640
    one = np.full((M, K), 2, np.uint8)  # 1.0
    byte = (np.full((M, -(-K // ref.BLOCK[fmt])), 0x38 if fmt == ref.NVFP4 else 127)).astype(np.uint8)
    code = (np.arange(N)[:, None] * 5 + np.arange(K)[None]) % 16
    byte_b = np.full((N, byte.shape[1]), byte[0, 0], np.uint8)
    a, b = ref.pack(fmt, one, byte), ref.pack(fmt, code.astype(np.uint8), byte_b)
    c = torch.empty(M, N, device="cuda")
    sgemm.gemm_mx4(fmt, 0, pkg.m_type.f32, c, dev(a[0]), dev(a[1]), dev(b[0]), dev(b[1]), M, N, K)
    want = ref.values(fmt, one, byte) @ ref.values(fmt, code.astype(np.uint8), byte_b).T
    assert np.array_equal(c.cpu().numpy(), want)


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("other", [1, 2, 200])
def test_product_of_nan_blocks_is_nan(sgemm, fmt, other):
    M, N, K = 40, other, 300
    x = torch.randn(M, K)
    x[7, 290] = float("nan")
    x[39, 0] = float("inf")
    a = quantize(sgemm, fmt, x.cuda(), M, K, "f32")
    b = operand(fmt, N, K, 5)
    c, t = torch.zeros(M, N, device="cuda"), torch.zeros(N, M, device="cuda")
    sgemm.gemm_mx4(fmt, 0, pkg.m_type.f32, c, a[0], a[1], b[0], b[1], M, N, K)
    sgemm.gemm_mx4(fmt, 0, pkg.m_type.f32, t, b[0], b[1], a[0], a[1], N, M, K)
    for nan in (torch.isnan(c), torch.isnan(t.T)):
        assert nan[7].all() and nan[39].all()
        assert nan.sum().item() == 2 * N


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("few", [1, 2, 3])
def test_product_of_nan_blocks_of_the_short_side(sgemm, fmt, few):
    M, N, K = few, 300, 1100
    x = torch.randn(M, K)
    x[M - 1, 777] = float("nan")
    a = quantize(sgemm, fmt, x.cuda(), M, K, "f32")
    b = operand(fmt, N, K, 5)
    c, t = torch.zeros(M, N, device="cuda"), torch.zeros(N, M, device="cuda")
    sgemm.gemm_mx4(fmt, 0, pkg.m_type.f32, c, a[0], a[1], b[0], b[1], M, N, K)
    sgemm.gemm_mx4(fmt, 0, pkg.m_type.f32, t, b[0], b[1], a[0], a[1], N, M, K)
    for nan in (torch.isnan(c), torch.isnan(t.T)):
        assert nan[M - 1].all() and nan.sum().item() == N


def grouped_case(fmt, counts, N, K, rows=None, seed=0):
    counts = np.array(counts, np.int32)
    offsets = np.concatenate([[0], np.cumsum(-(-counts // 128) * 128)]).astype(np.int32)
    rows = rows or max(int(offsets[-1]), 1)
    a = operand(fmt, rows, K, seed + 1)
    parts = [operand(fmt, N, K, seed + 10 + e) for e in range(len(counts))]
    b = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]), [p[2] for p in parts]
    return a, b, offsets, counts, rows


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("counts,N,K", [([1], 1, 1), ([3, 0, 130, 1], 200, 300), ([0, 0, 5], 128, 256), ([33, 64, 20, 0, 300], 130, 1000),
                                        ([1] * 40, 300, 2048), ([0, 0], 64, 64), ([500, 700], 520, 512), ([40, 100, 1, 32, 64, 33, 65, 0, 0, 0, 0, 0, 0, 0, 0, 0], 130, 300), ([300, 0, 129, 700, 256, 1, 512, 400], 2200, 512)],
                         ids=lambda v: "-".join(map(str, v[:5])) if isinstance(v, list) else str(v))
@pytest.mark.parametrize("hint", [0, 1])
def test_grouped(sgemm, fmt, dtype, counts, N, K, hint):
    a, b, offsets, counts, rows = grouped_case(fmt, counts, N, K)
    g = None if fmt == ref.MXFP4 else torch.linspace(0.5, 1.5, len(counts), device="cuda")
    c = torch.full((rows, N + 1), 3.0, dtype=TYPES[dtype], device="cuda")
    sgemm.gemm_mx4_grouped(fmt, pkg.m_type[dtype], c, a[0], a[1], b[0], b[1], rows, N, K, len(counts), dev(offsets), dev(counts),
                           ldc=N + 1, used_rows=int(counts.sum()) * hint, global_b=g)
    assert sgemm.mx4_device_status() == 0
    got, left = c.cpu(), torch.ones(rows, dtype=torch.bool)
    for e, n in enumerate(counts):
        at = slice(int(offsets[e]), int(offsets[e]) + int(n))
        left[at] = False
        f = 1.0 if g is None else float(g[e])
        want = a[2][at] @ b[2][e].T * f
        if n:
            check(got[at, :N], want, ref.product_bound(a[2][at], b[2][e] * f, want, dtype))
    assert (got[left] == 3).all() and (got[:, N] == 3).all()


@gpu
def test_grouped_leaves_out_groups_that_do_not_fit(sgemm):
    N, K = 130, 128
    a, b, offsets, counts, rows = grouped_case(ref.NVFP4, [5, 5, 5, 5, 5, 200], N, K)
    offsets, counts = offsets.copy(), counts.copy()
    offsets[1] = 64          # not a multiple of 128
    offsets[2] = -128
    counts[3] = rows         # behind the matrix
    counts[4] = -1
    c = torch.full((rows, N), 3.0, device="cuda")
    sgemm.gemm_mx4_grouped(ref.NVFP4, pkg.m_type.f32, c, a[0], a[1], b[0], b[1], rows, N, K, 6, dev(offsets), dev(counts))
    assert sgemm.mx4_device_status() == 2
    assert sgemm.mx4_device_status() == 0
    c = c.cpu()
    for e in (0, 5):
        at = slice(int(offsets[e]), int(offsets[e]) + int(counts[e]))
        want = a[2][at] @ b[2][e].T
        check(c[at], want, ref.product_bound(a[2][at], b[2][e], want, "f32"))
        c[at] = 3
    assert (c == 3).all()
    # groups on top of each other: more tiles than the rows make
    c = torch.full((rows, N), 3.0, device="cuda")
    sgemm.gemm_mx4_grouped(ref.NVFP4, pkg.m_type.f32, c, a[0], a[1], b[0], b[1], rows, N, K, 6, dev(np.zeros(6, np.int32)),
                           dev(np.full(6, rows, np.int32)))
    assert sgemm.mx4_device_status() == 2 and (c == 3).all()


# ---- as a program uses them ------------------------------------------------------------------------------------------

@gpu
def test_captured_and_replayed(sgemm):
    """Quantise and multiply inside a graph, replayed on two streams at once with a second graph: nothing is shared."""
    K, N = 2048, 1024
    graphs = []
    for M, seed in ((3, 1), (5, 2)):
        x = torch.randn(M, K, device="cuda")
        b = operand(ref.NVFP4, N, K, seed)
        nc, ns = sgemm.mx4_sizes(ref.NVFP4, M, K)
        codes, scales = torch.empty(nc, dtype=torch.uint8, device="cuda"), torch.empty(ns, dtype=torch.uint8, device="cuda")
        c = torch.zeros(M, N, device="cuda")

        def step(x=x, b=b, codes=codes, scales=scales, c=c, M=M):
            sgemm.mx4_quantize(ref.NVFP4, 0, pkg.m_type.f32, x, M, K, codes, scales)
            sgemm.gemm_mx4(ref.NVFP4, 0, pkg.m_type.f32, c, codes, scales, b[0], b[1], M, N, K)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append((graph, x, c, step))
    want = []
    for graph, x, c, step in graphs:
        x.copy_(torch.randn_like(x))
        step()
        want.append(c.clone())
        c.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for s, (graph, *_) in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for w, (_, _, c, _) in zip(want, graphs):
        assert torch.equal(w, c)
    assert sgemm.mx4_device_status() == 0


@gpu
def test_linear_layer_and_its_gradients(sgemm):
    """y = x w^T and both gradients, each from two quantisations along its own summed dimension: the products agree with
    those of the dequantised matrices."""
    M, N, K = 200, 320, 260
    x, w, dy = (torch.randn(s, device="cuda") for s in ((M, K), (N, K), (M, N)))

    def product(p, p_layout, q, q_layout, m, n, k):
        qa, qb = quantize(sgemm, ref.MXFP4, p, m, k, "f32", p_layout), quantize(sgemm, ref.MXFP4, q, n, k, "f32", q_layout)
        c = torch.empty(m, n, device="cuda")
        sgemm.gemm_mx4(ref.MXFP4, 0, pkg.m_type.f32, c, *qa, *qb, m, n, k)
        a, b = (ref.values(ref.MXFP4, *ref.quantize(ref.MXFP4, v.double().cpu().numpy()))
                for v in (p if p_layout == 0 else p.T, q if q_layout == 0 else q.T))
        want = a @ b.T
        check(c, want, ref.product_bound(a, b, want, "f32"))

    product(x, 0, w, 0, M, N, K)    # y[m, n]: sum over k
    product(dy, 0, w, 1, M, K, N)   # dx[m, k]: sum over n; w's transpose is its columns
    product(dy, 1, x, 1, N, K, M)   # dw[n, k]: sum over m
    assert sgemm.mx4_device_status() == 0


@gpu
def test_leading_dimensions_beyond_32_bits(sgemm):
    """Elements whose offset passes 2^31, on every side that takes a leading dimension."""
    rows, K, ld = 2100, 96, 1 << 20
    bf16, f32 = pkg.m_type.bf16, pkg.m_type.f32
    x = torch.randn(rows, K, device="cuda").bfloat16()
    big = torch.empty(rows, ld, dtype=torch.bfloat16, device="cuda")
    big[:, :K] = x
    packed, strided = quantize(sgemm, ref.NVFP4, x, rows, K, "bf16"), quantize(sgemm, ref.NVFP4, big, rows, K, "bf16", ldx=ld)
    assert all(torch.equal(p, s) for p, s in zip(packed, strided))
    # columns: K of them 2^20 apart
    packed_t = quantize(sgemm, ref.MXFP4, x, K, rows, "bf16", 1)
    strided_t = quantize(sgemm, ref.MXFP4, big, K, rows, "bf16", 1, ldx=ld)
    assert all(torch.equal(p, s) for p, s in zip(packed_t, strided_t))
    out = torch.empty(rows, K, dtype=torch.bfloat16, device="cuda")
    sgemm.mx4_dequantize(ref.NVFP4, bf16, *packed, rows, K, out)
    big[:, :K] = 0
    sgemm.mx4_dequantize(ref.NVFP4, bf16, *packed, rows, K, big, ldx=ld)
    assert torch.equal(big[:, :K], out)
    w = quantize(sgemm, ref.NVFP4, torch.randn(K, K, device="cuda"), K, K, "f32")
    for layout_c in (0, 1):
        c = torch.empty(rows, K, dtype=torch.bfloat16, device="cuda")
        big[:, :K] = 0
        a, b, m, n = (packed, w, rows, K) if layout_c == 0 else (w, packed, K, rows)
        sgemm.gemm_mx4(ref.NVFP4, layout_c, bf16, c, *a, *b, m, n, K)
        sgemm.gemm_mx4(ref.NVFP4, layout_c, bf16, big, *a, *b, m, n, K, ldc=ld)
        assert torch.equal(big[:, :K], c)
    assert sgemm.mx4_device_status() == 0


@gpu
def test_codes_beyond_32_bits(sgemm):
    """A matrix whose codes take more than 2^32 bytes: its last rows, quantised, read back and multiplied."""
    rows, K, last = (1 << 17) + 40, 1 << 16, 100
    bf16 = pkg.m_type.bf16
    x = torch.zeros(rows, K, dtype=torch.bfloat16, device="cuda")
    tail = torch.randn(last, K, device="cuda").bfloat16()
    x[-last:] = tail
    codes, scales = quantize(sgemm, ref.MXFP4, x, rows, K, "bf16")
    assert codes.numel() > 1 << 32
    code, byte = ref.quantize(ref.MXFP4, tail.double().cpu().numpy())
    values = ref.values(ref.MXFP4, code, byte)
    assert np.array_equal(codes.view(rows, -1)[-last:].cpu().numpy().reshape(-1), ref.pack(ref.MXFP4, code, byte)[0])
    sgemm.mx4_dequantize(ref.MXFP4, bf16, codes, scales, rows, K, x)
    assert np.array_equal(x[-last:].double().cpu().numpy(), values)
    assert not x[:1000].any() and not x[rows // 2:rows // 2 + 1000].any()
    del x
    for m in (1, 3):
        a = operand(ref.MXFP4, m, K, 6)
        want = a[2] @ values.T
        bound = ref.product_bound(a[2], values, want, "f32")
        c = torch.empty(m, rows, device="cuda")
        sgemm.gemm_mx4(ref.MXFP4, 0, pkg.m_type.f32, c, a[0], a[1], codes, scales, m, rows, K)
        check(c[:, -last:], want, bound)
        assert not c[:, :-last].any()
    assert sgemm.mx4_device_status() == 0
