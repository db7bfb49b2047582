"""The ways in which the dispatcher cuts a 4-bit product (columns of a tile, CTAs that share its K): each is run."""
import math
import random
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

import mx4_reference as ref
import rocm_sgemm_b200 as pkg

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FORMATS = [ref.NVFP4, ref.MXFP4]
fmt_ids = lambda f: ("nvfp4", "mxfp4")[f]  # noqa: E731
SMS = 148

# (layout of C, M, N, K) by (columns, split); the same for all types.  No extent fits a tile; with K beyond 2^15 FP16 results are
# added in parts
CASES = {(64, 1): [(0, 5, 9477, 515), (1, 5190, 137, 206)],
         (64, 2): [(0, 701, 699, 8190), (0, 131, 2373, 7000), (1, 131, 1046, 3543)],
         (64, 4): [(1, 130, 397, 2369), (0, 1726, 3, 32781)],
         (64, 8): [(0, 130, 397, 2369), (1, 5, 5, 1796), (0, 3, 5, 32843)],
         (128, 1): [(0, 5190, 137, 206), (0, 131, 9001, 2190)],
         (128, 2): [(0, 131, 4097, 8190), (1, 131, 2373, 7000)],
         (128, 4): [(0, 509, 517, 8190), (0, 1039, 147, 5668)],
         (128, 8): [(0, 403, 131, 12150), (1, 130, 386, 35641)],
         (256, 1): [(0, 9643, 142, 1863)]}
# (used rows, N, K, counts) by columns and type
GROUPED = {(256, "f32"): (2053, 4090, 2040, [600, 0, 129, 511, 257, 300, 255, 1]), (256, "f16"): (1171, 2051, 1100, [300, 1, 870, 0]),
           (128, "f32"): (1171, 2051, 1100, [300, 1, 870, 0]), (128, "bf16"): (516, 1239, 300, [100, 0, 200, 1, 3, 60, 150, 2]),
           (64, "f32"): (101, 65, 65, [33, 0, 68]), (64, "f16"): (101, 65, 65, [33, 0, 68])}


def plan(layout, dtype, M, N, K, groups=0):
    return pkg.mx4_plan(layout, pkg.m_type[dtype], M, N, K, groups, SMS)


def test_plan_refuses(sgemm):
    ok = dict(layout=0, type=0, M=4, N=8, K=32, groups=0, sms=148)

    def call(**kw):
        import ctypes
        a, b = ctypes.c_int(0), ctypes.c_int(0)
        return sgemm.lib().b200_sgemm_mx4_plan(*{**ok, **kw}.values(), ctypes.byref(a), ctypes.byref(b))

    assert call() == pkg.OK
    for kw in (dict(layout=2), dict(type=3), dict(M=0), dict(N=0), dict(K=0), dict(sms=0), dict(layout=1, groups=2)):
        assert call(**kw) == pkg.INVALID_ARGUMENT, kw
    for kw in (dict(M=1 << 31), dict(N=1 << 31), dict(K=1 << 31), dict(groups=1025), dict(groups=1024, N=1 << 22)):
        assert call(**kw) == pkg.UNSUPPORTED_SIZE, kw
    assert sgemm.lib().b200_sgemm_mx4_plan(0, 0, 4, 8, 32, 0, 148, None, None) == pkg.INVALID_ARGUMENT
    assert call(sms=1) == pkg.INVALID_ARGUMENT and call(sms=2) == pkg.OK  # a pair of CTAs needs two
    assert plan(0, "f32", 1, 4096, 4096) == (0, 1)


def test_cases_visit_every_cut(sgemm):
    """The cases below take the cuts that they stand for, and sizes all over the range take no others."""
    for cut, cases in CASES.items():
        for layout, M, N, K in cases:
            for dtype in TYPES:
                assert plan(layout, dtype, M, N, K) == cut, (cut, dtype, layout, M, N, K)
    for (columns, dtype), (used, N, K, counts) in GROUPED.items():
        assert used == sum(counts) and plan(0, dtype, used, N, K, len(counts)) == (columns, 1), (columns, dtype)
    r = random.Random(3)
    size = lambda lo, hi: int(math.exp(r.uniform(math.log(lo), math.log(hi))))  # noqa: E731
    for _ in range(20000):
        M, N, K, groups = size(1, 30000), size(1, 30000), size(1, 1 << 20), r.choice([0, 0, 1, 7, 64, 300])
        dtype, layout = r.choice(sorted(TYPES)), 0 if groups else r.choice([0, 1])
        cut = plan(layout, dtype, M, N, K, groups)
        assert cut in CASES or cut == (0, 1), (cut, M, N, K)
        assert groups == 0 or cut[1] == 1


def operand(fmt, rows, K, seed):
    """Codes and scales over a few powers of two, and their float64 values on the device."""
    r = np.random.default_rng(seed)
    code = r.integers(0, 16, (rows, K)).astype(np.uint8)
    low, high = (24, 56) if fmt == ref.NVFP4 else (125, 129)
    byte = r.integers(low, high, (rows, -(-K // ref.BLOCK[fmt]))).astype(np.uint8)
    codes, scales = (torch.from_numpy(v).cuda() for v in ref.pack(fmt, code, byte))
    return codes, scales, torch.from_numpy(ref.values(fmt, code, byte)).cuda()


def check(got, a, b, dtype):
    """As mx4_reference.product_bound, on the device."""
    want, size, K = a @ b.T, a.abs() @ b.abs().T, a.shape[1]
    steps = -(-K // 64)
    err = size * (min(steps, 32) * 2.0 ** -22 + -(-K // 1024) * 2.0 ** -24 if dtype == "f32" else steps * 2.0 ** -22)
    err += want.abs() * (4 * 2.0 ** -24 + ref.TYPE_EPS[dtype] / 2) + (2.0 ** -25 if dtype == "f16" else 0) + 1e-300
    off = ((got.double() - want).abs() / err).max().item()
    assert off <= 1, f"{off:.3g} times the bound"


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("case", [c for cases in CASES.values() for c in cases], ids=lambda c: "x".join(map(str, c)))
def test_product_of_every_cut(sgemm, fmt, case):
    layout, M, N, K = case
    assert torch.cuda.get_device_properties(0).multi_processor_count == SMS
    a, b = operand(fmt, M, K, 1), operand(fmt, N, K, 2)
    alpha = 2.0 ** -12  # keeps FP16 results in range
    n, m = (M, N) if layout == 0 else (N, M)
    for dtype in TYPES:
        c = [torch.full((n, m + 3), 9.0, dtype=TYPES[dtype], device="cuda") for _ in range(2)]
        for out in c:
            sgemm.gemm_mx4(fmt, layout, pkg.m_type[dtype], out, a[0], a[1], b[0], b[1], M, N, K, ldc=m + 3, alpha=alpha)
        assert sgemm.mx4_device_status() == 0
        assert torch.equal(*c) and (c[0][:, m:] == 9).all()
        check(c[0][:, :m] if layout == 0 else c[0][:, :m].T, a[2], b[2] * alpha, dtype)


@gpu
@pytest.mark.parametrize("fmt", FORMATS, ids=fmt_ids)
@pytest.mark.parametrize("columns,dtype", sorted(GROUPED))
def test_grouped_of_every_tile(sgemm, fmt, columns, dtype):
    used, N, K, counts = GROUPED[columns, dtype]
    offsets = np.concatenate([[0], np.cumsum(-(-np.array(counts) // 128) * 128)]).astype(np.int32)
    rows, alpha = int(offsets[-1]) + 128, 2.0 ** -12
    a, parts = operand(fmt, rows, K, 3), [operand(fmt, N, K, 10 + e) for e in range(len(counts))]
    codes, scales = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    c = torch.full((rows, N), 9.0, dtype=TYPES[dtype], device="cuda")
    sgemm.gemm_mx4_grouped(fmt, pkg.m_type[dtype], c, a[0], a[1], codes, scales, rows, N, K, len(counts),
                           torch.from_numpy(offsets).cuda(), torch.tensor(counts, dtype=torch.int32, device="cuda"), used_rows=used,
                           alpha=alpha)
    assert sgemm.mx4_device_status() == 0
    for e, n in enumerate(counts):
        at = slice(int(offsets[e]), int(offsets[e]) + n)
        if n:
            check(c[at], a[2][at], parts[e][2] * alpha, dtype)
        c[at] = 9
    assert (c == 9).all()


@gpu
def test_products_at_once(sgemm):
    """Every kind of cut from threads of their own, on streams of their own, at the same time: the bits of calls made alone."""
    shapes = [(1, 4096, 2048), (5, 5, 1796), (130, 397, 2369), (509, 517, 4094), (403, 131, 6150), (2100, 2300, 700), (1500, 700, 300)]
    work = []
    for i, (M, N, K) in enumerate(shapes):
        fmt, dtype = FORMATS[i % 2], sorted(TYPES)[i % 3]
        a, b = operand(fmt, M, K, 1), operand(fmt, N, K, 2)
        c = [torch.zeros(M, N, dtype=TYPES[dtype], device="cuda") for _ in range(2)]
        call = lambda out, stream, a=a, b=b, fmt=fmt, t=pkg.m_type[dtype], n=(M, N, K): sgemm.gemm_mx4(  # noqa: E731
            fmt, 0, t, out, a[0], a[1], b[0], b[1], *n, alpha=2.0 ** -12, stream=stream)
        call(c[0], torch.cuda.current_stream())
        work.append((call, c, torch.cuda.Stream()))
    torch.cuda.synchronize()

    def repeat(call, c, stream):
        for _ in range(200):
            call(c[1], stream)

    with ThreadPoolExecutor(len(work)) as pool:
        for done in [pool.submit(repeat, *w) for w in work]:
            done.result()
    torch.cuda.synchronize()
    assert sgemm.mx4_device_status() == 0
    for _, c, _ in work:
        assert torch.isfinite(c[0]).all() and c[0].any() and torch.equal(*c)
