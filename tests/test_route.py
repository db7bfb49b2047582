"""Routing (b200_sgemm_route_*): slots sorted by expert, rows there and back, and their gradients, against 64-bit numpy."""
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

import mx4_reference as ref
import rocm_sgemm_b200 as pkg

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def sort_reference(ids, experts, align, rows):
    slot_row = np.full(ids.size, -1, np.int32)
    row_slot = np.full(rows, -1, np.int32)
    offsets, counts = np.zeros(experts + 1, np.int32), np.zeros(experts, np.int32)
    at = 0
    for e in range(experts):
        slots = np.nonzero(ids.reshape(-1) == e)[0]
        offsets[e], counts[e] = at, slots.size
        slot_row[slots] = at + np.arange(slots.size)
        row_slot[at:at + slots.size] = slots
        at += -(-slots.size // align) * align
    offsets[experts] = at
    return offsets, counts, slot_row, row_slot


def run_sort(sgemm, ids, experts, align, extra=0):
    tokens, top_k = ids.shape
    rows = sgemm.route_capacity(tokens, top_k, experts, align) + extra
    out = [torch.full((n,), 99, dtype=torch.int32, device="cuda") for n in (experts + 1, experts, tokens * top_k, rows)]
    sgemm.route_sort(dev(ids), tokens, top_k, experts, align, *out, rows)
    return out, rows


# ---- without a device ------------------------------------------------------------------------------------------------

def test_capacity(sgemm):
    assert sgemm.route_capacity(10, 2, 4, 1) == 20
    assert sgemm.route_capacity(10, 2, 4, 128) == 20 + 4 * 127
    assert sgemm.route_capacity(1, 2, 64, 128) == 2 + 2 * 127
    for bad in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (1, 1, 1025, 1)):
        assert sgemm.route_capacity(*bad) == 0


def test_refusals(sgemm):
    l = sgemm.lib()

    def calls(name, ok, bad, large=()):
        f = getattr(l, name)
        for kw in bad:
            assert f(*{**ok, **kw}.values(), None) == pkg.INVALID_ARGUMENT, (name, kw)
        for kw in large:
            assert f(*{**ok, **kw}.values(), None) == pkg.UNSUPPORTED_SIZE, (name, kw)

    calls("b200_sgemm_route_sort", dict(ids=256, tokens=4, top_k=2, experts=8, align=128, off=256, cnt=256, sr=256, rs=256, rows=2000),
          [dict(ids=None), dict(off=None), dict(cnt=None), dict(sr=None), dict(rs=None), dict(tokens=0), dict(top_k=0), dict(experts=0),
           dict(align=0), dict(rows=8), dict(rows=8 + 8 * 127 - 1), dict(ids=2), dict(off=2), dict(cnt=2), dict(sr=2), dict(rs=2)],
          [dict(experts=1025), dict(tokens=1 << 31), dict(tokens=1 << 20, top_k=1 << 11), dict(rows=1 << 31)])
    calls("b200_sgemm_route_dispatch", dict(type=0, X=256, tokens=4, width=8, ldx=0, sr=256, top_k=2, Xs=256, rows=9, lds=0),
          [dict(type=3), dict(X=None), dict(tokens=0), dict(width=0), dict(ldx=7), dict(sr=None), dict(top_k=0), dict(Xs=None),
           dict(rows=0), dict(lds=7), dict(X=258), dict(Xs=258), dict(sr=2)],
          [dict(tokens=1 << 31), dict(width=1 << 31), dict(ldx=1 << 31), dict(rows=1 << 31)])
    calls("b200_sgemm_route_combine", dict(type=2, Y=256, rows=9, width=8, ldy=0, sr=256, tokens=4, top_k=2, w=None, out=256, ldo=0),
          [dict(type=-1), dict(Y=None), dict(rows=0), dict(width=0), dict(ldy=7), dict(sr=None), dict(tokens=0), dict(top_k=0),
           dict(out=None), dict(ldo=7), dict(Y=257), dict(out=257), dict(w=2), dict(sr=2)],
          [dict(tokens=1 << 31), dict(ldo=1 << 31)])
    calls("b200_sgemm_route_combine_backward",
          dict(type=0, dout=256, ldo=0, Y=256, rows=9, width=8, ldy=0, sr=256, tokens=4, top_k=2, w=256, dY=256, lddy=0, dw=256),
          [dict(type=3), dict(dout=None), dict(ldo=7), dict(Y=None), dict(rows=0), dict(width=0), dict(ldy=7), dict(sr=None),
           dict(tokens=0), dict(top_k=0), dict(dY=None, dw=None), dict(lddy=7), dict(dout=258), dict(Y=258), dict(dY=258), dict(w=2),
           dict(dw=2)],
          [dict(tokens=1 << 31), dict(lddy=1 << 31)])


# ---- sorting ---------------------------------------------------------------------------------------------------------

@gpu
@pytest.mark.parametrize("tokens,top_k,experts", [(1, 1, 1), (1, 8, 64), (7, 3, 5), (64, 8, 128), (700, 4, 33), (4097, 1, 256), (5000, 3, 1024),
                                                  (20000, 2, 16), (3001, 11, 7)])
@pytest.mark.parametrize("align", [1, 8, 128])
def test_sort(sgemm, tokens, top_k, experts, align):
    r = np.random.default_rng(tokens + experts)
    ids = np.minimum(r.integers(-1, experts + 2, (tokens, top_k)), r.integers(0, experts + 2, (tokens, top_k))).astype(np.int32)
    got, rows = run_sort(sgemm, ids, experts, align, extra=tokens % 3)
    for g, w in zip(got, sort_reference(ids, experts, align, rows)):
        assert np.array_equal(g.cpu().numpy(), w)


@gpu
def test_sort_all_to_one_and_none(sgemm):
    for ids in (np.full((6000, 3), 4, np.int32), np.full((300, 2), -1, np.int32), np.full((5, 2), 2 ** 31 - 1, np.int32)):
        got, rows = run_sort(sgemm, ids, 9, 128)
        for g, w in zip(got, sort_reference(ids, 9, 128, rows)):
            assert np.array_equal(g.cpu().numpy(), w)


@gpu
def test_sort_from_several_threads(sgemm):
    """Calls that need different amounts of shared memory, at once from four threads on streams of their own."""
    r = np.random.default_rng(5)
    cases = []
    for experts in (1024, 450, 700, 3):
        ids = r.integers(0, experts, (16384, 2)).astype(np.int32)
        out, rows = run_sort(sgemm, ids, experts, 8)
        cases.append((dev(ids), experts, out, rows, sort_reference(ids, experts, 8, rows), torch.cuda.Stream()))
        for o in out:
            o.fill_(99)
    torch.cuda.synchronize()

    def work(ids, experts, out, rows, want, stream):
        for _ in range(500):
            sgemm.route_sort(ids, 16384, 2, experts, 8, *out, rows, stream=stream)

    with ThreadPoolExecutor(len(cases)) as pool:
        for done in [pool.submit(work, *c) for c in cases]:
            done.result()
    torch.cuda.synchronize()
    for _, _, out, _, want, _ in cases:
        for g, w in zip(out, want):
            assert np.array_equal(g.cpu().numpy(), w)


# ---- rows there and back ---------------------------------------------------------------------------------------------

def case(tokens, top_k, width, dtype, seed, pad=0, rows=None):
    """Random rows for the slots, some dropped (two of them by a row that is not there), and leading dimensions."""
    r = np.random.default_rng(seed)
    rows = rows or tokens * top_k + 5
    slot_row = r.permutation(rows)[:tokens * top_k].astype(np.int32)
    slot_row[r.random(slot_row.size) < 0.2] = -1
    slot_row[0] = rows
    new = lambda n: torch.from_numpy(r.standard_normal((n, width + pad))).to(TYPES[dtype])  # noqa: E731
    return r, slot_row, rows, new


SHAPES = [(1, 1, 1), (5, 3, 33), (64, 8, 256), (100, 2, 1030), (33, 12, 4096), (300, 4, 8)]


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("pad", [0, 1, 8])
@pytest.mark.parametrize("tokens,top_k,width", SHAPES)
def test_dispatch_and_combine(sgemm, dtype, pad, tokens, top_k, width):
    r, slot_row, rows, new = case(tokens, top_k, width, dtype, width, pad)
    kept = (slot_row >= 0) & (slot_row < rows)
    token = np.arange(slot_row.size) // top_k
    ld = width + pad
    x, y = new(tokens), new(rows)
    xs = torch.full((rows, ld), 5.0, dtype=TYPES[dtype], device="cuda")
    sgemm.route_dispatch(pkg.m_type[dtype], x.cuda(), tokens, width, dev(slot_row), top_k, xs, rows, ldx=ld, lds=ld)
    want = torch.full((rows, ld), 5.0, dtype=TYPES[dtype])
    want[slot_row[kept], :width] = x[token[kept], :width]
    assert torch.equal(xs.cpu(), want)
    for weighted in (True, False):
        w = r.standard_normal((tokens, top_k)).astype(np.float32)
        out = torch.full((tokens, ld), 5.0, dtype=TYPES[dtype], device="cuda")
        sgemm.route_combine(pkg.m_type[dtype], y.cuda(), rows, width, dev(slot_row), tokens, top_k, out,
                            weights=dev(w) if weighted else None, ldy=ld, ldo=ld)
        assert (out[:, width:] == 5).all()
        terms = np.zeros((tokens, top_k, width))
        terms.reshape(-1, width)[kept] = y[slot_row[kept], :width].double().numpy()
        if weighted:
            terms *= w[..., None].astype(np.float64)
        exact = terms.sum(1)
        # every fused multiply-add rounds a partial sum by at most 2^-24 of the magnitudes; the result is rounded once
        bound = np.abs(terms).sum(1) * top_k * 2.0 ** -24 + np.abs(exact) * ref.TYPE_EPS[dtype] / 2 + (2.0 ** -25 if dtype == "f16" else 0)
        assert (np.abs(out[:, :width].double().cpu().numpy() - exact) <= bound * (1 + 2.0 ** -20) + 1e-300).all()


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("pad", [0, 1])
@pytest.mark.parametrize("tokens,top_k,width", SHAPES)
def test_combine_backward(sgemm, dtype, pad, tokens, top_k, width):
    r, slot_row, rows, new = case(tokens, top_k, width, dtype, width + 1, pad)
    kept = (slot_row >= 0) & (slot_row < rows)
    token = np.arange(slot_row.size) // top_k
    ld = width + pad
    dout, y = new(tokens), new(rows)
    w = r.standard_normal(slot_row.size).astype(np.float32)
    results = {}
    for what in ("both", "dy", "dw", "unweighted"):
        dy = torch.full((rows, ld), 5.0, dtype=TYPES[dtype], device="cuda") if what != "dw" else None
        dw = torch.full((slot_row.size,), 5.0, device="cuda") if what != "dy" else None
        sgemm.route_combine_backward(pkg.m_type[dtype], dout.cuda(), y.cuda() if dw is not None else None, rows, width, dev(slot_row),
                                     tokens, top_k, dev(w) if what != "unweighted" else None, dy, dw, ldo=ld, ldy=ld, lddy=ld)
        results[what] = dy, dw
    assert torch.equal(results["both"][0], results["dy"][0]) and torch.equal(results["both"][1], results["dw"][1])
    for what, weight in (("both", w), ("unweighted", np.ones_like(w))):
        dy, dw = (v.double().cpu().numpy() for v in results[what])
        g = dout[:, :width].double().numpy()[token]
        want = np.full((rows, ld), 5.0)
        want[slot_row[kept], :width] = weight[kept, None].astype(np.float64) * g[kept]
        bound = np.abs(want) * (2.0 ** -24 + ref.TYPE_EPS[dtype] / 2 * (1 + 2.0 ** -20)) + (2.0 ** -25 if dtype == "f16" else 0)
        assert (np.abs(dy - want) <= bound).all()
        terms = np.zeros((slot_row.size, width))
        terms[kept] = y[slot_row[kept], :width].double().numpy() * g[kept]
        # a partial sum has at most width / 256 + 13 terms on its way: each addition 2^-24 of the magnitudes
        steps = -(-width // 256) + 13 + 8
        assert (np.abs(dw - terms.sum(1)) <= np.abs(terms).sum(1) * steps * 2.0 ** -24 + 1e-300).all()
        assert (dw[~kept] == 0).all()


@gpu
def test_leading_dimensions_beyond_32_bits(sgemm):
    tokens, top_k, width, ld = 1100, 2, 64, 1 << 20
    rows, t = tokens * top_k, pkg.m_type.bf16
    slot_row = torch.randperm(rows, device="cuda").to(torch.int32)
    token = torch.arange(rows, device="cuda") // top_k
    x, w = torch.randn(tokens, width, device="cuda").bfloat16(), torch.rand(tokens, top_k, device="cuda")
    big = torch.empty(rows, ld, dtype=torch.bfloat16, device="cuda")
    sgemm.route_dispatch(t, x, tokens, width, slot_row, top_k, big, rows, lds=ld)
    y = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    y[slot_row.long()] = x[token]
    assert torch.equal(big[:, :width], y)
    outs = [torch.empty(tokens, width, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    sgemm.route_combine(t, big, rows, width, slot_row, tokens, top_k, outs[0], weights=w, ldy=ld)
    sgemm.route_combine(t, y, rows, width, slot_row, tokens, top_k, outs[1], weights=w)
    assert torch.equal(*outs)
    dw, dw_big = torch.empty_like(w), torch.empty_like(w)
    dy = torch.empty_like(y)
    sgemm.route_combine_backward(t, x, y, rows, width, slot_row, tokens, top_k, w, dy, dw)
    sgemm.route_combine_backward(t, x, big, rows, width, slot_row, tokens, top_k, w, None, dw_big, ldy=ld)
    assert torch.equal(dw, dw_big)
    sgemm.route_combine_backward(t, x, None, rows, width, slot_row, tokens, top_k, w, big, None, lddy=ld)
    assert torch.equal(big[:, :width], dy)


@gpu
def test_gradients_against_differences(sgemm):
    """The two gradients of combine, and of dispatch, against central differences of the forward pass (which is linear in
    each argument, so differences are exact up to rounding)."""
    tokens, top_k, width, experts = 6, 3, 40, 4
    r = np.random.default_rng(5)
    ids = r.integers(-1, experts, (tokens, top_k)).astype(np.int32)
    (_, _, slot_row, _), rows = run_sort(sgemm, ids, experts, 8)
    f32 = pkg.m_type.f32
    x, y, cot, cots = (torch.randn(n, width, device="cuda") for n in (tokens, rows, tokens, rows))
    w = torch.randn(tokens, top_k, device="cuda")

    def combine(y, w):
        out = torch.empty(tokens, width, device="cuda")
        sgemm.route_combine(f32, y, rows, width, slot_row, tokens, top_k, out, weights=w)
        return (out.double() * cot.double()).sum().item()

    def dispatch(x):
        xs = torch.zeros(rows, width, device="cuda")
        sgemm.route_dispatch(f32, x, tokens, width, slot_row, top_k, xs, rows)
        return (xs.double() * cots.double()).sum().item()

    dy, dw, dx = torch.zeros_like(y), torch.empty_like(w), torch.empty_like(x)
    sgemm.route_combine_backward(f32, cot, y, rows, width, slot_row, tokens, top_k, w, dy, dw)
    sgemm.route_combine(f32, cots, rows, width, slot_row, tokens, top_k, dx)
    for grad, value, f in ((dy, y, lambda v: combine(v, w)), (dw, w, lambda v: combine(y, v)), (dx, x, dispatch)):
        for _ in range(5):
            d = torch.randn_like(value)
            diff = (f(value + d) - f(value - d)) / 2
            # sums of at most rows * width products of numbers below 8 in magnitude, rounded in FP32 on the way
            assert abs(diff - (grad.double() * d.double()).sum().item()) <= rows * width * 64 * 2.0 ** -23


@gpu
@pytest.mark.parametrize("fmt", [ref.NVFP4, ref.MXFP4], ids=["nvfp4", "mxfp4"])
def test_experts_from_tokens_to_tokens(sgemm, fmt):
    """A layer of experts as a model runs it, captured into a graph: sort, quantise the sorted tokens, the experts'
    product, back with weights; a second routing is replayed through the same graph."""
    tokens, top_k, experts, K, N = 50, 3, 6, 160, 200
    rows = sgemm.route_capacity(tokens, top_k, experts, 128)
    r = np.random.default_rng(8)
    weights64, codes, scales = [], [], []
    for e in range(experts):
        code, byte = ref.quantize(fmt, r.standard_normal((N, K)))
        c, s = ref.pack(fmt, code, byte)
        codes.append(c), scales.append(s), weights64.append(ref.values(fmt, code, byte))
    b = dev(np.concatenate(codes)), dev(np.concatenate(scales))
    ids = torch.empty(tokens, top_k, dtype=torch.int32, device="cuda")
    x, w = torch.empty(tokens, K, device="cuda"), torch.empty(tokens, top_k, device="cuda")
    new = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
    offsets, counts, slot_row, row_slot = new(experts + 1), new(experts), new(tokens * top_k), new(rows)
    nc, ns = sgemm.mx4_sizes(fmt, rows, K)
    a = torch.empty(nc, dtype=torch.uint8, device="cuda"), torch.empty(ns, dtype=torch.uint8, device="cuda")
    y, out = torch.empty(rows, N, device="cuda"), torch.empty(tokens, N, device="cuda")
    f32 = pkg.m_type.f32

    def layer():
        sgemm.route_sort(ids, tokens, top_k, experts, 128, offsets, counts, slot_row, row_slot, rows)
        sgemm.mx4_quantize(fmt, 0, f32, x, rows, K, *a, row_index=row_slot, source_rows=tokens, index_div=top_k)
        sgemm.gemm_mx4_grouped(fmt, f32, y, *a, *b, rows, N, K, experts, offsets, counts, used_rows=tokens * top_k)
        sgemm.route_combine(f32, y, rows, N, slot_row, tokens, top_k, out, weights=w)

    def fill(seed):
        q = np.random.default_rng(seed)
        i = q.integers(-1, experts, (tokens, top_k)).astype(np.int32)
        xv, wv = q.standard_normal((tokens, K)).astype(np.float32), q.random((tokens, top_k)).astype(np.float32)
        ids.copy_(dev(i)), x.copy_(dev(xv)), w.copy_(dev(wv))
        xq = ref.values(fmt, *ref.quantize(fmt, xv.astype(np.float64)))
        want, size = np.zeros((tokens, N)), np.zeros((tokens, N))
        for t in range(tokens):
            for j in range(top_k):
                if i[t, j] >= 0:
                    want[t] += wv[t, j] * (weights64[i[t, j]] @ xq[t])
                    size[t] += wv[t, j] * (np.abs(weights64[i[t, j]]) @ np.abs(xq[t]))
        return want, size

    def close(want, size):  # the product's bound for K <= 512 (8 instructions), then top_k additions
        assert (np.abs(out.double().cpu().numpy() - want) <= size * (8 * 2.0 ** -22 + (top_k + 3) * 2.0 ** -24)).all()

    want = fill(1)
    layer()
    close(*want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for seed in (2, 3):
        want = fill(seed)
        graph.replay()
        close(*want)
    assert sgemm.mx4_device_status() == 0
