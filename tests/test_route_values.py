"""Routing of values that are not finite: rows that no kept slot names are not read, those that one names come through."""
import numpy as np
import pytest

import rocm_sgemm_b200 as pkg

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BITS = {"f32": torch.int32, "f16": torch.int16, "bf16": torch.int16}


@gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("tokens,top_k,width", [(6, 3, 40), (6, 3, 33), (3000, 2, 512), (3000, 5, 65), (1, 40, 24)])
def test_values_that_are_not_finite(sgemm, dtype, tokens, top_k, width):
    t, r = pkg.m_type[dtype], np.random.default_rng(width)
    slots, rows = tokens * top_k, tokens * top_k + 9
    slot_row = r.permutation(rows)[:slots].astype(np.int32)
    dropped = r.random(slots) < 0.3
    slot_row[dropped] = r.choice([-1, rows, 2 ** 31 - 1, -2 ** 31], dropped.sum())
    kept, token = np.nonzero(~dropped)[0], np.arange(slots) // top_k
    at = torch.from_numpy(slot_row).cuda()
    new = lambda n: torch.from_numpy(r.standard_normal((n, width))).to(TYPES[dtype])  # noqa: E731

    # dispatch copies bits: infinities, NaN of either sign, -0
    x = new(tokens)
    x.view(-1)[::7], x.view(-1)[3::11], x.view(-1)[5::13], x.view(-1)[1::17] = float("inf"), float("nan"), -float("nan"), -0.0
    xs = torch.full((rows, width), 5.0, dtype=TYPES[dtype], device="cuda")
    sgemm.route_dispatch(t, x.cuda(), tokens, width, at, top_k, xs, rows)
    want = torch.full((rows, width), 5.0, dtype=TYPES[dtype])
    want[slot_row[kept]] = x[token[kept]]
    assert torch.equal(xs.cpu().view(BITS[dtype]), want.view(BITS[dtype]))

    # rows without a kept slot are NaN, as are the weights of dropped slots: neither is seen
    y, w = new(rows), r.standard_normal(slots).astype(np.float32)
    named = np.zeros(rows, bool)
    named[slot_row[kept]] = True
    y[~named] = float("nan")
    w[dropped] = np.nan
    wt, out = torch.from_numpy(w).cuda(), torch.empty(tokens, width, dtype=TYPES[dtype], device="cuda")
    for weights in (wt, None):
        sgemm.route_combine(t, y.cuda(), rows, width, at, tokens, top_k, out, weights=weights)
        assert torch.isfinite(out).all()
    dout = new(tokens)
    dy, dw = torch.full((rows, width), 5.0, dtype=TYPES[dtype], device="cuda"), torch.empty(slots, device="cuda")
    sgemm.route_combine_backward(t, dout.cuda(), y.cuda(), rows, width, at, tokens, top_k, wt, dy, dw)
    assert torch.isfinite(dy).all() and (dy[torch.from_numpy(~named).cuda()] == 5).all()
    assert torch.isfinite(dw).all() and not dw[torch.from_numpy(dropped).cuda()].any()

    # an infinity in a row that a slot names reaches that token, that column and that weight, and nothing else
    s = kept[len(kept) // 2]
    y[slot_row[s], width // 2] = float("inf")
    w[s] = 0.5
    wt = torch.from_numpy(w).cuda()
    sgemm.route_combine(t, y.cuda(), rows, width, at, tokens, top_k, out, weights=wt)
    hit = torch.zeros(tokens, width, dtype=torch.bool)
    hit[token[s], width // 2] = True
    assert torch.equal(torch.isinf(out).cpu(), hit) and not torch.isnan(out).any()
    dout[token[s], width // 2] = -2.0
    sgemm.route_combine_backward(t, dout.cuda(), y.cuda(), rows, width, at, tokens, top_k, wt, dy, dw)
    hit = torch.zeros(slots, dtype=torch.bool)
    hit[s] = True
    assert torch.equal(torch.isinf(dw).cpu(), hit) and dw[s] == -float("inf") and torch.isfinite(dy).all()
