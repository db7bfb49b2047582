"""Operators of the 4-bit product path, in plain form and through the library.

Four operators, as a program that serves or trains a model with 4-bit weights uses them:

  quantise   a matrix to microscaled 4-bit floating point, and back to the values it stands for
  product    of two such matrices, C = alpha * global_a * global_b * A B
  experts    the same product for rows sorted by expert, each expert with weights of its own
  routing    tokens sorted by expert and back with weights applied, and the gradients of both

Formats.  "nvfp4": e2m1 codes, one e4m3 scale per 16 values of k, times one FP32 scale g for the matrix.
"mxfp4": e2m1 codes, one power of two (e8m0) per 32 values of k.  Codes lie as rows of ceil(K/32)*16 bytes, the lower
k in the lower half of a byte; scales as tiles of 128 rows x 4 scales, 512 bytes each (row r, scale c at
(r % 32) * 16 + r % 128 // 32 * 4 + c % 4), the tiles of one band of 128 rows one after the other.
"""
import math

import numpy as np
import torch

own = False

BLOCK = {"nvfp4": 16, "mxfp4": 32}
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # what the codes 0..7 stand for; 8..15 are their negatives
ALIGN = 128  # the first row of each expert is a multiple of this


# ---- cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # activations of a batch of 16 tokens on their way into a 4-bit product, one token each
        {"name": "quantise 16 tokens", "op": "quantise", "fmt": "nvfp4", "layout": 0, "type": "bf16", "rows": 16, "k": 8192},
        # weights when they are loaded, or activations of a long prefill
        {"name": "quantise 16384x8192", "op": "quantise", "fmt": "nvfp4", "layout": 0, "type": "bf16", "rows": 16384, "k": 8192},
        # training quantises the same matrix along its other axis too; no size fits a tile
        {"name": "quantise columns 4097x2050", "op": "quantise", "fmt": "mxfp4", "layout": 1, "type": "f32", "rows": 4097, "k": 2050},
        # one token against a weight matrix: the bytes of the weights are all there is
        {"name": "product 1x16384x4096", "op": "product", "fmt": "nvfp4", "layout_c": 0, "type": "bf16", "m": 1, "n": 16384, "k": 4096},
        # a small ragged product, K not a multiple of any block
        {"name": "product 1000x1030x515", "op": "product", "fmt": "mxfp4", "layout_c": 0, "type": "f32", "m": 1000, "n": 1030, "k": 515},
        # the headline cube of this library, FP32 result, column-major
        {"name": "product 4096 cube f32", "op": "product", "fmt": "nvfp4", "layout_c": 1, "type": "f32", "m": 4096, "n": 4096, "k": 4096},
        # a long prefill through a wide layer
        {"name": "product 8192 cube", "op": "product", "fmt": "nvfp4", "layout_c": 0, "type": "bf16", "m": 8192, "n": 8192, "k": 8192},
        # a few tokens in flight: most experts hold a handful of rows or none
        {"name": "experts 8 tokens", "op": "experts", "fmt": "nvfp4", "type": "bf16", "tokens": 8, "top_k": 8, "experts": 64, "n": 2048, "k": 4096},
        # a prefill: every expert holds many rows, unevenly
        {"name": "experts 8192 tokens", "op": "experts", "fmt": "mxfp4", "type": "bf16", "tokens": 8192, "top_k": 4, "experts": 32, "n": 4096, "k": 2048},
        # routing of a decode step
        {"name": "routing 64 tokens", "op": "routing", "pass": "forward", "type": "bf16", "tokens": 64, "top_k": 8, "experts": 128, "width": 4096, "dropped": 0.0},
        # routing of a prefill
        {"name": "routing 8192 tokens", "op": "routing", "pass": "forward", "type": "bf16", "tokens": 8192, "top_k": 4, "experts": 32, "width": 4096, "dropped": 0.05},
        # the gradients of a training step, some tokens over their expert's capacity
        {"name": "routing gradient 8191 tokens", "op": "routing", "pass": "backward", "type": "f32", "tokens": 8191, "top_k": 2, "experts": 16, "width": 2048, "dropped": 0.1},
    ]


def draw(rng):
    def spread(lo, hi):  # even over the logarithm; every other one falls on a multiple of 16 where there is room
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        return max(lo, v // 16 * 16) if v >= 64 and rng.random() < 0.5 else v

    op = rng.choice(["quantise", "product", "product", "experts", "routing"])
    if op == "quantise":
        rows = spread(1, 16384)
        return {"op": op, "fmt": rng.choice(sorted(BLOCK)), "layout": rng.choice([0, 1]), "type": rng.choice(sorted(TYPES)),
                "rows": rows, "k": spread(1, 8192)}
    if op == "product":
        return {"op": op, "fmt": rng.choice(sorted(BLOCK)), "layout_c": rng.choice([0, 0, 1]), "type": rng.choice(sorted(TYPES)),
                "m": spread(1, 8192), "n": spread(64, 8192), "k": spread(16, 8192)}
    if op == "experts":
        return {"op": op, "fmt": rng.choice(sorted(BLOCK)), "type": rng.choice(sorted(TYPES)), "tokens": spread(1, 4096),
                "top_k": rng.choice([1, 2, 4, 8]), "experts": rng.choice([8, 9, 16, 32]), "n": spread(64, 4096), "k": spread(64, 2048)}
    return {"op": op, "pass": rng.choice(["forward", "backward"]), "type": rng.choice(sorted(TYPES)), "tokens": spread(1, 8192),
            "top_k": rng.choice([1, 2, 3, 4, 8]), "experts": rng.choice([4, 8, 33, 64, 256]), "width": spread(8, 2048),
            "dropped": rng.choice([0.0, 0.1])}


def capacity(case):
    """Rows of the sorted buffers: every slot, and what rounding each expert up to ALIGN rows can add."""
    slots = case["tokens"] * case["top_k"]
    return slots + min(slots, case["experts"]) * (ALIGN - 1)


def quantised_bytes(fmt, rows, k):
    return rows * k / 2 + rows * -(-k // BLOCK[fmt])


def work(case):
    op = case["op"]
    if op == "quantise":
        size = TYPES[case["type"]].itemsize
        n = case["rows"] * case["k"]
        # the matrix in, codes and scales out; codes and scales in, FP32 values out
        return {"bytes": n * size + 2 * quantised_bytes(case["fmt"], case["rows"], case["k"]) + 4 * n, "flops": 4 * n}
    size = TYPES[case["type"]].itemsize
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": quantised_bytes(case["fmt"], m, k) + quantised_bytes(case["fmt"], n, k) + m * n * size, "flops": 2 * m * n * k}
    slots = case["tokens"] * case["top_k"]
    if op == "experts":
        used = min(slots, case["experts"] * (1 - (1 - 1 / case["experts"]) ** slots))  # experts that hold a row, on average
        return {"bytes": quantised_bytes(case["fmt"], slots, case["k"]) + used * quantised_bytes(case["fmt"], case["n"], case["k"])
                + slots * case["n"] * size, "flops": 2 * slots * case["n"] * case["k"]}
    tokens, width = case["tokens"], case["width"]
    if case["pass"] == "forward":  # ids in, order out; X in, its rows out; the experts' rows in, their sum out
        return {"bytes": slots * 12 + slots * 4 + 2 * (tokens + slots) * width * size, "flops": 2 * slots * width}
    # d(out), Y and weights in, dY and d(weights) out; d(rows) in, dX out
    return {"bytes": slots * 12 + (2 * tokens + 3 * slots) * width * size, "flops": 4 * slots * width}


# ---- what a program has in hand --------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"quantise": _prepare_quantise, "product": _prepare_product, "experts": _prepare_experts,
            "routing": _prepare_routing}[case["op"]](case, g)


def _normal(g, *shape, scale=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale


def _activations(g, rows, k):
    """Rows of a residual stream: normal, with a few channels tens of times larger."""
    x = _normal(g, rows, k)
    loud = torch.rand(k, generator=g, device="cuda") < 0.01
    return x * torch.where(loud, 20.0, 1.0)


def _global_scale(fmt, x):
    """The matrix's own scale, which puts its largest value at the top of both ranges; mxfp4 has none."""
    if fmt != "nvfp4":
        return None
    return (x.abs().amax().float() / (6 * 448)).reshape(1)


def _prepare_quantise(case, g):
    rows, k, dtype = case["rows"], case["k"], TYPES[case["type"]]
    x = _activations(g, rows, k).to(dtype)
    state = {"case": case, "x": x if case["layout"] == 0 else x.T.contiguous(), "g": _global_scale(case["fmt"], x)}
    code_bytes, scale_bytes = _sizes(case["fmt"], rows, k)
    state["codes"] = torch.empty(code_bytes, dtype=torch.uint8, device="cuda")
    state["scales"] = torch.empty(scale_bytes, dtype=torch.uint8, device="cuda")
    state["out"] = torch.empty(rows, k, dtype=torch.float32, device="cuda")
    return state


def _sizes(fmt, rows, k):
    return rows * (-(-k // 32) * 16), -(-rows // 128) * -(-k // (4 * BLOCK[fmt])) * 512


def _quantised(fmt, x):
    """(codes, scales, g) of x [rows, k] as they are stored."""
    g = _global_scale(fmt, x)
    levels, scale_bytes = _quantise_plain(fmt, x, g)
    return _pack_codes(levels), _tile_scales(scale_bytes), g


def _prepare_product(case, g):
    m, n, k = case["m"], case["n"], case["k"]
    a, b = _quantised(case["fmt"], _activations(g, m, k)), _quantised(case["fmt"], _normal(g, n, k, scale=0.02))
    shape = (m, n) if case["layout_c"] == 0 else (n, m)
    return {"case": case, "a": a, "b": b, "c": torch.empty(shape, dtype=TYPES[case["type"]], device="cuda")}


def _expert_ids(case, g):
    """The experts each token picks, different ones and some experts more often than others; -1 where a slot is dropped."""
    tokens, top_k, experts = case["tokens"], case["top_k"], case["experts"]
    liking = _normal(g, experts, scale=0.5) + _normal(g, tokens, experts)
    if top_k <= experts:
        ids = liking.topk(top_k, dim=1).indices.to(torch.int32)
    else:
        ids = torch.randint(experts, (tokens, top_k), generator=g, device="cuda", dtype=torch.int32)
    drop = torch.rand(tokens, top_k, generator=g, device="cuda") < case.get("dropped", 0.0)
    return torch.where(drop, torch.full_like(ids, -1), ids)


def _prepare_experts(case, g):
    experts, n, k, rows = case["experts"], case["n"], case["k"], capacity(case)
    ids = _expert_ids(case, g)
    offsets, counts, slot_row, row_slot = _sort_plain(ids, experts, rows)
    x = _activations(g, case["tokens"], k)
    sorted_x = torch.where((row_slot >= 0)[:, None], x[row_slot.clamp(min=0).long() // case["top_k"]], 0.0)
    a = _quantised(case["fmt"], sorted_x)
    del sorted_x
    parts = [_quantised(case["fmt"], _normal(g, n, k, scale=0.02)) for _ in range(experts)]
    codes, scales = torch.stack([p[0] for p in parts]), torch.stack([p[1] for p in parts])
    gb = torch.cat([p[2] for p in parts]) if case["fmt"] == "nvfp4" else None
    return {"case": case, "a": a, "b": (codes, scales, gb), "offsets": offsets, "counts": counts,
            "most": int(counts.max()), "c": torch.zeros(rows, n, dtype=TYPES[case["type"]], device="cuda")}


def _prepare_routing(case, g):
    tokens, top_k, width, rows, dtype = case["tokens"], case["top_k"], case["width"], capacity(case), TYPES[case["type"]]
    ids = _expert_ids(case, g)
    weights = torch.softmax(_normal(g, tokens, top_k), dim=1)
    state = {"case": case, "ids": ids, "weights": weights, "rows": rows, "y": _normal(g, rows, width).to(dtype)}
    if case["pass"] == "forward":
        new = lambda n: torch.empty(n, dtype=torch.int32, device="cuda")  # noqa: E731
        state |= {"x": _activations(g, tokens, width).to(dtype), "offsets": new(case["experts"] + 1), "counts": new(case["experts"]),
                  "slot_row": new(tokens * top_k), "row_slot": new(rows), "xs": torch.zeros(rows, width, dtype=dtype, device="cuda"),
                  "out": torch.empty(tokens, width, dtype=dtype, device="cuda")}
    else:
        _, _, slot_row, _ = _sort_plain(ids, case["experts"], rows)
        state |= {"slot_row": slot_row, "dout": _normal(g, tokens, width).to(dtype), "dxs": _normal(g, rows, width).to(dtype),
                  "dx": torch.empty(tokens, width, dtype=dtype, device="cuda"), "dy": torch.zeros(rows, width, dtype=dtype, device="cuda"),
                  "dw": torch.empty(tokens, top_k, dtype=torch.float32, device="cuda")}
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        return {"quantise": _own_quantise, "product": _own_product, "experts": _own_experts, "routing": _own_routing}[op](state)
    return {"quantise": _run_quantise, "product": _run_product, "experts": _run_experts, "routing": _run_routing}[op](state)


def _own_quantise(s):
    import rocm_sgemm_b200 as sg
    c = s["case"]
    fmt, dtype = sg.mx4_format[c["fmt"]], sg.m_type[c["type"]]
    sg.mx4_quantize(fmt, c["layout"], dtype, s["x"], c["rows"], c["k"], s["codes"], s["scales"], global_scale=s["g"])
    sg.mx4_dequantize(fmt, sg.m_type.f32, s["codes"], s["scales"], c["rows"], c["k"], s["out"], global_scale=s["g"])
    return s["out"]


def _own_product(s):
    import rocm_sgemm_b200 as sg
    c, a, b = s["case"], s["a"], s["b"]
    sg.gemm_mx4(sg.mx4_format[c["fmt"]], c["layout_c"], sg.m_type[c["type"]], s["c"], a[0], a[1], b[0], b[1], c["m"], c["n"], c["k"],
                global_a=a[2], global_b=b[2])
    return s["c"]


def _own_experts(s):
    import rocm_sgemm_b200 as sg
    c, a, b = s["case"], s["a"], s["b"]
    sg.gemm_mx4_grouped(sg.mx4_format[c["fmt"]], sg.m_type[c["type"]], s["c"], a[0], a[1], b[0], b[1], s["c"].shape[0], c["n"], c["k"],
                        c["experts"], s["offsets"], s["counts"], used_rows=c["tokens"] * c["top_k"], global_a=a[2], global_b=b[2])
    return s["c"]


def _own_routing(s):
    import rocm_sgemm_b200 as sg
    c, dtype = s["case"], sg.m_type[s["case"]["type"]]
    tokens, top_k, width, rows = c["tokens"], c["top_k"], c["width"], s["rows"]
    if c["pass"] == "forward":
        sg.route_sort(s["ids"], tokens, top_k, c["experts"], ALIGN, s["offsets"], s["counts"], s["slot_row"], s["row_slot"], rows)
        sg.route_dispatch(dtype, s["x"], tokens, width, s["slot_row"], top_k, s["xs"], rows)
        sg.route_combine(dtype, s["y"], rows, width, s["slot_row"], tokens, top_k, s["out"], weights=s["weights"])
        return [s["offsets"], s["counts"], s["slot_row"], s["row_slot"], s["xs"], s["out"]]
    sg.route_combine(dtype, s["dxs"], rows, width, s["slot_row"], tokens, top_k, s["dx"])
    sg.route_combine_backward(dtype, s["dout"], s["y"], rows, width, s["slot_row"], tokens, top_k, s["weights"], s["dy"], s["dw"])
    return [s["dx"], s["dy"], s["dw"]]


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _power(e):
    return torch.ldexp(torch.ones_like(e, dtype=torch.float64), e)


def _quantise_plain(fmt, x, g):
    """Signed levels [rows, k] and the scales as bytes [rows, ceil(k / block)].  In 64 bits: a value on the border between
    two levels has to be seen to lie on it."""
    rows, k = x.shape
    block = BLOCK[fmt]
    x = torch.nn.functional.pad(x.double(), (0, -k % block)).view(rows, -1, block)
    amax = x.abs().amax(-1)
    if fmt == "mxfp4":  # the power of two that puts the largest value into [4, 8); codes saturate at 6
        e = (torch.frexp(amax).exponent - 3).clamp(-127, 127)
        e = torch.where(amax > 0, e, torch.full_like(e, -127))
        scale, byte = _power(e), e + 127
    else:
        q = amax / (6 * g.double())
        e = (torch.frexp(q).exponent - 1).clamp(min=-6)
        step = _power(e - 3)
        scale = (torch.round(q / step) * step).clamp(max=448.0)
        e = (torch.frexp(scale).exponent - 1).clamp(min=-6)
        low = (scale / _power(e - 3)).to(torch.int32)  # 8..15, or 0..7 below the smallest power of two
        byte = torch.where(low >= 8, (e + 7) * 8 + low - 8, low)
        scale = scale * g.double()
    y = x / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None]
    y = torch.where((scale > 0)[..., None], y, torch.zeros_like(y))
    size = y.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    levels = torch.round(y / step) * step  # ties to even, which is the even code too
    return levels.clamp(-6, 6).view(rows, -1)[:, :k].float(), byte.to(torch.uint8)


def _pack_codes(levels):
    rows, k = levels.shape
    size = torch.nn.functional.pad(levels, (0, -k % 32)).abs()
    code = (size * 2).to(torch.uint8)
    code = torch.where(size == 3, 5, torch.where(size == 4, 6, torch.where(size == 6, 7, code))).to(torch.uint8)
    code |= torch.nn.functional.pad(torch.signbit(levels), (0, -k % 32)).to(torch.uint8) << 3
    return code[:, 0::2] | code[:, 1::2] << 4


def _tile_scales(byte):
    rows, cols = byte.shape
    t = torch.nn.functional.pad(byte, (0, -cols % 4, 0, -rows % 128))
    return t.view(-1, 4, 32, t.shape[1] // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _unpack(fmt, codes, scales, rows, k, dtype=torch.float32):
    """The values that codes and scales stand for, without the matrix's scale; any leading dimensions."""
    lead = codes.shape[:-2]
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=dtype, device=codes.device)
    levels = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], -1).flatten(-2)[..., :k]
    cols = -(-k // BLOCK[fmt])
    t = scales.view(*lead, -(-rows // 128), -(-cols // 4), 32, 4, 4)
    t = t.movedim(-2, -4).movedim(-3, -2)  # band, quarter, column tile, row, scale -> band, quarter, row, column tile, scale
    byte = t.reshape(*lead, -(-rows // 128) * 128, -1)[..., :rows, :cols].int()
    if fmt == "mxfp4":
        scale = torch.ldexp(torch.ones_like(byte, dtype=dtype), byte - 127)
    else:
        e, low = byte >> 3, byte & 7
        scale = torch.ldexp(torch.where(e > 0, low + 8, low).to(dtype), e.clamp(min=1) - 10)
    return levels * scale.repeat_interleave(BLOCK[fmt], -1)[..., :k]


def _run_quantise(s):
    c = s["case"]
    x = s["x"] if c["layout"] == 0 else s["x"].T
    levels, byte = _quantise_plain(c["fmt"], x, s["g"])
    values = _unpack(c["fmt"], _pack_codes(levels), _tile_scales(byte), c["rows"], c["k"])
    return values if s["g"] is None else values * s["g"]


def _factor(a, b):
    return 1.0 if a[2] is None else a[2] * b[2]


def _run_product(s):
    c, a, b = s["case"], s["a"], s["b"]
    x, y = _unpack(c["fmt"], a[0], a[1], c["m"], c["k"]), _unpack(c["fmt"], b[0], b[1], c["n"], c["k"])
    r = (x @ y.T if c["layout_c"] == 0 else y @ x.T) * _factor(a, b)
    return r.to(TYPES[c["type"]])


def _grouped(s, dtype, product):
    """Rows sorted by expert times their expert's weights, by a batch padded to the largest expert."""
    c, a, b, rows = s["case"], s["a"], s["b"], s["c"].shape[0]
    x, w = _unpack(c["fmt"], a[0], a[1], rows, c["k"], dtype), _unpack(c["fmt"], b[0], b[1], c["n"], c["k"], dtype)
    at = s["offsets"][:-1, None].long() + torch.arange(max(s["most"], 1), device="cuda")
    r = product(x[at.clamp(max=rows - 1)], w)  # [experts, most, n]
    row = torch.arange(rows, device="cuda")
    e = (torch.searchsorted(s["offsets"].long(), row, right=True) - 1).clamp(max=c["experts"] - 1)
    place = row - s["offsets"][e].long()
    if a[2] is not None:
        r = r * (a[2].to(dtype) * b[2].to(dtype))[:, None, None]
    return torch.where((place < s["counts"][e])[:, None], r[e, place.clamp(max=r.shape[1] - 1)], 0.0)


def _run_experts(s):
    return _grouped(s, torch.float32, lambda x, w: x @ w.transpose(1, 2)).to(TYPES[s["case"]["type"]])


def _sort_plain(ids, experts, rows):
    """offsets [experts + 1], counts [experts], slot_row [slots], row_slot [rows]: slots in order within each expert."""
    flat = ids.reshape(-1).long()
    key = torch.where((flat >= 0) & (flat < experts), flat, torch.full_like(flat, experts))
    slots = key.numel()
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=ids.device).scatter_add_(0, key, torch.ones_like(key))
    ends = torch.cumsum(counts, 0)
    padded = torch.cumsum((counts[:experts] + ALIGN - 1) // ALIGN * ALIGN, 0)
    offsets = torch.cat([torch.zeros_like(padded[:1]), padded])
    order = torch.argsort(key, stable=True)
    by = key[order]
    place = torch.arange(slots, device=ids.device) - (ends - counts)[by]
    row = torch.where(by < experts, offsets[by] + place, torch.full_like(by, rows))
    row_slot = torch.full((rows + 1,), -1, dtype=torch.int32, device=ids.device).scatter_(0, row, order.int())[:rows]
    slot_row = torch.empty_like(row).scatter_(0, order, torch.where(row < rows, row, torch.full_like(row, -1)))
    return offsets.int(), counts[:experts].int(), slot_row.int(), row_slot


def _rows_of(s, y, slot_row, dtype):
    """y's row of each slot [tokens, top_k, width], zero where the slot is dropped."""
    at = slot_row.view(s["case"]["tokens"], s["case"]["top_k"]).long()
    return torch.where((at >= 0)[..., None], y[at.clamp(min=0)].to(dtype), 0.0)


def _run_routing(s):
    c, dtype = s["case"], TYPES[s["case"]["type"]]
    if c["pass"] == "forward":
        offsets, counts, slot_row, row_slot = _sort_plain(s["ids"], c["experts"], s["rows"])
        xs = torch.where((row_slot >= 0)[:, None], s["x"][row_slot.clamp(min=0).long() // c["top_k"]], torch.zeros((), dtype=dtype, device="cuda"))
        out = (_rows_of(s, s["y"], slot_row, torch.float32) * s["weights"][..., None]).sum(1)
        return [offsets, counts, slot_row, row_slot, xs, out.to(dtype)]
    dx = _rows_of(s, s["dxs"], s["slot_row"], torch.float32).sum(1).to(dtype)
    dout = s["dout"].float()
    dw = (_rows_of(s, s["y"], s["slot_row"], torch.float32) * dout[:, None]).sum(-1)
    at = s["slot_row"].long()
    dy = torch.zeros(s["rows"] + 1, c["width"], dtype=dtype, device="cuda")
    dy[torch.where(at >= 0, at, torch.full_like(at, s["rows"]))] = (s["weights"][..., None] * dout[:, None]).view(-1, c["width"]).to(dtype)
    return [dx, dy[:-1], dw]


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"quantise": _exact_quantise, "product": _exact_product, "experts": _exact_experts, "routing": _exact_routing}[case["op"]](s)


def _exact_quantise(s):
    """Every level and scale found by comparing with the midpoints between neighbours; a midpoint goes to the even one."""
    c = s["case"]
    x = (s["x"] if c["layout"] == 0 else s["x"].T).double()
    rows, k, block = c["rows"], c["k"], BLOCK[c["fmt"]]
    out = torch.empty(rows, k, dtype=torch.float64, device="cuda")
    levels = torch.tensor(LEVELS, dtype=torch.float64, device="cuda")
    if c["fmt"] == "nvfp4":
        scales = torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1],
                              dtype=torch.float64, device="cuda")
        g = s["g"].double()
    for r in range(0, rows, 2048):
        part = torch.nn.functional.pad(x[r:r + 2048], (0, -k % block)).reshape(-1, block)
        amax = part.abs().amax(1)
        if c["fmt"] == "nvfp4":
            scale = scales[_nearest(amax / (6 * g), scales)] * g
        else:
            scale = torch.exp2(torch.floor(torch.log2(amax.clamp(min=1e-300))) - 2).clamp(2.0 ** -127, 2.0 ** 127)
        y = torch.where(scale[:, None] > 0, part.abs() / scale[:, None].clamp(min=1e-300), 0.0)
        v = levels[_nearest(y, levels)] * scale[:, None] * torch.sign(part)
        out[r:r + 2048] = v.view(-1, v.numel() // min(2048, rows - r))[:, :k]
    return out


def _nearest(v, table):
    """Index of the nearest entry of an ascending table, midpoints to the even index."""
    mid = (table[1:] + table[:-1]) / 2
    below, upto = torch.bucketize(v, mid), torch.bucketize(v, mid, right=True)  # they differ where v is a midpoint
    return torch.where(below % 2 == 0, below, upto)


def _exact_product(s):
    c, a, b = s["case"], s["a"], s["b"]
    x, y = (_exact_values(c["fmt"], t, rows, c["k"]) for t, rows in ((a, c["m"]), (b, c["n"])))
    r = x @ y.T
    return r if c["layout_c"] == 0 else r.T.contiguous()


def _exact_values(fmt, t, rows, k):
    """Values with the matrix's scale, each scale byte looked up by the address the format gives it."""
    codes, scales, g = t
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64, device="cuda")
    kk = torch.arange(k, device="cuda")
    code = codes[:, kk // 2].int() >> (kk % 2 * 4) & 15
    r, c = torch.arange(rows, device="cuda")[:, None], torch.arange(-(-k // BLOCK[fmt]), device="cuda")[None]
    tile = r // 128 * -(-c.shape[1] // 4) + c // 4
    byte = scales[tile * 512 + r % 32 * 16 + r % 128 // 32 * 4 + c % 4].double()
    if fmt == "mxfp4":
        scale = torch.exp2(byte - 127)
    else:
        e, low = torch.floor(byte / 8), byte % 8
        scale = torch.where(e > 0, (1 + low / 8) * torch.exp2(e - 7), low * 2.0 ** -9) * g.double()
    return table[code.long()] * scale[:, kk // BLOCK[fmt]]


def _exact_experts(s):
    c, a, (codes, scales, gb), rows = s["case"], s["a"], s["b"], s["c"].shape[0]
    x = _exact_values(c["fmt"], a, rows, c["k"])
    out = torch.zeros(rows, c["n"], dtype=torch.float64, device="cuda")
    first, count = s["offsets"].tolist(), s["counts"].tolist()
    for e in range(c["experts"]):
        if count[e]:
            w = _exact_values(c["fmt"], (codes[e], scales[e], None if gb is None else gb[e]), c["n"], c["k"])
            out[first[e]:first[e] + count[e]] = x[first[e]:first[e] + count[e]] @ w.T
    return out


def _exact_routing(s):
    c = s["case"]
    tokens, top_k, width, experts = c["tokens"], c["top_k"], c["width"], c["experts"]
    ids = s["ids"].reshape(-1).cpu().numpy()
    kept = np.nonzero((ids >= 0) & (ids < experts))[0]
    by = kept[np.argsort(ids[kept], kind="stable")]  # slots in sorted order
    counts = np.bincount(ids[kept], minlength=experts)
    offsets = np.concatenate([[0], np.cumsum(-(-counts // ALIGN) * ALIGN)])
    row = offsets[ids[by]] + np.arange(by.size) - (np.cumsum(counts) - counts)[ids[by]]
    slot, row = (torch.from_numpy(np.ascontiguousarray(v)).cuda() for v in (by, row))
    token, weights = slot // top_k, s["weights"].double().reshape(-1)
    sums = lambda v: torch.zeros(tokens, width, dtype=torch.float64, device="cuda").index_add_(0, token, v)  # noqa: E731
    rows_of = lambda v: torch.zeros(s["rows"], width, dtype=torch.float64, device="cuda").index_copy_(0, row, v)  # noqa: E731
    y = s["y"].double()[row]
    if c["pass"] == "forward":
        return [None, None, None, None, rows_of(s["x"].double()[token]), sums(y * weights[slot, None])]
    dout = s["dout"].double()[token]
    dw = torch.zeros(tokens * top_k, dtype=torch.float64, device="cuda").index_copy_(0, slot, (y * dout).sum(1))
    return [sums(s["dxs"].double()[row]), rows_of(dout * weights[slot, None]), dw.view(tokens, top_k)]
