"""The quantiser's gather (row_index): what becomes of every byte of codes and scales, rows that are left out included."""
import numpy as np
import pytest

import mx4_reference as ref
import rocm_sgemm_b200 as pkg

torch = pytest.importorskip("torch")
gpu = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def scale_rows(fmt, scales, rows, K):
    """Scale bytes of all rows that the tiles hold, behind the last row and behind K too."""
    bands, tiles = -(-rows // 128), -(-K // (4 * ref.BLOCK[fmt]))
    return scales.reshape(bands, tiles, 32, 4, 4).transpose(0, 3, 2, 1, 4).reshape(bands * 128, tiles * 4)


@gpu
@pytest.mark.parametrize("fmt", [ref.NVFP4, ref.MXFP4], ids=["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,K,div,none", [(400, 96, 3, (128, 256)), (400, 70, 1, (384, 400)), (300, 1030, 2, (0, 128)), (1, 33, 1, (0, 0)),
                                             (130, 512, 5, (0, 130))], ids=lambda v: str(v))
@pytest.mark.parametrize("bad", [False, True])
def test_gather_writes_these_bytes_and_no_others(sgemm, fmt, dtype, rows, K, div, none, bad):
    n = 37
    r = np.random.default_rng(rows + K)
    x = torch.from_numpy(r.standard_normal((n, K))).to(TYPES[dtype])
    index = r.integers(0, n * div, rows).astype(np.int32)
    index[r.random(rows) < 0.3] = -1
    far = r.random(rows) < 0.1
    index[far] = r.choice([n * div, n * div + 1, 2 ** 31 - 1, -2 ** 31], far.sum())
    index[none[0]:none[1]] = -1
    used = (index >= 0) & (index // div < n)
    if bad:  # a row of X that no index names is not read, one that an index names makes its blocks NaN
        x[n - 1] = float("nan")
        index[used & (index // div == n - 1)] = -1
        x[0, K - 1] = float("inf")
        used = (index >= 0) & (index // div < n)
    codes, scales = (torch.full((m,), 0xA5, dtype=torch.uint8, device="cuda") for m in sgemm.mx4_sizes(fmt, rows, K))
    sgemm.mx4_quantize(fmt, 0, pkg.m_type[dtype], x.cuda(), rows, K, codes, scales, row_index=dev(index), source_rows=n, index_div=div)
    code, byte = ref.quantize(fmt, x.double().numpy())
    want_codes = np.full((rows, -(-K // 32) * 16), 0xA5, np.uint8)
    packed = ref.pack(fmt, code, byte)[0].reshape(n, -1)
    want_codes[used] = packed[index[used] // div]
    assert np.array_equal(codes.cpu().numpy().reshape(rows, -1), want_codes)
    got = scale_rows(fmt, scales.cpu().numpy(), rows, K)
    want = np.zeros_like(got)
    at = np.nonzero(used)[0]
    want[at, :byte.shape[1]] = byte[index[used] // div]
    for band in range(0, got.shape[0], 128):
        if not used[band:band + 128].any():
            want[band:band + 128] = 0xA5
    assert np.array_equal(got, want)
