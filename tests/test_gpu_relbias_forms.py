"""Attention with a bucketed relative-position bias: every dispatched form of the kernels in both types, other scales than the
default, and the log-sum-exp within its derived error, against the definition in 64 bits (tolerances: test_gpu_relbias.py).

The log-sum-exp in float32: a score is a sum of D + 1 terms rounded some D + 3 times, each by at most 2^-24 of the sum of the
terms' magnitudes (`size`, the largest over all pairs); the sum of Tk exponentials, each off by two steps, is off by at most
(Tk + 2) 2^-24 of itself, so its logarithm by as much; reference, logarithm and the change of base round to 2^-24 of at most
|lse| + log Tk + size a few times:  (D + 11) size + Tk + 4 (|lse| + log Tk + 1), in units of 2^-24.
"""
import math

import pytest
import torch

from test_gpu_relbias import DEV, check_all, make, reference, within

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def lib():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    from css_amd import ops, ops_bwd
    ops.lib()
    return ops, ops_bwd


def check_lse(lse, q, k, table, scale, want):
    D, Tk = q.shape[3], k.shape[1]
    H, Hk = q.shape[2], k.shape[2]
    size = 0.0
    for h in range(H):
        a, b = q[:, :, h].float().cpu().abs(), k[:, :, h * Hk // H].float().cpu().abs()
        size = max(size, max(float((x @ y.t()).max()) for x, y in zip(a, b)) * scale + float(table[:, h].abs().max()))
    l, finite = lse.cpu().double(), torch.isfinite(want)
    assert torch.equal(torch.isfinite(l), finite)
    tol = 2.0 ** -24 * ((D + 11) * size + Tk + 4 * (want[finite].abs() + math.log(Tk) + 1))
    worst = float(((l - want)[finite].abs() / tol).max())
    assert worst <= 1.0, worst


@pytest.mark.parametrize("scale", [0.02, 1.0, 3.0])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Tq,Tk,H,Hk,D,causal,off", [
    (2, 200, 200, 4, 2, 64, False, 0),       # rows in tiles of 128
    (1, 130, 250, 2, 2, 128, True, 120),
    (1, 3, 700, 4, 2, 64, False, 697),       # few rows
    (1, 2, 3000, 8, 2, 128, True, 2998),     # few rows, keys split
    (1, 500, 130, 6, 2, 32, False, 5),       # backward split over queries
])
def test_scales(lib, B, Tq, Tk, H, Hk, D, causal, off, dtype, scale):
    q, k, v, table, do = make(41, dtype, B, Tq, Tk, H, Hk, D, 32)
    size = min(1.0, (0.25 / scale) ** 0.5)   # scores of ordinary size
    q, k = (q * size).to(dtype), (k * size).to(dtype)
    out, lse, _ = check_all(lib, q, k, v, table, do, (32, 128), causal=causal, offset=off, scale=scale)
    check_lse(lse, q, k, table, scale, reference(q, k, v, table, (32, 128), causal=causal, offset=off, scale=scale)[0]["lse"])


@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D,causal", [(9, 12, 6, 520, 300, 64, False), (22, 6, 2, 520, 430, 56, True), (7, 11, 11, 300, 390, 32, True),
                                                  (9, 6, 3, 520, 300, 128, True)])
def test_many_workgroups_in_fp16(lib, B, H, Hk, Tq, Tk, D, causal):
    """three waves a SIMD in the row-gradient kernel (the first two), hundreds of workgroups"""
    q, k, v, table, do = make(42, torch.float16, B, Tq, Tk, H, Hk, D, 32)
    check_all(lib, q, k, v, table, do, (32, 128), causal=causal, offset=Tk - Tq)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("causal", [False, True])
def test_few_rows_in_many_workgroups(lib, D, dtype, causal):
    """single frames of a serving batch: 640 workgroups of four waves, contexts of different lengths, an idle slot"""
    ops, _ = lib
    B, Tk, H, Hk = 32, 2100, 16, 4
    q, k, v, table, _ = make(43, dtype, B, 1, Tk, H, Hk, D, 32)
    lens = torch.tensor([0] + [Tk - 65 * b for b in range(1, B)], dtype=torch.int32, device=DEV)
    for b, n in enumerate(lens.tolist()):
        k[b, n:], v[b, n:] = math.nan, math.inf
    off = (lens - 1).clamp_min(0).int()
    out, lse = ops.mha_relbias(q, k, v, table, (32, 128), want_lse=True, causal=causal, offset=off, k_lens=lens)
    ref, mag = reference(q, k, v, table, (32, 128), causal=causal, offset=off, k_lens=lens)
    within("out", out, ref["out"], mag["out"], dtype, Tk, float(torch.nan_to_num(v.float(), 0.0, 0.0, 0.0).abs().max()))
    check_lse(lse, q, torch.nan_to_num(k), table, D ** -0.5, ref["lse"])
    assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
    # without a split, many workgroups too
    q, k, v, table, do = make(44, dtype, 40, 2, 500, 8, 8, D, 32)
    check_all(lib, q, k, v, table, do, (32, 128), causal=causal, offset=498)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_more_key_ranges_than_lanes(lib, D, dtype):
    """67 ranges of keys, joined 64 at a time: the largest scores in the first ones, in the last ones, and in both.  A float32 sum runs
    over the 512 keys of a range and then over the ranges, so the errors stay those of some 600 terms."""
    ops, _ = lib
    Tk = 34000
    for first, last in ((0, 1), (1, 0), (1, 1)):
        q, k, v, table, _ = make(45, dtype, 1, 3, Tk, 2, 1, D, 32)
        k[:, :300 * first] += 0.5 * q[:, :1, :1]
        k[:, Tk - 300 * last :] += 0.5 * q[:, 1:2, 1:]
        out, lse = ops.mha_relbias(q, k, v, table, (32, 128), want_lse=True, offset=Tk - 3)
        ref, mag = reference(q, k, v, table, (32, 128), offset=Tk - 3)
        within("out", out, ref["out"], mag["out"], dtype, Tk, float(v.float().abs().max()))
        check_lse(lse, q, k, table, D ** -0.5, ref["lse"])
