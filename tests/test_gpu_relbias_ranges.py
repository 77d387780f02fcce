"""Attention with a bucketed relative-position bias: values far from 1 - small and large probabilities, gradients, values, scales -
against the definition in 64 bits.

u = 2^-11 is half a step of fp16 relative to the value.  Where signs are random a 2-norm over many results is compared: dq, dk and dv
are rounded once and are sums of products whose left operand was rounded once, each rounding independent and u / sqrt(3) on
average at most, so u sqrt(2 / 3) in all: below BOTH = 2 u = 2^-10.  What fp16 cannot hold of a result (steps of 2^-24 below 2^-14) is
the caller's choice of scale: half a step per element, `floor`.
"""
import math

import pytest
import torch

from test_gpu_relbias import DEV, U, make, reference, within

pytestmark = pytest.mark.gpu

BOTH = 2.0 ** -10


@pytest.fixture(scope="module")
def lib():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    from css_amd import ops, ops_bwd
    ops.lib()
    return ops, ops_bwd


def gradients(lib, q, k, v, table, do, buckets, **how):
    ops, ob = lib
    out, lse = ops.mha_relbias(q, k, v, table, buckets, want_lse=True, **how)
    got = dict(zip(("dq", "dk", "dv", "dtable"), ob.mha_relbias_bwd(q, k, v, table, out, lse, do, buckets, **how)))
    return got, reference(q, k, v, table, buckets, dout=do, out=out, **how)


def near(name, got, want):
    # beyond 65504 fp16 has nothing but infinities: both sides are cut there, which brings no two numbers further apart
    got, want = got.cpu().double().clamp(-65504, 65504), want.clamp(-65504, 65504)
    floor = want.numel() ** 0.5 * 2.0 ** -25
    off, size = float((got - want).norm()), float(want.norm())
    assert off < BOTH * size + floor, f"{name}: {off / size:.2e} of its norm"


@pytest.mark.parametrize("D,far,gap,up", [(64, 6001, -9.0, 1024.0), (64, 6001, -6.0, 1024.0), (120, 3001, -9.0, 1024.0),
                                          (32, 3001, -14.0, 8192.0)])
def test_value_gradients_of_weakly_attended_keys_in_fp16(lib, D, far, gap, up):
    """keys beyond a distance get little of every query: some 2^-22 at -9, 2^-29 (below all that fp16 holds) at -14"""
    B, Tq, H = 1, 300, 2
    q, k, v, table, do = make(31, torch.float16, B, Tq, far, H, 1, D, 32)
    do = (do * up).half()
    table[15] = table[31] = gap  # the last bucket of either side
    got, (ref, _) = gradients(lib, q, k, v, table, do, (32, 128))
    behind = Tq + 128
    near("dv far", got["dv"][:, behind:], ref["dv"][:, behind:])
    near("dv near", got["dv"][:, :behind], ref["dv"][:, :behind])


@pytest.mark.parametrize("D,Tq,Tk,size,up", [(64, 40, 6001, 0.02, 8.0), (64, 200, 6001, 0.001, 64.0), (128, 70, 3001, 0.001, 64.0),
                                             (32, 300, 3001, 2.0 ** -14, 1024.0)])
def test_gradients_of_small_values_and_many_keys_in_fp16(lib, D, Tq, Tk, size, up):
    """dS = P (dout . v - delta) has the size of v / Tk, whatever dout's"""
    q, k, v, table, do = make(32, torch.float16, 1, Tq, Tk, 2, 1, D, 32)
    k, q, v, do = (k * 8).half(), (q / 8).half(), (v * size).half(), (do * up).half()
    got, (ref, _) = gradients(lib, q, k, v, table, do, (32, 128))
    for name in ("dq", "dk", "dv"):
        near(name, got[name], ref[name])
    # float32: a probability is off by at most (D + 3) 2^-24 |s| with |s| up to 12 in log2 units (9.4e-5 of it at 128), signs random
    assert float((got["dtable"].cpu().double() - ref["dtable"]).norm() / ref["dtable"].norm()) < 1e-4


@pytest.mark.parametrize("Tk", [40, 333])
def test_gradients_of_large_values_in_fp16(lib, Tk):
    """rows of v of norm 240000 along dout: dS in units of dout's norm is beyond fp16, dq and dk are not"""
    q, k, v, table, do = make(33, torch.float16, 1, Tk, Tk, 2, 2, 64, 32)
    v = (torch.where(v > 0, 30000.0, -30000.0)).half()
    do = (v.float() * 2.0 ** -30).half()
    table[0] = math.log(Tk)  # distance 0: about half of each row's probability
    got, (ref, _) = gradients(lib, q, k, v, table, do, (32, 128))
    for name in ("dq", "dk"):
        assert torch.isfinite(got[name]).all()
        near(name, got[name], ref[name])


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_that_change_size_along_a_sum_in_fp16(lib, D):
    """values 2^12 larger (and then as small again) along the keys, gradients 2^14 larger along the queries: the factors of dq's and
    dk's sums go down in the middle of them, by different steps in different rows"""
    for flip in (False, True):
        q, k, v, table, do = make(36, torch.float16, 1, 400, 700, 2, 1, D, 32)
        v, do = v * 2.0 ** -6, do * 2.0 ** -6
        v[:, 300:450] *= 2.0 ** 12
        do[:, ::3] *= 2.0 ** 5
        do[:, 200:] *= 2.0 ** 14
        v, do = v.half(), do.half()
        if flip:
            v, do = v.flip(1), do.flip(1)
        got, (ref, _) = gradients(lib, q, k, v, table, do, (32, 128))
        for name in ("dq", "dk", "dv"):
            near(name, got[name], ref[name])
        small = slice(200, 400) if flip else slice(0, 200)  # these rows of dq by themselves
        near("dq of small gradients", got["dq"][:, small], ref["dq"][:, small])


def test_one_key_with_nearly_all_of_a_row_in_fp16(lib):
    """The first key takes each row, its value is 0; the others have 2^-25.5 of it each, and the sum of thousands of them is the
    result.  Tolerance: fp16 holds P down to 2^-32 of the row's largest in steps of that size (n 2^-32 max|v|), else as everywhere."""
    ops, _ = lib
    for B, Tq, Tk, H in ((1, 1000, 1000, 16), (2, 3, 4000, 4), (1, 200, 900, 2)):
        q = torch.ones(B, Tq, H, 64, device=DEV).half()
        k = (torch.randn(B, Tk, H, 64, generator=torch.Generator().manual_seed(34)).to(DEV) * 0.05).half()
        k[:, 0] = 25.5 * math.log(2.0) / 8
        v = torch.full((B, Tk, H, 64), 1000.0, device=DEV).half()
        v[:, 0] = 0
        table = torch.zeros(32, H, device=DEV)
        out, lse = ops.mha_relbias(q, k, v, table, (32, 128), want_lse=True)
        ref, mag = reference(q, k, v, table, (32, 128))
        want, got = ref["out"], out.cpu().double()
        tol = 1.01 * U[torch.float16] * want + (U[torch.float16] + 4e-4) * mag["out"] + Tk * 2.0 ** -32 * 1000.0 + 1e-6
        worst = float(((got - want).abs() / tol).max())
        assert worst <= 1.0, (B, Tq, Tk, H, worst)
        assert float((lse.cpu().double() - ref["lse"]).abs().max()) < 1e-4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_cache_that_is_not_yet_written_behind_the_newest_frame(lib, dtype):
    """causal, no lengths: keys behind every query's position are seen by none and may hold anything, as an allocated cache does"""
    ops, ob = lib
    for B, Tq, H, Hk, D, T, off in ((2, 5, 4, 2, 64, 700, 333), (1, 100, 2, 1, 64, 200, 29), (2, 1, 8, 2, 128, 3000, 0), (1, 300, 4, 4, 32, 310, -2)):
        q, k, v, table, do = make(35, dtype, B, Tq, T, H, Hk, D, 32)
        n = off + Tq
        k[:, n:], v[:, n:] = math.nan, math.inf
        each = torch.full((B,), off, dtype=torch.int32, device=DEV)
        lens = torch.full((B,), n, dtype=torch.int32)
        for o in (off, each):
            out, lse = ops.mha_relbias(q, k, v, table, (32, 128), want_lse=True, causal=True, offset=o)
            got = dict(zip(("dq", "dk", "dv", "dtable"), ob.mha_relbias_bwd(q, k, v, table, out, lse, do, (32, 128), causal=True, offset=o)))
            ref, mag = reference(q, k, v, table, (32, 128), causal=True, offset=off, k_lens=lens, dout=do, out=out)
            within("out", out, ref["out"], mag["out"], dtype, T, float(v[:, :n].float().abs().max()))
            for name, top in (("dq", k[:, :n]), ("dk", q), ("dv", do)):
                within(name, got[name], ref[name], mag[name], dtype, T * H // Hk, float(top.float().abs().max()))
            assert torch.isfinite(got["dtable"]).all()
            assert (got["dk"][:, n:] == 0).all() and (got["dv"][:, n:] == 0).all()


@pytest.mark.parametrize("D", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_overflowed_and_absent_gradients(lib, dtype, D):
    """an infinity in dout (a loss scale that was too large) is seen in every gradient it belongs to and in no other sequence's or
    head's; a gradient of zeros gives zeros"""
    ops, ob = lib
    q, k, v, table, do = make(37, dtype, 2, 150, 170, 4, 2, D, 32)
    out, lse = ops.mha_relbias(q, k, v, table, (32, 128), want_lse=True)
    bad = do.clone()
    bad[0, 77, 1] = math.inf
    dq, dk, dv, dt = ob.mha_relbias_bwd(q, k, v, table, out, lse, bad, (32, 128))
    want = ob.mha_relbias_bwd(q, k, v, table, out, lse, do, (32, 128))
    assert not torch.isfinite(dq[0, 77, 1]).any() and not torch.isfinite(dv[0, :, 0]).any() and not torch.isfinite(dk[0, :, 0]).any()
    assert not torch.isfinite(dt[:, 1]).all()
    others = torch.ones(2, 150, 4, dtype=torch.bool, device=DEV)
    others[0, 77, 1] = False
    assert torch.equal(dq[others], want[0][others])
    for a, b in ((dk, want[1]), (dv, want[2])):
        assert torch.equal(a[1], b[1]) and torch.equal(a[0, :, 1], b[0, :, 1])
    assert torch.equal(dt[:, [0, 2, 3]], want[3][:, [0, 2, 3]])
    for g in ob.mha_relbias_bwd(q, k, v, table, out, lse, torch.zeros_like(do), (32, 128)):
        assert (g == 0).all()


def test_two_threads_on_streams_of_their_own(lib):
    """forward and backward of both types at once, with settings that neither thread has used before: the same bits as alone"""
    import threading
    ops, ob = lib
    jobs = []
    for n, dtype in enumerate((torch.bfloat16, torch.float16)):
        x = make(50 + n, dtype, 2, 200, 300, 4, 2, 64, 24)
        jobs.append((x, torch.cuda.Stream(), []))
    torch.cuda.synchronize()
    together = threading.Barrier(2, timeout=30)

    def work(x):
        out, lse = ops.mha_relbias(*x[:4], (24, 119), want_lse=True)
        step = ops.mha_relbias(x[0][:, -1:], *x[1:4], (24, 119), offset=299)
        return (out, lse, step, *ob.mha_relbias_bwd(*x[:4], out, lse, x[4], (24, 119)))

    def thread(x, stream, got):
        with torch.cuda.stream(stream):
            together.wait()
            for _ in range(20):
                got.append(work(x))
        stream.synchronize()

    threads = [threading.Thread(target=thread, args=j) for j in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    for x, _, got in jobs:
        alone = work(x)
        torch.cuda.synchronize()
        assert len(got) == 20
        for g in got:
            assert all(torch.equal(a, b) for a, b in zip(alone, g))
