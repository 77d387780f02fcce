"""Attention with a bucketed relative-position bias (csship_relbias_fwd / _bwd) against the definition in 64 bits.

The reference takes the kernels' inputs as they are (bf16 / fp16 values) and computes in float64 on the CPU.  Tolerances, per
element, with u half a step of the type relative to the value (bf16 2^-8, fp16 2^-11):
  * a result is rounded once: u |x|;
  * the left operands of the second products (P, dS) are rounded once each: u times the sum of the products' magnitudes,
    sum_j P_ij |v_jd| for out, sum_j |dS_ij| |k_jd| scale for dq, and so on; fp16 values below 2^-14 are rounded to multiples of
    2^-24 instead: at most 2^-25 per product, counted as n 2^-25 max|operand|;
  * everything else is float32: a score of size s (in log2 units) is off by at most (D + 3) 2^-24 |s|max, an exponential by that
    times its value; sums of n terms in float32 by n 2^-24 of the sum of magnitudes at the very most.  With D <= 128, n <= 2100
    and scores up to 32 this stays below REL = 4e-4 of the sums of magnitudes, and below 2^-24 * 32 * 131 = 2.6e-4 for P; the
    float32 results (lse, dtable) get F32 = 1e-4 of their sums of magnitudes, sqrt(n) growth instead of n (n = 10^5: 2e-5).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
REL, F32 = 4e-4, 1e-4


@pytest.fixture(scope="module")
def lib():
    assert torch.cuda.is_available(), "GPU tests need an MI355X"
    from css_amd import ops, ops_bwd
    ops.lib()
    return ops, ops_bwd


def bucket(n, far, two, r):
    """the bucket of one distance, from the formula's logarithms"""
    first = 0
    if two:
        n //= 2
        first, d = n * (r > 0), abs(r)
    else:
        d = max(-r, 0)
    e = n // 2
    if d < e:
        return first + d
    return first + min(n - 1, e + math.floor(math.log(d / e) / math.log(far / e) * (n - e) + 1e-9))


def reference(q, k, v, table, buckets, causal=False, offset=0, k_lens=None, q_lens=None, scale=None, dout=None, out=None):
    """float64 on the CPU; sequence by sequence, head by head, valid rows only.  With dout: the gradients, from the kernel's own
    rounded out (delta = dout . out belongs to the definition)."""
    q, k, v, table = (x.detach().cpu().double() for x in (q, k, v, table))
    B, Tq, H, D = q.shape
    Tk, Hk = k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    n, far, two = (*buckets, True)[:3]
    z = torch.zeros
    o, om, lse = z(B, Tq, H, D).double(), z(B, Tq, H, D).double(), torch.full((B, H, Tq), -math.inf).double()
    g = {x: z(y.shape).double() for x, y in (("dq", q), ("dk", k), ("dv", v), ("dtable", table))}
    gm = {x: torch.zeros_like(y) for x, y in g.items()}
    for b in range(B):
        kl = Tk if k_lens is None else min(max(int(k_lens[b]), 0), Tk)
        ql = Tq if q_lens is None else min(max(int(q_lens[b]), 0), Tq)
        off = int(offset[b]) if isinstance(offset, torch.Tensor) else offset
        if not kl or not ql:
            continue
        r = torch.arange(kl)[None] - (torch.arange(ql)[:, None] + off)
        lo, hi = int(r.min()), int(r.max())
        place = torch.tensor([bucket(n, far, two, x) for x in range(lo, hi + 1)])[r - lo]
        for h in range(H):
            c = h * Hk // H
            qq, kk, vv = q[b, :ql, h], k[b, :kl, c], v[b, :kl, c]
            w = table[:, h]
            w = torch.where(w <= -2.0 ** 20, torch.tensor(-math.inf).double(), w.clamp_max(2.0 ** 20))
            x = qq @ kk.t() * scale + w[place]
            if causal:
                x = x.masked_fill(r > 0, -math.inf)
            tot = torch.logsumexp(x, 1)
            p = torch.where(tot[:, None] > -math.inf, torch.exp(x - tot.clamp_min(-1e300)[:, None]), 0.0)
            lse[b, h, :ql] = tot
            o[b, :ql, h], om[b, :ql, h] = p @ vv, p @ vv.abs()
            if dout is None:
                continue
            do, oo = dout[b, :ql, h].detach().cpu().double(), out[b, :ql, h].detach().cpu().double()
            ds = p * (do @ vv.t() - (do * oo).sum(1, keepdim=True))
            mag = p * (do.abs() @ vv.abs().t() + (do * oo).abs().sum(1, keepdim=True))  # what dS is made of
            g["dq"][b, :ql, h], gm["dq"][b, :ql, h] = ds @ kk * scale, mag @ kk.abs() * scale
            g["dk"][b, :kl, c] += ds.t() @ qq * scale
            gm["dk"][b, :kl, c] += mag.t() @ qq.abs() * scale
            g["dv"][b, :kl, c] += p.t() @ do
            gm["dv"][b, :kl, c] += p.t() @ do.abs()
            g["dtable"][:, h].index_add_(0, place.flatten(), ds.flatten())
            gm["dtable"][:, h].index_add_(0, place.flatten(), mag.flatten())
    return dict(out=o, lse=lse, **g), dict(out=om, **gm)


def within(name, got, want, mag, dtype, n, top):
    """per element: u |x| + u (sum of magnitudes of the rounded products) + float32"""
    got = got.detach().cpu().double()
    assert torch.isfinite(got).all(), name
    u = U[dtype]
    tol = 1.01 * u * want.abs() + (u + REL) * mag + n * TINY[dtype] * top + 1e-6
    worst = float(((got - want).abs() / tol).max()) if got.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.2f} times its tolerance"


def make(seed, dtype, B, Tq, Tk, H, Hk, D, n, size=1.0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, do = (rnd(*s).mul(size).to(dtype).to(DEV) for s in ((B, Tq, H, D), (B, Tk, Hk, D), (B, Tk, Hk, D), (B, Tq, H, D)))
    return q, k, v, rnd(n, H).to(DEV), do


def check_all(lib, q, k, v, table, do, buckets, **how):
    ops, ob = lib
    out, lse = ops.mha_relbias(q, k, v, table, buckets, want_lse=True, **how)
    got = dict(zip(("dq", "dk", "dv", "dtable"), ob.mha_relbias_bwd(q, k, v, table, out, lse, do, buckets, **how)))
    ref, mag = reference(q, k, v, table, buckets, dout=do, out=out, **how)
    dt, Tk, Tq = q.dtype, k.shape[1], q.shape[1]
    fin = lambda x: float(torch.nan_to_num(x.detach().float(), 0.0, 0.0, 0.0).abs().max()) if x.numel() else 0.0  # noqa: E731
    within("out", out, ref["out"], mag["out"], dt, Tk, fin(v))
    finite = torch.isfinite(ref["lse"])
    l = lse.cpu().double()
    assert torch.equal(torch.isfinite(l), finite) and (l[~finite] == -math.inf).all()
    assert float((l - ref["lse"])[finite].abs().max() if finite.any() else 0.0) < F32 * 32
    G = q.shape[2] // k.shape[2]
    for name, n, top in (("dq", Tk, fin(k)), ("dk", Tq * G, fin(q)), ("dv", Tq * G, fin(do))):
        within(name, got[name], ref[name], mag[name], dt, n, top)
    off = (got["dtable"].cpu().double() - ref["dtable"]).abs()
    assert (off <= F32 * mag["dtable"] + 1e-6).all(), float((off / (F32 * mag["dtable"] + 1e-6)).max())
    return out, lse, got


SHAPES = [  # B, Tq, Tk, H, Hk, D, buckets, far, two-sided, causal, offset
    (1, 1, 1, 1, 1, 8, 2, 5, False, False, 0),
    (1, 1, 1, 1, 1, 64, 32, 128, True, True, 0),
    (2, 5, 7, 2, 1, 32, 4, 3, True, False, 2),
    (1, 31, 33, 3, 3, 40, 32, 128, True, False, 0),
    (2, 64, 64, 4, 2, 64, 32, 128, True, True, 0),
    (1, 65, 130, 4, 4, 64, 32, 20, True, False, -7),
    (3, 128, 129, 2, 2, 96, 33, 77, False, True, 1),
    (1, 150, 150, 6, 2, 128, 320, 800, True, False, 0),
    (1, 200, 333, 2, 2, 64, 16, 40, False, True, 133),
    (2, 400, 400, 2, 2, 64, 32, 128, True, False, 0),
    (1, 513, 700, 2, 1, 128, 64, 256, True, True, 187),
    (1, 1, 900, 4, 1, 64, 32, 128, False, True, 899),
    (1, 300, 40, 2, 2, 80, 32, 128, True, True, -100),  # the first 100 queries see no key
    (1, 700, 20, 1, 1, 16, 512, 1024, True, False, 0),
    # few query rows: one workgroup for all keys, keys split over workgroups, several row blocks, groups of heads in a block
    (2, 1, 31, 2, 2, 64, 32, 128, True, False, 30),
    (1, 3, 1500, 8, 2, 128, 32, 128, False, True, 1497),
    (2, 9, 2100, 12, 4, 64, 320, 800, True, False, 1000),
    (1, 5, 1100, 14, 2, 32, 16, 40, True, True, 700),
    (1, 100, 1300, 2, 1, 48, 32, 128, True, False, 1200),
    (3, 2, 1025, 4, 4, 112, 32, 128, True, True, 0),
    (1, 1, 2049, 33, 1, 8, 32, 128, True, True, -1),
    (1, 4, 1400, 16, 1, 64, 320, 800, True, True, 1396),  # tables too wide for the LDS copy
    # the key side of the backward split over workgroups
    (1, 700, 130, 6, 2, 128, 32, 128, True, False, 5),
    (1, 1100, 90, 1, 1, 64, 32, 128, True, True, -300),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_definition(lib, shape, dtype):
    B, Tq, Tk, H, Hk, D, n, far, two, causal, off = shape
    q, k, v, table, do = make(1, dtype, B, Tq, Tk, H, Hk, D, n)
    check_all(lib, q, k, v, table, do, (n, far, two), causal=causal, offset=off)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_batch_reads_nothing_behind_its_ends(lib, dtype, causal):
    """lengths of 0, 1, inside a tile, at a tile's border and full; NaN and infinities behind every sequence's end"""
    B, T, H, Hk, D = 7, 200, 4, 2, 64
    lens = [200, 0, 1, 64, 65, 127, 199]
    q, k, v, table, do = make(2, dtype, B, T, T, H, Hk, D, 32)
    for b, n in enumerate(lens):
        for i, x in enumerate((q, k, v, do)):
            x[b, n:] = (math.nan, math.inf, -math.inf, math.nan)[i]
    kl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out, lse, got = check_all(lib, q, k, v, table, do, (32, 128), causal=causal, k_lens=kl, q_lens=kl)
    for b, n in enumerate(lens):
        assert (out[b, n:] == 0).all() and (lse[b, :, n:] == -math.inf).all()
        for name in ("dq", "dk", "dv"):
            assert (got[name][b, n:] == 0).all(), name


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_batch_of_wide_heads(lib, dtype, causal):
    """the same at 120 columns, where tiles of the key gradients have 32 rows; groups of three heads, steps split over workgroups"""
    lens = [190, 0, 1, 31, 32, 33, 96, 161]
    q, k, v, table, do = make(13, dtype, len(lens), 190, 190, 6, 2, 120, 32)
    for b, n in enumerate(lens):
        for i, x in enumerate((q, k, v, do)):
            x[b, n:] = (math.inf, math.nan, math.nan, -math.inf)[i]
    kl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out, lse, got = check_all(lib, q, k, v, table, do, (32, 128), causal=causal, k_lens=kl, q_lens=kl)
    for b, n in enumerate(lens):
        assert (out[b, n:] == 0).all() and (lse[b, :, n:] == -math.inf).all()
        for name in ("dq", "dk", "dv"):
            assert (got[name][b, n:] == 0).all(), name


def test_serving_batch_of_single_frames(lib):
    """few rows, split keys, lengths and offsets per sequence; an idle slot and garbage behind the kept keys"""
    lens = [1700, 1, 0, 1024, 33, 1699]
    q, k, v, table, do = make(8, torch.bfloat16, 6, 1, 1700, 8, 2, 64, 32)
    for b, n in enumerate(lens):
        k[b, n:], v[b, n:] = math.nan, math.inf
    kl = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for causal in (False, True):
        out, lse, _ = check_all(lib, q, k, v, table, do, (32, 128), causal=causal, k_lens=kl, offset=(kl - 1).int())
        assert (out[2] == 0).all() and (lse[2] == -math.inf).all()


def test_offsets_per_sequence_and_lengths_outside_the_tensors(lib):
    """offsets on the device, far beyond the keys on both sides; lengths below 0 and above the tensors' are cut"""
    q, k, v, table, do = make(3, torch.bfloat16, 5, 40, 70, 2, 2, 64, 32)
    off = torch.tensor([30, -500, 100000, 0, 7], dtype=torch.int32, device=DEV)
    kl = torch.tensor([70, 70, 999, -3, 33], dtype=torch.int32, device=DEV)
    ql = torch.tensor([40, 1000, 40, 40, 0], dtype=torch.int32, device=DEV)
    for causal in (False, True):
        check_all(lib, q, k, v, table, do, (32, 128), causal=causal, offset=off, k_lens=kl, q_lens=ql)


def test_strided_operands(lib):
    """q | k | v as views of one packed projection, a cache in head-major order, an expanded (stride 0) value, a misaligned view"""
    ops, ob = lib
    B, T, H, Hk, D = 2, 100, 4, 2, 64
    table = torch.randn(32, H, device=DEV)
    packed = torch.randn(B, T, (H + 2 * Hk) * D, device=DEV).bfloat16()
    q, k, v = (x.view(B, T, -1, D) for x in packed.split((H * D, Hk * D, Hk * D), -1))
    do = torch.randn(B, T, H * D + 8, device=DEV).bfloat16()[..., 8:].view(B, T, H, D)
    check_all(lib, q, k, v, table, do, (32, 128))
    cache = torch.randn(2, B, Hk, 150, D, device=DEV).bfloat16()
    k, v = (x.transpose(1, 2)[:, :T] for x in cache)
    check_all(lib, q, k, v, table, do, (32, 128))
    check_all(lib, q, k, v[:1].expand(B, -1, -1, -1), table, do.sum(0, keepdim=True).expand(B, -1, -1, -1), (32, 128))
    odd = torch.randn(B * T * H * D + 3, device=DEV).bfloat16()[3:].view(B, T, H, D)
    check_all(lib, odd, k, v, table.t().contiguous().t(), do, (32, 128))


def test_empty_tensors(lib):
    ops, ob = lib
    for B, Tq, Tk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, table, do = make(4, torch.bfloat16, B, Tq, Tk, 2, 2, 32, 8)
        out, lse, got = check_all(lib, q, k, v, table, do, (8, 16))
        assert (out == 0).all() and (lse == -math.inf).all() and all((x == 0).all() for x in got.values())


def test_large_scores_and_banned_distances(lib):
    """scores up to some hundreds; a table with -inf, the type's lowest value and -10^9 (all ban), one large positive entry; rows
    whose every distance is banned"""
    q, k, v, table, do = make(5, torch.bfloat16, 1, 90, 90, 2, 1, 64, 32, size=1.0)
    check_all(lib, q * 4, k * 4, v, table, do, (32, 128))
    table[3, 0], table[4, 0], table[20, 1], table[1, 1], table[25, 0] = -math.inf, torch.finfo(torch.float32).min, -1e9, -2.0 ** 20, 30.0
    check_all(lib, q, k, v, table, do, (32, 128))
    table[:, 1] = -math.inf
    out, lse, got = check_all(lib, q, k, v, table, do, (32, 128))
    assert (out[:, :, 1] == 0).all() and (lse[:, 1] == -math.inf).all() and (got["dtable"][:, 1] == 0).all()


def test_same_bits_every_time(lib):
    ops, ob = lib
    q, k, v, table, do = make(6, torch.bfloat16, 4, 300, 300, 4, 2, 64, 32)
    first = None
    for _ in range(5):
        out, lse = ops.mha_relbias(q, k, v, table, (32, 128), want_lse=True)
        got = (out, lse, *ob.mha_relbias_bwd(q, k, v, table, out, lse, do, (32, 128)))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("B,H,Hk,Tq,Tk,D,causal", [(8, 10, 5, 520, 520, 32, True), (7, 11, 11, 300, 390, 32, True), (9, 12, 4, 270, 270, 32, False),
                                                  (1, 3, 3, 1400, 1400, 32, True), (9, 12, 6, 520, 300, 64, False), (22, 6, 2, 520, 430, 56, True)])
def test_many_workgroups(lib, B, H, Hk, Tq, Tk, D, causal):
    """hundreds of workgroups whose heads do not fall on the 256 or 32 of one round of the chip: every tile is taken, and once"""
    q, k, v, table, do = make(12, torch.bfloat16, B, Tq, Tk, H, Hk, D, 32)
    stale = [torch.full((n,), float("nan"), device="cuda") for n in [1 << 24] * 4 + [1 << 17] * 16]     # what a tile left out shows
    del stale
    check_all(lib, q, k, v, table, do, (32, 128), causal=causal, offset=Tk - Tq)


def test_small_gradients_in_fp16(lib):
    """dS has the size of the incoming gradient: 2^-14 here, and a thousandth of that per key.  Rounded as it is, dS would lie among
    fp16's subnormals (relative error 10^-2 and more); roundings to full precision are independent, u / sqrt(3) each at most
    on average, and dq and dk are rounded twice: below 2 u = 2^-10 in the 2-norm.  One head's gradient comes 2^12 larger from query
    150 on: the running factor of dk goes down in the middle of the sum."""
    ops, ob = lib
    q, k, v, table, do = make(9, torch.float16, 1, 300, 200, 2, 1, 64, 32)
    k = (k * 8).half()
    q = (q / 8).half()
    for late in (1.0, 4096.0):
        d = do.float() * 2.0 ** -14
        d[:, 150:, 1] *= late
        d = d.half()
        out, lse = ops.mha_relbias(q, k, v, table, (32, 128), want_lse=True)
        got = dict(zip(("dq", "dk", "dv", "dtable"), ob.mha_relbias_bwd(q, k, v, table, out, lse, d, (32, 128))))
        ref, _ = reference(q, k, v, table, (32, 128), dout=d, out=out)
        # dq, in multiples of what fp16 can hold at this size: its own subnormals are the caller's choice of scale
        for name in ("dq", "dk"):
            want = ref[name]
            floor = want.numel() ** 0.5 * 2.0 ** -25
            assert float((got[name].cpu().double() - want).norm()) < 2.0 ** -10 * float(want.norm()) + floor, (name, late)
        off = (got["dtable"].cpu().double() - ref["dtable"]).norm() / ref["dtable"].norm()
        assert float(off) < 2e-5


def test_cache_beyond_32_bit_offsets(lib):
    """keys and values as the last heads of a cache of 5.2 GB: element offsets above 2^31, in both forward forms and the backward"""
    B, T, D = 1, 5200, 128
    cache = torch.empty(B, T, 3904, D, dtype=torch.bfloat16, device=DEV)
    cache[:, :, 3902:] = torch.randn(B, T, 2, D, device=DEV).bfloat16()
    k, v = cache[:, :, 3902:3903], cache[:, :, 3903:]
    for Tq in (2, 150):
        q, _, _, table, do = make(10, torch.bfloat16, B, Tq, 1, 1, 1, D, 32)
        check_all(lib, q, k, v, table, do, (32, 128), offset=T - Tq)


def test_other_streams_and_graph_replays(lib):
    """side stream; a captured forward + backward replayed on new inputs with eager work between the replays, and two captured
    graphs in turn: every replay equals the eager result bit for bit"""
    ops, ob = lib
    buckets = (32, 128)

    def work(x):
        out, lse = ops.mha_relbias(*x[:4], buckets, want_lse=True)
        step = ops.mha_relbias(x[0][:, -1:], *x[1:4], buckets, offset=x[1].shape[1] - 1)
        return (out, lse, step, *ob.mha_relbias_bwd(*x[:4], out, lse, x[4], buckets))

    shapes = ((2, 150, 150, 4, 2, 64), (1, 130, 1500, 2, 1, 128))
    graphs = []
    for n, sh in enumerate(shapes):
        x = list(make(20 + n, torch.bfloat16, *sh, 32))
        want = work(x)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = work(x)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = work(x)
        graphs.append((g, x, y, sh))
    for turn in range(3):
        for n, (g, x, y, sh) in enumerate(graphs):
            for a, b in zip(x, make(40 + 2 * turn + n, torch.bfloat16, *sh, 32)):
                a.copy_(b)
            g.replay()
            eager = work(x)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(y, eager)), (turn, n)


def test_first_use_under_capture_is_refused(lib):
    ops, _ = lib
    q, k, v, table, _ = make(11, torch.bfloat16, 1, 8, 8, 2, 2, 64, 32)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(g):
            ops.mha_relbias(q, k, v, table, (32, 97))
    torch.cuda.synchronize()
    ops.mha_relbias(q, k, v, table, (32, 97))


def test_autograd_layer(lib):
    """a layer as a user writes it - packed projection, padded batch, bias table, output projection - trained through autograd:
    gradients of all parameters against float64 autograd of the formulas.  Tolerance: operands, out and the gradients between the
    operators are bf16, about eight roundings of 2^-8 in a row, each independent over the elements and at most u / sqrt(3) on
    average: 8^0.5 2^-8 / 3^0.5 = 6.4e-3 in the 2-norm, doubled."""
    from css_amd.autograd import mha_relbias
    torch.manual_seed(5)
    B, T, H, Hk, D, M = 3, 90, 4, 2, 32, 96
    lens = torch.tensor([90, 41, 64], dtype=torch.int32, device=DEV)
    w1 = (torch.randn((H + 2 * Hk) * D, M, device=DEV) / M ** 0.5).requires_grad_()
    w2 = (torch.randn(M, H * D, device=DEV) / (H * D) ** 0.5).requires_grad_()
    table = torch.randn(32, H, device=DEV, requires_grad=True)
    x = torch.randn(B, T, M, device=DEV)
    up = torch.randn(B, T, M, device=DEV)
    inside = (torch.arange(T, device=DEV)[None] < lens[:, None])[..., None]

    def layer(x, w1, w2, table, attend):
        p = x @ w1.t()
        q, k, v = p.split((H * D, Hk * D, Hk * D), -1)
        o = attend(q.view(B, T, H, D), k.view(B, T, Hk, D), v.view(B, T, Hk, D), table)
        return ((o.reshape(B, T, H * D) @ w2.t()) * up.to(x.dtype) * inside).sum()

    def ours(q, k, v, table):
        return mha_relbias(q.bfloat16(), k.bfloat16(), v.bfloat16(), table, (32, 128), k_lens=lens, q_lens=lens).to(q.dtype)

    def plain(q, k, v, table):
        r = torch.arange(T)[None] - torch.arange(T)[:, None]
        place = torch.tensor([bucket(32, 128, True, x) for x in range(-T + 1, T)])[r + T - 1].to(DEV)
        kk, vv = (y.repeat_interleave(H // Hk, 2).transpose(1, 2) for y in (k, v))
        s = (q.transpose(1, 2) @ kk.transpose(2, 3).contiguous()) * D ** -0.5 + table[place].permute(2, 0, 1)
        s = s.masked_fill(~inside[:, None, None, :, 0], -math.inf)
        return (torch.softmax(s, -1) @ vv).transpose(1, 2) * inside[..., None]

    layer(x, w1, w2, table, ours).backward()
    got = [t.grad.clone() for t in (w1, w2, table)]
    d = [t.detach().double().requires_grad_() for t in (w1, w2, table)]
    layer(x.double(), *d, plain).backward()
    for a, b in zip(got, d):
        assert float((a.double() - b.grad).norm() / b.grad.norm()) < 2 * 6.4e-3
    # differences: along the gradient the loss moves as its square says (float64 formulas at both ends)
    with torch.no_grad():
        h, ends = 1e-4, []
        for sign in (1, -1):
            moved = [t.detach().double() + sign * h * g.double() / g.double().norm() for t, g in zip((w1, w2, table), got)]
            ends.append(float(layer(x.double(), *moved, plain)))
        slope = (ends[0] - ends[1]) / (2 * h)
        want = sum(float(g.double().norm()) for g in got)
        assert abs(slope - want) < 2e-2 * want
    q = torch.randn(1, 4, 2, 32, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    y = mha_relbias(q, q, q, table[:, :2], (32, 128))
    g, = torch.autograd.grad(y.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative
        g.sum().backward()


def test_broadcast_gradient_and_shared_heads(lib):
    """an expanded (stride 0) upstream gradient and values expanded over the batch: gradients land on the one copy"""
    from css_amd.autograd import mha_relbias
    torch.manual_seed(6)
    q = torch.randn(4, 50, 4, 32, device=DEV).bfloat16().requires_grad_()
    k = torch.randn(4, 50, 1, 32, device=DEV).bfloat16().requires_grad_()
    v1 = torch.randn(1, 50, 1, 32, device=DEV).bfloat16().requires_grad_()
    table = torch.randn(16, 4, device=DEV, requires_grad=True)
    y = mha_relbias(q, k, v1.expand(4, -1, -1, -1), table, (16, 40))
    y.sum().backward()
    ref, mag = reference(q, k, v1.expand(4, -1, -1, -1), table, (16, 40), dout=torch.ones_like(y), out=y)
    want, m = ref["dv"].sum(0, keepdim=True), mag["dv"].sum(0, keepdim=True)
    # four rounded gradients are added in bf16: three more roundings
    assert ((v1.grad.cpu().double() - want).abs() <= 4 * 2.0 ** -8 * m + 1e-6).all()
    within("dk", k.grad, ref["dk"], mag["dk"], torch.bfloat16, 200, 1.0)


def test_refusals(lib):
    ops, ob = lib
    q, k, v, table, do = make(7, torch.bfloat16, 2, 8, 8, 4, 2, 64, 32)
    ok = (32, 128)
    lens = torch.ones(2, dtype=torch.int32, device=DEV)
    bad = [
        (TypeError, (q.float(), k, v, table, ok), {}),
        (TypeError, (q, k.half(), v, table, ok), {}),
        (RuntimeError, (q[0], k, v, table, ok), {}),
        (RuntimeError, (q.cpu(), k, v, table, ok), {}),
        (RuntimeError, (q, k[:, :4], v, table, ok), {}),
        (RuntimeError, (q[:, :, :3], k, v, table, ok), {}),
        (RuntimeError, (q[..., :60], k[..., :60], v[..., :60], table, ok), {}),
        (RuntimeError, (q, k, v, table[:16], ok), {}),
        (TypeError, (q, k, v, table.double(), ok), {}),
        (RuntimeError, (q, k, v, table, (32, 8)), {}),
        (RuntimeError, (q, k, v, table, (32, 5000)), {}),
        (RuntimeError, (q, k, v, table[:31], (31, 128)), {}),
        (RuntimeError, (q, k, v, table, ok), dict(k_lens=lens.long())),
        (RuntimeError, (q, k, v, table, ok), dict(k_lens=lens[:1])),
        (TypeError, (q, k, v, table, ok), dict(q_lens=[1, 2])),
        (RuntimeError, (q, k, v, table, ok), dict(offset=lens.cpu())),
        (RuntimeError, (q, k, v, table, ok), dict(offset=1 << 30)),
        (RuntimeError, (q, k, v, table, ok), dict(offset=0.5)),
        (RuntimeError, (q, k, v, table, ok), dict(scale=0.0)),
    ]
    for kind, args, how in bad:
        with pytest.raises(kind):
            ops.mha_relbias(*args, **how)
    out, lse = ops.mha_relbias(q, k, v, table, ok, want_lse=True)
    for o, l, d in ((out[:, :4], lse, do), (out, lse[:, :2], do), (out, lse, do.half()), (out, lse.double(), do), (out, lse, do[:, :4])):
        with pytest.raises((RuntimeError, TypeError)):
            ob.mha_relbias_bwd(q, k, v, table, o, l, d, ok)
