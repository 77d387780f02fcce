"""Cases of the attention with a bucketed relative-position bias, for the timing of its kernels.

Three kinds of pass ("op" of a case):
  fwd   one attention layer's forward in training: out and the rows' log-sum-exp
  step  a few new frames against the keys kept so far (streaming): out alone
  bwd   the layer's backward: gradients of q, k, v and of the bias table

A query i of sequence b sits at position i + offset[b], a key j at position j; r = j - position of the query:

  s[i, j] = scale * q_i . k_j + table[bucket(r), h]     over the keys j < k_lens[b] (and r <= 0 where the case is causal)
  out_i = sum_j softmax_j(s[i, :]) v_j,  lse_i = log sum_j exp(s[i, j]);  a row without keys: out 0, lse -inf
"""
import math

import torch

own = False

NEG = float("-inf")

_DEFAULTS = dict(op="fwd", dtype="bf16", B=1, Tq=1, Tk=1, H=4, Hk=4, D=64, buckets=32, max_distance=128, two_sided=True,
                 causal=False, ragged=False)


def _case(name, **kw):
    return dict(_DEFAULTS, name=name, **kw)


def listed():
    return [
        # ---- forward
        # the training chunk of the repository's benchmark: 32 x 400 frames, 4 heads of 64
        _case("fwd chunk 32x400", op="fwd", B=32, Tq=400, Tk=400),
        # separation windows of 2.4 s (150 frames), padded to the longest of the batch, a wide bucket table, fp16
        _case("fwd ragged windows", op="fwd", dtype="fp16", B=24, Tq=150, Tk=150, H=8, Hk=8, buckets=320, max_distance=800, ragged=True),
        # a decoder-like stack: causal, one-sided buckets, grouped heads of 128, an odd length
        _case("fwd causal grouped", op="fwd", B=2, Tq=2047, Tk=2047, H=16, Hk=4, D=128, two_sided=False, causal=True),
        # a whole recording in one pass (three minutes of frames)
        _case("fwd long", op="fwd", B=1, Tq=11250, Tk=11250, H=8, Hk=8),
        # ---- a few new frames against kept keys
        # the smallest call: one stream, one new frame, eight seconds of context
        _case("step one stream", op="step", B=1, Tq=1, Tk=500, H=4, Hk=4),
        # a serving batch of single frames, contexts of different lengths, one slot idle
        _case("step batch", op="step", B=32, Tq=1, Tk=8192, H=16, Hk=4, D=128, two_sided=False, causal=True, ragged=True),
        # a chunk of eight frames against a long recording, fp16, an odd number of keys
        _case("step chunk long", op="step", dtype="fp16", B=4, Tq=8, Tk=30001, H=8, Hk=8),
        # ---- backward
        _case("bwd chunk 32x400", op="bwd", B=32, Tq=400, Tk=400),
        _case("bwd ragged windows", op="bwd", dtype="fp16", B=24, Tq=150, Tk=150, H=8, Hk=8, buckets=320, max_distance=800, ragged=True),
        _case("bwd causal grouped", op="bwd", B=2, Tq=2047, Tk=2047, H=16, Hk=4, D=128, two_sided=False, causal=True),
        _case("bwd long", op="bwd", B=1, Tq=6001, Tk=6001, H=8, Hk=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["fwd", "step", "bwd"])
        H = rng.choice([2, 4, 6, 8, 12, 16])
        Hk = rng.choice([h for h in (1, 2, 3, 4, 6, 8, 12, 16) if H % h == 0])
        causal = rng.random() < 0.35
        n, far = rng.choice([(32, 128), (32, 128), (64, 256), (320, 800), (16, 40)])
        if op == "step":
            Tq, Tk, B = _log(rng, 1, 16), _log(rng, 64, 30001), _log(rng, 1, 32)
        else:
            Tk, B = _log(rng, 17, 11250 if op == "fwd" else 6001), _log(rng, 1, 48)
            Tq = Tk if rng.random() < 0.8 else _log(rng, 17, Tk)
        c = dict(_DEFAULTS, op=op, dtype=rng.choice(["bf16", "bf16", "fp16"]), B=B, Tq=min(Tq, Tk), Tk=Tk, H=H, Hk=Hk,
                 D=rng.choice([32, 64, 64, 80, 96, 128]), buckets=n, max_distance=far,
                 two_sided=(not causal) or rng.random() < 0.3, causal=causal, ragged=B > 1 and rng.random() < 0.5)
        w = work(c)
        top = {"fwd": 2.6e11, "step": 1e10, "bwd": 1.84e11}[op]
        if w["flops"] <= top and w["bytes"] <= 4.5e8 and 4.0 * B * H * c["Tq"] * Tk <= 4.2e9:
            return c


# ------------------------------------------------------------------------------------------------ lengths and work
def _k_lens(c):
    """Lengths of the batch: the longest first, down to half of it; a serving batch has one idle slot, its last."""
    if not c["ragged"]:
        return [c["Tk"]] * c["B"]
    got = [c["Tk"] - (b * c["Tk"]) // (2 * c["B"]) for b in range(c["B"])]
    if c["op"] == "step":
        got[-1] = 0
    return got


def _q_lens(c):
    return [min(c["Tq"], n) for n in _k_lens(c)] if c["op"] != "step" else [c["Tq"]] * c["B"]


def _offsets(c):
    """Streaming queries are the newest frames; otherwise the queries' last position is the keys' last."""
    return [max(0, n - c["Tq"]) for n in _k_lens(c)] if c["op"] == "step" else [c["Tk"] - c["Tq"]] * c["B"]


def _pairs(c):
    total = 0
    for ql, kl, off in zip(_q_lens(c), _k_lens(c), _offsets(c)):
        if not c["causal"]:
            total += ql * kl
        else:
            full = max(0, min(ql, kl - off))  # queries i < full see i + off + 1 keys, the others all
            total += full * off + full * (full + 1) // 2 + (ql - full) * kl
    return total * c["H"]


def work(c):
    nq, nk = sum(_q_lens(c)), sum(_k_lens(c))
    q, kv, table = nq * c["H"] * c["D"] * 2, nk * c["Hk"] * c["D"] * 2, c["buckets"] * c["H"] * 4
    rows = nq * c["H"] * 4
    pairs = _pairs(c)
    if c["op"] == "bwd":  # q, out, dout, lse, k, v, table in; dq, dk, dv, d table out
        return {"bytes": 4 * q + rows + 4 * kv + 2 * table, "flops": 10 * c["D"] * pairs}
    return {"bytes": 2 * q + (rows if c["op"] == "fwd" else 0) + 2 * kv + table, "flops": 4 * c["D"] * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _dtype(c):
    return {"bf16": torch.bfloat16, "fp16": torch.float16}[c["dtype"]]


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    t, B, Tq, Tk, H, Hk, D = _dtype(c), c["B"], c["Tq"], c["Tk"], c["H"], c["Hk"], c["D"]
    s = {"case": c}
    if c["op"] != "step" and Tq == Tk:  # the projections' packed rows, as the layer in front writes them
        packed = normal(B, Tk, (H + 2 * Hk) * D).to(t)
        s["q"] = packed[..., : H * D].view(B, Tq, H, D)
        s["k"] = packed[..., H * D : (H + Hk) * D].view(B, Tk, Hk, D)
        s["v"] = packed[..., (H + Hk) * D :].view(B, Tk, Hk, D)
    else:
        s["q"], s["k"], s["v"] = normal(B, Tq, H, D).to(t), normal(B, Tk, Hk, D).to(t), normal(B, Tk, Hk, D).to(t)
    s["table"] = normal(c["buckets"], H)
    s["k_lens"] = torch.tensor(_k_lens(c), dtype=torch.int32, device="cuda") if c["ragged"] else None
    s["q_lens"] = torch.tensor(_q_lens(c), dtype=torch.int32, device="cuda") if c["ragged"] and c["op"] != "step" else None
    s["offset"] = torch.tensor(_offsets(c), dtype=torch.int32, device="cuda") if c["ragged"] and c["op"] == "step" else _offsets(c)[0]
    if c["op"] == "bwd":  # what the forward left, and the gradient that comes from above
        s["dout"] = normal(B, Tq, H, D).to(t)
        s["out"], s["lse"] = _forward(s)
    return s


# ------------------------------------------------------------------------------------------------ plain form
def _per_batch(v, B, fill):
    """[B] lengths or offsets on the device from a tensor, a number or nothing."""
    if isinstance(v, torch.Tensor):
        return v.long()
    return torch.full((B,), fill if v is None else v, dtype=torch.long, device="cuda")


def _bucket(c, r):
    """Bucket of the distance r = key position - query position (whole numbers).  The logarithms are taken in 64 bits and
    lifted by 1e-9: a quotient that is a whole number in the formula must not end just below it."""
    n, first = c["buckets"], 0
    if c["two_sided"]:
        n //= 2
        first = (r > 0) * n
        d = r.abs()
    else:
        d = (-r).clamp_min(0)
    e = n // 2
    far = torch.log(d.clamp_min(1).double() / e) / math.log(c["max_distance"] / e) * (n - e)
    far = (e + torch.floor(far + 1e-9).long()).clamp_max(n - 1)
    return first + torch.where(d < e, d, far)


def _heads(x, H):
    """[B, T, Hk, D] -> f32 [B, H, T, D], a key head repeated for the query heads that share it."""
    x = x.float().transpose(1, 2)
    return x.repeat_interleave(H // x.shape[1], dim=1)


def _scores(s):
    """f32 [B, H, Tq, Tk] scores, -inf where a query does not see a key, and the operands of the products."""
    c = s["case"]
    B, Tq, Tk, H = c["B"], c["Tq"], c["Tk"], c["H"]
    qi, kj = torch.arange(Tq, device="cuda"), torch.arange(Tk, device="cuda")
    off = _per_batch(s["offset"], B, 0)
    kl, ql = _per_batch(s["k_lens"], B, Tk), _per_batch(s["q_lens"], B, Tq)
    if not isinstance(s["offset"], torch.Tensor):
        off = off[:1]  # one position for the whole batch
    r = kj[None, None, :] - (qi[None, :, None] + off[:, None, None])
    bias = s["table"][_bucket(c, r)].permute(0, 3, 1, 2)  # [B or 1, H, Tq, Tk]
    seen = (kj[None, None, :] < kl[:, None, None]) & (qi[None, :, None] < ql[:, None, None])
    if c["causal"]:
        seen = seen & (r <= 0)
    # what lies behind a sequence's end never enters a product: it may hold anything
    inside = (kj[None, :] < kl[:, None])[:, None, :, None]
    q = _heads(s["q"], H)
    k, v = (torch.where(inside, _heads(s[n], H), 0.0) for n in ("k", "v"))
    x = torch.matmul(q, k.transpose(2, 3)).mul_(c["D"] ** -0.5).add_(bias)
    return x.masked_fill_(~seen[:, None], NEG), q, k, v, r


def _softmax(x):
    """(probabilities, log-sum-exp) over the last axis; a row of -inf gives zeros and -inf."""
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(m == NEG, 0.0, m))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, 1.0, total)
    return p, (torch.log(total) + m).squeeze(-1)


def _forward(s):
    x, _, _, v, _ = _scores(s)
    p, lse = _softmax(x)
    return torch.matmul(p, v).transpose(1, 2).to(_dtype(s["case"])).contiguous(), lse


def _backward(s):
    c = s["case"]
    B, Tq, Tk, H, Hk, D, t = c["B"], c["Tq"], c["Tk"], c["H"], c["Hk"], c["D"], _dtype(c)
    scale = D ** -0.5
    x, q, k, v, r = _scores(s)
    lse = s["lse"][..., None]
    p = torch.exp(x - torch.where(lse == NEG, 0.0, lse))
    do, o = _heads(s["dout"], H), _heads(s["out"], H)
    d = (do * o).sum(-1, keepdim=True)
    ds = torch.matmul(do, v.transpose(2, 3)).sub_(d).mul_(p)
    dq = torch.matmul(ds, k).mul_(scale).transpose(1, 2).to(t)
    dk = torch.matmul(ds.transpose(2, 3), q).mul_(scale).view(B, Hk, H // Hk, Tk, D).sum(2).transpose(1, 2).to(t)
    dv = torch.matmul(p.transpose(2, 3), do).view(B, Hk, H // Hk, Tk, D).sum(2).transpose(1, 2).to(t)
    # one sum per diagonal (distances run along them): the rows in reverse order in rows one element shorter put each
    # diagonal into a column; long sums of both signs, so in 64 bits
    W = Tq + Tk
    skew = torch.nn.functional.pad(ds.flip(2), (0, Tq)).view(B, H, Tq * W)[..., : Tq * (W - 1)].view(B, H, Tq, W - 1)
    diagonal = skew.sum((0, 2), dtype=torch.float64)  # [H, Tq + Tk - 1], distance = column - (Tq - 1) - offset
    at = _bucket(c, torch.arange(W - 1, device="cuda") - (Tq - 1) - int(s["offset"]))
    one = (at[:, None] == torch.arange(c["buckets"], device="cuda")[None, :]).double()
    return dq, dk, dv, torch.matmul(diagonal, one).t().float()


def run(s):
    c = s["case"]
    if own:
        from css_amd import ops, ops_bwd

        how = dict(buckets=(c["buckets"], c["max_distance"], c["two_sided"]), causal=c["causal"], offset=s["offset"],
                   k_lens=s["k_lens"], q_lens=s["q_lens"])
        if c["op"] == "bwd":
            return ops_bwd.mha_relbias_bwd(s["q"], s["k"], s["v"], s["table"], s["out"], s["lse"], s["dout"], **how)
        return ops.mha_relbias(s["q"], s["k"], s["v"], s["table"], want_lse=c["op"] == "fwd", **how)
    if c["op"] == "bwd":
        return _backward(s)
    out, lse = _forward(s)
    return (out, lse) if c["op"] == "fwd" else out


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _first_distances(n, e, far):
    """first[t]: the smallest distance whose logarithmic bucket is e + t, decided in whole numbers:
    (n - e) log(d / e) / log(far / e) >= t  <=>  d^(n-e) e^t >= e^(n-e) far^t."""
    first, d = [], e
    for t in range(n - e):
        while d ** (n - e) * e ** t < e ** (n - e) * far ** t:
            d += 1
        first.append(d)
    return first


def exact(c, seed):
    s = prepare(c, seed)
    B, Tq, Tk, H, Hk, D = c["B"], c["Tq"], c["Tk"], c["H"], c["Hk"], c["D"]
    f64 = dict(dtype=torch.float64, device="cuda")
    n = c["buckets"] // 2 if c["two_sided"] else c["buckets"]
    e = n // 2
    border = torch.tensor(list(range(1, e)) + _first_distances(n, e, c["max_distance"]), device="cuda")  # first distance of bucket 1, 2, ...
    out, lse = torch.zeros(B, Tq, H, D, **f64), torch.full((B, H, Tq), NEG, **f64)
    dq, dk, dv = torch.zeros(B, Tq, H, D, **f64), torch.zeros(B, Tk, Hk, D, **f64), torch.zeros(B, Tk, Hk, D, **f64)
    dtable = torch.zeros(c["buckets"], H, **f64)
    for b, (ql, kl, off) in enumerate(zip(_q_lens(c), _k_lens(c), _offsets(c))):
        if ql == 0 or kl == 0:
            continue
        r = torch.arange(kl, device="cuda")[None, :] - torch.arange(off, off + ql, device="cuda")[:, None]
        place = torch.bucketize((r.abs() if c["two_sided"] else (-r).clamp_min(0)).contiguous(), border, right=True)
        if c["two_sided"]:
            place = place + n * (r > 0)
        for h in range(H):
            q, k, v = s["q"][b, :ql, h].double(), s["k"][b, :kl, h * Hk // H].double(), s["v"][b, :kl, h * Hk // H].double()
            x = q @ k.t() / math.sqrt(D) + s["table"][:, h].double()[place]
            if c["causal"]:
                x = x.masked_fill(r > 0, NEG)
            if c["op"] != "bwd":
                total = torch.logsumexp(x, 1)
                w = torch.exp(x - total.masked_fill(total == NEG, 0.0)[:, None])
                out[b, :ql, h], lse[b, h, :ql] = w @ v, total
                continue
            given = s["lse"][b, h, :ql].double()
            w = torch.exp(x - given.masked_fill(given == NEG, 0.0)[:, None])
            do = s["dout"][b, :ql, h].double()
            ds = w * (do @ v.t() - (do * s["out"][b, :ql, h].double()).sum(1, keepdim=True))
            dq[b, :ql, h] = ds @ k / math.sqrt(D)
            dk[b, :kl, h * Hk // H] += ds.t() @ q / math.sqrt(D)
            dv[b, :kl, h * Hk // H] += w.t() @ do
            for m in range(c["buckets"]):
                dtable[m, h] += torch.where(place == m, ds, 0.0).sum()
    if c["op"] == "bwd":
        return dq, dk, dv, dtable
    return (out, lse) if c["op"] == "fwd" else out
