"""Attention with a bucketed relative-position bias, host side: the bucket tables shared by threads and the argument checks."""
import threading

import pytest
import torch

from css_amd import _lib, ops


def test_two_threads_at_first_use_get_the_tables_that_are_kept(monkeypatch):
    """A launch holds the tables by address: what a caller is handed has to be what stays, also where two threads build at once."""
    both = threading.Barrier(2, timeout=60)
    build = ops.relbias_bucket_map

    def slow(*args):
        both.wait()  # neither returns before the other has begun
        return build(*args)

    monkeypatch.setattr(ops, "relbias_bucket_map", slow)
    monkeypatch.setattr(ops, "_RELBIAS_BUCKETS", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    got = [None, None]

    def use(n):
        got[n] = ops.relbias_buckets((32, 113, True), torch.device("cpu"))

    threads = [threading.Thread(target=use, args=(n,)) for n in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    (kept,) = ops._RELBIAS_BUCKETS.values()
    for g in got:
        assert g is not None and all(a is b for a, b in zip(g, kept))


def packed(B, Tq, Tk, H, Hk, D, n, q_stride=None, k_stride=None):
    """csship_relbias with addresses that are never used"""
    q_stride, k_stride = q_stride or (Tq * H * D, H * D, D), k_stride or (Tk * Hk * D, Hk * D, D)
    return _lib.RELBIAS.pack(256, 256, 256, *q_stride, *k_stride, *k_stride, 256, 256, 256, 0, 0, 0, _lib.RELBIAS_BF16, B, Tq, Tk, H, Hk, D,
                             n, 128, 0, 0, 1.0)


def test_tables_beyond_32_bit_indexes_are_refused():
    """heads x buckets number the table's entries in 32 bits in the kernels, and the backward's grid by waves"""
    h, bad = _lib.lib(), -1
    s3 = _lib.STRIDE3.pack(8, 8, 8)
    for H, n, fwd, bwd in ((600000, 4094, False, False), (65536, 32767, True, False), (4096, 16384, True, False), (4096, 16383, True, True)):
        p = packed(1, 1, 1, H, 1, 8, n, q_stride=(H * 8, H * 8, 8))
        # a null result is refused only behind the shape: nothing is launched either way
        assert (h.csship_relbias_fwd(p, None, s3, None, None, 0, None) == bad) == (not fwd)
        assert (h.csship_relbias_bwd(p, *[256, s3, 256, 256, s3, 256, s3, 256, s3, 256, s3], None, 256, 0, None) == bad) == (not bwd)


@pytest.mark.parametrize("buckets", [(32, 128, True, 4), (32,), (32.5, 128), (32, 128.5, True), ("32", 128), 32, None])
def test_malformed_bucket_settings_are_refused(buckets, monkeypatch):
    """not cut to the first three, not rounded"""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with pytest.raises((RuntimeError, TypeError), match="buckets"):
        ops.relbias_buckets(buckets, torch.device("cpu"))


def test_tables_made_ahead_serve_the_device_that_is_meant(monkeypatch):
    """a capture is prepared by ops.relbias_buckets(settings, "cuda"): the entry a tensor's device finds is that one"""
    monkeypatch.setattr(ops, "_RELBIAS_BUCKETS", {})
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch, "tensor", lambda x, dtype, make=torch.tensor: type("T", (), {"to": lambda self, d: make(x, dtype=dtype)})())
    kept = ops.relbias_buckets((32, 128), torch.device("cuda", 0))
    assert len(ops._RELBIAS_BUCKETS) == 1
    for device in ("cuda", "cuda:0", torch.device("cuda"), 0):
        assert ops.relbias_buckets((32, 128), device) is kept
    assert len(ops._RELBIAS_BUCKETS) == 1
