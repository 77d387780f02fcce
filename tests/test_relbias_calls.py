"""Attention with a bucketed relative-position bias, host side: the bucket tables shared by threads and the argument checks."""
import threading

import torch

from css_amd import ops


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
