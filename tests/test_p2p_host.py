"""The direct all-reduce's handshake where the runtime has no interprocess events, without a GPU: streams and events are stand-ins."""
import threading
import time

import numpy as np
import pytest
import torch

from css_amd import parallel


class NoRecord:
    def __init__(self, **kw):
        assert kw["interprocess"]

    def record(self, stream):
        raise RuntimeError("HIP error: invalid argument\nSearch for hipErrorInvalidValue")


class Recorded(NoRecord):
    def record(self, stream):
        self.on = stream


def test_refused_events_are_reported(monkeypatch):
    monkeypatch.setattr(torch.cuda, "Event", NoRecord)
    assert parallel.interprocess_events(3, "s") == (None, "HIP error: invalid argument")
    monkeypatch.setattr(torch.cuda, "Event", Recorded)
    events, reason = parallel.interprocess_events(3, "s")
    assert reason is None and [e.on for e in events] == ["s"] * 3


def ranks(world, timeout_s=20.0):
    seqs = np.zeros((parallel.P2PAllReduce.PHASES, world), dtype=np.int64)
    made = []
    for r in range(world):
        p = object.__new__(parallel.P2PAllReduce)
        p.rank, p.world, p.seq, p.by_events, p.timeout_s, p._seqs = r, world, 0, False, timeout_s, seqs
        made.append(p)
    return made


def test_host_handshake_publishes_only_finished_work():
    """every rank's work of a phase is done before any rank leaves the phase, call after call"""
    world, done, wrong = 3, [0, 0, 0], []

    class Stream:
        def __init__(self, r):
            self.r = r

        def synchronize(self):
            time.sleep(0.002 * (self.r + 1))
            done[self.r] += 1

    def rank(p):
        n = 0
        for _ in range(5):
            p.seq += 1
            for k in range(p.PHASES):
                n += 1
                p._phase(k, Stream(p.rank))
                if min(done) < n:
                    wrong.append((p.rank, n, list(done)))

    threads = [threading.Thread(target=rank, args=(p,)) for p in ranks(world)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and done == [15] * 3


def test_host_handshake_ends_where_a_rank_is_missing():
    class Stream:
        def synchronize(self):
            pass

    p = ranks(2, timeout_s=0.2)[0]
    p.seq = 1
    with pytest.raises(RuntimeError, match="rank 1 did not reach phase 0"):
        p._phase(0, Stream())
