"""The host side of the attention with a bucketed relative-position bias: the bucket map and the refusals that need no GPU."""
import math

import pytest
import torch

from css_amd import ops, ops_bwd


def formula(n, far, two, r):
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


@pytest.mark.parametrize("n,far,two", [(32, 128, True), (32, 128, False), (64, 256, True), (320, 800, True), (16, 40, True),
                                       (33, 77, False), (4, 2, True), (2, 1024, False), (512, 1024, True), (2048, 1024, True)])
def test_bucket_map_is_the_formula(n, far, two):
    if n == 2048:  # half of a side's buckets must stay below the largest distance
        far = 513
    m = ops.relbias_bucket_map(n, far, two)
    assert m == [formula(n, far, two, r) for r in range(-far, far + 1)]
    assert min(m) >= 0 and max(m) < n
    runs = [b for i, b in enumerate(m) if i == 0 or m[i - 1] != b]
    assert len(runs) == len(set(runs))  # a bucket's distances are contiguous


def test_bucket_map_refusals():
    for n, far, two in ((31, 128, True), (2, 128, True), (1, 128, False), (32, 8, True), (32, 1025, True), (32, 16, False)):
        with pytest.raises(RuntimeError):
            ops.relbias_bucket_map(n, far, two)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    table = torch.zeros(32, 2)
    with pytest.raises(RuntimeError):
        ops.mha_relbias(q, q, q, table, (32, 128))
    with pytest.raises(RuntimeError):
        ops_bwd.mha_relbias_bwd(q, q, q, table, q, torch.zeros(1, 2, 4), q, (32, 128))
