"""Batches of many heads in which one sequence, or a few, have most of the rows, and so most of the partial results, against float64."""
import math

import pytest
import torch

from tests.test_gpu_paged import _cache, _check, _gen

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,D,e4m3", [(1, 1, 128, False), (8, 1, 128, False), (8, 1, 64, False), (6, 2, 128, True), (16, 1, 64, True), (32, 1, 128, False),
                                           (32, 1, 128, True), (34, 1, 64, False), (3, 3, 128, False)])
@pytest.mark.parametrize("longest", [2100, 9000, 60000])
@pytest.mark.parametrize("others", [0, 20, 700])
def test_one_long_sequence_beside_many(Hq, Hkv, D, e4m3, longest, others):
    import tyr_amd
    g = _gen(longest + others + Hq)
    lens_ = [(others * (i % 7)) // 3 for i in range(70)]
    lens_[33], lens_[34], lens_[69] = longest, longest // 2, longest // 5
    (k, v), table, ks, vs = _cache(g, lens_, 16, Hkv, D, e4m3)
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
    q = torch.randn(70, Hq, 1, D, generator=g, device="cuda").bfloat16()
    o, lse = tyr_amd.paged_decode(q, k, v, table, lens, k_scale=ks, v_scale=vs)
    _check(o, lse, q, k, v, table, lens_, 1 / math.sqrt(D), ks=ks, vs=vs, only=[0, 1, 6, 32, 33, 34, 35, 68, 69])
    again = tyr_amd.paged_decode(q, k, v, table, lens, k_scale=ks, v_scale=vs)
    assert torch.equal(again[0], o) and torch.equal(again[1], lse)


@pytest.mark.parametrize("Hq,Hkv", [(8, 1), (5, 5)])
def test_captured_batch_whose_lengths_become_one_sequence_s(Hq, Hkv):
    """Which heads are joined by a wave and which by four follows the lengths of the replay."""
    import tyr_amd
    B, D, n = 64, 128, 30000
    g = _gen(3)
    (k, v), table, _, _ = _cache(g, [n] + [1000] * (B - 1), 16, Hkv, D, False)
    q = torch.randn(B, Hq, 1, D, generator=g, device="cuda").bfloat16()
    lens = torch.full((B,), 1000, dtype=torch.int32, device="cuda")
    tyr_amd.paged_decode(q, k, v, table, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = tyr_amd.paged_decode(q, k, v, table, lens)
    for first, rest in ((1000, 1000), (n, 7), (n, 1000), (3, 900), (n, 0), (0, 0), (n, 40)):
        lens[0], lens[1:] = first, rest
        o.zero_(), lse.zero_()
        want = tyr_amd.paged_decode(q, k, v, table, lens)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1]), (first, rest)
        _check(o, lse, q, k, v, table, lens.tolist(), 1 / math.sqrt(D), only=[0, 1, 63])
