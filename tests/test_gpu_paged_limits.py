"""A decode near the limits that the C ABI names, against float64 on the sequences that have rows."""
import math

import pytest
import torch

from tests.test_gpu_paged import _check, _gen

pytestmark = pytest.mark.gpu


def test_a_billion_steps_of_all_heads():
    """2^25 sequences in tables of 960 rows: 30 steps each are 1.007e9 of them, 33 with the turn from one to the next."""
    import tyr_amd
    B, D, width = 1 << 25, 64, 60
    g = _gen(1)
    k, v = (torch.randn(500, 1, 16, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    lens = torch.full((B,), 960, dtype=torch.int32, device="cuda")
    lens[1:-1] = 0
    some = [0, 1, 63, 64, 65, 1000003, B // 2, B - 65, B - 2, B - 1]
    for i, b in enumerate(some[1:-1]):
        lens[b] = 100 * i + 1
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    for b in some:
        table[b] = torch.randperm(500, generator=g, device="cuda")[:width].to(torch.int32)
    q = torch.ones(B, 1, 1, D, dtype=torch.bfloat16, device="cuda")
    for b in some:
        q[b] = torch.randn(1, 1, D, generator=g, device="cuda").bfloat16()
    o, lse = tyr_amd.paged_decode(q, k, v, table, lens)
    _check(o, lse, q, k, v, table, {b: int(lens[b]) for b in some}, 1 / math.sqrt(D), only=some)
    for t in (o, lse):
        t[torch.tensor(some, device="cuda")] = 0 if t is o else -math.inf
    assert not bool(o.view(torch.int16).any()) and bool((lse == -math.inf).all())
