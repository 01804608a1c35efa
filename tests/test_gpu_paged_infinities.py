"""Attention over pages whose visible V holds infinities, against the definition in float64: sum of p V with every p > 0, so a column
with infinities of one sign is that infinity, one with both signs or a NaN is NaN, and the others are what they are without them."""
import math

import pytest
import torch

from tests.test_gpu_paged import _cache, _gen

pytestmark = pytest.mark.gpu


def _definition(q, k, v, table, n, scale):
    """O and the room of a finite column, of one sequence of n rows in the pages of a table row."""
    Hq, D = q.shape
    Hkv, page = k.shape[1:3]
    rows = torch.arange(n, device="cuda")
    ids = table.long()[rows // page]
    assert bool(((ids >= 0) & (ids < k.shape[0])).all())
    kk, vv = (p[ids, :, rows % page].double().permute(1, 0, 2).contiguous() for p in (k, v))
    qq = q.double().view(Hkv, Hq // Hkv, D)
    s = torch.matmul(qq, kk.transpose(1, 2).contiguous()) * scale
    ds = (D + 2) * 2.0 ** -24 * scale * torch.matmul(qq.abs(), kk.abs().transpose(1, 2).contiguous()).amax(-1, keepdim=True)
    p = torch.softmax(s, -1)
    # as sums of products over the rows, one by one where an infinity is among them
    fine = torch.where(vv.isfinite(), vv, 0.0)
    o = torch.matmul(p, fine)
    up, down, nan = (x.any(1)[:, None, :].expand_as(o) for x in (vv == math.inf, vv == -math.inf, vv.isnan()))
    o = torch.where(up, math.inf, o)
    o = torch.where(down, -math.inf, o)
    o = torch.where(up & down | nan, math.nan, o)
    # an f32 sum's and the two parts' errors as in the tests of finite V, the rounding to bf16 (2^-8)
    room = 2.0 ** -8 * o.abs() + (2 * ds + 2.0 ** -15) * torch.matmul(p, fine.abs())
    return o.view(Hq, D), room.view(Hq, D)


def _compare(o, want, room, what):
    bad = ~want.isfinite()
    assert torch.equal(o[bad].float().nan_to_num(nan=7.0), want[bad].float().nan_to_num(nan=7.0)), what
    assert bool(((o.double() - want).abs()[~bad] <= room[~bad]).all()), what


# one block of query heads; waves side by side; two blocks a wave (a table wide enough for it); tables that are not cut
@pytest.mark.parametrize("Hq,Hkv,D,width", [(1, 1, 64, 200), (4, 4, 128, 200), (8, 2, 128, 200), (8, 2, 64, 200), (32, 1, 128, 200), (32, 1, 64, 9000),
                                            (17, 1, 64, 200), (8, 2, 128, 16), (8, 2, 64, 16), (32, 1, 128, 16)])
@pytest.mark.parametrize("seed", [1, 2])
def test_infinite_v_in_visible_rows(Hq, Hkv, D, width, seed):
    import tyr_amd
    lens_ = [1, 2, 20, 100, 256] if width == 16 else [1, 2, 20, 100, 700, 3001]
    g = _gen(seed)
    (k, v), table, _, _ = _cache(g, lens_, 16, Hkv, D, False, width=width)
    for b, n in enumerate(lens_):
        def put(row, col, x):
            v[table[b, row // 16].long(), :, row % 16, col] = x
        put(0, 3, math.inf)                             # the first row, the last, all of a column, some of both signs, a NaN beside
        put(n - 1, 5, -math.inf)
        for row in range(n):
            put(row, 7, -math.inf)
        for row in range(0, n, 3):
            put(row, 11, math.inf)
        put(n // 2, 13, math.inf)
        if n > 1:
            put(0, 17, math.inf)
            put(n - 1, 17, -math.inf)
        put(n // 3, 19, math.nan)
        if n % 16:                                      # rows that nobody sees may hold what they like
            v[table[b, n // 16].long(), :, n % 16:, 23] = math.inf
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
    q = torch.randn(len(lens_), Hq, 1, D, generator=g, device="cuda").bfloat16()
    scale = 1 / math.sqrt(D)
    o, lse = tyr_amd.paged_decode(q, k, v, table, lens)
    assert bool(lse.isfinite().all())
    for b, n in enumerate(lens_):
        _compare(o[b, :, 0], *_definition(q[b, :, 0], k, v, table[b], n, scale), (b, n))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [40, 2000])
@pytest.mark.parametrize("place", [0.0, 0.5, 1.0])
def test_infinite_v_in_rows_of_low_probability(D, n, place):
    """e^-60 of the largest, 2^-87, before rows that take the maximum and behind them."""
    import tyr_amd
    g = _gen(3)
    (k, v), table, _, _ = _cache(g, [n], 16, 1, D, False, width=200)
    k[...] = 0
    row = int(place * (n - 1))
    at = table[0, row // 16].long()
    k[at, 0, row % 16, 0] = -60.0
    v[at, 0, row % 16, 2::7] = math.inf
    v[at, 0, row % 16, 3::7] = -math.inf
    q = torch.zeros(1, 1, 1, D, device="cuda").bfloat16()
    q[..., 0] = 1.0
    o, _ = tyr_amd.paged_decode(q, k, v, table, torch.tensor([n], dtype=torch.int32, device="cuda"), scale=1.0)
    _compare(o[0, :, 0], *_definition(q[0, :, 0], k, v, table[0], n, 1.0), row)
