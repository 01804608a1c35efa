"""The cache in pages: appending to it and attention of one token over it, against float64 on the same rows.

Tolerance of the attention.  A score is an f32 sum of D exact products: off by at most ds = (D + 2) 2^-24 scale sum |q_i k_i|, so a
probability by a factor 1 +- 2 ds (its own score and the sum's).  exp2, the joins of pieces and the two-part probabilities are below
2^-15.  O is then rounded once to bf16, 2^-8 of its size.  LSE: ds, and 2^-17 for its sum and logarithm."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(g, lens, page, Hkv, D, e4m3, spare=3, width=None):
    """Pools with every row written (hidden ones too), a table in random order with -1 behind each sequence's pages, factors."""
    need = [-(-max(0, n) // page) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width or max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    pools = [torch.randn(total, Hkv, page, D, generator=g, device="cuda") for _ in range(2)]
    if not e4m3:
        return [p.bfloat16() for p in pools], table, None, None
    ks, vs = ((0.75 + 0.5 * torch.rand(Hkv, generator=g, device="cuda")) / 100.0 for _ in range(2))
    return [(p / s[:, None, None]).clamp(-448, 448).to(E4M3) for p, s in zip(pools, (ks, vs))], table, ks, vs


def _seen(n, window, sinks):
    rows = torch.arange(max(0, n), device="cuda")
    return rows if not window else rows[(rows < sinks) | (rows >= n - window)]


def _check(o, lse, q, k, v, table, lens, scale, window=0, sinks=0, ks=None, vs=None, only=None):
    B, Hq, _, D = q.shape
    P, Hkv, page, _ = k.shape
    G = Hq // Hkv
    for b in (range(B) if only is None else only):
        n = min(max(0, int(lens[b])), table.shape[1] * page)
        rows = _seen(n, window, sinks)
        ids = table[b].long()[rows // page]
        there = (ids >= 0) & (ids < P)
        rows, ids = rows[there], ids[there]
        if rows.numel() == 0:
            assert not bool(o[b].float().any()) and bool((lse[b] == -math.inf).all()), b
            continue
        kk, vv = (p[ids, :, rows % page].double().permute(1, 0, 2).contiguous() for p in (k, v))          # [Hkv, rows, D]
        if ks is not None:
            kk, vv = kk * ks.double()[:, None, None], vv * vs.double()[:, None, None]
        qq = q[b, :, 0].double().view(Hkv, G, D)
        s = torch.matmul(qq, kk.transpose(1, 2).contiguous()) * scale
        ds = (D + 2) * 2.0 ** -24 * scale * torch.matmul(qq.abs(), kk.abs().transpose(1, 2).contiguous()).amax(-1, keepdim=True)
        want_l = torch.logsumexp(s, -1)
        p = torch.exp(s - want_l[..., None])
        want = torch.matmul(p, vv)
        room = 2.0 ** -8 * want.abs() + (2 * ds + 2.0 ** -15) * torch.matmul(p, vv.abs())
        off = (o[b, :, 0].double().view(Hkv, G, D) - want).abs()
        assert bool((off <= room).all()), (b, n, float((off - room).max()))
        off_l = (lse[b].double().view(Hkv, G) - want_l).abs()
        assert bool((off_l <= ds[..., 0] + 2.0 ** -17 * (1 + want_l.abs())).all()), (b, n, float(off_l.max()))


LENS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 100, 127, 129, 255, 257, 500, 1000, 3001]


@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (8, 2), (32, 8), (16, 1), (34, 2), (48, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 48, 256])
@pytest.mark.parametrize("e4m3", [False, True])
def test_decode_lengths_heads_and_pages(Hq, Hkv, D, page, e4m3):
    import tyr_amd
    g = _gen(Hq * 1000 + D + page)
    (k, v), table, ks, vs = _cache(g, LENS, page, Hkv, D, e4m3)
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    q = torch.randn(len(LENS), Hq, 1, D, generator=g, device="cuda").bfloat16()
    o, lse = tyr_amd.paged_decode(q, k, v, table, lens, k_scale=ks, v_scale=vs)
    _check(o, lse, q, k, v, table, LENS, 1 / math.sqrt(D), ks=ks, vs=vs)


@pytest.mark.parametrize("Hq,Hkv", [(17, 1), (32, 1), (66, 2), (33, 1), (130, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("rows", [256, 3100, 70000])
def test_decode_many_query_heads_of_a_kv_head(Hq, Hkv, D, e4m3, rows):
    """Blocks of query heads, apart and together, and waves side by side: which of them depends on the tables' width."""
    import tyr_amd
    lens_ = [0, 1, 17, 31, 33, 100, rows // 2 - 5, 255, rows]
    g = _gen(Hq * 31 + D + rows)
    (k, v), table, ks, vs = _cache(g, lens_, 16, Hkv, D, e4m3, width=-(-rows // 16))
    copies = 8 if rows == 70000 else 1               # the same sequences again
    lens_ = lens_ * copies
    table = table.repeat(copies, 1)
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
    q = torch.randn(len(lens_), Hq, 1, D, generator=g, device="cuda").bfloat16()
    for window, sinks in ((0, 0), (300, 7), (60, 0)):
        o, lse = tyr_amd.paged_decode(q, k, v, table, lens, window=window, sinks=sinks, k_scale=ks, v_scale=vs)
        _check(o, lse, q, k, v, table, lens_, 1 / math.sqrt(D), window, sinks, ks, vs, only=range(9 * copies - 9, 9 * copies) if copies > 1 else None)
        again, lse2 = tyr_amd.paged_decode(q, k, v, table, lens, window=window, sinks=sinks, k_scale=ks, v_scale=vs)
        assert torch.equal(o, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("D,e4m3", [(64, False), (64, True), (128, False), (128, True)])
def test_decode_many_short_sequences_of_many_query_heads(D, e4m3):
    import tyr_amd
    lens_ = [(37 * i) % 257 for i in range(2050)]
    g = _gen(21 + D)
    (k, v), table, ks, vs = _cache(g, lens_, 16, 1, D, e4m3, width=16)
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
    q = torch.randn(2050, 20, 1, D, generator=g, device="cuda").bfloat16()
    o, lse = tyr_amd.paged_decode(q, k, v, table, lens, k_scale=ks, v_scale=vs)
    _check(o, lse, q, k, v, table, lens_, 1 / math.sqrt(D), ks=ks, vs=vs, only=[*range(0, 2050, 41), 2049])


@pytest.mark.parametrize("Hq,Hkv,D", [(4, 4, 128), (8, 2, 64), (34, 2, 128), (16, 1, 64)])
@pytest.mark.parametrize("page,rows", [(16, 256), (48, 240), (256, 256), (16, 272)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_decode_short_tables(Hq, Hkv, D, page, rows, e4m3):
    """Tables up to and just beyond the rows from which sequences are cut, also more of them than lanes."""
    import tyr_amd
    lens_ = [0, 1, 15, 16, 17, 100, 129, rows - 1, rows] * 8
    g = _gen(Hq * 7 + D + page + rows)
    (k, v), table, ks, vs = _cache(g, lens_, page, Hkv, D, e4m3, width=-(-rows // page))
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
    q = torch.randn(len(lens_), Hq, 1, D, generator=g, device="cuda").bfloat16()
    for window, sinks in ((0, 0), (60, 5)):
        o, lse = tyr_amd.paged_decode(q, k, v, table, lens, window=window, sinks=sinks, k_scale=ks, v_scale=vs)
        _check(o, lse, q, k, v, table, lens_, 1 / math.sqrt(D), window, sinks, ks, vs)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (17, 16), (100, 0), (100, 17), (1000, 64), (33, 300), (5000, 4), (2 ** 40, 2 ** 40)])
@pytest.mark.parametrize("page,e4m3,D", [(16, False, 128), (48, True, 128), (64, False, 64)])
def test_decode_windows_and_sinks(window, sinks, page, e4m3, D):
    import tyr_amd
    g = _gen(window % 1000 + sinks % 1000 + page)
    (k, v), table, ks, vs = _cache(g, LENS, page, 2, D, e4m3)
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    q = torch.randn(len(LENS), 8, 1, D, generator=g, device="cuda").bfloat16()
    # pages between the sinks and the window may be anything: given back, or another sequence's
    for b, n in enumerate(LENS):
        for p in range(table.shape[1]):
            if not bool(((_seen(n, window, sinks) // page) == p).any()):
                table[b, p] = [-1, 2 ** 31 - 1, -2 ** 31, 0][(b + p) % 4]
    o, lse = tyr_amd.paged_decode(q, k, v, table, lens, scale=0.11, window=window, sinks=sinks, k_scale=ks, v_scale=vs)
    _check(o, lse, q, k, v, table, LENS, 0.11, window, sinks, ks, vs)
    if window > 3001:
        whole = tyr_amd.paged_decode(q, k, v, table, lens, scale=0.11, k_scale=ks, v_scale=vs)
        assert torch.equal(o, whole[0]) and torch.equal(lse, whole[1])


def test_window_beyond_64_bits_is_all_rows():
    import tyr_amd
    g = _gen(78)
    (k, v), table, _, _ = _cache(g, [700], 16, 2, 64, False)
    lens = torch.tensor([700], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 1, 64, generator=g, device="cuda").bfloat16()
    want = tyr_amd.paged_decode(q, k, v, table, lens)
    for n in (2 ** 31 - 1, 2 ** 63, 2 ** 64 + 5):
        got = tyr_amd.paged_decode(q, k, v, table, lens, window=n, sinks=n)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(tyr_amd.TyrGpuError, match="negative"):
        tyr_amd.paged_decode(q, k, v, table, lens, window=-2 ** 70)


@pytest.mark.parametrize("e4m3", [False, True])
def test_what_hidden_rows_hold_does_not_matter(e4m3):
    import tyr_amd
    page, D, lens_ = 16, 128, [5, 40, 300, 777]
    g = _gen(77)
    (k, v), table, ks, vs = _cache(g, lens_, page, 2, D, e4m3)
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
    q = torch.randn(4, 8, 1, D, generator=g, device="cuda").bfloat16()
    args = dict(window=130, sinks=3, k_scale=ks, v_scale=vs)
    want = tyr_amd.paged_decode(q, k, v, table, lens, **args)
    seen = torch.zeros(k.shape[0], page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens_):
        rows = _seen(n, 130, 3)
        seen[table[b].long()[rows // page], rows % page] = True
    for fill in ([float("nan")] if e4m3 else [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min]):
        for pool in (k, v):
            f = pool.float()
            f[~seen[:, None, :].expand(-1, 2, -1)] = fill
            pool.copy_(f.to(pool.dtype))
        got = tyr_amd.paged_decode(q, k, v, table, lens, **args)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), fill


def test_nan_in_a_visible_row_is_seen():
    import tyr_amd
    g = _gen(5)
    for lens_ in ([3, 700], [3, 100]):                  # in pieces, and whole
        (k, v), table, _, _ = _cache(g, lens_, 16, 1, 64, False)
        lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
        q = torch.randn(2, 1, 1, 64, generator=g, device="cuda").bfloat16()
        k[table[1, 2].long(), 0, 5] = float("nan")
        o, lse = tyr_amd.paged_decode(q, k, v, table, lens)
        assert bool(o[1].isnan().all()) and bool(lse[1].isnan().all()) and not bool(o[0].isnan().any())


def test_pages_outside_the_pool_and_lengths_outside_the_table():
    import tyr_amd
    lens_ = [64, 200, 333, 80, 48]
    g = _gen(6)
    (k, v), table, _, _ = _cache(g, lens_, 16, 2, 128, False, width=30)
    table[0, :4] = torch.tensor([-1, -7, k.shape[0], 2 ** 31 - 1], dtype=torch.int32)      # nothing there
    table[1, 3] = k.shape[0] + 5
    table[2, 20] = -1                                                            # the last, part of a page
    given = torch.tensor([64, 200, 333, 2 ** 31 - 1, -5], dtype=torch.int32, device="cuda")
    q = torch.randn(5, 4, 1, 128, generator=g, device="cuda").bfloat16()
    o, lse = tyr_amd.paged_decode(q, k, v, table, given)
    _check(o, lse, q, k, v, table, given.tolist(), 1 / math.sqrt(128))
    assert bool((lse[4] == -math.inf).all())


@pytest.mark.parametrize("B,longest,Hq,Hkv", [(1, 20000, 8, 2), (1, 33000, 2, 1), (63, 900, 4, 4), (64, 900, 4, 4), (65, 900, 4, 4), (200, 2000, 8, 2), (1500, 300, 2, 2),
                                              (3, 5000, 1200, 600)])
def test_batches_of_unequal_lengths(B, longest, Hq, Hkv):
    """One sequence in hundreds of pieces; batches that the search for a piece walks in several rounds; more heads than the aim of pieces."""
    import tyr_amd
    D = 64
    g = _gen(B)
    lens_ = [max(0, round(longest ** (i / max(1, B - 1))) - 1) if B > 1 else longest for i in torch.randperm(B).tolist()]
    (k, v), table, _, _ = _cache(g, lens_, 32, Hkv, D, False)
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
    q = torch.randn(B, Hq, 1, D, generator=g, device="cuda").bfloat16()
    o, lse = tyr_amd.paged_decode(q, k, v, table, lens)
    _check(o, lse, q, k, v, table, lens_, 1 / math.sqrt(D), only=range(0, B, max(1, B // 40)))
    again = tyr_amd.paged_decode(q, k, v, table, lens)
    assert torch.equal(o, again[0]) and torch.equal(lse, again[1])


@pytest.mark.parametrize("e4m3", [False, True])
def test_far_pages(e4m3):
    """Pages beyond 4 GiB of a pool: 2^32 bytes and more from its start, written by the append and read."""
    import tyr_amd
    Hkv, page, D = 8, 64, 128
    P = (9 << 30 if e4m3 else 9 << 29) // (Hkv * page * D)           # 9 GiB a pool
    k, v = (torch.empty(P, Hkv, page, D, dtype=E4M3 if e4m3 else torch.bfloat16, device="cuda") for _ in range(2))
    n = 200
    table = torch.tensor([[P - 1, P // 2, 0, P - 2], [P - 3, 1, P // 2 + 1, P - 4]], dtype=torch.int32, device="cuda")
    g = _gen(9)
    kn, vn = (torch.randn(2, n, Hkv, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(2, n, 8, D, generator=g, device="cuda").bfloat16()
    cos, sin = torch.ones(n, D // 2, device="cuda"), torch.zeros(n, D // 2, device="cuda")
    ks = vs = torch.full((Hkv,), 1 / 64, device="cuda") if e4m3 else None
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    qr = tyr_amd.paged_rope_append(q, kn, vn, cos, sin, k, v, table, pos, k_scale=ks, v_scale=vs)
    assert torch.equal(qr, q)
    j = torch.arange(n, device="cuda")
    for pool, new, s in ((k, kn, ks), (v, vn, vs)):
        for b in range(2):
            got = pool.view(torch.uint8 if e4m3 else torch.int16)[table[b].long()[j // page], :, j % page]
            want = (new[b].float() / s[:, None]).to(E4M3).view(torch.uint8) if e4m3 else new[b].view(torch.int16)
            assert torch.equal(got, want)
    lens = torch.tensor([n, n - 9], dtype=torch.int32, device="cuda")
    qd = q[:, -1].contiguous().view(2, 8, 1, D)
    o, lse = tyr_amd.paged_decode(qd, k, v, table, lens, k_scale=ks, v_scale=vs)
    _check(o, lse, qd, k, v, table, lens.tolist(), 1 / math.sqrt(D), ks=ks, vs=vs)


def test_e4m3_pages_without_factors():
    import tyr_amd
    g = _gen(10)
    (k, v), table, _, _ = _cache(g, [300, 20], 16, 2, 128, True)
    lens = torch.tensor([300, 20], dtype=torch.int32, device="cuda")
    q = (torch.randn(2, 4, 1, 128, generator=g, device="cuda") / 64).bfloat16()
    one = torch.ones(2, device="cuda")
    for a, b in ((None, None), (one, None), (None, one), (one, one)):
        o, lse = tyr_amd.paged_decode(q, k, v, table, lens, k_scale=a, v_scale=b)
        _check(o, lse, q, k, v, table, [300, 20], 1 / math.sqrt(128), ks=one, vs=one)


@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 5)])
def test_factors_of_zero_and_below(window, sinks):
    """A kv head of factor 0 has scores of 0 (its rows count alike) or values of 0; a negative factor turns them round.  What is hidden
    stays hidden."""
    import tyr_amd
    lens_ = [1, 17, 100, 777]
    g = _gen(12)
    (k, v), table, ks, vs = _cache(g, lens_, 16, 3, 128, True)
    ks[0], vs[1] = 0.0, 0.0
    ks[2], vs[2] = -ks[2], -vs[2]
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
    q = torch.randn(4, 12, 1, 128, generator=g, device="cuda").bfloat16()
    o, lse = tyr_amd.paged_decode(q, k, v, table, lens, window=window, sinks=sinks, k_scale=ks, v_scale=vs)
    _check(o, lse, q, k, v, table, lens_, 1 / math.sqrt(128), window, sinks, ks, vs)


def test_equals_the_contiguous_decode():
    """The same rows in a contiguous cache: both are within their rounding of the same result."""
    import tyr_amd
    B, Hq, Hkv, L, D, page = 3, 16, 4, 1000, 128, 16
    g = _gen(11)
    kc, vc = (torch.randn(B, Hkv, L, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn(B, Hq, 1, D, generator=g, device="cuda").bfloat16()
    width = -(-L // page)
    order = torch.randperm(B * width, generator=g, device="cuda")
    table = order.to(torch.int32).view(B, width)
    k, v = (torch.zeros(B * width, Hkv, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    j = torch.arange(L, device="cuda")
    for b in range(B):
        for pool, c in ((k, kc), (v, vc)):
            pool[table[b].long()[j // page], :, j % page] = c[b].transpose(0, 1)
    lens = torch.tensor([1000, 1, 537], dtype=torch.int32, device="cuda")
    for window in (0, 200):
        o, lse = tyr_amd.paged_decode(q, k, v, table, lens, window=window)
        wo, wl = tyr_amd.gqa_decode(q, kc, vc, kv_lens=lens, window=window)
        assert float((o.float() - wo.float()).abs().max()) <= 2e-2 and float((lse - wl).abs().max()) <= 1e-3


# ---- append


def _rotate(x, c, s):
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * c - b * s, a * s + b * c), -1)


@pytest.mark.parametrize("T", [1, 5, 100])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 128, 16), (3, 3, 64, 48), (16, 1, 128, 64)])
@pytest.mark.parametrize("e4m3", [False, True])
def test_append(T, Hq, Hkv, D, page, e4m3):
    """Rows that are written bit for bit, every other row as it was: padding, a free place of the batch, tokens beyond the tables and on
    pages that are not there."""
    import tyr_amd
    first = [0, 15, 16, 47, 300, -1, -2 ** 31, 411 - T, 460, 2 ** 31 - 1]
    new = [T, max(0, T - 1), T, 0, T, T, T, T, T, T]
    B, S, width = len(first), 470, -(-512 // page)
    g = _gen(T * 7 + page)
    total = B * width + 2
    table = torch.randperm(total, generator=g, device="cuda")[:B * width].to(torch.int32).view(B, width)
    table[4, 300 // page] = -1
    table[2, 16 // page] = total
    dtype = E4M3 if e4m3 else torch.bfloat16
    pools = [torch.randn(total, Hkv, page, D, generator=g, device="cuda").to(dtype) for _ in range(2)]
    before = [p.clone() for p in pools]
    q, kn, vn = (torch.randn(B, T, h, D, generator=g, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv))
    ang = torch.randn(S, D // 2, generator=g, device="cuda")
    cos, sin = torch.cos(ang), torch.sin(ang)
    ks, vs = ((0.5 + torch.rand(Hkv, generator=g, device="cuda")) / 50 for _ in range(2)) if e4m3 else (None, None)
    pos, lens = (torch.tensor(t, dtype=torch.int32, device="cuda") for t in (first, new))
    kept = q.clone()
    qr = tyr_amd.paged_rope_append(q, kn, vn, cos, sin, *pools, table, pos, new_lens=lens, k_scale=ks, v_scale=vs)
    assert torch.equal(q, kept) and qr.shape == q.shape
    for b in range(B):
        for t in range(T):
            p = first[b] + t
            if first[b] < 0 or p >= S:
                assert not bool(qr[b, t].float().any())
                continue
            assert torch.equal(qr[b, t], _rotate(q[b, t], cos[p], sin[p]).bfloat16())
            page_of = int(table[b, p // page]) if p // page < width else -1
            if t >= new[b] or not 0 <= page_of < total:
                continue
            for i, (x, s) in enumerate(((_rotate(kn[b, t], cos[p], sin[p]), ks), (vn[b, t].float(), vs))):
                before[i].view(torch.uint8 if e4m3 else torch.int16)[page_of, :, p % page] = (
                    (x / s[:, None]).clamp(-448, 448).to(E4M3).view(torch.uint8) if e4m3 else x.bfloat16().view(torch.int16))
    for a, b in zip(pools, before):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_append_without_lengths_equals_the_contiguous_append():
    import tyr_amd
    B, Hq, Hkv, L, D, pos = 3, 8, 2, 64, 128, 37
    g = _gen(12)
    q, kn, vn = (torch.randn(B, h, 1, D, generator=g, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv))
    ang = torch.randn(L, D // 2, generator=g, device="cuda")
    cos, sin = torch.cos(ang), torch.sin(ang)
    kc, vc = (torch.randn(B, Hkv, L, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    k, v = kc.clone(), vc.clone()                         # one page a sequence: the same memory layout
    table = torch.arange(B, dtype=torch.int32, device="cuda").view(B, 1)
    want = tyr_amd.decode_rope_append(q, kn, vn, cos[pos:pos + 1].contiguous(), sin[pos:pos + 1].contiguous(), kc, vc, pos)
    got = tyr_amd.paged_rope_append(q.view(B, 1, Hq, D), kn.view(B, 1, Hkv, D), vn.view(B, 1, Hkv, D), cos, sin, k, v, table,
                                    torch.full((B,), pos, dtype=torch.int32, device="cuda"))
    assert torch.equal(got.view(want.shape), want) and torch.equal(k, kc) and torch.equal(v, vc)


def test_append_saturates_and_keeps_nan():
    import tyr_amd
    D = 64
    q = torch.ones(1, 1, 1, D, device="cuda").bfloat16()
    x = q.clone()
    x[..., :4] = torch.tensor([1e4, -1e4, float("nan"), float("inf")])
    cos, sin = torch.ones(1, D // 2, device="cuda"), torch.zeros(1, D // 2, device="cuda")
    k, v = (torch.zeros(1, 1, 16, D, device="cuda").to(E4M3) for _ in range(2))
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    tyr_amd.paged_rope_append(q, q, x, cos, sin, k, v, zero.view(1, 1), zero)
    row = v[0, 0, 0].float()
    assert row[:2].tolist() == [448.0, -448.0] and bool(row[2].isnan()) and float(row[3]) == 448.0 and bool((row[4:] == 1).all())


# ---- together


@pytest.mark.parametrize("e4m3", [False, True])
def test_generation_over_pages(e4m3):
    """A prompt batch of unequal lengths and then ten tokens, one layer as a server runs it: norm to e4m3, quantised projection,
    rotate and append, paged attention, projection, norm.  Attention is checked at every step against float64 over the rows that the
    cache holds, whose bytes are checked against the new tokens'; the products against the float64 of their operands."""
    import tyr_amd
    B, Hq, Hkv, D, page, d = 3, 8, 2, 64, 16, 512
    prompt = [37, 5, 64]
    T, steps, S = max(prompt), 10, 128
    g = _gen(20)
    w_norm = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).bfloat16()
    n_out = (Hq + 2 * Hkv) * D
    wq, sw = tyr_amd.quantize_e4m3(torch.randn(n_out, d, generator=g, device="cuda") * d ** -0.5)
    col = torch.full((n_out,), sw, device="cuda")
    wo = (torch.randn(d, Hq * D, generator=g, device="cuda") * (Hq * D) ** -0.5).bfloat16()
    ang = torch.outer(torch.arange(S, device="cuda", dtype=torch.float32), 10000.0 ** (-torch.arange(0, D, 2, device="cuda") / D))
    cos, sin = torch.cos(ang), torch.sin(ang)
    width = S // page
    table = torch.randperm(B * width, generator=g, device="cuda").to(torch.int32).view(B, width)
    k, v = (torch.zeros(B * width, Hkv, page, D, device="cuda").to(E4M3 if e4m3 else torch.bfloat16) for _ in range(2))
    ks, vs = (torch.full((Hkv,), 1 / 64, device="cuda") for _ in range(2)) if e4m3 else (None, None)

    def project(x, resid):
        rows = x.shape[0]
        a, s, h = tyr_amd.rmsnorm_residual_fp8(x, resid, w_norm)
        qkv = tyr_amd.gemm_fp8_scaled(a, wq, s, col, out_dtype=torch.bfloat16, trans_b=True)
        want = (a.double() * s.double()[:, None]) @ (wq.double() * sw).t().contiguous()
        # f32 sums of 512 exact products, one rounding
        size = (a.double() * s.double()[:, None]).abs() @ (wq.double() * sw).abs().t().contiguous()
        assert bool(((qkv.double() - want).abs() <= 2.0 ** -8 * want.abs() + 520 * 2.0 ** -24 * size).all())
        return [t.contiguous() for t in qkv.split([Hq * D, Hkv * D, Hkv * D], 1)], h

    def stored(row, s):
        return row if s is None else (row.float() / s[:, None]).clamp(-448, 448).to(E4M3)

    x = torch.randn(B * T, d, generator=g, device="cuda").bfloat16()
    (qp, kp, vp), _ = project(x, torch.zeros_like(x))
    lens = torch.tensor(prompt, dtype=torch.int32, device="cuda")
    pos = torch.zeros(B, dtype=torch.int32, device="cuda")
    tyr_amd.paged_rope_append(qp.view(B, T, Hq, D), kp.view(B, T, Hkv, D), vp.view(B, T, Hkv, D), cos, sin, k, v, table, pos, new_lens=lens,
                              k_scale=ks, v_scale=vs)
    x, resid = torch.randn(B, d, generator=g, device="cuda").bfloat16(), torch.randn(B, d, generator=g, device="cuda").bfloat16()
    for step in range(steps):
        (q1, k1, v1), h = project(x, resid)
        qr = tyr_amd.paged_rope_append(q1.view(B, 1, Hq, D), k1.view(B, 1, Hkv, D), v1.view(B, 1, Hkv, D), cos, sin, k, v, table, lens,
                                       k_scale=ks, v_scale=vs)
        for b in range(B):
            at = prompt[b] + step
            got = v[table[b, at // page].long(), :, at % page]
            assert torch.equal(got.view(torch.uint8), stored(v1.view(B, Hkv, D)[b], vs).view(torch.uint8))
        lens = lens + 1
        qd = qr.view(B, Hq, 1, D)
        o, lse = tyr_amd.paged_decode(qd, k, v, table, lens, window=40, sinks=2, k_scale=ks, v_scale=vs)
        _check(o, lse, qd, k, v, table, lens.tolist(), 1 / math.sqrt(D), 40, 2, ks, vs)
        x, resid = tyr_amd.gemm_bf16(o.view(B, Hq * D), wo, trans_b=True), h


def test_captured_step_follows_lengths_and_pages():
    """One captured step replayed while lengths, positions and the table change in place: each replay equals the eager call."""
    import tyr_amd
    B, Hq, Hkv, D, page, S = 5, 8, 2, 128, 16, 2048
    g = _gen(21)
    width = S // page
    table = torch.randperm(B * width, generator=g, device="cuda").to(torch.int32).view(B, width).contiguous()
    k0, v0 = (torch.randn(B * width, Hkv, page, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    q, kn, vn = (torch.randn(B, 1, h, D, generator=g, device="cuda").bfloat16() for h in (Hq, Hkv, Hkv))
    ang = torch.randn(S, D // 2, generator=g, device="cuda")
    cos, sin = torch.cos(ang), torch.sin(ang)
    pos, lens = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))

    def step(k, v):
        qr = tyr_amd.paged_rope_append(q, kn, vn, cos, sin, k, v, table, pos)
        return tyr_amd.paged_decode(qr.view(B, Hq, 1, D), k, v, table, lens)
    kg, vg = k0.clone(), v0.clone()
    step(kg, vg)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = step(kg, vg)
    for replay, at in enumerate(([0, 1, 2, 3, 4], [100, 2047, 16, 15, 1000], [-1, 5, 2000, 2000, 2000], [7, 7, 7, 7, 7])):
        pos.copy_(torch.tensor(at, dtype=torch.int32))
        lens.copy_(pos + 1)
        table.copy_(table.flip(0))
        kg.copy_(k0)
        vg.copy_(v0)
        ke, ve = k0.clone(), v0.clone()
        want = step(ke, ve)
        o.zero_()
        lse.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1]) and torch.equal(kg, ke) and torch.equal(vg, ve), replay


@pytest.mark.parametrize("Hq,D,e4m3,width", [(32, 128, False, 200), (33, 128, False, 200), (32, 128, True, 9000), (40, 64, False, 9000), (32, 128, True, 200)])
def test_captured_decode_of_many_query_heads(Hq, D, e4m3, width):
    """One captured call replayed, on a side stream too, while lengths and the table change in place; pages that are not there, NaN in
    rows that are not seen."""
    import tyr_amd
    B, page, full = 64, 16, 200 * 16
    g = _gen(31 + Hq)
    (k, v), table, ks, vs = _cache(g, [full] * B, page, 1, D, e4m3, width=width)
    table[3, 5], table[4, :200] = -7, k.shape[0]
    k[table[6, 1].long(), :, 9:] = float("nan")      # behind 25 rows of sequence 6
    v[table[6, 1].long(), :, 9:] = float("nan")
    q = torch.randn(B, Hq, 1, D, generator=g, device="cuda").bfloat16()
    lens = torch.full((B,), 25, dtype=torch.int32, device="cuda")

    def call(**kw):
        return tyr_amd.paged_decode(q, k, v, table, lens, k_scale=ks, v_scale=vs, **kw)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = call()
    side = torch.cuda.Stream()
    for replay, (shortest, longest) in enumerate(((25, 25), (0, full), (full - 40, full), (0, 70), (0, full))):
        n = torch.randint(shortest, longest + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        n[6] = 25
        lens.copy_(n)
        want = call()
        side.wait_stream(torch.cuda.current_stream())
        beside = call(stream=side)
        o.zero_()
        lse.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for got in ((o, lse), beside):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), replay
        _check(o, lse, q, k, v, table, lens.tolist(), 1 / math.sqrt(D), ks=ks, vs=vs, only=(0, 3, 4, 5, 6, 63))


def test_on_a_side_stream():
    import tyr_amd
    g = _gen(22)
    lens_ = [3000, 17, 900]
    (k, v), table, _, _ = _cache(g, lens_, 16, 2, 128, False)
    lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
    q = torch.randn(3, 8, 1, 128, generator=g, device="cuda").bfloat16()
    want = tyr_amd.paged_decode(q, k, v, table, lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for handle in (side, side.cuda_stream):
        got = tyr_amd.paged_decode(q, k, v, table, lens, stream=handle)
        junk = [torch.full((1 << 20,), float(i), device="cuda") for i in range(8)]
        side.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        del junk


def test_shared_pages_and_large_ones():
    """Sequences that share the pages of a common beginning; a page longer than any sequence; one row."""
    import tyr_amd
    g = _gen(24)
    (k, v), table, _, _ = _cache(g, [333, 333], 16, 2, 128, False)
    table[1, :15] = table[0, :15]
    lens = torch.tensor([333, 300], dtype=torch.int32, device="cuda")
    q = torch.randn(2, 8, 1, 128, generator=g, device="cuda").bfloat16()
    o, lse = tyr_amd.paged_decode(q, k, v, table, lens)
    _check(o, lse, q, k, v, table, [333, 300], 1 / math.sqrt(128))
    for e4m3 in (False, True):
        (k, v), table, ks, vs = _cache(g, [900, 1, 4000], 4096, 2, 64, e4m3, spare=1)
        lens = torch.tensor([900, 1, 4000], dtype=torch.int32, device="cuda")
        q = torch.randn(3, 4, 1, 64, generator=g, device="cuda").bfloat16()
        for window, sinks in ((0, 0), (50, 20)):
            o, lse = tyr_amd.paged_decode(q, k, v, table, lens, window=window, sinks=sinks, k_scale=ks, v_scale=vs)
            _check(o, lse, q, k, v, table, [900, 1, 4000], 0.125, window, sinks, ks, vs)


def test_calls_at_the_same_time():
    """Calls of unlike batches on two streams, queued without a wait: each has its own scratch."""
    import tyr_amd
    g = _gen(25)
    work = []
    for lens_, Hq, Hkv, D, e4m3 in (([9000, 100, 3000], 8, 2, 128, False), ([50, 20000], 16, 1, 64, True)):
        (k, v), table, ks, vs = _cache(g, lens_, 16, Hkv, D, e4m3)
        lens = torch.tensor(lens_, dtype=torch.int32, device="cuda")
        q = torch.randn(len(lens_), Hq, 1, D, generator=g, device="cuda").bfloat16()
        work.append(lambda s=None, a=(q, k, v, table, lens), f=(ks, vs): tyr_amd.paged_decode(*a, k_scale=f[0], v_scale=f[1], stream=s))
    want = [f() for f in work]
    streams = [torch.cuda.Stream() for _ in work]
    torch.cuda.synchronize()
    got = [[f(s) for f, s in zip(work, streams)] for _ in range(20)]
    torch.cuda.synchronize()
    for round_ in got:
        for a, b in zip(round_, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_refusals():
    import tyr_amd
    E = tyr_amd.TyrGpuError
    g = _gen(23)
    (k, v), table, _, _ = _cache(g, [40, 40], 16, 2, 128, False)
    (k8, v8), _, ks, vs = _cache(g, [40, 40], 16, 2, 128, True)
    lens = torch.tensor([40, 40], dtype=torch.int32, device="cuda")
    q = torch.zeros(2, 4, 1, 128, device="cuda").bfloat16()
    ok = dict(q=q, k_pages=k, v_pages=v, page_table=table, kv_lens=lens)
    tyr_amd.paged_decode(**ok)
    for change, msg in ((dict(q=q.float()), "bfloat16"), (dict(q=q.view(1, 2, 4, 128)), "shape"), (dict(v_pages=v[:1]), "same shape"),
                        (dict(v_pages=v8), "bfloat16"), (dict(k_pages=k8, v_pages=v), "float8"), (dict(page_table=table.long()), "int32"),
                        (dict(page_table=table[:1]), "one row per sequence"), (dict(kv_lens=lens[:1]), "one value per sequence"),
                        (dict(kv_lens=lens.cpu()), "CUDA"), (dict(k_scale=ks), "float8_e4m3fn pages"), (dict(scale=0.0), "not supported"),
                        (dict(window=-1), "negative"), (dict(sinks=-1), "negative"), (dict(q=q[:, :3].contiguous()), "extents"),
                        (dict(k_pages=k[:, :, :8].contiguous(), v_pages=v[:, :, :8].contiguous()), "not supported"),
                        (dict(k_pages=k[:, :, :, :96].contiguous(), v_pages=v[:, :, :, :96].contiguous(), q=q[..., :96].contiguous()), "not supported"),
                        (dict(k_pages=k.transpose(1, 2), v_pages=v.transpose(1, 2)), "contiguous"), (dict(k_pages=k[:0], v_pages=v[:0]), "extents"),
                        (dict(page_table=table[:, :0]), "extents"), (dict(k_pages=k8, v_pages=v8, k_scale=ks[:1]), "one factor per kv head")):
        with pytest.raises(E, match=msg):
            tyr_amd.paged_decode(**{**ok, **change})
    x = torch.zeros(2, 1, 2, 128, device="cuda").bfloat16()
    cos = torch.zeros(64, 64, device="cuda")
    ok = dict(q=q.view(2, 1, 4, 128), k_new=x, v_new=x, cos=cos, sin=cos, k_pages=k, v_pages=v, page_table=table, positions=lens)
    tyr_amd.paged_rope_append(**ok)
    for change, msg in ((dict(k_new=x[:, :, :1].contiguous()), "T, Hkv, D"), (dict(v_new=x[:1]), "T, Hkv, D"), (dict(sin=cos[:3]), "S, D/2"),
                        (dict(cos=cos[:, :32].contiguous(), sin=cos[:, :32].contiguous()), "S, D/2"), (dict(positions=lens.long()), "int32"),
                        (dict(new_lens=lens[:1]), "one value per sequence"), (dict(v_scale=vs), "float8_e4m3fn pages"),
                        (dict(page_table=table[:1]), "one row per sequence"), (dict(cos=cos[:0], sin=cos[:0]), "extents"),
                        (dict(q=q.view(1, 2, 4, 128)), "one row per sequence")):
        with pytest.raises(E, match=msg):
            tyr_amd.paged_rope_append(**{**ok, **change})
