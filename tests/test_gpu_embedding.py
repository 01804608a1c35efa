"""The embedding's lookup and the gradient of its table against the formulas in float64.

Tolerances.  The lookup is one f32 product, rounded once more: its bits are known.  A row of the gradient of c tokens is a sum in f32 of 32 rows
at most in turn, of 1/8 of the pieces of 8 or 32 tokens that the token reaches into, and of 8: fewer than 64 + c/64 roundings of 2^-24 of the
terms' sizes (a factor and an addition to what was there among them), and one of the result: 2^-8 (bf16), 2^-24 (f32).  Few tokens are up to 128
rows in turn, the k-th rounding of which is one of k/128 of the sizes: 64 and what is in the other term."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def _rows(n, d, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + n * 31 + d)
    return torch.randn(n, d, generator=g, device="cuda").to(dtype)


def _ids(kind, n, vocab, seed=0):
    """Tokens of a text, with padding on both sides of the table."""
    g = torch.Generator(device="cuda").manual_seed(seed + n)
    if kind == "one":
        return torch.full((n,), vocab - 1, device="cuda")
    if kind == "none":
        return torch.where(torch.arange(n, device="cuda") % 2 == 0, -1, vocab)
    if kind == "each":
        return torch.randperm(n, generator=g, device="cuda") % vocab
    ids = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * torch.tensor(vocab + 1.0).log().item()).exp().floor().long() - 1
    ids = ids.clamp(0, vocab - 1)
    r = torch.rand(n, generator=g, device="cuda")
    return torch.where(r < 0.05, -100, torch.where(r < 0.1, vocab + 3, ids))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n,vocab,d", [(1, 1, 8), (3, 5, 64), (257, 100, 72), (1000, 333, 1024), (64, 999, 2048), (130, 40, 5000), (5, 77, 12296)])
def test_lookup(n, vocab, d, dtype):
    import tyr_amd
    table = _rows(vocab, d, TYPES[dtype], 1)
    ids = _ids("text", n, vocab)
    real = (ids >= 0) & (ids < vocab)
    for scale in (1.0, 0.125, 45.254833995939045):
        want = torch.where(real[:, None], (table[ids.clamp(0, vocab - 1)].float() * scale).to(TYPES[dtype]), torch.zeros((), dtype=TYPES[dtype], device="cuda"))
        for index in (ids, ids.int()):
            out = tyr_amd.embedding(index, table, scale=scale)
            assert out.dtype == TYPES[dtype] and torch.equal(out, want)


def test_lookup_of_any_extents_and_ids_beyond_32_bits():
    import tyr_amd
    table = _rows(10, 64, torch.bfloat16, 2)
    ids = torch.tensor([[0, 9, 2 ** 32], [2 ** 32 + 1, -2 ** 63, 2 ** 31]], device="cuda")
    out = tyr_amd.embedding(ids.view(1, 2, 3), table)
    assert out.shape == (1, 2, 3, 64)
    assert torch.equal(out.view(6, 64)[:2], table[[0, 9]]) and not bool(out.view(6, 64)[2:].any())
    assert tyr_amd.embedding(ids[0, 1], table).shape == (64,)


def test_rows_of_padding_do_not_matter():
    """NaN in the rows of d_out that no token has, and in the table where no token is."""
    import tyr_amd
    table = _rows(6, 64, torch.float32, 3)
    table[3] = float("nan")
    ids = torch.tensor([0, -1, 5, 6], device="cuda")
    assert not bool(tyr_amd.embedding(ids, table).isnan().any())
    g = _rows(4, 64, torch.float32, 4)
    g[1] = g[3] = float("nan")
    out = tyr_amd.embedding_bwd(g, ids, 6)
    assert torch.equal(out[0], g[0]) and torch.equal(out[5], g[2]) and not bool(out[1:5].any())


def _check(got, g, ids, vocab, scale, base):
    g, dtype = g.reshape(-1, g.shape[-1]), g.dtype
    ids = ids.reshape(-1).long()
    real = (ids >= 0) & (ids < vocab)
    want = torch.zeros(vocab, g.shape[1], dtype=torch.float64, device="cuda")
    size, count = torch.zeros_like(want), torch.zeros(vocab, dtype=torch.float64, device="cuda")
    scale = float(torch.tensor(scale, dtype=torch.float32))
    want.index_add_(0, ids[real], g[real].double() * scale)
    size.index_add_(0, ids[real], g[real].double().abs() * abs(scale))
    count.index_add_(0, ids[real], torch.ones_like(ids[real], dtype=torch.float64))
    if base is not None:
        want, size = want + base.double(), size + base.double().abs()
        assert torch.equal(got[count == 0], base[count == 0])
    else:
        assert not bool(got[count == 0].any())
    limit = HALF_STEP[dtype] * want.abs() + (64 + count / 64)[:, None] * 2.0 ** -24 * size
    assert bool(((got.double() - want).abs() <= limit).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kind", ["text", "one", "none", "each"])
@pytest.mark.parametrize("n,vocab,d", [(1, 3, 64), (7, 5, 8), (8, 300, 64), (9, 4, 520), (64, 17, 1032), (65, 1, 256), (900, 1111, 256), (2049, 50, 4104),
                                       (8192, 700, 64), (8193, 700, 64), (8200, 3, 2056), (20000, 513, 128), (12345, 262150, 8), (140000, 1000, 64)])
def test_gradient(n, vocab, d, kind, dtype):
    import tyr_amd
    g, ids = _rows(n, d, TYPES[dtype], 5), _ids(kind, n, vocab)
    got = tyr_amd.embedding_bwd(g, ids, vocab, scale=0.75)
    _check(got, g, ids, vocab, 0.75, None)
    assert torch.equal(got, tyr_amd.embedding_bwd(g, ids.int(), vocab, scale=0.75))
    base = _rows(vocab, d, TYPES[dtype], 6)
    into = base.clone()
    assert tyr_amd.embedding_bwd(g, ids, vocab, scale=0.75, into=into).data_ptr() == into.data_ptr()
    _check(into, g, ids, vocab, 0.75, base)


def test_a_frequent_token_among_rare_ones():
    """Runs that begin and end anywhere in a piece, fill pieces, and reach over many."""
    import tyr_amd
    for n in (500, 9000):
        for long in (7, 8, 9, 16, 31, 33, 64, 65, 300, n - 2):
            for front in (0, 1, 5, 31):
                m = min(long, n - front)
                ids = torch.arange(n, device="cuda") + 10
                ids[front:front + m] = 3 + n + 20
                ids = ids[torch.randperm(n, generator=torch.Generator(device="cuda").manual_seed(front), device="cuda")]
                g = _rows(n, 64, torch.bfloat16, 8)
                _check(tyr_amd.embedding_bwd(g, ids, n + 40), g, ids, n + 40, 1.0, None)


@pytest.mark.parametrize("n,vocab,d,dtype", [(3000, 40001, 1024, "bf16"), (300, 50, 1 << 19, "f32"), (33000, 60001, 1024, "f32"), (300, 270000, 512, "bf16")])
def test_tables_larger_than_what_is_cleared_beside_the_sort(n, vocab, d, dtype):
    """The rows without a token that the sums' launch clears, and those before it; the memory held NaN."""
    import tyr_amd
    g, ids = _rows(n, 512, TYPES[dtype], 15).repeat(1, d // 512), _ids("text", n, vocab)
    for index in (ids, vocab - 1 - ids):                        # tokens are frequent at the beginning of the table, or at its end
        held = torch.full((vocab, d), float("nan"), dtype=TYPES[dtype], device="cuda")
        del held
        got = tyr_amd.embedding_bwd(g, index, vocab, scale=0.75)
        _check(got, g, index, vocab, 0.75, None)
        assert torch.equal(got, tyr_amd.embedding_bwd(g, index, vocab, scale=0.75))
        del got


def test_runs_over_many_pieces_end_anywhere():
    import tyr_amd
    n = 32000
    for runs in ((515, 17, 600, 1, 4096, 9, 2050, 24000), (31000, 5, 700), (8 * 64, 8 * 65 - 3, 8 * 66 + 1, 8 * 129, 8 * 193 + 5, 25000), (1, 32 * 65 - 1, 2, 32 * 200, 32 * 513)):
        ids = torch.repeat_interleave(torch.arange(len(runs)), torch.tensor(runs))[:n].to("cuda")
        ids = ids[torch.randperm(len(ids), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")]
        for d in (64, 2048):                                     # pieces of 8, of 32
            g = _rows(len(ids), d, torch.bfloat16, 16)
            base = _rows(9, d, torch.bfloat16, 17)
            _check(tyr_amd.embedding_bwd(g, ids, 9), g, ids, 9, 1.0, None)
            _check(tyr_amd.embedding_bwd(g, ids, 9, into=base.clone()), g, ids, 9, 1.0, base)


def test_gradient_against_differences():
    """The lookup is linear: its difference quotient in the table is exact in float64."""
    import tyr_amd
    table, g = _rows(30, 64, torch.float32, 9), _rows(200, 64, torch.float32, 10)
    ids = _ids("text", 200, 30)
    v = _rows(30, 64, torch.float32, 11)
    d = tyr_amd.embedding_bwd(g, ids, 30, scale=2.0)
    up, down = (tyr_amd.embedding(ids, table + s * v, scale=2.0).double() for s in (0.5, -0.5))
    want, got = float(((up - down) * g.double()).sum()), float((d.double() * v.double()).sum())
    # 12800 products, each of values rounded by 2^-24 of up to 16
    assert abs(got - want) <= 12800 * 16 * 2.0 ** -23


def test_offsets_beyond_32_bits():
    import tyr_amd
    vocab, d = 530000, 4096                                # 4.3 GB
    table = torch.zeros(vocab, d, dtype=torch.bfloat16, device="cuda")
    table[-5:] = _rows(5, d, torch.bfloat16, 12)
    ids = torch.arange(vocab - 5, vocab, device="cuda")
    assert torch.equal(tyr_amd.embedding(ids, table), table[-5:])
    g = _rows(5, d, torch.bfloat16, 13)
    out = tyr_amd.embedding_bwd(g, ids, vocab, into=table.zero_())
    assert torch.equal(out[-5:], g) and not bool(out[:-5].any())
    out.fill_(1.0)
    del table, out
    assert torch.equal(tyr_amd.embedding_bwd(g, ids, vocab)[-5:], g)


def test_refusals():
    import tyr_amd
    t, i = _rows(10, 64, torch.bfloat16, 14), torch.zeros(4, dtype=torch.int64, device="cuda")
    g = _rows(4, 64, torch.bfloat16, 15)
    for call, message in [
            (lambda: tyr_amd.embedding(i.float(), t), "ids must have dtype"), (lambda: tyr_amd.embedding(i, t.half()), "table must have dtype"),
            (lambda: tyr_amd.embedding(i, t.t()), "table must be contiguous"), (lambda: tyr_amd.embedding(i, t[0]), "table must have dim == 2"),
            (lambda: tyr_amd.embedding(i.cpu(), t), "ids must be a CUDA tensor"), (lambda: tyr_amd.embedding(i[:0], t), "status -2"),
            (lambda: tyr_amd.embedding(i, _rows(10, 60, torch.bfloat16, 1)), "status -3"), (lambda: tyr_amd.embedding(i.view(1, 1, 2, 2), t), "dim <= 3"),
            (lambda: tyr_amd.embedding_bwd(g, i[:3], 10), "dOut must have the shape"), (lambda: tyr_amd.embedding_bwd(g, i, 0), "status -2"),
            (lambda: tyr_amd.embedding_bwd(g, i, -1), "vocab must not be negative"), (lambda: tyr_amd.embedding_bwd(g, i, 2 ** 40), "status -2"),
            (lambda: tyr_amd.embedding_bwd(g, i, 10, into=t[:9]), "into must be"), (lambda: tyr_amd.embedding_bwd(g, i, 10, into=t.float()), "into must have dtype"),
            (lambda: tyr_amd.embedding_bwd(g[:, :60].contiguous(), i, 10), "status -3"), (lambda: tyr_amd.embedding_bwd(g, i, 1 << 26), "status -2"),
            (lambda: tyr_amd.embedding_bwd(g, i, 4, into=g), "into must not overlap dOut"),
            (lambda: tyr_amd.embedding_bwd(t[2:6], i, 4, into=t[5:9]), "into must not overlap dOut")]:
        with pytest.raises(tyr_amd.TyrGpuError, match=message):
            call()
