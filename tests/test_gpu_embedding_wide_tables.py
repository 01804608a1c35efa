"""The gradient of the embedding's table for tables up to the 262144 tokens that residue classes take, around the numbers of tokens where another
form is taken; and the lookup of such tables.

The rows of d_out are small whole numbers, the factor is 1: every sum of them is a whole number below 2^24, which f32 holds, so the result is the
sum's one rounding to its type and its bits are known."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _whole(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-8, 9, shape, generator=g, device="cuda").to(dtype)


def _ids(kind, n, vocab, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if kind == "last":                                           # one token, the table's last
        ids = torch.full((n,), vocab - 1, device="cuda")
    elif kind == "class":                                        # one residue class, all of its quotients
        ids = (vocab - 1) % 256 + 256 * torch.randint(0, (vocab - 1) // 256 + 1, (n,), generator=g, device="cuda")
    elif kind == "text":                                         # few frequent ones, padding, the ends of the table
        ids = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) * torch.tensor(vocab + 1.0).log().item()).exp().long() - 1
        r = torch.rand(n, generator=g, device="cuda")
        ids = torch.where(r < 0.05, -1, torch.where(r < 0.1, vocab, torch.where(r < 0.15, vocab - 1, ids.clamp(0, vocab - 1))))
    else:
        ids = torch.randint(0, vocab, (n,), generator=g, device="cuda")
    assert int(ids.max()) <= vocab
    return ids


def _check(got, g, ids, base):
    """The rows of each token, side by side, summed as differences of a running sum."""
    real = (ids >= 0) & (ids < got.shape[0])
    tokens, order = ids[real].sort()
    run = g[real][order].double().cumsum(0)
    last = torch.ones_like(tokens, dtype=torch.bool)
    last[:-1] = tokens[1:] != tokens[:-1]
    sums = run[last]
    sums[1:] -= run[last][:-1]
    want = torch.zeros_like(got) if base is None else base.clone()
    tokens = tokens[last]
    sums += want[tokens].double()
    assert not len(sums) or float(sums.abs().max()) < 2 ** 24
    want[tokens] = sums.to(torch.float32).to(got.dtype)
    assert torch.equal(got, want), (got.double() - want.double()).abs().amax(1).nonzero()[:5, 0].tolist()


@pytest.mark.parametrize("kind", ["last", "class", "text", "any"])
@pytest.mark.parametrize("vocab", [65537, 131073, 151936, 262143, 262144, 262145])
@pytest.mark.parametrize("n", [1, 300, 2048, 2049, 24576, 24577])
def test_gradient(n, vocab, kind):
    import tyr_amd
    ids = _ids(kind, n, vocab, n + vocab)
    for dtype, d in (("bf16", 8), ("f32", 36)):
        g = _whole((n, d), TYPES[dtype], n)
        for index in (ids, ids.int()):
            got = tyr_amd.embedding_bwd(g, index, vocab)
            _check(got, g, ids, None)
        base = _whole((vocab, d), TYPES[dtype], vocab)
        _check(tyr_amd.embedding_bwd(g, ids, vocab, into=base.clone()), g, ids, base)


@pytest.mark.parametrize("kind", ["last", "text"])
@pytest.mark.parametrize("n,vocab,d,dtype", [(512, 200064, 2048, "bf16"), (513, 200064, 2048, "bf16"), (5000, 151936, 1032, "bf16"), (24576, 131073, 520, "f32"),
                                             (20000, 262144, 256, "bf16")])
def test_gradient_of_wide_rows(n, vocab, d, dtype, kind):
    import tyr_amd
    ids, g = _ids(kind, n, vocab, 7), _whole((n, d), TYPES[dtype], 3)
    held = torch.full((vocab, d), float("nan"), dtype=TYPES[dtype], device="cuda")
    del held
    got = tyr_amd.embedding_bwd(g, ids, vocab)
    _check(got, g, ids, None)
    del got
    base = _whole((vocab, d), TYPES[dtype], 5)
    _check(tyr_amd.embedding_bwd(g, ids, vocab, into=base.clone()), g, ids, base)


@pytest.mark.parametrize("dtype,d", [("bf16", 4608), ("bf16", 5120), ("bf16", 5640), ("bf16", 7680), ("f32", 2304), ("f32", 3580), ("bf16", 8192), ("bf16", 8712)])
def test_few_rows_of_a_frequent_token_that_one_group_of_waves_adds(dtype, d):
    """Rows of 9 blocks of 64 lanes and more leave no second group of waves: all n rows in turn.  The sums of whole numbers are exact all the same; of
    others, n additions in turn: at most n roundings of 2^-24 of the terms' sizes, and the result's."""
    import tyr_amd
    n = 2048 // -(-d * (2 if dtype == "bf16" else 4) // 1024)
    for ids in (torch.full((n,), 9, device="cuda"), torch.where(torch.arange(n, device="cuda") % 3 == 0, 265, 9)):
        g = _whole((n, d), TYPES[dtype], n)
        _check(tyr_amd.embedding_bwd(g, ids, 300), g, ids, None)
        g = torch.randn(n, d, generator=torch.Generator(device="cuda").manual_seed(n), device="cuda").to(TYPES[dtype])
        want, size = (torch.zeros(300, d, dtype=torch.float64, device="cuda").index_add_(0, ids, v) for v in (g.double(), g.double().abs()))
        got = tyr_amd.embedding_bwd(g, ids, 300)
        half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
        assert bool(((got.double() - want).abs() <= half * want.abs() + n * 2.0 ** -24 * size).all())


@pytest.mark.parametrize("vocab", [151936, 262144])
def test_lookup(vocab):
    import tyr_amd
    ids = _ids("text", 5000, vocab, 1)
    real = (ids >= 0) & (ids < vocab)
    for dtype in TYPES.values():
        table = _whole((vocab, 72), dtype, 4)
        want = torch.where(real[:, None], table[ids.clamp(0, vocab - 1)], torch.zeros((), dtype=dtype, device="cuda"))
        assert torch.equal(tyr_amd.embedding(ids, table), want) and torch.equal(tyr_amd.embedding(ids.int(), table), want)
