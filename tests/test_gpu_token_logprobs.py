"""Log probabilities, entropy, alternatives and their gradient against the formulas in float64.

Tolerances.  An element's exponential: the hardware's 2^-23 and the rounding of its exponent, |x - m| 2^-23 of its size, which the exponential
itself outweighs: 2^-22.  Their sum: some 32 in turn, blocks of 32 in turn, lanes, waves and parts in a tree: below 64 roundings up to 2^17 logits a
row, 2^-18.  So ln s is within 2^-17, and logp = x - m - ln s within 2^-17 + 2^-23 (|x - m| + |logp|); lse adds 2^-23 |lse|.  The entropy
ln s - t / s adds 2^-17 of t / s, the mean of m - x.

The gradient is compared with its formula at the given f32 lse and entropy: p is within (|ln p| + 8) 2^-22 of its size, and so is each term."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SHAPES = [(1, 1, 1), (3, 2, 7), (5, 64, 64), (33, 101, 101), (4, 509, 512), (257, 1000, 1000), (7, 2049, 2049), (2, 5003, 5008), (3, 32768, 32768), (1, 50001, 50001),
          (1, 131073, 131080), (1100, 4097, 4097), (1030, 8200, 8200)]


def _logits(rows, width, dtype, seed=0, scale=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + rows * 31 + width)
    return (torch.randn(rows, width, generator=g, device="cuda") * scale).to(dtype)


def _targets(rows, vocab, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + rows + vocab)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    r = torch.rand(rows, generator=g, device="cuda")
    return torch.where((r < 0.1) & (rows > 2), -100, torch.where((r > 0.9) & (rows > 2), vocab, t))


def _check(out, x, targets, vocab, top):
    """`out` as token_logprobs returns it, for rows with a finite logit."""
    logp, lse, entropy, top_logp, top_ids = out
    t = targets.long()
    for at in range(0, x.shape[0], 64):
        s = slice(at, at + 64)
        z = x[s, :vocab].double()
        m = z.amax(-1)
        z = z - m[:, None]                                   # beside logits of 1e38 float64 too would lose the sum's logarithm
        want = torch.logsumexp(z, -1)
        assert bool(((lse[s].double() - m - want).abs() <= 2.0 ** -17 + 2.0 ** -23 * (want.abs() + m.abs())).all())
        real = (t[s] >= 0) & (t[s] < vocab)
        given = z.gather(1, t[s].clamp(0, vocab - 1)[:, None])[:, 0]
        w = torch.where(real, given - want, 0.0)
        limit = 2.0 ** -17 + 2.0 ** -23 * (w.abs() + given.abs())
        assert bool(((logp[s].double() - w).abs() <= limit)[w > -torch.inf].all()) and bool((logp[s][w == -torch.inf] == -torch.inf).all())
        assert not bool(logp[s][~real].any())
        if entropy is not None:
            l = z - want[:, None]
            p = l.exp()
            h = -(p * l.clamp_min(-1e300)).sum(-1)
            mean = -(p * z.clamp_min(-1e300)).sum(-1)
            assert bool(((entropy[s].double() - h).abs() <= 2.0 ** -17 * (1.0 + mean)).all())
            assert bool((entropy[s] >= 0).all())
        if top:
            values, ids = z.sort(dim=-1, descending=True, stable=True)
            assert torch.equal(top_ids[s].long(), ids[:, :top])
            w = values[:, :top] - want[:, None]
            limit = 2.0 ** -17 + 2.0 ** -23 * (w.abs() + values[:, :top].abs())
            assert bool(((top_logp[s].double() - w).abs() <= limit)[w > -torch.inf].all()) and bool((top_logp[s][w == -torch.inf] == -torch.inf).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,width", SHAPES)
def test_forward(rows, vocab, width, dtype):
    import tyr_amd
    x, t = _logits(rows, width, TYPES[dtype]), _targets(rows, vocab)
    if width > vocab:
        x[:, vocab:] = float("nan")                          # not looked at
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(64, vocab)}):
        out = tyr_amd.token_logprobs(x, t, vocab=vocab, top=top)
        _check(out, x, t, vocab, top)
        again = tyr_amd.token_logprobs(x, t.int(), vocab=vocab, top=top, entropy=False)
        assert again[2] is None and (top or (again[3] is None and again[4] is None))
        assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])
        assert not top or (torch.equal(out[3], again[3]) and torch.equal(out[4], again[4]))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(2, 5), (1, 300), (3, 5000), (1, 40000), (1100, 3000)])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "few values", "periodic", "signed zeros", "one finite"])
def test_alternatives_of_ties_and_sorted_rows(rows, vocab, dtype, kind):
    import tyr_amd
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    x = {"equal": torch.full_like(i, -1.5), "rising": i * 0.01 - 7, "falling": 5 - i * 0.01, "few values": (i * 7919 % 3) - 1.0,
         "periodic": -(i % 2048), "signed zeros": torch.where(i % 2 == 0, -0.0, 0.0), "one finite": torch.where(i == vocab // 2, 1.0, -torch.inf)}[kind]
    x = x.to(TYPES[dtype]).expand(rows, vocab).contiguous()
    t = torch.arange(rows, device="cuda") % vocab
    for top in sorted({1, min(5, vocab), min(64, vocab)}):
        _check(tyr_amd.token_logprobs(x, t, top=top), x, t, vocab, top)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab", [(1, 40000), (2, 131072), (20, 70001), (1, 400000)])
def test_alternatives_of_rows_in_parts(rows, vocab, dtype):
    """As many from each part, all from one of them, and ties across them, around the numbers where another way is taken."""
    import tyr_amd
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    spread, equal, dense = -((i * 7919) % 8191), torch.full_like(i, 2.0), _logits(1, vocab, torch.float32, scale=2.0 ** -9)[0] + 10.0
    together = torch.where((i > vocab - 300) & (i < vocab - 200), 20.0 - (i % 13), spread)
    for x in (spread, together, equal, dense):
        x = x.to(TYPES[dtype]).expand(rows, vocab).contiguous()
        t = torch.arange(rows, device="cuda") * 5
        for top in (2, 4, 8, 15, 24, 25, 40):
            _check(tyr_amd.token_logprobs(x, t, top=top), x, t, vocab, top)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab", [3, 70, 3001, 40007])
def test_masked_and_extreme_rows(vocab, dtype):
    import tyr_amd
    low = torch.finfo(TYPES[dtype]).min
    x = _logits(14, vocab, torch.float32, 3)
    x[0] = -torch.inf                                        # nothing left
    x[1, 1:] = -torch.inf                                    # one left
    x[2, ::2] = -torch.inf
    x[3] = low                                               # everything masked by the lowest value: the same probabilities
    x[4, 1:] = low
    x[5] *= 200
    x[6] = x[6] * 0.01 + 5000
    x[7] = x[7] * 0.01 - 5000
    x[8] = x[8] * 1e4 + 1e6
    x[9] = 3e38
    x[10, 0] = -torch.inf
    x[11, vocab // 2] = torch.nan
    x[12, vocab // 2] = torch.inf
    x[13, -1] = -torch.nan
    x = x.to(TYPES[dtype])
    t = torch.full((14,), vocab - 1, device="cuda")
    top = min(3, vocab)
    logp, lse, entropy, top_logp, top_ids = out = tyr_amd.token_logprobs(x, t, top=top)
    fine = list(range(1, 11))
    _check(tuple(o[fine] for o in out), x[fine], t[fine], vocab, top)
    assert float(lse[0]) == float(logp[0]) == -torch.inf and float(entropy[0]) == 0.0
    assert top_ids[0].tolist() == list(range(top)) and bool((top_logp[0] == -torch.inf).all())
    for r in (11, 12, 13):
        assert bool(lse[r].isnan()) and bool(logp[r].isnan()) and bool(entropy[r].isnan()) and bool(top_logp[r].isnan().all())
        assert bool(((top_ids[r] >= 0) & (top_ids[r] < vocab)).all()) and len(set(top_ids[r].tolist())) == top
    # the whole row is NaN: places that are there, all different
    ids = tyr_amd.token_logprobs(torch.full_like(x, torch.nan), t, top=top)[4]
    assert ids.tolist() == [list(range(top))] * 14
    # gradients: nothing where nothing was left, finite elsewhere
    g = torch.ones(14, device="cuda")
    d = tyr_amd.token_logprobs_bwd(g, x, t, lse, entropy=entropy, d_entropy=g)
    assert not bool(d[0].any()) and bool(d[1:11].isfinite().all())
    _check_gradient(d[1:11], x[1:11], t[1:11], vocab, lse[1:11], entropy[1:11], g[1:11], g[1:11], None)


def _check_gradient(got, x, targets, vocab, lse, entropy, d_logp, d_entropy, d_lse):
    rows, width = x.shape
    t = targets.long()
    real = (t >= 0) & (t < vocab)
    z = x[:, :vocab].double() - lse.double()[:, None]
    z = z.clamp_min(-1e30)
    p = z.exp()
    zero = torch.zeros(rows, dtype=torch.float64, device="cuda")
    g = torch.where(real, d_logp.double(), 0.0) if d_logp is not None else zero
    gh = d_entropy.double() if d_entropy is not None else zero
    gl = d_lse.double() if d_lse is not None else zero
    h = entropy.double() if d_entropy is not None else zero
    want = p * (gl - g - gh * h)[:, None] - torch.where(p > 0, p * z * gh[:, None], 0.0)
    size = p * ((gl.abs() + g.abs() + (gh * h).abs())[:, None] + (z * gh[:, None]).abs())
    size = torch.where(p > 0, size * (z.abs() + 8) * 2.0 ** -22, 0.0)
    # the rounding of lse log2(e), below 2^-23 |lse|, is taken back by a term that is rounded itself, in its three operations: 2^-22 of it
    size = size + (gh.abs() * 2.0 ** -45 * lse.double().abs())[:, None] * p
    at = t.clamp(0, vocab - 1)[:, None]
    want.scatter_add_(1, at, g[:, None])
    size.scatter_add_(1, at, g.abs()[:, None] * 2.0 ** -23)
    # below the least normal f32 number the exponential may be 0
    assert bool(((got[:, :vocab].double() - want).abs() <= HALF_STEP[x.dtype] * want.abs() + size + 2.0 ** -100).all())
    assert not bool(got[:, vocab:].any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,vocab,width", SHAPES)
def test_gradient(rows, vocab, width, dtype):
    import tyr_amd
    x, t = _logits(rows, width, TYPES[dtype], 4), _targets(rows, vocab, 4)
    x[:, vocab:] = float("nan")
    logp, lse, entropy, _, _ = tyr_amd.token_logprobs(x, t, vocab=vocab)
    gen = torch.Generator(device="cuda").manual_seed(5)
    g, gh, gl = (torch.randn(rows, generator=gen, device="cuda") for _ in range(3))
    for a, b, c in ((g, None, None), (g, gh, gl), (None, gh, None), (None, None, gl)):
        kw = dict(vocab=vocab, entropy=entropy, d_entropy=b, d_lse=c)
        d = tyr_amd.token_logprobs_bwd(a, x, t, lse, **kw)
        _check_gradient(d, x, t, vocab, lse, entropy, a, b, c)
        assert torch.equal(d, tyr_amd.token_logprobs_bwd(a, x, t.int(), lse, **kw))
        own = x.clone()
        assert tyr_amd.token_logprobs_bwd(a, own, t, lse, in_place=True, **kw).data_ptr() == own.data_ptr() and torch.equal(own, d)


def test_gradient_against_differences():
    """Of the kernel's own forward in f32 along a direction, which moves every logit by at most h: the error of a difference quotient is that of
    the forward's two values, 2^-16 a row and output, over 2 h, and h^2 times the third derivative, below 8 for such directions."""
    import tyr_amd
    rows, vocab = 40, 999
    x, v = _logits(rows, vocab, torch.float32, 6), _logits(rows, vocab, torch.float32, 7, 1.0).clamp(-1, 1)
    t = _targets(rows, vocab, 6)
    gen = torch.Generator(device="cuda").manual_seed(8)
    g, gh, gl = (torch.randn(rows, generator=gen, device="cuda") for _ in range(3))

    def loss(y):
        logp, lse, entropy, _, _ = tyr_amd.token_logprobs(y, t)
        return float((logp.double() * g + entropy.double() * gh + lse.double() * gl).sum())
    h = 2.0 ** -7
    _, lse, entropy, _, _ = tyr_amd.token_logprobs(x, t)
    d = tyr_amd.token_logprobs_bwd(g, x, t, lse, entropy=entropy, d_entropy=gh, d_lse=gl)
    total = float((g.abs() + 8 * gh.abs() + gl.abs()).sum())
    assert abs((loss(x + h * v) - loss(x - h * v)) / (2 * h) - float((d.double() * v.double()).sum())) <= total * (2.0 ** -16 / h + 8 * h * h)


def test_rows_without_a_gradient_are_not_looked_at():
    """Padding: zeros, whatever the row holds; the other rows are what they are alone."""
    import tyr_amd
    x = _logits(6, 3000, torch.bfloat16, 9)
    t = torch.tensor([5, -1, 7, 3000, 2, 1], device="cuda")
    lse = tyr_amd.token_logprobs(x, t)[1]
    g = torch.ones(6, device="cuda")
    want = tyr_amd.token_logprobs_bwd(g, x, t, lse)
    g[1] = g[3] = torch.nan
    x[1], x[3], lse[3] = torch.nan, torch.inf, torch.nan
    assert torch.equal(tyr_amd.token_logprobs_bwd(g, x, t, lse), want) and not bool(want[1].any()) and not bool(want[3].any())


def test_leading_extents():
    import tyr_amd
    x, t = _logits(24, 700, torch.bfloat16, 10), _targets(24, 700, 10)
    flat = tyr_amd.token_logprobs(x, t, top=4)
    for a, b in zip(tyr_amd.token_logprobs(x.view(2, 3, 4, 700), t.view(2, 3, 4), top=4), flat):
        assert a.shape[:3] == (2, 3, 4) and torch.equal(a.reshape(b.shape), b)
    one = tyr_amd.token_logprobs(x[3], t[3], top=4)
    assert one[0].shape == () and one[3].shape == (4,) and torch.equal(one[4], flat[4][3])
    d = tyr_amd.token_logprobs_bwd(one[0], x[3], t[3], one[1])
    assert d.shape == (700,) and torch.equal(d, tyr_amd.token_logprobs_bwd(flat[0], x, t, flat[1])[3])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_logits_that_begin_anywhere(dtype):
    """A view into other logits, at every place of 16 bytes; the gradient's memory begins at another one, or is the same."""
    import tyr_amd
    for vocab in (1, 5, 40, 5003):
        flat = _logits(1, 4 * vocab + 16, TYPES[dtype], 12).view(-1)
        t, g = _targets(4, vocab, 12), torch.ones(4, device="cuda")
        for at in range(9):
            x = flat[at:at + 4 * vocab].view(4, vocab)
            out = tyr_amd.token_logprobs(x, t, top=min(3, vocab))
            _check(out, x, t, vocab, min(3, vocab))
            d = tyr_amd.token_logprobs_bwd(g, x, t, out[1], entropy=out[2], d_entropy=g)
            _check_gradient(d, x, t, vocab, out[1], out[2], g, g, None)
            before = flat.clone()
            own = tyr_amd.token_logprobs_bwd(g, x, t, out[1], entropy=out[2], d_entropy=g, in_place=True)
            assert torch.equal(own, d) and torch.equal(flat[:at], before[:at]) and torch.equal(flat[at + 4 * vocab:], before[at + 4 * vocab:])
            flat.copy_(before)


def test_offsets_beyond_32_bits():
    """4.5 GB of logits: the last rows."""
    import tyr_amd
    rows, vocab = 17200, 131071
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    last = _logits(1030, vocab, torch.bfloat16, 11)
    x[-1030:] = last
    t = torch.arange(rows, device="cuda")
    out = tyr_amd.token_logprobs(x, t, top=3)
    _check(tuple(o[-1030:] for o in out), last, t[-1030:], vocab, 3)
    d = tyr_amd.token_logprobs_bwd(out[0], x, t, out[1], in_place=True)
    for at in (-1030, -70):
        s = slice(at, at + 70 if at + 70 else None)
        _check_gradient(d[s], last[s], t[s], vocab, out[1][s], None, out[0][s], None, None)


def test_refusals():
    import tyr_amd
    x, t = _logits(4, 100, torch.bfloat16), torch.zeros(4, dtype=torch.int64, device="cuda")
    v = torch.zeros(4, device="cuda")
    bwd = tyr_amd.token_logprobs_bwd
    for call, message in [
            (lambda: tyr_amd.token_logprobs(x.half(), t), "logits must have dtype"), (lambda: tyr_amd.token_logprobs(x, t.float()), "targets must have dtype"),
            (lambda: tyr_amd.token_logprobs(x, t[:3]), "targets must have the shape"), (lambda: tyr_amd.token_logprobs(x[:, :50], t), "logits must be contiguous"),
            (lambda: tyr_amd.token_logprobs(x, t, vocab=101), "vocab must not exceed"), (lambda: tyr_amd.token_logprobs(x, t, vocab=0), "status -2"),
            (lambda: tyr_amd.token_logprobs(x, t, vocab=10, top=11), "status -2"), (lambda: tyr_amd.token_logprobs(x, t, top=65), "status -3"),
            (lambda: tyr_amd.token_logprobs(x, t, top=-1), "top must not be negative"), (lambda: tyr_amd.token_logprobs(x[:0], t[:0]), "status -2"),
            (lambda: tyr_amd.token_logprobs(x, t, vocab=-5), "vocab must not be negative"),
            (lambda: bwd(v, x, t, v[:3]), "lse must have the shape"), (lambda: bwd(v.double(), x, t, v), "dLogp must have dtype"),
            (lambda: bwd(v, x, t, v, d_entropy=v), "needs the forward's entropy"), (lambda: bwd(v.cpu(), x, t, v), "dLogp must be a CUDA tensor"),
            (lambda: bwd(v, x, t, v, d_lse=v[:2]), "dLse must have the shape"), (lambda: bwd(v, x, t, v, vocab=0), "status -2")]:
        with pytest.raises(tyr_amd.TyrGpuError, match=message):
            call()
