"""The gradient of the token log probabilities where a row's terms are masked: an entropy of NaN, which the forward leaves for a row with a NaN or
an infinite logit, beside a d_entropy of 0."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("vocab,width", [(1, 1), (37, 37), (3001, 3008), (9003, 9003)])
def test_rows_whose_gradients_are_all_zero_get_zeros(vocab, width, dtype):
    """Whatever they and their results hold; the other rows are what they are alone.  Rows of 37, 3001 and 9003 begin anywhere in 16 bytes."""
    import tyr_amd
    rows = 7
    gen = torch.Generator(device="cuda").manual_seed(vocab)
    x = torch.randn(rows, width, generator=gen, device="cuda").to(TYPES[dtype])
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    g, gh, gl = (torch.randn(rows, generator=gen, device="cuda") for _ in range(3))
    fine = torch.tensor([0, 3, 6], device="cuda")
    padded, masked = [1, 2], [4, 5]                              # no target; a target whose gradient is 0
    t[1], t[2] = -1, vocab
    g[padded] = torch.nan
    g[masked] = 0.0
    gh[padded + masked] = gl[padded + masked] = 0.0
    x[1], x[2, vocab // 2], x[4], x[5, -1 if width == vocab else vocab - 1] = torch.nan, torch.inf, torch.inf, torch.nan
    _, lse, entropy, _, _ = tyr_amd.token_logprobs(x, t, vocab=vocab)
    assert bool(entropy[padded + masked].isnan().all())
    for dh, dl in ((gh, gl), (gh, None), (torch.zeros_like(gh), None)):
        d = tyr_amd.token_logprobs_bwd(g, x, t, lse, vocab=vocab, entropy=entropy, d_entropy=dh, d_lse=dl)
        assert not bool(d[padded + masked].any())
        alone = tyr_amd.token_logprobs_bwd(g[fine], x[fine], t[fine], lse[fine], vocab=vocab, entropy=entropy[fine], d_entropy=dh[fine],
                                           d_lse=None if dl is None else dl[fine])
        assert bool(alone.isfinite().all()) and torch.equal(d[fine], alone)
        own = x.clone()
        assert tyr_amd.token_logprobs_bwd(g, own, t, lse, vocab=vocab, entropy=entropy, d_entropy=dh, d_lse=dl, in_place=True).data_ptr() == own.data_ptr()
        assert torch.equal(own, d)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_an_entropy_without_a_gradient_is_not_looked_at(dtype):
    """Rows with other gradients: as if the entropy had been 0."""
    import tyr_amd
    gen = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(5, 3001, generator=gen, device="cuda").to(TYPES[dtype])
    t = torch.randint(0, 3001, (5,), generator=gen, device="cuda")
    g = torch.randn(5, generator=gen, device="cuda")
    _, lse, entropy, _, _ = tyr_amd.token_logprobs(x, t)
    gh = torch.tensor([0.0, 0.5, -0.0, -1.0, 0.0], device="cuda")
    want = tyr_amd.token_logprobs_bwd(g, x, t, lse, entropy=torch.where(gh == 0, 0.0, entropy), d_entropy=gh)
    got = tyr_amd.token_logprobs_bwd(g, x, t, lse, entropy=torch.where(gh == 0, torch.nan, entropy), d_entropy=gh)
    assert torch.equal(got, want) and bool(got.isfinite().all())
