"""Layer norm and its gradients on rows whose elements are all equal: n = 0 and rho = eps^-1/2, whatever their size and width.

Tolerances.  The mean of equal bf16 numbers is one of them: their sums are whole multiples of it, below 2^14 of its 8 bits, and so exact in f32, and
the quotient is.  So out is the bias and dw is 0, exactly.  dx = rho (a - mean a) + d_resid with a = d_out w: fewer than 64 roundings of 2^-24 of the
terms' sizes, 2^-18; 2^-17 leaves room for the root; the result is rounded once, 2^-8."""
import pytest
import torch

pytestmark = pytest.mark.gpu
WIDTHS = [8, 64, 104, 256, 488, 512, 1000, 1032, 2040, 2560, 4096, 4104, 5112, 8192]


def _rows(values, d):
    return torch.tensor(values, device="cuda").bfloat16()[:, None].expand(-1, d).contiguous()


def _weights(d):
    g = torch.Generator(device="cuda").manual_seed(d)
    return [(k + 0.3 * torch.randn(d, generator=g, device="cuda")).bfloat16() for k in (1.0, 0.0)]


def _check_forward(values, d, eps):
    import tyr_amd
    x, (w, b) = _rows(values, d), _weights(d)
    for res in (None, torch.zeros_like(x)):
        out, _ = tyr_amd.layernorm_residual(x, res, w, b, eps)
        assert torch.equal(out, b.expand_as(out)), [values[i] for i in range(len(values)) if not torch.equal(out[i], b)]
        assert not bool(tyr_amd.layernorm_residual(x, res, w, None, eps)[0].any())


def _check_gradients(values, d, eps):
    import tyr_amd
    x, (w, _) = _rows(values, d), _weights(d)
    gen = torch.Generator(device="cuda").manual_seed(d + 1)
    g, dr = (torch.randn(x.shape, generator=gen, device="cuda").bfloat16() for _ in range(2))
    a, rho = g.double() * w.double(), float(torch.tensor(eps, dtype=torch.float32).double()) ** -0.5
    for r in (dr, None):
        dx, dw, db = tyr_amd.layernorm_residual_bwd(g, x, w, eps, d_resid=r)
        want, size = rho * (a - a.mean(-1, keepdim=True)), rho * (a.abs() + a.abs().mean(-1, keepdim=True))
        if r is not None:
            want, size = want + r.double(), size + r.double().abs()
        bad = ~((dx.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -17 * size).all(-1)
        assert not bool(bad.any()), [values[i] for i in bad.nonzero()[:, 0].tolist()]
        assert not bool(dw.any())
        s = g.double()
        assert bool(((db.double() - s.sum(0)).abs() <= 2.0 ** -8 * s.sum(0).abs() + 2.0 ** -20 * s.abs().sum(0)).all())


@pytest.mark.parametrize("d", WIDTHS)
def test_rows_of_any_width(d):
    """Their number of elements has a reciprocal that f32 rounds, or one of their waves has."""
    values = [3.0, -0.1, 99840.0, -1.5e7, 1.1e18, 1.7e9, 2.0 ** 30 * 1.9921875]
    _check_forward(values, d, 1e-5)
    _check_gradients(values, d, 1e-5)


@pytest.mark.parametrize("eps", [1e-5, 1e-25, 1e-38, 1e-40])
@pytest.mark.parametrize("d", WIDTHS)
def test_rows_beyond_f32(d, eps):
    """Their sum is, or their squares, or eps beside them."""
    values = [3.0, 2.0 ** 90 * 1.25, -(2.0 ** 118 * 1.171875), 2.0 ** 126 * 1.9, -3.38e38, 2.0 ** -90 * 1.4, 2.0 ** -130 * 1.25, 0.0]
    _check_forward(values, d, eps)
    _check_gradients(values, d, eps)


@pytest.mark.parametrize("d", [104, 1000, 4096])
def test_one_such_row_among_others(d):
    """It does not reach the gradients of the weights, and the other rows are what they are without it."""
    import tyr_amd
    gen = torch.Generator(device="cuda").manual_seed(d)
    x, g = (torch.randn(50, d, generator=gen, device="cuda").bfloat16() for _ in range(2))
    w, b = _weights(d)
    g[17] = 0.0                                                  # row 17 adds nothing to dw, whatever it holds
    out, _ = tyr_amd.layernorm_residual(x, None, w, b)
    dx, dw, db = tyr_amd.layernorm_residual_bwd(g, x, w)
    other = [i for i in range(50) if i != 17]
    for value in (2.0 ** 126, -3.38e38, 2.0 ** 90 * 1.25, 2.0 ** 15 * 1.546875):
        x[17] = value
        out2, _ = tyr_amd.layernorm_residual(x, None, w, b)
        assert torch.equal(out2[17], b) and torch.equal(out2[other], out[other])
        dx2, dw2, db2 = tyr_amd.layernorm_residual_bwd(g, x, w)
        assert not bool(dx2[17].any()) and torch.equal(dx2[other], dx[other]) and torch.equal(dw2, dw) and torch.equal(db2, db)
