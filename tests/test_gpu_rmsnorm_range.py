"""RMS norm and its gradients of rows whose squares are beyond f32, large and small, against the formulas in float64.

A row's scale is a power of two that takes part in every term alike, so the bounds are those of ordinary rows."""
import pytest
import torch

from tests.test_gpu_rmsnorm import BF16, F32, LENGTHS, _check_grads, _data, _norm64

pytestmark = pytest.mark.gpu
SIZES = [2.0 ** 40, 2.0 ** 58, 2.0 ** 62, 2.0 ** 64, 2.0 ** 70, 2.0 ** 100, 2.0 ** 123, 2.0 ** -30, 2.0 ** -36, 2.0 ** -60, 2.0 ** -75, 2.0 ** -110]


def _rows(d, seed, n, sizes=SIZES):
    """Rows of every size beside ordinary ones, so that both kinds share workgroups and waves."""
    size = torch.tensor([s for pair in zip(sizes, [1.0] * len(sizes)) for s in pair], device="cuda")
    (x, *more), w = _data(len(size), d, seed, n)
    return (x.float() * size[:, None]).bfloat16(), more, w


def _check_forward(x, r, w, eps):
    import tyr_amd
    out, h = tyr_amd.rmsnorm_residual(x, r, w, eps)
    assert torch.equal(h, x if r is None else (x.float() + r.float()).bfloat16())
    y = _norm64(h, w, eps)
    off = (out.double() - y).abs() - (BF16 + F32) * y.abs() - 2.0 ** -126              # below it bf16 has fewer bits
    assert bool((off <= 0).all()), off.amax(-1)
    q, s, h8 = tyr_amd.rmsnorm_residual_fp8(x, r, w, eps)
    assert torch.equal(h8, h)
    top = y.abs().amax(-1)
    usual = top >= 2.0 ** -99
    assert bool(((s.double() * 448.0 - top).abs() <= F32 * top)[usual].all()) and bool((s[top < 2.0 ** -101] == 1.0).all())
    back = q.double() * s.double()[:, None]
    assert bool(((back - y).abs() <= (2.0 ** -4 + F32) * y.abs() + 2.0 ** -10 * s.double()[:, None]).all())


@pytest.mark.parametrize("d", LENGTHS)
@pytest.mark.parametrize("eps", [0.0, 1e-6, 2.0 ** -80])
def test_forward(d, eps):
    x, (r,), w = _rows(d, 31, 2)
    _check_forward(x, None, w, eps)
    small = (r.float() * 2.0 ** -20).bfloat16()
    small[1::2] = r[1::2]
    _check_forward(x, small, w, eps)


@pytest.mark.parametrize("d", LENGTHS)
def test_loud_elements(d):
    """One element decides the row's size; the others are ordinary and vanish beside it, or are all there is of a row of zeros."""
    x, _, w = _rows(d, 32, 1)
    x[1::2, 1:] = 0
    x[::2, 0] = (x[::2, 0].float() * 4.0).bfloat16()
    x[5, d - 1] = 3.0e38
    _check_forward(x, None, w, 0.0)


@pytest.mark.parametrize("d", LENGTHS)
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_backward(d, eps):
    """Up to rows whose gradients, their reciprocals, are ordinary bf16 numbers."""
    import tyr_amd
    x, (g, dr), w = _rows(d, 33, 3, [min(s, 2.0 ** 100) for s in SIZES])
    for r in (dr, None):
        _check_grads(tyr_amd.rmsnorm_residual_bwd(g, x, w, eps, d_resid=r), g, x, w, eps, r)
        for rows in (1, 4, 9):                           # one launch of few rows
            _check_grads(tyr_amd.rmsnorm_residual_bwd(g[:rows], x[:rows], w, eps, d_resid=None if r is None else r[:rows]),
                         g[:rows], x[:rows], w, eps, None if r is None else r[:rows])


@pytest.mark.parametrize("d", [64, 1000, 2304, 4096, 16384])
def test_ordinary_rows_do_not_change_beside_them(d):
    import tyr_amd
    x, (g,), w = _rows(d, 34, 2)
    plain = x.clone()
    plain[::2] = 1.0
    for fn in (tyr_amd.rmsnorm_residual, tyr_amd.rmsnorm_residual_fp8):
        for a, b in zip(fn(x, None, w)[:-1], fn(plain, None, w)[:-1]):
            assert torch.equal(a[1::2].contiguous().view(torch.uint8), b[1::2].contiguous().view(torch.uint8))
    assert torch.equal(tyr_amd.rmsnorm_residual_bwd(g, x, w)[0][1::2], tyr_amd.rmsnorm_residual_bwd(g, plain, w)[0][1::2])
