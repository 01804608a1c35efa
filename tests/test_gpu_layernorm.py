"""Layer norm without a residual or a bias, and the gradients of all forms, against the formulas in float64.

Tolerances.  A bf16 result is one rounding of an f32 value: at most 2^-8 of its size.  The f32 value's own error: sums of a row are at most 16 terms
a lane and a tree of some 12 levels over lanes and waves, each factor adds a rounding: less than 64 roundings of 2^-24, 2^-18, of the sum of the
terms' sizes; 2^-17 leaves room for rsqrt.  A difference from the mean is as exact as its two terms."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -17
BF16 = 2.0 ** -8
LENGTHS = [8, 64, 72, 128, 136, 256, 264, 512, 520, 1024, 1032, 2048, 2056, 2560, 3000, 4096, 4104, 5120, 8192]


def _data(rows, d, seed, n=1):
    g = torch.Generator(device="cuda").manual_seed(seed * 100003 + rows * 17 + d)
    x = [(torch.randn(rows, d, generator=g, device="cuda") + 0.5).bfloat16() for _ in range(n)]
    w, b = ((1.0 - k + 0.3 * torch.randn(d, generator=g, device="cuda")).bfloat16() for k in range(2))
    return x, w, b


def _statistics(h, eps):
    """Normalised rows, rho, and the sizes of the terms that the normalised values are made of."""
    h = h.double()
    mean = h.mean(-1, keepdim=True)
    c = h - mean
    rho = (c.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    return c * rho, rho, (c.abs() + h.abs() + h.abs().mean(-1, keepdim=True)) * rho


def _check_forward(out, h, w, b, eps):
    n, _, size = _statistics(h, eps)
    y, size = n * w.double(), size * w.double().abs()
    if b is not None:
        y, size = y + b.double(), size + b.double().abs()
    assert bool(((out.double() - y).abs() <= BF16 * y.abs() + F32 * size).all())


@pytest.mark.parametrize("rows", [1, 3, 33])
@pytest.mark.parametrize("d", LENGTHS)
def test_forward(rows, d):
    import tyr_amd
    (x, r), w, b = _data(rows, d, 1, 2)
    for res in (None, r):
        for bias in (None, b):
            out, h = tyr_amd.layernorm_residual(x, res, w, bias, 1e-5)
            want = x if res is None else (x.float() + res.float()).bfloat16()
            assert torch.equal(h, want) and (res is not None or h.data_ptr() == x.data_ptr())
            _check_forward(out, want, w, bias, 1e-5)


def test_forms_agree():
    """A residual of zeros is none, and so is a bias of zeros."""
    import tyr_amd
    for d in (64, 520, 4096, 8192):
        (x,), w, b = _data(77, d, 2)
        zero, none = torch.zeros_like(x), torch.zeros_like(b)
        full, h = tyr_amd.layernorm_residual(x, zero, w, b)
        assert torch.equal(h, x) and torch.equal(full, tyr_amd.layernorm_residual(x, None, w, b)[0])
        assert torch.equal(tyr_amd.layernorm_residual(x, None, w, none)[0], tyr_amd.layernorm_residual(x, None, w, None)[0])


@pytest.mark.parametrize("d", [64, 1000, 4096, 8192])
@pytest.mark.parametrize("residual", [False, True])
def test_extreme_rows(d, residual):
    """Rows beyond f32's squares on both sides; constant rows; NaN and infinity stay in their rows.  The gradients of the same rows."""
    import tyr_amd
    x = torch.randn(9, d, generator=torch.Generator(device="cuda").manual_seed(d), device="cuda")
    x[1] *= 2.0 ** 100
    x[2] *= 2.0 ** 70
    x[3] *= 2.0 ** -60
    x[4] = 3.0
    x[5, 3] = float("nan")
    x[6, 5] = float("inf")
    x[7] = x[7] * 2.0 ** 64 + 2.0 ** 66
    x[8] = x[8].sign() * 2.0 ** 127 * 0.99
    x = x.bfloat16()
    (g,), w, b = _data(9, d, 4)
    res = torch.zeros_like(x) if residual else None
    for eps in (1e-5, 1e-30):
        out, _ = tyr_amd.layernorm_residual(x, res, w, b, eps)
        dx, dw, db = tyr_amd.layernorm_residual_bwd(g, x, w, eps)
        for rows in ([0, 1, 2], [3, 4], [7, 8]):
            _check_forward(out[rows], x[rows], w, b, eps)
            want, size = _grads64(g[rows], x[rows], w, eps, None)[:2]
            # a gradient below the least normal f32 number or bf16 step is rounded to a multiple of that
            assert bool(((dx[rows].double() - want).abs() <= BF16 * want.abs() + F32 * size + 2.0 ** -126).all()), rows
        assert bool(out[5].isnan().all()) and bool(out[6].isnan().all()) and bool(dx[5].isnan().all()) and bool(dx[6].isnan().all())
        assert bool(dw.isnan().all()) and not bool(db.isnan().any())
        fine = [0, 1, 2, 3, 4, 7, 8]
        _check_grads(tyr_amd.layernorm_residual_bwd(g[fine].contiguous(), x[fine].contiguous(), w, eps), g[fine], x[fine], w, eps, None)


def _grads64(g, h, w, eps, dr):
    """dx, dw, dbias, each with the sizes of the terms that its f32 sums are made of."""
    n, rho, n_size = _statistics(h, eps)
    g = g.double()
    a = g * w.double()
    dx = rho * (a - a.mean(-1, keepdim=True) - n * (a * n).mean(-1, keepdim=True))
    size = rho * (a.abs() + a.abs().mean(-1, keepdim=True) + n_size * (a.abs() * n_size).mean(-1, keepdim=True))
    if dr is not None:
        dx, size = dx + dr.double(), size + dr.double().abs()
    return dx, size, (g * n).sum(0), (g.abs() * n_size).sum(0), g.sum(0), g.abs().sum(0)


def _check_grads(got, g, h, w, eps, dr):
    dx, size, dw, dw_size, db, db_size = _grads64(g, h, w, eps, dr)
    assert bool(((got[0].double() - dx).abs() <= BF16 * dx.abs() + F32 * size + 2.0 ** -126).all())
    # dw and dbias: up to some 256 rows in turn, then up to 512 parts by 32 in turn and 32: below 512 roundings, 2^-15
    assert bool(((got[1].double() - dw).abs() <= BF16 * dw.abs() + 2.0 ** -15 * dw_size).all())
    assert bool(((got[2].double() - db).abs() <= BF16 * db.abs() + 2.0 ** -15 * db_size).all())


@pytest.mark.parametrize("rows", [1, 2, 5, 40, 700])
@pytest.mark.parametrize("d", LENGTHS)
def test_backward(rows, d):
    import tyr_amd
    (h, g, dr), w, _ = _data(rows, d, 7, 3)
    for r in (dr, None):
        got = tyr_amd.layernorm_residual_bwd(g, h, w, 1e-5, d_resid=r)
        _check_grads(got, g, h, w, 1e-5, r)
        again = tyr_amd.layernorm_residual_bwd(g, h, w, 1e-5, d_resid=r, bias=False)
        assert all(torch.equal(a, b) for a, b in zip(got[:2], again[:2])) and again[2] is None


@pytest.mark.parametrize("rows,d", [(1, 2304), (2, 2056), (1601, 2560), (257, 4104), (4095, 4616), (4097, 5120), (300, 8184), (20003, 512), (70001, 64)])
def test_backward_of_many_rows(rows, d):
    import tyr_amd
    (h, g, dr), w, _ = _data(rows, d, 14, 3)
    for r in (dr, None):
        _check_grads(tyr_amd.layernorm_residual_bwd(g, h, w, 1e-5, d_resid=r), g, h, w, 1e-5, r)


def test_large_launch_equals_small_ones():
    """Beyond the size from which a launch streams past the last-level cache, and rows that do not fill a workgroup."""
    import tyr_amd
    (x, g, dr), w, b = _data(45003, 1024, 5, 3)
    assert torch.equal(tyr_amd.layernorm_residual(x, None, w, b)[0][-77:], tyr_amd.layernorm_residual(x[-77:].contiguous(), None, w, b)[0])
    dx = tyr_amd.layernorm_residual_bwd(g, x, w, d_resid=dr)[0]
    assert torch.equal(dx[-77:], tyr_amd.layernorm_residual_bwd(g[-77:].contiguous(), x[-77:].contiguous(), w, d_resid=dr[-77:].contiguous())[0])


def test_leading_extents():
    import tyr_amd
    (x, g), w, b = _data(60, 264, 6, 2)
    flat = tyr_amd.layernorm_residual_bwd(g, x, w)
    for a, c in zip(tyr_amd.layernorm_residual_bwd(g.view(3, 4, 5, 264), x.view(3, 4, 5, 264), w), flat):
        assert torch.equal(a.reshape(c.shape), c)
    assert torch.equal(tyr_amd.layernorm_residual(x[7], None, w, b)[0], tyr_amd.layernorm_residual(x, None, w, b)[0][7])


def test_gradients_against_differences():
    """Directional differences of the definition in float64, at the rounded inputs."""
    import tyr_amd
    (x, g), w, b = _data(50, 520, 8, 2)
    dx, dw, db = tyr_amd.layernorm_residual_bwd(g, x, w)
    (vx, ), vw, vb = _data(50, 520, 9)
    h = 1e-4

    def loss(s):
        xs, ws, bs = x.double() + s * vx.double(), w.double() + s * vw.double(), b.double() + s * vb.double()
        c = xs - xs.mean(-1, keepdim=True)
        return float(((c * (c.pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt() * ws + bs) * g.double()).sum())
    want = (loss(h) - loss(-h)) / (2 * h)
    terms = [(dx, vx), (dw, vw), (db, vb)]
    got = sum(float((a.double() * v.double()).sum()) for a, v in terms)
    # half a bf16 step of every gradient, and the third derivative's h^2
    assert abs(got - want) <= BF16 * sum(float((a.double() * v.double()).abs().sum()) for a, v in terms)


def test_refusals():
    import tyr_amd
    (x, r), w, b = _data(4, 64, 10, 2)
    for call, message in [
            (lambda: tyr_amd.layernorm_residual(x, r[:3], w, b), "residual must match"), (lambda: tyr_amd.layernorm_residual(x, None, w, b[:8]), "bias must be"),
            (lambda: tyr_amd.layernorm_residual(x[:0], None, w, b), "status -2"), (lambda: tyr_amd.layernorm_residual(x, None, w.float(), b), "weight must have dtype"),
            (lambda: tyr_amd.layernorm_residual(x.t(), None, w, b), "x must be contiguous"), (lambda: tyr_amd.layernorm_residual(x, None, w, b, -1.0), "status -3"),
            (lambda: tyr_amd.layernorm_residual_bwd(x, r, w.float()), "weight must have dtype"), (lambda: tyr_amd.layernorm_residual_bwd(x, r[:2], w), "dOut and dResid"),
            (lambda: tyr_amd.layernorm_residual_bwd(x, r, w, d_resid=x[:1]), "dOut and dResid"), (lambda: tyr_amd.layernorm_residual_bwd(x, r, w, float("nan")), "status -3")]:
        with pytest.raises(tyr_amd.TyrGpuError, match=message):
            call()
    big = torch.zeros(2, 8200, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(tyr_amd.TyrGpuError, match="status -3"):
        tyr_amd.layernorm_residual_bwd(big, big, big[0])
