"""RMS norm with residual (bf16 and e4m3 out) and its gradients, against the formulas in float64.

Tolerances.  A bf16 result is one rounding of an f32 value: at most 2^-8 of its size.  The f32 value's own error: sums of a row are
at most 16 terms a lane and a tree of some 12 levels over lanes and waves, and each factor adds a rounding, so less than 64 roundings of
2^-24, 2^-18, of the sum of the terms' sizes; 2^-17 leaves room for rsqrt.  e4m3: half a step is 2^-4 of a value, 2^-10 below 2^-6."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F32 = 2.0 ** -17
BF16 = 2.0 ** -8
LENGTHS = [8, 64, 72, 128, 136, 256, 264, 512, 520, 1024, 1032, 2048, 2056, 3000, 4096, 4104, 8192, 8200, 16384]


def _data(rows, d, seed, n=1):
    g = torch.Generator(device="cuda").manual_seed(seed * 100003 + rows * 17 + d)
    x = [torch.randn(rows, d, generator=g, device="cuda").bfloat16() for _ in range(n)]
    w = (1.0 + 0.3 * torch.randn(d, generator=g, device="cuda")).bfloat16()
    return x, w


def _norm64(h, w, eps):
    h = h.double()
    return h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("rows", [1, 3, 33])
@pytest.mark.parametrize("d", LENGTHS)
@pytest.mark.parametrize("residual", [True, False])
def test_forward(rows, d, residual):
    import tyr_amd
    (x, r), w = _data(rows, d, 1, 2)
    out, h = tyr_amd.rmsnorm_residual(x, r if residual else None, w, 1e-6)
    want_h = (x.float() + r.float()).bfloat16() if residual else x
    assert torch.equal(h, want_h) and (residual or h.data_ptr() == x.data_ptr())
    y = _norm64(want_h, w, 1e-6)
    assert bool(((out.double() - y).abs() <= (BF16 + F32) * y.abs()).all())
    q, s, h8 = tyr_amd.rmsnorm_residual_fp8(x, r if residual else None, w, 1e-6)
    assert torch.equal(h8, want_h) and s.shape == (rows,) and q.shape == x.shape and q.dtype == torch.float8_e4m3fn
    top = y.abs().amax(-1)
    assert bool(((s.double() * 448.0 - top).abs() <= F32 * top).all())
    back = q.double() * s.double()[:, None]
    assert bool(((back - y).abs() <= (2.0 ** -4 + F32) * y.abs() + 2.0 ** -10 * s.double()[:, None]).all())
    assert bool((q.float().abs().amax(-1) == 448.0).all())


@pytest.mark.parametrize("shape", [(5, 7, 3, 128), (4, 300, 64), (2, 2, 1024), (513,)])
def test_leading_extents(shape):
    import tyr_amd
    if shape == (513,):
        shape = (512,)
    g = torch.Generator(device="cuda").manual_seed(3)
    x, r = (torch.randn(*shape, generator=g, device="cuda").bfloat16() for _ in range(2))
    w = torch.randn(shape[-1], generator=g, device="cuda").bfloat16()
    flat = tyr_amd.rmsnorm_residual(x.view(-1, shape[-1]), r.view(-1, shape[-1]), w)
    for a, b in zip(tyr_amd.rmsnorm_residual(x, r, w), flat):
        assert a.shape == x.shape and torch.equal(a.view(b.shape), b)
    q, s, _ = tyr_amd.rmsnorm_residual_fp8(x, r, w)
    q2, s2, _ = tyr_amd.rmsnorm_residual_fp8(x.view(-1, shape[-1]), r.view(-1, shape[-1]), w)
    assert s.shape == x.shape[:-1] and torch.equal(s.reshape(-1), s2) and torch.equal(q.view(torch.uint8).view(q2.shape), q2.view(torch.uint8))


@pytest.mark.parametrize("d", [64, 1000, 4096])
def test_extreme_rows(d):
    """Rows of zeros, of one loud value, of tiny and of huge values; NaN and infinity stay in their rows."""
    import tyr_amd
    x = torch.zeros(8, d, device="cuda")
    x[1, d // 2] = 1.0
    x[2] = 2.0 ** -120
    x[3] = 2.0 ** 50                                   # its square is finite in f32 also summed over a row
    x[4] = torch.linspace(-1, 1, d, device="cuda")
    x[5], x[5, 3] = 1.0, float("nan")
    x[6], x[6, 5] = 1.0, float("inf")
    x[7] = -3.0
    x = x.bfloat16()
    w = torch.ones(d, device="cuda").bfloat16()
    eps = 1e-6
    out, _ = tyr_amd.rmsnorm_residual(x, None, w, eps)
    q, s, _ = tyr_amd.rmsnorm_residual_fp8(x, None, w, eps)
    fine = [0, 1, 2, 3, 4, 7]
    y = _norm64(x, w, eps)[fine]
    assert bool(((out[fine].double() - y).abs() <= (BF16 + F32) * y.abs()).all())
    back = q[fine].double() * s[fine].double()[:, None]
    assert bool(((back - y).abs() <= (2.0 ** -4 + F32) * y.abs() + 2.0 ** -10 * s[fine].double()[:, None]).all())
    assert float(s[0]) == 1.0 and float(s[2]) == 1.0 and not bool(q[0].float().any()) and not bool(q[2].float().any())
    assert bool(out[5].isnan().all()) and bool(out[6, 5].isnan()) and not bool(out[6, :5].float().any())
    assert bool(q[5].float().isnan().all()) and bool(s[5].isnan()) and bool(q[6, 5].float().isnan())


def test_zero_eps_and_zero_weights():
    import tyr_amd
    (x,), w = _data(9, 520, 4)
    w[::3] = 0
    y = _norm64(x, w, 0.0)
    out, _ = tyr_amd.rmsnorm_residual(x, None, w, 0.0)
    assert bool(((out.double() - y).abs() <= (BF16 + F32) * y.abs()).all())


def test_large_launch_equals_small_ones():
    """Beyond the size from which a launch streams past the last-level cache, and rows that do not fill a workgroup."""
    import tyr_amd
    (x, r), w = _data(20003, 1024, 5, 2)               # 246 MB with the outputs
    for fn in (tyr_amd.rmsnorm_residual, tyr_amd.rmsnorm_residual_fp8):
        for a, b in zip(fn(x, r, w), fn(x[-77:].contiguous(), r[-77:].contiguous(), w)):
            assert torch.equal(a[-77:].contiguous().view(torch.uint8), b.view(torch.uint8))
    (g, dr), _ = _data(20003, 1024, 6, 2)
    dx, _ = tyr_amd.rmsnorm_residual_bwd(g, x, w, d_resid=dr)
    part, _ = tyr_amd.rmsnorm_residual_bwd(g[-77:].contiguous(), x[-77:].contiguous(), w, d_resid=dr[-77:].contiguous())
    assert torch.equal(dx[-77:], part)


def _grads64(g, h, w, eps, dr):
    """dx, dw and the sizes of the terms that their f32 sums are made of."""
    g, h, w = g.double(), h.double(), w.double()
    rho = (h.pow(2).mean(-1, keepdim=True) + eps).rsqrt()
    a = g * w
    k = rho.pow(3) / h.shape[-1]
    dx = rho * a - k * (a * h).sum(-1, keepdim=True) * h
    size = (rho * a).abs() + k * (a * h).abs().sum(-1, keepdim=True) * h.abs()
    if dr is not None:
        dx, size = dx + dr.double(), size + dr.double().abs()
    t = g * h * rho
    return dx, size, t.sum(0), t.abs().sum(0)


def _check_grads(got, g, h, w, eps, dr):
    dx, size, dw, dw_size = _grads64(g, h, w, eps, dr)
    assert bool(((got[0].double() - dx).abs() <= BF16 * dx.abs() + F32 * size).all())
    # dw: up to some 200 rows in turn, then 1024 parts by 32 in turn and 32: below 512 roundings, 2^-15
    assert bool(((got[1].double() - dw).abs() <= BF16 * dw.abs() + 2.0 ** -15 * dw_size).all())


@pytest.mark.parametrize("rows", [1, 2, 5, 40, 700])
@pytest.mark.parametrize("d", LENGTHS)
def test_backward(rows, d):
    import tyr_amd
    (h, g, dr), w = _data(rows, d, 7, 3)
    for r in (dr, None):
        got = tyr_amd.rmsnorm_residual_bwd(g, h, w, 1e-5, d_resid=r)
        _check_grads(got, g, h, w, 1e-5, r)
        again = tyr_amd.rmsnorm_residual_bwd(g, h, w, 1e-5, d_resid=r)
        assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("rows,d", [(1, 2560), (2, 2056), (3, 2304), (4, 2560), (771, 2088), (1601, 2560), (1, 5120), (257, 4104), (4095, 4616), (4097, 5120)])
def test_backward_of_rows_of_five_and_ten_waves(rows, d):
    import tyr_amd
    (h, g, dr), w = _data(rows, d, 14, 3)
    for r in (dr, None):
        _check_grads(tyr_amd.rmsnorm_residual_bwd(g, h, w, 1e-6, d_resid=r), g, h, w, 1e-6, r)


@pytest.mark.parametrize("d", [64, 1000, 16384])
@pytest.mark.parametrize("size", [1e-15, 1e15])
def test_backward_of_large_and_small_rows(d, size):
    """rho^3 is beyond f32; the gradients are not."""
    import tyr_amd
    (h, g), w = _data(20, d, 13, 2)
    h = (h.float() * size).bfloat16()
    _check_grads(tyr_amd.rmsnorm_residual_bwd(g, h, w, 0.0), g, h, w, 0.0, None)


@pytest.mark.parametrize("rows,d", [(60000, 72), (9000, 1024), (3001, 4096), (1030, 16384)])
def test_backward_of_many_rows(rows, d):
    """More row groups than workgroups."""
    import tyr_amd
    (h, g, dr), w = _data(rows, d, 8, 3)
    _check_grads(tyr_amd.rmsnorm_residual_bwd(g, h, w, 1e-6, d_resid=dr), g, h, w, 1e-6, dr)


@pytest.mark.parametrize("rows,d", [(3, 64), (17, 520)])
def test_backward_against_differences(rows, d):
    """Directional derivatives of the float64 norm by central differences: error of the step t^2 and rounding 2^-52 / t are
    far below the bf16 rounding of the gradients, 2^-8 of each."""
    import tyr_amd
    (x, r, g, u), w = _data(rows, d, 9, 4)
    out, h = tyr_amd.rmsnorm_residual(x, r, w, 1e-6)
    dx, dw = tyr_amd.rmsnorm_residual_bwd(g, h, w, 1e-6)
    v = u[0].double()
    t = 1e-4

    def loss(hh, ww):
        return float((g.double() * hh / torch.sqrt(hh.pow(2).mean(-1, keepdim=True) + 1e-6) * ww).sum())
    h64, w64, u64 = h.double(), w.double(), u.double()
    by_x = (loss(h64 + t * u64, w64) - loss(h64 - t * u64, w64)) / (2 * t)
    by_w = (loss(h64, w64 + t * v) - loss(h64, w64 - t * v)) / (2 * t)
    _, size, _, dw_size = _grads64(g, h, w, 1e-6, None)
    room_x = float((BF16 * dx.double().abs() * u64.abs() + F32 * size * u64.abs()).sum()) + 1e-5
    room_w = float((BF16 * dw.double().abs() * v.abs() + F32 * dw_size * v.abs()).sum()) + 1e-5
    assert abs(float((dx.double() * u64).sum()) - by_x) <= room_x
    assert abs(float((dw.double() * v).sum()) - by_w) <= room_w


def test_two_layers_forward_and_back():
    """Two norms as a decoder chains them (the residual stream goes on, its gradient comes back through both ways), each step
    against the formulas on the tensors that reached it."""
    import tyr_amd
    rows, d = 333, 2048
    (x, r, f, g2, gr), w1 = _data(rows, d, 10, 5)
    w2 = w1.flip(0).contiguous()
    y1, h1 = tyr_amd.rmsnorm_residual(x, r, w1)
    branch = (y1.float() * f.float()).bfloat16()                      # stands for attention
    y2, h2 = tyr_amd.rmsnorm_residual(branch, h1, w2)
    assert torch.equal(h2, (branch.float() + h1.float()).bfloat16())
    dh2, dw2 = tyr_amd.rmsnorm_residual_bwd(g2, h2, w2, d_resid=gr)   # gradient of branch and of h1
    _check_grads((dh2, dw2), g2, h2, w2, 1e-6, gr)
    dy1 = (dh2.float() * f.float()).bfloat16()
    dx, dw1 = tyr_amd.rmsnorm_residual_bwd(dy1, h1, w1, d_resid=dh2)
    _check_grads((dx, dw1), dy1, h1, w1, 1e-6, dh2)


def test_captured_and_on_a_side_stream():
    import tyr_amd
    (x, r, g, dr), w = _data(300, 1024, 11, 4)

    def step(**kw):
        q, s, h = tyr_amd.rmsnorm_residual_fp8(x, r, w, **kw)
        y, _ = tyr_amd.rmsnorm_residual(x, r, w, **kw)
        return (q.view(torch.uint8), s, h, y) + tyr_amd.rmsnorm_residual_bwd(g, h, w, d_resid=dr, **kw)
    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for handle in (side, side.cuda_stream):
        got = step(stream=handle)
        junk = [torch.full((1 << 20,), float(i), device="cuda") for i in range(8)]
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del junk
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for replay in range(3):
        for t in got:
            t.zero_()
        x.copy_(x.flip(0))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), replay


def test_refusals():
    import tyr_amd
    (x, r), w = _data(4, 64, 12, 2)
    E = tyr_amd.TyrGpuError
    for bad, msg in (((x.float(), r, w), "bfloat16"), ((x, r[:2], w), "residual must match"), ((x, r, w[:8]), r"weight must be \[d_model\]"),
                     ((x[:, ::2], None, w[:32]), "contiguous"), ((x.cpu(), r, w), "CUDA"), ((x, r.cpu(), w), "CUDA"),
                     ((x[:0], None, w), "extents"), ((x[:, :12].contiguous(), None, w[:12]), "not supported")):
        for fn in (tyr_amd.rmsnorm_residual, tyr_amd.rmsnorm_residual_fp8):
            with pytest.raises(E, match=msg):
                fn(*bad)
    wide = torch.zeros(1, 16392, device="cuda").bfloat16()
    with pytest.raises(E, match="not supported"):
        tyr_amd.rmsnorm_residual(wide, None, wide[0])
    with pytest.raises(E, match="not supported"):
        tyr_amd.rmsnorm_residual(x, r, w, -1.0)
    for bad in ((x[:2], x, w), (x, x, w[:8]), (x.float(), x, w)):
        with pytest.raises(E):
            tyr_amd.rmsnorm_residual_bwd(*bad)
    with pytest.raises(E, match="dResid"):
        tyr_amd.rmsnorm_residual_bwd(x, x, w, d_resid=r[:2])
    off = torch.zeros(4 * 64 + 1, device="cuda").bfloat16()[1:].view(4, 64)
    with pytest.raises(E, match="aligned"):
        tyr_amd.rmsnorm_residual(off, None, w)
