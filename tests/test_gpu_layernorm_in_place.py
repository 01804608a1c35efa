"""The layer norm's C entry point where its outputs are its inputs: the bits that separate memory gives, also of rows whose squares f32 does not
hold, which are read twice."""
import pytest
import torch

pytestmark = pytest.mark.gpu
WIDTHS = [8, 64, 200, 512, 520, 1024, 1032, 2048, 3000, 4096, 4104, 8192]


def _rows(rows, d, seed):
    """Every second or third one is large, tiny, or of equal elements: neighbours of either kind."""
    g = torch.Generator(device="cuda").manual_seed(seed + d)
    x = torch.randn(rows, d, generator=g, device="cuda")
    x[1::6] *= 2.0 ** 100
    x[2::9] *= 2.0 ** -60
    x[4::6] = 2.0 ** 126
    return x.bfloat16()


def _call(x, res, w, b, out, out_resid, eps=1e-30):
    from tyr_amd import _lib
    p = lambda t: None if t is None else t.data_ptr()
    rc = _lib.load().tyr_hip_layernorm_residual(p(x), p(res), p(w), p(b), p(out), p(out_resid), x.shape[0], x.shape[1], eps,
                                                torch.cuda.current_stream().cuda_stream)
    assert rc == 0


@pytest.mark.parametrize("rows", [1, 7, 1001])
@pytest.mark.parametrize("d", WIDTHS)
def test_without_a_residual(rows, d):
    x, w, b = _rows(rows, d, 1), _rows(3, d, 2)[0], _rows(3, d, 3)[0]
    for bias in (b, None):
        want, own = torch.empty_like(x), x.clone()
        _call(x, None, w, bias, want, None)
        _call(own, None, w, bias, own, None)
        assert bool(want.isfinite().all()) and torch.equal(own, want)


@pytest.mark.parametrize("rows", [1, 7, 1001])
@pytest.mark.parametrize("d", WIDTHS)
def test_with_a_residual(rows, d):
    x, r, w, b = _rows(rows, d, 1), _rows(rows, d, 4), _rows(3, d, 2)[0], _rows(3, d, 3)[0]
    r[4::6] = 0.0
    want, h = torch.empty_like(x), torch.empty_like(x)
    _call(x, r, w, b, want, h)
    assert torch.equal(h, (x.float() + r.float()).bfloat16()) and bool(want.isfinite().all())
    for out, out_resid in (("x", None), ("r", None), (None, "x"), (None, "r"), ("x", "r"), ("r", "x")):
        own = {"x": x.clone(), "r": r.clone()}
        o, s = own.get(out, torch.empty_like(x)), own.get(out_resid, torch.empty_like(x))
        _call(own["x"], own["r"], w, b, o, s)
        assert torch.equal(o, want) and torch.equal(s, h), (out, out_resid)
        assert out == "x" or out_resid == "x" or torch.equal(own["x"], x)
        assert out == "r" or out_resid == "r" or torch.equal(own["r"], r)
