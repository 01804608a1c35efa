"""Host validation of the RMS norm and paged-cache entry points: nothing is launched on bad arguments (no GPU needed)."""
import pytest

from tyr_amd import _lib

P = 0x1000                                             # never dereferenced
NULL, SHAPE, UNSUP, MISAL, WS = -1, -2, -3, -4, -5
BIG = 1 << 40


def test_rmsnorm():
    L = _lib.load()

    def fwd(x=P, res=P, w=P, out=P, out_res=P, scale=None, rows=4, d=64, eps=1e-6, dtype=0):
        return L.tyr_hip_rmsnorm_residual(x, res, w, out, out_res, scale, rows, d, eps, dtype, None)
    assert fwd(x=None) == fwd(w=None) == fwd(out=None) == fwd(res=None) == fwd(out_res=None) == NULL
    assert fwd(dtype=2) == NULL                        # e4m3 needs row scales
    assert fwd(rows=0) == fwd(d=0) == fwd(rows=BIG) == SHAPE
    assert fwd(d=60) == fwd(d=16392) == fwd(dtype=1) == fwd(dtype=7) == fwd(eps=-1.0) == fwd(eps=float("nan")) == UNSUP
    assert fwd(x=P + 2) == fwd(res=P + 8) == fwd(w=P + 8) == fwd(out=P + 4) == fwd(out_res=P + 8) == fwd(scale=P + 2, dtype=2) == MISAL

    # threads of a launch: eight elements each up to a row of 512, then sixteen
    for rows, d in ((1 << 29, 64), (1 << 29, 8), (1 << 28, 72), (1 << 26, 512), (1 << 26, 520), (1 << 22, 8200), (1 << 22, 16384)):
        assert fwd(rows=rows, d=d) == SHAPE and fwd(rows=rows, d=d, x=P + 2) == SHAPE and fwd(rows=rows - 32, d=d, x=P + 2) == MISAL, (rows, d)

    def bwd(g=P, dr=P, h=P, w=P, dx=P, dw=P, rows=4, d=64, eps=1e-6, ws=P, n=BIG):
        return L.tyr_hip_rmsnorm_residual_bwd(g, dr, h, w, dx, dw, rows, d, eps, ws, n, None)
    assert bwd(g=None) == bwd(h=None) == bwd(w=None) == bwd(dx=None) == bwd(dw=None) == NULL
    assert bwd(rows=0) == bwd(d=0) == bwd(rows=BIG) == SHAPE
    assert bwd(d=60) == bwd(d=16392) == bwd(eps=-1.0) == UNSUP
    assert bwd(g=P + 8) == bwd(dr=P + 8) == bwd(h=P + 8) == bwd(w=P + 8) == bwd(dx=P + 8) == bwd(dw=P + 8) == bwd(ws=P + 8) == MISAL
    for rows, d in ((1, 8), (4, 64), (5000, 72), (65536, 1024), (3, 16384)):
        need = L.tyr_hip_rmsnorm_residual_bwd_workspace_bytes(rows, d)
        assert need >= d * 4 and need % (d * 4) == 0 and bwd(rows=rows, d=d, n=need - 1) == bwd(rows=rows, d=d, ws=None) == WS
    assert L.tyr_hip_rmsnorm_residual_bwd_workspace_bytes(0, 64) == L.tyr_hip_rmsnorm_residual_bwd_workspace_bytes(4, 60) == 0


def test_paged_decode():
    L = _lib.load()

    def call(q=P, k=P, v=P, table=P, lens=P, ks=None, vs=None, o=P, lse=P, B=2, Hq=8, Hkv=2, D=128, pages=10, page=16, width=100, window=0, sinks=0,
             dtype=0, scale=0.1, ws=P, n=BIG):
        return L.tyr_hip_paged_decode(q, k, v, table, lens, ks, vs, o, lse, B, Hq, Hkv, D, pages, page, width, window, sinks, dtype, scale, ws, n, None)
    assert call(q=None) == call(k=None) == call(v=None) == call(table=None) == call(lens=None) == call(o=None) == NULL
    for name in ("B", "Hq", "Hkv", "D", "pages", "page", "width"):
        assert call(**{name: 0}) == SHAPE, name
    assert call(Hq=7) == call(B=BIG) == call(Hq=BIG) == call(pages=BIG) == call(width=BIG) == call(page=BIG) == SHAPE
    assert call(B=1 << 20, Hq=1 << 14) == SHAPE                       # B * Hq
    assert call(width=1 << 27, page=16) == SHAPE                      # rows of a sequence
    assert call(pages=1 << 30) == SHAPE                               # tiles of the pool
    assert call(B=2 ** 31 - 1, Hq=1, Hkv=1) == call(B=1 << 26, Hq=1, Hkv=1, width=1) == SHAPE       # waves
    assert call(B=1 << 16, Hq=1, Hkv=1, width=1 << 15) == SHAPE       # steps of all heads
    assert call(D=96) == call(page=24) == call(page=8) == call(dtype=2) == call(scale=0.0) == call(scale=float("nan")) == call(scale=float("inf")) == UNSUP
    assert call(ks=P) == call(vs=P) == UNSUP                          # factors of bf16 pages
    assert call(q=P + 8) == call(k=P + 8) == call(v=P + 8) == call(o=P + 8) == call(table=P + 2) == call(lens=P + 2) == call(lse=P + 2) == MISAL
    assert call(ks=P + 2, dtype=1) == call(ws=P + 8) == MISAL
    need = L.tyr_hip_paged_decode_workspace_bytes(2, 8, 2, 128, 16, 100)
    assert need > 0 and call(n=need - 1) == call(ws=None) == WS
    # sequences of at most one piece need none
    assert L.tyr_hip_paged_decode_workspace_bytes(2, 8, 2, 128, 16, 1) == 0
    assert L.tyr_hip_paged_decode_workspace_bytes(2, 7, 2, 128, 16, 100) == L.tyr_hip_paged_decode_workspace_bytes(2, 8, 2, 128, 24, 100) == 0


def test_paged_append():
    L = _lib.load()
    names = ("q", "kn", "vn", "cos", "sin", "q_out", "k", "v", "table", "pos")

    def call(new=None, ks=None, vs=None, B=2, T=3, Hq=8, Hkv=2, D=128, pages=10, page=16, width=100, S=64, dtype=0, **ptr):
        p = [ptr.get(n, P) for n in names]
        return L.tyr_hip_paged_rope_append(*p, new, ks, vs, B, T, Hq, Hkv, D, pages, page, width, S, dtype, None)
    for n in names:
        assert call(**{n: None}) == NULL, n
        assert call(**{n: P + 2}) == MISAL, n
    for n in ("B", "T", "Hq", "Hkv", "D", "pages", "page", "width", "S"):
        assert call(**{n: 0}) == SHAPE, n
    assert call(Hq=7) == call(T=BIG) == call(S=BIG) == call(B=1 << 20, T=1 << 20) == SHAPE
    assert call(B=1 << 16, T=1 << 10, Hq=8, Hkv=8) == SHAPE           # threads
    assert call(D=96) == call(page=24) == call(dtype=5) == call(ks=P) == call(vs=P) == UNSUP
    assert call(new=P + 1) == call(ks=P + 2, dtype=1) == MISAL


def test_python_entry_points_refuse_cpu_tensors():
    import torch
    import tyr_amd
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    with pytest.raises(tyr_amd.TyrGpuError, match="x must be a CUDA tensor"):
        tyr_amd.rmsnorm_residual(x, None, x[0])
    with pytest.raises(tyr_amd.TyrGpuError, match="x must be a CUDA tensor"):
        tyr_amd.rmsnorm_residual_fp8(x, x, x[0])
    with pytest.raises(tyr_amd.TyrGpuError, match="dOut must be a CUDA tensor"):
        tyr_amd.rmsnorm_residual_bwd(x, x, x[0])
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    t = torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(tyr_amd.TyrGpuError, match="q must be a CUDA tensor"):
        tyr_amd.paged_decode(q, q, q, t, t[0])
    with pytest.raises(tyr_amd.TyrGpuError, match="q must be a CUDA tensor"):
        tyr_amd.paged_rope_append(q, q, q, x.float(), x.float(), q, q, t, t[0])
    with pytest.raises(tyr_amd.TyrGpuError, match="must be a tensor"):
        tyr_amd.rmsnorm_residual(1, None, x[0])
