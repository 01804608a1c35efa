"""Host validation of the embedding, layer norm and token log probability entry points: nothing is launched on bad arguments (no GPU needed)."""
import pytest

from tyr_amd import _lib

P = 0x1000                                             # never dereferenced
NULL, SHAPE, UNSUP, MISAL, WS = -1, -2, -3, -4, -5
BIG = 1 << 40
F32, BF16, I32, I64 = 0, 1, 0, 1
NAN = float("nan")


def test_the_numbers_of_the_types():
    L = _lib.load()
    # a multiple of 4 elements is a whole number of 16-byte pieces of f32 alone
    assert L.tyr_hip_embedding_bwd_workspace_bytes(4096, 100, 4, F32) > 0 == L.tyr_hip_embedding_bwd_workspace_bytes(4096, 100, 4, BF16)


def test_embedding():
    L = _lib.load()

    def fwd(ids=P, kind=I64, table=P, out=P, n=4, vocab=10, d=64, dtype=BF16):
        return L.tyr_hip_embedding(ids, kind, table, out, n, vocab, d, 1.0, dtype, None)
    assert fwd(ids=None) == fwd(table=None) == fwd(out=None) == NULL
    assert fwd(n=0) == fwd(vocab=0) == fwd(d=0) == fwd(n=BIG) == fwd(vocab=BIG) == fwd(n=1 << 25, d=1024) == SHAPE
    assert fwd(d=60) == fwd(d=62, dtype=F32) == fwd(dtype=2) == fwd(dtype=-1) == fwd(kind=2) == fwd(kind=-1) == fwd(d=(1 << 20) + 8) == UNSUP
    assert fwd(ids=P + 4) == fwd(ids=P + 2, kind=I32) == fwd(table=P + 8) == fwd(out=P + 8) == MISAL
    assert fwd(d=60, dtype=F32, out=P + 8) == fwd(ids=P + 4, kind=I32, out=P + 8) == MISAL

    def bwd(g=P, ids=P, kind=I64, table=P, n=4096, vocab=1000, d=64, into=0, dtype=BF16, ws=P, size=BIG):
        return L.tyr_hip_embedding_bwd(g, ids, kind, table, n, vocab, d, 1.0, into, dtype, ws, size, None)
    assert bwd(g=None) == bwd(ids=None) == bwd(table=None) == NULL
    assert bwd(n=0) == bwd(vocab=0) == bwd(d=0) == bwd(n=BIG) == bwd(vocab=BIG) == bwd(n=(1 << 30) + 1) == bwd(vocab=1 << 26) == SHAPE
    assert bwd(d=60) == bwd(dtype=2) == bwd(kind=2) == UNSUP
    assert bwd(g=P + 8) == bwd(ids=P + 4) == bwd(ids=P + 2, kind=I32) == bwd(table=P + 8) == bwd(ws=P + 8) == MISAL
    for n, vocab, d, dtype in ((4096, 1000, 64, BF16), (40000, 1000, 8, BF16), (3000, 300000, 4, F32)):
        need = L.tyr_hip_embedding_bwd_workspace_bytes(n, vocab, d, dtype)
        assert need > 0 and bwd(n=n, vocab=vocab, d=d, dtype=dtype, size=need - 1) == bwd(n=n, vocab=vocab, d=d, dtype=dtype, ws=None) == WS
    # few tokens need none
    assert L.tyr_hip_embedding_bwd_workspace_bytes(4, 1000, 64, BF16) == 0
    bad = [(0, 10, 64), (4, 0, 64), (4, 10, 0), (4, 10, 60), (BIG, 10, 64), ((1 << 30) + 1, 10, 64), (4, 1 << 26, 64)]
    assert all(L.tyr_hip_embedding_bwd_workspace_bytes(*b, BF16) == 0 for b in bad) and L.tyr_hip_embedding_bwd_workspace_bytes(4096, 10, 64, 9) == 0


def test_layernorm():
    L = _lib.load()

    def fwd(x=P, res=P, w=P, b=P, out=P, out_res=P, rows=4, d=64, eps=1e-5):
        return L.tyr_hip_layernorm_residual(x, res, w, b, out, out_res, rows, d, eps, None)
    assert fwd(x=None) == fwd(w=None) == fwd(out=None) == fwd(res=None) == fwd(out_res=None) == NULL
    assert fwd(b=None, x=P + 2) == fwd(res=None, out_res=None, x=P + 2) == MISAL                # both may be left out
    assert fwd(rows=0) == fwd(d=0) == fwd(rows=BIG) == SHAPE and fwd(d=60) == fwd(d=8200) == fwd(eps=-1.0) == fwd(eps=NAN) == UNSUP
    assert fwd(x=P + 2) == fwd(res=P + 8) == fwd(w=P + 8) == fwd(b=P + 8) == fwd(out=P + 4) == fwd(out_res=P + 8) == MISAL

    def bwd(g=P, dr=P, h=P, w=P, dx=P, dw=P, db=P, rows=4, d=64, eps=1e-5, ws=P, n=BIG):
        return L.tyr_hip_layernorm_residual_bwd(g, dr, h, w, dx, dw, db, rows, d, eps, ws, n, None)
    assert bwd(g=None) == bwd(h=None) == bwd(w=None) == bwd(dx=None) == bwd(dw=None) == NULL
    assert bwd(dr=None, db=None, g=P + 8) == MISAL
    assert bwd(rows=0) == bwd(d=0) == bwd(rows=BIG) == SHAPE and bwd(d=60) == bwd(d=8200) == bwd(eps=-1.0) == bwd(eps=NAN) == UNSUP
    for name in ("g", "dr", "h", "w", "dx", "dw", "db", "ws"):
        assert bwd(**{name: P + 8}) == MISAL, name
    for rows, d in ((1, 8), (4, 64), (5000, 72), (65536, 1024), (3, 8192)):
        need = L.tyr_hip_layernorm_residual_bwd_workspace_bytes(rows, d)
        assert need >= d * 8 and need % (d * 8) == 0 and bwd(rows=rows, d=d, n=need - 1) == bwd(rows=rows, d=d, ws=None) == WS
    assert L.tyr_hip_layernorm_residual_bwd_workspace_bytes(0, 64) == L.tyr_hip_layernorm_residual_bwd_workspace_bytes(4, 60) == 0


def test_token_logprobs():
    L = _lib.load()

    def fwd(x=P, t=P, kind=I64, logp=P, lse=P, h=P, tl=P, ti=P, rows=4, vocab=50000, width=50048, top=5, dtype=BF16, ws=P, n=BIG):
        return L.tyr_hip_token_logprobs(x, t, kind, logp, lse, h, tl, ti, rows, vocab, width, top, dtype, ws, n, None)
    assert fwd(x=None) == fwd(t=None) == fwd(logp=None) == fwd(lse=None) == fwd(tl=None) == fwd(ti=None) == NULL
    assert fwd(h=None, tl=None, ti=None, top=0, lse=P + 2) == MISAL                              # both may be left out
    assert fwd(rows=0) == fwd(vocab=0) == fwd(width=49999) == fwd(rows=BIG) == fwd(rows=1 << 24) == fwd(vocab=1 << 30, width=1 << 30) == SHAPE
    assert fwd(width=1 << 31) == fwd(vocab=4, top=5) == fwd(rows=1 << 21) == SHAPE               # 2^21 rows of 13 workgroups
    assert fwd(top=65) == fwd(dtype=2) == fwd(kind=2) == UNSUP and fwd(top=BIG) == SHAPE
    assert fwd(x=P + 1) == fwd(x=P + 2, dtype=F32) == fwd(t=P + 4) == fwd(t=P + 2, kind=I32) == MISAL
    for name in ("logp", "lse", "h", "tl", "ti"):
        assert fwd(**{name: P + 2}) == MISAL, name
    need = L.tyr_hip_token_logprobs_workspace_bytes(4, 50000, 5, BF16)
    assert need > 0 and fwd(n=need - 1) == fwd(ws=None) == WS and fwd(ws=P + 8) == MISAL
    assert L.tyr_hip_token_logprobs_workspace_bytes(4096, 50000, 5, BF16) == 0                   # whole rows
    assert L.tyr_hip_token_logprobs_workspace_bytes(4, 50000, 65, BF16) == L.tyr_hip_token_logprobs_workspace_bytes(0, 50000, 5, BF16) == 0
    assert L.tyr_hip_token_logprobs_workspace_bytes(4, 4, 5, BF16) == L.tyr_hip_token_logprobs_workspace_bytes(4, 50000, 5, 7) == 0

    def bwd(x=P, t=P, kind=I64, lse=P, h=P, g=P, gh=P, gl=P, dx=P, rows=4, vocab=50000, width=50048, dtype=BF16):
        return L.tyr_hip_token_logprobs_bwd(x, t, kind, lse, h, g, gh, gl, dx, rows, vocab, width, dtype, None)
    assert bwd(x=None) == bwd(t=None) == bwd(lse=None) == bwd(dx=None) == bwd(h=None) == NULL
    assert bwd(h=None, gh=None, g=None, gl=None, x=P + 1) == MISAL                               # they may be left out
    assert bwd(rows=0) == bwd(vocab=0) == bwd(width=49999) == bwd(rows=BIG) == bwd(width=1 << 31) == SHAPE
    assert bwd(dtype=2) == bwd(kind=2) == UNSUP
    for name, by in (("x", 1), ("dx", 1), ("t", 4), ("lse", 2), ("h", 2), ("g", 2), ("gh", 2), ("gl", 2)):
        assert bwd(**{name: P + by}) == MISAL, name


def test_python_entry_points_refuse_cpu_tensors():
    import torch
    import tyr_amd
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    ids = torch.zeros(4, dtype=torch.int64)
    f = torch.zeros(4)
    for call, name in ((lambda: tyr_amd.embedding(ids, x), "ids"), (lambda: tyr_amd.embedding_bwd(x, ids, 10), "dOut"),
                       (lambda: tyr_amd.layernorm_residual(x, None, x[0], None), "x"), (lambda: tyr_amd.layernorm_residual_bwd(x, x, x[0]), "dOut"),
                       (lambda: tyr_amd.token_logprobs(x, ids), "logits"), (lambda: tyr_amd.token_logprobs_bwd(f, x, ids, f), "logits")):
        with pytest.raises(tyr_amd.TyrGpuError, match=f"{name} must be a CUDA tensor"):
            call()
    with pytest.raises(tyr_amd.TyrGpuError, match="must be a tensor"):
        tyr_amd.embedding([1, 2], x)
