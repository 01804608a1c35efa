"""Host-side mirror of the Lean entry points ``Tyr.GPU.GFX950.*`` for torch tensors.

Same names, argument meaning and error behaviour as the Lean declarations in
``tyr_amd/lean/Tyr/GPU/GFX950.lean`` (which bind ``lean_tyr_gpu_*`` in
``csrc/lean_shim.cpp``): outputs are freshly allocated and returned, every tensor argument
is checked the way the reference's generated launcher checks it
(Tyr/GPU/Codegen/Attribute.lean:334-336: device, contiguity, rank <= 4) and a failed
check or a negative status from the C ABI raises ``TyrGpuError`` -- the analogue of the
``IO.userError`` the Lean wrappers return.  torch is used for device memory and the
current stream only; all arithmetic happens in ``libtyr_hip.so``.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib


class TyrGpuError(RuntimeError):
    """Raised where the Lean wrapper would return ``IO.userError msg``."""


# Checks, allocation and the C ABI call of every entry point below are native code (csrc/torch_binding.cpp): in Python
# they took longer than most of the kernels they launch.
_n = _lib.load_binding(TyrGpuError)
_flash_attn_fwd, _flash_attn_bwd, _gqa_decode, _decode_rope_append = _n.flash_attn_fwd, _n.flash_attn_bwd, _n.gqa_decode, _n.decode_rope_append
_rope_fwd, _layernorm_residual, _copy, _matmul_bf16, _gemm_bf16 = _n.rope_fwd, _n.layernorm_residual, _n.copy, _n.matmul_bf16, _n.gemm_bf16
_gemm_fp8, _gemm_fp8_scaled, _mse_loss_grad, _sgd_step = _n.gemm_fp8, _n.gemm_fp8_scaled, _n.mse_loss_grad, _n.sgd_step
_layernorm_residual_bwd, _embedding, _embedding_bwd = _n.layernorm_residual_bwd, _n.embedding, _n.embedding_bwd
_token_logprobs, _token_logprobs_bwd = _n.token_logprobs, _n.token_logprobs_bwd
_rmsnorm_residual, _rmsnorm_residual_bwd, _paged_rope_append, _paged_decode = _n.rmsnorm_residual, _n.rmsnorm_residual_bwd, _n.paged_rope_append, _n.paged_decode


def library_path() -> str:
    return _lib.LIB_PATH


def _raise(rc: int, what: str) -> None:
    if rc != 0:
        msg = _lib.load().tyr_hip_strerror(rc).decode()
        raise TyrGpuError(f"{what}: {msg} (status {rc})")


@contextlib.contextmanager
def _launch_stream(stream):
    """Outputs and scratch come from torch's caching allocator, which ties a block to the stream that was
    current when it was allocated and may hand a freed block to the next allocation on that stream.  The kernels
    run on the caller's ``stream``; when that is not torch's current stream it is made current for the call, so the
    blocks belong to it and a scratch tensor dropped on return (its kernels still queued) can only be reused by
    work queued behind them.  ``stream`` may be a ``torch.cuda.Stream`` or a raw ``hipStream_t`` handle."""
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream)) if int(stream) else torch.cuda.default_stream()
    with torch.cuda.stream(stream):
        yield


def _on_stream(stream, fn, *args):
    with _launch_stream(stream):
        return fn(*args)


def device_info(device: int = 0) -> dict:
    L = _lib.load()
    name = ctypes.create_string_buffer(64)
    cu, lds, clk = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    hbm = ctypes.c_size_t()
    _raise(L.tyr_hip_device_info(device, name, 64, ctypes.byref(cu), ctypes.byref(lds), ctypes.byref(clk),
                                 ctypes.byref(hbm)), "device_info")
    return {"arch": name.value.decode(), "compute_units": cu.value, "lds_bytes_per_cu": lds.value,
            "clock_mhz": clk.value, "hbm_bytes": hbm.value}


def flash_attn_fwd(q, k, v, causal: bool = True, scale: float | None = None, window: int = 0, kv_lens=None,
                   key_mask=None, stream=None):
    """O, LSE = flashAttnFwd q k v causal scale.

    q bf16 [B,Hq,N,D]; k, v bf16 [B,Hkv,N,D] with Hq % Hkv == 0 (query head h reads kv head h / (Hq/Hkv));
    ``window`` > 0 (causal only) lets query i see keys (i - window, i]; ``kv_lens`` (int32 [B] on the device)
    masks the keys at or beyond each sequence's length; ``key_mask`` (bool / uint8 [B,N] on the device, nonzero =
    visible) hides any set of keys per sequence instead.  -> (bf16 [B,Hq,N,D], f32 [B,Hq,N])."""
    if stream is None:
        return _flash_attn_fwd(q, k, v, causal, scale, window, kv_lens, key_mask)
    return _on_stream(stream, _flash_attn_fwd, q, k, v, causal, scale, window, kv_lens, key_mask)


def flash_attn_bwd(q, k, v, o, lse, d_o, causal: bool = True, scale: float | None = None, window: int = 0,
                   kv_lens=None, key_mask=None, stream=None):
    """dQ, dK, dV = flashAttnBwd q k v o lse dO causal scale.

    q, o, d_o bf16 [B,Hq,N,D]; k, v bf16 [B,Hkv,N,D]; lse f32 [B,Hq,N]; o and lse as returned by
    flash_attn_fwd for the same q, k, v, causal, scale, window, kv_lens and key_mask.  Returns dQ [B,Hq,N,D] and
    dK, dV [B,Hkv,N,D] (summed over the query heads of each kv head), bf16."""
    if stream is None:
        return _flash_attn_bwd(q, k, v, o, lse, d_o, causal, scale, window, kv_lens, key_mask)
    return _on_stream(stream, _flash_attn_bwd, q, k, v, o, lse, d_o, causal, scale, window, kv_lens, key_mask)


def gqa_decode(q, k, v, scale: float | None = None, num_splits: int = 0, kv_len: int | None = None,
               kv_lens=None, window: int = 0, stream=None):
    """O, LSE = gqaDecode q k v scale numSplits.

    q bf16 [B,Hq,1,D]; k, v bf16 [B,Hkv,Lmax,D] (the preallocated cache); the first ``kv_len``
    rows (default all) of every (batch, kv head) are attended to.  ``kv_lens`` (int32 [B] on the device)
    gives every sequence its own length in [0, kv_len] (a length of 0 yields O = 0, LSE = -inf); ``window`` > 0 restricts each sequence to its last
    ``window`` rows.  -> (bf16 [B,Hq,1,D], f32 [B,Hq]).
    """
    if stream is None:
        return _gqa_decode(q, k, v, scale, num_splits, kv_len, kv_lens, window)
    return _on_stream(stream, _gqa_decode, q, k, v, scale, num_splits, kv_len, kv_lens, window)


def decode_rope_append(q, k_new, v_new, cos, sin, k_cache, v_cache, pos: int, stream=None):
    """qRot = decodeRopeAppend q kNew vNew cos sin kCache vCache pos.

    q bf16 [B,Hq,1,D] (or [B,1,Hq,D]); k_new, v_new bf16 [B,Hkv,1,D]; cos, sin f32 [1,D/2] (or [D/2]) for
    position ``pos``; caches bf16 [B,Hkv,maxLen,D], row ``pos`` of each is overwritten in place.  Returns the
    rotated q with q's shape."""
    if stream is None:
        return _decode_rope_append(q, k_new, v_new, cos, sin, k_cache, v_cache, pos)
    return _on_stream(stream, _decode_rope_append, q, k_new, v_new, cos, sin, k_cache, v_cache, pos)


def rope_fwd(x, cos, sin, stream=None):
    """y = applyRotaryEmb x cos sin.  x f32 or bf16 [B,S,H,D]; cos, sin f32 [S,D/2]."""
    if stream is None:
        return _rope_fwd(x, cos, sin)
    return _on_stream(stream, _rope_fwd, x, cos, sin)


def layernorm_residual(x, residual, weight, bias, eps: float = 1e-5, stream=None):
    """(out, outResid) = fusedLayerNormResidual x residual weight bias.  bf16; x, residual [..., d]; weight, bias [d].
    Without a residual (None) outResid is x itself; without a bias (None) none is added."""
    if stream is None:
        return _layernorm_residual(x, residual, weight, bias, eps, False)
    return _on_stream(stream, _layernorm_residual, x, residual, weight, bias, eps, True)


def layernorm_residual_bwd(d_out, resid, weight, eps: float = 1e-5, d_resid=None, bias: bool = True, stream=None):
    """(dX, dWeight, dBias) = layerNormResidualBwd dOut resid weight: gradients of layernorm_residual, bf16.  resid [..., d] is
    the outResid that the forward returned, d_out the gradient of its out and d_resid (or None) the one that reaches outResid
    from the layers behind.  dX [..., d] is the gradient of x and of the residual alike; dWeight, dBias [d] (``bias`` False:
    dBias is None)."""
    if stream is None:
        return _layernorm_residual_bwd(d_out, resid, weight, eps, d_resid, bias, False)
    return _on_stream(stream, _layernorm_residual_bwd, d_out, resid, weight, eps, d_resid, bias, True)


def rmsnorm_residual(x, residual, weight, eps: float = 1e-6, stream=None):
    """(out, outResid) = rmsNormResidual x residual weight: outResid = x + residual, out = outResid * weight /
    sqrt(mean(outResid^2) + eps) over the last axis.  bf16; x, residual [..., d]; weight [d].  Without a residual (None)
    outResid is x itself."""
    if stream is None:
        return _rmsnorm_residual(x, residual, weight, eps, False, False)
    return _on_stream(stream, _rmsnorm_residual, x, residual, weight, eps, False, True)


def rmsnorm_residual_fp8(x, residual, weight, eps: float = 1e-6, stream=None):
    """(out, rowScale, outResid) = rmsNormResidualE4M3 x residual weight: as rmsnorm_residual, with out as e4m3 [..., d] and
    an f32 scale per row [...], out * rowScale being the norm: the ``aq`` and ``row_scale`` of gemm_fp8_scaled.  The
    largest value of a row is +-448."""
    if stream is None:
        return _rmsnorm_residual(x, residual, weight, eps, True, False)
    return _on_stream(stream, _rmsnorm_residual, x, residual, weight, eps, True, True)


def rmsnorm_residual_bwd(d_out, resid, weight, eps: float = 1e-6, d_resid=None, stream=None):
    """(dX, dWeight) = rmsNormResidualBwd dOut resid weight: gradients of rmsnorm_residual, bf16.  resid [..., d] is the
    outResid that the forward returned, d_out the gradient of its out and d_resid (or None) the one that reaches outResid
    from the layers behind.  dX [..., d] is the gradient of x and of the residual alike; dWeight [d]."""
    if stream is None:
        return _rmsnorm_residual_bwd(d_out, resid, weight, eps, d_resid, False)
    return _on_stream(stream, _rmsnorm_residual_bwd, d_out, resid, weight, eps, d_resid, True)


def paged_rope_append(q, k_new, v_new, cos, sin, k_pages, v_pages, page_table, positions, new_lens=None, k_scale=None, v_scale=None,
                      stream=None):
    """qRot = pagedRopeAppend q kNew vNew cos sin kPages vPages pageTable positions: rotates T new tokens of every sequence
    and writes their k (rotated) and v into the pages, in place.

    q bf16 [B,T,Hq,D]; k_new, v_new bf16 [B,T,Hkv,D]; cos, sin f32 [S,D/2], the whole rotary table; k_pages, v_pages
    [pages,Hkv,page_size,D] bf16, or e4m3 with the factors k_scale, v_scale (f32 [Hkv], None = ones) that a stored value is
    multiplied with; page_table int32 [B,width]; positions int32 [B], where each sequence's first new token stands (negative:
    it has none); new_lens int32 [B], how many of the T tokens are real (None = all).  Row j of a sequence is row
    j % page_size of page page_table[b, j / page_size].  Padding, tokens beyond the tables, and tokens on a page outside the
    pool are not written.  Returns the rotated q [B,T,Hq,D] (0 where a token has no place in the rotary table)."""
    if stream is None:
        return _paged_rope_append(q, k_new, v_new, cos, sin, k_pages, v_pages, page_table, positions, new_lens, k_scale, v_scale, False)
    return _on_stream(stream, _paged_rope_append, q, k_new, v_new, cos, sin, k_pages, v_pages, page_table, positions, new_lens, k_scale,
                      v_scale, True)


def paged_decode(q, k_pages, v_pages, page_table, kv_lens, scale: float | None = None, window: int = 0, sinks: int = 0, k_scale=None,
                 v_scale=None, stream=None):
    """O, LSE = pagedDecode q kPages vPages pageTable kvLens scale window sinks: attention of one new token over its pages.

    q bf16 [B,Hq,1,D]; pages, page_table and scales as for paged_rope_append; kv_lens int32 [B], rows of each sequence, the new
    token's among them (0: O = 0, LSE = -inf).  ``window`` > 0 restricts a sequence to its last ``window`` rows and its first
    ``sinks``; table entries of pages without a visible row may hold anything.  -> (bf16 [B,Hq,1,D], f32 [B,Hq])."""
    if stream is None:
        return _paged_decode(q, k_pages, v_pages, page_table, kv_lens, scale, window, sinks, k_scale, v_scale, False)
    return _on_stream(stream, _paged_decode, q, k_pages, v_pages, page_table, kv_lens, scale, window, sinks, k_scale, v_scale, True)


def embedding(ids, table, scale: float = 1.0, stream=None):
    """out = embedding ids table scale: out[..., :] = scale * table[ids[...]].  ids int32 or int64, any extents up to three;
    table bf16 or f32 [vocab, d] -> [..., d] of its type.  An id outside of [0, vocab) (padding) gives zeros."""
    if stream is None:
        return _embedding(ids, table, scale, False)
    return _on_stream(stream, _embedding, ids, table, scale, True)


def embedding_bwd(d_out, ids, vocab: int, scale: float = 1.0, into=None, stream=None):
    """dTable = embeddingBwd dOut ids: row v is scale times the sum of the rows of d_out whose id is v, zero where there are
    none.  d_out bf16 or f32 [..., d]; ids int32 or int64 [...]; -> [vocab, d] of d_out's type.  Ids outside of [0, vocab) add
    nothing.  With ``into`` (a gradient that is there, [vocab, d] of d_out's type: tied weights, accumulated batches) the sums
    are added to its rows, in place, and it is returned.  The result is reproducible."""
    if stream is None:
        return _embedding_bwd(d_out, ids, vocab, scale, into, False)
    return _on_stream(stream, _embedding_bwd, d_out, ids, vocab, scale, into, True)


def token_logprobs(logits, targets, vocab: int | None = None, top: int = 0, entropy: bool = True, stream=None):
    """(logp, lse, entropy, topLogp, topIds) = tokenLogprobs logits targets: for every row of logits (bf16 or f32 [..., width])
    the log of the sum of exponentials, the log probability of its target (int32 or int64 [...]; 0 for one outside of
    [0, vocab): padding), the entropy, and the ``top`` (up to 64) largest log probabilities with their ids (int32), largest
    first, equal ones by id.  The first ``vocab`` columns count (None: all); the others are the padding of the product that
    made the logits.  logp, lse, entropy f32 [...]; topLogp, topIds [..., top]; what was not asked for is None.  Logits of
    -infinity have no probability; a row of nothing else has logp = lse = -infinity and entropy 0."""
    if stream is None:
        return _token_logprobs(logits, targets, vocab, top, entropy, False)
    return _on_stream(stream, _token_logprobs, logits, targets, vocab, top, entropy, True)


def token_logprobs_bwd(d_logp, logits, targets, lse, vocab: int | None = None, entropy=None, d_entropy=None, d_lse=None,
                       in_place: bool = False, stream=None):
    """dLogits = tokenLogprobsBwd dLogp logits targets lse: the gradient of token_logprobs' logp, entropy and lse with respect
    to the logits, of their type and shape (zeros in the columns from ``vocab`` on).  lse and, with d_entropy, entropy are the
    forward's; d_logp, d_entropy, d_lse f32 [...] or None (zeros).  ``in_place`` overwrites the logits instead of
    allocating."""
    if stream is None:
        return _token_logprobs_bwd(d_logp, logits, targets, lse, vocab, entropy, d_entropy, d_lse, in_place, False)
    return _on_stream(stream, _token_logprobs_bwd, d_logp, logits, targets, lse, vocab, entropy, d_entropy, d_lse, in_place, True)


def copy(src, stream=None):
    """out = copy src (any dtype, contiguous)."""
    if stream is None:
        return _copy(src)
    return _on_stream(stream, _copy, src)


def matmul_bf16(a, b, trans_b: bool = False, stream=None):
    """C = matmul a b for operands of rank > 2 (`lean_torch_matmul`): a bf16 [..., M, K]; b bf16 [..., K, N] with
    the same leading extents, or a plain [K, N] matrix used for every batch entry (b is [..., N, K] / [N, K] with
    trans_b) -> bf16 [..., M, N]."""
    if stream is None:
        return _matmul_bf16(a, b, trans_b)
    return _on_stream(stream, _matmul_bf16, a, b, trans_b)


def gemm_bf16(a, b, trans_b: bool = False, stream=None):
    """C = gemmBf16 a b.  a bf16 [M,K]; b bf16 [K,N] (or [N,K] with trans_b) -> bf16 [M,N]."""
    if stream is None:
        return _gemm_bf16(a, b, trans_b)
    return _on_stream(stream, _gemm_bf16, a, b, trans_b)


def gemm_fp8(aq, bq, scale_a: float, scale_b: float, trans_b: bool = False, stream=None):
    """C = gemmFp8 aq bq scaleA scaleB.  aq e4m3 [M,K]; bq e4m3 [K,N] (or [N,K]) -> bf16 [M,N]."""
    if stream is None:
        return _gemm_fp8(aq, bq, scale_a, scale_b, trans_b)
    return _on_stream(stream, _gemm_fp8, aq, bq, scale_a, scale_b, trans_b)


def gemm_fp8_scaled(aq, bq, row_scale=None, col_scale=None, scale: float = 1.0, out_dtype=torch.float32,
                    trans_b: bool = False, stream=None):
    """C = gemmFp8Scaled aq bq rowScale colScale: out_dtype(scale * rowScale[m] * colScale[n] * (aq bq)[m, n]).

    The per-row / per-column dequantisation epilogue of `tkH100Fp8ScaledGemmFwd` (f32 out) and, with no scales and
    out_dtype = torch.float8_e4m3fn, the E4M3 epilogue of `tkH100Fp8E4M3GemmFwd`.  aq e4m3 [M,K]; bq e4m3 [K,N] (or
    [N,K] with trans_b); row_scale f32 [M], col_scale f32 [N] or None."""
    if stream is None:
        return _gemm_fp8_scaled(aq, bq, row_scale, col_scale, scale, out_dtype, trans_b)
    return _on_stream(stream, _gemm_fp8_scaled, aq, bq, row_scale, col_scale, scale, out_dtype, trans_b)


def mse_loss_grad(out, target, stream=None):
    """(loss, dO) = lossAndGradOut out target: loss = 0.5 mean((out - target)^2) as an f32 scalar tensor,
    dO = bf16((out - target) / numel).  out, target bf16, same shape, numel % 8 == 0."""
    if stream is None:
        return _mse_loss_grad(out, target)
    return _on_stream(stream, _mse_loss_grad, out, target)


def sgd_step(param, grad, lr: float, in_place: bool = False, stream=None):
    """(param', bf16 param') = sgdUpdate param grad lr: param' = param - f32(grad) * lr for an f32 master and a bf16
    gradient of the same shape, together with the bf16 cast the next step's kernels take.  ``in_place`` overwrites
    ``param`` instead of allocating."""
    if stream is None:
        return _sgd_step(param, grad, lr, in_place)
    return _on_stream(stream, _sgd_step, param, grad, lr, in_place)


def quantize_e4m3(x: torch.Tensor):
    """Per-tensor absmax quantisation used by the harness: s = absmax/448, xq = e4m3fn(x / s)."""
    s = float(x.abs().max()) / 448.0
    if s == 0.0:
        s = 1.0
    xq = (x.float() / s).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return xq, s
