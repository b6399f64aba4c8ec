"""Host-side mirror of the C ABI on torch CUDA tensors.

Every function here only allocates outputs (torch) and forwards device
pointers plus torch's current stream to libds4b200.so; the arithmetic lives in
the CUDA kernels.  Tensors must be contiguous CUDA tensors; nothing runs on CPU.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import (FP8_BLOCK64_POW2, FP8_ROW_AMAX, GLU_CLAMP_REF, GLU_CLAMP_SYM, GLU_PLAIN, KV_F32, KV_FP8_BLOCK64, KV_FP8_ROW,
                   TABLE_F16, TABLE_Q8_0, RopeParams, check)

__all__ = [
    "FP8_BLOCK64_POW2", "FP8_ROW_AMAX", "GLU_CLAMP_REF", "GLU_CLAMP_SYM", "GLU_PLAIN",
    "TABLE_F16", "TABLE_Q8_0", "RopeParams", "rope_params_for_layer", "rope_params_explicit",
    "add", "rms_norm_rows", "rms_norm_q8_0_rows", "quantize_q8_0_rows", "quantize_q8_K_rows", "embed_gather_rows", "rope_rows", "rope_table_rows", "rope_q8_0_rows", "fp8_kv_round_trip_rows",
    "rope_fp8_store_rows", "fp8_cache_load_rows", "kv_rows_to_raw", "swa_window_push_rows", "swiglu_rows", "hc_pre_rows", "hc_pre_norm_rows", "output_hc_head_rows", "hc_post_rows", "hc_sinkhorn_rows", "hc_sinkhorn_mix_rows",
    "e4m3_encode", "e4m3_decode", "e4m3_selfcheck", "div_selfcheck", "device_status", "compressor_step", "compressor_chunk", "swiglu_q8_K_rows",
    "KV_F32", "KV_FP8_BLOCK64", "KV_FP8_ROW", "PagedKv", "PagePool", "attn_workspace", "attn_decode_paged", "attn_window_paged",
    "pages_copy", "pages_fork", "pages_reserve", "pages_free", "pages_compact",
]


def _p(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("ds4cuda_b200 ops take CUDA tensors only")
    if not t.is_contiguous():
        raise ValueError("ds4cuda_b200 ops take contiguous tensors")
    return C.c_void_p(t.data_ptr())


def _s():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


def rope_params_for_layer(il: int, n_rot: int = 64) -> RopeParams:
    """Per-layer routing of the reference launcher (cuda/rope.cu:214-250)."""
    p = RopeParams()
    _lib.load().ds4b200_rope_params_for_layer(il, n_rot, C.byref(p))
    return p


def rope_params_explicit(freq_base: float, yarn_factor: float, n_ctx_orig: int,
                         n_rot: int = 64) -> RopeParams:
    p = RopeParams()
    _lib.load().ds4b200_rope_params_explicit(freq_base, yarn_factor, n_ctx_orig, n_rot, C.byref(p))
    return p


def device_status() -> int:
    return _lib.load().ds4b200_device_status()


def add(a, b):
    y = torch.empty_like(a)
    check(_lib.load().ds4b200_add_f32(_p(a), _p(b), _p(y), a.numel(), _s()))
    return y


def rms_norm_rows(x, w=None, residual=None, eps=1e-6, want_f32=True, want_bf16=False,
                  want_residual=False):
    """x [rows, n]; w None | [n] | [rows, n].  Returns (y_f32, y_bf16, residual_out)."""
    rows, n = x.shape
    weight_dim = 0 if w is None else w.numel()
    y = torch.empty_like(x) if want_f32 else None
    yb = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device) if want_bf16 else None
    ro = torch.empty_like(x) if want_residual else None
    check(_lib.load().ds4b200_rms_norm_rows_f32(_p(x), _p(residual), _p(w), weight_dim, _p(y),
                                                _p(yb), _p(ro), rows, n, eps, _s()))
    return y, yb, ro


def rms_norm_q8_0_rows(x, w=None, residual=None, eps=1e-6, want_f32=True, want_residual=False):
    """RMSNorm + Q8_0 activation quantiser.  Returns (y_f32, residual_out, xq int8 [rows, n], xscale [rows, n/32])."""
    rows, n = x.shape
    y = torch.empty_like(x) if want_f32 else None
    ro = torch.empty_like(x) if want_residual else None
    xq = torch.empty((rows, n), dtype=torch.int8, device=x.device)
    xs = torch.empty((rows, n // 32), dtype=torch.float32, device=x.device)
    check(_lib.load().ds4b200_rms_norm_q8_0_rows_f32(_p(x), _p(residual), _p(w), 0 if w is None else w.numel(), _p(y),
                                                     _p(ro), _p(xq), _p(xs), rows, n, eps, _s()))
    return y, ro, xq, xs


def rms_norm_q8_K_rows(x, w=None, residual=None, eps=1e-6, want_f32=True, want_residual=False, want_q8_0=False):
    """RMSNorm + Q8_K activation quantiser (and optionally the Q8_0 one on the same row).  Returns
    (y_f32, residual_out, (xq, xscale) or None, (kq int8 [rows, n], kscale [rows, n/256], kbsums int16 [rows, n/16]))."""
    rows, n = x.shape
    y = torch.empty_like(x) if want_f32 else None
    ro = torch.empty_like(x) if want_residual else None
    xq = torch.empty((rows, n), dtype=torch.int8, device=x.device) if want_q8_0 else None
    xs = torch.empty((rows, n // 32), dtype=torch.float32, device=x.device) if want_q8_0 else None
    kq = torch.empty((rows, n), dtype=torch.int8, device=x.device)
    ks = torch.empty((rows, n // 256), dtype=torch.float32, device=x.device)
    kb = torch.empty((rows, n // 16), dtype=torch.int16, device=x.device)
    check(_lib.load().ds4b200_rms_norm_q8_K_rows_f32(_p(x), _p(residual), _p(w), 0 if w is None else w.numel(), _p(y),
                                                     _p(ro), _p(xq), _p(xs), _p(kq), _p(ks), _p(kb), rows, n, eps,
                                                     _s()))
    return y, ro, ((xq, xs) if want_q8_0 else None), (kq, ks, kb)


def quantize_q8_0_rows(x):
    """x with numel % 32 == 0 -> (int8 like x, f32 scales [numel/32])."""
    xq = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    xs = torch.empty(x.numel() // 32, dtype=torch.float32, device=x.device)
    check(_lib.load().ds4b200_quantize_q8_0_rows_f32(_p(x), _p(xq), _p(xs), x.numel() // 32, _s()))
    return xq, xs


def quantize_q8_K_rows(x):
    """x with numel % 256 == 0 -> (int8 like x, f32 scales [numel/256], int16 sums [numel/16])."""
    nb = x.numel() // 256
    xq = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    xs = torch.empty(nb, dtype=torch.float32, device=x.device)
    bs = torch.empty(nb * 16, dtype=torch.int16, device=x.device)
    check(_lib.load().ds4b200_quantize_q8_K_rows_f32(_p(x), _p(xq), _p(xs), _p(bs), nb, _s()))
    return xq, xs, bs


def embed_gather_rows(table, table_dtype, ids, n_embd, residual=None, norm_w=None, eps=1e-6,
                      n_replicas=1, want_rows=True, want_f32=False, want_bf16=False):
    """Returns (rows [T, n_replicas, n_embd] f32, normed_f32, normed_bf16)."""
    T = ids.numel()
    dev = ids.device
    rows = torch.empty((T, n_replicas, n_embd), dtype=torch.float32, device=dev) if want_rows else None
    nf = torch.empty((T, n_embd), dtype=torch.float32, device=dev) if want_f32 else None
    nb = torch.empty((T, n_embd), dtype=torch.bfloat16, device=dev) if want_bf16 else None
    check(_lib.load().ds4b200_embed_gather_rows(_p(table), table_dtype, _p(ids), T, n_embd,
                                                _p(residual), _p(norm_w), eps, _p(rows), n_replicas,
                                                _p(nf), _p(nb), _s()))
    return rows, nf, nb


def rope_rows(x, pos, params, n_rot=64, inverse=False, unit_rms=False, eps=1e-6, out=None, table=None):
    """x [T, H, D], pos [T] int32; table: rope_table_rows(pos, params), in place of pos + params."""
    T, H, D = x.shape
    out = torch.empty_like(x) if out is None else out
    if table is not None:
        check(_lib.load().ds4b200_rope_rows_table_f32(_p(x), _p(out), T, H, D, n_rot, _p(table), int(inverse),
                                                      int(unit_rms), eps, _s()))
        return out
    check(_lib.load().ds4b200_rope_rows_f32(_p(x), _p(out), T, H, D, n_rot, _p(pos),
                                            C.byref(params), int(inverse), int(unit_rms), eps, _s()))
    return out


def rope_table_rows(pos, params, n_rot=64):
    """(cos, sin) multipliers of the n_rot/2 tail pairs at every position: [T, n_rot/2, 2]."""
    T = pos.numel()
    cs = torch.empty((T, n_rot // 2, 2), dtype=torch.float32, device=pos.device)
    check(_lib.load().ds4b200_rope_table_rows(_p(pos), C.byref(params), T, n_rot, _p(cs), _s()))
    return cs


def rope_q8_0_rows(x, pos, params, n_rot=64, inverse=False, unit_rms=False, eps=1e-6, want_f32=False, table=None):
    """rope_rows whose result leaves as Q8_0 blocks: (out f32 or None, xq int8 [T, H, D], xscale [T, H, D/32]).
    table: rope_table_rows(pos, params), in place of pos + params."""
    T, H, D = x.shape
    out = torch.empty_like(x) if want_f32 else None
    xq = torch.empty((T, H, D), dtype=torch.int8, device=x.device)
    xs = torch.empty((T, H, D // 32), dtype=torch.float32, device=x.device)
    check(_lib.load().ds4b200_rope_q8_0_rows_f32(_p(x), _p(out), _p(xq), _p(xs), T, H, D, n_rot, _p(pos),
                                                 None if params is None else C.byref(params), _p(table),
                                                 int(inverse), int(unit_rms), eps, _s()))
    return out, xq, xs


def fp8_kv_round_trip_rows(kv, n_rot=64, out=None):
    rows, D = kv.shape
    out = torch.empty_like(kv) if out is None else out
    check(_lib.load().ds4b200_fp8_kv_round_trip_rows_f32(_p(kv), _p(out), rows, D, n_rot, _s()))
    return out


def rope_fp8_store_rows(kv, pos, params, n_rot, scale_mode, codes, scales, slots=None,
                        norm_w=None, eps=1e-6, tail_out=None, rope_out=None, table=None):
    """Writes into the caller's cache tensors `codes` (uint8) and `scales` (f32).  `table` (rope_table_rows,
    one row per kv row) replaces pos + params."""
    rows, D = kv.shape
    if table is not None:
        check(_lib.load().ds4b200_rope_fp8_store_rows_table(
            _p(kv), rows, D, n_rot, _p(table), _p(norm_w), eps, scale_mode, _p(slots), _p(codes), _p(scales),
            _p(tail_out), _p(rope_out), _s()))
        return
    check(_lib.load().ds4b200_rope_fp8_store_rows(
        _p(kv), rows, D, n_rot, _p(pos), None if params is None else C.byref(params), _p(norm_w),
        eps, scale_mode, _p(slots), _p(codes), _p(scales), _p(tail_out), _p(rope_out), _s()))


def fp8_cache_load_rows(codes, scales, slots, n_rot, scale_mode, tail=None, f16_round=False):
    """Rows at `slots` of the byte cache -> f32 [len(slots), head_dim]."""
    D = codes.shape[1]
    out = torch.empty((slots.numel(), D), dtype=torch.float32, device=codes.device)
    check(_lib.load().ds4b200_fp8_cache_load_rows(_p(codes), _p(scales), _p(tail), _p(slots), slots.numel(), D, n_rot,
                                                  scale_mode, int(f16_round), _p(out), _s()))
    return out


def kv_rows_to_raw(kv, pos, params, raw_out, n_rot=64, slots=None, norm_w=None, eps=1e-6, table=None, table_out=None):
    """norm -> RoPE -> FP8 round trip -> f16 round, written to raw_out[slot] (f32 rows).  `table`
    (rope_table_rows, one row per kv row) replaces pos + params; `table_out` [rows, n_rot/2, 2] receives the
    angles this launch evaluates (the chunk's table, for the RoPE launches that follow)."""
    rows, D = kv.shape
    if table_out is not None:
        check(_lib.load().ds4b200_kv_rows_to_raw_table_out_f32(_p(kv), rows, D, n_rot, _p(pos), C.byref(params),
                                                               _p(norm_w), eps, _p(slots), _p(raw_out), _p(table_out), _s()))
        return raw_out
    if table is not None:
        check(_lib.load().ds4b200_kv_rows_to_raw_table_f32(_p(kv), rows, D, n_rot, _p(table), _p(norm_w), eps,
                                                           _p(slots), _p(raw_out), _s()))
        return raw_out
    check(_lib.load().ds4b200_kv_rows_to_raw_f32(_p(kv), rows, D, n_rot, _p(pos),
                                                 None if params is None else C.byref(params), _p(norm_w), eps,
                                                 _p(slots), _p(raw_out), _s()))
    return raw_out


def swa_window_push_rows(raw_kv, n_raw, new_rows):
    """raw_kv [cap, D] window with n_raw rows; pushes new_rows [n, D]; returns the new row count."""
    cap, D = raw_kv.shape
    after = C.c_int()
    check(_lib.load().ds4b200_swa_window_push_rows_f32(_p(raw_kv), cap, n_raw, _p(new_rows), new_rows.shape[0], D,
                                                       C.byref(after), _s()))
    return after.value


def compressor_chunk(is_attn, kv_cur, sc_cur, ape_f16, norm_w, head_dim, ratio, pos0, il, state_kv, state_score):
    """A window-aligned chunk of compressor steps at once; returns emits [T / ratio, head_dim]."""
    T = kv_cur.shape[0]
    emits = torch.empty((T // ratio, head_dim), dtype=torch.float32, device=kv_cur.device)
    check(_lib.load().ds4b200_compressor_chunk_f32(int(is_attn), _p(kv_cur), _p(sc_cur), _p(ape_f16), _p(norm_w),
                                                   head_dim, ratio, pos0, T, il, _p(state_kv), _p(state_score),
                                                   _p(emits), _s()))
    return emits


def swiglu_q8_K_rows(gate, up, weights=None, mode=GLU_PLAIN, clamp=0.0, fast_exp=False, want_f32=False):
    """gate/up [T, k, n] -> Q8_K blocks of the [T, k, n] SwiGLU rows: (xq int8 [T,k,n], scales [T,k,n/256],
    bsums int16 [T,k,n/256,16], mid f32 or None)."""
    T, k, n = gate.shape
    dev = gate.device
    xq = torch.empty((T, k, n), dtype=torch.int8, device=dev)
    xs = torch.empty((T, k, n // 256), dtype=torch.float32, device=dev)
    bs = torch.empty((T, k, n // 256, 16), dtype=torch.int16, device=dev)
    mid = torch.empty((T, k, n), dtype=torch.float32, device=dev) if want_f32 else None
    check(_lib.load().ds4b200_swiglu_q8_K_rows_f32(_p(gate), _p(up), _p(weights), _p(xq), _p(xs), _p(bs), _p(mid),
                                                   T, k, n, mode, clamp, int(fast_exp), _s()))
    return xq, xs, bs, mid


def compressor_step(is_attn, kv_cur, sc_cur, ape_f16, norm_w, head_dim, ratio, pos, il, state_kv, state_score,
                    emit_out):
    """One streaming-compressor step after its projections, in place; True when emit_out was written."""
    emitted = C.c_int()
    check(_lib.load().ds4b200_compressor_step_f32(int(is_attn), _p(kv_cur), _p(sc_cur), _p(ape_f16), _p(norm_w),
                                                  head_dim, ratio, pos, il, _p(state_kv), _p(state_score),
                                                  _p(emit_out), C.byref(emitted), _s()))
    return bool(emitted.value)


def swiglu_rows(gate, up, weights=None, mode=GLU_PLAIN, clamp=0.0, combine=False, fast_exp=False):
    """gate/up [T, k, n]; returns [T, n] when combine else [T, k, n]."""
    T, k, n = gate.shape
    out = torch.empty((T, n) if combine else (T, k, n), dtype=torch.float32, device=gate.device)
    check(_lib.load().ds4b200_swiglu_rows_f32(_p(gate), _p(up), _p(weights), _p(out), T, k, n, mode,
                                              clamp, int(combine), int(fast_exp), _s()))
    return out


def swiglu_q8_0_rows(gate, up, weights=None, mode=GLU_PLAIN, clamp=0.0, fast_exp=False, want_f32=False):
    """gate/up [T, k, n] -> (xq int8 [T, k, n], xscale [T, k, n/32], mid f32 or None): the SwiGLU rows as Q8_0 blocks."""
    T, k, n = gate.shape
    xq = torch.empty((T, k, n), dtype=torch.int8, device=gate.device)
    xs = torch.empty((T, k, n // 32), dtype=torch.float32, device=gate.device)
    mid = torch.empty((T, k, n), dtype=torch.float32, device=gate.device) if want_f32 else None
    check(_lib.load().ds4b200_swiglu_q8_0_rows_f32(_p(gate), _p(up), _p(weights), _p(xq), _p(xs), _p(mid), T, k, n, mode,
                                                   clamp, int(fast_exp), _s()))
    return xq, xs, mid


def hc_pre_rows(resid, fn_f16, scale3, base24, iters=20, eps=1e-6):
    """resid [T, 4, n]; fn_f16 [24, 4n] float16.  Returns (post [T,4], comb [T,16], out [T,n])."""
    T, _, n = resid.shape
    dev = resid.device
    post = torch.empty((T, 4), dtype=torch.float32, device=dev)
    comb = torch.empty((T, 16), dtype=torch.float32, device=dev)
    out = torch.empty((T, n), dtype=torch.float32, device=dev)
    check(_lib.load().ds4b200_hc_pre_rows_f32(_p(resid), _p(fn_f16), _p(scale3), _p(base24), _p(post),
                                              _p(comb), _p(out), T, n, iters, eps, _s()))
    return post, comb, out


def hc_pre_norm_rows(resid, fn_f16, scale3, base24, norm_w, iters=20, eps=1e-6, want_normed=True, want_q8=True):
    """hc_pre_rows followed by RMSNorm(out) * norm_w and its Q8_0 blocks.
    Returns (post, comb, out, normed or None, xq int8 [T, n] or None, xscale [T, n/32] or None)."""
    T, _, n = resid.shape
    dev = resid.device
    post = torch.empty((T, 4), dtype=torch.float32, device=dev)
    comb = torch.empty((T, 16), dtype=torch.float32, device=dev)
    out = torch.empty((T, n), dtype=torch.float32, device=dev)
    normed = torch.empty((T, n), dtype=torch.float32, device=dev) if want_normed else None
    xq = torch.empty((T, n), dtype=torch.int8, device=dev) if want_q8 else None
    xscale = torch.empty((T, n // 32), dtype=torch.float32, device=dev) if want_q8 else None
    check(_lib.load().ds4b200_hc_pre_norm_rows_f32(_p(resid), _p(fn_f16), _p(scale3), _p(base24), _p(norm_w), _p(post),
                                                   _p(comb), _p(out), _p(normed), _p(xq), _p(xscale), T, n, iters,
                                                   eps, _s()))
    return post, comb, out, normed, xq, xscale


def output_hc_head_rows(resid, fn_f16, scale1, base4, norm_w=None, eps=1e-6, want_out=True):
    """resid [T, 4, n]; fn_f16 [4, 4n].  Returns (out [T, n], normed [T, n] or None)."""
    T, _, n = resid.shape
    out = torch.empty((T, n), dtype=torch.float32, device=resid.device) if want_out else None
    normed = torch.empty((T, n), dtype=torch.float32, device=resid.device) if norm_w is not None else None
    check(_lib.load().ds4b200_output_hc_head_rows_f32(_p(resid), _p(fn_f16), _p(scale1), _p(base4), _p(norm_w),
                                                      _p(out), _p(normed), T, n, eps, _s()))
    return out, normed


def hc_post_rows(block_out, resid, post, comb, block_out2=None):
    T, _, n = resid.shape
    out = torch.empty_like(resid)
    check(_lib.load().ds4b200_hc_post_rows_f32(_p(block_out), _p(block_out2), _p(resid), _p(post),
                                               _p(comb), _p(out), T, n, _s()))
    return out


def hc_post_pre_rows(block_out, resid, post, comb, fn_f16, scale3, base24, block_out2=None, iters=20, eps=1e-6):
    """hc_post_rows then hc_pre_rows of its result.  Returns (out_hc [T,4,n], post [T,4], comb [T,16], out [T,n])."""
    T, _, n = resid.shape
    dev = resid.device
    out_hc = torch.empty_like(resid)
    post2 = torch.empty((T, 4), dtype=torch.float32, device=dev)
    comb2 = torch.empty((T, 16), dtype=torch.float32, device=dev)
    out = torch.empty((T, n), dtype=torch.float32, device=dev)
    check(_lib.load().ds4b200_hc_post_pre_rows_f32(_p(block_out), _p(block_out2), _p(resid), _p(post), _p(comb),
                                                   _p(fn_f16), _p(scale3), _p(base24), _p(out_hc), _p(post2), _p(comb2),
                                                   _p(out), T, n, iters, eps, _s()))
    return out_hc, post2, comb2, out


def hc_sinkhorn_rows(logits, iters=20, eps=1e-6):
    """logits [T, 16] -> comb [T, 16]."""
    comb = torch.empty_like(logits)
    check(_lib.load().ds4b200_hc_sinkhorn_rows_f32(_p(logits), _p(comb), logits.shape[0], iters, eps, _s()))
    return comb


def hc_sinkhorn_mix_rows(logits, resid, iters=20, eps=1e-6, want_comb=False):
    T, _, n = resid.shape
    out = torch.empty_like(resid)
    comb = torch.empty((T, 16), dtype=torch.float32, device=resid.device) if want_comb else None
    check(_lib.load().ds4b200_hc_sinkhorn_mix_rows_f32(_p(logits), _p(resid), _p(out), _p(comb), T, n,
                                                       iters, eps, _s()))
    return (out, comb) if want_comb else out


def e4m3_encode(x):
    codes = torch.empty(x.shape, dtype=torch.uint8, device=x.device)
    check(_lib.load().ds4b200_e4m3_encode_f32(_p(x), _p(codes), x.numel(), _s()))
    return codes


def e4m3_decode(codes):
    x = torch.empty(codes.shape, dtype=torch.float32, device=codes.device)
    check(_lib.load().ds4b200_e4m3_decode_f32(_p(codes), _p(x), codes.numel(), _s()))
    return x


def e4m3_selfcheck(first_bits: int, count: int) -> int:
    """Number of f32 bit patterns in the range whose hardware code differs from the table rule."""
    bad = torch.zeros(1, dtype=torch.int64, device="cuda")
    check(_lib.load().ds4b200_e4m3_selfcheck(first_bits, count, _p(bad), _s()))
    return int(bad.item())


def div_selfcheck(first: int, count: int) -> int:
    """Pairs (n, d in [1, 2]) for which the kernels' branch-free division differs from n / d."""
    bad = torch.zeros(1, dtype=torch.int64, device="cuda")
    check(_lib.load().ds4b200_div_selfcheck(first, count, _p(bad), _s()))
    return int(bad.item())


# ------------------------------------------------------------------ paged key-value cache

def _t(t, dtype, shape, what, device):
    """Device pointer of a tensor that has to have this type, shape and device."""
    if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.device != device or tuple(t.shape) != tuple(shape):
        have = f"{t.dtype} {tuple(t.shape)} on {t.device}" if isinstance(t, torch.Tensor) else type(t).__name__
        raise ValueError(f"{what}: expected {dtype} {tuple(shape)} on {device}, got {have}")
    return _p(t)


def _opt(t, dtype, shape, what, device):
    return None if t is None else _t(t, dtype, shape, what, device)


class PagedKv:
    """The pool's rows of one layer, as attention reads them: the tensors the store ops fill, seen as pages of
    `page_rows` rows.  codes uint8 [n_slots, head_dim] with scales f32 [n_slots, n_scales] (and tail f32
    [n_slots, n_rot] for KV_FP8_BLOCK64), or raw f32 [n_slots, head_dim]."""

    def __init__(self, row_format, page_rows, n_rot=64, codes=None, scales=None, tail=None, raw=None):
        rows = raw if row_format == KV_F32 else codes
        if rows is None or rows.dim() != 2:
            raise ValueError("PagedKv: codes / raw must be [n_slots, head_dim]")
        n, dim = rows.shape
        if page_rows < 1 or n % page_rows:
            raise ValueError("PagedKv: the rows must make whole pages")
        dev = rows.device
        k = self.struct = _lib.PagedKvStruct(row_format, dim, n_rot, page_rows, n // page_rows)
        if row_format == KV_F32:
            k.raw = _t(raw, torch.float32, (n, dim), "raw", dev)
        elif row_format in (KV_FP8_BLOCK64, KV_FP8_ROW):
            n_scales = (dim - n_rot) // 64 if row_format == KV_FP8_BLOCK64 else 1
            k.codes = _t(codes, torch.uint8, (n, dim), "codes", dev)
            k.scales = _t(scales, torch.float32, (n, n_scales), "scales", dev)
            if row_format == KV_FP8_BLOCK64 and n_rot:
                k.tail = _t(tail, torch.float32, (n, n_rot), "tail", dev)
        else:
            raise ValueError("PagedKv: unknown row format")
        self.tensors = (codes, scales, tail, raw)     # kept alive
        self.head_dim, self.page_rows, self.n_pages, self.device = dim, page_rows, n // page_rows, dev


def attn_workspace(n_heads, head_dim, device="cuda"):
    """Workspace of the attention ops below; calls that may overlap need one each."""
    n = _lib.load().ds4b200_attn_workspace_bytes(n_heads, head_dim)
    if n < 0:
        check(n)
    return torch.empty(n, dtype=torch.uint8, device=device)


def _attn(q, kv, page_table, kv_len, q_start, window, n_first, scale, sink, workspace, out, want_lse):
    if q.dim() != 3 or q.shape[2] != kv.head_dim:
        raise ValueError("attention: q must be [tokens, n_heads, head_dim] with the cache's head_dim")
    T, H, D = q.shape
    dev = kv.device
    n_seqs, width = page_table.shape
    if q_start is None and n_seqs != T:
        raise ValueError("attn_decode_paged: one token per sequence")
    if not (0 <= window < 1 << 31 and 0 <= n_first < 1 << 31):
        raise ValueError("attention: window and n_first must be in [0, 2^31)")
    if workspace is not None and workspace.device != dev:
        raise ValueError("attention: the workspace must be on the cache's device")
    with torch.cuda.device(dev):
        out = torch.empty_like(q) if out is None else out
        lse = torch.empty((T, H), dtype=torch.float32, device=dev) if want_lse else None
        ws = attn_workspace(H, D, dev) if workspace is None else workspace
        args = (page_table.data_ptr() if n_seqs == 0 else _t(page_table, torch.int32, (n_seqs, width), "page_table", dev), width,
                _t(kv_len, torch.int32, (n_seqs,), "kv_len", dev))
        rest = (n_seqs, H, D ** -0.5 if scale is None else scale, _opt(sink, torch.float32, (H,), "sink", dev), window, n_first,
                _t(out, torch.bfloat16, (T, H, D), "out", dev), _p(lse), _p(ws), ws.numel() * ws.element_size(), _s())
        qp = _t(q, torch.bfloat16, (T, H, D), "q", dev)
        if q_start is None:
            check(_lib.load().ds4b200_attn_decode_paged_bf16(qp, C.byref(kv.struct), *args, *rest))
        else:
            check(_lib.load().ds4b200_attn_window_paged_bf16(
                qp, T, C.byref(kv.struct), *args, _t(q_start, torch.int32, (n_seqs + 1,), "q_start", dev), *rest))
    return (out, lse) if want_lse else out


def attn_decode_paged(q, kv, page_table, kv_len, window=0, n_first=0, scale=None, sink=None, workspace=None, out=None,
                      want_lse=False):
    """Attention of one new token per sequence.  q bf16 [n_seqs, n_heads, head_dim], kv a PagedKv, page_table int32
    [n_seqs, width], kv_len int32 [n_seqs] (rows in the cache, the token's own among them).  The token sees the
    last `window` rows (0: all) and the `n_first` first ones.  scale: 1/sqrt(head_dim) by default; sink f32
    [n_heads]: a logit without a row.  At most 4096 sequences; `out` overlaps none of the inputs.  Returns out bf16 like q, with want_lse (out, lse f32 [n_seqs, n_heads])."""
    return _attn(q, kv, page_table, kv_len, None, window, n_first, scale, sink, workspace, out, want_lse)


def attn_window_paged(q, kv, page_table, kv_len, q_start, window=0, n_first=0, scale=None, sink=None, workspace=None, out=None,
                      want_lse=False):
    """Attention of a chunk: tokens q_start[b] .. q_start[b + 1] - 1 of q bf16 [tokens, n_heads, head_dim] are the last
    rows of sequence b, and each sees the rows up to its own, as in attn_decode_paged.  Rows of `out` outside
    [q_start[0], q_start[-1]) are left as they are."""
    return _attn(q, kv, page_table, kv_len, q_start, window, n_first, scale, sink, workspace, out, want_lse)


class PagePool:
    """The buffers whose pages move together (e.g. codes, scales and tail of every layer; each holds `n_pages` pages,
    by default its first dimension) and the workspace of the page ops on them."""

    def __init__(self, arrays, page_rows, n_seqs, table_width, n_pages=None, max_list=None):
        if not arrays and n_pages is None:
            raise ValueError("PagePool: n_pages is needed without arrays")
        self.n_pages = arrays[0].shape[0] if n_pages is None else n_pages
        self.page_rows, self.n_seqs, self.width = page_rows, n_seqs, table_width
        self.arrays = list(arrays)
        self.device = arrays[0].device if arrays else torch.device("cuda", torch.cuda.current_device())
        self.c_arrays = (_lib.PageArray * max(1, len(arrays)))()
        for i, a in enumerate(arrays):
            size = a.numel() * a.element_size()
            if a.device != self.device or size % max(1, self.n_pages):
                raise ValueError(f"PagePool: array {i} does not hold {self.n_pages} whole pages on {self.device}")
            self.c_arrays[i] = _lib.PageArray(_p(a), size // max(1, self.n_pages))
        self.max_list = n_seqs if max_list is None else max_list
        n = _lib.load().ds4b200_pages_workspace_bytes(self.n_pages, n_seqs, self.max_list)
        if n < 0:
            check(n)
        self.workspace = torch.empty(n, dtype=torch.uint8, device=self.device)

    def _ws(self):
        return _p(self.workspace), self.workspace.numel()

    def _tables(self, refs, table, lens, refs_out, table_out, lens_out):
        d, n = self.device, (self.n_seqs,)
        shape = (self.n_seqs, self.width)
        out = (refs if refs_out is None else refs_out, table if table_out is None else table_out, lens if lens_out is None else lens_out)
        ptrs = [_t(refs, torch.int32, (self.n_pages,), "refs", d), _t(out[0], torch.int32, (self.n_pages,), "refs_out", d),
                _t(table, torch.int32, shape, "table", d), _t(out[1], torch.int32, shape, "table_out", d)]
        if lens is not None:
            ptrs += [_t(lens, torch.int32, n, "lens", d), _t(out[2], torch.int32, n, "lens_out", d)]
        return ptrs, out

    def _status(self, status):
        return torch.empty(1, dtype=torch.int32, device=self.device) if status is None else status


def pages_copy(pool, moves, status=None):
    """Copies page moves[i, 0] to page moves[i, 1] (int32 [n, 2]) in every array; returns the status tensor."""
    with torch.cuda.device(pool.device):
        st = pool._status(status)
        n = moves.shape[0]
        check(_lib.load().ds4b200_pages_copy(pool.c_arrays, len(pool.arrays), pool.n_pages,
                                             _t(moves, torch.int32, (n, 2), "moves", pool.device), n,
                                             _t(st, torch.int32, (1,), "status", pool.device), *pool._ws(), _s()))
    return st


def pages_fork(pool, refs, table, lens, pairs, refs_out=None, table_out=None, lens_out=None, status=None):
    """Sequence pairs[i, 1] becomes a fork of sequence pairs[i, 0]: full pages shared, a part-filled last page
    copied.  In place unless *_out are given.  Returns (refs, table, lens, status): status int32 [1], 0 = done,
    > 0 = free pages missing, -1 = list not valid (nothing changed then)."""
    with torch.cuda.device(pool.device):
        ptrs, out = pool._tables(refs, table, lens, refs_out, table_out, lens_out)
        st = pool._status(status)
        n = pairs.shape[0]
        check(_lib.load().ds4b200_pages_fork(pool.c_arrays, len(pool.arrays), pool.n_pages, pool.page_rows, *ptrs, pool.n_seqs,
                                             pool.width, _t(pairs, torch.int32, (n, 2), "pairs", pool.device), n,
                                             _t(st, torch.int32, (1,), "status", pool.device), *pool._ws(), _s()))
    return (*out, st)


def pages_reserve(pool, refs, table, lens, new_lens, refs_out=None, table_out=None, lens_out=None, status=None):
    """Pages for new_lens[b] rows of every sequence.  Returns (refs, table, lens, status) as pages_fork."""
    with torch.cuda.device(pool.device):
        ptrs, out = pool._tables(refs, table, lens, refs_out, table_out, lens_out)
        st = pool._status(status)
        check(_lib.load().ds4b200_pages_reserve(pool.n_pages, pool.page_rows, *ptrs,
                                                _t(new_lens, torch.int32, (pool.n_seqs,), "new_lens", pool.device), pool.n_seqs,
                                                pool.width, _t(st, torch.int32, (1,), "status", pool.device), *pool._ws(), _s()))
    return (*out, st)


def pages_free(pool, refs, table, lens, seqs, refs_out=None, table_out=None, lens_out=None, status=None):
    """Takes the pages of the listed sequences (int32 [n]) from them.  Returns (refs, table, lens, status)."""
    with torch.cuda.device(pool.device):
        ptrs, out = pool._tables(refs, table, lens, refs_out, table_out, lens_out)
        st = pool._status(status)
        n = seqs.shape[0]
        check(_lib.load().ds4b200_pages_free(pool.n_pages, pool.page_rows, *ptrs, pool.n_seqs, pool.width,
                                             _t(seqs, torch.int32, (n,), "seqs", pool.device), n,
                                             _t(st, torch.int32, (1,), "status", pool.device), *pool._ws(), _s()))
    return (*out, st)


def pages_compact(pool, refs, table, refs_out=None, table_out=None, n_live=None):
    """Packs the pages in use to the pool's lower end.  Returns (refs, table, n_live int32 [1])."""
    with torch.cuda.device(pool.device):
        ptrs, out = pool._tables(refs, table, None, refs_out, table_out, None)
        n = pool._status(n_live)
        check(_lib.load().ds4b200_pages_compact(pool.c_arrays, len(pool.arrays), pool.n_pages, *ptrs, pool.n_seqs, pool.width,
                                                _t(n, torch.int32, (1,), "n_live", pool.device), *pool._ws(), _s()))
    return out[0], out[1], n
