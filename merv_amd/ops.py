"""
Tensor-level wrappers of the single-kernel C-ABI entry points (include/merv_hip.h, "single kernels" section).
Used by the parity tests and micro-benchmarks; the encoders themselves run through merv_encoder_forward.
All tensors must be contiguous CUDA (ROCm) tensors: bf16 activations / GEMM weights, fp32 vectors (the paged cache takes strides).
"""
from __future__ import annotations

import struct
from typing import Optional

import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib
from ._lib import ACT, DT_BF16, DT_F32, KV_BF16, KV_E4M3, PagedCache, check, current_stream_ptr, ptr


def _chk(t: Optional[torch.Tensor], dtype, name: str):
    if t is None:
        return
    if not t.is_cuda or t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous CUDA tensor of {dtype}, got {t.dtype} on {t.device}")


def gemm(a: torch.Tensor, w: torch.Tensor, bias=None, act: str = "none", lscale=None, res=None, res_row_mod: int = 0,
         out: Optional[torch.Tensor] = None, out_group: int = 0, out_stride: int = 0, out_off: int = 0) -> torch.Tensor:
    """out = res + lscale * act(a @ w.T + bias); a [M,K] bf16, w [N,K] bf16 (nn.Linear layout)."""
    _chk(a, torch.bfloat16, "a"); _chk(w, torch.bfloat16, "w"); _chk(bias, torch.float32, "bias")
    _chk(lscale, torch.float32, "lscale"); _chk(res, torch.bfloat16, "res")
    M, K = a.shape
    N = w.shape[0]
    if w.shape[1] != K:
        raise ValueError(f"gemm: K mismatch {a.shape} x {w.shape}")
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=a.device)
    _chk(out, torch.bfloat16, "out")
    lib = _lib.load()
    rc = lib.merv_gemm_bf16(ptr(a), ptr(w), ptr(out), ptr(bias), ptr(lscale), ptr(res), M, N, K, K, K, out.shape[-1],
                            res.shape[-1] if res is not None else 0, res_row_mod, out_group, out_stride, out_off,
                            ACT[act], current_stream_ptr(a.device))
    check(rc, "merv_gemm_bf16")
    return out


def layernorm(x: torch.Tensor, gamma, beta, eps: float, add=None, add_div: int = 1, add_mod: int = 1) -> torch.Tensor:
    """y = LN(x (+ add[(row // add_div) % add_mod], written back into x)). x [M,D] bf16."""
    _chk(x, torch.bfloat16, "x"); _chk(gamma, torch.float32, "gamma"); _chk(beta, torch.float32, "beta")
    _chk(add, torch.float32, "add")
    M, D = x.shape
    y = torch.empty_like(x)
    rc = _lib.load().merv_layernorm(ptr(x), ptr(y), ptr(gamma), ptr(beta), ptr(add), M, D, add_div, add_mod, eps,
                                    current_stream_ptr(x.device))
    check(rc, "merv_layernorm")
    return y


def attention(qkv: torch.Tensor, nseq: int, L: int, heads: int) -> torch.Tensor:
    """qkv [nseq*L, 3*D] bf16 -> [nseq*L, D] bf16, head_dim 64."""
    _chk(qkv, torch.bfloat16, "qkv")
    D = heads * 64
    if qkv.shape != (nseq * L, 3 * D):
        raise ValueError(f"attention: qkv shape {tuple(qkv.shape)} != {(nseq * L, 3 * D)}")
    out = torch.empty(nseq * L, D, dtype=torch.bfloat16, device=qkv.device)
    rc = _lib.load().merv_attention(ptr(qkv), ptr(out), nseq, L, heads, D, 0.125, current_stream_ptr(qkv.device))
    check(rc, "merv_attention")
    return out


def temporal_attention(qkv: torch.Tensor, nclips: int, t: int, ntok: int, heads: int) -> torch.Tensor:
    """Rows are frame-major (row = (clip*t + i) * ntok + token); attends over i for each (clip, token, head)."""
    _chk(qkv, torch.bfloat16, "qkv")
    D = heads * 64
    if qkv.shape != (nclips * t * ntok, 3 * D):
        raise ValueError("temporal_attention: bad qkv shape")
    out = torch.empty(nclips * t * ntok, D, dtype=torch.bfloat16, device=qkv.device)
    rc = _lib.load().merv_temporal_attention(ptr(qkv), ptr(out), nclips, t, ntok, heads, D, 0.125,
                                             current_stream_ptr(qkv.device))
    check(rc, "merv_temporal_attention")
    return out


def im2col(pix: torch.Tensor, layout: str, patch: int, tubelet: int, k_pad: int) -> torch.Tensor:
    """pix [B,F,3,H,W] ("BFCHW") or [B,3,F,H,W] ("BCFHW"), fp32 or bf16 -> [B*(F/tubelet)*hp*hp, k_pad] bf16."""
    if not pix.is_cuda or not pix.is_contiguous() or pix.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("im2col: contiguous CUDA fp32/bf16 pixels required")
    if layout == "BFCHW":
        B, Fr, _, H, W = pix.shape
        sB, sF, sC = Fr * 3 * H * W, 3 * H * W, H * W
    else:
        B, _, Fr, H, W = pix.shape
        sB, sC, sF = 3 * Fr * H * W, Fr * H * W, H * W
    hp = H // patch
    out = torch.empty(B * (Fr // tubelet) * hp * hp, k_pad, dtype=torch.bfloat16, device=pix.device)
    rc = _lib.load().merv_im2col(ptr(pix), DT_BF16 if pix.dtype == torch.bfloat16 else DT_F32, ptr(out), B, Fr, H, patch,
                                 tubelet, k_pad, sB, sF, sC, current_stream_ptr(pix.device))
    check(rc, "merv_im2col")
    return out


def pool3d(tokens: torch.Tensor, T: int, S: int, out_size: int) -> torch.Tensor:
    """tokens [B, T*S*S, C] bf16 -> [B, T*out*out, C] bf16 (AdaptiveAvgPool3d((T,out,out)))."""
    _chk(tokens, torch.bfloat16, "tokens")
    B, N, Cc = tokens.shape
    if N != T * S * S:
        raise ValueError("pool3d: token count != T*S*S")
    out = torch.empty(B, T * out_size * out_size, Cc, dtype=torch.bfloat16, device=tokens.device)
    rc = _lib.load().merv_pool3d(ptr(tokens), ptr(out), B, T, S, out_size, Cc, current_stream_ptr(tokens.device))
    check(rc, "merv_pool3d")
    return out


# ---- MXFP8 mode ----
def quantize_mxfp8(x: torch.Tensor):
    """bf16 [rows, K] -> (q uint8 [rows, K] OCP e4m3, scales uint8 in the GEMM's lane order); include/merv_hip.h."""
    lib = _lib.load()
    if x.dtype != torch.bfloat16 or x.dim() != 2 or x.stride(1) != 1 or not x.is_cuda:
        raise ValueError("quantize_mxfp8: expected a CUDA bf16 [rows, K] tensor with contiguous rows")
    rows, K = x.shape
    if K % 128:
        raise ValueError("quantize_mxfp8: K must be a multiple of 128")
    q = torch.empty(rows, K, dtype=torch.uint8, device=x.device)
    sc = torch.zeros(lib.merv_mxfp8_scale_bytes(rows, K), dtype=torch.uint8, device=x.device)
    check(lib.merv_quantize_mxfp8(ptr(x), rows, K, x.stride(0), ptr(q), ptr(sc), current_stream_ptr(x.device)), "merv_quantize_mxfp8")
    return q, sc


def mxfp8_scales_to_rows(sc: torch.Tensor, rows: int, K: int) -> torch.Tensor:
    """Un-permute the lane-order scale array to [rows, K/32] (tests / inspection)."""
    groups = (rows + 63) // 64
    s = sc.view(K // 128, groups, 4, 16, 4)  # [ktile][group][kblock%4][row%16][(row%64)/16]
    s = s.permute(1, 4, 3, 0, 2).reshape(groups * 64, K // 32)  # row = 64*group + 16*j + r ; kblock = 4*ktile + kq
    return s[:rows]


def gemm_mxfp8(aq, a_sc, wq, w_sc, bias=None, act="none", lscale=None, res=None, out=None):
    lib = _lib.load()
    M, K = aq.shape
    N = wq.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=torch.bfloat16, device=aq.device)
    check(lib.merv_gemm_mxfp8(ptr(aq), ptr(a_sc), ptr(wq), ptr(w_sc), ptr(out), ptr(bias), ptr(lscale), ptr(res), M, N, K,
                              aq.stride(0), wq.stride(0), out.stride(0), res.stride(0) if res is not None else 0, ACT[act],
                              current_stream_ptr(aq.device)), "merv_gemm_mxfp8")
    return out


# ---- paged key / value cache (PagedDecoder, paged.py): rows of unlike length on one pool of pages ----
# Pages are [n_pages, kv_heads, page_size, head_dim], bf16 or torch.float8_e4m3fn (then with uint8 scales [n_pages, kv_heads, page_size], a number
# standing for code * 2^(byte - 127)); table [rows, width] int32 names the page of positions i * page_size .. of a row. Any strides, last
# dimension contiguous. Row lengths, offsets and page numbers stay on the device (a captured step replays with new ones); the kernels check
# them: see include/merv_hip.h for what a bad one does. All of this is for inference: no gradients.
# These calls are made once a layer and token, so their checks read each attribute of a tensor once and build the C structure in one step.
_PAGED_CACHE = struct.Struct("@5P7q6i")  # merv_paged_cache


# a twentieth of torch.cuda.current_stream(dev).cuda_stream's 1.9 us; a torch without a GPU has neither (there the calls refuse their tensors before they need them)
_raw_stream, _raw_device = getattr(torch._C, "_cuda_getCurrentRawStream", None), getattr(torch._C, "_cuda_getDevice", None)
_E4M3, _BF16, _I32 = torch.float8_e4m3fn, torch.bfloat16, torch.int32


def _no_gradient(what: str, name: str, t: torch.Tensor) -> None:
    """What would need a gradient, or carries a tangent of forward-mode differentiation, is refused: there is no formula for either."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what}: {name} requires a gradient, and there is none: call it under torch.no_grad()")
    if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{what}: {name} carries a tangent, and there is none of the result")


def _paged_cache(what: str, k_pages, v_pages, table, k_scales, v_scales, written: bool = False):
    """-> (the C structure, device index, rows, kv_heads, head_dim, positions that a row's table can hold)."""
    kind, shape, st, dev = k_pages.dtype, k_pages.shape, k_pages.stride(), k_pages.get_device()
    if (kind is not _BF16 and kind is not _E4M3) or len(st) != 4 or dev < 0:
        raise ValueError(f"{what}: expected CUDA pages [n_pages, kv_heads, page_size, head_dim] of bfloat16 or float8_e4m3fn, got "
                         f"{kind} {tuple(shape)} on {k_pages.device}")
    if v_pages.dtype is not kind or v_pages.shape != shape or v_pages.stride() != st or v_pages.get_device() != dev:
        raise ValueError(f"{what}: v_pages must have the type, shape, strides and device of k_pages")
    if (k_pages.requires_grad or v_pages.requires_grad) and torch.is_grad_enabled():
        raise ValueError(f"{what}: the pages require a gradient, and there is none: call it under torch.no_grad()")
    if _forward_ad._current_level >= 0 and kind is _BF16:
        _no_gradient(what, "k_pages", k_pages)
        _no_gradient(what, "v_pages", v_pages)
    n_pages, kv_heads, page, hd = shape
    sp, sh, ss, last = st
    if last != 1:
        raise ValueError(f"{what}: the pages' last dimension must be contiguous")
    tst = table.stride()
    if len(tst) != 2 or table.dtype is not _I32 or table.get_device() != dev or (tst[1] != 1 and table.shape[1] > 1):
        raise ValueError(f"{what}: expected an int32 table [rows, width] on cuda:{dev} with contiguous rows")
    rows, width = table.shape
    kp, vp = k_pages.data_ptr(), v_pages.data_ptr()
    ks = vs = ssp = ssh = 0
    if kind is _E4M3:
        if k_scales is None or v_scales is None:
            raise ValueError(f"{what}: float8_e4m3fn pages need k_scales and v_scales")
        sst = k_scales.stride()
        for x in (k_scales, v_scales):
            if x.dtype is not torch.uint8 or x.shape != shape[:3] or x.get_device() != dev or x.stride() != sst or sst[2] != 1:
                raise ValueError(f"{what}: expected uint8 scales {tuple(shape[:3])} on cuda:{dev}, tokens contiguous, of the same strides")
        ks, vs, ssp, ssh = k_scales.data_ptr(), v_scales.data_ptr(), sst[0], sst[1]
    elif k_scales is not None or v_scales is not None:
        raise ValueError(f"{what}: bfloat16 pages take no scales")
    if n_pages == 1:  # the stride of a dimension of one means nothing
        sp = ssp = 0
    if kv_heads == 1:
        sh = ssh = 0
    if written and (kp == vp or ks and (ks == vs or ssp == 0 and n_pages > 1 or ssh == 0 and kv_heads > 1)
                    or sp == 0 and n_pages > 1 or sh == 0 and kv_heads > 1 or ss == 0) and n_pages:
        raise ValueError(f"{what}: pages and scales that are written must not share memory")
    c = PagedCache.from_buffer_copy(_PAGED_CACHE.pack(kp, vp, ks, vs, table.data_ptr(), n_pages, sp, sh, ss, ssp, ssh, tst[0] if rows > 1 else 0, rows, width,
                                                      kv_heads, hd, page, KV_BF16 if kind is _BF16 else KV_E4M3))
    return c, dev, rows, kv_heads, hd, width * page


def _paged_rows(what: str, name: str, t: torch.Tensor, shape, dev: int, out: bool = False):
    st = t.stride()
    if t.dtype is not _BF16 or t.shape != shape or t.get_device() != dev or st[2] != 1:
        raise ValueError(f"{what}: {name}: expected bfloat16 {tuple(shape)} on cuda:{dev} with contiguous last dimension, got {t.dtype} "
                         f"{tuple(t.shape)} on {t.device}")
    if t.requires_grad or _forward_ad._current_level >= 0:
        _no_gradient(what, name, t)
    s0, s1, _ = st
    if shape[0] <= 1:
        s0 = 0
    elif out and s0 == 0:
        raise ValueError(f"{what}: {name}: an output's rows must not share memory")
    if shape[1] <= 1:
        s1 = 0
    elif out and s1 == 0:
        raise ValueError(f"{what}: {name}: an output's rows must not share memory")
    return t.data_ptr(), s0, s1


def _paged_ints(what: str, name: str, t: Optional[torch.Tensor], n: int, dev: int) -> int:
    if t is None:
        return 0
    if t.dtype is not _I32 or t.shape != (n,) or t.get_device() != dev or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{what}: {name}: expected contiguous int32 [{n}] on cuda:{dev}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _paged_tables(what: str, cos: torch.Tensor, sin: torch.Tensor, hd: int, dev: int):
    st, shape = cos.stride(), cos.shape
    for name, t in (("cos", cos), ("sin", sin)):
        if t.dtype is not _BF16 or t.shape != shape or len(st) != 2 or shape[1] != hd or t.get_device() != dev or t.stride() != st or st[1] != 1:
            raise ValueError(f"{what}: expected bfloat16 rotary tables [positions, {hd}] on cuda:{dev} with contiguous rows, of the same strides")
        if t.requires_grad or _forward_ad._current_level >= 0:
            _no_gradient(what, name, t)
    return cos.data_ptr(), sin.data_ptr(), shape[0], st[0] if shape[0] > 1 else hd


def _launch_on(dev: int, call, what: str, *args) -> None:
    """call(*args, stream) on the device's current stream; the device is made current where it is not (its null stream has no device of its own)."""
    if _raw_device() == dev:
        rc = call(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = call(*args, _raw_stream(dev))
    if rc:
        check(rc, what)


def paged_cache_write(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, start: torch.Tensor,
                      offsets: Optional[torch.Tensor] = None, *, k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
                      q: Optional[torch.Tensor] = None, cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                      q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """New tokens k, v [T, kv_heads, head_dim] bf16 into the pages, in one launch with the rotary embedding of k and of q [T, heads, head_dim] where
    cos, sin [positions, head_dim] bf16 are given. Token t is row b's where offsets[b] <= t < offsets[b + 1] (int32 [rows + 1]; None: one token a
    row, t = b), at position start[b] + t - offsets[b]; rows with start[b] < 0 and tokens behind offsets[rows] are left alone, in every output. Returns
    the rotated queries (q_out, or a new tensor; q_out=q rotates in place), None without q; k_out takes the rotated keys as well (k_out=k: in place). Outputs share
    no memory with other operands. float8_e4m3fn pages:
    quantised with one power-of-two scale for each token and head (k_scales, v_scales); what is not finite becomes NaN. Two tokens of a call must not lie in
    the same place of a page (rows may share pages that are only read)."""
    what = "paged_cache_write"
    cache, dev, rows, kv_heads, hd, _ = _paged_cache(what, k_pages, v_pages, table, k_scales, v_scales, True)
    if k.dim() != 3:
        raise ValueError(f"{what}: k: expected [tokens, kv_heads, head_dim], got {tuple(k.shape)}")
    T = k.shape[0]
    shape = (T, kv_heads, hd)
    if T > 1 << 28:
        raise ValueError(f"{what}: at most 2^28 tokens a call")
    if offsets is None and T != rows:
        raise ValueError(f"{what}: without offsets there is one token for each row: {T} tokens, {rows} rows")
    kr, vr = _paged_rows(what, "k", k, shape, dev), _paged_rows(what, "v", v, shape, dev)
    off_p, start_p = _paged_ints(what, "offsets", offsets, rows + 1, dev), _paged_ints(what, "start", start, rows, dev)
    rope, heads, qr, qo, ko = (0, 0, 0, 0), 0, (0, 0, 0), (0, 0, 0), (0, 0, 0)
    if cos is not None and sin is not None:
        rope = _paged_tables(what, cos, sin, hd, dev)
    elif cos is not None or sin is not None or q is not None:
        raise ValueError(f"{what}: cos and sin come together, and q needs them")
    if q is not None:
        qshape = q.shape
        if len(qshape) != 3 or qshape[0] != T or qshape[2] != hd:
            raise ValueError(f"{what}: q: expected [{T}, heads, {hd}], got {tuple(qshape)}")
        heads = qshape[1]
        qr = _paged_rows(what, "q", q, qshape, dev)
        if q_out is None:
            q_out = torch.empty_like(q)
        qo = _paged_rows(what, "q_out", q_out, qshape, dev, True)
    elif q_out is not None:
        raise ValueError(f"{what}: q_out needs q")
    if k_out is not None:
        ko = _paged_rows(what, "k_out", k_out, shape, dev, True)
    _launch_on(dev, _lib.load().merv_paged_cache_write, what, cache, *kr, *vr, *qr, *rope, *qo, *ko, off_p, start_p, T, heads)
    return q_out


def paged_cache_read(k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, start: Optional[torch.Tensor], offsets: torch.Tensor,
                     total: int, *, k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None,
                     k_out: Optional[torch.Tensor] = None, v_out: Optional[torch.Tensor] = None):
    """Cached keys and values, back as bf16 [total, kv_heads, head_dim] each, rows one behind the other: output t is row b's position
    (start[b] or 0) + t - offsets[b] where offsets[b] <= t < offsets[b + 1]. Outputs behind offsets[rows], and those of rows with start[b] < 0, are
    not written. A position without a page reads as NaN. Numbers are given back exactly as the cache holds
    them; e4m3 rows with numbers of 248 x 2^120 and more (bf16's eight largest) hold 2^128 there, which bf16 has no finite number for: infinity."""
    what = "paged_cache_read"
    cache, dev, rows, kv_heads, hd, _ = _paged_cache(what, k_pages, v_pages, table, k_scales, v_scales)
    total = int(total)
    if not 0 <= total <= 1 << 27 or offsets is None:
        raise ValueError(f"{what}: total must not be negative or over 2^27, and offsets are needed")
    shape = (total, kv_heads, hd)
    off_p, start_p = _paged_ints(what, "offsets", offsets, rows + 1, dev), _paged_ints(what, "start", start, rows, dev)
    if k_out is None:
        k_out = torch.empty(shape, dtype=_BF16, device=k_pages.device)
    if v_out is None:
        v_out = torch.empty(shape, dtype=_BF16, device=k_pages.device)
    ko, vo = _paged_rows(what, "k_out", k_out, shape, dev, True), _paged_rows(what, "v_out", v_out, shape, dev, True)
    _launch_on(dev, _lib.load().merv_paged_cache_read, what, cache, *ko, *vo, off_p, start_p, total)
    return k_out, v_out


def paged_decode_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *,
                           k_scales: Optional[torch.Tensor] = None, v_scales: Optional[torch.Tensor] = None, scale: Optional[float] = None,
                           window: int = 0, out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of one token for each row, q [rows, heads, head_dim] bf16, over positions max(0, lens[b] - window) .. lens[b] - 1 of the row's pages
    (window 0: all of them; kv head = head // (heads // kv_heads); scale None: head_dim^-0.5). Returns out, or (out, lse [rows, heads] fp32, the
    natural logarithm of the softmax's sum). A row of length 0 gives zeros and -inf; a length over the table's capacity or a bad page gives
    that row NaN. Sums, softmax and the weights of the values are held in fp32; rounded to bf16 once, at the end."""
    what = "paged_decode_attention"
    cache, dev, rows, kv_heads, hd, capacity = _paged_cache(what, k_pages, v_pages, table, k_scales, v_scales)
    qshape = q.shape
    heads = qshape[1] if len(qshape) == 3 else 0
    if heads == 0 or qshape[0] != rows or qshape[2] != hd or heads % kv_heads:
        raise ValueError(f"{what}: q: expected [{rows}, heads, {hd}] with heads a multiple of {kv_heads}, got {tuple(qshape)}")
    if window < 0:
        raise ValueError(f"{what}: window must not be negative")
    qr, lens_p = _paged_rows(what, "q", q, qshape, dev), _paged_ints(what, "lens", lens, rows, dev)
    if out is None:
        out = torch.empty_like(q)
    orow = _paged_rows(what, "out", out, qshape, dev, True)
    lse = torch.empty((rows, heads), dtype=torch.float32, device=q.device) if return_lse else None
    lib = _lib.load()
    # a workspace of its own for each call (and each captured graph): nothing is shared by calls that run at the same time
    nbytes = lib.merv_paged_decode_attention_workspace_bytes(rows, heads, kv_heads, hd, capacity)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _launch_on(dev, lib.merv_paged_decode_attention, what, cache, *qr, *orow, 0 if lse is None else lse.data_ptr(), lens_p, heads, int(window),
               hd**-0.5 if scale is None else float(scale), 0 if ws is None else ws.data_ptr(), nbytes)
    return (out, lse) if return_lse else out
