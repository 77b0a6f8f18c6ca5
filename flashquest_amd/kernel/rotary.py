"""Appending a step's tokens to one layer's cache with the rotary embedding applied on the way, and reading a
cache's tokens back as values.

The reference's attention patch rotates the projections' q and k with transformers' apply_rotary_pos_emb and hands
the keys to the cache's update_quantized (src/flashquest/eager/llama_persistent_patch.py:186-194).  ``rotate_append``
does both, and the queries, in one launch: for the rotated channels i < R/2 of a row x and the cos / sin rows of
its position

    y[i] = x[i] cos[i] - x[i + R/2] sin[i]          y[i + R/2] = x[i + R/2] cos[i + R/2] + x[i] sin[i + R/2]

in fp32, rounded once to the tokens' type; channels from R on are unchanged.  What the cache then holds is
bit-identical to update_quantized of keys rotated like that.
"""
from __future__ import annotations

import contextlib

import torch

from .. import _host
from .. import _lib as L
from .. import _ops

_PLANES = {4: ("K_packed", "K_scale", "K_mn", "V_packed", "V_scale", "V_mn"),
           8: ("K_uint8", "K_scale", "K_mn", "V_uint8", "V_scale", "V_mn"),
           3: ("K_msb", "K_lsb", "K_scale_turbo", "V_msb", "V_lsb", "V_scale_turbo", "K_scale_raw", "K_mn_raw")}


def cache_bits(cache: dict) -> int:
    """4, 8 or 3 (TurboQuant): the family of a layer's buffers or views, by its keys."""
    for bits, names in _PLANES.items():
        if all(n in cache for n in names):
            return bits
    raise ValueError(f"not the buffers or views of an INT4, INT8 or TurboQuant cache layer: {sorted(cache)}")


def _layer_planes(cache: dict, bits: int) -> list:
    """The planes of one layer, their types checked (shapes are the callers')."""
    planes = [cache[n] for n in _PLANES[bits]]
    codes = (0, 3) if bits != 3 else (0, 1, 3, 4)
    for i, (n, t) in enumerate(zip(_PLANES[bits], planes)):
        if t.dim() != 4:
            raise ValueError(f"{n} must be one layer's, (B, H_kv, ...); got {tuple(t.shape)}")
        if (t.dtype == torch.uint8) != (i in codes) or (i not in codes and t.dtype not in (torch.bfloat16, torch.float16)):
            raise AssertionError(f"{n}: codes are uint8, metadata bf16 or fp16; got {t.dtype}")
        if bits == 3 and i not in codes and t.dtype != torch.bfloat16:
            raise AssertionError(f"{n} must be bf16; got {t.dtype}")
    if bits != 3 and planes[4].shape != planes[5].shape:
        raise ValueError(f"V_scale and V_mn must share one shape; got {tuple(planes[4].shape)} and {tuple(planes[5].shape)}")
    return planes


def on_device(t: torch.Tensor):
    """Launches for t's device: a context that makes it the current one where it is not."""
    if t.device.index is None or t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def same_device(*tensors) -> None:
    L.require_device(*tensors)
    if any(t.device != tensors[0].device for t in tensors):
        raise ValueError("the tensors are on different devices: " + ", ".join(sorted({str(t.device) for t in tensors})))


def _rows(t: torch.Tensor) -> torch.Tensor:
    return _ops._ensure_inner_contiguous(t, 16 // t.element_size())


def _check_tokens(q, k, v, cos, sin):
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape:
        raise ValueError(f"q must be (B, H_q, S, D), k and v one (B, H_kv, S, D) shape; got {tuple(q.shape)}, "
                         f"{tuple(k.shape)} and {tuple(v.shape)}")
    B, H_q, S, D = q.shape
    if (k.shape[0], k.shape[2], k.shape[3]) != (B, S, D):
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} disagree on the batch, the tokens or head_dim")
    if not (q.dtype == k.dtype == v.dtype):
        raise AssertionError("q, k and v must share a dtype")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"tokens must be bf16 or fp16; got {q.dtype}")
    if cos.shape != sin.shape or cos.dtype != sin.dtype or cos.dim() != 3:
        raise ValueError(f"cos and sin must share one (B or 1, S, R) shape and dtype; got {tuple(cos.shape)} "
                         f"{cos.dtype} and {tuple(sin.shape)} {sin.dtype}")
    if cos.shape[0] not in (1, B) or cos.shape[1] != S:
        raise ValueError(f"cos and sin are for {tuple(cos.shape[:2])} (batch, tokens), the tokens are ({B}, {S})")
    R = cos.shape[2]
    if R < 16 or R > D or R % 16:
        raise NotImplementedError(f"{R} rotated channels of {D}: a multiple of 16 is taken")
    if cos.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise NotImplementedError(f"cos and sin must be fp32, bf16 or fp16; got {cos.dtype}")


def _rotary(q, q_out, cos, sin, B):
    """The descriptor of one step's angles and queries, and the tensors it points into."""
    if cos.dtype not in (q.dtype, torch.float32):
        cos, sin = cos.float(), sin.float()
    q, cos, sin = _rows(q), _rows(cos), _rows(sin)

    def angle(t):
        st = t.stride()
        return L.I64x3(st[0] if t.shape[0] > 1 or B == 1 else 0, st[1], st[2])

    r = L.Rotary(cos.data_ptr(), angle(cos), sin.data_ptr(), angle(sin), L.dtype_code(cos.dtype), cos.shape[2],
                 q.data_ptr(), L.strides(q, 4), q_out.data_ptr(), L.strides(q_out, 4), q.shape[1])
    return r, (q, cos, sin)


def rotate(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor):
    """The rotation alone: (q, k) rotated, as contiguous tensors.  Arguments as rotate_append's."""
    _check_tokens(q, k, k, cos, sin)
    B, _, S, D = q.shape
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim={D} not in (64, 128)")
    same_device(q, k, cos, sin)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if q.numel() + k.numel() == 0:
        return q_out, k_out
    kr = _rows(k)
    r, keep = _rotary(q, q_out, cos, sin, B)
    with on_device(q):
        L.check(L.lib().fq_rotate(r, kr.data_ptr(), L.strides(kr, 4), k_out.data_ptr(), L.strides(k_out, 4),
                                  L.dtype_code(q.dtype), B, k.shape[1], S, D, L.stream_handle(q.device)), "rotate")
    return q_out, k_out


def rotate_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                  cache: dict, seen: int, *, page_size: int = 64) -> torch.Tensor:
    """Append the tokens k, v (B, H_kv, S, D) to one layer's cache, the keys rotated, and rotate the queries
    q (B, H_q, S, D) of the same positions.

    ``cos`` / ``sin`` (B or 1, S, R), fp32 or a 16-bit type, as transformers' rotary embedding gives them (both halves
    filled); R below D rotates the first R channels.  ``cache``: the layer's buffers at their full capacity
    (``PagedKVCache.buffers(layer)``), changed in place: K / V codes and V metadata (B, H_kv, capacity, ...), K scale and
    minimum (B, H_kv, pages, D), K_partial / V_partial (B, H_kv, 64, D) in the tokens' type.  ``seen``: the tokens the
    layer holds already; the caller counts on (``PagedKVCache.update_rotated`` does).  Pages that the tokens
    complete are quantised, the rest waits in the partial page; INT8 keeps the rows behind it at zero.
    Returns the rotated queries, contiguous (B, H_q, S, D).

    64-token pages and head_dim 64 or 128; other layouts raise NotImplementedError, before anything is changed.
    """
    host = _host.module() if q.is_cuda and page_size == 64 else None
    if host is not None:
        out = host.rotate_append(q, k, v, cos, sin, cache, seen, *_host.current())
        if out is not None:
            return out
    _check_tokens(q, k, v, cos, sin)
    bits = cache_bits(cache)
    names = _PLANES[bits]
    planes = _layer_planes(cache, bits)
    kp, vp = cache["K_partial"], cache["V_partial"]
    B, H_q, S, D = q.shape
    H_kv = k.shape[1]
    if page_size != 64:
        raise NotImplementedError(f"page_size={page_size}: 64-token pages are taken")
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim={D} not in (64, 128)")
    if H_kv < 1 or H_q % H_kv:
        raise ValueError(f"H_q={H_q} must be divisible by H_kv={H_kv}")
    if kp.shape != (B, H_kv, page_size, D) or vp.shape != kp.shape:
        raise ValueError(f"K_partial / V_partial must be {(B, H_kv, page_size, D)}; got {tuple(kp.shape)} and "
                         f"{tuple(vp.shape)}")
    if kp.dtype != q.dtype or vp.dtype != q.dtype:
        raise AssertionError(f"the partial page must have the tokens' type {q.dtype}; got {kp.dtype}, {vp.dtype}")
    capacity = planes[0].shape[2]
    width = {4: D // 2, 8: D, 3: D // 8}[bits]
    for n, t in zip(names, planes):
        pages = n.startswith("K_scale_raw") or n.startswith("K_mn") or (n == "K_scale" and bits != 3)
        want = (B, H_kv, -(-capacity // page_size) if pages else capacity)
        if t.dim() != 4 or t.shape[:2] != want[:2] or (t.shape[2] < want[2] if pages else t.shape[2] != want[2]):
            raise ValueError(f"{n} must be {want} and its channels; got {tuple(t.shape)}")
        if pages and t.shape[3] != D:
            raise ValueError(f"{n} must have {D} channels; got {tuple(t.shape)}")
        if t.stride(3) != 1 and t.shape[3] > 1:
            raise NotImplementedError(f"{n}: the innermost axis must be contiguous (it is written in place)")
    if planes[0].shape[3] != width or planes[3].shape[3] != width:
        raise ValueError(f"{names[0]} / {names[3]} must have {width} bytes a row; got {tuple(planes[0].shape)} and "
                         f"{tuple(planes[3].shape)}")
    seen = int(seen)
    if seen < 0:
        raise ValueError(f"seen={seen} tokens")
    if seen + S > capacity:
        raise RuntimeError(f"rotate_append: {seen} cached + {S} new tokens exceeds the capacity of {capacity}")
    same_device(q, k, v, cos, sin, *planes, kp, vp)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if S == 0 or B == 0:
        return q_out
    kr, vr = _rows(k), _rows(v)
    if bits == 3:
        _turbo_append(q, q_out, kr, vr, cos, sin, planes, kp, vp, seen, page_size)
        return q_out
    desc, keep = (_ops.int4_cache if bits == 4 else _ops.int8_cache)(*planes, page_size)
    if {t.data_ptr() for t in keep} - {t.data_ptr() for t in planes}:
        raise NotImplementedError("the cache's buffers need 16-byte aligned rows of K metadata and aligned codes")
    r, held = _rotary(q, q_out, cos, sin, B)
    fn = L.lib().fq_int4_cache_append_rotated if bits == 4 else L.lib().fq_int8_cache_append_rotated
    with on_device(q):
        L.check(fn(desc, 0, kp.data_ptr(), L.strides(kp, 5, 1), vp.data_ptr(), L.strides(vp, 5, 1),
                   L.dtype_code(kp.dtype), kr.data_ptr(), L.strides(kr, 4), vr.data_ptr(), L.strides(vr, 4), seen, S, r,
                   L.stream_handle(q.device)), "rotate_append")
    return q_out


def _turbo_append(q, q_out, k, v, cos, sin, planes, kp, vp, seen, page_size):
    """TurboQuant: the rotary rotation first (its row quantiser works on whole rows), then the append."""
    B, _, S, D = q.shape
    desc, keep = _ops.turbo_cache(*planes[:6], planes[6].shape[2], page_size)
    ksr, kmr = planes[6:]
    if {t.data_ptr() for t in keep} - {t.data_ptr() for t in planes}:
        raise NotImplementedError("the cache's planes need contiguous rows")
    r, held = _rotary(q, q_out, cos, sin, B)
    k_rot = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    lib, stream = L.lib(), L.stream_handle(q.device)
    append = (desc, ksr.data_ptr(), L.strides(ksr, 5, 1), kmr.data_ptr(), L.strides(kmr, 5, 1), 0, kp.data_ptr(),
              L.strides(kp, 5, 1), vp.data_ptr(), L.strides(vp, 5, 1), L.dtype_code(kp.dtype), k_rot.data_ptr(),
              L.strides(k_rot, 4), v.data_ptr(), L.strides(v, 4), seen)
    with on_device(q):
        L.check(lib.fq_turbo_cache_append(*append, 0, stream), "rotate_append")     # its checks, nothing appended
        L.check(lib.fq_rotate(r, k.data_ptr(), L.strides(k, 4), k_rot.data_ptr(), L.strides(k_rot, 4),
                              L.dtype_code(q.dtype), B, k.shape[1], S, D, stream), "rotate_append")
        L.check(lib.fq_turbo_cache_append(*append, S, stream), "rotate_append")


def dequantize_cache(cache: dict, length: int, *, start: int = 0, page_size: int = 64):
    """Tokens [start, length) of one layer's INT4 or INT8 cache as bf16 (K, V), (B, H_kv, length - start, D) each.

    ``cache``: the layer's buffers (``PagedKVCache.buffers``) or its views (get_views), holding ``length`` tokens: whole
    64-token pages in the planes, the others in K_partial / V_partial (bf16).  Page tokens are code * scale + min in
    fp32, rounded to bf16 (dequantize_k_int4 / dequantize_v_int4, src/flashquest/kernel/kv_quant.py:174-215,
    dequantize_k / dequantize_v, 64-97), in one launch with the partial page's rows, as
    llama_persistent_patch.py:143-156 puts them together for its eager attention.
    """
    host = _host.module() if page_size == 64 else None
    if host is not None and cache.get("K_partial") is not None and cache["K_partial"].is_cuda:
        res = host.dequantize(cache, length, start, *_host.current())
        if res is not None:
            return res
    bits = cache_bits(cache)
    if bits == 3:
        raise NotImplementedError("dequantize_cache reads INT4 and INT8 caches")
    names = _PLANES[bits]
    planes = _layer_planes(cache, bits)
    kp, vp = cache["K_partial"], cache["V_partial"]
    length, start = int(length), int(start)
    if not 0 <= start <= length:
        raise ValueError(f"start={start} outside the {length} tokens")
    if page_size != 64:
        raise NotImplementedError(f"page_size={page_size}: 64-token pages are taken")
    rest = length % page_size
    done = length - rest
    if kp.dim() != 4 or kp.shape[:2] != planes[0].shape[:2] or vp.shape != kp.shape:
        raise ValueError("cache tensors must be one layer's, (B, H_kv, ...)")
    B, H_kv, _, D = kp.shape
    if done > planes[0].shape[2] or done // page_size > planes[1].shape[2] or rest > kp.shape[2]:
        raise ValueError(f"the cache does not hold {length} tokens: {planes[0].shape[2]} slots, {planes[1].shape[2]} "
                         f"pages, {kp.shape[2]} rows in the partial page")
    if rest and (kp.dtype != torch.bfloat16 or vp.dtype != torch.bfloat16):
        raise NotImplementedError(f"the partial page must be bf16; got {kp.dtype}, {vp.dtype}")
    pages = done // page_size
    views = [t[:, :, :pages] if n in ("K_scale", "K_mn") else t[:, :, :done] for n, t in zip(names, planes)]
    if any(t.shape[:2] != (B, H_kv) for t in views) or any(t.shape[2] != done for t in (views[3], views[4], views[5])) or \
            views[2].shape[2] != pages:
        raise ValueError("the cache's tensors disagree on the batch, the heads or the tokens")
    width = D // 2 if bits == 4 else D
    if views[0].shape[3] != width or views[3].shape[3] != width or views[1].shape[3] != D or views[2].shape[3] != D:
        raise ValueError(f"the planes do not hold head_dim {D}")
    same_device(*planes, kp, vp)
    K = torch.empty(B, H_kv, length - start, D, dtype=torch.bfloat16, device=kp.device)
    V = torch.empty_like(K)
    if K.numel() == 0:
        return K, V
    desc, keep = (_ops.int4_cache if bits == 4 else _ops.int8_cache)(*views, page_size)
    tail, held = None, ()
    if rest:
        held = (_rows(kp[:, :, :rest]), _rows(vp[:, :, :rest]))
        tail = L.Tail(held[0].data_ptr(), L.strides(held[0], 5, 1), held[1].data_ptr(), L.strides(held[1], 5, 1),
                      L.FQ_BF16, rest, D)
    with on_device(kp):
        fn = L.lib().fq_dequant_int4 if bits == 4 else L.lib().fq_dequant_int8
        L.check(fn(desc, tail, start, K.data_ptr(), L.strides(K, 4), V.data_ptr(), L.strides(V, 4),
                   L.stream_handle(kp.device)), "dequantize_cache")
    return K, V
