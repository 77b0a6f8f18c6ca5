"""Attention of a batch whose sequences share a prefix (no reference counterpart).

A cache per sequence, as the reference keeps them, holds a prompt that B sequences share B times, and every step
reads it B times.  Here the prefix is one cache of one sequence, which a step reads once for the whole batch, and the
tokens that each sequence has of its own are a second cache of B sequences.
"""
from __future__ import annotations

import torch

from .. import _host
from .. import _lib as L
from .. import _ops
from ..kernel.rotary import _PLANES, _layer_planes, cache_bits, on_device, same_device


def _check_part(name, views, bits, D):
    """(batch, KV heads, tokens) of a cache layer's views."""
    planes = _layer_planes(views, bits)
    kt, vt = views["K_partial"], views["V_partial"]
    if kt.dim() != 4 or kt.shape != vt.shape:
        raise ValueError(f"{name}: one layer's views (B, H_kv, ...) are attended, K_partial and V_partial alike")
    B, H_kv, S, _ = planes[0].shape
    if kt.shape[:2] != (B, H_kv) or any(t.shape[:2] != (B, H_kv) for t in planes):
        raise ValueError(f"{name}: the cache's tensors disagree on the batch or the heads")
    if S % 64 or kt.shape[2] >= 64:
        raise ValueError(f"{name}: {S} tokens in pages of 64 and {kt.shape[2]} in the partial one: not a layer's views")
    if planes[1].shape[2] < S // 64 or planes[2].shape[2] < S // 64 or any(planes[i].shape[2] != S for i in (3, 4, 5)):
        raise ValueError(f"{name}: the cache's tensors disagree on the tokens")
    width = D // 2 if bits == 4 else D
    if any(planes[i].shape[3] != w for i, w in ((0, width), (1, D), (2, D), (3, width))) or kt.shape[3] != D:
        raise ValueError(f"{name}: the cache does not hold head_dim {D}")
    if kt.shape[2] and (kt.dtype != torch.bfloat16 or vt.dtype != torch.bfloat16):
        raise NotImplementedError(f"{name}: the partial page must be bf16; got {kt.dtype}, {vt.dtype}")
    return B, H_kv, S + kt.shape[2]


def _describe(views, bits, D):
    """The cache and tail descriptors of views, and the tensors they point into."""
    planes = [views[n] for n in _PLANES[bits]]
    planes[0] = _ops._ensure_inner_contiguous(planes[0], 16 if D * bits >= 512 else 8)
    desc, keep = (_ops.int4_cache if bits == 4 else _ops.int8_cache)(*planes, 64)
    kt, vt = views["K_partial"], views["V_partial"]
    if kt.shape[2] == 0:
        return desc, None, keep
    kt, vt = _ops._ensure_inner_contiguous(kt, 8), _ops._ensure_inner_contiguous(vt, 8)
    tail = L.Tail(kt.data_ptr(), L.strides(kt, 5, 1), vt.data_ptr(), L.strides(vt, 5, 1), L.FQ_BF16, kt.shape[2], D)
    return desc, tail, (keep, kt, vt)


def shared_prefix_attention(q: torch.Tensor, prefix: dict, suffix: dict, *, page_size: int = 64,
                            suffix_start: torch.Tensor | None = None, sm_scale: float | None = None,
                            return_lse: bool = False):
    """Attention of B sequences over a prefix that all share and each one's own tokens, for one layer.

    ``q`` (B, H_q, S_q, D), bf16 or fp16, the queries of the sequences' last S_q tokens (1 in a decode step, more when
    drafts are verified or the sequences' prompts go in).  ``prefix``: get_views(layer) of a cache of one sequence;
    ``suffix``: get_views(layer) of a cache of the same family with B sequences, the S_q tokens appended already.  Query
    i of sequence b attends all prefix tokens and the suffix tokens start[b] <= j <= S_suffix - S_q + i, where
    ``suffix_start`` (B,) int32 tells how many of a sequence's suffix tokens are left padding (None: none; read on the
    device, values outside 0 .. S_suffix count as the nearest).  A query with padding alone attends the prefix.

    Positions: the suffix's first token follows the prefix's last; the caches hold keys that are rotated already
    (PagedKVCache.update_rotated).  A value that is not finite reaches only the queries that attend it, whose outputs
    are then not finite; in a key it reaches all that attend its page, as the page's scales do.  INT4 and INT8 caches
    with 64-token pages and head_dim 64 or 128, at most 2^21 query rows (B H_q S_q).
    Returns O (B, H_q, S_q, D) in q's type, with return_lse also the natural-log sum of exponentials (B, H_q, S_q)
    fp32.
    """
    host = _host.module() if q.is_cuda and page_size == 64 else None
    if host is not None:
        res = host.shared_prefix(q, prefix, suffix, suffix_start, sm_scale, bool(return_lse), *_host.current())
        if res is not None:
            return res
    if q.dim() != 4:
        raise ValueError(f"q must be (B, H_q, S_q, D); got {tuple(q.shape)}")
    B, H_q, S_q, D = q.shape
    bits = cache_bits(prefix)
    if cache_bits(suffix) != bits:
        raise ValueError("prefix and suffix must be caches of one family")
    if bits == 3:
        raise NotImplementedError("shared_prefix_attention attends INT4 and INT8 caches")
    if page_size != 64:
        raise NotImplementedError(f"page_size={page_size}: 64-token pages are taken")
    if D not in (64, 128):
        raise NotImplementedError(f"head_dim={D} not in (64, 128)")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"q must be bf16 or fp16; got {q.dtype}")
    Bp, H_kv, n_prefix = _check_part("prefix", prefix, bits, D)
    Bs, H_s, n_suffix = _check_part("suffix", suffix, bits, D)
    if Bp != 1:
        raise ValueError(f"the prefix is one sequence; got a batch of {Bp}")
    if Bs != B or H_s != H_kv:
        raise ValueError(f"q has {B} sequences, the suffix {Bs}; the prefix has {H_kv} KV heads, the suffix {H_s}")
    if H_kv < 1 or H_q < 1 or H_q % H_kv:
        raise ValueError(f"H_q={H_q} must be divisible by H_kv={H_kv}")
    if n_prefix < 1:
        raise ValueError("the prefix has no tokens")
    if S_q < 1 or n_suffix < S_q:
        raise ValueError(f"S_q={S_q} query tokens, the suffix has {n_suffix} (they are its last)")
    if sm_scale is not None and not float(sm_scale) > 0.0:
        raise ValueError(f"sm_scale must be positive; got {sm_scale}")
    if suffix_start is not None:
        if suffix_start.shape != (B,) or suffix_start.dtype != torch.int32:
            raise ValueError(f"suffix_start must be ({B},) int32; got {tuple(suffix_start.shape)} {suffix_start.dtype}")
        suffix_start = suffix_start.contiguous()
    same_device(q, *(views[n] for views in (prefix, suffix) for n in _PLANES[bits] + ("K_partial", "V_partial")),
                *(() if suffix_start is None else (suffix_start,)))
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=q.device) if return_lse else None
    if B == 0:
        return (out, lse) if return_lse else out
    qr = _ops._ensure_inner_contiguous(q, 8)
    pd, pt, keep_p = _describe(prefix, bits, D)
    sd, st, keep_s = _describe(suffix, bits, D)
    query = L.SharedQuery(qr.data_ptr(), L.strides(qr, 4), out.data_ptr(), L.strides(out, 4), L.ptr(lse),
                          L.strides(lse, 3) if return_lse else L.I64x3(0, 0, 0), L.ptr(suffix_start),
                          L.dtype_code(q.dtype), B, H_q, S_q, 0.0 if sm_scale is None else float(sm_scale))
    lib = L.lib()
    with on_device(q):
        nbytes = lib.fq_shared_prefix_workspace_bytes(pd, pt, sd, st, query, bits)
        # a workspace of this call: captured graphs that run at the same time share none
        ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=q.device)
        fn = lib.fq_shared_prefix_int4 if bits == 4 else lib.fq_shared_prefix_int8
        L.check(fn(pd, pt, sd, st, query, ws.data_ptr(), nbytes, L.stream_handle(q.device)), "shared_prefix_attention")
    return (out, lse) if return_lse else out
