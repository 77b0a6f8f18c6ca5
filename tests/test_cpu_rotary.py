"""What rotate_append, rotate, dequantize_cache and their C entries refuse (host checks, no launch)."""
import ctypes

import pytest
import torch

from flashquest_amd import _lib as L
from flashquest_amd.cache import PersistentInt4KVCache, PersistentTurboKVCache
from flashquest_amd.kernel import dequantize_cache, rotate, rotate_append


def parts(B=2, H_q=4, H=2, S=3, D=128, room=128, dtype=torch.bfloat16, **kw):
    c = PersistentInt4KVCache(batch_size=B, num_layers=1, num_kv_heads=H, head_dim=D, max_seq_len=room, device="cpu", **kw)
    q, k = torch.zeros(B, H_q, S, D, dtype=dtype), torch.zeros(B, H, S, D, dtype=dtype)
    return dict(q=q, k=k, v=k, cos=torch.zeros(1, S, D), sin=torch.zeros(1, S, D), cache=c.buffers(0), seen=0)


def without(d, *names):
    return {n: t for n, t in d.items() if n not in names}


REFUSED = [
    (ValueError, lambda a: dict(k=a["k"][:1])),                               # another batch
    (ValueError, lambda a: dict(v=a["v"][:, :, :2])),                         # k and v differ
    (ValueError, lambda a: dict(q=a["q"][:, :, :2])),                         # q and k differ in tokens
    (ValueError, lambda a: dict(q=a["q"][:, :3])),                            # 3 query heads on 2 KV heads
    (ValueError, lambda a: dict(q=a["q"][0])),
    (AssertionError, lambda a: dict(q=a["q"].half())),                        # types differ
    (NotImplementedError, lambda a: dict(q=a["q"].float(), k=a["k"].float(), v=a["v"].float())),
    (ValueError, lambda a: dict(cos=a["cos"].half())),                        # cos and sin differ
    (ValueError, lambda a: dict(cos=a["cos"][0], sin=a["sin"][0])),           # no batch axis
    (ValueError, lambda a: dict(cos=a["cos"].expand(3, -1, -1), sin=a["sin"].expand(3, -1, -1))),
    (ValueError, lambda a: dict(cos=a["cos"][:, :2], sin=a["sin"][:, :2])),   # positions for 2 of 3 tokens
    (NotImplementedError, lambda a: dict(cos=a["cos"][..., :40], sin=a["sin"][..., :40])),
    (NotImplementedError, lambda a: dict(cos=torch.zeros(1, 3, 144), sin=torch.zeros(1, 3, 144))),
    (NotImplementedError, lambda a: dict(cos=a["cos"].double(), sin=a["sin"].double())),
    (NotImplementedError, lambda a: dict(page_size=32)),
    (ValueError, lambda a: dict(seen=-1)),
    (RuntimeError, lambda a: dict(seen=126)),                                 # 126 + 3 tokens in 128
    (ValueError, lambda a: dict(cache=without(a["cache"], "K_mn"))),
    (ValueError, lambda a: dict(cache=dict(a["cache"], K_partial=a["cache"]["K_partial"][:, :, :3]))),
    (ValueError, lambda a: dict(cache=dict(a["cache"], K_scale=a["cache"]["K_scale"][:, :, :1]))),
    (ValueError, lambda a: dict(cache=dict(a["cache"], K_scale=a["cache"]["K_scale"][..., :64]))),
    (ValueError, lambda a: dict(cache=dict(a["cache"], V_scale=a["cache"]["V_scale"][:, :1]))),
    (ValueError, lambda a: dict(cache=dict(a["cache"], V_packed=a["cache"]["V_packed"][..., :32]))),
    (AssertionError, lambda a: dict(cache=dict(a["cache"], V_partial=a["cache"]["V_partial"].half()))),
    (AssertionError, lambda a: {}),                                           # nothing wrong but the device
]


@pytest.mark.parametrize("i", range(len(REFUSED)))
def test_rotate_append_refuses(i):
    error, change = REFUSED[i]
    a = parts()
    a.update(change(a))
    with pytest.raises(error):
        rotate_append(**a)


def test_head_dim_and_turbo_refusals():
    a = parts(D=32)
    with pytest.raises(NotImplementedError):
        rotate_append(**a)
    with pytest.raises(NotImplementedError):
        rotate(a["q"], a["k"], a["cos"], a["sin"])
    t = PersistentTurboKVCache(batch_size=1, num_layers=1, num_kv_heads=1, head_dim=64, max_seq_len=64, device="cpu")
    with pytest.raises(NotImplementedError):
        dequantize_cache(t.buffers(0), 3)


def test_update_rotated_checks_the_layer_and_the_room_first():
    c = PersistentInt4KVCache(batch_size=1, num_layers=1, num_kv_heads=2, head_dim=64, max_seq_len=64, device="cpu")
    x = torch.zeros(1, 2, 65, 64, dtype=torch.bfloat16)
    a = torch.zeros(1, 65, 64)
    with pytest.raises(IndexError):
        c.update_rotated(x, x, x, a, a, 1)
    with pytest.raises(RuntimeError):
        c.update_rotated(x, x, x, a, a, 0)
    with pytest.raises(IndexError):
        c.buffers(-1)


@pytest.mark.parametrize("error,change,length,kw", [
    (ValueError, {}, 10, dict(start=11)),
    (ValueError, {}, 10, dict(start=-1)),
    (ValueError, {}, 200, {}),                            # more than the planes hold
    (NotImplementedError, {}, 10, dict(page_size=16)),
    (ValueError, dict(K_partial=lambda t: t[:, :, :5]), 10, {}),
    (ValueError, dict(K_scale=lambda t: t[:, :, :1]), 128, {}),
    (ValueError, dict(V_mn=lambda t: t[:, :, :64]), 128, {}),
    (ValueError, dict(V_packed=lambda t: t[..., :32]), 128, {}),
    (NotImplementedError, dict(K_partial=lambda t: t.half(), V_partial=lambda t: t.half()), 10, {}),
    (AssertionError, {}, 10, {}),                         # nothing wrong but the device
])
def test_dequantize_cache_refuses(error, change, length, kw):
    cache = parts()["cache"]
    cache.update({n: f(cache[n]) for n, f in change.items()})
    with pytest.raises(error):
        dequantize_cache(cache, length, **kw)


def _c_append(**kw):
    """fq_int4_cache_append_rotated on made-up addresses, 2 x 2 heads x 128 channels, 3 new tokens behind 10."""
    at = 1 << 20
    c = L.Int4Cache()
    for n in ("k_packed", "v_packed", "k_scale", "k_mn", "v_scale", "v_mn"):
        setattr(c, n, at)
    c.k_strides = c.v_strides = L.I64x5(0, 2 * 128 * 64, 128 * 64, 64, 1)
    c.ks_strides = c.km_strides = L.I64x5(0, 2 * 2 * 128, 2 * 128, 128, 1)
    c.vs_strides = c.vm_strides = L.I64x5(0, 2 * 128, 128, 1, 1)
    c.L, c.B, c.H_kv, c.S, c.P, c.D, c.page_size, c.v_groups = 1, 2, 2, 128, 2, 128, 64, 1
    for n in ("c_S", "c_D", "c_page_size"):
        if n in kw:
            setattr(c, n[2:], kw.pop(n))
    part, new = L.I64x5(0, 2 * 64 * 128, 64 * 128, 128, 1), L.I64x4(2 * 3 * 128, 3 * 128, 128, 1)
    r = L.Rotary(at, L.I64x3(0, 128, 1), at, L.I64x3(0, 128, 1), L.FQ_F32, 128, at, new, at, new, 4)
    none = kw.pop("no_rotary", False)
    for n in ("R", "dtype", "cos", "q", "cos_strides", "q_strides", "H_q"):
        if n in kw:
            setattr(r, n, kw.pop(n))
    args = dict(seen=10, S_new=3, k_new=at)
    args.update(kw)
    return L.lib().fq_int4_cache_append_rotated(c, 0, at, part, at, part, L.FQ_BF16, args["k_new"], new, at, new,
                                                args["seen"], args["S_new"], None if none else ctypes.byref(r), None)


@pytest.mark.parametrize("status,kw", [
    (L.FQ_ERR_INVALID, dict(no_rotary=True)),
    (L.FQ_ERR_UNSUPPORTED, dict(R=24)),
    (L.FQ_ERR_UNSUPPORTED, dict(R=0)),
    (L.FQ_ERR_UNSUPPORTED, dict(R=144)),
    (L.FQ_ERR_UNSUPPORTED, dict(dtype=L.FQ_F16)),                             # angles of a third type
    (L.FQ_ERR_INVALID, dict(cos=None)),
    (L.FQ_ERR_UNSUPPORTED, dict(cos=(1 << 20) + 4)),
    (L.FQ_ERR_UNSUPPORTED, dict(cos_strides=L.I64x3(0, 130, 1))),
    (L.FQ_ERR_UNSUPPORTED, dict(q_strides=L.I64x4(1536, 384, 128, 2))),
    (L.FQ_ERR_INVALID, dict(q=None)),
    (L.FQ_ERR_INVALID, dict(H_q=-1)),
    (L.FQ_ERR_INVALID, dict(k_new=None)),
    (L.FQ_ERR_INVALID, dict(seen=126)),
    (L.FQ_ERR_INVALID, dict(seen=-1)),
    (L.FQ_ERR_UNSUPPORTED, dict(c_page_size=32)),
    (L.FQ_ERR_UNSUPPORTED, dict(c_D=96)),
    (L.FQ_OK, dict(S_new=0)),
])
def test_c_append_rotated_checks(status, kw):
    assert _c_append(**kw) == status


def test_c_dequant_checks():
    lib, at = L.lib(), 1 << 20
    c = L.Int4Cache()
    c.L, c.B, c.H_kv, c.S, c.P, c.D, c.page_size, c.v_groups = 1, 1, 1, 0, 0, 128, 64, 1
    st = L.I64x4(64 * 128, 64 * 128, 128, 1)
    row = L.I64x5(0, 64 * 128, 64 * 128, 128, 1)
    tail = L.Tail(at, row, at, row, L.FQ_BF16, 5, 128)
    call = lambda t, start, k=at, s=st: lib.fq_dequant_int4(c, t, start, k, s, at, st, None)  # noqa: E731
    assert call(tail, 6) == L.FQ_ERR_INVALID                  # past the tokens
    assert call(tail, -1) == L.FQ_ERR_INVALID
    assert call(tail, 5) == L.FQ_OK                           # nothing to read
    assert call(None, 0) == L.FQ_OK
    assert call(tail, 0, k=None) == L.FQ_ERR_INVALID
    assert call(tail, 0, s=L.I64x4(8192, 8192, 129, 1)) == L.FQ_ERR_UNSUPPORTED
    for change in (dict(len=64), dict(D=64), dict(dtype=L.FQ_F16)):
        t = L.Tail(at, row, at, row, L.FQ_BF16, 5, 128)
        for n, x in change.items():
            setattr(t, n, x)
        assert call(t, 0) in (L.FQ_ERR_INVALID, L.FQ_ERR_UNSUPPORTED)
    c.S, c.P = 65, 2
    assert call(tail, 0) == L.FQ_ERR_INVALID                  # NULL planes
