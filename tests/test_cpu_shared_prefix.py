"""What shared_prefix_attention and its C entries refuse (host checks, no launch)."""
import ctypes

import pytest
import torch

from flashquest_amd import _lib as L
from flashquest_amd.cache import PersistentInt4KVCache, PersistentInt8KVCache, PersistentTurboKVCache
from flashquest_amd.eager import shared_prefix_attention


def views(cls, B, n, H=2, D=128, **kw):
    c = cls(batch_size=B, num_layers=1, num_kv_heads=H, head_dim=D, max_seq_len=256, device="cpu", **kw)
    c._seen_tokens[0] = n
    return c.get_views(0)


def call(bits=4, n_prefix=70, n_suffix=66, B=3, Hq=4, Sq=1, D=128, dtype=torch.bfloat16, **kw):
    cls = PersistentInt4KVCache if bits == 4 else PersistentInt8KVCache
    a = dict(q=torch.zeros(B, Hq, Sq, D, dtype=dtype), prefix=views(cls, 1, n_prefix, D=D), suffix=views(cls, B, n_suffix, D=D))
    a.update(kw)
    return shared_prefix_attention(**a)


INT4, INT8, TURBO = PersistentInt4KVCache, PersistentInt8KVCache, PersistentTurboKVCache


@pytest.mark.parametrize("error,kw", [
    (ValueError, dict(q=torch.zeros(3, 4, 128, dtype=torch.bfloat16))),
    (ValueError, dict(q=torch.zeros(2, 4, 1, 128, dtype=torch.bfloat16))),              # 2 of 3 sequences
    (ValueError, dict(Hq=3)),
    (NotImplementedError, dict(dtype=torch.float32)),
    (NotImplementedError, dict(D=32)),
    (NotImplementedError, dict(page_size=32)),
    (ValueError, dict(prefix=views(INT8, 1, 70))),                                      # two families
    (NotImplementedError, dict(prefix=views(TURBO, 1, 70), suffix=views(TURBO, 3, 66))),
    (ValueError, dict(prefix=views(INT4, 2, 70))),                                      # a prefix of two sequences
    (ValueError, dict(prefix=views(INT4, 1, 70, H=4))),
    (ValueError, dict(prefix=views(INT4, 1, 70, D=64))),
    (ValueError, dict(n_prefix=0)),
    (ValueError, dict(n_suffix=0)),
    (ValueError, dict(Sq=5, n_suffix=4)),
    (ValueError, dict(Sq=0)),
    (ValueError, dict(sm_scale=0.0)),
    (ValueError, dict(sm_scale=-1.0)),
    (ValueError, dict(sm_scale=float("nan"))),
    (ValueError, dict(suffix_start=torch.zeros(3, dtype=torch.int64))),
    (ValueError, dict(suffix_start=torch.zeros(2, dtype=torch.int32))),
    (ValueError, dict(prefix=dict(views(INT4, 1, 70), V_mn=views(INT4, 1, 10)["V_mn"]))),
    (ValueError, dict(prefix=dict(views(INT4, 1, 70), K_mn=views(INT4, 1, 10)["K_mn"]))),
    (ValueError, dict(prefix=dict(views(INT4, 1, 70), V_partial=views(INT4, 1, 68)["V_partial"]))),
    (ValueError, dict(prefix=dict(views(INT4, 1, 70), V_mn=views(INT4, 1, 70, v_group=32)["V_mn"]))),
    (ValueError, dict(prefix={n: t for n, t in views(INT4, 1, 70).items() if n != "K_scale"})),
    (NotImplementedError, dict(prefix=dict(views(INT4, 1, 70), K_partial=torch.zeros(1, 2, 6, 128),
                                           V_partial=torch.zeros(1, 2, 6, 128)))),
    (AssertionError, dict()),                                                           # nothing wrong but the device
])
def test_refusals(error, kw):
    with pytest.raises(error):
        call(**kw)


AT = 1 << 20


def c_cache(B, S, D=128, bits=4):
    c = L.Int4Cache()
    for n in ("k_packed", "v_packed", "k_scale", "k_mn", "v_scale", "v_mn"):
        setattr(c, n, AT)
    w = D * bits // 8
    c.k_strides = c.v_strides = L.I64x5(0, 2 * S * w, S * w, w, 1)
    c.ks_strides = c.km_strides = L.I64x5(0, S // 64 * 2 * D, S // 64 * D, D, 1)
    c.vs_strides = c.vm_strides = L.I64x5(0, 2 * S, S, 1, 1)
    c.L, c.B, c.H_kv, c.S, c.P, c.D, c.page_size, c.v_groups = 1, B, 2, S, max(1, S // 64), D, 64, 1
    return c


def c_tail(n, D=128):
    row = L.I64x5(0, 2 * 64 * D, 64 * D, D, 1)
    return L.Tail(AT, row, AT, row, L.FQ_BF16, n, D)


def c_query(B=3, Hq=4, Sq=1, D=128):
    st = L.I64x4(Hq * Sq * D, Sq * D, D, 1)
    return L.SharedQuery(AT, st, AT, st, None, L.I64x3(0, 0, 0), None, L.FQ_BF16, B, Hq, Sq, 0.0)


def changed(x, **kw):
    for n, v in kw.items():
        setattr(x, n, v)
    return x


@pytest.mark.parametrize("status,make", [
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (None, pt, s, st, q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, pt, s, st, None)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (changed(p, B=2), pt, s, st, q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, pt, changed(s, B=2), st, q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (changed(p, L=2), pt, s, st, q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (changed(p, S=65), pt, s, st, q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (changed(p, P=1), pt, s, st, q)),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (changed(p, page_size=32), pt, s, st, q)),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (changed(p, k_packed=AT + 8), pt, s, st, q)),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (changed(p, k_strides=L.I64x5(0, 1 << 20, 1 << 12, 72, 1)), pt, s, st, q)),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (changed(p, v_scale=AT + 1), pt, s, st, q)),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (p, pt, changed(s, meta_dtype=L.FQ_F16), st, q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, changed(pt, len=64), s, st, q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, changed(pt, len=-1), s, st, q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, changed(pt, D=64), s, st, q)),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (p, changed(pt, dtype=L.FQ_F16), s, st, q)),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (p, pt, s, changed(st, k=AT + 8), q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, pt, s, changed(st, v=None), q)),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, H_q=5))),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, S_q=0))),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, S_q=200))),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, H_q=1 << 24))),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, H_q=(1 << 21) // 3 + 2))),     # 2^21 rows at most
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, dtype=L.FQ_F32))),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, q=AT + 8))),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, o_strides=L.I64x4(512, 128, 130, 1)))),
    (L.FQ_ERR_UNSUPPORTED, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, o_strides=L.I64x4(512, 128, 128, 2)))),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, out=None))),
    (L.FQ_ERR_INVALID, lambda p, pt, s, st, q: (p, pt, s, st, changed(q, start=AT + 2))),
    (L.FQ_ERR_WORKSPACE, lambda p, pt, s, st, q: (p, pt, s, st, q)),
])
def test_c_checks(status, make):
    args = make(c_cache(1, 128), c_tail(6), c_cache(3, 64), c_tail(2), c_query())
    ref = [None if x is None else ctypes.byref(x) for x in args]
    assert L.lib().fq_shared_prefix_int4(*ref, AT, 0, None) == status
    if status != L.FQ_ERR_WORKSPACE and args[4] is not None and args[4].q == AT and args[4].out and not args[4].start \
            and args[4].o_strides[3] == 1 and args[4].o_strides[2] == 128:
        assert L.lib().fq_shared_prefix_workspace_bytes(*ref, 4) == 0
    assert L.lib().fq_shared_prefix_workspace_bytes(*ref, 3) == 0


def test_workspace_bytes_are_host_arithmetic():
    """Partial outputs, maxima and sums of every split: at least one of the prefix and one of the suffix per row."""
    q = c_query()
    n = L.lib().fq_shared_prefix_workspace_bytes(c_cache(1, 128), c_tail(6), c_cache(3, 64), c_tail(2), q, 4)
    assert n >= 2 * 3 * 4 * (128 + 2) * 4 and n % 8 == 0
    assert L.lib().fq_shared_prefix_int4(c_cache(1, 128), c_tail(6), c_cache(3, 64), c_tail(2), q, AT, n - 1, None) == \
        L.FQ_ERR_WORKSPACE
    assert L.lib().fq_shared_prefix_int4(c_cache(1, 128), c_tail(6), c_cache(3, 64), c_tail(2), q, AT + 4, n, None) == \
        L.FQ_ERR_INVALID
