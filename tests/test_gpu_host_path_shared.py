"""The native host path of rotate_append, dequantize_cache and shared_prefix_attention: plain calls go through it and
give the general way's results; calls it is not for do not."""
import pytest
import torch

from flashquest_amd import _host
from flashquest_amd.cache import PersistentInt4KVCache, PersistentInt8KVCache
from flashquest_amd.eager import shared_prefix_attention
from flashquest_amd.kernel import dequantize_cache, rotate_append

pytestmark = pytest.mark.gpu

DEV = "cuda"
CLASSES = {4: PersistentInt4KVCache, 8: PersistentInt8KVCache}


class Watched:
    """The module with its calls' answers kept: True where a call was taken."""

    def __init__(self, inner):
        self.inner, self.taken = inner, []

    def __getattr__(self, name):
        def call(*args):
            out = getattr(self.inner, name)(*args)
            self.taken.append(out is not None)
            return out
        return call


@pytest.fixture
def native(monkeypatch):
    inner = _host.module()
    assert inner is not None
    w = Watched(inner)
    monkeypatch.setattr(_host, "module", lambda: w)
    return w


def general(monkeypatch, f):
    with monkeypatch.context() as m:
        m.setattr(_host, "module", lambda: None)
        return f()


def cache(bits, B, n, gen, H=2, D=128, **kw):
    c = CLASSES[bits](batch_size=B, num_layers=2, num_kv_heads=H, head_dim=D, max_seq_len=320, device=DEV, **kw)
    k, v = (torch.randn(B, H, n, D, device=DEV, generator=gen).to(torch.bfloat16) for _ in range(2))
    if n:
        c.update_quantized(k, v, 1)
    return c


FORMS = [(4, 128, {}), (4, 128, dict(meta_dtype=torch.float16, v_group=32)), (4, 64, dict(v_group=32)), (8, 128, {}), (8, 64, {})]


@pytest.mark.parametrize("bits,D,kw", FORMS)
@pytest.mark.parametrize("seen,n", [(0, 1), (40, 3), (63, 1), (60, 200)])
def test_rotate_append(native, monkeypatch, bits, D, kw, seen, n):
    gen = torch.Generator(device=DEV).manual_seed(seen + n)
    q, k, v = (torch.randn(2, n, h, D, device=DEV, generator=gen).to(torch.bfloat16).transpose(1, 2) for h in (4, 2, 2))
    cos, sin = (torch.randn(b, n, D, device=DEV, generator=gen) for b in (1, 1))
    for c in (cos, cos.to(torch.bfloat16), cos.expand(2, -1, -1).contiguous()):
        s = sin.expand_as(c).to(c.dtype).contiguous()
        a, b = cache(bits, 2, seen, torch.Generator(device=DEV).manual_seed(1), D=D, **kw), None
        got = rotate_append(q, k, v, c, s, a.buffers(1), seen)
        b = cache(bits, 2, seen, torch.Generator(device=DEV).manual_seed(1), D=D, **kw)
        want = general(monkeypatch, lambda: rotate_append(q, k, v, c, s, b.buffers(1), seen))
        assert torch.equal(got, want)
        for name, t in a.buffers(1).items():
            assert torch.equal(t, b.buffers(1)[name]), name
    assert native.taken == [True] * 3


@pytest.mark.parametrize("bits,D,kw", FORMS)
@pytest.mark.parametrize("length,start", [(5, 0), (64, 1), (300, 70)])
def test_dequantize_cache(native, monkeypatch, bits, D, kw, length, start):
    c = cache(bits, 2, length, torch.Generator(device=DEV).manual_seed(2), D=D, **kw)
    for src in (c.buffers(1), c.get_views(1)):
        got = dequantize_cache(src, length, start=start)
        want = general(monkeypatch, lambda: dequantize_cache(src, length, start=start))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert native.taken == [True] * 2


@pytest.mark.parametrize("bits,D,kw", FORMS)
@pytest.mark.parametrize("prefix,suffix,n", [(5, 3, 1), (64, 64, 2), (130, 70, 70)])
def test_shared_prefix(native, monkeypatch, bits, D, kw, prefix, suffix, n):
    gen = torch.Generator(device=DEV).manual_seed(3)
    p, s = cache(bits, 1, prefix, gen, D=D, **kw).get_views(1), cache(bits, 3, suffix, gen, D=D, **kw).get_views(1)
    q = torch.randn(3, n, 6, D, device=DEV, generator=gen).to(torch.float16).transpose(1, 2)
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    for args in (dict(), dict(suffix_start=start, sm_scale=0.2), dict(return_lse=True)):
        got = shared_prefix_attention(q, p, s, **args)
        want = general(monkeypatch, lambda: shared_prefix_attention(q, p, s, **args))
        for x, y in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(x, y)
    assert native.taken == [True] * 3


def test_calls_it_is_not_for(native):
    gen = torch.Generator(device=DEV).manual_seed(4)
    c = cache(4, 2, 70, gen)
    q, k = (torch.zeros(2, h, 1, 128, dtype=torch.bfloat16, device=DEV) for h in (4, 2))
    a = torch.zeros(1, 1, 128, device=DEV)
    buf = c.buffers(1)
    with pytest.raises(RuntimeError):
        rotate_append(q, k, k, a, a, buf, 320)
    with pytest.raises(ValueError):
        rotate_append(q, k, k, a, a, buf, -1)
    with pytest.raises(ValueError):
        rotate_append(q[:1], k, k, a, a, buf, 70)
    with pytest.raises(ValueError):
        rotate_append(q, k, k, a, a, dict(buf, V_mn=buf["V_mn"][:, :, :64]), 70)
    with pytest.raises(ValueError):
        dequantize_cache(buf, 400)
    with pytest.raises(ValueError):
        dequantize_cache(buf, 70, start=71)
    with pytest.raises(ValueError):
        shared_prefix_attention(q, c.get_views(1), c.get_views(1))
    with pytest.raises(ValueError):
        shared_prefix_attention(q, cache(4, 1, 70, gen).get_views(1), c.get_views(0))
    with pytest.raises(ValueError):
        shared_prefix_attention(q, cache(4, 1, 70, gen).get_views(1), c.get_views(1), sm_scale=-1.0)
    rotate_append(q, k, k, a.half(), a.half(), buf, 70)                # angles of a third type: converted
    off = torch.zeros(q.numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view(q.shape)
    rotate_append(off, k, k, a, a, buf, 70)                            # copied to aligned rows
    assert native.taken == [False] * len(native.taken) and len(native.taken) == 11
