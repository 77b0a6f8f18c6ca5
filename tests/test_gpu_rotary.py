"""Appending rotated tokens (update_rotated, rotate_append) and reading a cache back (dequantize_cache).

The cache's contents are compared bit for bit with update_quantized of keys that were rotated by elementary fp32
operations: same products, same sums, same roundings.  The queries are also compared with the rotation in 64 bits:
two products and a sum of fp32 values lose at most 3 half steps of the largest product, the result one half step of
its 16-bit type.
"""
import pytest
import torch

from flashquest_amd.cache import PersistentInt4KVCache, PersistentInt8KVCache, PersistentTurboKVCache
from flashquest_amd.eager import prefill_attention_layer, sparse_decode_layer
from flashquest_amd.kernel import (dequantize_cache, dequantize_k, dequantize_k_int4, dequantize_v, dequantize_v_int4,
                                   rotate, rotate_append)

pytestmark = pytest.mark.gpu

DEV = "cuda"
CLASSES = {4: PersistentInt4KVCache, 8: PersistentInt8KVCache, 3: PersistentTurboKVCache}


def make_cache(bits, B=2, layers=2, H=2, D=128, room=320, **kw):
    return CLASSES[bits](batch_size=B, num_layers=layers, num_kv_heads=H, head_dim=D, max_seq_len=room, device=DEV, **kw)


def angles(B, pos, R, dtype, gen):
    """(B, len(pos), R) cos / sin of positions pos (+ an offset of its own for every row of the batch)."""
    at = pos[None].double() + torch.randint(0, 1000, (B, 1), device=DEV, generator=gen)
    turn = 10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
    a = (at[..., None] * turn).repeat(1, 1, 2)
    return a.cos().to(dtype), a.sin().to(dtype)


def turned(x, cos, sin):
    """fp32, every product and sum rounded by itself, once more to x's type."""
    h = cos.shape[-1] // 2
    c, s = cos.float()[:, None], sin.float()[:, None]
    a, b = x[..., :h].float(), x[..., h:2 * h].float()
    lo = a * c[..., :h] - b * s[..., :h]
    hi = b * c[..., h:] + a * s[..., h:]
    return torch.cat((lo, hi, x[..., 2 * h:].float()), -1).to(x.dtype)


def tokens(gen, B, H, S, D, dtype=torch.bfloat16, heads_first=False):
    x = torch.randn((B, H, S, D) if heads_first else (B, S, H, D), device=DEV, generator=gen).to(dtype)
    return x if heads_first else x.transpose(1, 2)


def same_buffers(a, b, layer):
    x, y = a.buffers(layer), b.buffers(layer)
    for n in x:
        assert torch.equal(x[n].view(torch.uint8) if x[n].dtype == torch.uint8 else x[n].view(torch.int16),
                           y[n].view(torch.uint8) if y[n].dtype == torch.uint8 else y[n].view(torch.int16)), n


# steps: the token counts of consecutive appends; pages end inside, at the end of and before a step
STEPS = ([1], [63], [64], [65], [5, 1, 57, 1, 1], [40, 40, 200], [63, 2, 63, 64], [128, 130])


@pytest.mark.parametrize("bits,D,R,H_q,angle,kw", [
    (4, 128, 128, 6, torch.bfloat16, {}),
    (4, 128, 64, 2, torch.float32, dict(meta_dtype=torch.float16, v_group=32)),
    (4, 64, 64, 14, torch.float32, {}),
    (8, 128, 128, 8, torch.float32, {}),
    (8, 64, 32, 2, torch.bfloat16, dict(meta_dtype=torch.float16)),
    (8, 128, 16, 2, torch.float16, {}),
    (3, 128, 128, 6, torch.bfloat16, {}),
    (3, 64, 48, 2, torch.float32, {}),
])
@pytest.mark.parametrize("steps", STEPS, ids=str)
def test_update_rotated_is_rotation_then_update_quantized(bits, D, R, H_q, angle, kw, steps):
    gen = torch.Generator(device=DEV).manual_seed(sum(steps) + D + R + bits)
    got, want = make_cache(bits, D=D, **kw), make_cache(bits, D=D, **kw)
    layer, seen = 1, 0
    for i, n in enumerate(steps):
        q = tokens(gen, 2, H_q, n, D, heads_first=i % 2 == 1)
        k, v = (tokens(gen, 2, 2, n, D, heads_first=i % 2 == 1) for _ in range(2))
        cos, sin = angles(2, seen + torch.arange(n, device=DEV), R, angle, gen)
        if i % 2:                # positions that the batch shares
            cos, sin = cos[:1], sin[:1]
        out = got.update_rotated(q, k, v, cos, sin, layer)
        want.update_quantized(turned(k, cos, sin), v, layer)
        assert out.shape == q.shape and out.is_contiguous()
        assert torch.equal(out, turned(q, cos, sin))
        seen += n
        assert got.get_seq_length(layer) == want.get_seq_length(layer) == seen
        same_buffers(got, want, layer)
    same_buffers(got, want, 0)           # the other layer is untouched


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("S", [1, 7, 1025])
def test_queries_against_64_bits(dtype, S):
    gen = torch.Generator(device=DEV).manual_seed(S)
    q, k = tokens(gen, 3, 5, S, 128, dtype), tokens(gen, 3, 1, S, 128, dtype)
    cos, sin = angles(3, torch.arange(S, device=DEV), 96, torch.float32, gen)
    gq, gk = rotate(q, k, cos, sin)
    for x, y in ((q, gq), (k, gk)):
        c, s, xd = cos.double()[:, None], sin.double()[:, None], x.double()
        part = torch.cat((-xd[..., 48:96], xd[..., :48]), -1)
        ref = torch.cat((xd[..., :96] * c + part * s, xd[..., 96:]), -1)
        size = torch.cat((xd[..., :96].abs() * c.abs() + part.abs() * s.abs(), xd[..., 96:].abs()), -1)
        tol = ref.abs() * (torch.finfo(dtype).eps / 2) * 1.001 + 3 * 2.0 ** -24 * size + torch.finfo(dtype).tiny * 2.0 ** -8
        assert bool(((y.double() - ref).abs() <= tol).all())


def test_many_heads_per_thread_and_rows_that_are_copied():
    """A step large enough that a thread rotates several heads; q, k and v that are not 16-byte aligned."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    S = 4200
    base = torch.randn(1, S, 26 * 128 + 1, device=DEV, generator=gen).to(torch.bfloat16)
    q = base[..., 1:22 * 128 + 1].view(1, S, 22, 128).transpose(1, 2)
    k = base[..., 22 * 128 + 1:24 * 128 + 1].view(1, S, 2, 128).transpose(1, 2)
    v = base[..., 24 * 128 + 1:].view(1, S, 2, 128).transpose(1, 2)
    cos, sin = angles(1, torch.arange(S, device=DEV), 128, torch.float32, gen)
    got, want = make_cache(8, B=1, layers=1, room=4224), make_cache(8, B=1, layers=1, room=4224)
    assert torch.equal(got.update_rotated(q, k, v, cos, sin, 0), turned(q, cos, sin))
    want.update_quantized(turned(k, cos, sin), v, 0)
    same_buffers(got, want, 0)


@pytest.mark.parametrize("bits", [4, 8])
def test_nan_and_infinities_stay_in_their_rows(bits):
    gen = torch.Generator(device=DEV).manual_seed(9)
    q, k, v = tokens(gen, 1, 2, 3, 128), tokens(gen, 1, 2, 3, 128).clone(), tokens(gen, 1, 2, 3, 128).clone()
    k[0, 0, 1, 5] = float("nan")
    v[0, 1, 2, 7] = float("inf")
    cos, sin = angles(1, torch.arange(3, device=DEV), 128, torch.float32, gen)
    c = make_cache(bits, B=1)
    c.update_rotated(q, k, v, cos, sin, 0)
    want = turned(k, cos, sin)
    part = c.K_partial[0][:, :, :3]
    assert torch.equal(part.isnan(), want.isnan()) and int(part.isnan().sum()) == 2       # the channel and its partner
    assert torch.equal(part.nan_to_num(), want.nan_to_num())
    assert torch.equal(c.V_partial[0][:, :, :3], v)


def test_other_page_sizes_and_token_types_take_the_two_step_way():
    gen = torch.Generator(device=DEV).manual_seed(11)
    for page, dtype in ((32, torch.bfloat16), (64, torch.float16)):
        a, b = make_cache(4, page_size=page), make_cache(4, page_size=page)
        q, k, v = (tokens(gen, 2, h, 150, 128, dtype) for h in (4, 2, 2))
        cos, sin = angles(2, torch.arange(150, device=DEV), 128, torch.float32, gen)
        assert torch.equal(a.update_rotated(q, k, v, cos, sin, 0), turned(q, cos, sin))
        b.update_quantized(turned(k, cos, sin), v, 0)
        same_buffers(a, b, 0)


def test_empty_steps_change_nothing():
    c = make_cache(4)
    z = torch.empty(2, 2, 0, 128, dtype=torch.bfloat16, device=DEV)
    out = c.update_rotated(z, z, z, torch.empty(1, 0, 128, device=DEV), torch.empty(1, 0, 128, device=DEV), 0)
    assert out.shape == z.shape and c.get_seq_length(0) == 0


def test_append_on_another_stream_and_replayed_from_a_graph():
    gen = torch.Generator(device=DEV).manual_seed(13)
    n, seen = 70, 40
    q, k, v = (tokens(gen, 2, h, n, 128) for h in (4, 2, 2))
    old = torch.randn(2, 2, 2, 64, 128, device=DEV, generator=gen).to(torch.bfloat16)
    cos, sin = angles(2, seen + torch.arange(n, device=DEV), 128, torch.float32, gen)
    c, w = make_cache(8), make_cache(8)
    for x in (c, w):
        x.K_partial[0].copy_(old[0])
        x.V_partial[0].copy_(old[1])
        x._seen_tokens[0] = seen
    w.update_quantized(turned(k, cos, sin), v, 0)
    buf = c.buffers(0)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        out = rotate_append(q, k, v, cos, sin, buf, seen)
    torch.cuda.current_stream().wait_stream(st)
    same_buffers(c, w, 0)
    assert torch.equal(out, turned(q, cos, sin))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = rotate_append(q, k, v, cos, sin, buf, seen)
    for i in range(3):
        q.copy_(q.flip(2))
        for t in buf.values():
            t.zero_()
        buf["K_partial"].copy_(old[0])
        buf["V_partial"].copy_(old[1])
        g.replay()
        torch.cuda.synchronize()
        same_buffers(c, w, 0)
        assert torch.equal(out, turned(q, cos, sin))


@pytest.mark.parametrize("bits,D,kw", [(4, 128, {}), (4, 128, dict(meta_dtype=torch.float16, v_group=32)), (4, 64, {}),
                                       (4, 64, dict(v_group=32)), (8, 128, dict(meta_dtype=torch.float16)),
                                       (8, 64, {})])
@pytest.mark.parametrize("length,start", [(1, 0), (63, 62), (64, 0), (64, 64), (65, 3), (300, 0), (300, 130), (300, 299)])
def test_dequantize_cache(bits, D, kw, length, start):
    gen = torch.Generator(device=DEV).manual_seed(length)
    c = make_cache(bits, D=D, **kw)
    k, v = (torch.randn(2, 2, length, D, device=DEV, generator=gen).to(torch.bfloat16) for _ in range(2))
    c.update_quantized(k, v, 1)
    w = c.get_views(1)
    if bits == 4:
        K = dequantize_k_int4(w["K_packed"], w["K_scale"], w["K_mn"], 64)
        V = dequantize_v_int4(w["V_packed"], w["V_scale"], w["V_mn"])
    else:
        K, V = dequantize_k(w["K_uint8"], w["K_scale"], w["K_mn"], 64), dequantize_v(w["V_uint8"], w["V_scale"], w["V_mn"])
    K, V = torch.cat((K, w["K_partial"]), 2)[:, :, start:], torch.cat((V, w["V_partial"]), 2)[:, :, start:]
    for src in (w, c.buffers(1)):
        gk, gv = dequantize_cache(src, length, start=start)
        assert torch.equal(gk, K) and torch.equal(gv, V)


@pytest.mark.parametrize("bits", [4, 8])
def test_offsets_past_32_bits(bits):
    """Heads of the cache, and of q, k and v, more than 2^32 bytes apart."""
    gen = torch.Generator(device=DEV).manual_seed(9)
    room = torch.empty(5 << 30, dtype=torch.uint8, device=DEV)
    at = [0]

    def far(t):
        size, st = t.element_size(), list(t.contiguous().stride())
        st[0], st[1] = (1 << 24) // size, ((1 << 32) + (1 << 12)) // size     # a batch's row holds all tensors, 2^18 apart
        x = room.view(t.dtype).as_strided(t.shape, st, at[0] // size)
        at[0] += 1 << 18
        x.copy_(t)
        return x

    c = make_cache(bits)
    buffers = {n: t.clone() for n, t in c.buffers(0).items()}
    spread = {n: far(t) for n, t in buffers.items()}
    seen = 0
    for n in (70, 1, 130):
        q, k, v = (tokens(gen, 2, 2, n, 128) for _ in range(3))
        cos, sin = angles(2, seen + torch.arange(n, device=DEV), 128, torch.float32, gen)
        want = rotate_append(q, k, v, cos, sin, buffers, seen)
        got = rotate_append(far(q), far(k), far(v), cos, sin, spread, seen)
        assert torch.equal(got, want)
        seen += n
        for name, t in buffers.items():
            assert torch.equal(spread[name], t), name
        gk, gv = dequantize_cache(spread, seen)
        wk, wv = dequantize_cache(buffers, seen)
        assert torch.equal(gk, wk) and torch.equal(gv, wv)


@pytest.mark.parametrize("bits", [4, 8, 3])
def test_a_prompt_and_decode_steps(bits):
    """A layer as a model runs it: the prompt rotated into the cache and attended, then steps of one token."""
    gen = torch.Generator(device=DEV).manual_seed(bits)
    got, want = make_cache(bits, B=1, layers=1), make_cache(bits, B=1, layers=1)
    seen = 0
    for n in (190, 1, 1, 1):
        q, k, v = (tokens(gen, 1, h, n, 128) for h in (6, 2, 2))
        cos, sin = angles(1, seen + torch.arange(n, device=DEV), 128, torch.bfloat16, gen)
        qr = got.update_rotated(q, k, v, cos, sin, 0)
        want.update_quantized(turned(k, cos, sin), v, 0)
        outs = []
        for c, x in ((got, qr), (want, turned(q, cos, sin).contiguous())):
            if n > 1:
                outs.append(prefill_attention_layer(x, c.get_views(0), page_size=64))
            else:
                outs.append(sparse_decode_layer(x, c.get_views(0), retention=0.5, num_sinks=1, window_pages=1, page_size=64))
        assert torch.equal(*outs)
        seen += n


def test_refusals_leave_the_cache_alone():
    c = make_cache(4)
    q = torch.zeros(2, 4, 2, 128, dtype=torch.bfloat16, device=DEV)
    k = q[:, :2]
    cos = torch.zeros(1, 2, 128, device=DEV)
    before = {n: t.clone() for n, t in c.buffers(0).items()}
    buf = c.buffers(0)
    off = torch.empty(2 * 2 * 5 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(2, 2, 5, 128)
    with pytest.raises(NotImplementedError):
        rotate_append(q, k, k, cos, cos, dict(buf, K_scale=off), 0)        # would have to be copied: written in place
    with pytest.raises(AssertionError):
        rotate_append(q, k, k, cos.cpu(), cos, buf, 0)
    with pytest.raises(RuntimeError):
        rotate_append(q, k, k, cos, cos, buf, 319)
    for n, t in c.buffers(0).items():
        assert torch.equal(t, before[n])
