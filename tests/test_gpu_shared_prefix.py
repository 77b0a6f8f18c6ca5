"""shared_prefix_attention against the softmax in 64 bits over the cache's own values.

Tolerance, from the roundings: the operands of both products are fp16 (half a step is u = 2^-11 of a value); queries
are exact.  A key's rounding moves a score by at most u sum |q_d k_d| sm_scale; keys are kept times 2^-6, so scale,
minimum and result are exact to 2^-19 each where they are small: a score's error is at most
e = (u sum |q_d k_d| + 3 2^-19 sum |q_d|) sm_scale, the largest over a row's keys.  A weight is rounded once (u), a value
once (u), and the weights' sum is that of the rounded ones, so a term p v is off by a factor within
e^(2 e) (1 + 3.1 u) of the row's common one:
|O - O*| <= (e^(2 e) (1 + 3.1 u) - 1 + 1e-5) sum p |v|, 1e-5 for the fp32 sums, plus 2^-25 for values below 2^-14,
N 2^-32 max |v| for weights below 2^-21 of the largest (fp16's smallest steps), and half a step of the output's type.
"""
import math

import pytest
import torch

from flashquest_amd import _lib as L
from flashquest_amd.cache import PersistentInt4KVCache, PersistentInt8KVCache
from flashquest_amd.eager import shared_prefix_attention
from flashquest_amd.eager.shared_prefix import _describe
from flashquest_amd.kernel import rotate_append

pytestmark = pytest.mark.gpu

DEV = "cuda"
CLASSES = {4: PersistentInt4KVCache, 8: PersistentInt8KVCache}


def filled(bits, gen, B, H, D, length, k_size=1.0, v_size=1.0, **kw):
    c = CLASSES[bits](batch_size=B, num_layers=1, num_kv_heads=H, head_dim=D, max_seq_len=max(64, length + 64),
                      device=DEV, **kw)
    if length:
        k = torch.randn(B, H, length, D, device=DEV, generator=gen) * k_size + 0.3 * k_size
        v = torch.randn(B, H, length, D, device=DEV, generator=gen) * v_size
        c.update_quantized(k.to(torch.bfloat16), v.to(torch.bfloat16), 0)
    return c


def values(views, bits):
    """The views' keys and values in 64 bits (B, H, S, D)."""
    def codes(x):
        if bits == 8:
            return x.double()
        return torch.stack((x & 15, x >> 4), -1).flatten(-2).double()
    kn, vn = ("K_packed", "V_packed") if bits == 4 else ("K_uint8", "V_uint8")
    S = views[kn].shape[2]
    page = torch.arange(S, device=DEV) // 64
    k = codes(views[kn]) * views["K_scale"].double()[:, :, page] + views["K_mn"].double()[:, :, page]
    D = k.shape[-1]
    G = views["V_scale"].shape[-1]
    grp = torch.arange(D, device=DEV) * G // D
    v = codes(views[vn]) * views["V_scale"].double()[..., grp] + views["V_mn"].double()[..., grp]
    return torch.cat((k, views["K_partial"].double()), 2), torch.cat((v, views["V_partial"].double()), 2)


def reference(q, prefix, suffix, bits, start=None, sm_scale=None):
    """(O, lse, tolerance) in 64 bits."""
    B, Hq, n, D = q.shape
    sm = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    kp, vp = values(prefix, bits)
    ks, vs = values(suffix, bits)
    H = kp.shape[1]
    k = torch.cat((kp.expand(B, -1, -1, -1), ks), 2).repeat_interleave(Hq // H, 1)
    v = torch.cat((vp.expand(B, -1, -1, -1), vs), 2).repeat_interleave(Hq // H, 1)
    Np, Ns = kp.shape[2], ks.shape[2]
    j = torch.arange(Ns, device=DEV)
    ok = (j[None] <= Ns - n + torch.arange(n, device=DEV)[:, None])[None].repeat(B, 1, 1)
    if start is not None:
        ok &= j >= start.long()[:, None, None]
    ok = torch.cat((torch.ones(B, n, Np, dtype=torch.bool, device=DEV), ok), 2)[:, None]
    qd = q.double()
    s = (qd @ k.transpose(2, 3) * sm).masked_fill(~ok, -math.inf)
    p = torch.softmax(s, -1)
    # values of padding tokens do not count, whatever they are
    vc = v.masked_fill(~ok.any(2)[..., None].expand(-1, Hq, -1, D), 0.0)
    o = p @ vc
    u = 2.0 ** -11
    size = ((qd.abs() @ k.abs().transpose(2, 3)) * u + qd.abs().sum(-1, True) * 3 * 2.0 ** -19) * sm
    size = size.masked_fill(~ok, 0.0).amax(-1, True)
    pv = p @ vc.abs()
    tol = (torch.exp(2 * size) * (1 + 3.1 * u) - 1 + 1e-5) * pv + 2.0 ** -25
    tol = tol + (Np + Ns) * 2.0 ** -32 * vc.abs().amax((2, 3), True)
    tol = tol + o.abs() * (torch.finfo(q.dtype).eps / 2)
    return o, torch.logsumexp(s, -1), tol, size[..., 0] + 2 * u


def check(q, prefix, suffix, bits, **kw):
    o, lse, tol, ltol = reference(q, prefix, suffix, bits, kw.get("suffix_start") if "suffix_start" in kw else None,
                                  kw.get("sm_scale"))
    got, glse = shared_prefix_attention(q, prefix, suffix, return_lse=True, **kw)
    assert got.shape == q.shape and got.dtype == q.dtype and glse.shape == q.shape[:-1]
    err = (got.double() - o).abs()
    assert bool((err <= tol).all()), f"{float((err / tol).max())} of the tolerance, at {float(err.max())}"
    assert bool(((glse.double() - lse).abs() <= ltol + 1e-5 * lse.abs()).all())
    return got


LENGTHS = [(1, 1), (63, 1), (64, 64), (65, 70), (127, 3), (200, 129), (1000, 37), (4099, 700)]


@pytest.mark.parametrize("bits,D,dtype,kw", [
    (4, 128, torch.bfloat16, {}),
    (4, 128, torch.float16, dict(meta_dtype=torch.float16, v_group=32)),
    (4, 64, torch.float16, dict(v_group=32)),
    (8, 128, torch.float16, dict(meta_dtype=torch.float16)),
    (8, 64, torch.bfloat16, {}),
])
@pytest.mark.parametrize("prefix,suffix", LENGTHS)
def test_one_token(bits, D, dtype, kw, prefix, suffix):
    gen = torch.Generator(device=DEV).manual_seed(prefix * 1000 + suffix)
    for B, Hq, H in ((1, 2, 2), (3, 6, 2), (9, 8, 1), (40, 3, 1)):
        p, s = filled(bits, gen, 1, H, D, prefix, **kw), filled(bits, gen, B, H, D, suffix, **kw)
        q = torch.randn(B, Hq, 1, D, device=DEV, generator=gen).to(dtype)
        check(q, p.get_views(0), s.get_views(0), bits)


@pytest.mark.parametrize("bits,D", [(4, 128), (8, 128), (4, 64), (8, 64)])
@pytest.mark.parametrize("B,Hq,H,n,prefix,suffix", [(2, 6, 2, 2, 70, 2), (5, 5, 1, 5, 128, 69), (3, 8, 2, 67, 333, 67),
                                                    (1, 4, 4, 130, 65, 257), (2, 14, 2, 3, 5, 64), (2, 8, 1, 64, 2000, 128)])
def test_several_tokens(bits, D, B, Hq, H, n, prefix, suffix):
    gen = torch.Generator(device=DEV).manual_seed(n + prefix)
    p, s = filled(bits, gen, 1, H, D, prefix), filled(bits, gen, B, H, D, suffix)
    q = torch.randn(B, Hq, n, D, device=DEV, generator=gen).to(torch.bfloat16)
    check(q, p.get_views(0), s.get_views(0), bits)


# enough rows for the row tiles in LDS, of 256 and of 128 rows, for both parts and for the prefix alone: pages that
# fill half a stage, no whole page in either part, rows that end inside a tile, splits
MANY = [(9, 48, 2, 100, 65, 100), (9, 48, 2, 100, 40, 100), (9, 32, 2, 63, 1823, 63), (9, 32, 2, 63, 95, 64),
        (9, 32, 2, 63, 65, 63), (9, 48, 2, 33, 40, 33), (5, 24, 1, 100, 4415, 140), (3, 24, 2, 60, 6011, 60),
        (4, 40, 1, 160, 2000, 1000)]


@pytest.mark.parametrize("bits,D,dtype,kw", [
    (4, 128, torch.bfloat16, {}),
    (4, 128, torch.float16, dict(meta_dtype=torch.float16, v_group=32)),
    (4, 64, torch.float16, dict(v_group=32)),
    (8, 128, torch.bfloat16, dict(meta_dtype=torch.float16)),
    (8, 64, torch.bfloat16, {}),
])
@pytest.mark.parametrize("B,Hq,H,n,prefix,suffix", MANY)
def test_many_rows(bits, D, dtype, kw, B, Hq, H, n, prefix, suffix):
    gen = torch.Generator(device=DEV).manual_seed(n + prefix + suffix)
    p, s = filled(bits, gen, 1, H, D, prefix, **kw), filled(bits, gen, B, H, D, suffix, **kw)
    q = torch.randn(B, Hq, n, D, device=DEV, generator=gen).to(dtype)
    check(q, p.get_views(0), s.get_views(0), bits)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n,suffix", [(100, 260), (37, 199)])
def test_many_rows_with_left_padding(bits, n, suffix):
    """Starts as in test_left_padding, among them ones that leave a query token none of its own keys."""
    gen = torch.Generator(device=DEV).manual_seed(7 + n)
    starts = torch.tensor([0, 1, 63, 64, 65, 128, suffix - n + 2, suffix, 1000, -5], dtype=torch.int32, device=DEV)
    B = len(starts)
    p = filled(bits, gen, 1, 2, 128, 130)
    s = CLASSES[bits](batch_size=B, num_layers=1, num_kv_heads=2, head_dim=128, max_seq_len=320, device=DEV)
    k, v = (torch.randn(B, 2, suffix, 128, device=DEV, generator=gen).to(torch.bfloat16) for _ in range(2))
    for b, x in enumerate(starts.tolist()):
        v[b, :, 0:max(0, min(x, suffix)):2] = float("nan")
        v[b, :, 1:max(0, min(x, suffix)):2] = float("inf")
    s.update_quantized(k, v, 0)
    q = torch.randn(B, 48, n, 128, device=DEV, generator=gen).to(torch.bfloat16)
    check(q, p.get_views(0), s.get_views(0), bits, suffix_start=starts)


@pytest.mark.parametrize("bits,D,kw", [(4, 128, {}), (4, 128, dict(v_group=32)), (4, 64, {}), (8, 128, {}), (8, 64, {})])
@pytest.mark.parametrize("B,Hq,H,n,prefix,suffix", [(3, 6, 2, 5, 100, 70), (2, 4, 2, 70, 65, 140), (9, 32, 2, 63, 95, 64),
                                                    (9, 48, 2, 100, 65, 128), (9, 48, 2, 100, 65, 100)])
def test_a_value_that_is_not_finite_stays_with_the_queries_that_attend_it(bits, D, kw, B, Hq, H, n, prefix, suffix):
    """NaN and infinities among the values of a step's own tokens, in whole pages and in the partial one, one sequence
    without: queries before the first of them are as without it, queries behind it are not finite."""
    gen = torch.Generator(device=DEV).manual_seed(n + suffix)
    p = filled(bits, gen, 1, H, D, prefix, **kw)
    k, v = (torch.randn(B, H, suffix, D, device=DEV, generator=gen).to(torch.bfloat16) for _ in range(2))
    first = torch.randint(suffix - n + 1, suffix, (B,), device=DEV, generator=gen)
    first[0], first[1], first[-1] = suffix - 1, suffix - n + 1, suffix       # the last query alone; all but one; none
    bad = v.clone()
    for b in range(B - 1):
        bad[b, :, first[b]] = (float("nan"), float("inf"), -float("inf"))[b % 3]
    q = torch.randn(B, Hq, n, D, device=DEV, generator=gen).to(torch.bfloat16)
    outs = []
    for x in (v, bad):
        s = CLASSES[bits](batch_size=B, num_layers=1, num_kv_heads=H, head_dim=D, max_seq_len=suffix + 64, device=DEV, **kw)
        s.update_quantized(k, x, 0)
        outs.append(shared_prefix_attention(q, p.get_views(0), s.get_views(0), return_lse=True))
    (want, wl), (got, gl) = outs
    before = torch.arange(n, device=DEV) + suffix - n < first[:, None]
    assert bool(before.any()) and not bool(before.all())
    assert torch.equal(got.transpose(1, 2)[before], want.transpose(1, 2)[before])
    assert torch.equal(gl, wl)
    assert not bool(got.transpose(1, 2)[~before].isfinite().any())


def far_apart(views):
    """The views' tensors with their heads more than 2^32 bytes apart, as slices of a long cache have them."""
    room = torch.empty((5 << 30), dtype=torch.uint8, device=DEV)
    out, at = dict(views), 0
    for name, t in views.items():
        if not torch.is_tensor(t) or t.numel() == 0:
            continue
        size = t.element_size()
        st = list(t.contiguous().stride())
        st[0], st[1] = (1 << 22) // size, ((1 << 32) + (1 << 12)) // size
        out[name] = room.view(t.dtype).as_strided(t.shape, st, at // size)
        out[name].copy_(t)
        at += 1 << 18
    return out


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("B,Hq,n,prefix,suffix", [(3, 6, 1, 150, 70), (9, 32, 63, 95, 70)])
def test_offsets_past_32_bits(bits, B, Hq, n, prefix, suffix):
    gen = torch.Generator(device=DEV).manual_seed(29)
    p, s = filled(bits, gen, 1, 2, 128, prefix), filled(bits, gen, B, 2, 128, suffix)
    q = torch.randn(B, Hq, n, 128, device=DEV, generator=gen).to(torch.bfloat16)
    want = shared_prefix_attention(q, p.get_views(0), s.get_views(0))
    assert torch.equal(shared_prefix_attention(q, far_apart(p.get_views(0)), far_apart(s.get_views(0))), want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("n", [1, 5])
def test_left_padding(bits, n):
    """Starts inside, at the ends of and beyond the pages, and past every token; padding holds NaN and infinities."""
    gen = torch.Generator(device=DEV).manual_seed(3 + n)
    starts = torch.tensor([0, 1, 63, 64, 65, 130, 199, 195, 200, 1000, -5], dtype=torch.int32, device=DEV)
    B = len(starts)
    p = filled(bits, gen, 1, 2, 128, 300)
    s = CLASSES[bits](batch_size=B, num_layers=1, num_kv_heads=2, head_dim=128, max_seq_len=256, device=DEV)
    k, v = (torch.randn(B, 2, 200, 128, device=DEV, generator=gen).to(torch.bfloat16) for _ in range(2))
    for b, x in enumerate(starts.tolist()):
        v[b, :, 0:max(0, min(x, 200)):2] = float("nan")
        v[b, :, 1:max(0, min(x, 200)):2] = float("inf")
    s.update_quantized(k, v, 0)
    views = s.get_views(0)
    q = torch.randn(B, 6, n, 128, device=DEV, generator=gen).to(torch.bfloat16)
    clean = dict(views)          # the reference takes the padding's values as 0
    for name in ("V_scale", "V_mn", "V_partial"):
        clean[name] = views[name].nan_to_num(0.0, 0.0, 0.0)
    o, lse, tol, _ = reference(q, p.get_views(0), clean, bits, starts)
    got = shared_prefix_attention(q, p.get_views(0), views, suffix_start=starts)
    assert bool(((got.double() - o).abs() <= tol).all())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("k_size,v_size,q_size", [(30.0, 1.0, 0.05), (1.0, 100.0, 3.0), (0.05, 0.02, 8.0), (4.0, 1.0, 4.0),
                                                  (1e-3, 1e-2, 1e3), (1.0, 1.0, 0.0)])
def test_sizes_of_keys_values_and_queries(bits, k_size, v_size, q_size):
    gen = torch.Generator(device=DEV).manual_seed(17)
    p, s = (filled(bits, gen, b, 2, 128, n, k_size, v_size) for b, n in ((1, 500), (4, 90)))
    q = (torch.randn(4, 6, 1, 128, device=DEV, generator=gen) * q_size).to(torch.bfloat16)
    check(q, p.get_views(0), s.get_views(0), bits)
    check(q, p.get_views(0), s.get_views(0), bits, sm_scale=0.3)


def test_a_long_prefix_far_above_a_sink():
    """65536 tokens, one key that takes most of the weight; the weights of the others are small but many."""
    gen = torch.Generator(device=DEV).manual_seed(23)
    p = filled(8, gen, 1, 1, 128, 65536 + 11, 0.1, 1.0)
    q = torch.randn(20, 2, 1, 128, device=DEV, generator=gen).to(torch.bfloat16)
    s = filled(8, gen, 20, 1, 128, 9)
    s.K_partial[0][:, :, 0] = (q[:, :1, 0] * 0.9).to(torch.bfloat16)
    check(q, p.get_views(0), s.get_views(0), 8)


def test_nan_in_a_row_stays_in_it_and_nan_keys_reach_every_row():
    gen = torch.Generator(device=DEV).manual_seed(29)
    p, s = filled(4, gen, 1, 2, 128, 200), filled(4, gen, 4, 2, 128, 70)
    q = torch.randn(4, 4, 1, 128, device=DEV, generator=gen).to(torch.bfloat16)
    good, _, tol, _ = reference(q, p.get_views(0), s.get_views(0), 4)
    bad = q.clone()
    bad[1, 2, 0, 5] = float("nan")
    bad[2, 0, 0, 7] = float("inf")
    got = shared_prefix_attention(bad, p.get_views(0), s.get_views(0))
    assert bool(got[1, 2].isnan().all()) and bool(got[2, 0].isnan().all())
    got = got.double()
    got[1, 2], got[2, 0] = good[1, 2], good[2, 0]
    assert bool(((got - good).abs() <= tol).all())
    s.K_partial[0][3, 1, 2] = float("nan")
    got = shared_prefix_attention(q, p.get_views(0), s.get_views(0))
    assert bool(got[3, 2:].isnan().all())
    got = got.double()
    got[3, 2:] = good[3, 2:]
    assert bool(((got - good).abs() <= tol).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_strides_and_alignments(bits):
    """Queries as projections leave them; planes with the tokens outside the heads, and misaligned ones (copied)."""
    gen = torch.Generator(device=DEV).manual_seed(31)
    p, s = filled(bits, gen, 1, 2, 128, 150), filled(bits, gen, 3, 2, 128, 150)
    q = torch.randn(3, 2, 8 * 128, device=DEV, generator=gen).to(torch.bfloat16)
    qt = q.view(3, 2, 8, 128).transpose(1, 2)
    want = shared_prefix_attention(qt.contiguous(), p.get_views(0), s.get_views(0))
    views = s.get_views(0)
    turned = {n: t.transpose(1, 2).contiguous().transpose(1, 2) if torch.is_tensor(t) else t for n, t in views.items()}

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)
    off = {n: shifted(t) if torch.is_tensor(t) else t for n, t in views.items()}
    base = torch.empty(3, 2, 8 * 128 + 1, dtype=torch.bfloat16, device=DEV)
    base[..., 1:] = q
    for qq, v in ((qt, views), (qt, turned), (qt, off), (base[..., 1:].unflatten(2, (8, 128)).transpose(1, 2), views)):
        assert torch.equal(shared_prefix_attention(qq, p.get_views(0), v), want)


def test_the_same_call_gives_the_same_bits_on_other_streams_and_from_graphs():
    gen = torch.Generator(device=DEV).manual_seed(37)
    p, s = filled(8, gen, 1, 2, 128, 3000), filled(8, gen, 12, 2, 128, 200)
    pv, sv = p.get_views(0), s.get_views(0)
    q = torch.randn(12, 8, 1, 128, device=DEV, generator=gen).to(torch.bfloat16)
    start = torch.arange(12, dtype=torch.int32, device=DEV) * 9
    want = shared_prefix_attention(q, pv, sv, suffix_start=start)
    st = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for x in st:
        x.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(x):
            outs.append(shared_prefix_attention(q, pv, sv, suffix_start=start))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    # two graphs of other queries, replayed at the same time
    qs = [q.clone(), q.flip(0).contiguous()]
    graphs = []
    for x in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = shared_prefix_attention(x, pv, sv, suffix_start=start)
        graphs.append((g, o))
    for i in range(3):
        for x in qs:
            x.copy_(torch.randn(x.shape, device=DEV, generator=gen))
        start.copy_((start + 7 * i) % 150)
        torch.cuda.synchronize()
        for (g, _), x in zip(graphs, st):
            with torch.cuda.stream(x):
                g.replay()
        torch.cuda.synchronize()
        for (_, o), x in zip(graphs, qs):
            assert torch.equal(o, shared_prefix_attention(x, pv, sv, suffix_start=start))


@pytest.mark.parametrize("B,Hq,n", [(7, 5, 3), (1, 1, 1), (33, 2, 1)])
def test_nothing_is_written_around_the_output_and_the_workspace(B, Hq, n):
    """Odd row counts: the kernels' row tiles reach past the last row, their stores do not."""
    gen = torch.Generator(device=DEV).manual_seed(41)
    p, s = filled(4, gen, 1, 1, 128, 130), filled(4, gen, B, 1, 128, 20)
    q = torch.randn(B, Hq, n, 128, device=DEV, generator=gen).to(torch.float16)
    pd, pt, k0 = _describe(p.get_views(0), 4, 128)
    sd, st, k1 = _describe(s.get_views(0), 4, 128)
    edge = 4096
    out = torch.full((2 * edge + q.numel(),), 7.0, dtype=torch.float16, device=DEV)
    lse = torch.full((2 * edge + B * Hq * n,), 7.0, device=DEV)
    o, l = out[edge:-edge].view(q.shape), lse[edge:-edge].view(B, Hq, n)
    query = L.SharedQuery(q.data_ptr(), L.strides(q, 4), o.data_ptr(), L.strides(o, 4), l.data_ptr(), L.strides(l, 3),
                          None, L.FQ_F16, B, Hq, n, 0.0)
    need = L.lib().fq_shared_prefix_workspace_bytes(pd, pt, sd, st, query, 4)
    ws = torch.full((2 * edge + need,), 77, dtype=torch.uint8, device=DEV)
    L.check(L.lib().fq_shared_prefix_int4(pd, pt, sd, st, query, ws[edge:].data_ptr(), need, L.stream_handle(q.device)))
    want, wl = shared_prefix_attention(q, p.get_views(0), s.get_views(0), return_lse=True)
    assert torch.equal(o, want) and torch.equal(l, wl)
    for t, x in ((out, 7.0), (lse, 7.0), (ws, 77)):
        assert bool((t[:edge] == x).all()) and bool((t[-edge:] == x).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_a_batch_as_it_runs(bits):
    """A prompt into the prefix cache, questions of their own into the suffix cache (left-padded), then tokens, all
    rotated at their own positions; against one cache per sequence in 64 bits, built from the same values."""
    gen = torch.Generator(device=DEV).manual_seed(43)
    B, Hq, H, D, n_prefix = 3, 6, 2, 128, 150
    turn = 10000.0 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)

    def angles(at):
        a = (at.double()[..., None] * turn).repeat(1, 1, 2)
        return a.cos().to(torch.bfloat16), a.sin().to(torch.bfloat16)

    def rows(b, h, n):
        return torch.randn(b, n, h, D, device=DEV, generator=gen).to(torch.bfloat16).transpose(1, 2)

    prefix = CLASSES[bits](batch_size=1, num_layers=1, num_kv_heads=H, head_dim=D, max_seq_len=256, device=DEV)
    suffix = CLASSES[bits](batch_size=B, num_layers=1, num_kv_heads=H, head_dim=D, max_seq_len=256, device=DEV)
    prefix.update_rotated(rows(1, Hq, n_prefix), rows(1, H, n_prefix), rows(1, H, n_prefix),
                          *angles(torch.arange(n_prefix, device=DEV)[None]), 0)
    start = torch.tensor([0, 9, 30], dtype=torch.int32, device=DEV)
    seen = 0
    for n in (62, 1, 1, 1, 4):
        at = (n_prefix + seen + torch.arange(n, device=DEV)[None] - start[:, None]).clamp_min(0)
        q = suffix.update_rotated(rows(B, Hq, n), rows(B, H, n), rows(B, H, n), *angles(at), 0)
        seen += n
        views = suffix.get_views(0)
        o, _, tol, _ = reference(q, prefix.get_views(0), views, bits, start)
        got = shared_prefix_attention(q, prefix.get_views(0), views, suffix_start=start)
        assert bool(((got.double() - o).abs() <= tol).all())


def test_a_cache_past_2_gib_of_a_layer():
    """Offsets past 32 bits: 64 sequences x 8 heads x 65600 tokens of INT8 codes a layer."""
    gen = torch.Generator(device=DEV).manual_seed(47)
    B, H, room, n = 64, 8, 65600, 100
    p = filled(8, gen, 1, H, 128, 64)
    s = CLASSES[8](batch_size=B, num_layers=1, num_kv_heads=H, head_dim=128, max_seq_len=room, device=DEV)
    k, v = (torch.randn(B, H, n, 128, device=DEV, generator=gen).to(torch.bfloat16) for _ in range(2))
    ones, zeros = torch.ones(1, n, 128, device=DEV), torch.zeros(1, n, 128, device=DEV)
    rotate_append(k, k, v, ones, zeros, s.buffers(0), 0)
    s._seen_tokens[0] = n
    q = torch.randn(B, H, 1, 128, device=DEV, generator=gen).to(torch.bfloat16)
    got = shared_prefix_attention(q, p.get_views(0), s.get_views(0))
    small = CLASSES[8](batch_size=B, num_layers=1, num_kv_heads=H, head_dim=128, max_seq_len=128, device=DEV)
    small.update_quantized(k, v, 0)
    assert torch.equal(got, shared_prefix_attention(q, p.get_views(0), small.get_views(0)))
