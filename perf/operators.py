"""Cases of the operators that put tokens into a paged cache and attend a prefix that a batch shares.

``append``: a step's query, key and value rows as the projections leave them, with the rotary cos / sin of
their positions: the queries and keys are rotated, the keys and values join one layer's packed cache (pages of
64 tokens are quantised once they are whole, the rest waits in the 16-bit partial page), and the tokens of the
pages concerned are read back as the values that the cache holds.

``shared``: a decode step (or a few tokens, or a chunk of a prompt) of B sequences over one prefix that all
share, held once, and each sequence's own tokens after it.

Both have their plain form here, in elementary torch operations in 32 bits, and the definition in 64 bits.
"""
import math

import torch

own = False

PAGE = 64
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ the cases --
def listed():
    return [
        # one user's next token: one row per head, nothing completes a page; the call's latency is all there is
        dict(name="append 1 token int4", op="append", bits=4, meta="bf16", v32=False, batch=1, hq=24, hkv=8, d=128,
             rot=128, seen=8229, new=1, angles="bf16"),
        # a batch's step of several accepted draft tokens, in the middle of a page
        dict(name="append 16x5 tokens int8", op="append", bits=8, meta="bf16", v32=False, batch=16, hq=32, hkv=8,
             d=128, rot=128, seen=4105, new=5, angles="bf16"),
        # a prompt chunk behind earlier pages; its last page stays partial
        dict(name="append 2047 tokens int4 d64", op="append", bits=4, meta="bf16", v32=False, batch=2, hq=32, hkv=8,
             d=64, rot=32, seen=1024, new=2047, angles="f32"),
        # a whole prompt, 32-channel value groups
        dict(name="append 32k prompt int4 v32", op="append", bits=4, meta="f16", v32=True, batch=1, hq=24, hkv=8,
             d=128, rot=128, seen=0, new=32768, angles="bf16"),
        # several prompts of one length at once
        dict(name="append 4x8191 tokens int8", op="append", bits=8, meta="bf16", v32=False, batch=4, hq=32, hkv=8,
             d=128, rot=128, seen=0, new=8191, angles="f32"),
        # a short system prompt and four users: latency
        dict(name="shared 4 seqs 1000 int4", op="shared", bits=4, meta="bf16", v32=False, batch=4, hq=24, hkv=8,
             d=128, prefix=1000, suffix=37, tokens=1, padded=False, dtype="bf16"),
        # a long document and 16 questions about it, left-padded to one length
        dict(name="shared 16 seqs 32k int4 v32", op="shared", bits=4, meta="f16", v32=True, batch=16, hq=24, hkv=8,
             d=128, prefix=32768, suffix=451, tokens=1, padded=True, dtype="f16"),
        # a few-shot prompt and a full batch
        dict(name="shared 64 seqs 8k int8", op="shared", bits=8, meta="bf16", v32=False, batch=64, hq=32, hkv=8,
             d=128, prefix=8192, suffix=300, tokens=1, padded=False, dtype="bf16"),
        # 64-channel heads, more of the batch's own tokens than of the prefix
        dict(name="shared 32 seqs 2k int8 d64", op="shared", bits=8, meta="bf16", v32=False, batch=32, hq=32, hkv=8,
             d=64, prefix=2085, suffix=1500, tokens=1, padded=True, dtype="bf16"),
        # draft tokens verified for wide groups of query heads
        dict(name="shared 8x5 tokens 16k int4", op="shared", bits=4, meta="bf16", v32=False, batch=8, hq=64, hkv=8,
             d=128, prefix=16384, suffix=200, tokens=5, padded=False, dtype="bf16"),
        # the questions themselves, a chunk of each, over a long document
        dict(name="shared 4x128 tokens 16k int8", op="shared", bits=8, meta="bf16", v32=False, batch=4, hq=32, hkv=8,
             d=128, prefix=16411, suffix=128, tokens=128, padded=False, dtype="bf16"),
        # the largest batch over the longest prompt
        dict(name="shared 128 seqs 32k int4", op="shared", bits=4, meta="bf16", v32=False, batch=128, hq=32, hkv=8,
             d=128, prefix=32768, suffix=640, tokens=1, padded=False, dtype="bf16"),
    ]


HEADS = ((24, 8), (32, 8), (64, 8), (8, 8), (40, 8), (6, 2))


def draw(rng):
    spread = lambda lo, hi: min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))  # noqa: E731
    bits = rng.choice((4, 8))
    hq, hkv = rng.choice(HEADS)
    c = dict(bits=bits, meta=rng.choice(("bf16", "f16")), v32=bits == 4 and rng.random() < 0.4, hq=hq, hkv=hkv,
             d=rng.choice((128, 128, 64)))
    if rng.random() < 0.4:
        c.update(op="append", batch=spread(1, 16), rot=rng.choice((c["d"], c["d"], c["d"] // 2)),
                 angles=rng.choice(("bf16", "f32")))
        new = spread(1, 32768)
        c["new"] = max(1, min(new, 32768 * 24 // (c["batch"] * hq)))
        pages = spread(1, 64) - 1
        # from the start of a page, or within one
        c["seen"] = PAGE * pages + (rng.randrange(PAGE - c["new"]) if c["new"] < PAGE else 0)
    else:
        c.update(op="shared", batch=spread(1, 128), tokens=rng.choice((1, 1, 1, spread(1, 128))),
                 padded=rng.random() < 0.4, dtype=rng.choice(("bf16", "bf16", "f16")))
        c["batch"] = max(1, min(c["batch"], 128 * 32 // (hq * c["tokens"])))
        rows = c["batch"] * hq * c["tokens"]
        c["prefix"] = spread(1, min(65536, 128 * 32 * 32768 // rows))
        c["suffix"] = max(c["tokens"], spread(1, min(2048, 128 * 32 * 2048 // rows)))
    return c


# ----------------------------------------------------------------------------------------------- the inputs --
def _type(name):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


def _key_pages(k, bits, meta):
    """Whole pages of keys (B, H, n, D), 16 bits: codes, and each page's scale and minimum of each channel.
    The scale's arithmetic is in the keys' type, the codes' in 32 bits."""
    p = k.unflatten(2, (-1, PAGE))
    mn, mx = p.amin(3), p.amax(3)
    scale = ((mx - mn).float() * torch.tensor(1.0 / (2 ** bits - 1), dtype=torch.float32, device=k.device)).to(k.dtype)
    scale = scale.clamp_min(EPS)
    codes = ((p.float() - mn.float()[:, :, :, None]) / scale.float()[:, :, :, None]).round().clamp(0, 2 ** bits - 1)
    return codes.flatten(2, 3).to(torch.uint8), scale.to(meta), mn.to(meta)


def _value_rows(v, bits, meta, groups):
    """Values (B, H, n, D): codes, and each token's (and channel group's) scale and minimum, in 32 bits."""
    g = v.float().unflatten(3, (groups, -1))
    mn, mx = g.amin(4), g.amax(4)
    scale = ((mx - mn) * torch.tensor(1.0 / (2 ** bits - 1), dtype=torch.float32, device=v.device)).clamp_min(EPS)
    codes = ((g - mn[..., None]) / scale[..., None]).round().clamp(0, 2 ** bits - 1)
    return codes.flatten(3, 4).to(torch.uint8), scale.to(meta), mn.to(meta)


def _packed(codes, bits):
    return codes if bits == 8 else codes[..., 0::2] | codes[..., 1::2] << 4


def _unpacked(packed, bits):
    return packed if bits == 8 else torch.stack((packed & 15, packed >> 4), -1).flatten(-2)


def _named(bits):
    return ("K_packed", "V_packed") if bits == 4 else ("K_uint8", "V_uint8")


def _cache(case, gen, batch, length):
    """One layer's cache of `length` tokens, as its views: the whole pages' planes and the partial page."""
    h, d, bits, meta = case["hkv"], case["d"], case["bits"], _type(case["meta"])
    groups = d // 32 if case["v32"] else 1
    # keys have channels of their own size and offset, values are spread around 0
    width = torch.exp(torch.randn(h, 1, d, device="cuda", generator=gen) * 0.6)
    middle = torch.randn(h, 1, d, device="cuda", generator=gen)
    k = (torch.randn(batch, h, length, d, device="cuda", generator=gen) * width + middle).to(torch.bfloat16)
    v = torch.randn(batch, h, length, d, device="cuda", generator=gen).to(torch.bfloat16)
    done = length // PAGE * PAGE
    kn, vn = _named(bits)
    kc, ks, km = _key_pages(k[:, :, :done], bits, meta)
    vc, vs, vm = _value_rows(v[:, :, :done], bits, meta, groups)
    return {kn: _packed(kc, bits), "K_scale": ks, "K_mn": km, vn: _packed(vc, bits), "V_scale": vs, "V_mn": vm,
            "K_partial": k[:, :, done:].contiguous(), "V_partial": v[:, :, done:].contiguous()}


def _buffers(case, gen):
    """One layer's buffers with room for the tokens, and `seen` % 64 tokens in the partial page."""
    b, h, d, bits, meta = case["batch"], case["hkv"], case["d"], case["bits"], _type(case["meta"])
    room = -(-(case["seen"] + case["new"]) // PAGE) * PAGE
    groups = d // 32 if case["v32"] else 1
    kn, vn = _named(bits)
    zeros = lambda *s, t: torch.zeros(*s, dtype=t, device="cuda")  # noqa: E731
    part = torch.randn(2, b, h, PAGE, d, device="cuda", generator=gen).to(torch.bfloat16)
    part[:, :, :, case["seen"] % PAGE:] = 0
    return {kn: zeros(b, h, room, d * bits // 8, t=torch.uint8), "K_scale": zeros(b, h, room // PAGE, d, t=meta),
            "K_mn": zeros(b, h, room // PAGE, d, t=meta), vn: zeros(b, h, room, d * bits // 8, t=torch.uint8),
            "V_scale": zeros(b, h, room, groups, t=meta), "V_mn": zeros(b, h, room, groups, t=meta),
            "K_partial": part[0].clone(), "V_partial": part[1].clone()}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    b, hq, hkv, d = case["batch"], case["hq"], case["hkv"], case["d"]
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    if case["op"] == "append":
        n = case["new"]
        # what the projections leave: (batch, token, head, channel), seen with the heads before the tokens
        q, k, v = (randn(b, n, h, d).mul_(1.5).to(torch.bfloat16).transpose(1, 2) for h in (hq, hkv, hkv))
        at = case["seen"] + torch.arange(n, device="cuda", dtype=torch.float64)
        turn = 500000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
        angle = (at[:, None] * turn).repeat(1, 2)[None]
        return dict(case=case, q=q, k=k, v=v, cos=angle.cos().to(_type(case["angles"])),
                    sin=angle.sin().to(_type(case["angles"])), cache=_buffers(case, gen))
    s = dict(case=case, q=(randn(b, hq, case["tokens"], d) * 1.2).to(_type(case["dtype"])),
             prefix=_cache(case, gen, 1, case["prefix"]), suffix=_cache(case, gen, b, case["suffix"]), start=None)
    if case["padded"]:      # the questions are of different lengths: padding comes before them
        most = max(1, (case["suffix"] - case["tokens"]) // 2 + 1)
        s["start"] = torch.randint(0, most, (b,), device="cuda", generator=gen, dtype=torch.int32)
    return s


# ---------------------------------------------------------------------------------------------- the one pass --
def run(state):
    case = state["case"]
    if case["op"] == "append":
        return _append_own(state) if own else _append_plain(state)
    return {"out": _shared_own(state) if own else _shared_plain(state)}


def _append_own(s):
    from flashquest_amd.kernel import dequantize_cache, rotate_append
    seen, new = s["case"]["seen"], s["case"]["new"]
    q = rotate_append(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["cache"], seen)
    k, v = dequantize_cache(s["cache"], seen + new, start=seen // PAGE * PAGE)
    return {"q": q, "k": k, "v": v}


def _shared_own(s):
    from flashquest_amd.eager import shared_prefix_attention
    return shared_prefix_attention(s["q"], s["prefix"], s["suffix"], suffix_start=s["start"])


def _rotated(x, cos, sin):
    half = cos.shape[-1] // 2
    a, b = x[..., :half].float(), x[..., half:2 * half].float()
    c, s = cos[:, None].float(), sin[:, None].float()
    lo = a * c[..., :half] - b * s[..., :half]
    hi = b * c[..., half:] + a * s[..., half:]
    return torch.cat((lo, hi, x[..., 2 * half:].float()), -1).to(x.dtype)


def _values(codes, scale, mn):
    """code * scale + minimum, the metadata broadcast over the last axis's groups of channels."""
    g = codes.float().unflatten(-1, (scale.shape[-1], -1))
    return (g * scale.float()[..., None] + mn.float()[..., None]).flatten(-2)


def _key_values(codes, scale, mn):
    p = codes.unflatten(2, (-1, PAGE)).float()
    return (p * scale.float()[:, :, :, None] + mn.float()[:, :, :, None]).flatten(2, 3)


def _append_plain(s):
    case, cache = s["case"], s["cache"]
    bits, meta = case["bits"], _type(case["meta"])
    held = case["seen"] % PAGE
    q, k = _rotated(s["q"], s["cos"], s["sin"]), _rotated(s["k"], s["cos"], s["sin"])
    k = torch.cat((cache["K_partial"][:, :, :held], k), 2)
    v = torch.cat((cache["V_partial"][:, :, :held], s["v"]), 2)
    done = k.shape[2] // PAGE * PAGE
    if done:
        ks = _key_pages(k[:, :, :done], bits, meta)
        vs = _value_rows(v[:, :, :done], bits, meta, cache["V_scale"].shape[-1])
        k = torch.cat((_key_values(*ks).to(torch.bfloat16), k[:, :, done:]), 2)
        v = torch.cat((_values(*vs).to(torch.bfloat16), v[:, :, done:]), 2)
    return {"q": q, "k": k, "v": v}


def _read(c, bits):
    """A cache's keys and values in 32 bits."""
    kn, vn = _named(bits)
    k = _key_values(_unpacked(c[kn], bits), c["K_scale"], c["K_mn"])
    v = _values(_unpacked(c[vn], bits), c["V_scale"], c["V_mn"])
    return torch.cat((k, c["K_partial"].float()), 2), torch.cat((v, c["V_partial"].float()), 2)


def _shared_plain(s):
    case, q = s["case"], s["q"]
    b, hq, n, d = q.shape
    hkv = case["hkv"]
    kp, vp = _read(s["prefix"], case["bits"])
    ks, vs = _read(s["suffix"], case["bits"])
    x = q.float().reshape(b, hkv, hq // hkv * n, d)
    # the prefix: the rows of all sequences against one set of keys
    rows = x.transpose(0, 1).reshape(1, hkv, -1, d)
    sp = (rows @ kp.transpose(2, 3)).reshape(hkv, b, hq // hkv * n, -1).transpose(0, 1) / math.sqrt(d)
    ss = (x @ ks.transpose(2, 3)) / math.sqrt(d)
    j = torch.arange(case["suffix"], device=q.device)
    last = case["suffix"] - n + torch.arange(n, device=q.device)
    seen = (j <= last[:, None])[None]
    if s["start"] is not None:
        seen = seen & (j >= s["start"][:, None, None])
    ss = ss.masked_fill(~seen.repeat(1, hq // hkv, 1)[:, None], -math.inf)
    top = torch.maximum(sp.amax(-1, True), ss.amax(-1, True))
    sp, ss = (sp - top).exp(), (ss - top).exp()
    out = (sp.transpose(0, 1).reshape(1, hkv, rows.shape[2], -1) @ vp).reshape(hkv, b, -1, d).transpose(0, 1) + ss @ vs
    return (out / (sp.sum(-1, True) + ss.sum(-1, True))).reshape(b, hq, n, d).to(q.dtype)


# ------------------------------------------------------------------------------------- the bytes and the sums --
def work(case):
    b, hq, hkv, d, bits = case["batch"], case["hq"], case["hkv"], case["d"], case["bits"]
    groups = d // 32 if case["v32"] else 1
    token = 2 * d * bits / 8 + 4 * groups + 4 * d / PAGE     # a token's codes and metadata, keys and values
    if case["op"] == "append":
        n, held = case["new"], case["seen"] % PAGE
        whole = (held + n) // PAGE * PAGE
        rest = held + n - whole
        angles = 2 * n * case["rot"] * (2 if case["angles"] == "bf16" else 4)
        rows = b * n * d * 2 * (2 * hq + 2 * hkv)               # q in and out, k and v in
        held_in = 4 * d * held if whole else 0                  # the partial page that becomes whole
        put = whole * token + 4 * d * (rest if whole else n)    # into the planes and the partial page
        back = whole * token + 4 * d * rest + 4 * d * (held + n)    # and back out, as values
        return {"bytes": rows + angles + b * hkv * (held_in + put + back),
                "flops": b * n * case["rot"] * 3 * (hq + hkv) + 12 * b * hkv * whole * d}
    n, pre, suf = case["tokens"], case["prefix"], case["suffix"]
    size = lambda t: t // PAGE * PAGE * token + t % PAGE * 4 * d  # noqa: E731
    kept = suf - (max(1, (suf - n) // 2 + 1) - 1) / 2 if case["padded"] else suf
    pairs = b * hq * (n * (pre + kept) - n * (n - 1) / 2)
    return {"bytes": hkv * (size(pre) + b * size(suf) * kept / suf) + 4 * b * hq * n * d, "flops": 4 * pairs * d}


# --------------------------------------------------------------------------------------- the definition, exact --
def exact(case, seed):
    s = prepare(case, seed)

    def appended():
        """Rotation by the definition, out[i] = x[i] cos[i] + r[i] sin[i] with r = (-x2, x1), in 64 bits. The cache's
        own definition rounds: tokens to bfloat16, a key page's range and scale to bfloat16, a value's scale and the
        quotients that become codes to 32 bits (values of 16 bits often lie between two codes), metadata to its type."""
        bits, meta, rot = case["bits"], _type(case["meta"]), case["rot"]
        steps, bf = 2 ** bits - 1, torch.bfloat16

        def turned(x):
            x = x.double()
            part = x[..., :rot]
            other = torch.cat((-part[..., rot // 2:], part[..., :rot // 2]), -1)
            part = part * s["cos"].double().unsqueeze(1) + other * s["sin"].double().unsqueeze(1)
            return torch.cat((part, x[..., rot:]), -1)

        held = case["seen"] % PAGE
        q = turned(s["q"])
        k = torch.cat((s["cache"]["K_partial"][:, :, :held].double(), turned(s["k"]).to(bf).double()), 2)
        v = torch.cat((s["cache"]["V_partial"][:, :, :held].double(), s["v"].double()), 2)
        fresh = turned(s["k"])                      # waiting tokens have no rounding of their own but the result's
        n = k.shape[2] // PAGE * PAGE
        k_out, v_out = k.clone(), v.clone()
        k_out[:, :, held:] = fresh
        for p in range(0, n, PAGE):
            x = k[:, :, p:p + PAGE]
            lo, hi = x.min(2, keepdim=True).values, x.max(2, keepdim=True).values
            width = (hi - lo).to(bf).double()
            step = (width / steps).to(bf).clamp_min(EPS).double()
            codes = torch.round(((x - lo) / step).float()).clamp(0, steps).double()
            k_out[:, :, p:p + PAGE] = codes * step.to(meta).double() + lo.to(meta).double()
        g = d = v.shape[3]
        if case["v32"]:
            g = 32
        for c in range(0, d, g):
            x = v[:, :, :n, c:c + g]
            lo, hi = x.min(3, keepdim=True).values, x.max(3, keepdim=True).values
            part = torch.tensor(1 / steps, dtype=torch.float32, device=x.device).double()
            step = ((hi - lo).float().double() * part).float().clamp_min(EPS).double()
            codes = torch.round(((x - lo) / step).float()).clamp(0, steps).double()
            v_out[:, :, :n, c:c + g] = codes * step.to(meta).double() + lo.to(meta).double()
        return {"q": q, "k": k_out, "v": v_out}

    def attended():
        """Each sequence by itself: softmax(q k^T / sqrt(d)) v over the prefix's and its own tokens up to its row's."""
        q = s["q"].double()
        b, hq, n, d = q.shape
        rep, bits = hq // case["hkv"], case["bits"]

        def tokens(c, i):
            kn, vn = _named(bits)
            codes = {}
            for name in (kn, vn):
                x = c[name][i]
                if bits == 4:
                    y = torch.empty(*x.shape[:-1], 2 * x.shape[-1], dtype=torch.float64, device=x.device)
                    y[..., ::2], y[..., 1::2] = (x % 16).double(), (x // 16).double()
                    x = y
                codes[name] = x.double()
            page = torch.arange(codes[kn].shape[1], device=q.device) // PAGE
            group = torch.arange(d, device=q.device) * c["V_scale"].shape[-1] // d
            k = codes[kn] * c["K_scale"][i].double()[:, page] + c["K_mn"][i].double()[:, page]
            v = codes[vn] * c["V_scale"][i].double()[..., group] + c["V_mn"][i].double()[..., group]
            return torch.cat((k, c["K_partial"][i].double()), 1), torch.cat((v, c["V_partial"][i].double()), 1)

        kp, vp = tokens(s["prefix"], 0)
        out = torch.empty_like(q)
        row = torch.arange(n, device=q.device)[:, None]
        for i in range(b):
            ks, vs = tokens(s["suffix"], i)
            first = 0 if s["start"] is None else int(s["start"][i])
            col = torch.arange(case["suffix"], device=q.device)
            hidden = (col > case["suffix"] - n + row) | (col < first)
            for h in range(case["hkv"]):
                k, v = torch.cat((kp[h], ks[h])), torch.cat((vp[h], vs[h]))
                for r in range(h * rep, h * rep + rep):
                    score = q[i, r] @ k.T * d ** -0.5
                    score[:, case["prefix"]:][hidden] = -math.inf
                    out[i, r] = torch.softmax(score, -1) @ v
        return out

    return appended() if case["op"] == "append" else {"out": attended()}
