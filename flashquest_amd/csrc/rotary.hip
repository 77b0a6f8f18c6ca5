// The append of a step's keys and values to one layer's INT4 / INT8 cache with the rotary
// position embedding applied on the way, and the step's queries rotated with it, in one
// launch; and the read of a cache's tokens back as values.
//
// Rotation of a row x by the cos / sin rows c, s of its position (R rotated channels, the
// halves paired as transformers' rotate_half does; src/flashquest/eager/
// llama_persistent_patch.py:186-194 applies it before update_quantized):
//   y[i] = x[i] c[i] - x[i + R/2] s[i],   y[i + R/2] = x[i + R/2] c[i + R/2] + x[i] s[i + R/2]
// for i < R/2, the channels from R on unchanged.  Products and sum are rounded to fp32 one
// by one (no contraction), the result once to the tokens' type: those are the tokens the
// cache holds, so pages, metadata and tail are bit-identical to rotating first and
// appending with update_quantized.
//
// Three kinds of workgroups by block index:
//   pages  one per (completed page, batch * KV head): quant_page with rotated keys.  The
//          workgroup of a head's first page is the only reader of the head's old partial
//          page, so after its last load it also stages what stays in the partial page.
//   rows   without a completed page, the new rows of K (rotated) and V to the partial page.
//   q      the query rows.
// All are bound by memory: every input is read once and every output written once, the angles
// by every head, for which the heads of a page or of a chunk of query rows run on one XCD (from
// its L2: 5 % of a long prompt).  A thread turns
// its query unit for 4 heads with one load of the angles; a short step, which would not fill the
// GPU so, for one (2^19 units: 8 waves a SIMD).  32768 tokens of 24 query and 8 KV heads of 128
// channels to an empty INT4 cache: 139 us for 0.61 GB (4.4 TB/s; a copy 5.2), of which the query
// rows run at 5.3; the pages' vector instructions, half of the time, are what keeps them below.
// One token: 3 us, the launch.
#include "fq_common.h"
#include "page_quant.h"

namespace fq {
namespace {

struct Rotary {
    const void* cos; int64_t cs[2];      // (b, t) element strides; channels contiguous
    const void* sin; int64_t ss[2];
    int R;                               // rotated channels, a multiple of 16, at most D
};

// 8 consecutive values of a type as floats.
template <int DT>
FQ_DEV void ld8(const void* p, int64_t e, float (&x)[8]) {
    if constexpr (DT == FQ_F32) {
        const uint4 a = *(const uint4*)((const char*)p + e * 4), c = *(const uint4*)((const char*)p + e * 4 + 16);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
        const uint4 a = *(const uint4*)((const char*)p + e * 2);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = DT == FQ_BF16 ? bf16_bits_to_f(w[i] & 0xFFFFu) : f16_bits_to_f(w[i] & 0xFFFFu);
            x[2 * i + 1] = DT == FQ_BF16 ? bf16_bits_to_f(w[i] >> 16) : f16_bits_to_f(w[i] >> 16);
        }
    }
}
template <int DT>
FQ_DEV void st8(void* p, int64_t e, const float (&x)[8]) {
    uint32_t w[4];
    if constexpr (DT == FQ_BF16) {
        // the conversion instruction, of two values at once: it agrees with f_to_bf16_bits on every
        // float but NaNs, whose payload it keeps
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        bool nan = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[i] = __builtin_bit_cast(uint32_t, bf2{(__bf16)x[2 * i], (__bf16)x[2 * i + 1]});
            nan |= __builtin_isunordered(x[2 * i], x[2 * i + 1]);
        }
        if (__builtin_amdgcn_ballot_w64(nan)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (uint32_t)f_to_bf16_bits(x[2 * i]) | (uint32_t)f_to_bf16_bits(x[2 * i + 1]) << 16;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)f_to_f16_bits(x[2 * i]) | (uint32_t)f_to_f16_bits(x[2 * i + 1]) << 16;
    }
    *(uint4*)((char*)p + e * 2) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows (b, h, t) of `src` to `dst`, rotated or not.  16-byte chunks; channels contiguous.
struct Rows {
    const void* src; int64_t ss[3];
    void* dst; int64_t ds[3];
    int H, n;                            // heads, tokens: src tokens src_t0 .., dst tokens dst_t0 ..
    int src_t0, dst_t0;
    int zero;                            // dst tokens after them that are set to 0
};

// The unit of a rotated row: channels 8u .. 8u + 7 and their partners R/2 further, or, past
// the R/16 rotated units, 16 unrotated channels from R on.
template <int DT>
FQ_DEV void unit_channels(const Rotary& r, int u, int& lo, int& hi) {
    const int nr = r.R >> 4;
    lo = u < nr ? 8 * u : r.R + 16 * (u - nr);
    hi = u < nr ? lo + (r.R >> 1) : lo + 8;
}

template <int CT>
struct Angles { float cl[8], ch[8], sl[8], sh[8]; };
template <int CT>
FQ_DEV void load_angles(const Rotary& r, int b, int t, int lo, int hi, Angles<CT>& a) {
    const int64_t c = b * r.cs[0] + t * r.cs[1], s = b * r.ss[0] + t * r.ss[1];
    ld8<CT>(r.cos, c + lo, a.cl);
    ld8<CT>(r.cos, c + hi, a.ch);
    ld8<CT>(r.sin, s + lo, a.sl);
    ld8<CT>(r.sin, s + hi, a.sh);
}
template <int CT>
FQ_DEV void rotate_pair(float (&x)[8], float (&y)[8], const Angles<CT>& a) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float p = x[i], q = y[i];
        x[i] = p * a.cl[i] - q * a.sl[i];
        y[i] = q * a.ch[i] + p * a.sh[i];
    }
}

// Blocks whose tokens share angles go to one XCD, one after another, so that its L2 has them: block
// ids go round the 8 XCDs, so items (heads) of chunk c get ids that are c modulo 8.
constexpr int kXcd = 8;
FQ_DEV void by_xcd(int64_t blk, int items, int& chunk, int& item) {
    const uint32_t local = (uint32_t)(blk / kXcd);
    chunk = (int)(local / items) * kXcd + (int)(blk % kXcd);
    item = (int)(local % items);
}
int64_t xcd_blocks(int64_t chunks, int64_t items) { return (chunks + kXcd - 1) / kXcd * kXcd * items; }

// One thread's share of Rows: unit u of token t (of n) for HPT heads from h0 on, rotated, all loads
// before the first store.
template <int DT, int CT, int HPT>
FQ_DEV void turn_heads(const Rows& w, const Rotary& r, int b, int t, int u, int h0) {
    int lo, hi;
    unit_channels<DT>(r, u, lo, hi);
    const bool turn = u < (r.R >> 4);
    Angles<CT> ang;
    if (turn) load_angles<CT>(r, b, w.src_t0 + t, lo, hi, ang);
    const uint16_t* in = (const uint16_t*)w.src + b * w.ss[0] + (int64_t)(w.src_t0 + t) * w.ss[2];
    uint16_t* out = (uint16_t*)w.dst + b * w.ds[0] + (int64_t)(w.dst_t0 + t) * w.ds[2];
    uint4 x[HPT], y[HPT];
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
        const uint16_t* p = in + min(h0 + i, w.H - 1) * w.ss[1];
        x[i] = *(const uint4*)(p + lo);
        y[i] = *(const uint4*)(p + hi);
    }
#pragma unroll
    for (int i = 0; i < HPT; ++i) {
        if (h0 + i >= w.H) break;
        uint16_t* p = out + (h0 + i) * w.ds[1];
        if (turn) {
            float xf[8], yf[8];
            ld8<DT>(&x[i], 0, xf);
            ld8<DT>(&y[i], 0, yf);
            rotate_pair<CT>(xf, yf, ang);
            st8<DT>(p, lo, xf);
            st8<DT>(p, hi, yf);
        } else {
            *(uint4*)(p + lo) = x[i];
            *(uint4*)(p + hi) = y[i];
        }
    }
}

// One thread's share of Rows: unit u of token t (of n + zero) for heads h0 .. h1 - 1.
template <int DT, int CT, bool ROT>
FQ_DEV void do_rows(const Rows& w, const Rotary& r, int b, int t, int u, int h0, int h1) {
    int lo = 16 * u, hi = lo + 8;
    if (ROT) unit_channels<DT>(r, u, lo, hi);
    const bool turn = ROT && u < (r.R >> 4) && t < w.n;
    Angles<CT> ang;
    if (turn) load_angles<CT>(r, b, w.src_t0 + t, lo, hi, ang);
    for (int h = h0; h < h1; ++h) {
        const int64_t s = b * w.ss[0] + h * w.ss[1] + (int64_t)(w.src_t0 + t) * w.ss[2];
        const int64_t d = b * w.ds[0] + h * w.ds[1] + (int64_t)(w.dst_t0 + t) * w.ds[2];
        uint16_t* out = (uint16_t*)w.dst;
        if (t >= w.n) {
            *(uint4*)(out + d + lo) = make_uint4(0u, 0u, 0u, 0u);
            *(uint4*)(out + d + hi) = make_uint4(0u, 0u, 0u, 0u);
        } else if (turn) {
            float x[8], y[8];
            ld8<DT>(w.src, s + lo, x);
            ld8<DT>(w.src, s + hi, y);
            rotate_pair<CT>(x, y, ang);
            st8<DT>(w.dst, d + lo, x);
            st8<DT>(w.dst, d + hi, y);
        } else {
            const uint16_t* in = (const uint16_t*)w.src;
            const uint4 x = *(const uint4*)(in + s + lo), y = *(const uint4*)(in + s + hi);
            *(uint4*)(out + d + lo) = x;
            *(uint4*)(out + d + hi) = y;
        }
    }
}

// Threads of a Rows: (b, group of `hpt` heads, token, unit), units fastest.
// chunks > 0 (many tokens, rotated, none set to 0): a block per (chunk of tokens, batch, group of 4
// heads) instead, placed by by_xcd.
struct RowGrid { int hpt, groups; int64_t threads; int chunks; };
RowGrid row_grid(const Rows& w, int B, int D, int hpt) {
    RowGrid g{hpt, (w.H + hpt - 1) / hpt, 0, 0};
    g.threads = (int64_t)B * g.groups * (w.n + w.zero) * (D / 16);
    return g;
}
template <int D, int DT, int CT, bool ROT>
FQ_DEV void rows_block(const Rows& w, const Rotary& r, const RowGrid& g, int64_t block) {
    if constexpr (ROT) {
        if (g.chunks > 0) {
            constexpr int TPB = kThreads / (D / 16);     // tokens of a block
            int chunk, item;
            by_xcd(block, (int)g.threads, chunk, item);
            const int t = chunk * TPB + threadIdx.x / (D / 16);
            if (t < w.n) turn_heads<DT, CT, 4>(w, r, item / g.groups, t, threadIdx.x % (D / 16), item % g.groups * 4);
            return;
        }
    }
    const int64_t i = block * kThreads + threadIdx.x;
    if (i >= g.threads) return;
    const int u = (int)(i % (D / 16));
    const int64_t j = i / (D / 16);
    const int t = (int)(j % (w.n + w.zero));
    const int64_t k = j / (w.n + w.zero);
    const int hg = (int)(k % g.groups), b = (int)(k / g.groups);
    do_rows<DT, CT, ROT>(w, r, b, t, u, hg * g.hpt, min(hg * g.hpt + g.hpt, w.H));
}

struct RotAppendParams {
    PageQuantParams pq;                  // pq.n_tok: tokens of the completed pages (0: none)
    Rotary r;
    Rows q, k, v;                        // k, v: what goes to the partial page
    RowGrid gq, gk, gv;
    int64_t page_blocks, k_blocks, v_blocks;    // then the query blocks
    int pages;
};

// Channels 8 c8 .. + 7 of a key of the stream, as load8, the new tokens rotated and rounded.
template <int DT, int CT>
FQ_DEV void load8_rotated(const TokSrc& s, const Rotary& r, int b, int h, int pos, int c8, float (&x)[8]) {
    const bool in_head = pos < s.head_len;
    const void* base = in_head ? s.head : s.tail;
    const int64_t* st = in_head ? s.hs : s.ts;
    const int t = in_head ? pos : pos - s.head_len;
    const int64_t e = b * st[0] + h * st[1] + t * st[2];
    const int ch = 8 * c8, half = r.R >> 1;
    const bool turn = !in_head && ch < r.R;
    const bool low = ch < half;
    // every load is unconditional: unrotated channels read themselves and channel 0's angles
    const int other = turn ? (low ? ch + half : ch - half) : ch;
    const int at = turn ? ch : 0, ta = in_head ? 0 : t;
    float y[8], c[8], sn[8];
    ld8<DT>(base, e + ch, x);
    ld8<DT>(base, e + other, y);
    ld8<CT>(r.cos, b * r.cs[0] + ta * r.cs[1] + at, c);
    ld8<CT>(r.sin, b * r.ss[0] + ta * r.ss[1] + at, sn);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float p = x[i] * c[i], q = y[i] * sn[i];
        const float v = low ? p - q : p + q;
        x[i] = turn ? round_to(v, DT) : x[i];
    }
}

// A page of new tokens only: the thread's rows at a pointer and uniform steps.
template <int D, int DT, int CT>
struct FreshPage {
    static constexpr int RPP = kThreads / (D / 8);       // rows between a thread's
    const uint16_t *k, *v;               // the thread's first row, its channels
    const void *cos, *sin;
    int64_t ce, se;                      // element offsets of its first row's angles
    int other;                           // channels to the partners
    bool turn;
    uint32_t flip;                       // sign bits of the partners' products

    FQ_DEV FreshPage(const RotAppendParams& a, int pg, int b, int h) {
        const TokSrc &ks = a.pq.k, &vs = a.pq.v;
        const int c8 = threadIdx.x % (D / 8), t = pg * kPage - ks.head_len + threadIdx.x / (D / 8), ch = 8 * c8, half = a.r.R >> 1;
        k = (const uint16_t*)ks.tail + b * ks.ts[0] + h * ks.ts[1] + t * ks.ts[2] + ch;
        v = (const uint16_t*)vs.tail + b * vs.ts[0] + h * vs.ts[1] + t * vs.ts[2] + ch;
        turn = ch < a.r.R;
        other = turn ? (ch < half ? half : -half) : 0;
        flip = ch < half ? 0x80008000u : 0u;
        cos = a.r.cos; sin = a.r.sin;
        ce = b * a.r.cs[0] + t * a.r.cs[1] + (turn ? ch : 0);        // (unrotated channels: loads without a use)
        se = b * a.r.ss[0] + t * a.r.ss[1] + (turn ? ch : 0);
    }
    FQ_DEV void key(const RotAppendParams& a, int u, float (&x)[8]) const {
        const uint16_t* p = k + u * (RPP * a.pq.k.ts[2]);
        uint4 y4 = *(const uint4*)(p + other);
        float y[8], c[8], s[8];
        ld8<DT>(p, 0, x);
        ld8<CT>(cos, ce + u * (RPP * a.r.cs[1]), c);
        ld8<CT>(sin, se + u * (RPP * a.r.ss[1]), s);
        y4 = make_uint4(y4.x ^ flip, y4.y ^ flip, y4.z ^ flip, y4.w ^ flip);
        ld8<DT>(&y4, 0, y);
        if (!turn) return;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float z = x[i] * c[i] + y[i] * s[i];
            x[i] = DT == FQ_BF16 ? (float)(__bf16)z : (float)(_Float16)z;    // (a NaN stays one)
        }
    }
    FQ_DEV void value(const RotAppendParams& a, int u, float (&x)[8]) const { ld8<DT>(v + u * (RPP * a.pq.v.ts[2]), 0, x); }
};

template <int D, int BITS, int DT, int CT>
__global__ __launch_bounds__(kThreads) void rotate_append_kernel(RotAppendParams a) {
    int64_t blk = blockIdx.x;
    if (blk < a.page_blocks) {
        int pg, bh;
        by_xcd(blk, a.pq.B * a.pq.H, pg, bh);
        if (pg >= a.pages) return;
        const int b = bh / a.pq.H, h = bh % a.pq.H;
        if (pg > 0 || a.pq.k.head_len == 0) {            // no token of the partial page
            const FreshPage<D, DT, CT> f(a, pg, b, h);
            quant_page<D, BITS, DT>(a.pq, pg, bh, [&](int u, int, int, float (&x)[8]) { f.key(a, u, x); },
                                    [&](int u, int, int, float (&x)[8]) { f.value(a, u, x); });
        } else {
            quant_page<D, BITS, DT>(a.pq, pg, bh, [&](int, int pos, int c8, float (&x)[8]) {
                load8_rotated<DT, CT>(a.pq.k, a.r, b, h, pos, c8, x);
            }, [&](int, int pos, int c8, float (&x)[8]) { load8<DT>(a.pq.v, b, h, pos, c8, x); });
        }
        if (pg == 0 && a.k.n + a.k.zero > 0) {
            __syncthreads();             // every thread has its rows of the old partial page
            const int units = D / 16, rows = a.k.n + a.k.zero;
            for (int i = threadIdx.x; i < rows * units; i += kThreads) {
                do_rows<DT, CT, true>(a.k, a.r, b, i / units, i % units, h, h + 1);
                do_rows<DT, CT, false>(a.v, a.r, b, i / units, i % units, h, h + 1);
            }
        }
        return;
    }
    blk -= a.page_blocks;
    if (blk < a.k_blocks) return rows_block<D, DT, CT, true>(a.k, a.r, a.gk, blk);
    blk -= a.k_blocks;
    if (blk < a.v_blocks) return rows_block<D, DT, CT, false>(a.v, a.r, a.gv, blk);
    rows_block<D, DT, CT, true>(a.q, a.r, a.gq, blk - a.v_blocks);
}

// Rows of two tensors rotated (fq_rotate).
struct RotateParams {
    Rotary r;
    Rows x[2];
    RowGrid g[2];
    int64_t blocks0;
};
template <int D, int DT, int CT>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotateParams a) {
    const int64_t blk = blockIdx.x;
    if (blk < a.blocks0) rows_block<D, DT, CT, true>(a.x[0], a.r, a.g[0], blk);
    else rows_block<D, DT, CT, true>(a.x[1], a.r, a.g[1], blk - a.blocks0);
}

// Tokens [start, S + tail) of a cache as values: code * scale + min in fp32 (an exact product,
// one rounding), rounded to bf16 (dequantize_k_int4 / dequantize_v_int4, kv_quant.py:174-215;
// dequantize_k / dequantize_v, 64-97), the partial page's rows as they are.  One workgroup
// per (page, batch * head) and one thread per 8 channels, as quant_page: bound by the bytes,
// 32768 tokens of 8 heads of 128 channels in INT4 31 us (0.17 GB, 5.5 TB/s).
struct DequantParams {
    Int4Cache c;
    TailArgs t;                          // 16-bit rows of the outputs' type (bf16)
    uint16_t* k; int64_t k_s[3];         // (b, h, t) element strides
    uint16_t* v; int64_t v_s[3];
    int start, page0;
};

template <int BITS>
FQ_DEV void codes8(const uint8_t* p, float (&x)[8]) {
    if constexpr (BITS == 4) {
        const uint32_t w = *(const uint32_t*)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)((w >> (4 * i)) & 15u);
    } else {
        const uint2 w = *(const uint2*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) { x[i] = (float)((w.x >> (8 * i)) & 255u); x[4 + i] = (float)((w.y >> (8 * i)) & 255u); }
    }
}

template <int D, int BITS, int META>
__global__ __launch_bounds__(kThreads) void dequant_cache_kernel(DequantParams a) {
    constexpr int CPR = D / 8, RPP = kThreads / CPR, TPT = kPage / RPP;
    const Int4Cache& c = a.c;
    const int c8 = threadIdx.x % CPR, r = threadIdx.x / CPR;
    const int b = blockIdx.y / c.Hkv, h = blockIdx.y % c.Hkv;
    const int pg = a.page0 + blockIdx.x;
    if (pg * kPage >= c.S) {             // the partial page
#pragma unroll
        for (int u = 0; u < TPT; ++u) {
            const int i = r + RPP * u;
            const int64_t o = (int64_t)c.S + i - a.start;
            if (i >= a.t.len || o < 0) continue;
            *(uint4*)(a.k + b * a.k_s[0] + h * a.k_s[1] + o * a.k_s[2] + 8 * c8) =
                *(const uint4*)((const uint16_t*)a.t.k + b * a.t.ks[1] + h * a.t.ks[2] + i * a.t.ks[3] + 8 * c8);
            *(uint4*)(a.v + b * a.v_s[0] + h * a.v_s[1] + o * a.v_s[2] + 8 * c8) =
                *(const uint4*)((const uint16_t*)a.t.v + b * a.t.vs[1] + h * a.t.vs[2] + i * a.t.vs[3] + 8 * c8);
        }
        return;
    }
    float sc[8], mn[8];
    ld8<META>(c.ksc, b * c.ksc_s[1] + h * c.ksc_s[2] + pg * c.ksc_s[3] + 8 * c8, sc);
    ld8<META>(c.kmn, b * c.kmn_s[1] + h * c.kmn_s[2] + pg * c.kmn_s[3] + 8 * c8, mn);
    const uint8_t* kr = c.kp + b * c.kp_s[1] + h * c.kp_s[2] + c8 * BITS;
    const uint8_t* vr = c.vp + b * c.vp_s[1] + h * c.vp_s[2] + c8 * BITS;
    const int64_t vs = b * c.vsc_s[1] + h * c.vsc_s[2], vm = b * c.vmn_s[1] + h * c.vmn_s[2];
    const int g = c.G == 1 ? 0 : c8 >> 2;
#pragma unroll
    for (int u = 0; u < TPT; ++u) {
        const int64_t t = (int64_t)pg * kPage + r + RPP * u, o = t - a.start;
        if (o < 0) continue;
        float kx[8], vx[8];
        codes8<BITS>(kr + t * c.kp_s[3], kx);
        codes8<BITS>(vr + t * c.vp_s[3], vx);
        const float s = half_to_f<std::conditional_t<META == FQ_BF16, bf16, f16>>(((const uint16_t*)c.vsc)[vs + t * c.vsc_s[3] + g]);
        const float m = half_to_f<std::conditional_t<META == FQ_BF16, bf16, f16>>(((const uint16_t*)c.vmn)[vm + t * c.vmn_s[3] + g]);
#pragma unroll
        for (int i = 0; i < 8; ++i) { kx[i] = fmaf(kx[i], sc[i], mn[i]); vx[i] = fmaf(vx[i], s, m); }
        st8<FQ_BF16>(a.k, b * a.k_s[0] + h * a.k_s[1] + o * a.k_s[2] + 8 * c8, kx);
        st8<FQ_BF16>(a.v, b * a.v_s[0] + h * a.v_s[1] + o * a.v_s[2] + 8 * c8, vx);
    }
}

// Heads a thread rotates with one load of its angles: 4 once one head a thread gives more
// waves than the GPU holds, so that short steps keep every lane busy.
RowGrid rotated_grid(const Rows& w, int B, int D) {
    const bool many = (int64_t)B * w.H * w.n * (D / 16) >= (1 << 19);
    RowGrid g = row_grid(w, B, D, many ? 4 : 1);
    if (many) {
        g.chunks = (w.n + kThreads / (D / 16) - 1) / (kThreads / (D / 16));
        g.threads = (int64_t)B * g.groups;       // items of a chunk
    }
    return g;
}

Rotary rotary_of(const fq_rotary& f) {
    Rotary r{};
    r.cos = f.cos; r.sin = f.sin;
    for (int i = 0; i < 2; ++i) { r.cs[i] = f.cos_strides[i]; r.ss[i] = f.sin_strides[i]; }
    r.R = f.R;
    return r;
}

int64_t blocks_of(const RowGrid& g) { return g.chunks > 0 ? xcd_blocks(g.chunks, g.threads) : (g.threads + kThreads - 1) / kThreads; }

template <typename F>
hipError_t by_type(int D, int dt, int ct, F f) {
#define FQ_T(D_, DT_, CT_) \
    if (D == D_ && dt == DT_ && ct == CT_) return f(std::integral_constant<int, D_>(), std::integral_constant<int, DT_>(), std::integral_constant<int, CT_>());
    FQ_T(128, FQ_BF16, FQ_BF16) FQ_T(128, FQ_BF16, FQ_F32) FQ_T(128, FQ_F16, FQ_F16) FQ_T(128, FQ_F16, FQ_F32)
    FQ_T(64, FQ_BF16, FQ_BF16) FQ_T(64, FQ_BF16, FQ_F32) FQ_T(64, FQ_F16, FQ_F16) FQ_T(64, FQ_F16, FQ_F32)
#undef FQ_T
    return hipErrorInvalidValue;
}

}  // namespace

// The append of S_new tokens to one layer (kv: partial page and new tokens as launch_kv_append
// takes them) with the keys and the queries of `f` rotated.
hipError_t launch_rotate_append(const Int4Cache& c, int layer, void* kpart, const int64_t* kpart_s, void* vpart,
                                const int64_t* vpart_s, int dtype, const void* knew, const int64_t* kn_s,
                                const void* vnew, const int64_t* vn_s, int seen, int S_new, const fq_rotary& f,
                                hipStream_t st) {
    const AppendPlan pl = plan_append(seen, S_new, c.page);
    const int64_t l = layer;
    RotAppendParams a{};
    a.r = rotary_of(f);
    a.pages = pl.n_complete;
    a.page_blocks = xcd_blocks(pl.n_complete, (int64_t)c.B * c.Hkv);
    if (pl.n_complete > 0) {
        PageQuantParams& p = a.pq;
        p.k = stream_src(kpart, kpart_s, l, knew, kn_s, pl.partial_len, dtype);
        p.v = stream_src(vpart, vpart_s, l, vnew, vn_s, pl.partial_len, dtype);
        p.do_k = true; p.k_codes = true; p.do_v = true;
        p.n_tok = pl.complete_len; p.tok_dst0 = pl.page_tok0;
        p.kp = (uint8_t*)c.kp + l * c.kp_s[0];
        p.vp = (uint8_t*)c.vp + l * c.vp_s[0];
        p.ks = (uint16_t*)c.ksc + l * c.ksc_s[0];
        p.km = (uint16_t*)c.kmn + l * c.kmn_s[0];
        p.vs = (uint16_t*)c.vsc + l * c.vsc_s[0];
        p.vm = (uint16_t*)c.vmn + l * c.vmn_s[0];
        for (int i = 0; i < 3; ++i) {
            p.kp_s[i] = c.kp_s[i + 1]; p.vp_s[i] = c.vp_s[i + 1];
            p.ks_s[i] = c.ksc_s[i + 1]; p.km_s[i] = c.kmn_s[i + 1];
            p.vs_s[i] = c.vsc_s[i + 1]; p.vm_s[i] = c.vmn_s[i + 1];
        }
        p.v_group = c.D / c.G;
        p.meta_dtype = c.meta_dtype;
    }
    a.pq.B = c.B; a.pq.H = c.Hkv;
    const bool done = pl.n_complete > 0;
    const int n = done ? pl.rest : S_new, dst0 = done ? 0 : pl.partial_len;
    auto part = [&](const void* src, const int64_t* ss, void* dst, const int64_t* ds) {
        Rows w{};
        w.src = src; w.dst = (char*)dst + l * ds[0] * 2;
        for (int i = 0; i < 3; ++i) { w.ss[i] = ss[i]; w.ds[i] = ds[i + 1]; }
        w.H = c.Hkv; w.n = n;
        w.src_t0 = done ? S_new - pl.rest : 0; w.dst_t0 = dst0;
        w.zero = c.bits == 8 ? c.page - (dst0 + n) : 0;      // as the INT8 cache keeps the rows after its tail
        return w;
    };
    a.k = part(knew, kn_s, kpart, kpart_s);
    a.v = part(vnew, vn_s, vpart, vpart_s);
    Rows& q = a.q;
    q.src = f.q; q.dst = f.q_out;
    for (int i = 0; i < 3; ++i) { q.ss[i] = f.q_strides[i]; q.ds[i] = f.qo_strides[i]; }
    q.H = f.H_q; q.n = S_new;
    a.gk = row_grid(a.k, c.B, c.D, 1);
    a.gv = row_grid(a.v, c.B, c.D, 1);
    a.gq = rotated_grid(q, c.B, c.D);
    a.k_blocks = done ? 0 : blocks_of(a.gk);
    a.v_blocks = done ? 0 : blocks_of(a.gv);
    const int64_t blocks = a.page_blocks + a.k_blocks + a.v_blocks + blocks_of(a.gq);
    if (blocks == 0) return hipSuccess;
    if (blocks * kThreads > 0xFFFFFFFFll) return hipErrorInvalidValue;
    return by_type(c.D, dtype, f.dtype, [&](auto D, auto DT, auto CT) {
        if (c.bits == 8) hipLaunchKernelGGL((rotate_append_kernel<D(), 8, DT(), CT()>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
        else hipLaunchKernelGGL((rotate_append_kernel<D(), 4, DT(), CT()>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
        return hipGetLastError();
    });
}

// Queries of `f` and keys k -> k_out rotated, (B, H, S, D) each.
hipError_t launch_rotate(const fq_rotary& f, const void* k, const int64_t* k_s, void* k_out, const int64_t* ko_s,
                         int dtype, int B, int H_kv, int S, int D, hipStream_t st) {
    RotateParams a{};
    a.r = rotary_of(f);
    auto rows = [&](const void* src, const int64_t* ss, void* dst, const int64_t* ds, int H) {
        Rows w{};
        w.src = src; w.dst = dst; w.H = H; w.n = S;
        for (int i = 0; i < 3; ++i) { w.ss[i] = ss[i]; w.ds[i] = ds[i]; }
        return w;
    };
    a.x[0] = rows(f.q, f.q_strides, f.q_out, f.qo_strides, f.H_q);
    a.x[1] = rows(k, k_s, k_out, ko_s, H_kv);
    for (int i = 0; i < 2; ++i) a.g[i] = rotated_grid(a.x[i], B, D);
    a.blocks0 = blocks_of(a.g[0]);
    const int64_t blocks = a.blocks0 + blocks_of(a.g[1]);
    if (blocks == 0) return hipSuccess;
    if (blocks * kThreads > 0xFFFFFFFFll) return hipErrorInvalidValue;
    return by_type(D, dtype, f.dtype, [&](auto D_, auto DT, auto CT) {
        hipLaunchKernelGGL((rotate_kernel<D_(), DT(), CT()>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a);
        return hipGetLastError();
    });
}

// Tokens [start, c.S + t.len) of one layer's cache to k / v (bf16, element strides b, h, t).
hipError_t launch_dequant_cache(const Int4Cache& c, const TailArgs& t, int start, void* k, const int64_t* k_s,
                                void* v, const int64_t* v_s, hipStream_t st) {
    DequantParams a{};
    a.c = c; a.t = t; a.start = start; a.page0 = start / kPage;
    a.k = (uint16_t*)k; a.v = (uint16_t*)v;
    for (int i = 0; i < 3; ++i) { a.k_s[i] = k_s[i]; a.v_s[i] = v_s[i]; }
    const int pages = (c.S + t.len + kPage - 1) / kPage - a.page0;
    if (pages <= 0 || c.B * c.Hkv == 0) return hipSuccess;
    const dim3 grid(pages, c.B * c.Hkv);
    const bool bf = c.meta_dtype == FQ_BF16;
#define FQ_DQ(D_, BITS_)                                                                                               \
    if (c.D == D_ && c.bits == BITS_) {                                                                                \
        if (bf) hipLaunchKernelGGL((dequant_cache_kernel<D_, BITS_, FQ_BF16>), grid, dim3(kThreads), 0, st, a);        \
        else hipLaunchKernelGGL((dequant_cache_kernel<D_, BITS_, FQ_F16>), grid, dim3(kThreads), 0, st, a);            \
        return hipGetLastError();                                                                                      \
    }
    FQ_DQ(128, 4) FQ_DQ(64, 4) FQ_DQ(128, 8) FQ_DQ(64, 8)
#undef FQ_DQ
    return hipErrorInvalidValue;
}

}  // namespace fq
