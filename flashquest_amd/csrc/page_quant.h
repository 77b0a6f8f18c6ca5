// One 64-token page of the INT4 / INT8 cache quantised by a workgroup of 256 threads,
// shared by the appends and the whole-tensor quantisers (cache.hip describes the
// arithmetic and what bounds it) and the append with rotated keys (rotary.hip).
#pragma once

#include "fq_common.h"

namespace fq {

namespace {

constexpr float kCacheEps = 1e-6f;                      // kv_quant.py:14
__device__ __constant__ float kCacheInv15 = 1.0f / 15.0f;
__device__ __constant__ float kCacheInv255 = 1.0f / 255.0f;    // the INT8 quantisers' "/ 255.0"

constexpr int kPage = 64;

// Positions [0, head_len) come from head, the rest from tail (position
// head_len is tail's token 0).  Element strides (b, h, t); channels contiguous.
struct TokSrc {
    const void* head; int64_t hs[3];
    const void* tail; int64_t ts[3];
    int head_len;
    int dtype;
};

struct PageQuantParams {
    TokSrc k, v;
    bool do_k, k_codes, do_v;
    int B, H, n_tok;
    int tok_dst0;                       // destination token of position 0 (a page boundary for K)
    uint8_t* kp; int64_t kp_s[3];       // (b, h, t) byte strides
    void* ks; int64_t ks_s[3];          // (b, h, page) element strides; channels contiguous
    void* km; int64_t km_s[3];
    uint8_t* vp; int64_t vp_s[3];
    void* vs; int64_t vs_s[3];          // (b, h, t); groups contiguous
    void* vm; int64_t vm_s[3];
    int v_group;
    int meta_dtype;
};

// Channels 8 c8 .. + 7 of a position as floats.  The type is a template argument:
// with a test of it per value, the page kernel waited for each load before the
// next one went out.
template <int DT>
FQ_DEV void load8(const TokSrc& s, int b, int h, int pos, int c8, float (&x)[8]) {
    const bool in_head = pos < s.head_len;
    const char* base = (const char*)(in_head ? s.head : s.tail);
    const int64_t* st = in_head ? s.hs : s.ts;
    const int t = in_head ? pos : pos - s.head_len;
    const int64_t e = b * st[0] + h * st[1] + t * st[2] + 8 * c8;
    if constexpr (DT == FQ_F32) {
        const uint4 a = *(const uint4*)(base + e * 4), c = *(const uint4*)(base + e * 4 + 16);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(w[i]);
    } else {
        const uint4 a = *(const uint4*)(base + e * 2);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = DT == FQ_BF16 ? bf16_bits_to_f(w[i] & 0xFFFFu) : f16_bits_to_f(w[i] & 0xFFFFu);
            x[2 * i + 1] = DT == FQ_BF16 ? bf16_bits_to_f(w[i] >> 16) : f16_bits_to_f(w[i] >> 16);
        }
    }
}

// A code rint(RN(d / s)) clamped to [0, 2^BITS - 1], d = x - mn, with the scale's
// reciprocal r = RN(1 / s), in the low bits of 2^23 + code (kCodeBias + code as an
// integer), which the fp32 add rounds to even as rint does.  q0 = d r is within 1.5
// ulp of d / s; one residual correction leaves an error of 2^-46 before its own
// rounding, and no quotient of two floats lies that close to a code's tie without
// being the tie (every significand of s with the 9 nearest d at each of the 255
// ties: no code differs from the division's).  That holds while nothing over- or
// underflows: quotients below 2^-100 round to 0 either way, and scales above 1e30
// (or NaN) take the division itself (quot_wide, per wave).  Scales are at least
// 1e-6.  A NaN's code is 0 (fmed3 gives the least of its other operands).
constexpr uint32_t kCodeBias = 0x4B000000u;          // 2^23
template <int BITS>
FQ_DEV uint32_t biased_code(float q) {
    return __float_as_uint(__builtin_amdgcn_fmed3f(q, 0.f, (float)((1 << BITS) - 1)) + 8388608.0f);
}
template <int BITS>
FQ_DEV uint32_t quot_code(float d, float s, float r) {
    const float q0 = d * r;
    return biased_code<BITS>(fmaf(fmaf(-q0, s, d), r, q0));
}
FQ_DEV bool quot_wide(bool ok) { return __builtin_amdgcn_ballot_w64(!ok) != 0; }   // any lane's scale out of range

// min / max over the lanes with the same (lane & 15): rows 0..3 of the wave.
template <bool MAX>
FQ_DEV float mm(float a, float b) { return MAX ? fmaxf(a, b) : fminf(a, b); }
template <bool MAX>
FQ_DEV float across_rows(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = mm<MAX>(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return mm<MAX>(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
// min / max over each run of `n` lanes (1, 2, 4, 8 or 16; uniform).
template <bool MAX>
FQ_DEV float across_run(float v, int n) {
    if (n > 1) v = mm<MAX>(v, dpp<kDppXor1>(v));
    if (n > 2) v = mm<MAX>(v, dpp<kDppXor2>(v));
    if (n > 4) v = mm<MAX>(v, dpp<kDppHalfMirror>(v));
    if (n > 8) v = mm<MAX>(v, dpp<kDppMirror>(v));
    return v;
}
constexpr int kDppRor8 = 0x128;      // lane i <- i ^ 8 within each 16

// The 8 codes (with their bias) of a thread's channels: BITS 4 packs two per byte
// (4 bytes), BITS 8 one per byte (8 bytes), at byte 8 * c8 * BITS / 8 of the row.
// The biases left of a code add up to one constant, taken off once.
template <int BITS>
FQ_DEV void store_codes(uint8_t* row, int c8, const uint32_t (&c)[8]) {
    if constexpr (BITS == 4) {
        uint32_t word = c[0] - (kCodeBias + (kCodeBias << 4));
#pragma unroll
        for (int i = 1; i < 8; ++i) word += c[i] << (4 * i);
        *(uint32_t*)(row + 4 * c8) = word;
    } else {
        uint2 w = make_uint2(c[0] - kCodeBias, c[4] - kCodeBias);
#pragma unroll
        for (int i = 1; i < 4; ++i) { w.x += c[i] << (8 * i); w.y += c[4 + i] << (8 * i); }
        *(uint2*)(row + 8 * c8) = w;
    }
}

// Page pg of batch * head bh.  DT: the type of K and V, which share it; load_k(u, pos, c8, x),
// load_v: channels 8 c8 .. + 7 of the token at a position, the thread's u-th, as floats.
// The rows of a thread are RPP apart, and a row's address is the one before it and a uniform
// step: 64-bit products per row and lane cost as much as the quantisation itself.
template <int D, int BITS, int DT, typename LoadK, typename LoadV>
FQ_DEV void quant_page(const PageQuantParams& a, int pg, int bh, LoadK load_k, LoadV load_v) {
    constexpr int CPR = D / 8;                  // threads per token row
    constexpr int RPP = kThreads / CPR;         // token rows per pass
    constexpr int TPT = kPage / RPP;            // tokens per thread
    const int tid = threadIdx.x;
    const int c8 = tid % CPR, r = tid / CPR;
    const int b = bh / a.H, h = bh % a.H;
    // a partial last page: tokens past the end re-read the last one (the same
    // page), which changes no minimum or maximum, and are not stored
    int pos[TPT], lpos[TPT];
    bool ok[TPT];
#pragma unroll
    for (int u = 0; u < TPT; ++u) {
        pos[u] = pg * kPage + r + RPP * u;
        ok[u] = pos[u] < a.n_tok;
        lpos[u] = min(pos[u], a.n_tok - 1);
    }

    if (a.do_k) {
        float x[TPT][8];
        float mn[8], mx[8];
#pragma unroll
        for (int u = 0; u < TPT; ++u) load_k(u, lpos[u], c8, x[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) { mn[i] = INFINITY; mx[i] = -INFINITY; }
#pragma unroll
        for (int u = 0; u < TPT; ++u)
#pragma unroll
            for (int i = 0; i < 8; ++i) { mn[i] = fminf(mn[i], x[u][i]); mx[i] = fmaxf(mx[i], x[u][i]); }
        // rows of this wave: lanes c8 + CPR * j
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (CPR == 8) {
                mn[i] = fminf(mn[i], dpp<kDppRor8>(mn[i]));
                mx[i] = fmaxf(mx[i], dpp<kDppRor8>(mx[i]));
            }
            mn[i] = across_rows<false>(mn[i]);
            mx[i] = across_rows<true>(mx[i]);
        }
        __shared__ float s_red[kThreads / 64][CPR][16];
        const int w = tid >> 6;
        if ((tid & 63) < CPR) {
#pragma unroll
            for (int i = 0; i < 8; ++i) { s_red[w][c8][i] = mn[i]; s_red[w][c8][8 + i] = mx[i]; }
        }
        __syncthreads();
        // one thread a channel: every row of threads doing it for its own eight was a third of the
        // vector instructions of K
        __shared__ __attribute__((aligned(16))) float s_ch[3][D];        // minimum, scale, its reciprocal
        if (tid < D) {
            float lo = INFINITY, hi = -INFINITY;
#pragma unroll
            for (int ww = 0; ww < kThreads / 64; ++ww) {
                lo = fminf(lo, s_red[ww][tid >> 3][tid & 7]);
                hi = fmaxf(hi, s_red[ww][tid >> 3][8 + (tid & 7)]);
            }
            // scale in the input dtype (kv_quant.py:131-149), as quant_k_kernel
            const float diff = round_to(hi - lo, DT);
            float sc = round_to(diff * (BITS == 8 ? kCacheInv255 : kCacheInv15), DT);
            sc = round_to(fmaxf(sc, kCacheEps), DT);
            s_ch[0][tid] = lo;
            s_ch[1][tid] = sc;
            s_ch[2][tid] = __fdiv_rn(1.0f, sc);
        }
        __syncthreads();
        float sc[8], rc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) { mn[i] = s_ch[0][8 * c8 + i]; sc[i] = s_ch[1][8 * c8 + i]; rc[i] = s_ch[2][8 * c8 + i]; }
        if (r == 0) {
            const int64_t p = a.tok_dst0 / kPage + pg;
            uint32_t sw[4], mw[4];
            auto pack = [&](auto bits) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sw[j] = bits(sc[2 * j]) | bits(sc[2 * j + 1]) << 16;
                    mw[j] = bits(mn[2 * j]) | bits(mn[2 * j + 1]) << 16;
                }
            };
            if (a.meta_dtype == FQ_BF16) pack([](float f) { return (uint32_t)f_to_bf16_bits(f); });      // uniform
            else pack([](float f) { return (uint32_t)f_to_f16_bits(f); });
            *(uint4*)((uint16_t*)a.ks + b * a.ks_s[0] + h * a.ks_s[1] + p * a.ks_s[2] + 8 * c8) =
                make_uint4(sw[0], sw[1], sw[2], sw[3]);
            *(uint4*)((uint16_t*)a.km + b * a.km_s[0] + h * a.km_s[1] + p * a.km_s[2] + 8 * c8) =
                make_uint4(mw[0], mw[1], mw[2], mw[3]);
        }
        if (a.k_codes) {
            bool fine = true;
#pragma unroll
            for (int i = 0; i < 8; ++i) fine &= sc[i] <= 1e30f;
            const bool wide = quot_wide(fine);
            uint8_t* row = a.kp + b * a.kp_s[0] + h * a.kp_s[1] + (int64_t)(a.tok_dst0 + pg * kPage + r) * a.kp_s[2];
#pragma unroll
            for (int u = 0; u < TPT; ++u) {
                uint32_t cd[8];
                if (wide) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) cd[i] = biased_code<BITS>(__fdiv_rn(x[u][i] - mn[i], sc[i]));
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) cd[i] = quot_code<BITS>(x[u][i] - mn[i], sc[i], rc[i]);
                }
                if (!ok[u]) continue;
                store_codes<BITS>(row + u * (RPP * a.kp_s[2]), c8, cd);
            }
        }
    }

    if (a.do_v) {
        const int lpg = a.v_group / 8;          // lanes per V group (a power of two <= CPR)
        const int g = (8 * c8) / a.v_group;
        const int64_t t0 = a.tok_dst0 + pg * kPage + r;
        uint8_t* row = a.vp + b * a.vp_s[0] + h * a.vp_s[1] + t0 * a.vp_s[2];
        const int64_t s0 = b * a.vs_s[0] + h * a.vs_s[1] + t0 * a.vs_s[2] + g, m0 = b * a.vm_s[0] + h * a.vm_s[1] + t0 * a.vm_s[2] + g;
        float x[TPT][8];
#pragma unroll
        for (int u = 0; u < TPT; ++u) load_v(u, lpos[u], c8, x[u]);
#pragma unroll
        for (int u = 0; u < TPT; ++u) {
            // every lane of the row takes part in the reductions; invalid tokens are not stored
            float mn = x[u][0], mx = x[u][0];
#pragma unroll
            for (int i = 1; i < 8; ++i) { mn = fminf(mn, x[u][i]); mx = fmaxf(mx, x[u][i]); }
            mn = across_run<false>(mn, lpg);
            mx = across_run<true>(mx, lpg);
            // fp32 (kv_quant.py:189-205; INT8: 78-89)
            const float s = fmaxf((mx - mn) * (BITS == 8 ? kCacheInv255 : kCacheInv15), kCacheEps);
            const float rc = __fdiv_rn(1.0f, s);
            uint32_t cd[8];
            if (quot_wide(s <= 1e30f)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) cd[i] = biased_code<BITS>(__fdiv_rn(x[u][i] - mn, s));
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) cd[i] = quot_code<BITS>(x[u][i] - mn, s, rc);
            }
            if (!ok[u]) continue;
            if (c8 % lpg == 0) {
                store_any(a.vs, a.meta_dtype, s0 + u * (RPP * a.vs_s[2]), s);
                store_any(a.vm, a.meta_dtype, m0 + u * (RPP * a.vm_s[2]), mn);
            }
            store_codes<BITS>(row + u * (RPP * a.vp_s[2]), c8, cd);
        }
    }
}

// The page arithmetic of an append: `seen` tokens were in the layer, S_new
// arrive; the stream (old tail, new tokens) completes n_complete pages
// starting at token page_tok0, and `rest` tokens stay in the tail.
struct AppendPlan {
    int partial_len, n_complete, complete_len, page_tok0, rest;
};
inline AppendPlan plan_append(int seen, int S_new, int page) {
    AppendPlan p{};
    p.partial_len = seen % page;
    p.n_complete = (p.partial_len + S_new) / page;
    p.complete_len = p.n_complete * page;
    p.page_tok0 = seen - p.partial_len;
    p.rest = p.partial_len + S_new - p.complete_len;
    return p;
}

// Token sources of the stream: the layer's tail rows, then the new tokens.
inline TokSrc stream_src(const void* part, const int64_t* part_s, int64_t layer, const void* fresh, const int64_t* fresh_s,
                  int partial_len, int dtype) {
    return TokSrc{(const char*)part + layer * part_s[0] * 2, {part_s[1], part_s[2], part_s[3]}, fresh,
                  {fresh_s[0], fresh_s[1], fresh_s[2]}, partial_len, dtype};
}

}  // namespace
}  // namespace fq
