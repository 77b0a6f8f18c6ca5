// Attention of a batch whose sequences share a prefix, over the packed INT4 / INT8 caches:
// the prefix is one cache (batch 1) that is read once for all sequences, the tokens that each
// sequence has of its own are another (batch B).
//
//   O = softmax([q Kp^T, q Ks^T + mask] sm_scale) [Vp; Vs]
//
// per sequence b, query head and query token i of S_q: all of the prefix's tokens, and the
// suffix's tokens start[b] <= j <= S_suffix - S_q + i (the S_q query tokens are the suffix's
// last).  Keys and values are code * scale + min of the pages, then the bf16 rows of the
// partial page, for prefix and suffix alike.
//
// The softmax over both parts is one: each workgroup keeps a running maximum, sum and output
// over its share of one part's keys, and shared_merge_kernel joins the shares,
//   m = max m_i, l = sum 2^(m_i - m) l_i, O = sum 2^(m_i - m) O_i / l.
//
// Rows.  Every (sequence, token, query head of the KV head's group) is a row of the prefix's
// products: B S_q G rows against one set of keys, so a page that was loaded and turned into
// operands serves all rows of a tile.  The suffix's rows are one sequence's S_q G.
//
// A wave takes 16 QB rows and every fourth page of its workgroup's range:
//   S^T = K Q^T     v_mfma_f32_16x16x32_f16, keys as the A operand
//   O^T += V^T P^T  the same, channels as the A operand
// The transposed products keep a row on one lane column: its statistics are per lane, and P
// leaves S^T's accumulator as the B operand of the second product.
//
// Operands are fp16, whose 11 bits leave errors below those of 16-bit outputs (bf16's 8 do
// not): q exact after a power of two per row (16-bit inputs), K and V one rounding of
// code * scale + min, K times 2^-6 (|K| up to 2e6 stays finite, |V| up to 3e4; K is exact to
// 2^-19, V to 2^-25, where they are small), P times 2^7 (exact to 2^-32 of a row's largest
// weight where it is small).  Sums, maxima and outputs are fp32.
#include <algorithm>
#include <type_traits>

#include "fq_common.h"

namespace fq {
namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kPg = 64;                  // tokens of a page
constexpr int kW = 4;                    // waves of a workgroup
constexpr float kLazy = 8.0f;            // the reference moves when a maximum exceeds it by 2^8
constexpr float kPShift = 7.0f;          // P is kept times 2^7
constexpr float kKExp = 0x1p-6f;         // K is kept times 2^-6

// One part of the keys: the prefix (one item) or the suffixes (an item per sequence).
struct SharedPart {
    Int4Cache c;
    TailArgs t;
    int keys;                            // c.S + t.len
    int rows;                            // rows of an item and KV head
    int items, tiles, splits;            // sequences, row tiles, key splits
    int pages, per_split;                // pages (the partial one last), pages of a split
    int64_t wgs;                         // items * Hkv * tiles * splits
    float* part;                         // [item][kv head][split][row]: D sums, then all (m, l)
};

struct SharedParams {
    SharedPart p[2];
    int first;                           // parts of this launch: [first, last]
    int last;
    const void* q; int64_t q_s[3];       // (b, h, i) element strides, channels contiguous
    void* out; int64_t o_s[3];
    float* lse; int64_t lse_s[3];
    const int32_t* start;
    int bf16;
    int B, Hq, Hkv, G, Sq;
    float qk_scale;                      // sm_scale * log2(e)
};

template <typename MT> FQ_DEV float meta_f(uint32_t bits) { return half_to_f<MT>(bits); }
FQ_DEV uint32_t h2_bits(h2 x) { return __builtin_bit_cast(uint32_t, x); }
FQ_DEV h2 bits_h2(uint32_t x) { return __builtin_bit_cast(h2, x); }
FQ_DEV uint32_t pack_h2(float a, float b) { return h2_bits(h2{(_Float16)a, (_Float16)b}); }
FQ_DEV v8h frag(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { return __builtin_bit_cast(v8h, u32x4{a, b, c, d}); }
FQ_DEV uint32_t fma_h2(uint32_t a, uint32_t b, uint32_t c) {
    return h2_bits(__builtin_elementwise_fma(bits_h2(a), bits_h2(b), bits_h2(c)));
}
FQ_DEV void lds_order() { __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront"); }

// Codes as fp16 without a conversion: a code c ORed under an exponent whose last place is
// 2^-s is 2^(10 - s) + c 2^-s, and the subtraction is exact.  INT4: c / 16, from bits 0..3
// (64 + c / 16) or bits 4..7 (4 + c / 16) of each half; INT8: c / 256 from bits 0..7 (4 + c / 256).
FQ_DEV uint32_t nib_lo(uint32_t w) {
    return h2_bits(bits_h2((w & 0x000F000Fu) | 0x54005400u) - h2{(_Float16)64.f, (_Float16)64.f});
}
FQ_DEV uint32_t nib_hi(uint32_t w) {
    return h2_bits(bits_h2((w & 0x00F000F0u) | 0x44004400u) - h2{(_Float16)4.f, (_Float16)4.f});
}
FQ_DEV uint32_t byte_pair(uint32_t w) {          // bytes already at bits 0..7 of each half, 0x44 above them
    return h2_bits(bits_h2(w) - h2{(_Float16)4.f, (_Float16)4.f});
}
template <int BITS> constexpr float kCodeUp = BITS == 4 ? 16.f : 256.f;      // scales take the code's factor back

FQ_DEV float rows_max(float v) {         // over lanes n, n + 16, n + 32, n + 48
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// A page as it is in memory: one lane's K bytes of keys 16 T + n (channels D/4 lg ..) and V
// bytes of 16 keys (channels D/16 n ..), and its share of the page's metadata.
template <int D, int BITS>
struct PageRaw {
    static constexpr int KD = D * BITS / 128;            // dwords of D/4 channels
    static constexpr int VD = D * BITS == 1024 ? 2 : 1;  // dwords (or one half) of D/16 channels
    uint32_t k[4][KD];
    uint32_t v[16][VD];
    uint32_t ks[2], km[2];               // two channels' K scale and minimum
    u32x2 vs, vm;                        // one token's V scales and minima
};

// A wave's LDS: the page's metadata as fp16, scales with the codes' factor.  K in operand order.
template <int D>
struct alignas(16) WaveMeta {
    uint16_t ks[D], km[D];
    uint16_t vs[4][kPg], vm[4][kPg];
};

// The keys of a lane's k-slots of step j of the second product: 32 j + 4 lg + {0..3}, then + 16.
FQ_DEV constexpr int slot_key(int u) { return (u & 3) + 16 * (u >> 2); }      // u = 0 .. 7, before 32 j + 4 lg

template <int D, int BITS, typename MT, int QB>
__global__ __launch_bounds__(64 * kW) void shared_attn_kernel(SharedParams a) {
    constexpr int NS = D / 32, NT = D / 16, RT = 16 * QB;
    constexpr int KB = D * BITS / 32;            // bytes of a lane's D/4 channels
    __shared__ WaveMeta<D> s_meta[kW];
    __shared__ v4f s_o[kW - 1][QB * NT][64];
    __shared__ float2 s_ml[kW - 1][QB][64];
    const int L = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
    const int n = L & 15, lg = L >> 4;
    WaveMeta<D>& M = s_meta[w];

    // KV heads vary fastest over the workgroups, so with 8 of them the row tiles of a head and
    // range run on one XCD and share its L2
    int64_t blk = blockIdx.x;
    const int pi = a.first < a.last && blk >= a.p[0].wgs ? 1 : a.first;
    if (pi > a.first) blk -= a.p[0].wgs;
    const SharedPart& P = a.p[pi];
    const int h = (int)(blk % a.Hkv);
    const int64_t r1 = blk / a.Hkv;
    const int tile = (int)(r1 % P.tiles);
    const int64_t r2 = r1 / P.tiles;
    const int split = (int)(r2 % P.splits), item = (int)(r2 / P.splits);
    const Int4Cache& c = P.c;
    const int code_pages = c.S / kPg;

    // The lane's rows: row0 + 16 qb + n
    const int row0 = tile * RT;
    int hi[QB];                                  // last key a row attends
    float rs[QB];                                // S^T -> scores in the log2 domain
    v8h qf[QB][NS];
    int lo = 0, hi_all = P.keys - 1;             // first key; the least hi of the tile
    if (pi == 1) {
        if (a.start) lo = min(max(a.start[item], 0), P.keys);
        hi_all = P.keys - a.Sq + row0 / a.G;
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const int row = min(row0 + 16 * qb + n, P.rows - 1);
        const int g = row % a.G, i = (row / a.G) % a.Sq, b = pi == 1 ? item : row / (a.G * a.Sq);
        hi[qb] = pi == 1 ? P.keys - a.Sq + i : P.keys - 1;
        const uint16_t* q = (const uint16_t*)a.q + b * a.q_s[0] + (int64_t)(h * a.G + g) * a.q_s[1] + i * a.q_s[2] +
                            (D / 4) * lg;
        float x[NS][8];
        float mx = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const u32x4 v = *(const u32x4*)(q + 8 * s);
            const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                x[s][2 * u] = a.bf16 ? bf16_bits_to_f(d[u] & 0xFFFFu) : f16_bits_to_f(d[u] & 0xFFFFu);
                x[s][2 * u + 1] = a.bf16 ? bf16_bits_to_f(d[u] >> 16) : f16_bits_to_f(d[u] >> 16);
                mx = fmaxf(mx, fmaxf(fabsf(x[s][2 * u]), fabsf(x[s][2 * u + 1])));
            }
        }
        mx = rows_max(mx);
        const int e = mx > 0.f && mx < INFINITY ? __builtin_amdgcn_frexp_expf(mx) : 0;      // mx = f 2^e, 1/2 <= f < 1
        rs[qb] = ldexpf(a.qk_scale / kKExp, e);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            uint32_t d[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {        // INT4: channels in the order the codes unpack
                const int c0 = BITS == 4 ? u : 2 * u, c1 = BITS == 4 ? u + 4 : 2 * u + 1;
                d[u] = pack_h2(ldexpf(x[s][c0], -e), ldexpf(x[s][c1], -e));
            }
            qf[qb][s] = frag(d[0], d[1], d[2], d[3]);
        }
    }

    v4f o[QB][NT], ol[QB];
    float m_run[QB];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        m_run[qb] = -INFINITY;
        ol[qb] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NT; ++i) o[qb][i] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    const v8h ones = frag(0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u);

    // One page of 64 keys: kf(T, s) and vf(j, i) give its operands, masked: some row's keys end
    // or begin inside it.
    auto page_step = [&](int page, bool masked, auto kf, auto vf) {
        v4f s[QB][4];
#pragma unroll
        for (int T = 0; T < 4; ++T) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) s[qb][T] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < NS; ++st) {
                const v8h k = kf(T, st);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) s[qb][T] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[qb][st], s[qb][T], 0, 0, 0);
            }
        }
        if (masked) {
            const int k0 = page * kPg + 4 * lg;
#pragma unroll
            for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                for (int T = 0; T < 4; ++T)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = k0 + 16 * T + r;
                        if (key < lo || key > hi[qb]) s[qb][T][r] = -INFINITY;
                    }
        }
        float mx[QB];
        bool moved = false;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            float t[4];
#pragma unroll
            for (int T = 0; T < 4; ++T) t[T] = fmaxf(fmaxf(s[qb][T][0], s[qb][T][1]), fmaxf(s[qb][T][2], s[qb][T][3]));
            mx[qb] = rows_max(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]))) * rs[qb];
            moved |= mx[qb] > m_run[qb] + kLazy;
        }
        if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                const float m_new = fmaxf(m_run[qb], mx[qb]);
                const float al = __builtin_amdgcn_exp2f(m_run[qb] - (m_new == -INFINITY ? 0.f : m_new));
                m_run[qb] = m_new;
                ol[qb] *= al;
#pragma unroll
                for (int i = 0; i < NT; ++i) o[qb][i] *= al;
            }
        }
        v8h pb[QB][2];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            const float ref = kPShift - (m_run[qb] == -INFINITY ? 0.f : m_run[qb]);
            uint32_t d[4][2];
#pragma unroll
            for (int T = 0; T < 4; ++T)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    d[T][r] = pack_h2(__builtin_amdgcn_exp2f(fmaf(s[qb][T][2 * r], rs[qb], ref)),
                                      __builtin_amdgcn_exp2f(fmaf(s[qb][T][2 * r + 1], rs[qb], ref)));
            pb[qb][0] = frag(d[0][0], d[0][1], d[1][0], d[1][1]);
            pb[qb][1] = frag(d[2][0], d[2][1], d[3][0], d[3][1]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const v8h v = vf(j, i);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb[qb][j], o[qb][i], 0, 0, 0);
            }
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) ol[qb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[qb][j], ol[qb], 0, 0, 0);
        }
    };

    // The item's slices; a page's part of an address is uniform, a lane's the same for every page.
    const uint8_t* kb = c.kp + item * c.kp_s[1] + h * c.kp_s[2] + n * c.kp_s[3] + KB * lg;
    const uint8_t* vb = c.vp + item * c.vp_s[1] + h * c.vp_s[2] + 4 * lg * c.vp_s[3] + (D * BITS / 128) * n;
    // two channels of a lane whose fp16 values are neighbours in operand order
    const int mc0 = BITS == 4 ? 8 * (L >> 2) + (L & 3) : 2 * L, mc1 = BITS == 4 ? mc0 + 4 : mc0 + 1;
    const int mcl = 2 * L < D ? 0 : 1;           // D = 64: lanes 32 .. 63 have none and repeat channel 0
    const uint16_t* ksb = (const uint16_t*)c.ksc + item * c.ksc_s[1] + h * c.ksc_s[2];
    const uint16_t* kmb = (const uint16_t*)c.kmn + item * c.kmn_s[1] + h * c.kmn_s[2];
    const uint16_t* vsb = (const uint16_t*)c.vsc + item * c.vsc_s[1] + h * c.vsc_s[2] + L * c.vsc_s[3];
    const uint16_t* vmb = (const uint16_t*)c.vmn + item * c.vmn_s[1] + h * c.vmn_s[2] + L * c.vmn_s[3];
    const int G = c.G;

    auto load = [&](PageRaw<D, BITS>& r, int page) {
        const int64_t t0 = (int64_t)page * kPg;
        const uint8_t* kp = kb + t0 * c.kp_s[3];
#pragma unroll
        for (int T = 0; T < 4; ++T) {
            const uint8_t* p = kp + 16 * T * c.kp_s[3];
            if constexpr (KB == 8) {
                const u32x2 x = *(const u32x2*)p;
                r.k[T][0] = x.x; r.k[T][1] = x.y;
            } else {
#pragma unroll
                for (int u = 0; u < KB / 16; ++u) {
                    const u32x4 x = *(const u32x4*)(p + 16 * u);
                    r.k[T][4 * u] = x.x; r.k[T][4 * u + 1] = x.y; r.k[T][4 * u + 2] = x.z; r.k[T][4 * u + 3] = x.w;
                }
            }
        }
        const uint8_t* vp = vb + t0 * c.vp_s[3];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const uint8_t* p = vp + (32 * (u >> 3) + slot_key(u & 7)) * c.vp_s[3];
            if constexpr (D * BITS == 256) r.v[u][0] = *(const uint16_t*)p;
            else if constexpr (D * BITS == 512) r.v[u][0] = *(const uint32_t*)p;
            else { const u32x2 x = *(const u32x2*)p; r.v[u][0] = x.x; r.v[u][1] = x.y; }
        }
        const int64_t ks = page * c.ksc_s[3], km = page * c.kmn_s[3];
        r.ks[0] = ksb[ks + (mcl ? 0 : mc0)]; r.ks[1] = ksb[ks + (mcl ? 0 : mc1)];
        r.km[0] = kmb[km + (mcl ? 0 : mc0)]; r.km[1] = kmb[km + (mcl ? 0 : mc1)];
        const uint16_t* vs = vsb + t0 * c.vsc_s[3];
        const uint16_t* vm = vmb + t0 * c.vmn_s[3];
        r.vs = u32x2{vs[0], 0u}; r.vm = u32x2{vm[0], 0u};
        if (G > 1) {
            r.vs.x |= (uint32_t)vs[1] << 16; r.vm.x |= (uint32_t)vm[1] << 16;
            if (G > 2) {
                r.vs.y = vs[2] | (uint32_t)vs[3] << 16;
                r.vm.y = vm[2] | (uint32_t)vm[3] << 16;
            }
        }
    };

    auto code_page = [&](const PageRaw<D, BITS>& r, int page) {
        // metadata through LDS: every lane converts its share, all read it in operand order
        constexpr float up = kCodeUp<BITS>;
        lds_order();
        if (!mcl) {
            *(uint32_t*)&M.ks[2 * L] = pack_h2(meta_f<MT>(r.ks[0]) * (up * kKExp), meta_f<MT>(r.ks[1]) * (up * kKExp));
            *(uint32_t*)&M.km[2 * L] = pack_h2(meta_f<MT>(r.km[0]) * kKExp, meta_f<MT>(r.km[1]) * kKExp);
        }
        const bool on = page * kPg + L >= lo;            // values of padding tokens count as 0, whatever they are
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (g >= G) break;
            const uint32_t sb = (g < 2 ? r.vs.x : r.vs.y) >> (16 * (g & 1)), mb = (g < 2 ? r.vm.x : r.vm.y) >> (16 * (g & 1));
            M.vs[g][L] = on ? f_to_f16_bits(meta_f<MT>(sb) * up) : 0;
            M.vm[g][L] = on ? f_to_f16_bits(meta_f<MT>(mb)) : 0;
        }
        lds_order();
        u32x4 sk[NS], mk[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            sk[s] = *(const u32x4*)&M.ks[(D / 4) * lg + 8 * s];
            mk[s] = *(const u32x4*)&M.km[(D / 4) * lg + 8 * s];
        }
        const int vg = n * G >> 4;
        u32x2 sv[2][2], mv[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                sv[j][u] = *(const u32x2*)&M.vs[vg][32 * j + 16 * u + 4 * lg];
                mv[j][u] = *(const u32x2*)&M.vm[vg][32 * j + 16 * u + 4 * lg];
            }
        auto kf = [&](int T, int s) {
            uint32_t x[4];
            if constexpr (BITS == 4) {
                const uint32_t wd = r.k[T][s], w8 = wd >> 8;
                x[0] = nib_lo(wd); x[1] = nib_hi(wd); x[2] = nib_lo(w8); x[3] = nib_hi(w8);
            } else {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t wd = r.k[T][2 * s + u];
                    x[2 * u] = byte_pair(__builtin_amdgcn_perm(0x44444444u, wd, 0x04010400u));
                    x[2 * u + 1] = byte_pair(__builtin_amdgcn_perm(0x44444444u, wd, 0x04030402u));
                }
            }
            return frag(fma_h2(x[0], sk[s].x, mk[s].x), fma_h2(x[1], sk[s].y, mk[s].y), fma_h2(x[2], sk[s].z, mk[s].z),
                        fma_h2(x[3], sk[s].w, mk[s].w));
        };
        auto vf = [&](int j, int i) {                    // channel D/16 n + i of 8 keys
            uint32_t x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {                // keys 2u, 2u + 1 of the slots
                const uint32_t wa = r.v[8 * j + 2 * u][BITS == 8 ? i >> 2 : 0], wb = r.v[8 * j + 2 * u + 1][BITS == 8 ? i >> 2 : 0];
                const uint32_t y = BITS == 4 ? i >> 1 : i & 3;
                if constexpr (BITS == 4) {
                    const uint32_t pr = __builtin_amdgcn_perm(wb, wa, 0x0C000C00u | y | (y + 4) << 16);
                    x[u] = i & 1 ? nib_hi(pr) : nib_lo(pr);
                } else {
                    const uint32_t pr = __builtin_amdgcn_perm(wb, wa, 0x0C000C00u | y | (y + 4) << 16);
                    x[u] = byte_pair(pr | 0x44004400u);
                }
            }
            return frag(fma_h2(x[0], sv[j][0].x, mv[j][0].x), fma_h2(x[1], sv[j][0].y, mv[j][0].y),
                        fma_h2(x[2], sv[j][1].x, mv[j][1].x), fma_h2(x[3], sv[j][1].y, mv[j][1].y));
        };
        page_step(page, page * kPg < lo || page * kPg + kPg - 1 > hi_all, kf, vf);
    };

    // The partial page: bf16 rows, the last one repeated past the end (masked; values 0).
    auto tail_page = [&](int page) {
        const TailArgs& t = P.t;
        const uint16_t* kt = (const uint16_t*)t.k + item * t.ks[1] + h * t.ks[2] + (D / 4) * lg;
        const uint16_t* vt = (const uint16_t*)t.v + item * t.vs[1] + h * t.vs[2] + (D / 16) * n;
        auto kf = [&](int T, int s) {
            const u32x4 v = *(const u32x4*)(kt + (int64_t)min(16 * T + n, t.len - 1) * t.ks[3] + 8 * s);
            float x[8];
            const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                x[2 * u] = bf16_bits_to_f(d[u] & 0xFFFFu) * kKExp;
                x[2 * u + 1] = bf16_bits_to_f(d[u] >> 16) * kKExp;
            }
            if constexpr (BITS == 4) return frag(pack_h2(x[0], x[4]), pack_h2(x[1], x[5]), pack_h2(x[2], x[6]), pack_h2(x[3], x[7]));
            else return frag(pack_h2(x[0], x[1]), pack_h2(x[2], x[3]), pack_h2(x[4], x[5]), pack_h2(x[6], x[7]));
        };
        uint32_t tv[16][NT / 2];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const int key = 32 * (u >> 3) + slot_key(u & 7) + 4 * lg;
            const uint16_t* p = vt + (int64_t)min(key, t.len - 1) * t.vs[3];
            const bool on = key < t.len && page * kPg + key >= lo;
            if constexpr (NT == 8) {
                const u32x4 x = *(const u32x4*)p;
                tv[u][0] = on ? x.x : 0u; tv[u][1] = on ? x.y : 0u; tv[u][2] = on ? x.z : 0u; tv[u][3] = on ? x.w : 0u;
            } else {
                const u32x2 x = *(const u32x2*)p;
                tv[u][0] = on ? x.x : 0u; tv[u][1] = on ? x.y : 0u;
            }
        }
        auto vf = [&](int j, int i) {
            uint32_t x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t wa = tv[8 * j + 2 * u][i >> 1], wb = tv[8 * j + 2 * u + 1][i >> 1];
                x[u] = i & 1 ? pack_h2(bf16_bits_to_f(wa >> 16), bf16_bits_to_f(wb >> 16))
                             : pack_h2(bf16_bits_to_f(wa & 0xFFFFu), bf16_bits_to_f(wb & 0xFFFFu));
            }
            return frag(x[0], x[1], x[2], x[3]);
        };
        page_step(page, true, kf, vf);
    };

    // This wave's pages, every fourth of the workgroup's range; pages before the first key or
    // behind the last row's are left out.
    const int p_first = max(split * P.per_split, lo / kPg);
    const int hi_top = pi == 1 ? P.keys - a.Sq + min(row0 + RT - 1, P.rows - 1) / a.G : P.keys - 1;
    const int p_end = min(min((split + 1) * P.per_split, P.pages), hi_top / kPg + 1);
    int page = p_first + w;
    const int code_end = min(p_end, code_pages);
    if (page < code_end) {
        PageRaw<D, BITS> cur, nxt;
        load(cur, page);
        while (true) {
            const int np = page + kW;
            const bool more = np < code_end;
            load(nxt, more ? np : page);                 // unconditional: in flight while this page is computed
            code_page(cur, page);
            page = np;
            if (!more) break;
            cur = nxt;
        }
    }
    if (page < p_end) tail_page(page);                   // page == code_pages: only the partial one is left

    // The waves' states meet in wave 0.
    if (w > 0) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            s_ml[w - 1][qb][L] = make_float2(m_run[qb], ol[qb][0]);
#pragma unroll
            for (int i = 0; i < NT; ++i) s_o[w - 1][qb * NT + i][L] = o[qb][i];
        }
    }
    __syncthreads();
    if (w > 0) return;
    const int64_t base = ((int64_t)(item * a.Hkv + h) * P.splits + split) * P.rows;
    const int64_t all = (int64_t)P.items * a.Hkv * P.splits * P.rows;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        float m[kW], l[kW], mm = m_run[qb];
        m[0] = m_run[qb]; l[0] = ol[qb][0];
#pragma unroll
        for (int u = 1; u < kW; ++u) {
            const float2 x = s_ml[u - 1][qb][L];
            m[u] = x.x; l[u] = x.y;
            mm = fmaxf(mm, m[u]);
        }
        const float mu = mm == -INFINITY ? 0.f : mm;
        float wt[kW], ls = 0.f;
#pragma unroll
        for (int u = 0; u < kW; ++u) {
            wt[u] = __builtin_amdgcn_exp2f(m[u] - mu);
            ls = fmaf(wt[u], l[u], ls);
        }
        float x[4][NT];                                  // [r][i]: channel D/16 (4 lg + r) + i
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            v4f t = o[qb][i] * wt[0];
#pragma unroll
            for (int u = 1; u < kW; ++u) {
                const v4f y = s_o[u - 1][qb * NT + i][L];
#pragma unroll
                for (int r = 0; r < 4; ++r) t[r] = fmaf(wt[u], y[r], t[r]);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r][i] = t[r];
        }
        const int row = row0 + 16 * qb + n;
        if (row >= P.rows) continue;
        float* dst = P.part + (base + row) * D + (D / 4) * lg;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < NT; i += 4) *(v4f*)(dst + NT * r + i) = v4f{x[r][i], x[r][i + 1], x[r][i + 2], x[r][i + 3]};
        if (lg == 0) *(float2*)(P.part + all * D + 2 * (base + row)) = make_float2(mm, ls);
    }
}

// Joins the shares of a row: prefix splits, then suffix splits, in order.  D/4 lanes a row,
// four channels a lane.
template <int D>
__global__ __launch_bounds__(kThreads) void shared_merge_kernel(SharedParams a) {
    constexpr int LPR = D / 4;
    const int64_t idx = ((int64_t)blockIdx.x * kThreads + threadIdx.x) / LPR;
    const int ch = 4 * (threadIdx.x % LPR);
    if (idx >= (int64_t)a.B * a.Hq * a.Sq) return;
    // rows as the prefix has them: ((kv head, b), i, g)
    const int g = (int)(idx % a.G), i = (int)(idx / a.G % a.Sq);
    const int b = (int)(idx / (a.G * a.Sq) % a.B), h = (int)(idx / ((int64_t)a.G * a.Sq * a.B));
    float M = -INFINITY, l = 0.f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const SharedPart& P = a.p[p];
        const int item = p == 1 ? b : 0;
        const int row = p == 1 ? i * a.G + g : (b * a.Sq + i) * a.G + g;
        const int64_t all = (int64_t)P.items * a.Hkv * P.splits * P.rows;
        const int64_t base = (int64_t)(item * a.Hkv + h) * P.splits * P.rows + row;
        for (int s0 = 0; s0 < P.splits; s0 += 4) {
            float2 ml[4];
            v4f x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t at = base + (int64_t)min(s0 + u, P.splits - 1) * P.rows;
                ml[u] = *(const float2*)(P.part + all * D + 2 * at);
                x[u] = *(const v4f*)(P.part + at * D + ch);
            }
            float mn = M;
#pragma unroll
            for (int u = 0; u < 4; ++u) mn = fmaxf(mn, ml[u].x);
            if (mn == -INFINITY) {       // nothing so far, but a NaN stays one
#pragma unroll
                for (int u = 0; u < 4; ++u) if (s0 + u < P.splits) { l += ml[u].y; o += x[u]; }
                continue;
            }
            const float al = __builtin_amdgcn_exp2f(M - mn);
            l *= al;
            o *= al;
            M = mn;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (s0 + u >= P.splits) break;
                const float wt = __builtin_amdgcn_exp2f(ml[u].x - mn);
                l = fmaf(wt, ml[u].y, l);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[r] = fmaf(wt, x[u][r], o[r]);
            }
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;         // a row without keys: O = 0, lse = -inf
    const int hq = h * a.G + g;
    uint16_t* out = (uint16_t*)a.out + b * a.o_s[0] + hq * a.o_s[1] + i * a.o_s[2] + ch;
    uint16_t y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = a.bf16 ? f_to_bf16_bits(o[r] * inv) : f_to_f16_bits(o[r] * inv);
    *(u32x2*)out = u32x2{(uint32_t)y[0] | (uint32_t)y[1] << 16, (uint32_t)y[2] | (uint32_t)y[3] << 16};
    if (a.lse && ch == 0)
        a.lse[b * a.lse_s[0] + hq * a.lse_s[1] + i * a.lse_s[2]] =
            l == 0.f ? -INFINITY : (M - kPShift + __log2f(l)) * kLn2;
}

// Rows a wave takes: 16 where they hold an item's rows, else 32.
int row_blocks(int rows) { return rows <= 16 ? 1 : 2; }

// Key splits of a part: enough workgroups for the GPU's slots, at least 4 pages (one a wave) each.
void plan_part(SharedPart& p, int Hkv, int qb) {
    const int slots = 512;
    p.tiles = (p.rows + 16 * qb - 1) / (16 * qb);
    p.pages = (p.keys + kPg - 1) / kPg;
    const int64_t groups = (int64_t)p.items * Hkv * p.tiles;
    const int most = std::max(1, (p.pages + kW - 1) / kW);
    int64_t s = std::max<int64_t>(1, slots / std::max<int64_t>(1, groups));
    s = std::min<int64_t>(s, most);
    p.per_split = (int)((p.pages + s - 1) / s);
    if (p.per_split < 1) p.per_split = 1;
    p.splits = std::max(1, (p.pages + p.per_split - 1) / p.per_split);
    p.wgs = groups * p.splits;
}

size_t part_floats(const SharedPart& p, int Hkv, int D) {
    return (size_t)p.items * Hkv * p.splits * p.rows * (D + 2);
}

}  // namespace

// prefix / suffix: the two caches and their partial pages (checked; S whole pages, keys > 0);
// q (B, Hq, Sq, D).  ws null: returns the workspace bytes in *bytes.
hipError_t launch_shared_prefix(const Int4Cache& pc, const TailArgs& pt, const Int4Cache& sc, const TailArgs& st_,
                                const fq_shared_query& q, float qk_scale, void* ws, size_t* bytes, hipStream_t st) {
    SharedParams a{};
    const int G = q.H_q / pc.Hkv;
    a.p[0].c = pc; a.p[0].t = pt; a.p[0].keys = pc.S + pt.len; a.p[0].items = 1; a.p[0].rows = q.B * q.S_q * G;
    a.p[1].c = sc; a.p[1].t = st_; a.p[1].keys = sc.S + st_.len; a.p[1].items = q.B; a.p[1].rows = q.S_q * G;
    int qb[2];
    for (int i = 0; i < 2; ++i) {
        qb[i] = row_blocks(a.p[i].rows);
        plan_part(a.p[i], pc.Hkv, qb[i]);
    }
    if (!ws) {
        *bytes = (part_floats(a.p[0], pc.Hkv, pc.D) + part_floats(a.p[1], pc.Hkv, pc.D)) * sizeof(float);
        return hipSuccess;
    }
    if (a.p[0].wgs + a.p[1].wgs > 0x7FFFFFFF) return hipErrorInvalidValue;
    a.p[0].part = (float*)ws;
    a.p[1].part = a.p[0].part + part_floats(a.p[0], pc.Hkv, pc.D);
    a.q = q.q; a.out = q.out; a.lse = q.lse; a.start = q.start;
    for (int i = 0; i < 3; ++i) { a.q_s[i] = q.q_strides[i]; a.o_s[i] = q.o_strides[i]; a.lse_s[i] = q.lse_strides[i]; }
    a.bf16 = q.dtype == FQ_BF16;
    a.B = q.B; a.Hq = q.H_q; a.Hkv = pc.Hkv; a.G = G; a.Sq = q.S_q;
    a.qk_scale = qk_scale;
    auto attend = [&](int first, int last, int nb) {
        a.first = first; a.last = last;
        int64_t wgs = 0;
        for (int i = first; i <= last; ++i) wgs += a.p[i].wgs;
        const dim3 grid((unsigned)wgs);
        const bool bf = pc.meta_dtype == FQ_BF16;
#define FQ_SP(D_, B_, Q_)                                                                                              \
    if (pc.D == D_ && pc.bits == B_ && nb == Q_) {                                                                     \
        if (bf) hipLaunchKernelGGL((shared_attn_kernel<D_, B_, struct bf16, Q_>), grid, dim3(64 * kW), 0, st, a);      \
        else hipLaunchKernelGGL((shared_attn_kernel<D_, B_, f16, Q_>), grid, dim3(64 * kW), 0, st, a);                 \
        return hipGetLastError();                                                                                      \
    }
#define FQ_SPQ(D_, B_) FQ_SP(D_, B_, 1) FQ_SP(D_, B_, 2)
        FQ_SPQ(128, 4) FQ_SPQ(128, 8) FQ_SPQ(64, 4) FQ_SPQ(64, 8)
#undef FQ_SPQ
#undef FQ_SP
        return hipErrorInvalidValue;
    };
    hipError_t e;
    if (qb[0] == qb[1]) {
        e = attend(0, 1, qb[0]);
    } else {
        e = attend(0, 0, qb[0]);
        if (e == hipSuccess) e = attend(1, 1, qb[1]);
    }
    if (e != hipSuccess) return e;
    const int64_t threads = (int64_t)q.B * q.H_q * q.S_q * (pc.D / 4);
    const dim3 grid((unsigned)((threads + kThreads - 1) / kThreads));
    if (pc.D == 128) hipLaunchKernelGGL(shared_merge_kernel<128>, grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL(shared_merge_kernel<64>, grid, dim3(kThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace fq
