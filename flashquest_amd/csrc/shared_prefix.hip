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
// Both kernels compute the transposed products
//   S^T = K Q^T     v_mfma_f32_16x16x32_f16, keys as the A operand
//   O^T += V^T P^T  the same, channels as the A operand
// which keep a row on one lane column: its statistics are per lane, and P leaves S^T's
// accumulator as the B operand of the second product.  shared_attn_kernel (few rows) turns the
// codes into operands in registers, 16 rows a wave; shared_tile_kernel (many) once per workgroup
// of 128 or 256 rows, through LDS.  plan_forms chooses, per part.
//
// What bounds them: reading the packed caches is the floor of short batches (37 MB of codes and
// metadata for 32768 tokens of 8 KV heads in INT4: 7 us), the products that of long ones, and
// between the two it is the vector instructions that turn codes into operands and scores into
// weights: beyond two vector instructions a matrix instruction each further one adds its own
// four cycles, so they have to be few of each page.
//
// Operands are fp16: errors of 4e-4 of the outputs' size, an fp16 output's own rounding (2e-4)
// included; a bf16 output's is 1.7e-3.  (bf16 operands, with 8 bits for 11, would leave eight times
// as much.)  q is exact after a power of two per row (16-bit inputs), K and V one rounding of
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
    int pages, per_split;                // pages (the partial one last), pages (row-tile kernel: stages) of a split
    uint32_t wgs;                        // items * Hkv * tiles * splits
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
FQ_DEV uint32_t opaque_v(uint32_t x) {           // a constant held in a vector register: v_and_or_b32 takes one scalar
    asm("" : "+v"(x));
    return x;
}
FQ_DEV uint32_t nib_lo(uint32_t w) {
    return h2_bits(bits_h2((w & 0x000F000Fu) | opaque_v(0x54005400u)) - h2{(_Float16)64.f, (_Float16)64.f});
}
FQ_DEV uint32_t nib_hi(uint32_t w) {
    return h2_bits(bits_h2((w & 0x00F000F0u) | opaque_v(0x44004400u)) - h2{(_Float16)4.f, (_Float16)4.f});
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

// A row's query as B operands: step s holds the 8 channels of q[s], in the order the codes unpack
// (INT4: u, u + 4 side by side).  q times 2^-e with the largest of the row below
// 1 is exact in fp16 (16-bit inputs: what underflows is below 2^-24 of it); returns the
// factor from S^T to scores in the log2 domain.
template <int D, int BITS>
FQ_DEV float turn_query(const u32x4 (&q)[D / 32], bool bf, float qk_scale, v8h (&qf)[D / 32]) {
    float x[D / 32][8];
    float mx = 0.f;
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
        const uint32_t d[4] = {q[s].x, q[s].y, q[s].z, q[s].w};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            x[s][2 * u] = bf ? bf16_bits_to_f(d[u] & 0xFFFFu) : f16_bits_to_f(d[u] & 0xFFFFu);
            x[s][2 * u + 1] = bf ? bf16_bits_to_f(d[u] >> 16) : f16_bits_to_f(d[u] >> 16);
            mx = fmaxf(mx, fmaxf(fabsf(x[s][2 * u]), fabsf(x[s][2 * u + 1])));
        }
    }
    mx = rows_max(mx);
    const int e = mx > 0.f && mx < INFINITY ? __builtin_amdgcn_frexp_expf(mx) : 0;      // mx = f 2^e, 1/2 <= f < 1
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
        uint32_t d[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c0 = BITS == 4 ? u : 2 * u, c1 = BITS == 4 ? u + 4 : 2 * u + 1;
            d[u] = pack_h2(ldexpf(x[s][c0], -e), ldexpf(x[s][c1], -e));
        }
        qf[s] = frag(d[0], d[1], d[2], d[3]);
    }
    return ldexpf(qk_scale / kKExp, e);
}

// 8 channels of K codes as fp16 pairs (times 1 / kCodeUp), in the queries' order.
template <int BITS>
FQ_DEV void key_codes(const uint32_t* w, uint32_t (&x)[4]) {
    if constexpr (BITS == 4) {
        const uint32_t w8 = w[0] >> 8;
        x[0] = nib_lo(w[0]); x[1] = nib_hi(w[0]); x[2] = nib_lo(w8); x[3] = nib_hi(w8);
    } else {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            x[2 * u] = byte_pair(__builtin_amdgcn_perm(0x44444444u, w[u], 0x04010400u));
            x[2 * u + 1] = byte_pair(__builtin_amdgcn_perm(0x44444444u, w[u], 0x04030402u));
        }
    }
}
// Channel i of two tokens' V codes (i counted within INT8's dword) as an fp16 pair.
template <int BITS>
FQ_DEV uint32_t value_pair(uint32_t wa, uint32_t wb, int i) {
    const uint32_t y = BITS == 4 ? i >> 1 : i & 3;
    const uint32_t pr = __builtin_amdgcn_perm(wb, wa, 0x0C000C00u | y | (y + 4) << 16);
    if constexpr (BITS == 4) return i & 1 ? nib_hi(pr) : nib_lo(pr);
    else return byte_pair(pr | 0x44004400u);
}
// The partial page's bf16: 8 channels of a key, one channel of two tokens.
template <int BITS>
FQ_DEV u32x4 tail_keys(const uint16_t* p) {
    const u32x4 v = *(const u32x4*)p;
    float x[8];
    const uint32_t d[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        x[2 * u] = bf16_bits_to_f(d[u] & 0xFFFFu) * kKExp;
        x[2 * u + 1] = bf16_bits_to_f(d[u] >> 16) * kKExp;
    }
    if constexpr (BITS == 4) return u32x4{pack_h2(x[0], x[4]), pack_h2(x[1], x[5]), pack_h2(x[2], x[6]), pack_h2(x[3], x[7])};
    else return u32x4{pack_h2(x[0], x[1]), pack_h2(x[2], x[3]), pack_h2(x[4], x[5]), pack_h2(x[6], x[7])};
}
FQ_DEV uint32_t tail_pair(uint32_t wa, uint32_t wb, int odd) {
    return odd ? pack_h2(bf16_bits_to_f(wa >> 16), bf16_bits_to_f(wb >> 16))
               : pack_h2(bf16_bits_to_f(wa & 0xFFFFu), bf16_bits_to_f(wb & 0xFFFFu));
}

// A workgroup's share: KV heads vary fastest, so with 8 of them the row tiles of a head and
// range run on one XCD and share its L2.
struct WgPlace { int h, tile, split, item; };
FQ_DEV WgPlace place(const SharedPart& P, uint32_t blk, int Hkv) {
    const uint32_t r1 = blk / Hkv, r2 = r1 / P.tiles;
    return {(int)(blk - r1 * Hkv), (int)(r1 - r2 * P.tiles), (int)(r2 % P.splits), (int)(r2 / P.splits)};
}

// A row of a part: head in the group, token, sequence (item: the suffix's).
struct RowPlace { int g, i, b; };
FQ_DEV RowPlace row_place(uint32_t row, int G, int Sq, bool suffix, int item) {
    const uint32_t t = row / G;
    const uint32_t b = suffix ? 0 : t / Sq;
    return {(int)(row - t * G), (int)(t - b * Sq), suffix ? item : (int)b};
}

// One step of the running softmax over a product's scores s (S^T: a lane's rows are its column's,
// keys 16 T + 4 lg + r): p = 2^(s rs - reference + kPShift) as the B operands of the second
// product.  The reference is the largest score seen, but moves only when one exceeds it by 2^8:
// sums and outputs are then rescaled, until then nothing is.
template <int QB, int NK, int NT>
FQ_DEV void softmax_step(v4f (&s)[QB][NK], const float (&rs)[QB], float (&m_run)[QB], v4f (&o)[QB][NT], v4f (&ol)[QB],
                         v8h (&pb)[QB][NK / 2]) {
    float ref[QB], mx[QB];
    bool moved = false;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const bool none = m_run[qb] == -INFINITY;
        ref[qb] = kPShift - (none ? 0.f : m_run[qb]);
        // exponents before the maximum: products of their own need no canonicalising moves, and
        // they are final unless the reference moves
#pragma unroll
        for (int T = 0; T < NK; ++T)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[qb][T][r] = fmaf(s[qb][T][r], rs[qb], ref[qb]);
        float m = fmaxf(fmaxf(s[qb][0][0], s[qb][0][1]), s[qb][0][2]);
        m = fmaxf(m, s[qb][0][3]);
#pragma unroll
        for (int T = 1; T < NK; ++T) {
            m = fmaxf(fmaxf(m, s[qb][T][0]), s[qb][T][1]);
            m = fmaxf(fmaxf(m, s[qb][T][2]), s[qb][T][3]);
        }
        mx[qb] = m;                              // of this lane's keys: joined over the row's lanes if it matters
        moved |= m > (none ? -INFINITY : kPShift + kLazy);
    }
    if (__builtin_amdgcn_ballot_w64(moved)) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            const float m_new = fmaxf(m_run[qb], rows_max(mx[qb]) - ref[qb]);
            const float nref = kPShift - (m_new == -INFINITY ? 0.f : m_new);
            const float al = __builtin_amdgcn_exp2f(m_run[qb] + nref - kPShift), by = nref - ref[qb];
            m_run[qb] = m_new;
            ol[qb] *= al;
#pragma unroll
            for (int i = 0; i < NT; ++i) o[qb][i] *= al;
#pragma unroll
            for (int T = 0; T < NK; ++T)
#pragma unroll
                for (int r = 0; r < 4; ++r) s[qb][T][r] += by;
        }
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        uint32_t d[NK][2];
#pragma unroll
        for (int T = 0; T < NK; ++T)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                d[T][r] = pack_h2(__builtin_amdgcn_exp2f(s[qb][T][2 * r]), __builtin_amdgcn_exp2f(s[qb][T][2 * r + 1]));
#pragma unroll
        for (int j = 0; j < NK / 2; ++j) pb[qb][j] = frag(d[2 * j][0], d[2 * j][1], d[2 * j + 1][0], d[2 * j + 1][1]);
    }
}

// Scores of keys outside lo .. hi, key0 the lane's first.
template <int QB, int NK>
FQ_DEV void mask_step(v4f (&s)[QB][NK], int key0, int lo, const int (&hi)[QB]) {
    asm volatile("");        // keeps the branch round it: most steps mask nothing
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int T = 0; T < NK; ++T)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = key0 + 16 * T + r;
                if (key < lo || key > hi[qb]) s[qb][T][r] = -INFINITY;
            }
}

// Values that are not finite, where a sequence has several query tokens: a weight of 0 times one is
// not 0, so rows that end before it would not be free of it.  Such values are taken as 0, and rows
// that give them a weight get NaN.  It costs 3 to 8 % of the row tiles' time (their registers).  (Keys that are not finite need none of this: scores of keys that
// a row does not attend are replaced.)
//
// 0xFFFF for each half where the scale or the minimum is not finite (fp16).
FQ_DEV uint32_t not_finite(uint32_t s, uint32_t m) {
    typedef uint16_t us2 __attribute__((ext_vector_type(2)));
    const us2 x = __builtin_elementwise_max(__builtin_bit_cast(us2, s & 0x7FFF7FFFu), __builtin_bit_cast(us2, m & 0x7FFF7FFFu));
    return (x.x >= 0x7C00u ? 0xFFFFu : 0u) | (x.y >= 0x7C00u ? 0xFFFF0000u : 0u);
}
// Whether any of 2 N bf16 values is not finite in fp16.
template <int N>
FQ_DEV uint32_t tail_not_finite(const uint32_t (&x)[N]) {
    uint32_t b = 0;
#pragma unroll
    for (int k = 0; k < N; ++k) b |= (x[k] & 0x7FFFu) >= 0x4780u || (x[k] & 0x7FFF0000u) >= 0x47800000u;     // 2^16 and more
    return b;
}
// bad[T]: such masks of the lane's keys 16 T + 4 lg + {0, 1}, {2, 3}; pb: the weights.
template <int QB, int NT>
FQ_DEV void spoil_rows(const u32x2 (&bad)[4], const v8h (&pb)[QB][2], v4f (&o)[QB][NT]) {
    uint32_t hit[QB], any = 0;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const u32x4 p = __builtin_bit_cast(u32x4, pb[qb][0]), q = __builtin_bit_cast(u32x4, pb[qb][1]);
        hit[qb] = (p.x & bad[0].x) | (p.y & bad[0].y) | (p.z & bad[1].x) | (p.w & bad[1].y) |
                  (q.x & bad[2].x) | (q.y & bad[2].y) | (q.z & bad[3].x) | (q.w & bad[3].y);
        any |= hit[qb];
    }
    if (!__builtin_amdgcn_ballot_w64(any != 0)) return;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const float x = rows_max(hit[qb] ? 1.f : 0.f) > 0.f ? NAN : 0.f;
#pragma unroll
        for (int i = 0; i < NT; ++i) o[qb][i] += x;
    }
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
    uint16_t bad[kPg];                   // spoil_rows' masks
};

// The keys of a lane's k-slots of step j of the second product: 32 j + 4 lg + {0..3}, then + 16.
FQ_DEV constexpr int slot_key(int u) { return (u & 3) + 16 * (u >> 2); }      // u = 0 .. 7, before 32 j + 4 lg

constexpr int attn_waves(int d) { return d == 64 ? 3 : 2; }      // a SIMD, as the registers allow

// Few rows: a wave takes 16 rows and every fourth page of its workgroup's range, its loads and
// operands its own, and the four waves' states meet in LDS.  The next page's metadata, keys and
// values are loaded into the registers of this one's as each has been used: a second set would
// leave room for one wave a SIMD instead of two (the suffixes of 64 sequences, INT8: 24 us then,
// 13.5 now; three or four waves a SIMD spill and are slower).  128 suffixes of 640 tokens of 8 KV
// heads in INT4: 27 us for 92 MB (3.4 TB/s), half of it waits for a page, half vector issue.
template <int D, int BITS, typename MT>
__global__ __launch_bounds__(64 * kW) __attribute__((amdgpu_waves_per_eu(attn_waves(D), attn_waves(D))))
void shared_attn_kernel(SharedParams a) {
    constexpr int QB = 1;
    constexpr int NS = D / 32, NT = D / 16, RT = 16 * QB;
    constexpr int KB = D * BITS / 32;            // bytes of a lane's D/4 channels
    __shared__ WaveMeta<D> s_meta[kW];
    __shared__ v4f s_o[kW - 1][QB * NT][64];
    __shared__ float2 s_ml[kW - 1][QB][64];
    const int L = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
    const int n = L & 15, lg = L >> 4;
    WaveMeta<D>& M = s_meta[w];

    const int pi = a.first < a.last && blockIdx.x >= a.p[0].wgs ? 1 : a.first;
    const SharedPart& P = a.p[pi];
    const WgPlace at = place(P, blockIdx.x - (pi > a.first ? a.p[0].wgs : 0u), a.Hkv);
    const int h = at.h, tile = at.tile, split = at.split, item = at.item;
    const Int4Cache& c = P.c;
    const int code_pages = c.S / kPg;

    // The lane's rows: row0 + 16 qb + n
    const int row0 = tile * RT;
    int hi[QB];                                  // last key a row attends
    float rs[QB];                                // S^T -> scores in the log2 domain
    v8h qf[QB][NS];
    u32x4 qr[QB][NS];                            // turned when the first keys are on their way
    int lo = 0, hi_all = P.keys - 1;             // first key; the least hi of the tile
    if (pi == 1) {
        if (a.start) lo = min(max(a.start[item], 0), P.keys);
        hi_all = P.keys - a.Sq + row0 / a.G;
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const int row = min(row0 + 16 * qb + n, P.rows - 1);
        const RowPlace r = row_place(row, a.G, a.Sq, pi == 1, item);
        hi[qb] = pi == 1 ? P.keys - a.Sq + r.i : P.keys - 1;
        const uint16_t* q = (const uint16_t*)a.q + r.b * a.q_s[0] + (int64_t)(h * a.G + r.g) * a.q_s[1] + r.i * a.q_s[2];
#pragma unroll
        for (int s = 0; s < NS; ++s) qr[qb][s] = *(const u32x4*)(q + (D / 4) * lg + 8 * s);
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

    const bool several = pi == 1 && a.Sq > 1;    // rows of several query tokens

    // One page of 64 keys: kf(T, s) and vf(j, i) give its operands, masked: some row's keys end
    // or begin inside it.
    auto page_step = [&](int page, bool masked, auto kf, auto vf, auto k_done) __attribute__((always_inline)) {
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
        k_done();
        if (masked) mask_step(s, page * kPg + 4 * lg, lo, hi);
        v8h pb[QB][2];
        softmax_step(s, rs, m_run, o, ol, pb);
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
        if (several) {
            asm volatile("");
            u32x2 bad[4];
#pragma unroll
            for (int T = 0; T < 4; ++T) bad[T] = *(const u32x2*)&M.bad[16 * T + 4 * lg];
            spoil_rows(bad, pb, o);
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

    auto load_k = [&](PageRaw<D, BITS>& r, int page) __attribute__((always_inline)) {
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
    };
    auto load_v = [&](PageRaw<D, BITS>& r, int page) __attribute__((always_inline)) {
        const uint8_t* vp = vb + (int64_t)page * kPg * c.vp_s[3];
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const uint8_t* p = vp + (32 * (u >> 3) + slot_key(u & 7)) * c.vp_s[3];
            if constexpr (D * BITS == 256) r.v[u][0] = *(const uint16_t*)p;
            else if constexpr (D * BITS == 512) r.v[u][0] = *(const uint32_t*)p;
            else { const u32x2 x = *(const u32x2*)p; r.v[u][0] = x.x; r.v[u][1] = x.y; }
        }
    };
    auto load_meta = [&](PageRaw<D, BITS>& r, int page) __attribute__((always_inline)) {
        const int64_t t0 = (int64_t)page * kPg, ks = page * c.ksc_s[3], km = page * c.kmn_s[3];
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

    auto code_page = [&](PageRaw<D, BITS>& r, int page, int next) __attribute__((always_inline)) {
        // metadata through LDS: every lane converts its share, all read it in operand order
        constexpr float up = kCodeUp<BITS>;
        lds_order();
        if (!mcl) {
            *(uint32_t*)&M.ks[2 * L] = pack_h2(meta_f<MT>(r.ks[0]) * (up * kKExp), meta_f<MT>(r.ks[1]) * (up * kKExp));
            *(uint32_t*)&M.km[2 * L] = pack_h2(meta_f<MT>(r.km[0]) * kKExp, meta_f<MT>(r.km[1]) * kKExp);
        }
        bool on = page * kPg + L >= lo;                  // values of padding tokens count as 0, whatever they are
        if (several) {
            asm volatile("");
            bool fine = true;
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (g >= G) break;
                const uint32_t sb = (g < 2 ? r.vs.x : r.vs.y) >> (16 * (g & 1)), mb = (g < 2 ? r.vm.x : r.vm.y) >> (16 * (g & 1));
                fine &= fabsf(meta_f<MT>(sb)) * up < 65520.f && fabsf(meta_f<MT>(mb)) < 65520.f;         // finite in fp16; false for NaN
            }
            M.bad[L] = on && !fine ? 0xFFFFu : 0u;
            on = on && fine;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (g >= G) break;
            const uint32_t sb = (g < 2 ? r.vs.x : r.vs.y) >> (16 * (g & 1)), mb = (g < 2 ? r.vm.x : r.vm.y) >> (16 * (g & 1));
            M.vs[g][L] = on ? f_to_f16_bits(meta_f<MT>(sb) * up) : 0;
            M.vm[g][L] = on ? f_to_f16_bits(meta_f<MT>(mb)) : 0;
        }
        if (next) load_meta(r, next);
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
            key_codes<BITS>(&r.k[T][BITS == 4 ? s : 2 * s], x);
            return frag(fma_h2(x[0], sk[s].x, mk[s].x), fma_h2(x[1], sk[s].y, mk[s].y), fma_h2(x[2], sk[s].z, mk[s].z),
                        fma_h2(x[3], sk[s].w, mk[s].w));
        };
        auto vf = [&](int j, int i) {                    // channel D/16 n + i of 8 keys
            uint32_t x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {                // keys 2u, 2u + 1 of the slots
                const int d = BITS == 8 ? i >> 2 : 0;
                x[u] = value_pair<BITS>(r.v[8 * j + 2 * u][d], r.v[8 * j + 2 * u + 1][d], i);
            }
            return frag(fma_h2(x[0], sv[j][0].x, mv[j][0].x), fma_h2(x[1], sv[j][0].y, mv[j][0].y),
                        fma_h2(x[2], sv[j][1].x, mv[j][1].x), fma_h2(x[3], sv[j][1].y, mv[j][1].y));
        };
        page_step(page, page * kPg < lo || page * kPg + kPg - 1 > hi_all, kf, vf, [&]() __attribute__((always_inline)) {
            if (next) load_k(r, next);
        });
        if (next) load_v(r, next);
    };

    // The partial page: bf16 rows, the last one repeated past the end (masked; values 0).
    auto tail_page = [&](int page) {
        const TailArgs& t = P.t;
        const uint16_t* kt = (const uint16_t*)t.k + item * t.ks[1] + h * t.ks[2] + (D / 4) * lg;
        const uint16_t* vt = (const uint16_t*)t.v + item * t.vs[1] + h * t.vs[2] + (D / 16) * n;
        auto kf = [&](int T, int s) {
            return __builtin_bit_cast(v8h, tail_keys<BITS>(kt + (int64_t)min(16 * T + n, t.len - 1) * t.ks[3] + 8 * s));
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
        if (several) {
            asm volatile("");
            lds_order();
            M.bad[L] = 0;
            lds_order();
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                const uint32_t b = tail_not_finite(tv[u]);
                if (b) M.bad[32 * (u >> 3) + slot_key(u & 7) + 4 * lg] = 0xFFFFu;        // (any lane that has one)
#pragma unroll
                for (int k = 0; k < NT / 2; ++k) tv[u][k] = b ? 0u : tv[u][k];
            }
            lds_order();
        }
        auto vf = [&](int j, int i) {
            uint32_t x[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                x[u] = tail_pair(tv[8 * j + 2 * u][i >> 1], tv[8 * j + 2 * u + 1][i >> 1], i & 1);
            }
            return frag(x[0], x[1], x[2], x[3]);
        };
        page_step(page, true, kf, vf, [] {});
    };

    // This wave's pages, every fourth of the workgroup's range; pages before the first key or
    // behind the last row's are left out.
    const int p_first = max(split * P.per_split, lo / kPg);
    const int hi_top = pi == 1 ? P.keys - a.Sq + min(row0 + RT - 1, P.rows - 1) / a.G : P.keys - 1;
    const int p_end = min(min((split + 1) * P.per_split, P.pages), hi_top / kPg + 1);
    int page = p_first + w;
    const int code_end = min(p_end, code_pages);
    auto turn = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) rs[qb] = turn_query<D, BITS>(qr[qb], a.bf16, a.qk_scale, qf[qb]);
    };
    if (page < code_end) {
        PageRaw<D, BITS> r;
        load_meta(r, page);
        load_k(r, page);
        load_v(r, page);
        turn();
        while (true) {
            const int next = page + kW < code_end ? page + kW : 0;
            code_page(r, page, next);
            page += kW;
            if (!next) break;
        }
    }
    if (page == p_first + w) turn();                     // (no page yet)
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

// ---- many rows: keys and values staged in LDS ------------------------------------------
// With more rows than a wave or two take, turning a page into operands once per 16 rows is what
// the time goes into.  Here a workgroup turns each stage of two pages into fp16 once, K as
// [key][channel] and V as [channel][key] in LDS, while the stage before is attended: 256 / KG rows
// times KG groups of keys, key group kg taking keys 128 kg / KG .. of every stage for its rows; the
// groups' states meet in LDS at the end.  Metadata is turned into fp16 once, through LDS too.  The
// codes are loaded a stage ahead, their metadata two: no wait on memory in the loop but the one for
// loads that are a stage old.
//
// KG = 1: 8 waves of 32 rows, two a SIMD, each thread turning K and V; an operand read from LDS
// feeds two matrix instructions.  KG = 2: 16 waves of 16 rows, four a SIMD, the lower ones turning K
// and the upper ones V; a read feeds one (1.9 ns of LDS to 1.8 of the four matrix cores), but three
// other waves have work while one waits.  512 rows over 32768 tokens in INT4: 102 us with 8 waves for
// KG = 1, 106 with 16; 128 rows: 49 with 8 for KG = 2, 47 with 16; 320 rows over 16384: 60 and 49.
//
// 4 x 512 rows over 16411 tokens of 8 KV heads in INT8: 151 us, 0.92 PFLOP/s (a large fp16 product
// reaches 1.17).  A matrix instruction takes 7.1 ns of a SIMD and hides two vector instructions of the
// other wave; each further one adds 2.3 ns.  Left out one at a time, the products were 63 %, scores to
// weights 20 % and the operands' making 16 % of the time: hardly any overlap.  Keeping the two waves of
// a SIMD in different parts by barriers did not bring it (a part then lasts as long as one wave's
// serial instructions).
//
// SEVERAL: a launch with suffixes of several query tokens (spoil_rows); without it a step of one token
// is 1 to 2 % faster.
//
// LDS holds a plane for each lane group lg of the operands: K's plane has a row per key of the
// chunks (8 channels, 16 bytes) 4 st + lg, V's a row per channel of the chunks (8 keys) 4 jb + lg.
// A 16-byte read of 64 lanes is served 16 lanes at a time, 8 of one lg and the other 8 n of the
// next; with chunk x of row r at x ^ (r / rows of 256 bytes) those 16 hit all banks once, and so
// do the writes (planes 64 bytes apart modulo 256; not for K with D = 64, 4 on a bank).  V's
// channels are dealt to the tiles as the codes unpack (tile i: channels D/16 n + i), so that the
// 16 lanes that write channel i of their codes write neighbouring rows.
constexpr int kST = 2 * kPg;             // keys of a stage
// Scheduling groups: n LDS reads, then (m matrix instructions, one read) until the reads are out,
// then the rest: operand reads stay n ahead of their use (left alone, the scheduler puts each
// right before it and every pair of matrix instructions waits for LDS).
template <int READS, int AHEAD, int MFMA_PER_READ>
FQ_DEV void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
    for (int i = 0; i < READS - AHEAD; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, MFMA_PER_READ, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD * MFMA_PER_READ, 0);
}
constexpr int tile_waves(int kg) { return kg == 1 ? 8 : 16; }

template <int D> struct StageLds {
    static constexpr int NS = D / 32;
    static constexpr int KROW = 16 * NS, KPL = kST * KROW + (D == 128 ? 64 : 0), KB = 4 * KPL;
    static constexpr int VROW = 64, VPL = D * VROW + 64, VB = 4 * VPL;
    FQ_DEV static int k_at(int lg, int key, int st) { return lg * KPL + key * KROW + 16 * (st ^ ((key / (16 / NS)) & (NS - 1))); }
    FQ_DEV static int v_at(int lg, int row, int jb) { return lg * VPL + row * VROW + 16 * (jb ^ ((row >> 2) & 3)); }
};

template <int D, int BITS, typename MT, int KG, bool SEVERAL>
__global__ __launch_bounds__(64 * tile_waves(KG)) __attribute__((amdgpu_waves_per_eu(tile_waves(KG) / 4, tile_waves(KG) / 4)))
void shared_tile_kernel(SharedParams a) {
    constexpr int kTW = tile_waves(KG), QB = 16 / kTW, NS = D / 32, NT = D / 16, VC = D / 16;
    constexpr int RG = kTW / KG;                 // row groups
    constexpr int RT = 16 * QB * RG;                  // rows of the workgroup
    constexpr int NK = kPg / 16, NJ = kPg / 32, NSUB = 2 / KG;       // of a product of 64 keys: 16-key tiles, 32-key steps; products a stage
    constexpr int TPP = 256;                     // threads of a page (KG = 2: for K and for V)
    constexpr int CPR = D / 8, KPT = kPg * CPR / TPP;        // K: chunks of a row, rows a thread turns
    constexpr int KW = BITS / 4, VW = VC * BITS / 8 == 8 ? 2 : 1;            // dwords of 8 K channels, of VC V channels
    constexpr int AHEAD = QB == 2 ? 6 : 2;                    // operand reads in flight
    using Lds = StageLds<D>;
    __shared__ __attribute__((aligned(16))) uint8_t s_k[2][Lds::KB];
    __shared__ __attribute__((aligned(16))) uint8_t s_v[2][Lds::VB];
    // metadata as fp16, scales with the codes' factor: [stage & 1][page] [scale, minimum] of K's
    // channels in operand order, and of V's tokens by channel group
    __shared__ __attribute__((aligned(16))) uint16_t s_bad[2][2][kPg];       // spoil_rows' masks of a stage
    __shared__ __attribute__((aligned(16))) uint16_t s_km[2][2][2][D], s_vm[2][2][4][2][kPg];
    const int tid = threadIdx.x, L = lane_id(), w = __builtin_amdgcn_readfirstlane(wave_id());
    const int n = L & 15, lg = L >> 4;

    const int pi = a.first < a.last && blockIdx.x >= a.p[0].wgs ? 1 : a.first;
    const SharedPart& P = a.p[pi];
    const WgPlace at = place(P, blockIdx.x - (pi > a.first ? a.p[0].wgs : 0u), a.Hkv);
    const int h = at.h, tile = at.tile, split = at.split, item = at.item;
    const Int4Cache& c = P.c;
    const int code_pages = c.S / kPg;
    const int kg = w / RG;                       // key group
    const int wg_row0 = tile * RT, row0 = wg_row0 + (w % RG) * (16 * QB);

    const bool wave_on = row0 < P.rows;
    const bool several = SEVERAL && pi == 1;     // rows of several query tokens

    int hi[QB], lo = 0, hi_all = P.keys - 1;
    float rs[QB];
    v8h qf[QB][NS];
    if (pi == 1) {
        if (a.start) lo = min(max(a.start[item], 0), P.keys);
        hi_all = P.keys - a.Sq + min(row0, P.rows - 1) / a.G;
    }
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const int row = min(row0 + 16 * qb + n, P.rows - 1);
        const RowPlace r = row_place(row, a.G, a.Sq, pi == 1, item);
        hi[qb] = pi == 1 ? P.keys - a.Sq + r.i : P.keys - 1;
        const uint16_t* q = (const uint16_t*)a.q + r.b * a.q_s[0] + (int64_t)(h * a.G + r.g) * a.q_s[1] + r.i * a.q_s[2];
        u32x4 qr[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) qr[s] = *(const u32x4*)(q + 8 * lg + 32 * s);
        rs[qb] = turn_query<D, BITS>(qr, a.bf16, a.qk_scale, qf[qb]);
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

    // This thread's part of a stage, of its page 2 t + pg: KPT keys' 8 channels of K, or 4 keys' VC
    // channels of V, or both.
    const bool upper = w >= kTW / 2;
    constexpr auto takes_k = [](auto up) { return KG == 1 || !decltype(up)::value; };
    constexpr auto takes_v = [](auto up) { return KG == 1 || decltype(up)::value; };
    const int ti = tid & (TPP - 1), pg = (w >> 2) & 1;
    const int kc = ti % CPR, kr = ti / CPR;      // K: chunk, first key
    const int vc = ti & 15, vt = ti >> 4;        // V: channels VC vc .., keys 4 vq .. (a wave's four vq fill whole 16-byte chunks)
    const int vq = (vt & 8) | (vt & 1) << 2 | ((vt >> 1) & 3);
    const uint8_t* kb = c.kp + item * c.kp_s[1] + h * c.kp_s[2] + kr * c.kp_s[3] + kc * BITS;
    const uint8_t* vb = c.vp + item * c.vp_s[1] + h * c.vp_s[2] + vc * (VC * BITS / 8) + 4 * vq * c.vp_s[3];
    struct Raw { uint32_t k[KPT * KW], v[4 * VW]; };
    // and of its metadata: K's scale or minimum of one channel, V's of one token in groups mg, mg + 2
    const int mt = ti & 63, mg = __builtin_amdgcn_readfirstlane(ti >> 7);
    const bool mv = ti & 64;
    const uint16_t* vmeta = mv ? (const uint16_t*)c.vmn + item * c.vmn_s[1] + h * c.vmn_s[2] + mt * c.vmn_s[3] + mg
                               : (const uint16_t*)c.vsc + item * c.vsc_s[1] + h * c.vsc_s[2] + mt * c.vsc_s[3] + mg;
    const int64_t vmeta_s = kPg * (mv ? c.vmn_s[3] : c.vsc_s[3]);
    const float vmeta_f = mv ? 1.f : kCodeUp<BITS>;
    auto slot = [](int ch) { return BITS == 4 ? (ch & ~7) | (ch & 3) << 1 | ((ch >> 2) & 1) : ch; };      // operand order
    const int vg = vc * c.G >> 4;
    struct RawMeta { uint32_t k, v[2]; };
    const uint16_t* ksb = (const uint16_t*)c.ksc + item * c.ksc_s[1] + h * c.ksc_s[2] + (ti & (D - 1));
    const uint16_t* kmb = (const uint16_t*)c.kmn + item * c.kmn_s[1] + h * c.kmn_s[2] + (ti & (D - 1));
    const uint16_t* kmeta = ti & D ? kmb : ksb;
    const int64_t kmeta_s = ti & D ? c.kmn_s[3] : c.ksc_s[3];
    const int last_page = max(code_pages - 1, 0);        // later pages are not loaded ahead; S = 0: the host's dummies are read
    auto load_meta = [&](auto up, RawMeta& r, int t) __attribute__((always_inline)) {
        const int page = min(2 * t + pg, last_page);
        if constexpr (takes_v(up)) {
            const uint16_t* v = vmeta + page * vmeta_s;
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (mg + 2 * u < c.G) r.v[u] = v[2 * u];
        }
        if constexpr (takes_k(up)) r.k = kmeta[page * kmeta_s];
    };
    auto put_meta = [&](auto up, const RawMeta& r, int t) __attribute__((always_inline)) {
        if constexpr (takes_v(up)) {
            const bool on = (2 * t + pg) * kPg + mt >= lo;      // values of padding tokens count as 0, whatever they are
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (mg + 2 * u < c.G) s_vm[t & 1][pg][mg + 2 * u][mv][mt] = on ? f_to_f16_bits(meta_f<MT>(r.v[u]) * vmeta_f) : 0;
        }
        if constexpr (takes_k(up)) {
            const bool mn = ti & D;
            if (ti < 2 * D) s_km[t & 1][pg][mn][slot(ti & (D - 1))] = f_to_f16_bits(meta_f<MT>(r.k) * (mn ? kKExp : kCodeUp<BITS> * kKExp));
        }
    };
    auto load = [&](auto up, Raw& r, int t) __attribute__((always_inline)) {    // code pages; the partial one is read when it is written
        const int64_t t0 = (int64_t)min(2 * t + pg, last_page) * kPg;
        if constexpr (takes_k(up)) {
#pragma unroll
            for (int j = 0; j < KPT; ++j) {
                const uint8_t* p = kb + (t0 + TPP / CPR * j) * c.kp_s[3];
                if constexpr (KW == 1) r.k[j] = *(const uint32_t*)p;
                else { const u32x2 x = *(const u32x2*)p; r.k[2 * j] = x.x; r.k[2 * j + 1] = x.y; }
            }
        }
        if constexpr (takes_v(up)) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint8_t* p = vb + (t0 + j) * c.vp_s[3];
                if constexpr (VC * BITS == 16) r.v[j] = *(const uint16_t*)p;
                else if constexpr (VW == 1) r.v[j] = *(const uint32_t*)p;
                else { const u32x2 x = *(const u32x2*)p; r.v[2 * j] = x.x; r.v[2 * j + 1] = x.y; }
            }
        }
    };
    auto put_k = [&](int buf, int j, u32x4 x) __attribute__((always_inline)) {
        *(u32x4*)&s_k[buf][Lds::k_at(kc & 3, kPg * pg + kr + TPP / CPR * j, kc >> 2)] = x;
    };
    const int v_to = Lds::v_at(vq & 3, vc, 2 * pg + (vq >> 3)) + 8 * ((vq >> 2) & 1);
    auto put_v = [&](int buf, int i, u32x2 x) __attribute__((always_inline)) { *(u32x2*)&s_v[buf][v_to + 16 * i * Lds::VROW] = x; };
    auto write_k = [&](const Raw& r, int t) __attribute__((always_inline)) {
        const int page = 2 * t + pg, buf = t & 1;
        if (page < code_pages) {
            const u32x4 sk = *(const u32x4*)&s_km[buf][pg][0][8 * kc], mk = *(const u32x4*)&s_km[buf][pg][1][8 * kc];
#pragma unroll
            for (int j = 0; j < KPT; ++j) {
                uint32_t x[4];
                key_codes<BITS>(&r.k[j * KW], x);
                put_k(buf, j, u32x4{fma_h2(x[0], sk.x, mk.x), fma_h2(x[1], sk.y, mk.y), fma_h2(x[2], sk.z, mk.z), fma_h2(x[3], sk.w, mk.w)});
            }
        } else {                                 // the partial page, its last row repeated past the end; no keys: zeros
            const TailArgs& tl = P.t;
            const uint16_t* kt = (const uint16_t*)tl.k + item * tl.ks[1] + h * tl.ks[2] + 8 * kc;
#pragma unroll
            for (int j = 0; j < KPT; ++j) {
                u32x4 x = {0u, 0u, 0u, 0u};
                if (page * kPg < P.keys) x = tail_keys<BITS>(kt + (int64_t)min(kr + TPP / CPR * j, tl.len - 1) * tl.ks[3]);
                put_k(buf, j, x);
            }
        }
    };
    auto put_bad = [&](int buf, u32x2 b) __attribute__((always_inline)) {      // of any of a token's 16 threads
        uint32_t any[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            any[j] = (uint32_t)(__builtin_amdgcn_ballot_w64((b[j >> 1] >> (16 * (j & 1)) & 1u) != 0) >> (L & 48)) & 0xFFFFu ? 0xFFFFu : 0u;
        if (vc == 0) *(u32x2*)&s_bad[buf][pg][4 * vq] = u32x2{any[0] | any[1] << 16, any[2] | any[3] << 16};
    };
    auto write_v = [&](const Raw& r, int t) __attribute__((always_inline)) {
        const int page = 2 * t + pg, buf = t & 1;
        if (page < code_pages) {
            u32x2 sv = *(const u32x2*)&s_vm[buf][pg][vg][0][4 * vq], mv = *(const u32x2*)&s_vm[buf][pg][vg][1][4 * vq];
            if (several) {
                asm volatile("");
                const u32x2 b = {not_finite(sv.x, mv.x), not_finite(sv.y, mv.y)};
                sv = u32x2{sv.x & ~b.x, sv.y & ~b.y};
                mv = u32x2{mv.x & ~b.x, mv.y & ~b.y};
                put_bad(buf, b);
            }
#pragma unroll
            for (int i = 0; i < VC; ++i) {
                const int d = BITS == 8 ? i >> 2 : 0;
                put_v(buf, i, u32x2{fma_h2(value_pair<BITS>(r.v[d], r.v[VW + d], i), sv.x, mv.x),
                                    fma_h2(value_pair<BITS>(r.v[2 * VW + d], r.v[3 * VW + d], i), sv.y, mv.y)});
            }
        } else {                                 // past the end: masked, and values of 0
            const TailArgs& tl = P.t;
            const uint16_t* vt = (const uint16_t*)tl.v + item * tl.vs[1] + h * tl.vs[2] + VC * vc;
            uint32_t x[4][VC / 2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = page * kPg + 4 * vq + j;
#pragma unroll
                for (int k = 0; k < VC / 2; ++k) x[j][k] = 0u;
                if (key >= lo && key < P.keys) {
                    const uint32_t* p = (const uint32_t*)(vt + (int64_t)(4 * vq + j) * tl.vs[3]);
#pragma unroll
                    for (int k = 0; k < VC / 2; ++k) x[j][k] = p[k];
                }
            }
            if (several) {
                asm volatile("");
                uint32_t b[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    b[j] = tail_not_finite(x[j]) ? 0xFFFFu : 0u;
#pragma unroll
                    for (int k = 0; k < VC / 2; ++k) x[j][k] = b[j] ? 0u : x[j][k];
                }
                put_bad(buf, u32x2{b[0] | b[1] << 16, b[2] | b[3] << 16});
            }
#pragma unroll
            for (int i = 0; i < VC; ++i)
                put_v(buf, i, u32x2{tail_pair(x[0][i >> 1], x[1][i >> 1], i & 1), tail_pair(x[2][i >> 1], x[3][i >> 1], i & 1)});
        }
    };

    // Operand addresses of the lane: row n (rows 16 apart are a constant apart).
    int k_lane[NS];
#pragma unroll
    for (int st = 0; st < NS; ++st) k_lane[st] = Lds::k_at(lg, n, st);
    const int v_lane = Lds::v_at(lg, n, 0);      // its chunk bits XORed with the key block's
    static_assert(Lds::VPL % Lds::VROW == 0, "chunk bits are the low ones of a row");

    // The two products of a wave's 64 keys from key `k0` of a stage on.
    auto qk = [&](const uint8_t* sk, int k0, v4f (&s)[QB][NK]) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < NK; ++kb)
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) s[qb][kb] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < NS; ++st)
#pragma unroll
            for (int kb = 0; kb < NK; ++kb) {
                const v8h k = *(const v8h*)(sk + k_lane[st] + (k0 + 16 * kb) * Lds::KROW);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) s[qb][kb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qf[qb][st], s[qb][kb], 0, 0, 0);
            }
        reads_ahead<NS * NK, AHEAD, QB>();
    };
    auto pv = [&](const uint8_t* sv, int k0, const v8h (&pb)[QB][NJ]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const v8h v = *(const v8h*)(sv + (v_lane ^ 16 * (k0 / 32 + j)) + 16 * i * Lds::VROW);
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) o[qb][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pb[qb][j], o[qb][i], 0, 0, 0);
            }
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) ol[qb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ones, pb[qb][j], ol[qb], 0, 0, 0);
        }
        reads_ahead<NT * NJ, AHEAD, QB>();
        __builtin_amdgcn_sched_group_barrier(0x008, QB * NJ, 0);
    };

    // Stages of this workgroup: those of its split with keys between the first and the last
    // row's last.
    const int hi_top = pi == 1 ? P.keys - a.Sq + min(wg_row0 + RT - 1, P.rows - 1) / a.G : P.keys - 1;
    const int t_begin = max(split * P.per_split, lo / kST);
    const int t_end = min(min((split + 1) * P.per_split, (P.pages + 1) / 2), hi_top / kST + 1);
    auto run = [&](auto up) __attribute__((always_inline)) {
        constexpr bool UP = decltype(up)::value;
        Raw raw;
        RawMeta meta = {};
        auto write = [&](int t) __attribute__((always_inline)) {         // stage t, and what comes after it
            if constexpr (takes_k(up)) write_k(raw, t);
            if constexpr (takes_v(up)) write_v(raw, t);
            put_meta(up, meta, t + 1);           // stage t - 1's place: nobody has read that since the last barrier
            load(up, raw, t + 1);
            load_meta(up, meta, t + 2);
        };
        load_meta(up, meta, t_begin);
        load(up, raw, t_begin);
        put_meta(up, meta, t_begin);
        load_meta(up, meta, t_begin + 1);
        lds_barrier();
        write(t_begin);
        lds_barrier();
        for (int t = t_begin; t < t_end; ++t) {
            const int buf = t & 1;
            // a SIMD's waves take their vector-only part at opposite ends of the stage
            if (UP && t + 1 < t_end) write(t + 1);
            if (wave_on) {
                const int k0 = kg * (kST / KG);
                v8h pb[QB][NJ];
#pragma unroll 1
                for (int u = 0; u < NSUB; ++u) {
                    v4f s[QB][NK];
                    qk(s_k[buf], k0 + kPg * u, s);
                    const int key0 = t * kST + k0 + kPg * u;
                    if (key0 < lo || key0 + kPg - 1 > hi_all) mask_step(s, key0 + 4 * lg, lo, hi);
                    softmax_step(s, rs, m_run, o, ol, pb);
                    __builtin_amdgcn_sched_barrier(0);
                    pv(s_v[buf], k0 + kPg * u, pb);
                    __builtin_amdgcn_sched_barrier(0);
                    if (several) {
                        asm volatile("");
                        u32x2 bad[4];
#pragma unroll
                        for (int T = 0; T < 4; ++T) bad[T] = *(const u32x2*)&s_bad[buf][(k0 + kPg * u) / kPg][16 * T + 4 * lg];
                        spoil_rows(bad, pb, o);
                    }
                }
            }
            if (!UP && t + 1 < t_end) write(t + 1);
            lds_barrier();
        }
    };
    if (t_begin < t_end) {
        if (upper) run(std::true_type{});
        else run(std::false_type{});
    }

    // The key groups' states of a row group meet in key group 0's wave.
    if constexpr (KG > 1) {
        constexpr int NSL = QB * NT, kHalf = 2 * Lds::KB / 16;       // of each of the K and V buffers
        static_assert((kTW - RG) * NSL * 64 * 16 <= 2 * kHalf * 16, "states fit the stage buffers");
        __shared__ float2 s_ml[(kTW - RG) * QB * 64];
        v4f* st0 = (v4f*)&s_k[0][0];
        v4f* st1 = (v4f*)&s_v[0][0];
        auto state = [&](int i) -> v4f* { return i < kHalf ? st0 + i : st1 + (i - kHalf); };
        if (kg > 0) {
            const int src = w - RG;
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
                for (int i = 0; i < NT; ++i) *state((src * NSL + qb * NT + i) * 64 + L) = o[qb][i];
                s_ml[(src * QB + qb) * 64 + L] = make_float2(m_run[qb], ol[qb][0]);
            }
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            float m[KG], l[KG], mm = m_run[qb];
            m[0] = m_run[qb]; l[0] = ol[qb][0];
#pragma unroll
            for (int u = 1; u < KG; ++u) {
                const float2 x = s_ml[(((u - 1) * RG + w) * QB + qb) * 64 + L];
                m[u] = x.x; l[u] = x.y;
                mm = fmaxf(mm, m[u]);
            }
            const float mu = mm == -INFINITY ? 0.f : mm;
            float wt[KG], ls = 0.f;
#pragma unroll
            for (int u = 0; u < KG; ++u) {
                wt[u] = __builtin_amdgcn_exp2f(m[u] - mu);
                ls = fmaf(wt[u], l[u], ls);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                v4f t = o[qb][i] * wt[0];
#pragma unroll
                for (int u = 1; u < KG; ++u) {
                    const v4f y = *state((((u - 1) * RG + w) * NSL + qb * NT + i) * 64 + L);
#pragma unroll
                    for (int r = 0; r < 4; ++r) t[r] = fmaf(wt[u], y[r], t[r]);
                }
                o[qb][i] = t;
            }
            m_run[qb] = mm;
            ol[qb][0] = ls;
        }
    }
    const int64_t base = ((int64_t)(item * a.Hkv + h) * P.splits + split) * P.rows;
    const int64_t all = (int64_t)P.items * a.Hkv * P.splits * P.rows;
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const int row = row0 + 16 * qb + n;
        if (row >= P.rows) continue;
        float* dst = P.part + (base + row) * D + (D / 4) * lg;
#pragma unroll
        for (int r = 0; r < 4; ++r)              // channels D/16 (4 lg + r) + i
#pragma unroll
            for (int i = 0; i < NT; i += 4)
                *(v4f*)(dst + NT * r + i) = v4f{o[qb][i][r], o[qb][i + 1][r], o[qb][i + 2][r], o[qb][i + 3][r]};
        if (lg == 0) *(float2*)(P.part + all * D + 2 * (base + row)) = make_float2(m_run[qb], ol[qb][0]);
    }
}

// Joins the shares of a row: prefix splits, then suffix splits; 33 MB of shares in 9.5 us (3.5 TB/s).  D/4 lanes take four channels
// each of every MG-th share (its loads all go out before the first is used: the kernel is
// little but the latency of reading the shares), and the MG groups meet in LDS, in order.
template <int D, int MG>
__global__ __launch_bounds__(kThreads) void shared_merge_kernel(SharedParams a) {
    constexpr int LPR = D / 4, RPB = kThreads / (LPR * MG), NL = 8;
    __shared__ v4f s_o[MG][RPB][LPR];            // (group 0's stays in its registers)
    __shared__ float2 s_ml[MG][RPB];
    const int ln = threadIdx.x % LPR, mg = threadIdx.x / LPR % MG, rb = threadIdx.x / (LPR * MG);
    const uint32_t rows = a.B * a.Hq * a.Sq, at = blockIdx.x * RPB + rb;
    const bool on = at < rows;
    const int ch = 4 * ln;
    // rows as the prefix has them: ((kv head, b), i, g)
    const uint32_t idx = min(at, rows - 1), h = idx / a.p[0].rows, prow = idx - h * a.p[0].rows;
    const RowPlace rp = row_place(prow, a.G, a.Sq, false, 0);
    const int g = rp.g, i = rp.i, b = rp.b;
    const int n0 = a.p[0].splits, n = n0 + a.p[1].splits;
    const int64_t all0 = (int64_t)a.Hkv * n0 * a.p[0].rows, all1 = (int64_t)a.p[1].items * a.Hkv * a.p[1].splits * a.p[1].rows;
    const int64_t base0 = (int64_t)h * n0 * a.p[0].rows + prow;
    const int64_t base1 = (int64_t)(b * a.Hkv + h) * a.p[1].splits * a.p[1].rows + i * a.G + g;
    float M = -INFINITY, l = 0.f;
    v4f o = {0.f, 0.f, 0.f, 0.f};
    auto join = [&](float m, float pl, v4f x) __attribute__((always_inline)) {
        const float mn = fmaxf(M, m);
        if (mn == -INFINITY) {           // nothing so far, but a NaN stays one
            l += pl;
            o += x;
            return;
        }
        const float wa = __builtin_amdgcn_exp2f(M - mn), wb = __builtin_amdgcn_exp2f(m - mn);
        M = mn;
        l = fmaf(wb, pl, wa * l);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = fmaf(wb, x[r], wa * o[r]);
    };
    for (int s0 = mg; s0 < n; s0 += MG * NL) {
        float2 ml[NL];
        v4f x[NL];
#pragma unroll
        for (int u = 0; u < NL; ++u) {
            const int sp = s0 + MG * u;
            if (sp >= n) break;
            const bool pre = sp < n0;
            const float* part = pre ? a.p[0].part : a.p[1].part;
            const int64_t at = pre ? base0 + (int64_t)sp * a.p[0].rows : base1 + (int64_t)(sp - n0) * a.p[1].rows;
            ml[u] = *(const float2*)(part + (pre ? all0 : all1) * D + 2 * at);
            x[u] = *(const v4f*)(part + at * D + ch);
        }
#pragma unroll
        for (int u = 0; u < NL; ++u) {
            if (s0 + MG * u >= n) break;
            join(ml[u].x, ml[u].y, x[u]);
        }
    }
    if constexpr (MG > 1) {
        if (mg > 0) {
            s_o[mg][rb][ln] = o;
            if (ln == 0) s_ml[mg][rb] = make_float2(M, l);
        }
        __syncthreads();
    }
    if (mg > 0 || !on) return;
#pragma unroll
    for (int u = 1; u < MG; ++u) {
        const float2 ml = s_ml[u][rb];
        join(ml.x, ml.y, s_o[u][rb][ln]);
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

// How a part's rows are taken: 16 rows a wave (kg 0: shared_attn_kernel), or 256 / kg rows a
// workgroup over stages in LDS (kg 1, 2: shared_tile_kernel).
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A part under a form; `pages_a_wg`: what a workgroup of 16-row waves should take.
void plan_part(SharedPart& p, int Hkv, int kg, int64_t pages_a_wg) {
    const int rt = kg ? 256 / kg : 16;
    p.tiles = (int)ceil_div(p.rows, rt);
    p.pages = (int)ceil_div(p.keys, kPg);
    const int64_t groups = (int64_t)p.items * Hkv * p.tiles;
    if (kg) {       // one workgroup a CU; at least four pages each
        const int stages = (int)ceil_div(p.pages, 2);
        const int64_t s = std::min(std::max<int64_t>(1, 256 / groups), ceil_div(p.pages, 4));
        p.per_split = (int)ceil_div(stages, s);
        p.splits = (int)ceil_div(stages, p.per_split);
    } else {
        p.per_split = (int)std::min<int64_t>(p.pages, pages_a_wg);
        p.splits = (int)ceil_div(p.pages, p.per_split);
    }
    p.wgs = (uint32_t)(groups * p.splits);
}

// Forms of the two parts and their plans: the least time by a model, in us, fitted to 80 batches (32 ..
// 512 rows over 2048 .. 32768 tokens, suffixes of 1 and 1024, both widths and head sizes), each measured
// in five pairs of forms; what it takes is within 1 % of the best pair on average, and at most 11 %
// behind.  D = 128, INT4:
//   64 rows over 32768 tokens    35 with 16-row waves, 36 and 42 with row tiles of 128 and 256
//   128 rows                     55, 46 and 48
//   512 rows over 2048           31, 42 and 45
//   512 rows over 32768          174, 108 and 100
void plan_forms(SharedParams& a, int D, int bits, int (&kg)[2]) {
    const int slots = 256 * attn_waves(D);       // workgroups of 16-row waves that run at once
    constexpr double launch = 7., round = 3.2;   // a launch; a round of workgroups of 16-row waves
    const double wave = D == 64 ? 0.65e-3 : bits == 4 ? 0.9e-3 : 1.05e-3;                // a page of a 16-row wave
    const double first[3] = {0., 7., 4.};       // a row tile's start and shares, a stage of it
    const double stage[3] = {0., D == 128 ? 3.7 : 2.9, D == 128 ? 2.1 : 1.6};
    double best = 0.;
    SharedPart plan[2];
    for (int k0 = 0; k0 < 3; ++k0)
        for (int k1 = 0; k1 < 3; ++k1) {
            SharedPart p[2] = {a.p[0], a.p[1]};
            const int k[2] = {k0, k1};
            int64_t pages = 0, wgs = 0;          // of 16-row waves
            for (int i = 0; i < 2; ++i)
                if (!k[i]) pages += p[i].items * a.Hkv * ceil_div(p[i].rows, 16) * ceil_div(p[i].keys, kPg);
            const int64_t each = std::max<int64_t>(1, ceil_div(pages, kW * slots)) * kW;         // the waves take as many
            double t = (k0 == k1 ? 1 : 2) * launch + (double)pages * wave;
            for (int i = 0; i < 2; ++i) {
                plan_part(p[i], a.Hkv, k[i], each);
                if (k[i]) t += (double)ceil_div(p[i].wgs, 256) * (p[i].per_split * stage[k[i]] + first[k[i]]);
                else wgs += p[i].wgs;
            }
            if (wgs) t += round * std::max(1., (double)wgs / slots);
            if (best == 0. || t < best) {
                best = t;
                kg[0] = k0; kg[1] = k1;
                plan[0] = p[0]; plan[1] = p[1];
            }
        }
    a.p[0] = plan[0];
    a.p[1] = plan[1];
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
    a.Hkv = pc.Hkv;
    for (SharedPart& p : a.p) {
        if (p.c.S) continue;
        // no whole page: the loads that run ahead read the first query's channels, and nobody uses them
        p.c.kp = p.c.vp = (const uint8_t*)q.q;
        p.c.ksc = p.c.kmn = p.c.vsc = p.c.vmn = q.q;
        for (int i = 0; i < 4; ++i) p.c.kp_s[i] = p.c.vp_s[i] = p.c.ksc_s[i] = p.c.kmn_s[i] = p.c.vsc_s[i] = p.c.vmn_s[i] = 0;
    }
    int kg[2];
    plan_forms(a, pc.D, pc.bits, kg);
    if (!ws) {
        *bytes = (part_floats(a.p[0], pc.Hkv, pc.D) + part_floats(a.p[1], pc.Hkv, pc.D)) * sizeof(float);
        return hipSuccess;
    }
    a.p[0].part = (float*)ws;
    a.p[1].part = a.p[0].part + part_floats(a.p[0], pc.Hkv, pc.D);
    a.q = q.q; a.out = q.out; a.lse = q.lse; a.start = q.start;
    for (int i = 0; i < 3; ++i) { a.q_s[i] = q.q_strides[i]; a.o_s[i] = q.o_strides[i]; a.lse_s[i] = q.lse_strides[i]; }
    a.bf16 = q.dtype == FQ_BF16;
    a.B = q.B; a.Hq = q.H_q; a.G = G; a.Sq = q.S_q;
    a.qk_scale = qk_scale;
    auto attend = [&](int first, int last, int kg) {
        a.first = first; a.last = last;
        const dim3 grid((first == 0 ? a.p[0].wgs : 0) + (last == 1 ? a.p[1].wgs : 0));
        const bool bf = pc.meta_dtype == FQ_BF16, sev = a.Sq > 1 && last == 1;
#define FQ_SP(D_, B_)                                                                                                  \
    if (pc.D == D_ && pc.bits == B_ && kg == 0) {                                                                      \
        if (bf) hipLaunchKernelGGL((shared_attn_kernel<D_, B_, bf16>), grid, dim3(64 * kW), 0, st, a);                 \
        else hipLaunchKernelGGL((shared_attn_kernel<D_, B_, f16>), grid, dim3(64 * kW), 0, st, a);                     \
        return hipGetLastError();                                                                                      \
    }
#define FQ_ST(D_, B_, K_)                                                                                              \
    if (pc.D == D_ && pc.bits == B_ && kg == K_) {                                                                     \
        if (bf && !sev) hipLaunchKernelGGL((shared_tile_kernel<D_, B_, bf16, K_, false>), grid, dim3(64 * tile_waves(K_)), 0, st, a); \
        else if (!sev) hipLaunchKernelGGL((shared_tile_kernel<D_, B_, f16, K_, false>), grid, dim3(64 * tile_waves(K_)), 0, st, a);   \
        else if (bf) hipLaunchKernelGGL((shared_tile_kernel<D_, B_, bf16, K_, true>), grid, dim3(64 * tile_waves(K_)), 0, st, a);     \
        else hipLaunchKernelGGL((shared_tile_kernel<D_, B_, f16, K_, true>), grid, dim3(64 * tile_waves(K_)), 0, st, a);              \
        return hipGetLastError();                                                                                      \
    }
#define FQ_SPQ(D_, B_) FQ_SP(D_, B_) FQ_ST(D_, B_, 1) FQ_ST(D_, B_, 2)
        FQ_SPQ(128, 4) FQ_SPQ(128, 8) FQ_SPQ(64, 4) FQ_SPQ(64, 8)
#undef FQ_SPQ
#undef FQ_ST
#undef FQ_SP
        return hipErrorInvalidValue;
    };
    hipError_t e;
    if (kg[0] == kg[1]) {
        e = attend(0, 1, kg[0]);
    } else {
        e = attend(0, 0, kg[0]);
        if (e == hipSuccess) e = attend(1, 1, kg[1]);
    }
    if (e != hipSuccess) return e;
    const int64_t rows = (int64_t)q.B * q.H_q * q.S_q;
    // four groups of lanes a row where there are shares for them
    const int mg = a.p[0].splits + a.p[1].splits > 8 ? 4 : 1;
    const dim3 grid((unsigned)ceil_div(rows, kThreads / (pc.D / 4 * mg)));
    if (pc.D == 128 && mg == 4) hipLaunchKernelGGL((shared_merge_kernel<128, 4>), grid, dim3(kThreads), 0, st, a);
    else if (pc.D == 128) hipLaunchKernelGGL((shared_merge_kernel<128, 1>), grid, dim3(kThreads), 0, st, a);
    else if (mg == 4) hipLaunchKernelGGL((shared_merge_kernel<64, 4>), grid, dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((shared_merge_kernel<64, 1>), grid, dim3(kThreads), 0, st, a);
    return hipGetLastError();
}

}  // namespace fq
