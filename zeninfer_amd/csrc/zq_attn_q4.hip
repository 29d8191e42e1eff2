// zq_attn_q4.hip -- attention over the 4-bit KV cache of include/zq_kv.h.
//
// Rows are (query token, head of the kv head) pairs, r = t * G + g, of one
// (sequence, kv head): the G heads that share keys are rows of one matrix
// product, so a held row is read and decoded once for all of them.
//
//   s[r][p] = scale * q_r . k_p        p < visible(r)
//   out[r]  = sum_p exp(s - lse) v_p,  lse = log sum_p exp(s)
//   weight[p] (+)= sum_r exp(s - lse)
//
// The held values are exact in fp16 (11 significant bits), so they are single
// operands of the f16 MFMA; queries and softmax weights are fp32 and go in as two
// fp16 parts h + l (22 bits), accumulated in fp32.
#include "../../include/zq_hip.h"
#include "zq_attn_q4_at.hpp"
#include "zq_internal.hpp"
#include "zq_kv.hpp"

#include <math.h>

#include <algorithm>

namespace zq {
namespace {

typedef float v4f_t __attribute__((ext_vector_type(4)));

struct AttnQ4 {
    zq_kv_q4 c;
    const float* q;
    float* out;
    const int32_t* lens;
    const int32_t* counts;
    size_t stride;      // floats between the query tokens
    float* part;        // partial outputs [head][row][split][D], where splits > 1
    float* part_ml;     // their (max, sum) pairs [head][row][split][2]
    float* lse;         // [head][row], log2 units, where weights are wanted
    float* sc;          // with at most kScoreRows rows: their scores [head][row][capacity], log2 units
    // with many rows: the query operands [head][row][2 parts][D], rows padded to
    // whole tiles, and the factors that take their scale off
    _Float16* qop;
    float* qinv;
    uint32_t rows_pad;
    float scale2;       // scale * log2(e): scores are in log2 units
    uint32_t tokens, G, KH, heads_kv;  // heads_kv = seqs * KH
    uint32_t rows;      // tokens * G
    uint32_t splits;
    int full, add, many;
};

// What a sequence's rows see.
struct Seq {
    uint32_t s, kh, head, live, len;
};
__device__ __forceinline__ Seq seq_of(const AttnQ4& a, uint32_t head) {
    Seq x;
    x.head = head;
    x.s = head / a.KH;
    x.kh = head % a.KH;
    const int32_t n = a.counts ? a.counts[x.s] : int32_t(a.tokens);
    x.live = uint32_t(min(max(n, 0), int32_t(a.tokens)));  // live query tokens
    x.len = uint32_t(clamp_len(a.lens[x.s], a.c.capacity));
    return x;
}
// slots that query token t sees
__device__ __forceinline__ uint32_t visible(const AttnQ4& a, const Seq& x, uint32_t t) {
    return a.full ? x.len : uint32_t(min(uint64_t(x.len) + t + 1, uint64_t(a.c.capacity)));
}

// A weight as two fp16 parts.  unit is 1.0f in a register (unit_factor()): with a
// factor that the compiler does not know, the difference and its rounding are one
// v_fma_mix instruction.
__device__ __forceinline__ float unit_factor() {
    float x = 1.0f;
    asm("" : "+v"(x));
    return x;
}
// (two at a time: the packed conversion's result is what the differences read)
__device__ __forceinline__ void split_p2(float p0, float p1, float unit, h8_t& h, h8_t& l, int i) {
    uint32_t u = __builtin_bit_cast(uint32_t, h2_t{_Float16(p0), _Float16(p1)});
    asm("" : "+v"(u));
    const h2_t x = __builtin_bit_cast(h2_t, u);
    h[i] = x.x;
    h[i + 1] = x.y;
    l[i] = _Float16(fmaf(p0, unit, -float(x.x)));
    l[i + 1] = _Float16(fmaf(p1, unit, -float(x.y)));
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float max_groups(float v) {  // over the four lanes that share lane & 15
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float sum_groups(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// ---- few rows: 16 rows a workgroup, keys split over waves and workgroups ----------
// v_mfma_f32_16x16x32_f16 throughout, computed transposed (S^T = K Q^T, O^T = V^T
// P^T) so that nothing crosses lanes between the two products:
//  * lane (i = lane & 15, g = lane >> 4) loads codes of key 8 (i >> 2) + 4 t + (i & 3)
//    of a 32-key tile for the two 16-key products t = 0, 1, the g-th quarter of its
//    row; the dimension that a k slot stands for is the same for K and Q and need not
//    be in order.  Lane (i, g) then holds the scores of row i and keys 8 g ... 8 g + 7;
//  * which is what the second product's B operand wants of it.  Its A operand is V^T:
//    lane (i, g) loads the i-th 1/16 of the rows of keys 8 g ... 8 g + 7 and picks
//    one nibble position of two rows with one v_perm.
// K and V so go from HBM into the operands without LDS, a wave takes whole tiles on
// its own, and the running maximum is only moved (and the sums rescaled) when a score
// passes it by 2^8: weights stay below 2^14, within fp16.
// Bound by the rows' bytes with one row tile and many keys: 64 sequences of up to 8190 rows,
// 8 kv heads x 4, D = 128: 242 MB in 58.3 us, 4.1 TB/s (a large copy: 4.9), with vector
// instructions on 53 % of the issue slots.  By latency with one sequence: 24,001 rows 11.8 us
// (+ 3.9 for joining the splits), 601 rows 6.3 (+ 3.6).  By latency, and by the longest
// sequence, with several row tiles and uneven lengths: 16 sequences of up to 3001 rows, 4 kv heads
// x 7, D = 64, 6 tokens: 14.5 us (+ 5.3), 19 % of the issue slots and the matrix cores busy 4 %
// of the time.  Against the times of their step, tiles two deep on their way cost a wave a SIMD
// (65 for 60 us for the first), two row tiles a workgroup more registers than their shared
// decoding gives (16.5 for 15.2 for the last).
constexpr int kWaves = 4;
constexpr float kShift = 6.0f;  // weights are 2^(s - max + kShift)
constexpr float kSlack = 8.0f;  // how far a score may pass the running maximum

// The k-slot order of a dword's 8 nibbles (nibbles2 of w, w >> 4, w >> 8, w >> 12):
// elements 0, 2, 16, 18, 1, 3, 17, 19 of the block from the dword's first byte on.
__device__ __forceinline__ h8_t dequant8(uint32_t w, h2_t d, uint32_t one) {
    const h2_t a = nibbles2(w, one) * d, b = nibbles2(w >> 4, one) * d, c = nibbles2(w >> 8, one) * d,
               e = nibbles2(w >> 12, one) * d;
    return h8_t{a.x, a.y, b.x, b.y, c.x, c.y, e.x, e.y};
}

template <int D>
struct KTile {  // a wave's part of 32 keys
    static constexpr int KB = D / 8;   // bytes of a row that a lane takes
    static constexpr int KW = KB / 4;  // dwords, one an MFMA step
    static constexpr int NS = KB > 16 ? KB / 16 : 1;  // scales of a lane's part
    uint32_t w[2][KW];
    uint32_t sc[2][NS];
};
template <int D>
struct VTile {
    static constexpr int VB = D / 32;  // bytes of a row that a lane takes
    static constexpr int VW = VB > 4 ? VB / 4 : 1;
    uint32_t w[8][VW];
    h8_t sc;  // of the 8 keys
};

// (a base that is one for the wave, and 32-bit offsets of the lane)
template <int D>
__device__ __forceinline__ void load_k(KTile<D>& t, const AttnQ4& a, uint32_t head, uint32_t key0, int i, int g) {
    using K = KTile<D>;
    const size_t cap = a.c.capacity;
    const uint8_t* w = a.c.k + (size_t(head) * cap + key0) * (D / 2);
    const uint8_t* d = reinterpret_cast<const uint8_t*>(a.c.k_scale + size_t(head) * (D / 32) * cap + key0);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const uint32_t key = uint32_t(8 * (i >> 2) + 4 * u + (i & 3));
        const uint8_t* p = w + (key * (D / 2) + uint32_t(g * K::KB));
        if constexpr (K::KB == 8) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            t.w[u][0] = x.x;
            t.w[u][1] = x.y;
        } else {
#pragma unroll
            for (int j = 0; j < K::KW / 4; ++j) {
                const uint4 x = reinterpret_cast<const uint4*>(p)[j];
                t.w[u][4 * j] = x.x;
                t.w[u][4 * j + 1] = x.y;
                t.w[u][4 * j + 2] = x.z;
                t.w[u][4 * j + 3] = x.w;
            }
        }
#pragma unroll
        for (int j = 0; j < K::NS; ++j)
            t.sc[u][j] = *reinterpret_cast<const uint16_t*>(
                d + (uint32_t((g * K::KB) / 16 + j) * uint32_t(cap) + key) * 2u);
    }
}
template <int D>
__device__ __forceinline__ void load_v(VTile<D>& t, const AttnQ4& a, uint32_t head, uint32_t key0, int i, int g) {
    using V = VTile<D>;
    const size_t cap = a.c.capacity;
    const uint8_t* w = a.c.v + (size_t(head) * cap + key0) * (D / 2);
    const uint8_t* d = reinterpret_cast<const uint8_t*>(a.c.v_scale + size_t(head) * (D / 32) * cap + key0);
    const uint32_t off = uint32_t(8 * g * (D / 2) + i * V::VB);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const uint8_t* p = w + off + uint32_t(k * (D / 2));
        if constexpr (V::VB == 2) t.w[k][0] = *reinterpret_cast<const uint16_t*>(p);
        else if constexpr (V::VB == 4) t.w[k][0] = *reinterpret_cast<const uint32_t*>(p);
        else {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            t.w[k][0] = x.x;
            t.w[k][1] = x.y;
        }
    }
    t.sc = *reinterpret_cast<const h8_t*>(d + (uint32_t((i * V::VB) / 16) * uint32_t(cap) + uint32_t(8 * g)) * 2u);
}
// scores of 32 keys and 16 rows: s[4 u + r] = row i, key 8 g + 4 u + r
template <int D>
__device__ __forceinline__ void scores(const KTile<D>& t, const h8_t (&qh)[D / 32], const h8_t (&ql)[D / 32], uint32_t one,
                                       float (&s)[8]) {
    using K = KTile<D>;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        v4f_t acc = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < K::KW; ++j) {
            const _Float16 d = __builtin_bit_cast(_Float16, uint16_t(t.sc[u][K::NS > 1 ? j / 4 : 0]));
            const h8_t k = dequant8(t.w[u][j], h2_t{d, d}, one);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[j], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[j], acc, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) s[4 * u + r] = acc[r];
    }
}

// Query row r of a (sequence, kv head), as operands: scaled to its own power of two
// (the returned 2^-e takes it off the scores again), split into two fp16 parts.
// Rows past the live ones are zero.
template <int D>
__device__ __forceinline__ float load_q(const AttnQ4& a, const Seq& x, uint32_t r, bool ok, int g, h8_t (&qh)[D / 32],
                                        h8_t (&ql)[D / 32]) {
    constexpr int KB = D / 8;
    const uint32_t t = ok ? r / a.G : 0, hg = ok ? r % a.G : 0;
    const float* q = a.q + (size_t(x.s) * a.tokens + t) * a.stride + size_t(x.kh * a.G + hg) * D;
    float4 v[D / 32][2];
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        const int byte = g * KB + 4 * j, dim = byte / 16 * 32 + byte % 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            v[j][h] = ok ? *reinterpret_cast<const float4*>(q + dim + 16 * h) : make_float4(0, 0, 0, 0);
            v[j][h].x *= a.scale2;
            v[j][h].y *= a.scale2;
            v[j][h].z *= a.scale2;
            v[j][h].w *= a.scale2;
            m = fmaxf(m, fmaxf(fmaxf(fabsf(v[j][h].x), fabsf(v[j][h].y)), fmaxf(fabsf(v[j][h].z), fabsf(v[j][h].w))));
        }
    }
    m = max_groups(m);
    const int e = m > 0.0f ? min(max(15 - __builtin_amdgcn_frexp_expf(m), -120), 120) : 0;
    const float f = pow2f(e);
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        const float o[8] = {v[j][0].x, v[j][0].z, v[j][1].x, v[j][1].z, v[j][0].y, v[j][0].w, v[j][1].y, v[j][1].w};
#pragma unroll
        for (int k = 0; k < 8; ++k) split_h(o[k] * f, qh[j], ql[j], k);
    }
    return pow2f(-e);
}

// Tiles of 32 keys that a row tile's rows see, and how many a split takes.
struct Cut {
    uint32_t keys, tiles, per, used;
};
__device__ __forceinline__ Cut cut_of(const AttnQ4& a, const Seq& x, uint32_t r0) {
    Cut c;
    const uint32_t last = min(r0 + 15, x.live * a.G - 1) / a.G;
    c.keys = visible(a, x, last);
    c.tiles = (c.keys + 31) / 32;
    c.per = max((c.tiles + a.splits - 1) / a.splits, uint32_t(kWaves));
    c.used = max((c.tiles + c.per - 1) / c.per, 1u);
    return c;
}

template <int D>
__global__ __launch_bounds__(kWaves * 64, D == 64 ? 4 : D == 128 ? 3 : 2) void attn_q4_few_kernel(AttnQ4 a) {
    constexpr int NT = D / 16;  // 16-row O^T tiles
    using V = VTile<D>;
    __shared__ float so[kWaves][NT * 4][64];
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    // the (sequence, kv head) runs fastest: with 8 of them, all row tiles and splits
    // of one lie on one XCD and share its L2
    const uint32_t head = blockIdx.x % a.heads_kv, rest = blockIdx.x / a.heads_kv;
    const uint32_t sp = rest % a.splits, r0 = rest / a.splits * 16;
    const Seq x = seq_of(a, head);
    if (r0 >= x.live * a.G) return;
    const Cut cut = cut_of(a, x, r0);
    if (sp >= cut.used) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i = lane & 15, g = lane >> 4;
    const uint32_t r = r0 + i;
    const bool ok = r < x.live * a.G;
    const uint32_t lim = ok ? visible(a, x, r / a.G) : 0;
    // tiles below it need no mask: every live row sees them
    const uint32_t whole = visible(a, x, r0 / a.G) / 32;

    const uint32_t t1 = min((sp + 1) * cut.per, cut.tiles);
    uint32_t t = sp * cut.per + wave;
    // The next tile is loaded as soon as this one's registers are free, K and V apart.
    // Loads past the last tile repeat it: with a branch around them the compiler would
    // have to wait for all that are under way.
    KTile<D> kt;
    VTile<D> vt;
    auto key_of = [&](uint32_t tile) { return min(tile, t1 - 1) * 32; };
    if (t < t1) {
        load_k<D>(kt, a, head, t * 32, i, g);
        load_v<D>(vt, a, head, t * 32, i, g);
    }
    const uint32_t one = code_bits();
    const float unit = unit_factor();
    h8_t qh[D / 32], ql[D / 32];
    const float c = load_q<D>(a, x, r, ok, g, qh, ql);
    v4f_t o[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) o[n] = v4f_t{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    for (; t < t1; t += kWaves) {
        float s[8];
        scores<D>(kt, qh, ql, one, s);
        __builtin_amdgcn_sched_barrier(0);
        load_k<D>(kt, a, head, key_of(t + kWaves), i, g);
        h8_t vsc = vt.sc;
        if (t >= whole) {
            const uint32_t key = t * 32 + 8 * g;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                s[k] = key + k < lim ? s[k] : -INFINITY;
                vsc[k] = key + k < cut.keys ? vsc[k] : _Float16(0);  // rows that hold nothing: their scale may be any bits
            }
        }
        if (a.sc && ok) {
            float4* p = reinterpret_cast<float4*>(a.sc + (size_t(head) * a.rows + r) * a.c.capacity + t * 32 + 8 * g);
            p[0] = make_float4(s[0] * c, s[1] * c, s[2] * c, s[3] * c);
            p[1] = make_float4(s[4] * c, s[5] * c, s[6] * c, s[7] * c);
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), fmaxf(fmaxf(s[4], s[5]), fmaxf(s[6], s[7]))) * c;
        if (__any(mx > m + kSlack)) {
            const float mn = fmaxf(m, max_groups(mx));
            const float f = exp2_(m - (mn == -INFINITY ? 0.0f : mn));  // 0 where nothing was summed yet
            m = mn;
            l *= f;
#pragma unroll
            for (int n = 0; n < NT; ++n) o[n] *= f;
        }
        const float ms = (m == -INFINITY ? 0.0f : m) - kShift;
        h8_t ph, pl;
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
            const float p0 = exp2_(fmaf(s[k], c, -ms)), p1 = exp2_(fmaf(s[k + 1], c, -ms));
            l += p0 + p1;
            split_p2(p0, p1, unit, ph, pl, k);
        }
        h2_t d[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) d[k] = h2_t{vsc[2 * k], vsc[2 * k + 1]};
#pragma unroll
        for (int y = 0; y < V::VB; ++y) {  // byte y of a lane's part: two nibbles, two O^T tiles
            h8_t lo, hi;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t sel = 0x0c000c00u | uint32_t((4 + (y & 3)) << 16) | uint32_t(y & 3);
                const uint32_t u = __builtin_amdgcn_perm(vt.w[2 * k + 1][y / 4], vt.w[2 * k][y / 4], sel);
                const h2_t a0 = nibbles2(u, one) * d[k], a1 = nibbles2(u >> 4, one) * d[k];
                lo[2 * k] = a0.x;
                lo[2 * k + 1] = a0.y;
                hi[2 * k] = a1.x;
                hi[2 * k + 1] = a1.y;
            }
            o[2 * y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, ph, o[2 * y], 0, 0, 0);
            o[2 * y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo, pl, o[2 * y], 0, 0, 0);
            o[2 * y + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, ph, o[2 * y + 1], 0, 0, 0);
            o[2 * y + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(hi, pl, o[2 * y + 1], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        load_v<D>(vt, a, head, key_of(t + kWaves), i, g);
    }
    // ---- the four waves' sums as one ----
    l = sum_groups(l);
    if (g == 0) {
        sm[wave][i] = m;
        sl[wave][i] = l;
    }
    __syncthreads();
    float M = sm[0][i], L = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sm[w][i]);
    const float Ms = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) L += sl[w][i] * exp2_(sm[w][i] - Ms);
    const float f = exp2_(m - Ms);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k) so[wave][n * 4 + k][lane] = o[n][k] * f;
    __syncthreads();
    if (!ok) return;
    const bool direct = cut.used == 1;
    const size_t row = size_t(head) * a.rows + r;
    if (wave == 0 && g == 0) {
        if (!direct) {
            float* ml = a.part_ml + (row * a.splits + sp) * 2;
            ml[0] = M;
            ml[1] = L;
        } else if (a.lse) {
            a.lse[row] = M - kShift + log2f(L);
        }
    }
    float* dst = direct ? a.out + ((size_t(x.s) * a.tokens + r / a.G) * a.KH * a.G + x.kh * a.G + r % a.G) * D
                        : a.part + (row * a.splits + sp) * D;
    const float inv = direct ? (L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L)) : 1.0f;  // no key: 0; NaN stays
    // lane (i, g), register k of tile n = 2 y + h: row i, byte (4 g + k) VB + y of the
    // codes, its low or high nibble.  Wave w takes k = w.
    {
        const int k = wave;
        const int byte = (4 * g + k) * V::VB, dim = byte / 16 * 32 + byte % 16;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[V::VB];
#pragma unroll
            for (int y = 0; y < V::VB; ++y) {
                float t = 0.0f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) t += so[w][(2 * y + h) * 4 + k][lane];
                v[y] = t * inv;
            }
            float* p = dst + dim + 16 * h;
            if constexpr (V::VB == 2) {
                *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
            } else {
#pragma unroll
                for (int y = 0; y < V::VB; y += 4)
                    *reinterpret_cast<float4*>(p + y) = make_float4(v[y], v[y + 1], v[y + 2], v[y + 3]);
            }
        }
    }
}

// ---- many rows: tiles of 128 rows, keys decoded once a tile into LDS ----------------
// v_mfma_f32_32x32x16_f16, transposed as above.  A workgroup takes 128 rows; its
// eight waves stand in four groups of 32 rows, twice, so a SIMD holds two waves whose
// matrix and vector work overlap.  For D <= 128 each half has its 32 keys of every staged
// 64, and their sums are merged at the end.  For D = 256 that would take more than the 256
// registers of a wave: each half has its 128 dimensions of every staged 32 keys, of the
// queries and of the output, and the two waves of a row group exchange their parts of the
// scores through LDS (both then compute the weights).  Four waves with the whole dimension
// each, one a SIMD, took 20 % longer.
//  * the keys of a step are decoded into LDS as fp16, K row-major with the dwords' own
//    element order, V transposed, into two buffers each, one barrier a step: decoding
//    a value takes two vector instructions, which 128 rows share;
//  * row rho of the S^T product reads key rho with bits 2 and 3 exchanged, so that a
//    lane's 16 scores are those of keys 8 h .. 8 h + 7 and 16 + 8 h .. (h = lane >> 5):
//    the B operands of the second product as they are, and V^T is read in 16-byte runs.
// Bound by the matrix products, twice those of the formula as both fp32 factors go in as two
// parts: 1024 tokens behind 7168 rows, 32 heads, D = 128: 258 GF in 250 us, 1.03 PF/s (a
// large f16 product: 1.34), the matrix cores busy 45 % of the time.  A whole prompt of 2048
// tokens takes 83 us, 0.83 PF/s: the first tiles see few keys, and a workgroup takes 5 us to
// stage its queries.  D = 256, 4 sequences of up to 1777 rows, 333 tokens, 4 heads: 41 us + 6
// for joining the splits: one workgroup a CU, of unequal lengths.  Two workgroups of four waves
// a CU instead of one of eight: 99 for 94 us for the prompt, at the clocks of that step.
constexpr uint32_t kTileRows = 128;
typedef float v16f_t __attribute__((ext_vector_type(16)));

template <int D>
struct Big {
    static constexpr int KG = D <= 128 ? 2 : 1;  // 32-key parts of a step, each with waves of its own
    static constexpr int DG = 2 / KG;            // parts of the head dimension, likewise
    static constexpr int T = 512;                // threads
    static constexpr int TK = StageShape<D>::TK;  // keys of a step
    // halves of a K row in LDS: the 16-byte parts of 16 rows lie on banks of their own (counted all the same, over
    // all of the kernel: conflicts are 14 % of the LDS cycles, 24 % at D = 256)
    static constexpr int HP = D + 8;
    static constexpr int KP = TK + 8;            // halves of a V^T row
    static constexpr int NT = D / 32 / DG, KS = D / 16 / DG;  // a wave's tiles of O^T, its steps of a score
    static constexpr int kTasks = StageShape<D>::kTasks;  // blocks of K, and 8-key column groups of V, of a step
    static constexpr size_t kK = size_t(TK) * HP, kV = size_t(D) * KP;  // halves of one buffer of each
    static constexpr size_t kMerge = KG == 2 ? size_t(4) * 64 * (NT * 16 + 2) * 4 : 0;
    static constexpr size_t kQ = size_t(kTileRows) * HP;  // halves of one part of the queries
    static constexpr size_t kSwap = DG == 2 ? size_t(8) * 16 * 64 : 0;  // floats: the waves' parts of a step's scores
    static constexpr size_t kLds = std::max({4 * (kK + kV) + 8 * kSwap, 4 * kQ, kMerge});
    static_assert(TK == 32 * KG && kTasks <= 256 && kTasks % 64 == 0, "one task a thread, whole waves");
};

// Task e of K: key e / (D / 32), block e % (D / 32).  Task e of V: 8 keys, two bytes
// of their rows (four dimensions); the key group's low bit runs fastest, so that the
// 16-byte LDS writes of 16 lanes meet all banks.
template <int D>
struct KStage {
    uint4 w;
    _Float16 d;
};
template <int D>
struct VStage {
    uint16_t w[8];
    h8_t d;
};
template <int D>
__device__ __forceinline__ void load_kstage(KStage<D>& r, const AttnQ4& a, uint32_t head, uint32_t key0, int e) {
    const size_t cap = a.c.capacity;
    const StageAt at = stage_k_at<D>(uint32_t(cap), key0, uint32_t(e));
    // a base that is one for the wave, and 32-bit offsets of the lane
    const uint8_t* w = a.c.k + (size_t(head) * cap + key0) * (D / 2);
    const uint8_t* d = reinterpret_cast<const uint8_t*>(a.c.k_scale + size_t(head) * (D / 32) * cap + key0);
    r.w = *reinterpret_cast<const uint4*>(w + at.codes);
    r.d = *reinterpret_cast<const _Float16*>(d + at.scales);
}
template <int D>
__device__ __forceinline__ void store_kstage(const KStage<D>& r, _Float16* kt, uint32_t one, int e) {
    const int key = e / (D / 32), b = e % (D / 32);
    const h2_t d = {r.d, r.d};
    h8_t* p = reinterpret_cast<h8_t*>(kt + key * Big<D>::HP + b * 32);
    p[0] = dequant8(r.w.x, d, one);
    p[1] = dequant8(r.w.y, d, one);
    p[2] = dequant8(r.w.z, d, one);
    p[3] = dequant8(r.w.w, d, one);
}
template <int D>
__device__ __forceinline__ void load_vstage(VStage<D>& r, const AttnQ4& a, uint32_t head, uint32_t key0, int e) {
    const size_t cap = a.c.capacity;
    const StageAt at = stage_v_at<D>(uint32_t(cap), key0, uint32_t(e));
    const uint8_t* w = a.c.v + (size_t(head) * cap + key0) * (D / 2);
    const uint8_t* d = reinterpret_cast<const uint8_t*>(a.c.v_scale + size_t(head) * (D / 32) * cap + key0);
#pragma unroll
    for (int k = 0; k < 8; ++k) r.w[k] = *reinterpret_cast<const uint16_t*>(w + at.codes + uint32_t(k * (D / 2)));
    r.d = *reinterpret_cast<const h8_t*>(d + at.scales);
}
// MASK: only `keys` of the step's keys hold rows that are seen (the others' scale may be
// any bits)
template <int D, bool MASK>
__device__ __forceinline__ void store_vstage(const VStage<D>& r, _Float16* vt, uint32_t keys, uint32_t one, int e) {
    const StageV task = stage_v_task<D>(uint32_t(e));
    const int ch = int(task.ch), o = int(task.o);
    h8_t s = r.d;
    if (MASK)
#pragma unroll
        for (int k = 0; k < 8; ++k) s[k] = uint32_t(8 * o + k) < keys ? s[k] : _Float16(0);
    const int dim = ch / 8 * 32 + 2 * (ch % 8);
#pragma unroll
    for (int y = 0; y < 2; ++y) {
        h8_t lo, hi;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t u = __builtin_amdgcn_perm(uint32_t(r.w[2 * k + 1]), uint32_t(r.w[2 * k]),
                                                     0x0c000c00u | uint32_t((4 + y) << 16) | uint32_t(y));
            const h2_t d = {s[2 * k], s[2 * k + 1]};
            const h2_t a0 = nibbles2(u, one) * d, a1 = nibbles2(u >> 4, one) * d;
            lo[2 * k] = a0.x;
            lo[2 * k + 1] = a0.y;
            hi[2 * k] = a1.x;
            hi[2 * k + 1] = a1.y;
        }
        *reinterpret_cast<h8_t*>(vt + (dim + y) * Big<D>::KP + 8 * o) = lo;
        *reinterpret_cast<h8_t*>(vt + (dim + y + 16) * Big<D>::KP + 8 * o) = hi;
    }
}

// Steps of `unit` keys that a tile's rows see, and how many a split takes.
__device__ __forceinline__ Cut big_cut(const AttnQ4& a, const Seq& x, uint32_t r0, uint32_t unit) {
    Cut c;
    const uint32_t last = min(r0 + kTileRows - 1, x.live * a.G - 1) / a.G;
    c.keys = visible(a, x, last);
    c.tiles = (c.keys + unit - 1) / unit;
    c.per = max((c.tiles + a.splits - 1) / a.splits, 1u);
    c.used = max((c.tiles + c.per - 1) / c.per, 1u);
    return c;
}

// The tile's query rows into LDS as operands (a row's own power of two taken off, two
// fp16 parts, the dwords' element order): whole rows are read by neighbouring lanes,
// where operand loads straight from memory would touch 64 lines each.
template <int D, int T, int N>
struct QStage {  // what a thread of T holds of N rows
    static constexpr int RL = D / 4, J = N * RL / T;  // lanes of a row, passes
    float4 v[J];
};
template <int D, int T, int N>
__device__ __forceinline__ void load_qstage(QStage<D, T, N>& s, const AttnQ4& a, const Seq& x, uint32_t r0, int tid) {
    using S = QStage<D, T, N>;
#pragma unroll
    for (int j = 0; j < S::J; ++j) {
        const uint32_t r = r0 + uint32_t(j * (T / S::RL) + tid / S::RL);
        const uint32_t t = r / a.G, hg = r % a.G;
        s.v[j] = r < x.live * a.G ? *reinterpret_cast<const float4*>(a.q + (size_t(x.s) * a.tokens + t) * a.stride +
                                                                     size_t(x.kh * a.G + hg) * D + tid % S::RL * 4)
                                  : make_float4(0, 0, 0, 0);
    }
}
template <int D, int T, int N>
__device__ __forceinline__ void store_qstage(const QStage<D, T, N>& s, float scale2, _Float16* hi, _Float16* lo,
                                             float* inv, int tid) {
    using S = QStage<D, T, N>;
    constexpr int HP = D + 8;
    const int l = tid % S::RL, dim = 4 * l;
    const int pos = (dim / 32 * 4 + dim % 16 / 4) * 8 + (dim % 32 >= 16 ? 2 : 0);
#pragma unroll
    for (int j = 0; j < S::J; ++j) {
        const int row = j * (T / S::RL) + tid / S::RL;
        const float4 v = make_float4(s.v[j].x * scale2, s.v[j].y * scale2, s.v[j].z * scale2, s.v[j].w * scale2);
        float m = fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w)));
#pragma unroll
        for (int o = S::RL / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        const int e = m > 0.0f ? min(max(15 - __builtin_amdgcn_frexp_expf(m), -120), 120) : 0;
        const float f = pow2f(e);
        if (l == 0) inv[row] = pow2f(-e);
        h4_t h, w;
        split_h(v.x * f, h, w, 0);
        split_h(v.z * f, h, w, 1);
        split_h(v.y * f, h, w, 2);
        split_h(v.w * f, h, w, 3);
        _Float16* ph = hi + row * HP + pos;
        _Float16* pl = lo + row * HP + pos;
        *reinterpret_cast<h2_t*>(ph) = h2_t{h.x, h.y};
        *reinterpret_cast<h2_t*>(ph + 4) = h2_t{h.z, h.w};
        *reinterpret_cast<h2_t*>(pl) = h2_t{w.x, w.y};
        *reinterpret_cast<h2_t*>(pl + 4) = h2_t{w.z, w.w};
    }
}

template <int D>
__global__ __launch_bounds__(Big<D>::T) void attn_q4_many_kernel(AttnQ4 a) {
    using B = Big<D>;
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ float inv_q[kTileRows];
    const uint32_t head = blockIdx.x % a.heads_kv, rest = blockIdx.x / a.heads_kv;
    const uint32_t sp = rest % a.splits, tiles = (a.rows + kTileRows - 1) / kTileRows;
    const uint32_t r0 = (tiles - 1 - rest / a.splits) * kTileRows;  // the tiles that see most come first
    const Seq x = seq_of(a, head);
    const uint32_t rows = x.live * a.G;
    if (r0 >= rows) return;
    const Cut cut = big_cut(a, x, r0, B::TK);
    if (sp >= cut.used) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31, lh = lane >> 5;
    const int kg = B::KG == 2 ? wave >> 2 : 0, dg = B::DG == 2 ? wave >> 2 : 0;
    const uint32_t rw = r0 + 32 * (wave & 3), r = rw + l32;
    const bool ok = r < rows;
    const uint32_t lim = ok ? visible(a, x, r / a.G) : 0;
    // of the wave's rows: keys that some see, and that all (live ones) see
    const uint32_t most = rw < rows ? visible(a, x, min(rw + 31, rows - 1) / a.G) : 0;
    const uint32_t whole = rw < rows ? visible(a, x, rw / a.G) : 0;

    const uint32_t t0 = sp * cut.per, t1 = min(t0 + cut.per, cut.tiles);
    _Float16* kbuf = reinterpret_cast<_Float16*>(lds);
    _Float16* vbuf = kbuf + 2 * B::kK;
    float* swap = reinterpret_cast<float*>(vbuf + 2 * B::kV) + lane;
    // K by the first 256 threads, V by the others
    const int e = tid & 255;
    const bool kr = tid < 256 && e < B::kTasks, vr = tid >= 256 && e < B::kTasks;
    const int em = min(e, B::kTasks - 1);  // a thread without a task loads the last one's
    const uint32_t one = code_bits();
    const float unit = unit_factor();
    KStage<D> ks;
    VStage<D> vs;
    if (t0 < t1) {
        if (kr) load_kstage<D>(ks, a, head, t0 * B::TK, e);
        if (vr) load_vstage<D>(vs, a, head, t0 * B::TK, e);
    }
    h8_t qh[B::KS], ql[B::KS];
    {
        QStage<D, B::T, int(kTileRows)> qs;
        load_qstage(qs, a, x, r0, tid);
        store_qstage(qs, a.scale2, kbuf, kbuf + B::kQ, inv_q, tid);
    }
    __syncthreads();
    const int qrow = 32 * (wave & 3) + l32;
    const float c = inv_q[qrow];
#pragma unroll
    for (int j = 0; j < B::KS; ++j) {
        qh[j] = *reinterpret_cast<const h8_t*>(kbuf + qrow * B::HP + (dg * B::KS + j) * 16 + 8 * lh);
        ql[j] = *reinterpret_cast<const h8_t*>(kbuf + B::kQ + qrow * B::HP + (dg * B::KS + j) * 16 + 8 * lh);
    }
    if (a.qop && sp == 0) {  // the operands once more, for the weights
        const size_t row = size_t(head) * a.rows_pad + r0;
        h8_t* dst = reinterpret_cast<h8_t*>(a.qop + row * 2 * D);
        constexpr int P = D / 8;  // 16-byte parts of a row's one operand
#pragma unroll 4
        for (int j = tid; j < int(kTileRows) * 2 * P; j += B::T) {
            const int rr = j / (2 * P), part = j / P % 2, e8 = j % P;
            dst[j] = *reinterpret_cast<const h8_t*>(kbuf + part * B::kQ + rr * B::HP + e8 * 8);
        }
        if (tid < int(kTileRows)) a.qinv[row + tid] = inv_q[tid];
    }
    __syncthreads();  // K and V take its place
    v16f_t o[B::NT], s;
#pragma unroll
    for (int n = 0; n < B::NT; ++n)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[n][v] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    if (t0 < t1) {
        if (kr) {
            store_kstage<D>(ks, kbuf + (t0 & 1) * B::kK, one, e);
            if (t0 + 1 < t1) {
                load_kstage<D>(ks, a, head, (t0 + 1) * B::TK, e);
                store_kstage<D>(ks, kbuf + ((t0 + 1) & 1) * B::kK, one, e);
            }
        }
        if (vr) store_vstage<D, true>(vs, vbuf + (t0 & 1) * B::kV, cut.keys - t0 * B::TK, one, e);
    }
    __syncthreads();
    // this lane's part of a K row: bits 2 and 3 of the row exchanged
    const int krow = 32 * kg + ((l32 & 0x13) | (l32 & 4) << 1 | (l32 & 8) >> 1), koff = krow * B::HP + 16 * B::KS * dg + 8 * lh;
    const int voff = (32 * B::NT * dg + l32) * B::KP + 32 * kg + 8 * lh;
    auto product = [&](uint32_t t) {
        const _Float16* kt = kbuf + (t & 1) * B::kK + koff;
        v16f_t y;
#pragma unroll
        for (int v = 0; v < 16; ++v) y[v] = 0.0f;
#pragma unroll
        for (int j = 0; j < B::KS; ++j) {
            const h8_t k = *reinterpret_cast<const h8_t*>(kt + j * 16);
            y = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qh[j], y, 0, 0, 0);
            y = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[j], y, 0, 0, 0);
        }
        return y;
    };
    // DG == 2: a wave's scores are those of its half of the dimension; step t adds the other
    // wave's, who has left them in one of two places by t (what stood there is read in t - 2)
    auto give = [&](uint32_t t) {
        if constexpr (B::DG == 2)
#pragma unroll
            for (int v = 0; v < 16; ++v) swap[(t & 1) * B::kSwap + (wave * 16 + v) * 64] = s[v];
    };
    auto take = [&](uint32_t t) {
        if constexpr (B::DG == 2)
#pragma unroll
            for (int v = 0; v < 16; ++v) s[v] += swap[(t & 1) * B::kSwap + ((wave ^ 4) * 16 + v) * 64];
    };
    if (t0 < t1) {
        s = product(t0);
        give(t0);
    }
    // Step t: the weights of its scores, the next step's scores, the second product and
    // the decoding of later keys (K two steps ahead, V one) stand in one run of code,
    // whose vector and matrix instructions the compiler mixes.  Past the last step the
    // last one is loaded and decoded again, for nothing.
    auto fetch = [&](uint32_t t, auto k_role, auto v_role) {  // what step t decodes
        if constexpr (decltype(k_role)::value) load_kstage<D>(ks, a, head, min(t + 2, t1 - 1) * B::TK, em);
        if constexpr (decltype(v_role)::value) load_vstage<D>(vs, a, head, min(t + 1, t1 - 1) * B::TK, em);
    };
    auto step = [&](uint32_t t, auto k_role, auto v_role, auto last) {
        __syncthreads();  // K of t + 1 and V of t are written, K of t and V of t - 1 are read no more
        auto decode = [&] {
            if (B::kTasks == 256 || e < B::kTasks) {
                if constexpr (decltype(k_role)::value) store_kstage<D>(ks, kbuf + (t & 1) * B::kK, one, e);
                if constexpr (decltype(v_role)::value)
                    store_vstage<D, decltype(last)::value>(vs, vbuf + ((t + 1) & 1) * B::kV,
                                                           cut.keys - min(t + 1, t1 - 1) * B::TK, one, e);
            }
            fetch(t + 1, k_role, v_role);
        };
        const uint32_t key0 = t * B::TK + 32 * kg;
        if (key0 >= most) {  // uniform in the wave, and so for every later step
            decode();
            asm volatile("s_nop 0");  // else the two copies of decode() become one, behind the matrix instructions
            return;
        }
        take(t);
        if (key0 + 32 > whole) {
#pragma unroll
            for (int v = 0; v < 16; ++v) s[v] = key0 + 16 * (v >> 3) + 8 * lh + (v & 7) < lim ? s[v] : -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int v = 1; v < 16; ++v) mx = fmaxf(mx, s[v]);
        mx *= c;
        if (__any(mx > m + kSlack)) {
            const float mn = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32)));
            const float f = exp2_(m - (mn == -INFINITY ? 0.0f : mn));
            m = mn;
            l *= f;
#pragma unroll
            for (int n = 0; n < B::NT; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) o[n][v] *= f;
        }
        const float ms = (m == -INFINITY ? 0.0f : m) - kShift;
        const v16f_t next = product(t + 1);
        h8_t ph[2], pl[2];
#pragma unroll
        for (int v = 0; v < 16; v += 2) {
            const float p0 = exp2_(fmaf(s[v], c, -ms)), p1 = exp2_(fmaf(s[v + 1], c, -ms));
            l += p0 + p1;
            split_p2(p0, p1, unit, ph[v >> 3], pl[v >> 3], v & 7);
        }
        s = next;
        give(t + 1);
        const _Float16* vt = vbuf + (t & 1) * B::kV + voff;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int n = 0; n < B::NT; ++n) {
                const h8_t v = *reinterpret_cast<const h8_t*>(vt + 32 * n * B::KP + 16 * u);
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph[u], o[n], 0, 0, 0);
                o[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl[u], o[n], 0, 0, 0);
            }
        // the last two steps' masked decoding stays apart: mixed in, it costs more registers than there are
        if constexpr (decltype(last)::value) __builtin_amdgcn_sched_barrier(0);
        decode();
    };
    using yes = std::true_type;
    using no = std::false_type;
    uint32_t t = t0;
    if (tid < 256) {
        if (t < t1) fetch(t, yes{}, no{});
        for (; t < t1; ++t) step(t, yes{}, no{}, no{});
    } else {
        if (t < t1) fetch(t, no{}, yes{});
        for (; t + 2 < t1; ++t) step(t, no{}, yes{}, no{});
        for (; t < t1; ++t) step(t, no{}, yes{}, yes{});
    }
    // ---- the two key halves of a row as one ----
    l += __shfl_xor(l, 32);
    float M = m, L = l;
    if constexpr (B::KG == 2) {
        float* mrg = reinterpret_cast<float*>(lds) + size_t(wave & 3) * 64 * (B::NT * 16 + 2);
        __syncthreads();  // the buffers are read no more
        if (kg == 1) {
#pragma unroll
            for (int n = 0; n < B::NT; ++n)
#pragma unroll
                for (int v = 0; v < 16; ++v) mrg[(n * 16 + v) * 64 + lane] = o[n][v];
            mrg[B::NT * 16 * 64 + lane] = m;
            mrg[(B::NT * 16 + 1) * 64 + lane] = l;
        }
        __syncthreads();
        if (kg == 1) return;
        const float m1 = mrg[B::NT * 16 * 64 + lane], l1 = mrg[(B::NT * 16 + 1) * 64 + lane];
        M = fmaxf(m, m1);
        const float Ms = M == -INFINITY ? 0.0f : M;
        const float f0 = exp2_(m - Ms), f1 = exp2_(m1 - Ms);
        L = l * f0 + l1 * f1;
#pragma unroll
        for (int n = 0; n < B::NT; ++n)
#pragma unroll
            for (int v = 0; v < 16; ++v) o[n][v] = o[n][v] * f0 + mrg[(n * 16 + v) * 64 + lane] * f1;
    }
    if (!ok) return;
    const bool direct = cut.used == 1;
    const size_t row = size_t(head) * a.rows + r;
    if (lh == 0 && dg == 0) {
        if (!direct) {
            float* ml = a.part_ml + (row * a.splits + sp) * 2;
            ml[0] = M;
            ml[1] = L;
        } else if (a.lse) {
            a.lse[row] = M - kShift + log2f(L);
        }
    }
    float* dst = (direct ? a.out + ((size_t(x.s) * a.tokens + r / a.G) * a.KH * a.G + x.kh * a.G + r % a.G) * D
                         : a.part + (row * a.splits + sp) * D) + 32 * B::NT * dg;
    const float inv = direct ? (L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L)) : 1.0f;
#pragma unroll
    for (int n = 0; n < B::NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4*>(dst + 32 * n + 8 * j + 4 * lh) =
                make_float4(o[n][4 * j] * inv, o[n][4 * j + 1] * inv, o[n][4 * j + 2] * inv, o[n][4 * j + 3] * inv);
}

// The splits' partial outputs of a row as one, by a workgroup of one wave (many rows,
// few splits) or four: D / 4 lanes take a split's output, so WAVES * 256 / D splits are
// read at a time.  Bound by latency, 3 to 6 us (one wave a row for all: 29 us at 96 splits).
template <int D, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void attn_q4_combine_kernel(AttnQ4 a) {
    constexpr int RL = D / 4, P = 64 * WAVES / RL;
    __shared__ float wgt[128];
    __shared__ float4 sum[P][RL];
    const uint32_t head = blockIdx.x / a.rows, r = blockIdx.x % a.rows;
    const Seq x = seq_of(a, head);
    if (r >= x.live * a.G) return;
    const Cut cut = a.many ? big_cut(a, x, r / kTileRows * kTileRows, Big<D>::TK) : cut_of(a, x, r / 16 * 16);
    if (cut.used == 1) return;  // written by the split itself
    const int tid = threadIdx.x, lane = tid & 63;
    const size_t row = size_t(head) * a.rows + r;
    // every wave finds the maximum and the sum of them all (at most 128 splits)
    const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + row * a.splits;
    const float2 none = make_float2(-INFINITY, 0.0f);
    const float2 p0 = uint32_t(lane) < cut.used ? ml[lane] : none;
    const float2 p1 = uint32_t(lane) + 64 < cut.used ? ml[lane + 64] : none;
    const uint32_t p = uint32_t(tid) / RL, l = uint32_t(tid) % RL;
    const float4* part = reinterpret_cast<const float4*>(a.part + row * a.splits * D) + l;
    constexpr int N = 4;  // splits that a lane has on the way
    float4 v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = p + j * P < cut.used ? part[size_t(p + j * P) * RL] : make_float4(0, 0, 0, 0);
    const float M = wave_max(fmaxf(p0.x, p1.x)), Ms = M == -INFINITY ? 0.0f : M;
    const float w0 = exp2_(p0.x - Ms), w1 = exp2_(p1.x - Ms);
    const float L = wave_sum(p0.y * w0 + p1.y * w1);
    if (tid < 64) {
        wgt[lane] = w0;
        wgt[lane + 64] = w1;
    }
    __syncthreads();
    float4 acc = make_float4(0, 0, 0, 0);
    for (uint32_t j0 = p; j0 < cut.used; j0 += N * P) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float w = j0 + j * P < cut.used ? wgt[j0 + j * P] : 0.0f;
            acc = make_float4(fmaf(v[j].x, w, acc.x), fmaf(v[j].y, w, acc.y), fmaf(v[j].z, w, acc.z), fmaf(v[j].w, w, acc.w));
            const uint32_t n = j0 + (N + j) * P;
            if (n < cut.used) v[j] = part[size_t(n) * RL];
        }
    }
    sum[p][l] = acc;
    __syncthreads();
    if (tid >= RL) return;
#pragma unroll
    for (int j = 1; j < P; ++j) {
        const float4 t = sum[j][l];
        acc = make_float4(acc.x + t.x, acc.y + t.y, acc.z + t.z, acc.w + t.w);
    }
    const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);
    reinterpret_cast<float4*>(a.out + ((size_t(x.s) * a.tokens + r / a.G) * a.KH * a.G + x.kh * a.G + r % a.G) * D)[l] =
        make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    if (a.lse && tid == 0) a.lse[row] = M - kShift + log2f(L);
}

// ---- the rows' weights ----------------------------------------------------------
// At most kScoreRows rows, one row tile (a decode step): the attention kernel has left its
// scores, 4 bytes a row and key beside the key's 72 to 288, and what is left is their sum;
// bound by reading them.  Whole call with its weights, us, scores stored against the
// products of the kernel below: 16 sequences x 8 kv heads, 4000 rows held: D = 128, 4 rows
// 28 / 44, 16 rows 38 / 48, 32 rows (if two row tiles stored theirs) 68 / 68; D = 64, 4 rows
// 23 / 29, 16 rows 32 / 32, 32 rows 54 / 45; D = 256 (4 kv heads) 16 rows 42 / 62.  1 sequence,
// 8000 rows, D = 128, 4 rows: 15 / 18.
constexpr uint32_t kScoreRows = 16;
__global__ __launch_bounds__(256) void attn_q4_weights_sum_kernel(AttnQ4 a) {
    const uint32_t head = blockIdx.x % a.heads_kv, key = (blockIdx.x / a.heads_kv * 256 + threadIdx.x) * 4;
    const Seq x = seq_of(a, head);
    if (!x.live) return;
    const uint32_t rows = x.live * a.G, keys = visible(a, x, x.live - 1);
    if (key >= keys) return;
    float4 v[kScoreRows];
    const float* s = a.sc + size_t(head) * a.rows * a.c.capacity + key;
#pragma unroll
    for (uint32_t r = 0; r < kScoreRows; ++r)
        if (r < rows) v[r] = *reinterpret_cast<const float4*>(s + size_t(r) * a.c.capacity);
    float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t r = 0; r < kScoreRows; ++r) {
        if (r < rows) {
            const float e = a.lse[size_t(head) * a.rows + r];
            const uint32_t n = visible(a, x, r / a.G);
            const float t[4] = {v[r].x, v[r].y, v[r].z, v[r].w};
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) w[i] += key + i < n ? exp2_(t[i] - e) : 0.0f;
        }
    }
    float* dst = a.c.weight + size_t(head) * a.c.capacity + key;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i)
        if (key + i < keys) dst[i] = a.add ? dst[i] + w[i] : w[i];
}

// More rows: S = Q K^T again, with the sums of the rows known (lse): a lane's 16 results are 16
// query rows of one key, so a key's weight is a sum in one register.  A wave keeps 64
// keys (D = 256: 32) as operands; query rows pass by in LDS, 64 at a time.  Every key's sum has one
// owner (or two halves, added in order) and one order.
typedef float acc16_t __attribute__((ext_vector_type(16)));
constexpr int kWgtRows = 64;

template <int D>
struct Wgt {
    static constexpr int HP = D + 8, KS = D / 16;
    static constexpr int KU = D <= 128 ? 2 : 1;           // a wave's keys, by 32: what registers hold
    static constexpr uint32_t kKeys = 128 * KU;           // a workgroup's
    static constexpr size_t kQ = size_t(kWgtRows) * HP;   // halves of one part of the queries
};
// what a row tile's scores need beside the operands
struct __align__(16) WgtMeta {
    float inv[kWgtRows], lse[kWgtRows];
    int32_t lim[kWgtRows];
};
__device__ __forceinline__ void row_meta(WgtMeta& m, const AttnQ4& a, const Seq& x, uint32_t r, int tid) {
    const bool ok = r < x.live * a.G;
    m.lse[tid] = ok ? a.lse[size_t(x.head) * a.rows + r] : INFINITY;  // a row past the live ones: weights 0
    m.lim[tid] = ok ? int32_t(visible(a, x, r / a.G)) : 0;
}
// The wave's keys from key0 on as B operands: lane (l32, lh) holds half a row of keys l32
// and 32 + l32.  The last keys may lie past the capacity: their lanes take its last row.
template <int D>
struct KeyCodes {
    uint4 w[Wgt<D>::KU][D / 64];
    _Float16 d[Wgt<D>::KU][D / 64];
};
template <int D>
__device__ __forceinline__ void load_keys(KeyCodes<D>& k, const AttnQ4& a, uint32_t head, uint32_t key0, int l32, int lh) {
    const size_t cap = a.c.capacity;
#pragma unroll
    for (int u = 0; u < Wgt<D>::KU; ++u) {
        const size_t key = min(size_t(key0) + 32 * u + l32, cap - 1);
        const uint4* p = reinterpret_cast<const uint4*>(a.c.k + (size_t(head) * cap + key) * (D / 2) + lh * (D / 4));
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            k.w[u][j] = p[j];
            k.d[u][j] = __builtin_bit_cast(_Float16, a.c.k_scale[(size_t(head) * (D / 32) + lh * (D / 64) + j) * cap + key]);
        }
    }
}
template <int D>
__device__ __forceinline__ void decode_keys(h8_t (&kf)[Wgt<D>::KU][D / 16], const KeyCodes<D>& k, uint32_t one) {
#pragma unroll
    for (int u = 0; u < Wgt<D>::KU; ++u)
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            const uint4 w = k.w[u][j];
            const h2_t d = {k.d[u][j], k.d[u][j]};
            kf[u][4 * j] = dequant8(w.x, d, one);
            kf[u][4 * j + 1] = dequant8(w.y, d, one);
            kf[u][4 * j + 2] = dequant8(w.z, d, one);
            kf[u][4 * j + 3] = dequant8(w.w, d, one);
        }
}
// scores of 32 rows (q: this lane's row and half) and the wave's keys
template <int D>
__device__ __forceinline__ void row_scores(const _Float16* q, const h8_t (&kf)[Wgt<D>::KU][D / 16],
                                           acc16_t (&s)[Wgt<D>::KU]) {
    constexpr int KU = Wgt<D>::KU;
#pragma unroll
    for (int u = 0; u < KU; ++u)
#pragma unroll
        for (int v = 0; v < 16; ++v) s[u][v] = 0.0f;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
        const h8_t h = *reinterpret_cast<const h8_t*>(q + 8 * j);
        const h8_t l = *reinterpret_cast<const h8_t*>(q + Wgt<D>::kQ + 8 * j);
#pragma unroll
        for (int u = 0; u < KU; ++u) {
            s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(h, kf[u][j], s[u], 0, 0, 0);
            s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(l, kf[u][j], s[u], 0, 0, 0);
        }
    }
}
// their softmax weights onto w.  Result v of a lane: row row0 + 8 (v >> 2) + 4 lh + (v & 3),
// key l32.  CUT: some rows do not see all of the keys.
template <bool CUT, int KU>
__device__ __forceinline__ void add_weights(float (&w)[KU], const acc16_t (&s)[KU], const WgtMeta& m, int row0, int key,
                                            int lh) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int at = row0 + 8 * j + 4 * lh;
        const float4 c = *reinterpret_cast<const float4*>(&m.inv[at]);
        const float4 e = *reinterpret_cast<const float4*>(&m.lse[at]);
        const float cc[4] = {c.x, c.y, c.z, c.w}, ee[4] = {e.x, e.y, e.z, e.w};
        int n[4] = {0, 0, 0, 0};
        if constexpr (CUT) {
            const int4 t = *reinterpret_cast<const int4*>(&m.lim[at]);
            n[0] = t.x, n[1] = t.y, n[2] = t.z, n[3] = t.w;
        }
#pragma unroll
        for (int u = 0; u < KU; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = exp2_(fmaf(s[u][4 * j + i], cc[i], -ee[i]));
                w[u] += !CUT || key + 32 * u < n[i] ? p : 0.0f;
            }
    }
}

// the weight of the key that a lane stands for: both lane halves' rows added, lane = key
template <int KU>
__device__ __forceinline__ float lane_weight(const float (&w)[KU], int lh) {
    float v = w[0] + __shfl_xor(w[0], 32);
    if constexpr (KU == 2) {
        const float t = w[1] + __shfl_xor(w[1], 32);
        v = lh ? t : v;
    }
    return v;
}

// Up to 64 rows, staged once: four waves, which go on to further keys.  Bound by the keys'
// decoding and the exponentials: 16 sequences x 8 kv heads, 4000 rows held, 32 rows, D = 128:
// 24 us (8.4 GF in two parts: 0.35 PF/s).
template <int D>
__global__ __launch_bounds__(256) void attn_q4_weights_few_kernel(AttnQ4 a, uint32_t blocks) {
    using W = Wgt<D>;
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ WgtMeta meta;
    _Float16* qbuf = reinterpret_cast<_Float16*>(lds);
    const uint32_t head = blockIdx.x % a.heads_kv, first = blockIdx.x / a.heads_kv;
    const Seq x = seq_of(a, head);
    if (!x.live) return;
    const uint32_t rows = x.live * a.G, keys = visible(a, x, x.live - 1);
    const uint32_t nb = (keys + W::kKeys - 1) / W::kKeys;
    if (first >= nb) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31,
              lh = lane >> 5;
    const uint32_t one = code_bits();
    // the first keys on their way before the queries, and each next ones before their turn
    auto key_of = [&](uint32_t kb) { return min(kb, nb - 1) * W::kKeys + 32 * W::KU * wave; };
    KeyCodes<D> k;
    load_keys<D>(k, a, head, key_of(first), l32, lh);
    {
        QStage<D, 256, kWgtRows> qs;
        load_qstage(qs, a, x, 0, tid);
        store_qstage(qs, a.scale2, qbuf, qbuf + W::kQ, meta.inv, tid);
        if (tid < kWgtRows) row_meta(meta, a, x, tid, tid);
    }
    __syncthreads();
    for (uint32_t kb = first; kb < nb; kb += blocks) {
        const uint32_t key0 = key_of(kb);
        if (key0 >= keys) break;  // uniform in the wave
        h8_t kf[W::KU][W::KS];
        decode_keys<D>(kf, k, one);
        load_keys<D>(k, a, head, key_of(kb + blocks), l32, lh);
        float w[W::KU] = {};
        for (uint32_t row0 = 0; row0 < rows; row0 += 32) {
            acc16_t s[W::KU];
            row_scores<D>(qbuf + (row0 + l32) * W::HP + lh * (D / 2), kf, s);
            if (key0 + 32 * W::KU > visible(a, x, row0 / a.G)) add_weights<true>(w, s, meta, int(row0), int(key0 + l32), lh);
            else add_weights<false>(w, s, meta, int(row0), int(key0 + l32), lh);
        }
        const float v = lane_weight(w, lh);
        if (lane < 32 * W::KU && key0 + lane < keys) {
            float* dst = a.c.weight + size_t(head) * a.c.capacity + key0 + lane;
            *dst = a.add ? *dst + v : v;
        }
    }
}

// Many rows: eight waves, four on each half of the passing 64
// rows, whose operands the attention kernel has left in memory.  The next tile's
// products stand between this one's exponentials; operands are loaded two tiles ahead.
// Bound by the products: 1024 tokens x 32 heads over 8192 rows, D = 128: 129 GF in two parts
// in 118 us, 1.09 PF/s (a large f16 product: 1.34; with the operands made here again the
// kernel took 233 for 139 us at that step).
template <int D>
__global__ __launch_bounds__(512) void attn_q4_weights_many_kernel(AttnQ4 a) {
    using W = Wgt<D>;
    constexpr int P = D / 8, J = kWgtRows * 2 * P / 512;  // 16-byte parts of a row's one operand; parts a thread moves
    extern __shared__ __align__(16) uint8_t lds[];
    __shared__ WgtMeta meta[3];
    __shared__ float half[256];
    _Float16* qbuf = reinterpret_cast<_Float16*>(lds);
    const uint32_t head = blockIdx.x % a.heads_kv, kb = blockIdx.x / a.heads_kv;
    const Seq x = seq_of(a, head);
    if (!x.live) return;
    const uint32_t rows = x.live * a.G, keys = visible(a, x, x.live - 1);
    if (kb * W::kKeys >= keys) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l32 = lane & 31,
              lh = lane >> 5, kg = wave & 3, rh = wave >> 2;
    const uint32_t one = code_bits(), key0 = kb * W::kKeys + 32 * W::KU * kg;
    const bool mine = key0 < keys;  // uniform in the wave
    // rows before the first token that sees the block's first key see none of it
    const uint32_t ta = a.full || kb * W::kKeys < x.len ? 0 : kb * W::kKeys - x.len;
    const uint32_t t0 = ta * a.G / kWgtRows, t1 = (rows + kWgtRows - 1) / kWgtRows;
    h8_t st[J];
    float st_inv = 0.0f;
    auto fetch = [&](uint32_t t) {  // tile t (past the last one: that again)
        const size_t row = size_t(head) * a.rows_pad + min(t, t1 - 1) * kWgtRows;
        const h8_t* q = reinterpret_cast<const h8_t*>(a.qop + row * 2 * D);
#pragma unroll
        for (int j = 0; j < J; ++j) st[j] = q[tid + j * 512];
        if (tid < kWgtRows) st_inv = a.qinv[row + tid];
    };
    auto put = [&](uint32_t t) {
        _Float16* q = qbuf + (t & 1) * 2 * W::kQ;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int e = tid + j * 512, r = e / (2 * P), part = e / P % 2, e8 = e % P;
            *reinterpret_cast<h8_t*>(q + part * W::kQ + r * W::HP + e8 * 8) = st[j];
        }
        if (tid < kWgtRows) {
            WgtMeta& m = meta[t % 3];
            m.inv[tid] = st_inv;
            row_meta(m, a, x, t * kWgtRows + tid, tid);
        }
    };
    fetch(t0);
    h8_t kf[W::KU][W::KS];
    if (mine) {
        KeyCodes<D> k;
        load_keys<D>(k, a, head, key0, l32, lh);
        decode_keys<D>(kf, k, one);
    }
    put(t0);
    fetch(t0 + 1);
    put(t0 + 1);
    fetch(t0 + 2);
    __syncthreads();
    const int row0 = 32 * rh;
    const _Float16* q = qbuf + (row0 + l32) * W::HP + lh * (D / 2);
    acc16_t s[W::KU];
    if (mine) row_scores<D>(q + (t0 & 1) * 2 * W::kQ, kf, s);
    float w[W::KU] = {};
    for (uint32_t t = t0; t < t1; ++t) {
        __syncthreads();  // tile t + 1 is written, the buffer of tile t is read no more
        if (mine) {
            acc16_t next[W::KU];
            const bool cut = key0 + 32 * W::KU > visible(a, x, min(t * kWgtRows + row0, rows - 1) / a.G);
            if (cut) {
                add_weights<true>(w, s, meta[t % 3], row0, int(key0 + l32), lh);
                row_scores<D>(q + ((t + 1) & 1) * 2 * W::kQ, kf, next);
            } else {
                row_scores<D>(q + ((t + 1) & 1) * 2 * W::kQ, kf, next);
                add_weights<false>(w, s, meta[t % 3], row0, int(key0 + l32), lh);
            }
#pragma unroll
            for (int u = 0; u < W::KU; ++u) s[u] = next[u];
        }
        put(t + 2);  // (past the last tile: written, read no more)
        fetch(t + 3);
    }
    float v = lane_weight(w, lh);
    if (rh == 1) half[64 * kg + lane] = v;
    __syncthreads();
    if (rh == 0 && lane < 32 * W::KU && key0 + lane < keys) {
        v += half[64 * kg + lane];
        float* dst = a.c.weight + size_t(head) * a.c.capacity + key0 + lane;
        *dst = a.add ? *dst + v : v;
    }
}

// Which kernel takes a call, and how many workgroups share a row tile's keys.
struct Plan {
    bool many;
    uint32_t splits;
};
// The 16-row kernel reads and decodes the keys for every 16 rows, the 128-row kernel once,
// but a workgroup of it starts and ends slower (its queries pass through LDS, its sums are
// merged): it pays from more than 48 rows on, three row tiles, where there are row tiles for
// half the CUs.  us, 16-row against 128-row kernel:
//   16 sequences x 8 kv heads, 3000 rows held, D = 128: 48 rows 51 / 53, 64 rows 63 / 54,
//   128 rows 110 / 70; 16 x 4, D = 64: 28 rows 18 / 24, 56 rows 29 / 27; 16 x 4, D = 256:
//   48 rows 51 / 61, 56 rows 71 / 62;  1 sequence x 8, 8000 rows, D = 128: 64 rows 21 / 25,
//   192 rows 33 / 35, 256 rows 40 / 39; 4 x 4, 1777 rows, D = 256: 100 rows 37 / 40, 160
//   rows 46 / 45.
// With weights it takes more than 64 rows, whose weights need its operands (the other way
// holds all rows in LDS).  us, 16-row against 128-row kernel, weights and all: 16 x 8, 4000
// rows held, D = 128: 32 rows 68 / 105, 64 rows 103 / 111; D = 64: 64 rows 69 / 85; 16 x 4,
// D = 256: 64 rows 120 / 149.
Plan plan_of(const zq_kv_q4& c, size_t rows, bool weights) {
    Plan p;
    const size_t heads = c.seqs * c.kv_heads, cus = size_t(device_cu_count());
    p.many = weights ? rows > size_t(kWgtRows)
                     : rows > 48 && heads * ((rows + 15) / 16) > cus / 2;
    const size_t tile = p.many ? kTileRows : 16;
    const size_t base = heads * ((rows + tile - 1) / tile);
    size_t want, most;
    if (p.many) {  // one workgroup a CU
        want = cus / base;
        most = (c.capacity + 255) / 256;
    } else {
        // Two workgroups a CU, or three where that leaves each less to do (192 row tiles: three splits 25.0 us, four
        // 23.0; 8 row tiles, 24,000 rows: two workgroups a CU 15.4, three 16.7; 64, 2000 rows: 15.0 / 17.1).  Where
        // there is a row tile for every CU, three splits even out what sequences of uneven length leave to do (64
        // sequences x 8 of up to 8190 rows: 1 split 76, 2 70, 3 60, 4 63, 6 65 us; 32 x 8 of 4000 rows each: 3 splits
        // 40.8, 6 43.6), fewer from two row tiles a CU on.
        const size_t two = 2 * cus / base, three = 3 * cus / base;
        want = base < cus ? (3 * two < 2 * three ? three : two) : std::min<size_t>(3, (6 * cus + base - 1) / base);
        most = (c.capacity / 32 + kWaves - 1) / kWaves;
    }
    p.splits = uint32_t(std::max<size_t>(1, std::min<size_t>({want, most, 128})));
    return p;
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t pad_rows(size_t rows) { return (rows + kTileRows - 1) / kTileRows * kTileRows; }

}  // namespace

size_t attention_q4_bytes(const zq_kv_q4& c, size_t tokens, size_t heads, int flags) {
    const size_t rows = tokens * (heads / c.kv_heads), all = c.seqs * c.kv_heads * rows;
    const Plan plan = plan_of(c, rows, (flags & ZQ_ATTN_Q4_WEIGHTS) != 0);
    size_t n = 0;
    if (plan.splits > 1) n += up256(all * plan.splits * c.head_dim * 4) + up256(all * plan.splits * 8);
    if (flags & ZQ_ATTN_Q4_WEIGHTS) {
        n += up256(all * 4);
        const size_t pad = c.seqs * c.kv_heads * pad_rows(rows);
        if (plan.many) n += up256(pad * c.head_dim * 4) + up256(pad * 4);
        else if (rows <= kScoreRows) n += up256(all * c.capacity * 4);
    }
    return n;
}

hipError_t launch_attention_q4(const zq_kv_q4& c, const float* q, float* out, size_t tokens, size_t heads, size_t stride,
                               const int32_t* lens, const int32_t* counts, float scale, int flags, void* ws,
                               hipStream_t stream) {
    AttnQ4 a{};
    a.c = c;
    a.q = q;
    a.out = out;
    a.lens = lens;
    a.counts = counts;
    a.stride = stride;
    a.scale2 = float(double(scale) * 1.4426950408889634);
    a.tokens = uint32_t(tokens);
    a.KH = uint32_t(c.kv_heads);
    a.G = uint32_t(heads / c.kv_heads);
    a.heads_kv = uint32_t(c.seqs * c.kv_heads);
    a.rows = uint32_t(tokens) * a.G;
    const Plan plan = plan_of(c, a.rows, (flags & ZQ_ATTN_Q4_WEIGHTS) != 0);
    a.splits = plan.splits;
    a.many = plan.many;
    a.full = (flags & ZQ_ATTN_Q4_FULL) != 0;
    a.add = (flags & ZQ_ATTN_Q4_ADD) != 0;
    const size_t all = size_t(a.heads_kv) * a.rows;
    uint8_t* p = static_cast<uint8_t*>(ws);
    if (a.splits > 1) {
        a.part = reinterpret_cast<float*>(p);
        p += up256(all * a.splits * c.head_dim * 4);
        a.part_ml = reinterpret_cast<float*>(p);
        p += up256(all * a.splits * 8);
    }
    if (flags & ZQ_ATTN_Q4_WEIGHTS) {
        a.lse = reinterpret_cast<float*>(p);
        p += up256(all * 4);
        if (a.many) {
            a.rows_pad = uint32_t(pad_rows(a.rows));
            const size_t pad = size_t(a.heads_kv) * a.rows_pad;
            a.qop = reinterpret_cast<_Float16*>(p);
            p += up256(pad * c.head_dim * 4);
            a.qinv = reinterpret_cast<float*>(p);
        } else if (a.rows <= kScoreRows) {
            a.sc = reinterpret_cast<float*>(p);
        }
    }
    const size_t tile = a.many ? kTileRows : 16;
    const size_t blocks = size_t(a.heads_kv) * a.splits * ((a.rows + tile - 1) / tile);
    const size_t per_block = c.head_dim == 256 ? Wgt<256>::kKeys : Wgt<128>::kKeys;
    const size_t all_blocks = (c.capacity + per_block - 1) / per_block, fill = size_t(device_cu_count()) * 4 / a.heads_kv + 1;
    const size_t wblocks = a.many ? all_blocks : std::min(all_blocks, fill), key_blocks = a.heads_kv * wblocks;
    if (a.many && a.lse && key_blocks * 512 > kMaxThreads) return hipErrorInvalidValue;  // over 150 GB of rows
#define ZQ_ATTN_D(KERNEL, GRID, THREADS)                                                                \
    do {                                                                                                \
        if (c.head_dim == 64) hipLaunchKernelGGL(KERNEL<64>, dim3(uint32_t(GRID)), dim3(THREADS), 0, stream, a);        \
        else if (c.head_dim == 128) hipLaunchKernelGGL(KERNEL<128>, dim3(uint32_t(GRID)), dim3(THREADS), 0, stream, a); \
        else hipLaunchKernelGGL(KERNEL<256>, dim3(uint32_t(GRID)), dim3(THREADS), 0, stream, a);                        \
        const hipError_t e = hipGetLastError();                                                         \
        if (e != hipSuccess) return e;                                                                  \
    } while (0)
    if (a.many) {
#define ZQ_ATTN_MANY(DD)                                                                                          \
    hipLaunchKernelGGL(attn_q4_many_kernel<DD>, dim3(uint32_t(blocks)), dim3(Big<DD>::T), Big<DD>::kLds, stream, a)
        if (c.head_dim == 64) ZQ_ATTN_MANY(64);
        else if (c.head_dim == 128) ZQ_ATTN_MANY(128);
        else ZQ_ATTN_MANY(256);
#undef ZQ_ATTN_MANY
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    } else {
        ZQ_ATTN_D(attn_q4_few_kernel, blocks, kWaves * 64);
    }
    if (a.splits > 1) {
#define ZQ_ATTN_C(DD)                                                                                              \
    do {                                                                                                           \
        if (a.many) hipLaunchKernelGGL((attn_q4_combine_kernel<DD, 1>), dim3(uint32_t(all)), dim3(64), 0, stream, a); \
        else hipLaunchKernelGGL((attn_q4_combine_kernel<DD, 4>), dim3(uint32_t(all)), dim3(256), 0, stream, a);    \
    } while (0)
        if (c.head_dim == 64) ZQ_ATTN_C(64);
        else if (c.head_dim == 128) ZQ_ATTN_C(128);
        else ZQ_ATTN_C(256);
#undef ZQ_ATTN_C
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
#undef ZQ_ATTN_D
    if (!a.lse) return hipSuccess;
    if (a.sc) {
        const size_t grid = a.heads_kv * ((c.capacity + 1023) / 1024);
        hipLaunchKernelGGL(attn_q4_weights_sum_kernel, dim3(uint32_t(grid)), dim3(256), 0, stream, a);
        return hipGetLastError();
    }
#define ZQ_ATTN_W(DD)                                                                                               \
    do {                                                                                                            \
        const dim3 grid{uint32_t(key_blocks)};                                                                      \
        if (a.many)                                                                                                 \
            hipLaunchKernelGGL(attn_q4_weights_many_kernel<DD>, grid, dim3(512), 8 * Wgt<DD>::kQ, stream, a);       \
        else                                                                                                        \
            hipLaunchKernelGGL(attn_q4_weights_few_kernel<DD>, grid, dim3(256), 4 * Wgt<DD>::kQ, stream, a,         \
                               uint32_t(wblocks));                                                                  \
    } while (0)
    if (c.head_dim == 64) ZQ_ATTN_W(64);
    else if (c.head_dim == 128) ZQ_ATTN_W(128);
    else ZQ_ATTN_W(256);
#undef ZQ_ATTN_W
    return hipGetLastError();
}

}  // namespace zq
