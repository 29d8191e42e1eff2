// zq_attn_paged.hip -- attention of single query tokens over the paged KV cache of
// include/zq_paged.h.
//
//   s[r][p] = scale * q_r . k_p        p: rows that the query sees, in its pages
//   out[r]  = sum_p exp(s - max) v_p / sum_p exp(s - max)
//
// Rows r are the heads of one kv head, up to 16 of them at once: they are the rows
// of one matrix product, so a held row is read once for all of them.
#include "zq_entry.hpp"
#include "zq_internal.hpp"
#include "zq_paged.hpp"

#include <math.h>

namespace zq {
namespace {

typedef float v4f_t __attribute__((ext_vector_type(4)));
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef uint32_t v4u_t __attribute__((ext_vector_type(4)));

struct Cut {
    uint32_t query, kh, rows, parts;  // parts 0: none
    uint64_t slot;                    // of the first part; part j > 0 has slot 2 (w + j)
};
struct AttnPaged {
    const uint8_t* k;
    const uint8_t* v;
    const int32_t* table;
    const int32_t* select;
    const float* q;
    float* out;
    float* part;     // partial outputs [2 W][RS][D]
    float* part_ml;  // their (max, sum) [2 W][RS][2]
    Cut* cut;        // [W] the pair that a share's end cuts, if the share has its start
    Queries see;
    size_t stride;   // floats between queries
    float scale2;    // scale * log2(e): scores are in log2 units
    uint32_t width, pages, KH, G, keep, lp;
    uint32_t start;  // units that a pair's start counts as
    uint32_t P, RS, RL;  // queries of a group at most, rows of a partial and of a workgroup
};

// ---- work of a workgroup ---------------------------------------------------------
// The rows of a (query, kv head) pair are cut into units of kUnit keys, and these are
// shared out evenly (zq_paged.hpp).  A pair that a share's end cuts is put together by
// the join kernel.  Starting on a pair and writing its outputs takes as long as `start`
// units more, which count as units without keys at its start.
constexpr int kT = kShareT, kWaves = kShareWaves;
// More workgroups than CUs only where each has this many units: 100,000 rows of one kv head take 23 us so, 37 with a unit
// each (768 partials to join).
constexpr uint32_t kFew = 6;
template <int TYPE>
struct Tile {
    static constexpr int kKeys = TYPE == ZQ_KV_F32 ? 16 : 32;  // keys of a wave's tile
    static constexpr int H = kKeys / 16;                        // 16-key parts of it
    static constexpr int kUnit = kKeys * kWaves;
};

__device__ __forceinline__ uint32_t entries_of(const AttnPaged& a, uint32_t rows) {  // pages that count
    const uint32_t pages = (rows + (1u << a.lp) - 1) >> a.lp;
    return a.select ? min(pages, a.keep) : pages;
}
// Queries of one sequence that lie next to each other, as drafted tokens and prompts do,
// share a product where their heads fit 16 rows (GROUP; not with selected pages): the
// first one of every P (by number) and of every sequence stands for those behind it.
struct Group {
    Seen first;
    uint32_t queries, most, least;  // rows that they see
};
template <int GROUP>
__device__ __forceinline__ Group group_of(const AttnPaged& a, const ShareScan& sh, uint32_t i) {
    Group x{seen_held(a.see, sh, i), 1, 0, 0};
    x.most = x.least = x.first.rows;
    if constexpr (GROUP != 0) {
        for (uint32_t j = i + 1; x.first.seq >= 0 && j < a.see.n && j % a.P; ++j) {
            const Seen y = seen_held(a.see, sh, j);
            if (y.seq != x.first.seq) break;
            ++x.queries;
            x.most = max(x.most, y.rows);
            x.least = min(x.least, y.rows);
        }
    }
    return x;
}
template <int TYPE, int GROUP>
__device__ __forceinline__ uint32_t units_of(const AttnPaged& a, const ShareScan& sh, uint32_t i) {
    const Group x = group_of<GROUP>(a, sh, i);
    if (x.first.seq < 0) return 0;
    if (GROUP && i % a.P && seen_held(a.see, sh, i - 1).seq == x.first.seq) return 0;
    const uint32_t rows = a.select ? entries_of(a, x.most) << a.lp : x.most;
    return a.start + max((rows + Tile<TYPE>::kUnit - 1) / Tile<TYPE>::kUnit, 1u);  // no rows: a unit that writes zeros
}

// Where row r (query, head) of a group goes; without groups r is a head, G of them and no more.
__device__ __forceinline__ size_t out_row(const AttnPaged& a, uint32_t query, uint32_t kh, uint32_t r) {
    return size_t(query + r / a.G) * a.KH * a.G + size_t(kh) * a.G + r % a.G;
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

// Weights are 2^(s - m + kShift) with m the running maximum, which a score may pass by kSlack before the sums are scaled
// anew.  An fp16 cache's weights are two fp16 parts, multiples of 2^-24 at most 2^15: as far up as they go, a weight has 22
// bits down to 2^-17 of the largest and is off by 2^-39 of that below; with 6 and 8 as elsewhere it was 2^-31, which 1200
// rows 2^-20 below a first one showed as 1.3e-4 of their share.  (Sums are scaled more often so, which costs no time:
// 64 sequences of up to 8190 rows: 176 us either way.)
template <int TYPE>
constexpr float kShift = TYPE == ZQ_KV_F16 ? 14.0f : 6.0f;
template <int TYPE>
constexpr float kSlack = TYPE == ZQ_KV_F16 ? 1.0f : 8.0f;

// An fp32 factor as operands of the cache's type: fp16 in two parts (22 bits; the
// factors are scaled so that the second one stays normal), bf16 in three (exact: 8
// bits each, cut off), fp32 as it is.
__device__ __forceinline__ uint32_t f_bits(float x) { return __float_as_uint(x); }
__device__ __forceinline__ float bits_f(uint32_t x) { return __uint_as_float(x); }
template <int TYPE>
struct Parts;
template <>
struct Parts<ZQ_KV_F16> {
    static constexpr int N = 2;
    h8_t x[N];
    __device__ __forceinline__ void set2(int i, float a, float b) {
        x[0][i] = _Float16(a);
        x[0][i + 1] = _Float16(b);
        x[1][i] = _Float16(a - float(x[0][i]));
        x[1][i + 1] = _Float16(b - float(x[0][i + 1]));
    }
    __device__ __forceinline__ v4u_t bits(int n) const { return __builtin_bit_cast(v4u_t, x[n]); }
};
template <>
struct Parts<ZQ_KV_BF16> {
    static constexpr int N = 3;
    v4u_t x[N];
    __device__ __forceinline__ void set2(int i, float a, float b) {
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            x[n][i / 2] = __builtin_amdgcn_perm(f_bits(b), f_bits(a), 0x07060302u);  // the upper halves
            a -= bits_f(f_bits(a) & 0xffff0000u);
            b -= bits_f(f_bits(b) & 0xffff0000u);
        }
    }
    __device__ __forceinline__ v4u_t bits(int n) const { return x[n]; }
};

template <int TYPE>
__device__ __forceinline__ v4f_t mma(v4u_t held, v4u_t part, v4f_t c) {
    if constexpr (TYPE == ZQ_KV_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8_t, held), __builtin_bit_cast(h8_t, part), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8_t, held), __builtin_bit_cast(b8_t, part), c, 0, 0, 0);
}

template <int TYPE, int D>
struct Shape {
    static constexpr int ES = TYPE == ZQ_KV_F32 ? 4 : 2;
    static constexpr int H = Tile<TYPE>::H;
    static constexpr int KC = D * ES / 64;                          // 16-byte loads of a key
    static constexpr int VE = TYPE == ZQ_KV_F32 ? 4 : D == 64 ? 4 : 8;  // elements of a V load
    static constexpr int VC = D / (16 * VE);                        // V loads of a row
    static constexpr int VW = VE * ES / 4;                          // dwords of one
    static constexpr int VR = 4 * H;                                // rows whose V a lane loads
    static constexpr int NP = TYPE == ZQ_KV_F32 ? 1 : TYPE == ZQ_KV_F16 ? 2 : 3;
    static constexpr int QL = TYPE == ZQ_KV_F32 ? 1 : 2;            // 16-byte loads of q for 16 bytes of a key
};

// The softmax weights of a lane's rows as operands, and what they add to one tile of O^T.
template <int TYPE, int VR>
struct Weights {
    Parts<TYPE> x;
    __device__ __forceinline__ explicit Weights(const float (&p)[VR]) {
#pragma unroll
        for (int r = 0; r < VR; r += 2) x.set2(r, p[r], p[r + 1]);
    }
};
template <int VR>
struct Weights<ZQ_KV_F32, VR> {
    float x[VR];
    __device__ __forceinline__ explicit Weights(const float (&p)[VR]) {
#pragma unroll
        for (int r = 0; r < VR; ++r) x[r] = p[r];
    }
};
// (word(r): the dword of row r that has the tile's element e of every V load)
template <int TYPE, int VR, int PARTS = Shape<TYPE, 128>::NP, class F>
__device__ __forceinline__ v4f_t add_pv(F word, const Weights<TYPE, VR>& p, int e, v4f_t o) {
    if constexpr (TYPE == ZQ_KV_F32) {
#pragma unroll
        for (int r = 0; r < VR; ++r) o = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f(word(r)), p.x[r], o, 0, 0, 0);
    } else {
        v4u_t w;
#pragma unroll
        for (int z = 0; z < 4; ++z)
            w[z] = __builtin_amdgcn_perm(word(2 * z + 1), word(2 * z), e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int y = PARTS - 1; y >= 0; --y) o = mma<TYPE>(w, p.x.bits(y), o);
    }
    return o;
}
// Infinities and NaN of a dword's values: ones in their places, and zeros in the dword.
template <int TYPE>
__device__ __forceinline__ uint32_t take_odd(uint32_t& w) {
    constexpr uint32_t m = TYPE == ZQ_KV_F32 ? 0x7f800000u : TYPE == ZQ_KV_F16 ? 0x7c00u : 0x7f80u;
    constexpr uint32_t one = TYPE == ZQ_KV_F32 ? 0x3f800000u : TYPE == ZQ_KV_F16 ? 0x3c00u : 0x3f80u;
    constexpr uint32_t all = TYPE == ZQ_KV_F32 ? 0xffffffffu : 0xffffu;
    uint32_t gone = (w & m) == m ? all : 0u, ones = gone & one;
    if constexpr (TYPE != ZQ_KV_F32) {
        const bool hi = (w & m << 16) == m << 16;
        gone |= hi ? all << 16 : 0u;
        ones |= hi ? one << 16 : 0u;
    }
    w &= ~gone;
    return ones;
}
// Whether there are any.
template <int TYPE>
__device__ __forceinline__ bool not_finite(uint32_t w) {
    if (TYPE == ZQ_KV_F32) return (w & 0x7f800000u) == 0x7f800000u;
    const uint32_t m = TYPE == ZQ_KV_F16 ? 0x7c00u : 0x7f80u;
    return (w & m) == m || (w >> 16 & m) == m;
}

// A held row's bytes: read by one workgroup alone, or (GROUP) by those of other queries of its sequence too.
template <bool GROUP, class V>
__device__ __forceinline__ V load_held(const uint8_t* p) {
    return GROUP ? *reinterpret_cast<const V*>(p) : load_once<V>(p);
}

// ---- the kernel ------------------------------------------------------------------
// Both products are computed transposed (S^T = K Q^T, O^T = V^T P^T) on 16x16 tiles,
// so that nothing crosses lanes between them.  With lane (i = lane & 15, g = lane >> 4):
//  * K: lane loads 16 bytes of key i at a time, the g-th quarter of every 64 bytes of
//    the row; the dimension that a k slot stands for is the same for K and Q and need
//    not be in order.  It then holds the scores of row i and keys 4 g .. 4 g + 3 of
//    each 16-key part;
//  * which is what the second product's B operand wants of it.  Its A operand is V^T:
//    the lane loads the i-th 16 bytes (8 for D = 64) of the rows of those keys, and
//    pairs the same element of two rows with one v_perm (fp32: no pairing, one key a
//    product).
// K and V go from HBM into the operands without LDS, in whole rows.  A 16-key part lies
// in one page: its place is one readlane of the table entries that the wave loaded, 64
// parts at once.  The next tile's K is asked for when this one's scores are there, the
// next V when this one is used.
// Bound by HBM from some hundred rows a workgroup on.  What a wave has under way is a tile
// of K and one of V, 8 to 16 KB each; with two workgroups a CU that is enough to read at 6.0
// to 6.2 TB/s (131,072 bf16 rows of 8 kv heads of 128, 537 MB: 89 us; 64 sequences of up to
// 8190 fp16 rows, 1.09 GB: 175), where a copy moves 5.1.  load_once is a part of that: 4.8
// TB/s without.  Of a product's 16 rows a decode step uses the heads of a kv head only, but
// the matrix cores are not what it waits for, which is why both factors may go in as parts.
// A short pair is bound by its chain of round trips (length, table, K and V) and the merge of
// the four waves' sums: 600 rows take 8.9 us.
// One (query or group, kv head) pair, or the units u0 .. u1 of it, by a workgroup.
// whole: straight into the output; else into partial `slot`.
template <int TYPE, int D, int GROUP, class F>
__device__ __forceinline__ void attend(const AttnPaged& a, float* dyn, float (&sm)[kWaves][16], float (&sl)[kWaves][16], uint32_t qi,
                                       uint32_t kh, const Group& x, uint32_t row0, uint32_t u0, uint32_t u1, bool whole,
                                       size_t slot, F rows_of, bool has_ahead = false, uint32_t ahead = 0) {
    using S = Shape<TYPE, D>;
    constexpr int H = S::H, KC = S::KC, VE = S::VE, VC = S::VC, VW = S::VW, VR = S::VR, NP = S::NP;
    constexpr int RT = GROUP ? GROUP : 1;  // tiles of 16 rows
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const size_t head_rows = size_t(1) << a.lp;
    v4u_t* held_q = reinterpret_cast<v4u_t*>(dyn + kWaves * a.RL * (D + 4));  // q's operands [RT][KC][NP][64]
    const uint32_t R = GROUP ? x.queries * a.G : min(a.G - row0, 16u);  // rows: query, head
    const bool two = RT > 1 && R > 16;
    const uint32_t entries = entries_of(a, x.most);
    const uint32_t parts = a.select ? entries << (a.lp - 4) : (x.most + 15) >> 4;  // 16-key parts of the pair
    const uint32_t tiles = (parts + H - 1) / H;
    const uint32_t t0 = u0 * kWaves + wave, t1 = min(u1 * kWaves, tiles);
    const uint32_t nt = t0 < t1 ? (t1 - t0 + kWaves - 1) / kWaves : 0;  // tiles of this wave
    const int32_t* table = a.table + size_t(x.first.seq) * a.width;
    const int32_t* select = a.select ? a.select + (size_t(qi) * a.KH + kh) * a.keep : nullptr;

    // ---- the wave's tiles ----
    v4u_t kt[H][KC];
    // (vectors: with dwords of their own a build, not kept, had two of four loaded over before their use; in today's code neither
    // form has, and a test of the generated code looks for it)
    typedef uint32_t vw_t __attribute__((ext_vector_type(VW)));
    vw_t vt[VR][VC];
    uint32_t place = 0;  // lane p: page | rows there << 24 of the p-th part that the wave has ahead
    // byte offset of the wave's part p (of 64) from the cache's start
    auto part_at = [&](uint32_t p, uint32_t part) {
        const uint32_t page = uint32_t(__builtin_amdgcn_readlane(int(place), int(p))) & 0xffffffu;
        const uint32_t in = (part << 4) & (uint32_t(head_rows) - 1);
        return ((size_t(page) * a.KH + kh) * head_rows + in) * (D * S::ES);
    };
    auto rows_at = [&](uint32_t p) { return uint32_t(__builtin_amdgcn_readlane(int(place), int(p))) >> 24; };
    constexpr uint32_t kBatch = 64 / H;  // tiles whose places a wave holds
    uint32_t b = 0;  // the first tile of the batch
    auto load_places = [&] {
        const uint32_t j = b + lane / H, part = (t0 + j * kWaves) * H + lane % H, e = part >> (a.lp - 4);
        place = 0;
        if (j < nt && e < entries) {
            const uint32_t y = select ? uint32_t(select[e]) : e;  // place in the sequence
            if (y < a.width && (y << a.lp) < x.most) {
                const uint32_t page = has_ahead && b == 0 ? ahead : uint32_t(table[y]);
                const uint32_t first = (y << a.lp) + ((part << 4) & (uint32_t(head_rows) - 1));
                if (page < a.pages && first < x.most) place = page | min(x.most - first, 16u) << 24;
            }
        }
    };
    auto load_k = [&](uint32_t j) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const uint8_t* p = a.k + part_at(j * H + h, (t0 + (b + j) * kWaves) * H + h);
#pragma unroll
            for (int k = 0; k < KC; ++k)
                kt[h][k] = load_held<GROUP != 0, v4u_t>(p + uint32_t(i * D * S::ES + k * 64 + g * 16));
        }
    };
    auto load_v = [&](uint32_t j) {
        asm volatile("" ::: "memory");  // behind K: a wait for K is none for V
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const uint8_t* p = a.v + part_at(j * H + h, (t0 + (b + j) * kWaves) * H + h);
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int n = 0; n < VC; ++n) {
                    const uint8_t* at = p + uint32_t((4 * g + r) * D * S::ES + (n * 16 + i) * VE * S::ES);
                    vt[h * 4 + r][n] = load_held<GROUP != 0, vw_t>(at);
                }
        }
    };
    load_places();

    // ---- the queries as operands ----
    uint32_t my_rows[RT];  // that this lane's query sees
    float c[RT];           // takes a score into log2 units
    auto load_q = [&](int t, float4 (&x0)[KC][S::QL]) {
        const uint32_t at = uint32_t(t * 16 + i), row = min(at, R - 1), member = GROUP ? row / a.G : 0u;
        const float* qrow = a.q + (qi + member) * a.stride + (size_t(kh) * a.G + row0 + row - member * a.G) * D;
        my_rows[t] = GROUP ? rows_of(qi + member) : 0u;
#pragma unroll
        for (int k = 0; k < KC; ++k)
#pragma unroll
            for (int j = 0; j < S::QL; ++j) {
                x0[k][j] = *reinterpret_cast<const float4*>(qrow + ((4 * k + g) * S::QL + j) * 4);
                if (at >= R) x0[k][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
    };
    auto make_q = [&](int t, const float4 (&x0)[KC][S::QL]) {
        c[t] = a.scale2;
        float up = 1.0f;
        if constexpr (TYPE == ZQ_KV_F16) {  // the row's largest element to 2^14 .. 2^15
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int j = 0; j < S::QL; ++j)
                    most = fmaxf(most, fmaxf(fmaxf(fabsf(x0[k][j].x), fabsf(x0[k][j].y)), fmaxf(fabsf(x0[k][j].z), fabsf(x0[k][j].w))));
            most = max_groups(most);
            if (most > 0.0f) {
                const int e = min(max(15 - __builtin_amdgcn_frexp_expf(most), -113), 126);
                up = pow2f(e);
                c[t] *= pow2f(-e);
            }
        }
#pragma unroll
        for (int k = 0; k < KC; ++k) {
            v4u_t op[NP];
            if constexpr (TYPE == ZQ_KV_F32) {
                op[0] = v4u_t{f_bits(x0[k][0].x), f_bits(x0[k][0].y), f_bits(x0[k][0].z), f_bits(x0[k][0].w)};
            } else {
                Parts<TYPE> p;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    p.set2(4 * j, x0[k][j].x * up, x0[k][j].y * up);
                    p.set2(4 * j + 2, x0[k][j].z * up, x0[k][j].w * up);
                }
#pragma unroll
                for (int n = 0; n < NP; ++n) op[n] = p.bits(n);
            }
            if (k % kWaves == wave)
#pragma unroll
                for (int n = 0; n < NP; ++n) held_q[((t * KC + k) * NP + n) * 64 + lane] = op[n];
        }
    };
    {
        float4 x0[KC][S::QL];
        if (RT > 1) my_rows[RT - 1] = 0, c[RT - 1] = 0.0f;
        if (two) {
            load_q(RT - 1, x0);
            make_q(RT - 1, x0);
        }
        load_q(0, x0);
        // (asked for behind the queries, which are waited for first; a wave without tiles reads rows of page 0)
        load_k(0);
        load_v(0);
        make_q(0, x0);
    }
    __syncthreads();

    v4f_t o[RT][VC][VE];
    float m[RT], l[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        m[t] = -INFINITY;
        l[t] = 0.0f;
#pragma unroll
        for (int n = 0; n < VC; ++n)
#pragma unroll
            for (int e = 0; e < VE; ++e) o[t][n][e] = v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
    }
    auto step = [&](uint32_t j, auto last) {
        v4f_t s[RT][H];
        asm volatile("" ::: "memory");  // q is read again, not held
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int h = 0; h < H; ++h) s[t][h] = v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
            if (t && !two) break;  // uniform
#pragma unroll
            for (int k = 0; k < KC; ++k) {
                v4u_t op[NP];
#pragma unroll
                for (int n = 0; n < NP; ++n) op[n] = held_q[((t * KC + k) * NP + n) * 64 + lane];
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    if constexpr (TYPE == ZQ_KV_F32) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            s[t][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f(kt[h][k][e]), bits_f(op[0][e]), s[t][h], 0, 0, 0);
                    } else {
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n) s[t][h] = mma<TYPE>(kt[h][k], op[n], s[t][h]);
                    }
                }
            }
        }
        const uint32_t key0 = (t0 + (b + j) * kWaves) * H * 16;  // (without selected pages) the tile's first key
        uint32_t rows[H];
        bool cut = false;
#pragma unroll
        for (int h = 0; h < H; ++h) {
            rows[h] = rows_at(j * H + h);
            cut |= rows[h] < 16;
            if (GROUP) cut |= key0 + h * 16 + 16 > x.least;
        }
        if constexpr (!decltype(last)::value) load_k(j + 1);
        auto cut_v = [&] {  // rows behind the last one
            if (!cut) return;  // uniform
#pragma unroll
            for (int r = 0; r < VR; ++r) {
                const uint32_t keep = uint32_t(4 * g + r % 4) < rows[r / 4] ? 0xffffffffu : 0u;
#pragma unroll
                for (int n = 0; n < VC; ++n) vt[r][n] &= keep;
            }
        };
        if (GROUP) cut_v();
        // a value that is no number must not reach (0 times it) the queries that do not see its row
        bool odd = false;
        if (GROUP && cut && x.least < x.most) {
#pragma unroll
            for (int r = 0; r < VR; ++r)
#pragma unroll
                for (int n = 0; n < VC; ++n)
#pragma unroll
                    for (int z = 0; z < VW; ++z) odd |= not_finite<TYPE>(vt[r][n][z]);
            odd = __any(odd);
        }
        if (odd) {  // per element: how many such values a query sees; more than none gives NaN
            uint32_t ln = threadIdx.x;
            asm volatile("" : "+v"(ln));  // made here, not held through the tiles
            const uint32_t og = (ln >> 4) & 3;
#pragma unroll
            for (int n = 0; n < VC; ++n)
#pragma unroll
                for (int z = 0; z < VW; ++z) {
                    uint32_t ones[VR];
#pragma unroll
                    for (int r = 0; r < VR; ++r) {
                        uint32_t w = vt[r][n][z];
                        ones[r] = take_odd<TYPE>(w);
                        vt[r][n][z] = w;
                    }
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
                        float sees[VR];
#pragma unroll
                        for (int r = 0; r < VR; ++r) sees[r] = key0 + r / 4 * 16 + 4 * og + r % 4 < my_rows[t] ? 1.0f : 0.0f;
                        const Weights<TYPE, VR> ps(sees);
#pragma unroll
                        for (int e = 0; e < VE / VW; ++e) {
                            const v4f_t y = add_pv<TYPE, VR, 1>([&](int r) { return ones[r]; }, ps, e, v4f_t{0.0f, 0.0f, 0.0f, 0.0f});
                            v4f_t& to = o[t][n][z * (VE / VW) + e];
#pragma unroll
                            for (int k = 0; k < 4; ++k) to[k] = y[k] > 0.0f ? NAN : to[k];
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);  // one after the other: in few registers
                }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            if (t && !two) break;
#pragma unroll
            for (int h = 0; h < H; ++h) s[t][h] *= c[t];
            if (cut) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    uint32_t n = rows[h];
                    if (GROUP) n = min(n, uint32_t(max(int32_t(my_rows[t] - (key0 + h * 16)), 0)));
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (uint32_t(4 * g + r) >= n) s[t][h][r] = -INFINITY;
                }
            }
            float most = -INFINITY;
#pragma unroll
            for (int h = 0; h < H; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) most = fmaxf(most, s[t][h][r]);
            if (__any(most > m[t] + kSlack<TYPE>)) {
                const float to = fmaxf(m[t], max_groups(most));
                const float f = to == -INFINITY ? 1.0f : exp2_(m[t] - to);
                m[t] = to;
                l[t] *= f;
#pragma unroll
                for (int n = 0; n < VC; ++n)
#pragma unroll
                    for (int e = 0; e < VE; ++e) o[t][n][e] *= f;
            }
            const float ms = (m[t] == -INFINITY ? 0.0f : m[t]) - kShift<TYPE>;
            float p[VR];
#pragma unroll
            for (int r = 0; r < VR; ++r) {
                p[r] = exp2_(s[t][r / 4][r % 4] - ms);
                l[t] += p[r];
            }
            if (!GROUP) cut_v();  // (as late as it can be: it waits for V)
            const Weights<TYPE, VR> pw(p);
#pragma unroll
            for (int n = 0; n < VC; ++n)
#pragma unroll
                for (int e = 0; e < VE; ++e)
                    o[t][n][e] = add_pv<TYPE, VR>([&](int r) { return uint32_t(vt[r][n][e * VW / VE]); }, pw, e, o[t][n][e]);
        }
        if constexpr (!decltype(last)::value) load_v(j + 1);
    };
    while (b < nt) {
        const uint32_t count = min(nt - b, kBatch);
        for (uint32_t j = 0; j + 1 < count; ++j) step(j, std::false_type{});
        step(count - 1, std::true_type{});
        b += kBatch;
        if (b < nt) {
            load_places();
            load_k(0);
            load_v(0);
        }
    }

    // ---- the four waves' sums as one ----
    uint32_t ln = threadIdx.x;
    asm volatile("" : "+v"(ln));  // the addresses below are made here, not held through the tiles
    const uint32_t mi = ln & 15, mg = (ln >> 4) & 3;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        if (t && !two) break;
        const uint32_t rows = min(R - t * 16, 16u);
        l[t] = sum_groups(l[t]);
        if (mg == 0) {
            sm[wave][mi] = m[t];
            sl[wave][mi] = l[t];
        }
        if (mi < rows) {
            float* to = dyn + (size_t(wave) * a.RL + mi) * (D + 4);
#pragma unroll
            for (int n = 0; n < VC; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < VE; e += 4)
                        *reinterpret_cast<float4*>(to + n * 16 * VE + VE * (4 * mg + r) + e) =
                            make_float4(o[t][n][e][r], o[t][n][e + 1][r], o[t][n][e + 2][r], o[t][n][e + 3][r]);
        }
        __syncthreads();
        for (uint32_t z = ln; z < rows * (D / 4); z += kT) {
            const uint32_t r = z / (D / 4), d = z % (D / 4) * 4, at = t * 16 + r;
            float M = sm[0][r];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sm[w][r]);
            const float Ms = M == -INFINITY ? 0.0f : M;
            float L = 0.0f;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = exp2_(sm[w][r] - Ms);
                const float4 q = *reinterpret_cast<const float4*>(dyn + (w * a.RL + r) * (D + 4) + d);
                L += sl[w][r] * f;
                y.x += q.x * f, y.y += q.y * f, y.z += q.z * f, y.w += q.w * f;
            }
            if (whole) {
                const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);  // no row: 0; NaN stays
                y.x *= inv, y.y *= inv, y.z *= inv, y.w *= inv;
            } else if (d == 0) {
                a.part_ml[(slot + at) * 2] = M;
                a.part_ml[(slot + at) * 2 + 1] = L;
            }
            float* to = whole ? out_row(a, qi, kh, row0 + at) * D + a.out : a.part + (slot + at) * D;
            *reinterpret_cast<float4*>(to + d) = y;
        }
        __syncthreads();
    }
}

// The share of workgroup b of `used`: those of an XCD, which b % 8 says, are neighbours, so that the groups of a sequence
// that are at the same rows find them in one L2 (drafted tokens of 16 sequences at D = 64: 24.9, 23.7 us).
__device__ __forceinline__ uint32_t share_by_xcd(uint32_t b, uint32_t used) {
    if (b >= used) return b;
    const uint32_t x = b % 8;
    return x * (used / 8) + min(x, used % 8) + b / 8;
}

// Shares of all pairs' units, as they come.  (With D = 256 there is a workgroup a CU: a wave may have all registers.)
template <int TYPE, int D, int GROUP>
__global__ __launch_bounds__(kT, D == 256 ? 1 : GROUP > 1 ? 2 : D == 64 ? 4 : 3) void attn_paged_kernel(AttnPaged a) {
    extern __shared__ float dyn[];  // [waves][rows][D + 4], then q's operands
    __shared__ ShareScan scan;
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    const uint32_t row0 = GROUP ? 0u : blockIdx.y * 16;  // the first head of this workgroup's
    const auto units = [&](uint32_t n) { return units_of<TYPE, GROUP>(a, scan, n); };
    hold_seen(a.see, scan);
    uint32_t mine, own;
    const Shares sh = scan_units(a.see.n, a.KH, gridDim.x, kFew, units, scan, mine, own);
    const uint32_t share = GROUP ? share_by_xcd(blockIdx.x, sh.used) : blockIdx.x;
    if (threadIdx.x == 0 && blockIdx.y == 0) a.cut[share].parts = 0;
    if (share >= sh.used) return;
    const uint64_t begin = share_start(sh, share), end = share_start(sh, share + 1);
    const Found at_begin = find_query(a.see.n, a.KH, units, scan, begin, mine, own);
    uint32_t qi = at_begin.query, before = at_begin.before;
    uint64_t pos = begin;
    while (pos < end) {
        const uint32_t u = uniform(units(qi));
        if (pos >= uint64_t(before + u) * a.KH) {
            before += u;
            ++qi;
            continue;
        }
        const uint32_t rel = uint32_t(pos - uint64_t(before) * a.KH), kh = rel / u, v0 = rel % u;
        const uint32_t v1 = uint32_t(min(uint64_t(u), v0 + (end - pos)));
        const uint32_t u0 = v0 > a.start ? v0 - a.start : 0u, u1 = v1 > a.start ? v1 - a.start : 0u;  // with keys
        if (u1 == 0) {
            pos += v1 - v0;
            continue;
        }
        Group x = group_of<GROUP>(a, scan, qi);
        x.first.seq = int32_t(uniform(uint32_t(x.first.seq)));
        x.queries = uniform(x.queries), x.most = uniform(x.most), x.least = uniform(x.least);
        const bool whole = u0 == 0 && v1 == u;
        const size_t at = size_t(share) * 2 + (pos != begin);
        if (u0 == 0 && v1 < u && threadIdx.x == 0 && blockIdx.y == 0) {
            // shares with a part of the pair: up to the last one that starts below its end
            uint64_t all = sh.all;
            asm volatile("" : "+s"(all));  // its reciprocal is made here, not held through the pairs
            const uint64_t last = ((pos - v0 + u) * sh.used + all - 1) / all - 1;
            a.cut[share] = {qi, kh, GROUP ? x.queries * a.G : a.G, uint32_t(last - share + 1), at};
        }
        attend<TYPE, D, GROUP>(a, dyn, sm, sl, qi, kh, x, row0, u0, u1, whole, at * a.RS + row0,
                                       [&](uint32_t n) { return seen_held(a.see, scan, n).rows; });
        pos += v1 - v0;
    }
}

// The group that query i leads, by a wave whose lanes each look at one query of those that
// might be in it; queries 0 where it leads none.  rows: what query base + lane sees.
struct GroupLanes {
    Group x;
    uint32_t base, rows;
};
__device__ __forceinline__ GroupLanes group_by_lanes(const AttnPaged& a, uint32_t i) {
    const uint32_t lane = threadIdx.x & 63, base = i / a.P * a.P, o = i - base;  // P <= 16
    Seen s{-1, 0};
    if (lane < a.P && base + lane < a.see.n) s = seen_by(a.see, base + lane);
    const int32_t seq = __builtin_amdgcn_readlane(s.seq, int(o));
    const uint64_t same = __ballot(s.seq == seq) >> o;
    GroupLanes g{{{seq, 0}, 0, 0, 0}, base, s.rows};
    if (seq < 0 || (o && __builtin_amdgcn_readlane(s.seq, int(o) - 1) == seq)) return g;
    const uint32_t n = min(uint32_t(__builtin_ctzll(~same)), a.P - o);
    g.x.queries = n;
    uint32_t most = 0, least = 0xffffffffu;
    if (lane >= o && lane < o + n) most = least = s.rows;
#pragma unroll
    for (int m = 1; m < 16; m *= 2) {
        most = max(most, uint32_t(__shfl_xor(int(most), m)));
        least = min(least, uint32_t(__shfl_xor(int(least), m)));
    }
    g.x.most = uniform(most), g.x.least = uniform(least);
    return g;
}

// A workgroup for every pair: nothing to share out and nothing to join.  (32 sequences with
// 2048 selected rows each, 8 kv heads of 128: 268 MB in 48 us, 5.6 TB/s.)
template <int TYPE, int D, bool GROUP>
__global__ __launch_bounds__(kT, D == 64 ? 4 : GROUP ? 256 / D : D == 128 ? 3 : 2) void attn_paged_pair_kernel(AttnPaged a) {
    extern __shared__ float dyn[];
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    const uint32_t qi = blockIdx.x / a.KH, kh = blockIdx.x % a.KH;
    const auto units = [&](uint32_t most) {
        const uint32_t rows = a.select ? entries_of(a, most) << a.lp : most;
        return max((rows + Tile<TYPE>::kUnit - 1) / Tile<TYPE>::kUnit, 1u);
    };
    if constexpr (GROUP) {
        const GroupLanes g = group_by_lanes(a, qi);
        if (g.x.queries == 0) return;
        attend<TYPE, D, 1>(a, dyn, sm, sl, qi, kh, g.x, 0, 0, units(g.x.most), true, 0,
                              [&](uint32_t q) { return uint32_t(__shfl(int(g.rows), int(q - g.base))); });
    } else {
        // the table entries of a wave's first parts, asked for before it is known how many there are
        constexpr uint32_t H = Tile<TYPE>::H;
        const uint32_t lane = threadIdx.x & 63, e = ((lane / H * kWaves + threadIdx.x / 64) * H + lane % H) >> (a.lp - 4);
        const bool has_ahead = !a.see.seq_of && !a.select;
        uint32_t ahead = 0;
        if (has_ahead && e < a.width) ahead = uint32_t(a.table[size_t(qi) * a.width + e]);
        const Seen s = seen_by(a.see, qi);
        if (s.seq < 0) return;
        attend<TYPE, D, 0>(a, dyn, sm, sl, qi, kh, Group{s, 1, s.rows, s.rows}, blockIdx.y * 16, 0, units(s.rows), true, 0,
                               [](uint32_t) { return 0u; }, has_ahead, ahead);
    }
}

// ---- join ------------------------------------------------------------------------
// Workgroup (w, r) puts row r of the pair together that the end of share w cuts.  A launch
// and three round trips (the share's record, the maxima, the partials), whatever its bytes
// (512 partials of 4 rows of 128: 1 MB): 4.7 us.
template <int D>
__global__ __launch_bounds__(kT) void attn_paged_join_kernel(AttnPaged a) {
    constexpr int E = D / 64;  // elements of a lane
    __shared__ float acc[kWaves][D];
    __shared__ float wm[kWaves], wl[kWaves];
    const uint32_t w = blockIdx.x, r = blockIdx.y;
    const Cut c = a.cut[w];
    if (r >= c.rows || c.parts == 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto slot = [&](uint32_t j) { return (j ? size_t(w + j) * 2 : size_t(c.slot)) * a.RS + r; };
    float M = -INFINITY;
    for (uint32_t j = threadIdx.x; j < c.parts; j += kT) M = fmaxf(M, a.part_ml[slot(j) * 2]);
    M = wave_max(M);
    if (lane == 0) wm[wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    const float Ms = M == -INFINITY ? 0.0f : M;
    float L = 0.0f, y[E] = {};
#pragma unroll 8
    for (uint32_t j = wave; j < c.parts; j += kWaves) {
        const size_t at = slot(j);
        const float f = exp2_(a.part_ml[at * 2] - Ms);
        L += a.part_ml[at * 2 + 1] * f;
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] += a.part[at * D + lane * E + e] * f;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) acc[wave][lane * E + e] = y[e];
    if (lane == 0) wl[wave] = L;
    __syncthreads();
    L = (wl[0] + wl[1]) + (wl[2] + wl[3]);
    const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);
    float* out = a.out + out_row(a, c.query, c.kh, r) * D;
    for (uint32_t d = threadIdx.x; d < D; d += kT) out[d] = ((acc[0][d] + acc[1][d]) + (acc[2][d] + acc[3][d])) * inv;
}

// Whether every pair gets a workgroup of its own.  The host knows how long a pair may be (the tables' width, or the pages
// selected), not how long it is.  us, such workgroups and shares, of 8 kv heads of 128 and fp16 if not said otherwise:
//  - pairs of up to 320 KB of rows: few pairs cross between 280 and 350 KB, more later (pages all over 4 GB: a sequence of
//    272 KB 8.6, 9.9; 320 KB 9.8, 10.4; 368 KB 11.7, 10.5; bf16, D = 64, 284 KB 9.7, 9.7; 336 KB 11.3, 10.0; fp32, 4 kv heads
//    of 256, 288 KB 11.0, 13.3; 352 KB 13.7, 13.3; 4 sequences of 272 KB 10.5, 10.9; 320 KB 11.9, 11.4; 16 of 320 KB 14.7,
//    18.3; of up to 520 KB 18.5, 18.0);
//  - two pairs for every CU of up to 1.1 MB (64 sequences of up to 1 MB 54, 55; 1.1 MB 56, 56; 1.5 MB 78, 74; 2 MB 103, 95;
//    512 of up to 200 KB 84, 110);
//  - as many selected pages each of up to 1.1 MB where the pairs fill rounds of a workgroup a CU (1 MB of longer sequences: 24
//    sequences 66, 70; 29: 73, 80; 32: 71, 79; 33: 107, 91; 40: 104, 97; 48: 122, 115; 60: 136, 143).  Such pairs gain at 2 MB
//    too (32: 123, 131), but where lengths are below what may be selected they are of all sizes: 32 sequences of up to 0.5 MB
//    23, 32; 1 MB 39, 38; 2 MB 70, 58.
// Of groups, all but the first query's workgroups have nothing to do: only where these are few, or all of them (62 sequences
// of 6 rows with 8 drafted tokens, 2 kv heads: 18, 25; 100 of up to 200 with 2 of 8 heads, 8 kv heads: 26, 28; 128 of up to
// 300 with 8 of one head, 8: 37, 40; 100 of up to 300 with 4 of 4, 8: 47, 36; two prompts of 500 tokens, 8: 130, 62).
bool by_pairs(const AttnPaged& a, size_t row_bytes) {
    const uint64_t cap = a.see.cap, picked = a.select ? uint64_t(a.keep) << a.lp : cap;
    const uint64_t bytes = (picked < cap ? picked : cap) * 2 * row_bytes, all = uint64_t(a.see.n) * a.KH, pairs = all / a.P;
    if (a.P > 1 && all > 2048 && pairs > 512) return false;
    const uint64_t rounds = (pairs + 255) / 256;
    return bytes <= 320 * 1024 || (bytes <= 1100 * 1024 && (pairs >= 512 || (a.select && pairs * 10 >= rounds * 256 * 9)));
}

// What a pair's start counts as, in units, with groups in that many tiles (0: none).  us with 2, 3 and 4 in two: 8 drafted
// tokens of 8 sequences at D = 128: 50, 47, 41; in one, of 32 sequences, 3 and 4: 68, 70; without groups 1, 2 and 3: 128
// sequences of up to 2000 rows, D = 256: 198, 187, 187.
constexpr uint32_t kMostStart = 4;
uint32_t start_units(int tiles) { return uint32_t(2 + tiles); }
// Workgroups for a call, as many as there are units at most: two a CU, and a third (all that are resident) where there
// are so many pairs that every one starts on several of them; with D = 256 one, with two tiles two.  (512, 768, 1536
// workgroups, us: 64 sequences of up to 8190 rows, 512 pairs: 175, 177, 182; 512 of up to 400, 4096 pairs: 114, 110, 104;
// 131,072 rows of one: 89, 91, 100; 32 of up to 8000, bf16, D = 256, with 256, 512 and 1024: 97, 110, 131.)
uint32_t shares_of(const zq_kv_paged& c, const zq_page_tables& t, size_t queries, int tiles) {
    const size_t unit = c.type == ZQ_KV_F32 ? 64 : 128, pairs = queries * c.kv_heads;
    const size_t most = pairs * ((t.width * t.page_size + unit - 1) / unit + kMostStart);
    const size_t want = 256 * (c.head_dim == 256 ? 1 : tiles > 1 || pairs < 2048 ? 2 : 3);
    return uint32_t(most < want ? most : want);
}

// Queries of a group at most, and rows of a partial, for G heads of a kv head.
uint32_t group_most(size_t G, int tiles) { return G * 2 <= size_t(16 * tiles) ? uint32_t(16 * tiles / G) : 1; }
size_t part_rows(size_t G) { return G * group_most(G, 2); }

template <class K>
hipError_t allow_lds(K kernel, size_t lds) {
    if (lds <= 64 * 1024) return hipSuccess;
    return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
}

template <int TYPE, int D, int GROUP>
hipError_t run_attention(const AttnPaged& a, uint32_t W, hipStream_t stream) {
    using S = Shape<TYPE, D>;
    const size_t lds = size_t(kWaves) * a.RL * (D + 4) * 4 + size_t(GROUP ? GROUP : 1) * S::KC * S::NP * 64 * 16;
    const uint32_t tiles = GROUP ? 1 : (a.G + 15) / 16;
    if constexpr (GROUP < 2)
        if (by_pairs(a, D * S::ES)) {
            const hipError_t e = allow_lds(&attn_paged_pair_kernel<TYPE, D, GROUP != 0>, lds);
            if (e != hipSuccess) return e;
            hipLaunchKernelGGL((attn_paged_pair_kernel<TYPE, D, GROUP != 0>), dim3(a.see.n * a.KH, tiles), dim3(kT), lds, stream, a);
            return hipGetLastError();
        }
    hipError_t e = allow_lds(&attn_paged_kernel<TYPE, D, GROUP>, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((attn_paged_kernel<TYPE, D, GROUP>), dim3(W, tiles), dim3(kT), lds, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess || W == 1) return e;
    hipLaunchKernelGGL(attn_paged_join_kernel<D>, dim3(W - 1, a.RS), dim3(kT), 0, stream, a);
    return hipGetLastError();
}
template <int TYPE, int GROUP>
hipError_t run_attention(const AttnPaged& a, uint32_t W, size_t D, hipStream_t stream) {
    return D == 64 ? run_attention<TYPE, 64, GROUP>(a, W, stream)
                   : D == 128 ? run_attention<TYPE, 128, GROUP>(a, W, stream) : run_attention<TYPE, 256, GROUP>(a, W, stream);
}
template <int TYPE>
hipError_t run_attention(const AttnPaged& a, uint32_t W, size_t D, int group, hipStream_t stream) {
    return group == 2   ? run_attention<TYPE, 2>(a, W, D, stream)
           : group == 1 ? run_attention<TYPE, 1>(a, W, D, stream) : run_attention<TYPE, 0>(a, W, D, stream);
}

// Tiles of 16 rows for groups of queries of one sequence: 0: no groups; 2, which halve the times that keys are read, where
// sequences have more queries on average than one tile takes and keys are many; not at D = 256, where the registers for two
// leave few for loads.  us, 1 and 2 tiles: 8 sequences of up to 4000 rows with 8 queries of 8 heads: 53, 41; 30 of up to 9000
// with 2 of 16, D = 64: 187, 125; 16 of up to 3001 with 5 of 7, D = 64: 25, 30; 40 of up to 1379 with 8 of 4, D = 256: 38, 46.
int group_tiles(const zq_kv_paged& c, const zq_page_tables& t, size_t queries, size_t G, bool may) {
    const size_t bytes = t.width * t.page_size * 2 * c.head_dim * (c.type == ZQ_KV_F32 ? 4 : 2);
    if (!may || group_most(G, 2) == 1) return 0;
    if (c.head_dim < 256 && queries > t.seqs * group_most(G, 1) && bytes >= 1024 * 1024) return 2;
    return group_most(G, 1) > 1 ? 1 : 0;
}

size_t workspace(const zq_kv_paged& c, const zq_page_tables& t, size_t queries, size_t heads) {
    const size_t W = shares_of(c, t, queries, 0), rows = W * 2 * part_rows(heads / c.kv_heads);
    return (W * sizeof(Cut) + rows * (c.head_dim + 2) * 4 + 255) / 256 * 256;
}

}  // namespace
}  // namespace zq

extern "C" {

size_t zq_hip_attention_paged_workspace_bytes(const zq_kv_paged* cache, const zq_page_tables* tables, size_t queries,
                                              size_t heads) {
    if (!zq::kv_paged_ok(cache) || !zq::page_tables_ok(tables) ||
        !zq::queries_ok(*cache, *tables, queries, heads, tables->table))
        return 0;
    return zq::workspace(*cache, *tables, queries, heads);
}

int zq_hip_attention_paged_dev(const zq_kv_paged* cache, const zq_page_tables* tables, const float* q, float* out,
                               size_t queries, size_t heads, size_t stride, const int32_t* seq_of, const int32_t* lens,
                               const int32_t* counts, const int32_t* select, size_t keep, float scale, int flags,
                               void* workspace, size_t workspace_bytes, void* stream) {
    using zq::a16;
    using zq::a4;
    if (!zq::kv_paged_ok(cache) || !zq::page_tables_ok(tables) || !zq::queries_ok(*cache, *tables, queries, heads, seq_of) ||
        !q || !out || !lens || !a16(q) || !a16(out) || !a4(lens) || !a4(counts) || !a4(seq_of) || !a4(select) ||
        (flags & ~ZQ_ATTN_PAGED_FULL) || (select && (!keep || keep > zq::kPgMaxTokens / 16)))
        return ZQ_ERR_ARG;
    const size_t width = heads * cache->head_dim;
    if (!stride) stride = width;
    if (stride < width || stride % 4 || stride > zq::kPgMaxStride) return ZQ_ERR_ARG;
    if (!workspace || !a16(workspace) || workspace_bytes < zq::workspace(*cache, *tables, queries, heads)) return ZQ_ERR_ARG;
    const zq::OnDeviceOf dev(cache->k);
    if (dev.status() != ZQ_OK) return dev.status();
    const uint32_t G = uint32_t(heads / cache->kv_heads);
    zq::AttnPaged a{};
    a.k = static_cast<const uint8_t*>(cache->k);
    a.v = static_cast<const uint8_t*>(cache->v);
    a.table = tables->table;
    a.select = select;
    a.q = q;
    a.out = out;
    const int group = zq::group_tiles(*cache, *tables, queries, G, seq_of && !select);
    const uint32_t W = zq::shares_of(*cache, *tables, queries, group);
    a.P = group ? zq::group_most(G, group) : 1;
    a.start = zq::start_units(group);
    a.RS = a.P * G;
    a.RL = a.RS < 16 ? a.RS : 16;
    a.part = static_cast<float*>(workspace);
    a.cut = reinterpret_cast<zq::Cut*>(a.part + size_t(W) * 2 * a.RS * cache->head_dim);
    a.part_ml = reinterpret_cast<float*>(a.cut + W);
    a.see = {seq_of, lens, counts, uint32_t(queries), uint32_t(tables->seqs), uint32_t(tables->width * tables->page_size),
             flags & ZQ_ATTN_PAGED_FULL};
    a.stride = stride;
    a.scale2 = scale * 1.4426950408889634f;
    a.width = uint32_t(tables->width);
    a.pages = uint32_t(tables->pages);
    a.KH = uint32_t(cache->kv_heads);
    a.G = G;
    a.keep = uint32_t(keep);
    a.lp = zq::log2_of(tables->page_size);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    return zq::status(cache->type == ZQ_KV_F32   ? zq::run_attention<ZQ_KV_F32>(a, W, cache->head_dim, group, st)
                      : cache->type == ZQ_KV_F16 ? zq::run_attention<ZQ_KV_F16>(a, W, cache->head_dim, group, st)
                                                 : zq::run_attention<ZQ_KV_BF16>(a, W, cache->head_dim, group, st));
}

}  // extern "C"
