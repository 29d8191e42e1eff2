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
typedef uint32_t v2u_t __attribute__((ext_vector_type(2)));

struct AttnPaged {
    const uint8_t* k;
    const uint8_t* v;
    const int32_t* table;
    const int32_t* select;
    const float* q;
    float* out;
    float* part;     // partial outputs [2 W][G][D]
    float* part_ml;  // their (max, sum) [2 W][G][2]
    Queries see;
    size_t stride;   // floats between queries
    float scale2;    // scale * log2(e): scores are in log2 units
    uint32_t width, pages, KH, G, keep, lp;
};

// ---- work of a workgroup ---------------------------------------------------------
// The rows of a (query, kv head) pair are cut into units of kUnit keys, and these are
// shared out evenly (zq_paged.hpp).  A pair that a share's end cuts is put together by
// the join kernel.
constexpr int kT = kShareT, kWaves = kShareWaves;
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
template <int TYPE>
__device__ __forceinline__ uint32_t units_of(const AttnPaged& a, uint32_t i) {
    const Seen x = seen_by(a.see, i);
    if (x.seq < 0) return 0;
    const uint32_t rows = a.select ? entries_of(a, x.rows) << a.lp : x.rows;
    return max((rows + Tile<TYPE>::kUnit - 1) / Tile<TYPE>::kUnit, 1u);  // no rows: a unit that writes zeros
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

constexpr float kShift = 6.0f;  // weights are 2^(s - max + kShift)
constexpr float kSlack = 8.0f;  // how far a score may pass the running maximum

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
    static constexpr bool kQInLds = true;
};

template <int TYPE, int D>
__global__ __launch_bounds__(kT, D == 64 ? 4 : D == 128 ? 3 : 2) void attn_paged_kernel(AttnPaged a) {
    using S = Shape<TYPE, D>;
    constexpr int H = S::H, KC = S::KC, VE = S::VE, VC = S::VC, VW = S::VW, VR = S::VR, NP = S::NP;
    extern __shared__ float dyn[];  // [4 waves][rows][D + 4], then q's operands where they are kept here
    __shared__ ShareScan scan;
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t row0 = blockIdx.y * 16, R = min(a.G - row0, 16u);  // rows of this workgroup
    const auto units = [&](uint32_t n) { return units_of<TYPE>(a, n); };
    uint32_t mine, own;
    const Shares sh = scan_units(a.see.n, a.KH, gridDim.x, units, scan, mine, own);
    if (blockIdx.x >= sh.used) return;
    const uint64_t begin = share_start(sh, blockIdx.x), end = share_start(sh, blockIdx.x + 1);
    find_query(a.see.n, a.KH, units, scan, begin, mine, own);
    uint32_t qi = scan.query, before = scan.before;
    uint64_t pos = begin;
    const size_t head_rows = size_t(1) << a.lp;
    while (pos < end) {
        const uint32_t u = units(qi);
        if (pos >= uint64_t(before + u) * a.KH) {
            before += u;
            ++qi;
            continue;
        }
        const uint32_t rel = uint32_t(pos - uint64_t(before) * a.KH), kh = rel / u, u0 = rel % u;
        const uint32_t u1 = uint32_t(min(uint64_t(u), u0 + (end - pos)));
        const Seen x = seen_by(a.see, qi);
        const uint32_t entries = entries_of(a, x.rows);
        const uint32_t parts = a.select ? entries << (a.lp - 4) : (x.rows + 15) >> 4;  // 16-key parts of the pair
        const uint32_t tiles = (parts + H - 1) / H;
        const uint32_t t0 = u0 * kWaves + wave, t1 = min(u1 * kWaves, tiles);
        const uint32_t nt = t0 < t1 ? (t1 - t0 + kWaves - 1) / kWaves : 0;  // tiles of this wave
        const int32_t* table = a.table + size_t(x.seq) * a.width;
        const int32_t* select = a.select ? a.select + (size_t(qi) * a.KH + kh) * a.keep : nullptr;

        // ---- the queries as operands ----
        const float* qrow = a.q + qi * a.stride + (size_t(kh) * a.G + row0 + min(uint32_t(i), R - 1)) * D;
        v4u_t qop[S::kQInLds ? 1 : KC][NP];
        float c = a.scale2;  // takes a score into log2 units
        {
            float4 x0[KC][TYPE == ZQ_KV_F32 ? 1 : 2];
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < KC; ++k)
#pragma unroll
                for (int j = 0; j < (TYPE == ZQ_KV_F32 ? 1 : 2); ++j) {
                    float4 y = *reinterpret_cast<const float4*>(qrow + (4 * k + g) * (TYPE == ZQ_KV_F32 ? 4 : 8) + 4 * j);
                    if (uint32_t(i) >= R) y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x0[k][j] = y;
                    most = fmaxf(most, fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
                }
            float up = 1.0f;
            if constexpr (TYPE == ZQ_KV_F16) {  // the row's largest element to 2^14 .. 2^15
                most = max_groups(most);
                if (most > 0.0f) {
                    const int e = min(max(15 - __builtin_amdgcn_frexp_expf(most), -113), 126);
                    up = pow2f(e);
                    c *= pow2f(-e);
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
                if constexpr (S::kQInLds) {
                    v4u_t* at = reinterpret_cast<v4u_t*>(dyn + kWaves * R * (D + 4));
                    if (k % kWaves == wave)
#pragma unroll
                        for (int n = 0; n < NP; ++n) at[(k * NP + n) * 64 + lane] = op[n];
                } else {
#pragma unroll
                    for (int n = 0; n < NP; ++n) qop[k][n] = op[n];
                }
            }
        }
        if constexpr (S::kQInLds) __syncthreads();

        // ---- the wave's tiles ----
        v4u_t kt[H][KC];
        uint32_t vt[VR][VC][VW];
        v4f_t o[VC][VE];
#pragma unroll
        for (int n = 0; n < VC; ++n)
#pragma unroll
            for (int e = 0; e < VE; ++e) o[n][e] = v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -INFINITY, l = 0.0f;
        uint32_t place = 0;  // lane p: page | rows there << 24 of the p-th part that the wave has ahead
        // byte offset of the wave's part p (of 64) from the cache's start
        auto part_at = [&](uint32_t p, uint32_t part) {
            const uint32_t page = uint32_t(__builtin_amdgcn_readlane(int(place), int(p))) & 0xffffffu;
            const uint32_t in = (part << 4) & (uint32_t(head_rows) - 1);
            return ((size_t(page) * a.KH + kh) * head_rows + in) * (D * S::ES);
        };
        auto rows_at = [&](uint32_t p) { return uint32_t(__builtin_amdgcn_readlane(int(place), int(p))) >> 24; };
        constexpr uint32_t kBatch = 64 / H;  // tiles whose places a wave holds
        for (uint32_t b = 0; b < nt; b += kBatch) {
            {
                const uint32_t j = b + lane / H, part = (t0 + j * kWaves) * H + lane % H, e = part >> (a.lp - 4);
                place = 0;
                if (j < nt && e < entries) {
                    const uint32_t y = select ? uint32_t(select[e]) : e;  // place in the sequence
                    if (y < a.width && (y << a.lp) < x.rows) {
                        const uint32_t page = uint32_t(table[y]);
                        const uint32_t first = (y << a.lp) + ((part << 4) & (uint32_t(head_rows) - 1));
                        if (page < a.pages && first < x.rows) place = page | min(x.rows - first, 16u) << 24;
                    }
                }
            }
            const uint32_t count = min(nt - b, kBatch);
            auto load_k = [&](uint32_t j) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const uint8_t* p = a.k + part_at(j * H + h, (t0 + (b + j) * kWaves) * H + h);
#pragma unroll
                    for (int k = 0; k < KC; ++k)
                        kt[h][k] = *reinterpret_cast<const v4u_t*>(p + uint32_t(i * D * S::ES + k * 64 + g * 16));
                }
            };
            auto load_v = [&](uint32_t j) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const uint8_t* p = a.v + part_at(j * H + h, (t0 + (b + j) * kWaves) * H + h);
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int n = 0; n < VC; ++n) {
                            const uint8_t* at = p + uint32_t((4 * g + r) * D * S::ES + (n * 16 + i) * VE * S::ES);
                            if constexpr (VW == 4) {
                                const v4u_t w = *reinterpret_cast<const v4u_t*>(at);
#pragma unroll
                                for (int z = 0; z < 4; ++z) vt[h * 4 + r][n][z] = w[z];
                            } else {
                                const v2u_t w = *reinterpret_cast<const v2u_t*>(at);
                                vt[h * 4 + r][n][0] = w[0];
                                vt[h * 4 + r][n][1] = w[1];
                            }
                        }
                }
            };
            load_k(0);
            load_v(0);
            auto step = [&](uint32_t j, auto last) {
                v4f_t s[H];
#pragma unroll
                for (int h = 0; h < H; ++h) s[h] = v4f_t{0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (S::kQInLds) asm volatile("" ::: "memory");  // q is read again, not held
#pragma unroll
                for (int k = 0; k < KC; ++k) {
                    v4u_t op[NP];
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        if constexpr (S::kQInLds)
                            op[n] = reinterpret_cast<const v4u_t*>(dyn + kWaves * R * (D + 4))[(k * NP + n) * 64 + lane];
                        else
                            op[n] = qop[k][n];
                    }
#pragma unroll
                    for (int h = 0; h < H; ++h) {
                        if constexpr (TYPE == ZQ_KV_F32) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f(kt[h][k][e]), bits_f(op[0][e]), s[h], 0, 0, 0);
                        } else {
#pragma unroll
                            for (int n = NP - 1; n >= 0; --n) s[h] = mma<TYPE>(kt[h][k], op[n], s[h]);
                        }
                    }
                }
                uint32_t rows[H];
                bool cut = false;
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    rows[h] = rows_at(j * H + h);
                    cut |= rows[h] < 16;
                }
                if constexpr (!decltype(last)::value) load_k(j + 1);
#pragma unroll
                for (int h = 0; h < H; ++h) s[h] *= c;
                if (cut) {  // uniform
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (uint32_t(4 * g + r) >= rows[h]) s[h][r] = -INFINITY;
                }
                float most = -INFINITY;
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) most = fmaxf(most, s[h][r]);
                if (__any(most > m + kSlack)) {
                    const float to = fmaxf(m, max_groups(most));
                    const float f = to == -INFINITY ? 1.0f : exp2_(m - to);
                    m = to;
                    l *= f;
#pragma unroll
                    for (int n = 0; n < VC; ++n)
#pragma unroll
                        for (int e = 0; e < VE; ++e) o[n][e] *= f;
                }
                const float ms = (m == -INFINITY ? 0.0f : m) - kShift;
                float p[VR];
#pragma unroll
                for (int h = 0; h < H; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        p[h * 4 + r] = exp2_(s[h][r] - ms);
                        l += p[h * 4 + r];
                    }
                if (cut) {
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (uint32_t(4 * g + r) >= rows[h])
#pragma unroll
                                for (int n = 0; n < VC; ++n)
#pragma unroll
                                    for (int z = 0; z < VW; ++z) vt[h * 4 + r][n][z] = 0;
                }
                if constexpr (TYPE == ZQ_KV_F32) {
#pragma unroll
                    for (int n = 0; n < VC; ++n)
#pragma unroll
                        for (int e = 0; e < VE; ++e)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                o[n][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(bits_f(vt[r][n][e]), p[r], o[n][e], 0, 0, 0);
                } else {
                    Parts<TYPE> pp;
#pragma unroll
                    for (int r = 0; r < VR; r += 2) pp.set2(r, p[r], p[r + 1]);
#pragma unroll
                    for (int n = 0; n < VC; ++n)
#pragma unroll
                        for (int e = 0; e < VE; ++e) {
                            v4u_t w;
#pragma unroll
                            for (int z = 0; z < 4; ++z)
                                w[z] = __builtin_amdgcn_perm(vt[2 * z + 1][n][e / 2], vt[2 * z][n][e / 2],
                                                             e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                            for (int y = NP - 1; y >= 0; --y) o[n][e] = mma<TYPE>(w, pp.bits(y), o[n][e]);
                        }
                }
                if constexpr (!decltype(last)::value) load_v(j + 1);
            };
            for (uint32_t j = 0; j + 1 < count; ++j) step(j, std::false_type{});
            step(count - 1, std::true_type{});
        }

        // ---- the four waves' sums as one ----
        l = sum_groups(l);
        if (g == 0) {
            sm[wave][i] = m;
            sl[wave][i] = l;
        }
        if (uint32_t(i) < R) {
            float* to = dyn + (size_t(wave) * R + i) * (D + 4);
#pragma unroll
            for (int n = 0; n < VC; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < VE; e += 4)
                        *reinterpret_cast<float4*>(to + n * 16 * VE + VE * (4 * g + r) + e) =
                            make_float4(o[n][e][r], o[n][e + 1][r], o[n][e + 2][r], o[n][e + 3][r]);
        }
        __syncthreads();
        const bool whole = u0 == 0 && u1 == u;
        const size_t slot = (size_t(blockIdx.x) * 2 + (pos != begin)) * a.G + row0;
        float* out = whole ? a.out + (size_t(qi) * a.KH * a.G + size_t(kh) * a.G + row0) * D : a.part + slot * D;
        for (uint32_t z = threadIdx.x; z < R * (D / 4); z += kT) {
            const uint32_t r = z / (D / 4), d = z % (D / 4) * 4;
            float M = sm[0][r];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sm[w][r]);
            const float Ms = M == -INFINITY ? 0.0f : M;
            float L = 0.0f;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = exp2_(sm[w][r] - Ms);
                const float4 t = *reinterpret_cast<const float4*>(dyn + (w * R + r) * (D + 4) + d);
                L += sl[w][r] * f;
                y.x += t.x * f, y.y += t.y * f, y.z += t.z * f, y.w += t.w * f;
            }
            if (whole) {
                const float inv = L > 0.0f ? 1.0f / L : (L == 0.0f ? 0.0f : L);  // no row: 0; NaN stays
                y.x *= inv, y.y *= inv, y.z *= inv, y.w *= inv;
            } else if (d == 0) {
                a.part_ml[(slot + r) * 2] = M;
                a.part_ml[(slot + r) * 2 + 1] = L;
            }
            *reinterpret_cast<float4*>(out + size_t(r) * D + d) = y;
        }
        __syncthreads();
        pos += u1 - u0;
    }
}

// ---- join ------------------------------------------------------------------------
// Workgroup (b, r) puts row r of the pair together that the end of share b cuts, if
// it is the first share's end in that pair.
template <int TYPE, int D>
__global__ __launch_bounds__(kT) void attn_paged_join_kernel(AttnPaged a, uint32_t W) {
    constexpr int E = D / 64;  // elements of a lane
    __shared__ ShareScan scan;
    __shared__ float acc[kWaves][D];
    __shared__ float wm[kWaves], wl[kWaves];
    const auto units = [&](uint32_t n) { return units_of<TYPE>(a, n); };
    uint32_t mine, own;
    const Shares sh = scan_units(a.see.n, a.KH, W, units, scan, mine, own);
    const uint32_t b = blockIdx.x + 1;
    if (b >= sh.used) return;
    const uint64_t x = share_start(sh, b), x0 = share_start(sh, b - 1);
    find_query(a.see.n, a.KH, units, scan, x, mine, own);
    const uint32_t qi = scan.query, u = units(qi);
    const uint64_t base = uint64_t(scan.before) * a.KH;
    const uint32_t kh = uint32_t(x - base) / u;
    const uint64_t first = base + uint64_t(kh) * u;  // the pair's units: first .. first + u
    if (x == first || x0 > first) return;
    // partials: of share b - 1, then of shares b, b + 1, ... that start below the pair's end
    const uint32_t r = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    auto slot = [&](uint32_t w) { return (size_t(w) * 2 + (w == b - 1 && x0 != first)) * a.G + r; };
    uint32_t n = uint32_t(((first + u) * sh.used - 1) / sh.all) - (b - 1) + 1;  // shares with a part of it
    while (share_start(sh, b - 1 + n) < first + u) ++n;
    while (n > 1 && share_start(sh, b - 1 + n - 1) >= first + u) --n;
    float M = -INFINITY;
    for (uint32_t j = threadIdx.x; j < n; j += kT) M = fmaxf(M, a.part_ml[slot(b - 1 + j) * 2]);
    M = wave_max(M);
    if (lane == 0) wm[wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(wm[0], wm[1]), fmaxf(wm[2], wm[3]));
    const float Ms = M == -INFINITY ? 0.0f : M;
    float L = 0.0f, y[E] = {};
#pragma unroll 4
    for (uint32_t j = wave; j < n; j += kWaves) {
        const size_t at = slot(b - 1 + j);
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
    for (uint32_t d = threadIdx.x; d < D; d += kT)
        a.out[(size_t(qi) * a.KH * a.G + size_t(kh) * a.G + r) * D + d] = ((acc[0][d] + acc[1][d]) + (acc[2][d] + acc[3][d])) * inv;
}

// Workgroups for a call: three a CU are resident (two with D = 256), and as many as
// there are units at most.
uint32_t shares_of(const zq_kv_paged& c, const zq_page_tables& t, size_t queries) {
    const size_t unit = c.type == ZQ_KV_F32 ? 64 : 128;
    const size_t most = queries * c.kv_heads * ((t.width * t.page_size + unit - 1) / unit);
    const size_t want = 256 * (c.head_dim == 256 ? 2 : 3);
    return uint32_t(most < want ? most : want);
}

template <int TYPE, int D>
hipError_t run_attention(const AttnPaged& a, uint32_t W, hipStream_t stream) {
    using S = Shape<TYPE, D>;
    const uint32_t R = a.G < 16 ? a.G : 16;
    const size_t lds = size_t(kWaves) * R * (D + 4) * 4 + (S::kQInLds ? size_t(S::KC) * S::NP * 64 * 16 : 0);
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_paged_kernel<TYPE, D>),
                                                 hipFuncAttributeMaxDynamicSharedMemorySize, int(lds));
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((attn_paged_kernel<TYPE, D>), dim3(W, (a.G + 15) / 16), dim3(kT), lds, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || W == 1) return e;
    hipLaunchKernelGGL((attn_paged_join_kernel<TYPE, D>), dim3(W - 1, a.G), dim3(kT), 0, stream, a, W);
    return hipGetLastError();
}
template <int TYPE>
hipError_t run_attention(const AttnPaged& a, uint32_t W, size_t D, hipStream_t stream) {
    return D == 64 ? run_attention<TYPE, 64>(a, W, stream)
                   : D == 128 ? run_attention<TYPE, 128>(a, W, stream) : run_attention<TYPE, 256>(a, W, stream);
}

size_t workspace(const zq_kv_paged& c, const zq_page_tables& t, size_t queries, size_t heads) {
    const size_t rows = size_t(shares_of(c, t, queries)) * 2 * (heads / c.kv_heads);
    return (rows * (c.head_dim + 2) * 4 + 255) / 256 * 256;
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
    const uint32_t W = zq::shares_of(*cache, *tables, queries), G = uint32_t(heads / cache->kv_heads);
    zq::AttnPaged a{};
    a.k = static_cast<const uint8_t*>(cache->k);
    a.v = static_cast<const uint8_t*>(cache->v);
    a.table = tables->table;
    a.select = select;
    a.q = q;
    a.out = out;
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + size_t(W) * 2 * G * cache->head_dim;
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
    return zq::status(cache->type == ZQ_KV_F32   ? zq::run_attention<ZQ_KV_F32>(a, W, cache->head_dim, st)
                      : cache->type == ZQ_KV_F16 ? zq::run_attention<ZQ_KV_F16>(a, W, cache->head_dim, st)
                                                 : zq::run_attention<ZQ_KV_BF16>(a, W, cache->head_dim, st));
}

}  // extern "C"
