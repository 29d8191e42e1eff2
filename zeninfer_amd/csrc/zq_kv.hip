// zq_kv.hip -- the 4-bit KV cache of include/zq_kv.h: append, read-back,
// eviction, and the C entry points (the attention's kernels are in
// zq_attn_q4.hip).
#include "../../include/zq_hip.h"
#include "zq_internal.hpp"
#include "zq_kv.hpp"

#include <math.h>

namespace zq {
namespace {

constexpr int kT = 256;

// ---- append ------------------------------------------------------------------
// One lane takes four consecutive elements of a row's key and of its value, so 8
// lanes hold a block and D / 4 lanes a row; a wave takes 256 / D rows (one row =
// one token of one kv head).  Bound by its launch and two dependent round trips to
// memory, then by the fp32 rows it reads, 8 D bytes a row against D + D / 8 written: 1024
// tokens of 8 kv heads, D = 128, 9.6 MB, take 6.2 us, 1.5 TB/s; 26 tokens 3.7 us.
// The block's scale is an eighth of its element of largest magnitude, negated,
// so that this element gets code 0 and all 16 codes are in use.  m / -8 is exact;
// rounding it to bf16 leaves (code - 8) * d with at most 11 significant bits,
// which fp16 holds exactly: the attention's matrix operands need no second part.
// The quotient x / d of the correctly rounded division lies on a half only if the
// exact one does (x is on d's grid near such a quotient, and the next x on either
// side is a relative 2^-24 away, at least half a spacing of the quotient), so
// rintf gives the nearest code of the exact quotient.
struct Q4Block {
    uint32_t codes;  // lanes 0..3 of the block's 8: bytes 4 l .. 4 l + 3
    uint16_t scale;
};
__device__ __forceinline__ uint32_t group8_max(uint32_t v) {
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), kDppXor1, 0xF, 0xF, false)));
    v = max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), kDppXor2, 0xF, 0xF, false)));
    return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), kDppHalfMirror, 0xF, 0xF, false)));
}
__device__ __forceinline__ Q4Block quantize_block(float4 x, bool poison, bool is_key) {
    const float e[4] = {x.x, x.y, x.z, x.w};
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(e[i]) & 0x7fffffffu);
    m = group8_max(m);
    // the first element that has the largest magnitude: as 2 * (32 - index) + sign, so the max is the first
    const uint32_t l8 = threadIdx.x & 7u;
    uint32_t at = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        const uint32_t u = __float_as_uint(e[i]);
        if ((u & 0x7fffffffu) == m) at = 2u * (32u - (4u * l8 + uint32_t(i))) + (u >> 31);
    }
    at = group8_max(at);
    const float top = __uint_as_float(m | ((at & 1u) << 31));
    uint32_t u = __float_as_uint(top / -8.0f);
    u = (u + 0x7fffu + ((u >> 16) & 1u)) & 0xffff0000u;  // bf16, to nearest even (m is finite here or unused)
    const _Float16 h = _Float16(fminf(fmaxf(__uint_as_float(u), -4096.0f), 4096.0f));
    const float d = float(h);
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float r = d != 0.0f ? fminf(fmaxf(rintf(e[i] / d), -8.0f), 7.0f) : 0.0f;
        c |= (poison ? 8u : uint32_t(int(r) + 8)) << (8 * i);
    }
    Q4Block b;
    const uint32_t hi = uint32_t(__shfl(int(c), int(threadIdx.x & 63u) ^ 4));  // elements 16 on: the block's lanes 4..7
    b.codes = c | (hi << 4);
    b.scale = poison ? (is_key ? 0x7e00u : 0u) : (d != 0.0f ? __builtin_bit_cast(uint16_t, h) : uint16_t(0));
    return b;
}

// Four elements of a row's key and value, by the D / 4 lanes of a row, into `slot`
// (every lane of the wave takes part; a row with live = false writes nothing).
template <int D>
__device__ __forceinline__ void append_row(const zq_kv_q4& c, size_t head, size_t slot, float4 kx, float4 vx, int32_t pos,
                                           bool live) {
    constexpr uint32_t RL = D / 4;  // lanes of a row
    const uint32_t l = threadIdx.x % RL;
    auto odd = [](float4 x) {  // any exponent of all ones: NaN or infinity
        const uint32_t e = 0x7f800000u;
        return (__float_as_uint(x.x) & e) == e || (__float_as_uint(x.y) & e) == e || (__float_as_uint(x.z) & e) == e ||
               (__float_as_uint(x.w) & e) == e;
    };
    const uint64_t bad = __ballot(odd(kx) || odd(vx));
    const uint32_t row0 = (threadIdx.x & 63u) / RL * RL;  // first lane of this row in the wave
    const bool poison = ((bad >> row0) & (RL == 64 ? ~uint64_t(0) : (uint64_t(1) << (RL & 63u)) - 1)) != 0;
    const Q4Block bk = quantize_block(kx, poison, true);
    const Q4Block bv = quantize_block(vx, poison, false);
    if (!live) return;
    const size_t at = head * c.capacity + slot;
    const uint32_t b = l / 8, l8 = l % 8;
    if (l8 < 4) {
        *reinterpret_cast<uint32_t*>(c.k + at * (D / 2) + b * 16 + l8 * 4) = bk.codes;
        *reinterpret_cast<uint32_t*>(c.v + at * (D / 2) + b * 16 + l8 * 4) = bv.codes;
    } else if (l8 == 4) {
        const size_t sc = (head * (D / 32) + b) * c.capacity + slot;
        c.k_scale[sc] = bk.scale;
        c.v_scale[sc] = bv.scale;
    }
    if (l == 0) {
        if (c.weight) c.weight[at] = 0.0f;
        if (c.pos) c.pos[at] = pos;
    }
}

template <int D>
__global__ __launch_bounds__(kT) void kv_q4_append_kernel(const float* __restrict__ k, const float* __restrict__ v,
                                                          zq_kv_q4 c, uint32_t tokens, size_t stride,
                                                          const int32_t* __restrict__ lens,
                                                          const int32_t* __restrict__ counts,
                                                          const int32_t* __restrict__ first_pos, uint32_t rows) {
    constexpr uint32_t RL = D / 4;
    const uint32_t KH = uint32_t(c.kv_heads);
    const uint32_t id = blockIdx.x * (kT / RL) + threadIdx.x / RL, l = threadIdx.x % RL;
    const uint32_t row = min(id, rows - 1);  // every lane of a wave takes part in the block's reductions
    const uint32_t kh = row % KH, st = row / KH, t = st % tokens, s = st / tokens;
    const int32_t len = lens[s];
    const int32_t n = counts ? counts[s] : int32_t(tokens);
    const bool live = id < rows && int32_t(t) < n && len >= 0 && size_t(len) + t < c.capacity;
    const size_t slot = live ? size_t(len) + t : 0;
    const size_t src = size_t(st) * stride + size_t(kh) * D + 4 * l;
    const float4 z = make_float4(0, 0, 0, 0);
    const float4 kx = live ? *reinterpret_cast<const float4*>(k + src) : z;
    const float4 vx = live ? *reinterpret_cast<const float4*>(v + src) : z;
    append_row<D>(c, size_t(s) * KH + kh, slot, kx, vx, (first_pos ? first_pos[s] : len) + int32_t(t), live);
}

// The decoder's form: rows are the heads of a token, H query heads and then the kv
// heads.  Pairs (2 i, 2 i + 1) of a float4 rotate by positions' factors; elements past
// 2 * pairs are left (rope(), :317-328 of the reference runtime).  Bound as the append:
// 32 + 8 heads of D = 128, one token 3.8 us, 1024 tokens (43 MB, most of it q) 16.4, 2.6 TB/s.
template <int D>
__global__ __launch_bounds__(kT) void rope_kv_q4_kernel(zq_kv_q4 c, const float* q, float* q_out,
                                                        const float* __restrict__ k, const float* __restrict__ v,
                                                        const float* __restrict__ cos_tab,
                                                        const float* __restrict__ sin_tab,
                                                        const int32_t* __restrict__ len_ptr,
                                                        const uint32_t* __restrict__ pos_ptr, uint32_t H, uint32_t pairs,
                                                        uint32_t ldq, uint32_t ldkv, uint32_t rows) {
    constexpr uint32_t RL = D / 4;
    const uint32_t heads = H + uint32_t(c.kv_heads);
    const uint32_t id = blockIdx.x * (kT / RL) + threadIdx.x / RL, l = threadIdx.x % RL;
    const uint32_t row = min(id, rows - 1), t = row / heads, h = row % heads;
    const bool is_q = h < H;
    const uint32_t kh = is_q ? 0 : h - H;
    const int32_t len = *len_ptr;
    const uint32_t pos = *pos_ptr + t;
    const float4 x = is_q ? *reinterpret_cast<const float4*>(q + size_t(t) * ldq + size_t(h) * D + 4 * l)
                          : *reinterpret_cast<const float4*>(k + size_t(t) * ldkv + size_t(kh) * D + 4 * l);
    const float4 vx = is_q ? make_float4(0, 0, 0, 0)
                           : *reinterpret_cast<const float4*>(v + size_t(t) * ldkv + size_t(kh) * D + 4 * l);
    float4 y = x;
    const uint32_t i = 2 * l;  // the float4's pairs
    if (i < pairs) {
        const float c0 = cos_tab[size_t(pos) * pairs + i], s0 = sin_tab[size_t(pos) * pairs + i];
        y.x = x.x * c0 - x.y * s0;
        y.y = x.x * s0 + x.y * c0;
    }
    if (i + 1 < pairs) {
        const float c1 = cos_tab[size_t(pos) * pairs + i + 1], s1 = sin_tab[size_t(pos) * pairs + i + 1];
        y.z = x.z * c1 - x.w * s1;
        y.w = x.z * s1 + x.w * c1;
    }
    const bool live = id < rows && !is_q && len >= 0 && size_t(len) + t < c.capacity;
    append_row<D>(c, kh, live ? size_t(len) + t : 0, y, vx, int32_t(pos), live);
    if (id < rows && is_q) *reinterpret_cast<float4*>(q_out + (size_t(t) * H + h) * D + 4 * l) = y;
}

// ---- read ----------------------------------------------------------------------
// A lane gives four elements (the low or the high nibbles of four bytes), so a
// row's stores are as wide as its fp32 elements allow: bound by those.  262,144 rows,
// D = 128: 54 us, 5.7 TB/s; 8192 rows 4.8 us.
template <int D>
__global__ __launch_bounds__(kT) void kv_q4_read_kernel(zq_kv_q4 c, float* __restrict__ k, float* __restrict__ v,
                                                        uint32_t tokens, const int32_t* __restrict__ first,
                                                        const int32_t* __restrict__ counts, uint32_t rows) {
    constexpr uint32_t RL = D / 4;
    const uint32_t KH = uint32_t(c.kv_heads);
    const uint32_t row = blockIdx.x * (kT / RL) + threadIdx.x / RL, l = threadIdx.x % RL;
    if (row >= rows) return;
    const uint32_t kh = row % KH, st = row / KH, t = st % tokens, s = st / tokens;
    const int32_t f = first[s];
    if (int32_t(t) >= (counts ? counts[s] : int32_t(tokens)) || f < 0 || size_t(f) + t >= c.capacity) return;
    const size_t slot = size_t(f) + t, head = size_t(s) * KH + kh, at = head * c.capacity + slot;
    const uint32_t b = l / 8, l8 = l % 8;
    const size_t code = at * (D / 2) + b * 16 + (l8 & 3u) * 4, sc = (head * (D / 32) + b) * c.capacity + slot;
    const size_t dst = (size_t(st) * KH + kh) * D + 4 * l;
    auto four = [&](const uint8_t* codes, const uint16_t* scales) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(codes + code) >> (l8 & 4u);
        const float d = half_bits_to_float(scales[sc]);
        return make_float4(float(int(w & 15u) - 8) * d, float(int((w >> 8) & 15u) - 8) * d,
                           float(int((w >> 16) & 15u) - 8) * d, float(int((w >> 24) & 15u) - 8) * d);
    };
    if (k) *reinterpret_cast<float4*>(k + dst) = four(c.k, c.k_scale);
    if (v) *reinterpret_cast<float4*>(v + dst) = four(c.v, c.v_scale);
}

// ---- evict ---------------------------------------------------------------------
// One workgroup a (sequence, kv head) finds the rows that stay and, for every slot
// below the new length, the slot its row comes from; it also moves weight and pos.
// Free slots are filled from above the new length, so what is written and what is read
// never meet, in place or not, and only evicted slots are written in place.
// A second launch copies the rows' codes and scales (the one workgroup would take 11 us
// for 1024 rows of D = 64 where that launch takes 3).
// Bound by latency: the keys in one read, three digits of an LDS histogram, the ranks.
// 128 of them with 8192 rows take 19 us (14 where an L2 holds their weights), 8 with 1153
// rows 7; a decoder's 256, 1024 rows more than the 2048 that stay, 15.
constexpr int kEvT = 1024, kEvWaves = kEvT / 64;
constexpr int kEvHeld = 24;  // keys a thread holds at most: caches up to 24576 rows are read once

// Order of a row: protected ones, then by weight (-0 = +0), a NaN last.
__device__ __forceinline__ uint32_t evict_key(float w, bool held) {
    if (held) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Sums of v over the lanes below this one, and of all lanes: DPP shifts within rows of
// 16 lanes, then the rows' sums on to the rows behind them.
__device__ __forceinline__ uint32_t wave_before(uint32_t v, uint32_t& all) {
    auto step = [](uint32_t s, auto ctrl, auto rows) {
        return s + uint32_t(__builtin_amdgcn_update_dpp(0, int(s), decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
    };
    using std::integral_constant;
    uint32_t s = v;
    s = step(s, integral_constant<int, 0x111>{}, integral_constant<int, 0xF>{});  // row_shr:1, 2, 4, 8
    s = step(s, integral_constant<int, 0x112>{}, integral_constant<int, 0xF>{});
    s = step(s, integral_constant<int, 0x114>{}, integral_constant<int, 0xF>{});
    s = step(s, integral_constant<int, 0x118>{}, integral_constant<int, 0xF>{});
    s = step(s, integral_constant<int, 0x142>{}, integral_constant<int, 0xA>{});  // row_bcast:15 into rows 1 and 3
    s = step(s, integral_constant<int, 0x143>{}, integral_constant<int, 0xC>{});  // row_bcast:31 into rows 2 and 3
    all = uint32_t(__builtin_amdgcn_readlane(int(s), 63));
    return s - v;
}

// N: keys a thread holds, for caches of up to N * 1024 rows; the largest N reads longer ones
// again for every digit.  A cache takes the smallest N that holds it, as every pass over the
// keys is N steps: 128 caches of 8192 rows take 14 us with N = 8 (20 from HBM), 23 with 16; 24,000 rows 36
// with 24, 41 with 32 (registers spilled); 40,000 rows 107.
template <int N>
__device__ __forceinline__ void evict_rows(const zq_kv_q4& c, const zq_kv_q4& dst, int in_place, uint32_t head, uint32_t n,
                                           uint32_t keep, int64_t newest, uint32_t first, int32_t* __restrict__ ws) {
    constexpr int kBins = 2048;
    __shared__ uint32_t hist[2][kBins];
    __shared__ uint32_t pick[2];           // the digit found, and the rows wanted among those that have it
    __shared__ uint32_t sums[kEvWaves];
    __shared__ uint32_t counts[N][kEvWaves];
    const uint32_t kept = keep;  // n > keep
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float* w = c.weight + size_t(head) * c.capacity;
    const int32_t* pos = c.pos + size_t(head) * c.capacity;
    float* dw = dst.weight + size_t(head) * dst.capacity;
    int32_t* dp = dst.pos + size_t(head) * dst.capacity;
    int32_t* from = ws + size_t(head) * 3 * keep;  // [keep] the slot that slot j's row comes from
    int32_t* holes = from + keep;                  // free slots below the new length, ascending
    int32_t* above = holes + keep;                 // kept slots from the new length on, ascending
    auto key = [&](uint32_t i) {
        const int32_t p = pos[i];
        return evict_key(w[i], p >= 0 && (int64_t(p) >= newest || p < int64_t(first)));
    };
    const bool held = N < kEvHeld || n <= uint32_t(kEvHeld * kEvT);  // uniform
    uint32_t mine[N];
    // (loads past the end take the last row: no branch between them, all are under way at once)
    auto load_keys = [&](uint32_t i0) {
#pragma unroll
        for (int j = 0; j < N; ++j) mine[j] = key(min(i0 + uint32_t(j * kEvT + tid), n - 1));
    };
    if (held) load_keys(0);
    // the key of rank `kept`, by digits of 11, 11 and 10 bits from the top: want = rows still to be found among
    // those that share its digits so far.  (A first digit of sign, exponent and two bits spreads weights over
    // enough bins that the LDS atomics of a wave seldom meet.)
    uint32_t prefix = 0, want = kept;
    hist[0][tid] = hist[0][tid + kEvT] = 0;
    __syncthreads();
    for (int d = 0; d < 3; ++d) {
        const int shift = d == 0 ? 21 : d == 1 ? 10 : 0, up = d == 0 ? 32 : d == 1 ? 21 : 10;
        const uint32_t mask = d == 2 ? 1023u : 2047u;
        uint32_t* bins = hist[d & 1];
        auto count = [&](uint32_t x) {
            if (d == 0 || (x >> up) == (prefix >> up)) atomicAdd(&bins[(x >> shift) & mask], 1u);
        };
        if (held) {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (uint32_t(j * kEvT) < n && uint32_t(j * kEvT + tid) < n) count(mine[j]);
        } else {
            for (uint32_t i = tid; i < n; i += kEvT) count(key(i));
        }
        __syncthreads();
        // thread t holds bins 2047 - 2 t and 2046 - 2 t; rows in higher bins than its own by two scans
        const uint32_t h0 = bins[kBins - 1 - 2 * tid], h1 = bins[kBins - 2 - 2 * tid];
        hist[(d + 1) & 1][tid] = hist[(d + 1) & 1][tid + kEvT] = 0;  // the next digit's
        uint32_t all;
        uint32_t before = wave_before(h0 + h1, all);
        if (lane == 0) sums[wave] = all;
        __syncthreads();
        for (int k = 0; k < kEvWaves; ++k) before += k < wave ? sums[k] : 0u;
        if (before < want && want <= before + h0) {
            pick[0] = uint32_t(kBins - 1 - 2 * tid);
            pick[1] = want - before;
        } else if (before + h0 < want && want <= before + h0 + h1) {
            pick[0] = uint32_t(kBins - 2 - 2 * tid);
            pick[1] = want - before - h0;
        }
        __syncthreads();
        prefix |= pick[0] << shift;
        want = pick[1];
    }
    // in slot order: a row stays if its key is above the found one, or equal and among the first `want`
    const uint64_t below = (uint64_t(1) << lane) - 1;
    uint32_t equal = 0, free_n = 0, above_n = 0;  // of the passes over N * 1024 rows before this one
    for (uint32_t i0 = 0; i0 < n; i0 += N * kEvT) {
        if (!held) load_keys(i0);
        // counts of [j][wave], then what stands before each of them in slot order; returns the sum of all
        constexpr int SW = (N * kEvWaves + 63) / 64;  // waves that scan
        auto scan_counts = [&] {
            __syncthreads();
            if (wave < SW) {
                uint32_t& at = counts[tid / kEvWaves][tid % kEvWaves];
                uint32_t all;
                const uint32_t b = wave_before(tid < N * kEvWaves ? at : 0u, all);
                if (tid < N * kEvWaves) at = b;
                if (lane == 0) sums[wave] = all;
            }
            __syncthreads();
            uint32_t all = 0;
            for (int k = 0; k < SW; ++k) all += sums[k];
            return all;
        };
        auto before = [&](int j) {  // of this wave's part of [j]
            uint32_t b = counts[j][wave];
            const int q = j * kEvWaves / 64;  // the scanning wave that part belonged to
            for (int k = 0; k < q; ++k) b += sums[k];
            return b;
        };
        __syncthreads();
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = i0 + uint32_t(j * kEvT + tid);
            uint64_t eq = 0;
            if (i0 + uint32_t(j * kEvT) < n) eq = __ballot(i < n && mine[j] == prefix);  // uniform
            if (lane == 0) counts[j][wave] = uint32_t(__popcll(eq));
        }
        const uint32_t eq_all = scan_counts();
        uint32_t stay = 0;  // bit j: row j stays
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = i0 + uint32_t(j * kEvT + tid);
            if (i0 + uint32_t(j * kEvT) < n) {  // uniform
                const bool eq = i < n && mine[j] == prefix;
                const uint64_t b = __ballot(eq);
                const uint32_t r = equal + before(j) + uint32_t(__popcll(b & below));
                if (i < n && (mine[j] > prefix || (eq && r < want))) stay |= 1u << j;
            }
        }
        equal += eq_all;
        __syncthreads();  // the counts are read
        // holes and kept rows above, counted together: 16 bits each (at most 24576 in a pass)
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = i0 + uint32_t(j * kEvT + tid);
            const bool st = (stay >> j) & 1u;
            uint64_t h = 0, u = 0;
            if (i0 + uint32_t(j * kEvT) < n) h = __ballot(i < kept && !st), u = __ballot(i >= kept && st);
            if (lane == 0) counts[j][wave] = uint32_t(__popcll(h)) | uint32_t(__popcll(u)) << 16;
        }
        const uint32_t both = scan_counts();
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t i = i0 + uint32_t(j * kEvT + tid);
            if (i0 + uint32_t(j * kEvT) < n) {
                const bool st = (stay >> j) & 1u, hole = i < kept && !st, up = i >= kept && st;
                const uint64_t h = __ballot(hole), u = __ballot(up);
                const uint32_t b = before(j);
                if (hole) holes[free_n + (b & 0xffffu) + uint32_t(__popcll(h & below))] = int32_t(i);
                if (up) above[above_n + (b >> 16) + uint32_t(__popcll(u & below))] = int32_t(i);
                if (i < kept && st) {
                    from[i] = int32_t(i);
                    if (!in_place) {
                        dw[i] = w[i];
                        dp[i] = pos[i];
                    }
                }
            }
        }
        free_n += both & 0xffffu;
        above_n += both >> 16;
    }
    __syncthreads();  // the lists, written by other waves of this workgroup
    for (uint32_t x = tid; x < free_n; x += kEvT) {
        const int32_t h = holes[x], a = above[x];
        from[h] = a;
        dw[h] = w[a];
        dp[h] = pos[a];
    }
    __syncthreads();  // every moved weight and pos has been read
    if (in_place)
        for (uint32_t i = kept + tid; i < n; i += kEvT) {
            dw[i] = -INFINITY;
            dp[i] = -1;
        }
}

__global__ __launch_bounds__(kEvT) void kv_q4_evict_kernel(zq_kv_q4 c, zq_kv_q4 dst, int in_place,
                                                           const int32_t* __restrict__ lens, uint32_t keep,
                                                           uint32_t recent, uint32_t first,
                                                           const int32_t* __restrict__ next_pos,
                                                           int32_t* __restrict__ ws) {
    const uint32_t head = blockIdx.x, s = head / uint32_t(c.kv_heads);
    const uint32_t n = uint32_t(clamp_len(lens[s], c.capacity));
    if (n <= keep) {  // everything stays
        int32_t* from = ws + size_t(head) * 3 * keep;
        const size_t at = size_t(head) * c.capacity, to = size_t(head) * dst.capacity;
        for (uint32_t i = threadIdx.x; i < n; i += kEvT) {
            from[i] = int32_t(i);
            if (!in_place) {
                dst.weight[to + i] = c.weight[at + i];
                dst.pos[to + i] = c.pos[at + i];
            }
        }
        return;
    }
    const int64_t newest = int64_t(next_pos ? next_pos[s] : int32_t(n)) - recent;
    if (n <= 2 * kEvT) evict_rows<2>(c, dst, in_place, head, n, keep, newest, first, ws);
    else if (n <= 8 * kEvT) evict_rows<8>(c, dst, in_place, head, n, keep, newest, first, ws);
    else if (n <= 16 * kEvT) evict_rows<16>(c, dst, in_place, head, n, keep, newest, first, ws);
    else evict_rows<kEvHeld>(c, dst, in_place, head, n, keep, newest, first, ws);
}

// A workgroup copies 64 rows of one (sequence, kv head): codes in 16-byte parts, scales
// one by one from their planes, all loads before the stores.  Kept rows lie anywhere, so a
// row's 64 bytes of codes bring a line of 128 and a scale one of its own: 262,144 rows,
// D = 128, another cache: 32 us for 75 MB that are used; in place, 256 caches that keep 2048
// rows each: 26 us.
constexpr uint32_t kMoveRows = 64;
template <int D>
__global__ __launch_bounds__(kT) void kv_q4_evict_move_kernel(zq_kv_q4 c, zq_kv_q4 dst, int in_place,
                                                              const int32_t* __restrict__ lens, uint32_t keep,
                                                              const int32_t* __restrict__ ws, uint32_t parts) {
    constexpr uint32_t P = D / 32;  // 16-byte parts of a row's codes, and its scales
    constexpr uint32_t I = (kMoveRows * P + kT - 1) / kT;
    __shared__ int32_t from[kMoveRows];
    const uint32_t head = blockIdx.x / parts, j0 = blockIdx.x % parts * kMoveRows, s = head / uint32_t(c.kv_heads);
    const uint32_t kept = min(uint32_t(clamp_len(lens[s], c.capacity)), keep);
    if (j0 >= kept) return;
    const uint32_t n = min(kept - j0, kMoveRows), tid = threadIdx.x;
    if (tid < kMoveRows) from[tid] = ws[size_t(head) * 3 * keep + j0 + min(tid, n - 1)];
    __syncthreads();
    const size_t src = size_t(head) * c.capacity, to = size_t(head) * dst.capacity + j0;
    uint4 k[I], v[I];
    uint16_t ks[I], vs[I];
#pragma unroll
    for (uint32_t i = 0; i < I; ++i) {  // element e: part e % P of row e / P, and scale e / 64 of row e % 64
        const uint32_t e = min(tid + i * kT, kMoveRows * P - 1);
        const size_t a = (src + uint32_t(from[e / P])) * P + e % P;
        k[i] = reinterpret_cast<const uint4*>(c.k)[a];
        v[i] = reinterpret_cast<const uint4*>(c.v)[a];
        const size_t b = (size_t(head) * P + e / kMoveRows) * c.capacity + uint32_t(from[e % kMoveRows]);
        ks[i] = c.k_scale[b];
        vs[i] = c.v_scale[b];
    }
#pragma unroll
    for (uint32_t i = 0; i < I; ++i) {
        const uint32_t e = tid + i * kT;
        if (e >= kMoveRows * P) break;
        const uint32_t j = e / P, js = e % kMoveRows;
        if (j < n && !(in_place && uint32_t(from[j]) == j0 + j)) {
            const size_t b = (to + j) * P + e % P;
            reinterpret_cast<uint4*>(dst.k)[b] = k[i];
            reinterpret_cast<uint4*>(dst.v)[b] = v[i];
        }
        if (js < n && !(in_place && uint32_t(from[js]) == j0 + js)) {
            const size_t b = (size_t(head) * P + e / kMoveRows) * dst.capacity + j0 + js;
            dst.k_scale[b] = ks[i];
            dst.v_scale[b] = vs[i];
        }
    }
}

}  // namespace

bool kv_q4_ok(const zq_kv_q4* c) {
    auto a16 = [](const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    auto a4 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; };
    return c && a16(c->k) && a16(c->v) && a16(c->k_scale) && a16(c->v_scale) && a4(c->weight) && a4(c->pos) &&
           (c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256) && c->capacity && c->capacity % 32 == 0 &&
           c->capacity <= kKvMaxCapacity && c->seqs && c->kv_heads && c->seqs <= kKvMaxHeads &&
           c->kv_heads <= kKvMaxHeads && c->seqs * c->kv_heads <= kKvMaxHeads;
}

hipError_t launch_kv_q4_append(const zq_kv_q4& c, const float* k, const float* v, size_t tokens, size_t stride,
                               const int32_t* lens, const int32_t* counts, const int32_t* first_pos,
                               hipStream_t stream) {
    const uint32_t rows = uint32_t(c.seqs * tokens * c.kv_heads);
    const uint32_t per = uint32_t(kT / (c.head_dim / 4));
    const dim3 grid((rows + per - 1) / per);
#define ZQ_KV(DD)                                                                                                \
    hipLaunchKernelGGL(kv_q4_append_kernel<DD>, grid, dim3(kT), 0, stream, k, v, c, uint32_t(tokens), stride, lens, \
                       counts, first_pos, rows)
    if (c.head_dim == 64) ZQ_KV(64);
    else if (c.head_dim == 128) ZQ_KV(128);
    else ZQ_KV(256);
#undef ZQ_KV
    return hipGetLastError();
}

hipError_t launch_rope_kv_q4(const zq_kv_q4& c, const float* q, float* q_out, const float* k, const float* v,
                             const float* cos_tab, const float* sin_tab, const int32_t* len, const uint32_t* pos,
                             uint32_t T, uint32_t H, uint32_t pairs, uint32_t ld, hipStream_t stream) {
    const uint32_t D = uint32_t(c.head_dim), KH = uint32_t(c.kv_heads);
    auto a16 = [](const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
    if (!kv_q4_ok(&c) || c.seqs != 1 || !a16(q) || !a16(q_out) || !a16(k) || !a16(v) || !cos_tab || !sin_tab || !len ||
        !pos || !T || !H || !pairs || pairs > D / 2 || ld % 4 || (ld && ld < (H + 2 * KH) * D))
        return hipErrorInvalidValue;
    const uint32_t rows = T * (H + KH), per = uint32_t(kT) / (D / 4);
    const dim3 grid((rows + per - 1) / per);
#define ZQ_KV(DD)                                                                                                  \
    hipLaunchKernelGGL(rope_kv_q4_kernel<DD>, grid, dim3(kT), 0, stream, c, q, q_out, k, v, cos_tab, sin_tab, len, pos, \
                       H, pairs, ld ? ld : H * D, ld ? ld : KH * D, rows)
    if (D == 64) ZQ_KV(64);
    else if (D == 128) ZQ_KV(128);
    else ZQ_KV(256);
#undef ZQ_KV
    return hipGetLastError();
}

hipError_t launch_kv_q4_read(const zq_kv_q4& c, float* k, float* v, size_t tokens, const int32_t* first,
                             const int32_t* counts, hipStream_t stream) {
    const uint32_t rows = uint32_t(c.seqs * tokens * c.kv_heads);
    const uint32_t per = uint32_t(kT / (c.head_dim / 4));
    const dim3 grid((rows + per - 1) / per);
#define ZQ_KV(DD) \
    hipLaunchKernelGGL(kv_q4_read_kernel<DD>, grid, dim3(kT), 0, stream, c, k, v, uint32_t(tokens), first, counts, rows)
    if (c.head_dim == 64) ZQ_KV(64);
    else if (c.head_dim == 128) ZQ_KV(128);
    else ZQ_KV(256);
#undef ZQ_KV
    return hipGetLastError();
}

size_t kv_q4_evict_bytes(const zq_kv_q4& c, size_t keep) {
    return c.seqs * c.kv_heads * 3 * (keep < c.capacity ? keep : c.capacity) * sizeof(int32_t);
}

hipError_t launch_kv_q4_evict(const zq_kv_q4& c, const zq_kv_q4& dst, bool in_place, const int32_t* lens, size_t keep,
                              size_t recent, size_t first, const int32_t* next_pos, void* ws, hipStream_t stream) {
    const uint32_t heads = uint32_t(c.seqs * c.kv_heads), kp = uint32_t(keep < c.capacity ? keep : c.capacity);
    hipLaunchKernelGGL(kv_q4_evict_kernel, dim3(heads), dim3(kEvT), 0, stream, c, dst, in_place ? 1 : 0, lens, kp,
                       uint32_t(recent), uint32_t(first), next_pos, static_cast<int32_t*>(ws));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const uint32_t parts = (kp + kMoveRows - 1) / kMoveRows;
#define ZQ_KV(DD)                                                                                                  \
    hipLaunchKernelGGL(kv_q4_evict_move_kernel<DD>, dim3(heads * parts), dim3(kT), 0, stream, c, dst, in_place ? 1 : 0, \
                       lens, kp, static_cast<const int32_t*>(ws), parts)
    if (c.head_dim == 64) ZQ_KV(64);
    else if (c.head_dim == 128) ZQ_KV(128);
    else ZQ_KV(256);
#undef ZQ_KV
    return hipGetLastError();
}

}  // namespace zq

// ---- C entry points --------------------------------------------------------------
namespace {

bool a16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool a4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

int status(hipError_t e) { return e == hipSuccess ? ZQ_OK : e == hipErrorInvalidValue ? ZQ_ERR_ARG : ZQ_ERR_HIP; }

// The device that holds the cache made current for the call's launches, and the
// caller's device again after it.
class OnDeviceOf {
public:
    explicit OnDeviceOf(const void* p) {
        hipPointerAttribute_t a;
        if (hipPointerGetAttributes(&a, p) != hipSuccess) {
            (void)hipGetLastError();
            int n = 0;
            st_ = hipGetDeviceCount(&n) == hipSuccess && n > 0 ? ZQ_ERR_ARG : ZQ_ERR_NO_DEVICE;
            (void)hipGetLastError();
            return;
        }
        if (a.type != hipMemoryTypeDevice && a.type != hipMemoryTypeManaged) {
            st_ = ZQ_ERR_ARG;  // an address of the host: a kernel that used it would fault
            return;
        }
        dev_ = a.device;
        if (hipGetDevice(&was_) != hipSuccess) st_ = ZQ_ERR_HIP;
        else if (a.device != was_) {
            moved_ = hipSetDevice(a.device) == hipSuccess;
            if (!moved_) st_ = ZQ_ERR_HIP;
        }
    }
    ~OnDeviceOf() {
        if (moved_) (void)hipSetDevice(was_);
    }
    int status() const { return st_; }
    // p is memory of that device, too
    bool holds(const void* p) const {
        hipPointerAttribute_t a;
        if (hipPointerGetAttributes(&a, p) != hipSuccess) {
            (void)hipGetLastError();
            return false;
        }
        return (a.type == hipMemoryTypeDevice || a.type == hipMemoryTypeManaged) && a.device == dev_;
    }

private:
    int was_ = 0, dev_ = 0, st_ = ZQ_OK;
    bool moved_ = false;
};

// Some array of b meets some array of a.
bool arrays_meet(const zq_kv_q4& a, const zq_kv_q4& b) {
    struct Range {
        uintptr_t at;
        size_t bytes;
    };
    auto ranges = [](const zq_kv_q4& c, Range (&r)[6]) {
        const size_t rows = c.seqs * c.kv_heads * c.capacity, codes = rows * (c.head_dim / 2), scales = rows * (c.head_dim / 16);
        const void* p[6] = {c.k, c.v, c.k_scale, c.v_scale, c.weight, c.pos};
        const size_t n[6] = {codes, codes, scales, scales, rows * 4, rows * 4};
        for (int i = 0; i < 6; ++i) r[i] = {reinterpret_cast<uintptr_t>(p[i]), n[i]};
    };
    Range x[6], y[6];
    ranges(a, x);
    ranges(b, y);
    for (const Range& i : x)
        for (const Range& j : y)
            if (i.at < j.at + j.bytes && j.at < i.at + i.bytes) return true;
    return false;
}

bool tokens_ok(const zq_kv_q4& c, size_t tokens, size_t heads) {
    return tokens && tokens <= zq::kKvMaxRows && heads <= zq::kKvMaxHeads && c.seqs * heads <= zq::kKvMaxRows / tokens;
}

}  // namespace

extern "C" {

size_t zq_kv_q4_bytes(size_t kv_heads, size_t head_dim, size_t capacity) {
    if (!kv_heads || kv_heads > zq::kKvMaxHeads || (head_dim != 64 && head_dim != 128 && head_dim != 256) || !capacity ||
        capacity % 32 || capacity > zq::kKvMaxCapacity)
        return 0;
    return 2 * kv_heads * capacity * (head_dim / 2 + head_dim / 16);
}

int zq_hip_kv_q4_append_dev(const zq_kv_q4* cache, const float* k, const float* v, size_t tokens, size_t stride,
                            const int32_t* lens, const int32_t* counts, const int32_t* first_pos, void* stream) {
    if (!zq::kv_q4_ok(cache) || !k || !v || !lens || !a16(k) || !a16(v) || !a4(lens) || !a4(counts) || !a4(first_pos) ||
        !tokens_ok(*cache, tokens, cache->kv_heads))
        return ZQ_ERR_ARG;
    const size_t width = cache->kv_heads * cache->head_dim;
    if (!stride) stride = width;
    if (stride < width || stride % 4 || stride > (size_t(1) << 31)) return ZQ_ERR_ARG;
    const OnDeviceOf dev(cache->k);
    if (dev.status() != ZQ_OK) return dev.status();
    return status(zq::launch_kv_q4_append(*cache, k, v, tokens, stride, lens, counts, first_pos,
                                          static_cast<hipStream_t>(stream)));
}

int zq_hip_kv_q4_read_dev(const zq_kv_q4* cache, float* k, float* v, size_t tokens, const int32_t* first,
                          const int32_t* counts, void* stream) {
    if (!zq::kv_q4_ok(cache) || (!k && !v) || !first || !a16(k) || !a16(v) || !a4(first) || !a4(counts) ||
        !tokens_ok(*cache, tokens, cache->kv_heads))
        return ZQ_ERR_ARG;
    const OnDeviceOf dev(cache->k);
    if (dev.status() != ZQ_OK) return dev.status();
    return status(zq::launch_kv_q4_read(*cache, k, v, tokens, first, counts, static_cast<hipStream_t>(stream)));
}

size_t zq_hip_attention_q4_workspace_bytes(const zq_kv_q4* cache, size_t tokens, size_t heads, int flags) {
    if (!zq::kv_q4_ok(cache) || !heads || heads % cache->kv_heads || !tokens_ok(*cache, tokens, heads)) return 0;
    return zq::attention_q4_bytes(*cache, tokens, heads, flags);
}

int zq_hip_attention_q4_dev(const zq_kv_q4* cache, const float* q, float* out, size_t tokens, size_t heads,
                            size_t stride, const int32_t* lens, const int32_t* counts, float scale, int flags,
                            void* workspace, size_t workspace_bytes, void* stream) {
    if (!zq::kv_q4_ok(cache) || !q || !out || !lens || !a16(q) || !a16(out) || !a4(lens) || !a4(counts) || !heads ||
        heads % cache->kv_heads || !tokens_ok(*cache, tokens, heads))
        return ZQ_ERR_ARG;
    const int known = ZQ_ATTN_Q4_FULL | ZQ_ATTN_Q4_WEIGHTS | ZQ_ATTN_Q4_ADD;
    if ((flags & ~known) || ((flags & ZQ_ATTN_Q4_ADD) && !(flags & ZQ_ATTN_Q4_WEIGHTS)) ||
        ((flags & ZQ_ATTN_Q4_WEIGHTS) && !cache->weight))
        return ZQ_ERR_ARG;
    const size_t width = heads * cache->head_dim;
    if (!stride) stride = width;
    if (stride < width || stride % 4 || stride > (size_t(1) << 31)) return ZQ_ERR_ARG;
    const size_t need = zq::attention_q4_bytes(*cache, tokens, heads, flags);
    if (need && (!workspace || workspace_bytes < need || !a16(workspace))) return ZQ_ERR_ARG;
    const OnDeviceOf dev(cache->k);
    if (dev.status() != ZQ_OK) return dev.status();
    return status(zq::launch_attention_q4(*cache, q, out, tokens, heads, stride, lens, counts, scale, flags, workspace,
                                          static_cast<hipStream_t>(stream)));
}

size_t zq_hip_kv_q4_evict_workspace_bytes(const zq_kv_q4* cache, size_t keep) {
    if (!zq::kv_q4_ok(cache) || !keep) return 0;
    return zq::kv_q4_evict_bytes(*cache, keep);
}

int zq_hip_kv_q4_evict_dev(const zq_kv_q4* cache, const zq_kv_q4* dst, const int32_t* lens, size_t keep, size_t recent,
                           size_t first, const int32_t* next_pos, void* workspace, size_t workspace_bytes,
                           void* stream) {
    if (!zq::kv_q4_ok(cache) || !cache->weight || !cache->pos || !lens || !a4(lens) || !a4(next_pos) || !keep ||
        recent > keep || first > keep - recent || !workspace || !a16(workspace))
        return ZQ_ERR_ARG;
    if (recent > 0x7fffffffu || first > 0x7fffffffu) return ZQ_ERR_ARG;
    if (!dst) dst = cache;
    const bool in_place = dst->k == cache->k;
    if (in_place) {
        if (dst->v != cache->v || dst->k_scale != cache->k_scale || dst->v_scale != cache->v_scale ||
            dst->weight != cache->weight || dst->pos != cache->pos || dst->seqs != cache->seqs ||
            dst->kv_heads != cache->kv_heads || dst->head_dim != cache->head_dim || dst->capacity != cache->capacity)
            return ZQ_ERR_ARG;
    } else if (!zq::kv_q4_ok(dst) || !dst->weight || !dst->pos || dst->seqs != cache->seqs ||
               dst->kv_heads != cache->kv_heads || dst->head_dim != cache->head_dim ||
               dst->capacity < (keep < cache->capacity ? keep : cache->capacity) || arrays_meet(*cache, *dst)) {
        return ZQ_ERR_ARG;
    }
    if (workspace_bytes < zq::kv_q4_evict_bytes(*cache, keep)) return ZQ_ERR_ARG;
    const size_t parts = ((keep < cache->capacity ? keep : cache->capacity) + 63) / 64;
    if (parts * cache->seqs * cache->kv_heads * 256 > zq::kMaxThreads) return ZQ_ERR_ARG;
    const OnDeviceOf dev(cache->k);
    if (dev.status() != ZQ_OK) return dev.status();
    if (!in_place && !dev.holds(dst->k)) return ZQ_ERR_ARG;
    return status(zq::launch_kv_q4_evict(*cache, *dst, in_place, lens, keep, recent, first, next_pos, workspace,
                                         static_cast<hipStream_t>(stream)));
}

}  // extern "C"
