// zq_paged.hpp -- the paged KV cache inside the library: what the tables and
// append (zq_paged.hip), attention (zq_attn_paged.hip) and selection
// (zq_page_select.hip) share.
#pragma once
#include "../../include/zq_paged.h"
#include "zq_device.hpp"

namespace zq {

// Bounds that keep every index in range: a token's place in its sequence and its
// row of a call fit 31 bits, rows of a pool and byte offsets are 64-bit.
constexpr size_t kPgMaxSeqs = 8192, kPgMaxPages = size_t(1) << 24, kPgMaxTokens = size_t(1) << 24;
constexpr size_t kPgMaxHeads = 1024, kPgMaxStride = size_t(1) << 31;

// Shape, pointers and alignment, as include/zq_paged.h asks for them.
bool page_tables_ok(const zq_page_tables* t);
bool kv_paged_ok(const zq_kv_paged* c);
// The arguments that attention and selection share (after the two above).
bool queries_ok(const zq_kv_paged& c, const zq_page_tables& t, size_t queries, size_t heads, const int32_t* seq_of);

inline uint32_t log2_of(size_t x) { return uint32_t(__builtin_ctzll(x)); }

#if defined(__HIPCC__)
// The queries of a call and what each sees.
struct Queries {
    const int32_t* seq_of;
    const int32_t* lens;
    const int32_t* counts;
    uint32_t n, seqs, cap;  // cap = width * page_size
    int full;
};
struct Seen {
    int32_t seq;    // -1: idle
    uint32_t rows;
};
__device__ __forceinline__ Seen seen_by(const Queries& a, uint32_t i) {
    const int32_t s = a.seq_of ? a.seq_of[i] : int32_t(i);
    const int32_t c = a.counts ? a.counts[i] : 1;
    const int32_t n = min(max(a.lens[i], 0), int32_t(a.cap));
    if (uint32_t(s) >= a.seqs || c <= 0) return {-1, 0};
    return {s, a.full ? uint32_t(n) : min(uint32_t(n) + uint32_t(c), a.cap)};
}

// Sums over the lanes below this one, and over all, of values whose sums may pass
// 31 bits: they stay at 2^31 - 1 then.
__device__ __forceinline__ uint32_t add_sat31(uint32_t a, uint32_t b) { return min(a + b, 0x7fffffffu); }
__device__ __forceinline__ uint32_t wave_before_sat(uint32_t v, uint32_t& all) {
    auto step = [](uint32_t s, auto ctrl, auto rows) {
        return add_sat31(s, uint32_t(__builtin_amdgcn_update_dpp(0, int(s), decltype(ctrl)::value, decltype(rows)::value, 0xF, false)));
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
    const uint32_t up = uint32_t(__builtin_amdgcn_update_dpp(0, int(s), 0x138, 0xF, 0xF, false));  // wave_shr:1
    return (threadIdx.x & 63) == 0 ? 0u : up;
}

// The exponent and the codes that values of magnitude up to `most` are held with:
// the least e in -50 .. 50 with most <= 127 * 2^e.  127 = 127/128 * 2^7.
__device__ __forceinline__ int bound_exp(float most) {
    if (!(most > 0.0f)) return -50;
    if (most == INFINITY) return 50;
    const int e = __builtin_amdgcn_frexp_expf(most) - (__builtin_amdgcn_frexp_mantf(most) <= 127.0f / 128.0f ? 7 : 6);
    return min(max(e, -50), 50);
}
__device__ __forceinline__ int bound_code(float x) { return int(fminf(fmaxf(x, -127.0f), 127.0f)); }

// ---- even shares of uneven work ------------------------------------------------
// Query i has units(i) units of work for each of `mult` kv heads (0 where it is idle);
// the units of all, one behind the other, are cut into equal shares, one a workgroup,
// whatever the lengths are.  Every workgroup of 256 takes the sums by itself, and holds
// what the queries see in LDS where they are few: what follows then waits for no memory.
constexpr int kShareT = 256, kShareWaves = kShareT / 64;
constexpr uint32_t kSeenHeld = 1024;
struct ShareScan {
    int32_t seq[kSeenHeld];
    uint32_t rows[kSeenHeld];
    uint32_t part[kShareWaves];
    uint32_t query, before;
};
struct Shares {
    uint32_t units;  // of all queries, for one kv head
    uint64_t all;    // of all kv heads
    uint32_t used;   // workgroups that have a share
};
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return uint32_t(__builtin_amdgcn_readfirstlane(int(x))); }
__device__ __forceinline__ uint64_t share_start(const Shares& s, uint32_t w) {
    const uint64_t x = uint64_t(w) * s.all / s.used;
    return uint64_t(uniform(uint32_t(x))) | uint64_t(uniform(uint32_t(x >> 32))) << 32;
}
__device__ __forceinline__ void hold_seen(const Queries& a, ShareScan& sh) {
    if (a.n > kSeenHeld) return;
    for (uint32_t i = threadIdx.x; i < a.n; i += kShareT) {
        const Seen x = seen_by(a, i);
        sh.seq[i] = x.seq;
        sh.rows[i] = x.rows;
    }
    __syncthreads();
}
__device__ __forceinline__ Seen seen_held(const Queries& a, const ShareScan& sh, uint32_t i) {
    if (a.n > kSeenHeld) return seen_by(a, i);
    return {sh.seq[i], sh.rows[i]};
}
// The sums; mine: before this thread's queries (t * each ...), own: of them.  W: workgroups; with more than one a CU
// each gets `few` units at least.
template <class F>
__device__ __forceinline__ Shares scan_units(uint32_t n, uint32_t mult, uint32_t W, uint32_t few, F units, ShareScan& sh, uint32_t& mine,
                                             uint32_t& own) {
    const uint32_t tid = threadIdx.x, each = (n + kShareT - 1) / kShareT, i0 = tid * each, i1 = min(i0 + each, n);
    own = 0;
    for (uint32_t i = i0; i < i1; ++i) own += units(i);
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t all;
    mine = wave_before_sat(own, all);
    if (lane == 0) sh.part[wave] = all;
    __syncthreads();
    Shares s{};
    for (int w = 0; w < kShareWaves; ++w) {
        if (w == wave) mine += s.units;
        s.units += sh.part[w];
    }
    s.units = uint32_t(__builtin_amdgcn_readfirstlane(int(s.units)));  // one for the workgroup
    s.all = uint64_t(s.units) * mult;
    constexpr uint32_t kCUs = 256;
    s.used = uint32_t(min(min(uint64_t(W), s.all), max(uint64_t(kCUs), s.all / few)));
    return s;
}
// The query that has unit x (< all) of all kv heads, and the units of one kv head before it.
struct Found {
    uint32_t query, before;
};
template <class F>
__device__ __forceinline__ Found find_query(uint32_t n, uint32_t mult, F units, ShareScan& sh, uint64_t x, uint32_t mine,
                                            uint32_t own) {
    if (x >= uint64_t(mine) * mult && x < uint64_t(mine + own) * mult) {
        uint32_t i = threadIdx.x * ((n + kShareT - 1) / kShareT), before = mine;
        for (;;) {  // ends: the unit is one of this thread's queries
            const uint32_t u = units(i);
            if (x < uint64_t(before + u) * mult) break;
            before += u;
            ++i;
        }
        sh.query = i;
        sh.before = before;
    }
    __syncthreads();
    return {uint32_t(__builtin_amdgcn_readfirstlane(int(sh.query))), uint32_t(__builtin_amdgcn_readfirstlane(int(sh.before)))};
}
// A read of bytes that no other workgroup reads: they need not stay in a cache.
template <class V>
__device__ __forceinline__ V load_once(const void* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
}
#endif

}  // namespace zq
