// zq_paged.hip -- the paged KV cache of include/zq_paged.h: page tables, append
// with the pages' bounds, and their C entry points (attention is in
// zq_attn_paged.hip, selection in zq_page_select.hip).
#include "zq_entry.hpp"
#include "zq_paged.hpp"

#include <math.h>

namespace zq {
namespace {

// ---- page tables -----------------------------------------------------------------
// A step in numbers: sequence s fits with c_s new tokens, lacks need_s pages; P, C the
// sums of need and c up to and with s.  It is served where P and C are within the free
// pages and the rows; both only grow, so those served come first, and their sums are
// the last served one's.  A workgroup takes all the sums by itself (8 sequences a
// thread at most) into LDS; then every packed row finds its sequence by bisection and
// its page without any other row: the page of a new one is as far below the top of the
// stack as P says.  With few rows one workgroup does it all; with many, each of a grid
// repeats the sums, and a second launch writes what the first one still reads (the
// counts may be the granted ones' array, the free pages' number its own successor).
constexpr int kTabT = 1024, kTabWaves = kTabT / 64;
constexpr uint32_t kExpand = 1, kCommit = 2;

struct StepArgs {
    int32_t* table;
    const int32_t* free_pages;
    const int32_t* lens;
    const int32_t* counts;
    const int32_t* free_count;
    int32_t* free_left;
    int32_t* granted;
    int32_t* start;
    int64_t* slots;
    int32_t* positions;
    int32_t* seq_of;
    uint32_t seqs, width, pages, lp, tokens;
};

// Sums before a thread's own value over the workgroup (v: two values), and their totals.
struct Sums2 {
    uint32_t a, b;
};
__device__ __forceinline__ Sums2 block_before2(Sums2 v, uint32_t (&part)[2][kTabWaves], Sums2& all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t wa, wb;
    Sums2 x{wave_before_sat(v.a, wa), wave_before_sat(v.b, wb)};
    if (lane == 0) {
        part[0][wave] = wa;
        part[1][wave] = wb;
    }
    __syncthreads();
    all = {0, 0};
    for (int w = 0; w < kTabWaves; ++w) {
        if (w == wave) {
            x.a = add_sat31(x.a, all.a);
            x.b = add_sat31(x.b, all.b);
        }
        all.a = add_sat31(all.a, part[0][w]);
        all.b = add_sat31(all.b, part[1][w]);
    }
    __syncthreads();
    return x;
}
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t lp) { return (tokens + (1u << lp) - 1) >> lp; }

__global__ __launch_bounds__(kTabT) void page_step_kernel(StepArgs a, uint32_t role) {
    __shared__ uint32_t end[kPgMaxSeqs];   // granted tokens up to and with a sequence
    __shared__ uint32_t taken[kPgMaxSeqs]; // pages taken before it
    __shared__ uint32_t part[2][kTabWaves];
    __shared__ uint32_t total[2];
    const uint32_t tid = threadIdx.x, each = (a.seqs + kTabT - 1) / kTabT, s0 = tid * each, s1 = min(s0 + each, a.seqs);
    const uint32_t cap = a.width << a.lp, fc = uint32_t(min(max(a.free_count[0], 0), int32_t(a.pages)));
    auto len_of = [&](uint32_t s) { return uint32_t(min(max(a.lens[s], 0), int32_t(cap))); };
    struct Want {
        uint32_t tokens, pages;
        bool fits;
    };
    auto want = [&](uint32_t s) {
        const uint32_t n = len_of(s), c = uint32_t(max(a.counts[s], 0));
        if (c > cap - n) return Want{0, 0, false};
        return Want{c, pages_of(n + c, a.lp) - pages_of(n, a.lp), true};
    };
    Sums2 own{0, 0}, all;
    for (uint32_t s = s0; s < s1; ++s) {
        const Want w = want(s);
        own.a = add_sat31(own.a, w.tokens);
        own.b = add_sat31(own.b, w.pages);
    }
    if (tid < 2) total[tid] = 0;
    Sums2 at = block_before2(own, part, all);
    uint32_t tok = 0, pg = 0;  // the sums of the last one served
    for (uint32_t s = s0; s < s1; ++s) {
        const Want w = want(s);
        taken[s] = at.b;
        at.a = add_sat31(at.a, w.tokens);
        at.b = add_sat31(at.b, w.pages);
        end[s] = at.a;
        if (w.fits && at.a <= a.tokens && at.b <= fc) tok = at.a, pg = at.b;
    }
    if (tok) atomicMax(&total[0], tok);
    if (pg) atomicMax(&total[1], pg);
    __syncthreads();
    const uint32_t served = total[0], taken_all = total[1];
    if (role & kExpand) {
        for (uint32_t r = blockIdx.x * kTabT + tid; r < a.tokens; r += gridDim.x * kTabT) {
            int64_t slot = -1;
            int32_t pos = -1, seq = -1;
            if (r < served) {
                uint32_t lo = 0, hi = a.seqs - 1;  // the first sequence whose end is past r
                while (lo < hi) {
                    const uint32_t mid = (lo + hi) >> 1;
                    if (end[mid] > r) hi = mid;
                    else lo = mid + 1;
                }
                const uint32_t n = len_of(lo), p = n + r - (lo ? end[lo - 1] : 0u), j = p >> a.lp, old = pages_of(n, a.lp);
                const uint32_t page = uint32_t(j < old ? a.table[size_t(lo) * a.width + j]
                                                       : a.free_pages[fc - 1 - (taken[lo] + j - old)]);
                const uint32_t row = p & ((1u << a.lp) - 1);
                if (row == 0) a.table[size_t(lo) * a.width + j] = int32_t(page);  // a new page's first token is a new one
                if (page < a.pages) slot = (int64_t(page) << a.lp) + row;
                pos = int32_t(p);
                seq = int32_t(lo);
            }
            a.slots[r] = slot;
            if (a.positions) a.positions[r] = pos;
            if (a.seq_of) a.seq_of[r] = seq;
        }
    }
    if (role & kCommit) {
        for (uint32_t s = tid; s < a.seqs; s += kTabT) {
            const uint32_t e = min(end[s], served), b = s ? min(end[s - 1], served) : 0u;
            a.start[s] = int32_t(b);
            a.granted[s] = int32_t(e - b);
        }
        if (tid == 0) {
            a.start[a.seqs] = int32_t(served);
            a.free_left[0] = int32_t(fc - taken_all);
        }
    }
}

// The pages that the sequences do not need, by the same sums: page x of all that go
// back, in order of sequence and place, is x below the new top.
struct ReleaseArgs {
    const int32_t* table;
    int32_t* free_pages;
    const int32_t* lens;
    const int32_t* keep;
    const int32_t* free_count;
    int32_t* free_left;
    uint32_t seqs, width, pages, lp;
};
__global__ __launch_bounds__(kTabT) void page_release_kernel(ReleaseArgs a, uint32_t role) {
    __shared__ uint32_t end[kPgMaxSeqs];
    __shared__ uint32_t part[2][kTabWaves];
    const uint32_t tid = threadIdx.x, each = (a.seqs + kTabT - 1) / kTabT, s0 = tid * each, s1 = min(s0 + each, a.seqs);
    const uint32_t cap = a.width << a.lp, fc = uint32_t(min(max(a.free_count[0], 0), int32_t(a.pages)));
    struct Span {
        uint32_t from, to;
    };
    auto span = [&](uint32_t s) {
        const uint32_t n = uint32_t(min(max(a.lens[s], 0), int32_t(cap)));
        const uint32_t k = min(uint32_t(max(a.keep[s], 0)), n);
        return Span{pages_of(k, a.lp), pages_of(n, a.lp)};
    };
    Sums2 own{0, 0}, all;
    for (uint32_t s = s0; s < s1; ++s) {
        const Span x = span(s);
        own.a = add_sat31(own.a, x.to - x.from);
    }
    Sums2 at = block_before2(own, part, all);
    for (uint32_t s = s0; s < s1; ++s) {
        const Span x = span(s);
        end[s] = at.a = add_sat31(at.a, x.to - x.from);
    }
    __syncthreads();
    const uint32_t n = all.a;
    if (role & kExpand) {
        for (uint32_t x = blockIdx.x * kTabT + tid; x < n; x += gridDim.x * kTabT) {
            uint32_t lo = 0, hi = a.seqs - 1;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) >> 1;
                if (end[mid] > x) hi = mid;
                else lo = mid + 1;
            }
            const uint32_t j = span(lo).from + x - (lo ? end[lo - 1] : 0u), to = fc + (n - 1 - x);
            if (to < a.pages) a.free_pages[to] = a.table[size_t(lo) * a.width + j];
        }
    }
    if ((role & kCommit) && tid == 0) a.free_left[0] = int32_t(min(fc + n, a.pages));
}

// Rows up to which one workgroup does it all.
constexpr size_t kOneTable = 4096;

// ---- append ----------------------------------------------------------------------
template <int TYPE>
struct Held {
    typedef float type;
};
template <>
struct Held<ZQ_KV_F16> {
    typedef _Float16 type;
};
template <>
struct Held<ZQ_KV_BF16> {
    typedef __bf16 type;
};

struct AppendArgs {
    uint8_t* k;
    uint8_t* v;
    int8_t* bounds;
    int8_t* bounds_exp;
    const float* src_k;
    const float* src_v;
    const int64_t* slots;
    size_t stride;
    int64_t all_slots;
    uint32_t rows, KH, lp;
};

// A lane takes 16 bytes of a held row, so a row (one token of one kv head) is
// head_dim * size / 16 lanes.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
    typedef typename Held<TYPE>::type T;
    constexpr int E = 16 / sizeof(T), L = D / E;
    const uint32_t row = blockIdx.x * (256 / L) + threadIdx.x / L, l = threadIdx.x % L;
    if (row >= a.rows) return;
    const uint32_t t = row / a.KH, h = row % a.KH;
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.all_slots) return;
    const size_t from = t * a.stride + h * D + l * E;
    typedef T vec __attribute__((ext_vector_type(E)));
    vec k, v;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(a.src_k + from + i);
        const float4 y = *reinterpret_cast<const float4*>(a.src_v + from + i);
        k[i] = T(x.x), k[i + 1] = T(x.y), k[i + 2] = T(x.z), k[i + 3] = T(x.w);
        v[i] = T(y.x), v[i + 1] = T(y.y), v[i + 2] = T(y.z), v[i + 3] = T(y.w);
    }
    const size_t ps = size_t(1) << a.lp;
    const size_t to = (((size_t(slot) >> a.lp) * a.KH + h) * ps + (size_t(slot) & (ps - 1))) * D + l * E;
    *reinterpret_cast<vec*>(a.k + to * sizeof(T)) = k;
    *reinterpret_cast<vec*>(a.v + to * sizeof(T)) = v;
}

// Bounds of the pages that got rows: a wave for every (token, kv head), which goes on
// where the token is the last of its page in this call.
template <int TYPE, int D>
__global__ __launch_bounds__(256) void paged_bounds_kernel(AppendArgs a) {
    typedef typename Held<TYPE>::type T;
    constexpr int E = 16 / sizeof(T), L = D / E, R = 64 / L;  // elements a lane, lanes a row, rows at once
    const uint32_t row = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / 64);
    const int lane = threadIdx.x & 63, l = lane % L;
    if (row >= a.rows) return;
    const uint32_t t = row / a.KH, h = row % a.KH;
    const int64_t slot = a.slots[t], ps = int64_t(1) << a.lp;
    if (slot < 0 || slot >= a.all_slots) return;
    const int last = int(slot & (ps - 1));
    if ((row / a.KH + 1) * a.KH < a.rows && last + 1 < ps && a.slots[t + 1] == slot + 1) return;
    const size_t head = size_t(slot >> a.lp) * a.KH + h;
    const T* p = reinterpret_cast<const T*>(a.k) + (head << a.lp) * D + l * E;
    float lo[E], hi[E];
#pragma unroll
    for (int i = 0; i < E; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
    typedef T vec __attribute__((ext_vector_type(E)));
    for (int r = lane / L; r <= last; r += R) {
        const vec x = *reinterpret_cast<const vec*>(p + size_t(r) * D);
#pragma unroll
        for (int i = 0; i < E; ++i) {
            lo[i] = fminf(lo[i], float(x[i]));
            hi[i] = fmaxf(hi[i], float(x[i]));
        }
    }
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
#pragma unroll
        for (int m = L; m < 64; m *= 2) {
            lo[i] = fminf(lo[i], __shfl_xor(lo[i], m));
            hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], m));
        }
        if (lo[i] > hi[i]) lo[i] = hi[i] = 0.0f;  // NaN only
        most = fmaxf(most, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
    }
#pragma unroll
    for (int m = 1; m < L; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
    const int e = bound_exp(most);
    uint32_t w[2][(E + 3) / 4] = {};
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int c0 = bound_code(floorf(ldexpf(lo[i], -e))), c1 = bound_code(ceilf(ldexpf(hi[i], -e)));
        w[0][i / 4] |= uint32_t(c0 & 255) << (8 * (i % 4));
        w[1][i / 4] |= uint32_t(c1 & 255) << (8 * (i % 4));
    }
    if (lane < L) {
        int8_t* b = a.bounds + head * 2 * D + l * E;
#pragma unroll
        for (int i = 0; i < E / 4; ++i) {
            reinterpret_cast<uint32_t*>(b)[i] = w[0][i];
            reinterpret_cast<uint32_t*>(b + D)[i] = w[1][i];
        }
        if (lane == 0) a.bounds_exp[head] = int8_t(e);
    }
}

template <int TYPE, int D>
void run_append(const AppendArgs& a, hipStream_t stream) {
    constexpr uint32_t per = 256 / (D * sizeof(typename Held<TYPE>::type) / 16);
    hipLaunchKernelGGL((paged_append_kernel<TYPE, D>), dim3((a.rows + per - 1) / per), dim3(256), 0, stream, a);
    if (a.bounds)
        hipLaunchKernelGGL((paged_bounds_kernel<TYPE, D>), dim3((a.rows + 3) / 4), dim3(256), 0, stream, a);
}
template <int TYPE>
void run_append(const AppendArgs& a, size_t D, hipStream_t stream) {
    if (D == 64) run_append<TYPE, 64>(a, stream);
    else if (D == 128) run_append<TYPE, 128>(a, stream);
    else run_append<TYPE, 256>(a, stream);
}

bool page_size_ok(size_t n) { return n >= 16 && n <= 256 && (n & (n - 1)) == 0; }

}  // namespace

bool page_tables_ok(const zq_page_tables* t) {
    return t && t->table && a4(t->table) && a4(t->free_pages) && t->seqs && t->seqs <= kPgMaxSeqs && t->pages &&
           t->pages <= kPgMaxPages && page_size_ok(t->page_size) && t->width && t->width <= kPgMaxTokens / t->page_size;
}

bool kv_paged_ok(const zq_kv_paged* c) {
    return c && c->k && c->v && a16(c->k) && a16(c->v) && a16(c->bounds) && !c->bounds == !c->bounds_exp && c->pages &&
           c->pages <= kPgMaxPages && c->kv_heads && c->kv_heads <= kPgMaxHeads &&
           (c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256) && page_size_ok(c->page_size) &&
           (c->type == ZQ_KV_F32 || c->type == ZQ_KV_F16 || c->type == ZQ_KV_BF16);
}

bool queries_ok(const zq_kv_paged& c, const zq_page_tables& t, size_t queries, size_t heads, const int32_t* seq_of) {
    return t.pages <= c.pages && t.page_size == c.page_size && queries && queries <= kPgMaxSeqs && heads &&
           heads <= kPgMaxHeads && heads % c.kv_heads == 0 && (seq_of || queries <= t.seqs);
}

}  // namespace zq

// ---- C entry points --------------------------------------------------------------
using zq::OnDeviceOf;
using zq::a16;
using zq::a4;

extern "C" {

int zq_hip_page_tables_step_dev(const zq_page_tables* tables, const int32_t* lens, const int32_t* counts,
                                const int32_t* free_count, int32_t* free_left, int32_t* granted, int32_t* start,
                                int64_t* slots, int32_t* positions, int32_t* seq_of, size_t tokens, void* stream) {
    if (!zq::page_tables_ok(tables) || !tables->free_pages || !lens || !counts || !free_count || !free_left || !granted ||
        !start || !slots || !a4(lens) || !a4(counts) || !a4(free_count) || !a4(free_left) || !a4(granted) || !a4(start) ||
        (reinterpret_cast<uintptr_t>(slots) & 7u) || !a4(positions) || !a4(seq_of) || !tokens ||
        tokens > zq::kPgMaxTokens)
        return ZQ_ERR_ARG;
    const OnDeviceOf dev(tables->table);
    if (dev.status() != ZQ_OK) return dev.status();
    const zq::StepArgs a{tables->table, tables->free_pages, lens, counts, free_count, free_left, granted, start, slots,
                         positions, seq_of, uint32_t(tables->seqs), uint32_t(tables->width), uint32_t(tables->pages),
                         zq::log2_of(tables->page_size), uint32_t(tokens)};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (tokens <= zq::kOneTable) {
        hipLaunchKernelGGL(zq::page_step_kernel, dim3(1), dim3(zq::kTabT), 0, st, a, zq::kExpand | zq::kCommit);
    } else {
        const size_t blocks = (tokens + zq::kTabT - 1) / zq::kTabT;
        hipLaunchKernelGGL(zq::page_step_kernel, dim3(uint32_t(blocks < 512 ? blocks : 512)), dim3(zq::kTabT), 0, st, a,
                           zq::kExpand);
        hipLaunchKernelGGL(zq::page_step_kernel, dim3(1), dim3(zq::kTabT), 0, st, a, zq::kCommit);
    }
    return zq::status(hipGetLastError());
}

int zq_hip_page_tables_release_dev(const zq_page_tables* tables, const int32_t* lens, const int32_t* keep,
                                   const int32_t* free_count, int32_t* free_left, void* stream) {
    if (!zq::page_tables_ok(tables) || !tables->free_pages || !lens || !keep || !free_count || !free_left || !a4(lens) ||
        !a4(keep) || !a4(free_count) || !a4(free_left))
        return ZQ_ERR_ARG;
    const OnDeviceOf dev(tables->table);
    if (dev.status() != ZQ_OK) return dev.status();
    const zq::ReleaseArgs a{tables->table, tables->free_pages, lens, keep, free_count, free_left, uint32_t(tables->seqs),
                            uint32_t(tables->width), uint32_t(tables->pages), zq::log2_of(tables->page_size)};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const size_t most = tables->seqs * tables->width < tables->pages ? tables->seqs * tables->width : tables->pages;
    if (most <= zq::kOneTable) {
        hipLaunchKernelGGL(zq::page_release_kernel, dim3(1), dim3(zq::kTabT), 0, st, a, zq::kExpand | zq::kCommit);
    } else {
        const size_t blocks = (most + zq::kTabT - 1) / zq::kTabT;
        hipLaunchKernelGGL(zq::page_release_kernel, dim3(uint32_t(blocks < 256 ? blocks : 256)), dim3(zq::kTabT), 0, st, a,
                           zq::kExpand);
        hipLaunchKernelGGL(zq::page_release_kernel, dim3(1), dim3(zq::kTabT), 0, st, a, zq::kCommit);
    }
    return zq::status(hipGetLastError());
}

int zq_hip_kv_paged_append_dev(const zq_kv_paged* cache, const float* k, const float* v, size_t tokens, size_t stride,
                               const int64_t* slots, void* stream) {
    if (!zq::kv_paged_ok(cache) || !k || !v || !slots || !a16(k) || !a16(v) || (reinterpret_cast<uintptr_t>(slots) & 7u) ||
        !tokens || tokens > zq::kPgMaxTokens || tokens * cache->kv_heads > (size_t(1) << 25))
        return ZQ_ERR_ARG;
    const size_t width = cache->kv_heads * cache->head_dim;
    if (!stride) stride = width;
    if (stride < width || stride % 4 || stride > zq::kPgMaxStride) return ZQ_ERR_ARG;
    const OnDeviceOf dev(cache->k);
    if (dev.status() != ZQ_OK) return dev.status();
    const zq::AppendArgs a{static_cast<uint8_t*>(cache->k), static_cast<uint8_t*>(cache->v), cache->bounds,
                           cache->bounds_exp, k, v, slots, stride, int64_t(cache->pages * cache->page_size),
                           uint32_t(tokens * cache->kv_heads), uint32_t(cache->kv_heads), zq::log2_of(cache->page_size)};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (cache->type == ZQ_KV_F32) zq::run_append<ZQ_KV_F32>(a, cache->head_dim, st);
    else if (cache->type == ZQ_KV_F16) zq::run_append<ZQ_KV_F16>(a, cache->head_dim, st);
    else zq::run_append<ZQ_KV_BF16>(a, cache->head_dim, st);
    return zq::status(hipGetLastError());
}

}  // extern "C"
