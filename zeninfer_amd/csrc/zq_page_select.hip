// zq_page_select.hip -- which pages of the paged KV cache of include/zq_paged.h a
// query attends to.
//
//   score(page) = max_h 2^(eq_h + e) sum_d max(c_hd lo_d, c_hd hi_d)
//
// with c the query's 8-bit codes and lo, hi, e the page's bounds.  max(c lo, c hi) is c hi
// where c > 0 and c lo where c < 0, so the sum is one product of [lo | hi] with
// [min(c, 0) | max(c, 0)], 2 D long: int8 MFMA, pages by heads.  |sum| <= 127 * 127 * D <
// 2^23, the exponents lie in -100 .. 100: the score is exact in fp32, whatever the order.
#include "zq_entry.hpp"
#include "zq_internal.hpp"
#include "zq_paged.hpp"

#include <math.h>

namespace zq {
namespace {

typedef int32_t v4i_t __attribute__((ext_vector_type(4)));

struct SelectArgs {
    const int8_t* bounds;
    const int8_t* bounds_exp;
    const int32_t* table;
    const float* q;
    int32_t* select;
    float* score;  // [queries][KH][pitch]
    Queries see;
    size_t stride;
    uint32_t width, pitch, pages, KH, G, lp, keep, recent, first;  // pitch: width in whole groups of 4
};
__device__ __forceinline__ uint32_t pages_seen(const SelectArgs& a, const Seen& x) {
    return (x.rows + (1u << a.lp) - 1) >> a.lp;
}

// ---- scores ----------------------------------------------------------------------
// A wave takes B tiles of 16 pages at once, all their bounds under way together; a
// workgroup's four waves are a unit of 64 B pages of one (query, kv head), shared out
// evenly.  v_mfma_i32_16x16x64_i8: lane (i, g) loads bytes 64 k + 16 g of page i's
// bounds; it then holds the sums of head i and pages 4 g .. 4 g + 3.  The bounds are
// asked for before the query's codes are made, of which each wave makes a quarter.
// Bound by HBM latency: a kv head's bounds are 2 D bytes a page, in a place of their own, and
// a workgroup has a few units.  4 sequences of 8192 pages, 8 kv heads of 128, 67 MB: 16 us,
// 4.1 TB/s; 32 of up to 938 pages, 32 MB: 11.6 us.
template <int D>
struct ScoreShape {
    static constexpr int B = D == 256 ? 2 : 4;
    static constexpr uint32_t kUnit = 64 * B;
    static constexpr int KC = 2 * D / 64;
};
template <int D>
__global__ __launch_bounds__(kShareT, 3) void page_score_kernel(SelectArgs a) {
    using S = ScoreShape<D>;
    __shared__ ShareScan scan;
    __shared__ v4i_t held_q[S::KC][64];  // [min(c, 0) | max(c, 0)] as operands
    __shared__ float largest[kShareWaves][16];
    hold_seen(a.see, scan);
    const auto units = [&](uint32_t i) {
        const Seen x = seen_held(a.see, scan, i);
        const uint32_t n = x.seq < 0 ? 0u : pages_seen(a, x);
        return n > a.keep ? (n + S::kUnit - 1) / S::kUnit : 0u;
    };
    uint32_t mine, own;
    const Shares sh = scan_units(a.see.n, a.KH, gridDim.x, 1, units, scan, mine, own);
    if (blockIdx.x >= sh.used) return;
    uint64_t pos = share_start(sh, blockIdx.x);
    const uint64_t end = share_start(sh, blockIdx.x + 1);
    const Found at = find_query(a.see.n, a.KH, units, scan, pos, mine, own);
    uint32_t qi = at.query, before = at.before;
    const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    while (pos < end) {
        const uint32_t u = uniform(units(qi));
        if (pos >= uint64_t(before + u) * a.KH) {
            before += u;
            ++qi;
            continue;
        }
        const uint32_t rel = uint32_t(pos - uint64_t(before) * a.KH), kh = rel / u, u0 = rel % u;
        const uint32_t u1 = uint32_t(min(uint64_t(u), u0 + (end - pos)));
        Seen x = seen_held(a.see, scan, qi);
        x.seq = int32_t(uniform(uint32_t(x.seq)));
        const uint32_t n = uniform(pages_seen(a, x));
        const int32_t* table = a.table + size_t(x.seq) * a.width;
        float* score = a.score + (size_t(qi) * a.KH + kh) * a.pitch;
        v4i_t b[S::B][S::KC];
        float scale;
        // pages of unit t: lane l < 16 B has the l-th (past the last one: the last one's place is read)
        auto load_page = [&](uint32_t t) {
            const uint32_t j = (t * kShareWaves + wave) * 16 * S::B + uint32_t(lane % (16 * S::B));
            return uint32_t(table[min(j, n - 1)]);
        };
        auto load_bounds = [&](uint32_t page) {
            const bool good = page < a.pages;
            if (!good) page = 0;
            const int e = a.bounds_exp[size_t(page) * a.KH + kh];
#pragma unroll
            for (int w = 0; w < S::B; ++w) {
                const uint32_t pg = uint32_t(__shfl(int(page), w * 16 + i));
                const int8_t* from = a.bounds + (size_t(pg) * a.KH + kh) * 2 * D + g * 16;
#pragma unroll
                for (int k = 0; k < S::KC; ++k) b[w][k] = *reinterpret_cast<const v4i_t*>(from + k * 64);
            }
            scale = good ? pow2f(e) : -1.0f;
        };
        for (uint32_t h0 = 0; h0 < a.G; h0 += 16) {  // 16 heads at once
            const uint32_t first_page = load_page(u0);
            // codes of head h0 + i, elements 64 k + 16 g ..: this wave's are dword `wave` of every 16 bytes
            const uint32_t R = min(a.G - h0, 16u);
            const float* q = a.q + qi * a.stride + (size_t(kh) * a.G + h0 + min(uint32_t(i), R - 1)) * D + g * 16 + wave * 4;
            float4 y[D / 64];
            float most = 0.0f;
#pragma unroll
            for (int k = 0; k < D / 64; ++k) y[k] = *reinterpret_cast<const float4*>(q + k * 64);
            load_bounds(first_page);
#pragma unroll
            for (int k = 0; k < D / 64; ++k)
                most = fmaxf(most, fmaxf(fmaxf(fabsf(y[k].x), fabsf(y[k].y)), fmaxf(fabsf(y[k].z), fabsf(y[k].w))));
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            if (g == 0) largest[wave][i] = most;
            __syncthreads();  // (and the operands before these have been read)
            most = fmaxf(fmaxf(largest[0][i], largest[1][i]), fmaxf(largest[2][i], largest[3][i]));
            const int eq = bound_exp(most);
            const float unit = pow2f(-eq), up = pow2f(eq);
#pragma unroll
            for (int k = 0; k < D / 64; ++k) {
                const float e[4] = {y[k].x, y[k].y, y[k].z, y[k].w};
                uint32_t neg = 0, plus = 0;
#pragma unroll
                for (int c4 = 0; c4 < 4; ++c4) {
                    const float f = rintf(e[c4] * unit);
                    const int c = f != f ? 0 : bound_code(f);
                    neg |= (uint32_t(min(c, 0)) & 255u) << (8 * c4);
                    plus |= uint32_t(max(c, 0)) << (8 * c4);
                }
                reinterpret_cast<uint32_t*>(&held_q[k][lane])[wave] = neg;
                reinterpret_cast<uint32_t*>(&held_q[D / 64 + k][lane])[wave] = plus;
            }
            __syncthreads();
            for (uint32_t t = u0; t < u1; ++t) {
                if (t != u0) load_bounds(load_page(t));
                float mine_s = 0.0f;
                v4i_t s[S::B];
#pragma unroll
                for (int w = 0; w < S::B; ++w) s[w] = v4i_t{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < S::KC; ++k) {
                    const v4i_t op = held_q[k][lane];
#pragma unroll
                    for (int w = 0; w < S::B; ++w) s[w] = __builtin_amdgcn_mfma_i32_16x16x64_i8(b[w][k], op, s[w], 0, 0, 0);
                }
#pragma unroll
                for (int w = 0; w < S::B; ++w)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float f = uint32_t(i) < R ? float(s[w][r]) * up : -INFINITY;
                        f = fmaxf(f, dpp_f<kDppXor1>(f));
                        f = fmaxf(f, dpp_f<kDppXor2>(f));
                        f = fmaxf(f, dpp_f<kDppHalfMirror>(f));
                        f = fmaxf(f, dpp_f<kDppMirror>(f));
                        // of page w * 16 + 4 g + r, which is lane w * 16 + 4 g + r's
                        const float of = __shfl(f, ((lane >> 2) & 3) * 16);
                        if ((lane >> 4) == w && (lane & 3) == r) mine_s = of;
                    }
                const uint32_t j = (t * kShareWaves + wave) * 16 * S::B + uint32_t(lane);
                if (j < n && lane < 16 * S::B) {
                    float f = scale > 0.0f ? mine_s * scale : -INFINITY;
                    if (h0) f = fmaxf(f, score[j]);
                    score[j] = f;
                }
            }
        }
        pos += u1 - u0;
    }
}

// ---- the largest ---------------------------------------------------------------------
// A workgroup for every (query, kv head).  Thread t holds pages t N .. t N + N - 1 (of
// every N * 1024), as whole numbers in the order of the scores, from the least one on.
// The score of rank `want` is found by digits of 11 bits from the highest bit there is,
// counted in LDS, until all that share its digits stay; one scan of (pages above it,
// pages at it) then gives every page that stays its place: what stays, and where, does not
// depend on the order of the counts.  Bound by a digit's chain (LDS atomics, a scan over the
// bins, four barriers): 8192 pages 9.8 us, 938 5.9.
constexpr int kTopT = 1024, kTopWaves = kTopT / 64, kBins = 2048;

__device__ __forceinline__ uint32_t score_key(float f) {
    const uint32_t u = __float_as_uint(f + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

template <int N>
__device__ __forceinline__ void top_pages(const SelectArgs& a, const float* score, int32_t* to, uint32_t n,
                                          uint32_t (&hist)[2][kBins], uint32_t (&pick)[3], uint32_t (&part)[2][kTopWaves]) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lo = a.first, hi = n - a.recent;  // the others stay; n > keep >= first + recent
    const bool held = n <= uint32_t(N * kTopT);
    uint32_t key[N], least = 0;
    auto load = [&](uint32_t i0) {
        const uint32_t p = i0 + uint32_t(tid * N);
        if constexpr (N % 4 == 0) {  // (within the pitch; what lies behind the scores is not looked at)
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                const float4 x = *reinterpret_cast<const float4*>(score + min(p + j, a.pitch - 4));
                key[j] = score_key(x.x) - least, key[j + 1] = score_key(x.y) - least;
                key[j + 2] = score_key(x.z) - least, key[j + 3] = score_key(x.w) - least;
            }
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) key[j] = score_key(score[min(p + j, n - 1)]) - least;
        }
    };
    auto each = [&](auto f) {  // f(key) of every candidate
        for (uint32_t i0 = 0; i0 < n; i0 += N * kTopT) {
            if (!held) load(i0);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t p = i0 + uint32_t(tid * N + j);
                if (p >= lo && p < hi) f(key[j]);
            }
        }
    };
    if (held) load(0);
    // of the candidates, those from `top` on stay, and the first `want` of those from `at` on below it
    uint32_t want = a.keep - a.first - a.recent, at = 0xffffffffu, top = 0xffffffffu;
    if (want) {
        uint32_t low = 0xffffffffu, most = 0;
        each([&](uint32_t k) {
            low = min(low, k);
            most = max(most, k);
        });
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            low = min(low, uint32_t(__shfl_xor(int(low), m)));
            most = max(most, uint32_t(__shfl_xor(int(most), m)));
        }
        if (lane == 0) part[0][wave] = low, part[1][wave] = most;
        hist[0][tid] = hist[0][tid + kTopT] = 0;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kTopWaves; ++w) low = min(low, part[0][w]), most = max(most, part[1][w]);
        least = low;
        if (held)
#pragma unroll
            for (int j = 0; j < N; ++j) key[j] -= least;
        int bits = 32 - __clz(int(most - low));  // of the largest key (0: all are equal)
        uint32_t prefix = 0;
        bool all_stay = false;
        for (int d = 0; bits > 0 && !all_stay; ++d) {
            const int shift = max(bits - 11, 0);
            uint32_t* bins = hist[d & 1];
            const uint64_t up = uint64_t(prefix) >> bits;
            const uint32_t mask = (1u << (bits - shift)) - 1;
            each([&](uint32_t k) {
                if (uint64_t(k) >> bits == up) atomicAdd(&bins[(k >> shift) & mask], 1u);
            });
            __syncthreads();
            const uint32_t h0 = bins[kBins - 1 - 2 * tid], h1 = bins[kBins - 2 - 2 * tid];
            hist[(d + 1) & 1][tid] = hist[(d + 1) & 1][tid + kTopT] = 0;
            uint32_t all;
            uint32_t before = wave_before_sat(h0 + h1, all);
            if (lane == 0) part[0][wave] = all;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < kTopWaves; ++w) before += w < wave ? part[0][w] : 0u;
            if (before < want && want <= before + h0) {
                pick[0] = uint32_t(kBins - 1 - 2 * tid);
                pick[1] = want - before;
                pick[2] = h0;
            } else if (before + h0 < want && want <= before + h0 + h1) {
                pick[0] = uint32_t(kBins - 2 - 2 * tid);
                pick[1] = want - before - h0;
                pick[2] = h1;
            }
            __syncthreads();
            prefix |= pick[0] << shift;
            want = pick[1];
            all_stay = pick[2] == want;
            bits = shift;
        }
        at = prefix;
        top = all_stay ? prefix : prefix + 1;  // (a key is below 2^32 - 1: the largest score's is)
    }
    // pages that stay, in order: those held anyway, those above, and the first `want` at it
    uint32_t done = 0, equal = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += N * kTopT) {
        if (!held) load(i0);
        uint32_t sure = 0, some = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t p = i0 + uint32_t(tid * N + j);
            if (p < n) {
                const bool must = p < lo || p >= hi;
                sure += must || key[j] >= top;
                some += !must && key[j] >= at && key[j] < top;
            }
        }
        uint32_t all_s, all_e;
        uint32_t bs = wave_before_sat(sure, all_s), be = wave_before_sat(some, all_e);
        __syncthreads();
        if (lane == 0) part[0][wave] = all_s, part[1][wave] = all_e;
        __syncthreads();
        uint32_t ts = 0, te = 0;
#pragma unroll
        for (int w = 0; w < kTopWaves; ++w) {
            if (w == wave) bs += ts, be += te;
            ts += part[0][w];
            te += part[1][w];
        }
        bs += done;
        be += equal;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t p = i0 + uint32_t(tid * N + j);
            if (p < n) {
                const bool must = p < lo || p >= hi, yes = must || key[j] >= top, eq = !yes && key[j] >= at;
                if (yes || (eq && be < want)) to[bs + min(be, want)] = int32_t(p);
                bs += yes;
                be += eq;
            }
        }
        done += ts;
        equal += te;
    }
}

__global__ __launch_bounds__(kTopT) void page_top_kernel(SelectArgs a) {
    const uint32_t qi = blockIdx.y, pair = qi * a.KH + blockIdx.x;
    const Seen x = seen_by(a.see, qi);
    if (x.seq < 0) return;
    const uint32_t n = pages_seen(a, x);
    int32_t* to = a.select + size_t(pair) * a.keep;
    if (n <= a.keep) {
        for (uint32_t j = threadIdx.x; j < a.keep; j += kTopT) to[j] = j < n ? int32_t(j) : -1;
        return;
    }
    const float* score = a.score + size_t(pair) * a.pitch;
    __shared__ uint32_t hist[2][kBins];
    __shared__ uint32_t pick[3];
    __shared__ uint32_t part[2][kTopWaves];
    if (n <= kTopT) top_pages<1>(a, score, to, n, hist, pick, part);
    else if (n <= 4 * kTopT) top_pages<4>(a, score, to, n, hist, pick, part);
    else top_pages<8>(a, score, to, n, hist, pick, part);
}

uint32_t score_shares(const zq_kv_paged& c, const zq_page_tables& t, size_t queries) {
    const size_t unit = c.head_dim == 256 ? 128 : 256;
    const size_t most = queries * c.kv_heads * ((t.width + unit - 1) / unit);
    return uint32_t(most < 768 ? most : 768);
}

uint32_t pitch_of(const zq_page_tables& t) { return uint32_t(t.width + 3) / 4 * 4; }
size_t select_bytes(const zq_kv_paged& c, const zq_page_tables& t, size_t queries) {
    return (queries * c.kv_heads * pitch_of(t) * 4 + 255) / 256 * 256;
}

template <int D>
void run_scores(const SelectArgs& a, uint32_t W, hipStream_t stream) {
    hipLaunchKernelGGL(page_score_kernel<D>, dim3(W), dim3(kShareT), 0, stream, a);
}

}  // namespace
}  // namespace zq

extern "C" {

size_t zq_hip_page_select_workspace_bytes(const zq_kv_paged* cache, const zq_page_tables* tables, size_t queries,
                                          size_t heads, size_t keep) {
    if (!zq::kv_paged_ok(cache) || !zq::page_tables_ok(tables) || !keep ||
        !zq::queries_ok(*cache, *tables, queries, heads, tables->table))
        return 0;
    return zq::select_bytes(*cache, *tables, queries);
}

int zq_hip_page_select_dev(const zq_kv_paged* cache, const zq_page_tables* tables, const float* q, int32_t* select,
                           size_t queries, size_t heads, size_t stride, const int32_t* seq_of, const int32_t* lens,
                           const int32_t* counts, size_t keep, size_t recent, size_t first, int flags, void* workspace,
                           size_t workspace_bytes, void* stream) {
    using zq::a16;
    using zq::a4;
    if (!zq::kv_paged_ok(cache) || !cache->bounds || !zq::page_tables_ok(tables) ||
        !zq::queries_ok(*cache, *tables, queries, heads, seq_of) || !q || !select || !lens || !a16(q) || !a4(select) ||
        !a4(lens) || !a4(counts) || !a4(seq_of) || (flags & ~ZQ_ATTN_PAGED_FULL) || !keep || keep > zq::kPgMaxTokens / 16 ||
        recent > keep || first > keep - recent)
        return ZQ_ERR_ARG;
    const size_t width = heads * cache->head_dim;
    if (!stride) stride = width;
    if (stride < width || stride % 4 || stride > zq::kPgMaxStride) return ZQ_ERR_ARG;
    if (!workspace || !a16(workspace) || workspace_bytes < zq::select_bytes(*cache, *tables, queries)) return ZQ_ERR_ARG;
    const zq::OnDeviceOf dev(cache->k);
    if (dev.status() != ZQ_OK) return dev.status();
    zq::SelectArgs a{};
    a.bounds = cache->bounds;
    a.bounds_exp = cache->bounds_exp;
    a.table = tables->table;
    a.q = q;
    a.select = select;
    a.score = static_cast<float*>(workspace);
    a.see = {seq_of, lens, counts, uint32_t(queries), uint32_t(tables->seqs), uint32_t(tables->width * tables->page_size),
             flags & ZQ_ATTN_PAGED_FULL};
    a.stride = stride;
    a.width = uint32_t(tables->width);
    a.pitch = zq::pitch_of(*tables);
    a.pages = uint32_t(tables->pages);
    a.KH = uint32_t(cache->kv_heads);
    a.G = uint32_t(heads / cache->kv_heads);
    a.lp = zq::log2_of(tables->page_size);
    a.keep = uint32_t(keep);
    a.recent = uint32_t(recent);
    a.first = uint32_t(first);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (tables->width > keep) {
        const uint32_t W = zq::score_shares(*cache, *tables, queries);
        if (cache->head_dim == 64) zq::run_scores<64>(a, W, st);
        else if (cache->head_dim == 128) zq::run_scores<128>(a, W, st);
        else zq::run_scores<256>(a, W, st);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return zq::status(e);
    }
    // (in two dimensions: 2^23 workgroups of 1024 are more than one dimension takes)
    hipLaunchKernelGGL(zq::page_top_kernel, dim3(a.KH, uint32_t(queries)), dim3(zq::kTopT), 0, st, a);
    return zq::status(hipGetLastError());
}

}  // extern "C"
