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
// the last served one's.  A workgroup takes all the sums by itself (N sequences a
// thread) into LDS; then every packed row finds its sequence by bisection and its page
// without any other row: the page of a new one is as far below the top of the stack as
// P says.  Every workgroup of a grid repeats the sums, so that one launch will do; where
// an output is an input too (the granted ones' array the counts', the number of free
// pages its own successor) and one workgroup is too few, a second launch writes them.
// Bound by dependent round trips, not by bytes: lens, counts and the number of free pages; an
// old page's entry or a new page's; the stores; and two barriers.  With a sequence a thread
// (N = 1) the entries and the stack's top are asked for before the sums.  256 decoding
// sequences: 6.2 us; 600 with 198,280 new tokens, 3.3 MB (0.6 us of a copy): 9.2.
constexpr uint32_t kExpand = 1, kCommit = 2;
constexpr size_t kOneTable = 4096;  // rows up to which one workgroup does it all then

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

// Sums before a thread's own values over a workgroup of W waves, and their totals.
struct Sums2 {
    uint32_t a, b;
};
template <int W>
__device__ __forceinline__ Sums2 block_before2(Sums2 v, uint32_t (&part)[2][W], Sums2& all) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t wa, wb;
    Sums2 x{wave_before_sat(v.a, wa), wave_before_sat(v.b, wb)};
    if (lane == 0) {
        part[0][wave] = wa;
        part[1][wave] = wb;
    }
    __syncthreads();
    all = {0, 0};
#pragma unroll
    for (int w = 0; w < W; ++w) {
        if (w == wave) {
            x.a = add_sat31(x.a, all.a);
            x.b = add_sat31(x.b, all.b);
        }
        all.a = add_sat31(all.a, part[0][w]);
        all.b = add_sat31(all.b, part[1][w]);
    }
    return x;
}
__device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t lp) { return (tokens + (1u << lp) - 1) >> lp; }

template <int T, int N>
__global__ __launch_bounds__(T) void page_step_kernel(StepArgs a, uint32_t role) {
    __shared__ uint32_t end[T * N];    // granted tokens up to and with a sequence
    __shared__ uint32_t taken[T * N];  // pages taken before it
    __shared__ uint32_t held[T * N];   // tokens it holds
    __shared__ uint32_t part[2][T / 64];
    __shared__ uint32_t total[3];
    __shared__ int32_t top[N == 1 ? T : 1];
    const uint32_t tid = threadIdx.x, cap = a.width << a.lp;
    const uint32_t fc = uint32_t(min(max(a.free_count[0], 0), int32_t(a.pages)));
    auto len_of = [&](uint32_t s) { return uint32_t(min(max(a.lens[s], 0), int32_t(cap))); };
    uint32_t n[N], c[N], need[N];
    bool fits[N];
    if (tid < 3) total[tid] = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t s = tid * N + j, at = min(s, a.seqs - 1);
        n[j] = len_of(at);
        c[j] = s < a.seqs ? uint32_t(max(a.counts[at], 0)) : 0u;
    }
    Sums2 own{0, 0}, all;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        fits[j] = c[j] <= cap - n[j];
        if (!fits[j]) c[j] = 0;
        need[j] = pages_of(n[j] + c[j], a.lp) - pages_of(n[j], a.lp);
        own.a = add_sat31(own.a, c[j]);
        own.b = add_sat31(own.b, need[j]);
    }
    // (the page that the first new token of this thread's sequence continues, if it does: asked for before the sums)
    const uint32_t row_n = n[0] & ((1u << a.lp) - 1);
    // and the stack's top, one page a sequence
    int32_t last_page = -1, top_page = -1;
    if (N == 1 && tid < a.seqs && c[0] && row_n) last_page = a.table[size_t(tid) * a.width + (n[0] >> a.lp)];
    if (N == 1 && tid < fc) top_page = a.free_pages[fc - 1 - tid];
    Sums2 at = block_before2<T / 64>(own, part, all);
    uint32_t tok = 0, pg = 0;  // the sums of the last one served
    const Sums2 first = at;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        taken[tid * N + j] = at.b;
        held[tid * N + j] = n[j];
        at.a = add_sat31(at.a, c[j]);
        at.b = add_sat31(at.b, need[j]);
        end[tid * N + j] = at.a;
        if (fits[j] && at.a <= a.tokens && at.b <= fc) tok = at.a, pg = at.b;
    }
    if (tok) atomicMax(&total[0], tok);
    if (pg) atomicMax(&total[1], pg);
    if (N == 1 && c[0] > 1) total[2] = 1;
    if (N == 1) top[tid] = top_page;
    __syncthreads();
    const uint32_t served = total[0], taken_all = total[1];
    if (role & kExpand) {
        auto put = [&](uint32_t r, int64_t slot, int32_t pos, int32_t seq) {
            a.slots[r] = slot;
            if (a.positions) a.positions[r] = pos;
            if (a.seq_of) a.seq_of[r] = seq;
        };
        if (N == 1 && !total[2]) {  // a decode step: a thread's sequence has one row at most
            if (blockIdx.x == 0 && c[0] && at.a <= served) {
                uint32_t page = uint32_t(last_page);
                if (!row_n) {
                    page = uint32_t(top[first.b]);  // (a page each: below T)
                    a.table[size_t(tid) * a.width + (n[0] >> a.lp)] = int32_t(page);
                }
                put(first.a, page < a.pages ? (int64_t(page) << a.lp) + row_n : -1, int32_t(n[0]), int32_t(tid));
            }
            for (uint32_t r = served + blockIdx.x * T + tid; r < a.tokens; r += gridDim.x * T) put(r, -1, -1, -1);
        } else {
            for (uint32_t r = blockIdx.x * T + tid; r < a.tokens; r += gridDim.x * T) {
                int64_t slot = -1;
                int32_t pos = -1, seq = -1;
                if (r < served) {
                    uint32_t lo = 0, hi = a.seqs - 1;  // the first sequence whose end is past r
                    while (lo < hi) {
                        const uint32_t mid = (lo + hi) >> 1;
                        if (end[mid] > r) hi = mid;
                        else lo = mid + 1;
                    }
                    const uint32_t len = held[lo], p = len + r - (lo ? end[lo - 1] : 0u), j = p >> a.lp;
                    const uint32_t old = pages_of(len, a.lp), row = p & ((1u << a.lp) - 1);
                    const uint32_t page = uint32_t(j < old ? a.table[size_t(lo) * a.width + j]
                                                           : a.free_pages[fc - 1 - (taken[lo] + j - old)]);
                    if (row == 0) a.table[size_t(lo) * a.width + j] = int32_t(page);  // a new page's first token is a new one
                    if (page < a.pages) slot = (int64_t(page) << a.lp) + row;
                    pos = int32_t(p);
                    seq = int32_t(lo);
                }
                put(r, slot, pos, seq);
            }
        }
    }
    if ((role & kCommit) && blockIdx.x == 0) {
        uint32_t b = min(first.a, served);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const uint32_t s = tid * N + j, e = min(end[s], served);
            if (s < a.seqs) {
                a.start[s] = int32_t(b);
                a.granted[s] = int32_t(e - b);
            }
            b = e;
        }
        if (tid == 0) {
            a.start[a.seqs] = int32_t(served);
            a.free_left[0] = int32_t(fc - taken_all);
        }
    }
}

// The pages that the sequences do not need go back: of all entries of theirs, in order of sequence and place, those that
// are pages; a page lies as far above the old top as there are pages behind it.  Entries that are none (pages given up)
// must not be handed out again, so a workgroup has to know how many of the entries behind its own 1024 are pages, and
// reads all of these: a wave its part of them, four sequences and up to 256 neighbours of each at once (8 and 256: the
// same; 8 and 128 or 4 and 512: 10 and 14 % slower); the sequence comes from a ballot over the ends that its lanes hold.
// 1024 entries and fewer are one workgroup's: 33 pages 3.6 us, as without; 2139 5.3; 512 sequences that give back 32,896
// 9.1, of which more than half are these reads and what finds their addresses.
struct ReleaseArgs {
    const int32_t* table;
    int32_t* free_pages;
    const int32_t* lens;
    const int32_t* keep;
    const int32_t* free_count;
    int32_t* free_left;
    uint32_t seqs, width, pages, lp;
};
constexpr int kReleaseT = 1024, kReleaseWaves = kReleaseT / 64;
template <int N>
__global__ __launch_bounds__(kReleaseT) void page_release_kernel(ReleaseArgs a, uint32_t role) {
    constexpr int T = kReleaseT, W = kReleaseWaves;
    __shared__ uint32_t end[T * N];
    __shared__ uint32_t from[T * N];  // the first entry of a sequence that goes back
    __shared__ uint32_t part[2][W];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = uint32_t(__builtin_amdgcn_readfirstlane(int(tid >> 6)));
    const uint32_t cap = a.width << a.lp;
    const uint32_t fc = uint32_t(min(max(a.free_count[0], 0), int32_t(a.pages)));
    uint32_t back[N];
    Sums2 own{0, 0}, all;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t s = min(tid * N + j, a.seqs - 1), n = uint32_t(min(max(a.lens[s], 0), int32_t(cap)));
        const uint32_t k = pages_of(min(uint32_t(max(a.keep[s], 0)), n), a.lp);
        from[tid * N + j] = k;
        back[j] = tid * N + j < a.seqs ? pages_of(n, a.lp) - k : 0u;
        own.a = add_sat31(own.a, back[j]);
    }
    Sums2 at = block_before2<W>(own, part, all);
#pragma unroll
    for (int j = 0; j < N; ++j) end[tid * N + j] = at.a = add_sat31(at.a, back[j]);
    __syncthreads();
    const uint32_t n = uniform(all.a);
    auto sequence_of = [&](uint32_t x) {  // the first one whose end is past x (< n)
        uint32_t lo = 0, hi = a.seqs - 1;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (end[mid] > x) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    };
    // entry x of sequence s is at this plus x (modulo 2^32) in its row
    auto row_off = [&](uint32_t s) { return from[s] - (s ? end[s - 1] : 0u); };
    // this workgroup's entries: c0 .. c1 - 1
    const uint32_t groups = role & kExpand ? gridDim.x : 1u;
    const uint32_t chunk = max((n + groups - 1) / groups, uint32_t(T));
    const uint32_t c0 = uint32_t(min(uint64_t(blockIdx.x) * chunk, uint64_t(n))), c1 = role & kExpand ? min(c0 + chunk, n) : 0u;
    if (blockIdx.x && c0 >= n) return;
    // how many of those behind them are no pages, a part of these a wave
    const uint32_t each = (n - c1 + W - 1) / W, x0 = min(c1 + wave * each, n), x1 = min(x0 + each, n);
    uint32_t none = 0;
    if (x0 < x1) {
        uint32_t s0 = uniform(sequence_of(x0)), my_end, my_off;  // of sequence s0 + lane
        auto hold = [&] {
            const uint32_t s = min(s0 + lane, a.seqs - 1);
            my_end = s0 + lane < a.seqs ? end[s] : 0u;
            my_off = row_off(s);
        };
        hold();
        for (uint32_t x = x0; x < x1;) {
            constexpr int U = 4, Q = 4;  // sequences at once, and reads of each
            int32_t v[U][Q];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint32_t i = 0, count = 0;
                if (x < x1) {
                    uint64_t past = __ballot(my_end > x);
                    while (!past) {  // ends: x is below the last sequence's end
                        s0 += 64;
                        hold();
                        past = __ballot(my_end > x);
                    }
                    i = uint32_t(__builtin_ctzll(past));
                    count = min(min(uint32_t(__builtin_amdgcn_readlane(int(my_end), int(i))), x1) - x, 64u * Q);
                }
                const uint32_t j = count ? uint32_t(__builtin_amdgcn_readlane(int(my_off), int(i))) + x : 0u;
                const int32_t* at = a.table + (count ? size_t(s0 + i) * a.width + j : 0);
                // (lanes past the entries read nothing, and get 0, which is a page)
                const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<int32_t*>(at), 0, int(count * 4), 0x00020000);
#pragma unroll
                for (int k = 0; k < Q; ++k) v[u][k] = int32_t(__builtin_amdgcn_raw_buffer_load_b32(r, lane * 4 + 256 * k, 0, 0));
                x += count;
            }
            asm volatile("" ::: "memory");  // all of them are asked for before the first is looked at
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int k = 0; k < Q; ++k) none += uint32_t(v[u][k]) >= a.pages;
        }
    }
    uint32_t in_wave;
    wave_before_sat(none, in_wave);
    if (lane == 0) part[1][wave] = in_wave;
    __syncthreads();
    uint32_t sum = n - c1;  // pages behind
#pragma unroll
    for (int w = 0; w < W; ++w) sum -= part[1][w];
    for (uint32_t b = c1; b > c0;) {  // from the last entry on: a page's place is behind those of the pages behind it
        const uint32_t x = b - 1 - tid;
        int32_t v = -1;
        if (tid < b - c0) {
            const uint32_t s = sequence_of(x);
            v = a.table[size_t(s) * a.width + (row_off(s) + x)];
        }
        const bool is = uint32_t(v) < a.pages;
        const uint64_t m = __ballot(is);
        __syncthreads();
        if (lane == 0) part[0][wave] = uint32_t(__popcll(m));
        __syncthreads();
        uint32_t place = fc + sum + uint32_t(__popcll(m & ((uint64_t(1) << lane) - 1)));
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (uint32_t(w) < wave) place += part[0][w];
            sum += part[0][w];
        }
        if (is && place < a.pages) a.free_pages[place] = v;
        b -= min(b - c0, uint32_t(T));
    }
    if ((role & kCommit) && blockIdx.x == 0 && tid == 0) a.free_left[0] = int32_t(min(fc + sum, a.pages));
}

// Workgroups of T threads for `rows` rows; where what one writes is what others read, one workgroup or two launches.
template <class F>
void expand_and_commit(size_t rows, int T, bool overlap, F launch) {
    const size_t blocks = (rows + T - 1) / T, most = 1024;
    const uint32_t g = uint32_t(blocks < most ? blocks : most);
    if (!overlap) return launch(g, kExpand | kCommit);
    if (rows <= kOneTable) return launch(1u, kExpand | kCommit);
    launch(g, kExpand);
    launch(1u, kCommit);
}
void run_step(const StepArgs& a, hipStream_t stream) {
    const bool overlap = a.granted == a.counts || a.free_left == a.free_count;
    auto run = [&](auto kernel, int T) {
        expand_and_commit(a.tokens, T, overlap, [&](uint32_t g, uint32_t role) {
            hipLaunchKernelGGL(kernel, dim3(g), dim3(T), 0, stream, a, role);
        });
    };
    if (a.seqs <= 256) run(page_step_kernel<256, 1>, 256);
    else if (a.seqs <= 1024) run(page_step_kernel<256, 4>, 256);
    else run(page_step_kernel<1024, 8>, 1024);
}
void run_release(const ReleaseArgs& a, hipStream_t stream) {
    const size_t all = size_t(a.seqs) * a.width, entries = all < a.pages ? all : a.pages, most = size_t(256) * kReleaseT;
    auto run = [&](auto kernel) {  // (at most a workgroup a CU)
        expand_and_commit(entries < most ? entries : most, kReleaseT, a.free_left == a.free_count, [&](uint32_t g, uint32_t role) {
            hipLaunchKernelGGL(kernel, dim3(g), dim3(kReleaseT), 0, stream, a, role);
        });
    };
    if (a.seqs <= kReleaseT) run(page_release_kernel<1>);
    else run(page_release_kernel<8>);
}

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
// head_dim * size / 16 lanes.  Each byte moves once: bound by HBM, and for a step's few
// rows by a launch and two round trips (the slot, then the row).
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

// The same with the bounds of the pages that get rows.  The rows of one page in a call
// are neighbours: C waves share such a run for one kv head, write its rows, read the
// page's rows before them, and have the bounds without reading the new rows back.  A
// workgroup looks for the runs that end in its B tokens: one token where there are few
// (a decode step), else about a page's, as a workgroup that finds none has cost a wait.
// Bound by HBM where rows are many (8218 tokens of 24 sequences, 8 kv heads of 128, bf16,
// 102 MB: 22 to 27 us, 3.8 to 4.4 TB/s; a copy of as many bytes takes 20), else by the chain
// of slots, held rows and bounds: 64 decoding sequences: 5.0 us.  With the bounds in a launch
// of their own, which reads the new rows back, these took 41 and 6.7.
template <int TYPE, int D, int C>
__global__ __launch_bounds__(256) void paged_append_bounds_kernel(AppendArgs a, uint32_t tokens, uint32_t B) {
    typedef typename Held<TYPE>::type T;
    constexpr int E = 16 / sizeof(T), L = D / E, R = 64 / L;  // elements a lane, lanes a row, rows at once
    constexpr int U = 4;
    typedef T vec __attribute__((ext_vector_type(E)));
    __shared__ float ends_of[2][C][2][D];  // with C > 1: least and greatest of waves 1 ..
    const int lane = threadIdx.x & 63, l = lane % L, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int part = C > 1 ? wave : 0;
    const uint32_t h = blockIdx.x % a.KH, block0 = blockIdx.x / a.KH * B;
    const int64_t ps = int64_t(1) << a.lp;
    auto slot_at = [&](uint32_t t) { return t < tokens ? a.slots[t] : int64_t(-1); };
    int z = 0;  // runs so far (the same in every wave)
    for (uint32_t t0 = block0; t0 < block0 + B && t0 < tokens; t0 += 64) {
        const int64_t mine = uint32_t(lane) < block0 + B - t0 ? slot_at(t0 + lane) : -1, next = slot_at(t0 + lane + 1);
        uint64_t runs = __ballot(mine >= 0 && mine < a.all_slots && !(next == mine + 1 && (next & (ps - 1)) != 0));
        for (; runs; ++z) {
            const int at = __builtin_ctzll(runs);
            runs &= runs - 1;
            if (C == 1 && z % 4 != wave) continue;
            const uint32_t t = t0 + uint32_t(at);  // the run's last token
            const uint64_t slot = uint64_t(uint32_t(__builtin_amdgcn_readlane(int(mine), at))) |
                                  uint64_t(uint32_t(__builtin_amdgcn_readlane(int(mine >> 32), at))) << 32;
            const int last = int(slot & uint64_t(ps - 1));
            int n = 0;  // rows of the run
            for (bool more = true; more; n += 64) {  // ends: at token 0, at the page's first row, or before
                const int64_t back = int64_t(n) + lane;
                const bool same = back <= last && back <= int64_t(t) && a.slots[int64_t(t) - back] == int64_t(slot) - back;
                const uint64_t m = ~__ballot(same);
                if (m) {
                    n += __builtin_ctzll(m) - 64;
                    more = false;
                }
            }
            const size_t head = size_t(slot >> a.lp) * a.KH + h;
            const size_t base = (head << a.lp) * D + l * E;
            T* pk = reinterpret_cast<T*>(a.k) + base;
            T* pv = reinterpret_cast<T*>(a.v) + base;
            float lo[E], hi[E];
#pragma unroll
            for (int i = 0; i < E; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
            auto take = [&](const vec& x) {
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    lo[i] = fminf(lo[i], float(x[i]));
                    hi[i] = fmaxf(hi[i], float(x[i]));
                }
            };
            const int first = last + 1 - n;
#pragma unroll 4
            for (int r = part * R + lane / L; r < first; r += C * R) take(*reinterpret_cast<const vec*>(pk + size_t(r) * D));
            const size_t src = size_t(t - uint32_t(n - 1)) * a.stride + h * D + l * E;
            // U rows' loads before their stores: a load behind a store waits until that is done
            for (int r0 = part * R + lane / L; r0 < n; r0 += U * C * R) {
                float4 x[U][E / 4], y[U][E / 4];
#pragma unroll
                for (int j = 0; j < U; ++j)
#pragma unroll
                    for (int i = 0; i < E / 4; ++i) {
                        const size_t from = src + min(r0 + j * C * R, n - 1) * a.stride + 4 * i;
                        x[j][i] = *reinterpret_cast<const float4*>(a.src_k + from);
                        y[j][i] = *reinterpret_cast<const float4*>(a.src_v + from);
                    }
#pragma unroll
                for (int j = 0; j < U; ++j) {
                    const int r = r0 + j * C * R;
                    if (r >= n) break;
                    vec k, v;
#pragma unroll
                    for (int i = 0; i < E / 4; ++i) {
                        const float4 p = x[j][i], q = y[j][i];
                        k[4 * i] = T(p.x), k[4 * i + 1] = T(p.y), k[4 * i + 2] = T(p.z), k[4 * i + 3] = T(p.w);
                        v[4 * i] = T(q.x), v[4 * i + 1] = T(q.y), v[4 * i + 2] = T(q.z), v[4 * i + 3] = T(q.w);
                    }
                    *reinterpret_cast<vec*>(pk + size_t(first + r) * D) = k;
                    *reinterpret_cast<vec*>(pv + size_t(first + r) * D) = v;
                    take(k);
                }
            }
#pragma unroll
            for (int i = 0; i < E; ++i)
#pragma unroll
                for (int m = L; m < 64; m *= 2) {
                    lo[i] = fminf(lo[i], __shfl_xor(lo[i], m));
                    hi[i] = fmaxf(hi[i], __shfl_xor(hi[i], m));
                }
            // (two buffers: a wave that is a run ahead has passed the barrier that the first one came to after reading)
            if constexpr (C > 1) {
                if (wave && lane < L)
#pragma unroll
                    for (int i = 0; i < E; ++i) ends_of[z & 1][wave][0][l * E + i] = lo[i], ends_of[z & 1][wave][1][l * E + i] = hi[i];
                __syncthreads();
                if (wave) continue;
            }
            float most = 0.0f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
#pragma unroll
                for (int w = 1; w < C; ++w) {
                    lo[i] = fminf(lo[i], ends_of[z & 1][w][0][l * E + i]);
                    hi[i] = fmaxf(hi[i], ends_of[z & 1][w][1][l * E + i]);
                }
                if (lo[i] > hi[i]) lo[i] = hi[i] = 0.0f;  // NaN only
                most = fmaxf(most, fmaxf(fabsf(lo[i]), fabsf(hi[i])));
            }
#pragma unroll
            for (int m = 1; m < L; m *= 2) most = fmaxf(most, __shfl_xor(most, m));
            const int e = bound_exp(most);
            uint32_t w[2][E / 4] = {};
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
    }
}
constexpr uint32_t kFewRows = 8192;

template <int TYPE, int D>
void run_append(const AppendArgs& a, hipStream_t stream) {
    if (a.bounds) {
        // us with C = 4 and a workgroup a (token, head), and with C = 1 in blocks: 300 decoding sequences of 8 kv heads, pages of
        // 256, fp32: 37, 124; 1000 tokens of two prompts, pages of 16: 16, 10; 2000: 30, 11.  Blocks of 16 and 32: 8200 tokens,
        // pages of 16: 22, 23; of 32: 26, 22.
        const uint32_t tokens = a.rows / a.KH, ps = 1u << a.lp;
        auto run = [&](auto kernel, uint32_t threads, uint32_t B) {
            hipLaunchKernelGGL(kernel, dim3((tokens + B - 1) / B * a.KH), dim3(threads), 0, stream, a, tokens, B);
        };
        if (a.rows <= kFewRows) run(paged_append_bounds_kernel<TYPE, D, 4>, 256, 1);
        else run(paged_append_bounds_kernel<TYPE, D, 1>, 256, ps < 32 || a.rows <= 4 * kFewRows ? 16 : 32);
        return;
    }
    constexpr uint32_t per = 256 / (D * sizeof(typename Held<TYPE>::type) / 16);
    hipLaunchKernelGGL((paged_append_kernel<TYPE, D>), dim3((a.rows + per - 1) / per), dim3(256), 0, stream, a);
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
    zq::run_step(a, static_cast<hipStream_t>(stream));
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
    zq::run_release(a, static_cast<hipStream_t>(stream));
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
