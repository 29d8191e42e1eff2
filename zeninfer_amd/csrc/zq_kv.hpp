// zq_kv.hpp -- the 4-bit KV cache inside the library: what the append, read,
// evict (zq_kv.hip) and attention (zq_attn_q4.hip) launchers share, and the
// device-side decode of its rows.
#pragma once
#include "../../include/zq_kv.h"
#include "zq_device.hpp"

namespace zq {

// Bounds that keep every index of the kernels in range: rows of one call fit 31
// bits, a launch's threads (64 a row at most) 32, as HIP asks; byte offsets are size_t.
constexpr size_t kKvMaxCapacity = size_t(1) << 24, kKvMaxHeads = size_t(1) << 20, kKvMaxRows = size_t(1) << 25;
constexpr size_t kMaxThreads = (size_t(1) << 32) - 1;  // of a launch

// Shape, pointers and alignment of a cache, as include/zq_kv.h asks for them.
bool kv_q4_ok(const zq_kv_q4* c);

hipError_t launch_kv_q4_append(const zq_kv_q4& c, const float* k, const float* v, size_t tokens, size_t stride,
                               const int32_t* lens, const int32_t* counts, const int32_t* first_pos,
                               hipStream_t stream);
hipError_t launch_kv_q4_read(const zq_kv_q4& c, float* k, float* v, size_t tokens, const int32_t* first,
                             const int32_t* counts, hipStream_t stream);
hipError_t launch_kv_q4_evict(const zq_kv_q4& c, const zq_kv_q4& dst, bool in_place, const int32_t* lens, size_t keep,
                              size_t recent, size_t first, const int32_t* next_pos, void* ws, hipStream_t stream);
size_t kv_q4_evict_bytes(const zq_kv_q4& c, size_t keep);
// RoPE (adjacent pairs) of T tokens' q into q_out ([T][H * D]) and of their k, then
// k and v appended to one sequence's cache at slots *len on, positions *pos on.
// q, k, v: rows ld floats apart (0: dense).
hipError_t launch_rope_kv_q4(const zq_kv_q4& c, const float* q, float* q_out, const float* k, const float* v,
                             const float* cos_tab, const float* sin_tab, const int32_t* len, const uint32_t* pos,
                             uint32_t T, uint32_t H, uint32_t pairs, uint32_t ld, hipStream_t stream);
// attention: dims of the call, the workspace it needs, the launch
size_t attention_q4_bytes(const zq_kv_q4& c, size_t tokens, size_t heads, int flags);
hipError_t launch_attention_q4(const zq_kv_q4& c, const float* q, float* out, size_t tokens, size_t heads, size_t stride,
                               const int32_t* lens, const int32_t* counts, float scale, int flags, void* ws,
                               hipStream_t stream);

#if defined(__HIPCC__)
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));

// Two nibbles at bits 0..3 and 16..19 of u as fp16 code - 8: 0x6400 | n is
// 1024 + n, and the difference to 1032 is exact.  `one` is 0x64006400 in a vector
// register (code_bits()): with it the mask and the or are one instruction, which
// takes no two literals.
__device__ __forceinline__ uint32_t code_bits() {
    uint32_t x = 0x64006400u;
    asm("" : "+v"(x));  // no constant to the compiler
    return x;
}
__device__ __forceinline__ h2_t nibbles2(uint32_t u, uint32_t one) {
    const h2_t x = __builtin_bit_cast(h2_t, (u & 0x000f000fu) | one);
    return x - h2_t{_Float16(1032.0f), _Float16(1032.0f)};
}
__device__ __forceinline__ int32_t clamp_len(int32_t n, size_t most) {
    return n < 0 ? 0 : (size_t(n) > most ? int32_t(most) : n);
}
#endif

}  // namespace zq
