// zq_attn_q4_at.hpp -- where the 128-row attention kernel of the 4-bit KV cache
// reads: offsets of what one thread stages of a step's keys.  Plain C++, so that a
// host program can check every address.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define ZQ_HD __host__ __device__ __forceinline__
#else
#define ZQ_HD inline
#endif

namespace zq {

// Keys of a step, and tasks of K and of V that its threads share.
template <int D>
struct StageShape {
    static constexpr int TK = D <= 128 ? 64 : 32;
    static constexpr int kTasks = TK * D / 32;
};

// Byte offsets of a task's codes and scales from those of the step's first key on (key0,
// below the capacity).  A capacity is a multiple of 32, so a step of 64 keys may pass it:
// the tasks past it take the last key, or the last 8 keys, and what they give is masked.
struct StageAt {
    uint32_t codes, scales;
};
// Task e of K: 16 bytes of key e / (D / 32), its block e % (D / 32), and that block's scale.
template <int D>
ZQ_HD StageAt stage_k_at(uint32_t capacity, uint32_t key0, uint32_t e) {
    uint32_t key = e / (D / 32);
    const uint32_t b = e % (D / 32);
    if (StageShape<D>::TK > 32 && key > capacity - 1 - key0) key = capacity - 1 - key0;
    return {key * (D / 2) + b * 16, (b * capacity + key) * 2u};
}
// Task e of V: two bytes, column pair ch, of the 8 keys of group o (rows D / 2 apart), and 8 scales.
struct StageV {
    uint32_t ch, o;
};
template <int D>
ZQ_HD StageV stage_v_task(uint32_t e) {
    return {(e >> 1) % (D / 4), (e & 1) + 2 * (e / (D / 2))};
}
template <int D>
ZQ_HD StageAt stage_v_at(uint32_t capacity, uint32_t key0, uint32_t e) {
    const StageV t = stage_v_task<D>(e);
    uint32_t key = 8 * t.o;
    if (StageShape<D>::TK > 32 && key > capacity - 8 - key0) key = capacity - 8 - key0;
    return {key * (D / 2) + 2 * t.ch, (t.ch / 8 * capacity + key) * 2u};
}

}  // namespace zq
