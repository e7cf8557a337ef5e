// What the kernels over K / V pages of 16-bit numbers share: their number types and
// the request of a token.
#pragma once
#include "attn.h"

namespace v1 {
namespace paged {

using namespace attn;

constexpr int kDim = 128;

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Two numbers of T (__bf16 or _Float16) in a register <-> fp32; to T by nearest even.
template <class T>
using Pair = __attribute__((ext_vector_type(2))) T;

template <class T>
__device__ __forceinline__ uint32_t pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), Pair<T>));
}

template <class T>
__device__ __forceinline__ f32x2 unpack(uint32_t w) {
    return __builtin_convertvector(__builtin_bit_cast(Pair<T>, w), f32x2);
}

// The last of 0 .. n - 1 whose start (ascending) is `at` or less; 0: none is.  64 of
// them are looked at at a time, by a whole wave.
template <class Start>
__device__ __forceinline__ int32_t last_at_most(int32_t n, int32_t at, Start start) {
    const int32_t lane = (int32_t)threadIdx.x % kWave;
    int32_t from = 0;
    while (n > 1) {
        const int32_t step = (n + kWave - 1) / kWave, i = lane * step;
        const bool past = i >= n || start(from + min(i, n - 1)) > at;
        const int32_t skip = (max(__popcll(__ballot(!past)), 1) - 1) * step;
        from += skip;
        n = min(step, n - skip);
    }
    return __builtin_amdgcn_readfirstlane(from);
}

// The request that holds token t: cu[r] <= t < cu[r + 1]; -1: none.
__device__ __forceinline__ int32_t request_of(const int32_t* cu, int32_t requests, int32_t t) {
    const int32_t r = last_at_most(requests, t, [&](int32_t i) __attribute__((always_inline)) { return cu[i]; });
    return cu[r] <= t && t < cu[r + 1] ? r : -1;
}

}  // namespace paged
}  // namespace v1
