// code_common.hpp -- 8-bit codes of numbers by their largest, shared by the
// cache's append and the quantised rows; and accesses of 16 bytes at any
// alignment of their elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace manta {

// As one vector: of a struct's elements the compiler makes several accesses.
typedef uint32_t Words4 __attribute__((ext_vector_type(4)));
typedef Words4 Words4Any __attribute__((aligned(2)));
template <class P>
__device__ __forceinline__ P load16_any(const void* p) {
    static_assert(sizeof(P) == 16, "16 bytes");
    return __builtin_bit_cast(P, (Words4)*(const Words4Any*)p);
}
template <class P>
__device__ __forceinline__ void store16_any(void* p, const P& v) {
    static_assert(sizeof(P) == 16, "16 bytes");
    *(Words4Any*)p = __builtin_bit_cast(Words4, v);
}
// Of data that is too large to be found in a cache afterwards.
template <class P>
__device__ __forceinline__ void store16_past(void* p, const P& v) {
    static_assert(sizeof(P) == 16, "16 bytes");
    __builtin_nontemporal_store(__builtin_bit_cast(Words4, v), (Words4Any*)p);
}

// Four codes, t[j] / max rounded half to even, the division left out where it
// cannot matter: t * (1 / max) is within 127 * 3 * 2^-24 < 2^-15 of it (three
// roundings), so only what lies closer than that to a half is divided.  Adding
// 1.5 * 2^23 rounds, and leaves the code in the low byte.  |t| <= 127 max, but
// for t beyond the largest number; `exact`: there may be such a t (max >= 2^121;
// its code is 127 or -127), or 1 / max is not a normal number.
__device__ __forceinline__ uint32_t ratio_codes(const float* t, float max, float inv, bool exact) {
#pragma clang fp contract(off)  // (here, not in the file: what includes it has its own rule)
    constexpr float kRound = 12582912.0f;
    uint32_t b[4];
    float far = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float q = t[j] * inv, n = q + kRound;
        far = fmaxf(far, fabsf(q - (n - kRound)));
        b[j] = __float_as_uint(n);
    }
    if (exact || far > 0.5f - 0x1p-15f) {
#pragma unroll
        for (int j = 0; j < 4; j++)
            b[j] = (uint32_t)(int)fminf(127.0f, fmaxf(-127.0f, __builtin_rintf(__fdiv_rn(t[j], max))));
    }
    const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), hi = __builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u);
    return lo | hi << 16;
}

}  // namespace manta
