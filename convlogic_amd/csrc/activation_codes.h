// Activations in 8 bits: 128 elements, in the order in which they lie in memory, share their lowest value and a step; element i is scales[i / 128].x +
// codes[i] scales[i / 128].y.
#pragma once

#include "row_tile.h"

constexpr int kCodeGroup = 128;

#if defined(__HIPCC__)

template <typename A>
struct CodeScale {                                                    // NaN: a group that cannot be told in codes
    A low, step;
};

// VEC coded float32 elements from the flat index i on.  RAGGED: i is any index, and the elements may be of two groups.
typedef uint32_t u32_any __attribute__((aligned(1)));
template <int VEC, bool RAGGED>
__device__ __forceinline__ void decode_at(const uint8_t *__restrict__ codes, const CodeScale<float> *__restrict__ scales, int64_t i, float (&v)[VEC])
{
    static_assert(VEC == 1 || VEC == 4, "a byte or a word of codes");
    const CodeScale<float> first = scales[i / kCodeGroup];
    if constexpr (VEC == 1) {
        v[0] = __builtin_fmaf((float)codes[i], first.step, first.low);
    } else {
        uint32_t c;
        if constexpr (RAGGED) c = *reinterpret_cast<const u32_any *>(codes + i);
        else c = *reinterpret_cast<const uint32_t *>(codes + i);
        CodeScale<float> second = first;
        if constexpr (RAGGED) second = scales[(i + 3) / kCodeGroup];
        const int left = kCodeGroup - (int)(i & (kCodeGroup - 1));    // elements of the first group
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const CodeScale<float> s = !RAGGED || k < left ? first : second;
            v[k] = __builtin_fmaf((float)((c >> 8 * k) & 255u), s.step, s.low);
        }
    }
}

#endif  // __HIPCC__
