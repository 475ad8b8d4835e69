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

// rint((x - low) 255 / size) in 64-bit arithmetic, of VEC elements as bytes; `bad`: an element is NaN.  Of 32-bit elements the quotient in 32 bits is within 8 *
// 10^-5 of the exact one, which decides all but those next to a half; there (x - low) 255 is compared with a half more of size, both exact.  (With a 64-bit
// division for each element 777 x 50001 bfloat16 took 44 us, not 25.)
struct Coder {
    double low, size, divisor;
    float low32, scale;                                               // scale 0: the 32-bit quotient does not do
    __device__ __forceinline__ Coder(double low_, double high) : low(low_), size(high - low_), divisor(size > 0 ? size : 1.0), low32((float)low_)
    {
        const float range = (float)size;
        scale = range > 1e-30f && range < 1e30f ? 255.f * __builtin_amdgcn_rcpf(range) : 0.f;
    }
    template <int VEC>
    __device__ __forceinline__ void operator()(const float (&x)[VEC], uint32_t (&c)[VEC / 4], bool &bad) const
    {
        bool sure = scale != 0.f, known[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float u = (x[k] - low32) * scale, q = __builtin_rintf(u);
            known[k] = __builtin_fabsf(u - q) < 0.5f - 0x1p-12f;
            sure &= known[k];
            c[k / 4] = __builtin_amdgcn_cvt_pk_u8_f32(q, k % 4, k % 4 ? c[k / 4] : 0);
        }
        if (sure) return;
#pragma unroll
        for (int k = 0; k < VEC; ++k)
            if (scale == 0.f || !known[k]) {
                bad |= x[k] != x[k];
                c[k / 4] = __builtin_amdgcn_cvt_pk_u8_f32((float)of((double)x[k]), k % 4, c[k / 4]);
            }
    }
    template <int VEC>
    __device__ __forceinline__ void operator()(const double (&x)[VEC], uint32_t (&c)[VEC / 4], bool &bad) const
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            bad |= x[k] != x[k];
            c[k / 4] = __builtin_amdgcn_cvt_pk_u8_f32((float)rint((x[k] - low) * 255.0 / divisor), k % 4, k % 4 ? c[k / 4] : 0);
        }
    }
    __device__ __forceinline__ double of(double x) const
    {
        const double part = (x - low) * 255.0;
        double q = scale != 0.f ? rint((double)(((float)x - low32) * scale)) : rint(part / divisor);
        const double rest = __builtin_fma(-q, size, part), half = 0.5 * size;
        const bool odd = (int)q & 1;
        if (rest > half || (rest == half && odd)) q += 1;
        if (rest < -half || (rest == -half && odd)) q -= 1;
        return q;
    }
};

__device__ __forceinline__ float min_of(float a, float b) { return __builtin_fminf(a, b); }
__device__ __forceinline__ double min_of(double a, double b) { return __builtin_fmin(a, b); }

// The scale of a group from its lowest and highest element; bad: NaN
template <typename A>
__device__ __forceinline__ CodeScale<A> scale_of(A low, const Coder &code, bool bad)
{
    double step = code.size * (1 / 255.0);                            // (code.size / 255, without a division)
    step = __builtin_fma(__builtin_fma(-step, 255.0, code.size), 1 / 255.0, step);
    CodeScale<A> s = {low, (A)step};
    // (the highest code may not stand for infinity)
    if (!(__builtin_fabs((double)(A)__builtin_fma(255.0, (double)s.step, (double)low)) <= __DBL_MAX__)) s.step = s.step * (A)(1 - 0x1p-23);
    if (bad) s.low = s.step = (A)__builtin_nanf("");
    return s;
}

constexpr int kCodeLanes = 16, kCodeEach = kCodeGroup / kCodeLanes;   // a row of DPP has a group, a lane eight elements of it
template <typename T>
struct EightOf {                                                      // as they lie in memory, at any element's address
    static constexpr int VEC = Vec16<T>::N < kCodeEach ? Vec16<T>::N : kCodeEach, PIECES = kCodeEach / VEC;
    typedef typename Vec16<T>::type V;
};

// Groups first, first + step, ... of n elements become codes, by rows of 16 lanes.
template <typename T>
__device__ __forceinline__ void encode_groups(const T *__restrict__ x, int64_t n, uint8_t *__restrict__ codes, CodeScale<typename Wide<T>::type> *__restrict__ scales,
                                              int64_t first, int64_t step)
{
    typedef typename Wide<T>::type A;
    typedef typename EightOf<T>::V V;
    const int lane = threadIdx.x % kCodeLanes;
    const int64_t groups = (n + kCodeGroup - 1) / kCodeGroup;
    for (int64_t g = first; g < groups; g += step) {
        const int64_t at = g * kCodeGroup + lane * kCodeEach;
        const bool whole = (g + 1) * kCodeGroup <= n;
        A v[kCodeEach];
        if (whole) {
#pragma unroll
            for (int p = 0; p < EightOf<T>::PIECES; ++p) {
                const V u = *reinterpret_cast<const V *>(x + at + p * EightOf<T>::VEC);
#pragma unroll
                for (int k = 0; k < EightOf<T>::VEC; ++k) v[p * EightOf<T>::VEC + k] = (A)u[k];
            }
        } else {                                                      // (what is missing is as the last element)
#pragma unroll
            for (int k = 0; k < kCodeEach; ++k) v[k] = (A)x[at + k < n ? at + k : n - 1];
        }
        A low = v[0], high = v[0];                                    // (NaN is passed over, and found by the coder)
#pragma unroll
        for (int k = 1; k < kCodeEach; ++k) low = min_of(low, v[k]), high = max_of(high, v[k]);
        low = -row16_max(-low);
        high = row16_max(high);
        const Coder code((double)low, (double)high);
        bool bad = !(code.size * 255.0 <= __DBL_MAX__);
        uint32_t c[2];
        code(v, c, bad);
        bad = (__ballot(bad) >> (threadIdx.x & 48) & 0xFFFF) != 0;
        if (bad) c[0] = c[1] = 0;
        if (whole) {
            *reinterpret_cast<u32x2 *>(codes + at) = u32x2{c[0], c[1]};
        } else {
#pragma unroll
            for (int k = 0; k < kCodeEach; ++k)
                if (at + k < n) codes[at + k] = (uint8_t)(c[k / 4] >> 8 * (k % 4));
        }
        if (lane == 0) scales[g] = scale_of(low, code, bad);
    }
}

// VEC coded float32 elements from a flat index on, as they are loaded, and their values.  RAGGED: the index is any, and the elements may be of two groups.
typedef uint32_t u32_any __attribute__((aligned(1)));
template <int VEC, bool RAGGED>
struct Coded {
    static_assert(VEC == 1 || VEC == 4, "a byte or a word of codes");
    uint32_t c;
    CodeScale<float> first, second;
    int left;                                                         // elements of the first group
    template <typename I>
    __device__ __forceinline__ void load(const uint8_t *__restrict__ codes, const CodeScale<float> *__restrict__ scales, I i)
    {
        first = scales[i / kCodeGroup];
        if constexpr (VEC == 1) {
            c = codes[i];
        } else if constexpr (RAGGED) {
            c = *reinterpret_cast<const u32_any *>(codes + i);
            second = scales[(i + 3) / kCodeGroup];
            left = kCodeGroup - (int)(i & (kCodeGroup - 1));
        } else {
            c = *reinterpret_cast<const uint32_t *>(codes + i);
        }
    }
    __device__ __forceinline__ void values(float (&v)[VEC]) const
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const CodeScale<float> s = !(RAGGED && VEC > 1) || k < left ? first : second;
            v[k] = __builtin_fmaf((float)(VEC == 1 ? c : (c >> 8 * k) & 255u), s.step, s.low);
        }
    }
};

#endif  // __HIPCC__
