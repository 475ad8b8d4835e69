// Rows of scores as the kernels over classes, vocabularies and experts hold them: element types, tiles in registers, sums and maxima over a workgroup.
#pragma once

#include "clg_common.h"

#if defined(__HIPCC__)

template <typename T>
struct Wide {                                                         // what sums and softmax values of T are held in
    typedef float type;
};
template <>
struct Wide<double> {
    typedef double type;
};

// 16 bytes of a row.  Rows of an odd number of 2-byte elements start at any even address, which a wide access to global memory takes as it is.
template <typename T>
struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

__device__ __forceinline__ float lowest(float) { return -__builtin_inff(); }
__device__ __forceinline__ double lowest(double) { return -__builtin_inf(); }
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_fmaxf(a, b); }
__device__ __forceinline__ double max_of(double a, double b) { return __builtin_fmax(a, b); }

// e^(x / temperature) for x <= 0 up to the sign of rounding: scale is log2(e) / temperature for floats, 1 / temperature for doubles
__device__ __forceinline__ float exp_scaled(float x, float scale) { return __builtin_amdgcn_exp2f(x * scale); }
__device__ __forceinline__ double exp_scaled(double x, double scale) { return exp(x * scale); }
template <typename A>
__host__ __device__ inline A exp_scale(double temperature)
{
    return (A)((sizeof(A) == 4 ? 1.4426950408889634074 : 1.0) / temperature);
}

// a maximum as the sums subtract it: an infinite one is left out, so that rows of -inf sum to 0, rows with +inf to inf and NaN stays NaN
template <typename A>
__device__ __forceinline__ A finite_or_zero(A m)
{
    return __builtin_isinf(m) ? A(0) : m;
}

// the sum s of exponentials relative to the maximum `from` as one relative to `to`, which is no lower (a sum over -inf alone is 0, or NaN)
template <typename A>
__device__ __forceinline__ A rescaled(A s, A from, A to, A scale)
{
    return from == lowest(A(0)) ? s : s * exp_scaled(finite_or_zero(from) - finite_or_zero(to), scale);
}

// Maximum over the 64 lanes (NaN is passed over), valid in all of them.
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ float dpp_keep(float v)
{
    const int u = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(u, u, CTRL, ROW_MASK, 0xF, false));
}
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ double dpp_keep(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const int l = (int)(uint32_t)u, h = (int)(uint32_t)(u >> 32);
    const uint32_t lo = __builtin_amdgcn_update_dpp(l, l, CTRL, ROW_MASK, 0xF, false), hi = __builtin_amdgcn_update_dpp(h, h, CTRL, ROW_MASK, 0xF, false);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ float last_lane(float v) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63)); }
__device__ __forceinline__ double last_lane(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, 63), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
template <typename A>
__device__ __forceinline__ A wave_max(A v)
{
    v = max_of(v, dpp_keep<0xB1, 0xF>(v));
    v = max_of(v, dpp_keep<0x4E, 0xF>(v));
    v = max_of(v, dpp_keep<0x141, 0xF>(v));
    v = max_of(v, dpp_keep<0x140, 0xF>(v));
    v = max_of(v, dpp_keep<0x142, 0xA>(v));
    v = max_of(v, dpp_keep<0x143, 0xC>(v));
    return last_lane(v);
}

// Columns base .. of one row in the registers of a workgroup: thread t holds the 16-byte pieces t, t + THREADS, ... and, of what is left of a row
// behind its last whole piece, one element.  What is behind the row is -inf.
template <typename T, int THREADS, int NV>
struct RowTile {
    static constexpr int VEC = Vec16<T>::N, COLS = THREADS * NV * VEC;
    typedef typename Vec16<T>::type V;
    V v[NV];
    T last;
    int whole, tail;                                                  // whole pieces in the tile, elements behind them

    __device__ __forceinline__ void load(const T *__restrict__ row, int64_t base, int64_t cols)
    {
        const int n = (int)(cols - base < COLS ? cols - base : COLS), tid = threadIdx.x;
        whole = n / VEC;
        tail = n % VEC;
        const T none = (T)lowest(0.f);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int p = j * THREADS + tid;
            if (j * THREADS < whole) {                                // (of the workgroup; lanes behind the row read its last piece again)
                v[j] = *reinterpret_cast<const V *>(row + base + (int64_t)(p < whole ? p : whole - 1) * VEC);
                if (p >= whole) v[j] = (V)none;
            } else {
                v[j] = (V)none;
            }
        }
        last = tid < tail ? row[base + (int64_t)whole * VEC + tid] : none;
    }
    // f(element, column in the tile) for the row's elements that this thread holds
    template <typename F>
    __device__ __forceinline__ void each(F f)
    {
        const int tid = threadIdx.x;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (j * THREADS >= whole) break;
            if (j * THREADS + tid >= whole) break;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                T x = v[j][i];
                f(x, (j * THREADS + tid) * VEC + i);
                v[j][i] = x;
            }
        }
        if (tid < tail) f(last, whole * VEC + tid);
    }
    // the same columns of `row` = f(element); f's result is A
    template <typename F>
    __device__ __forceinline__ void store(T *__restrict__ row, int64_t base, F f) const
    {
        const int tid = threadIdx.x;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int p = j * THREADS + tid;
            if (j * THREADS >= whole) break;
            V out;
#pragma unroll
            for (int i = 0; i < VEC; ++i) out[i] = (T)f(v[j][i]);
            if (p < whole) *reinterpret_cast<V *>(row + base + (int64_t)p * VEC) = out;
        }
        if (tid < tail) row[base + (int64_t)whole * VEC + tid] = (T)f(last);
    }
};

// Sums (SUM) or maxima of COUNT values per thread over the workgroup, valid in all threads; the order is fixed.  `room`: COUNT values per wavefront.
// The caller has a barrier between two uses of the same room.
template <bool SUM, int THREADS, int COUNT, typename A>
__device__ __forceinline__ void block_reduce(A (&x)[COUNT], A *room)
{
#pragma unroll
    for (int c = 0; c < COUNT; ++c) x[c] = SUM ? wave_sum(x[c]) : wave_max(x[c]);
    if constexpr (THREADS > kWave) {
        constexpr int WAVES = THREADS / kWave;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int c = 0; c < COUNT; ++c) room[(threadIdx.x >> 6) * COUNT + c] = x[c];
        __syncthreads();
#pragma unroll
        for (int c = 0; c < COUNT; ++c) {
            A r = room[c];
            for (int w = 1; w < WAVES; ++w) r = SUM ? r + room[w * COUNT + c] : max_of(r, room[w * COUNT + c]);
            x[c] = r;
        }
    }
}

// element i of an array of one of the C ABI's types, as a double
__device__ __forceinline__ double load_any(const void *p, int dtype, int64_t i)
{
    switch (dtype) {
    case CLG_F64: return static_cast<const double *>(p)[i];
    case CLG_F16: return (double)(float)static_cast<const _Float16 *>(p)[i];
    case CLG_BF16: return (double)(float)static_cast<const __bf16 *>(p)[i];
    default: return (double)static_cast<const float *>(p)[i];
    }
}

#endif  // __HIPCC__

static inline bool clg_score_type(int dtype) { return dtype == CLG_F32 || dtype == CLG_F64 || dtype == CLG_F16 || dtype == CLG_BF16; }
static inline int clg_elem_bytes(int dtype) { return dtype == CLG_F64 ? 8 : dtype == CLG_F32 ? 4 : 2; }

// call(T()) with the element type of a dtype code that clg_score_type has checked
template <typename F>
static inline int clg_with_type(int dtype, F call)
{
    switch (dtype) {
    case CLG_F64: return call(double());
    case CLG_F16: return call((_Float16)0);
    case CLG_BF16: return call((__bf16)0);
    default: return call(float());
    }
}
