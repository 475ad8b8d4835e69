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

// a maximum as the sums subtract it: an infinite one is left out, so that rows of -inf sum to 0, rows with +inf to inf and NaN stays NaN
template <typename A>
__device__ __forceinline__ A finite_or_zero(A m)
{
    return __builtin_isinf(m) ? A(0) : m;
}

// Exponentials of z / temperature relative to that of a value m.  Floats: 2^(scale z - at) in one multiply-add and the instruction for 2^x, with
// scale = log2(e) / temperature and at = scale m as it is rounded; residue() is what that rounding moved, in 64 bits, for the few values that are not such
// sums.  It is at most 64 (a factor of 2^64 in every exponential of a row) while |at| < 2^31.  From there on another value than m is at least 2^-24 |m| away,
// its exponential at most 2^-128 of m's: nothing next to it, whatever the scale, which is then the power of two that puts `at` between 2^31 and 2^32, exactly.
template <typename A>
struct Exps;
template <>
struct Exps<float> {
    float scale, at;
    __host__ __device__ static double unit(double temperature) { return 1.4426950408889634074 / temperature; }
    __device__ __forceinline__ Exps(float m, float unit_)
    {
#pragma clang fp contract(off)                                        // (`at` is the rounded product in all that is computed of it)
        m = finite_or_zero(m);
        const float whole = m * unit_;
        const uint32_t power = (uint32_t)(127 + 31 + 127) << 23;          // (2^31 over the power of two in m)
        scale = __builtin_fabsf(whole) < 0x1p31f ? unit_ : __builtin_bit_cast(float, power - (__builtin_bit_cast(uint32_t, m) & 0x7F800000u));
        at = m * scale;
    }
    __device__ __forceinline__ float operator()(float z) const { return __builtin_amdgcn_exp2f(__builtin_fmaf(z, scale, -at)); }
    // the factor that makes a sum relative to this one of one relative to `to`, which is of a value no lower
    __device__ __forceinline__ float factor(const Exps &to) const { return scale == to.scale ? __builtin_amdgcn_exp2f(at - to.at) : 0.f; }
    // natural logarithm of the sum 1 relative to m
    __device__ __forceinline__ double residue(float m) const { return ((double)at - (double)finite_or_zero(m) * (double)scale) * 0.69314718055994530942; }
};
template <>
struct Exps<double> {
    double scale, at;
    __host__ __device__ static double unit(double temperature) { return 1.0 / temperature; }
    __device__ __forceinline__ Exps(double m, double unit_) : scale(unit_), at(finite_or_zero(m)) {}
    __device__ __forceinline__ double operator()(double z) const { return exp((z - at) * scale); }
    __device__ __forceinline__ double factor(const Exps &to) const { return exp((at - to.at) * scale); }
    __device__ __forceinline__ double residue(double) const { return 0.0; }
};
// the sum s of exponentials relative to `from` as one relative to `to` (a sum over -inf alone is 0, or NaN)
template <typename A>
__device__ __forceinline__ A rescaled(A s, A m_from, const Exps<A> &from, const Exps<A> &to)
{
    return m_from == lowest(A(0)) ? s : s * from.factor(to);
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
__device__ __forceinline__ float of_lane(float v, int lane) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane)); }
__device__ __forceinline__ double of_lane(double v, int lane)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
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
    return of_lane(v, 63);
}

// Columns base .. of one row in the registers of a team of LANES threads (a workgroup, or a part of a wavefront): thread t holds the 16-byte pieces t, t +
// LANES, ... and, of what is left of a row behind its last whole piece, one element.  What is behind the row is -inf.  STREAM: loads (1) and stores (2) past the caches.
template <typename T, int LANES, int NV, int STREAM>
struct RowTile {
    static constexpr int VEC = Vec16<T>::N, COLS = LANES * NV * VEC;
    typedef typename Vec16<T>::type V;
    typedef typename Wide<T>::type A;
    V v[NV];
    T last;
    int tid, whole, tail;                                             // of the team; whole pieces in the tile, elements behind them

    __device__ __forceinline__ explicit RowTile(int tid_) : tid(tid_) {}

    __device__ __forceinline__ void load(const T *__restrict__ row, int64_t base, int64_t cols)
    {
        const int n = (int)(cols - base < COLS ? cols - base : COLS);
        whole = n / VEC;
        tail = n % VEC;
        const T none = (T)lowest(0.f);
        const T *at = row + base;
        // (all loads before anything waits for one: lanes behind the row read its last piece again, which trim() drops)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int p = j * LANES + tid;
            if (j * LANES < whole) v[j] = load_vec<(STREAM & 1) != 0>(reinterpret_cast<const V *>(reinterpret_cast<const char *>(at) + (uint32_t)(p < whole ? p : whole - 1) * 16u));
            else v[j] = (V)none;
        }
        last = none;
        if (tid < tail) last = at[whole * VEC + tid];
    }
    // the second half of load, which waits for the row
    __device__ __forceinline__ void trim()
    {
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (j * LANES < whole && (j + 1) * LANES > whole && j * LANES + tid >= whole) v[j] = (V)(T)lowest(0.f);
    }
    // keeps the values of the next pass apart from those of the last: both in registers at once would be twice the row
    __device__ __forceinline__ void fence()
    {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            u32x4 r = __builtin_bit_cast(u32x4, v[j]);
            asm volatile("" : "+v"(r));
            v[j] = __builtin_bit_cast(V, r);
        }
        asm volatile("" : "+s"(whole));                               // (compared again rather than kept as a condition per piece)
    }
    // the highest of each piece
    __device__ __forceinline__ void peaks(A (&high)[NV]) const
    {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            high[j] = lowest(A(0));
            if (j * LANES >= whole) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) high[j] = max_of(high[j], (A)v[j][i]);
        }
    }
    // the columns with a bit become -inf
    __device__ __forceinline__ void drop(const uint32_t *bits)
    {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (j * LANES >= whole) break;
            const int c = (j * LANES + tid) * VEC;
            const uint32_t b = bits[c >> 5] >> (c & 31) & ((1u << VEC) - 1);
            if (b)
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (b >> i & 1) v[j][i] = (T)lowest(0.f);
        }
        const int c = whole * VEC + tid;
        if (tid < tail && (bits[c >> 5] >> (c & 31) & 1)) last = (T)lowest(0.f);
    }
    __device__ __forceinline__ A highest() const
    {
        A m = (A)last;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (j * LANES >= whole) break;
#pragma unroll
            for (int i = 0; i < VEC; ++i) m = max_of(m, (A)v[j][i]);
        }
        return m;
    }
    __device__ __forceinline__ A sum(const Exps<A> &e) const
    {
        A s = e((A)last);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (j * LANES >= whole) break;
#pragma unroll
            for (int i = 0; i < VEC; ++i) s += e((A)v[j][i]);
        }
        return s;
    }
    // the same columns of `row` = f(element); f's result is A
    template <typename F>
    __device__ __forceinline__ void store(T *__restrict__ row, int64_t base, F f) const
    {
        T *at = row + base;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int p = j * LANES + tid;
            if (j * LANES >= whole) break;
            V out;
#pragma unroll
            for (int i = 0; i < VEC; ++i) out[i] = (T)f((A)v[j][i]);
            if (p < whole) store_vec<(STREAM & 2) != 0>(reinterpret_cast<V *>(reinterpret_cast<char *>(at) + (uint32_t)p * 16u), out);
        }
        if (tid < tail) at[whole * VEC + tid] = (T)f((A)last);
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
        static_assert(WAVES <= 16, "one row of lanes");
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int c = 0; c < COUNT; ++c) {
            const A r = lane < WAVES ? room[lane * COUNT + c] : SUM ? A(0) : lowest(A(0));
            x[c] = of_lane(SUM ? row16_sum(r) : row16_max(r), 0);
        }
    }
}

// The same for sums of two types at once; `some`, of a wavefront: whether its y are other than 0.
template <int THREADS, int CA, int CB, typename A, typename B>
__device__ __forceinline__ void block_sums(A (&x)[CA], B (&y)[CB], A *room_x, B *room_y, bool some)
{
#pragma unroll
    for (int c = 0; c < CA; ++c) x[c] = wave_sum(x[c]);
    if (some)
#pragma unroll
        for (int c = 0; c < CB; ++c) y[c] = wave_sum(y[c]);
    if constexpr (THREADS > kWave) {
        constexpr int WAVES = THREADS / kWave;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int c = 0; c < CA; ++c) room_x[(threadIdx.x >> 6) * CA + c] = x[c];
#pragma unroll
            for (int c = 0; c < CB; ++c) room_y[(threadIdx.x >> 6) * CB + c] = y[c];
        }
        __syncthreads();
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int c = 0; c < CA; ++c) x[c] = of_lane(row16_sum(lane < WAVES ? room_x[lane * CA + c] : A(0)), 0);
#pragma unroll
        for (int c = 0; c < CB; ++c) y[c] = of_lane(row16_sum(lane < WAVES ? room_y[lane * CB + c] : B(0)), 0);
    }
}

// The team that has a row: a workgroup of THREADS, or LANES = 16 of them, one row of DPP.
template <int THREADS, int LANES>
struct Team {
    static constexpr bool kWhole = THREADS == LANES;
    static_assert(kWhole || LANES == 16, "a workgroup or a row of lanes");
    template <bool SUM, int COUNT, typename A>
    __device__ __forceinline__ static void reduce(A (&x)[COUNT], A *room)
    {
        if constexpr (kWhole) {
            block_reduce<SUM, THREADS>(x, room);
        } else {
#pragma unroll
            for (int c = 0; c < COUNT; ++c) x[c] = SUM ? row16_sum(x[c]) : row16_max(x[c]);
        }
    }
    template <int CA, int CB, typename A>
    __device__ __forceinline__ static void sums(A (&x)[CA], double (&y)[CB], A *room_x, double *room_y, bool some)
    {
        if constexpr (kWhole) {
            block_sums<THREADS>(x, y, room_x, room_y, some);
        } else {
            reduce<true>(x, room_x);
            reduce<true>(y, room_y);
        }
    }
    template <typename A>
    __device__ __forceinline__ static A from(A v, int lane)             // of the team's first wavefront
    {
        if constexpr (kWhole) return of_lane(v, lane);
        else return __shfl(v, lane, 16);
    }
};

// 1 / v, to the last few bits
__device__ __forceinline__ double quick_inverse(double v)
{
    double r = __builtin_amdgcn_rcp(v);
    r = __builtin_fma(__builtin_fma(-v, r, 1.0), r, r);
    return __builtin_fma(__builtin_fma(-v, r, 1.0), r, r);
}

// element i of an array of one of the C ABI's types: its bits, which may still be on their way, and its value
__device__ __forceinline__ uint64_t load_bits(const void *p, int dtype, int64_t i)
{
    switch (dtype) {
    case CLG_F64: return static_cast<const uint64_t *>(p)[i];
    case CLG_F32: return static_cast<const uint32_t *>(p)[i];
    default: return static_cast<const uint16_t *>(p)[i];
    }
}
__device__ __forceinline__ double value_of_bits(uint64_t u, int dtype)
{
    switch (dtype) {
    case CLG_F64: return __builtin_bit_cast(double, u);
    case CLG_F16: return (double)(float)__builtin_bit_cast(_Float16, (uint16_t)u);
    case CLG_BF16: return (double)__builtin_bit_cast(float, (uint32_t)u << 16);
    default: return (double)__builtin_bit_cast(float, (uint32_t)u);
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
