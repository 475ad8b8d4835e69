// Activations in 8 bits.  Of 128 elements with the lowest value l and the highest h, element x becomes the code rint((x - l) 255 / (h - l)) and stands for
// l + code * step, step = (h - l) / 255: off by at most step / 2 and the rounding of l + code * step.  The codes are those of 64-bit arithmetic, in which
// (x - l) 255 is exact for 32-bit elements of like magnitude, so that a half is a half.
#include "activation_codes.h"

namespace {

constexpr int kLanes = 16, kEach = kCodeGroup / kLanes;               // a row of DPP has a group, a lane eight elements of it

template <typename T>
struct Eight {                                                        // as they lie in memory, at any element's address
    static constexpr int VEC = Vec16<T>::N < kEach ? Vec16<T>::N : kEach, PIECES = kEach / VEC;
    typedef typename Vec16<T>::type V;
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

// Bound by memory: 1 GiB of float32 in 222 us, 6.1 TB/s of reads and writes (a copy of 1 GiB 5.1), of bfloat16 in 300.  (Loads past the caches: 232, and 9 us
// more for 128 MiB, which other kernels have just left there.)
template <typename T>
__global__ __launch_bounds__(256) void encode_kernel(const T *__restrict__ x, int64_t n, uint8_t *__restrict__ codes,
                                                   CodeScale<typename Wide<T>::type> *__restrict__ scales)
{
    typedef typename Wide<T>::type A;
    typedef typename Eight<T>::V V;
    const int lane = threadIdx.x % kLanes;
    const int64_t groups = (n + kCodeGroup - 1) / kCodeGroup;
    for (int64_t g = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes; g < groups; g += (int64_t)gridDim.x * (256 / kLanes)) {
        const int64_t at = g * kCodeGroup + lane * kEach;
        const bool whole = (g + 1) * kCodeGroup <= n;
        A v[kEach];
        if (whole) {
#pragma unroll
            for (int p = 0; p < Eight<T>::PIECES; ++p) {
                const V u = *reinterpret_cast<const V *>(x + at + p * Eight<T>::VEC);
#pragma unroll
                for (int k = 0; k < Eight<T>::VEC; ++k) v[p * Eight<T>::VEC + k] = (A)u[k];
            }
        } else {                                                      // (what is missing is as the last element)
#pragma unroll
            for (int k = 0; k < kEach; ++k) v[k] = (A)x[at + k < n ? at + k : n - 1];
        }
        A low = v[0], high = v[0];                                    // (NaN is passed over, and found by the coder)
#pragma unroll
        for (int k = 1; k < kEach; ++k) low = min_of(low, v[k]), high = max_of(high, v[k]);
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
            for (int k = 0; k < kEach; ++k)
                if (at + k < n) codes[at + k] = (uint8_t)(c[k / 4] >> 8 * (k % 4));
        }
        if (lane == 0) {
            double step = code.size * (1 / 255.0);                    // (code.size / 255, without a division)
            step = __builtin_fma(__builtin_fma(-step, 255.0, code.size), 1 / 255.0, step);
            CodeScale<A> s = {low, (A)step};
            // (the highest code may not stand for infinity)
            if (!(__builtin_fabs((double)(A)__builtin_fma(255.0, (double)s.step, (double)low)) <= __DBL_MAX__)) s.step = s.step * (A)(1 - 0x1p-23);
            if (bad) s.low = s.step = (A)__builtin_nanf("");
            scales[g] = s;
        }
    }
}

// 1 GiB of float32 in 253 us, 5.4 TB/s of reads and writes, of bfloat16 in 286.
template <typename T>
__global__ __launch_bounds__(256) void decode_kernel(const uint8_t *__restrict__ codes, const CodeScale<typename Wide<T>::type> *__restrict__ scales, int64_t n,
                                                   T *__restrict__ x)
{
    typedef typename Wide<T>::type A;
    typedef typename Eight<T>::V V;
    const int lane = threadIdx.x % kLanes;
    const int64_t groups = (n + kCodeGroup - 1) / kCodeGroup;
    for (int64_t g = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes; g < groups; g += (int64_t)gridDim.x * (256 / kLanes)) {
        const int64_t at = g * kCodeGroup + lane * kEach;
        const CodeScale<A> s = scales[g];
        if ((g + 1) * kCodeGroup <= n) {
            const u32x2 c = *reinterpret_cast<const u32x2 *>(codes + at);
#pragma unroll
            for (int p = 0; p < Eight<T>::PIECES; ++p) {
                V u;
#pragma unroll
                for (int k = 0; k < Eight<T>::VEC; ++k) {
                    const int i = p * Eight<T>::VEC + k;
                    u[k] = (T)fma_t((A)((c[i / 4] >> 8 * (i % 4)) & 255u), s.step, s.low);
                }
                *reinterpret_cast<V *>(x + at + p * Eight<T>::VEC) = u;
            }
        } else {
            for (int k = 0; k < kEach; ++k)
                if (at + k < n) x[at + k] = (T)fma_t((A)codes[at + k], s.step, s.low);
        }
    }
}

dim3 grid_of(int64_t n)
{
    const int64_t blocks = clg_ceil_div(n, 256 / kLanes * kCodeGroup);
    return dim3((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
}

int check_codes(const char *name, int dtype, const void *x, const void *codes, const void *scales, int64_t n)
{
    CLG_REQUIRE(clg_score_type(dtype), "%s: dtype must be CLG_F32, CLG_F64, CLG_F16 or CLG_BF16, got %d", name, dtype);
    CLG_REQUIRE(n >= 0, "%s: negative number of elements", name);
    CLG_REQUIRE(!n || (x && codes && scales), "%s: null pointer", name);
    CLG_REQUIRE(reinterpret_cast<uintptr_t>(codes) % 8 == 0 && reinterpret_cast<uintptr_t>(scales) % 16 == 0, "%s: codes must be aligned to 8 bytes, scales to 16",
                name);
    return CLG_OK;
}

}  // namespace

extern "C" int64_t clg_codes_groups(int64_t n) { return n <= 0 ? 0 : clg_ceil_div(n, kCodeGroup); }

extern "C" int clg_codes_encode(int dtype, const void *x, int64_t n, uint8_t *codes, void *scales, void *stream)
{
    if (const int rc = check_codes("clg_codes_encode", dtype, x, codes, scales, n)) return rc;
    if (!n) return CLG_OK;
    const int rc = clg_with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        auto *s = static_cast<CodeScale<typename Wide<T>::type> *>(scales);
        encode_kernel<T><<<grid_of(n), dim3(256), 0, clg_stream(stream)>>>(static_cast<const T *>(x), n, codes, s);
        return CLG_OK;
    });
    if (rc) return rc;
    CLG_CHECK_LAUNCH("clg_codes_encode");
    return CLG_OK;
}

extern "C" int clg_codes_decode(int dtype, const uint8_t *codes, const void *scales, int64_t n, void *x, void *stream)
{
    if (const int rc = check_codes("clg_codes_decode", dtype, x, codes, scales, n)) return rc;
    if (!n) return CLG_OK;
    const int rc = clg_with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        const auto *s = static_cast<const CodeScale<typename Wide<T>::type> *>(scales);
        decode_kernel<T><<<grid_of(n), dim3(256), 0, clg_stream(stream)>>>(codes, s, n, static_cast<T *>(x));
        return CLG_OK;
    });
    if (rc) return rc;
    CLG_CHECK_LAUNCH("clg_codes_decode");
    return CLG_OK;
}
