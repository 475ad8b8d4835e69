// Activations in 8 bits.  Of 128 elements with the lowest value l and the highest h, element x becomes the code rint((x - l) 255 / (h - l)) and stands for
// l + code * step, step = (h - l) / 255: off by at most step / 2 and the rounding of l + code * step.  The codes are those of 64-bit arithmetic, in which
// (x - l) 255 is exact for 32-bit elements of like magnitude, so that a half is a half.
#include "activation_codes.h"

namespace {

// Bound by memory: 1 GiB of float32 in 222 us, 6.1 TB/s of reads and writes (a copy of 1 GiB 5.1), of bfloat16 in 340.  (Loads past the caches: 232, and 9 us
// more for 128 MiB, which other kernels have just left there.)
template <typename T>
__global__ __launch_bounds__(256) void encode_kernel(const T *__restrict__ x, int64_t n, uint8_t *__restrict__ codes,
                                                   CodeScale<typename Wide<T>::type> *__restrict__ scales)
{
    encode_groups(x, n, codes, scales, (int64_t)blockIdx.x * (256 / kCodeLanes) + threadIdx.x / kCodeLanes, (int64_t)gridDim.x * (256 / kCodeLanes));
}

// 1 GiB of float32 in 253 us, 5.4 TB/s of reads and writes, of bfloat16 in 286.
template <typename T>
__global__ __launch_bounds__(256) void decode_kernel(const uint8_t *__restrict__ codes, const CodeScale<typename Wide<T>::type> *__restrict__ scales, int64_t n,
                                                   T *__restrict__ x)
{
    typedef typename Wide<T>::type A;
    typedef typename EightOf<T>::V V;
    const int lane = threadIdx.x % kCodeLanes;
    const int64_t groups = (n + kCodeGroup - 1) / kCodeGroup;
    for (int64_t g = (int64_t)blockIdx.x * (256 / kCodeLanes) + threadIdx.x / kCodeLanes; g < groups; g += (int64_t)gridDim.x * (256 / kCodeLanes)) {
        const int64_t at = g * kCodeGroup + lane * kCodeEach;
        const CodeScale<A> s = scales[g];
        if ((g + 1) * kCodeGroup <= n) {
            const u32x2 c = *reinterpret_cast<const u32x2 *>(codes + at);
#pragma unroll
            for (int p = 0; p < EightOf<T>::PIECES; ++p) {
                V u;
#pragma unroll
                for (int k = 0; k < EightOf<T>::VEC; ++k) {
                    const int i = p * EightOf<T>::VEC + k;
                    u[k] = (T)fma_t((A)((c[i / 4] >> 8 * (i % 4)) & 255u), s.step, s.low);
                }
                *reinterpret_cast<V *>(x + at + p * EightOf<T>::VEC) = u;
            }
        } else {
            for (int k = 0; k < kCodeEach; ++k)
                if (at + k < n) x[at + k] = (T)fma_t((A)codes[at + k], s.step, s.low);
        }
    }
}

dim3 grid_of(int64_t n)
{
    const int64_t blocks = clg_ceil_div(n, 256 / kCodeLanes * kCodeGroup);
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
