// The sum of a loss over rows, in a fixed order: of all rows by one workgroup, or of kSlice to a workgroup first.  (One workgroup: 3 us for 10000 rows, 6 for
// 40000, 9 for 65536, of loads that wait; in slices 5 for 65537, two launches.)
#pragma once

#include "row_tile.h"

namespace {

constexpr int kSlice = 16384;

#if defined(__HIPCC__)
__device__ __forceinline__ double sum_of(const double *v, int64_t n, double *room)
{
    double s[1] = {0};
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < n; i += 1024) s[0] += v[i];
    block_reduce<true, 1024>(s, room);
    return s[0];
}
__global__ __launch_bounds__(1024) void sum_slices_kernel(const double *row_loss, int64_t rows, double *slices)
{
    __shared__ double room[16];
    const int64_t first = (int64_t)blockIdx.x * kSlice;
    const double s = sum_of(row_loss + first, rows - first < kSlice ? rows - first : kSlice, room);
    if (threadIdx.x == 0) slices[blockIdx.x] = s;
}
template <typename A>
__global__ __launch_bounds__(1024) void sum_rows_kernel(const double *row_loss, int64_t rows, const double *per_count, A *out)
{
    __shared__ double room[16];
    const double s = sum_of(row_loss, rows, room);
    if (threadIdx.x == 0) *out = (A)(s * (per_count ? *per_count : 1));
}

// *loss (of the type that dtype's sums are held in) = the rows' losses, times *per_count where that is not NULL; slices: a value for every kSlice rows
inline int sum_rows(const char *name, int dtype, const double *row_loss, int64_t rows, double *slices, const double *per_count, void *loss, hipStream_t stream)
{
    int64_t n = rows;
    if (rows > 4 * kSlice) {
        n = clg_ceil_div(rows, kSlice);
        sum_slices_kernel<<<dim3((unsigned)n), dim3(1024), 0, stream>>>(row_loss, rows, slices);
        CLG_CHECK_LAUNCH(name);
        row_loss = slices;
    }
    if (dtype == CLG_F64) sum_rows_kernel<double><<<dim3(1), dim3(1024), 0, stream>>>(row_loss, n, per_count, static_cast<double *>(loss));
    else sum_rows_kernel<float><<<dim3(1), dim3(1024), 0, stream>>>(row_loss, n, per_count, static_cast<float *>(loss));
    CLG_CHECK_LAUNCH(name);
    return CLG_OK;
}
#endif

}  // namespace
