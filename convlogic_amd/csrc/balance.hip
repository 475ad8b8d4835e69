// How evenly rows choose among experts: with p = softmax(z) of a row's logits over E experts, the k highest of each row chosen (of equal ones the lowest),
// c_e rows that chose expert e and n rows in all,
//     loss = E / (k n^2) sum_e c_e sum_t p_te,        d loss / d z_ti = p_ti (w_i - sum_e w_e p_te),        w_e = E c_e / (k n^2)
// (1 where the experts are chosen equally; the choice itself has no gradient).  The gates of a neuron are 16 experts of which it takes one: several tensors
// of logits, a network's layers, go in one launch, each with a loss of its own, of which the mean is taken.
#include <type_traits>

#include "row_tile.h"

namespace {

constexpr int kSegments = 16, kThreads = 256, kMaxExperts = 1024, kEach = 16;

// Logits from so many MB on are read past the caches, gradients written so: smaller ones are still in the last-level cache when the backward pass
// reads them again (131072 rows of 256 experts, 134 MB: 81 us a step through the caches, 87 past them; the gates of 79 M logits, 316 MB: 201 and 179).
constexpr int kPastMb = 192;

struct Segments {
    const void *z[kSegments];
    void *grad[kSegments];
    int64_t rows[kSegments], stride[kSegments];
    int first[kSegments + 1];                                         // workgroups first[i] .. first[i + 1] - 1 take segment i
    int n;
};

struct BalanceArgs {
    Segments seg;
    int experts, k;
    const uint8_t *mask;                                              // of the only segment, or NULL
    float *sums;                                                      // [workgroups][experts] sums of probabilities
    int *counts;                                                      // [workgroups][experts + 1] rows per expert, rows in all
    int *ticket;                                                      // 0 for the launch behind
    const void *w;                                                    // [segments][experts] in A
    const void *upstream;                                             // A
};

// Reductions over groups of G lanes, in all of them: up to 16 lanes by DPP, beyond by LDS permutation.
template <int CTRL>
__device__ __forceinline__ int of_lanes(int v)                        // (every lane has a source: one instruction with what takes the value)
{
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ uint32_t of_lanes(uint32_t v)
{
    return (uint32_t)of_lanes<CTRL>((int)v);
}
template <int CTRL>
__device__ __forceinline__ float of_lanes(float v)
{
    return __builtin_bit_cast(float, of_lanes<CTRL>(__builtin_bit_cast(int, v)));
}
template <int CTRL>
__device__ __forceinline__ double of_lanes(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)of_lanes<CTRL>((int)(uint32_t)u), hi = (uint32_t)of_lanes<CTRL>((int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
template <int G, typename A, typename F>
__device__ __forceinline__ A group_reduce(A v, F f)
{
    if constexpr (G > 1) v = f(v, of_lanes<0xB1>(v));                 // quad_perm [1,0,3,2]
    if constexpr (G > 2) v = f(v, of_lanes<0x4E>(v));                 // quad_perm [2,3,0,1]
    if constexpr (G > 4) v = f(v, of_lanes<0x141>(v));                // row_half_mirror
    if constexpr (G > 8) v = f(v, of_lanes<0x140>(v));                // row_mirror
    if constexpr (G > 16) v = f(v, (A)__shfl_xor(v, 16));
    if constexpr (G > 32) v = f(v, (A)__shfl_xor(v, 32));
    return v;
}
struct Max {
    template <typename A>
    __device__ __forceinline__ A operator()(A a, A b) const { return max_of(a, b); }
};
struct Sum {
    template <typename A>
    __device__ __forceinline__ A operator()(A a, A b) const { return a + b; }
};

// the logits of a row that a lane holds: pieces lane, lane + G, ... of 16 bytes; -inf behind the row
template <typename T, int G, int NV, bool STREAM>
struct RowPart {
    typedef typename Wide<T>::type A;
    static constexpr int VEC = Vec16<T>::N, N = NV * VEC, kLanes = G;
    A x[N];
    __device__ __forceinline__ static int expert(int lane, int i) { return ((i / VEC) * G + lane) * VEC + i % VEC; }
    __device__ __forceinline__ void load(const T *row, int lane, int experts)
    {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = (j * G + lane) * VEC;
            if (e + VEC <= experts) {
                const auto v = load_vec<STREAM>(reinterpret_cast<const typename Vec16<T>::type *>(row + e));
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[j * VEC + i] = (A)v[i];
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) x[j * VEC + i] = e + i < experts ? (A)row[e + i] : lowest(A(0));
            }
        }
    }
    __device__ __forceinline__ A highest() const
    {
        A m = x[0];
#pragma unroll
        for (int i = 1; i < N; ++i) m = max_of(m, x[i]);
        return group_reduce<G>(m, Max());
    }
    // e = exponentials relative to the row's highest, m -> their sum: 0 for a row of -inf alone, NaN for one with a NaN
    __device__ __forceinline__ A exponentials(A m, A (&e)[N]) const
    {
        const Exps<A> f(m, (A)Exps<A>::unit(1.0));
        A s = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            e[i] = f(x[i]);
            s += e[i];
        }
        return group_reduce<G>(s, Sum());
    }
};

__device__ __forceinline__ int segment_of(const Segments &s)
{
    int at = 0;
    for (int i = 1; i < s.n; ++i) at += (int)blockIdx.x >= s.first[i];
    return at;
}

// Rows that a group of lanes has in flight.  Sums alone, as here and with one: 1 M rows of 16 float32 24 and 27 us, 65536 of 64 bfloat16 21 and 21, 131072 of 256 float32
// 38 and 38; but 20000 of 60 float32 19 and 15, of 100 float64 26 and 21, where a group has few rows.
template <int N>
constexpr int kAhead = N <= 4 ? 4 : N <= 8 ? 2 : 1;

// (off by one step of its type at most, as the exponentials are)
__device__ __forceinline__ float reciprocal(float v) { return __builtin_amdgcn_rcpf(v); }
__device__ __forceinline__ double reciprocal(double v) { return 1.0 / v; }

// the choice of one row, one expert at a time: the lowest of the highest that are left
template <typename Part, int N>
__device__ __forceinline__ void choose(Part &part, int lane, int k, int (&c)[N])
{
    typedef typename Part::A A;
    const A none = lowest(A(0));
#pragma unroll
    for (int i = 0; i < N; ++i) part.x[i] = part.x[i] != part.x[i] ? -none : part.x[i];
#pragma unroll 1
    for (int pick = 0; pick < k; ++pick) {
        const A top = part.highest();
        if (top == none) break;
        int which = kMaxExperts;
#pragma unroll
        for (int i = N - 1; i >= 0; --i) which = part.x[i] == top ? Part::expert(lane, i) : which;
        which = group_reduce<Part::kLanes>(which, [](int u, int v) { return u < v ? u : v; });
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const bool it = Part::expert(lane, i) == which;
            c[i] += it;
            part.x[i] = it ? none : part.x[i];
        }
    }
}

// order of a 16-bit logit, then of its expert, from the lowest; 0 for -inf, as +inf for NaN (and so never ~0)
__device__ __forceinline__ uint32_t choice_key(float x, int expert)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f), ordered = x != x ? 0xFF800000u : u ^ (u >> 31 ? ~0u : 0x80000000u);
    return x == lowest(0.f) ? 0 : (ordered & ~0x1FFFu) | (uint32_t)(0x1FFF - expert);
}
__device__ __forceinline__ uint32_t choice_key(double, int) { return 0; }                // (not of this type)

// Sums and counts of a workgroup's rows.  131072 rows of 256 experts: 25 us with the logits in the last-level cache, 39 without; 79 M gate logits 60 us, 5.2 TB/s;
// 65536 rows of 64 bfloat16 experts of which 8 are chosen 11 us, of vector instructions (69 to 75 % of the time in all three).
template <typename T, int G, int NV, bool STREAM>
__global__ __launch_bounds__(kThreads) void balance_kernel(BalanceArgs a)
{
    typedef RowPart<T, G, NV, STREAM> Part;
    typedef typename Part::A A;
    constexpr int N = Part::N, kGroups = kThreads / G, R = kAhead<N>;
    __shared__ A room_p[kThreads / 64][G * N];
    __shared__ int room_c[kThreads / 64][G * N + 1];
    const int tid = threadIdx.x, lane = tid % G, seg = segment_of(a.seg);
    const int64_t rows = a.seg.rows[seg], groups = (int64_t)(a.seg.first[seg + 1] - a.seg.first[seg]) * kGroups;
    const T *z = static_cast<const T *>(a.seg.z[seg]);
    A p[N] = {};
    int c[N] = {}, n = 0;
    for (int64_t row0 = (int64_t)((int)blockIdx.x - a.seg.first[seg]) * kGroups + tid / G; row0 < rows; row0 += R * groups) {
        Part part[R];
        bool kept[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + r * groups;
            kept[r] = row < rows && !(a.mask && !a.mask[row]);
            part[r].load(z + (kept[r] ? row : row0) * a.seg.stride[seg], lane, a.experts);
        }
        // (rows that do not count go the same way with a weight of 0: the steps of R rows fill one another's waits)
        A m[R], e[R][N], s[R];
        bool odd = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
            for (int i = 0; i < N; ++i) part[r].x[i] = kept[r] ? part[r].x[i] : A(0);
            m[r] = part[r].highest();
        }
#pragma unroll
        for (int r = 0; r < R; ++r) s[r] = part[r].exponentials(m[r], e[r]);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            kept[r] = kept[r] && !(s[r] == 0);
            n += kept[r];
        }
        if constexpr (sizeof(T) == 2) {
            // The choice of 16-bit logits, of which many are equal: the k highest keys of a logit's order and, in the bits that a float32 of it does not use,
            // the expert.  No two are equal; -inf has none.
            uint32_t key[R][N], least[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                least[r] = ~0u;
#pragma unroll
                for (int i = 0; i < N; ++i) key[r][i] = choice_key(part[r].x[i], Part::expert(lane, i));
            }
#pragma unroll 1
            for (int pick = 0; pick < a.k; ++pick)
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    uint32_t next = 0;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const uint32_t below = key[r][i] < least[r] ? key[r][i] : 0;
                        next = below > next ? below : next;
                    }
                    least[r] = group_reduce<G>(next, [](uint32_t u, uint32_t v) { return u > v ? u : v; });
                }
#pragma unroll
            for (int r = 0; r < R; ++r) {
                least[r] = least[r] == 0 ? 1 : least[r];
#pragma unroll
                for (int i = 0; i < N; ++i) c[i] += kept[r] && key[r][i] >= least[r];
            }
        } else {
            // The choice: k times the highest below the last one.  -inf is none, NaN is above everything.  Where values are equal, or too few are there,
            // these are too many or too few experts, and the slow way takes one at a time, the lowest of the highest.
            A least[R];
#pragma unroll
            for (int r = 0; r < R; ++r) {
                least[r] = m[r];
                odd |= s[r] != s[r];
            }
#pragma unroll 1
            for (int pick = 1; pick < a.k; ++pick) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    A next = lowest(A(0));
#pragma unroll
                    for (int i = 0; i < N; ++i) next = max_of(next, part[r].x[i] < least[r] ? part[r].x[i] : lowest(A(0)));
                    least[r] = group_reduce<G>(next, Max());
                }
            }
            int want = 0, have = 0;                                   // of the wavefront
#pragma unroll
            for (int r = 0; r < R; ++r) {
                odd |= kept[r] && least[r] == lowest(A(0));
                want += __popcll(__ballot(kept[r]));
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const bool it = kept[r] && part[r].x[i] >= least[r];
                    have += __popcll(__ballot(it));
                    c[i] += it;
                }
            }
            if (__any(odd) || have * G != want * a.k) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
#pragma unroll
                    for (int i = 0; i < N; ++i) c[i] -= kept[r] && part[r].x[i] >= least[r];
                    if (kept[r]) choose(part[r], lane, a.k, c);
                }
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const A inv = kept[r] ? reciprocal(s[r]) : A(0);
#pragma unroll
            for (int i = 0; i < N; ++i) p[i] += e[r][i] * inv;
        }
    }
    // groups of a wavefront, then its four wavefronts, in a fixed order
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int by = G; by < 64; by <<= 1) {
            p[i] += __shfl_xor(p[i], by);
            c[i] += __shfl_xor(c[i], by);
        }
#pragma unroll
    for (int by = G; by < 64; by <<= 1) n += __shfl_xor(n, by);
    if ((tid & 63) < G) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            room_p[tid >> 6][Part::expert(lane, i)] = p[i];
            room_c[tid >> 6][Part::expert(lane, i)] = c[i];
        }
        if (lane == 0) room_c[tid >> 6][G * N] = n;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) *a.ticket = 0;
    A *sums = reinterpret_cast<A *>(a.sums) + (int64_t)blockIdx.x * a.experts;
    int *counts = a.counts + (int64_t)blockIdx.x * (a.experts + 1);
    for (int e = tid; e <= a.experts; e += kThreads) {
        const int s = e < a.experts ? e : G * N;
        int cc = 0;
        A pp = 0;
        for (int w = 0; w < kThreads / 64; ++w) {
            cc += room_c[w][s];
            if (e < a.experts) pp += room_p[w][s];
        }
        counts[e] = cc;
        if (e < a.experts) sums[e] = pp;
    }
}

struct FinishArgs {
    Segments seg;
    int experts, k;
    const void *sums;
    const int *counts;
    double weight;
    void *loss, *w;                                                   // A, [segments][experts] in A
    int64_t *count_out;                                               // [segments][experts]
    double *terms;                                                    // [segments][blocks of experts]
    int *ticket;
};

// One workgroup per 16 experts of a segment, 64 slices of its workgroups' sums at once: rows per expert and in all, the coefficients of the gradient and
// these experts' part of the loss.  The workgroup that is done last adds the parts up, in their order.  4.5 to 9 us: loads that wait.  (64 experts to a workgroup: 10 us in place of 5 for
// the 512 KB of sums of 64 experts.)
template <typename A>
__global__ __launch_bounds__(1024) void balance_finish_kernel(FinishArgs a)
{
    constexpr int EACH = kEach, SLICES = 1024 / EACH;
    __shared__ double room[16], sum_p[1024];
    __shared__ int64_t sum_c[1024];
    const int seg = blockIdx.y, tid = threadIdx.x, first = a.seg.first[seg], end = a.seg.first[seg + 1];
    const int e = (int)blockIdx.x * EACH + tid % EACH;
    double n[1] = {0};
    for (int w = first + tid; w < end; w += 1024) n[0] += a.counts[(int64_t)w * (a.experts + 1) + a.experts];
    double p = 0;
    int64_t c = 0;
    if (e < a.experts) {
        for (int w0 = first + tid / EACH; w0 < end; w0 += 8 * SLICES) {       // (eight rows of sums on their way at once)
            A p8[8];
            int c8[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int w = w0 + u * SLICES < end ? w0 + u * SLICES : w0;
                p8[u] = static_cast<const A *>(a.sums)[(int64_t)w * a.experts + e];
                c8[u] = a.counts[(int64_t)w * (a.experts + 1) + e];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const bool there = w0 + u * SLICES < end;
                p += there ? (double)p8[u] : 0.0;
                c += there ? c8[u] : 0;
            }
        }
    }
    sum_p[tid] = p;
    sum_c[tid] = c;
    block_reduce<true, 1024>(n, room);
    if (tid >= kWave) return;
    // the first wavefront: 64 / EACH parts of the slices, then these
    p = 0, c = 0;
    for (int s = tid / EACH; s < SLICES; s += kWave / EACH) {
        p += sum_p[s * EACH + tid % EACH];
        c += sum_c[s * EACH + tid % EACH];
    }
#pragma unroll
    for (int by = EACH; by < kWave; by <<= 1) {
        p += __shfl_xor(p, by);
        c += __shfl_xor(c, by);
    }
    double term = 0;
    if (tid < EACH && e < a.experts) {
        const double w = n[0] == 0 ? 0 : a.weight * a.experts * (double)c / ((double)a.k * n[0] * n[0]);
        a.count_out[(int64_t)seg * a.experts + e] = c;
        static_cast<A *>(a.w)[(int64_t)seg * a.experts + e] = (A)w;
        term = w * p;
    }
    term = wave_sum(term);
    const int blocks = gridDim.x * gridDim.y;
    if (blocks > 1) {
        int mine = 0;
        if (tid == 0) {
            __hip_atomic_store(a.terms + seg * gridDim.x + blockIdx.x, term, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            mine = __hip_atomic_fetch_add(a.ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        }
        if (__builtin_amdgcn_readfirstlane(mine) != blocks - 1) return;
        term = 0;
        for (int i = tid; i < blocks; i += kWave) term += __hip_atomic_load(a.terms + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        term = wave_sum(term);
    }
    if (tid == 0) *static_cast<A *>(a.loss) = (A)term;
}

// The gradient, from a second pass over the logits (the coefficients need the counts of every row): 79 M gate logits 112 us, 5.6 TB/s read and written;
// 131072 rows of 256 experts 43 us, 6.2 TB/s with the logits from the last-level cache.
template <typename T, int G, int NV, bool STREAM>
__global__ __launch_bounds__(kThreads) void balance_grad_kernel(BalanceArgs a)
{
    typedef RowPart<T, G, NV, STREAM> Part;
    typedef typename Part::A A;
    typedef typename Vec16<T>::type V;
    constexpr int N = Part::N, VEC = Part::VEC, kGroups = kThreads / G, R = kAhead<N>;
    const int tid = threadIdx.x, lane = tid % G, seg = segment_of(a.seg);
    const int64_t rows = a.seg.rows[seg], groups = (int64_t)(a.seg.first[seg + 1] - a.seg.first[seg]) * kGroups;
    const T *z = static_cast<const T *>(a.seg.z[seg]);
    T *grad = static_cast<T *>(a.seg.grad[seg]);
    const A up = *static_cast<const A *>(a.upstream);
    A w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = Part::expert(lane, i);
        w[i] = e < a.experts ? static_cast<const A *>(a.w)[(int64_t)seg * a.experts + e] : A(0);
    }
    for (int64_t row0 = (int64_t)((int)blockIdx.x - a.seg.first[seg]) * kGroups + tid / G; row0 < rows; row0 += R * groups) {
        Part part[R];
        bool kept[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + r * groups;
            kept[r] = row < rows && !(a.mask && !a.mask[row]);
            if (kept[r]) part[r].load(z + row * a.seg.stride[seg], lane, a.experts);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int64_t row = row0 + r * groups;
            if (row >= rows) break;
            A e[N], inv = 0, mean = 0;
            if (kept[r]) {
                const A s = part[r].exponentials(part[r].highest(), e);
                kept[r] = !(s == 0);
                inv = reciprocal(s);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    e[i] *= inv;
                    mean += w[i] * e[i];
                }
                mean = group_reduce<G>(mean, Sum());
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int at = (j * G + lane) * VEC;
                V v;
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] = kept[r] ? (T)(e[j * VEC + i] * (w[j * VEC + i] - mean) * up) : (T)0.f;
                T *out = grad + row * a.experts + at;
                if (at + VEC <= a.experts) {
                    store_vec<STREAM>(reinterpret_cast<V *>(out), v);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i)
                        if (at + i < a.experts) out[i] = v[i];
                }
            }
        }
    }
}

// call(lanes per row, pieces per lane) for a number of experts
template <typename T, typename F>
void with_part(int experts, F call)
{
    const int pieces = (experts + Vec16<T>::N - 1) / Vec16<T>::N;
    if (pieces <= 1) return call(std::integral_constant<int, 1>(), std::integral_constant<int, 1>());
    if (pieces <= 2) return call(std::integral_constant<int, 2>(), std::integral_constant<int, 1>());
    if (pieces <= 4) return call(std::integral_constant<int, 4>(), std::integral_constant<int, 1>());
    if (pieces <= 8) return call(std::integral_constant<int, 8>(), std::integral_constant<int, 1>());
    if (pieces <= 16) return call(std::integral_constant<int, 16>(), std::integral_constant<int, 1>());
    if (pieces <= 32) return call(std::integral_constant<int, 16>(), std::integral_constant<int, 2>());
    if (pieces <= 64) return call(std::integral_constant<int, 16>(), std::integral_constant<int, 4>());
    if (pieces <= 128) return call(std::integral_constant<int, 64>(), std::integral_constant<int, 2>());
    call(std::integral_constant<int, 64>(), std::integral_constant<int, (kMaxExperts / 64 / Vec16<T>::N > 2 ? kMaxExperts / 64 / Vec16<T>::N : 2)>());
}

template <typename T>
int lanes_of(int experts)
{
    int g = 0;
    with_part<T>(experts, [&](auto lanes, auto) { g = decltype(lanes)::value; });
    return g;
}

constexpr int kTerms = kSegments * (kMaxExperts / kEach);               // of the loss
// Workgroups of the sums: 1 M rows of 16 float32 26, 24 and 26 us by 512, 1024 and 2048, 131072 of 256 40, 38 and 46, 20000 of 1000 41, 36 and 43; 65536 of 64
// bfloat16 19, 21 and 32, 200000 of 8 11, 15 and 14, where adding 1024 of them up is a good part.
constexpr int kMostGroups = 1024;

// workgroups per segment, `most` in all or a few more: by rows, one at least
int64_t share_out(Segments &s, int64_t per_group, int64_t most)
{
    int64_t total = 0;
    for (int i = 0; i < s.n; ++i) total += s.rows[i];
    int64_t at = 0;
    for (int i = 0; i < s.n; ++i) {
        s.first[i] = (int)at;
        const int64_t need = clg_ceil_div(s.rows[i], per_group), fair = total ? (int64_t)((double)most * s.rows[i] / total) : 0;
        at += need < fair ? need : fair < 1 ? 1 : fair;
        if (at == s.first[i]) ++at;
    }
    s.first[s.n] = (int)at;
    return at;
}

int check_segments(const char *name, int dtype, int n, const void *const *logits, const int64_t *rows, const int64_t *strides, int64_t experts, int64_t k,
                   const uint8_t *mask, Segments &s)
{
    CLG_REQUIRE(clg_score_type(dtype), "%s: unsupported dtype %d", name, dtype);
    CLG_REQUIRE(n >= 1 && n <= kSegments && logits && rows && strides, "%s: 1 to %d tensors, got %d", name, kSegments, n);
    CLG_REQUIRE(experts >= 1 && experts <= kMaxExperts, "%s: 1 to %d experts, got %lld", name, kMaxExperts, (long long)experts);
    CLG_REQUIRE(k >= 1 && k <= experts, "%s: a row chooses 1 to %lld experts, got %lld", name, (long long)experts, (long long)k);
    CLG_REQUIRE(!mask || n == 1, "%s: a mask is of one tensor", name);
    s.n = n;
    for (int i = 0; i < n; ++i) {
        CLG_REQUIRE(rows[i] >= 0 && rows[i] < (int64_t)1 << 31, "%s: %lld rows", name, (long long)rows[i]);
        CLG_REQUIRE(logits[i] || !rows[i], "%s: null pointer", name);
        CLG_REQUIRE(strides[i] >= 0, "%s: negative row stride", name);
        s.z[i] = logits[i], s.rows[i] = rows[i], s.stride[i] = strides[i], s.grad[i] = nullptr;
    }
    return CLG_OK;
}

}  // namespace

extern "C" int64_t clg_balance_scratch_bytes(int dtype, int64_t experts)
{
    if (!clg_score_type(dtype) || experts < 1 || experts > kMaxExperts) return 0;
    const int64_t groups = kMostGroups + kSegments;
    return groups * experts * (dtype == CLG_F64 ? 8 : 4) + groups * (experts + 1) * 4 + kTerms * 8 + 8 + 8;
}

extern "C" int clg_balance_forward(int dtype, int n, const void *const *logits, const int64_t *rows, const int64_t *row_strides, int64_t experts, int64_t k,
                                   const uint8_t *mask, double weight, void *loss, int64_t *counts, void *coefs, void *scratch, void *stream)
{
    BalanceArgs a{};
    if (const int rc = check_segments("clg_balance_forward", dtype, n, logits, rows, row_strides, experts, k, mask, a.seg)) return rc;
    CLG_REQUIRE(loss && counts && coefs && scratch, "clg_balance_forward: null pointer");
    const bool f64 = dtype == CLG_F64;
    double *terms = static_cast<double *>(scratch);
    a.experts = (int)experts, a.k = (int)k, a.mask = mask;
    a.ticket = reinterpret_cast<int *>(terms + kTerms);
    a.sums = reinterpret_cast<float *>(terms + kTerms + 1);
    a.counts = reinterpret_cast<int *>(reinterpret_cast<char *>(a.sums) + (kMostGroups + kSegments) * experts * (f64 ? 8 : 4));
    int64_t elements = 0;
    for (int i = 0; i < n; ++i) elements += rows[i] * experts;
    const int rc = clg_with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        const int64_t grid = share_out(a.seg, kThreads / lanes_of<T>(a.experts), kMostGroups);
        with_part<T>(a.experts, [&](auto g, auto nv) {
            const auto run = [&](auto past) {
                balance_kernel<T, decltype(g)::value, decltype(nv)::value, decltype(past)::value><<<dim3((unsigned)grid), dim3(kThreads), 0, clg_stream(stream)>>>(a);
            };
            if (clg_past_caches(elements * sizeof(T), kPastMb)) run(std::true_type());
            else run(std::false_type());
        });
        return CLG_OK;
    });
    if (rc) return rc;
    CLG_CHECK_LAUNCH("clg_balance_forward");
    const FinishArgs f{a.seg, a.experts, a.k, a.sums, a.counts, weight / n, loss, coefs, counts, terms, a.ticket};
    const dim3 blocks((unsigned)clg_ceil_div(experts, kEach), n);
    if (f64) balance_finish_kernel<double><<<blocks, dim3(1024), 0, clg_stream(stream)>>>(f);
    else balance_finish_kernel<float><<<blocks, dim3(1024), 0, clg_stream(stream)>>>(f);
    CLG_CHECK_LAUNCH("clg_balance_forward");
    return CLG_OK;
}

extern "C" int clg_balance_backward(int dtype, int n, const void *const *logits, const int64_t *rows, const int64_t *row_strides, int64_t experts,
                                    const uint8_t *mask, const void *coefs, const void *upstream, void *const *grads, void *stream)
{
    BalanceArgs a{};
    if (const int rc = check_segments("clg_balance_backward", dtype, n, logits, rows, row_strides, experts, 1, mask, a.seg)) return rc;
    CLG_REQUIRE(coefs && upstream && grads, "clg_balance_backward: null pointer");
    for (int i = 0; i < n; ++i) {
        CLG_REQUIRE(grads[i] || !rows[i], "clg_balance_backward: null pointer");
        a.seg.grad[i] = grads[i];
    }
    a.experts = (int)experts, a.mask = mask, a.w = coefs, a.upstream = upstream;
    int64_t elements = 0;
    for (int i = 0; i < n; ++i) elements += rows[i] * experts;
    const int rc = clg_with_type(dtype, [&](auto t) {
        typedef decltype(t) T;
        // (of the gradient: 2048 to 16384 workgroups are within 2 % at all of these sizes)
        const int64_t grid = share_out(a.seg, kThreads / lanes_of<T>(a.experts), 8192);
        with_part<T>(a.experts, [&](auto g, auto nv) {
            const auto run = [&](auto past) {
                balance_grad_kernel<T, decltype(g)::value, decltype(nv)::value, decltype(past)::value><<<dim3((unsigned)grid), dim3(kThreads), 0, clg_stream(stream)>>>(a);
            };
            if (clg_past_caches(elements * sizeof(T), kPastMb)) run(std::true_type());
            else run(std::false_type());
        });
        return CLG_OK;
    });
    if (rc) return rc;
    CLG_CHECK_LAUNCH("clg_balance_backward");
    return CLG_OK;
}
