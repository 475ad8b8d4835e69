// Softmax cross entropy of group sums.  A row has k classes of G features each; with the scores s_c = (sum of the class's features) / tau, the highest M, the row's
// target t, O = sum over c != t of exp(s_c - M), Z = O + exp(s_t - M) and the smoothing e:
//     loss = w [ (1 - e) (M - s_t + log Z) + e (log Z + mean_c (M - s_c)) ]
//     d loss / d feature of c = w / tau [ exp(s_c - M) / Z - e / k ],  of t  w / tau [ -O / Z + e - e / k ]
// Where the target is the highest, log Z = log1p(O): with O apart, losses and gradients near 0 keep their digits.  A score is a long sum, and its rounding is a
// relative error of its exponential: sums over features and the differences of scores that exponentials are taken of are in 64 bits, but for rows_kernel's floats.
//
// Rows in memory ("rows", features dense): a workgroup has a row, whose scores stay in LDS from the sums to the gradient, so the features are read once (rows_kernel);
// rows of more classes than LDS holds, or too few rows to fill the chip, go in pieces of the classes, once for the sums and the highest (row_stats_kernel) and once
// more for the gradient (row_grad_kernel).  A feature per row in memory ("columns"): lanes are samples, in pieces of the classes likewise; where a class has few
// features the gradient is from the features again, else from the classes' sums, and large classes in a few of them go in slices (column_stats_kernel joins these).
#include "row_sums.h"

namespace {

// Exponentials of scores, as the sums take them: of differences of classes' sums, which are 64-bit numbers, times `unit` over tau, rounded to A; 2^x by one instruction
// for float.  (Differences before the factor, not after it: the rounding of a product of 10^38 is many powers of two.)
template <typename A>
struct Unit;
template <>
struct Unit<float> {
    static constexpr double unit = 1.4426950408889634074;
    __device__ __forceinline__ static float power(float u) { return __builtin_amdgcn_exp2f(u); }
};
template <>
struct Unit<double> {
    static constexpr double unit = 1.0;
    __device__ __forceinline__ static double power(double u) { return exp(u); }
};

struct CeArgs {
    const void *x;
    void *grad;                                                       // or NULL
    int64_t rows, stride;                                             // stride: from row to row of x ("rows")
    int k, group;
    const void *targets;
    int targets64;
    double inv_tau, smoothing, scale;                                 // scale: weight, over the rows where their number is known to be all
    int reduction, count;                                             // count: to be counted here (1), or in per_count (2)
    double *per_count, *row_loss;                                     // 1 / rows that count; [rows]
    double *final;                                                    // [rows][4]: the highest sum, O, Z
    void *out;                                                        // [rows] in A, or NULL
    const void *upstream;                                             // in A, [rows] for CLG_REDUCE_NONE, or NULL for 1
    int if_changed;                                                   // nothing to do for an upstream gradient of 1
    // pieces
    int pieces, per_piece;                                            // of the classes
    double *stats, *target_sum;                                       // [pieces][rows][4], [rows]
    double *scores, *partial;                                         // "columns": [k][rows], [slices][k][rows], or NULL
    int slices, lanes_log2;                                           // of a class's features; lanes to a class, or samples side by side
};

__device__ __forceinline__ int64_t target_of(const CeArgs &a, int64_t row)
{
    return a.targets64 ? static_cast<const int64_t *>(a.targets)[row] : static_cast<const int32_t *>(a.targets)[row];
}
// behind the last class of the piece that begins with `first`
__device__ __forceinline__ int end_of(const CeArgs &a, int first) { return a.k - first > a.per_piece ? first + a.per_piece : a.k; }
template <typename A>
__device__ __forceinline__ bool nothing_to_do(const CeArgs &a) { return a.if_changed && *static_cast<const A *>(a.upstream) == A(1); }

// 1 / number of rows that count, by the whole workgroup; 1 where it does not matter
template <int THREADS>
__device__ __forceinline__ double per_row(const CeArgs &a, double *room)
{
    if (a.count == 2) return *a.per_count;
    if (a.count == 0) return 1;
    double n[1] = {0};
    for (int64_t i = threadIdx.x; i < a.rows; i += THREADS) n[0] += target_of(a, i) >= 0;
    block_reduce<true, THREADS>(n, room);
    return n[0] == 0 ? 0 : 1 / n[0];
}

// The statistics of a part of a row's classes, of their sums: the highest so far, O and the sum of (highest - sum) relative to it, and the number of
// classes.  Differences are taken in 64 bits before anything is rounded to A: relative to a score that is not the highest -- a masked class's, the first one's --
// those of all others would lose their digits.
template <typename A>
struct Stats {
    double m = lowest(0.0), others = 0, down = 0, n = 0;
    __device__ __forceinline__ void add(double sum, bool is_target, bool smooth, double unit)
    {
        if (sum > m) {
            if (m != lowest(0.0)) {
                others *= (double)Unit<A>::power((A)((m - sum) * unit));
                down += n * (sum - m);
            }
            m = sum;
        }
        const A e = sum == lowest(0.0) ? A(0) : Unit<A>::power((A)((sum - m) * unit));
        others += is_target ? 0.0 : (double)e;
        if (smooth) {
            down += sum == lowest(0.0) ? -lowest(0.0) : m - sum;
            n += 1;
        }
    }
};
// The same of several threads, relative to `m`.
template <typename A>
struct Joint {
    double m = lowest(0.0), others = 0, down = 0, n = 0;
    __device__ __forceinline__ Joint() {}
    __device__ __forceinline__ explicit Joint(const Stats<A> &s) : m(s.m), others(s.others), down(s.down), n(s.n) {}
    __device__ __forceinline__ explicit Joint(const double *p) : m(p[0]), others(p[1]), down(p[2]), n(p[3]) {}
    __device__ __forceinline__ void store(double *p) const { p[0] = m, p[1] = others, p[2] = down, p[3] = n; }
    __device__ __forceinline__ void raise(double to, double unit)
    {
        if (!(to > m)) return;
        if (m != lowest(0.0)) {
            others *= (double)Unit<A>::power((A)((m - to) * unit));
            down += n * (to - m);
        }
        m = to;
    }
    __device__ __forceinline__ void join(Joint b, double unit)
    {
        raise(b.m, unit);
        b.raise(m, unit);
        others += b.others;
        down += b.down;
        n += b.n;
    }
};

// What a row's loss and gradient are made of.
struct Row {
    double others, total;
    // margin: M - s_t, down: sum of M - s_c
    __device__ __forceinline__ double loss(double margin, double down, int k, double smoothing) const
    {
        const double log_total = margin == 0 ? log1p(others) : log(total);
        double l = margin + log_total;
        if (smoothing != 0) l = (1 - smoothing) * l + smoothing * (log_total + down / k);
        return l;
    }
};
// the gradient of class c is e(c) * factor - off, of the target `target`
struct Grad {
    double factor, off, target;
    __device__ __forceinline__ Grad(const Row &r, double scale, double smoothing, int k)
        : factor(scale / r.total), off(scale * smoothing / k), target(scale * (smoothing - smoothing / k - r.others / r.total))
    {
    }
};

// ---- rows in memory ------------------------------------------------------------------------------------------------------------
// (Rows have up to 2^31 - 1 features: indexes do not go beyond the last one, or are differences.)
// The classes of a row by THREADS threads.  PACK != 0: G = PACK features, of which a 16-byte piece holds a whole number of classes; a thread takes
// pieces.  PACK == 0: teams of 1 to 64 lanes take a class each, by pieces of 16 bytes and what is left behind them.
template <typename T, int THREADS, int PACK>
struct Classes {
    static constexpr int E = Vec16<T>::N, EACH = PACK ? E / PACK : 1;
    typedef typename Vec16<T>::type V;
    int group, lanes, lane, team, teams;
    __device__ __forceinline__ Classes(int group_, int lanes_log2)
        : group(group_), lanes(1 << lanes_log2), lane(threadIdx.x & (lanes - 1)), team(threadIdx.x >> lanes_log2), teams(THREADS >> lanes_log2)
    {
    }
    // sum of a class's features, in all lanes of the team
    __device__ __forceinline__ double sum(const T *__restrict__ p) const
    {
        const int pieces = group / E;
        double s = 0;
        int i = lane;
        for (; i + 3 * lanes < pieces; i += 4 * lanes) {
            V v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = reinterpret_cast<const V *>(p)[i + u * lanes];
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
                for (int j = 0; j < E; ++j) s += (double)(typename Wide<T>::type)v[u][j];
        }
        for (; i < pieces; i += lanes) {
            const V v = reinterpret_cast<const V *>(p)[i];
#pragma unroll
            for (int j = 0; j < E; ++j) s += (double)(typename Wide<T>::type)v[j];
        }
        for (i = lane; i < group - pieces * E; i += lanes) s += (double)(typename Wide<T>::type)p[pieces * E + i];
        for (int by = lanes >> 1; by > 0; by >>= 1) s += __shfl_xor(s, by);
        return s;
    }
    // the first N of `count` elements and the last N: all of N to 2 N
    template <int N>
    __device__ __forceinline__ static void fill_twice(T *p, int count, T value)
    {
        typedef T P __attribute__((ext_vector_type(N), aligned(sizeof(T))));
        *reinterpret_cast<P *>(p) = (P)value;
        *reinterpret_cast<P *>(p + count - N) = (P)value;
    }
    // the class's features = value; the end of its last 16 bytes is written along with what is in front of it, with the same
    __device__ __forceinline__ void fill(T *__restrict__ p, T value) const
    {
        const int pieces = group / E;
        if (pieces > 0) {
            for (int i = lane; i < pieces + (group > pieces * E); i += lanes) *reinterpret_cast<V *>(p + (i < pieces ? i * E : group - E)) = (V)value;
            return;
        }
        if (lane != 0) return;
        if constexpr (E >= 4)
            if (group >= E / 2) return fill_twice<E / 2>(p, group, value);
        if constexpr (E >= 8)
            if (group >= E / 4) return fill_twice<E / 4>(p, group, value);
        for (int i = 0; i < group; ++i) p[i] = value;
    }
    // f(c, sum) in all lanes of a team for the classes from `first` to `end` of at most a piece of 16 bytes for each lane, with the pieces of four classes on their way
    // at once.  What is left behind a class's whole pieces is the end of its last 16 bytes; a class of less than a piece is a part of one.  last: features of the row.
    template <typename F>
    __device__ __forceinline__ void short_sums(const T *__restrict__ row, int first, int end, int64_t last, F f) const
    {
        typedef typename Wide<T>::type A;
        constexpr int U = sizeof(T) == 8 ? 2 : 4;
        const int pieces = group / E, rest = group - pieces * E;
        const auto place = [&](int64_t at) {                          // of the lane's piece of the class at `at`
            if (pieces > 0) return at + (lane < pieces ? lane * E : group - E);
            return at + E <= last ? at : last - E;
        };
        if (last < E) {
            for (int c = first + team; c < end; c += teams) f(c, sum(row + (int64_t)c * group));
            return;
        }
        for (int c0 = first + team; c0 < end; c0 += U * teams) {
            V v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const V *>(row + place((int64_t)(c0 + u * teams < end ? c0 + u * teams : end - 1) * group));
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * teams;
                if (c >= end) break;
                int from = 0, to = E;                                 // elements of the piece that are the lane's
                if (pieces == 0) {
                    from = (int)((int64_t)c * group - place((int64_t)c * group)), to = from + group;
                } else if (lane >= pieces) {
                    from = lane == pieces ? E - rest : E;
                }
                double s = 0;
#pragma unroll
                for (int j = 0; j < E; ++j) s += j >= from && j < to ? (double)(A)v[u][j] : 0.0;
                for (int by = lanes >> 1; by > 0; by >>= 1) s += __shfl_xor(s, by);
                f(c, s);
            }
        }
    }
    __device__ __forceinline__ bool is_short() const { return group <= lanes * E; }
    // f(c, sum of the features, whether this thread is to account for it) for the classes from `first` to `end`; every lane of a team calls it
    template <typename F>
    __device__ __forceinline__ void sums(const T *__restrict__ row, int first, int end, int64_t last, F f) const
    {
        if constexpr (PACK == 0) {
            if (is_short()) return short_sums(row, first, end, last, [&](int c, double s) { f(c, s, lane == 0); });
            for (int c = first + team; c < end; c += teams) f(c, sum(row + (int64_t)c * group), lane == 0);
        } else {
            const T *p = row + (int64_t)first * PACK;
            const int pieces = (end - first) / EACH;
            const auto of = [&](int i, const V &v) {
#pragma unroll
                for (int q = 0; q < EACH; ++q) {
                    double s = 0;
#pragma unroll
                    for (int j = 0; j < PACK; ++j) s += (double)(typename Wide<T>::type)v[q * PACK + j];
                    f(first + i * EACH + q, s, true);
                }
            };
            int i = threadIdx.x;
            for (; i + 3 * THREADS < pieces; i += 4 * THREADS) {
                V v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = reinterpret_cast<const V *>(p)[i + u * THREADS];
#pragma unroll
                for (int u = 0; u < 4; ++u) of(i + u * THREADS, v[u]);
            }
            for (; i < pieces; i += THREADS) of(i, reinterpret_cast<const V *>(p)[i]);
            const int left = pieces * EACH + (int)threadIdx.x, c = first + left;
            if (left < end - first) {
                double s = 0;
#pragma unroll
                for (int j = 0; j < PACK; ++j) s += (double)(typename Wide<T>::type)row[(int64_t)c * PACK + j];
                f(c, s, true);
            }
        }
    }
    // every feature of class c of `to` = value(c, sum of c's features in `row`)
    template <typename F>
    __device__ __forceinline__ void both(const T *__restrict__ row, T *__restrict__ to, int first, int end, int64_t last, F value) const
    {
        if constexpr (PACK == 0) {
            sums(row, first, end, last, [&](int c, double s, bool) { fill(to + (int64_t)c * group, (T)value(c, s)); });
        } else {
            const T *p = row + (int64_t)first * PACK;
            T *o = to + (int64_t)first * PACK;
            const int pieces = (end - first) / EACH;
            const auto of = [&](int i, V v) {
#pragma unroll
                for (int q = 0; q < EACH; ++q) {
                    double s = 0;
#pragma unroll
                    for (int j = 0; j < PACK; ++j) s += (double)(typename Wide<T>::type)v[q * PACK + j];
                    const T u = (T)value(first + i * EACH + q, s);
#pragma unroll
                    for (int j = 0; j < PACK; ++j) v[q * PACK + j] = u;
                }
                reinterpret_cast<V *>(o)[i] = v;
            };
            int i = threadIdx.x;
            for (; i + 3 * THREADS < pieces; i += 4 * THREADS) {
                V v[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) v[u] = reinterpret_cast<const V *>(p)[i + u * THREADS];
#pragma unroll
                for (int u = 0; u < 4; ++u) of(i + u * THREADS, v[u]);
            }
            for (; i < pieces; i += THREADS) of(i, reinterpret_cast<const V *>(p)[i]);
            const int left = pieces * EACH + (int)threadIdx.x, c = first + left;
            if (left < end - first) {
                double s = 0;
#pragma unroll
                for (int j = 0; j < PACK; ++j) s += (double)(typename Wide<T>::type)row[(int64_t)c * PACK + j];
                const T u = (T)value(c, s);
#pragma unroll
                for (int j = 0; j < PACK; ++j) to[(int64_t)c * PACK + j] = u;
            }
        }
    }
    // every feature of class c = value(c)
    template <typename F>
    __device__ __forceinline__ void store(T *__restrict__ row, int first, int end, F value) const
    {
        if constexpr (PACK == 0) {
            for (int c = first + team; c < end; c += teams) fill(row + (int64_t)c * group, (T)value(c));
        } else {
            T *p = row + (int64_t)first * PACK;
            const int pieces = (end - first) / EACH;
            for (int i = threadIdx.x; i < pieces; i += THREADS) {
                V v;
#pragma unroll
                for (int q = 0; q < EACH; ++q) {
                    const T u = (T)value(first + i * EACH + q);
#pragma unroll
                    for (int j = 0; j < PACK; ++j) v[q * PACK + j] = u;
                }
                reinterpret_cast<V *>(p)[i] = v;
            }
            const int left = pieces * EACH + (int)threadIdx.x, c = first + left;
            if (left < end - first) {
                const T u = (T)value(c);
#pragma unroll
                for (int j = 0; j < PACK; ++j) row[(int64_t)c * PACK + j] = u;
            }
        }
    }
};

// A workgroup per row.  Its classes' sums are in LDS as S; those of up to 64 features as floats, twice as many: scores in units relative to the highest of the classes
// in the row's first 64 features, or, where these do not fill 16-byte pieces, of the first class and the middle one.  Where the row's highest turns out to be more than kFar
// from that, as where these classes are masked, they are made again relative to the highest.  Near the highest a score is then off by half a step of a float under
// kFar, 2^-18, as any argument of that size of an exponential is.  (Relative to the target's, which is seldom masked, but whose place has to be read first: loss_tokens
// 398 us, not 385.)  Bound by memory: 4096 rows of 32768 classes of 4 bfloat16 with their gradient, 2.1 GB, 375 us, 5.7 TB/s (with the next pieces loaded under the sums of
// these 392); of 1 bfloat16 422 us in all, and 490 where the first 64 classes are -10^4.
constexpr int kNear = 64;
constexpr float kFar = 128;
constexpr double kLevel = 1 << 28;                                    // units up to which a multiply-add with the rounded product of another sum is a difference
// wavefronts that a SIMD shall hold of rows_kernel: 2000 rows of 6000 classes of 5 bfloat16 79 us with five, 82 with the four that 99 registers leave
constexpr int rows_waves(int threads, int pack, size_t held) { return threads != 256 || held == 8 ? 1 : pack == 0 ? 5 : 4; }
template <typename T, int THREADS, int PACK, typename S>
__global__ __launch_bounds__(THREADS, rows_waves(THREADS, PACK, sizeof(S))) void rows_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    extern __shared__ char lds[];
    __shared__ double room[32], shared[2];
    S *score = reinterpret_cast<S *>(lds);
    constexpr bool kFloats = sizeof(S) == 4;
    const double unit = a.inv_tau * Unit<A>::unit;
    const Classes<T, THREADS, PACK> classes(a.group, a.lanes_log2);
    const double per = per_row<THREADS>(a, room);
    if (a.count == 1 && blockIdx.x == 0 && threadIdx.x == 0) *a.per_count = per;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.stride;
        T *grad = a.grad ? static_cast<T *>(a.grad) + row * ((int64_t)a.k * a.group) : nullptr;
        const int64_t t = target_of(a, row);
        if (t < 0 || t >= a.k) {                                      // a row that does not count, or has no such class
            const double v = t < 0 ? 0.0 : __builtin_nan("");
            if (threadIdx.x == 0) {
                if (a.row_loss) a.row_loss[row] = v;
                if (a.out) static_cast<A *>(a.out)[row] = (A)v;
            }
            if (grad) classes.store(grad, 0, a.k, [&](int) { return (A)v; });
            continue;
        }
        double at = 0;                                                // what floats are relative to
        if constexpr (kFloats) {                                      // (each wavefront finds it for itself)
            const int lane = threadIdx.x & 63;
            if constexpr (PACK == 0) {
                const T *other = x + (int64_t)(a.k / 2) * a.group;
                const double v = lane < a.group ? (double)(A)x[lane] : 0.0, w = lane < a.group ? (double)(A)other[lane] : 0.0;
                at = max_of(wave_sum(v), wave_sum(w));
            } else {
                const bool there = lane < a.k * PACK;
                double v = there ? (double)(A)x[lane] : 0.0;
                if constexpr (PACK > 1) v += dpp_zero<0xB1, 0xF>(v);
                if constexpr (PACK > 2) v += dpp_zero<0x4E, 0xF>(v);
                if constexpr (PACK > 4) v += dpp_zero<0x141, 0xF>(v);
                at = wave_max(there ? v : lowest(0.0));
            }
            at *= unit;
            if (!(__builtin_fabs(at) <= kLevel)) at = 0;
        }
        S m[1];
        for (bool again = false;; again = true) {
            m[0] = lowest(S(0));
            classes.sums(x, 0, a.k, (int64_t)a.k * a.group, [&](int c, double s, bool mine) {
                const S u = (S)(kFloats ? s * unit - at : s);
                if (mine) score[c] = u;
                m[0] = max_of(m[0], u);
            });
            __syncthreads();                                          // (also: room is free again)
            block_reduce<false, THREADS>(m, reinterpret_cast<S *>(room));
            if (!kFloats || again || __builtin_fabs(m[0]) <= kFar || !(__builtin_fabs(at + (double)m[0]) <= kLevel)) break;
            at += (double)m[0];                                       // the highest but for 2^-24 of its distance, 32 units at most
            __syncthreads();                                          // (room is read)
        }
        double highest = kFloats ? (at + (double)m[0]) / unit : (double)m[0];
        // (for rows that are further off, or whose scores are beyond kLevel, by plain loops that take no registers from the others)
        const auto plain_sum = [&](int c) {
            double s = 0;
#pragma unroll 1
            for (int j = 0; j < a.group; ++j) s += (double)(A)x[c * a.group + j];
            return s;
        };
        if (kFloats && !(__builtin_fabs(m[0]) <= kFar)) {
            double top[1] = {lowest(0.0)};
            for (int c = threadIdx.x; c < a.k; c += THREADS) top[0] = max_of(top[0], plain_sum(c));
            __syncthreads();
            block_reduce<false, THREADS>(top, room);
            highest = top[0];
            const double from = __builtin_isinf(highest) ? 0 : highest;
            for (int c = threadIdx.x; c < a.k; c += THREADS) score[c] = (S)((plain_sum(c) - from) * unit);
            m[0] = (S)(highest - from);
            __syncthreads();
        }
        const double to_score = kFloats ? 1 / Unit<A>::unit : a.inv_tau;
        double sums[2] = {0, 0};
        for (int c = threadIdx.x; c < a.k; c += THREADS) {
            const S u = score[c];
            const A e = Unit<A>::power(kFloats ? (A)(u - m[0]) : (A)((u - m[0]) * unit));
            if (c == t) {
                shared[0] = (double)u;
                shared[1] = (double)e;
            } else {
                sums[0] += (double)e;
            }
            if (a.smoothing != 0) sums[1] += (double)m[0] - (double)u;
            score[c] = (S)e;
        }
        __syncthreads();
        block_reduce<true, THREADS>(sums, room);
        __syncthreads();
        if (kFloats && (sums[1] == -lowest(0.0) || shared[0] == lowest(0.0))) {
            // a score further below the highest than floats reach: what the loss takes of it
            double down[1] = {0};
            __syncthreads();                                          // (everyone has seen the target's)
            for (int c = threadIdx.x; c < a.k; c += THREADS) {
                const double d = (highest - plain_sum(c)) * unit;
                down[0] += d;
                if (c == t) shared[0] = (double)m[0] - d;
            }
            block_reduce<true, THREADS>(down, room);
            __syncthreads();
            sums[1] = down[0];
        }
        const Row r{sums[0], sums[0] + shared[1]};
        const double scale = a.scale * per;
        const Grad g(r, scale * a.inv_tau, a.smoothing, a.k);
        if (threadIdx.x == 0) {
            const double loss = r.loss(((double)m[0] - shared[0]) * to_score, sums[1] * to_score, a.k, a.smoothing) * scale;
            if (a.row_loss) a.row_loss[row] = loss;
            if (a.out) static_cast<A *>(a.out)[row] = (A)loss;
            double *f = a.final + 4 * row;
            f[0] = highest, f[1] = r.others, f[2] = r.total;
        }
        if (grad) {
            const A factor = (A)g.factor, off = (A)g.off, target = (A)g.target;
            const int at = (int)t;
            classes.store(grad, 0, a.k, [&](int c) { return c == at ? target : __builtin_elementwise_fma((A)score[c], factor, -off); });
        }
        __syncthreads();                                              // the scores are read
    }
}

// Few short rows, by one workgroup: 16 lanes to a row, a lane has classes l, l + 16, ...  The call is one launch, not two: 100 rows of 10 classes with gradient 9.3 us
// in all, 10.6 with a workgroup for each row and one that adds their losses; 128 rows of 64 13 and 10, and a launch less for the host; 256 of 10 17 and 11.
constexpr int kFewRows = 128, kFewFeatures = 64;
template <typename T>
__global__ __launch_bounds__(1024) void few_rows_kernel(CeArgs a, void *out_sum)
{
    typedef typename Wide<T>::type A;
    constexpr int EACH = kFewFeatures / 16;
    __shared__ double room[16], more[16];
    const double per = per_row<1024>(a, room);
    if (a.count == 1 && threadIdx.x == 0) *a.per_count = per;
    const int l = threadIdx.x % 16;
    const double unit = a.inv_tau * Unit<A>::unit;
    double sum[1] = {0};
    for (int64_t row = threadIdx.x / 16; row < a.rows; row += 64) {
        const T *x = static_cast<const T *>(a.x) + row * a.stride;
        T *grad = a.grad ? static_cast<T *>(a.grad) + row * ((int64_t)a.k * a.group) : nullptr;
        const int64_t t = target_of(a, row);
        double s[EACH], s_target = lowest(0.0), m = lowest(0.0), others = 0, of_target = 0, down = 0;
        A e[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int c = l + 16 * i;
            s[i] = 0;
            if (c >= a.k) continue;
            for (int j = 0; j < a.group; ++j) s[i] += (double)(A)x[c * a.group + j];
            m = max_of(m, s[i]);
            if (c == t) s_target = s[i];
        }
        m = row16_max(m);
        // (one lane has the target's; a NaN there is found by the exponential)
        s_target = row16_max(s_target);
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int c = l + 16 * i;
            e[i] = c < a.k ? Unit<A>::power((A)((s[i] - m) * unit)) : A(0);
            if (c >= a.k) continue;
            if (c == t) of_target = (double)e[i];
            else others += (double)e[i];
            down += m - s[i];
        }
        others = row16_sum(others), of_target = row16_sum(of_target), down = row16_sum(down);
        const Row r{others, others + of_target};
        const bool counts = t >= 0 && t < a.k;
        const double scale = a.scale * per, none = t < 0 ? 0.0 : __builtin_nan("");
        const Grad g(r, scale * a.inv_tau, a.smoothing, a.k);
        const double loss = counts ? r.loss((m - s_target) * a.inv_tau, down * a.inv_tau, a.k, a.smoothing) * scale : none;
        if (l < 3) a.final[4 * row + l] = l == 0 ? m : l == 1 ? r.others : r.total;
        if (l == 0) {
            sum[0] += loss;
            if (a.out) static_cast<A *>(a.out)[row] = (A)loss;
        }
        if (!grad) continue;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int c = l + 16 * i;
            if (c >= a.k) continue;
            const A v = !counts ? (A)none : c == t ? (A)g.target : __builtin_elementwise_fma(e[i], (A)g.factor, -(A)g.off);
            for (int j = 0; j < a.group; ++j) grad[c * a.group + j] = (T)v;
        }
    }
    if (!out_sum) return;
    block_reduce<true, 1024>(sum, more);
    if (threadIdx.x == 0) *static_cast<A *>(out_sum) = (A)sum[0];
}

// Statistics over THREADS threads, valid in thread 0.
template <int THREADS, typename A>
__device__ __forceinline__ Joint<A> block_stats(const Stats<A> &mine, double unit, double *room)
{
    Joint<A> s(mine);
    double m[1] = {s.m};
    block_reduce<false, THREADS>(m, room);
    s.raise(m[0], unit);
    double sums[3] = {s.others, s.down, s.n};
    __syncthreads();
    block_reduce<true, THREADS>(sums, room);
    __syncthreads();
    s.m = m[0], s.others = sums[0], s.down = sums[1], s.n = sums[2];
    return s;
}

constexpr int kPart = 256;                                            // threads of a piece

// 7 rows of 50001 classes of 5 float16, 3.5 MB: 7.2 us, 3.5 for the join, 6.8 for the gradient; what a launch takes to start, load and end.
template <typename T, int PACK>
__global__ __launch_bounds__(kPart) void row_stats_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    __shared__ double room[3 * kPart / kWave];
    const Classes<T, kPart, PACK> classes(a.group, a.lanes_log2);
    const bool smooth = a.smoothing != 0;
    const double unit = a.inv_tau * Unit<A>::unit;
    for (int64_t task = blockIdx.x; task < a.rows * a.pieces; task += gridDim.x) {
        const int64_t row = task / a.pieces;
        const int piece = (int)(task % a.pieces), first = piece * a.per_piece, end = end_of(a, first);
        const int64_t t = target_of(a, row);
        const T *x = static_cast<const T *>(a.x) + row * a.stride;
        Stats<A> s;
        if (t >= 0 && t < a.k) {
            classes.sums(x, first, end, (int64_t)a.k * a.group, [&](int c, double sum, bool mine) {
                if (!mine) return;
                s.add(sum, c == t, smooth, unit);
                if (c == t) a.target_sum[row] = sum;
            });
        }
        const Joint<A> all = block_stats<kPart>(s, unit, room);
        if (threadIdx.x == 0) all.store(a.stats + 4 * ((int64_t)piece * a.rows + row));
    }
}

// A row's loss from its statistics, which become the highest sum, O and Z.
template <typename A>
__device__ __forceinline__ double row_of(const CeArgs &a, int64_t row, Joint<A> s, double target, double per)
{
    if (__builtin_isinf(s.m)) s.others = __builtin_nan("");
    const Row r{s.others, s.others + (double)Unit<A>::power((A)((target - s.m) * (a.inv_tau * Unit<A>::unit)))};
    a.final[4 * row] = s.m, a.final[4 * row + 1] = r.others, a.final[4 * row + 2] = r.total;
    return r.loss((s.m - target) * a.inv_tau, s.down * a.inv_tau, a.k, a.smoothing) * a.scale * per;
}
// The statistics of a row's pieces into the highest sum, O, Z and the loss: LANES to a row.  One workgroup for all rows (`out_sum`) also adds their losses.
template <typename A, int LANES, int THREADS>
__global__ __launch_bounds__(THREADS) void join_kernel(CeArgs a, void *out_sum)
{
    constexpr int ROWS = THREADS / LANES;
    __shared__ double room[16], more[16];
    const double per = per_row<THREADS>(a, room);
    if (a.count == 1 && blockIdx.x == 0 && threadIdx.x == 0) *a.per_count = per;
    const int l = threadIdx.x % LANES;
    const double unit = a.inv_tau * Unit<A>::unit;
    double sum[1] = {0};
    for (int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES; row < a.rows; row += (int64_t)gridDim.x * ROWS) {
        const int64_t t = target_of(a, row);
        double loss = t < 0 ? 0.0 : __builtin_nan("");
        if (t >= 0 && t < a.k) {
            Joint<A> s;
            for (int p = l; p < a.pieces; p += LANES) s.join(Joint<A>(a.stats + 4 * ((int64_t)p * a.rows + row)), unit);
            if constexpr (LANES == 16) {
                s.raise(row16_max(s.m), unit);
                s.others = row16_sum(s.others), s.down = row16_sum(s.down);
            } else {
                s.raise(wave_max(s.m), unit);
                s.others = wave_sum(s.others), s.down = wave_sum(s.down);
            }
            if (l == 0) loss = row_of(a, row, s, a.target_sum[row], per);
        }
        if (l != 0) continue;
        sum[0] += loss;
        if (a.row_loss) a.row_loss[row] = loss;
        if (a.out) static_cast<A *>(a.out)[row] = (A)loss;
    }
    if (!out_sum) return;
    block_reduce<true, THREADS>(sum, more);
    if (threadIdx.x == 0) *static_cast<A *>(out_sum) = (A)sum[0];
}

// What a gradient is computed from: the highest sum and the factors.
template <typename A>
struct GradOf {
    double m, unit;
    A factor, off, target;
    __device__ __forceinline__ GradOf() {}
    __device__ __forceinline__ GradOf(const CeArgs &a, int64_t row)
    {
        const double *f = a.final + 4 * row;
        const double up = a.upstream ? (double)static_cast<const A *>(a.upstream)[a.reduction == CLG_REDUCE_NONE ? row : 0] : 1.0;
        const Grad g(Row{f[1], f[2]}, a.scale * (a.count ? *a.per_count : 1.0) * a.inv_tau * up, a.smoothing, a.k);
        m = f[0], unit = a.inv_tau * Unit<A>::unit;
        factor = (A)g.factor, off = (A)g.off, target = (A)g.target;
    }
    __device__ __forceinline__ A operator()(double sum, bool is_target) const
    {
        const A e = Unit<A>::power((A)((sum - m) * unit));
        return is_target ? target : __builtin_elementwise_fma(e, factor, -off);
    }
};

template <typename T, int PACK>
__global__ __launch_bounds__(kPart) void row_grad_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    if (nothing_to_do<A>(a)) return;
    const Classes<T, kPart, PACK> classes(a.group, a.lanes_log2);
    for (int64_t task = blockIdx.x; task < a.rows * a.pieces; task += gridDim.x) {
        const int64_t row = task / a.pieces;
        const int piece = (int)(task % a.pieces), first = piece * a.per_piece, end = end_of(a, first);
        const int64_t t = target_of(a, row);
        T *grad = static_cast<T *>(a.grad) + row * ((int64_t)a.k * a.group);
        if (t < 0 || t >= a.k) {
            const A v = t < 0 ? A(0) : (A)__builtin_nan("");
            classes.store(grad, first, end, [&](int) { return v; });
            continue;
        }
        const GradOf<A> g(a, row);
        classes.both(static_cast<const T *>(a.x) + row * a.stride, grad, first, end, (int64_t)a.k * a.group, [&](int c, double sum) { return g(sum, c == t); });
    }
}

// ---- columns: x [k G][rows] ----------------------------------------------------------------------------------------------------
// A wavefront has 64 V samples, V to a lane; or (V = 1) 1 << lanes_log2 samples side by side and, beside them, as many features of a class as its lanes hold.  The
// wavefronts of a workgroup have a class each.  The last lanes of a row that V does not divide take the last V samples, some of them twice.
template <int V>
struct Column {
    int64_t row;                                                      // the first sample
    int sub, subs, wave;
    bool live;
    __device__ __forceinline__ explicit Column(const CeArgs &a)
    {
        const int lane = threadIdx.x & 63;
        wave = uniform(threadIdx.x >> 6);
        if constexpr (V == 1) {
            row = ((int64_t)blockIdx.x << a.lanes_log2) + (lane & ((1 << a.lanes_log2) - 1));
            sub = lane >> a.lanes_log2, subs = 64 >> a.lanes_log2;
        } else {
            row = ((int64_t)blockIdx.x * 64 + lane) * V;
            sub = 0, subs = 1;
        }
        live = row < a.rows;
        if (row + V > a.rows) row = a.rows - V;
    }
};
// the classes of the wavefront that has a part of a piece's
__device__ __forceinline__ void wave_classes(int first, int end, int wave, int &c0, int &c1)
{
    constexpr int WAVES = kPart / kWave;
    const int n = end - first, run = n / WAVES + (n % WAVES != 0), from = wave * run < n ? wave * run : n;
    c0 = first + from;
    c1 = n - from > run ? c0 + run : end;
}
template <typename T>
__device__ __forceinline__ double column_sum(const CeArgs &a, const Column<1> &col, int64_t from, int64_t to)
{
    typedef typename Wide<T>::type A;
    const T *x = static_cast<const T *>(a.x) + col.row;
    double s = 0;
    int64_t i = from + col.sub;
    for (; i + 7 * col.subs < to; i += 8 * col.subs) {
        T v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = x[(i + u * col.subs) * a.rows];
#pragma unroll
        for (int u = 0; u < 8; ++u) s += (double)(A)v[u];
    }
    for (; i < to; i += col.subs) s += (double)(A)x[i * a.rows];
    for (int by = 1 << a.lanes_log2; by < 64; by <<= 1) s += __shfl_xor(s, by);
    return s;
}
// V values of a row, at any element's address
template <typename T, int V>
struct Some {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
template <typename T>
struct Some<T, 1> {
    typedef T type;
};
template <int V, typename U>
__device__ __forceinline__ auto part_of(const U &v, int i)
{
    if constexpr (V == 1) return v;
    else return v[i];
}
template <int V, typename T, typename S>
__device__ __forceinline__ void store_part(T *p, const S (&s)[V])
{
    typename Some<T, V>::type v;
    if constexpr (V == 1) v = (T)s[0];
    else
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)s[i];
    *reinterpret_cast<typename Some<T, V>::type *>(p) = v;
}

// f(class, sums) for the classes from `first` on whose features are rows `from` to `to` of x one after the other, `group` each, with the next rows on their way
template <int V, typename T, typename F>
__device__ __forceinline__ void column_stream(const CeArgs &a, const Column<V> &col, const T *x, int first, int64_t from, int64_t to, int group, F f)
{
    typedef typename Wide<T>::type A;
    typedef typename Some<T, V>::type P;
    constexpr int U = V * sizeof(T) >= 16 ? 4 : V * sizeof(T) <= 2 ? 16 : 8;
    x += col.row;
    const auto load = [&](int64_t i, P (&v)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const P *>(x + (i + u < to ? i + u : to - 1) * a.rows);
    };
    P now[U], then[U];
    int c = first, left = group;
    double s[V] = {};
    load(from, now);
    for (int64_t i = from; i < to; i += U) {
        if (i + U < to) load(i + U, then);
        if (left > U && i + U <= to) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int v = 0; v < V; ++v) s[v] += (double)(A)part_of<V>(now[u], v);
            left -= U;
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (i + u >= to) break;
#pragma unroll
                for (int v = 0; v < V; ++v) s[v] += (double)(A)part_of<V>(now[u], v);
                if (--left == 0) {
                    f(c, s);
                    ++c, left = group;
#pragma unroll
                    for (int v = 0; v < V; ++v) s[v] = 0;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) now[u] = then[u];
    }
}
// Statistics of the workgroup's wavefronts, V samples a lane: valid in the first wavefront's, after which `finish` is called for each sample.
template <typename A, int V, int WAVES, typename F>
__device__ __forceinline__ void column_finish(const Column<V> &col, const Stats<A> (&s)[V], double unit, double (&room)[WAVES][V][kWave][4], F finish)
{
#pragma unroll
    for (int v = 0; v < V; ++v) Joint<A>(s[v]).store(room[col.wave][v][threadIdx.x & 63]);
    __syncthreads();
    if (col.wave != 0 || col.sub != 0 || !col.live) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        Joint<A> all(s[v]);
        for (int w = 1; w < WAVES; ++w) all.join(Joint<A>(room[w][v][threadIdx.x & 63]), unit);
        finish(v, all);
    }
}

// Sums over the features of a class, or a slice of them; statistics of the classes of a piece where the sums are whole.  Bound by loads in flight: 1111 rows of 1000
// classes of 30 float32, 133 MB, 30 us, 4.5 TB/s; 256 rows of 10 of 8192 in 64 slices, 84 MB, 21 to 27 us.
template <typename T, int V>
__global__ __launch_bounds__(kPart) void column_sums_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    __shared__ double room[kPart / kWave][V][kWave][4];
    const Column<V> col(a);
    const int first = (int)blockIdx.y * a.per_piece, end = end_of(a, first), slice = blockIdx.z;
    const int64_t from = (int64_t)a.group * slice / a.slices, to = (int64_t)a.group * (slice + 1) / a.slices;
    int64_t t[V];
#pragma unroll
    for (int v = 0; v < V; ++v) t[v] = target_of(a, col.row + v);
    const bool smooth = a.smoothing != 0, store = col.live && col.sub == 0;
    const double unit = a.inv_tau * Unit<A>::unit;
    Stats<A> s[V];
    const auto score = [&](int c, const double (&sum)[V]) {
        if (a.slices > 1) {
            if (store) store_part<V>(a.partial + ((int64_t)slice * a.k + c) * a.rows + col.row, sum);
            return;
        }
        if (store && a.scores) store_part<V>(a.scores + (int64_t)c * a.rows + col.row, sum);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            s[v].add(sum[v], c == t[v], smooth, unit);
            if (store && c == t[v]) a.target_sum[col.row + v] = sum[v];
        }
    };
    const T *x = static_cast<const T *>(a.x);
    int c0, c1;
    wave_classes(first, end, col.wave, c0, c1);
    if (V == 1 && col.subs > 1) {
        if constexpr (V == 1)
            for (int c = c0; c < c1; ++c) {
                const double sum[1] = {column_sum<T>(a, col, (int64_t)c * a.group + from, (int64_t)c * a.group + to)};
                score(c, sum);
            }
    } else if (a.slices > 1) {
        for (int c = c0; c < c1; ++c) column_stream(a, col, x, c, (int64_t)c * a.group + from, (int64_t)c * a.group + to, (int)(to - from), score);
    } else if (c0 < c1) {
        column_stream(a, col, x, c0, (int64_t)c0 * a.group, (int64_t)c1 * a.group, a.group, score);
    }
    if (a.slices == 1)
        column_finish(col, s, unit, room, [&](int v, const Joint<A> &all) { all.store(a.stats + 4 * ((int64_t)blockIdx.y * a.rows + col.row + v)); });
}
// The same from the sums of the slices, of all classes by one workgroup, which ends the rows' losses too.
template <typename T>
__global__ __launch_bounds__(1024) void column_stats_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    constexpr int WAVES = 1024 / kWave;
    __shared__ double room[WAVES][1][kWave][4], more[WAVES];
    const double per = per_row<1024>(a, more);
    if (a.count == 1 && blockIdx.x == 0 && threadIdx.x == 0) *a.per_count = per;
    const Column<1> col(a);
    const int64_t t = target_of(a, col.row);
    const bool smooth = a.smoothing != 0, store = col.live && col.sub == 0;
    const double unit = a.inv_tau * Unit<A>::unit;
    Stats<A> s[1];
    for (int c = col.wave; c < a.k; c += WAVES) {
        double sum = 0;
#pragma unroll 8
        for (int i = col.sub; i < a.slices; i += col.subs) sum += a.partial[((int64_t)i * a.k + c) * a.rows + col.row];
        for (int by = 1 << a.lanes_log2; by < 64; by <<= 1) sum += __shfl_xor(sum, by);
        s[0].add(sum, c == t, smooth, unit);
        if (store) a.scores[(int64_t)c * a.rows + col.row] = sum;
        if (store && c == t) a.target_sum[col.row] = sum;
    }
    column_finish(col, s, unit, room, [&](int, const Joint<A> &all) {       // (behind a barrier: the target's score is there)
        const double loss = t < 0 ? 0.0 : t >= a.k ? __builtin_nan("") : row_of(a, col.row, all, a.target_sum[col.row], per);
        if (a.row_loss) a.row_loss[col.row] = loss;
        if (a.out) static_cast<A *>(a.out)[col.row] = (A)loss;
    });
}
// Gradient from the sums of the classes, or from the features again.  256 rows of 10 classes of 8192 float32, 84 MB from the sums: 16 us, 5.3 TB/s.
template <typename T, int V>
__global__ __launch_bounds__(kPart) void column_grad_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    if (nothing_to_do<A>(a)) return;
    const Column<V> col(a);
    const int first = (int)blockIdx.y * a.per_piece, end = end_of(a, first), slice = blockIdx.z;
    const int64_t from = (int64_t)a.group * slice / a.slices, to = (int64_t)a.group * (slice + 1) / a.slices;
    int64_t t[V];
    GradOf<A> g[V];
#pragma unroll
    for (int v = 0; v < V; ++v) t[v] = target_of(a, col.row + v), g[v] = GradOf<A>(a, col.row + v);
    T *grad = static_cast<T *>(a.grad) + col.row;
    const auto store = [&](int c, const double (&sum)[V]) {
        A value[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            value[v] = g[v](sum[v], c == t[v]);
            if (t[v] < 0 || t[v] >= a.k) value[v] = t[v] < 0 ? A(0) : (A)__builtin_nan("");
        }
        if (!col.live) return;
        T *p = grad + ((int64_t)c * a.group + from + col.sub) * a.rows;
        for (int64_t i = from + col.sub; i < to; i += col.subs, p += col.subs * a.rows) store_part<V>(p, value);
    };
    int c0, c1;
    wave_classes(first, end, col.wave, c0, c1);
    if (c0 >= c1) return;
    if (V > 1 || col.subs == 1) {
        if (a.scores) column_stream(a, col, a.scores, c0, c0, c1, 1, store);
        else column_stream(a, col, static_cast<const T *>(a.x), c0, (int64_t)c0 * a.group, (int64_t)c1 * a.group, a.group, store);
    } else if constexpr (V == 1) {
        for (int c = c0; c < c1; ++c) {
            const double sum[1] = {a.scores ? a.scores[(int64_t)c * a.rows + col.row]
                                            : column_sum<T>(a, col, (int64_t)c * a.group, (int64_t)(c + 1) * a.group)};
            store(c, sum);
        }
    }
}

// 1 / number of rows that count, by one workgroup
__global__ __launch_bounds__(1024) void count_kernel(CeArgs a)
{
    __shared__ double room[16];
    a.count = 1;
    const double per = per_row<1024>(a, room);
    if (threadIdx.x == 0) *a.per_count = per;
}

// ---- host ----------------------------------------------------------------------------------------------------------------------
constexpr int64_t kCounted = 1024;                                    // rows that every workgroup counts for itself
constexpr int kLds = 144 << 10;                                       // of a row's scores
constexpr int64_t kMostBlocks = 1 << 20;
constexpr int64_t kSliced = 256;                                      // classes whose features may go in slices

// How a call goes, by its sizes alone.
struct Plan {
    bool rows, whole, few;                                            // layout; a workgroup per row, or for all
    int64_t n, k, group, features;
    int size;                                                         // bytes of an element
    int lanes_log2, samples, pieces, per_piece, slices;               // samples: of a lane ("columns")
    bool scores, kept_scores;                                         // "columns"
};
int log2_up(int64_t v)
{
    int l = 0;
    while ((1ll << l) < v) ++l;
    return l;
}
int64_t chunks_of(const Plan &p) { return clg_ceil_div(p.n, p.samples > 1 ? 64ll * p.samples : 1ll << p.lanes_log2); }
int packed(const Plan &p)
{
    const int e = 16 / p.size;
    return p.group <= e && e % p.group == 0 ? (int)p.group : 0;
}
Plan plan_of(int dtype, bool rows, int64_t n, int64_t features, int64_t k)
{
    Plan p{rows, false, false, n, k, features / k, features, clg_elem_bytes(dtype), 0, 1, 1, (int)k, 1, false, false};
    const auto cut = [&](int64_t pieces, int64_t unit) {              // pieces of a multiple of `unit` classes
        const int64_t each = clg_ceil_div(clg_ceil_div(k, pieces < 1 ? 1 : pieces), unit) * unit;
        p.per_piece = (int)(each < k ? each : k);
        p.pieces = (int)clg_ceil_div(k, p.per_piece);
    };
    p.few = rows && n <= kFewRows && features <= kFewFeatures;
    if (rows) {
        // a lane for each piece of a class, up to a wavefront: what the lanes load at once is then in one place (a lane for four pieces, two lanes to a class
        // of 61 bfloat16 features: 2.1 TB/s)
        const int e = 16 / p.size;
        p.lanes_log2 = p.group < e ? 0 : log2_up(clg_ceil_div(p.group, e));
        if (p.lanes_log2 > 6) p.lanes_log2 = 6;
        const int64_t lds = k * (dtype == CLG_F64 || p.group > kNear ? 8 : 4);
        // a workgroup for a row of 256 KB (1000 classes of 64 float32) takes 26, 28, 28 and 33 us for 32, 64, 96 and 192 of them, pieces 22, 26, 36 and 50; for
        // rows of 240 KB (30000 of 4 bfloat16) 23, 25 and 31 for 32, 64 and 192, pieces 19, 25 and 45; for 16 and 96 of 32 KB 15 and 15, pieces 16 and 21
        p.whole = lds <= kLds && (n > 64 || features * p.size <= 64 << 10);
        // else about 1024 workgroups, of 16 KiB of features at least
        int64_t want = clg_ceil_div(1024, n), most = clg_ceil_div(features * p.size, 16 << 10);
        cut(want < most ? want : most, 16);
    } else {
        p.lanes_log2 = log2_up(n < 64 ? n : 64);
        // several samples to a lane where that leaves few lanes idle and workgroups enough (4 to a lane and 1: 4802 rows of 1759 classes of 27 float32 543
        // and 657 us, but the sums of 256 rows of 10 classes of 8192 28 and 21)
        for (int v = dtype == CLG_F64 ? 2 : 4; v > 1 && p.samples == 1; v /= 2)
            if (n >= v * 64 && clg_ceil_div(n, v * 64) * v * 64 * 3 <= n * 4 &&
                clg_ceil_div(n, v * 64) * clg_ceil_div(k, 4) * (p.group < 128 || k > kSliced ? 1 : p.group > 4096 ? 64 : p.group / 64) >= 768)
                p.samples = v;
        const int64_t chunks = chunks_of(p), want = clg_ceil_div(1024, chunks);
        cut(want < clg_ceil_div(k, 4) ? want : clg_ceil_div(k, 4), 4);
        // Slices of 64 features at least, for up to three workgroups to a CU (few classes: the workgroup that joins the slices has all of them).  768, 1024 and 1536
        // workgroups: 512 rows of 10 classes of 8192 float32 88, 94 and 96 us, 1000 of 7 of 3000 54, 54 and 59; up to 64 and 256 slices: 64 rows of 2 of 65536
        // 115 and 50.
        const int64_t slices = 768 / (chunks * p.pieces), most = k <= kSliced ? p.group / 64 : 1;
        p.slices = (int)(slices < most ? slices : most);
        if (p.slices < 1) p.slices = 1;
        if (p.slices > 256) p.slices = 256;
        // The sums of the classes are written out for the gradient where that is less than to read the features again: without and with, 1024 rows of 4096 classes
        // of 4 float32 features 66 and 69 us, of 5 71 and 67, of 16 190 and 157; of 8 bfloat16 69 and 66, of 16 118 and 92.  Those that are no more than a
        // sixteenth of the features are kept for a backward pass with another upstream gradient.
        p.kept_scores = p.slices > 1 || p.group * p.size >= 128;
        p.scores = p.kept_scores || p.group * p.size > 16;
    }
    return p;
}

// Workspaces: what a backward pass reads again (per_count, final, scores), and the rest.
struct Rooms {
    int64_t kept, scratch;
};
Rooms rooms_of(const Plan &p, CeArgs *a, void *kept, void *scratch)
{
    int64_t at = 0;
    const auto take = [&](void *base, int64_t n) {
        double *v = base ? static_cast<double *>(base) + at : nullptr;
        at += n;
        return v;
    };
    CeArgs none;
    CeArgs &r = a ? *a : none;
    r.per_count = take(kept, 2);
    r.final = take(kept, 4 * p.n);
    if (p.kept_scores) r.scores = take(kept, p.k * p.n);
    const int64_t bytes = at * 8;
    at = 0;
    if (p.few) return {bytes, 0};
    r.row_loss = take(scratch, p.n);
    take(scratch, clg_ceil_div(p.n, kSlice));
    if (!p.whole) {
        r.target_sum = take(scratch, p.n);
        r.stats = take(scratch, 4 * p.pieces * p.n);
    }
    if (p.scores && !p.kept_scores) r.scores = take(scratch, p.k * p.n);
    if (p.slices > 1) r.partial = take(scratch, (int64_t)p.slices * p.k * p.n);
    return {bytes, at * 8};
}

template <typename T, typename F>
void with_pack(int pack, F call)
{
    constexpr int E = 16 / sizeof(T);
    const std::integral_constant<int, 0> team;
    switch (pack) {
    case 1: return call(std::integral_constant<int, 1>());
    case 2: return call(std::integral_constant<int, 2>());
    case 4:
        if constexpr (E >= 4) return call(std::integral_constant<int, 4>());
    case 8:
        if constexpr (E >= 8) return call(std::integral_constant<int, 8>());
    default: return call(team);
    }
}

template <typename T, typename F>
void with_samples(int samples, F call)
{
    if (samples == 1) call(std::integral_constant<int, 1>());
    else if (sizeof(T) == 8 || samples == 2) call(std::integral_constant<int, 2>());
    else call(std::integral_constant<int, sizeof(T) == 8 ? 2 : 4>());
}

unsigned blocks(int64_t n) { return (unsigned)(n < kMostBlocks ? n : kMostBlocks); }

template <typename T, int THREADS, int PACK, typename S>
int launch_rows(const char *name, const CeArgs &a, hipStream_t stream)
{
    const size_t lds = a.k * sizeof(S);
    if (lds > 48 << 10) {                                             // (of all calls the same: another thread's may come between this one and the launch)
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(rows_kernel<T, THREADS, PACK, S>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds);
        if (e != hipSuccess) {
            clg_set_error("%s: %s", name, hipGetErrorString(e));
            return CLG_ELAUNCH;
        }
    }
    rows_kernel<T, THREADS, PACK, S><<<dim3(blocks(a.rows)), dim3(THREADS), lds, stream>>>(a);
    CLG_CHECK_LAUNCH(name);
    return CLG_OK;
}
// Threads of a row.  64, 256 and 1024 of them, 2000 rows of 4 KB of float32 19, 21 and 45 us, of 16 KB 24, 27 and 48, of 64 KB 68, 66 and 86, of 256 KB 278, 248
// and 224, of bfloat16 32 KB 46, 38 and 68, 128 KB 160, 130 and 139; 500 rows of 4 KB 14, 12 and 17, of 64 KB 49, 25 and 28, of 256 KB 180, 70 and 64; 150 rows of 4
// KB 13, 11 and 12, of 64 KB 44, 21 and 17.
template <typename T, int PACK, typename S>
int launch_rows(const char *name, const CeArgs &a, hipStream_t stream)
{
    const int64_t bytes = (int64_t)a.k * a.group * sizeof(T);
    const bool many = a.rows >= 1024;
    if (bytes <= (many ? 16 << 10 : 2 << 10)) return launch_rows<T, 64, PACK, S>(name, a, stream);
    if (bytes <= (many ? 128 << 10 : 32 << 10)) return launch_rows<T, 256, PACK, S>(name, a, stream);
    return launch_rows<T, 1024, PACK, S>(name, a, stream);
}

template <typename T>
int forward(const char *name, const Plan &p, const CeArgs &a, void *out_sum, hipStream_t stream)
{
    int rc = CLG_OK;
    if (p.few) {
        few_rows_kernel<T><<<dim3(1), dim3(1024), 0, stream>>>(a, out_sum);
        CLG_CHECK_LAUNCH(name);
        return CLG_OK;
    }
    if (p.whole) {
        with_pack<T>(packed(p), [&](auto pack) {
            constexpr int PACK = decltype(pack)::value;
            if (p.group > kNear) rc = launch_rows<T, 0, double>(name, a, stream);
            else rc = launch_rows<T, PACK, typename Wide<T>::type>(name, a, stream);
        });
        return rc;
    }
    const dim3 columns((unsigned)chunks_of(p), (unsigned)p.pieces, (unsigned)p.slices);
    if (p.rows) {
        with_pack<T>(packed(p), [&](auto pack) { row_stats_kernel<T, decltype(pack)::value><<<dim3(blocks(p.n * p.pieces)), dim3(kPart), 0, stream>>>(a); });
    } else {
        with_samples<T>(p.samples, [&](auto v) { column_sums_kernel<T, decltype(v)::value><<<columns, dim3(kPart), 0, stream>>>(a); });
        CLG_CHECK_LAUNCH(name);
        // 4 samples to a workgroup, and 16 lanes to a class's slices: this kernel of 256 rows of 10 classes in 64 slices 7.5 us, with 16 samples 10.9; of 1024 rows
        // of 256 classes in 5 slices 20.9 and 18.2
        if (p.slices > 1) {
            CeArgs b = a;
            b.lanes_log2 = p.lanes_log2 < 2 ? p.lanes_log2 : 2;
            column_stats_kernel<T><<<dim3((unsigned)clg_ceil_div(p.n, 1ll << b.lanes_log2)), dim3(1024), 0, stream>>>(b);
        }
    }
    CLG_CHECK_LAUNCH(name);
    if (!p.rows && p.slices > 1) return CLG_OK;
    typedef typename Wide<T>::type A;
    // In one workgroup that adds the losses too, 16 lanes to a row, or 64 where it has more than 32 pieces (then of up to 16 rows): 40 rows of 16 pieces 5.2 and 8.4
    // us, 16 of them 4.6 and 5.5.  Else four rows to a workgroup, 64 lanes each: 100 rows of 256 pieces 5.9 us, with 16 lanes 10.9; 1024 rows of 256 7.2 and 11.2,
    // with 16 rows to a workgroup, whose lanes have a line of memory each, 10.2.
    if (!out_sum) join_kernel<A, 64, 256><<<dim3(blocks(clg_ceil_div(p.n, 4))), dim3(256), 0, stream>>>(a, nullptr);
    else if (p.pieces <= 32) join_kernel<A, 16, 1024><<<dim3(1), dim3(1024), 0, stream>>>(a, out_sum);
    else join_kernel<A, 64, 1024><<<dim3(1), dim3(1024), 0, stream>>>(a, out_sum);
    CLG_CHECK_LAUNCH(name);
    return CLG_OK;
}
template <typename T>
int gradient(const char *name, const Plan &p, const CeArgs &a, hipStream_t stream)
{
    if (p.rows) with_pack<T>(packed(p), [&](auto pack) { row_grad_kernel<T, decltype(pack)::value><<<dim3(blocks(p.n * p.pieces)), dim3(kPart), 0, stream>>>(a); });
    else with_samples<T>(p.samples, [&](auto v) {
            column_grad_kernel<T, decltype(v)::value><<<dim3((unsigned)chunks_of(p), (unsigned)p.pieces, (unsigned)p.slices), dim3(kPart), 0, stream>>>(a);
        });
    CLG_CHECK_LAUNCH(name);
    return CLG_OK;
}

int check_call(const char *name, int dtype, const void *x, int64_t stride, int64_t rows, int64_t features, int64_t k, const void *targets, int targets_bits, double tau,
               double smoothing, int reduction)
{
    CLG_REQUIRE(clg_score_type(dtype), "%s: unsupported dtype %d", name, dtype);
    CLG_REQUIRE(rows >= 0 && rows < 1ll << 31 && k >= 1 && features >= 1 && features < 1ll << 31, "%s: bad shape [%lld, %lld] of %lld classes", name, (long long)rows,
                (long long)features, (long long)k);
    CLG_REQUIRE(features % k == 0, "%s: %lld features are no multiple of %lld classes", name, (long long)features, (long long)k);
    CLG_REQUIRE(targets_bits == 32 || targets_bits == 64, "%s: targets must have 32 or 64 bits, got %d", name, targets_bits);
    CLG_REQUIRE(stride >= -1, "%s: negative row stride", name);
    CLG_REQUIRE(tau > 0 && tau < 1e30, "%s: tau must be positive and finite", name);
    CLG_REQUIRE(smoothing >= 0 && smoothing <= 1, "%s: the smoothing must be between 0 and 1", name);
    CLG_REQUIRE(reduction == CLG_REDUCE_NONE || reduction == CLG_REDUCE_SUM || reduction == CLG_REDUCE_MEAN, "%s: bad reduction %d", name, reduction);
    CLG_REQUIRE(!rows || (x && targets), "%s: null pointer", name);
    return CLG_OK;
}
CeArgs args_of(const Plan &p, const void *x, int64_t stride, const void *targets, int targets_bits, double tau, double smoothing, double weight, int reduction)
{
    CeArgs a{};
    a.x = x, a.rows = p.n, a.stride = stride, a.k = (int)p.k, a.group = (int)p.group;
    a.targets = targets, a.targets64 = targets_bits == 64;
    a.inv_tau = 1 / tau, a.smoothing = smoothing, a.scale = weight, a.reduction = reduction;
    a.pieces = p.pieces, a.per_piece = p.per_piece, a.slices = p.slices, a.lanes_log2 = p.lanes_log2;
    return a;
}

}  // namespace

extern "C" int64_t clg_group_ce_kept_bytes(int dtype, int columns, int64_t rows, int64_t features, int64_t k)
{
    if (!clg_score_type(dtype) || rows <= 0 || k < 1 || features < k || features % k || features >= 1ll << 31) return 0;
    return rooms_of(plan_of(dtype, !columns, rows, features, k), nullptr, nullptr, nullptr).kept;
}
extern "C" int64_t clg_group_ce_scratch_bytes(int dtype, int columns, int64_t rows, int64_t features, int64_t k)
{
    if (!clg_score_type(dtype) || rows <= 0 || k < 1 || features < k || features % k || features >= 1ll << 31) return 0;
    return rooms_of(plan_of(dtype, !columns, rows, features, k), nullptr, nullptr, nullptr).scratch;
}

extern "C" int clg_group_ce_forward(int dtype, const void *x, int64_t row_stride, int64_t rows, int64_t features, int64_t k, const void *targets, int targets_bits,
                                    double tau, double smoothing, double weight, int reduction, void *loss, void *grad, void *kept, void *scratch, void *stream)
{
    const char *name = "clg_group_ce_forward";
    if (const int rc = check_call(name, dtype, x, row_stride, rows, features, k, targets, targets_bits, tau, smoothing, reduction)) return rc;
    CLG_REQUIRE(loss || (reduction == CLG_REDUCE_NONE && !rows), "%s: null pointer", name);
    CLG_REQUIRE(!rows || kept, "%s: null workspace", name);
    CLG_REQUIRE(!grad || reduction != CLG_REDUCE_NONE, "%s: the gradient of a loss per row is clg_group_ce_backward's", name);
    hipStream_t st = clg_stream(stream);
    if (!rows) return reduction == CLG_REDUCE_NONE ? CLG_OK : sum_rows(name, dtype, nullptr, 0, nullptr, nullptr, loss, st);
    const Plan p = plan_of(dtype, row_stride >= 0, rows, features, k);
    CeArgs a = args_of(p, x, row_stride, targets, targets_bits, tau, smoothing, weight, reduction);
    const Rooms rooms = rooms_of(p, &a, kept, scratch);
    CLG_REQUIRE(!rooms.scratch || scratch, "%s: null workspace", name);
    double *row_loss = a.row_loss;
    if (reduction == CLG_REDUCE_NONE) a.out = loss, a.row_loss = nullptr;
    if (reduction == CLG_REDUCE_MEAN) {
        a.count = 2;
        if (rows <= kCounted) {                                       // by the workgroups of the rows, or the one that joins them
            a.count = 1;
        } else {
            count_kernel<<<dim3(1), dim3(1024), 0, st>>>(a);
            CLG_CHECK_LAUNCH(name);
        }
    }
    const bool at_once = p.whole || p.few;                            // gradient and all
    // one workgroup also adds the losses: all of few rows, or the joint statistics of so many
    const bool add = reduction != CLG_REDUCE_NONE && (p.few || (!p.whole && p.slices == 1 && rows <= (p.pieces <= 32 ? 64 : 16)));
    if (at_once) a.grad = grad;
    if (!grad && !p.kept_scores) a.scores = nullptr;
    int rc = clg_with_type(dtype, [&](auto t) { return forward<decltype(t)>(name, p, a, add ? loss : nullptr, st); });
    if (rc) return rc;
    if (grad && !at_once) {
        a.grad = grad;
        if (a.count) a.count = 2;
        rc = clg_with_type(dtype, [&](auto t) { return gradient<decltype(t)>(name, p, a, st); });
        if (rc) return rc;
    }
    return reduction == CLG_REDUCE_NONE || add ? CLG_OK : sum_rows(name, dtype, row_loss, rows, row_loss + rows, nullptr, loss, st);
}

extern "C" int clg_group_ce_backward(int dtype, const void *x, int64_t row_stride, int64_t rows, int64_t features, int64_t k, const void *targets, int targets_bits,
                                     double tau, double smoothing, double weight, int reduction, const void *upstream, void *grad, int has_grad, const void *kept,
                                     void *stream)
{
    const char *name = "clg_group_ce_backward";
    if (const int rc = check_call(name, dtype, x, row_stride, rows, features, k, targets, targets_bits, tau, smoothing, reduction)) return rc;
    if (!rows) return CLG_OK;
    CLG_REQUIRE(upstream && grad && kept, "%s: null pointer", name);
    CLG_REQUIRE(!has_grad || reduction != CLG_REDUCE_NONE, "%s: there is no gradient of a loss per row yet", name);
    const Plan p = plan_of(dtype, row_stride >= 0, rows, features, k);
    CeArgs a = args_of(p, x, row_stride, targets, targets_bits, tau, smoothing, weight, reduction);
    a.grad = grad, a.upstream = upstream, a.if_changed = has_grad, a.count = reduction == CLG_REDUCE_MEAN ? 2 : 0;
    rooms_of(p, &a, const_cast<void *>(kept), nullptr);
    if (!p.kept_scores) a.scores = nullptr;
    return clg_with_type(dtype, [&](auto t) { return gradient<decltype(t)>(name, p, a, clg_stream(stream)); });
}
