// Softmax cross entropy of group sums.  A row has k classes of G features each; with the scores s_c = (sum of the class's features) / tau, the highest M, the row's
// target t, O = sum over c != t of exp(s_c - M), Z = O + exp(s_t - M) and the smoothing e:
//     loss = w [ (1 - e) (M - s_t + log Z) + e (log Z + mean_c (M - s_c)) ]
//     d loss / d feature of c = w / tau [ exp(s_c - M) / Z - e / k ],  of t  w / tau [ -O / Z + e - e / k ]
// Where the target is the highest, log Z = log1p(O): with O apart, losses and gradients near 0 keep their digits.  A score is a long sum, and its rounding is a
// relative error of its exponential: sums over features, and what is taken of a score before its exponential, are in 64 bits.
//
// Rows in memory ("rows", features dense): a workgroup has a row, whose scores stay in LDS from the sums to the gradient, so the features are read once (rows_kernel);
// rows of more classes than LDS holds, or too few rows to fill the chip, go in pieces of the classes, once for the sums and the highest (row_stats_kernel) and once
// more for the gradient (row_grad_kernel).  A feature per row in memory ("columns"): lanes are samples, in pieces of the classes likewise.
#include "row_sums.h"

namespace {

// exp(x - m) as the sums take it: the difference in 64 bits, the exponential in A
__device__ __forceinline__ float exp_of(double x, double m, float) { return __builtin_amdgcn_exp2f((float)((x - m) * 1.4426950408889634074)); }
__device__ __forceinline__ double exp_of(double x, double m, double) { return exp(x - m); }

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
    double *final;                                                    // [rows][3]: M, O, Z
    void *out;                                                        // [rows] in A, or NULL
    const void *upstream;                                             // in A, [rows] for CLG_REDUCE_NONE, or NULL for 1
    int if_changed;                                                   // nothing to do for an upstream gradient of 1
    // pieces
    int pieces, per_piece;                                            // of the classes
    double *stats, *target_score;                                     // [pieces][rows][4], [rows]
    double *scores, *partial;                                         // "columns": [k][rows], [slices][k][rows], or NULL
    int slices, lanes_log2;                                           // of a class's features; lanes to a class, or samples side by side
};

__device__ __forceinline__ int64_t target_of(const CeArgs &a, int64_t row)
{
    return a.targets64 ? static_cast<const int64_t *>(a.targets)[row] : static_cast<const int32_t *>(a.targets)[row];
}
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

// The statistics of a part of a row's classes.
struct Stats {
    double m = lowest(0.0), others = 0, down = 0, n = 0;             // highest, O and sum of (m - s) relative to it, classes
    template <typename A>
    __device__ __forceinline__ void add(double s, bool is_target, A type)
    {
        if (!(s <= m)) raise(s == s ? s : m, type);
        const double e = s == m ? 1.0 : (double)exp_of(s, m, type);
        others += is_target ? 0.0 : s == s ? e : s;
        down += m - s;
        n += 1;
    }
    template <typename A>
    __device__ __forceinline__ void raise(double to, A type)
    {
        if (!(to > m)) return;
        if (m != lowest(0.0)) {
            others *= (double)exp_of(m, to, type);
            down += n * (to - m);
        } else {
            others = others == others ? 0.0 : others;
            down = n == 0 ? 0.0 : -lowest(0.0);                       // (classes of -inf)
        }
        m = to;
    }
    template <typename A>
    __device__ __forceinline__ void join(const Stats &o, A type)
    {
        Stats b = o;
        raise(b.m, type);
        b.raise(m, type);
        others += b.others;
        down += b.down;
        n += b.n;
    }
    __device__ __forceinline__ void store(double *p) const { p[0] = m, p[1] = others, p[2] = down, p[3] = n; }
    __device__ __forceinline__ static Stats load(const double *p)
    {
        Stats s;
        s.m = p[0], s.others = p[1], s.down = p[2], s.n = p[3];
        return s;
    }
};

// What a row's loss and gradient are made of.
struct Row {
    double m, others, total;
    __device__ __forceinline__ double loss(double s_target, double down, int k, double smoothing) const
    {
        const double margin = m - s_target, log_total = margin == 0 ? log1p(others) : log(total);
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
        for (i = pieces * E + lane; i < group; i += lanes) s += (double)(typename Wide<T>::type)p[i];
        for (int by = lanes >> 1; by > 0; by >>= 1) s += __shfl_xor(s, by);
        return s;
    }
    __device__ __forceinline__ void fill(T *__restrict__ p, T value) const
    {
        const int pieces = group / E;
        for (int i = lane; i < pieces; i += lanes) reinterpret_cast<V *>(p)[i] = (V)value;
        for (int i = pieces * E + lane; i < group; i += lanes) p[i] = value;
    }
    // f(c, sum of the features, whether this thread is to account for it) for the classes from `first` to `end`; every lane of a team calls it
    template <typename F>
    __device__ __forceinline__ void sums(const T *__restrict__ row, int first, int end, F f) const
    {
        if constexpr (PACK == 0) {
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
            const int c = first + pieces * EACH + (int)threadIdx.x;
            if (c < end) {
                double s = 0;
#pragma unroll
                for (int j = 0; j < PACK; ++j) s += (double)(typename Wide<T>::type)row[(int64_t)c * PACK + j];
                f(c, s, true);
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
            const int c = first + pieces * EACH + (int)threadIdx.x;
            if (c < end) {
                const T u = (T)value(c);
#pragma unroll
                for (int j = 0; j < PACK; ++j) row[(int64_t)c * PACK + j] = u;
            }
        }
    }
};

// A workgroup per row.  The scores are in LDS as the arguments of their exponentials, relative to a value near them (of the first features of class 0): as 32-bit
// numbers they are then as exact as a 32-bit exponential can tell.
template <typename T, int THREADS, int PACK>
__global__ __launch_bounds__(THREADS) void rows_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    extern __shared__ char lds[];
    __shared__ double room[32], shared[2];
    A *score = reinterpret_cast<A *>(lds);
    constexpr bool kFloat = sizeof(A) == 4;
    constexpr double kUnit = kFloat ? 1.4426950408889634074 : 1.0;    // exponentials are 2^x, or e^x
    const auto power = [](A x) {
        if constexpr (kFloat) return __builtin_amdgcn_exp2f(x);
        else return exp(x);
    };
    const Classes<T, THREADS, PACK> classes(a.group, a.lanes_log2);
    const int lane = threadIdx.x & 63;
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
        const int near = a.group < 64 ? a.group : 64;
        double pivot = kFloat ? wave_sum(lane < near ? (double)(A)x[lane] : 0.0) * ((double)a.group / near) * a.inv_tau * kUnit : 0.0;
        if (!(__builtin_fabs(pivot) <= __DBL_MAX__)) pivot = 0;
        A m[1] = {lowest(A(0))};
        classes.sums(x, 0, a.k, [&](int c, double s, bool mine) {
            const A u = (A)(s * (a.inv_tau * kUnit) - pivot);
            if (mine) score[c] = u;
            m[0] = max_of(m[0], u);
        });
        __syncthreads();                                              // (also: room is free again)
        block_reduce<false, THREADS>(m, reinterpret_cast<A *>(room));
        double sums[2] = {0, 0};
        for (int c = threadIdx.x; c < a.k; c += THREADS) {
            const A u = score[c], e = power(u - m[0]);
            if (c == t) {
                shared[0] = (double)u;
                shared[1] = (double)e;
            } else {
                sums[0] += (double)e;
            }
            if (a.smoothing != 0) sums[1] += (double)m[0] - (double)u;
            score[c] = e;
        }
        __syncthreads();
        block_reduce<true, THREADS>(sums, room);
        __syncthreads();
        const Row r{((double)m[0] + pivot) / kUnit, sums[0], sums[0] + shared[1]};
        const double margin = ((double)m[0] - shared[0]) / kUnit;
        const double scale = a.scale * per;
        const Grad g(r, scale * a.inv_tau, a.smoothing, a.k);
        if (threadIdx.x == 0) {
            const double loss = Row{margin, r.others, r.total}.loss(0, sums[1] / kUnit, a.k, a.smoothing) * scale;
            if (a.row_loss) a.row_loss[row] = loss;
            if (a.out) static_cast<A *>(a.out)[row] = (A)loss;
            if (a.final) a.final[3 * row] = r.m, a.final[3 * row + 1] = r.others, a.final[3 * row + 2] = r.total;
        }
        if (grad) {
            const A factor = (A)g.factor, off = (A)g.off, target = (A)g.target;
            const int at = (int)t;
            classes.store(grad, 0, a.k, [&](int c) { return c == at ? target : __builtin_elementwise_fma(score[c], factor, -off); });
        }
        __syncthreads();                                              // the scores are read
    }
}

// Statistics over THREADS threads, valid in thread 0.
template <int THREADS, typename A>
__device__ __forceinline__ Stats block_stats(Stats s, double *room, A type)
{
    double m[1] = {s.m};
    block_reduce<false, THREADS>(m, room);
    s.raise(m[0], type);
    double sums[3] = {s.others, s.down, s.n};
    __syncthreads();
    block_reduce<true, THREADS>(sums, room);
    __syncthreads();
    s.m = m[0], s.others = sums[0], s.down = sums[1], s.n = sums[2];
    return s;
}

constexpr int kPart = 256;                                            // threads of a piece

template <typename T, int PACK>
__global__ __launch_bounds__(kPart) void row_stats_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    __shared__ double room[3 * kPart / kWave];
    const Classes<T, kPart, PACK> classes(a.group, a.lanes_log2);
    for (int64_t task = blockIdx.x; task < a.rows * a.pieces; task += gridDim.x) {
        const int64_t row = task / a.pieces;
        const int piece = (int)(task % a.pieces), first = piece * a.per_piece, end = first + a.per_piece < a.k ? first + a.per_piece : a.k;
        const int64_t t = target_of(a, row);
        Stats s;
        if (t >= 0 && t < a.k) {
            classes.sums(static_cast<const T *>(a.x) + row * a.stride, first, end, [&](int c, double sum, bool mine) {
                if (!mine) return;
                const double v = sum * a.inv_tau;
                if (c == t) a.target_score[row] = v;
                s.add(v, c == t, A());
            });
            s = block_stats<kPart>(s, room, A());
        }
        if (threadIdx.x == 0) s.store(a.stats + 4 * ((int64_t)piece * a.rows + row));
    }
}

// The statistics of a row's pieces into M, O, Z and the loss: a thread per row.  (One workgroup also counts the rows.)
__global__ __launch_bounds__(1024) void join_kernel(CeArgs a, int dtype)
{
    __shared__ double room[16];
    const double per = per_row<1024>(a, room);
    if (a.count == 1 && threadIdx.x == 0) *a.per_count = per;
    const int64_t row = (int64_t)blockIdx.x * 1024 + threadIdx.x;
    if (row >= a.rows) return;
    const int64_t t = target_of(a, row);
    double loss = t < 0 ? 0.0 : __builtin_nan("");
    if (t >= 0 && t < a.k) {
        Stats s;
        const auto join = [&](auto type) {
            for (int p = 0; p < a.pieces; ++p) s.join(Stats::load(a.stats + 4 * ((int64_t)p * a.rows + row)), type);
            return (double)exp_of(a.target_score[row], s.m, type);
        };
        const double of_target = dtype == CLG_F64 ? join(double()) : join(float());
        if (__builtin_isinf(s.m)) s.others = __builtin_nan("");
        const Row r{s.m, s.others, s.others + of_target};
        loss = r.loss(a.target_score[row], s.down, a.k, a.smoothing) * a.scale * per;
        if (a.final) a.final[3 * row] = r.m, a.final[3 * row + 1] = r.others, a.final[3 * row + 2] = r.total;
    }
    if (a.row_loss) a.row_loss[row] = loss;
    if (a.out && dtype == CLG_F64) static_cast<double *>(a.out)[row] = loss;
    else if (a.out) static_cast<float *>(a.out)[row] = (float)loss;
}

// Gradient of a row from its M, O and Z.
template <typename A>
__device__ __forceinline__ Grad grad_of(const CeArgs &a, int64_t row)
{
    const Row r{a.final[3 * row], a.final[3 * row + 1], a.final[3 * row + 2]};
    const double up = a.upstream ? (double)static_cast<const A *>(a.upstream)[a.reduction == CLG_REDUCE_NONE ? row : 0] : 1.0;
    return Grad(r, a.scale * (a.count ? *a.per_count : 1.0) * a.inv_tau * up, a.smoothing, a.k);
}

template <typename T, int PACK>
__global__ __launch_bounds__(kPart) void row_grad_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    if (nothing_to_do<A>(a)) return;
    const Classes<T, kPart, PACK> classes(a.group, a.lanes_log2);
    for (int64_t task = blockIdx.x; task < a.rows * a.pieces; task += gridDim.x) {
        const int64_t row = task / a.pieces;
        const int piece = (int)(task % a.pieces), first = piece * a.per_piece, end = first + a.per_piece < a.k ? first + a.per_piece : a.k;
        const int64_t t = target_of(a, row);
        T *grad = static_cast<T *>(a.grad) + row * ((int64_t)a.k * a.group);
        if (t < 0 || t >= a.k) {
            const A v = t < 0 ? A(0) : (A)__builtin_nan("");
            classes.store(grad, first, end, [&](int) { return v; });
            continue;
        }
        const Grad g = grad_of<A>(a, row);
        const double m = a.final[3 * row];
        const A factor = (A)g.factor, off = (A)g.off, target = (A)g.target;
        classes.sums(static_cast<const T *>(a.x) + row * a.stride, first, end, [&](int c, double sum, bool) {
            const A v = c == t ? target : __builtin_elementwise_fma(exp_of(sum * a.inv_tau, m, A()), factor, -off);
            if constexpr (PACK == 0) {
                classes.fill(grad + (int64_t)c * a.group, (T)v);
            } else {
#pragma unroll
                for (int j = 0; j < PACK; ++j) grad[(int64_t)c * PACK + j] = (T)v;
            }
        });
    }
}

// ---- columns: x [k G][rows] ----------------------------------------------------------------------------------------------------
// A wavefront has 1 << lanes_log2 samples side by side and, beside them, as many features of a class as its lanes hold; the wavefronts of a workgroup have a class each.
struct Column {
    int64_t row;                                                      // sample
    int sub, subs, wave;
    bool live;
    __device__ __forceinline__ explicit Column(const CeArgs &a)
    {
        const int lane = threadIdx.x & 63;
        row = ((int64_t)blockIdx.x << a.lanes_log2) + (lane & ((1 << a.lanes_log2) - 1));
        sub = lane >> a.lanes_log2, subs = 64 >> a.lanes_log2, wave = uniform(threadIdx.x >> 6);
        live = row < a.rows;
        if (!live) row = a.rows - 1;
    }
};
template <typename T>
__device__ __forceinline__ double column_sum(const CeArgs &a, const Column &col, int64_t from, int64_t to)
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
// statistics of the workgroup's wavefronts, a sample each lane
template <typename A>
__device__ __forceinline__ void store_stats(const CeArgs &a, const Column &col, const Stats &s, double (&room)[kPart / kWave][kWave][4], A type)
{
    s.store(room[col.wave][threadIdx.x & 63]);
    __syncthreads();
    if (col.wave != 0 || col.sub != 0 || !col.live) return;
    Stats all = s;
    for (int w = 1; w < kPart / kWave; ++w) all.join(Stats::load(room[w][threadIdx.x & 63]), type);
    all.store(a.stats + 4 * ((int64_t)blockIdx.y * a.rows + col.row));
}

// Sums over the features of a class, or a slice of them; statistics of the classes of a piece where the sums are whole.
template <typename T>
__global__ __launch_bounds__(kPart) void column_sums_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    __shared__ double room[kPart / kWave][kWave][4];
    const Column col(a);
    const int first = (int)blockIdx.y * a.per_piece, end = first + a.per_piece < a.k ? first + a.per_piece : a.k, slice = blockIdx.z;
    const int64_t from = (int64_t)a.group * slice / a.slices, to = (int64_t)a.group * (slice + 1) / a.slices;
    const int64_t t = target_of(a, col.row);
    Stats s;
    for (int c = first + col.wave; c < end; c += kPart / kWave) {
        const double sum = column_sum<T>(a, col, (int64_t)c * a.group + from, (int64_t)c * a.group + to);
        if (a.slices > 1) {
            if (col.live && col.sub == 0) a.partial[((int64_t)slice * a.k + c) * a.rows + col.row] = sum;
            continue;
        }
        const double v = sum * a.inv_tau;
        if (col.live && col.sub == 0) {
            if (a.scores) a.scores[(int64_t)c * a.rows + col.row] = v;
            if (c == t) a.target_score[col.row] = v;
        }
        s.add(v, c == t, A());
    }
    if (a.slices == 1) store_stats(a, col, s, room, A());
}
// the same from the sums of the slices
template <typename A>
__global__ __launch_bounds__(kPart) void column_stats_kernel(CeArgs a)
{
    __shared__ double room[kPart / kWave][kWave][4];
    const Column col(a);
    const int first = (int)blockIdx.y * a.per_piece, end = first + a.per_piece < a.k ? first + a.per_piece : a.k;
    const int64_t t = target_of(a, col.row);
    Stats s;
    for (int c = first + col.wave; c < end; c += kPart / kWave) {
        double sum = 0;
#pragma unroll 8
        for (int i = col.sub; i < a.slices; i += col.subs) sum += a.partial[((int64_t)i * a.k + c) * a.rows + col.row];
        for (int by = 1 << a.lanes_log2; by < 64; by <<= 1) sum += __shfl_xor(sum, by);
        const double v = sum * a.inv_tau;
        if (col.live && col.sub == 0) {
            a.scores[(int64_t)c * a.rows + col.row] = v;
            if (c == t) a.target_score[col.row] = v;
        }
        s.add(v, c == t, A());
    }
    store_stats(a, col, s, room, A());
}
// Gradient from the scores, or from the features again.
template <typename T>
__global__ __launch_bounds__(kPart) void column_grad_kernel(CeArgs a)
{
    typedef typename Wide<T>::type A;
    if (nothing_to_do<A>(a)) return;
    const Column col(a);
    const int first = (int)blockIdx.y * a.per_piece, end = first + a.per_piece < a.k ? first + a.per_piece : a.k, slice = blockIdx.z;
    const int64_t from = (int64_t)a.group * slice / a.slices, to = (int64_t)a.group * (slice + 1) / a.slices;
    const int64_t t = target_of(a, col.row);
    const bool counts = t >= 0 && t < a.k;
    const Grad g = grad_of<A>(a, counts ? col.row : 0);
    const double m = a.final[3 * col.row];
    const A factor = (A)g.factor, off = (A)g.off, target = (A)g.target;
    T *grad = static_cast<T *>(a.grad) + col.row;
    for (int c = first + col.wave; c < end; c += kPart / kWave) {
        const double s = a.scores ? a.scores[(int64_t)c * a.rows + col.row] : column_sum<T>(a, col, (int64_t)c * a.group, (int64_t)(c + 1) * a.group) * a.inv_tau;
        A v = c == t ? target : __builtin_elementwise_fma(exp_of(s, m, A()), factor, -off);
        if (!counts) v = t < 0 ? A(0) : (A)__builtin_nan("");
        if (!col.live) continue;
        const T u = (T)v;
        for (int64_t i = (int64_t)c * a.group + from + col.sub; i < (int64_t)c * a.group + to; i += col.subs) grad[i * a.rows] = u;
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

// How a call goes, by its sizes alone.
struct Plan {
    bool rows, whole;                                                 // layout; a workgroup per row
    int64_t n, k, group, features;
    int size;                                                         // bytes of an element
    int lanes_log2, pieces, per_piece, slices;
    bool scores, kept_scores;                                         // "columns"
};
int log2_up(int64_t v)
{
    int l = 0;
    while ((1ll << l) < v) ++l;
    return l;
}
int packed(const Plan &p)
{
    const int e = 16 / p.size;
    return p.group <= e && e % p.group == 0 ? (int)p.group : 0;
}
Plan plan_of(int dtype, bool rows, int64_t n, int64_t features, int64_t k)
{
    Plan p{rows, false, n, k, features / k, features, clg_elem_bytes(dtype), 0, 1, (int)k, 1, false, false};
    const auto cut = [&](int64_t pieces, int64_t unit) {              // pieces of a multiple of `unit` classes
        const int64_t each = clg_ceil_div(clg_ceil_div(k, pieces < 1 ? 1 : pieces), unit) * unit;
        p.per_piece = (int)(each < k ? each : k);
        p.pieces = (int)clg_ceil_div(k, p.per_piece);
    };
    if (rows) {
        const int64_t pieces = clg_ceil_div(p.group, 16 / p.size);    // of a class; a lane takes about four
        p.lanes_log2 = pieces <= 4 ? 0 : log2_up(clg_ceil_div(pieces, 4));
        if (p.lanes_log2 > 6) p.lanes_log2 = 6;
        const int64_t lds = k * (dtype == CLG_F64 ? 8 : 4);
        p.whole = lds <= kLds && (n >= 128 || features * p.size <= 64 << 10);
        // else about 1024 workgroups, of 16 KiB of features at least
        int64_t want = clg_ceil_div(1024, n), most = clg_ceil_div(features * p.size, 16 << 10);
        cut(want < most ? want : most, 16);
    } else {
        p.lanes_log2 = log2_up(n < 64 ? n : 64);
        const int64_t chunks = clg_ceil_div(n, 1ll << p.lanes_log2), want = clg_ceil_div(1024, chunks);
        cut(want < clg_ceil_div(k, 4) ? want : clg_ceil_div(k, 4), 4);
        const int64_t slices = clg_ceil_div(1024, chunks * p.pieces), most = p.group / 64;
        p.slices = (int)(slices < most ? slices : most);
        if (p.slices < 1) p.slices = 1;
        if (p.slices > 64) p.slices = 64;
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
    r.final = take(kept, 3 * p.n);
    if (p.kept_scores) r.scores = take(kept, p.k * p.n);
    const int64_t bytes = at * 8;
    at = 0;
    r.row_loss = take(scratch, p.n);
    take(scratch, clg_ceil_div(p.n, kSlice));
    if (!p.whole) {
        r.target_score = take(scratch, p.n);
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

unsigned blocks(int64_t n) { return (unsigned)(n < kMostBlocks ? n : kMostBlocks); }

template <typename T, int THREADS, int PACK>
int launch_rows(const char *name, const CeArgs &a, hipStream_t stream)
{
    const size_t lds = a.k * sizeof(typename Wide<T>::type);
    if (lds > 48 << 10) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(rows_kernel<T, THREADS, PACK>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) {
            clg_set_error("%s: %s", name, hipGetErrorString(e));
            return CLG_ELAUNCH;
        }
    }
    rows_kernel<T, THREADS, PACK><<<dim3(blocks(a.rows)), dim3(THREADS), lds, stream>>>(a);
    CLG_CHECK_LAUNCH(name);
    return CLG_OK;
}

template <typename T>
int forward(const char *name, const Plan &p, CeArgs a, int dtype, hipStream_t stream)
{
    int rc = CLG_OK;
    if (p.rows && p.whole) {
        with_pack<T>(packed(p), [&](auto pack) {
            constexpr int PACK = decltype(pack)::value;
            if (p.features <= 2048) rc = launch_rows<T, 64, PACK>(name, a, stream);
            else if (p.features <= 16384) rc = launch_rows<T, 256, PACK>(name, a, stream);
            else rc = launch_rows<T, 1024, PACK>(name, a, stream);
        });
        return rc;
    }
    const dim3 columns((unsigned)clg_ceil_div(p.n, 1ll << p.lanes_log2), (unsigned)p.pieces, (unsigned)p.slices);
    if (p.rows) {
        with_pack<T>(packed(p), [&](auto pack) { row_stats_kernel<T, decltype(pack)::value><<<dim3(blocks(p.n * p.pieces)), dim3(kPart), 0, stream>>>(a); });
    } else {
        column_sums_kernel<T><<<columns, dim3(kPart), 0, stream>>>(a);
        CLG_CHECK_LAUNCH(name);
        if (p.slices > 1) column_stats_kernel<typename Wide<T>::type><<<dim3(columns.x, columns.y), dim3(kPart), 0, stream>>>(a);
    }
    CLG_CHECK_LAUNCH(name);
    join_kernel<<<dim3((unsigned)clg_ceil_div(p.n, 1024)), dim3(1024), 0, stream>>>(a, dtype);
    CLG_CHECK_LAUNCH(name);
    return CLG_OK;
}
template <typename T>
int gradient(const char *name, const Plan &p, const CeArgs &a, hipStream_t stream)
{
    if (p.rows) with_pack<T>(packed(p), [&](auto pack) { row_grad_kernel<T, decltype(pack)::value><<<dim3(blocks(p.n * p.pieces)), dim3(kPart), 0, stream>>>(a); });
    else column_grad_kernel<T><<<dim3((unsigned)clg_ceil_div(p.n, 1ll << p.lanes_log2), (unsigned)p.pieces, (unsigned)p.slices), dim3(kPart), 0, stream>>>(a);
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
    CLG_REQUIRE(!rows || (kept && scratch), "%s: null workspace", name);
    CLG_REQUIRE(!grad || reduction != CLG_REDUCE_NONE, "%s: the gradient of a loss per row is clg_group_ce_backward's", name);
    hipStream_t st = clg_stream(stream);
    if (!rows) return reduction == CLG_REDUCE_NONE ? CLG_OK : sum_rows(name, dtype, nullptr, 0, nullptr, nullptr, loss, st);
    const Plan p = plan_of(dtype, row_stride >= 0, rows, features, k);
    CeArgs a = args_of(p, x, row_stride, targets, targets_bits, tau, smoothing, weight, reduction);
    rooms_of(p, &a, kept, scratch);
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
    if (p.whole) a.grad = grad;
    int rc = clg_with_type(dtype, [&](auto t) { return forward<decltype(t)>(name, p, a, dtype, st); });
    if (rc) return rc;
    if (grad && !p.whole) {
        a.grad = grad;
        if (a.count) a.count = 2;
        rc = clg_with_type(dtype, [&](auto t) { return gradient<decltype(t)>(name, p, a, st); });
        if (rc) return rc;
    }
    return reduction == CLG_REDUCE_NONE ? CLG_OK : sum_rows(name, dtype, row_loss, rows, row_loss + rows, nullptr, loss, st);
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
