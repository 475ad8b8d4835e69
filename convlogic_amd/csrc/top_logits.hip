// The k highest logits of each row in descending order, the columns they are in (of equal ones the lowest, NaN above everything) and the logsumexp of the
// whole row, in one pass over the logits.
//
// No row is sorted.  The k-th highest of the threads' own maxima is a value that at least k elements reach, and hardly more do: they alone are written
// to LDS, where each counts the candidates before it.  Rows with more candidates than room (equal values, the highest next to one another) find the
// threshold bit by bit instead.
#include "row_tile.h"

namespace {

// values as integers in the same order: -0 and +0 equal, NaN on top; 0 is below every value
__device__ __forceinline__ uint32_t ordered(float v)
{
    const uint32_t u = __builtin_bit_cast(uint32_t, v + 0.0f);
    return v != v ? 0xFFFFFFFFu : (u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u));
}
__device__ __forceinline__ uint64_t ordered(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v + 0.0);
    return v != v ? ~0ull : (u ^ ((u >> 63) ? ~0ull : 1ull << 63));
}
__device__ __forceinline__ float value_of(uint32_t o) { return __builtin_bit_cast(float, (o >> 31) ? o ^ 0x80000000u : ~o); }
__device__ __forceinline__ double value_of(uint64_t o) { return __builtin_bit_cast(double, (o >> 63) ? o ^ (1ull << 63) : ~o); }

// candidates in the order of the answer: by value, of equal ones by column
template <typename A>
struct Cand;
template <>
struct Cand<float> {
    typedef uint32_t K;
    uint64_t v;
    __device__ __forceinline__ Cand(K key, uint32_t column) : v((uint64_t)key << 32 | ~column) {}
    __device__ __forceinline__ uint32_t column() const { return ~(uint32_t)v; }
    __device__ __forceinline__ K key() const { return (K)(v >> 32); }
    __device__ __forceinline__ bool before(const Cand &o) const { return v > o.v; }
};
template <>
struct Cand<double> {
    typedef uint64_t K;
    K k;
    uint64_t c;
    __device__ __forceinline__ Cand(K key, uint32_t column) : k(key), c(column) {}
    __device__ __forceinline__ uint32_t column() const { return (uint32_t)c; }
    __device__ __forceinline__ K key() const { return k; }
    __device__ __forceinline__ bool before(const Cand &o) const { return k > o.k || (k == o.k && c < o.c); }
};

struct TopArgs {
    const void *z;
    int64_t rows, cols, row_stride;
    int k, room;                                                      // room: candidates that LDS holds
    double temperature;
    void *values;                                                     // [rows][k]
    int64_t *columns;                                                 // [rows][k]
    void *lse;                                                        // [rows] in A
};

// A value that at least `want` of the keys of a wavefront reach, the greatest or one that no more than `enough` reach.
template <int PER, typename K>
__device__ __forceinline__ K wave_threshold(const K (&x)[PER], int want, int enough)
{
    K t = 0;
#pragma unroll 1
    for (int b = 8 * sizeof(K) - 1; b >= 0; --b) {
        const K next = t | (K)1 << b;
        int n = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) n += __popcll(__ballot(x[i] >= next));
        if (n < want) continue;
        t = next;
        if (n <= enough) break;
    }
    return t;
}

// The same of all values of a workgroup: count(t) of this thread's are t or more.
template <int THREADS, typename K, typename F>
__device__ __forceinline__ K threshold(int want, int enough, double *sums, F count)
{
    K t = 0;
#pragma unroll 1
    for (int b = 8 * sizeof(K) - 1; b >= 0; --b) {
        const K next = t | (K)1 << b;
        double n[1] = {(double)count(next)};
        __syncthreads();
        block_reduce<true, THREADS>(n, sums);
        if (n[0] < want) continue;
        t = next;
        if (n[0] <= enough) break;
    }
    return t;
}

template <typename C>
size_t top_lds(int threads, int room, int best)
{
    return 16 * 8 + 16 + (size_t)(room + best) * sizeof(C) + (size_t)threads * sizeof(typename C::K);
}

// One workgroup per row.  MULTI: rows that its registers do not hold go tile by tile, the k best so far in front of each tile's candidates.
template <typename T, int THREADS, int NV, bool MULTI>
__global__ __launch_bounds__(THREADS, 4) void top_kernel(TopArgs a)
{
    typedef typename Wide<T>::type A;
    typedef Cand<A> C;
    typedef typename C::K K;
    typedef RowTile<T, THREADS, NV> Tile;
    extern __shared__ char lds[];
    double *sums = reinterpret_cast<double *>(lds);                   // 16
    K *shared = reinterpret_cast<K *>(sums + 16);                     // the threshold
    int *count = reinterpret_cast<int *>(sums + 17);
    C *cand = reinterpret_cast<C *>(sums + 18), *best = cand + a.room, *next = best + a.k;            // (best, next: MULTI)
    K *maxima = reinterpret_cast<K *>(best + (MULTI ? 2 * a.k : 0));
    const int tid = threadIdx.x, k = a.k;
    const A unit = (A)Exps<A>::unit(a.temperature);
    const int64_t row = blockIdx.x;
    const T *z = static_cast<const T *>(a.z) + row * a.row_stride;

    A m_t = lowest(A(0)), s_t = 0;
    int have = 0;                                                     // in best
#pragma unroll 1
    for (int64_t base = 0; base < a.cols; base += Tile::COLS) {
        Tile tile;
        tile.load(z, base, a.cols);
        const int n = (int)(a.cols - base < Tile::COLS ? a.cols - base : Tile::COLS);
        const A mine = tile.highest();
        if (have == 0) maxima[tid] = ordered(mine);
        if (tid == 0) *count = 0;
        tile.fence();
        const A m = max_of(m_t, mine);
        const Exps<A> e(m, unit);
        if (MULTI) s_t = rescaled(s_t, m_t, Exps<A>(m_t, unit), e);
        s_t += tile.sum(e);
        m_t = m;
        const bool nan = s_t != s_t;                                  // (of this thread, now or in an earlier tile; it is in no maximum)
        tile.fence();
        __syncthreads();
        // what has to be exceeded
        K from;
        if (have) from = best[k - 1].key();                           // (a later column has to be higher than the k-th, not equal)
        else {
            if (tid < kWave) {
                constexpr int PER = THREADS / kWave;
                K x[PER];
#pragma unroll
                for (int i = 0; i < PER; ++i) x[i] = maxima[i * kWave + tid];
                const K t = wave_threshold(x, k, k + k / 4);
                if (tid == 0) *shared = t - (t != 0);
            }
            __syncthreads();
            from = *shared;
        }
        const A least = value_of((K)(from + (from != ~(K)0)));
        const bool all = from < ordered(lowest(A(0))) || nan;
        const auto collect = [&](auto wanted) {
            tile.pieces([&](A high, auto each) {
                if (high >= least || all)
                    each([&](A x, int c) {
                        const K o = ordered(x);
                        if (wanted(o, c)) {
                            const int i = atomicAdd(count, 1);
                            if (i < a.room) cand[i] = C(o, (uint32_t)(base + c));
                        }
                    });
            });
        };
        collect([&](K o, int) { return o > from; });
        __syncthreads();
        int found = *count;
        if (found > a.room) {
            // more than there is room for: the value that at least k reach, then the last column of those that equal it
            const K value = threshold<THREADS, K>(k, a.room, sums, [&](K t) {
                int c_t = 0;
                tile.each([&](T x, int) { c_t += ordered((A)x) >= t; });
                tile.fence();
                return c_t;
            });
            double reach[2] = {0, 0};
            tile.each([&](T x, int) {
                const K o = ordered((A)x);
                reach[0] += o > value;
                reach[1] += o == value;
            });
            tile.fence();
            __syncthreads();
            block_reduce<true, THREADS>(reach, sums);
            uint32_t last = ~0u;                                      // equal ones up to this column of the tile
            if (reach[0] + reach[1] > a.room) {
                // (columns counted from the end, so that those that reach a threshold are the lowest)
                last = ~threshold<THREADS, uint32_t>(k - (int)reach[0], k - (int)reach[0], sums, [&](uint32_t t) {
                    int c_t = 0;
                    tile.each([&](T x, int c) { c_t += ordered((A)x) == value && ~(uint32_t)c >= t; });
                    tile.fence();
                    return c_t;
                });
            }
            __syncthreads();
            if (tid == 0) *count = 0;
            __syncthreads();
            collect([&](K o, int c) { return o > value || (o == value && (uint32_t)c <= last); });
            __syncthreads();
            found = *count;
        }
        // ranks: earlier tiles' best, then the candidates
        const bool end = !MULTI || base + Tile::COLS >= a.cols;
#pragma unroll 1
        for (int i = tid; i < have + found; i += THREADS) {
            const C mine = i < have ? best[i] : cand[i - have];
            int rank = 0;
            for (int j = 0; j < have; ++j) rank += best[j].before(mine);
            for (int j = 0; j < found; ++j) rank += cand[j].before(mine);
            if (rank >= k) continue;
            if (end) {
                static_cast<T *>(a.values)[row * k + rank] = z[mine.column()];
                a.columns[row * k + rank] = mine.column();
            } else if (MULTI) {
                next[rank] = mine;
            }
        }
        if (MULTI) {
            __syncthreads();
            C *const spare = best;
            best = next, next = spare;
            have = k;
        }
    }
    if (!a.lse) return;
    A top[1] = {m_t};
    __syncthreads();
    block_reduce<false, THREADS>(top, reinterpret_cast<A *>(sums));
    const Exps<A> e(top[0], unit);
    double s[1] = {(double)rescaled(s_t, m_t, Exps<A>(m_t, unit), e)};
    __syncthreads();
    block_reduce<true, THREADS>(s, sums);
    if (tid == 0) static_cast<A *>(a.lse)[row] = (A)((double)finite_or_zero(top[0]) / a.temperature + log(s[0]) + e.residue(top[0]));
}

template <typename T, int THREADS, int NV, bool MULTI>
void launch_as(TopArgs a, hipStream_t stream)
{
    // (up to 64 KB of LDS: 1024 entries of a long row are 48 KB, in float64 60)
    if (sizeof(T) == 8) a.room = a.k <= 128 ? 256 : a.k <= 512 ? 2 * a.k : a.k + a.k / 2;
    else a.room = a.k <= 64 ? 256 : 4 * a.k;
    const size_t lds = top_lds<Cand<typename Wide<T>::type>>(THREADS, a.room, MULTI ? 2 * a.k : 0);
    top_kernel<T, THREADS, NV, MULTI><<<dim3((unsigned)a.rows), dim3(THREADS), lds, stream>>>(a);
}

template <typename T>
void launch(const TopArgs &a, hipStream_t stream)
{
    const int64_t pieces = (a.cols + Vec16<T>::N - 1) / Vec16<T>::N;
    if (pieces <= 64) return launch_as<T, 64, 1, false>(a, stream);
    if (pieces <= 64 * 4) return launch_as<T, 64, 4, false>(a, stream);
    if (pieces <= 256 * 4) return launch_as<T, 256, 4, false>(a, stream);
    if (pieces <= 256 * 16) return launch_as<T, 256, 16, false>(a, stream);
    if (pieces <= 512 * 16) return launch_as<T, 512, 16, false>(a, stream);
    if (pieces <= 1024 * 16) return launch_as<T, 1024, 16, false>(a, stream);
    launch_as<T, 512, 8, true>(a, stream);
}

constexpr int kMaxTop = 1024;

}  // namespace

extern "C" int clg_top_logits(int dtype, const void *logits, int64_t row_stride, int64_t rows, int64_t cols, int64_t k, double temperature, void *values,
                              int64_t *columns, void *lse, void *stream)
{
    CLG_REQUIRE(clg_score_type(dtype), "clg_top_logits: unsupported dtype %d", dtype);
    CLG_REQUIRE(rows >= 0 && rows < (int64_t)1 << 31 && cols >= 1 && cols < (int64_t)1 << 31, "clg_top_logits: bad shape [%lld, %lld]", (long long)rows,
                (long long)cols);
    CLG_REQUIRE(k >= 1 && k <= kMaxTop && k <= cols, "clg_top_logits: 1 to %d logits of %lld, got %lld", kMaxTop, (long long)cols, (long long)k);
    CLG_REQUIRE(row_stride >= 0, "clg_top_logits: negative row stride");
    CLG_REQUIRE(temperature > 0 && temperature < 1e30, "clg_top_logits: the temperature must be positive and finite");
    if (!rows) return CLG_OK;
    CLG_REQUIRE(logits && values && columns, "clg_top_logits: null pointer");
    TopArgs a{logits, rows, cols, row_stride, (int)k, 0, temperature, values, columns, lse};
    const int rc = clg_with_type(dtype, [&](auto t) {
        launch<decltype(t)>(a, clg_stream(stream));
        return CLG_OK;
    });
    if (rc) return rc;
    CLG_CHECK_LAUNCH("clg_top_logits");
    return CLG_OK;
}
