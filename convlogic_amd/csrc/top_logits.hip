// The k highest logits of each row in descending order, the columns they are in (of equal ones the lowest, NaN above everything) and the logsumexp of the
// whole row, in one pass over the logits.
//
// No row is sorted.  The k-th highest of the threads' own maxima is a value that at least k elements reach, and hardly more do: they alone are written
// to LDS, where each counts the candidates before it.  Rows with more candidates than room (equal values, ascending order) find the
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
template <typename A>
struct Key {
    typedef uint32_t type;
};
template <>
struct Key<double> {
    typedef uint64_t type;
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

// Greatest t that at least `want` of the workgroup's values reach, or any such t that no more than `enough` reach: count(t) values of this thread
// are t or more.
template <int THREADS, typename K, typename F>
__device__ __forceinline__ K search(int want, int enough, double *sums, F count)
{
    K t = 0;
    for (int b = 8 * sizeof(K) - 1; b >= 0; --b) {
        const K next = t | (K)1 << b;
        double n[1] = {(double)count(next)};
        __syncthreads();
        block_reduce<true, THREADS>(n, sums);
        if (n[0] >= want) t = next;
        if (n[0] >= want && n[0] <= enough) break;
    }
    return t;
}

// One workgroup per row.  MULTI: rows that its registers do not hold go tile by tile, the k best so far before each tile's candidates.
template <typename T, int THREADS, int NV, bool MULTI>
__global__ __launch_bounds__(THREADS) void top_kernel(TopArgs a)
{
    typedef typename Wide<T>::type A;
    typedef typename Key<A>::type K;
    typedef RowTile<T, THREADS, NV> Tile;
    extern __shared__ char lds[];
    double *sums = reinterpret_cast<double *>(lds);                   // 16
    int *count = reinterpret_cast<int *>(sums + 16);                  // (2 words)
    K *cand = reinterpret_cast<K *>(sums + 17), *best = cand + a.room;                // candidates; the best so far, twice (MULTI)
    uint32_t *at = reinterpret_cast<uint32_t *>(best + (MULTI ? 2 * a.k : 0)), *best_at = at + a.room;
    const int tid = threadIdx.x, k = a.k;
    K *next = best + k;
    uint32_t *next_at = best_at + k;
    const A scale = exp_scale<A>(a.temperature);
    const int64_t row = blockIdx.x;
    const T *z = static_cast<const T *>(a.z) + row * a.row_stride;

    A m_t = lowest(A(0)), s_t = 0;
    int have = 0;                                                     // in best
    for (int64_t base = 0; base < a.cols; base += Tile::COLS) {
        Tile tile;
        tile.load(z, base, a.cols);
        const int n = (int)(a.cols - base < Tile::COLS ? a.cols - base : Tile::COLS);
        // logsumexp, and the thread's highest
        A m = lowest(A(0));
        tile.each([&](T &x, int) { m = max_of(m, (A)x); });
        const A both = max_of(m_t, m), safe = finite_or_zero(both);
        if (MULTI) s_t = rescaled(s_t, m_t, both, scale);
        tile.each([&](T &x, int) { s_t += exp_scaled((A)x - safe, scale); });
        m_t = both;
        const bool nan = s_t != s_t;                                  // (NaN of this thread, now or in an earlier tile)
        // the threshold
        K from;
        if (have == k) from = best[k - 1];                            // (later columns have to be higher than the k-th, not equal)
        else {
            const K mine = nan ? ~(K)0 : ordered(m);
            from = search<THREADS, K>(k, k + k / 4, sums, [&](K t) { return mine >= t; });
            from -= from != 0;
        }
        // what is above it
        __syncthreads();
        if (tid == 0) *count = 0;
        __syncthreads();
        tile.each([&](T &x, int c) {
            const K o = ordered((A)x);
            if (o > from && c < n) {
                const int i = atomicAdd(count, 1);
                if (i < a.room) cand[i] = o, at[i] = (uint32_t)(base + c);
            }
        });
        __syncthreads();
        int found = *count;
        if (found > a.room) {
            // more than there is room for: the value that at least k reach, then the last column of those that equal it
            const K value = search<THREADS, K>(k, a.room, sums, [&](K t) {
                int c_t = 0;
                tile.each([&](T &x, int c) { c_t += c < n && ordered((A)x) >= t; });
                return c_t;
            });
            double reach[2] = {0, 0};
            tile.each([&](T &x, int c) {
                const K o = ordered((A)x);
                reach[0] += c < n && o > value;
                reach[1] += c < n && o == value;
            });
            __syncthreads();
            block_reduce<true, THREADS>(reach, sums);
            uint32_t last = ~0u;                                      // equal ones up to this column of the tile
            if (reach[0] + reach[1] > a.room) {
                const uint32_t less = search<THREADS, uint32_t>(k - (int)reach[0], k - (int)reach[0], sums, [&](uint32_t t) {
                    int c_t = 0;                                      // (columns counted from the end, so that t or more are the lowest columns)
                    tile.each([&](T &x, int c) { c_t += c < n && ordered((A)x) == value && ~(uint32_t)c >= t; });
                    return c_t;
                });
                last = ~less;
            }
            __syncthreads();
            if (tid == 0) *count = 0;
            __syncthreads();
            tile.each([&](T &x, int c) {
                const K o = ordered((A)x);
                if (c < n && (o > value || (o == value && (uint32_t)c <= last))) {
                    const int i = atomicAdd(count, 1);
                    if (i < a.room) cand[i] = o, at[i] = (uint32_t)(base + c);
                }
            });
            __syncthreads();
            found = *count;
        }
        // ranks: earlier tiles' best, then the candidates
        const bool end = !MULTI || base + Tile::COLS >= a.cols;
        for (int i = tid; i < have + found; i += THREADS) {
            const K mine = i < have ? best[i] : cand[i - have];
            const uint32_t c = i < have ? best_at[i] : at[i - have];
            int rank = 0;
            for (int j = 0; j < have; ++j) rank += best[j] > mine || (best[j] == mine && best_at[j] < c);
            for (int j = 0; j < found; ++j) rank += cand[j] > mine || (cand[j] == mine && at[j] < c);
            if (rank >= k) continue;
            if (end) {
                static_cast<T *>(a.values)[row * k + rank] = z[c];
                a.columns[row * k + rank] = c;
            } else if (MULTI) {
                next[rank] = mine, next_at[rank] = c;
            }
        }
        if (MULTI) {
            __syncthreads();
            K *const spare = best;
            uint32_t *const spare_at = best_at;
            best = next, best_at = next_at, next = spare, next_at = spare_at;
            have = k;
        }
    }
    if (!a.lse) return;
    A top[1] = {m_t};
    __syncthreads();
    block_reduce<false, THREADS>(top, reinterpret_cast<A *>(sums));
    double s[1] = {(double)rescaled(s_t, m_t, top[0], scale)};
    __syncthreads();
    block_reduce<true, THREADS>(s, sums);
    if (tid == 0) static_cast<A *>(a.lse)[row] = (A)((double)finite_or_zero(top[0]) / a.temperature + log(s[0]));
}

template <typename T, int THREADS, int NV, bool MULTI>
void launch_as(TopArgs a, hipStream_t stream)
{
    typedef typename Key<typename Wide<T>::type>::type K;
    a.room = a.k <= 128 ? 256 : 2 * a.k;
    const size_t lds = 17 * 8 + (size_t)(a.room + (MULTI ? 2 * a.k : 0)) * (sizeof(K) + 4);
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
    if (pieces <= 1024 * 8) return launch_as<T, 1024, 8, false>(a, stream);
    if (pieces <= 1024 * 16) return launch_as<T, 1024, 16, false>(a, stream);
    launch_as<T, 1024, 8, true>(a, stream);
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
