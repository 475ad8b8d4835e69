// The k highest logits of each row in descending order, the columns they are in (of equal ones the lowest, NaN above everything) and the logsumexp of the
// whole row, in one pass over the logits.
//
// No row is sorted.  A workgroup goes over its row in tiles, the next one on its way while it looks at one, and each thread keeps the maximum of what it
// has seen: the k-th highest of these is a value that at least k elements reach, and of a random row hardly more do.  It is found anew after 1, 2, 4, ...
// tiles and at the end.  The pass itself only notes which 16-byte pieces reach it; at the end these are read again, each of their elements that
// reaches the last value is a candidate, and each candidate counts those before it.  Where pieces or candidates become more than there is room for, the
// best k so far are kept and the lowest of those is what has to be exceeded from then on.
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
    int k;
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

// Maxima that the first threshold is made of: the threads' own, or of each piece where k is more than a third of the threads.
template <int THREADS, int NV>
__host__ __device__ __forceinline__ bool of_pieces(int k)
{
    return NV > 1 && 3 * k > THREADS;
}

constexpr int kSpare = 512;                                           // candidates that there is room for beside the k best
constexpr int kNoted = 512;                                           // pieces that may be noted when a tile begins

// LDS of a workgroup: reduction room, counters, candidates, the best k, maxima, noted pieces
template <typename T, int THREADS, int NV>
struct TopRoom {
    typedef Cand<typename Wide<T>::type> C;
    int room, maxima, notes;
    size_t bytes;
    __host__ __device__ explicit TopRoom(int k)
        : room(k + (k > kSpare ? k : kSpare)), maxima(THREADS * (of_pieces<THREADS, NV>(k) ? NV : 1)), notes(THREADS * NV + Vec16<T>::N + kNoted),
          bytes(18 * 8 + (size_t)(room + k) * sizeof(C) + (size_t)maxima * sizeof(typename C::K) + (size_t)notes * 4)
    {
    }
};

// One workgroup per row; MULTI: of more than one tile.
template <typename T, int THREADS, int NV, bool MULTI>
__global__ __launch_bounds__(THREADS) void top_kernel(TopArgs a)
{
    typedef typename Wide<T>::type A;
    typedef Cand<A> C;
    typedef typename C::K K;
    typedef RowTile<T, THREADS, NV> Tile;
    extern __shared__ char lds[];
    const TopRoom<T, THREADS, NV> size(a.k);
    double *sums = reinterpret_cast<double *>(lds);                   // of 16 wavefronts
    K *shared = reinterpret_cast<K *>(sums + 16);                     // the threshold
    int *noted = reinterpret_cast<int *>(sums + 17), *count = noted + 1;
    C *cand = reinterpret_cast<C *>(sums + 18), *best = cand + size.room;
    K *maxima = reinterpret_cast<K *>(best + a.k);
    uint32_t *note = reinterpret_cast<uint32_t *>(maxima + size.maxima);             // first columns
    const int tid = threadIdx.x, k = a.k;
    const A unit = (A)Exps<A>::unit(a.temperature);
    const int64_t row = blockIdx.x;
    const T *z = static_cast<const T *>(a.z) + row * a.row_stride;
    const int64_t whole = a.cols / Tile::VEC * Tile::VEC;

    int found = 0;                                                    // candidates
    C from(0, 0);                                                     // what a candidate has to be before

    // the candidates that have less than k before them, to where f(candidate, how many) puts them
    const auto rank = [&](auto f) {
#pragma unroll 1
        for (int i = tid; i < found; i += THREADS) {
            const C mine = cand[i];
            int before = 0;
#pragma unroll 8
            for (int j = 0; j < found; ++j) before += cand[j].before(mine);
            if (before < k) f(mine, before);
        }
    };
    const auto keep_best = [&]() {
        if (found <= k) return;
        rank([&](C c, int at) { best[at] = c; });
        __syncthreads();
        for (int j = tid; j < k; j += THREADS) cand[j] = best[j];
        if (best[k - 1].before(from)) from = best[k - 1];
        found = k;
    };
    // the elements of noted pieces i0 .. i0 + n - 1 that are candidates, behind those that are there; how many there would be in all
    const auto take = [&](int i0, int n) {
        if (tid == 0) *count = found;
        __syncthreads();
#pragma unroll 1
        for (int i = i0 + tid; i < i0 + n; i += THREADS) {
            const uint32_t c = note[i];
            const bool piece = c < whole;
            typename Tile::V v;
            if (piece) v = *reinterpret_cast<const typename Tile::V *>(z + c);
            else v[0] = z[c];
#pragma unroll
            for (int e = 0; e < Tile::VEC; ++e) {
                const C mine(ordered((A)v[e]), c + e);
                if ((e == 0 || piece) && mine.before(from)) {
                    const int at = atomicAdd(count, 1);
                    if (at < size.room) cand[at] = mine;
                }
            }
        }
        __syncthreads();
        const int now = *count;
        __syncthreads();
        return now;
    };
    // all noted pieces to candidates
    const auto take_all = [&](int n) {
        int most = n;
#pragma unroll 1
        for (int i = 0; i < n;) {
            int some = n - i < most ? n - i : most;
            int now = take(i, some);
            if (now > size.room) {                                    // too many: the best k, and as many pieces as there is room for in any case
                keep_best();
                most = kSpare / Tile::VEC;
                some = some < most ? some : most;
                now = take(i, some);
            }
            found = now < size.room ? now : size.room;
            i += some;
        }
    };

    A m_t = lowest(A(0)), s_t = 0, seen[NV];                          // seen: highest by piece, of the tiles so far
#pragma unroll
    for (int j = 0; j < NV; ++j) seen[j] = lowest(A(0));
    const bool pieces = of_pieces<THREADS, NV>(k);
    // the k-th highest of the maxima, by the first wavefront, between two barriers
    const auto show = [&]() {
        if (pieces) {
#pragma unroll
            for (int j = 0; j < NV; ++j) maxima[j * THREADS + tid] = ordered(seen[j]);
        } else {
            maxima[tid] = ordered(m_t);
        }
    };
    const auto search = [&]() {
        if (tid >= kWave) return;
        constexpr int PER = THREADS / kWave;
        K t;
        if (pieces) {
            K x[PER * NV];
#pragma unroll
            for (int i = 0; i < PER * NV; ++i) x[i] = maxima[i * kWave + tid];
            t = wave_threshold(x, k, k + k / 4);
        } else {
            K x[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) x[i] = maxima[i * kWave + tid];
            t = wave_threshold(x, k, k + k / 4);
        }
        if (tid == 0) *shared = t - (t != 0);
    };
    // (what was found of a threshold is below what the best k of candidates have given)
    const auto raise = [&]() {
        const C now(*shared, 0);
        if (now.key() > from.key()) from = now;
    };

    Tile tile, coming;
    coming.load(z, 0, a.cols);
    if (tid == 0) *noted = 0;
#pragma unroll 1
    for (int64_t base = 0, tiles = 1; base < a.cols; base += Tile::COLS, ++tiles) {
        tile = coming;
        if (MULTI && base + Tile::COLS < a.cols) coming.load(z, base + Tile::COLS, a.cols);
        A high[NV], m = max_of(m_t, (A)tile.last);
        tile.peaks(high);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            m = max_of(m, high[j]);
            seen[j] = max_of(seen[j], high[j]);
        }
        seen[0] = max_of(seen[0], (A)tile.last);
        tile.fence();
        const Exps<A> e(m, unit);
        if (MULTI) s_t = rescaled(s_t, m_t, Exps<A>(m_t, unit), e);
        s_t += tile.sum(e);
        m_t = m;
        const bool nan = s_t != s_t;                                  // (of this thread, now or in an earlier tile; it is in no maximum)
        if (base == 0) {
            show();
            __syncthreads();
            search();
            __syncthreads();
            raise();
        }
        // the pieces that matter: higher than the value of `from`, which is of an earlier column or below a threshold
        const K above = from.key();
        const A least = value_of((K)(above + (above != ~(K)0)));
        const bool all = above < ordered(lowest(A(0))) || nan;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int p = j * THREADS + tid;
            if (p < tile.whole && (high[j] >= least || all)) note[atomicAdd(noted, 1)] = (uint32_t)(base + p * Tile::VEC);
        }
        if (tid < tile.tail && ((A)tile.last >= least || all)) note[atomicAdd(noted, 1)] = (uint32_t)(base + tile.whole * Tile::VEC + tid);
        if (MULTI) {
            const bool last = base + Tile::COLS >= a.cols, anew = base && (last || (tiles & (tiles - 1)) == 0);
            if (anew) show();
            __syncthreads();
            if (anew) search();
            const int n = *noted;
            if (n > kNoted && !last) {
                take_all(n);
                keep_best();
                if (tid == 0) *noted = 0;
            }
            __syncthreads();
            if (anew) raise();
        }
    }
    if (!MULTI) __syncthreads();
    take_all(*noted);
    rank([&](C c, int i) {
        static_cast<T *>(a.values)[row * k + i] = z[c.column()];
        a.columns[row * k + i] = c.column();
    });
    if (!a.lse) return;
    A top[1] = {m_t};
    block_reduce<false, THREADS>(top, reinterpret_cast<A *>(sums));
    const Exps<A> e(top[0], unit);
    double s[1] = {(double)rescaled(s_t, m_t, Exps<A>(m_t, unit), e)};
    __syncthreads();
    block_reduce<true, THREADS>(s, sums);
    if (tid == 0) static_cast<A *>(a.lse)[row] = (A)((double)finite_or_zero(top[0]) / a.temperature + log(s[0]) + e.residue(top[0]));
}

template <typename T, int THREADS, int NV, bool MULTI>
void launch_as(const TopArgs &a, hipStream_t stream)
{
    top_kernel<T, THREADS, NV, MULTI><<<dim3((unsigned)a.rows), dim3(THREADS), TopRoom<T, THREADS, NV>(a.k).bytes, stream>>>(a);
}

template <typename T>
void launch(const TopArgs &a, hipStream_t stream)
{
    const int64_t pieces = (a.cols + Vec16<T>::N - 1) / Vec16<T>::N;
    if (pieces <= 64) return launch_as<T, 64, 1, false>(a, stream);
    if (pieces <= 64 * 4) return launch_as<T, 64, 4, false>(a, stream);
    if (pieces <= 256 * 4) return launch_as<T, 256, 4, false>(a, stream);
    if (a.rows > 512) return launch_as<T, 256, 4, true>(a, stream);
    launch_as<T, sizeof(T) == 8 ? 256 : 1024, 4, true>(a, stream);
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
    TopArgs a{logits, rows, cols, row_stride, (int)k, temperature, values, columns, lse};
    const int rc = clg_with_type(dtype, [&](auto t) {
        launch<decltype(t)>(a, clg_stream(stream));
        return CLG_OK;
    });
    if (rc) return rc;
    CLG_CHECK_LAUNCH("clg_top_logits");
    return CLG_OK;
}
