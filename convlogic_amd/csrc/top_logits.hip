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
    int64_t rows, cols, row_stride, first_row;                        // (first_row: of this launch)
    int k;
    double temperature;
    void *values;                                                     // [rows][k]
    int64_t *columns;                                                 // [rows][k]
    void *lse;                                                        // [rows] in A
    int parts;                                                        // of a row, each with a workgroup of its own
    int64_t width;                                                    // columns of a part
    void *part_best;                                                  // [rows][parts][k] candidates in order
    double *part_lse;                                                 // [rows][parts]
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

// Maxima that the threshold is made of: the threads' own, or where k is more than a third of the threads up to four of each.  5000 rows of 8000 bfloat16, 256
// threads, us by threads and by pieces: k = 60 39 and 44, 85 42 and 46, 120 49 and 51, 200 606 and 72; 20000 of 1000 float32, 64 threads: k = 15 34 and 37,
// 22 37 and 39, 30 44 and 42, 60 607 and 58.
template <int THREADS, int NV>
constexpr int kSeen = THREADS >= 1024 ? 1 : NV < 4 ? NV : 4;
template <int THREADS, int NV>
__host__ __device__ __forceinline__ bool by_pieces(int k)
{
    return kSeen<THREADS, NV> > 1 && 3 * k > THREADS;
}

constexpr int kSpare = 512;                                           // candidates that there is room for beside the k best
constexpr int kAllRanked = 64;                                        // columns of rows without a threshold (20000 of 64 float32 20 us, 23 with one; of 20 17, 24)
constexpr int kNoted = 1024;                                          // pieces that may be noted when a tile begins

// LDS of a workgroup: reduction room, counters, candidates, the best k, maxima, noted pieces
template <typename T, int THREADS, int NV, bool MULTI>
struct TopRoom {
    typedef Cand<typename Wide<T>::type> C;
    int room, maxima, notes;
    size_t bytes;
    __host__ __device__ explicit TopRoom(int k)
        : room(k + (k > kSpare ? k : kSpare)), maxima(THREADS * (by_pieces<THREADS, NV>(k) ? kSeen<THREADS, NV> : 1)), notes(THREADS * NV + Vec16<T>::N + (MULTI ? kNoted : 0)),
          bytes(18 * 8 + (size_t)(room + k) * sizeof(C) + (size_t)maxima * sizeof(typename C::K) + (size_t)notes * 4)
    {
    }
};

// One workgroup per row; MULTI: of more than one tile.  The best 64 of 65536 bfloat16, 4096 rows: 113 us, 4.8 TB/s with the vector units busy 71 % of the time
// under the counters; the best 20 of 131071 in one row, 31 parts: 8 us and 7 to merge them, two launches that wait for their loads.
// Registers for six wavefronts to a SIMD: 4096 x 65536 bfloat16 125 us, for four 136, for eight 132 (20000 x 3000 95, 94, 88; 20000 x 1000 float32 33, 33, 35).
// float64, for two: 1000 x 65536 148 to 154 us, for four 139; 20000 x 1000 148 and 149.
template <typename T, int THREADS, int NV, bool MULTI, bool STREAM>
__global__ __launch_bounds__(THREADS, sizeof(T) == 8 ? 2 : 6) void top_kernel(TopArgs a)
{
    typedef typename Wide<T>::type A;
    typedef Cand<A> C;
    typedef typename C::K K;
    typedef RowTile<T, THREADS, NV, STREAM> Tile;
    extern __shared__ char lds[];
    const TopRoom<T, THREADS, NV, MULTI> size(a.k);
    double *sums = reinterpret_cast<double *>(lds);                   // of 16 wavefronts
    K *shared = reinterpret_cast<K *>(sums + 16);                     // the threshold
    int *noted = reinterpret_cast<int *>(sums + 17), *count = noted + 1;
    C *cand = reinterpret_cast<C *>(sums + 18), *best = cand + size.room;
    K *maxima = reinterpret_cast<K *>(best + a.k);
    uint32_t *note = reinterpret_cast<uint32_t *>(maxima + size.maxima);             // first columns
    const int tid = threadIdx.x, part = blockIdx.y;
    const A unit = (A)Exps<A>::unit(a.temperature);
    const int64_t row = a.first_row + blockIdx.x, start = part * a.width, cols = a.cols - start < a.width ? a.cols - start : a.width, whole = cols / Tile::VEC * Tile::VEC;
    const int k = a.k < cols ? a.k : (int)cols;
    const T *z = static_cast<const T *>(a.z) + row * a.row_stride + start;

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

    A m_t = lowest(A(0)), s_t = 0, seen[kSeen<THREADS, NV>];          // seen: highest of the tiles so far, in parts
    constexpr int SEEN = kSeen<THREADS, NV>;
#pragma unroll
    for (int j = 0; j < SEEN; ++j) seen[j] = lowest(A(0));
    const bool pieces = by_pieces<THREADS, NV>(k);
    // the k-th highest of the maxima, by the first wavefront, between two barriers
    const auto show = [&]() {
        if (pieces) {
#pragma unroll
            for (int j = 0; j < SEEN; ++j) maxima[j * THREADS + tid] = ordered(seen[j]);
        } else {
            maxima[tid] = ordered(m_t);
        }
    };
    const auto search = [&](const Tile &tile) {
        if (tid >= kWave) return;
        constexpr int PER = THREADS / kWave;
        K t;
        if (!MULTI && THREADS == kWave && 2 * k > tile.whole) {       // (too many for maxima of pieces: of the elements, which this wavefront has)
            K x[NV * Tile::VEC + 1];
#pragma unroll
            for (int i = 0; i < NV * Tile::VEC; ++i) x[i] = i / Tile::VEC * THREADS + tid < tile.whole ? ordered((A)tile.v[i / Tile::VEC][i % Tile::VEC]) : K(0);
            x[NV * Tile::VEC] = tid < tile.tail ? ordered((A)tile.last) : K(0);
            t = wave_threshold(x, k, k + k / 4 + 8);
        } else if (pieces) {
            K x[PER * SEEN];
#pragma unroll
            for (int i = 0; i < PER * SEEN; ++i) x[i] = maxima[i * kWave + tid];
            t = wave_threshold(x, k, k + k / 4 + 8);
        } else {
            K x[PER];
#pragma unroll
            for (int i = 0; i < PER; ++i) x[i] = maxima[i * kWave + tid];
            t = wave_threshold(x, k, k + k / 4 + 8);
        }
        if (tid == 0) *shared = t - (t != 0);
    };
    // (what was found of a threshold is below what the best k of candidates have given)
    const auto raise = [&]() {
        const C now(*shared, 0);
        if (now.key() > from.key()) from = now;
    };

    Tile tile(tid);
    if (tid == 0) *noted = 0;
#pragma unroll 1
    for (int64_t base = 0, tiles = 1; base < cols; base += Tile::COLS, ++tiles) {
        tile.load(z, base, cols);
        tile.trim();
        A high[NV], m = max_of(m_t, (A)tile.last);
        tile.peaks(high);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            m = max_of(m, high[j]);
            seen[j % SEEN] = max_of(seen[j % SEEN], high[j]);
        }
        seen[0] = max_of(seen[0], (A)tile.last);
        tile.fence();
        const Exps<A> e(m, unit);
        if (MULTI) s_t = rescaled(s_t, m_t, Exps<A>(m_t, unit), e);
        s_t += tile.sum(e);
        m_t = m;
        const bool nan = s_t != s_t;                                  // (of this thread, now or in an earlier tile; it is in no maximum)
        if (!MULTI && NV == 1 && cols <= kAllRanked) {                // (a short row: every element is a candidate)
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = (j * THREADS + tid) * Tile::VEC;
#pragma unroll
                for (int i = 0; i < Tile::VEC; ++i)
                    if (c + i < tile.whole * Tile::VEC) cand[c + i] = C(ordered((A)tile.v[j][i]), c + i);
            }
            const int c = tile.whole * Tile::VEC + tid;
            if (tid < tile.tail) cand[c] = C(ordered((A)tile.last), c);
            found = (int)cols;
            break;
        }
        if (base == 0) {
            show();
            __syncthreads();
            search(tile);
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
            const bool last = base + Tile::COLS >= cols, anew = base && (last || (tiles & (tiles - 1)) == 0);
            if (anew) show();
            __syncthreads();
            if (anew) search(tile);
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
    C *const mine = static_cast<C *>(a.part_best) + (row * a.parts + part) * a.k;
    rank([&](C c, int i) {
        if (a.parts > 1) {
            mine[i] = C(c.key(), (uint32_t)start + c.column());
        } else {
            static_cast<T *>(a.values)[row * k + i] = z[c.column()];
            a.columns[row * k + i] = c.column();
        }
    });
    if (a.parts > 1)
        for (int i = k + tid; i < a.k; i += THREADS) mine[i] = C(0, ~0u);
    if (!a.lse) return;
    A top[1] = {m_t};
    block_reduce<false, THREADS>(top, reinterpret_cast<A *>(sums));
    const Exps<A> e(top[0], unit);
    double s[1] = {(double)rescaled(s_t, m_t, Exps<A>(m_t, unit), e)};
    __syncthreads();
    block_reduce<true, THREADS>(s, sums);
    if (tid != 0) return;
    const double lse = (double)finite_or_zero(top[0]) / a.temperature + log(s[0]) + e.residue(top[0]);
    if (a.parts > 1) a.part_lse[row * a.parts + part] = lse;
    else static_cast<A *>(a.lse)[row] = (A)lse;
}

// Rows of up to 16 columns, 16 lanes each: a lane has an element and meets the others on its way around the row of lanes.  256 rows of 10: 3.4 us, a launch;
// the best 3 of 10 in 100000 rows 13 us, 58 by the kernel above.
template <int BY>
__device__ __forceinline__ uint32_t rotated(uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + BY, 0xF, 0xF, true);           // row_ror
}
template <int BY>
__device__ __forceinline__ uint64_t rotated(uint64_t v)
{
    return (uint64_t)rotated<BY>((uint32_t)(v >> 32)) << 32 | rotated<BY>((uint32_t)v);
}
template <int BY, typename K>
__device__ __forceinline__ int count_before(K mine, int lane)
{
    if constexpr (BY == 16) {
        return 0;
    } else {
        const K other = rotated<BY>(mine);                            // of lane - BY, around the row
        return (other > mine || (other == mine && lane >= BY)) + count_before<BY + 1>(mine, lane);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void top_small_kernel(TopArgs a)
{
    typedef typename Wide<T>::type A;
    const int lane = threadIdx.x % 16;
    const int64_t row = a.first_row + (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (row >= a.rows) return;
    const bool there = lane < a.cols;
    const T z = there ? static_cast<const T *>(a.z)[row * a.row_stride + lane] : (T)lowest(0.f);
    const int before = count_before<1>(there ? ordered((A)z) : typename Cand<A>::K(0), lane);
    if (there && before < a.k) {
        static_cast<T *>(a.values)[row * a.k + before] = z;
        a.columns[row * a.k + before] = lane;
    }
    if (!a.lse) return;
    A top[1] = {(A)z};
    Team<256, 16>::reduce<false>(top, (A *)nullptr);
    if (top[0] != top[0]) top[0] = 0;                                 // (NaN, as the sum will be)
    const Exps<A> e(top[0], (A)Exps<A>::unit(a.temperature));
    A s[1] = {e((A)z)};
    Team<256, 16>::reduce<true>(s, (A *)nullptr);
    if (lane == 0) static_cast<A *>(a.lse)[row] = (A)((double)finite_or_zero(top[0]) / a.temperature + log((double)s[0]) + e.residue(top[0]));
}

constexpr int kMostParts = 64, kMerged = 1024;                        // parts of a row, and their candidates

// The parts of a row together: the candidates that reach a value which k of them reach, by rank.
template <typename T>
__global__ __launch_bounds__(256) void top_merge_kernel(TopArgs a)
{
    typedef typename Wide<T>::type A;
    typedef Cand<A> C;
    typedef typename C::K K;
    extern __shared__ char lds[];
    const int64_t row = blockIdx.x;
    const int n = a.parts * a.k, tid = threadIdx.x;
    K *shared = reinterpret_cast<K *>(lds);
    int *count = reinterpret_cast<int *>(lds + 8);
    C *all = reinterpret_cast<C *>(lds + 16), *some = all + n;
    const C *mine = static_cast<const C *>(a.part_best) + row * n;
    const T *z = static_cast<const T *>(a.z) + row * a.row_stride;
    for (int i = tid; i < n; i += 256) all[i] = mine[i];
    if (tid == 0) *count = 0;
    __syncthreads();
    if (tid < kWave) {
        K x[kMerged / kWave];
#pragma unroll
        for (int i = 0; i < kMerged / kWave; ++i) x[i] = i * kWave + tid < n ? all[i * kWave + tid].key() : K(0);
        const K t = wave_threshold(x, a.k, a.k + a.k / 4 + 8);
        if (tid == 0) *shared = t;
    }
    __syncthreads();
    const K least = *shared;
    for (int i = tid; i < n; i += 256) {
        const C c = all[i];
        if (c.key() >= least && c.key() != 0) some[atomicAdd(count, 1)] = c;
    }
    __syncthreads();
    const int m = *count;
    for (int i = tid; i < m; i += 256) {
        const C c = some[i];
        int before = 0;
#pragma unroll 8
        for (int j = 0; j < m; ++j) before += some[j].before(c);
        if (before >= a.k) continue;
        static_cast<T *>(a.values)[row * a.k + before] = z[c.column()];
        a.columns[row * a.k + before] = c.column();
    }
    if (!a.lse || tid >= kWave) return;
    const double l = tid < a.parts ? a.part_lse[row * a.parts + tid] : lowest(0.0), top = finite_or_zero(wave_max(l)), s = wave_sum(exp(l - top));
    if (tid == 0) static_cast<A *>(a.lse)[row] = (A)(top + log(s));
}

template <typename T, int THREADS, int NV, bool MULTI, bool STREAM>
void launch_as(const TopArgs &a, hipStream_t stream)
{
    TopArgs some = a;
    constexpr int64_t kMost = ((int64_t)1 << 31) / THREADS;           // rows of a launch: 2^31 threads
    for (; some.first_row < a.rows; some.first_row += kMost) {
        const int64_t rows = a.rows - some.first_row < kMost ? a.rows - some.first_row : kMost;
        top_kernel<T, THREADS, NV, MULTI, STREAM><<<dim3((unsigned)rows, a.parts), dim3(THREADS), TopRoom<T, THREADS, NV, MULTI>(a.k).bytes, stream>>>(some);
    }
}

template <typename T, bool STREAM>
void launch_rows(const TopArgs &a, hipStream_t stream)
{
    const int64_t pieces = (a.width + Vec16<T>::N - 1) / Vec16<T>::N;
    if (a.cols <= 16) {
        TopArgs some = a;
        constexpr int64_t kMost = (int64_t)1 << 27;                   // rows of a launch: 2^31 threads
        for (; some.first_row < a.rows; some.first_row += kMost)
            top_small_kernel<T><<<dim3((unsigned)clg_ceil_div(a.rows - some.first_row < kMost ? a.rows - some.first_row : kMost, 16)), dim3(256), 0, stream>>>(some);
        return;
    }
    if (pieces <= 64) launch_as<T, 64, 1, false, STREAM>(a, stream);
    else if (pieces <= 64 * 4) launch_as<T, 64, 4, false, STREAM>(a, stream);
    else if (pieces <= 256 * 4) launch_as<T, 256, 4, false, STREAM>(a, stream);
    // (1024 threads where there are few workgroups.  bfloat16, 256 and 1024 threads: 256 x 131072 36 and 28 us, 128 34 and 24, 1 29 and 20; 1024 58 and 95, 600 47 and 70.
    // 256 threads are sooner from more rows than one to a CU on, which this takes as 512 workgroups: 384 x 131072 40 and 49, 300 x 20000 15 and 22)
    else if (a.rows * a.parts > 512) launch_as<T, 256, 8, true, STREAM>(a, stream);
    else launch_as<T, sizeof(T) == 8 ? 256 : 1024, 8, true, STREAM>(a, stream);
    if (a.parts > 1)
        top_merge_kernel<T><<<dim3((unsigned)a.rows), dim3(256), 16 + (size_t)a.parts * a.k * 2 * sizeof(Cand<typename Wide<T>::type>), stream>>>(a);
}

template <typename T>
void launch(const TopArgs &a, hipStream_t stream)
{
    // (past the caches: 256 MB behind a pass over other memory 104 -> 67 us, 32 MB 31 -> 27, the same where the logits were in the caches)
    if (clg_past_caches(a.rows * a.cols * sizeof(T), 16)) launch_rows<T, true>(a, stream);
    else launch_rows<T, false>(a, stream);
}

// Few long rows are shared out among workgroups, whose best are merged by a second launch.  In us whole and in parts, bfloat16, k = 20: 1 row of 131072 20 and 15,
// 64 23 and 19 (of 200000 34 and 21), 128 25 and 23 (36 and 28), 192 26 and 28 (38 and 34): rows up to 64, well before the crossing.  1 row of 65536 13 and 15,
// of 80000 18 and 15.  The width of a part hardly counts: 1 row of 131072, k = 8, 14 us from 1024 to 8192 columns, 17 at 16384.  What a part finds does, by which the merge
// gets longer: of 131072 columns in 10 parts (k = 100) 23 and 22, in 5 (k = 200) 25 and 27, in 4 (k = 256) 27 and 33, in 3 (k = 300) 28 and 36.
int parts_of(int64_t rows, int64_t cols, int64_t k)
{
    if (rows > 64 || rows == 0) return 1;
    if (cols <= 65536) return 1;
    int64_t parts = cols / 4096;
    if (parts > kMostParts) parts = kMostParts;
    if (parts * k > kMerged) parts = kMerged / k;
    if (parts * rows > 1024) parts = 1024 / rows;
    return parts < 4 ? 1 : (int)parts;
}

constexpr int kMaxTop = 1024;

}  // namespace

extern "C" int64_t clg_top_logits_scratch_bytes(int dtype, int64_t rows, int64_t cols, int64_t k)
{
    if (!clg_score_type(dtype) || rows < 0 || cols < 1 || k < 1 || k > kMaxTop) return 0;
    const int parts = parts_of(rows, cols, k);
    return parts == 1 ? 0 : rows * parts * (k * (dtype == CLG_F64 ? 16 : 8) + 8);
}

extern "C" int clg_top_logits(int dtype, const void *logits, int64_t row_stride, int64_t rows, int64_t cols, int64_t k, double temperature, void *values,
                              int64_t *columns, void *lse, void *scratch, void *stream)
{
    CLG_REQUIRE(clg_score_type(dtype), "clg_top_logits: unsupported dtype %d", dtype);
    CLG_REQUIRE(rows >= 0 && rows < (int64_t)1 << 31 && cols >= 1 && cols < (int64_t)1 << 31, "clg_top_logits: bad shape [%lld, %lld]", (long long)rows,
                (long long)cols);
    CLG_REQUIRE(k >= 1 && k <= kMaxTop && k <= cols, "clg_top_logits: 1 to %d logits of %lld, got %lld", kMaxTop, (long long)cols, (long long)k);
    CLG_REQUIRE(row_stride >= 0, "clg_top_logits: negative row stride");
    CLG_REQUIRE(temperature > 0 && temperature < 1e30, "clg_top_logits: the temperature must be positive and finite");
    if (!rows) return CLG_OK;
    CLG_REQUIRE(logits && values && columns, "clg_top_logits: null pointer");
    TopArgs a{logits, rows, cols, row_stride, 0, (int)k, temperature, values, columns, lse, parts_of(rows, cols, k), cols, nullptr, nullptr};
    if (a.parts > 1) {
        CLG_REQUIRE(scratch, "clg_top_logits: null scratch");
        a.width = clg_ceil_div(clg_ceil_div(cols, a.parts), 64) * 64;
        a.parts = (int)clg_ceil_div(cols, a.width);
        a.part_lse = static_cast<double *>(scratch);
        a.part_best = a.part_lse + rows * a.parts;
    }
    const int rc = clg_with_type(dtype, [&](auto t) {
        launch<decltype(t)>(a, clg_stream(stream));
        return CLG_OK;
    });
    if (rc) return rc;
    CLG_CHECK_LAUNCH("clg_top_logits");
    return CLG_OK;
}
