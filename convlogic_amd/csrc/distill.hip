// Distillation from a teacher's top logits: the loss of each row and, in the same pass, its gradient w.r.t. the student's logits.
//
// With u = z / tau, q = softmax(u), entries (t_j, c_j) of the teacher and p_j their probabilities (over the entries alone, or with the teacher's
// logsumexp L over all columns, p_j = exp(t_j / tau - L), and p_r = 1 - sum p_j for everything else):
//     loss = tau^2 [ sum_j p_j (log p_j - log q_{c_j}) + p_r (log p_r - log q_r) ],        q_r = sum of q over the columns that are not listed
//     d loss / d z_v = tau [ M q_v - sum_{j: c_j = v} p_j ]  listed,    tau q_v [ M - p_r / q_r ]  not listed,        M = sum_j p_j + p_r
// q_r may be small, so it is no difference of sums: listed columns leave the row first (a bit per column in LDS), their few exponentials are added to the
// sum of the others afterwards.  Where the student agrees with its teacher the loss is a small difference of its terms: those exponentials and what takes the
// others' sum to the row's highest are 64-bit numbers, and a relative error d of that sum, in 32 bits, moves the loss by tau^2 (M q_r - p_r) d only.
#include <stdlib.h>

#include "row_tile.h"

namespace {

struct DistillArgs {
    const void *z;                                                    // [rows][cols] with a stride between rows
    int64_t rows, cols, row_stride, first_row;                        // (first_row: of this launch)
    const void *values, *columns, *lse;                               // [rows][k], [rows][k], [rows] or NULL
    int values_type, lse_type, columns64, k;
    const uint8_t *mask;                                              // [rows] or NULL
    double temperature, inv_tau, loss_scale, grad_scale;
    const double *per_count;                                          // factor of both that is known on the device only, or NULL
    double *row_loss;                                                 // [rows] or NULL
    void *out;                                                        // [rows] losses in A, or NULL
    void *grad;                                                       // [rows][cols] or NULL
    void *applied;                                                    // [rows] in A: the factor that `grad` was written with, or NULL
    const void *upstream;                                             // A, [rows] with upstream_rows, or NULL for 1
    int upstream_rows, only_changed;
};

constexpr int kFlagTwice = 1, kFlagListed = 2, kFlagBad = 4;

// LDS of a team: reduction room (16 wavefronts of 4 doubles, for a workgroup), flags, entries (probability, logit, column), bits of a tile
__host__ __device__ inline int distill_lds(bool workgroup, int k, int cols_of_tile /* whole words of bits */)
{
    return ((workgroup ? 16 * 4 * 8 : 0) + 16 + k * (8 + 8 + 4) + cols_of_tile / 32 * 4 + 15) & ~15;
}

// whether entry j is the first of its column, and with all the others' probabilities on it
__device__ __forceinline__ bool first_of(const int *column, int j)
{
    bool first = true;
    for (int i = 0; i < j && first; ++i) first = column[i] != column[j];
    return first;
}
__device__ __forceinline__ double all_of(const int *column, const double *prob, int j, int k)
{
    double p = prob[j];
    for (int i = j + 1; i < k; ++i) p += column[i] == column[j] ? prob[i] : 0;
    return p;
}

// A team of LANES threads per row: a workgroup, or 16 lanes where there are many short rows.  A row that fits its registers (COLS columns) is read from memory
// once, for the sum and for the gradient; longer ones (MULTI) tile by tile, twice.
// 4096 rows of 131072 bfloat16 with gradient: 465 to 508 us, 4.2 to 4.6 TB/s of the 5.1 that a copy reaches; 122 registers of 1024 threads are all that a CU
// has, so a row's loads, sums and stores follow one another (vector units 60 % of the time).  777 of 50001 float16, 3 rows to a CU and two at a time: 47 us.
// 10000 of 1000 float32 without gradient, 16 lanes each: 16 us, of latency: 2500 wavefronts are 2.4 to a SIMD, each once through its chain of loads, sums and
// logarithms; they wait half of their time, the vector units are busy 44 % of it.
template <typename T, int THREADS, int LANES, int NV, bool MULTI, int STREAM>
__global__ __launch_bounds__(THREADS, 4) void distill_kernel(DistillArgs a)
{
    typedef typename Wide<T>::type A;
    typedef RowTile<T, LANES, NV, STREAM> Tile;
    typedef Team<THREADS, LANES> Mine;
    constexpr int TEAMS = THREADS / LANES, ROOM = Mine::kWhole ? 16 * 4 : 0;
    static_assert(TEAMS == 1 || THREADS == kWave, "teams share a wavefront, where LDS is in order");
    extern __shared__ char lds[];
    const int tid = Mine::kWhole ? threadIdx.x : threadIdx.x % LANES, team = Mine::kWhole ? 0 : threadIdx.x / LANES, k = a.k;
    double *room = reinterpret_cast<double *>(lds + team * distill_lds(Mine::kWhole, k, Tile::COLS)), *prob = room + ROOM + 2, *logit = prob + k;
    int *flags = reinterpret_cast<int *>(room + ROOM);
    int *column = reinterpret_cast<int *>(logit + k);
    uint32_t *bits = reinterpret_cast<uint32_t *>(column + k);
    const A unit = (A)Exps<A>::unit(a.temperature);

    const int64_t row = a.first_row + (Mine::kWhole ? (int64_t)blockIdx.x : (int64_t)blockIdx.x * TEAMS + team);
    if (TEAMS > 1 && row >= a.rows) return;
    const A up = a.upstream ? static_cast<const A *>(a.upstream)[a.upstream_rows ? row : 0] : A(1);
    if (a.only_changed && static_cast<const A *>(a.applied)[row] == up) return;
    T *grad = a.grad ? static_cast<T *>(a.grad) + row * a.cols : nullptr;
    const bool kept = !a.mask || a.mask[row];
    const T *z = static_cast<const T *>(a.z) + row * a.row_stride;
    // The teacher's entries in front of the row: the logits in their columns are a load behind theirs, and of a workgroup most wavefronts have none and go
    // on to the row.  What this thread's first entry loads is taken up after the row is on its way.
    if (tid == 0) *flags = 0;
    __syncthreads();
    A tops[2] = {lowest(A(0)), lowest(A(0))};                         // highest of the student's listed logits, of the others
    double top_t[1] = {lowest(0.0)};                                  // of the teacher's values
    T first_logit = (T)0.f;
    uint64_t first_value = 0, lse_bits = 0;
    bool first_there = false;
    const auto enter = [&](int j, T logit_j, uint64_t value) {
        const double v = value_of_bits(value, a.values_type);
        const A l = (A)logit_j;
        prob[j] = v;
        logit[j] = (double)l;
        top_t[0] = max_of(top_t[0], v);
        tops[0] = max_of(tops[0], l);
    };
    if (kept) {
        int seen = 0;
#pragma unroll 1
        for (int j = tid; j < k; j += LANES) {
            const int64_t at = row * k + j, c = a.columns64 ? static_cast<const int64_t *>(a.columns)[at] : static_cast<const int32_t *>(a.columns)[at];
            const uint64_t value = load_bits(a.values, a.values_type, at);
            const bool there = c >= 0 && c < a.cols;
            seen |= there ? kFlagListed : c >= a.cols ? kFlagBad : 0;
            column[j] = there ? (int)c : -1;
            if (!there) continue;
            if (j == tid) {
                first_there = true;
                first_value = value;
                first_logit = z[c];
            } else {
                enter(j, z[c], value);
            }
        }
        if (seen) atomicOr(flags, seen);
        if (a.lse) lse_bits = load_bits(a.lse, a.lse_type, row);
    }
    Tile tile(tid);
    if (kept) tile.load(z, 0, a.cols);
    // the sum over what is not listed
    A m_t = lowest(A(0)), s_t = 0;
    const auto look = [&](int64_t base) {
        const int n = (int)(a.cols - base < Tile::COLS ? a.cols - base : Tile::COLS);
        for (int w = tid; w < (n + 31) / 32; w += LANES) bits[w] = 0;
        __syncthreads();
#pragma unroll 1
        for (int j = tid; j < k; j += LANES) {
            const int64_t c = (int64_t)column[j] - base;
            if (column[j] < 0 || c < 0 || c >= n) continue;
            if (atomicOr(&bits[c >> 5], 1u << (c & 31)) >> (c & 31) & 1) atomicOr(flags, kFlagTwice);
        }
        __syncthreads();
        if (base == 0 && first_there) enter(tid, first_logit, first_value);
        tile.trim();
        tile.drop(bits);
        tile.fence();
        const A m = max_of(m_t, tile.highest());
        const Exps<A> e(m, unit);
        if (MULTI) s_t = rescaled(s_t, m_t, Exps<A>(m_t, unit), e);
        tile.fence();
        s_t += tile.sum(e);
        m_t = m;
        tile.fence();
    };
    if (kept) {
        look(0);
        if (MULTI)
            for (int64_t base = Tile::COLS; base < a.cols; base += Tile::COLS) {
                __syncthreads();
                tile.load(z, base, a.cols);
                look(base);
            }
    }
    __syncthreads();
    const int flag = *flags;
    if (!kept || !(flag & (kFlagListed | kFlagBad))) {                // a row that says nothing
        if (tid == 0) {
            if (a.row_loss) a.row_loss[row] = 0;
            if (a.out) static_cast<A *>(a.out)[row] = 0;
            if (a.applied) static_cast<A *>(a.applied)[row] = up;
        }
        if (grad) {
            for (int64_t c = (int64_t)tid * Tile::VEC; c + Tile::VEC <= a.cols; c += LANES * Tile::VEC)
                *reinterpret_cast<typename Tile::V *>(grad + c) = (typename Tile::V)(T)0.f;
            if (tid < a.cols % Tile::VEC) grad[a.cols - 1 - tid] = (T)0.f;
        }
        return;
    }
    tops[1] = m_t;
    Mine::template reduce<false>(tops, reinterpret_cast<A *>(room));
    // (the teacher's highest is exact: relative to one that was rounded, or rounded over the temperature, its exponentials may all be 0, or infinite)
    if (!a.lse) Mine::template reduce<false>(top_t, room + 32);
    const A m_u = tops[1], m = max_of(tops[0], m_u);
    const Exps<A> of_rest(m_u, unit);
    __syncthreads();

    // sums: the others' exponentials relative to m_u; in 64 bits the teacher's, its share times the difference of the logarithms, and the student's listed
    // exponentials relative to m
    A sums[1] = {rescaled(s_t, m_t, Exps<A>(m_t, unit), of_rest)};
    double parts[3] = {0, 0, 0};
    const double lse = a.lse ? value_of_bits(lse_bits, a.lse_type) : 0, base_t = a.lse ? 0 : finite_or_zero(top_t[0]);
#pragma unroll 1
    for (int j = tid; j < k; j += LANES) {
        if (column[j] < 0) continue;
        const double l = logit[j], u = (l - (double)m) * a.inv_tau, t = (prob[j] - base_t) * a.inv_tau - lse, e = exp(t), q = l == lowest(0.0) ? 0 : exp(u);
        if (!(flag & kFlagTwice) || first_of(column, j)) parts[2] += q;
        parts[0] += e;
        if (e != 0) parts[1] += e * (t - u);
        prob[j] = e;
        logit[j] = q;
    }
    // what makes an exponential of the others, as it is summed, one relative to m: by the first wavefront, beside the entries
    const double log_of_u = ((double)m_u - (double)m) * a.inv_tau + of_rest.residue(m_u);
    if (!Mine::kWhole || tid < kWave) room[ROOM + 1] = m_u == lowest(A(0)) ? 1 : exp(log_of_u);
    Mine::sums(sums, parts, reinterpret_cast<A *>(room), room + 16, uniform(tid & ~63) < k);
    const double s_u = sums[0], mass_p = parts[0], of_u = room[ROOM + 1], total = s_u * of_u + parts[2];
    bool all_listed = false;                                          // (then there is nothing else)
    if (a.lse && k >= a.cols) {
        A n[1] = {0};
#pragma unroll 1
        for (int j = tid; j < k; j += LANES) n[0] += column[j] >= 0 && first_of(column, j);
        __syncthreads();
        Mine::template reduce<true>(n, reinterpret_cast<A *>(room));
        all_listed = n[0] == (A)a.cols;
    }
    double rest = 0;
    if (a.lse && !all_listed) rest = mass_p != mass_p ? mass_p : max_of(0.0, 1 - mass_p);
    // four logarithms and three inverses at once, one in a lane
    const int lane = tid & 63;
    const double value = lane == 0 ? total : lane == 1 ? s_u : lane == 2 ? rest : mass_p, logs = log(value), inverses = quick_inverse(value);
    const double log_total = Mine::from(logs, 0);
    double mass, loss, per = 1;                                       // per: of an entry's exponential
    if (a.lse) {
        mass = mass_p + rest;
        loss = parts[1] + mass_p * log_total;
        if (rest != 0) loss += rest * (Mine::from(logs, 2) - (log_of_u + Mine::from(logs, 1) - log_total));
    } else {
        per = mass_p == 0 ? 0 : Mine::from(inverses, 3);
        mass = mass_p * per;
        loss = mass_p == 0 ? 0 : parts[1] * per + log_total - Mine::from(logs, 3);
    }
    if ((flag & kFlagBad) || m == -lowest(A(0))) loss = mass = __builtin_nan("");        // (a logit of +inf)
    const double factor = a.per_count ? *a.per_count : 1;
    if (tid == 0) {
        if (a.row_loss) a.row_loss[row] = loss * a.loss_scale;
        if (a.out) static_cast<A *>(a.out)[row] = (A)(loss * a.loss_scale * factor);
        if (a.applied) static_cast<A *>(a.applied)[row] = up;
    }
    if (!grad) return;
    const double g = a.grad_scale * factor * (double)up, of_listed = mass * Mine::from(inverses, 0);
    const A others = s_u == 0 && total > 0 && mass == mass
                         ? A(0)
                         : (A)(g * (of_listed * of_u - (rest == 0 ? 0 : rest * Mine::from(inverses, 1))));
    const auto of = [&](A x) { return of_rest(x) * others; };
    if (MULTI) {
        for (int64_t base = 0; base < a.cols; base += Tile::COLS) {
            tile.load(z, base, a.cols);
            tile.store(grad, base, of);
        }
    } else {
        tile.store(grad, 0, of);                                      // (no loop: in one, all values come before the first store)
    }
    __syncthreads();                                                  // the listed columns' own values go over those
#pragma unroll 1
    for (int j = tid; j < k; j += LANES) {
        if (column[j] < 0) continue;
        double p = prob[j];
        if (flag & kFlagTwice) {
            if (!first_of(column, j)) continue;
            p = all_of(column, prob, j, k);
        }
        grad[column[j]] = (T)(A)(g * (of_listed * logit[j] - p * per));
    }
}

// 1 / number of kept rows, 0 where there are none, by one workgroup: a byte a row, 16 at a time
__global__ __launch_bounds__(1024) void count_kept_kernel(const uint8_t *mask, int64_t rows, double *per_count)
{
    typedef uint32_t Four __attribute__((ext_vector_type(4), aligned(1)));
    __shared__ double room[16];
    int64_t count = 0;
    const int64_t whole = rows / 16;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < whole; i += 1024) {
        const Four x = reinterpret_cast<const Four *>(mask)[i];
#pragma unroll
        for (int w = 0; w < 4; ++w) count += __popc(((x[w] & 0x7F7F7F7Fu) + 0x7F7F7F7Fu | x[w]) & 0x80808080u);     // bytes that are not 0
    }
    if (threadIdx.x < rows % 16) count += mask[rows - 1 - threadIdx.x] != 0;
    double n[1] = {(double)count};
    block_reduce<true, 1024>(n, room);
    if (threadIdx.x == 0) *per_count = n[0] == 0 ? 0 : 1 / n[0];
}

// The sum of the rows' losses, in a fixed order: of all rows, or of kSlice to a workgroup first.  (One workgroup: 3 us for 10000 rows, 6 for 40000, 9 for
// 65536, of loads that wait; in slices 5 for 65537, two launches.)
constexpr int kSlice = 16384;
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

template <typename T, int THREADS, int LANES, int NV, bool MULTI, int STREAM>
void launch_as(const DistillArgs &a, hipStream_t stream)
{
    typedef RowTile<T, LANES, NV, STREAM> Tile;
    static_assert(Tile::COLS % 32 == 0, "bits of a tile fill whole words");
    constexpr int TEAMS = THREADS / LANES;
    const size_t lds = (size_t)TEAMS * distill_lds(TEAMS == 1, a.k, Tile::COLS);
    DistillArgs part = a;
    constexpr int64_t kMost = (int64_t)1 << 31;                       // threads of a launch
    for (; part.first_row < a.rows; part.first_row += kMost / LANES) {
        const int64_t rows = a.rows - part.first_row < kMost / LANES ? a.rows - part.first_row : kMost / LANES;
        distill_kernel<T, THREADS, LANES, NV, MULTI, STREAM><<<dim3((unsigned)clg_ceil_div(rows, TEAMS)), dim3(THREADS), lds, stream>>>(part);
    }
}

template <typename T, int STREAM>
void launch_rows(const DistillArgs &a, hipStream_t stream)
{
    const int64_t pieces = (a.cols + Vec16<T>::N - 1) / Vec16<T>::N;
    // 16 lanes to a row: what is done once for a row is done for four at a time, most of the work of short rows; with fewer rows than fill the chip so, longer
    // ones are done sooner by 64 lanes each.  A pass in us by 64 and by 16 lanes, float32 with gradient: 8192 rows of 100 columns 23 and 15 (2048: 13 and 12,
    // 512: 12 and 11), 32768 of 500 66 and 50 (8192: 25 and 21, 2048: 15 and 17), 8192 of 1000 29 and 26 (2048: 16 and 19); entries beyond 32 take a lane as long as
    // its part of 1000 columns (32768 rows, k = 33: 80 and 91).  The loss alone: 8192 of 100 17 and 10, of 500 18 and 14 (2048: 10 and 11), of 1000 21 and
    // 18 (2048: 11 and 12).  bfloat16 with gradient: 8192 of 1000 27 and 24 (2048: 15 and 18), 32768 of 2000 84 and 82; with k = 33, where the rule takes
    // 64 lanes, 32768 of 1000 78 and 66.  float64: 8192 of 500 33 and 33, 32768 91 and 88 (2048: 18 and 24).  16 pieces in 16 lanes are all 128 registers and
    // 28 to 44 bytes of scratch beyond.
    const char *lanes = clg_knob(K_DISTILL_LANES);
    const bool few = a.k <= 64 && (lanes ? atoi(lanes) == 16 : pieces <= 16 || (pieces <= 64 ? a.rows >= 2048 : a.k <= 32 && a.rows >= 8192));
    if (few && pieces <= 16) return launch_as<T, 64, 16, 1, false, STREAM>(a, stream);
    if (few && pieces <= 16 * 4) return launch_as<T, 64, 16, 4, false, STREAM>(a, stream);
    if (few && pieces <= 16 * 16) return launch_as<T, 64, 16, 16, false, STREAM>(a, stream);
    if (pieces <= 64 * 4) return launch_as<T, 64, 64, 4, false, STREAM>(a, stream);
    if (pieces <= 64 * 16) return launch_as<T, 64, 64, 16, false, STREAM>(a, stream);
    if (pieces <= 256 * 16) return launch_as<T, 256, 256, 16, false, STREAM>(a, stream);
    if (pieces <= 512 * 16) return launch_as<T, 512, 512, 16, false, STREAM>(a, stream);
    if (pieces <= 1024 * 16) return launch_as<T, 1024, 1024, 16, false, STREAM>(a, stream);
    // (rows in tiles of 1024 threads where they do not fill the chip: 16 of 200000 bfloat16 48 -> 43 us a step, but 300 of them 102 -> 122)
    if (a.rows <= 128) return launch_as<T, 1024, 1024, 8, true, STREAM>(a, stream);
    launch_as<T, 512, 512, 8, true, STREAM>(a, stream);
}

template <typename T>
void launch(const DistillArgs &a, hipStream_t stream)
{
    // Past the caches from 16 MB on: the lines that other kernels left there modified have to be written out first to take rows that are read once (32768
    // columns behind a pass over 512 MB of other memory: 256 MB of logits 138 us through the caches, 118 past them, 32 MB 36 and 29; where the logits
    // were in the caches, the same either way).  Gradient rows that are no whole cache lines are written through the caches, which put the lines together.
    if (!clg_past_caches(a.rows * a.cols * sizeof(T), 16)) launch_rows<T, 0>(a, stream);
    else if (a.cols * sizeof(T) % 128 != 0) launch_rows<T, 1>(a, stream);
    else launch_rows<T, 3>(a, stream);
}

}  // namespace

constexpr int kMaxEntries = 1024;

// what both entry points require of a call
static int check_call(const char *name, int dtype, const void *logits, int64_t row_stride, const void *values, int values_dtype, const void *columns,
                      int columns_bits, const void *lse, int lse_dtype, int64_t rows, int64_t cols, int64_t k, double temperature)
{
    CLG_REQUIRE(clg_score_type(dtype), "%s: unsupported dtype %d", name, dtype);
    CLG_REQUIRE(clg_score_type(values_dtype) && (!lse || clg_score_type(lse_dtype)), "%s: unsupported dtype of the teacher's values", name);
    CLG_REQUIRE(columns_bits == 32 || columns_bits == 64, "%s: columns must have 32 or 64 bits, got %d", name, columns_bits);
    CLG_REQUIRE(rows >= 0 && cols >= 1 && cols < (int64_t)1 << 31, "%s: bad shape [%lld, %lld]", name, (long long)rows, (long long)cols);
    CLG_REQUIRE(k >= 1 && k <= kMaxEntries, "%s: 1 to %d entries per row, got %lld", name, kMaxEntries, (long long)k);
    CLG_REQUIRE(rows < (int64_t)1 << 31, "%s: %lld rows are more than a launch holds", name, (long long)rows);
    CLG_REQUIRE(row_stride >= 0, "%s: negative row stride", name);
    CLG_REQUIRE(temperature > 0 && temperature < 1e30, "%s: the temperature must be positive and finite", name);
    CLG_REQUIRE(!rows || (logits && values && columns), "%s: null pointer", name);
    return CLG_OK;
}

extern "C" int64_t clg_distill_scratch_bytes(int64_t rows) { return rows < 0 ? 0 : (rows + 2 + clg_ceil_div(rows, kSlice)) * 8; }

extern "C" int clg_distill_forward(int dtype, const void *logits, int64_t row_stride, const void *values, int values_dtype, const void *columns,
                                   int columns_bits, const void *lse, int lse_dtype, const uint8_t *mask, int64_t rows, int64_t cols, int64_t k,
                                   double temperature, double weight, int reduction, void *loss, void *grad, void *applied, void *scratch, void *stream)
{
    if (const int rc = check_call("clg_distill_forward", dtype, logits, row_stride, values, values_dtype, columns, columns_bits, lse, lse_dtype, rows, cols, k,
                                  temperature))
        return rc;
    CLG_REQUIRE(reduction == CLG_REDUCE_NONE || reduction == CLG_REDUCE_SUM || reduction == CLG_REDUCE_MEAN, "clg_distill_forward: bad reduction %d", reduction);
    CLG_REQUIRE(loss || (reduction == CLG_REDUCE_NONE && !rows), "clg_distill_forward: null pointer");
    CLG_REQUIRE(reduction == CLG_REDUCE_NONE || scratch, "clg_distill_forward: null scratch");
    CLG_REQUIRE(!grad == !applied, "clg_distill_forward: grad and applied come together");
    CLG_REQUIRE(!grad || reduction != CLG_REDUCE_NONE, "clg_distill_forward: the gradient of a loss per row is clg_distill_backward's");
    double *row_loss = static_cast<double *>(scratch), *per_count = row_loss ? row_loss + rows : nullptr;
    DistillArgs a{};
    a.z = logits, a.rows = rows, a.cols = cols, a.row_stride = row_stride;
    a.values = values, a.columns = columns, a.lse = lse, a.values_type = values_dtype, a.lse_type = lse_dtype, a.columns64 = columns_bits == 64, a.k = (int)k;
    a.mask = mask, a.temperature = temperature, a.inv_tau = 1 / temperature, a.loss_scale = temperature * temperature * weight, a.grad_scale = temperature * weight;
    a.grad = grad, a.applied = applied;
    if (reduction == CLG_REDUCE_NONE) a.out = loss;
    else a.row_loss = row_loss;
    if (reduction == CLG_REDUCE_MEAN && mask && rows) {
        count_kept_kernel<<<dim3(1), dim3(1024), 0, clg_stream(stream)>>>(mask, rows, per_count);
        CLG_CHECK_LAUNCH("clg_distill_forward");
        a.per_count = per_count;
    } else if (reduction == CLG_REDUCE_MEAN && rows) {
        a.loss_scale /= rows, a.grad_scale /= rows;
    }
    if (rows) {
        const int rc = clg_with_type(dtype, [&](auto t) {
            launch<decltype(t)>(a, clg_stream(stream));
            return CLG_OK;
        });
        if (rc) return rc;
        CLG_CHECK_LAUNCH("clg_distill_forward");
    }
    if (reduction == CLG_REDUCE_NONE) return CLG_OK;
    const double *terms = row_loss;
    int64_t n = rows;
    if (rows > 4 * kSlice) {
        n = clg_ceil_div(rows, kSlice);
        sum_slices_kernel<<<dim3((unsigned)n), dim3(1024), 0, clg_stream(stream)>>>(row_loss, rows, per_count + 1);
        CLG_CHECK_LAUNCH("clg_distill_forward");
        terms = per_count + 1;
    }
    if (dtype == CLG_F64) sum_rows_kernel<double><<<dim3(1), dim3(1024), 0, clg_stream(stream)>>>(terms, n, a.per_count, static_cast<double *>(loss));
    else sum_rows_kernel<float><<<dim3(1), dim3(1024), 0, clg_stream(stream)>>>(terms, n, a.per_count, static_cast<float *>(loss));
    CLG_CHECK_LAUNCH("clg_distill_forward");
    return CLG_OK;
}

extern "C" int clg_distill_backward(int dtype, const void *logits, int64_t row_stride, const void *values, int values_dtype, const void *columns,
                                    int columns_bits, const void *lse, int lse_dtype, const uint8_t *mask, int64_t rows, int64_t cols, int64_t k,
                                    double temperature, double weight, int reduction, const void *upstream, void *grad, void *applied, void *scratch,
                                    void *stream)
{
    if (const int rc = check_call("clg_distill_backward", dtype, logits, row_stride, values, values_dtype, columns, columns_bits, lse, lse_dtype, rows, cols,
                                  k, temperature))
        return rc;
    CLG_REQUIRE(reduction == CLG_REDUCE_NONE || reduction == CLG_REDUCE_SUM || reduction == CLG_REDUCE_MEAN, "clg_distill_backward: bad reduction %d", reduction);
    if (!rows) return CLG_OK;
    CLG_REQUIRE(upstream && grad, "clg_distill_backward: null pointer");
    DistillArgs a{};
    a.z = logits, a.rows = rows, a.cols = cols, a.row_stride = row_stride;
    a.values = values, a.columns = columns, a.lse = lse, a.values_type = values_dtype, a.lse_type = lse_dtype, a.columns64 = columns_bits == 64, a.k = (int)k;
    a.mask = mask, a.temperature = temperature, a.inv_tau = 1 / temperature, a.grad_scale = temperature * weight;
    a.grad = grad, a.applied = applied, a.only_changed = applied != nullptr, a.upstream = upstream, a.upstream_rows = reduction == CLG_REDUCE_NONE;
    if (reduction == CLG_REDUCE_MEAN && mask) {
        CLG_REQUIRE(scratch, "clg_distill_backward: null scratch");
        a.per_count = static_cast<const double *>(scratch) + rows;
        if (!applied) {
            count_kept_kernel<<<dim3(1), dim3(1024), 0, clg_stream(stream)>>>(mask, rows, static_cast<double *>(scratch) + rows);
            CLG_CHECK_LAUNCH("clg_distill_backward");
        }
    } else if (reduction == CLG_REDUCE_MEAN) {
        a.grad_scale /= rows;
    }
    const int rc = clg_with_type(dtype, [&](auto t) {
        launch<decltype(t)>(a, clg_stream(stream));
        return CLG_OK;
    });
    if (rc) return rc;
    CLG_CHECK_LAUNCH("clg_distill_backward");
    return CLG_OK;
}
