// Backward pass of a LogicLayer whose input was kept in codes (activation_codes.h): both gradients from the codes themselves, float32.
//
// y_j = c_1 + c_a a + c_b b + c_ab a b with a, b two rows of x [in_dim, batch].  Per neuron the sums over the batch of g, g a, g b and g a b give the gradient of
// its 16 logits; per input, the gradient is the sum over the operands it is of g (c_a + c_ab b) or g (c_b + c_ab a).
#include "activation_codes.h"

namespace {

constexpr int kWaves = 4, kBlock = kWaves * kWave;
constexpr int64_t kFull = 256 * 32, kTurns = 4;                       // wavefronts that the chip holds; items that one takes, from there on
typedef float f32x4_row __attribute__((ext_vector_type(4), aligned(4)));

template <int VEC>
__device__ __forceinline__ void load_floats(const float *__restrict__ p, float (&v)[VEC])
{
    if constexpr (VEC == 4) {
        const f32x4_row u = *reinterpret_cast<const f32x4_row *>(p);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = u[k];
    } else {
        v[0] = *p;
    }
}
template <int VEC>
__device__ __forceinline__ void store_floats(float *__restrict__ p, const float (&v)[VEC])
{
    if constexpr (VEC == 4) *reinterpret_cast<f32x4_row *>(p) = f32x4_row{v[0], v[1], v[2], v[3]};
    else *p = v[0];
}

// What a backward pass needs of a neuron, in one line of memory (its wiring and its coefficients in tables of their own were three lines for each visit): the inputs
// of its operands and the coefficients, as the forward pass leaves them.
struct __attribute__((aligned(16))) Neuron {
    int32_t in_a, in_b;
    float ab, a, b, one, unused[2];
};

// The lane's samples: VEC of them from `at` on.  The last lane of a row that VEC does not divide steps back to its last VEC samples, of which `again` are its
// neighbour's: written twice with the same values, and left out of sums.
template <int VEC, bool RAGGED>
struct Samples {
    int64_t at;
    int again;
    bool live;
    __device__ __forceinline__ Samples(int64_t s, int64_t batch) : live(s < batch)
    {
        at = live ? s : 0;
        again = 0;
        if (RAGGED && live && s + VEC > batch) at = batch - VEC, again = (int)(s - at);
    }
};

// sums of one neuron over the lane's samples: g a b, g a, g b, g
struct Sums {
    float ab = 0, a = 0, b = 0, one = 0;
    template <int VEC>
    __device__ __forceinline__ void add(const float (&g)[VEC], const float (&x)[VEC], const float (&y)[VEC], int from)
    {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const float v = k >= from ? g[k] : 0.f;
            ab = __builtin_fmaf(v, x[k] * y[k], ab);
            a = __builtin_fmaf(v, x[k], a);
            b = __builtin_fmaf(v, y[k], b);
            one += v;
        }
    }
    // over LPR lanes, valid in the last 16
    template <int LPR>
    __device__ __forceinline__ void over_lanes()
    {
        ab = lane_group_sum<float, LPR>(ab);
        a = lane_group_sum<float, LPR>(a);
        b = lane_group_sum<float, LPR>(b);
        one = lane_group_sum<float, LPR>(one);
    }
    // their sums over LPR lanes, of which l is this one, at `to`: every exchange between rows of 16 lanes halves the number of values that a row has
    template <int LPR>
    __device__ __forceinline__ void store(float4 *to, int l) const
    {
        float *at = reinterpret_cast<float *>(to);
        if constexpr (LPR == 64) {
            const float v = row16_sum(swap_add16(swap_add32(ab, b), swap_add32(a, one)));      // row 0: ab, 1: a, 2: b, 3: one
            if ((l & 15) == 0) at[l >> 4] = v;
        } else if constexpr (LPR == 32) {
            const float u = row16_sum(swap_add16(ab, a)), v = row16_sum(swap_add16(b, one));
            if ((l & 15) == 0) at[l >> 4] = u, at[2 + (l >> 4)] = v;
        } else {
            const float4 v = {row16_sum(ab), row16_sum(a), row16_sum(b), row16_sum(one)};
            if (l == 0) *to = v;
        }
    }
    __device__ __forceinline__ float of_logit(int q, float p) const { return softmax16_backward(coef_transpose_row<float>(q, ab, a, b, one), p); }
};

struct Layer {
    uint8_t *codes;
    CodeScale<float> *scales;
    Neuron *neurons;
    const int64_t *a, *b, *start, *list;
    const float *x, *logits, *gy;
    float *probs, *y, *gx, *gl;
    float4 *sums;                                                     // [chunks][out_dim]
    int64_t in_dim, out_dim, batch;
};

// The 128 samples that 32 lanes have of an input become codes.
__device__ __forceinline__ float over_rows(float v, bool highest)     // of two rows of 16 lanes, the same in both
{
    const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const float p = __builtin_bit_cast(float, (unsigned)r[0]), q = __builtin_bit_cast(float, (unsigned)r[1]);
    return highest ? max_of(p, q) : min_of(p, q);
}
__device__ __forceinline__ void encode_row(const Layer &L, int64_t at, const float (&v)[4])
{
    float low = min_of(min_of(v[0], v[1]), min_of(v[2], v[3])), high = max_of(max_of(v[0], v[1]), max_of(v[2], v[3]));
    low = over_rows(-row16_max(-low), false);
    high = over_rows(row16_max(high), true);
    const Coder code((double)low, (double)high);
    bool bad = !(code.size * 255.0 <= __DBL_MAX__);
    uint32_t c[1];
    code(v, c, bad);
    bad = (uint32_t)(__ballot(bad) >> (threadIdx.x & 32)) != 0;
    *reinterpret_cast<uint32_t *>(L.codes + at) = bad ? 0 : c[0];
    if ((threadIdx.x & 31) == 0) L.scales[at / kCodeGroup] = scale_of(low, code, bad);
}

// Forward pass from the logits, with the arithmetic of clg_fc_forward_logits; a neuron takes LPR lanes.  ENCODE: every input is read by one operand only, whose
// neuron also makes its codes, and the batch is a multiple of 128, so that a row of 32 lanes has a group: x is then read once, not twice (163840 inputs, batch 256,
// forward pass and codes 76 us, not 95; with 64 lanes, two groups at a time, 79; batch 384 109, 143 and 117).  Else the workgroups from neuron_blocks on make them.
// The wiring and the logits of a wavefront's next neurons are on their way while the rows of these are.  131072 -> 1310720 neurons, batch 128: 350 us for 1.5 GB read,
// 1.3 of them rows of x, which are in no XCD's cache, and 0.8 written, 6.6 TB/s.
template <int VEC, bool RAGGED, int LPR, bool ENCODE>
__global__ __launch_bounds__(kBlock) void forward_kernel(Layer L, int neuron_blocks)
{
    constexpr int ROWS = kWave / LPR;
    if (!ENCODE && (int)blockIdx.x >= neuron_blocks) {
        encode_groups(L.x, L.in_dim * L.batch, L.codes, L.scales, (int64_t)(blockIdx.x - neuron_blocks) * (kBlock / kCodeLanes) + threadIdx.x / kCodeLanes,
                      (int64_t)(gridDim.x - neuron_blocks) * (kBlock / kCodeLanes));
        return;
    }
    const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x >> 6), sub = lane / LPR, l = lane % LPR, q = lane & 15;
    const Fold16<float> fold(q);
    const int64_t step = (int64_t)neuron_blocks * kWaves * ROWS;
    struct Wiring {
        int64_t a, b;
        float logit;
        __device__ __forceinline__ Wiring(const Layer &L, int64_t j, int q) : a(L.a[j]), b(L.b[j]), logit(L.logits[j * 16 + q]) {}
    };
    int64_t j0 = ((int64_t)blockIdx.x * kWaves + wave) * ROWS;
    if (j0 >= L.out_dim) return;
    const auto neuron = [&](int64_t first) { return first + sub < L.out_dim ? first + sub : L.out_dim - 1; };
    for (Wiring next(L, neuron(j0), q); j0 < L.out_dim; j0 += step) {
        const bool valid = j0 + sub < L.out_dim;
        const int64_t j = neuron(j0);                                 // every lane takes part in the sums
        const int32_t ia = (int32_t)clamp_index(next.a, L.in_dim), ib = (int32_t)clamp_index(next.b, L.in_dim);
        const float logit = next.logit;
        float x[VEC], y[VEC], out[VEC];
        int64_t s = (int64_t)l * VEC;
        Samples<VEC, RAGGED> mine(s, L.batch);
        load_floats(L.x + ia * L.batch + mine.at, x);
        load_floats(L.x + ib * L.batch + mine.at, y);
        if (j0 + step < L.out_dim) next = Wiring(L, neuron(j0 + step), q);
        float p;
        const Coef<float> c = fold(logit, p);
        if (valid && l < 16) {
            L.probs[j * 16 + q] = p;
            const float wiring = __builtin_bit_cast(float, q == 0 ? ia : ib), coef = q == 2 ? c.ab : q == 3 ? c.a : q == 4 ? c.b : c.one;
            if (q < 6) reinterpret_cast<float *>(L.neurons + j)[q] = q < 2 ? wiring : coef;
        }
        if (!valid) continue;
        while (s < L.batch) {
#pragma unroll
            for (int k = 0; k < VEC; ++k) out[k] = gate(c, x[k], y[k]);
            store_floats(L.y + j * L.batch + mine.at, out);
            if constexpr (ENCODE) {
                encode_row(L, ia * L.batch + mine.at, x);
                encode_row(L, ib * L.batch + mine.at, y);
            }
            s += LPR * VEC;
            if (s >= L.batch) break;
            mine = Samples<VEC, RAGGED>(s, L.batch);
            load_floats(L.x + ia * L.batch + mine.at, x);
            load_floats(L.x + ib * L.batch + mine.at, y);
        }
    }
}

// A neuron takes LPR lanes, which go through its three rows; with GX every input is read by one operand only, whose neuron writes its gradient.  Bound by memory:
// 163840 -> 81920 neurons, batch 256, 0.31 GB, 52 us, 6 TB/s.
template <int VEC, bool RAGGED, int LPR, bool GX>
__global__ __launch_bounds__(kBlock) void neurons_kernel(Layer L)
{
    constexpr int ROWS = kWave / LPR;
    const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x >> 6), sub = lane / LPR, l = lane % LPR, q = lane & 15;
    for (int64_t j0 = ((int64_t)blockIdx.x * kWaves + wave) * ROWS; j0 < L.out_dim; j0 += (int64_t)gridDim.x * kWaves * ROWS) {
        const bool valid = j0 + sub < L.out_dim;
        const int64_t j = valid ? j0 + sub : L.out_dim - 1;           // every lane takes part in the sums
        const Neuron c = L.neurons[j];
        const int64_t ia = c.in_a * L.batch, ib = c.in_b * L.batch;
        const float p = L.probs[j * 16 + q];
        Sums sums;
        for (int64_t s = (int64_t)l * VEC; s < L.batch; s += LPR * VEC) {
            const Samples<VEC, RAGGED> mine(s, L.batch);
            float x[VEC], y[VEC], g[VEC];
            load_floats(L.gy + j * L.batch + mine.at, g);
            Coded<VEC, RAGGED> cx, cy;
            cx.load(L.codes, L.scales, ia + mine.at);
            cy.load(L.codes, L.scales, ib + mine.at);
            cx.values(x);
            cy.values(y);
            sums.add(g, x, y, mine.again);
            if (GX && valid) {
                float ga[VEC], gb[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    ga[k] = __builtin_fmaf(c.ab, y[k], c.a) * g[k];
                    gb[k] = __builtin_fmaf(c.ab, x[k], c.b) * g[k];
                }
                store_floats(L.gx + ia + mine.at, ga);
                store_floats(L.gx + ib + mine.at, gb);
            }
        }
        sums.over_lanes<LPR>();
        if (l >= LPR - 16) {
            const float gl = sums.of_logit(q, p);
            if (valid) L.gl[j * 16 + q] = gl;
        }
    }
}

// value of lane `at` of the LPR lanes of a row, in all of them
template <int LPR>
__device__ __forceinline__ int32_t from_lane(int32_t v, int at)
{
    if constexpr (LPR == kWave) return __builtin_amdgcn_readlane(v, at);
    else return __shfl(v, at, LPR);
}
template <int LPR>
__device__ __forceinline__ float from_lane(float v, int at) { return __builtin_bit_cast(float, from_lane<LPR>(__builtin_bit_cast(int32_t, v), at)); }
template <int LPR>
__device__ __forceinline__ uint32_t from_lane(uint32_t v, int at) { return (uint32_t)from_lane<LPR>((int32_t)v, at); }
template <int LPR>
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int at)
{
    return (uint64_t)from_lane<LPR>((uint32_t)(v >> 32), at) << 32 | from_lane<LPR>((uint32_t)v, at);
}

// LPR lanes take `each` inputs one after the other and go through the operands these are, which follow one another in `list`, for PARTS * LPR * VEC samples.  The
// visit that reaches a neuron through its first operand has all its rows and forms its sums as well (SUMS): the gradient of its logits if the samples are the
// whole batch (kWhole), else for gradients_kernel (kParts).  A neuron wired to an input twice is listed twice, and is its second operand the second time.
// The way to a row -- list entry, neuron, row -- is three trips to memory: the lanes first go it for as many operands as they are, one each, and then
// take these one by one, with the rows of the next two on their way (of the next four: 28 to 57 registers more, and 8000 -> 8000 neurons, batch 100, 9.7 us, not
// 7.9); an input's own row is read with its first operand's and stays in registers (with every operand's: 30001 -> 60000, batch 333, 67 us, not 58).  I: what holds
// an index into x and gy.
// 131072 -> 1310720 neurons, batch 128: 370 us for 2.2 GB that leave the memory side -- 1.3 of gradients, each read twice, 0.3 of codes, the rest wiring and
// coefficients by the line -- 6 TB/s; a walk operand by operand, with the wiring and the coefficients in tables of their own, took 623.
enum { kNoSums, kWhole, kParts };
constexpr int kEachMost = 15;
template <int VEC, bool RAGGED, int LPR, int PARTS, int SUMS, typename I>
__global__ __launch_bounds__(kBlock) void inputs_kernel(Layer L, int each)
{
    constexpr int ROWS = kWave / LPR;
    constexpr int kOwner = 15, kFirst = 16, kLast = 32, kOpens = 64;
    const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x >> 6), sub = lane / LPR, l = lane % LPR, q = lane & 15;
    const int64_t groups = (L.in_dim + each - 1) / each, most = 2 * L.out_dim;
    const I batch = (I)L.batch;
    struct Part {
        I at;
        int again;
        bool live;
    } part[PARTS];                                                    // LPR * VEC samples apart
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        const Samples<VEC, RAGGED> s((((int64_t)blockIdx.y * PARTS + p) * LPR + l) * VEC, L.batch);
        part[p] = {(I)s.at, s.live ? s.again : VEC, s.live};
    }
    struct Rows {
        Coded<VEC, RAGGED> x[PARTS], own[PARTS];
        float g[PARTS][VEC];
        int mark;
    };
    for (int64_t it = ((int64_t)blockIdx.x * kWaves + wave) * ROWS; it < groups; it += (int64_t)gridDim.x * kWaves * ROWS) {
        const bool valid = it + sub < groups;
        const int64_t i0 = valid ? (it + sub) * each : 0;
        const int count = !valid ? 0 : L.in_dim - i0 < each ? (int)(L.in_dim - i0) : each;
        const int64_t begin = clamp_index(L.start[i0], most + 1);
        const int ends = (int)(clamp_index(L.start[i0 + (l < count ? l + 1 : count)], most + 1) - begin);       // lane l: behind input l, from `begin` on
        const int edges = valid ? max(from_lane<LPR>(ends, count > 0 ? count - 1 : 0), 0) : 0;
        int longest = edges;                                          // of the rows of a wavefront
        if constexpr (LPR <= 32) longest = max(longest, __shfl_xor(longest, 32));
        if constexpr (LPR <= 16) longest = max(longest, __shfl_xor(longest, 16));
        longest = uniform(longest);
        const I own_at = (I)i0 * batch;                               // the first input's
        float acc[PARTS][VEC] = {}, own[PARTS][VEC];                  // gradient and values of the input that has its turn
        for (int base = 0; base < longest; base += LPR) {
            // an operand for each lane
            const int at = base + l;
            const bool there = at < edges;
            const int64_t place = begin + (there ? at : 0);
            const int32_t j = (int32_t)clamp_index(L.list[place < most ? place : most - 1], L.out_dim);
            const int32_t before = (int32_t)L.list[place > 0 ? (place < most ? place : most - 1) - 1 : 0];
            const Neuron n = L.neurons[j];
            int owner = 0, opened = 0, closed = edges;                // input, from the first; its operands are opened .. closed
            for (int k = 0; k < each; ++k) {
                const int e = from_lane<LPR>(ends, k);
                if (k < count - 1 && e <= at) owner = k + 1, opened = e;
            }
            for (int k = each - 1; k >= 0; --k) {
                const int e = from_lane<LPR>(ends, k);
                if (k < count && k >= owner) closed = e;
            }
            const int32_t i = (int32_t)i0 + owner;
            const bool as_a = n.in_a == i && !(n.in_b == i && at > opened && before == j);
            const int mark = owner | (there && as_a ? kFirst : 0) | (there && at + 1 == closed ? kLast : 0) | (at == opened ? kOpens : 0);
            const I row_x = there ? (I)(as_a ? n.in_b : n.in_a) * batch : I(0), row_g = there ? (I)j * batch : I(0);
            const float c_ab = there ? n.ab : 0.f, c_own = there ? (as_a ? n.a : n.b) : 0.f;
            const int steps = longest - base < LPR ? longest - base : LPR;
            const auto load = [&](int e, Rows &r) {
                const int from = e < LPR ? e : LPR - 1;               // (what is behind the last of a row is dropped)
                r.mark = from_lane<LPR>(mark, from);
                const I at_g = from_lane<LPR>(row_g, from), at_x = from_lane<LPR>(row_x, from), at_own = own_at + (I)(r.mark & kOwner) * batch;
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    load_floats(L.gy + (at_g + part[p].at), r.g[p]);
                    r.x[p].load(L.codes, L.scales, (I)(at_x + part[p].at));
                    if (SUMS != kNoSums && r.mark & kOpens) r.own[p].load(L.codes, L.scales, (I)(at_own + part[p].at));
                }
            };
            const auto take = [&](int e, const Rows &r) {
                if (e >= steps) return;
                const float ab = from_lane<LPR>(c_ab, e), lin = from_lane<LPR>(c_own, e);
                float x[PARTS][VEC];
#pragma unroll
                for (int p = 0; p < PARTS; ++p) r.x[p].values(x[p]);
                // (an operand that is not there has coefficients 0, and a gradient that may be infinite)
                if (LPR == kWave || base + e < edges) {
#pragma unroll
                    for (int p = 0; p < PARTS; ++p)
#pragma unroll
                        for (int k = 0; k < VEC; ++k) acc[p][k] = __builtin_fmaf(__builtin_fmaf(ab, x[p][k], lin), r.g[p][k], acc[p][k]);
                }
                if (SUMS != kNoSums) {
                    const int32_t to = from_lane<LPR>(j, e);
                    if (r.mark & kOpens) {
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) r.own[p].values(own[p]);
                    }
                    if (r.mark & kFirst) {                            // uniform over the lanes of a row
                        Sums sums;
#pragma unroll
                        for (int p = 0; p < PARTS; ++p) sums.add(r.g[p], own[p], x[p], part[p].again);
                        if constexpr (SUMS == kWhole) {
                            sums.over_lanes<LPR>();
                            if (l >= LPR - 16) L.gl[(int64_t)to * 16 + q] = sums.of_logit(q, L.probs[(int64_t)to * 16 + q]);
                        } else {
                            sums.store<LPR>(L.sums + (int64_t)blockIdx.y * L.out_dim + to, l);
                        }
                    }
                }
                if (r.mark & kLast) {
#pragma unroll
                    for (int p = 0; p < PARTS; ++p) {
                        if (part[p].live) store_floats(L.gx + (own_at + (I)(r.mark & kOwner) * batch + part[p].at), acc[p]);
#pragma unroll
                        for (int k = 0; k < VEC; ++k) acc[p][k] = 0.f;
                    }
                }
            };
            constexpr int AHEAD = 2;
            Rows rows[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) load(u, rows[u]);
            for (int e = 0; e < steps; e += AHEAD) {
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    take(e + u, rows[u]);
                    load(e + u + AHEAD, rows[u]);
                }
            }
        }
        // inputs that nobody reads
        for (int k = 0; k < each; ++k) {
            const int e = from_lane<LPR>(ends, k), b = k ? from_lane<LPR>(ends, k - 1) : 0;
            if (k < count && e <= b) {
                const float none[VEC] = {};
#pragma unroll
                for (int p = 0; p < PARTS; ++p)
                    if (part[p].live) store_floats(L.gx + (own_at + (I)k * batch + part[p].at), none);
            }
        }
    }
}

// The gradient of the logits from the sums of inputs_kernel's parts of the batch, added in their order: four lanes to a neuron, with four logits each.
__global__ __launch_bounds__(kBlock) void gradients_kernel(const float4 *__restrict__ sums, const float4 *__restrict__ probs, float4 *__restrict__ gl, int64_t out_dim,
                                                         int chunks)
{
    const int i = (threadIdx.x & 3) * 4;
    for (int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x; e < out_dim * 4; e += (int64_t)gridDim.x * kBlock) {
        const float4 v = probs[e];
        float4 s = sums[e / 4];
        for (int c = 1; c < chunks; ++c) {
            const float4 u = sums[c * out_dim + e / 4];
            s.x += u.x, s.y += u.y, s.z += u.z, s.w += u.w;
        }
        const float p[4] = {v.x, v.y, v.z, v.w};
        float g[4], mean = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) g[k] = coef_transpose_row<float>(i + k, s.x, s.y, s.z, s.w), mean = __builtin_fmaf(p[k], g[k], mean);
        mean += dpp_zero<0xB1, 0xF>(mean);
        mean += dpp_zero<0x4E, 0xF>(mean);
        gl[e] = float4{p[0] * (g[0] - mean), p[1] * (g[1] - mean), p[2] * (g[2] - mean), p[3] * (g[3] - mean)};
    }
}

// Four samples to a lane from 17 samples on, or where they divide the batch (up to 16, one to a lane is one pass as well: 30001 -> 60000 neurons, batch 9, 23 us and
// 27 with four).
bool fours(int64_t batch) { return batch % 4 == 0 || batch > 16; }
// Lanes of a row: as many as it takes, up to a wavefront.
int lanes_of(int64_t batch)
{
    const int64_t lanes = fours(batch) ? clg_ceil_div(batch, 4) : batch;
    return lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
}
// How inputs_kernel takes a batch: LANES to a row, PARTS of LANES x 4 samples to a lane, so that up to 512 samples go one way to their rows.  inputs_kernel alone,
// with the shape taken and the next best: 30001 -> 60000 neurons, batch 150 36.8 us and 41.9 (64 lanes), 190 40.6 and 46.6, 200 39.9 and 46.7 (16 lanes, 3 parts),
// 300 48.6 and 55.1 (64, 2), 333 67.2 and 72.2 (16, 3, two chunks of the batch), 400 59.8 and 65.2 (64, two chunks); 300000 -> 500000, batch 300 439 and 479, with
// three chunks of 32 lanes 588.  Two parts where one does: batch 256 43.0 us for 41.0, batch 128 23.6 for 22.1.  Behind 512 samples chunks of 64 lanes: batch 700
// 109 us, with three parts of 32 lanes 111, with two of 64 115.
struct Shape {
    int lanes, parts;
};
Shape shape_of(int64_t batch)
{
    if (batch > 128 && batch <= 192) return {16, 3};
    if (batch > 256 && batch <= 384) return {32, 3};
    if (batch > 384 && batch <= 512) return {64, 2};
    return {lanes_of(batch), 1};
}
int64_t chunks_of(int64_t batch)
{
    const Shape s = shape_of(batch);
    return clg_ceil_div(batch, (int64_t)s.lanes * s.parts * (fours(batch) ? 4 : 1));
}

// Whether gradients_kernel ends the sums, also those of one chunk: with and without it 34.8 + 3.9 and 39.2 us for 30001 -> 60000 neurons, batch 256, 69.0 + 4.7 and
// 78.6 for 100000 -> 100000; batch 64 14.5 + 3.8 and 16.1, 24.8 + 4.1 and 26.7.
bool in_parts(int64_t out_dim, int64_t batch) { return chunks_of(batch) > 1 || out_dim * batch >= 1 << 24; }

// Inputs that a row of lanes takes: about 16 operands, worth the way to them, and rows enough to fill the chip.  inputs_kernel with 1, 4 and 15 inputs each: 100000
// -> 100000 neurons, batch 256, 94, 70 and 72 us; 30001 -> 60000, batch 150, 37, 34 and 77; batch 333 73, 69 and 72; 8000 -> 8000, batch 100, 8, 11 and 27; 131072
// -> 1310720, batch 128, 389, 397 and 453.
int inputs_each(int64_t in_dim, int64_t out_dim, int64_t chunks, int rows)
{
    const int64_t fan = clg_ceil_div(2 * out_dim, in_dim), by_fan = 16 / fan, by_rows = in_dim * chunks / (rows * 4096);
    const int64_t each = by_fan < by_rows ? by_fan : by_rows;
    return (int)(each < 1 ? 1 : each > kEachMost ? kEachMost : each);
}

// call(VEC, RAGGED, LPR) of the batch as integral constants
template <typename F>
void with_rows(int64_t batch, int row_lanes, F call)
{
    const auto lanes = [&](auto vec, auto ragged) {
        switch (row_lanes) {
        case 16: return call(vec, ragged, std::integral_constant<int, 16>());
        case 32: return call(vec, ragged, std::integral_constant<int, 32>());
        default: return call(vec, ragged, std::integral_constant<int, 64>());
        }
    };
    const std::integral_constant<int, 1> one;
    const std::integral_constant<int, 4> four;
    if (!fours(batch)) call(one, std::true_type(), std::integral_constant<int, 16>());
    else if (batch % 4 == 0) lanes(four, std::false_type());
    else lanes(four, std::true_type());
}

unsigned blocks_of(int64_t wavefronts)
{
    const int64_t blocks = clg_ceil_div(wavefronts, (int64_t)kWaves);
    return (unsigned)(blocks < (1 << 20) ? blocks : 1 << 20);
}

}  // namespace

extern "C" int64_t clg_fc_codes_scratch_bytes(int64_t out_dim, int64_t batch)
{
    if (out_dim <= 0 || batch <= 0) return 0;
    return in_parts(out_dim, batch) ? chunks_of(batch) * out_dim * (int64_t)sizeof(float4) : 0;
}

static int check_layer(const char *name, int64_t in_dim, int64_t out_dim, int64_t batch, int sole)
{
    CLG_REQUIRE(in_dim > 0 && out_dim > 0 && batch > 0, "%s: in_dim, out_dim and batch must be positive (%lld, %lld, %lld)", name, (long long)in_dim,
                (long long)out_dim, (long long)batch);
    CLG_REQUIRE(in_dim < (1ll << 31) && out_dim < (1ll << 30), "%s: 2^31 inputs and 2^30 neurons are not supported", name);
    CLG_REQUIRE(chunks_of(batch) <= 65535, "%s: a batch of %lld is not supported", name, (long long)batch);
    CLG_REQUIRE(!sole || 2 * out_dim == in_dim, "%s: sole needs 2 out_dim == in_dim, got %lld and %lld", name, (long long)out_dim, (long long)in_dim);
    return CLG_OK;
}

extern "C" int clg_fc_codes_forward(const float *x, const int64_t *a, const int64_t *b, const float *logits, float *probs, void *neurons, float *y, uint8_t *codes,
                                    void *scales, int64_t in_dim, int64_t out_dim, int64_t batch, int sole, void *stream)
{
    const char *name = "clg_fc_codes_forward";
    if (const int rc = check_layer(name, in_dim, out_dim, batch, sole)) return rc;
    CLG_REQUIRE(x && a && b && logits && probs && neurons && y && codes && scales, "%s: null pointer argument", name);
    CLG_REQUIRE(reinterpret_cast<uintptr_t>(neurons) % 16 == 0 && reinterpret_cast<uintptr_t>(codes) % 8 == 0, "%s: neurons must be aligned to 16 bytes, codes to 8", name);
    Layer L{};
    L.codes = codes, L.scales = static_cast<CodeScale<float> *>(scales), L.neurons = static_cast<Neuron *>(neurons), L.a = a, L.b = b;
    L.x = x, L.logits = logits, L.probs = probs, L.y = y, L.in_dim = in_dim, L.out_dim = out_dim, L.batch = batch;
    hipStream_t st = clg_stream(stream);
    const bool encode = sole && batch % kCodeGroup == 0;
    with_rows(batch, encode ? 32 : lanes_of(batch), [&](auto vec, auto ragged, auto lpr) {
        constexpr int VEC = decltype(vec)::value, LPR = decltype(lpr)::value;
        constexpr bool RAGGED = decltype(ragged)::value;
        // (up to four neurons one after the other, from where the chip is full)
        const int64_t wavefronts = clg_ceil_div(out_dim, (int64_t)(kWave / LPR)), turns = wavefronts / kFull;
        const int neurons = (int)blocks_of(clg_ceil_div(wavefronts, turns < 1 ? 1 : turns > kTurns ? kTurns : turns));
        const int coders = encode ? 0 : (int)blocks_of(clg_ceil_div(in_dim * batch, 4 * (int64_t)kCodeLanes * kCodeEach));
        const dim3 grid((unsigned)(neurons + coders));
        if constexpr (!RAGGED && LPR == 32)
            if (encode) return forward_kernel<VEC, RAGGED, LPR, true><<<grid, dim3(kBlock), 0, st>>>(L, neurons);
        forward_kernel<VEC, RAGGED, LPR, false><<<grid, dim3(kBlock), 0, st>>>(L, neurons);
    });
    CLG_CHECK_LAUNCH(name);
    return CLG_OK;
}

extern "C" int clg_fc_codes_backward(const uint8_t *codes, const void *scales, const void *neurons, const float *probs, const float *grad_y, const int64_t *csr_start,
                                     const int64_t *csr_list, float *grad_x, float *grad_logits, int64_t in_dim, int64_t out_dim, int64_t batch, int sole,
                                     void *scratch, void *stream)
{
    const char *name = "clg_fc_codes_backward";
    if (const int rc = check_layer(name, in_dim, out_dim, batch, sole)) return rc;
    CLG_REQUIRE(codes && scales && neurons && grad_y && (grad_x || grad_logits), "%s: null pointer argument", name);
    CLG_REQUIRE(!grad_x || (csr_start && csr_list), "%s: null pointer argument", name);
    CLG_REQUIRE(!grad_logits || probs, "%s: null pointer argument", name);
    const bool parts = grad_x && grad_logits && !sole && in_parts(out_dim, batch);
    CLG_REQUIRE(!parts || scratch, "%s: null scratch", name);
    Layer L{};
    L.codes = const_cast<uint8_t *>(codes), L.scales = static_cast<CodeScale<float> *>(const_cast<void *>(scales));
    L.neurons = static_cast<Neuron *>(const_cast<void *>(neurons)), L.start = csr_start, L.list = csr_list;
    L.probs = const_cast<float *>(probs), L.gy = grad_y, L.gx = grad_x, L.gl = grad_logits, L.sums = static_cast<float4 *>(scratch);
    L.in_dim = in_dim, L.out_dim = out_dim, L.batch = batch;
    hipStream_t st = clg_stream(stream);
    const bool by_neurons = !grad_x || (sole && grad_logits);
    const Shape shape = shape_of(batch);
    with_rows(batch, by_neurons ? lanes_of(batch) : shape.lanes, [&](auto vec, auto ragged, auto lpr) {
        constexpr int VEC = decltype(vec)::value, LPR = decltype(lpr)::value, ROWS = kWave / LPR;
        constexpr bool RAGGED = decltype(ragged)::value;
        if (by_neurons) {
            const dim3 grid(blocks_of(clg_ceil_div(out_dim, (int64_t)ROWS)));
            if (grad_x) neurons_kernel<VEC, RAGGED, LPR, true><<<grid, dim3(kBlock), 0, st>>>(L);
            else neurons_kernel<VEC, RAGGED, LPR, false><<<grid, dim3(kBlock), 0, st>>>(L);
            return;
        }
        const int each = inputs_each(in_dim, out_dim, chunks_of(batch), ROWS);
        const dim3 grid(blocks_of(clg_ceil_div(clg_ceil_div(in_dim, each), (int64_t)ROWS)), (unsigned)chunks_of(batch));
        const auto launch = [&](auto index) {
            typedef decltype(index) I;
            const auto with = [&](auto n) {
                constexpr int PARTS = decltype(n)::value;
                if (!grad_logits) inputs_kernel<VEC, RAGGED, LPR, PARTS, kNoSums, I><<<grid, dim3(kBlock), 0, st>>>(L, each);
                else if (parts) inputs_kernel<VEC, RAGGED, LPR, PARTS, kParts, I><<<grid, dim3(kBlock), 0, st>>>(L, each);
                else inputs_kernel<VEC, RAGGED, LPR, PARTS, kWhole, I><<<grid, dim3(kBlock), 0, st>>>(L, each);
            };
            if constexpr (VEC == 4)
                if (shape.parts > 1) return with(std::integral_constant<int, LPR == 64 ? 2 : 3>());
            with(std::integral_constant<int, 1>());
        };
        // (the batch behind the last row: what lanes that are dropped read is in front of it)
        if ((in_dim > out_dim ? in_dim : out_dim) * batch < 1ll << 30) launch(uint32_t());
        else launch(uint64_t());
    });
    CLG_CHECK_LAUNCH(name);
    if (parts) {
        gradients_kernel<<<dim3(blocks_of(clg_ceil_div(out_dim, 16))), dim3(kBlock), 0, st>>>(L.sums, reinterpret_cast<const float4 *>(probs),
                                                                                         reinterpret_cast<float4 *>(grad_logits), out_dim, (int)chunks_of(batch));
        CLG_CHECK_LAUNCH(name);
    }
    return CLG_OK;
}
