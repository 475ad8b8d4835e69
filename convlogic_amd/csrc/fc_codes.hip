// Backward pass of a LogicLayer whose input was kept in codes (activation_codes.h): both gradients from the codes themselves, float32.
//
// y_j = c_1 + c_a a + c_b b + c_ab a b with a, b two rows of x [in_dim, batch].  Per neuron the sums over the batch of g, g a, g b and g a b give the gradient of
// its 16 logits; per input, the gradient is the sum over the operands it is of g (c_a + c_ab b) or g (c_b + c_ab a).
#include "activation_codes.h"

namespace {

constexpr int kWaves = 4, kBlock = kWaves * kWave;
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

// Coefficients of a neuron as clg_fc_fold leaves them.
struct Gate {
    float ab, a, b;
    __device__ __forceinline__ explicit Gate(const float *__restrict__ folded)
    {
        const float4 v = *reinterpret_cast<const float4 *>(folded);
        ab = v.x, a = v.y, b = v.z;
    }
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
    __device__ __forceinline__ float of_logit(int q, float p) const { return softmax16_backward(coef_transpose_row<float>(q, ab, a, b, one), p); }
};

struct Layer {
    const uint8_t *codes;
    const CodeScale<float> *scales;
    const int64_t *a, *b, *start, *list;
    const float *folded, *probs, *gy;
    float *gx, *gl;
    float4 *sums;                                                     // [chunks][out_dim]
    int64_t in_dim, out_dim, batch;
};

// A neuron takes LPR lanes, which go through its three rows; with GX every input is read by one operand only, whose neuron writes its gradient.
template <int VEC, bool RAGGED, int LPR, bool GX>
__global__ __launch_bounds__(kBlock) void neurons_kernel(Layer L)
{
    constexpr int ROWS = kWave / LPR;
    const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x >> 6), sub = lane / LPR, l = lane % LPR, q = lane & 15;
    for (int64_t j0 = ((int64_t)blockIdx.x * kWaves + wave) * ROWS; j0 < L.out_dim; j0 += (int64_t)gridDim.x * kWaves * ROWS) {
        const bool valid = j0 + sub < L.out_dim;
        const int64_t j = valid ? j0 + sub : L.out_dim - 1;           // every lane takes part in the sums
        const int64_t ia = clamp_index(L.a[j], L.in_dim) * L.batch, ib = clamp_index(L.b[j], L.in_dim) * L.batch;
        const Gate c(L.folded + j * 4);
        const float p = L.probs[j * 16 + q];
        Sums sums;
        for (int64_t s = (int64_t)l * VEC; s < L.batch; s += LPR * VEC) {
            const Samples<VEC, RAGGED> mine(s, L.batch);
            float x[VEC], y[VEC], g[VEC];
            load_floats(L.gy + j * L.batch + mine.at, g);
            decode_at<VEC, RAGGED>(L.codes, L.scales, ia + mine.at, x);
            decode_at<VEC, RAGGED>(L.codes, L.scales, ib + mine.at, y);
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

// An input takes LPR lanes, which walk the operands it is (`list`) for LPR * VEC samples.  With SUMS != kNoSums the visit that reaches a neuron through its first
// operand has all its rows and forms its sums as well: the gradient of its logits if the samples are the whole batch (kWhole), else for gradients_kernel (kParts).
// A neuron wired to an input twice is listed twice, and is its second operand the second time.
// Operands go by fours, with a sum of their own per place: the rows of four are fetched and used while the wiring of the next four and the list entries of
// those behind are on their way.  All loads are from valid addresses, and what does not count is dropped afterwards: a load under a lane's condition
// would be waited for at the end of its branch.
enum { kNoSums, kWhole, kParts };
template <int VEC, bool RAGGED, int LPR, int SUMS>
__global__ __launch_bounds__(kBlock) void inputs_kernel(Layer L)
{
    constexpr int ROWS = kWave / LPR;
    struct Operands {
        int32_t j[4], other[4];                                       // neuron (-1: none), input of its other operand
        float c_ab[4], c_own[4], p[4];
        bool first[4];
    };
    const int lane = threadIdx.x & (kWave - 1), wave = uniform(threadIdx.x >> 6), sub = lane / LPR, l = lane % LPR, q = lane & 15;
    const int64_t groups = (L.in_dim + ROWS - 1) / ROWS, last = 2 * L.out_dim - 1;
    const Samples<VEC, RAGGED> mine(((int64_t)blockIdx.y * LPR + l) * VEC, L.batch);
    for (int64_t it = (int64_t)blockIdx.x * kWaves + wave; it < groups; it += (int64_t)gridDim.x * kWaves) {
        const bool valid = it * ROWS + sub < L.in_dim;
        const int64_t i = valid ? it * ROWS + sub : L.in_dim - 1;
        const int64_t begin = clamp_index(L.start[i], last + 2), end = valid ? clamp_index(L.start[i + 1], last + 2) : begin;
        const bool live = valid && mine.live;
        const auto entries = [&](int64_t at, int32_t (&j)[4]) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int32_t v = (int32_t)clamp_index(L.list[at + u < last ? at + u : last], L.out_dim);
                j[u] = at + u < end ? v : -1;
            }
        };
        const auto wiring = [&](const int32_t (&j)[4], int32_t before, Operands &m) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t jj = j[u] < 0 ? 0 : j[u];
                const int64_t ja = clamp_index(L.a[jj], L.in_dim), jb = clamp_index(L.b[jj], L.in_dim);
                const Gate c(L.folded + jj * 4);
                if (SUMS == kWhole) m.p[u] = L.probs[jj * 16 + q];
                const bool as_a = ja == i && !(jb == i && before == j[u]);
                m.j[u] = j[u];
                m.first[u] = j[u] >= 0 && as_a;
                m.other[u] = (int32_t)(as_a ? jb : ja);
                m.c_ab[u] = j[u] >= 0 ? c.ab : 0.f;
                m.c_own[u] = j[u] >= 0 ? (as_a ? c.a : c.b) : 0.f;
                before = j[u];
            }
        };
        float own[VEC];
        if (SUMS != kNoSums) decode_at<VEC, RAGGED>(L.codes, L.scales, i * L.batch + mine.at, own);
        float part[4][VEC];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int k = 0; k < VEC; ++k) part[u][k] = 0.f;
        int32_t next[4], after[4];
        Operands now, then;
        entries(begin, next);
        wiring(next, -1, now);
        entries(begin + 4, next);
        for (int64_t at = begin; at < end; at += 4) {                 // (the lanes of a row leave the loop together)
            float x[4][VEC], g[4][VEC];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                decode_at<VEC, RAGGED>(L.codes, L.scales, (int64_t)now.other[u] * L.batch + mine.at, x[u]);
                load_floats(L.gy + (int64_t)(now.j[u] < 0 ? 0 : now.j[u]) * L.batch + mine.at, g[u]);
            }
            wiring(next, now.j[3], then);
            entries(at + 8, after);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (now.j[u] < 0) continue;
#pragma unroll
                for (int k = 0; k < VEC; ++k) part[u][k] = __builtin_fmaf(__builtin_fmaf(now.c_ab[u], x[u][k], now.c_own[u]), g[u][k], part[u][k]);
                if (SUMS != kNoSums && now.first[u]) {                // uniform over the lanes of a row
                    Sums sums;
                    sums.add(g[u], own, x[u], mine.live ? mine.again : VEC);
                    sums.over_lanes<LPR>();
                    if (SUMS == kWhole && l >= LPR - 16) L.gl[(int64_t)now.j[u] * 16 + q] = sums.of_logit(q, now.p[u]);
                    if (SUMS == kParts && l == LPR - 1) L.sums[(int64_t)blockIdx.y * L.out_dim + now.j[u]] = float4{sums.ab, sums.a, sums.b, sums.one};
                }
            }
            now = then;
#pragma unroll
            for (int u = 0; u < 4; ++u) next[u] = after[u];
        }
        float sum[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) sum[k] = (part[0][k] + part[1][k]) + (part[2][k] + part[3][k]);
        if (live) store_floats(L.gx + i * L.batch + mine.at, sum);
    }
}

// The gradient of the logits from the sums of inputs_kernel's parts of the batch, added in their order: 16 lanes to a neuron.
__global__ __launch_bounds__(kBlock) void gradients_kernel(const float4 *__restrict__ sums, const float *__restrict__ probs, float *__restrict__ gl, int64_t out_dim,
                                                         int chunks)
{
    for (int64_t e = (int64_t)blockIdx.x * kBlock + threadIdx.x; e < out_dim * 16; e += (int64_t)gridDim.x * kBlock) {
        Sums s;
        for (int c = 0; c < chunks; ++c) {
            const float4 v = sums[c * out_dim + e / 16];
            s.ab += v.x, s.a += v.y, s.b += v.z, s.one += v.w;
        }
        gl[e] = s.of_logit((int)(e & 15), probs[e]);
    }
}

// Four samples to a lane from 17 samples on, or where they divide the batch.
bool fours(int64_t batch) { return batch % 4 == 0 || batch > 16; }
int lanes_of(int64_t batch)
{
    const int64_t lanes = fours(batch) ? clg_ceil_div(batch, 4) : batch;
    return lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
}
int64_t chunks_of(int64_t batch) { return clg_ceil_div(batch, (int64_t)lanes_of(batch) * (fours(batch) ? 4 : 1)); }

// call(VEC, RAGGED, LPR) of the batch as integral constants
template <typename F>
void with_rows(int64_t batch, F call)
{
    const auto lanes = [&](auto vec, auto ragged) {
        switch (lanes_of(batch)) {
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
    const int64_t chunks = chunks_of(batch);
    return chunks > 1 ? chunks * out_dim * (int64_t)sizeof(float4) : 0;
}

extern "C" int clg_fc_codes_backward(const uint8_t *codes, const void *scales, const int64_t *a, const int64_t *b, const float *folded, const float *probs,
                                     const float *grad_y, const int64_t *csr_start, const int64_t *csr_list, float *grad_x, float *grad_logits, int64_t in_dim,
                                     int64_t out_dim, int64_t batch, int sole, void *scratch, void *stream)
{
    const char *name = "clg_fc_codes_backward";
    CLG_REQUIRE(in_dim > 0 && out_dim > 0 && batch > 0, "%s: in_dim, out_dim and batch must be positive (%lld, %lld, %lld)", name, (long long)in_dim,
                (long long)out_dim, (long long)batch);
    CLG_REQUIRE(in_dim < (1ll << 31) && out_dim < (1ll << 30) && chunks_of(batch) <= 65535, "%s: 2^31 inputs, 2^30 neurons and batches of more than 65535 times 256 are not supported", name);
    CLG_REQUIRE(codes && scales && a && b && folded && grad_y && (grad_x || grad_logits), "%s: null pointer argument", name);
    CLG_REQUIRE(!grad_x || (csr_start && csr_list), "%s: null pointer argument", name);
    CLG_REQUIRE(!grad_logits || probs, "%s: null pointer argument", name);
    CLG_REQUIRE(!sole || 2 * out_dim == in_dim, "%s: sole needs 2 out_dim == in_dim, got %lld and %lld", name, (long long)out_dim, (long long)in_dim);
    const bool parts = grad_x && grad_logits && !sole && chunks_of(batch) > 1;
    CLG_REQUIRE(!parts || scratch, "%s: null scratch", name);
    const Layer L{codes, static_cast<const CodeScale<float> *>(scales), a, b, csr_start, csr_list, folded, probs, grad_y, grad_x, grad_logits, static_cast<float4 *>(scratch),
                  in_dim, out_dim, batch};
    hipStream_t st = clg_stream(stream);
    with_rows(batch, [&](auto vec, auto ragged, auto lpr) {
        constexpr int VEC = decltype(vec)::value, LPR = decltype(lpr)::value, ROWS = kWave / LPR;
        constexpr bool RAGGED = decltype(ragged)::value;
        if (!grad_x || (sole && grad_logits)) {
            const dim3 grid(blocks_of(clg_ceil_div(out_dim, (int64_t)ROWS)));
            if (grad_x) neurons_kernel<VEC, RAGGED, LPR, true><<<grid, dim3(kBlock), 0, st>>>(L);
            else neurons_kernel<VEC, RAGGED, LPR, false><<<grid, dim3(kBlock), 0, st>>>(L);
            return;
        }
        const dim3 grid(blocks_of(clg_ceil_div(in_dim, (int64_t)ROWS)), (unsigned)chunks_of(batch));
        if (!grad_logits) inputs_kernel<VEC, RAGGED, LPR, kNoSums><<<grid, dim3(kBlock), 0, st>>>(L);
        else if (parts) inputs_kernel<VEC, RAGGED, LPR, kParts><<<grid, dim3(kBlock), 0, st>>>(L);
        else inputs_kernel<VEC, RAGGED, LPR, kWhole><<<grid, dim3(kBlock), 0, st>>>(L);
    });
    CLG_CHECK_LAUNCH(name);
    if (parts) {
        gradients_kernel<<<dim3(blocks_of(clg_ceil_div(out_dim, 4))), dim3(kBlock), 0, st>>>(L.sums, probs, grad_logits, out_dim, (int)chunks_of(batch));
        CLG_CHECK_LAUNCH(name);
    }
    return CLG_OK;
}
