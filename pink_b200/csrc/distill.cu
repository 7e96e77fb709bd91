// Distillation: the loss of a head's scores against the routes of a map, and its gradient (pink_b200_op_distill*).
//
//   q = softmax(s / T) over the neurons that take part; p_j: the weights of a row's targets, or the softmax of their logits over T
//   loss = scale * (sum of p_j log(p_j / q_j) + r log(r / q_rest)),  r = 1 - sum p_j,  q_rest = sum of q over the other neurons
//   dscores_e = dloss * scale / T * (q_e (sum p_j + r) - [e a target] p_e - [e another] r q_e / q_rest)
//
// Bound by memory: a row is read once and stays in the registers of a warp or a block, which needs one barrier for it.  Every warp forms
// its exponentials relative to its own maximum, and the warps' maxima and sums meet in shared memory.  The targets are left out of
// these sums -- each warp finds its own by a ballot over the row's list -- and join them afterwards, so that the others' sum is one of positive
// terms, however little is left for them beside the targets.
#include "readout.cuh"

namespace pinkb {
namespace {

struct DistillArgs
{
    uint64_t n;
    uint32_t N, k, logits, rest;
    float inv_t, exp2_t, scale;      // 1 / T, log2(e) / T
    const void* scores; uint64_t ld;
    const uint8_t* mask;
    const uint32_t* neurons; const float* targets;
    const float* dloss;              // null: 1 for every row
    void* dscores; uint64_t ld_d;
    float* loss;
    uint32_t whole_mask, whole_d;    // the mask may be read, and dscores written, a chunk at a time
};

__device__ __forceinline__ float exp2_fast(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

__device__ __forceinline__ float redux_max(float v)      // (a NaN is passed over; it shows in the sums)
{
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// exp((v - m) / T); m = -infinity stands for a set without members.
__device__ __forceinline__ float relative(float v, float m, float exp2_t) { return exp2_fast((v - (m == -INFINITY ? 0.0f : m)) * exp2_t); }

// What the first warp of a row tells the others about its targets.
struct Row
{
    float p[32];                     // weight of a target; 0 where it is absent
    uint32_t neuron[32];             // kNoNeuron where it is absent
    float most, sum;                 // of the targets' exponentials
    float mass, rest;                // sum of p, and 1 minus it (0 without a.rest)
    uint32_t present;
    float warp_most[32], warp_sum[32];
};

// The targets of a row, a lane each.  `value` is the score of the lane's neuron, -infinity where it takes no part or the lane has none.
__device__ __forceinline__ void gather_targets(const DistillArgs& a, uint32_t lane, uint32_t neuron, float target, float value, Row* s)
{
    const bool there = value != -INFINITY;               // (also for a NaN, which shows in the loss)
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, there ? neuron : 0x80000000u + lane);
    const bool first = there && __ffs(same) - 1 == (int)lane;      // a neuron listed twice is one neuron
    const uint32_t present = __ballot_sync(0xFFFFFFFFu, there);
    const float most = redux_max(first ? value : -INFINITY);
    const float sum = warp_sum(first ? relative(value, most, a.exp2_t) : 0.0f);
    float p = target, mass = 1.0f, rest = 0.0f;
    if (a.logits) {
        const float t = there ? fminf(target, FLT_MAX) : -INFINITY, high = redux_max(t);
        p = there ? expf((t - high) * a.inv_t) : 0.0f;
        const float all = warp_sum(p);
        p = there ? p / all : 0.0f;
    } else if (a.rest) {
        double m = there ? (double)p : 0.0;              // (the rest is a difference)
#pragma unroll
        for (int o = 16; o; o >>= 1) m += __shfl_xor_sync(0xFFFFFFFFu, m, o);
        mass = (float)m;
        rest = fmaxf((float)(1.0 - m), 0.0f);
    } else {
        mass = warp_sum(there ? p : 0.0f);
    }
    s->p[lane] = there ? p : 0.0f;
    s->neuron[lane] = there ? neuron : kNoNeuron;
    if (lane == 0) {
        s->most = most;
        s->sum = sum;
        s->mass = mass;
        s->rest = rest;
        s->present = present;
    }
}

// Words with -infinity in the places that `out` marks, a bit an element.
template <typename T>
__device__ __forceinline__ uint4 without(const uint4& c, uint32_t out)
{
    constexpr uint32_t kNone = std::is_same<T, __nv_bfloat16>::value ? 0xFF80u : std::is_same<T, __half>::value ? 0xFC00u : 0xFF800000u;
    uint32_t w[4] = { c.x, c.y, c.z, c.w };
#pragma unroll
    for (uint32_t v = 0; v < kChunk<T>; ++v)
        if (out >> v & 1) {
            if constexpr (sizeof(T) == 4) w[v] = kNone;
            else w[v / 2] = v % 2 ? (w[v / 2] & 0xFFFFu) | kNone << 16 : (w[v / 2] & 0xFFFF0000u) | kNone;
        }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The same for neurons whose mask is zero: bytes of a whole chunk.
template <typename T>
__device__ __forceinline__ uint4 masked(const uint4& c, const uint8_t* mask)
{
    if constexpr (sizeof(T) == 4) {
        const uint32_t m = *reinterpret_cast<const uint32_t*>(mask);
        return make_uint4(m & 0xFFu ? c.x : 0xFF800000u, m & 0xFF00u ? c.y : 0xFF800000u, m & 0xFF0000u ? c.z : 0xFF800000u, m & 0xFF000000u ? c.w : 0xFF800000u);
    } else {
        constexpr uint32_t kNone = std::is_same<T, __nv_bfloat16>::value ? 0xFF80FF80u : 0xFC00FC00u;
        const uint2 m = *reinterpret_cast<const uint2*>(mask);
        const uint32_t a = __vcmpeq4(m.x, 0), b = __vcmpeq4(m.y, 0);           // 255 where an element is left out
        auto put = [&](uint32_t w, uint32_t out) { return (w & ~out) | (kNone & out); };
        return make_uint4(put(c.x, __byte_perm(a, 0, 0x1100)), put(c.y, __byte_perm(a, 0, 0x3322)), put(c.z, __byte_perm(b, 0, 0x1100)), put(c.w, __byte_perm(b, 0, 0x3322)));
    }
}

// The larger of two words of elements, element by element; a NaN is passed over.
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b)
{
    if constexpr (sizeof(T) == 4) return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    else {
        using Two = std::conditional_t<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>;
        const Two m = __hmax2(*reinterpret_cast<const Two*>(&a), *reinterpret_cast<const Two*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
}

constexpr uint32_t kDistillWarps = 4;                    // rows of a block, where a row is a warp's

// A row in the registers of a warp, or (BLOCK) of a block, CH chunks a thread.  The elements stay as they are (16-bit ones packed) and their exponentials are
// formed again for the gradient.
template <typename T, bool BLOCK, int CH, int ALIGN, bool GRAD>
__global__ void __launch_bounds__(BLOCK ? 512 : 32 * kDistillWarps) distill_kernel(const DistillArgs a)
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int P = kPairs<T>;
    using In = RowOf<T, ALIGN>;
    __shared__ Row rows_s[BLOCK ? 1 : kDistillWarps];
    const uint32_t lane = threadIdx.x & 31, warp = BLOCK ? threadIdx.x >> 5 : 0, warps = BLOCK ? blockDim.x >> 5 : 1;
    const uint32_t threads = warps * 32, t = warp * 32 + lane;
    Row* s = &rows_s[BLOCK ? 0 : threadIdx.x >> 5];
    const uint64_t row = BLOCK ? blockIdx.x : (uint64_t)blockIdx.x * kDistillWarps + (threadIdx.x >> 5);
    follow();
    if (!BLOCK && row >= a.n) return;
    const In in(a.scores, a.ld, row, a.n, a.N);
    const T* x = static_cast<const T*>(a.scores) + row * a.ld;
    typename In::Chunk on_way[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if ((t + i * threads) * V < a.N) on_way[i] = in.load((t + i * threads) * V);

    // the row's list: a target counts if its neuron exists and its weight is positive (its logit above -infinity)
    uint32_t neuron = kNoNeuron;
    float target = 0.0f;
    if (lane < a.k) {
        neuron = a.neurons[row * a.k + lane];
        target = a.targets[row * a.k + lane];
    }
    if (neuron >= a.N || !(a.logits ? target > -INFINITY : target > 0.0f)) neuron = kNoNeuron;
    if (warp == 0) {
        float value = -INFINITY;
        if (neuron != kNoNeuron && !(a.mask && !a.mask[neuron])) value = to_float(x[neuron]);
        gather_targets(a, lane, neuron, target, value, s);
    }
    // which of this thread's elements are in it
    uint64_t hits = 0;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t start = (i * threads + warp * 32) * V, at = neuron - start;
        uint32_t in_warp = __ballot_sync(0xFFFFFFFFu, neuron != kNoNeuron && at < 32 * V);
        while (in_warp) {
            const uint32_t e = __shfl_sync(0xFFFFFFFFu, at, __ffs(in_warp) - 1);
            if (e / V == lane) hits |= 1ull << (i * V + e % V);
            in_warp &= in_warp - 1;
        }
    }

    uint4 w[CH];
    uint32_t top[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) top[j] = 0;
    bool any = false;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t c = (t + i * threads) * V;
        if (c >= a.N) break;
        w[i] = in.all(on_way[i]);
        uint32_t out = (uint32_t)(hits >> (i * V)) & ((1u << V) - 1);          // elements that are left out of the sums
        const bool whole = c + V <= a.N;
        if (!whole) out |= 0xFFFFFFFFu << (a.N - c);
        if (a.mask) {
            if (a.whole_mask && whole) w[i] = masked<T>(w[i], a.mask + c);
            else
#pragma unroll
                for (uint32_t v = 0; v < V; ++v) out |= (uint32_t)(c + v < a.N && !a.mask[c + v]) << v;
        }
        if (out) w[i] = without<T>(w[i], out);
        const uint32_t v[4] = { w[i].x, w[i].y, w[i].z, w[i].w };
#pragma unroll
        for (int j = 0; j < 4; ++j) top[j] = i == 0 ? v[j] : larger<T>(top[j], v[j]);
        any = true;
    }
    float most = -INFINITY;
    if (any) {
        const F2 m0 = pair_of<T>(make_uint4(top[0], top[1], top[2], top[3]), 0);
        most = fmaxf(fmaxf(most, m0.lo()), m0.hi());
#pragma unroll
        for (int j = 1; j < P; ++j) {
            const F2 m = pair_of<T>(make_uint4(top[0], top[1], top[2], top[3]), j);
            most = fmaxf(most, fmaxf(m.lo(), m.hi()));
        }
    }
    most = redux_max(most);
    const F2 below = two(most == -INFINITY ? 0.0f : -most), by_t = two(a.exp2_t);
    auto exponentials = [&](const uint4& c, int j) {
        const F2 e = mul2(add2(pair_of<T>(c, j), below), by_t);
        return two(exp2_fast(e.lo()), exp2_fast(e.hi()));
    };
    F2 sum2 = two(0.0f);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if ((t + i * threads) * V >= a.N) break;
#pragma unroll
        for (int j = 0; j < P; ++j) sum2 = add2(sum2, exponentials(w[i], j));
    }
    const float sum = warp_sum(sum2.lo() + sum2.hi());

    // the others' maximum and sum, and those of all
    float rest_most = most, rest_sum = sum;
    if constexpr (BLOCK) {
        if (lane == 0) { s->warp_most[warp] = most; s->warp_sum[warp] = sum; }
        __syncthreads();
        const float m = lane < warps ? s->warp_most[lane] : -INFINITY;
        rest_most = redux_max(m);
        rest_sum = warp_sum(lane < warps ? s->warp_sum[lane] * relative(m, rest_most, a.exp2_t) : 0.0f);
    } else {
        __syncwarp();
    }
    const float all_most = fmaxf(rest_most, s->most);
    const float all_sum = s->sum * relative(s->most, all_most, a.exp2_t) + rest_sum * relative(rest_most, all_most, a.exp2_t);
    const float r = rest_most != -INFINITY ? s->rest : 0.0f;

    if (a.loss && warp == 0) {
        float term = 0.0f;
        const float p = s->p[lane];
        if (p > 0.0f) term = p * (logf(p) - ((to_float(x[s->neuron[lane]]) - all_most) * a.inv_t - logf(all_sum)));
        float loss = warp_sum(term);
        if (r > 0.0f) {
            // r / q_rest is near 1 where the targets have little: 1 / q_rest = 1 + x, x what they have over the others' sum
            const float x = s->sum / rest_sum * expf((s->most - rest_most) * a.inv_t), z = fmaf(r, x, -s->mass);
            if (x > FLT_MAX) loss += r * (logf(r) + (s->most - rest_most) * a.inv_t + logf(s->sum / rest_sum));
            else loss += r * (z > -0.5f ? log1pf(z) : logf(r) + log1pf(x));
        }
        if (lane == 0) a.loss[row] = s->present ? a.scale * loss : 0.0f;
    }
    if constexpr (GRAD) {
        const float by = s->present ? (a.dloss ? a.dloss[row] : 1.0f) * a.scale * a.inv_t : 0.0f;
        const float of_q = by * (s->mass + r) / all_sum, of_rest = r > 0.0f ? by * r / rest_sum : 0.0f;
        const float factor = of_q * relative(most, all_most, a.exp2_t) - of_rest * relative(most, rest_most, a.exp2_t);
        const bool finite = s->present && fabsf(factor) <= FLT_MAX;
        const F2 f2 = two(factor);
        T* d = static_cast<T*>(a.dscores) + row * a.ld_d;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const uint32_t c = (t + i * threads) * V;
            if (c >= a.N) break;
            F2 o[P];
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const F2 e = exponentials(w[i], j);
                o[j] = mul2(e, f2);
                if (!finite)                             // what takes no part stays zero beside a NaN, and a row without targets is zero whatever its scores
                    o[j] = two(e.lo() == 0.0f || !s->present ? 0.0f : o[j].lo(), e.hi() == 0.0f || !s->present ? 0.0f : o[j].hi());
            }
            store_pairs<T>(d + c, o, a.N - c, a.whole_d);
        }
        // the targets among them, one by one, behind their chunks
        while (hits) {
            const uint32_t b = __ffsll((long long)hits) - 1, e = (t + b / V * threads) * V + b % V;
            hits &= hits - 1;
            float p = 0.0f;
            bool there = false;
            for (uint32_t j = 0; j < a.k; ++j)
                if (s->neuron[j] == e) { p += s->p[j]; there = true; }
            // (a target whose neuron takes no part has no gradient)
            d[e] = from_float<T>(there ? fmaf(of_q, relative(to_float(x[e]), all_most, a.exp2_t), -by * p) : 0.0f);
        }
    }
}

template <typename T, int ALIGN, bool GRAD>
cudaError_t run_distill(const DistillArgs& a, cudaStream_t st)
{
    const uint32_t chunks = (a.N + kChunk<T> - 1) / kChunk<T>;
    const dim3 of_warps((unsigned)((a.n + kDistillWarps - 1) / kDistillWarps)), of_blocks((unsigned)a.n);
    if (chunks <= 32) return launch_following(distill_kernel<T, false, 1, ALIGN, GRAD>, of_warps, 32 * kDistillWarps, 0, st, a);
    if (chunks <= 64) return launch_following(distill_kernel<T, false, 2, ALIGN, GRAD>, of_warps, 32 * kDistillWarps, 0, st, a);
    if (chunks <= 128) return launch_following(distill_kernel<T, false, 4, ALIGN, GRAD>, of_warps, 32 * kDistillWarps, 0, st, a);
    if (a.n >= 1024 || chunks > 4 * 512) {
        const uint32_t warps = (chunks + 32 * 8 - 1) / (32 * 8);
        if (chunks <= 256) return launch_following(distill_kernel<T, false, 8, ALIGN, GRAD>, of_warps, 32 * kDistillWarps, 0, st, a);
        if constexpr (sizeof(T) == 4) if (warps > 16) return launch_following(distill_kernel<T, true, 16, ALIGN, GRAD>, of_blocks, 512, 0, st, a);
        return launch_following(distill_kernel<T, true, 8, ALIGN, GRAD>, of_blocks, 32 * warps, 0, st, a);
    }
    return launch_following(distill_kernel<T, true, 4, ALIGN, GRAD>, of_blocks, (chunks + 127) / 128 * 32, 0, st, a);
}

int distill(const pink_b200_distill_config* cfg, uint64_t n, uint32_t type, const void* scores, uint64_t ld, const uint8_t* mask, const uint32_t* neurons,
            const float* targets, const float* dloss, void* dscores, uint64_t ld_d, float* loss, bool grad, cudaStream_t st)
{
    if (!cfg) return report_error(PINK_B200_EINVAL, "null argument");
    if (cfg->n_neurons == 0 || cfg->n_neurons > PINK_B200_MAX_ROUTED_NEURONS) return report_error(PINK_B200_EINVAL, "1 to 32768 neurons");
    if (cfg->top_k == 0 || cfg->top_k > PINK_B200_MAX_ROUTES) return report_error(PINK_B200_EINVAL, "top_k must be 1 to 32");
    if (cfg->teacher > PINK_B200_TEACHER_LOGITS) return report_error(PINK_B200_EINVAL, "unknown teacher");
    if (cfg->rest > 1) return report_error(PINK_B200_EINVAL, "rest must be 0 or 1");
    if (cfg->rest && cfg->teacher == PINK_B200_TEACHER_LOGITS) return report_error(PINK_B200_EINVAL, "the softmax of logits leaves no rest");
    if (!(cfg->temperature >= 1e-3f) || !(cfg->temperature <= 1e3f)) return report_error(PINK_B200_EINVAL, "temperature must be 0.001 to 1000");
    if (!(cfg->scale > 0.0f) || !(cfg->scale <= FLT_MAX)) return report_error(PINK_B200_EINVAL, "scale must be positive and finite");
    if (type > PINK_B200_F16) return report_error(PINK_B200_EINVAL, "unknown element type");
    if (n > 0x7FFFFFFFull) return report_error(PINK_B200_EINVAL, "too many rows");
    if (ld < cfg->n_neurons || (grad && ld_d < cfg->n_neurons)) return report_error(PINK_B200_EINVAL, "leading dimension smaller than the row");
    if (n == 0) return PINK_B200_OK;
    if (!scores || !neurons || !targets || !(grad ? dscores : loss)) return report_error(PINK_B200_EINVAL, "null argument");
    const double inv = 1.0 / (double)cfg->temperature;
    DistillArgs a{n, cfg->n_neurons, cfg->top_k, cfg->teacher, cfg->rest, (float)inv, (float)(inv * 1.4426950408889634), cfg->scale, scores, ld, mask, neurons,
                  targets, dloss, dscores, ld_d, loss, 0, 0};
    return launch_status(with_type(type, [&](auto t) {
        using T = decltype(t);
        a.whole_mask = reinterpret_cast<uintptr_t>(mask) % kChunk<T> == 0;
        a.whole_d = RowAlign().add(dscores, ld_d, sizeof(T)).elements(sizeof(T), kChunk<T>) == kChunk<T>;
        return with_alignment(alignment_of(RowAlign().add(scores, ld, sizeof(T)), sizeof(T)), [&](auto align) {
            constexpr int ALIGN = decltype(align)::value;
            return grad ? run_distill<T, ALIGN, true>(a, st) : run_distill<T, ALIGN, false>(a, st);
        });
    }), grad ? "distillation gradient" : "distillation");
}

} // namespace
} // namespace pinkb

using namespace pinkb;

extern "C" {

int pink_b200_op_distill(const pink_b200_distill_config* cfg, uint64_t n, uint32_t type, const void* dev_scores, uint64_t ld_scores, const uint8_t* dev_mask,
                         const uint32_t* dev_neurons, const float* dev_targets, float* dev_loss, void* stream)
{
    return distill(cfg, n, type, dev_scores, ld_scores, dev_mask, dev_neurons, dev_targets, nullptr, nullptr, 0, dev_loss, false, static_cast<cudaStream_t>(stream));
}

int pink_b200_op_distill_backward(const pink_b200_distill_config* cfg, uint64_t n, uint32_t type, const void* dev_scores, uint64_t ld_scores,
                                  const uint8_t* dev_mask, const uint32_t* dev_neurons, const float* dev_targets, const float* dev_dloss,
                                  void* dev_dscores, uint64_t ld_dscores, float* dev_loss, void* stream)
{
    return distill(cfg, n, type, dev_scores, ld_scores, dev_mask, dev_neurons, dev_targets, dev_dloss, dev_dscores, ld_dscores, dev_loss, true,
                   static_cast<cudaStream_t>(stream));
}

} // extern "C"
