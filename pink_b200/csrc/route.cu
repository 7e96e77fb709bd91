// Routing of images to neurons and its gradient (pink_b200_op_route*): logits, choice of the top k under a bias and groups,
// weights from softmax or sigmoid scores.
//
// With l = fl(slope * value) and c = fl(l + bias), both rounded to float32 once, the choice is a function of exact numbers: it
// does not depend on how a softmax is summed, so that equal inputs choose equal neurons in every kernel here.
#include "readout.cuh"

namespace pinkb {
namespace {

struct RouteArgs
{
    uint64_t n;
    uint32_t N, k, softmax, renormalise, groups, top_groups, group_best;
    float slope, scale;
    const void* values; uint64_t ld;
    const float* bias; const uint8_t* mask;
    uint32_t* neurons; float* weights; uint32_t* load;
    void* scores; uint64_t ld_scores;
};

constexpr float kNone = -INFINITY;     // logit or choice of a neuron that takes no part

// Logit of a value; kNone where the neuron takes no part.  (Adding zero turns -0 into +0, so that both compare and sort alike.)
__device__ __forceinline__ float logit_of(float v, float slope)
{
    const float l = __fadd_rn(__fmul_rn(slope, v), 0.0f);
    return l == l ? fminf(l, FLT_MAX) : kNone;
}

__device__ __forceinline__ float choice_of(float l, float bias)
{
    if (l == kNone) return kNone;
    const float c = __fadd_rn(__fadd_rn(l, bias), 0.0f);
    return c == c ? fminf(c, FLT_MAX) : kNone;
}

// Unsigned word that orders as the float does.
__device__ __forceinline__ uint32_t ordered(float v)
{
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float sigmoid_of(float l)
{
    // exp of a non-positive number only: no overflow, and full accuracy in both tails
    const float e = expf(-fabsf(l));
    return (l >= 0.0f ? 1.0f : e) / (1.0f + e);
}

constexpr uint32_t kRowThreads = 256, kRowWarps = kRowThreads / 32;

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* scratch, Op op)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    __syncthreads();                                     // the scratch's earlier readers are done
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (uint32_t w = 1; w < kRowWarps; ++w) v = op(v, scratch[w]);
    return v;
}

struct Max { template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; } };
struct Sum { __device__ float operator()(float a, float b) const { return a + b; } };

// The k chosen neurons of a row, lane by lane of one warp: weights, counters and results.  `l` is the logit of the lane's neuron
// (kNone where it has none), p its score where it is not renormalised.
__device__ __forceinline__ void write_routes(const RouteArgs& a, uint64_t row, uint32_t lane, uint32_t neuron, float l, float p)
{
    float w = p;
    if (a.renormalise) {
        // relative to the largest: softmax exp(l) and sigmoid exp(min(l, 0)) / (1 + exp(-|l|)) over one common exponential
        const float e = a.softmax ? l : fminf(l, 0.0f);
        const float most = warp_max(e);
        w = neuron == kNoNeuron ? 0.0f : expf(e - most) / (a.softmax ? 1.0f : 1.0f + expf(-fabsf(l)));
        const float sum = warp_sum(w);
        w = neuron == kNoNeuron ? 0.0f : w / sum;
    }
    if (lane < a.k) {
        a.neurons[row * a.k + lane] = neuron;
        a.weights[row * a.k + lane] = neuron == kNoNeuron ? 0.0f : a.scale * w;
        if (a.load && neuron != kNoNeuron) atomicAdd(&a.load[neuron], 1u);
    }
}

// Best of a group and, with group_best = 2, its sum with the second best, held to the range of finite floats.
__device__ __forceinline__ float group_value(float best, float second, uint32_t group_best)
{
    if (group_best == 2 && second != kNone)
        best = fmaxf(fminf(__fadd_rn(__fadd_rn(best, second), 0.0f), FLT_MAX), -FLT_MAX);
    return best;
}

// Key whose maximum is the largest choice and, of equal ones, the first; 0: nothing to choose.
__device__ __forceinline__ unsigned long long choice_key(float c, uint32_t j)
{
    return c == kNone ? 0ull : (unsigned long long)ordered(c) << 32 | (0xFFFFFFFFu - j);
}

// A block per image; the row's choices lie in shared memory.  Serves every size.
template <typename T, typename S>
__global__ void __launch_bounds__(kRowThreads) route_row_kernel(const RouteArgs a)
{
    extern __shared__ float choice[];                    // [N] choices, then [groups] values
    __shared__ float fscratch[kRowWarps];
    __shared__ unsigned long long kscratch[kRowWarps];
    __shared__ uint32_t kept[PINK_B200_MAX_ROUTE_GROUPS / 32];
    __shared__ uint32_t chosen[PINK_B200_MAX_ROUTES];
    const uint64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.values) + row * a.ld;
    const uint32_t t = threadIdx.x;
    auto logit = [&](uint32_t j) { return a.mask && !a.mask[j] ? kNone : logit_of(to_float(x[j]), a.slope); };

    float most = kNone;
    for (uint32_t j = t; j < a.N; j += kRowThreads) {
        const float l = logit(j);
        most = fmaxf(most, l);
        choice[j] = a.bias ? choice_of(l, a.bias[j]) : l;
    }
    const bool dense = a.scores || !a.renormalise;       // the scores of all neurons matter
    float inv = 0.0f;
    if (a.softmax && dense) {
        most = block_reduce(most, fscratch, Max());
        float sum = 0.0f;
        if (most != kNone)
            for (uint32_t j = t; j < a.N; j += kRowThreads) sum += expf(logit(j) - most);
        sum = block_reduce(sum, fscratch, Sum());
        inv = sum > 0.0f ? 1.0f / sum : 0.0f;            // a row without neurons has no scores
    }
    auto score = [&](float l) { return l == kNone ? 0.0f : a.softmax ? expf(l - most) * inv : sigmoid_of(l); };
    if (a.scores) {
        S* out = static_cast<S*>(a.scores) + row * a.ld_scores;
        for (uint32_t j = t; j < a.N; j += kRowThreads) out[j] = from_float<S>(score(logit(j)));
    }
    __syncthreads();
    const uint32_t size = a.N / a.groups;
    if (a.groups > 1) {
        float* gvalue = choice + a.N;
        for (uint32_t g = t; g < a.groups; g += kRowThreads) {
            float best = kNone, second = kNone;
            for (uint32_t j = g * size; j < (g + 1) * size; ++j) {
                const float c = choice[j];
                if (c > best) { second = best; best = c; }
                else if (c > second) second = c;
            }
            gvalue[g] = group_value(best, second, a.group_best);
        }
        if (t < PINK_B200_MAX_ROUTE_GROUPS / 32) kept[t] = 0;
        __syncthreads();
        for (uint32_t r = 0; r < a.top_groups; ++r) {
            unsigned long long best = 0;
            for (uint32_t g = t; g < a.groups; g += kRowThreads) best = Max()(best, choice_key(gvalue[g], g));
            best = block_reduce(best, kscratch, Max());
            if (best == 0) break;
            const uint32_t g = 0xFFFFFFFFu - (uint32_t)best;
            if (t == g % kRowThreads) { gvalue[g] = kNone; kept[g >> 5] |= 1u << (g & 31); }   // (its reader in the next round)
            __syncthreads();
        }
        for (uint32_t j = t; j < a.N; j += kRowThreads) {
            const uint32_t g = j / size;
            if (!(kept[g >> 5] >> (g & 31) & 1u)) choice[j] = kNone;
        }
    }
    if (t < PINK_B200_MAX_ROUTES) chosen[t] = kNoNeuron;
    for (uint32_t r = 0; r < a.k; ++r) {
        unsigned long long best = 0;
        for (uint32_t j = t; j < a.N; j += kRowThreads) best = Max()(best, choice_key(choice[j], j));
        best = block_reduce(best, kscratch, Max());
        if (best == 0) break;
        const uint32_t j = 0xFFFFFFFFu - (uint32_t)best;
        if (t == j % kRowThreads) choice[j] = kNone;     // (its reader in the next round)
        if (t == 0) chosen[r] = j;
    }
    __syncthreads();
    if (t < 32) {
        const uint32_t j = chosen[t];
        const float l = j == kNoNeuron ? kNone : logit(j);
        write_routes(a, row, t, j, l, score(l));
    }
}

// ---- gradient ------------------------------------------------------------------------------------------------------------

struct RouteGradArgs
{
    uint64_t n;
    uint32_t N, k, softmax, renormalise;
    float slope, scale;
    const void* values; uint64_t ld;
    const uint8_t* mask;
    const uint32_t* neurons; const float* weights; const float* dweights;
    const void* dscores; uint64_t ld_dscores;
    void* dvalues; uint64_t ld_dvalues;
};

// A block per image.  With g the gradient of a weight and G that of a score (G = dscores, plus scale * g at the routes where
// they are not renormalised):
//   softmax   dl = p (G - sum G p),   renormalised routes add  w (g - sum g w / scale)
//   sigmoid   dl = G p (1 - p),       renormalised routes add  w (g - sum g w / scale) (1 - p)
template <typename T>
__global__ void __launch_bounds__(kRowThreads) route_grad_row_kernel(const RouteGradArgs a)
{
    extern __shared__ float grad[];                      // [N] what the routes add: to G, or (renormalised) to dl
    __shared__ float fscratch[kRowWarps];
    const uint64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(a.values) + row * a.ld;
    const T* ds = a.dscores ? static_cast<const T*>(a.dscores) + row * a.ld_dscores : nullptr;
    T* out = static_cast<T*>(a.dvalues) + row * a.ld_dvalues;
    const uint32_t t = threadIdx.x;
    auto logit = [&](uint32_t j) { return a.mask && !a.mask[j] ? kNone : logit_of(to_float(x[j]), a.slope); };

    for (uint32_t j = t; j < a.N; j += kRowThreads) grad[j] = 0.0f;
    __syncthreads();
    if (t < 32) {
        const uint32_t j = t < a.k ? a.neurons[row * a.k + t] : kNoNeuron;
        const bool there = j < a.N;
        const float g = there ? a.dweights[row * a.k + t] : 0.0f, w = there ? a.weights[row * a.k + t] : 0.0f;
        float d = a.scale * g;
        if (a.renormalise) {
            const float mean = warp_sum(g * w) / a.scale;
            d = w * (g - mean);
            if (!a.softmax && there) d *= sigmoid_of(-logit(j));
        }
        // a neuron may be listed twice: one lane after the other
        for (uint32_t r = 0; r < a.k; ++r) {
            if (t == r && there) grad[j] += d;
            __syncwarp();
        }
    }
    __syncthreads();
    const bool dense = ds || !a.renormalise;
    float most = kNone, inv = 0.0f, mean = 0.0f;
    if (a.softmax && dense) {
        for (uint32_t j = t; j < a.N; j += kRowThreads) most = fmaxf(most, logit(j));
        most = block_reduce(most, fscratch, Max());
        float sum = 0.0f, dot = 0.0f;
        if (most != kNone)
            for (uint32_t j = t; j < a.N; j += kRowThreads) {
                const float l = logit(j);
                if (l == kNone) continue;
                const float e = expf(l - most), G = (ds ? to_float(ds[j]) : 0.0f) + (a.renormalise ? 0.0f : grad[j]);
                sum += e;
                dot += e * G;
            }
        sum = block_reduce(sum, fscratch, Sum());
        dot = block_reduce(dot, fscratch, Sum());
        inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        mean = dot * inv;
    }
    for (uint32_t j = t; j < a.N; j += kRowThreads) {
        const float l = logit(j);
        float d = 0.0f;
        if (l != kNone) {
            if (dense) {
                const float G = (ds ? to_float(ds[j]) : 0.0f) + (a.renormalise ? 0.0f : grad[j]);
                d = a.softmax ? expf(l - most) * inv * (G - mean) : G * sigmoid_of(l) * sigmoid_of(-l);
            }
            if (a.renormalise) d += grad[j];
        }
        out[j] = from_float<T>(l == kNone ? 0.0f : a.slope * d);
    }
}

// ---- balance -------------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(1024) balance_kernel(uint32_t N, const uint32_t* load, const uint8_t* mask, float rate,
                                                       const float* bias, float* out)
{
    __shared__ unsigned long long total_s, members_s;
    if (threadIdx.x == 0) total_s = members_s = 0;
    __syncthreads();
    unsigned long long total = 0, members = 0;
    for (uint32_t j = threadIdx.x; j < N; j += blockDim.x)
        if (!mask || mask[j]) { total += load[j]; ++members; }
    for (int o = 16; o; o >>= 1) {
        total += __shfl_xor_sync(0xFFFFFFFFu, total, o);
        members += __shfl_xor_sync(0xFFFFFFFFu, members, o);
    }
    if ((threadIdx.x & 31) == 0) { atomicAdd(&total_s, total); atomicAdd(&members_s, members); }
    __syncthreads();
    total = total_s; members = members_s;
    for (uint32_t j = threadIdx.x; j < N; j += blockDim.x) {
        float b = bias[j];
        if (!mask || mask[j]) {
            const unsigned long long mine = members * load[j];       // < 2^15 * 2^32
            if (total > mine) b += rate;
            else if (total < mine) b -= rate;
        }
        out[j] = b;
    }
}

int check_route(const pink_b200_route_config* c, uint64_t n, uint32_t type, uint64_t ld)
{
    if (!c) return report_error(PINK_B200_EINVAL, "null argument");
    if (c->n_neurons == 0 || c->n_neurons > PINK_B200_MAX_ROUTED_NEURONS)
        return report_error(PINK_B200_EINVAL, "a route chooses from 1 to 32768 neurons");
    if (c->top_k == 0 || c->top_k > PINK_B200_MAX_ROUTES || c->top_k > c->n_neurons)
        return report_error(PINK_B200_EINVAL, "top_k must be 1 to 32 and at most the number of neurons");
    if (c->score > PINK_B200_SCORE_SIGMOID) return report_error(PINK_B200_EINVAL, "unknown score function");
    if (c->renormalise > 1) return report_error(PINK_B200_EINVAL, "renormalise must be 0 or 1");
    if (!(c->slope == c->slope) || c->slope - c->slope != 0.0f) return report_error(PINK_B200_EINVAL, "slope must be finite");
    if (!(c->scale > 0.0f) || c->scale - c->scale != 0.0f) return report_error(PINK_B200_EINVAL, "scale must be positive and finite");
    if (type > PINK_B200_F16) return report_error(PINK_B200_EINVAL, "unknown element type");
    if (n > 0x7FFFFFFFull) return report_error(PINK_B200_EINVAL, "at most 2147483647 rows");
    if (ld < c->n_neurons) return report_error(PINK_B200_EINVAL, "leading dimension smaller than the number of neurons");
    return PINK_B200_OK;
}

} // namespace
} // namespace pinkb

using namespace pinkb;

extern "C" {

int pink_b200_op_route(const pink_b200_route_config* cfg, uint64_t n, uint32_t type, const void* dev_values, uint64_t ld_values,
                       const float* dev_bias, const uint8_t* dev_mask, uint32_t* dev_neurons, float* dev_weights,
                       uint32_t* dev_load, uint32_t scores_type, void* dev_scores, uint64_t ld_scores, void* stream)
{
    const int rc = check_route(cfg, n, type, ld_values);
    if (rc) return rc;
    if (cfg->n_groups == 0 || cfg->n_groups > PINK_B200_MAX_ROUTE_GROUPS || cfg->n_neurons % cfg->n_groups)
        return report_error(PINK_B200_EINVAL, "n_groups must be 1 to 256 and divide the number of neurons");
    if (cfg->top_groups == 0 || cfg->top_groups > cfg->n_groups)
        return report_error(PINK_B200_EINVAL, "top_groups must be 1 to n_groups");
    if (cfg->n_groups > 1 && (uint64_t)cfg->top_groups * (cfg->n_neurons / cfg->n_groups) < cfg->top_k)
        return report_error(PINK_B200_EINVAL, "top_groups groups have fewer than top_k neurons");
    if (cfg->group_best != 1 && cfg->group_best != 2) return report_error(PINK_B200_EINVAL, "group_best must be 1 or 2");
    if (dev_scores && (scores_type > PINK_B200_F16 || ld_scores < cfg->n_neurons))
        return report_error(PINK_B200_EINVAL, "bad element type or leading dimension of the dense scores");
    if (n == 0) return PINK_B200_OK;
    if (!dev_values || !dev_neurons || !dev_weights) return report_error(PINK_B200_EINVAL, "null argument");
    RouteArgs a{n, cfg->n_neurons, cfg->top_k, cfg->score == PINK_B200_SCORE_SOFTMAX, cfg->renormalise, cfg->n_groups, cfg->top_groups,
                cfg->group_best, cfg->slope, cfg->scale, dev_values, ld_values, dev_bias, dev_mask, dev_neurons, dev_weights, dev_load,
                dev_scores, ld_scores};
    const size_t smem = (a.N + (a.groups > 1 ? a.groups : 0)) * sizeof(float);
    return launch_status(with_type(type, [&](auto v) {
        return with_type(dev_scores ? scores_type : PINK_B200_F32, [&](auto s) {
            auto* kernel = route_row_kernel<decltype(v), decltype(s)>;
            cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return e;
            kernel<<<(unsigned)n, kRowThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
            return cudaGetLastError();
        });
    }), "route kernel");
}

int pink_b200_op_route_backward(const pink_b200_route_config* cfg, uint64_t n, uint32_t type, const void* dev_values, uint64_t ld_values,
                                const uint8_t* dev_mask, const uint32_t* dev_neurons, const float* dev_weights,
                                const float* dev_dweights, const void* dev_dscores, uint64_t ld_dscores, void* dev_dvalues,
                                uint64_t ld_dvalues, void* stream)
{
    const int rc = check_route(cfg, n, type, ld_values);
    if (rc) return rc;
    if (ld_dvalues < cfg->n_neurons || (dev_dscores && ld_dscores < cfg->n_neurons))
        return report_error(PINK_B200_EINVAL, "leading dimension smaller than the number of neurons");
    if (n == 0) return PINK_B200_OK;
    if (!dev_values || !dev_neurons || !dev_weights || !dev_dweights || !dev_dvalues) return report_error(PINK_B200_EINVAL, "null argument");
    RouteGradArgs a{n, cfg->n_neurons, cfg->top_k, cfg->score == PINK_B200_SCORE_SOFTMAX, cfg->renormalise, cfg->slope, cfg->scale,
                    dev_values, ld_values, dev_mask, dev_neurons, dev_weights, dev_dweights, dev_dscores, ld_dscores, dev_dvalues, ld_dvalues};
    const size_t smem = a.N * sizeof(float);
    return launch_status(with_type(type, [&](auto v) {
        auto* kernel = route_grad_row_kernel<decltype(v)>;
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        kernel<<<(unsigned)n, kRowThreads, smem, static_cast<cudaStream_t>(stream)>>>(a);
        return cudaGetLastError();
    }), "route gradient kernel");
}

int pink_b200_op_route_balance(uint32_t n_neurons, const uint32_t* dev_load, const uint8_t* dev_mask, float rate, const float* dev_bias,
                               float* dev_new_bias, void* stream)
{
    if (n_neurons == 0 || n_neurons > PINK_B200_MAX_ROUTED_NEURONS)
        return report_error(PINK_B200_EINVAL, "a route chooses from 1 to 32768 neurons");
    if (!(rate == rate) || rate - rate != 0.0f) return report_error(PINK_B200_EINVAL, "rate must be finite");
    if (!dev_load || !dev_bias || !dev_new_bias) return report_error(PINK_B200_EINVAL, "null argument");
    balance_kernel<<<1, n_neurons < 1024 ? 256 : 1024, 0, static_cast<cudaStream_t>(stream)>>>(n_neurons, dev_load, dev_mask, rate,
                                                                                           dev_bias, dev_new_bias);
    return launch_status(cudaGetLastError(), "balance kernel");
}

} // extern "C"
