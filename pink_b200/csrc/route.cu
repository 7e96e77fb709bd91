// Routing of images to neurons and its gradient (pink_b200_op_route*): logits, choice of the top k under a bias and groups,
// weights from softmax or sigmoid scores.
//
// With l = fl(slope * value) and c = fl(l + bias), both rounded to float32 once, the choice is a function of exact numbers: it
// does not depend on how a softmax is summed, so that equal inputs choose equal neurons in every kernel here.
//
// The kernels of an element type are a module of their own (PINK_ROUTE_TYPE = 0, 1, 2: float32, bfloat16, float16), so that a process
// loads what it uses; without the macro this file holds the entry points.
#include "readout.cuh"

namespace pinkb {

struct RouteArgs
{
    uint64_t n;
    uint32_t N, k, softmax, renormalise, groups, top_groups, group_best;
    float slope, scale;
    const void* values; uint64_t ld;
    const float* bias; const uint8_t* mask;
    uint32_t* neurons; float* weights; uint32_t* load;
    uint32_t scores_type; void* scores; uint64_t ld_scores;
};

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

template <typename T> cudaError_t run_route(const RouteArgs& a, cudaStream_t st);
template <typename T> cudaError_t run_route_grad(const RouteGradArgs& a, cudaStream_t st);

#ifdef PINK_ROUTE_TYPE

namespace {

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

// Maximum over a warp in one instruction.
__device__ __forceinline__ float warp_max_redux(float v)
{
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// The k chosen neurons of a row, lane by lane of one warp: weights, counters and results.  `l` is the logit of the lane's neuron
// (kNone where it has none), p its score where it is not renormalised.
__device__ __forceinline__ void write_routes(const RouteArgs& a, uint64_t row, uint32_t lane, uint32_t neuron, float l, float p)
{
    float w = p;
    if (a.renormalise) {
        // relative to the largest: softmax exp(l) and sigmoid exp(min(l, 0)) / (1 + exp(-|l|)) over one common exponential
        const float e = a.softmax ? l : fminf(l, 0.0f);
        const float most = warp_max_redux(e);
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

__device__ __forceinline__ void store_score(void* scores, uint32_t type, uint64_t at, float p)
{
    if (type == PINK_B200_F32) static_cast<float*>(scores)[at] = p;
    else if (type == PINK_B200_BF16) static_cast<__nv_bfloat16*>(scores)[at] = from_float<__nv_bfloat16>(p);
    else static_cast<__half*>(scores)[at] = from_float<__half>(p);
}

// A block per image; the row's choices lie in shared memory.  For rows that do not fit the registers of route_kernel below.
template <typename T>
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
    if (a.scores)
        for (uint32_t j = t; j < a.N; j += kRowThreads) store_score(a.scores, a.scores_type, row * a.ld_scores + j, score(logit(j)));
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

// ---- rows in registers ---------------------------------------------------------------------------------------------------
// WARPS warps per image, whose values stay in registers: element i * 32 * WARPS + t is the i-th of thread t.  The chosen neurons are
// found without sorting the row: the k-th largest of the threads' maxima (within a warp; the largest over the warps) is a bound that
// k elements reach, so only the few that reach it can be chosen; they are collected in shared memory, and the place of each is the number
// of those that beat it.  Should more reach it than fit (many equal values), the k are taken one after the other.
//
// Measured, 65,536 images of 2,791 neurons, eight routes and a bias: 211 us, 3.5 TB/s of the 6.45 a copy reaches.  A row passes through
// phases that wait for one another (its load, the bound, the candidates, the weights), and eight rows an SM do not hide all of that.
// Instructions are the other limit, so an element costs few of them: its product with the slope (and, with a bias, a
// minimum and a sum) is all that is formed for every element.  NaN needs no test of its own, since fmaxf passes it over and no comparison
// holds for it; +infinity is caught by holding the bound to finite floats, and -infinity as well.

constexpr uint32_t kRegThreads = 128;                    // threads of a block of one-warp images
constexpr uint32_t kCandidates = 128;

// As logit_of, in fewer instructions: fmaxf turns NaN into kNone.  (-0 stays: it compares as +0 does.)
__device__ __forceinline__ float held(float v) { return fminf(fmaxf(v, kNone), FLT_MAX); }

// min(v, FLT_MAX), NaN where v is.
__device__ __forceinline__ float below_infinity(float v)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(FLT_MAX));
    return r;
}

// The largest of three (NaN passed over), in one instruction.
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// e^v for v <= 0 in two instructions (results below 2^-126 are zero).  The product rounds once more than in expf: |v| units of 2^-24.
__device__ __forceinline__ float exp_of(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v * 1.44269504f));
    return r;
}

template <int WARPS> __host__ __device__ constexpr uint32_t images_per_block() { return WARPS * 32 < kRegThreads ? kRegThreads / (WARPS * 32) : 1; }

// Barrier of the threads of one image: a warp, or a block.
template <int WARPS> __device__ __forceinline__ void row_sync()
{
    static_assert(WARPS == 1 || images_per_block<WARPS>() == 1, "images of several warps have a block each");
    if (WARPS == 1) __syncwarp();
    else __syncthreads();
}

// Reduction over the threads of an image; `scratch` has a word per warp.
template <int WARPS, typename V, typename Op>
__device__ __forceinline__ V row_reduce(V v, V* scratch, uint32_t t, Op op)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    if (WARPS == 1) return v;
    row_sync<WARPS>();
    if ((t & 31) == 0) scratch[t >> 5] = v;
    row_sync<WARPS>();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) v = op(v, scratch[w]);
    return v;
}

// Two sums at once.
template <int WARPS>
__device__ __forceinline__ float2 row_sums(float2 v, float2* scratch, uint32_t t)
{
    v.x = warp_sum(v.x);
    v.y = warp_sum(v.y);
    if (WARPS == 1) return v;
    if ((t & 31) == 0) scratch[t >> 5] = v;
    row_sync<WARPS>();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) { v.x += scratch[w].x; v.y += scratch[w].y; }
    return v;
}

// fn(i, j, in) for the thread's elements j = i * THREADS + t, eight at a time: whole eights without a test, eights beyond N not at all.
// AHEAD lets the compiler load for later eights before it is done with one: wanted for the row itself, which is held
// anyway; elsewhere it would cost a register per element.
constexpr int kChunk = 8;

template <int ITEMS, uint32_t THREADS, bool AHEAD = false, typename Fn>
__device__ __forceinline__ void each_item(uint32_t N, uint32_t t, Fn fn)
{
    static_assert(ITEMS % kChunk == 0, "whole chunks");
    asm volatile("" : "+r"(N));                          // the tests below are made anew in every pass, not kept in registers
#pragma unroll
    for (int c = 0; c < ITEMS; c += kChunk) {
        if (!AHEAD) asm volatile("" ::: "memory");
        if ((c + kChunk) * THREADS <= N) {
#pragma unroll
            for (int i = c; i < c + kChunk; ++i) fn(i, i * THREADS + t, true);
        } else if (c * THREADS < N) {
#pragma unroll
            for (int i = c; i < c + kChunk; ++i) fn(i, i * THREADS + t, i * THREADS + t < N);
        }
    }
}

template <typename T, int WARPS, int ITEMS>
__global__ void __launch_bounds__(WARPS * 32 < kRegThreads ? kRegThreads : WARPS * 32, WARPS > 4 ? 1 : ITEMS > 16 ? 8 : 10) route_kernel(const RouteArgs a)
{
    constexpr uint32_t kThreads = WARPS * 32, kImages = images_per_block<WARPS>();
    __shared__ unsigned long long cand_s[kImages][kCandidates];
    __shared__ uint32_t count_s[kImages];
    __shared__ float cand_logit_s[kImages][kCandidates];
    __shared__ uint32_t chosen_s[kImages][PINK_B200_MAX_ROUTES];
    __shared__ float logit_s[kImages][PINK_B200_MAX_ROUTES];
    __shared__ float fscratch_s[kImages][WARPS], bounds_s[kImages][WARPS];
    __shared__ unsigned long long kscratch_s[kImages][WARPS];
    extern __shared__ float group_s[];                   // with groups: per image [N] choices, [groups] values and [groups] marks
    const uint32_t image = kImages > 1 ? threadIdx.x / kThreads : 0, t = kImages > 1 ? threadIdx.x % kThreads : threadIdx.x;
    const uint64_t row = (uint64_t)blockIdx.x * kImages + image;
    follow();
    if (kImages > 1 && row >= a.n) return;               // (all threads of the image, which wait for no other's)
    const T* x = static_cast<const T*>(a.values) + row * a.ld;

    float l[ITEMS];                                      // values, then logits, then choices
    each_item<ITEMS, kThreads, true>(a.N, t, [&](int i, uint32_t j, bool in) { l[i] = in ? to_float(x[j]) : NAN; });
    if (t < PINK_B200_MAX_ROUTES) chosen_s[image][t] = kNoNeuron;
    if (t == 0) count_s[image] = 0;
    float top[4] = { kNone, kNone, kNone, kNone };       // the thread's largest choice, in four parts that do not wait for one another
    float most = kNone, inv = 0.0f;
    if (!a.mask && !a.scores && a.renormalise && a.groups == 1) {
        // nothing but the choice is asked for: one pass
        if (a.bias)
            each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t j, bool in) {
                l[i] = __fadd_rn(below_infinity(__fmul_rn(a.slope, l[i])), in ? a.bias[j] : 0.0f);
                if (i & 1) top[i / 2 & 3] = max3(top[i / 2 & 3], l[i - 1], l[i]);
            });
        else
            each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) {
                l[i] = __fmul_rn(a.slope, l[i]);
                if (i & 1) top[i / 2 & 3] = max3(top[i / 2 & 3], l[i - 1], l[i]);
            });
    } else {
        each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) { l[i] = __fmul_rn(a.slope, l[i]); });
        if (a.mask) each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t j, bool in) { if (in && !a.mask[j]) l[i] = kNone; });
        if (a.scores || !a.renormalise) {                // the scores of all neurons matter
            each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) { l[i] = held(l[i]); });
            if (a.softmax) {
                each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) { if (i & 1) top[i / 2 & 3] = max3(top[i / 2 & 3], l[i - 1], l[i]); });
                most = row_reduce<WARPS>(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), fscratch_s[image], t, Max());
                const float m = most == kNone ? 0.0f : most;
                float sum[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
                each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) { sum[i & 3] += exp_of(l[i] - m); });      // (kNone: zero)
                const float all = row_reduce<WARPS>(sum[0] + sum[1] + (sum[2] + sum[3]), fscratch_s[image], t, Sum());
                inv = all > 0.0f ? 1.0f / all : 0.0f;
            }
        }
        if (a.scores)
            each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t j, bool in) {
                if (in) store_score(a.scores, a.scores_type, row * a.ld_scores + j, l[i] == kNone ? 0.0f : a.softmax ? exp_of(l[i] - most) * inv : sigmoid_of(l[i]));
            });
        if (a.bias) each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t j, bool in) { if (in) l[i] = __fadd_rn(below_infinity(l[i]), a.bias[j]); });

        if (a.groups > 1) {
            const uint32_t size = a.N / a.groups;
            float* choice = group_s + (size_t)image * (a.N + 2 * a.groups);
            float* value = choice + a.N;
            uint32_t* kept = reinterpret_cast<uint32_t*>(value + a.groups);
            each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t j, bool in) { if (in) choice[j] = held(l[i]); });
            row_sync<WARPS>();
            for (uint32_t g = t; g < a.groups; g += kThreads) {
                float best = kNone, second = kNone;
#pragma unroll 4
                for (uint32_t j = g * size; j < (g + 1) * size; ++j) {
                    const float c = choice[j];
                    second = fmaxf(second, fminf(best, c));
                    best = fmaxf(best, c);
                }
                value[g] = group_value(best, second, a.group_best);
            }
            row_sync<WARPS>();
            for (uint32_t g = t; g < a.groups; g += kThreads) {
                const float v = value[g];
                uint32_t better = 0;
#pragma unroll 4
                for (uint32_t h = 0; h < a.groups; ++h) better += value[h] > v || (value[h] == v && h < g);
                kept[g] = better < a.top_groups;
            }
            row_sync<WARPS>();
            // j / size as a product: exact for j, size < 2^16
            const uint32_t magic = size > 1 ? 0xFFFFFFFFu / size + 1 : 0;
            each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t j, bool in) { if (in && !kept[magic ? __umulhi(j, magic) : j]) l[i] = kNone; });
        }
        top[0] = top[1] = top[2] = top[3] = kNone;
        each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) { if (i & 1) top[i / 2 & 3] = max3(top[i / 2 & 3], l[i - 1], l[i]); });
    }
    auto score = [&](float v) { return v == kNone ? 0.0f : a.softmax ? exp_of(v - most) * inv : sigmoid_of(v); };

    // the bound
    const float mine = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    float bound, left = mine;
    for (uint32_t r = 0;;) {                             // (equal maxima go together: the bound is no higher for it)
        bound = warp_max_redux(left);
        if (++r == a.k) break;
        if (left == bound) left = kNone;
    }
    if (WARPS > 1) {
        if ((t & 31) == 0) bounds_s[image][t >> 5] = bound;
        row_sync<WARPS>();
#pragma unroll
        for (int w = 0; w < WARPS; ++w) bound = fmaxf(bound, bounds_s[image][w]);
    } else {
        __syncwarp();                                    // the counter is zero
    }
    bound = fminf(fmaxf(bound, -FLT_MAX), FLT_MAX);

    // the elements that reach it (none of them masked or left out by its group), with their logits
    if (mine >= bound) {
        static_assert(ITEMS <= 32, "a bit per element");
        uint32_t reach = 0;
        each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) { if (l[i] >= bound) reach |= 1u << i; });
        for (; reach; reach &= reach - 1) {
            const uint32_t at = atomicAdd(&count_s[image], 1u);
            const uint32_t j = (__ffs(reach) - 1) * kThreads + t;
            if (at < kCandidates) {
                const float v = __fmul_rn(a.slope, to_float(x[j]));
                const float c = held(a.bias ? __fadd_rn(below_infinity(v), a.bias[j]) : v);
                cand_s[image][at] = choice_key(c + 0.0f, j);                 // (-0 becomes +0, as keys need it)
                cand_logit_s[image][at] = held(v);
            }
        }
    }
    row_sync<WARPS>();
    const uint32_t count = count_s[image];
    if (count <= kCandidates) {
        for (uint32_t c = t; c < count; c += kThreads) {
            const unsigned long long key = cand_s[image][c];
            uint32_t better = 0;
#pragma unroll 4
            for (uint32_t h = 0; h < count; ++h) better += cand_s[image][h] > key;
            if (better < a.k) {
                chosen_s[image][better] = 0xFFFFFFFFu - (uint32_t)key;
                logit_s[image][better] = cand_logit_s[image][c];
            }
        }
    } else {
        unsigned long long last = ~0ull;
        for (uint32_t r = 0; r < a.k; ++r) {
            unsigned long long best = 0;
            each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t j, bool) {
                float c = l[i];
                asm volatile("" : "+f"(c));              // (keys formed here, not held over the rounds)
                const unsigned long long key = choice_key(held(c) + 0.0f, j);
                if (key < last && key > best) best = key;
            });
            best = row_reduce<WARPS>(best, kscratch_s[image], t, Max());
            if (best == 0) break;
            if (t == 0) {
                const uint32_t j = 0xFFFFFFFFu - (uint32_t)best;
                chosen_s[image][r] = j;
                logit_s[image][r] = held(__fmul_rn(a.slope, to_float(x[j])));
            }
            last = best;
        }
    }
    row_sync<WARPS>();
    if (t < 32) {
        const uint32_t j = chosen_s[image][t];
        const float v = j == kNoNeuron ? kNone : logit_s[image][t];
        write_routes(a, row, t, j, v, a.renormalise ? 0.0f : score(v));
    }
}

template <typename T, int WARPS, int ITEMS>
cudaError_t launch_route(const RouteArgs& a, cudaStream_t st)
{
    constexpr uint32_t kImages = images_per_block<WARPS>();
    const size_t smem = a.groups > 1 ? kImages * (a.N + 2 * a.groups) * sizeof(float) : 0;       // at most 36 KB
    return launch_following(route_kernel<T, WARPS, ITEMS>, (unsigned)((a.n + kImages - 1) / kImages), kImages * WARPS * 32, smem, st, a);
}

// ---- gradient ------------------------------------------------------------------------------------------------------------

// Every neuron has a gradient (dense scores, or routes that are not renormalised); a block per image.  With g the gradient of a weight
// and G that of a score (G = dscores, plus scale * g at the routes where they are not renormalised):
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
    float most = kNone, inv = 0.0f, mean = 0.0f;
    if (a.softmax) {
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
            const float G = (ds ? to_float(ds[j]) : 0.0f) + (a.renormalise ? 0.0f : grad[j]);
            d = a.softmax ? expf(l - most) * inv * (G - mean) : G * sigmoid_of(l) * sigmoid_of(-l);
            if (a.renormalise) d += grad[j];
        }
        out[j] = from_float<T>(l == kNone ? 0.0f : a.slope * d);
    }
}

// The same with the row in registers.  Routes are few: their part of the sums is added by one warp, and their elements are written
// again after the others.  Measured, 16,384 images of 2,791 neurons with dense gradients: 121 us = 4.5 TB/s of the 6.45 a copy reaches.
template <typename T, int WARPS, int ITEMS>
__global__ void __launch_bounds__(WARPS * 32 < kRegThreads ? kRegThreads : WARPS * 32) route_grad_kernel(const RouteGradArgs a)
{
    constexpr uint32_t kThreads = WARPS * 32, kImages = images_per_block<WARPS>();
    __shared__ float fscratch_s[kImages][WARPS];
    __shared__ float2 pair_s[kImages][WARPS];
    const uint32_t image = kImages > 1 ? threadIdx.x / kThreads : 0, t = kImages > 1 ? threadIdx.x % kThreads : threadIdx.x;
    const uint64_t row = (uint64_t)blockIdx.x * kImages + image;
    follow();
    if (kImages > 1 && row >= a.n) return;               // (all threads of the image, which wait for no other's)
    const T* x = static_cast<const T*>(a.values) + row * a.ld;
    const T* ds = a.dscores ? static_cast<const T*>(a.dscores) + row * a.ld_dscores : nullptr;
    T* out = static_cast<T*>(a.dvalues) + row * a.ld_dvalues;

    float l[ITEMS], G[ITEMS];
    float most = kNone, inv = 0.0f, mean = 0.0f;
    each_item<ITEMS, kThreads, true>(a.N, t, [&](int i, uint32_t j, bool in) { l[i] = in ? to_float(x[j]) : NAN; });
    if (ds) each_item<ITEMS, kThreads, true>(a.N, t, [&](int i, uint32_t j, bool in) { G[i] = in ? to_float(ds[j]) : 0.0f; });
    else each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) { G[i] = 0.0f; });
    if (a.mask) each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t j, bool in) { if (in && !a.mask[j]) l[i] = NAN; });
    each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) {
        l[i] = held(__fmul_rn(a.slope, l[i]));
        if (l[i] == kNone) G[i] = 0.0f;              // (what stands there is not looked at)
        most = fmaxf(most, l[i]);
    });
    // the routes: a lane each; of equal neurons the first lane stands for all
    uint32_t j = kNoNeuron;
    bool first = false;
    float lr = kNone, d = 0.0f, Gr = 0.0f;
    if (t < 32) {
        j = t < a.k ? a.neurons[row * a.k + t] : kNoNeuron;
        const bool there = j < a.N;
        if (!there) j = kNoNeuron;
        const float g = there ? a.dweights[row * a.k + t] : 0.0f, w = there ? a.weights[row * a.k + t] : 0.0f;
        if (there && !(a.mask && !a.mask[j])) lr = held(__fmul_rn(a.slope, to_float(x[j])));
        d = a.scale * g;
        if (a.renormalise) {
            const float m = warp_sum(g * w) / a.scale;
            d = w * (g - m);
            if (!a.softmax && there) d *= sigmoid_of(-lr);
        }
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, j);
        first = there && __ffs(same) - 1 == (int)t;
        float all = 0.0f;
        for (uint32_t r = 0; r < a.k; ++r) {
            const float dr = __shfl_sync(0xFFFFFFFFu, d, r);
            if (same >> r & 1u) all += dr;
        }
        d = all;
        if (ds && first && lr != kNone) Gr = to_float(ds[j]);
    }
    if (a.softmax) {
        most = row_reduce<WARPS>(most, fscratch_s[image], t, Max());
        const float m = most == kNone ? 0.0f : most;
        float sums[2] = { 0.0f, 0.0f }, dots[2] = { 0.0f, 0.0f };
        each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t, bool) {
            l[i] = exp_of(l[i] - m);                     // (kNone: zero)
            sums[i & 1] += l[i];
            dots[i & 1] = fmaf(l[i], G[i], dots[i & 1]);
        });
        if (!a.renormalise && first && lr != kNone) dots[0] = fmaf(exp_of(lr - m), d, dots[0]);
        const float2 both = row_sums<WARPS>(make_float2(sums[0] + sums[1], dots[0] + dots[1]), pair_s[image], t);
        const float sum = both.x, dot = both.y;
        inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        mean = dot * inv;
        const float by = a.slope * inv;
        each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t e, bool in) { if (in) out[e] = from_float<T>(by * l[i] * (G[i] - mean)); });
    } else {
        each_item<ITEMS, kThreads>(a.N, t, [&](int i, uint32_t e, bool in) {
            if (in) out[e] = from_float<T>(l[i] == kNone ? 0.0f : a.slope * G[i] * sigmoid_of(l[i]) * sigmoid_of(-l[i]));
        });
    }
    row_sync<WARPS>();
    if (first) {
        float v = 0.0f;
        if (lr != kNone) {
            if (!a.renormalise) Gr += d;
            v = a.softmax ? exp_of(lr - most) * inv * (Gr - mean) : Gr * sigmoid_of(lr) * sigmoid_of(-lr);
            if (a.renormalise) v += d;
        }
        out[j] = from_float<T>(a.slope * v);
    }
}

// Renormalised routes without dense gradients: zeros but for the routes, whose own logits are all that is read.  The zeros go out
// as whole 16-byte words while the routes arrive.  (65,536 images of 2,791 neurons: 236 us by the kernel above, whose registers
// leave room for five images an SM.)
template <typename T, int WARPS>
__global__ void __launch_bounds__(kRegThreads) route_grad_sparse_kernel(const RouteGradArgs a)
{
    constexpr uint32_t kThreads = WARPS * 32, kImages = images_per_block<WARPS>(), kWord = 16 / sizeof(T);
    const uint32_t image = kImages > 1 ? threadIdx.x / kThreads : 0, t = kImages > 1 ? threadIdx.x % kThreads : threadIdx.x;
    const uint64_t row = (uint64_t)blockIdx.x * kImages + image;
    follow();
    if (kImages > 1 && row >= a.n) return;               // (all threads of the image, which wait for no other's)
    T* out = static_cast<T*>(a.dvalues) + row * a.ld_dvalues;
    uint32_t j = kNoNeuron;
    float g = 0.0f, w = 0.0f;
    if (t < a.k) {
        j = a.neurons[row * a.k + t];
        g = a.dweights[row * a.k + t];
        w = a.weights[row * a.k + t];
    }
    const uint32_t head = min(a.N, ((16u - ((uint32_t)reinterpret_cast<uintptr_t>(out) & 15u)) & 15u) / (uint32_t)sizeof(T));
    const uint32_t words = (a.N - head) / kWord, tail = head + words * kWord;
    if (t < head) out[t] = from_float<T>(0.0f);
    for (uint32_t i = t; i < words; i += kThreads) reinterpret_cast<uint4*>(out + head)[i] = make_uint4(0, 0, 0, 0);
    if (tail + t < a.N) out[tail + t] = from_float<T>(0.0f);
    float d = 0.0f;
    bool first = false;
    if (t < 32) {
        const bool there = j < a.N;
        if (!there) { j = kNoNeuron; g = w = 0.0f; }
        float lr = kNone;
        if (there && !(a.mask && !a.mask[j])) lr = held(__fmul_rn(a.slope, to_float(static_cast<const T*>(a.values)[row * a.ld + j])));
        const float m = warp_sum(g * w) / a.scale;
        float mine = w * (g - m);
        if (!a.softmax && there) mine *= sigmoid_of(-lr);
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, j);
        first = there && __ffs(same) - 1 == (int)t;      // of equal neurons the first lane stands for all
        for (uint32_t r = 0; r < a.k; ++r) {
            const float dr = __shfl_sync(0xFFFFFFFFu, mine, r);
            if (same >> r & 1u) d += dr;
        }
        if (lr == kNone) d = 0.0f;
    }
    row_sync<WARPS>();
    if (first) out[j] = from_float<T>(a.slope * d);
}

template <typename T, int WARPS, int ITEMS>
cudaError_t launch_route_grad(const RouteGradArgs& a, cudaStream_t st)
{
    constexpr uint32_t kImages = images_per_block<WARPS>();
    return launch_following(route_grad_kernel<T, WARPS, ITEMS>, (unsigned)((a.n + kImages - 1) / kImages), kImages * WARPS * 32, 0, st, a);
}

} // namespace

template <typename T>
cudaError_t run_route(const RouteArgs& a, cudaStream_t st)
{
    // Four warps an image (65,536 images, eight routes and a bias: 161 us at 1,600 neurons where two warps take 197; 211 at 2,791,
    // where two take 266 and eight 348); one where a warp holds the row; more for few images, which then have less to do each.
    if (a.N <= 512) return launch_route<T, 1, 16>(a, st);
    if (a.N <= 4096 && a.n <= 256) return launch_route<T, 8, 16>(a, st);
    if (a.N <= 2048) return launch_route<T, 4, 16>(a, st);
    if (a.N <= 4096) return launch_route<T, 4, 32>(a, st);
    if (a.N <= 8192) return launch_route<T, 16, 16>(a, st);
    const size_t smem = (a.N + (a.groups > 1 ? a.groups : 0)) * sizeof(float);
    auto* kernel = route_row_kernel<T>;
    const cudaError_t e = allow_shared(kernel, smem, (PINK_B200_MAX_ROUTED_NEURONS + PINK_B200_MAX_ROUTE_GROUPS) * sizeof(float));
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)a.n, kRowThreads, smem, st>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t run_route_grad(const RouteGradArgs& a, cudaStream_t st)
{
    if (a.renormalise && !a.dscores) {
        if (a.N <= 512) return launch_following(route_grad_sparse_kernel<T, 1>, (unsigned)((a.n + images_per_block<1>() - 1) / images_per_block<1>()), kRegThreads, 0, st, a);
        return launch_following(route_grad_sparse_kernel<T, 4>, (unsigned)a.n, kRegThreads, 0, st, a);
    }
    // two values a place are held here (logit and gradient), so rows are spread over more warps than in the forward pass
    if (a.N <= 512) return launch_route_grad<T, 1, 16>(a, st);
    if (a.N <= 2048) return launch_route_grad<T, 4, 16>(a, st);
    if (a.N <= 4096) return launch_route_grad<T, 4, 32>(a, st);
    if (a.N <= 8192) return launch_route_grad<T, 8, 32>(a, st);
    const size_t smem = a.N * sizeof(float);
    auto* kernel = route_grad_row_kernel<T>;
    const cudaError_t e = allow_shared(kernel, smem, PINK_B200_MAX_ROUTED_NEURONS * sizeof(float));
    if (e != cudaSuccess) return e;
    kernel<<<(unsigned)a.n, kRowThreads, smem, st>>>(a);
    return cudaGetLastError();
}

#if PINK_ROUTE_TYPE == 0
using RouteType = float;
#elif PINK_ROUTE_TYPE == 1
using RouteType = __nv_bfloat16;
#else
using RouteType = __half;
#endif
template cudaError_t run_route<RouteType>(const RouteArgs&, cudaStream_t);
template cudaError_t run_route_grad<RouteType>(const RouteGradArgs&, cudaStream_t);

} // namespace pinkb

#else // PINK_ROUTE_TYPE

namespace {

// ---- balance -------------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(1024) balance_kernel(uint32_t N, const uint32_t* load, const uint8_t* mask, float rate,
                                                       const float* bias, float* out)
{
    __shared__ unsigned long long total_s, members_s;
    follow();
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

__global__ void __launch_bounds__(256) route_rotations_kernel(const uint32_t* rot, uint32_t N, const uint32_t* neurons, uint64_t routes, uint32_t k,
                                                              uint32_t* out)
{
    for (uint64_t r = (uint64_t)blockIdx.x * 256 + threadIdx.x; r < routes; r += (uint64_t)gridDim.x * 256) {
        const uint32_t e = neurons[r];
        out[r] = e < N ? rot[r / k * N + e] : kNoNeuron;
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

cudaError_t launch_route_rotations(const uint32_t* rot, uint32_t n_neurons, const uint32_t* neurons, uint32_t n_img, uint32_t k, uint32_t* out,
                                   cudaStream_t st)
{
    const uint64_t routes = (uint64_t)n_img * k;
    route_rotations_kernel<<<(unsigned)((routes + 255) / 256), 256, 0, st>>>(rot, n_neurons, neurons, routes, k, out);
    return cudaGetLastError();
}

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
                scores_type, dev_scores, ld_scores};
    return launch_status(with_type(type, [&](auto v) { return run_route<decltype(v)>(a, static_cast<cudaStream_t>(stream)); }), "route kernel");
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
    return launch_status(with_type(type, [&](auto v) { return run_route_grad<decltype(v)>(a, static_cast<cudaStream_t>(stream)); }), "route gradient kernel");
}

int pink_b200_op_route_balance(uint32_t n_neurons, const uint32_t* dev_load, const uint8_t* dev_mask, float rate, const float* dev_bias,
                               float* dev_new_bias, void* stream)
{
    if (n_neurons == 0 || n_neurons > PINK_B200_MAX_ROUTED_NEURONS)
        return report_error(PINK_B200_EINVAL, "a route chooses from 1 to 32768 neurons");
    if (!(rate == rate) || rate - rate != 0.0f) return report_error(PINK_B200_EINVAL, "rate must be finite");
    if (!dev_load || !dev_bias || !dev_new_bias) return report_error(PINK_B200_EINVAL, "null argument");
    return launch_status(launch_following(balance_kernel, 1, n_neurons < 1024 ? 256 : 1024, 0, static_cast<cudaStream_t>(stream), n_neurons, dev_load,
                                          dev_mask, rate, dev_bias, dev_new_bias), "balance kernel");
}

} // extern "C"

#endif // PINK_ROUTE_TYPE
