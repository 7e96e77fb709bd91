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
//
// The kernels of an element type are a module of their own (PINK_DISTILL_TYPE = 0, 1, 2: float32, bfloat16, float16), so that a process
// loads what it uses; without the macro this file holds the entry points.
#include "ring.cuh"

namespace pinkb {

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
    uint32_t per_thread;             // 2^32 over a block's threads, rounded up
    uint32_t whole_mask, whole_d;    // the mask may be read, and dscores written, a chunk at a time
};

// align: of the rows of scores (kAny, kEight, kSixteen).
template <typename T> cudaError_t run_distill(const DistillArgs& a, int align, bool grad, cudaStream_t st);

#ifdef PINK_DISTILL_TYPE

namespace {

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

// A row's targets, as one warp finds them for all.  What the loss needs of them: their share of it relative to their own maximum, where
//   sum of p log(p / q) = share + mass ((all_most - most) / T + log all_sum),  share = sum of p (log p - (score - most) / T)
struct Targets
{
    float most, sum;                 // maximum and sum of their exponentials
    float share, mass, rest;         // mass: the sum of p; rest: 1 minus it (0 without a.rest)
    uint32_t present;
};

struct Row
{
    float p[32];                     // weight of a target; 0 where it is absent
    float value[32];                 // its score
    uint32_t neuron[32];             // kNoNeuron where it is absent
    Targets all;
    float warp_most[16], warp_sum[16];
};

// The targets of a row, a lane each.  `value` is the score of the lane's neuron, -infinity where it takes no part or the lane has none.
__device__ __forceinline__ Targets gather_targets(const DistillArgs& a, uint32_t lane, uint32_t neuron, float target, float value, Row* s)
{
    Targets o;
    const bool there = value != -INFINITY;               // (also for a NaN, which shows in the loss)
    const uint32_t same = __match_any_sync(0xFFFFFFFFu, there ? neuron : 0x80000000u + lane);
    const bool first = there && __ffs(same) - 1 == (int)lane;      // a neuron listed twice is one neuron
    o.present = __ballot_sync(0xFFFFFFFFu, there);
    o.most = redux_max(first ? value : -INFINITY);
    o.sum = warp_sum(first ? relative(value, o.most, a.exp2_t) : 0.0f);
    float p = target;
    o.mass = 1.0f;
    o.rest = 0.0f;
    if (a.logits) {
        const float t = there ? fminf(target, FLT_MAX) : -INFINITY, high = redux_max(t);
        p = there ? expf((t - high) * a.inv_t) : 0.0f;
        const float all = warp_sum(p);
        p = there ? p / all : 0.0f;
    } else if (a.rest) {
        double m = there ? (double)p : 0.0;              // (the rest is a difference)
#pragma unroll
        for (int o = 16; o; o >>= 1) m += __shfl_xor_sync(0xFFFFFFFFu, m, o);
        o.mass = (float)m;
        o.rest = fmaxf((float)(1.0 - m), 0.0f);
    } else {
        o.mass = warp_sum(there ? p : 0.0f);
    }
    o.share = 0.0f;
    s->p[lane] = there ? p : 0.0f;
    s->value[lane] = value;
    s->neuron[lane] = there ? neuron : kNoNeuron;
    if (lane == 0) s->all = o;
    return o;
}

// A chunk with -infinity in the places that `out` marks, a bit an element.
template <typename T>
__device__ __forceinline__ uint4 without(const uint4& c, uint32_t out)
{
    constexpr uint32_t kNone = std::is_same<T, __nv_bfloat16>::value ? 0xFF80u : std::is_same<T, __half>::value ? 0xFC00u : 0xFF800000u;
    uint32_t w[4] = { c.x, c.y, c.z, c.w };
    while (out) {                                        // (a loop that stays one: it hardly ever runs)
        const uint32_t v = __ffs(out) - 1, at = sizeof(T) == 4 ? v : v / 2;
        const uint32_t keep = sizeof(T) == 4 ? 0u : v % 2 ? 0xFFFFu : 0xFFFF0000u, put = sizeof(T) == 4 || v % 2 == 0 ? kNone : kNone << 16;
        out &= out - 1;
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q)
            if (q == at) w[q] = (w[q] & keep) | put;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The same in the places of neurons whose mask is zero; the bytes of a whole chunk.
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

// Which of a thread's elements are targets: a bit each in kWords words, and the element behind the chunks.  A warp's own targets set the bits in
// its part of shared memory, a word for every lane.
template <int WORDS>
struct Marks
{
    uint32_t bits[WORDS];
    bool behind;
    uint32_t any;                    // of the warp

    // neuron: the lane's target; slot, owner: place of its chunk among the threads' slots and threads; mine: it belongs to this warp
    template <uint32_t V>
    __device__ __forceinline__ void set(uint32_t (*words)[32], uint32_t lane, uint32_t neuron, uint32_t chunks, uint32_t slot, uint32_t owner, bool mine)
    {
        any = __ballot_sync(0xFFFFFFFFu, mine);
        behind = false;
#pragma unroll
        for (int q = 0; q < WORDS; ++q) bits[q] = 0;
        if (!any) return;
#pragma unroll
        for (int q = 0; q <= WORDS; ++q) words[q][lane] = 0;
        __syncwarp();
        if (mine) {
            const bool end = neuron >= chunks * V;
            const uint32_t bit = slot * V + neuron % V, q = end ? WORDS : bit / 32;
            atomicOr(&words[q][end ? neuron - chunks * V : owner & 31], 1u << (bit & 31));
        }
        __syncwarp();
#pragma unroll
        for (int q = 0; q < WORDS; ++q) bits[q] = words[q][lane];
        behind = words[WORDS][lane] != 0;
    }
};

// The targets' share of the loss, by the warp that has gathered them.
__device__ __forceinline__ float share_of(const DistillArgs& a, const Row* s, float most, uint32_t lane)
{
    const float p = s->p[lane];
    return warp_sum(p > 0.0f ? p * (logf(p) - (s->value[lane] - most) * a.inv_t) : 0.0f);
}

// What a row's warps come to together: the others' maximum and sum.
struct Others { float most, sum; };

__device__ __forceinline__ Others others_of(const DistillArgs& a, const Row* s, uint32_t lane, uint32_t warps)
{
    if (warps > 4) {
        const float m = lane < warps ? s->warp_most[lane] : -INFINITY, most = redux_max(m);
        return { most, warp_sum(lane < warps ? s->warp_sum[lane] * relative(m, most, a.exp2_t) : 0.0f) };
    }
    float most = s->warp_most[0], sum = 0.0f;
    for (uint32_t w = 1; w < warps; ++w) most = fmaxf(most, s->warp_most[w]);
    for (uint32_t w = 0; w < warps; ++w) sum = fmaf(s->warp_sum[w], relative(s->warp_most[w], most, a.exp2_t), sum);
    return { most, sum };
}

// And with the targets: maximum and sum of all.
struct Whole { float most, sum, r; };

__device__ __forceinline__ Whole whole_of(const DistillArgs& a, const Targets& t, const Others& o)
{
    Whole w;
    w.most = fmaxf(o.most, t.most);
    w.sum = t.sum * relative(t.most, w.most, a.exp2_t) + o.sum * relative(o.most, w.most, a.exp2_t);
    w.r = o.most != -INFINITY ? t.rest : 0.0f;
    return w;
}

__device__ __forceinline__ float loss_of(const DistillArgs& a, const Targets& t, const Others& o)
{
    if (!t.present) return 0.0f;
    const Whole w = whole_of(a, t, o);
    float loss = fmaf(t.mass, fmaf(w.most - t.most, a.inv_t, logf(w.sum)), t.share);
    if (w.r > 0.0f) {
        // r / q_rest is near 1 where the targets have little: 1 / q_rest = 1 + x, x what they have over the others' sum
        const float x = t.sum / o.sum * expf((t.most - o.most) * a.inv_t), z = fmaf(w.r, x, -t.mass);
        if (x > FLT_MAX) loss += w.r * (logf(w.r) + (t.most - o.most) * a.inv_t + logf(t.sum / o.sum));
        else loss += w.r * (z > -0.5f ? log1pf(z) : logf(w.r) + log1pf(x));
    }
    return a.scale * loss;
}

// The gradient's factors: of q at a target, and of this warp's exponentials.
struct Factors { float by, of_q, all_most, mine; bool present, finite; };

__device__ __forceinline__ Factors factors_of(const DistillArgs& a, const Targets& t, const Others& o, float dloss, float most)
{
    const Whole w = whole_of(a, t, o);
    Factors f;
    f.present = t.present != 0;
    f.by = f.present ? dloss * a.scale * a.inv_t : 0.0f;
    f.of_q = f.by * (t.mass + w.r) / w.sum;
    f.all_most = w.most;
    const float of_rest = w.r > 0.0f ? f.by * w.r / o.sum : 0.0f;
    f.mine = f.of_q * relative(most, w.most, a.exp2_t) - of_rest * relative(most, o.most, a.exp2_t);
    f.finite = f.present && fabsf(f.mine) <= FLT_MAX;
    return f;
}

// The gradient of this thread's elements where the row's factor is not finite.  A NaN or a +infinity among the scores that take part makes NaN of all of them,
// whatever is left of their exponentials; what takes no part, and beside an infinite factor what has underflowed, stays zero.  From memory again, an element
// at a time.  (A call, so that other rows hold no registers for it: inline in the loop over the chunks it took 32 of them, 102 us for 75 at 16,384 x 2,791 float32.)
template <typename T>
__device__ __noinline__ void unusual_gradient(const DistillArgs a, float factor, float most, uint64_t row, uint32_t t, uint32_t threads, uint32_t e1)
{
    constexpr uint32_t V = kChunk<T>;
    const T* x = static_cast<const T*>(a.scores) + row * a.ld;
    T* d = static_cast<T*>(a.dscores) + row * a.ld_d;
    auto element = [&](uint32_t e) {
        const float v = a.mask && !a.mask[e] ? -INFINITY : to_float(x[e]), q = relative(v, most, a.exp2_t);
        d[e] = from_float<T>(v == -INFINITY || (q == 0.0f && factor == factor) ? 0.0f : q * factor);
    };
    const uint32_t chunks = a.N / V;
#pragma unroll 1
    for (uint32_t c = t; c < chunks; c += threads)
#pragma unroll 1
        for (uint32_t v = 0; v < V; ++v) element(c * V + v);
    if (e1 < a.N && t < V) element(e1);
}

// A warp's elements: the chunks' sums and gradients are the same whichever way a row has come.
template <typename T, int CH>
struct Elements
{
    static constexpr int P = kPairs<T>;
    uint4 w[CH];
    float f1, most;                  // the element behind the chunks; the warp's maximum
    F2 below, by_t;

    template <typename On>
    __device__ __forceinline__ float sum(const DistillArgs& a, On on)
    {
        uint32_t top[4];
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (on(i)) {
                const uint32_t v[4] = { w[i].x, w[i].y, w[i].z, w[i].w };
#pragma unroll
                for (int j = 0; j < 4; ++j) top[j] = i == 0 ? v[j] : larger<T>(top[j], v[j]);
            }
        most = f1;
        if (CH > 1 || on(0)) {
            if constexpr (sizeof(T) == 2) {
                const F2 m = pair_of<T>(make_uint4(larger<T>(larger<T>(top[0], top[1]), larger<T>(top[2], top[3])), 0, 0, 0), 0);
                most = fmaxf(most, fmaxf(m.lo(), m.hi()));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) most = fmaxf(most, __uint_as_float(top[j]));
            }
        }
        if (!(most == most)) most = -INFINITY;           // (a NaN shows in the sums)
        most = redux_max(most);
        below = two(most == -INFINITY ? 0.0f : -most);
        by_t = two(a.exp2_t);
        F2 s = two(relative(f1, most, a.exp2_t), 0.0f);
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (on(i)) {
#pragma unroll
                for (int j = 0; j < P; ++j) s = add2(s, exponentials(w[i], j));
            }
        return warp_sum(s.lo() + s.hi());
    }

    __device__ __forceinline__ F2 exponentials(const uint4& c, int j) const
    {
        const float2 e = mul2(add2(pair_of<T>(c, j), below), by_t).both();
        return two(exp2_fast(e.x), exp2_fast(e.y));
    }

    // dscores of a row, of which this thread has the chunks t, t + threads, ... and element e1 behind them (beyond N: none).
    template <typename On, typename M>
    __device__ __forceinline__ void gradient(const DistillArgs& a, const Row* s, const Factors& f, const M& marks, uint64_t row, T* d, uint32_t t, uint32_t threads, uint32_t e1,
                                             On on) const
    {
        constexpr uint32_t V = kChunk<T>;
        if (__builtin_expect(f.finite, 1)) {
            const F2 f2 = two(f.mine);
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (on(i)) {
                    F2 v[P];
#pragma unroll
                    for (int j = 0; j < P; ++j) v[j] = mul2(exponentials(w[i], j), f2);
                    store_pairs<T>(d + (t + i * threads) * V, v, V, a.whole_d);
                }
            if (e1 < a.N && t < V) d[e1] = from_float<T>(relative(f1, most, a.exp2_t) * f.mine);
        } else if (f.present) {
            unusual_gradient<T>(a, f.mine, most, row, t, threads, e1);
        } else {                                         // a row without targets, whatever its scores
            F2 none[P];
#pragma unroll
            for (int j = 0; j < P; ++j) none[j] = two(0.0f);
#pragma unroll 1
            for (int i = 0; i < CH; ++i)
                if (on(i)) store_pairs<T>(d + (t + i * threads) * V, none, V, a.whole_d);
            if (e1 < a.N && t < V) d[e1] = from_float<T>(0.0f);
        }
        // the targets, one by one, behind their chunks
        if (!marks.any) return;
        auto target_gradient = [&](uint32_t e) {
            float p = 0.0f, value = -INFINITY;
            for (uint32_t j = 0; j < a.k; ++j)
                if (s->neuron[j] == e) { p += s->p[j]; value = s->value[j]; }
            // (a target whose neuron takes no part has no gradient)
            d[e] = from_float<T>(value != -INFINITY ? fmaf(f.of_q, relative(value, f.all_most, a.exp2_t), -f.by * p) : 0.0f);
        };
#pragma unroll
        for (int q = 0; q < (int)((CH * V + 31) / 32); ++q)
            for (uint32_t bits = marks.bits[q]; bits; bits &= bits - 1) {
                const uint32_t b = q * 32 + __ffs(bits) - 1;
                target_gradient((t + b / V * threads) * V + b % V);
            }
        if (marks.behind) target_gradient(e1);
    }
};

// Leaves out of a chunk what the mask and the targets take from it.
template <typename T>
__device__ __forceinline__ uint4 left_in(const DistillArgs& a, uint4 c, uint32_t col, uint32_t marked)
{
    if (a.mask) {
        if (a.whole_mask) {
            c = masked<T>(c, a.mask + col);
        } else {
#pragma unroll
            for (uint32_t v = 0; v < kChunk<T>; ++v) marked |= (uint32_t)(!a.mask[col + v]) << v;
        }
    }
    return without<T>(c, marked);
}

// The lane's target of a row, kNoNeuron where it does not count: its neuron exists and its weight is positive (its logit above -infinity).
__device__ __forceinline__ uint32_t counted(const DistillArgs& a, uint32_t neuron, float target)
{
    return neuron < a.N && (a.logits ? target > -INFINITY : target > 0.0f) ? neuron : kNoNeuron;
}

constexpr uint32_t kDistillWarps = 4;                    // rows of a block, where a row is a warp's

// Few rows: a row in the registers of a warp, or (BLOCK) of a block, CH chunks a thread.  Whole chunks are dealt to the threads in turn, and the fewer than V
// elements behind the last go one to a lane of the first warp.  ALL: any slot but the first may be empty; otherwise (CH - 1) threads <= chunks, so
// that only a thread's last slot has to look for the row's end.
template <typename T, bool BLOCK, int CH, bool ALL, int ALIGN, bool GRAD>
__global__ void __launch_bounds__(BLOCK ? 512 : 32 * kDistillWarps) distill_kernel(const __grid_constant__ DistillArgs a)
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int kWords = (CH * V + 31) / 32;
    using In = RowOf<T, ALIGN>;
    __shared__ Row rows_s[BLOCK ? 1 : kDistillWarps];
    __shared__ uint32_t words[BLOCK ? 16 : kDistillWarps][kWords + 1][32];
    const uint32_t lane = threadIdx.x & 31, warp = BLOCK ? threadIdx.x >> 5 : 0, warps = BLOCK ? blockDim.x >> 5 : 1;
    const uint32_t threads = warps * 32, t = warp * 32 + lane, N = a.N, chunks = N / V;
    Row* s = &rows_s[BLOCK ? 0 : threadIdx.x >> 5];
    const uint64_t row = BLOCK ? blockIdx.x : (uint64_t)blockIdx.x * kDistillWarps + (threadIdx.x >> 5);
    follow();
    if (!BLOCK && row >= a.n) return;
    const In in(a.scores, a.ld, row, a.n, chunks * V);   // (its whole chunks)
    const T* x = static_cast<const T*>(a.scores) + row * a.ld;
    const bool last = t + (CH - 1) * threads < chunks;   // this thread's last slot has a chunk
    auto on = [&](int i) { return ALL ? t + i * threads < chunks : i + 1 < CH || last; };
    typename In::Chunk on_way[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (on(i)) on_way[i] = in.load((t + i * threads) * V);
    const uint32_t e1 = chunks * V + t;                  // the element behind the chunks that is this thread's
    Elements<T, CH> own;
    own.f1 = e1 < N && t < V && !(a.mask && !a.mask[e1]) ? to_float(x[e1]) : -INFINITY;

    uint32_t neuron = kNoNeuron;
    float target = 0.0f;
    if (lane < a.k) {
        neuron = a.neurons[row * a.k + lane];
        target = a.targets[row * a.k + lane];
    }
    neuron = counted(a, neuron, target);
    if (warp == 0) gather_targets(a, lane, neuron, target, neuron != kNoNeuron && !(a.mask && !a.mask[neuron]) ? to_float(x[neuron]) : -INFINITY, s);
    const uint32_t chunk = neuron / V, slot = chunk / threads, owner = chunk % threads;
    Marks<kWords> marks;
    marks.template set<V>(words[threadIdx.x >> 5], lane, neuron, chunks, slot, owner, neuron != kNoNeuron && (chunk >= chunks ? 0 : owner >> 5) == warp);
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (on(i)) own.w[i] = left_in<T>(a, in.all(on_way[i]), (t + i * threads) * V, marks.bits[i * V / 32] >> (i * V % 32) & ((1u << V) - 1));
    if (marks.behind) own.f1 = -INFINITY;
    const float sum = own.sum(a, on);
    if constexpr (BLOCK) {
        if (lane == 0) { s->warp_most[warp] = own.most; s->warp_sum[warp] = sum; }
        __syncthreads();
    } else {
        __syncwarp();
    }
    const Others o = BLOCK ? others_of(a, s, lane, warps) : Others{ own.most, sum };
    if (a.loss && warp == 0) {
        Targets targets = s->all;
        targets.share = share_of(a, s, targets.most, lane);
        const float loss = loss_of(a, targets, o);
        if (lane == 0) a.loss[row] = loss;
    }
    if constexpr (GRAD)
        own.gradient(a, s, factors_of(a, s->all, o, a.dloss ? a.dloss[row] : 1.0f, own.most), marks, row, static_cast<T*>(a.dscores) + row * a.ld_d, t, threads, e1, on);
}

// Many rows: a block takes a row at a time, which arrives through the ring in shared memory.  Its last warp has no elements but the row's list, which it
// gathers while the others sum the row, and the losses, which it forms for 32 rows at once, a lane each: neither is on the others' way.
constexpr uint32_t kDistillRing = 2;                     // stages: a row is in registers when its sums meet, and its stage free for the next but one

template <typename T, int CH, int ALIGN, bool GRAD>
__global__ void __launch_bounds__(544) distill_ring_kernel(const DistillArgs a)
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int kWords = (CH * V + 31) / 32;
    extern __shared__ __align__(16) uint8_t ring[];      // [kDistillRing] rows, then [warps][kWords + 1][32] of Marks
    __shared__ Row rows_s[2];
    const uint32_t t = threadIdx.x, threads = blockDim.x - 32, lane = t & 31, warp = t >> 5, warps = threads >> 5, N = a.N, chunks = N / V, n = (uint32_t)a.n, step = gridDim.x;
    const uint32_t stage = staged_bytes(N, sizeof(T)), e1 = chunks * V + t;
    uint32_t r = blockIdx.x;
    follow();
    Staged<T, CH> x(a.scores, a.ld, r, step, N, smem_u32(ring), threads);
    uint32_t neuron = kNoNeuron;
    float target = 0.0f, dloss = 1.0f;
    auto list = [&](uint32_t row) {                      // (read a row ahead)
        if (row < n && lane < a.k) {
            neuron = a.neurons[(uint64_t)row * a.k + lane];
            target = a.targets[(uint64_t)row * a.k + lane];
        }
        if constexpr (GRAD) if (row < n && a.dloss) dloss = a.dloss[row];
    };
    list(r);
    uint32_t slot = 0, turn = 0;
    if (warp == warps) {
        Targets mine{};
        Others others{};
        uint32_t held = 0, first = r;                    // rows whose losses are due, the first of them
        auto write = [&] {
            if (a.loss && lane < held) a.loss[first + (uint64_t)lane * step] = loss_of(a, mine, others);
        };
        __syncthreads();
        for (; r < n; r += step, slot = slot + 1 == kDistillRing ? 0 : slot + 1, ++turn) {
            Row* s = &rows_s[turn & 1];
            const uint32_t e = counted(a, neuron, target);
            const bool there = e != kNoNeuron && !(a.mask && !a.mask[e]);
            Targets o = gather_targets(a, lane, e, target, there ? staged_element<T>(x.place(slot * stage) + e * (uint32_t)sizeof(T)) : -INFINITY, s);
            list(r + step);
            __syncthreads();
            if (a.loss) {
                const Others all = others_of(a, s, lane, warps);
                o.share = share_of(a, s, o.most, lane);
                if (lane == held) { mine = o; others = all; }
                if (++held == 32) {
                    write();
                    held = 0;
                    first = r + step;
                }
            }
            x.advance();
        }
        write();
        return;
    }
    const bool last = t + (CH - 1) * threads < chunks, wide = a.ld * sizeof(T) >= 16;
    auto on = [&](int i) { return i + 1 < CH || last; };
    const bool one = e1 < N && t < V && !(a.mask && !a.mask[e1]);
    uint32_t ahead = r;
    auto copy = [&](uint32_t slot) {
        if (ahead < n) x.copy(slot * stage, wide && ahead > 0, wide && ahead + 1 < n);
        ahead += step;
        copies_committed();
    };
    for (uint32_t i = 0; i < kDistillRing; ++i) copy(i);
    copies_waited<kDistillRing - 1>();
    __syncthreads();
    T* d = GRAD ? static_cast<T*>(a.dscores) + r * a.ld_d : nullptr;
    const uint64_t d_pace = step * a.ld_d;
    for (; r < n; r += step, slot = slot + 1 == kDistillRing ? 0 : slot + 1, ++turn, d += d_pace) {
        const uint32_t here = x.place(slot * stage);
        Row* s = &rows_s[turn & 1];
        Elements<T, CH> own;
        const uint32_t e = counted(a, neuron, target);
        const float by = dloss;
        list(r + step);
        const uint32_t chunk = e / V, place = __umulhi(chunk, a.per_thread), owner = chunk - place * threads;
        Marks<kWords> marks;
        marks.template set<V>(reinterpret_cast<uint32_t(*)[32]>(ring + kDistillRing * stage) + warp * (kWords + 1), lane, e, chunks, place, owner, e != kNoNeuron && (chunk >= chunks ? 0 : owner >> 5) == warp);
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (on(i)) own.w[i] = left_in<T>(a, staged_chunk<T, ALIGN>(here + (t + i * threads) * 16), (t + i * threads) * V, marks.bits[i * V / 32] >> (i * V % 32) & ((1u << V) - 1));
        own.f1 = one && !marks.behind ? staged_element<T>(here + e1 * (uint32_t)sizeof(T)) : -INFINITY;
        const float sum = own.sum(a, on);
        if (lane == 0) { s->warp_most[warp] = own.most; s->warp_sum[warp] = sum; }
        copies_waited<kDistillRing - 2>();               // this thread's part of the next row is there
        __syncthreads();
        copy(slot);
        if constexpr (GRAD) own.gradient(a, s, factors_of(a, s->all, others_of(a, s, lane, warps), by, own.most), marks, r, d, t, threads, e1, on);
        x.advance();
    }
}

template <typename T, int ALIGN, bool GRAD>
cudaError_t run_distill_at(DistillArgs a, cudaStream_t st)
{
    const uint32_t chunks = a.N / kChunk<T>, smem = kDistillRing * staged_bytes(a.N, sizeof(T));
    uint32_t threads = 0;
    auto takes = [&](uint32_t per) { return (threads = ring_threads(chunks, per)) != 0; };
    const dim3 of_warps((unsigned)((a.n + kDistillWarps - 1) / kDistillWarps)), of_blocks((unsigned)a.n);
    auto warp_rows = [&](auto kernel) { return launch_following(kernel, of_warps, 32 * kDistillWarps, 0, st, a); };
    auto block_rows = [&](auto kernel) { return launch_following(kernel, of_blocks, threads, 0, st, a); };
    if (a.n >= 8 * (uint64_t)sm_count()) {
        // Many chunks a thread, so that fewer warps share what a row costs beside its elements (64 rows an SM with the gradient, bfloat16: 8,192 neurons 83 us with eight
        // chunks, 100 with two; 2,791 43 with six, 45 with two).  16-bit rows take the ring (65,536 x 2,791: 120 us; a block a row in registers 162; gradient, 2,791, at 4, 8, 16
        // and 64 rows an SM: 5.3, 8.5, 12.8, 43.4; in registers with two chunks 6.2, 9.2, 14.2, 51.7 -- rows of one warp may lose by it: 900 neurons at 64 rows an SM 22.6 for 21.4,
        // 400 neurons 16.2 for 12.3, and at 16 rows gain, 7.9 for 9.1 and 5.9 for 7.2), float32 rows registers: twice the bytes for an element's instructions
        // (16,384 x 2,791 with the gradient: 75 us; the ring 79; at 4, 8 and 16 rows an SM with eight chunks a thread 6.8, 7.7 and 13.9, with two 5.7, 9.8 and 18.8).
        if constexpr (sizeof(T) == 2) {
            auto ring = [&](auto kernel, uint32_t words) {
                a.per_thread = (uint32_t)((0x100000000ull + threads - 1) / threads);
                return launch_ring(kernel, a.n, threads + 32, smem + threads * 4 * (words + 1), st, a);
            };
            if (takes(8)) return ring(distill_ring_kernel<T, 8, ALIGN, GRAD>, 2);
            if (takes(6)) return ring(distill_ring_kernel<T, 6, ALIGN, GRAD>, 2);
            if (takes(4)) return ring(distill_ring_kernel<T, 4, ALIGN, GRAD>, 1);
            if (takes(2)) return ring(distill_ring_kernel<T, 2, ALIGN, GRAD>, 1);
            if (takes(1)) return ring(distill_ring_kernel<T, 1, ALIGN, GRAD>, 1);
        } else {
            if (takes(8)) return threads == 32 ? warp_rows(distill_kernel<T, false, 8, false, ALIGN, GRAD>) : block_rows(distill_kernel<T, true, 8, false, ALIGN, GRAD>);
            if (takes(4)) return threads == 32 ? warp_rows(distill_kernel<T, false, 4, false, ALIGN, GRAD>) : block_rows(distill_kernel<T, true, 4, false, ALIGN, GRAD>);
        }
    }
    if (takes(2)) return threads == 32 ? warp_rows(distill_kernel<T, false, 2, false, ALIGN, GRAD>) : block_rows(distill_kernel<T, true, 2, false, ALIGN, GRAD>);
    if (takes(1)) return threads == 32 ? warp_rows(distill_kernel<T, false, 1, false, ALIGN, GRAD>) : block_rows(distill_kernel<T, true, 1, false, ALIGN, GRAD>);
    threads = 512;                                       // 1,024 to 8,192 chunks
    if (chunks <= 4 * 512) return block_rows(distill_kernel<T, true, 4, true, ALIGN, GRAD>);
    if (chunks <= 8 * 512) return block_rows(distill_kernel<T, true, 8, true, ALIGN, GRAD>);
    if constexpr (sizeof(T) == 4) return block_rows(distill_kernel<T, true, 16, true, ALIGN, GRAD>);
    return cudaErrorInvalidValue;                        // (not reached: 4,096 chunks of 16-bit elements are 8 a thread)
}

} // namespace

template <typename T>
cudaError_t run_distill(const DistillArgs& a, int align, bool grad, cudaStream_t st)
{
    return with_alignment(align, [&](auto at) {
        constexpr int ALIGN = decltype(at)::value;
        return grad ? run_distill_at<T, ALIGN, true>(a, st) : run_distill_at<T, ALIGN, false>(a, st);
    });
}

#if PINK_DISTILL_TYPE == 0
using DistillType = float;
#elif PINK_DISTILL_TYPE == 1
using DistillType = __nv_bfloat16;
#else
using DistillType = __half;
#endif
template cudaError_t run_distill<DistillType>(const DistillArgs&, int, bool, cudaStream_t);

} // namespace pinkb

#else // PINK_DISTILL_TYPE

namespace {

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
                  targets, dloss, dscores, ld_d, loss, 0, 0, 0};
    return launch_status(with_type(type, [&](auto t) {
        using T = decltype(t);
        a.whole_mask = reinterpret_cast<uintptr_t>(mask) % kChunk<T> == 0;
        a.whole_d = RowAlign().add(dscores, ld_d, sizeof(T)).elements(sizeof(T), kChunk<T>) == kChunk<T>;
        return run_distill<T>(a, alignment_of(RowAlign().add(scores, ld, sizeof(T)), sizeof(T)), grad, st);
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

#endif // PINK_DISTILL_TYPE
