// Read-out of routed neurons and its gradient (pink_b200_op_read_out*).
//
//   out_i = sum_j w_ij V[e_ij] (+ residual_i),   dw_ij = <dout_i, V[e_ij]>,   dV[e] = sum over the routes to e of w_ij dout_i
//
// The forward pass and dw are gathers.  dV would be a scatter with floating-point atomics, whose order changes the result; here
// the routes are sorted by neuron first (a stable counting sort), and every neuron's routes are added up in a fixed order.
#include "readout.cuh"

#include <algorithm>

namespace pinkb {
namespace {

constexpr uint32_t kThreads = 256;

struct ReadOutArgs
{
    uint64_t n; uint32_t N, D, k;
    const void* values; uint64_t ld;
    const uint32_t* neurons; const float* weights;
    const void* residual; uint64_t ld_residual;
    void* out; uint64_t ld_out;
    uint32_t tx_shift;               // log2 of the threads along the columns of a row
};

// Threads along the columns of a row, PARTS vectors of VEC elements each.  With one vector a thread the kernel is bound by
// instructions (the route, its weight and the row's address for every vector); two share them (four hold too many registers for the
// loads in flight).  Measured, 2,000 rows of 8,192 bfloat16, eight routes each of 2,791: 34 us, 7.7 TB/s gathered, all but the first touch from
// L2; rows of 8,100, whose places allow loads of 8 bytes only: 45 us.
template <typename T, int VEC, int PARTS>
__global__ void __launch_bounds__(kThreads) read_out_kernel(const ReadOutArgs a)
{
    const uint32_t width = 1u << a.tx_shift;
    const uint32_t tx = threadIdx.x & (width - 1), ty = threadIdx.x >> a.tx_shift;
    const uint64_t row = (uint64_t)blockIdx.x * (kThreads >> a.tx_shift) + ty;
    const uint32_t col = (blockIdx.y * PARTS * width + tx) * VEC, step = width * VEC;
    if (row >= a.n || col >= a.D) return;
    const uint32_t* e = a.neurons + row * a.k;
    const float* w = a.weights + row * a.k;
    const T* values = static_cast<const T*>(a.values) + col;
    float acc[PARTS][VEC];
#pragma unroll
    for (int p = 0; p < PARTS; ++p)
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[p][v] = 0.0f;
    constexpr uint32_t kTogether = 2;                    // routes whose loads are in flight together
    for (uint32_t j0 = 0; j0 < a.k; j0 += kTogether) {
        uint32_t id[kTogether];
        float wj[kTogether];
        Pack<T, VEC> x[kTogether][PARTS];
#pragma unroll
        for (uint32_t q = 0; q < kTogether; ++q) {
            id[q] = j0 + q < a.k ? e[j0 + q] : kNoNeuron;
            wj[q] = j0 + q < a.k ? w[j0 + q] : 0.0f;
        }
#pragma unroll
        for (uint32_t q = 0; q < kTogether; ++q)
#pragma unroll
            for (int p = 0; p < PARTS; ++p)
                if (id[q] < a.N && (p == 0 || col + p * step < a.D))
                    x[q][p] = Pack<T, VEC>::load(values + id[q] * a.ld + p * step);
#pragma unroll
        for (uint32_t q = 0; q < kTogether; ++q)
            if (id[q] < a.N)
#pragma unroll
                for (int p = 0; p < PARTS; ++p) {
                    float f[VEC];
                    x[q][p].floats(f);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) acc[p][v] = fmaf(wj[q], f[v], acc[p][v]);
                }
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        if (p != 0 && col + p * step >= a.D) break;
        if (a.residual) {
            const Pack<T, VEC> r = Pack<T, VEC>::load(static_cast<const T*>(a.residual) + row * a.ld_residual + col + p * step);
            float f[VEC];
            r.floats(f);
#pragma unroll
            for (int v = 0; v < VEC; ++v) acc[p][v] += f[v];
        }
        Pack<T, VEC>::of(acc[p]).store(static_cast<T*>(a.out) + row * a.ld_out + col + p * step);
    }
}

// ---- gradient of the weights ----------------------------------------------------------------------------------------------

struct ReadOutGradArgs
{
    uint64_t n; uint32_t N, D, k;
    const void* values; uint64_t ld;
    const uint32_t* neurons; const float* weights;
    const void* dout; uint64_t ld_dout;
    void* dvalues; uint64_t ld_dvalues;
    float* dweights;
    // the sorted routes (see sort_plan)
    uint32_t routes, chunks, per_chunk;
    uint32_t segment;                // routes of a segment
    uint32_t tiles;                  // column tiles of a row (wider rows)
    uint32_t* counts;                // [chunks][N] routes of a chunk to a neuron, then where they start among the neuron's
    uint32_t* total;                 // [N] routes to a neuron
    uint32_t* first;                 // [N] where a neuron's routes start in `sorted`
    uint32_t* seg_first;             // [N] its first segment
    uint32_t* part_first;            // [N + 1] its first row of partial sums (neurons of several segments)
    uint32_t* n_segments;            // their number
    uint32_t most_segments;          // and room: N + routes / segment
    uint4* segments;                 // [N + routes / segment] {first place in `sorted`, routes, neuron, row of partial sums or kNoNeuron}
    uint2* sorted;                   // [routes] {route (image * k + position), weight} by neuron, in order
    float* dots;                     // wider rows: [blocks along the columns][routes] products of their columns; null without dweights
    float* parts;                    // partial sums of the segments of neurons that have several
    uint32_t part_ld;
    uint32_t tx_shift;
};

// G threads per image, k_now <= 8 routes at a time.
template <typename T, int VEC, int G>
__global__ void __launch_bounds__(kThreads) dweights_kernel(const ReadOutGradArgs a)
{
    constexpr uint32_t kRows = kThreads / G;
    __shared__ float part[G > 32 ? kThreads / 32 : 1][8];
    const uint32_t tx = threadIdx.x % G;
    const uint64_t row = (uint64_t)blockIdx.x * kRows + threadIdx.x / G;
    const bool live = row < a.n;                          // (no thread leaves: the reductions below are for whole warps)
    const T* dout = static_cast<const T*>(a.dout) + (live ? row : 0) * a.ld_dout;
    for (uint32_t j0 = 0; j0 < a.k; j0 += 8) {
        const T* v[8];
        float acc[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const uint32_t id = live && j0 + j < a.k ? a.neurons[row * a.k + j0 + j] : kNoNeuron;
            v[j] = id < a.N ? static_cast<const T*>(a.values) + id * a.ld : nullptr;
            acc[j] = 0.0f;
        }
        if (live)
            for (uint32_t col = tx * VEC; col < a.D; col += G * VEC) {
                const Pack<T, VEC> d = Pack<T, VEC>::load(dout + col);
                float g[VEC];
                d.floats(g);
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    if (!v[j]) continue;
                    float f[VEC];
                    Pack<T, VEC>::load(v[j] + col).floats(f);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[j] = fmaf(g[i], f[i], acc[j]);
                }
            }
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
#pragma unroll
            for (int o = (G < 32 ? G : 32) / 2; o; o >>= 1) acc[j] += __shfl_xor_sync(0xFFFFFFFFu, acc[j], o);
        if constexpr (G > 32) {
            __syncthreads();
            if ((threadIdx.x & 31) == 0)
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) part[threadIdx.x >> 5][j] = acc[j];
            __syncthreads();
            if (live && tx < 8 && j0 + tx < a.k) {
                float s = 0.0f;
#pragma unroll
                for (uint32_t w = 0; w < G / 32; ++w) s += part[w][tx];
                a.dweights[row * a.k + j0 + tx] = s;
            }
        } else if (live && tx == 0) {
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j)
                if (j0 + j < a.k) a.dweights[row * a.k + j0 + j] = acc[j];
        }
    }
}

// ---- routes sorted by neuron ----------------------------------------------------------------------------------------------
// The routes are cut into chunks, a block each, and a chunk into one range per warp.  Blocks count their routes per neuron
// (count_kernel); the counts are turned into starting places, first along the chunks (column_kernel), then along the neurons
// (offsets_kernel); every warp then walks its range in order and puts its routes there (place_kernel): stable, so that a neuron's routes
// stay in the order of the images.

__global__ void __launch_bounds__(kThreads) count_kernel(const ReadOutGradArgs a)
{
    follow();
    extern __shared__ uint32_t bins[];                   // [N]
    for (uint32_t e = threadIdx.x; e < a.N; e += kThreads) bins[e] = 0;
    __syncthreads();
    const uint32_t lo = blockIdx.x * a.per_chunk, hi = min(lo + a.per_chunk, a.routes);
#pragma unroll 4
    for (uint32_t r = lo + threadIdx.x; r < hi; r += kThreads) {
        const uint32_t id = a.neurons[r];
        if (id < a.N) atomicAdd(&bins[id], 1u);
        else if (a.dweights) a.dweights[r] = 0.0f;       // (narrow_kernel, which walks the sorted routes, does not come by absent ones)
    }
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < a.N; e += kThreads) a.counts[(size_t)blockIdx.x * a.N + e] = bins[e];
}

// Running sums along the chunks: a block takes 32 neurons, its eight warps a range of chunks each, kMaxChunks at a time.
constexpr uint32_t kMaxChunks = 256;
__global__ void __launch_bounds__(kThreads) column_kernel(const ReadOutGradArgs a)
{
    __shared__ uint32_t part[8][32];
    follow();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    uint32_t carry = 0;
    for (uint32_t c0 = 0; c0 < a.chunks; c0 += kMaxChunks) {
        const uint32_t here = min(kMaxChunks, a.chunks - c0), per = (here + 7) / 8;
        const uint32_t lo = c0 + min(warp * per, here), hi = min(lo + per, c0 + here);
        uint32_t v[kMaxChunks / 8], sum = 0;
#pragma unroll
        for (uint32_t c = 0; c < kMaxChunks / 8; ++c) v[c] = e < a.N && lo + c < hi ? a.counts[(size_t)(lo + c) * a.N + e] : 0;
#pragma unroll
        for (uint32_t c = 0; c < kMaxChunks / 8; ++c) sum += v[c];
        part[warp][lane] = sum;
        __syncthreads();
        uint32_t run = carry, all = 0;
#pragma unroll
        for (uint32_t w = 0; w < 8; ++w) {
            if (w < warp) run += part[w][lane];
            all += part[w][lane];
        }
#pragma unroll
        for (uint32_t c = 0; c < kMaxChunks / 8; ++c) {
            if (e < a.N && lo + c < hi) a.counts[(size_t)(lo + c) * a.N + e] = run;
            run += v[c];
        }
        carry += all;
        __syncthreads();
    }
    if (warp == 0 && e < a.N) a.total[e] = carry;
}

// A neuron's routes are added up in segments.  A block (a warp, for narrow rows) walks its segment in a few steps of loads that depend on
// nothing before them, so that a popular neuron does not hold up the others.
constexpr uint32_t kSegmentWide = 32, kSegmentNarrow = 64;

__device__ __forceinline__ uint32_t segments_of(const ReadOutGradArgs& a, uint32_t routes) { return max((routes + a.segment - 1) / a.segment, 1u); }

// One block: running sums over the neurons of routes, segments and partial rows.
__global__ void __launch_bounds__(1024) offsets_kernel(const ReadOutGradArgs a)
{
    follow();
    __shared__ uint32_t warp_sums[3][32];
    uint32_t carry[3] = { 0, 0, 0 };
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint32_t e0 = 0; e0 < a.N; e0 += 1024) {
        const uint32_t e = e0 + threadIdx.x;
        uint32_t own[3] = { 0, 0, 0 }, run[3];
        if (e < a.N) {
            own[0] = a.total[e];
            own[1] = segments_of(a, own[0]);
            own[2] = own[1] > 1 ? own[1] : 0;
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            run[q] = own[q];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, run[q], o);
                if (lane >= (uint32_t)o) run[q] += v;
            }
            if (lane == 31) warp_sums[q][warp] = run[q];
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            uint32_t w = warp_sums[q][lane];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, w, o);
                if (lane >= (uint32_t)o) w += v;
            }
            run[q] += carry[q] - own[q] + (warp ? __shfl_sync(0xFFFFFFFFu, w, warp - 1) : 0u);
            carry[q] += __shfl_sync(0xFFFFFFFFu, w, 31);
        }
        if (e < a.N) {
            a.first[e] = run[0];
            a.part_first[e] = run[2];
        }
        if (e < a.N) a.seg_first[e] = run[1];
        __syncthreads();
    }
    if (threadIdx.x == 0) { a.part_first[a.N] = carry[2]; *a.n_segments = carry[1]; }
}

// A warp's counters of its routes per neuron are 16 bits wide, two in a word: routes are cut so that a block has fewer than 2^16.
constexpr uint32_t kPlaceWarps = 16;

// Counts the routes mine .. end of a warp.
__device__ __forceinline__ void count_range(const ReadOutGradArgs& a, uint32_t* own, uint32_t mine, uint32_t end, uint32_t lane, bool clear_absent)
{
    constexpr uint32_t kAhead = 4;                       // groups of 32 routes loaded ahead
    for (uint32_t r0 = mine + lane; r0 < end; r0 += 32 * kAhead) {
        uint32_t ids[kAhead];
#pragma unroll
        for (uint32_t q = 0; q < kAhead; ++q) ids[q] = r0 + 32 * q < end ? a.neurons[r0 + 32 * q] : kNoNeuron;
#pragma unroll
        for (uint32_t q = 0; q < kAhead; ++q) {
            if (ids[q] < a.N) atomicAdd(&own[ids[q] >> 1], ids[q] & 1u ? 0x10000u : 1u);
            else if (clear_absent && r0 + 32 * q < end) a.dweights[r0 + 32 * q] = 0.0f;
        }
    }
}

// Turns the warps' counts into the counts of the warps before (both halves of a word at once: their sums stay below 2^16, as the
// block's routes do) and returns the sum of all.
__device__ __forceinline__ uint32_t counts_before(uint32_t* counters, uint32_t warps, uint32_t pitch, uint32_t word)
{
    uint32_t before = 0;
    for (uint32_t w = 0; w < warps; ++w) {
        const uint32_t c = counters[w * pitch + word];
        counters[w * pitch + word] = before;
        before += c;
    }
    return before;
}

// Puts the routes of a warp, in order, at base[neuron] + next[neuron].
__device__ __forceinline__ void place_range(const ReadOutGradArgs& a, const uint32_t* base, uint16_t* next, uint32_t mine, uint32_t end, uint32_t lane)
{
    constexpr uint32_t kAhead = 4;
    for (uint32_t r0 = mine; r0 < end; r0 += 32 * kAhead) {
        uint32_t ids[kAhead];
        float w[kAhead];
#pragma unroll
        for (uint32_t q = 0; q < kAhead; ++q) {
            const uint32_t r = r0 + q * 32 + lane;
            ids[q] = r < end ? a.neurons[r] : kNoNeuron;
            w[q] = r < end ? a.weights[r] : 0.0f;
        }
#pragma unroll
        for (uint32_t q = 0; q < kAhead; ++q) {
            const uint32_t id = ids[q];
            const bool there = id < a.N;
            const uint32_t same = __match_any_sync(0xFFFFFFFFu, there ? id : kNoNeuron);
            const uint32_t rank = __popc(same & ((1u << lane) - 1));
            const uint32_t at = there ? next[id] : 0;
            __syncwarp();
            if (there) {
                a.sorted[base[id] + at + rank] = make_uint2(r0 + q * 32 + lane, __float_as_uint(w[q]));
                if (rank == 0) next[id] = (uint16_t)(at + __popc(same));
            }
            __syncwarp();
        }
    }
}

__device__ __forceinline__ void write_segments(const ReadOutGradArgs& a, uint32_t e, uint32_t routes, uint32_t first, uint32_t seg, uint32_t part)
{
    const uint32_t count = segments_of(a, routes);
    for (uint32_t g = 0; g < count; ++g)
        a.segments[seg + g] = make_uint4(first + g * a.segment, min(a.segment, routes - g * a.segment), e, count > 1 ? part + g : kNoNeuron);
}

// As many warps (up to kPlaceWarps) as have room for counters of their own; `base` holds where the chunk's routes to a neuron begin.
__global__ void __launch_bounds__(kPlaceWarps * 32) place_kernel(const ReadOutGradArgs a)
{
    extern __shared__ uint32_t base[];                   // [N], then [warps][N rounded up to 2] 16-bit counters
    follow();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, pitch = (a.N + 1) / 2;
    const uint32_t lo = blockIdx.x * a.per_chunk, hi = min(lo + a.per_chunk, a.routes);
    // the segments of the neurons, which the blocks share out
    for (uint32_t e = blockIdx.x * blockDim.x + threadIdx.x; e < a.N; e += gridDim.x * blockDim.x)
        write_segments(a, e, a.total[e], a.first[e], a.seg_first[e], a.part_first[e]);
    const uint32_t per = (a.per_chunk + warps * 32 - 1) / (warps * 32) * 32;             // routes of a warp
    const uint32_t mine = min(lo + warp * per, hi), end = min(mine + per, hi);
    uint32_t* counters = base + a.N;
    for (uint32_t q = threadIdx.x; q < warps * pitch; q += blockDim.x) counters[q] = 0;
#pragma unroll 4
    for (uint32_t e = threadIdx.x; e < a.N; e += blockDim.x) base[e] = a.first[e] + a.counts[(size_t)blockIdx.x * a.N + e];
    __syncthreads();
    uint32_t* own = counters + warp * pitch;
    count_range(a, own, mine, end, lane, false);
    __syncthreads();
    for (uint32_t q = threadIdx.x; q < pitch; q += blockDim.x) counts_before(counters, warps, pitch, q);
    __syncthreads();
    place_range(a, base, reinterpret_cast<uint16_t*>(own), mine, end, lane);
}

// Few routes: the whole sort in one block, in place of the four kernels above (1,024 images of four routes, 400 neurons: 14 us in four
// launches).
constexpr uint32_t kSmallRoutes = 8192, kSmallNeurons = 4096;

__global__ void __launch_bounds__(kPlaceWarps * 32) sort_small_kernel(const ReadOutGradArgs a)
{
    extern __shared__ uint32_t base[];                   // [N rounded up to 2] routes of a neuron, then where they begin; [warps][N rounded up to 2] counters
    __shared__ uint32_t warp_sums[3][kPlaceWarps];
    follow();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pitch = (a.N + 1) / 2;
    const uint32_t per = (a.routes + kPlaceWarps * 32 - 1) / (kPlaceWarps * 32) * 32;
    const uint32_t mine = min(warp * per, a.routes), end = min(mine + per, a.routes);
    uint32_t* counters = base + 2 * pitch;
    for (uint32_t q = threadIdx.x; q < kPlaceWarps * pitch; q += kPlaceWarps * 32) counters[q] = 0;
    __syncthreads();
    uint32_t* own = counters + warp * pitch;
    count_range(a, own, mine, end, lane, a.dweights != nullptr);
    __syncthreads();
    for (uint32_t q = threadIdx.x; q < pitch; q += kPlaceWarps * 32) {
        const uint32_t all = counts_before(counters, kPlaceWarps, pitch, q);
        base[2 * q] = all & 0xFFFFu;
        base[2 * q + 1] = all >> 16;
    }
    __syncthreads();
    // running sums of routes, segments and partial rows: a run of neurons per thread
    const uint32_t run = (a.N + kPlaceWarps * 32 - 1) / (kPlaceWarps * 32), e0 = min(threadIdx.x * run, a.N), e1 = min(e0 + run, a.N);
    uint32_t own3[3] = { 0, 0, 0 }, at[3];
    for (uint32_t e = e0; e < e1; ++e) {
        const uint32_t routes = base[e], count = segments_of(a, routes);
        own3[0] += routes;
        own3[1] += count;
        own3[2] += count > 1 ? count : 0;
    }
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        at[q] = own3[q];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, at[q], o);
            if (lane >= (uint32_t)o) at[q] += v;
        }
        if (lane == 31) warp_sums[q][warp] = at[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 3; ++q) {
        at[q] -= own3[q];
        for (uint32_t w = 0; w < warp; ++w) at[q] += warp_sums[q][w];
    }
    for (uint32_t e = e0; e < e1; ++e) {
        const uint32_t routes = base[e], count = segments_of(a, routes);
        write_segments(a, e, routes, at[0], at[1], at[2]);
        a.part_first[e] = at[2];
        base[e] = at[0];
        at[0] += routes;
        at[1] += count;
        at[2] += count > 1 ? count : 0;
    }
    if (threadIdx.x == kPlaceWarps * 32 - 1) { a.part_first[a.N] = at[2]; *a.n_segments = at[1]; }
    __syncthreads();
    place_range(a, base, reinterpret_cast<uint16_t*>(own), mine, end, lane);
}

// ---- gradient of the values -----------------------------------------------------------------------------------------------

// Wider rows: a block per segment of a neuron's routes, PARTS vectors a thread, walking the column tiles blockIdx.y, blockIdx.y +
// gridDim.y, ...: what leads to a segment's first load is a chain of three, which few routes a neuron do not hide.  The gradient of the
// weights comes with it, since the neuron's row and the images' gradients are at hand.
template <typename T, int VEC, int PARTS>
__global__ void __launch_bounds__(kThreads) dvalues_kernel(const ReadOutGradArgs a)
{
    follow();
    __shared__ uint2 route_s[kSegmentWide];
    __shared__ float dot_s[kThreads / 32][kSegmentWide];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint4 seg = a.segments[blockIdx.x];            // (whatever it is beyond the last: there is room for a segment per block)
    if (blockIdx.x >= *a.n_segments) return;
    const uint32_t count = seg.y, e = seg.z;
    for (uint32_t p = threadIdx.x; p < count; p += blockDim.x) route_s[p] = a.sorted[seg.x + p];
    dot_s[warp][lane] = 0.0f;
    __syncthreads();
    const uint32_t step = blockDim.x * VEC;
    for (uint32_t tile = blockIdx.y; tile < a.tiles; tile += gridDim.y) {
        const uint32_t col = tile * PARTS * step + threadIdx.x * VEC;
        float acc[PARTS][VEC], own[PARTS][VEC];
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) acc[q][v] = own[q][v] = 0.0f;
            if (a.dots && count && col + q * step < a.D)
                Pack<T, VEC>::load(static_cast<const T*>(a.values) + e * a.ld + col + q * step).floats(own[q]);
        }
        const T* dout = static_cast<const T*>(a.dout) + col;
        constexpr uint32_t kTogether = 4;                // routes whose loads are in flight together
        static_assert(kTogether == 4 && kSegmentWide % kTogether == 0, "the sum over a warp below is made for four");
        for (uint32_t p0 = 0; p0 < count; p0 += kTogether) {
            Pack<T, VEC> d[kTogether][PARTS];
            float dot[kTogether];
#pragma unroll
            for (uint32_t h = 0; h < kTogether; ++h) {
                if (p0 + h >= count) continue;
                const T* src = dout + (uint64_t)(route_s[p0 + h].x / a.k) * a.ld_dout;
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
                    if (col + q * step < a.D) d[h][q] = Pack<T, VEC>::load(src + q * step);
            }
#pragma unroll
            for (uint32_t h = 0; h < kTogether; ++h) {
                dot[h] = 0.0f;
                if (p0 + h >= count) continue;
                const float w = __uint_as_float(route_s[p0 + h].y);
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
                    if (col + q * step < a.D) {
                        float g[VEC];
                        d[h][q].floats(g);
#pragma unroll
                        for (int v = 0; v < VEC; ++v) {
                            acc[q][v] = fmaf(w, g[v], acc[q][v]);
                            dot[h] = fmaf(g[v], own[q][v], dot[h]);
                        }
                    }
            }
            if (a.dots) {
                // four sums over the warp at once: lanes 8 h .. 8 h + 7 end with that of route h
                const float u0 = (lane & 16 ? dot[2] : dot[0]) + __shfl_xor_sync(0xFFFFFFFFu, lane & 16 ? dot[0] : dot[2], 16);
                const float u1 = (lane & 16 ? dot[3] : dot[1]) + __shfl_xor_sync(0xFFFFFFFFu, lane & 16 ? dot[1] : dot[3], 16);
                float u = (lane & 8 ? u1 : u0) + __shfl_xor_sync(0xFFFFFFFFu, lane & 8 ? u0 : u1, 8);
#pragma unroll
                for (int o = 4; o; o >>= 1) u += __shfl_xor_sync(0xFFFFFFFFu, u, o);
                if ((lane & 7) == 0) dot_s[warp][p0 + (lane >> 3)] += u;
            }
        }
#pragma unroll
        for (int q = 0; q < PARTS; ++q) {
            if (col + q * step >= a.D) break;
            if (seg.w == kNoNeuron) {
                Pack<T, VEC>::of(acc[q]).store(static_cast<T*>(a.dvalues) + e * a.ld_dvalues + col + q * step);
            } else {
                float* dst = a.parts + (size_t)seg.w * a.part_ld + col + q * step;
#pragma unroll
                for (int v = 0; v < VEC; ++v) dst[v] = acc[q][v];
            }
        }
    }
    if (a.dots) {
        __syncthreads();
        if (threadIdx.x < count) {
            float s = 0.0f;
            for (uint32_t w = 0; w < blockDim.x / 32; ++w) s += dot_s[w][threadIdx.x];
            a.dots[(size_t)blockIdx.y * a.routes + route_s[threadIdx.x].x] = s;
        }
    }
}

// Narrow rows (a warp holds one or more of them): a warp per segment, lanes along the columns and along the routes.  The gradient of
// the weights comes with it: the neuron's row and the image's gradient are at hand.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) narrow_kernel(const ReadOutGradArgs a)
{
    follow();
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t seg_at = blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const uint4 seg = a.segments[min(seg_at, a.most_segments - 1)];
    if (seg_at >= *a.n_segments) return;
    const uint32_t e = seg.z, begin = seg.x, end = seg.x + seg.y;
    const uint32_t width = 1u << a.tx_shift, height = 32u >> a.tx_shift;
    const uint32_t tx = lane & (width - 1), ty = lane >> a.tx_shift, col = tx * VEC;
    const bool in = col < a.D;
    float acc[VEC], own[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) { acc[v] = 0.0f; own[v] = 0.0f; }
    if (a.dweights && in) {
        Pack<T, VEC>::load(static_cast<const T*>(a.values) + e * a.ld + col).floats(own);
    }
    constexpr uint32_t kAhead = 4;                       // rows of routes in flight
    for (uint32_t p0 = begin; p0 < end; p0 += height * kAhead) {
        uint32_t r[kAhead];
        float w[kAhead];
        Pack<T, VEC> d[kAhead];
#pragma unroll
        for (uint32_t q = 0; q < kAhead; ++q) {
            const uint32_t p = p0 + q * height + ty;
            const uint2 s = p < end ? a.sorted[p] : make_uint2(kNoNeuron, 0u);
            r[q] = s.x;
            w[q] = __uint_as_float(s.y);
        }
#pragma unroll
        for (uint32_t q = 0; q < kAhead; ++q) {
            if (r[q] == kNoNeuron) continue;
            if (in) d[q] = Pack<T, VEC>::load(static_cast<const T*>(a.dout) + (uint64_t)(r[q] / a.k) * a.ld_dout + col);
        }
#pragma unroll
        for (uint32_t q = 0; q < kAhead; ++q) {
            float dot = 0.0f;
            if (r[q] != kNoNeuron && in) {
                float g[VEC];
                d[q].floats(g);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    acc[v] = fmaf(w[q], g[v], acc[v]);
                    dot = fmaf(g[v], own[v], dot);
                }
            }
            if (a.dweights) {
                for (uint32_t o = width / 2; o; o >>= 1) dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
                if (tx == 0 && r[q] != kNoNeuron) a.dweights[r[q]] = dot;
            }
        }
    }
#pragma unroll
    for (int v = 0; v < VEC; ++v)
        for (uint32_t o = 16; o >= width; o >>= 1) acc[v] += __shfl_xor_sync(0xFFFFFFFFu, acc[v], o);
    if (ty != 0 || !in) return;
    if (seg.w == kNoNeuron) {
        Pack<T, VEC>::of(acc).store(static_cast<T*>(a.dvalues) + e * a.ld_dvalues + col);
    } else {
        float* dst = a.parts + (size_t)seg.w * a.part_ld + col;
#pragma unroll
        for (int v = 0; v < VEC; ++v) dst[v] = acc[v];
    }
}

// Sums of the partial rows of the neurons that have several segments, and of the products of the blocks along the columns.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_kernel(const ReadOutGradArgs a, uint32_t column_blocks)
{
    follow();
    if (a.dots && blockIdx.y == 0)
        for (uint32_t r = blockIdx.x * kThreads + threadIdx.x; r < a.routes; r += gridDim.x * kThreads) {
            float s = 0.0f;
            if (a.neurons[r] < a.N)
                for (uint32_t t = 0; t < column_blocks; ++t) s += a.dots[(size_t)t * a.routes + r];
            a.dweights[r] = s;
        }
    if (a.D > 128) {                                     // wide: the block along the columns
        for (uint32_t e = blockIdx.x; e < a.N; e += gridDim.x) {
            const uint32_t lo = a.part_first[e], hi = a.part_first[e + 1];
            if (lo == hi) continue;
            for (uint32_t col = blockIdx.y * kThreads + threadIdx.x; col < a.D; col += gridDim.y * kThreads) {
                float acc = 0.0f;
#pragma unroll 8
                for (uint32_t p = lo; p < hi; ++p) acc += a.parts[(size_t)p * a.part_ld + col];
                static_cast<T*>(a.dvalues)[e * a.ld_dvalues + col] = from_float<T>(acc);
            }
        }
        return;
    }
    // narrow (a popular neuron has hundreds of rows): lanes along the columns, the warps along the rows, whose sums meet in order
    __shared__ float meet[kThreads / 32][32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint32_t e = blockIdx.x; e < a.N; e += gridDim.x) {
        const uint32_t lo = a.part_first[e], hi = a.part_first[e + 1];
        if (lo == hi) continue;
        for (uint32_t c0 = blockIdx.y * 32; c0 < a.D; c0 += gridDim.y * 32) {
            const uint32_t col = c0 + lane;
            float acc = 0.0f;
            if (col < a.D)
#pragma unroll 4
                for (uint32_t p = lo + warp; p < hi; p += kThreads / 32) acc += a.parts[(size_t)p * a.part_ld + col];
            meet[warp][lane] = acc;
            __syncthreads();
            if (warp == 0 && col < a.D) {
#pragma unroll
                for (uint32_t w = 1; w < kThreads / 32; ++w) acc += meet[w][lane];
                static_cast<T*>(a.dvalues)[e * a.ld_dvalues + col] = from_float<T>(acc);
            }
            __syncthreads();
        }
    }
}

// Whether a warp's lanes cover a row in vectors of `vec`: narrow_kernel's case.
bool is_narrow(uint32_t D, uint32_t vec) { return (D + vec - 1) / vec <= 32; }

// Where the pieces of the workspace lie, and how the sort is cut.
struct SortPlan
{
    uint32_t chunks, per_chunk, segment, tiles, part_rows, part_ld;
    uint64_t counts, total, first, seg_first, part_first, n_segments, segments, sorted, dots, parts, bytes;
};

// vec 0: enough for whatever alignment the call will find.
SortPlan sort_plan(uint32_t N, uint32_t D, uint64_t routes, uint32_t vec)
{
    SortPlan p{};
    // every chunk costs a row of N counts: 1024 routes each at least, and at most kMaxChunks of them -- unless they would be too long
    // for the 16-bit counters of place_kernel
    p.chunks = (uint32_t)std::max(std::min<uint64_t>(kMaxChunks, (routes + 1023) / 1024), (routes + 65279) / 65280);
    p.per_chunk = (uint32_t)((routes + p.chunks - 1) / p.chunks);
    p.segment = vec && is_narrow(D, vec) ? kSegmentNarrow : kSegmentWide;
    // column tiles of a block: two vectors a thread where there are that many
    const uint32_t v = vec ? vec : 1, vectors = (D + v - 1) / v;
    p.tiles = vectors >= 2 * kThreads ? (vectors + 2 * kThreads - 1) / (2 * kThreads) : (vectors + kThreads - 1) / kThreads;
    // a neuron with several segments has more routes than one holds: fewer than 2 * routes / segment such segments in all
    p.part_rows = (uint32_t)(2 * routes / p.segment);
    p.part_ld = (D + 3) / 4 * 4;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) { const uint64_t here = at; at += (bytes + 15) / 16 * 16; return here; };
    p.counts = take((uint64_t)p.chunks * N * 4);
    p.total = take((uint64_t)N * 4);
    p.first = take((uint64_t)N * 4);
    p.seg_first = take((uint64_t)N * 4);
    p.part_first = take(((uint64_t)N + 1) * 4);
    p.n_segments = take(4);
    p.segments = take((N + routes / p.segment) * 16);
    p.sorted = take(routes * 8);
    p.dots = take(vec && is_narrow(D, vec) ? 0 : p.tiles * routes * 4);
    p.parts = take((uint64_t)p.part_rows * p.part_ld * 4);
    p.bytes = at;
    return p;
}

// Shared memory of sort_small_kernel and of a warp's counters in place_kernel, and the warps of the latter: as many as leave room for two
// blocks an SM, one at least.
constexpr size_t small_shared(size_t n_neurons) { return (n_neurons + 1) / 2 * (8 + kPlaceWarps * 4); }
constexpr size_t counter_bytes(size_t n_neurons) { return (n_neurons + 1) / 2 * 4; }

uint32_t place_warps_for(uint32_t n_neurons)
{
    const size_t base = std::min<size_t>(n_neurons * sizeof(uint32_t), 64 * 1024);
    return (uint32_t)std::max<size_t>(1, std::min<size_t>(kPlaceWarps, (110 * 1024 - base) / counter_bytes(n_neurons)));
}

// (Up to 16,384 neurons a block has at most 110 KB; beyond, one warp's counters, or 46 KB of them, beside the neurons' words.)
constexpr size_t kMostPlaceShared = PINK_B200_MAX_ROUTED_NEURONS * sizeof(uint32_t) + counter_bytes(PINK_B200_MAX_ROUTED_NEURONS);

uint32_t log2_threads(uint32_t columns)                  // threads along a row: the smallest power of two that covers it, at most kThreads
{
    uint32_t s = 0;
    while (s < 8 && (1u << s) < columns) ++s;
    return s;
}

// Calls fn(T value, integral constant) with the element type and the widest load that alignment and row length allow.
template <typename Fn>
cudaError_t with_vector(uint32_t type, uint32_t vec, Fn fn)
{
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int full = 16 / sizeof(T);
        if (vec >= full) return fn(t, std::integral_constant<int, full>());
        if (full == 8 && vec == 4) return fn(t, std::integral_constant<int, 4>());
        if (vec >= 2) return fn(t, std::integral_constant<int, 2>());
        return fn(t, std::integral_constant<int, 1>());
    });
}

uint32_t vector_width(uint32_t type, uint32_t D, RowAlign align)
{
    const uint32_t size = (uint32_t)element_size(type);
    uint32_t v = align.elements(size, 16 / size);
    while (v > 1 && D % v) v >>= 1;
    return v;
}

int check_read_out(uint32_t type, uint32_t N, uint32_t D, uint64_t ld, uint64_t n, uint32_t k)
{
    if (type > PINK_B200_F16) return report_error(PINK_B200_EINVAL, "unknown element type");
    if (N == 0 || N == kNoNeuron) return report_error(PINK_B200_EINVAL, "n_neurons must be 1 to 4294967294");
    if (D == 0 || D > 1u << 24) return report_error(PINK_B200_EINVAL, "dims must be 1 to 16777216");
    if (k == 0 || k > PINK_B200_MAX_ROUTES) return report_error(PINK_B200_EINVAL, "top_k must be 1 to 32");
    if (n > 0x7FFFFFFFull) return report_error(PINK_B200_EINVAL, "at most 2147483647 rows");
    if (ld < D) return report_error(PINK_B200_EINVAL, "leading dimension smaller than dims");
    return PINK_B200_OK;
}

} // namespace
} // namespace pinkb

using namespace pinkb;

extern "C" {

int pink_b200_op_read_out(uint32_t type, uint32_t n_neurons, uint32_t dims, const void* dev_values, uint64_t ld_values, uint64_t n,
                          uint32_t top_k, const uint32_t* dev_neurons, const float* dev_weights, const void* dev_residual,
                          uint64_t ld_residual, void* dev_out, uint64_t ld_out, void* stream)
{
    const int rc = check_read_out(type, n_neurons, dims, ld_values, n, top_k);
    if (rc) return rc;
    if (ld_out < dims || (dev_residual && ld_residual < dims)) return report_error(PINK_B200_EINVAL, "leading dimension smaller than dims");
    if (n == 0) return PINK_B200_OK;
    if (!dev_values || !dev_neurons || !dev_weights || !dev_out) return report_error(PINK_B200_EINVAL, "null argument");
    const size_t size = element_size(type);
    const uint32_t vec = vector_width(type, dims, RowAlign().add(dev_values, ld_values, size).add(dev_residual, ld_residual, size)
                                                      .add(dev_out, ld_out, size));
    ReadOutArgs a{n, n_neurons, dims, top_k, dev_values, ld_values, dev_neurons, dev_weights, dev_residual, ld_residual, dev_out, ld_out,
                  log2_threads((dims + vec - 1) / vec)};
    const uint32_t rows = kThreads >> a.tx_shift, columns = vec << a.tx_shift, tiles = (dims + columns - 1) / columns;
    const uint64_t row_blocks = (n + rows - 1) / rows;
    // two vectors a thread where that leaves every SM a few blocks (2,000 rows of 8,192 bfloat16, eight routes: 38 -> 34 us)
    const bool two = tiles >= 2 && row_blocks * ((tiles + 1) / 2) >= 512;
    const dim3 grid((unsigned)row_blocks, two ? (tiles + 1) / 2 : tiles);
    return launch_status(with_vector(type, vec, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int VEC = decltype(v)::value;
        if (two) read_out_kernel<T, VEC, 2><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
        else read_out_kernel<T, VEC, 1><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
        return cudaGetLastError();
    }), "read-out kernel");
}

uint64_t pink_b200_read_out_workspace(uint32_t n_neurons, uint32_t dims, uint64_t n, uint32_t top_k)
{
    if (n_neurons == 0 || n_neurons > PINK_B200_MAX_ROUTED_NEURONS || dims == 0 || top_k == 0 || top_k > PINK_B200_MAX_ROUTES) return 0;
    if (n == 0 || n > 0x7FFFFFFFull / top_k) return 0;
    return sort_plan(n_neurons, dims, n * top_k, 0).bytes;
}

int pink_b200_op_read_out_backward(uint32_t type, uint32_t n_neurons, uint32_t dims, const void* dev_values, uint64_t ld_values,
                                   uint64_t n, uint32_t top_k, const uint32_t* dev_neurons, const float* dev_weights,
                                   const void* dev_dout, uint64_t ld_dout, void* dev_dvalues, uint64_t ld_dvalues, float* dev_dweights,
                                   void* dev_workspace, uint64_t workspace_bytes, void* stream)
{
    const int rc = check_read_out(type, n_neurons, dims, dev_dweights ? ld_values : dims, n, top_k);
    if (rc) return rc;
    if (n_neurons > PINK_B200_MAX_ROUTED_NEURONS) return report_error(PINK_B200_EINVAL, "the gradient takes at most 32768 neurons");
    if (n > 0x7FFFFFFFull / top_k) return report_error(PINK_B200_EINVAL, "n * top_k must be below 2147483648");
    if ((n && ld_dout < dims) || (dev_dvalues && ld_dvalues < dims)) return report_error(PINK_B200_EINVAL, "leading dimension smaller than dims");
    if (n && (!dev_neurons || !dev_weights || !dev_dout || (dev_dweights && !dev_values))) return report_error(PINK_B200_EINVAL, "null argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const size_t size = element_size(type);
    if (n == 0) {                                        // no routes: the table's gradient is zero
        if (!dev_dvalues) return PINK_B200_OK;
        return launch_status(cudaMemset2DAsync(dev_dvalues, ld_dvalues * size, 0, dims * size, n_neurons, st), "clearing the gradient");
    }
    ReadOutGradArgs a{};
    a.n = n; a.N = n_neurons; a.D = dims; a.k = top_k;
    a.values = dev_values; a.ld = ld_values; a.neurons = dev_neurons; a.weights = dev_weights;
    a.dout = dev_dout; a.ld_dout = ld_dout; a.dvalues = dev_dvalues; a.ld_dvalues = ld_dvalues; a.dweights = dev_dweights;
    if (dev_dvalues) {
        if (!dev_workspace || workspace_bytes < pink_b200_read_out_workspace(n_neurons, dims, n, top_k))
            return report_error(PINK_B200_EINVAL, "workspace too small (pink_b200_read_out_workspace)");
        if (reinterpret_cast<uintptr_t>(dev_workspace) % 16) return report_error(PINK_B200_EINVAL, "the workspace must be 16-byte aligned");
        const uint32_t vec = vector_width(type, dims, RowAlign().add(dev_dout, ld_dout, size).add(dev_dvalues, ld_dvalues, size)
                                                          .add(dev_dweights ? dev_values : nullptr, ld_values, size));
        const bool narrow = is_narrow(dims, vec);
        const SortPlan p = sort_plan(n_neurons, dims, n * top_k, vec);
        uint8_t* base = static_cast<uint8_t*>(dev_workspace);
        auto at = [&](uint64_t off) { return reinterpret_cast<uint32_t*>(base + off); };
        a.routes = (uint32_t)(n * top_k); a.chunks = p.chunks; a.per_chunk = p.per_chunk; a.segment = p.segment;
        a.tiles = p.tiles;
        a.counts = at(p.counts); a.total = at(p.total); a.first = at(p.first); a.seg_first = at(p.seg_first); a.part_first = at(p.part_first); a.n_segments = at(p.n_segments);
        a.segments = reinterpret_cast<uint4*>(base + p.segments); a.sorted = reinterpret_cast<uint2*>(base + p.sorted); a.parts = reinterpret_cast<float*>(base + p.parts); a.part_ld = p.part_ld;
        a.dots = dev_dweights && !narrow ? reinterpret_cast<float*>(base + p.dots) : nullptr;
        a.tx_shift = log2_threads((dims + vec - 1) / vec);
        const size_t smem = n_neurons * sizeof(uint32_t);
        const uint32_t place_warps = place_warps_for(n_neurons);
        const size_t place_smem = smem + place_warps * counter_bytes(n_neurons);
        const uint32_t segments = n_neurons + a.routes / p.segment;          // one for every neuron, one more for every full segment
        a.most_segments = segments;
        // blocks along the columns: only as many as give every SM several blocks
        const uint32_t column_blocks = std::max(1u, std::min(p.tiles, 2368 / segments));
        return launch_status([&] {
            cudaError_t e = cudaSuccess;
            if (a.routes <= kSmallRoutes && n_neurons <= kSmallNeurons) {
                const size_t small = small_shared(n_neurons);
                e = allow_shared(sort_small_kernel, small, small_shared(kSmallNeurons));
                if (e == cudaSuccess) e = launch_following(sort_small_kernel, 1, kPlaceWarps * 32, small, st, a);
            } else {
                e = allow_shared(count_kernel, smem, PINK_B200_MAX_ROUTED_NEURONS * sizeof(uint32_t));
                if (e == cudaSuccess) e = allow_shared(place_kernel, place_smem, kMostPlaceShared);
                if (e == cudaSuccess) e = launch_following(count_kernel, a.chunks, kThreads, smem, st, a);
                if (e == cudaSuccess) e = launch_following(column_kernel, (n_neurons + 31) / 32, kThreads, 0, st, a);
                if (e == cudaSuccess) e = launch_following(offsets_kernel, 1, 1024, 0, st, a);
                if (e == cudaSuccess) e = launch_following(place_kernel, a.chunks, place_warps * 32, place_smem, st, a);
            }
            if (e != cudaSuccess) return e;
            e = with_vector(type, vec, [&](auto t, auto v) {
                using T = decltype(t);
                constexpr int VEC = decltype(v)::value;
                if (narrow) return launch_following(narrow_kernel<T, VEC>, (segments + kThreads / 32 - 1) / (kThreads / 32), kThreads, 0, st, a);
                const uint32_t vectors = (dims + VEC - 1) / VEC, threads = std::min(kThreads, (vectors + 31) / 32 * 32);
                if (vectors >= 2 * kThreads) return launch_following(dvalues_kernel<T, VEC, 2>, dim3(segments, column_blocks), kThreads, 0, st, a);
                return launch_following(dvalues_kernel<T, VEC, 1>, dim3(segments, column_blocks), threads, 0, st, a);
            });
            if (e != cudaSuccess || (!a.dots && p.part_rows < 2)) return e;
            return with_type(type, [&](auto t) {
                return launch_following(join_kernel<decltype(t)>, dim3(std::min(n_neurons, 592u), dims > 128 ? std::min((dims + kThreads - 1) / kThreads, 8u) : (dims + 31) / 32),
                                        kThreads, 0, st,
                                        a, column_blocks);
            });
        }(), "gradient of the values");
    }
    if (!dev_dweights) return PINK_B200_OK;
    const uint32_t vec = vector_width(type, dims, RowAlign().add(dev_dout, ld_dout, size).add(dev_values, ld_values, size));
    const uint32_t columns = (dims + vec - 1) / vec;
    return launch_status(with_vector(type, vec, [&](auto t, auto v) {
        using T = decltype(t);
        constexpr int VEC = decltype(v)::value;
        // threads per image: enough for a row of loads
        if (columns <= 8) dweights_kernel<T, VEC, 8><<<(unsigned)((n + 31) / 32), kThreads, 0, st>>>(a);
        else if (columns <= 128) dweights_kernel<T, VEC, 32><<<(unsigned)((n + 7) / 8), kThreads, 0, st>>>(a);
        else dweights_kernel<T, VEC, 256><<<(unsigned)n, kThreads, 0, st>>>(a);
        return cudaGetLastError();
    }), "gradient of the weights");
}

} // extern "C"
