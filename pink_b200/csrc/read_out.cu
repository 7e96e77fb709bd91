// Read-out of routed neurons and its gradient (pink_b200_op_read_out*).
//
//   out_i = sum_j w_ij V[e_ij] (+ residual_i),   dw_ij = <dout_i, V[e_ij]>,   dV[e] = sum over the routes to e of w_ij dout_i
//
// The forward pass and dw are gathers.  dV would be a scatter with floating-point atomics, whose order changes the result; here
// the routes are sorted by neuron first (a stable counting sort), and every neuron's routes are added up in a fixed order.
#include "readout.cuh"

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

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) read_out_kernel(const ReadOutArgs a)
{
    const uint32_t tx = threadIdx.x & ((1u << a.tx_shift) - 1), ty = threadIdx.x >> a.tx_shift;
    const uint64_t row = (uint64_t)blockIdx.x * (kThreads >> a.tx_shift) + ty;
    const uint32_t col = ((blockIdx.y << a.tx_shift) + tx) * VEC;
    if (row >= a.n || col >= a.D) return;
    const uint32_t* e = a.neurons + row * a.k;
    const float* w = a.weights + row * a.k;
    const T* values = static_cast<const T*>(a.values) + col;
    float acc[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
#pragma unroll 4
    for (uint32_t j = 0; j < a.k; ++j) {
        const uint32_t id = e[j];
        if (id >= a.N) continue;
        const float wj = w[j];
        const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC>*>(values + id * a.ld);
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = fmaf(wj, to_float(p.v[v]), acc[v]);
    }
    if (a.residual) {
        const Pack<T, VEC> r = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.residual) + row * a.ld_residual + col);
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] += to_float(r.v[v]);
    }
    Pack<T, VEC> o;
#pragma unroll
    for (int v = 0; v < VEC; ++v) o.v[v] = from_float<T>(acc[v]);
    *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.out) + row * a.ld_out + col) = o;
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
    uint32_t* counts;                // [chunks][N] routes of a chunk to a neuron, then where they start among the neuron's
    uint32_t* total;                 // [N] routes to a neuron
    uint32_t* first;                 // [N + 1] where a neuron's routes start in `sorted`
    uint32_t* seg_first;             // [N + 1] its first segment
    uint32_t* part_first;            // [N + 1] its first row of partial sums (neurons of several segments)
    uint32_t* sorted;                // [routes] route numbers (image * k + position) by neuron, in order
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
                const Pack<T, VEC> d = *reinterpret_cast<const Pack<T, VEC>*>(dout + col);
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    if (!v[j]) continue;
                    const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC>*>(v[j] + col);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[j] = fmaf(to_float(d.v[i]), to_float(p.v[i]), acc[j]);
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
// The routes are cut into chunks, one warp each.  A warp counts its routes per neuron (count), the counts are turned into
// starting places (columns, then neurons), and the warp walks its routes again in order and puts them there (place): stable,
// so that a neuron's routes stay in the order of the images.

__global__ void __launch_bounds__(32) count_kernel(const ReadOutGradArgs a)
{
    extern __shared__ uint32_t bins[];                   // [N]
    const uint32_t lane = threadIdx.x;
    for (uint32_t e = lane; e < a.N; e += 32) bins[e] = 0;
    __syncwarp();
    const uint64_t lo = (uint64_t)blockIdx.x * a.per_chunk, hi = min(lo + a.per_chunk, (uint64_t)a.routes);
    for (uint64_t r = lo + lane; r < hi; r += 32) {
        const uint32_t id = a.neurons[r];
        if (id < a.N) atomicAdd(&bins[id], 1u);
    }
    __syncwarp();
    for (uint32_t e = lane; e < a.N; e += 32) a.counts[(size_t)blockIdx.x * a.N + e] = bins[e];
}

__global__ void __launch_bounds__(kThreads) column_kernel(const ReadOutGradArgs a)
{
    const uint32_t e = blockIdx.x * kThreads + threadIdx.x;
    if (e >= a.N) return;
    uint32_t sum = 0;
#pragma unroll 8
    for (uint32_t c = 0; c < a.chunks; ++c) {
        const uint32_t v = a.counts[(size_t)c * a.N + e];
        a.counts[(size_t)c * a.N + e] = sum;
        sum += v;
    }
    a.total[e] = sum;
}

constexpr uint32_t kSegment = 128;                       // routes that one block adds up

__device__ __forceinline__ uint32_t segments_of(uint32_t routes) { return max((routes + kSegment - 1) / kSegment, 1u); }

// One block: running sums over the neurons of routes, segments and partial rows.
__global__ void __launch_bounds__(1024) offsets_kernel(const ReadOutGradArgs a)
{
    __shared__ uint32_t warp_sums[3][32];
    uint32_t carry[3] = { 0, 0, 0 };
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (uint32_t e0 = 0; e0 < a.N; e0 += 1024) {
        const uint32_t e = e0 + threadIdx.x;
        uint32_t own[3] = { 0, 0, 0 }, run[3];
        if (e < a.N) {
            own[0] = a.total[e];
            own[1] = segments_of(own[0]);
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
            uint32_t before = carry[q], all = 0;
            for (uint32_t w = 0; w < 32; ++w) {
                if (w < warp) before += warp_sums[q][w];
                all += warp_sums[q][w];
            }
            carry[q] += all;
            run[q] += before - own[q];
        }
        if (e < a.N) { a.first[e] = run[0]; a.seg_first[e] = run[1]; a.part_first[e] = run[2]; }
        __syncthreads();
    }
    if (threadIdx.x == 0) { a.first[a.N] = carry[0]; a.seg_first[a.N] = carry[1]; a.part_first[a.N] = carry[2]; }
}

__global__ void __launch_bounds__(32) place_kernel(const ReadOutGradArgs a)
{
    extern __shared__ uint32_t next[];                   // [N] place of the chunk's next route to a neuron
    const uint32_t lane = threadIdx.x;
    for (uint32_t e = lane; e < a.N; e += 32) next[e] = a.first[e] + a.counts[(size_t)blockIdx.x * a.N + e];
    __syncwarp();
    const uint64_t lo = (uint64_t)blockIdx.x * a.per_chunk, hi = min(lo + a.per_chunk, (uint64_t)a.routes);
    for (uint64_t r0 = lo; r0 < hi; r0 += 32) {
        const uint64_t r = r0 + lane;
        const uint32_t id = r < hi ? a.neurons[r] : kNoNeuron;
        const bool there = id < a.N;
        const uint32_t same = __match_any_sync(0xFFFFFFFFu, there ? id : kNoNeuron);
        const uint32_t rank = __popc(same & ((1u << lane) - 1));
        uint32_t at = there ? next[id] : 0;
        __syncwarp();
        if (there) {
            a.sorted[at + rank] = (uint32_t)r;
            if (rank == 0) next[id] = at + __popc(same);
        }
        __syncwarp();
    }
}

// ---- gradient of the values -----------------------------------------------------------------------------------------------

// A block per segment of a neuron's routes and tile of columns: threads along the columns and along the routes, whose sums
// meet in shared memory in order.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) dvalues_kernel(const ReadOutGradArgs a)
{
    __shared__ float meet[kThreads * VEC];
    const uint32_t seg = blockIdx.x;
    if (seg >= a.seg_first[a.N]) return;
    uint32_t lo = 0, hi = a.N;                           // the neuron of this segment: the last whose first segment is not beyond it
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (a.seg_first[mid] <= seg) lo = mid; else hi = mid;
    }
    const uint32_t e = lo, part = seg - a.seg_first[e];
    const uint32_t parts = a.seg_first[e + 1] - a.seg_first[e];
    const uint32_t begin = a.first[e] + part * kSegment, end = min(begin + kSegment, a.first[e + 1]);
    const uint32_t width = 1u << a.tx_shift, height = kThreads >> a.tx_shift;
    const uint32_t tx = threadIdx.x & (width - 1), ty = threadIdx.x >> a.tx_shift;
    const uint32_t col = (blockIdx.y * width + tx) * VEC;
    float acc[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
    if (col < a.D) {
#pragma unroll 4
        for (uint32_t p = begin + ty; p < end; p += height) {
            const uint32_t r = a.sorted[p];
            const float w = a.weights[r];
            const Pack<T, VEC> d = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.dout) + (uint64_t)(r / a.k) * a.ld_dout + col);
#pragma unroll
            for (int v = 0; v < VEC; ++v) acc[v] = fmaf(w, to_float(d.v[v]), acc[v]);
        }
    }
    if (height > 1) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) meet[v * kThreads + threadIdx.x] = acc[v];
        for (uint32_t h = height / 2; h; h >>= 1) {
            __syncthreads();
            if (ty < h)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    acc[v] += meet[v * kThreads + threadIdx.x + (h << a.tx_shift)];
                    meet[v * kThreads + threadIdx.x] = acc[v];
                }
        }
    }
    if (ty != 0 || col >= a.D) return;
    if (parts == 1) {
        Pack<T, VEC> o;
#pragma unroll
        for (int v = 0; v < VEC; ++v) o.v[v] = from_float<T>(acc[v]);
        *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.dvalues) + e * a.ld_dvalues + col) = o;
    } else {
        float* dst = a.parts + (size_t)(a.part_first[e] + part) * a.part_ld + col;
#pragma unroll
        for (int v = 0; v < VEC; ++v) dst[v] = acc[v];
    }
}

// Sums of the partial rows of the neurons that have several segments.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_kernel(const ReadOutGradArgs a)
{
    const uint32_t e = blockIdx.x, lo = a.part_first[e], hi = a.part_first[e + 1];
    if (lo == hi) return;
    for (uint32_t col = blockIdx.y * kThreads + threadIdx.x; col < a.D; col += gridDim.y * kThreads) {
        float acc = 0.0f;
        for (uint32_t p = lo; p < hi; ++p) acc += a.parts[(size_t)p * a.part_ld + col];
        static_cast<T*>(a.dvalues)[e * a.ld_dvalues + col] = from_float<T>(acc);
    }
}

// Where the pieces of the workspace lie, and how the sort is cut.
struct SortPlan { uint32_t chunks, per_chunk, part_rows, part_ld; uint64_t counts, total, first, seg_first, part_first, sorted, parts, bytes; };

SortPlan sort_plan(uint32_t N, uint32_t D, uint64_t routes)
{
    SortPlan p{};
    // a warp's walk over its chunk is serial, and every chunk costs a row of N counts: 256 routes each, at most 256 chunks
    p.chunks = (uint32_t)(routes <= 256 ? 1 : routes >= 65536 ? 256 : (routes + 255) / 256);
    p.per_chunk = (uint32_t)((routes + p.chunks - 1) / p.chunks);
    // a neuron with several segments has more than kSegment routes: fewer than 2 * routes / kSegment such segments in all
    p.part_rows = (uint32_t)(2 * routes / kSegment);
    p.part_ld = (D + 3) / 4 * 4;
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) { const uint64_t here = at; at += (bytes + 15) / 16 * 16; return here; };
    p.counts = take((uint64_t)p.chunks * N * 4);
    p.total = take((uint64_t)N * 4);
    p.first = take(((uint64_t)N + 1) * 4);
    p.seg_first = take(((uint64_t)N + 1) * 4);
    p.part_first = take(((uint64_t)N + 1) * 4);
    p.sorted = take(routes * 4);
    p.parts = take((uint64_t)p.part_rows * p.part_ld * 4);
    p.bytes = at;
    return p;
}

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
    const uint32_t rows = kThreads >> a.tx_shift, columns = vec << a.tx_shift;
    const dim3 grid((unsigned)((n + rows - 1) / rows), (dims + columns - 1) / columns);
    return launch_status(with_vector(type, vec, [&](auto t, auto v) {
        read_out_kernel<decltype(t), decltype(v)::value><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
        return cudaGetLastError();
    }), "read-out kernel");
}

uint64_t pink_b200_read_out_workspace(uint32_t n_neurons, uint32_t dims, uint64_t n, uint32_t top_k)
{
    if (n_neurons == 0 || n_neurons > PINK_B200_MAX_ROUTED_NEURONS || dims == 0 || top_k == 0 || top_k > PINK_B200_MAX_ROUTES) return 0;
    if (n == 0 || n > 0x7FFFFFFFull / top_k) return 0;
    return sort_plan(n_neurons, dims, n * top_k).bytes;
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
        const SortPlan p = sort_plan(n_neurons, dims, n * top_k);
        if (!dev_workspace || workspace_bytes < p.bytes) return report_error(PINK_B200_EINVAL, "workspace too small (pink_b200_read_out_workspace)");
        if (reinterpret_cast<uintptr_t>(dev_workspace) % 16) return report_error(PINK_B200_EINVAL, "the workspace must be 16-byte aligned");
        uint8_t* base = static_cast<uint8_t*>(dev_workspace);
        auto at = [&](uint64_t off) { return reinterpret_cast<uint32_t*>(base + off); };
        a.routes = (uint32_t)(n * top_k); a.chunks = p.chunks; a.per_chunk = p.per_chunk;
        a.counts = at(p.counts); a.total = at(p.total); a.first = at(p.first); a.seg_first = at(p.seg_first);
        a.part_first = at(p.part_first); a.sorted = at(p.sorted); a.parts = reinterpret_cast<float*>(base + p.parts); a.part_ld = p.part_ld;
        const size_t smem = n_neurons * sizeof(uint32_t);
        const int rc2 = launch_status([&] {
            cudaError_t e = cudaFuncSetAttribute(count_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
            if (e != cudaSuccess) return e;
            count_kernel<<<a.chunks, 32, smem, st>>>(a);
            column_kernel<<<(n_neurons + kThreads - 1) / kThreads, kThreads, 0, st>>>(a);
            offsets_kernel<<<1, 1024, 0, st>>>(a);
            place_kernel<<<a.chunks, 32, smem, st>>>(a);
            const uint32_t vec = vector_width(type, dims, RowAlign().add(dev_dout, ld_dout, size).add(dev_dvalues, ld_dvalues, size));
            a.tx_shift = log2_threads((dims + vec - 1) / vec);
            const uint32_t columns = vec << a.tx_shift;
            // a segment for every neuron, one more for every kSegment routes
            const dim3 grid(n_neurons + a.routes / kSegment, (dims + columns - 1) / columns);
            e = with_vector(type, vec, [&](auto t, auto v) {
                dvalues_kernel<decltype(t), decltype(v)::value><<<grid, kThreads, 0, st>>>(a);
                return cudaGetLastError();
            });
            if (e != cudaSuccess || p.part_rows < 2) return e;
            return with_type(type, [&](auto t) {
                join_kernel<decltype(t)><<<dim3(n_neurons, dims > 16384 ? 64 : (dims + kThreads - 1) / kThreads), kThreads, 0, st>>>(a);
                return cudaGetLastError();
            });
        }(), "gradient of the values");
        if (rc2) return rc2;
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
