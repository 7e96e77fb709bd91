// Dense product with bias, activation and residual, and its gradient (pink_b200_op_product*).
//
//   z = x W^T + b,  out = act(z) + r;     dz = dout * act'(z),  dx = dz W,  dw = dz^T x,  db = column sums of dz
//
// All three products are D[i][j] = sum_k A[i][k] B[j][k] on the 5th-generation tensor cores (tcgen05.mma kind::f16, float32
// sums in tensor memory).  An operand whose k runs along its rows is staged K-major, one whose k runs across its rows
// MN-major -- W by input, and every operand of dw -- so that nothing is ever transposed in memory.
#include "product.cuh"

namespace pinkb {
namespace {

// One 128 x n_tile tile of D (and one range of K) per block.
template <typename T, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GemmArgs p)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem);
    uint64_t* empty_bar = full_bar + kMaxRing;
    uint64_t* done_bar = empty_bar + kMaxRing;
    uint32_t* tmem_ptr_s = reinterpret_cast<uint32_t*>(done_bar + 1);
    uint8_t* ring = smem + kHeadBytes;
    float* staging = reinterpret_cast<float*>(ring + (size_t)p.ring * p.stage_bytes);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t m0 = blockIdx.x / p.tiles_n * kTileM, n0 = blockIdx.x % p.tiles_n * p.n_tile;
    const uint32_t kb0 = blockIdx.y * p.split_slices, num_kb = min(p.split_slices, p.slices - kb0);
    constexpr uint32_t a_bytes = kTileM * 128;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.ring; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
        mbar_init(done_bar, 1);
        mbar_fence_init();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_b);
    }
    if (warp == 1) { tmem_alloc(tmem_ptr_s, 256); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_ptr_s;
    follow();                            // (nothing above touches global memory)

    if (warp == 0) {
        if (elect_one()) {
            const uint32_t full0 = smem_u32(full_bar), empty0 = smem_u32(empty_bar), ring0 = smem_u32(ring);
            const uint32_t tx = a_bytes + p.n_tile * 128;
            uint32_t s = 0, ph = 0;
            for (uint32_t kb = 0; kb < num_kb; ++kb) {
                if (!mbar_wait(empty0 + 8 * s, ph ^ 1)) { report_timeout(p, kGemmTimeoutProducer); break; }
                const uint32_t bar = full0 + 8 * s, st = ring0 + s * p.stage_bytes;
                const int32_t k = (int32_t)((kb0 + kb) * kSliceK);
                mbar_expect_tx(bar, tx);
                if (A_MN) for (uint32_t c = 0; c < kTileM; c += 64) tma_load_2d(st + c * 128, &map_a, bar, (int32_t)(m0 + c), k);
                else tma_load_2d(st, &map_a, bar, k, (int32_t)m0);
                if (B_MN) for (uint32_t c = 0; c < p.n_tile; c += 64) tma_load_2d(st + a_bytes + c * 128, &map_b, bar, (int32_t)(n0 + c), k);
                else tma_load_2d(st + a_bytes, &map_b, bar, k, (int32_t)n0);
                if (++s == p.ring) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1) {
        if (elect_one()) {
            const uint32_t idesc = gemm_idesc<T, A_MN, B_MN>(kTileM, p.n_tile);
            const uint32_t full0 = smem_u32(full_bar), empty0 = smem_u32(empty_bar), ring0 = smem_u32(ring);
            uint32_t s = 0, ph = 0;
            for (uint32_t kb = 0; kb < num_kb; ++kb) {
                if (!mbar_wait(full0 + 8 * s, ph)) { report_timeout(p, kGemmTimeoutMma); break; }
                tc_fence_after();
                const uint64_t a = operand_desc(ring0 + s * p.stage_bytes, A_MN), b = operand_desc(ring0 + s * p.stage_bytes + a_bytes, B_MN);
#pragma unroll
                for (uint32_t k = 0; k < kSliceK / kStepK; ++k) {
                    // 16 k: 32 bytes inside a K-major row, 16 rows of an MN-major slice
                    const uint64_t da = (A_MN ? kStepK * 128 : kStepK * 2) * k >> 4, db = (B_MN ? kStepK * 128 : kStepK * 2) * k >> 4;
                    umma_f16(tmem_base, a + da, b + db, idesc, (kb | k) != 0);
                }
                umma_commit(empty0 + 8 * s);
                if (++s == p.ring) { s = 0; ph ^= 1; }
            }
            umma_commit(done_bar);
        }
    } else {
        const uint32_t quad = warp & 3;
        if (mbar_wait(done_bar, 0)) {
            tc_fence_after();
            finish_rows<T>(p, p.f, p.parts, tmem_base + ((quad * 32u) << 16), m0 + quad * 32, n0, blockIdx.y, (warp - 2) >> 2, staging + (warp - 2) * 32 * kStagePitch, lane, [] {});
        } else {
            report_timeout(p, kGemmTimeoutFinish);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, 256);
}

// ---- a few rows ------------------------------------------------------------------------------------------------------------
// Up to kFewRows rows of x: every weight is used a few times only, so the pass is bound by reading W.

constexpr uint32_t kFewRows = 8;

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// W by output: a warp per group of outputs, its lanes along k.
template <typename T, int VEC, int ROWS>
__global__ void __launch_bounds__(256) few_rows_kernel(const T* x, uint64_t ld_x, const T* w, uint64_t ld_w, uint32_t K, uint32_t M, const Finish f)
{
    constexpr uint32_t kOut = 2;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t m0 = ((uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * kOut;
    if (m0 >= M) return;
    float acc[kOut][ROWS];
#pragma unroll
    for (uint32_t o = 0; o < kOut; ++o)
#pragma unroll
        for (int i = 0; i < ROWS; ++i) acc[o][i] = 0.0f;
    for (uint64_t k = lane * VEC; k < K; k += 32 * VEC) {
        Pack<T, VEC> wv[kOut];
#pragma unroll
        for (uint32_t o = 0; o < kOut; ++o)
            wv[o] = Pack<T, VEC>::load(w + (m0 + o < M ? m0 + o : m0) * ld_w + k);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            float xf[VEC];
            Pack<T, VEC>::load(x + i * ld_x + k).floats(xf);
#pragma unroll
            for (uint32_t o = 0; o < kOut; ++o) {
                float wf[VEC];
                wv[o].floats(wf);
#pragma unroll
                for (int v = 0; v < VEC; ++v) acc[o][i] = fmaf(xf[v], wf[v], acc[o][i]);
            }
        }
    }
#pragma unroll
    for (uint32_t o = 0; o < kOut; ++o)
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const float s = warp_sum(acc[o][i]);
            if (lane == 0 && m0 + o < M) finish1<T>(f, i, (uint32_t)(m0 + o), s);
        }
}

// Measured, one row, 2791 x 8100 bfloat16, calls that follow one another in a graph with six tables in turn: 11.3 us (4.0 TB/s); by output, in rows
// of 2,784 elements, 11.1 us, of 2,791, read one by one, 21.2 us.
// W by input: lanes along the outputs; the eight warps of a block and the kFewBlocks blocks of a cluster along k.  The warps' sums
// meet in shared memory, the blocks' in distributed shared memory: one launch, no scratch, a fixed order.
constexpr uint32_t kFewBlocks = 8;

template <typename T, int VEC, int ROWS>
__global__ void __launch_bounds__(256, ROWS <= 2 ? 4 : 2) few_rows_by_input_kernel(const T* x, uint64_t ld_x, const T* w, uint64_t ld_w, uint32_t K, uint32_t M, const Finish f)
{
    constexpr uint32_t kCols = 32 * VEC;                 // outputs of the cluster
    constexpr uint32_t kStep = 8 * kFewBlocks;           // rows of W that the cluster takes at a time
    constexpr uint32_t kAhead = ROWS <= 2 ? 8 : 4;       // rows of W that a thread has in flight
    __shared__ float meet[8][kCols];
    __shared__ float sums[ROWS][kCols];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = cluster_ctarank();
    const uint32_t col0 = blockIdx.x / kFewBlocks * kCols, col = col0 + lane * VEC;
    float acc[ROWS][VEC];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[i][v] = 0.0f;
    if (col < M) {
        uint32_t k = rank * 8 + warp;
        const T* wp = w + k * ld_w + col;
        const T* xp = x + k;
        const uint64_t step = kStep * ld_w;
        for (; k + (kAhead - 1) * kStep < K; k += kAhead * kStep, wp += kAhead * step, xp += kAhead * kStep) {
            Pack<T, VEC> wv[kAhead];
            T xv[ROWS][kAhead];
#pragma unroll
            for (uint32_t q = 0; q < kAhead; ++q) wv[q] = Pack<T, VEC>::load(wp + q * step);
#pragma unroll
            for (int i = 0; i < ROWS; ++i)
#pragma unroll
                for (uint32_t q = 0; q < kAhead; ++q) xv[i][q] = xp[i * ld_x + q * kStep];
#pragma unroll
            for (uint32_t q = 0; q < kAhead; ++q) {
                float wf[VEC];
                wv[q].floats(wf);
#pragma unroll
                for (int i = 0; i < ROWS; ++i)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) acc[i][v] = fmaf(to_float(xv[i][q]), wf[v], acc[i][v]);
            }
        }
#pragma unroll 4
        for (; k < K; k += kStep, wp += step, xp += kStep) {
            float wf[VEC];
            Pack<T, VEC>::load(wp).floats(wf);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const float xv = to_float(xp[i * ld_x]);
#pragma unroll
                for (int v = 0; v < VEC; ++v) acc[i][v] = fmaf(xv, wf[v], acc[i][v]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < VEC; ++v) meet[warp][lane * VEC + v] = acc[i][v];
        __syncthreads();
        for (uint32_t c = threadIdx.x; c < kCols; c += 256) {
            float s = 0.0f;
#pragma unroll
            for (int q = 0; q < 8; ++q) s += meet[q][c];
            sums[i][c] = s;
        }
    }
    cluster_sync();
    // each block finishes its share of the outputs
    for (uint32_t t = threadIdx.x + 256 * rank; t < ROWS * kCols; t += 256 * kFewBlocks) {
        const uint32_t i = t / kCols, c = t % kCols;
        if (col0 + c >= M) continue;
        const uint32_t here = smem_u32(&sums[i][c]);
        float s = 0.0f;
#pragma unroll
        for (uint32_t q = 0; q < kFewBlocks; ++q) s += ld_cluster_f32(map_to_cta(here, q));
        finish1<T>(f, i, col0 + c, s);
    }
    cluster_sync();                                      // no block leaves while another reads its sums
}

// ---- gradient of the activation and the bias -------------------------------------------------------------------------------

constexpr uint32_t kDzRows = 32;                         // rows that one block adds up for the bias

// dz = dout * act'(z) enters the products in 16 bits, as the tensor cores want it: half a step of dz each, so that the results are about 1.4 times as
// far from 64 bits as their own rounding takes them (a second word for the remainder would double the products' time).
//
// The range of float16.  bfloat16 holds dz to half a step of its own, 2^-8 of dz,
// but in float16 it may be too large (GELU and SiLU are steeper than 1) or among the subnormals (a sigmoid's slope at z = 8 is 3e-4: with dout =
// 1e-4 an element was off by 78 %).  So dz is multiplied by the power of two that takes the largest finite |dout| to 2^14 .. 2^15 -- no slope
// exceeds 1.13 -- and the sums by its inverse, both exactly; what is 2^-28 of the largest or less still loses digits.  dout is read once
// more for it (4096 x 2791: 6 us of 240), and found in L2 by the pass that follows.  Without an activation dz is dout itself and nothing is rounded.
struct Peak { uint32_t* peaks; float* unscale; uint32_t count; };    // [count] largest finite |dout| of a block's part, as float16 bits

constexpr uint32_t kPeakBlocks = 512, kPeakChunks = 4;   // chunks of eight elements that a lane has in flight

__global__ void __launch_bounds__(256) peak_kernel(const Source m, uint32_t* peaks)
{
    __shared__ uint32_t part[8];
    follow();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // a warp takes 32 * kPeakChunks chunks of a row at a time
    const uint32_t chunks = (m.cols + 7) / 8, pieces = (chunks + 32 * kPeakChunks - 1) / (32 * kPeakChunks);
    const uint64_t items = m.rows * pieces;
    uint32_t most = 0;
    for (uint64_t t = (uint64_t)blockIdx.x * 8 + warp; t < items; t += (uint64_t)gridDim.x * 8) {
        const uint64_t row = t / pieces;
        const uint32_t c0 = (uint32_t)(t - row * pieces) * 32 * kPeakChunks + lane;
        Chunk v[kPeakChunks];
#pragma unroll
        for (uint32_t q = 0; q < kPeakChunks; ++q)
            if (c0 + 32 * q < chunks) v[q] = load_chunk(m, row, (c0 + 32 * q) * 8);
#pragma unroll
        for (uint32_t q = 0; q < kPeakChunks; ++q) {
            if (c0 + 32 * q >= chunks) continue;
            const uint4 j = joined(v[q]);
            const uint32_t w[4] = { j.x, j.y, j.z, j.w };
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = w[i] & 0x7FFFu, hi = w[i] >> 16 & 0x7FFFu;
                if (lo < 0x7C00u) most = max(most, lo);  // (infinities and NaN have no part in it)
                if (hi < 0x7C00u) most = max(most, hi);
            }
        }
    }
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if (lane == 0) part[warp] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) most = max(most, part[w]);
        peaks[blockIdx.x] = most;
    }
}

// The power of two for dz, 1 where dout has nothing but zeros; all threads of a block of 256 call it.
__device__ __forceinline__ float scale_of(const Peak& peak)
{
    __shared__ uint32_t part[8];
    uint32_t most = 0;
    for (uint32_t i = threadIdx.x; i < peak.count; i += 256) most = max(most, peak.peaks[i]);
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) most = max(most, part[w]);
    if (most == 0) return 1.0f;
    const uint32_t exponent = __float_as_uint(__half2float(__ushort_as_half((unsigned short)most))) >> 23;       // 103 .. 142
    return __uint_as_float((127 + 14 + 127 - exponent) << 23);
}

// dz (nullable) in rows a tensor map can describe, and column sums of kDzRows rows of the unrounded dz (nullable).  A block takes
// 256 columns, eight a thread, and its eight warps the rows in turn.
struct DzJob { Source dout, z; uint16_t* dz; uint64_t ld; float* sums; uint32_t act, row_blocks, col_blocks; Peak peak; };

template <typename T>
__device__ __forceinline__ void dz_block(const DzJob& job, uint32_t block, float (&meet)[8][32][9])
{
    float scale = 1.0f;
    if (job.peak.count) {
        scale = scale_of(job.peak);
        if (block == 0 && threadIdx.x == 0) *job.peak.unscale = 1.0f / scale;
    }
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rb = block / job.col_blocks;
    const uint64_t lo = (uint64_t)rb * kDzRows, hi = min(lo + kDzRows, job.dout.rows);
    const uint32_t cols = job.dout.cols;
    T* dz = reinterpret_cast<T*>(job.dz);
    for (uint32_t c0 = block % job.col_blocks * 256; c0 < cols; c0 += job.col_blocks * 256) {
        const uint32_t c = c0 + lane * 8;
        float sum[8] = { 0, 0, 0, 0, 0, 0, 0, 0 };
        if (c < cols) {
            for (uint64_t r = lo + warp; r < hi; r += 8) {
                const Chunk d = load_chunk(job.dout, r, c);
                Chunk b = d;
                if (job.z.p) b = load_chunk(job.z, r, c);
                float g[8], a[8];
                Pack<T, 8>{ joined(d) }.floats(g);
                Pack<T, 8>{ joined(b) }.floats(a);
                if (job.z.p) times_slope(g, a, job.act);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (c + i >= cols) g[i] = 0.0f;
                    sum[i] += g[i];
                }
                if (dz) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) g[i] *= scale;
                    Pack<T, 8>::of(g).store(dz + r * job.ld + c);
                }
            }
        }
        if (job.sums) {
#pragma unroll
            for (int i = 0; i < 8; ++i) meet[warp][lane][i] = sum[i];
            __syncthreads();
            const uint32_t m = threadIdx.x >> 3, i = threadIdx.x & 7;
            float s = 0.0f;
#pragma unroll
            for (int q = 0; q < 8; ++q) s += meet[q][m][i];
            if (c0 + threadIdx.x < cols) job.sums[(size_t)rb * cols + c0 + threadIdx.x] = s;
            __syncthreads();
        }
    }
}

// What the products need first, in one launch: dz (row_blocks 0: none) and up to two copies.  Reading memory for the copies and
// computing slopes for dz then share the SMs (4096 x 2791 and 4096 x 3969, GELU: 72 us in three launches).
template <typename T>
__global__ void __launch_bounds__(256, 3) prepare_kernel(const DzJob dz, const PackJob p0, const PackJob p1)
{
    __shared__ float meet[8][32][9];                     // (nine: no bank conflicts)
    follow();
    uint32_t block = blockIdx.x;
    const uint32_t n_dz = dz.row_blocks * dz.col_blocks, n0 = p0.row_blocks * p0.col_blocks;
    if (block < n_dz) { dz_block<T>(dz, block, meet); return; }
    block -= n_dz;
    if (block < n0) pack_block(p0, block);
    else pack_block(p1, block - n0);
}

// Column sums of the blocks' sums: a block takes 32 columns, its eight warps the row blocks in turn.
__global__ void __launch_bounds__(256) dbias_kernel(const float* sums, uint32_t blocks, uint32_t cols, float* dbias)
{
    __shared__ float meet[8][32];
    follow();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < cols)
#pragma unroll 8
        for (uint32_t b = warp; b < blocks; b += 8) s += sums[(size_t)b * cols + c];
    meet[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < cols) {
#pragma unroll
        for (int q = 1; q < 8; ++q) s += meet[q][lane];
        dbias[c] = s;
    }
}

// ---- tables between float32 and bfloat16 -------------------------------------------------------------------------------------

__global__ void __launch_bounds__(256) widen_kernel(const __nv_bfloat16* src, uint64_t ld, uint64_t rows, uint32_t cols, float* dst)
{
    for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x)
        for (uint32_t c = blockIdx.y * 256 + threadIdx.x; c < cols; c += gridDim.y * 256) dst[r * cols + c] = __bfloat162float(src[r * ld + c]);
}

__global__ void __launch_bounds__(256) narrow_kernel(const float* src, uint64_t rows, uint32_t cols, __nv_bfloat16* dst, uint64_t ld, uint8_t* infinite)
{
    for (uint64_t r = blockIdx.x; r < rows; r += gridDim.x)
        for (uint32_t c = blockIdx.y * 256 + threadIdx.x; c < cols; c += gridDim.y * 256) {
            const __nv_bfloat16 v = __float2bfloat16_rn(src[r * cols + c]);
            dst[r * ld + c] = v;
            if ((__bfloat16_as_ushort(v) & 0x7F80u) == 0x7F80u) infinite[r] = 1;       // (all who write it write the same)
        }
}

__global__ void __launch_bounds__(256) masked_rows_kernel(const uint4* src, const uint8_t* mask, uint32_t rows, uint32_t words, uint4* dst)
{
    for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const bool there = mask[r] != 0;
        for (uint32_t i = blockIdx.y * 256 + threadIdx.x; i < words; i += gridDim.y * 256)
            dst[(size_t)r * words + i] = there ? src[(size_t)r * words + i] : make_uint4(0, 0, 0, 0);
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------

// D = A B^T with A[i][k] and B[j][k]; a_mn / b_mn: the operand's memory has k across its rows.
template <typename T, bool A_MN, bool B_MN>
cudaError_t launch_gemm(const Matrix& a, const Matrix& b, const GemmPlan& p, uint32_t rows, uint32_t cols, float* parts, const Finish& f, int* status, cudaStream_t st)
{
    Maps<kPlain> maps;
    const uint32_t b_rows = p.pair ? p.n_tile / 2 : p.n_tile;
    if (!encode(&maps.a, a, A_MN ? kSliceK : kTileM) || !encode(&maps.b, b, B_MN ? kSliceK : b_rows)) return cudaErrorInvalidValue;
    const GemmArgs g = gemm_args(p, rows, cols, parts, f, status);
    cudaError_t e;
    if (p.pair) {
        e = launch_pairs<T, A_MN, B_MN, kPlain>(maps, p, g, st);
    } else {
        static thread_local int opted_in = -1;
        auto* kernel = gemm_kernel<T, A_MN, B_MN>;
        e = opt_in(kernel, &opted_in);
        if (e != cudaSuccess) return e;
        if (!status) g_used.store(true, std::memory_order_relaxed);
        t_launches += 1;
        e = launch_product(kernel, dim3(p.tiles_m * p.tiles_n, p.splits), 1, 1024 + kHeadBytes + (size_t)p.ring * p.stage_bytes + kStagingBytes, st, maps.a, maps.b, g);
    }
    if (e != cudaSuccess || p.splits == 1) return e;
    t_launches += 1;
    return launch_following(finish_kernel<T>, dim3(rows, std::min((cols + 1023) / 1024, 64u)), 256, 0, st, parts, p.splits, rows, cols, g.part_ld, f);
}

// One product: its plan, the copies of its operands (null: read in place) and its partial sums.
struct Job
{
    Matrix a, b;
    bool a_mn, b_mn;
    uint32_t rows, cols, K;
    Finish f;
    GemmPlan plan;
    uint16_t *pa, *pb;
    float* parts;
};

// (`made`: the operand that is read as it is, because its copy has been decided on already; null: none)
Job plan_job(Arena& ws, const Matrix& a, bool a_mn, const Matrix& b, bool b_mn, uint32_t rows, uint32_t cols, uint32_t K, const Finish& f,
             const Matrix* made = nullptr)
{
    Job j{a, b, a_mn, b_mn, rows, cols, K, f, plan_gemm(rows, cols, K, b_mn), nullptr, nullptr, nullptr};
    if (&a != made && needs_pack(a, j.plan.tiles_n)) j.pa = ws.take<uint16_t>(packed_elements(a));
    if (&b != made && needs_pack(b, j.plan.tiles_m)) j.pb = ws.take<uint16_t>(packed_elements(b));
    if (j.plan.splits > 1) j.parts = ws.take<float>((uint64_t)j.plan.splits * rows * ((cols + 3ull) / 4 * 4));
    return j;
}

template <typename T>
cudaError_t prepare(const DzJob& dz, const PackJob* jobs, cudaStream_t st)
{
    if (dz.peak.count) {
        t_launches += 1;
        const cudaError_t e = launch_following(peak_kernel, dim3(dz.peak.count), 256, 0, st, dz.dout, dz.peak.peaks);
        if (e != cudaSuccess) return e;
    }
    const uint64_t blocks = (uint64_t)dz.row_blocks * dz.col_blocks + (uint64_t)jobs[0].row_blocks * jobs[0].col_blocks
                          + (uint64_t)jobs[1].row_blocks * jobs[1].col_blocks;
    if (blocks == 0) return cudaSuccess;
    if (blocks > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    t_launches += 1;
    return launch_following(prepare_kernel<T>, dim3((unsigned)blocks), 256, 0, st, dz, jobs[0], jobs[1]);
}

template <typename T>
cudaError_t multiply(Job& j, int* status, cudaStream_t st)
{
    j.f.vec4 = vec4_rows(j.f, sizeof(T));
    if (j.a_mn) return launch_gemm<T, true, true>(j.a, j.b, j.plan, j.rows, j.cols, j.parts, j.f, status, st);
    if (j.b_mn) return launch_gemm<T, false, true>(j.a, j.b, j.plan, j.rows, j.cols, j.parts, j.f, status, st);
    return launch_gemm<T, false, false>(j.a, j.b, j.plan, j.rows, j.cols, j.parts, j.f, status, st);
}

uint32_t vector_of(const Matrix& x, const Matrix& w, bool by_input)
{
    RowAlign al;
    al.add(w.p, w.ld, 2);
    if (!by_input) al.add(x.p, x.ld, 2);
    uint32_t v = al.elements(2, 8);
    while (v > 1 && w.cols % v) v >>= 1;
    return v;
}

template <typename T, int VEC, int ROWS>
cudaError_t few_rows(bool launch, const Matrix& x, const Matrix& w, bool by_input, uint32_t K, uint32_t M, const Finish& f, cudaStream_t st)
{
    const T *xp = static_cast<const T*>(x.p), *wp = static_cast<const T*>(w.p);
    t_launches += launch;
    if (!by_input) {
        if (!launch) return cudaSuccess;
        few_rows_kernel<T, VEC, ROWS><<<(M + 15) / 16, 256, 0, st>>>(xp, x.ld, wp, w.ld, K, M, f);
        return cudaGetLastError();
    }
    if (!launch) return cudaSuccess;
    constexpr int V = VEC > 4 ? 4 : VEC;                 // (accumulators: rows x columns of a thread)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((M + 32ull * V - 1) / (32 * V) * kFewBlocks));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kFewBlocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, few_rows_by_input_kernel<T, V, ROWS>, xp, x.ld, wp, w.ld, K, M, f);
}

template <typename T, int VEC>
cudaError_t few_rows_n(uint32_t n, bool launch, const Matrix& x, const Matrix& w, bool by_input, uint32_t K, uint32_t M, const Finish& f, cudaStream_t st)
{
    switch (n) {
        case 1: return few_rows<T, VEC, 1>(launch, x, w, by_input, K, M, f, st);
        case 2: return few_rows<T, VEC, 2>(launch, x, w, by_input, K, M, f, st);
        case 3: return few_rows<T, VEC, 3>(launch, x, w, by_input, K, M, f, st);
        case 4: return few_rows<T, VEC, 4>(launch, x, w, by_input, K, M, f, st);
        case 5: return few_rows<T, VEC, 5>(launch, x, w, by_input, K, M, f, st);
        case 6: return few_rows<T, VEC, 6>(launch, x, w, by_input, K, M, f, st);
        case 7: return few_rows<T, VEC, 7>(launch, x, w, by_input, K, M, f, st);
        default: return few_rows<T, VEC, 8>(launch, x, w, by_input, K, M, f, st);
    }
}

int check_product(const pink_b200_product_config* c, uint64_t ld_x, uint64_t ld_w)
{
    if (!c) return report_error(PINK_B200_EINVAL, "null argument");
    if (c->type != PINK_B200_BF16 && c->type != PINK_B200_F16) return report_error(PINK_B200_EINVAL, "the product takes bfloat16 and float16");
    if (c->inputs == 0 || c->inputs > 0x7FFFFFF0u || c->outputs == 0 || c->outputs > 0x7FFFFFF0u || c->n > 0x7FFFFFF0ull)
        return report_error(PINK_B200_EINVAL, "rows, inputs and outputs must be below 2147483632, inputs and outputs not zero");
    if (c->by_input > 1) return report_error(PINK_B200_EINVAL, "by_input must be 0 or 1");
    if (c->activation > PINK_B200_ACT_SIGMOID) return report_error(PINK_B200_EINVAL, "unknown activation");
    if (c->reserved) return report_error(PINK_B200_EINVAL, "reserved must be 0");
    if (ld_x < c->inputs || ld_w < (c->by_input ? c->outputs : c->inputs))
        return report_error(PINK_B200_EINVAL, "leading dimension smaller than the row");
    if (ld_x >= 1ull << 38 || ld_w >= 1ull << 38) return report_error(PINK_B200_EINVAL, "leading dimension too large");
    // blocks of the products' grids: tiles of 128 rows and at least 16 columns
    auto tiles = [](uint64_t r, uint64_t c2) { return ((r + 127) / 128) * ((c2 + 15) / 16); };
    const uint64_t most = std::max(std::max(tiles(c->n, c->outputs), tiles(c->n, c->inputs)),
                                   std::max(tiles(c->outputs, c->inputs), tiles(c->inputs, c->outputs)));
    if (most > 0x7FFFFFFFull) return report_error(PINK_B200_EINVAL, "product too large");
    return PINK_B200_OK;
}

} // namespace

bool product_used() { return g_used.load(std::memory_order_relaxed); }

uint64_t product_launches() { return t_launches; }

cudaError_t launch_widen_bf16(const void* src, uint64_t ld, uint64_t rows, uint32_t cols, float* dst, cudaStream_t st)
{
    if (rows == 0) return cudaSuccess;
    widen_kernel<<<dim3((unsigned)std::min<uint64_t>(rows, 65536), std::min((cols + 255) / 256, 64u)), 256, 0, st>>>(
        static_cast<const __nv_bfloat16*>(src), ld, rows, cols, dst);
    return cudaGetLastError();
}

cudaError_t launch_narrow_bf16(const float* src, uint64_t rows, uint32_t cols, void* dst, uint64_t ld, uint8_t* infinite, cudaStream_t st)
{
    narrow_kernel<<<dim3((unsigned)std::min<uint64_t>(rows, 65536), std::min((cols + 255) / 256, 64u)), 256, 0, st>>>(
        src, rows, cols, static_cast<__nv_bfloat16*>(dst), ld, infinite);
    return cudaGetLastError();
}

cudaError_t launch_masked_rows(const void* src, const uint8_t* mask, uint32_t rows, uint32_t words, void* dst, cudaStream_t st)
{
    masked_rows_kernel<<<dim3(std::min(rows, 65536u), std::min((words + 255) / 256, 64u)), 256, 0, st>>>(static_cast<const uint4*>(src), mask, rows, words,
                                                                                                    static_cast<uint4*>(dst));
    return cudaGetLastError();
}

int product(const pink_b200_product_config* cfg, const void* dev_x, uint64_t ld_x, const void* dev_w, uint64_t ld_w, const float* dev_bias,
            const void* dev_residual, uint64_t ld_residual, void* dev_out, uint64_t ld_out, void* dev_z, uint64_t ld_z, void* dev_workspace,
            uint64_t* workspace_bytes, uint32_t size_only, int* status, cudaStream_t st)
{
    const int rc = check_product(cfg, ld_x, ld_w);
    if (rc) return rc;
    const uint32_t n = (uint32_t)cfg->n, K = cfg->inputs, M = cfg->outputs;
    if (ld_out < M || (dev_residual && ld_residual < M) || (dev_z && ld_z < M))
        return report_error(PINK_B200_EINVAL, "leading dimension smaller than the row");
    if (n == 0) {
        if (size_only && workspace_bytes) *workspace_bytes = 0;
        return PINK_B200_OK;
    }
    if (!dev_x || !dev_w || !dev_out) return report_error(PINK_B200_EINVAL, "null argument");
    const Matrix x{dev_x, ld_x, n, K};
    const Matrix w{dev_w, ld_w, cfg->by_input ? K : M, cfg->by_input ? M : K};
    Finish f{dev_bias, dev_residual, ld_residual, dev_out, ld_out, dev_z, ld_z, cfg->activation, 0};
    return with_workspace(dev_workspace, workspace_bytes, size_only, "product", [&](Arena& ws, bool launch) {
        return with_half_type(cfg->type, [&](auto t) {
            using T = decltype(t);
            if (n > kFewRows) {
                Job job = plan_job(ws, x, false, w, cfg->by_input != 0, n, M, K, f);
                if (!launch) return cudaSuccess;
                PackJob copies[2] = {};
                uint32_t n_copies = 0;
                take_copy(copies, &n_copies, &job.a, job.pa);
                take_copy(copies, &n_copies, &job.b, job.pb);
                const cudaError_t e = prepare<T>(DzJob{}, copies, st);
                return e != cudaSuccess ? e : multiply<T>(job, status, st);
            }
            f.vec4 = vec4_rows(f, sizeof(T));
            const uint32_t v = vector_of(x, w, cfg->by_input != 0);
            if (v == 8) return few_rows_n<T, 8>(n, launch, x, w, cfg->by_input != 0, K, M, f, st);
            if (v == 4) return few_rows_n<T, 4>(n, launch, x, w, cfg->by_input != 0, K, M, f, st);
            if (v == 2) return few_rows_n<T, 2>(n, launch, x, w, cfg->by_input != 0, K, M, f, st);
            return few_rows_n<T, 1>(n, launch, x, w, cfg->by_input != 0, K, M, f, st);
        });
    });
}

cudaError_t take_product_status(int* out) { return take_status(out); }

} // namespace pinkb

using namespace pinkb;

extern "C" {

int pink_b200_op_product(const pink_b200_product_config* cfg, const void* dev_x, uint64_t ld_x, const void* dev_w, uint64_t ld_w,
                         const float* dev_bias, const void* dev_residual, uint64_t ld_residual, void* dev_out, uint64_t ld_out,
                         void* dev_z, uint64_t ld_z, void* dev_workspace, uint64_t* workspace_bytes, uint32_t size_only, void* stream)
{
    return product(cfg, dev_x, ld_x, dev_w, ld_w, dev_bias, dev_residual, ld_residual, dev_out, ld_out, dev_z, ld_z, dev_workspace, workspace_bytes,
                   size_only, nullptr, static_cast<cudaStream_t>(stream));
}

int pink_b200_op_product_backward(const pink_b200_product_config* cfg, const void* dev_dout, uint64_t ld_dout, const void* dev_x, uint64_t ld_x,
                                  const void* dev_w, uint64_t ld_w, const void* dev_z, uint64_t ld_z, void* dev_dx, uint64_t ld_dx,
                                  void* dev_dw, uint64_t ld_dw, float* dev_dbias, void* dev_workspace, uint64_t* workspace_bytes,
                                  uint32_t size_only, void* stream)
{
    const int rc = check_product(cfg, ld_x, ld_w);
    if (rc) return rc;
    const uint32_t n = (uint32_t)cfg->n, K = cfg->inputs, M = cfg->outputs;
    const bool act = cfg->activation != PINK_B200_ACT_NONE;
    const uint32_t w_cols = cfg->by_input ? M : K;
    const uint64_t w_rows = cfg->by_input ? K : M;
    if (ld_dout < M || (act && ld_z < M) || (dev_dx && ld_dx < K) || (dev_dw && ld_dw < w_cols) || ld_dout >= 1ull << 38)
        return report_error(PINK_B200_EINVAL, "bad leading dimension");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (n == 0) {
        if (size_only) { if (workspace_bytes) *workspace_bytes = 0; return PINK_B200_OK; }
        cudaError_t e = cudaSuccess;
        if (dev_dw) e = cudaMemset2DAsync(dev_dw, ld_dw * 2, 0, (size_t)w_cols * 2, w_rows, st);
        if (e == cudaSuccess && dev_dbias) e = cudaMemsetAsync(dev_dbias, 0, (size_t)M * 4, st);
        return launch_status(e, "clearing the gradients");
    }
    if (!dev_dout || (act && !dev_z) || (dev_dw && !dev_x) || (dev_dx && !dev_w)) return report_error(PINK_B200_EINVAL, "null argument");
    return with_workspace(dev_workspace, workspace_bytes, size_only, "product gradient", [&](Arena& ws, bool launch) {
        return with_half_type(cfg->type, [&](auto t) {
            using T = decltype(t);
            const Matrix x{dev_x, ld_x, n, K}, w{dev_w, ld_w, w_rows, w_cols};
            Matrix dz{dev_dout, ld_dout, n, M};
            const bool products = dev_dx || dev_dw;
            // how often the tiles of the two products read dz: one copy of it serves both
            uint32_t reads = 0;
            if (dev_dx) reads += plan_gemm(n, K, M, !cfg->by_input).tiles_n;
            if (dev_dw) reads += cfg->by_input ? plan_gemm(K, M, n, true).tiles_m : plan_gemm(M, K, n, true).tiles_n;
            const bool make_dz = products && (act || needs_pack(dz, reads));
            const uint32_t blocks = (n + kDzRows - 1) / kDzRows;
            DzJob dzj{};
            if (make_dz || dev_dbias) {
                dzj.dout = Source{static_cast<const uint16_t*>(dev_dout), ld_dout, n, M};
                dzj.z = Source{act ? static_cast<const uint16_t*>(dev_z) : nullptr, ld_z, n, M};
                dzj.dz = make_dz ? ws.take<uint16_t>(packed_elements(dz)) : nullptr;
                dzj.sums = dev_dbias ? ws.take<float>((uint64_t)blocks * M) : nullptr;
                dzj.ld = packed_ld(M);
                dzj.act = cfg->activation;
                dzj.row_blocks = blocks;
                dzj.col_blocks = std::min((M + 255) / 256, 4096u);
                if (make_dz) { dz.p = dzj.dz; dz.ld = dzj.ld; }
            }
            if (make_dz && act && cfg->type == PINK_B200_F16) {
                const uint64_t pieces = (uint64_t)n * ((M + 255ull) / 256);          // (at least as many as peak_kernel's warps find)
                dzj.peak.count = (uint32_t)std::min<uint64_t>(kPeakBlocks, (pieces + 7) / 8);
                dzj.peak.peaks = ws.take<uint32_t>(kPeakBlocks);
                dzj.peak.unscale = ws.take<float>(1);
            }
            Finish fx{}, fw{};
            fx.unscale = fw.unscale = dzj.peak.unscale;
            fx.out = dev_dx; fx.ld_out = ld_dx;
            fw.out = dev_dw; fw.ld_out = ld_dw;
            Job jx{}, jw{};
            if (dev_dx) jx = plan_job(ws, dz, false, w, !cfg->by_input, n, K, M, fx, &dz);
            if (dev_dw) jw = cfg->by_input ? plan_job(ws, x, true, dz, true, K, M, n, fw, &dz) : plan_job(ws, dz, true, x, true, M, K, n, fw, &dz);
            if (!launch) return cudaSuccess;
            PackJob copies[2] = {};
            uint32_t n_copies = 0;
            if (dev_dx) take_copy(copies, &n_copies, &jx.b, jx.pb);
            if (dev_dw) take_copy(copies, &n_copies, cfg->by_input ? &jw.a : &jw.b, cfg->by_input ? jw.pa : jw.pb);
            cudaError_t e = prepare<T>(dzj, copies, st);
            if (e == cudaSuccess && dev_dx) e = multiply<T>(jx, nullptr, st);
            if (e == cudaSuccess && dev_dw) e = multiply<T>(jw, nullptr, st);
            if (e == cudaSuccess && dev_dbias) {
                t_launches += 1;
                e = launch_following(dbias_kernel, (M + 31) / 32, 256, 0, st, dzj.sums, blocks, M, dev_dbias);
            }
            return e;
        });
    });
}

} // extern "C"
