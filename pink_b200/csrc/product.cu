// Dense product with bias, activation and residual, and its gradient (pink_b200_op_product*).
//
//   z = x W^T + b,  out = act(z) + r;     dz = dout * act'(z),  dx = dz W,  dw = dz^T x,  db = column sums of dz
//
// All three products are D[i][j] = sum_k A[i][k] B[j][k] on the 5th-generation tensor cores (tcgen05.mma kind::f16, float32
// sums in tensor memory).  An operand whose k runs along its rows is staged K-major, one whose k runs across its rows
// MN-major -- W by input, and every operand of dw -- so that nothing is ever transposed in memory.
#include "ptx.cuh"
#include "readout.cuh"
#include "tensormap.cuh"

#include <algorithm>
#include <atomic>

namespace pinkb {
namespace {

// ---- element-wise pieces ---------------------------------------------------------------------------------------------------

// Results of these are rounded to 16 bits (11 significant ones at most), so the fast exponential and reciprocal -- a few units of
// 2^-24, and |z| of them in the exponential -- lose nothing that shows.  With expf and a full division the finishing warps of
// 8192 x 2791 x 8100 (sigmoid) took longer than the products.
__device__ __forceinline__ float sigmoid_f(float z)
{
    const float e = __expf(-fabsf(z));                   // never overflows
    return __fdividef(z >= 0.0f ? 1.0f : e, 1.0f + e);
}

// Phi(z), and e^(-z^2 / 2).  Phi(-|z|) = erfcx(|z| / sqrt 2) e^(-z^2 / 2) / 2, where erfcx(x) = e^(x^2) erfc(x) is smooth: a polynomial in
// 1 / (1 + 0.6 x), fitted for the smallest relative error over 0 <= x <= 12 (5e-7 as evaluated in float32); beyond, the exponential is zero.
__device__ __forceinline__ float normal_cdf(float z, float* gauss)
{
    const float x = fabsf(z) * 0.70710678f, e = __expf(-0.5f * z * z), t = __fdividef(1.0f, fmaf(0.6f, x, 1.0f));
    float p = -0.09208938f;
    p = fmaf(p, t, 0.41197607f);
    p = fmaf(p, t, -0.6445099f);
    p = fmaf(p, t, 0.28382227f);
    p = fmaf(p, t, 0.073382594f);
    p = fmaf(p, t, 0.29161027f);
    p = fmaf(p, t, 0.33724764f);
    p = fmaf(p, t, 0.33856016f);
    const float tail = 0.5f * e * (p * t);
    *gauss = e;
    return z < 0.0f ? tail : 1.0f - tail;
}

__device__ __forceinline__ float activate(float z, uint32_t act)
{
    float gauss;
    switch (act) {
        case PINK_B200_ACT_RELU: return z > 0.0f || z != z ? z : 0.0f;
        case PINK_B200_ACT_GELU: return z * normal_cdf(z, &gauss);
        case PINK_B200_ACT_SILU: return z * sigmoid_f(z);
        case PINK_B200_ACT_SIGMOID: return sigmoid_f(z);
        default: return z;
    }
}

template <int ROWS>
__device__ __forceinline__ void activate_all(float (&y)[ROWS][4], uint32_t act)
{
    auto each = [&](auto fn) {
#pragma unroll
        for (int q = 0; q < ROWS; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) y[q][i] = fn(y[q][i]);
    };
    if (act == PINK_B200_ACT_SIGMOID) each([](float z) { return sigmoid_f(z); });
    else if (act == PINK_B200_ACT_SILU) each([](float z) { return z * sigmoid_f(z); });
    else if (act == PINK_B200_ACT_GELU) each([](float z) { float gauss; return z * normal_cdf(z, &gauss); });
    else if (act == PINK_B200_ACT_RELU) each([](float z) { return z > 0.0f || z != z ? z : 0.0f; });
}

// z as a factor beside an exponential that is zero far out: an infinity counts as the largest float, so that the slope there is its limit
// and not infinity times zero (a float16 z below -65,504 is kept as -infinity, while SiLU and GELU are finite).  A NaN is in the other factor too.
__device__ __forceinline__ float finite_factor(float z) { return fminf(fmaxf(z, -FLT_MAX), FLT_MAX); }

// g times the slope of the activation at z, for eight elements whose instructions do not wait for one another.
__device__ __forceinline__ void times_slope(float (&g)[8], const float (&z)[8], uint32_t act)
{
    auto each = [&](auto slope) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= slope(z[i]);
    };
    if (act == PINK_B200_ACT_RELU) each([](float z) { return z > 0.0f ? 1.0f : 0.0f; });
    else if (act == PINK_B200_ACT_GELU) each([](float z) { float gauss; const float c = normal_cdf(z, &gauss); return fmaf(finite_factor(z) * 0.39894228f, gauss, c); });
    else if (act == PINK_B200_ACT_SILU) each([](float z) { const float s = sigmoid_f(z); return fmaf(finite_factor(z) * s, sigmoid_f(-z), s); });
    else if (act == PINK_B200_ACT_SIGMOID) each([](float z) { return sigmoid_f(z) * sigmoid_f(-z); });
}

// What follows the sums: out = act(sum + bias) + residual, z = sum + bias (nullable).
struct Finish
{
    const float* bias;
    const void* residual; uint64_t ld_residual;
    void* out; uint64_t ld_out;
    void* z; uint64_t ld_z;
    uint32_t act;
    uint32_t vec4;                   // rows of residual, out and z may be accessed four elements at a time
    const float* unscale;            // not null: the sums are multiplied by this power of two first (see Peak)
};

template <typename T>
__device__ __forceinline__ void finish1(const Finish& f, uint64_t row, uint32_t col, float sum, float by = 1.0f)
{
    sum = fmaf(sum, by, f.bias ? f.bias[col] : 0.0f);
    if (f.z) static_cast<T*>(f.z)[row * f.ld_z + col] = from_float<T>(sum);
    float y = activate(sum, f.act);
    if (f.residual) y += to_float(static_cast<const T*>(f.residual)[row * f.ld_residual + col]);
    static_cast<T*>(f.out)[row * f.ld_out + col] = from_float<T>(y);
}

template <typename T>
__device__ __forceinline__ void finish4(const Finish& f, uint64_t row, uint32_t col, float4 s, float by)
{
    float v[4] = { s.x * by, s.y * by, s.z * by, s.w * by };
    if (f.bias)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += f.bias[col + i];
    if (f.z) Pack<T, 4>::of(v).store(static_cast<T*>(f.z) + row * f.ld_z + col);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = activate(v[i], f.act);
    if (f.residual) {
        float r[4];
        Pack<T, 4>::load(static_cast<const T*>(f.residual) + row * f.ld_residual + col).floats(r);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += r[i];
    }
    Pack<T, 4>::of(v).store(static_cast<T*>(f.out) + row * f.ld_out + col);
}

// ---- tensor-core product ---------------------------------------------------------------------------------------------------

constexpr uint32_t kTileM = 128;                         // rows of D per block = TMEM lanes
constexpr uint32_t kSliceK = 64;                         // k per pipeline stage: 128 bytes of a 16-bit type
constexpr uint32_t kStepK = 16;                          // k per instruction
constexpr uint32_t kFinishWarps = 8;                     // two for every 32 rows, which take the columns in turn
constexpr uint32_t kGemmThreads = 64 + 32 * kFinishWarps;    // warp 0 loads, warp 1 multiplies, the others finish
constexpr uint32_t kMaxRing = 8;
constexpr uint32_t kStagePitch = 36;                     // floats per staged row of 32 columns: 16-byte rows without bank conflicts
constexpr uint32_t kHeadBytes = 1024;                    // barriers and the tensor-memory address
constexpr uint32_t kStagingBytes = kFinishWarps * 32 * kStagePitch * 4;

enum : int { kGemmTimeoutProducer = 31, kGemmTimeoutMma = 32, kGemmTimeoutFinish = 33 };

__device__ int g_status;                                 // code of the first bounded wait that expired in a call of the public entries
std::atomic<bool> g_used{false};
thread_local uint64_t t_launches = 0;

struct GemmArgs
{
    uint32_t rows, cols;                                 // of D
    uint32_t tiles_m, tiles_n, n_tile;                   // row tiles (of 256 for pairs); column tiles of n_tile (a multiple of 16, of 32 for pairs, at most 256)
    uint32_t slices, split_slices, splits;               // K slices in all and per range, and ranges
    uint32_t ring, stage_bytes;
    float* parts; uint32_t part_ld;                      // not null: raw sums of this K range go to parts[blockIdx.y][rows][part_ld]
    Finish f;
    int* status;                                         // receives the code of a wait that expired; null: g_status
};

__device__ __forceinline__ uint64_t operand_desc(uint32_t smem_addr, bool mn_major)
{
    // MN-major: rows of 64 elements along m or n, 128-byte swizzle; eight k are 1024 bytes (stride byte offset), the next 64
    // along m or n follow after all k of the slice (leading byte offset)
    uint64_t d = make_sw128_kmajor_desc(smem_addr);
    if (mn_major) d |= (uint64_t)(kSliceK * 128u >> 4) << 16;
    return d;
}

template <typename T> __host__ __device__ constexpr uint32_t format_code() { return std::is_same<T, __nv_bfloat16>::value ? 1u : 0u; }

template <typename T, bool A_MN, bool B_MN>
__host__ __device__ constexpr uint32_t gemm_idesc(uint32_t m, uint32_t n)
{
    return (1u << 4)                                     // float32 accumulator
         | (format_code<T>() << 7) | (format_code<T>() << 10)
         | ((A_MN ? 1u : 0u) << 15) | ((B_MN ? 1u : 0u) << 16)
         | ((n >> 3) << 17) | ((m >> 4) << 24);
}

__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n"
        :: "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void report_timeout(const GemmArgs& p, int code) { atomicCAS(p.status ? p.status : &g_status, 0, code); }

// Finishes 32 rows (a warp's TMEM lanes) of a tile: `taddr` their first column, `row0` and `col0` their place in D.  The sums pass
// through shared memory, 32 columns at a time, so that the lanes run along the columns of a row; the next columns leave tensor
// memory, and the residual arrives, while the current ones are finished.  Two warps (turn 0 and 1) share the columns.  drained() is
// called when this warp has read its part of the accumulator.
template <typename T, typename Drained>
__device__ __forceinline__ void finish_rows(const GemmArgs& p, uint32_t taddr, uint32_t row0, uint32_t col0, uint32_t split, uint32_t turn,
                                            float* st, uint32_t lane, Drained drained)
{
    const Finish& f = p.f;
    const uint32_t ncols = min(p.n_tile, p.cols - col0);
    const uint32_t nrows = row0 < p.rows ? min(32u, p.rows - row0) : 0u;
    uint32_t v[32];
    const uint32_t cq = (lane & 7) * 4, rq = lane >> 3;  // four columns a lane, four rows at a time
    const float by = f.unscale ? *f.unscale : 1.0f;
    const uint32_t first = 32 * turn;
    if (first < ncols) tmem_ld_32x32(taddr + first, v);
    else drained();
    for (uint32_t c0 = first; c0 < ncols; c0 += 64) {
        const uint32_t left = min(32u, ncols - c0), col = col0 + c0;
        const bool whole = f.vec4 && !p.parts && cq + 4 <= left;
        Pack<T, 4> res[8];
        float bias[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
        if (whole && f.residual) {
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q)
                if (rq + 4 * q < nrows)
                    res[q] = Pack<T, 4>::load(static_cast<const T*>(f.residual) + (uint64_t)(row0 + rq + 4 * q) * f.ld_residual + col + cq);
        }
        if (whole && f.bias)
#pragma unroll
            for (int i = 0; i < 4; ++i) bias[i] = f.bias[col + cq + i];
        tmem_ld_wait_on(v);
        __syncwarp();                                    // the staged columns before these have been read
#pragma unroll
        for (uint32_t q = 0; q < 32; q += 4)
            *reinterpret_cast<uint4*>(st + lane * kStagePitch + q) = make_uint4(v[q], v[q + 1], v[q + 2], v[q + 3]);
        __syncwarp();
        if (c0 + 64 < ncols) tmem_ld_32x32(taddr + c0 + 64, v);      // (a last read may pass n_tile, inside this accumulator's 256 columns)
        else drained();
        if (p.parts) {
            float* dst = p.parts + ((size_t)split * p.rows + row0) * p.part_ld + col + lane;
            if (lane < left) for (uint32_t r = 0; r < nrows; ++r) dst[(size_t)r * p.part_ld] = st[r * kStagePitch + lane];
        } else if (whole) {
            // step by step over all 32 values of the lane: each step's instructions do not wait for one another
            float y[8][4];
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q) {
                const float4 s = *reinterpret_cast<const float4*>(st + (rq + 4 * q) * kStagePitch + cq);
                y[q][0] = fmaf(s.x, by, bias[0]); y[q][1] = fmaf(s.y, by, bias[1]); y[q][2] = fmaf(s.z, by, bias[2]); y[q][3] = fmaf(s.w, by, bias[3]);
            }
            if (f.z) {
                T* dst = static_cast<T*>(f.z) + (uint64_t)(row0 + rq) * f.ld_z + col + cq;
#pragma unroll
                for (uint32_t q = 0; q < 8; ++q)
                    if (rq + 4 * q < nrows) Pack<T, 4>::of(y[q]).store(dst + 4 * q * f.ld_z);
            }
            activate_all(y, f.act);
            if (f.residual)
#pragma unroll
                for (uint32_t q = 0; q < 8; ++q) {
                    float add[4];
                    res[q].floats(add);
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[q][i] += add[i];
                }
            T* dst = static_cast<T*>(f.out) + (uint64_t)(row0 + rq) * f.ld_out + col + cq;
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q)
                if (rq + 4 * q < nrows) Pack<T, 4>::of(y[q]).store(dst + 4 * q * f.ld_out);
        } else if (f.vec4) {
            for (uint32_t r = rq; r < nrows; r += 4) {   // the last columns of a row
                const float* s = st + r * kStagePitch + cq;
                for (uint32_t i = 0; i < 3; ++i)
                    if (cq + i < left) finish1<T>(f, row0 + r, col + cq + i, s[i], by);
            }
        } else if (lane < left) {
            // rows at any pitch: a lane per column
            if (!f.bias && !f.z && !f.residual && f.act == PINK_B200_ACT_NONE) {
                T* dst = static_cast<T*>(f.out) + (uint64_t)row0 * f.ld_out + col + lane;
#pragma unroll 8
                for (uint32_t r = 0; r < nrows; ++r) dst[r * f.ld_out] = from_float<T>(st[r * kStagePitch + lane] * by);
            } else {
#pragma unroll 4
                for (uint32_t r = 0; r < nrows; ++r) finish1<T>(f, row0 + r, col + lane, st[r * kStagePitch + lane], by);
            }
        }
        __syncwarp();                                    // (the lanes of a ragged end took different ways)
    }
}

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
            finish_rows<T>(p, tmem_base + ((quad * 32u) << 16), m0 + quad * 32, n0, blockIdx.y, (warp - 2) >> 2, staging + (warp - 2) * 32 * kStagePitch, lane, [] {});
        } else {
            report_timeout(p, kGemmTimeoutFinish);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, 256);
}

__device__ __forceinline__ void umma_f16_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n"
        :: "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// Work item of the persistent kernel: a 256 x n_tile tile of D and a range of K.  Items run through kGroupM row tiles before
// they move to the next column tile, so that those in flight share operand rows in L2.
constexpr uint32_t kGroupM = 8;
struct Item { uint32_t m, n, split; };
__device__ __forceinline__ Item item_at(const GemmArgs& p, uint32_t t)
{
    const uint32_t per_split = p.tiles_m * p.tiles_n, split = t / per_split;
    t -= split * per_split;
    const uint32_t strip = t / (kGroupM * p.tiles_n), height = min(kGroupM, p.tiles_m - strip * kGroupM);
    t -= strip * kGroupM * p.tiles_n;
    return { strip * kGroupM + t % height, t / height, split };
}

// Pairs of blocks (cta_group::2) that stay resident and work through tiles of 256 x n_tile: each block stages its 128 rows of A and
// half of the tile's rows of B.  Two accumulators of 256 columns: one is finished while the next tile is multiplied.
// Measured, 8192 x 2791 x 8100 with sigmoid, residual and kept z: 254 us (1.46 PFLOP/s, tensor pipe active 85 %); a block a tile of
// 128 x 256 that finished it before the next began: 1209 us.
template <typename T, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const GemmArgs p)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem);          // [kMaxRing] in the even block: a slice of both blocks has arrived
    uint64_t* empty_bar = full_bar + kMaxRing;                       // [kMaxRing] this block's slice has been read
    uint64_t* done_bar = empty_bar + kMaxRing;                       // [2] an accumulator is complete
    uint64_t* free_bar = done_bar + 2;                               // [2] in the even block: both blocks have read an accumulator
    uint32_t* tmem_ptr_s = reinterpret_cast<uint32_t*>(free_bar + 2);
    uint8_t* ring = smem + kHeadBytes;
    float* staging = reinterpret_cast<float*>(ring + (size_t)p.ring * p.stage_bytes);

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t items = p.tiles_m * p.tiles_n * p.splits;
    const uint32_t half = p.n_tile / 2;
    constexpr uint32_t a_bytes = kTileM * 128;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.ring; ++s) { mbar_init(&full_bar[s], 2); mbar_init(&empty_bar[s], 1); }
        for (uint32_t b = 0; b < 2; ++b) { mbar_init(&done_bar[b], 1); mbar_init(&free_bar[b], 2 * kFinishWarps); }
        mbar_fence_init();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_b);
    }
    if (warp == 1) { tmem_alloc_pair(tmem_ptr_s, 512); tmem_relinquish_pair(); }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_ptr_s;
    follow();                            // (nothing above touches global memory)

    if (warp == 0) {
        if (elect_one()) {
            const uint32_t full0 = map_to_cta(smem_u32(full_bar), 0), empty0 = smem_u32(empty_bar), ring0 = smem_u32(ring);
            const uint32_t b_boxes = (half + 63) / 64;               // MN-major: rows of 64; the last may be partly another's
            const uint32_t tx = a_bytes + (B_MN ? b_boxes * kSliceK * 128 : half * 128);
            uint32_t s = 0, ph = 0, st = ring0;
            bool ok = true;
            for (uint32_t t = pair; t < items && ok; t += pairs) {
                const Item it = item_at(p, t);
                const int32_t m0 = (int32_t)((it.m * 2 + rank) * kTileM), n0 = (int32_t)(it.n * p.n_tile + rank * half);
                const uint32_t kb0 = it.split * p.split_slices, num_kb = min(p.split_slices, p.slices - kb0);
                int32_t k = (int32_t)(kb0 * kSliceK);
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait(empty0 + 8 * s, ph ^ 1)) { report_timeout(p, kGemmTimeoutProducer); ok = false; break; }
                    const uint32_t bar = full0 + 8 * s;
                    mbar_expect_tx_cluster(bar, tx);
                    if (A_MN) { tma_load_2d_pair(st, &map_a, bar, m0, k); tma_load_2d_pair(st + kSliceK * 128, &map_a, bar, m0 + 64, k); }
                    else tma_load_2d_pair(st, &map_a, bar, k, m0);
                    if (B_MN) for (uint32_t c = 0; c < b_boxes; ++c) tma_load_2d_pair(st + a_bytes + c * kSliceK * 128, &map_b, bar, n0 + (int32_t)(c * 64), k);
                    else tma_load_2d_pair(st + a_bytes, &map_b, bar, k, n0);
                    k += (int32_t)kSliceK;
                    st += p.stage_bytes;
                    if (++s == p.ring) { s = 0; ph ^= 1; st = ring0; }
                }
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            const uint32_t idesc = gemm_idesc<T, A_MN, B_MN>(2 * kTileM, p.n_tile);
            const uint32_t full0 = smem_u32(full_bar), ring0 = smem_u32(ring);
            const uint32_t empty0 = smem_u32(empty_bar), empty1 = map_to_cta(empty0, 1);
            const uint32_t done0 = smem_u32(done_bar), done1 = map_to_cta(done0, 1), free0 = smem_u32(free_bar);
            const uint64_t a0 = operand_desc(ring0, A_MN), b0 = operand_desc(ring0 + a_bytes, B_MN);
            uint32_t s = 0, ph = 0, off = 0, n_item = 0;
            bool ok = true;
            for (uint32_t t = pair; t < items && ok; t += pairs, ++n_item) {
                const uint32_t buf = n_item & 1, use = n_item >> 1;
                const uint32_t kb0 = item_at(p, t).split * p.split_slices, num_kb = min(p.split_slices, p.slices - kb0);
                if (!mbar_wait(free0 + 8 * buf, (use & 1) ^ 1)) { report_timeout(p, kGemmTimeoutMma); break; }
                tc_fence_after();
                const uint32_t d = tmem_base + buf * 256;
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait(full0 + 8 * s, ph)) { report_timeout(p, kGemmTimeoutMma); ok = false; break; }
                    tc_fence_after();
#pragma unroll
                    for (uint32_t k = 0; k < kSliceK / kStepK; ++k) {
                        const uint64_t da = (A_MN ? kStepK * 128 : kStepK * 2) * k >> 4, db = (B_MN ? kStepK * 128 : kStepK * 2) * k >> 4;
                        umma_f16_pair(d, a0 + off + da, b0 + off + db, idesc, (kb | k) != 0);
                    }
                    umma_commit_pair(empty0 + 8 * s);
                    umma_commit_pair(empty1 + 8 * s);
                    off += p.stage_bytes >> 4;
                    if (++s == p.ring) { s = 0; ph ^= 1; off = 0; }
                }
                umma_commit_pair(done0 + 8 * buf);
                umma_commit_pair(done1 + 8 * buf);
            }
        }
    } else {
        const uint32_t quad = warp & 3, free0 = map_to_cta(smem_u32(free_bar), 0);
        float* st = staging + (warp - 2) * 32 * kStagePitch;
        uint32_t n_item = 0;
        for (uint32_t t = pair; t < items; t += pairs, ++n_item) {
            const Item it = item_at(p, t);
            const uint32_t buf = n_item & 1, use = n_item >> 1;
            if (!mbar_wait(&done_bar[buf], use & 1)) { report_timeout(p, kGemmTimeoutFinish); break; }
            tc_fence_after();
            finish_rows<T>(p, tmem_base + buf * 256 + ((quad * 32u) << 16), (it.m * 2 + rank) * kTileM + quad * 32, it.n * p.n_tile, it.split, (warp - 2) >> 2, st, lane, [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(free0 + 8 * buf);
            });
        }
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();                      // neither block leaves while the other may still signal or read it
    if (warp == 1) tmem_dealloc_pair(tmem_base, 512);
}

// Sum of the K ranges' partial sums, in order, and what follows it.
template <typename T>
__global__ void __launch_bounds__(256) finish_kernel(const float* parts, uint32_t splits, uint32_t rows, uint32_t cols, uint32_t part_ld, const Finish f)
{
    follow();
    const uint64_t row = blockIdx.x;
    const size_t step = (size_t)rows * part_ld;
    const float by = f.unscale ? *f.unscale : 1.0f;
    for (uint32_t c = (blockIdx.y * 256 + threadIdx.x) * 4; c < cols; c += gridDim.y * 1024) {
        const float4* src = reinterpret_cast<const float4*>(parts + row * part_ld + c);
        float4 s = make_float4(0, 0, 0, 0);
#pragma unroll 4
        for (uint32_t k = 0; k < splits; ++k) {
            const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + k * step);
            s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
        }
        if (f.vec4 && c + 4 <= cols) finish4<T>(f, row, c, s, by);
        else {
            finish1<T>(f, row, c, s.x, by);
            if (c + 1 < cols) finish1<T>(f, row, c + 1, s.y, by);
            if (c + 2 < cols) finish1<T>(f, row, c + 2, s.z, by);
            if (c + 3 < cols) finish1<T>(f, row, c + 3, s.w, by);
        }
    }
}

using Source = Rows<uint16_t>;

constexpr uint32_t kPackRows = 4;                        // rows a thread copies: loads in flight

// Copy of a matrix with rows of any alignment into rows a tensor map can describe (at 2791 x 8100: 45 MB in, 45 MB out).
struct PackJob { Source m; uint16_t* dst; uint64_t ld; uint32_t row_blocks, col_blocks; };

__device__ __forceinline__ void pack_block(const PackJob& job, uint32_t block)
{
    const Source& m = job.m;
    const uint32_t chunks = (m.cols + 7) / 8;
    const uint64_t row0 = ((uint64_t)(block / job.col_blocks) * 8 + (threadIdx.x >> 5)) * kPackRows;
    for (uint32_t c = block % job.col_blocks * 32 + (threadIdx.x & 31); c < chunks; c += job.col_blocks * 32) {
        Chunk v[kPackRows];
#pragma unroll
        for (uint32_t r = 0; r < kPackRows; ++r)
            if (row0 + r < m.rows) v[r] = load_chunk(m, row0 + r, c * 8);
#pragma unroll
        for (uint32_t r = 0; r < kPackRows; ++r)
            if (row0 + r < m.rows) *reinterpret_cast<uint4*>(job.dst + (row0 + r) * job.ld + c * 8) = joined(v[r]);
    }
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

// A matrix in memory: `rows` rows of `cols` contiguous elements.
struct Matrix { const void* p; uint64_t ld, rows; uint32_t cols; };

bool mappable(const Matrix& m) { return reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.ld % 8 == 0; }

// Hands out pieces of the workspace; without one it only counts.
struct Arena
{
    uint8_t* base; uint64_t used = 0;
    template <typename P> P* take(uint64_t count)
    {
        uint8_t* here = base ? base + used : nullptr;
        used += (count * sizeof(P) + 255) / 256 * 256;
        return reinterpret_cast<P*>(here);
    }
};

bool encode(CUtensorMap* map, const Matrix& m, uint32_t box_rows)
{
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = { m.cols, m.rows };
    cuuint64_t strides[1] = { m.ld * 2 };
    cuuint32_t box[2] = { kSliceK, box_rows };
    cuuint32_t estr[2] = { 1, 1 };
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(m.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count()
{
    static thread_local int known_dev = -1, sms = 0;
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev != known_dev) { cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev); known_dev = dev; }
    return sms > 0 ? sms : 148;
}

struct GemmPlan { bool pair; uint32_t n_tile, tiles_m, tiles_n, slices, split_slices, splits, ring, stage_bytes; };

constexpr uint32_t kSmemBudget = 226u * 1024;

GemmPlan plan_gemm(uint32_t rows, uint32_t cols, uint32_t K, bool b_mn)
{
    GemmPlan p{};
    const uint32_t sms = (uint32_t)sm_count();
    p.slices = (K + kSliceK - 1) / kSliceK;
    p.pair = rows > kTileM;
    if (p.pair) {
        p.tiles_m = (rows + 2 * kTileM - 1) / (2 * kTileM);
        // the tile width whose waves over the pairs take least: a slice costs what an SM loads for it, 128 rows of A and half the
        // tile's of B (2791 x 3969 x 4096: 90 us with 160 columns, which multiplying alone would choose)
        uint64_t best = ~0ull;
        for (uint32_t w = 256; w >= 64; w -= 32) {
            const uint64_t tiles = (uint64_t)p.tiles_m * ((cols + w - 1) / w), waves = (tiles + sms / 2 - 1) / (sms / 2);
            const uint64_t cost = waves * (kTileM + w / 2);
            if (cost < best) { best = cost; p.n_tile = w; }
        }
        p.n_tile = std::min(p.n_tile, (cols + 31) / 32 * 32);
    } else {
        p.tiles_m = (rows + kTileM - 1) / kTileM;
        const uint32_t grain = b_mn ? 64 : 16;           // an MN-major tile is made of 64-element rows
        p.n_tile = std::min(256u, (cols + grain - 1) / grain * grain);
        while (p.n_tile > 64 && (uint64_t)p.tiles_m * ((cols + p.n_tile - 1) / p.n_tile) < (uint64_t)sms) p.n_tile = (p.n_tile / 2 + grain - 1) / grain * grain;
    }
    p.tiles_n = (cols + p.n_tile - 1) / p.n_tile;
    // fewer tiles than SMs (pairs of them): split K, into ranges of four slices at least
    const uint64_t tiles = (uint64_t)p.tiles_m * p.tiles_n;
    const uint32_t splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((p.pair ? sms / 2 : sms) / tiles, p.slices / 4));
    p.split_slices = (p.slices + splits - 1) / splits;
    p.splits = (p.slices + p.split_slices - 1) / p.split_slices;
    const uint32_t b_rows = p.pair ? p.n_tile / 2 : p.n_tile;
    p.stage_bytes = kTileM * 128 + (b_mn ? (b_rows + 63) / 64 * kSliceK * 128 : (b_rows * 128 + 1023) / 1024 * 1024);
    p.ring = std::min(kMaxRing, (kSmemBudget - 1024 - kHeadBytes - kStagingBytes) / p.stage_bytes);
    if (!p.pair) p.ring = std::min(p.ring, std::max(2u, p.split_slices));
    return p;
}

// D = A B^T with A[i][k] and B[j][k]; a_mn / b_mn: the operand's memory has k across its rows.
template <typename T, bool A_MN, bool B_MN>
cudaError_t launch_gemm(const Matrix& a, const Matrix& b, const GemmPlan& p, uint32_t rows, uint32_t cols, float* parts, const Finish& f, int* status, cudaStream_t st)
{
    CUtensorMap ma, mb;
    const uint32_t b_rows = p.pair ? p.n_tile / 2 : p.n_tile;
    if (!encode(&ma, a, A_MN ? kSliceK : kTileM) || !encode(&mb, b, B_MN ? kSliceK : b_rows)) return cudaErrorInvalidValue;
    auto* kernel = p.pair ? gemm_pair_kernel<T, A_MN, B_MN> : gemm_kernel<T, A_MN, B_MN>;
    // (A pair takes all of its SMs' shared memory that matters: no other kernel's pair, which would wait for the same tensor
    // memory in the other order, fits beside it.)
    const size_t smem = p.pair ? kSmemBudget : 1024 + kHeadBytes + (size_t)p.ring * p.stage_bytes + kStagingBytes;
    static thread_local int opted_in[2] = { -1, -1 };    // device of the last opt-in to large shared memory, per kernel
    int dev = 0;
    cudaGetDevice(&dev);
    cudaError_t e = cudaSuccess;
    if (opted_in[p.pair] != dev) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBudget);
        if (e != cudaSuccess) return e;
        opted_in[p.pair] = dev;
    }
    const GemmArgs g{rows, cols, p.tiles_m, p.tiles_n, p.n_tile, p.slices, p.split_slices, p.splits, p.ring, p.stage_bytes, p.splits > 1 ? parts : nullptr, (cols + 3) / 4 * 4, f, status};
    const uint64_t items = (uint64_t)p.tiles_m * p.tiles_n * p.splits;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = p.pair ? dim3((unsigned)(2 * std::min<uint64_t>(items, sm_count() / 2))) : dim3(p.tiles_m * p.tiles_n, p.splits);
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.pair ? 2 : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (!status) g_used.store(true, std::memory_order_relaxed);
    e = cudaLaunchKernelEx(&cfg, kernel, ma, mb, g);
    t_launches += p.splits > 1 ? 2 : 1;
    if (e != cudaSuccess || p.splits == 1) return e;
    return launch_following(finish_kernel<T>, dim3(rows, std::min((cols + 1023) / 1024, 64u)), 256, 0, st, parts, p.splits, rows, cols, g.part_ld, f);
}

// Rows of a packed matrix start on 128-byte lines.  (A box of 128 bytes that starts elsewhere takes five sectors of two lines from L2
// instead of four of one: 8192 x 2791 x 8100, plain: 323 us with rows of 2792 elements, 273 of 2800, 260 of 2816.)
uint64_t packed_ld(uint32_t cols) { return (cols + 63ull) / 64 * 64; }
uint64_t packed_elements(const Matrix& m) { return m.rows * packed_ld(m.cols); }

// Whether an operand is copied before the product: where a tensor map cannot describe it, and where its rows straddle lines and
// are read so often (once per tile along the other side) that the copy, two passes over memory, costs less: from about 24 times.
bool needs_pack(const Matrix& m, uint32_t reads) { return !mappable(m) || (m.ld % 16 != 0 && reads >= 24); }

bool vec4_rows(const Finish& f, size_t size)
{
    return RowAlign().add(f.residual, f.ld_residual, size).add(f.out, f.ld_out, size).add(f.z, f.ld_z, size).elements(size, 4) == 4;
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

// Queues an operand's copy and lets the product read that instead.
void take_copy(PackJob* jobs, uint32_t* n, Matrix* m, uint16_t* dst)
{
    if (!dst) return;
    const uint64_t ld = packed_ld(m->cols);
    const uint32_t chunks = (m->cols + 7) / 8;
    jobs[(*n)++] = PackJob{Source{static_cast<const uint16_t*>(m->p), m->ld, m->rows, m->cols}, dst, ld,
                           (uint32_t)((m->rows + 8 * kPackRows - 1) / (8 * kPackRows)), std::min((chunks + 31) / 32, 64u)};
    m->p = dst;
    m->ld = ld;
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

// Runs `step(arena, launch)` twice: to size the workspace, then -- where that was not all -- to launch.
template <typename Step>
int with_workspace(void* dev_workspace, uint64_t* workspace_bytes, uint32_t size_only, const char* what, Step step)
{
    Arena count{nullptr};
    step(count, false);
    if (size_only) {
        if (!workspace_bytes) return report_error(PINK_B200_EINVAL, "null argument");
        *workspace_bytes = count.used;
        return PINK_B200_OK;
    }
    if (count.used) {
        if (!dev_workspace || !workspace_bytes || *workspace_bytes < count.used)
            return report_error(PINK_B200_EINVAL, "workspace too small (ask with size_only)");
        if (reinterpret_cast<uintptr_t>(dev_workspace) % 16) return report_error(PINK_B200_EINVAL, "the workspace must be 16-byte aligned");
    }
    Arena arena{static_cast<uint8_t*>(dev_workspace)};
    return launch_status(step(arena, true), what);
}

template <typename Fn>
cudaError_t with_half_type(uint32_t type, Fn fn)
{
    if (type == PINK_B200_BF16) return fn(__nv_bfloat16());
    return fn(__half());
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

cudaError_t take_product_status(int* out)
{
    *out = 0;
    if (!product_used()) return cudaSuccess;
    cudaError_t e = cudaMemcpyFromSymbol(out, g_status, sizeof(int));
    const int zero = 0;
    if (e == cudaSuccess && *out) e = cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
    return e;
}

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
