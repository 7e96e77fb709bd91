// Shared pieces of the dense products (product.cu, gated.cu): activations, the tensor-core kernel of block pairs, copies into rows that a tensor
// map can describe, plans and workspaces.  Every source that includes this has its own of all of them.
#pragma once
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
    Finish f2;                                           // kGated: bias and z of the second product; kTwo: out of the second
    uint32_t first_slices;                               // kSum: slices of the first product
};

// What a launch of the pair kernel multiplies.  A kind other than kPlain has two products, whose operands lie in four matrices:
//   kGated  z = A B^T and z2 = A B2^T, a tile of each side by side in one accumulator; out = act(z + bias) (z2 + bias2)
//   kSum    D = A B^T + A2 B2^T, one K range after the other
//   kTwo    D = A B^T and D2 = A2 B2^T, the tiles of the second behind those of the first
enum : int { kPlain = 0, kGated = 1, kSum = 2, kTwo = 3 };

template <int KIND> struct Maps { CUtensorMap a, b, a2, b2; };
template <> struct Maps<kPlain> { CUtensorMap a, b; };

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
__device__ __forceinline__ void finish_rows(const GemmArgs& p, const Finish& f, float* parts, uint32_t taddr, uint32_t row0, uint32_t col0, uint32_t split, uint32_t turn,
                                            float* st, uint32_t lane, Drained drained)
{
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
        const bool whole = f.vec4 && !parts && cq + 4 <= left;
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
        if (parts) {
            float* dst = parts + ((size_t)split * p.rows + row0) * p.part_ld + col + lane;
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

// The same for the two halves of an accumulator, z in its first n_tile / 2 columns and z2 behind them: out = act(z + bias) * (z2 + bias2).
template <typename T, typename Drained>
__device__ __forceinline__ void finish_gated_rows(const GemmArgs& p, uint32_t taddr, uint32_t row0, uint32_t col0, uint32_t split, uint32_t turn,
                                                  float* st, uint32_t lane, Drained drained)
{
    const Finish &f = p.f, &f2 = p.f2;
    const uint32_t half = p.n_tile / 2, ncols = min(half, p.cols - col0);
    const uint32_t nrows = row0 < p.rows ? min(32u, p.rows - row0) : 0u;
    const uint32_t cq = (lane & 7) * 4, rq = lane >> 3;
    const uint32_t first = 32 * turn;
    uint32_t v[32], w[32];
    if (first < ncols) { tmem_ld_32x32(taddr + first, v); tmem_ld_32x32(taddr + half + first, w); }      // (may pass the halves, inside the 256 columns)
    else drained();
    for (uint32_t c0 = first; c0 < ncols; c0 += 64) {
        const uint32_t left = min(32u, ncols - c0), col = col0 + c0;
        float y[2][8][4];
        auto stage = [&](const uint32_t (&z)[32], float (&out)[8][4]) {
            __syncwarp();                                // the staged columns before these have been read
#pragma unroll
            for (uint32_t q = 0; q < 32; q += 4)
                *reinterpret_cast<uint4*>(st + lane * kStagePitch + q) = make_uint4(z[q], z[q + 1], z[q + 2], z[q + 3]);
            __syncwarp();
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q) {
                const float4 s = *reinterpret_cast<const float4*>(st + (rq + 4 * q) * kStagePitch + cq);
                out[q][0] = s.x; out[q][1] = s.y; out[q][2] = s.z; out[q][3] = s.w;
            }
        };
        tmem_ld_wait_on(v);
        tmem_ld_wait_on(w);
        stage(v, y[0]);
        stage(w, y[1]);
        if (c0 + 64 < ncols) { tmem_ld_32x32(taddr + c0 + 64, v); tmem_ld_32x32(taddr + half + c0 + 64, w); }
        else drained();
        auto rest = [&] {
            if (p.parts) {
#pragma unroll
                for (uint32_t q = 0; q < 8; ++q)
                    if (rq + 4 * q < nrows) {
                        float* dst = p.parts + ((size_t)split * p.rows + row0 + rq + 4 * q) * 2 * p.part_ld + col + cq;
                        *reinterpret_cast<float4*>(dst) = make_float4(y[0][q][0], y[0][q][1], y[0][q][2], y[0][q][3]);
                        *reinterpret_cast<float4*>(dst + p.part_ld) = make_float4(y[1][q][0], y[1][q][1], y[1][q][2], y[1][q][3]);
                    }
                return;
            }
            const bool whole = f.vec4 && cq + 4 <= left;
            if (f.bias) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float b = cq + i < left ? f.bias[col + cq + i] : 0.0f;
#pragma unroll
                    for (uint32_t q = 0; q < 8; ++q) y[0][q][i] += b;
                }
            }
            if (f2.bias) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float b = cq + i < left ? f2.bias[col + cq + i] : 0.0f;
#pragma unroll
                    for (uint32_t q = 0; q < 8; ++q) y[1][q][i] += b;
                }
            }
            auto write = [&](void* p0, uint64_t ld, const float (&out)[8][4]) {
                T* dst = static_cast<T*>(p0) + (uint64_t)(row0 + rq) * ld + col + cq;
#pragma unroll
                for (uint32_t q = 0; q < 8; ++q) {
                    if (rq + 4 * q >= nrows) continue;
                    if (whole) {
                        Pack<T, 4>::of(out[q]).store(dst + 4 * q * ld);
                    } else {
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i)
                            if (cq + i < left) dst[4 * q * ld + i] = from_float<T>(out[q][i]);
                    }
                }
            };
            if (f.z) write(f.z, f.ld_z, y[0]);
            if (f2.z) write(f2.z, f2.ld_z, y[1]);
            activate_all(y[0], f.act);
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q)
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) y[0][q][i] *= y[1][q][i];
            write(f.out, f.ld_out, y[0]);
        };
        if (cq < left) rest();
        __syncwarp();                                    // (the lanes of a ragged end took different ways)
    }
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
struct Item { uint32_t m, n, split, second; };
template <int KIND>
__device__ __forceinline__ Item item_at(const GemmArgs& p, uint32_t t)
{
    const uint32_t per_split = p.tiles_m * p.tiles_n;
    uint32_t split = t / per_split, second = 0;
    t -= split * per_split;
    if (KIND == kTwo && split >= p.splits) { split -= p.splits; second = 1; }
    const uint32_t strip = t / (kGroupM * p.tiles_n), height = min(kGroupM, p.tiles_m - strip * kGroupM);
    t -= strip * kGroupM * p.tiles_n;
    return { strip * kGroupM + t % height, t / height, split, second };
}

// Pairs of blocks (cta_group::2) that stay resident and work through tiles of 256 x n_tile: each block stages its 128 rows of A and
// half of the tile's rows of B.  Two accumulators of 256 columns: one is finished while the next tile is multiplied.
// Measured, 8192 x 2791 x 8100 with sigmoid, residual and kept z: 254 us (1.46 PFLOP/s, tensor pipe active 85 %); a block a tile of
// 128 x 256 that finished it before the next began: 1209 us.  kGated, 8192 x 3969 x 8100 (twice), GELU, both kept: 701 us (1.50 PFLOP/s, tensor pipe active
// 95 %); kSum and kTwo, the gradients of 4096 x 3969 x 2791: 123 and 128 us (1.47 and 1.42 PFLOP/s, 87 %; 288 tiles
// of 224 columns and 352 of 256, over 74 pairs).
template <typename T, bool A_MN, bool B_MN, int KIND>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_pair_kernel(const __grid_constant__ Maps<KIND> maps, const GemmArgs p)
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
    const uint32_t items = p.tiles_m * p.tiles_n * p.splits * (KIND == kTwo ? 2 : 1);
    const uint32_t half = p.n_tile / 2;
    constexpr uint32_t a_bytes = kTileM * 128;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.ring; ++s) { mbar_init(&full_bar[s], 2); mbar_init(&empty_bar[s], 1); }
        for (uint32_t b = 0; b < 2; ++b) { mbar_init(&done_bar[b], 1); mbar_init(&free_bar[b], 2 * kFinishWarps); }
        mbar_fence_init();
        tma_prefetch_desc(&maps.a);
        tma_prefetch_desc(&maps.b);
        if constexpr (KIND != kPlain) { tma_prefetch_desc(&maps.a2); tma_prefetch_desc(&maps.b2); }
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
                const Item it = item_at<KIND>(p, t);
                // (kGated: the even block stages rows of B, the odd one the same rows of B2)
                const int32_t m0 = (int32_t)((it.m * 2 + rank) * kTileM), n0 = (int32_t)(KIND == kGated ? it.n * half : it.n * p.n_tile + rank * half);
                const CUtensorMap *ma = &maps.a, *mb = &maps.b;
                if constexpr (KIND == kTwo) if (it.second) { ma = &maps.a2; mb = &maps.b2; }
                if constexpr (KIND == kGated) if (rank) mb = &maps.b2;
                const uint32_t kb0 = it.split * p.split_slices, num_kb = min(p.split_slices, p.slices - kb0);
                int32_t k = (int32_t)(kb0 * kSliceK);
                for (uint32_t kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait(empty0 + 8 * s, ph ^ 1)) { report_timeout(p, kGemmTimeoutProducer); ok = false; break; }
                    const uint32_t bar = full0 + 8 * s;
                    if constexpr (KIND == kSum) if (kb == 0 || kb0 + kb == p.first_slices) {
                        const bool second = kb0 + kb >= p.first_slices;
                        ma = second ? &maps.a2 : &maps.a;
                        mb = second ? &maps.b2 : &maps.b;
                        k = (int32_t)((kb0 + kb - (second ? p.first_slices : 0)) * kSliceK);
                    }
                    mbar_expect_tx_cluster(bar, tx);
                    if (A_MN) { tma_load_2d_pair(st, ma, bar, m0, k); tma_load_2d_pair(st + kSliceK * 128, ma, bar, m0 + 64, k); }
                    else tma_load_2d_pair(st, ma, bar, k, m0);
                    if (B_MN) for (uint32_t c = 0; c < b_boxes; ++c) tma_load_2d_pair(st + a_bytes + c * kSliceK * 128, mb, bar, n0 + (int32_t)(c * 64), k);
                    else tma_load_2d_pair(st + a_bytes, mb, bar, k, n0);
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
                const uint32_t kb0 = item_at<KIND>(p, t).split * p.split_slices, num_kb = min(p.split_slices, p.slices - kb0);
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
            const Item it = item_at<KIND>(p, t);
            const uint32_t buf = n_item & 1, use = n_item >> 1;
            if (!mbar_wait(&done_bar[buf], use & 1)) { report_timeout(p, kGemmTimeoutFinish); break; }
            tc_fence_after();
            auto drained = [&] {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(free0 + 8 * buf);
            };
            const uint32_t from = tmem_base + buf * 256 + ((quad * 32u) << 16), row0 = (it.m * 2 + rank) * kTileM + quad * 32, turn = (warp - 2) >> 2;
            if constexpr (KIND == kGated) {
                finish_gated_rows<T>(p, from, row0, it.n * half, it.split, turn, st, lane, drained);
            } else if constexpr (KIND == kTwo) {
                const Finish& f = it.second ? p.f2 : p.f;
                finish_rows<T>(p, f, p.parts ? p.parts + (size_t)it.second * p.splits * p.rows * p.part_ld : nullptr, from, row0, it.n * p.n_tile, it.split, turn, st, lane, drained);
            } else {
                finish_rows<T>(p, p.f, p.parts, from, row0, it.n * p.n_tile, it.split, turn, st, lane, drained);
            }
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
    using In = RowOf<__half, kAny>;                      // (any 16-bit elements)
    const Source& m = job.m;
    const uint32_t chunks = (m.cols + 7) / 8;
    const uint64_t row0 = ((uint64_t)(block / job.col_blocks) * 8 + (threadIdx.x >> 5)) * kPackRows;
    for (uint32_t c = block % job.col_blocks * 32 + (threadIdx.x & 31); c < chunks; c += job.col_blocks * 32) {
        In::Chunk v[kPackRows];
#pragma unroll
        for (uint32_t r = 0; r < kPackRows; ++r)
            if (row0 + r < m.rows) v[r] = In(m.p, m.ld, row0 + r, m.rows, m.cols).load(c * 8);
#pragma unroll
        for (uint32_t r = 0; r < kPackRows; ++r)
            if (row0 + r < m.rows) *reinterpret_cast<uint4*>(job.dst + (row0 + r) * job.ld + c * 8) = In(m.p, m.ld, row0 + r, m.rows, m.cols).all(v[r]);
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

uint32_t slices_of(uint32_t K) { return (K + kSliceK - 1) / kSliceK; }

// `wide`: columns of an accumulator that a column of D takes (kGated: 2); `products`: kTwo: 2; `range`: slices of a range of K, at least.
GemmPlan plan_gemm(uint32_t rows, uint32_t cols, uint32_t slices, bool b_mn, bool pair, uint32_t wide = 1, uint32_t products = 1,
                   uint32_t range = 4)
{
    GemmPlan p{};
    const uint32_t sms = (uint32_t)sm_count();
    p.slices = slices;
    p.pair = pair;
    if (p.pair) {
        p.tiles_m = (rows + 2 * kTileM - 1) / (2 * kTileM);
        // the tile width whose waves over the pairs take least: a slice costs what an SM loads for it, 128 rows of A and half the
        // tile's of B (2791 x 3969 x 4096: 90 us with 160 columns, which multiplying alone would choose)
        uint64_t best = ~0ull;
        for (uint32_t w = 256; w >= 64; w -= 32) {
            const uint64_t tiles = (uint64_t)products * p.tiles_m * ((cols + w / wide - 1) / (w / wide)), waves = (tiles + sms / 2 - 1) / (sms / 2);
            const uint64_t cost = waves * (kTileM + w / 2);
            if (cost < best) { best = cost; p.n_tile = w; }
        }
        p.n_tile = (uint32_t)std::min<uint64_t>(p.n_tile, ((uint64_t)cols * wide + 31) / 32 * 32);
    } else {
        p.tiles_m = (rows + kTileM - 1) / kTileM;
        const uint32_t grain = b_mn ? 64 : 16;           // an MN-major tile is made of 64-element rows
        p.n_tile = std::min(256u, (cols + grain - 1) / grain * grain);
        while (p.n_tile > 64 && (uint64_t)p.tiles_m * ((cols + p.n_tile - 1) / p.n_tile) < (uint64_t)sms) p.n_tile = (p.n_tile / 2 + grain - 1) / grain * grain;
    }
    p.tiles_n = (cols + p.n_tile / wide - 1) / (p.n_tile / wide);
    // fewer tiles than SMs (pairs of them): split K
    const uint64_t tiles = (uint64_t)products * p.tiles_m * p.tiles_n;
    const uint32_t splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>((p.pair ? sms / 2 : sms) / tiles, p.slices / range));
    p.split_slices = (p.slices + splits - 1) / splits;
    p.splits = (p.slices + p.split_slices - 1) / p.split_slices;
    const uint32_t b_rows = p.pair ? p.n_tile / 2 : p.n_tile;
    p.stage_bytes = kTileM * 128 + (b_mn ? (b_rows + 63) / 64 * kSliceK * 128 : (b_rows * 128 + 1023) / 1024 * 1024);
    p.ring = std::min(kMaxRing, (kSmemBudget - 1024 - kHeadBytes - kStagingBytes) / p.stage_bytes);
    if (!p.pair) p.ring = std::min(p.ring, std::max(2u, p.split_slices));
    return p;
}

GemmPlan plan_gemm(uint32_t rows, uint32_t cols, uint32_t K, bool b_mn) { return plan_gemm(rows, cols, slices_of(K), b_mn, rows > kTileM); }

// Opts a product's kernel into large shared memory, once per thread and device.
template <typename... P>
cudaError_t opt_in(void (*kernel)(P...), int* device)
{
    int dev = 0;
    cudaGetDevice(&dev);
    if (*device == dev) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBudget);
    if (e == cudaSuccess) *device = dev;
    return e;
}

GemmArgs gemm_args(const GemmPlan& p, uint32_t rows, uint32_t cols, float* parts, const Finish& f, int* status)
{
    return {rows, cols, p.tiles_m, p.tiles_n, p.n_tile, p.slices, p.split_slices, p.splits, p.ring, p.stage_bytes, p.splits > 1 ? parts : nullptr,
            (cols + 3) / 4 * 4, f, status, Finish{}, 0};
}

template <typename... P, typename... A>
cudaError_t launch_product(void (*kernel)(P...), dim3 grid, uint32_t cluster, size_t smem, cudaStream_t st, const A&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, bool A_MN, bool B_MN, int KIND>
cudaError_t launch_pairs(const Maps<KIND>& maps, const GemmPlan& p, const GemmArgs& g, cudaStream_t st)
{
    static thread_local int opted_in = -1;               // device of the last opt-in to large shared memory
    auto* kernel = gemm_pair_kernel<T, A_MN, B_MN, KIND>;
    const cudaError_t e = opt_in(kernel, &opted_in);
    if (e != cudaSuccess) return e;
    const uint64_t items = (uint64_t)p.tiles_m * p.tiles_n * p.splits * (KIND == kTwo ? 2 : 1);
    if (!g.status) g_used.store(true, std::memory_order_relaxed);
    t_launches += 1;
    // (A pair takes all of its SMs' shared memory that matters: no other kernel's pair, which would wait for the same tensor
    // memory in the other order, fits beside it.)
    return launch_product(kernel, dim3((unsigned)(2 * std::min<uint64_t>(items, sm_count() / 2))), 2, kSmemBudget, st, maps, g);
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

// Reads and clears the code of the first wait that expired in a call of this source's public entries.
cudaError_t take_status(int* out)
{
    *out = 0;
    if (!g_used.load(std::memory_order_relaxed)) return cudaSuccess;
    cudaError_t e = cudaMemcpyFromSymbol(out, g_status, sizeof(int));
    const int zero = 0;
    if (e == cudaSuccess && *out) e = cudaMemcpyToSymbol(g_status, &zero, sizeof(int));
    return e;
}

} // namespace
} // namespace pinkb
