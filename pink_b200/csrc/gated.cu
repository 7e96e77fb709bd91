// Gated projections and their gradient (pink_b200_op_gated*).
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = act(g) u
//   dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dbg, dbu = column sums of dg, du
//
// The products run on the kernel of block pairs in product.cuh.  Forward, one block of a pair stages rows of Wg and the other the same rows of
// Wu, so that a tile of g and the same tile of u lie side by side in one accumulator and meet in the epilogue: x is read once for both, and
// g and u reach memory only where they are kept.  Backward, dx is one product whose K runs through dg and Wg and then through du
// and Wu; the weights' gradients are the tiles of one launch.
#include "product.cuh"

namespace pinkb {
namespace {

// ---- a few rows ------------------------------------------------------------------------------------------------------------
// Up to kFewRows rows of x: bound by reading both weights once.  ROWS is the number of rows rounded up to a power of two; the rows beyond
// n repeat the last.

constexpr uint32_t kFewRows = 8;

struct FewArgs
{
    Source x, gate, up;
    uint32_t n, K, M;
    Finish f, f2;                    // as for kGated
};

template <typename T>
__device__ __forceinline__ void finish_gated1(const Finish& f, const Finish& f2, uint64_t row, uint32_t col, float g, float u)
{
    if (f.bias) g += f.bias[col];
    if (f2.bias) u += f2.bias[col];
    if (f.z) static_cast<T*>(f.z)[row * f.ld_z + col] = from_float<T>(g);
    if (f2.z) static_cast<T*>(f2.z)[row * f2.ld_z + col] = from_float<T>(u);
    static_cast<T*>(f.out)[row * f.ld_out + col] = from_float<T>(activate(g, f.act) * u);
}

// Weights by output: a block takes kFewOut outputs, its four warps a quarter of k each, in which a chunk of x serves all of its weights' rows -- so that
// four loads are on their way at once and x costs little.  The warps' sums meet in shared memory.  (One row, 2,791 x 8,100: 19.2 us among others of its kind;
// four outputs a block 22.6, eight warps 21.4.)
constexpr uint32_t kFewOut = 2, kFewWarps = 4;

template <typename T, int ALIGN, int ROWS>
__global__ void __launch_bounds__(32 * kFewWarps) gated_few_rows_kernel(const FewArgs a)
{
    using In = RowOf<T, ALIGN>;
    __shared__ float meet[kFewWarps][ROWS][2 * kFewOut];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, m0 = blockIdx.x * kFewOut;
    follow();
    F2 acc[ROWS][2 * kFewOut];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (uint32_t o = 0; o < 2 * kFewOut; ++o) acc[i][o] = two(0.0f);
    // (outputs beyond the last repeat it, rows beyond n the last, and are not written)
    auto weight = [&](uint32_t o) {
        const Source& w = o & 1 ? a.up : a.gate;
        return In(w.p, w.ld, min(m0 + o / 2, a.M - 1), a.M, a.K);
    };
    auto row = [&](uint32_t i) { return In(a.x.p, a.x.ld, min(i, a.n - 1), a.n, a.K); };
    const uint32_t chunks = (a.K + 7) / 8, part = (chunks + kFewWarps - 1) / kFewWarps, end = min(chunks, (warp + 1) * part);
    for (uint32_t k = warp * part + lane; k < end; k += 32) {
        typename In::Chunk w[2 * kFewOut];
#pragma unroll
        for (uint32_t o = 0; o < 2 * kFewOut; ++o) w[o] = weight(o).load(k * 8);
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
            const In x = row(i);
            const uint4 xv = x.all(x.load(k * 8));
#pragma unroll
            for (uint32_t o = 0; o < 2 * kFewOut; ++o) {
                const uint4 wv = weight(o).all(w[o]);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][o] = fma2(pair_of<T>(xv, j), pair_of<T>(wv, j), acc[i][o]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (uint32_t o = 0; o < 2 * kFewOut; ++o) {
            const float s = warp_sum(acc[i][o].lo() + acc[i][o].hi());
            if (lane == 0) meet[warp][i][o] = s;
        }
    __syncthreads();
    const uint32_t i = threadIdx.x / kFewOut, m = threadIdx.x % kFewOut;
    if (i >= a.n || m0 + m >= a.M) return;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (uint32_t q = 0; q < kFewWarps; ++q) { g += meet[q][i][2 * m]; u += meet[q][i][2 * m + 1]; }
    finish_gated1<T>(a.f, a.f2, i, m0 + m, g, u);
}

// Four elements at any alignment of a row, as load_chunk (readout.cuh) takes eight.
struct Four { uint2 a, b; uint32_t off; };

template <bool WHOLE>
__device__ __forceinline__ Four load_four(const Source& m, uint64_t row, uint32_t col)
{
    const uint16_t* src = m.p + row * m.ld + col;
    const uint32_t off = WHOLE ? 0u : (uint32_t)reinterpret_cast<uintptr_t>(src) & 7u;
    const uint16_t* lo = src - off / 2;
    if (col + 4 <= m.cols && (WHOLE || (lo >= m.p && lo + 8 <= m.p + (m.rows - 1) * m.ld + m.cols)))
        return { *reinterpret_cast<const uint2*>(lo), WHOLE ? make_uint2(0, 0) : *(reinterpret_cast<const uint2*>(lo) + 1), off };
    uint32_t w[2] = { 0, 0 };
#pragma unroll
    for (uint32_t q = 0; q < 4; ++q)
        if (col + q < m.cols) w[q / 2] |= (uint32_t)src[q] << (q & 1) * 16;
    return { make_uint2(w[0], w[1]), make_uint2(0, 0), 0u };
}

template <typename T, bool WHOLE>
__device__ __forceinline__ void floats_of(const Four& e, float (&f)[4])
{
    uint2 w = e.a;
    if constexpr (!WHOLE) {
        const uint32_t v[4] = { e.a.x, e.a.y, e.b.x, e.b.y }, s = e.off & 4u ? 1u : 0u, bits = (e.off & 2u) * 8u;
        w = make_uint2(__funnelshift_r(s ? v[1] : v[0], s ? v[2] : v[1], bits), __funnelshift_r(s ? v[2] : v[1], s ? v[3] : v[2], bits));
    }
    Pack<T, 4>{ w }.floats(f);
}

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}

// Weights by input: lanes along the outputs; the eight warps of a block and the kFewBlocks blocks of a cluster along k.  The warps' sums
// meet in shared memory, the blocks' in distributed shared memory: one launch, no scratch, a fixed order.
constexpr uint32_t kFewBlocks = 8, kFewCols = 128;

template <typename T, bool WHOLE, int ROWS>
__global__ void __launch_bounds__(256) gated_few_rows_by_input_kernel(const FewArgs a)
{
    constexpr uint32_t kStep = 8 * kFewBlocks, kAhead = ROWS <= 2 ? 4 : 2;
    __shared__ float meet[8][2][kFewCols];
    __shared__ float sums[ROWS][2][kFewCols];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rank = cluster_ctarank();
    const uint32_t col0 = blockIdx.x / kFewBlocks * kFewCols, col = col0 + lane * 4;
    float acc[ROWS][2][4];
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[i][0][v] = acc[i][1][v] = 0.0f;
    const T* x = reinterpret_cast<const T*>(a.x.p);
    if (col < a.M)
        for (uint64_t k0 = rank * 8 + warp; k0 < a.K; k0 += kAhead * kStep) {
            Four wg[kAhead], wu[kAhead];
            T xv[ROWS][kAhead];
#pragma unroll
            for (uint32_t q = 0; q < kAhead; ++q) {
                const uint64_t k = k0 + q * kStep;
                if (k >= a.K) break;
                wg[q] = load_four<WHOLE>(a.gate, k, col);
                wu[q] = load_four<WHOLE>(a.up, k, col);
#pragma unroll
                for (int i = 0; i < ROWS; ++i) xv[i][q] = x[min((uint32_t)i, a.n - 1) * a.x.ld + k];
            }
#pragma unroll
            for (uint32_t q = 0; q < kAhead; ++q) {
                if (k0 + q * kStep >= a.K) break;
                float gf[4], uf[4];
                floats_of<T, WHOLE>(wg[q], gf);
                floats_of<T, WHOLE>(wu[q], uf);
#pragma unroll
                for (int i = 0; i < ROWS; ++i)
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        acc[i][0][v] = fmaf(to_float(xv[i][q]), gf[v], acc[i][0][v]);
                        acc[i][1][v] = fmaf(to_float(xv[i][q]), uf[v], acc[i][1][v]);
                    }
            }
        }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < 4; ++v) { meet[warp][0][lane * 4 + v] = acc[i][0][v]; meet[warp][1][lane * 4 + v] = acc[i][1][v]; }
        __syncthreads();
        const uint32_t both = threadIdx.x >> 7, c = threadIdx.x & 127;
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < 8; ++q) s += meet[q][both][c];
        sums[i][both][c] = s;
    }
    cluster_sync();
    // each block finishes its share of the outputs
    for (uint32_t t = threadIdx.x + 256 * rank; t < a.n * kFewCols; t += 256 * kFewBlocks) {
        const uint32_t i = t / kFewCols, c = t % kFewCols;
        if (col0 + c >= a.M) continue;
        const uint32_t here = smem_u32(&sums[i][0][c]);
        float g = 0.0f, u = 0.0f;
#pragma unroll
        for (uint32_t q = 0; q < kFewBlocks; ++q) {
            const uint32_t there = map_to_cta(here, q);
            g += ld_cluster_f32(there);
            u += ld_cluster_f32(there + kFewCols * 4);
        }
        finish_gated1<T>(a.f, a.f2, i, col0 + c, g, u);
    }
    cluster_sync();                                      // no block leaves while another reads its sums
}

// Sum of the K ranges' partial sums, in order, and what follows it.
template <typename T>
__global__ void __launch_bounds__(256) finish_gated_kernel(const float* parts, uint32_t splits, uint32_t rows, uint32_t cols, uint32_t part_ld, const Finish f, const Finish f2)
{
    follow();
    const uint64_t row = blockIdx.x;
    const size_t step = (size_t)rows * 2 * part_ld;
    for (uint32_t c = blockIdx.y * 256 + threadIdx.x; c < cols; c += gridDim.y * 256) {
        const float* src = parts + row * 2 * part_ld + c;
        float g = 0.0f, u = 0.0f;
#pragma unroll 4
        for (uint32_t k = 0; k < splits; ++k) { g += src[k * step]; u += src[k * step + part_ld]; }
        finish_gated1<T>(f, f2, row, c, g, u);
    }
}

// ---- gradients of g and u ---------------------------------------------------------------------------------------------------


// x times a factor that its 16-bit type may have held as an infinity while it was finite: nothing where x is nothing.
__device__ __forceinline__ float times_limit(float x, float factor)
{
    const float p = x * finite_factor(factor);
    return fabsf(factor) == INFINITY && p != 0.0f ? p * INFINITY : p;
}

// Value and slope of the gate's activation.
template <uint32_t ACT>
__device__ __forceinline__ float2 gate_of(float z)
{
    if constexpr (ACT == PINK_B200_ACT_SILU) {
        const float q = __fdividef(1.0f, 1.0f + __expf(-z));               // (0 below -88)
        return make_float2(z * q, fmaf(z * q, 1.0f - q, q));               // (what 1 - q loses is lost beside the q that is added)
    } else if constexpr (ACT == PINK_B200_ACT_GELU) {
        float gauss;
        const float c = normal_cdf(z, &gauss);
        return make_float2(z * c, fmaf(z * 0.39894228f, gauss, c));
    } else if constexpr (ACT == PINK_B200_ACT_SIGMOID) {
        const float q = sigmoid_f(z);
        return make_float2(q, q * sigmoid_f(-z));
    } else if constexpr (ACT == PINK_B200_ACT_RELU) {
        return make_float2(z > 0.0f || z != z ? z : 0.0f, z > 0.0f ? 1.0f : 0.0f);
    } else {
        return make_float2(z, 1.0f);
    }
}

// dg and du of eight elements, whose instructions do not wait for one another.  An infinity that a 16-bit type holds for a finite g or u makes some
// of them NaN; the elements that have become NaN are formed again with the limits: of act and its slope where g is an infinity, and nothing where
// an infinity meets a gradient of zero.
template <uint32_t ACT>
__device__ __forceinline__ void gate_gradients(const float (&d)[8], const float (&g)[8], const float (&u)[8], float (&dg)[8], float (&du)[8])
{
    float check = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 a = gate_of<ACT>(g[i]);
        dg[i] = d[i] * a.y * u[i];
        du[i] = d[i] * a.x;
        check = fmaf(dg[i], 0.0f, fmaf(du[i], 0.0f, check));
    }
    if (__builtin_expect(check == 0.0f, 1)) return;      // (an infinity or a NaN among them makes a NaN of it)
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
        float z = 0.0f, dd = 0.0f, uu = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j == i) { z = g[j]; dd = d[j]; uu = u[j]; }
        float2 a = gate_of<ACT>(z);
        if (z == -INFINITY && ACT != PINK_B200_ACT_NONE) a = make_float2(0.0f, 0.0f);
        if (z == INFINITY && ACT != PINK_B200_ACT_SIGMOID) a = make_float2(INFINITY, 1.0f);
        const float x = times_limit(dd * a.y, uu), y = times_limit(dd, a.x);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j == i) { dg[j] = x; du[j] = y; }
    }
}

template <typename Fn>
__device__ __forceinline__ void with_activation(uint32_t act, Fn fn)
{
    if (act == PINK_B200_ACT_SILU) fn(std::integral_constant<uint32_t, PINK_B200_ACT_SILU>());
    else if (act == PINK_B200_ACT_GELU) fn(std::integral_constant<uint32_t, PINK_B200_ACT_GELU>());
    else if (act == PINK_B200_ACT_SIGMOID) fn(std::integral_constant<uint32_t, PINK_B200_ACT_SIGMOID>());
    else if (act == PINK_B200_ACT_RELU) fn(std::integral_constant<uint32_t, PINK_B200_ACT_RELU>());
    else fn(std::integral_constant<uint32_t, PINK_B200_ACT_NONE>());
}

// dg and du enter the products in 16 bits, as the tensor cores want it: half a step of each (2^-8 of it in bfloat16, 2^-11 in float16).  float16 has too little
// range for them as they are -- products of three numbers -- so they are multiplied by the power of two that takes the largest finite
// |dg| or |du| of the call to 2^14 .. 2^15, and the sums by its inverse, both exactly; what is 2^-28 of the largest or less loses
// digits.  The largest is found by a pass of its own over dh, g and u.
struct GradJob
{
    Source dh, g, u;
    uint16_t *dg, *du; uint64_t ld;                      // null: only the sums are asked for
    float *gate_sums, *up_sums;                          // [row_blocks][cols], null: not asked for
    uint32_t act, rows, row_blocks, col_blocks;          // rows that one block takes, and adds up for the biases
    uint32_t* peaks; float* unscale; uint32_t peak_count;
};

// A row of dh, g and u.
template <typename T>
struct Three
{
    using In = RowOf<T, kAny>;
    struct Loaded { typename In::Chunk d, g, u; };
    In d, g, u;
    __device__ __forceinline__ Three(const GradJob& job, uint64_t row)
        : d(job.dh.p, job.dh.ld, row, job.dh.rows, job.dh.cols), g(job.g.p, job.g.ld, row, job.g.rows, job.g.cols), u(job.u.p, job.u.ld, row, job.u.rows, job.u.cols) {}
    __device__ __forceinline__ Loaded load(uint32_t col) const { return { d.load(col), g.load(col), u.load(col) }; }
    __device__ __forceinline__ void floats(const Loaded& v, float (&df)[8], float (&gf)[8], float (&uf)[8]) const
    {
        Pack<T, 8>{ d.all(v.d) }.floats(df);
        Pack<T, 8>{ g.all(v.g) }.floats(gf);
        Pack<T, 8>{ u.all(v.u) }.floats(uf);
    }
};

template <typename T>
__global__ void __launch_bounds__(256) gated_peak_kernel(const GradJob job)
{
    __shared__ uint32_t part[8];
    follow();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t chunks = (job.dh.cols + 7) / 8, pieces = (chunks + 31) / 32;
    const uint64_t items = job.dh.rows * pieces;
    uint32_t most = 0;
    with_activation(job.act, [&](auto act) {
#pragma unroll 2
        for (uint64_t t = (uint64_t)blockIdx.x * 8 + warp; t < items; t += (uint64_t)gridDim.x * 8) {
            const uint64_t row = t / pieces;
            const uint32_t c = (uint32_t)(t - row * pieces) * 32 + lane;
            if (c >= chunks) continue;
            const Three<T> in(job, row);
            float df[8], gf[8], uf[8], dg[8], du[8];
            in.floats(in.load(c * 8), df, gf, uf);
            gate_gradients<decltype(act)::value>(df, gf, uf, dg, du);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t a = __float_as_uint(dg[i]) & 0x7FFFFFFFu, b = __float_as_uint(du[i]) & 0x7FFFFFFFu;
                if (a < 0x7F800000u) most = max(most, a);    // (infinities and NaN have no part in it)
                if (b < 0x7F800000u) most = max(most, b);
            }
        }
    });
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if (lane == 0) part[warp] = most;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) most = max(most, part[w]);
        job.peaks[blockIdx.x] = most;
    }
}

// The power of two for dg and du, 1 where they have nothing but zeros; all threads of a block of 256 call it.
__device__ __forceinline__ float gate_scale(const GradJob& job)
{
    __shared__ uint32_t part[8];
    uint32_t most = 0;
    for (uint32_t i = threadIdx.x; i < job.peak_count; i += 256) most = max(most, job.peaks[i]);
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) most = max(most, part[w]);
    if (most == 0) return 1.0f;
    const uint32_t exponent = max(most >> 23, 127u - 86u);           // (so that the power and its inverse are finite)
    return __uint_as_float((127 + 14 + 127 - exponent) << 23);
}

// A block takes job.rows rows and 256 columns, eight a thread, its eight warps the rows in turn; a warp's next row is on its way.  Measured, 4,096 x 2,791 SiLU: 41 us (2.8 TB/s),
// bound by instructions at two blocks an SM; with the limits of infinities formed for every element 55.
template <typename T, uint32_t ACT>
__device__ __forceinline__ void gradients_block(const GradJob& job, uint32_t block, float (&meet)[8][32][9])
{
    float scale = 1.0f;
    if (job.peak_count) {
        scale = gate_scale(job);
        if (block == 0 && threadIdx.x == 0) *job.unscale = 1.0f / scale;
    }
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, rb = block / job.col_blocks, cols = job.dh.cols;
    const uint64_t lo = (uint64_t)rb * job.rows, hi = min(lo + job.rows, job.dh.rows);
    for (uint32_t c0 = block % job.col_blocks * 256; c0 < cols; c0 += job.col_blocks * 256) {
        const uint32_t c = c0 + lane * 8;
        float sg[8] = { 0, 0, 0, 0, 0, 0, 0, 0 }, su[8] = { 0, 0, 0, 0, 0, 0, 0, 0 };
        if (c < cols) {
            uint64_t r = lo + warp;
            typename Three<T>::Loaded next;
            if (r < hi) next = Three<T>(job, r).load(c);
#pragma unroll 1
            for (; r < hi; r += 8) {
                float df[8], gf[8], uf[8], dg[8], du[8];
                Three<T>(job, r).floats(next, df, gf, uf);
                if (r + 8 < hi) next = Three<T>(job, r + 8).load(c);
                gate_gradients<ACT>(df, gf, uf, dg, du);
#pragma unroll
                for (int i = 0; i < 8; ++i) {            // (beyond the row dh is zero, and so are these)
                    sg[i] += dg[i];
                    su[i] += du[i];
                    dg[i] *= scale;
                    du[i] *= scale;
                }
                if (job.dg) {
                    Pack<T, 8>::of(dg).store(reinterpret_cast<T*>(job.dg) + r * job.ld + c);
                    Pack<T, 8>::of(du).store(reinterpret_cast<T*>(job.du) + r * job.ld + c);
                }
            }
        }
        auto add_up = [&](const float (&sum)[8], float* out) {
            if (!out) return;
#pragma unroll
            for (int i = 0; i < 8; ++i) meet[warp][lane][i] = sum[i];
            __syncthreads();
            const uint32_t m = threadIdx.x >> 3, i = threadIdx.x & 7;
            float s = 0.0f;
#pragma unroll
            for (int q = 0; q < 8; ++q) s += meet[q][m][i];
            if (c0 + threadIdx.x < cols) out[(size_t)rb * cols + c0 + threadIdx.x] = s;
            __syncthreads();
        };
        add_up(sg, job.gate_sums);
        add_up(su, job.up_sums);
    }
}

// dg and du, and (blocks behind them) up to three copies.
template <typename T>
__global__ void __launch_bounds__(256, 2) gated_prepare_kernel(const GradJob job, const PackJob p0, const PackJob p1, const PackJob p2)
{
    __shared__ float meet[8][32][9];                     // (nine: no bank conflicts)
    follow();
    uint32_t block = blockIdx.x;
    const uint32_t n_dz = job.row_blocks * job.col_blocks, n0 = p0.row_blocks * p0.col_blocks, n1 = p1.row_blocks * p1.col_blocks;
    if (block < n_dz) {
        with_activation(job.act, [&](auto act) { gradients_block<T, decltype(act)::value>(job, block, meet); });
        return;
    }
    block -= n_dz;
    if (block < n0) { pack_block(p0, block); return; }
    block -= n0;
    if (block < n1) pack_block(p1, block);
    else pack_block(p2, block - n1);
}

// Copies of operands where they are many: a kernel of its own, with registers for more blocks (x and both weights of 8,192 x 3,969 x 8,100: 58 us, 6.7 TB/s; in one launch
// with the gradients 88 us).
__global__ void __launch_bounds__(256, 5) gated_pack_kernel(const PackJob p0, const PackJob p1, const PackJob p2)
{
    follow();
    uint32_t block = blockIdx.x;
    const uint32_t n0 = p0.row_blocks * p0.col_blocks, n1 = p1.row_blocks * p1.col_blocks;
    if (block < n0) { pack_block(p0, block); return; }
    block -= n0;
    if (block < n1) pack_block(p1, block);
    else pack_block(p2, block - n1);
}

// Column sums of the blocks' sums, of the gate's and the other projection's bias: a block takes 32 columns, its eight warps the row blocks in turn.
__global__ void __launch_bounds__(256) gated_dbias_kernel(const float* gate_sums, const float* up_sums, uint32_t blocks, uint32_t cols, float* dgate, float* dup)
{
    __shared__ float meet[8][32];
    follow();
    const float* sums = blockIdx.y ? up_sums : gate_sums;
    float* out = blockIdx.y ? dup : dgate;
    if (!out) return;
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
        out[c] = s;
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------

// K ranges of so many slices at least: shorter ones take less time than joining them (331 x 961 x 400: dx in one range of 14 slices 9.2 us, and 4.6 for the joining).
constexpr uint32_t kRangeSlices = 16;

// Boxes of A and B that a block of a pair stages.
uint32_t box_a(bool mn) { return mn ? kSliceK : kTileM; }
uint32_t box_b(const GemmPlan& p, bool mn) { return mn ? kSliceK : p.n_tile / 2; }

template <bool A_MN, bool B_MN, int KIND>
bool encode_all(Maps<KIND>* maps, const GemmPlan& p, const Matrix& a, const Matrix& b, const Matrix& a2, const Matrix& b2)
{
    return encode(&maps->a, a, box_a(A_MN)) && encode(&maps->b, b, box_b(p, B_MN)) && encode(&maps->a2, a2, box_a(A_MN)) && encode(&maps->b2, b2, box_b(p, B_MN));
}

// The copies, and (T: with rows) dg and du: in one launch where that is a wave or less, which is quicker than two.
template <typename T>
cudaError_t launch_prepare(const GradJob& job, const PackJob* jobs, cudaStream_t st)
{
    const uint64_t gradients = (uint64_t)job.row_blocks * job.col_blocks;
    uint64_t copies = 0;
    for (int i = 0; i < 3; ++i) copies += (uint64_t)jobs[i].row_blocks * jobs[i].col_blocks;
    if (gradients + copies > 0x7FFFFFFFull) return cudaErrorInvalidValue;
    const bool both = gradients && (copies == 0 || gradients + copies <= 4ull * sm_count());
    const PackJob none{};
    if (gradients) {
        const cudaError_t e = launch_following(gated_prepare_kernel<T>, dim3((unsigned)(both ? gradients + copies : gradients)), 256, 0, st, job,
                                               both ? jobs[0] : none, both ? jobs[1] : none, both ? jobs[2] : none);
        if (e != cudaSuccess || both) return e;
    }
    if (copies == 0) return cudaSuccess;
    return launch_following(gated_pack_kernel, dim3((unsigned)copies), 256, 0, st, jobs[0], jobs[1], jobs[2]);
}

template <typename T, int ALIGN>
cudaError_t few_rows(const FewArgs& a, cudaStream_t st)
{
    auto launch = [&](auto kernel) { return launch_following(kernel, dim3((a.M + kFewOut - 1) / kFewOut), 32 * kFewWarps, 0, st, a); };
    if (a.n == 1) return launch(gated_few_rows_kernel<T, ALIGN, 1>);
    if (a.n == 2) return launch(gated_few_rows_kernel<T, ALIGN, 2>);
    if (a.n <= 4) return launch(gated_few_rows_kernel<T, ALIGN, 4>);
    return launch(gated_few_rows_kernel<T, ALIGN, 8>);
}

template <typename T, bool WHOLE>
cudaError_t few_rows_by_input(const FewArgs& a, cudaStream_t st)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.M + (uint64_t)kFewCols - 1) / kFewCols * kFewBlocks));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kFewBlocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (a.n == 1) return cudaLaunchKernelEx(&cfg, gated_few_rows_by_input_kernel<T, WHOLE, 1>, a);
    if (a.n == 2) return cudaLaunchKernelEx(&cfg, gated_few_rows_by_input_kernel<T, WHOLE, 2>, a);
    if (a.n <= 4) return cudaLaunchKernelEx(&cfg, gated_few_rows_by_input_kernel<T, WHOLE, 4>, a);
    return cudaLaunchKernelEx(&cfg, gated_few_rows_by_input_kernel<T, WHOLE, 8>, a);
}

int check_gated(const pink_b200_product_config* c, uint64_t ld_x, uint64_t ld_gate, uint64_t ld_up)
{
    if (!c) return report_error(PINK_B200_EINVAL, "null argument");
    if (c->type != PINK_B200_BF16 && c->type != PINK_B200_F16) return report_error(PINK_B200_EINVAL, "gated projections take bfloat16 and float16");
    if (c->inputs == 0 || c->inputs > 0x3FFFFFF0u || c->outputs == 0 || c->outputs > 0x3FFFFFF0u || c->n > 0x7FFFFFF0ull)
        return report_error(PINK_B200_EINVAL, "inputs and outputs must be 1 to 1073741808, rows at most 2147483632");
    if (c->by_input > 1) return report_error(PINK_B200_EINVAL, "by_input must be 0 or 1");
    if (c->activation > PINK_B200_ACT_SIGMOID) return report_error(PINK_B200_EINVAL, "unknown activation");
    if (c->reserved) return report_error(PINK_B200_EINVAL, "reserved must be 0");
    const uint64_t row = c->by_input ? c->outputs : c->inputs;
    if (ld_x < c->inputs || ld_gate < row || ld_up < row) return report_error(PINK_B200_EINVAL, "leading dimension smaller than the row");
    if (ld_x >= 1ull << 38 || ld_gate >= 1ull << 38 || ld_up >= 1ull << 38) return report_error(PINK_B200_EINVAL, "leading dimension too large");
    // tiles of 256 rows and at least 16 columns, of two products
    auto tiles = [](uint64_t r, uint64_t c2) { return 2 * ((r + 255) / 256) * ((c2 + 15) / 16); };
    const uint64_t most = std::max(std::max(tiles(c->n, c->outputs), tiles(c->n, c->inputs)),
                                   std::max(tiles(c->outputs, c->inputs), tiles(c->inputs, c->outputs)));
    if (most > 0x7FFFFFFFull) return report_error(PINK_B200_EINVAL, "product too large");
    return PINK_B200_OK;
}

} // namespace

bool gated_used() { return g_used.load(std::memory_order_relaxed); }

cudaError_t take_gated_status(int* out) { return take_status(out); }

} // namespace pinkb

using namespace pinkb;

extern "C" {

int pink_b200_op_gated(const pink_b200_product_config* cfg, const void* dev_x, uint64_t ld_x, const void* dev_gate, uint64_t ld_gate, const void* dev_up,
                       uint64_t ld_up, const float* dev_gate_bias, const float* dev_up_bias, void* dev_h, uint64_t ld_h, void* dev_g, uint64_t ld_g,
                       void* dev_u, uint64_t ld_u, void* dev_workspace, uint64_t* workspace_bytes, uint32_t size_only, void* stream)
{
    const int rc = check_gated(cfg, ld_x, ld_gate, ld_up);
    if (rc) return rc;
    const uint32_t n = (uint32_t)cfg->n, K = cfg->inputs, M = cfg->outputs;
    if (ld_h < M || (dev_g && ld_g < M) || (dev_u && ld_u < M)) return report_error(PINK_B200_EINVAL, "leading dimension smaller than the row");
    if (n == 0) {
        if (size_only && workspace_bytes) *workspace_bytes = 0;
        return PINK_B200_OK;
    }
    if (!dev_x || !dev_gate || !dev_up || !dev_h) return report_error(PINK_B200_EINVAL, "null argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const uint64_t w_rows = cfg->by_input ? K : M;
    const uint32_t w_cols = cfg->by_input ? M : K;
    const bool mn = cfg->by_input != 0;
    return with_workspace(dev_workspace, workspace_bytes, size_only, "gated projections", [&](Arena& ws, bool launch) {
        return with_half_type(cfg->type, [&](auto t) {
            using T = decltype(t);
            Matrix x{dev_x, ld_x, n, K}, gate{dev_gate, ld_gate, w_rows, w_cols}, up{dev_up, ld_up, w_rows, w_cols};
            Finish f{}, f2{};
            f.bias = dev_gate_bias; f.out = dev_h; f.ld_out = ld_h; f.z = dev_g; f.ld_z = ld_g; f.act = cfg->activation;
            f2.bias = dev_up_bias; f2.z = dev_u; f2.ld_z = ld_u;
            if (n <= kFewRows) {
                if (!launch) return cudaSuccess;
                auto source = [](const Matrix& m) { return Source{static_cast<const uint16_t*>(m.p), m.ld, m.rows, m.cols}; };
                const FewArgs a{source(x), source(gate), source(up), n, K, M, f, f2};
                const RowAlign al = RowAlign().add(gate.p, gate.ld, 2).add(up.p, up.ld, 2);
                if (mn) return al.elements(2, 4) == 4 ? few_rows_by_input<T, true>(a, st) : few_rows_by_input<T, false>(a, st);
                return with_alignment(alignment_of(RowAlign(al).add(x.p, x.ld, 2), 2), [&](auto align) { return few_rows<T, decltype(align)::value>(a, st); });
            }
            const GemmPlan plan = plan_gemm(n, M, slices_of(K), mn, true, 2, 1, kRangeSlices);
            uint16_t* px = needs_pack(x, plan.tiles_n) ? ws.take<uint16_t>(packed_elements(x)) : nullptr;
            const bool pack_gate = needs_pack(gate, plan.tiles_m), pack_up = needs_pack(up, plan.tiles_m);
            uint16_t* pg = pack_gate ? ws.take<uint16_t>(packed_elements(gate)) : nullptr;
            uint16_t* pu = pack_up ? ws.take<uint16_t>(packed_elements(up)) : nullptr;
            float* parts = plan.splits > 1 ? ws.take<float>((uint64_t)plan.splits * n * 2 * ((M + 3ull) / 4 * 4)) : nullptr;
            if (!launch) return cudaSuccess;
            PackJob copies[3] = {};
            uint32_t n_copies = 0;
            take_copy(copies, &n_copies, &x, px);
            take_copy(copies, &n_copies, &gate, pg);
            take_copy(copies, &n_copies, &up, pu);
            cudaError_t e = launch_prepare<T>(GradJob{}, copies, st);
            if (e != cudaSuccess) return e;
            f.vec4 = RowAlign().add(f.out, f.ld_out, 2).add(f.z, f.ld_z, 2).add(f2.z, f2.ld_z, 2).elements(2, 4) == 4;
            GemmArgs g = gemm_args(plan, n, M, parts, f, nullptr);
            g.f2 = f2;
            Maps<kGated> maps;
            if (mn ? !encode_all<false, true>(&maps, plan, x, gate, x, up) : !encode_all<false, false>(&maps, plan, x, gate, x, up)) return cudaErrorInvalidValue;
            e = mn ? launch_pairs<T, false, true, kGated>(maps, plan, g, st) : launch_pairs<T, false, false, kGated>(maps, plan, g, st);
            if (e != cudaSuccess || plan.splits == 1) return e;
            return launch_following(finish_gated_kernel<T>, dim3(n, std::min((M + 255) / 256, 64u)), 256, 0, st, parts, plan.splits, n, M, g.part_ld, f, f2);
        });
    });
}

int pink_b200_op_gated_backward(const pink_b200_product_config* cfg, const void* dev_dh, uint64_t ld_dh, const void* dev_x, uint64_t ld_x,
                                const void* dev_gate, uint64_t ld_gate, const void* dev_up, uint64_t ld_up, const void* dev_g, uint64_t ld_g,
                                const void* dev_u, uint64_t ld_u, void* dev_dx, uint64_t ld_dx, void* dev_dgate, uint64_t ld_dgate, void* dev_dup,
                                uint64_t ld_dup, float* dev_dgate_bias, float* dev_dup_bias, void* dev_workspace, uint64_t* workspace_bytes,
                                uint32_t size_only, void* stream)
{
    const int rc = check_gated(cfg, ld_x, ld_gate, ld_up);
    if (rc) return rc;
    const uint32_t n = (uint32_t)cfg->n, K = cfg->inputs, M = cfg->outputs;
    const uint64_t w_rows = cfg->by_input ? K : M;
    const uint32_t w_cols = cfg->by_input ? M : K;
    if (!dev_dgate != !dev_dup) return report_error(PINK_B200_EINVAL, "the gradients of both weights come together");
    if (!dev_dgate_bias != !dev_dup_bias) return report_error(PINK_B200_EINVAL, "the gradients of both biases come together");
    if (ld_dh < M || ld_g < M || ld_u < M || (dev_dx && ld_dx < K) || (dev_dgate && (ld_dgate < w_cols || ld_dup < w_cols)))
        return report_error(PINK_B200_EINVAL, "leading dimension smaller than the row");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (n == 0) {
        if (size_only) { if (workspace_bytes) *workspace_bytes = 0; return PINK_B200_OK; }
        cudaError_t e = cudaSuccess;
        if (dev_dgate) e = cudaMemset2DAsync(dev_dgate, ld_dgate * 2, 0, (size_t)w_cols * 2, w_rows, st);
        if (e == cudaSuccess && dev_dup) e = cudaMemset2DAsync(dev_dup, ld_dup * 2, 0, (size_t)w_cols * 2, w_rows, st);
        if (e == cudaSuccess && dev_dgate_bias) e = cudaMemsetAsync(dev_dgate_bias, 0, (size_t)M * 4, st);
        if (e == cudaSuccess && dev_dup_bias) e = cudaMemsetAsync(dev_dup_bias, 0, (size_t)M * 4, st);
        return launch_status(e, "clearing the gradients");
    }
    if (!dev_dh || !dev_g || !dev_u || (dev_dgate && !dev_x) || (dev_dx && (!dev_gate || !dev_up))) return report_error(PINK_B200_EINVAL, "null argument");
    const bool mn = cfg->by_input != 0;
    return with_workspace(dev_workspace, workspace_bytes, size_only, "gradient of gated projections", [&](Arena& ws, bool launch) {
        return with_half_type(cfg->type, [&](auto t) {
            using T = decltype(t);
            auto source = [&](const void* p, uint64_t ld) { return Source{static_cast<const uint16_t*>(p), ld, n, M}; };
            Matrix x{dev_x, ld_x, n, K}, gate{dev_gate, ld_gate, w_rows, w_cols}, up{dev_up, ld_up, w_rows, w_cols};
            Matrix dg{nullptr, packed_ld(M), n, M}, du = dg;
            const bool products = dev_dx || dev_dgate;
            GradJob job{};
            if (!products && !dev_dgate_bias) return cudaSuccess;
            job.dh = source(dev_dh, ld_dh);
            job.g = source(dev_g, ld_g);
            job.u = source(dev_u, ld_u);
            job.act = cfg->activation;
            job.col_blocks = std::min((M + 255) / 256, 4096u);
            job.rows = (uint64_t)(n / 32) * job.col_blocks < 2ull * sm_count() ? 8 : 32;      // (a row a warp where that fills the SMs no better)
            job.row_blocks = (n + job.rows - 1) / job.rows;
            job.ld = dg.ld;
            if (products) {
                dg.p = job.dg = ws.take<uint16_t>(packed_elements(dg));
                du.p = job.du = ws.take<uint16_t>(packed_elements(du));
            }
            if (dev_dgate_bias) {
                job.gate_sums = ws.take<float>((uint64_t)job.row_blocks * M);
                job.up_sums = ws.take<float>((uint64_t)job.row_blocks * M);
            }
            if (products && cfg->type == PINK_B200_F16) {
                const uint64_t pieces = (uint64_t)n * ((M + 255ull) / 256);
                job.peak_count = (uint32_t)std::min<uint64_t>(4ull * sm_count(), (pieces + 7) / 8);
                job.peaks = ws.take<uint32_t>(job.peak_count);
                job.unscale = ws.take<float>(1);
            }
            const uint32_t half_slices = slices_of(M);
            GemmPlan plan_x{}, plan_w{};
            uint16_t *pg = nullptr, *pu = nullptr, *px = nullptr;
            float *parts_x = nullptr, *parts_w = nullptr;
            const uint32_t rows_w = mn ? K : M, cols_w = mn ? M : K;
            if (dev_dx) {
                plan_x = plan_gemm(n, K, 2 * half_slices, !mn, true, 1, 1, kRangeSlices);
                if (needs_pack(gate, plan_x.tiles_m)) pg = ws.take<uint16_t>(packed_elements(gate));
                if (needs_pack(up, plan_x.tiles_m)) pu = ws.take<uint16_t>(packed_elements(up));
                if (plan_x.splits > 1) parts_x = ws.take<float>((uint64_t)plan_x.splits * n * ((K + 3ull) / 4 * 4));
            }
            if (dev_dgate) {
                plan_w = plan_gemm(rows_w, cols_w, slices_of(n), true, true, 1, 2, kRangeSlices);
                if (needs_pack(x, 2 * (mn ? plan_w.tiles_n : plan_w.tiles_m))) px = ws.take<uint16_t>(packed_elements(x));
                if (plan_w.splits > 1) parts_w = ws.take<float>(2ull * plan_w.splits * rows_w * ((cols_w + 3ull) / 4 * 4));
            }
            if (!launch) return cudaSuccess;
            PackJob copies[3] = {};
            uint32_t n_copies = 0;
            take_copy(copies, &n_copies, &gate, pg);
            take_copy(copies, &n_copies, &up, pu);
            take_copy(copies, &n_copies, &x, px);
            cudaError_t e = cudaSuccess;
            if (job.peak_count) e = launch_following(gated_peak_kernel<T>, dim3(job.peak_count), 256, 0, st, job);
            if (e == cudaSuccess) e = launch_prepare<T>(job, copies, st);
            if (e == cudaSuccess && dev_dx) {
                Finish f{};
                f.out = dev_dx; f.ld_out = ld_dx; f.unscale = job.unscale;
                f.vec4 = vec4_rows(f, 2);
                GemmArgs g = gemm_args(plan_x, n, K, parts_x, f, nullptr);
                g.first_slices = half_slices;
                Maps<kSum> maps;
                if (mn ? !encode_all<false, false>(&maps, plan_x, dg, gate, du, up) : !encode_all<false, true>(&maps, plan_x, dg, gate, du, up)) return cudaErrorInvalidValue;
                e = mn ? launch_pairs<T, false, false, kSum>(maps, plan_x, g, st) : launch_pairs<T, false, true, kSum>(maps, plan_x, g, st);
                if (e == cudaSuccess && plan_x.splits > 1)
                    e = launch_following(finish_kernel<T>, dim3(n, std::min((K + 1023) / 1024, 64u)), 256, 0, st, parts_x, plan_x.splits, n, K, g.part_ld, f);
            }
            if (e == cudaSuccess && dev_dgate) {
                Finish f{}, f2{};
                f.out = dev_dgate; f.ld_out = ld_dgate; f.unscale = job.unscale;
                f2.out = dev_dup; f2.ld_out = ld_dup; f2.unscale = job.unscale;
                f.vec4 = vec4_rows(f, 2);
                f2.vec4 = vec4_rows(f2, 2);
                GemmArgs g = gemm_args(plan_w, rows_w, cols_w, parts_w, f, nullptr);
                g.f2 = f2;
                Maps<kTwo> maps;
                if (mn ? !encode_all<true, true>(&maps, plan_w, x, dg, x, du) : !encode_all<true, true>(&maps, plan_w, dg, x, du, x)) return cudaErrorInvalidValue;
                e = launch_pairs<T, true, true, kTwo>(maps, plan_w, g, st);
                if (plan_w.splits > 1)
                    for (int second = 0; second < 2 && e == cudaSuccess; ++second)
                        e = launch_following(finish_kernel<T>, dim3(rows_w, std::min((cols_w + 1023) / 1024, 64u)), 256, 0, st,
                                             parts_w + (size_t)second * plan_w.splits * rows_w * g.part_ld, plan_w.splits, rows_w, cols_w, g.part_ld, second ? f2 : f);
            }
            if (e == cudaSuccess && dev_dgate_bias)
                e = launch_following(gated_dbias_kernel, dim3((M + 31) / 32, 2), 256, 0, st, job.gate_sums, job.up_sums, job.row_blocks, M, dev_dgate_bias, dev_dup_bias);
            return e;
        });
    });
}

} // extern "C"
