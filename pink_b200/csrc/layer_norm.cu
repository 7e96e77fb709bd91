// Layer norm and its gradient (pink_b200_op_layer_norm*).
//
//   m = mean of a row, s = 1 / sqrt(variance + eps), h = (x - m) s, y = h w + b
//   g = dy w,  dx = s (g - mean(g) - h mean(g h)) + r,  dw = column sums of dy h,  db = column sums of dy
//
// Both are bound by memory: a row is read once and kept in registers.  The squares are summed about m as rounded, or a number
// within two standard deviations of it, so that the variance is no difference of large sums; and what that number leaves in every element of a row -- as
// much as the whole spread where a row lies far from zero -- is summed beside it and taken out again: mean(x - m) in the forward pass, mean(h) in the backward pass.
//
// The kernels of an element type are a module of their own (PINK_NORM_TYPE = 0, 1, 2: float32, bfloat16, float16), so that a process
// loads what it uses; without the macro this file holds the entry points.
#include "ring.cuh"

#include <algorithm>

namespace pinkb {

struct NormArgs
{
    const void* x; uint64_t ld_x;
    const float *weight, *bias;
    void* y; uint64_t ld_y;
    float *mean, *rstd;
    uint64_t n;
    uint32_t D;
    float eps;
    uint32_t whole_y, whole_w;       // rows of y, and weight and bias, start on 16-byte boundaries
};

struct NormGradArgs
{
    const void* dy; uint64_t ld_dy;
    const void* x; uint64_t ld_x;
    const float *mean, *rstd, *weight;
    const void* residual; uint64_t ld_residual;
    void* dx; uint64_t ld_dx;
    float *dweight, *dbias;          // [blocks][D] each: sums of a block's rows; null: not asked for
    uint64_t n;
    uint32_t D;
    uint32_t whole_dx, whole_w;
};

// The means that a row's sums stand for: of g, of g h, and what the rounding of the row's mean has left in h.
struct Means { float c1, c2, off; };

// Which kernel takes the gradient, and its blocks: as many rows of partial sums.
struct NormGradPlan { uint32_t lanes, threads, parts, smem, per; };

// align: of the rows that are read (kAny, kEight, kSixteen).
template <typename T> cudaError_t run_norm(const NormArgs& a, int align, cudaStream_t st);
template <typename T> cudaError_t run_norm_grad(const NormGradArgs& a, const NormGradPlan& p, int align, Means* means, cudaStream_t st);

#ifdef PINK_NORM_TYPE

namespace {

// kChunk numbers of a float32 vector from col on, `left` of them inside it; what is beyond is `rest`.
template <uint32_t N>
__device__ __forceinline__ void load_vector(const float* p, uint32_t col, uint32_t left, bool whole, float rest, float (&f)[N])
{
    if (!p) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) f[i] = rest;
    } else if (whole && left >= N) {
#pragma unroll
        for (uint32_t i = 0; i < N; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + col + i);
            f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) f[i] = i < left ? p[col + i] : rest;
    }
}

// Sums over the threads of a row: LANES of a warp, or (0) the whole block.
template <int LANES, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], float (*scratch)[32][N], uint32_t turn)
{
    if constexpr (LANES == 0) {
        block_sums(v, scratch, turn);
    } else {
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
    }
}

// weight and bias of a chunk, as pairs.
template <typename T>
__device__ __forceinline__ void load_pairs(const float* p, uint32_t col, uint32_t left, bool whole, float rest, F2 (&f)[kPairs<T>])
{
    float v[kChunk<T>];
    load_vector<kChunk<T>>(p, col, left, whole, rest, v);
#pragma unroll
    for (int i = 0; i < kPairs<T>; ++i) f[i] = two(v[2 * i], v[2 * i + 1]);
}

template <typename T>
__device__ __forceinline__ void pairs_of(const uint4& c, F2 (&f)[kPairs<T>])
{
#pragma unroll
    for (int j = 0; j < kPairs<T>; ++j) f[j] = pair_of<T>(c, j);
}

// The moments of a row in one pass: sums of d = x - shift and of d^2, where the shift is the mean of eight elements spread over the row, each read by a
// lane of every warp.  The variance is then a difference, and good while the square of the sums' mean is not far above it; where it is (outliers among
// the eight, so hardly ever) a second pass takes the row's own mean as the shift.  It begins with the elements themselves, read again: x - shift has been
// rounded in steps of the far shift, beside which ordinary elements have lost their last bits.
constexpr uint32_t kSamples = 8;
constexpr float kFar = 4.0f;                             // (mean d)^2 over the variance from where the second pass runs: below it the difference loses log2(1 + 4) = 2.3 bits at most

__device__ __forceinline__ uint32_t sample_of(uint32_t D) { return (uint32_t)((uint64_t)(2 * (threadIdx.x % kSamples) + 1) * D / (2 * kSamples)); }

__device__ __forceinline__ float shift_of(float v)         // (v: the lane's sample)
{
    v *= 1.0f / kSamples;                                // (before the sum: a row of fewer elements than samples may be in range where eight of them are not)
#pragma unroll
    for (uint32_t o = kSamples / 2; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Adds a chunk's d = x - shift to the sums; what is beyond the row's end counts as zero.
template <typename T>
__device__ __forceinline__ void moments(F2 (&d)[kPairs<T>], F2 minus, uint32_t left, F2& s, F2& q)
{
#pragma unroll
    for (int j = 0; j < kPairs<T>; ++j) {
        d[j] = add2(d[j], minus);
        if (left < kChunk<T>) d[j] = two(2 * j < left ? d[j].lo() : 0.0f, 2 * j + 1 < left ? d[j].hi() : 0.0f);
        s = add2(s, d[j]);
        q = fma2(d[j], d[j], q);
    }
}

__device__ __forceinline__ bool far_off(const float (&s)[2], float inv_d)
{
    const float m = s[0] * inv_d;
    return m * m > kFar * fmaf(-m, m, s[1] * inv_d);
}

__device__ __forceinline__ float rstd_of(const float (&s)[2], float inv_d, float eps)
{
    const float m = s[0] * inv_d, var = fmaf(-m, m, s[1] * inv_d);
    return rsqrtf((var < 0.0f ? 0.0f : var) + eps);      // (a NaN stays)
}

// The second pass of a block's row, and what follows it, from memory.  (A call, so that the kernel's own way holds neither registers nor instructions for it: inline, a block of
// 384 threads took eleven registers more, two blocks an SM instead of three.)
template <typename T, int ALIGN>
__device__ __noinline__ void norm_far_row(const NormArgs& a, uint64_t row, float mean, float (*scratch)[32][2])
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int P = kPairs<T>;
    const RowOf<T, ALIGN> x(a.x, a.ld_x, row, a.n, a.D);
    const float inv_d = 1.0f / (float)a.D;
    F2 d[P], s2 = two(0.0f), q2 = two(0.0f);
#pragma unroll 1
    for (uint32_t c = threadIdx.x * V; c < a.D; c += blockDim.x * V) {
        pairs_of<T>(x.all(x.load(c)), d);
        moments<T>(d, two(-mean), a.D - c, s2, q2);
    }
    float s[2] = { s2.lo() + s2.hi(), q2.lo() + q2.hi() };
    block_sums(s, scratch, 1);
    const float rstd = rstd_of(s, inv_d, a.eps), away = s[0] * inv_d;
    if (threadIdx.x == 0 && a.mean) a.mean[row] = mean + away;
    if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
    T* y = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll 1
    for (uint32_t c = threadIdx.x * V; c < a.D; c += blockDim.x * V) {
        F2 w[P], b[P];
        load_pairs<T>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
        load_pairs<T>(a.bias, c, a.D - c, a.whole_w, 0.0f, b);
        pairs_of<T>(x.all(x.load(c)), d);
#pragma unroll
        for (int j = 0; j < P; ++j) d[j] = fma2(mul2(add2(add2(d[j], two(-mean)), two(-away)), two(rstd)), w[j], b[j]);
        store_pairs<T>(y + c, d, a.D - c, a.whole_y);
    }
}

// A row in the registers of LANES lanes (rows of a block side by side) or of a block (LANES 0), CH chunks a thread, chunks of a row dealt in turn.
template <typename T, int LANES, int CH, int ALIGN>
__global__ void __launch_bounds__(LANES ? 256 : 512) norm_kernel(const __grid_constant__ NormArgs a)
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int P = kPairs<T>;
    using In = RowOf<T, ALIGN>;
    __shared__ float scratch[2][32][2];
    const uint32_t threads = LANES ? LANES : blockDim.x, t = LANES ? threadIdx.x % threads : threadIdx.x;
    const uint64_t at = LANES ? (uint64_t)blockIdx.x * (256 / threads) + threadIdx.x / threads : blockIdx.x, row = min(at, a.n - 1);
    follow();
    const In in(a.x, a.ld_x, row, a.n, a.D);             // (rows behind the last repeat it, and are not written)
    typename In::Chunk on_way[CH];
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if ((t + i * threads) * V < a.D) on_way[i] = in.load((t + i * threads) * V);
    const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
    float shift = shift_of(to_float(x[sample_of(a.D)]));   // (a row is at least eight lanes': all samples are its own)
    const float inv_d = 1.0f / (float)a.D;
    F2 d[CH][P], s2 = two(0.0f), q2 = two(0.0f);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t c = (t + i * threads) * V;
        if (c >= a.D) break;
        const uint4 v = in.all(on_way[i]);
#pragma unroll
        for (int j = 0; j < P; ++j) d[i][j] = pair_of<T>(v, j);
        moments<T>(d[i], two(-shift), a.D - c, s2, q2);
    }
    float s[2] = { s2.lo() + s2.hi(), q2.lo() + q2.hi() };
    row_sums<LANES>(s, scratch, 0);
    const bool far = far_off(s, inv_d);
    // (rows that share a warp meet in its sums; each keeps its own, so that no row depends on the others)
    if (__builtin_expect(LANES > 0 ? __any_sync(0xFFFFFFFFu, far) : far, 0)) {
        if (far) shift += s[0] * inv_d;
        if constexpr (LANES == 0) {
            norm_far_row<T, ALIGN>(a, row, shift, scratch);
            return;
        }
        s2 = q2 = two(0.0f);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const uint32_t c = (t + i * threads) * V;
            if (!far || c >= a.D) break;
            pairs_of<T>(in.all(in.load(c)), d[i]);
            moments<T>(d[i], two(-shift), a.D - c, s2, q2);
        }
        float own[2] = { s2.lo() + s2.hi(), q2.lo() + q2.hi() };
        row_sums<LANES>(own, scratch, 1);
        if (far) { s[0] = own[0]; s[1] = own[1]; }
    }
    const float rstd = rstd_of(s, inv_d, a.eps), away = s[0] * inv_d;
    if (at >= a.n) return;
    if (t == 0) {
        if (a.mean) a.mean[row] = shift + away;
        if (a.rstd) a.rstd[row] = rstd;
    }
    T* y = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t c = (t + i * threads) * V;
        if (c >= a.D) break;
        F2 w[P], b[P];
        load_pairs<T>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
        load_pairs<T>(a.bias, c, a.D - c, a.whole_w, 0.0f, b);
#pragma unroll
        for (int j = 0; j < P; ++j) d[i][j] = fma2(mul2(add2(d[i][j], two(-away)), two(rstd)), w[j], b[j]);
        store_pairs<T>(y + c, d[i], a.D - c, a.whole_y);
    }
}

// Rows that do not fit the registers of a block: three passes, of which the second and third find the row in L2.
template <typename T, int ALIGN>
__global__ void __launch_bounds__(1024) norm_long_kernel(const NormArgs a)
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int P = kPairs<T>;
    __shared__ float scratch[2][32][2];
    const uint64_t row = blockIdx.x;
    const RowOf<T, ALIGN> x(a.x, a.ld_x, row, a.n, a.D);
    follow();
    auto each = [&](auto fn) {
#pragma unroll 2
        for (uint32_t c = threadIdx.x * V; c < a.D; c += 1024 * V) fn(x.all(x.load(c)), c);
    };
    float s1[2] = { 0.0f, 0.0f }, s2[2] = { 0.0f, 0.0f };
    each([&](uint4 v, uint32_t) {
#pragma unroll
        for (int j = 0; j < P; ++j) { const F2 f = pair_of<T>(v, j); s1[0] += f.lo() + f.hi(); }
    });
    block_sums(s1, scratch, 0);
    const float mean = s1[0] / (float)a.D;
    each([&](uint4 v, uint32_t c) {
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const F2 f = pair_of<T>(v, j);
            const float d0 = c + 2 * j < a.D ? f.lo() - mean : 0.0f, d1 = c + 2 * j + 1 < a.D ? f.hi() - mean : 0.0f;
            s2[0] += d0 + d1;
            s2[1] = fmaf(d0, d0, fmaf(d1, d1, s2[1]));
        }
    });
    block_sums(s2, scratch, 1);
    const float away = s2[0] / (float)a.D;
    const float var = s2[1] / (float)a.D - away * away, rstd = rsqrtf((var < 0.0f ? 0.0f : var) + a.eps);
    if (threadIdx.x == 0 && a.mean) a.mean[row] = mean + away;
    if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
    T* y = static_cast<T*>(a.y) + row * a.ld_y;
    each([&](uint4 v, uint32_t c) {
        F2 w[P], b[P], f[P];
        load_pairs<T>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
        load_pairs<T>(a.bias, c, a.D - c, a.whole_w, 0.0f, b);
#pragma unroll
        for (int j = 0; j < P; ++j) f[j] = fma2(mul2(add2(add2(pair_of<T>(v, j), two(-mean)), two(-away)), two(rstd)), w[j], b[j]);
        store_pairs<T>(y + c, f, a.D - c, a.whole_y);
    });
}

// Many rows: weight and bias stay in registers.  Measured, 65,536 x 3,969 bfloat16 at odd places: 220 us (4.7 TB/s); 510 instructions a warp and row, so bound by issue and by
// the latency of a row's one barrier at four blocks an SM.  With 16 columns a thread 286 us, with five blocks (100 registers, spills) 297.  Whole chunks are dealt to the threads in turn; the fewer than V elements behind the last go one to a
// lane of the first warp, and (CH - 1) threads <= chunks, so that only a thread's last slot has to look for the row's end.  (__grid_constant__: 32,768 x 4,096 bfloat16 in
// 100 us, 109 with the arguments by value; 16,384 x 8,100 float32 186, 197.)
template <typename T, int CH, int ALIGN>
__global__ void __launch_bounds__(512) norm_ring_kernel(const __grid_constant__ NormArgs a)
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int P = kPairs<T>;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float scratch[2][32][2];
    const uint32_t t = threadIdx.x, threads = blockDim.x, stage = staged_bytes(a.D, sizeof(T)), chunks = a.D / V, rest = a.D % V;
    const uint32_t step = gridDim.x, n = (uint32_t)a.n;
    const float inv_d = 1.0f / (float)a.D;
    const bool one = t < rest;
    F2 w[CH][P], b[CH][P];
    float w1 = 1.0f, b1 = 0.0f;
    follow();
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t c = (t + i * threads) * V;
#pragma unroll
        for (int j = 0; j < P; ++j) w[i][j] = b[i][j] = two(0.0f);
        if (i + 1 < CH || t + i * threads < chunks) {
            load_pairs<T>(a.weight, c, V, a.whole_w, 1.0f, w[i]);
            load_pairs<T>(a.bias, c, V, a.whole_w, 0.0f, b[i]);
        }
    }
    if (one) {
        if (a.weight) w1 = a.weight[chunks * V + t];
        if (a.bias) b1 = a.bias[chunks * V + t];
    }
    uint32_t r = blockIdx.x, ahead = r;
    Staged<T, CH> x(a.x, a.ld_x, r, step, a.D, smem_u32(ring), threads);
    auto copy = [&](uint32_t slot) {
        if (ahead < n) x.copy(slot * stage, ahead > 0, ahead + 1 < n);
        ahead += step;
        copies_committed();
    };
    for (uint32_t i = 0; i + 1 < kRing; ++i) copy(i);
    copies_waited<kRing - 2>();
    __syncthreads();
    T* y = static_cast<T*>(a.y) + r * a.ld_y + t * V;
    const uint64_t y_pace = step * a.ld_y;
    const uint32_t sample = sample_of(a.D) * (uint32_t)sizeof(T), last = (chunks * V + t) * (uint32_t)sizeof(T);
    uint32_t slot = 0, turn = 0;
    for (; r < n; r += step, slot = slot + 1 == kRing ? 0 : slot + 1, y += y_pace) {
        const uint32_t here = x.place(slot * stage);
        F2 d[CH][P];
        float d1 = 0.0f;
        float shift = shift_of(staged_element<T>(here + sample));
        float s[2];
        auto sums = [&] {
            F2 s2 = two(0.0f), q2 = two(0.0f);
#pragma unroll
            for (int i = 0; i < CH; ++i)
                if (i + 1 < CH || t + i * threads < chunks) {
                    pairs_of<T>(staged_chunk<T, ALIGN>(here + (t + i * threads) * 16), d[i]);
                    moments<T>(d[i], two(-shift), V, s2, q2);
                }
            s[0] = s2.lo() + s2.hi();
            s[1] = q2.lo() + q2.hi();
            if (one) {
                d1 = staged_element<T>(here + last) - shift;
                s[0] += d1;
                s[1] = fmaf(d1, d1, s[1]);
            }
        };
        sums();
        copies_waited<kRing - 3>();                      // this thread's part of the next row is there
        block_sums(s, scratch, turn++);
        if (__builtin_expect(far_off(s, inv_d), 0)) {    // (the row's stage is filled again behind the next row's barrier)
            shift += s[0] * inv_d;
            sums();
            block_sums(s, scratch, turn++);
        }
        const float rstd = rstd_of(s, inv_d, a.eps), away = s[0] * inv_d;
        if (t == 0) {
            if (a.mean) a.mean[r] = shift + away;
            if (a.rstd) a.rstd[r] = rstd;
        }
        const F2 minus = two(-away), by = two(rstd);
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i + 1 < CH || t + i * threads < chunks) {
#pragma unroll
                for (int j = 0; j < P; ++j) d[i][j] = fma2(mul2(add2(d[i][j], minus), by), w[i][j], b[i][j]);
                store_pairs<T>(y + i * threads * V, d[i], V, true);
            }
        if (one) y[(chunks - t) * V + t] = from_float<T>(fmaf((d1 - away) * rstd, w1, b1));
        copy(slot == 0 ? kRing - 1 : slot - 1);
        x.advance();
    }
}

// What a chunk adds to its row's sums -- of g, of g h and of h -- where g = dy w; h is formed on the way.  `left`: elements of the chunk inside the row.
template <typename T>
__device__ __forceinline__ void chunk_sums(const uint4& x, const F2 (&dy)[kPairs<T>], const F2 (&w)[kPairs<T>], float mean, float rstd, uint32_t left,
                                           F2 (&h)[kPairs<T>], F2 (&s)[3])
{
#pragma unroll
    for (int j = 0; j < kPairs<T>; ++j) {
        h[j] = mul2(add2(pair_of<T>(x, j), two(-mean)), two(rstd));
        if (left < kChunk<T>) h[j] = two(2 * j < left ? h[j].lo() : 0.0f, 2 * j + 1 < left ? h[j].hi() : 0.0f);
        const F2 g = mul2(dy[j], w[j]);
        s[0] = add2(s[0], g);
        s[1] = fma2(g, h[j], s[1]);
        s[2] = add2(s[2], h[j]);
    }
}

__device__ __forceinline__ Means means_of(float g, float gh, float h, float inv_d)
{
    const float c1 = g * inv_d, off = h * inv_d;
    return { c1, fmaf(gh, inv_d, -c1 * off), off };
}

// dx of a chunk, and what it adds to the columns' sums.
template <typename T>
__device__ __forceinline__ void chunk_gradient(const F2 (&h)[kPairs<T>], const F2 (&dy)[kPairs<T>], const F2 (&w)[kPairs<T>], const Means& m, float rstd,
                                               F2 (&dw)[kPairs<T>], F2 (&db)[kPairs<T>], F2 (&d)[kPairs<T>])
{
#pragma unroll
    for (int j = 0; j < kPairs<T>; ++j) {
        const F2 hj = add2(h[j], two(-m.off));
        dw[j] = fma2(dy[j], hj, dw[j]);
        db[j] = add2(db[j], dy[j]);
        d[j] = mul2(two(rstd), fma2(hj, two(-m.c2), fma2(dy[j], w[j], two(-m.c1))));
    }
}

template <typename T, int ALIGN>
__device__ __forceinline__ void add_residual(const NormGradArgs& a, uint64_t row, uint32_t c, F2 (&d)[kPairs<T>])
{
    const RowOf<T, ALIGN> r(a.residual, a.ld_residual, row, a.n, a.D);
    const uint4 v = r.all(r.load(c));
#pragma unroll
    for (int j = 0; j < kPairs<T>; ++j) d[j] = add2(d[j], pair_of<T>(v, j));
}

// Short rows, LANES lanes each, a chunk a lane.  A thread keeps its columns from row to row and adds up what they give for weight and bias.  The next row's
// elements are on their way while a row is summed.
template <typename T, int LANES, int ALIGN>
__global__ void __launch_bounds__(256) norm_grad_kernel(const NormGradArgs a)
{
    constexpr uint32_t V = kChunk<T>, kGroups = 256 / LANES;
    constexpr int P = kPairs<T>;
    using In = RowOf<T, ALIGN>;
    __shared__ float meet[kGroups][LANES * V];
    const uint32_t t = threadIdx.x % LANES, group = threadIdx.x / LANES, c = t * V;
    const uint64_t first = (uint64_t)blockIdx.x * kGroups, step = (uint64_t)gridDim.x * kGroups;
    const bool mine = c < a.D;
    const uint32_t left = mine ? a.D - c : 0;
    F2 dw[P], db[P], w[P];
#pragma unroll
    for (int j = 0; j < P; ++j) dw[j] = db[j] = w[j] = two(0.0f);
    follow();
    if (mine) load_pairs<T>(a.weight, c, left, a.whole_w, 1.0f, w);
    uint4 px = make_uint4(0, 0, 0, 0), pd = px;
    float mean = 0.0f, rstd = 0.0f;
    auto fetch = [&](uint64_t r) {
        if (r >= a.n || !mine) return;
        const In x(a.x, a.ld_x, r, a.n, a.D), dy(a.dy, a.ld_dy, r, a.n, a.D);
        const typename In::Chunk cx = x.load(c), cd = dy.load(c);
        px = x.all(cx);
        pd = dy.all(cd);
        mean = a.mean[r];
        rstd = a.rstd[r];
    };
    fetch(first + group);
    for (uint64_t r0 = first; r0 < a.n; r0 += step) {    // (all groups of a block take as many steps: their lanes meet)
        const uint64_t r = r0 + group;
        const bool there = r < a.n && mine;
        const float rs = rstd;
        F2 h[P], g[P], s2[3] = { two(0.0f), two(0.0f), two(0.0f) };
        pairs_of<T>(pd, g);
        chunk_sums<T>(px, g, w, mean, rs, left, h, s2);
        float s[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) s[i] = there ? s2[i].lo() + s2[i].hi() : 0.0f;
        fetch(r + step);
#pragma unroll
        for (int o = LANES / 2; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < 3; ++i) s[i] += __shfl_xor_sync(0xFFFFFFFFu, s[i], o);
        if (!there) continue;
        F2 d[P];
        chunk_gradient<T>(h, g, w, means_of(s[0], s[1], s[2], 1.0f / (float)a.D), rs, dw, db, d);
        if (!a.dx) continue;
        if (a.residual) add_residual<T, ALIGN>(a, r, c, d);
        store_pairs<T>(static_cast<T*>(a.dx) + r * a.ld_dx + c, d, left, a.whole_dx);
    }
    if (!a.dweight) return;
    for (int both = 0; both < 2; ++both) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < P; ++j) {
            const F2 v = both ? db[j] : dw[j];
            meet[group][c + 2 * j] = v.lo();
            meet[group][c + 2 * j + 1] = v.hi();
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < a.D; i += 256) {
            float s = 0.0f;
#pragma unroll 8
            for (uint32_t q = 0; q < kGroups; ++q) s += meet[q][i];
            (both ? a.dbias : a.dweight)[(size_t)blockIdx.x * a.D + i] = s;
        }
    }
}

// Sixteen columns a thread at most (their sums, 32 numbers, stay in registers: one block of 512 threads an SM).  Measured, 16,384 x 8,100 bfloat16 with a residual: 250 us
// (4.2 TB/s), bound by issue and three sums a row over 16 warps; with 8 columns and 1,024 threads 346.  Chunks and the elements behind them as in norm_ring_kernel.
template <typename T, int CH, int ALIGN>
__global__ void __launch_bounds__(512, 1) norm_grad_ring_kernel(const NormGradArgs a)
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int P = kPairs<T>;
    extern __shared__ __align__(16) uint8_t ring[];      // [kRing][x, dy, residual]
    __shared__ float scratch[2][32][3];
    const uint32_t t = threadIdx.x, threads = blockDim.x, bytes = staged_bytes(a.D, sizeof(T)), stage = (a.residual ? 3 : 2) * bytes;
    const uint32_t chunks = a.D / V, rest = a.D % V;
    const uint32_t step = gridDim.x, n = (uint32_t)a.n;
    const float inv_d = 1.0f / (float)a.D;
    const bool one = t < rest;
    F2 dw[CH][P], db[CH][P], w[CH][P];
    float dw1 = 0.0f, db1 = 0.0f, w1 = 1.0f;
    follow();
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
        for (int j = 0; j < P; ++j) dw[i][j] = db[i][j] = w[i][j] = two(0.0f);
        if (i + 1 < CH || t + i * threads < chunks) load_pairs<T>(a.weight, (t + i * threads) * V, V, a.whole_w, 1.0f, w[i]);
    }
    if (one && a.weight) w1 = a.weight[chunks * V + t];
    uint32_t r = blockIdx.x, ahead = r;
    Staged<T, CH> x(a.x, a.ld_x, r, step, a.D, smem_u32(ring), threads), dy(a.dy, a.ld_dy, r, step, a.D, smem_u32(ring) + bytes, threads);
    Staged<T, CH> res(a.residual, a.ld_residual, r, step, a.D, smem_u32(ring) + 2 * bytes, threads);
    auto copy = [&](uint32_t slot) {
        if (ahead < n) {
            const bool before = ahead > 0, behind = ahead + 1 < n;
            x.copy(slot * stage, before, behind);
            dy.copy(slot * stage, before, behind);
            if (a.residual) res.copy(slot * stage, before, behind);
        }
        ahead += step;
        copies_committed();
    };
    for (uint32_t i = 0; i + 1 < kRing; ++i) copy(i);
    copies_waited<kRing - 2>();
    auto row_stat = [&](const float* p, uint32_t row) { return row < n ? p[row] : 0.0f; };
    float mean = row_stat(a.mean, r), rstd = row_stat(a.rstd, r), mean1 = row_stat(a.mean, r + step), rstd1 = row_stat(a.rstd, r + step);      // (two rows ahead)
    __syncthreads();
    T* dx = static_cast<T*>(a.dx) + r * a.ld_dx + t * V;
    const uint64_t dx_pace = step * a.ld_dx;
    const uint32_t last = (chunks * V + t) * (uint32_t)sizeof(T);
    uint32_t slot = 0, turn = 0;
    for (; r < n; r += step, slot = slot + 1 == kRing ? 0 : slot + 1, ++turn, dx += dx_pace) {
        const uint32_t at = slot * stage, here_x = x.place(at), here_d = dy.place(at);
        const float rs = rstd;
        F2 h[CH][P], g[CH][P], s2[3] = { two(0.0f), two(0.0f), two(0.0f) };
        float h1 = 0.0f, g1 = 0.0f;
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i + 1 < CH || t + i * threads < chunks) {
                const uint32_t g16 = (t + i * threads) * 16;
                const uint4 vx = staged_chunk<T, ALIGN>(here_x + g16), vd = staged_chunk<T, ALIGN>(here_d + g16);
                pairs_of<T>(vd, g[i]);
                chunk_sums<T>(vx, g[i], w[i], mean, rs, V, h[i], s2);
            }
        float s[3] = { s2[0].lo() + s2[0].hi(), s2[1].lo() + s2[1].hi(), s2[2].lo() + s2[2].hi() };
        if (one) {
            g1 = staged_element<T>(here_d + last);
            h1 = (staged_element<T>(here_x + last) - mean) * rs;
            s[0] += g1 * w1;
            s[1] = fmaf(g1 * w1, h1, s[1]);
            s[2] += h1;
        }
        mean = mean1;
        rstd = rstd1;
        mean1 = row_stat(a.mean, r + 2 * step);
        rstd1 = row_stat(a.rstd, r + 2 * step);
        copies_waited<kRing - 3>();                      // this thread's part of the next row is there
        block_sums(s, scratch, turn);
        const Means m = means_of(s[0], s[1], s[2], inv_d);
        const uint32_t here_r = res.place(at);
#pragma unroll
        for (int i = 0; i < CH; ++i)
            if (i + 1 < CH || t + i * threads < chunks) {
                F2 d[P];
                chunk_gradient<T>(h[i], g[i], w[i], m, rs, dw[i], db[i], d);
                if (a.residual) {
                    const uint4 v = staged_chunk<T, ALIGN>(here_r + (t + i * threads) * 16);
#pragma unroll
                    for (int j = 0; j < P; ++j) d[j] = add2(d[j], pair_of<T>(v, j));
                }
                store_pairs<T>(dx + i * threads * V, d, V, true);
            }
        if (one) {
            h1 -= m.off;
            dw1 = fmaf(g1, h1, dw1);
            db1 += g1;
            const float d1 = rs * fmaf(-h1, m.c2, fmaf(g1, w1, -m.c1));
            dx[(chunks - t) * V + t] = from_float<T>(d1 + (a.residual ? staged_element<T>(here_r + last) : 0.0f));
        }
        copy(slot == 0 ? kRing - 1 : slot - 1);
        x.advance();
        dy.advance();
        res.advance();
    }
    if (!a.dweight) return;
    float *pw = a.dweight + (size_t)blockIdx.x * a.D, *pb = a.dbias + (size_t)blockIdx.x * a.D;
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (i + 1 < CH || t + i * threads < chunks)
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const uint32_t c = (t + i * threads) * V + 2 * j;
                pw[c] = dw[i][j].lo(); pb[c] = db[i][j].lo();
                pw[c + 1] = dw[i][j].hi(); pb[c + 1] = db[i][j].hi();
            }
    if (one) { pw[chunks * V + t] = dw1; pb[chunks * V + t] = db1; }
}

// Rows that are too long for that, first half: the means of every row.
template <typename T, int ALIGN>
__global__ void __launch_bounds__(512) norm_grad_means_kernel(const NormGradArgs a, Means* means)
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int P = kPairs<T>;
    __shared__ float scratch[2][32][3];
    const uint64_t row = blockIdx.x;
    const RowOf<T, ALIGN> x(a.x, a.ld_x, row, a.n, a.D), dy(a.dy, a.ld_dy, row, a.n, a.D);
    follow();
    const float mean = a.mean[row], rstd = a.rstd[row];
    F2 s2[3] = { two(0.0f), two(0.0f), two(0.0f) };
#pragma unroll 2
    for (uint32_t c = threadIdx.x * V; c < a.D; c += 512 * V) {
        const auto cx = x.load(c);
        const auto cd = dy.load(c);
        F2 h[P], g[P], w[P];
        load_pairs<T>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
        pairs_of<T>(dy.all(cd), g);
        chunk_sums<T>(x.all(cx), g, w, mean, rstd, a.D - c, h, s2);
    }
    float s[3] = { s2[0].lo() + s2[0].hi(), s2[1].lo() + s2[1].hi(), s2[2].lo() + s2[2].hi() };
    block_sums(s, scratch, 0);
    if (threadIdx.x == 0) means[row] = means_of(s[0], s[1], s[2], 1.0f / (float)a.D);
}

// Second half: a block takes 256 chunks' columns and every gridDim.y-th row.
template <typename T, int ALIGN>
__global__ void __launch_bounds__(256) norm_grad_long_kernel(const NormGradArgs a, const Means* means)
{
    constexpr uint32_t V = kChunk<T>;
    constexpr int P = kPairs<T>;
    const uint64_t c64 = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * V;
    follow();
    if (c64 >= a.D) return;
    const uint32_t c = (uint32_t)c64;
    F2 w[P], dw[P], db[P];
    load_pairs<T>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
#pragma unroll
    for (int j = 0; j < P; ++j) dw[j] = db[j] = two(0.0f);
#pragma unroll 2
    for (uint64_t r = blockIdx.y; r < a.n; r += gridDim.y) {
        const RowOf<T, ALIGN> x(a.x, a.ld_x, r, a.n, a.D), dy(a.dy, a.ld_dy, r, a.n, a.D);
        const auto cx = x.load(c);
        const auto cd = dy.load(c);
        const float mean = a.mean[r], rstd = a.rstd[r];
        const Means m = means[r];
        F2 h[P], g[P], d[P];
        const uint4 v = x.all(cx);
        pairs_of<T>(dy.all(cd), g);
#pragma unroll
        for (int j = 0; j < P; ++j) h[j] = mul2(add2(pair_of<T>(v, j), two(-mean)), two(rstd));
        chunk_gradient<T>(h, g, w, m, rstd, dw, db, d);
        if (!a.dx) continue;
        if (a.residual) add_residual<T, ALIGN>(a, r, c, d);
        store_pairs<T>(static_cast<T*>(a.dx) + r * a.ld_dx + c, d, a.D - c, a.whole_dx);
    }
    if (!a.dweight) return;
    float *pw = a.dweight + (size_t)blockIdx.y * a.D, *pb = a.dbias + (size_t)blockIdx.y * a.D;
#pragma unroll
    for (int j = 0; j < P; ++j) {
        if (c + 2 * j < a.D) { pw[c + 2 * j] = dw[j].lo(); pb[c + 2 * j] = db[j].lo(); }
        if (c + 2 * j + 1 < a.D) { pw[c + 2 * j + 1] = dw[j].hi(); pb[c + 2 * j + 1] = db[j].hi(); }
    }
}

template <typename T, int ALIGN>
cudaError_t run_norm_at(const NormArgs& a, cudaStream_t st)
{
    const uint32_t chunks = (a.D + kChunk<T> - 1) / kChunk<T>;
    auto lanes = [&](auto kernel, uint32_t per_row) {
        const uint64_t rows = 256 / per_row;
        return launch_following(kernel, dim3((unsigned)((a.n + rows - 1) / rows)), 256, 0, st, a);
    };
    if (chunks <= 8) return lanes(norm_kernel<T, 8, 1, ALIGN>, 8);
    if (chunks <= 32) return lanes(norm_kernel<T, 32, 1, ALIGN>, 32);
    const uint32_t sms = (uint32_t)sm_count(), smem = kRing * staged_bytes(a.D, sizeof(T)), whole = a.D / kChunk<T>;
    // (eight rows an SM or more: 3,969 bfloat16 at 4, 8, 16 and 64 rows an SM 4.9, 6.8, 11.4 and 36.8 us through the ring, 4.8, 6.8, 12.8 and 43.2 in registers; 2,791 float32 4.8, 7.3,
    // 12.1 and 38.4 for 5.0, 8.3, 13.8 and 45.4; 1,000 bfloat16 3.0, 3.5, 5.3 and 9.5 for 3.3, 3.5, 4.0 and 10.8)
    if (a.n >= 8 * sms && a.whole_y && smem <= kRingSmem) {
        auto ring = [&](auto kernel, uint32_t threads) { return launch_ring(kernel, a.n, threads, smem, st, a); };
        constexpr int MANY = 32 / kChunk<T>, FEW = 2;
        if (const uint32_t t = ring_threads(whole, MANY)) return ring(norm_ring_kernel<T, MANY, ALIGN>, t);
        if (const uint32_t t = ring_threads(whole, FEW)) return ring(norm_ring_kernel<T, FEW, ALIGN>, t);
    }
    if (chunks <= 128) return lanes(norm_kernel<T, 32, 4, ALIGN>, 32);
    if (chunks <= 4 * 512) return launch_following(norm_kernel<T, 0, 4, ALIGN>, dim3((unsigned)a.n), whole_warps((chunks + 3) / 4), 0, st, a);
    return launch_following(norm_long_kernel<T, ALIGN>, dim3((unsigned)a.n), 1024, 0, st, a);
}

template <typename T, int ALIGN>
cudaError_t run_norm_grad_at(const NormGradArgs& a, const NormGradPlan& p, Means* means, cudaStream_t st)
{
    if (p.lanes == 8) return launch_following(norm_grad_kernel<T, 8, ALIGN>, dim3(p.parts), p.threads, 0, st, a);
    if (p.lanes == 32) return launch_following(norm_grad_kernel<T, 32, ALIGN>, dim3(p.parts), p.threads, 0, st, a);
    if (p.smem) {
        auto ring = [&](auto kernel) {
            const cudaError_t e = allow_shared(kernel, p.smem, kRingSmem);
            return e != cudaSuccess ? e : launch_following(kernel, dim3(p.parts), p.threads, p.smem, st, a);
        };
        return p.per == 2 ? ring(norm_grad_ring_kernel<T, 2, ALIGN>) : ring(norm_grad_ring_kernel<T, 16 / kChunk<T>, ALIGN>);
    }
    const cudaError_t e = launch_following(norm_grad_means_kernel<T, ALIGN>, dim3((unsigned)a.n), 512, 0, st, a, means);
    if (e != cudaSuccess) return e;
    const uint64_t chunks = (a.D + kChunk<T> - 1) / kChunk<T>;
    return launch_following(norm_grad_long_kernel<T, ALIGN>, dim3((unsigned)((chunks + 255) / 256), p.parts), p.threads, 0, st, a, means);
}

} // namespace

template <typename T>
cudaError_t run_norm(const NormArgs& a, int align, cudaStream_t st)
{
    return with_alignment(align, [&](auto at) { return run_norm_at<T, decltype(at)::value>(a, st); });
}

template <typename T>
cudaError_t run_norm_grad(const NormGradArgs& a, const NormGradPlan& p, int align, Means* means, cudaStream_t st)
{
    return with_alignment(align, [&](auto at) { return run_norm_grad_at<T, decltype(at)::value>(a, p, means, st); });
}

#if PINK_NORM_TYPE == 0
using NormType = float;
#elif PINK_NORM_TYPE == 1
using NormType = __nv_bfloat16;
#else
using NormType = __half;
#endif
template cudaError_t run_norm<NormType>(const NormArgs&, int, cudaStream_t);
template cudaError_t run_norm_grad<NormType>(const NormGradArgs&, const NormGradPlan&, int, Means*, cudaStream_t);

} // namespace pinkb

#else // PINK_NORM_TYPE

namespace {

// Column sums of the blocks' sums: a block takes 32 columns, its eight warps the parts in turn.
__global__ void __launch_bounds__(256) norm_columns_kernel(const float* dw_parts, const float* db_parts, uint32_t parts, uint32_t D, float* dweight, float* dbias)
{
    __shared__ float meet[8][32];
    follow();
    const float* src = blockIdx.y ? db_parts : dw_parts;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float s = 0.0f;
    if (c < D)
#pragma unroll 8
        for (uint32_t p = warp; p < parts; p += 8) s += src[(size_t)p * D + c];
    meet[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < D) {
#pragma unroll
        for (int q = 1; q < 8; ++q) s += meet[q][lane];
        (blockIdx.y ? dbias : dweight)[c] = s;
    }
}

// ---- host side -------------------------------------------------------------------------------------------------------------

constexpr uint32_t kMaxRow = 1u << 24;

int norm_args(uint32_t type, uint32_t D, uint64_t n)
{
    if (type > PINK_B200_F16) return report_error(PINK_B200_EINVAL, "unknown element type");
    if (D == 0 || D > kMaxRow) return report_error(PINK_B200_EINVAL, "a row must have 1 to 16777216 elements");
    if (n > 0x7FFFFFFFull) return report_error(PINK_B200_EINVAL, "too many rows");
    return PINK_B200_OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

NormGradPlan plan_norm_grad(uint32_t type, uint32_t D, uint64_t n, bool residual, bool whole_dx)
{
    const uint32_t size = (uint32_t)element_size(type), V = 16 / size, chunks = (D + V - 1) / V, sms = (uint32_t)sm_count();
    NormGradPlan p{};
    if (chunks <= 32) {
        p.lanes = chunks <= 8 ? 8 : 32;
        p.threads = 256;
        const uint64_t rows = 256 / p.lanes;
        p.parts = (uint32_t)std::min<uint64_t>((n + rows - 1) / rows, 4 * sms);
        return p;
    }
    const uint64_t smem = (uint64_t)kRing * (residual ? 3 : 2) * staged_bytes(D, size);
    const uint32_t many = 16 / V, whole = D / V;
    p.per = ring_threads(whole, many) ? many : ring_threads(whole, 2) ? 2 : 0;
    if (p.per && smem <= kRingSmem && whole_dx) {
        p.threads = ring_threads(whole, p.per);
        p.smem = (uint32_t)smem;
        // as many blocks an SM as its registers (128 a thread) and shared memory hold
        const uint32_t blocks = std::min(512 / p.threads, kRingSmem / (p.smem + 2048));
        p.parts = (uint32_t)std::min<uint64_t>(n, (uint64_t)sms * std::max(1u, blocks));
        return p;
    }
    p.threads = 256;
    const uint64_t columns = (chunks + 255) / 256;
    p.parts = (uint32_t)std::min<uint64_t>((n + 7) / 8, std::max<uint64_t>(1, 8 * sms / columns));
    return p;
}

uint64_t sums_bytes(const NormGradPlan& p, uint32_t D) { return ((uint64_t)p.parts * D * 4 + 255) / 256 * 256; }
uint64_t means_bytes(const NormGradPlan& p, uint64_t n) { return p.lanes || p.smem ? 0 : n * sizeof(Means); }

} // namespace
} // namespace pinkb

using namespace pinkb;

extern "C" {

int pink_b200_op_layer_norm(uint32_t type, uint32_t dims, uint64_t n, const void* dev_x, uint64_t ld_x, const float* dev_weight, const float* dev_bias,
                            float eps, void* dev_y, uint64_t ld_y, float* dev_mean, float* dev_rstd, void* stream)
{
    const int rc = norm_args(type, dims, n);
    if (rc) return rc;
    if (!(eps > 0.0f) || !(eps <= FLT_MAX)) return report_error(PINK_B200_EINVAL, "eps must be positive and finite");
    if (ld_x < dims || ld_y < dims) return report_error(PINK_B200_EINVAL, "leading dimension smaller than the row");
    if (n == 0) return PINK_B200_OK;
    if (!dev_x || !dev_y) return report_error(PINK_B200_EINVAL, "null argument");
    return launch_status(with_type(type, [&](auto t) {
        using T = decltype(t);
        NormArgs a{dev_x, ld_x, dev_weight, dev_bias, dev_y, ld_y, dev_mean, dev_rstd, n, dims, eps, 0, 0};
        a.whole_y = RowAlign().add(dev_y, ld_y, sizeof(T)).elements(sizeof(T), kChunk<T>) == kChunk<T>;
        a.whole_w = aligned16(dev_weight) && aligned16(dev_bias);
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        return run_norm<T>(a, alignment_of(RowAlign().add(dev_x, ld_x, sizeof(T)), sizeof(T)), st);
    }), "layer norm");
}

uint64_t pink_b200_layer_norm_workspace(uint32_t type, uint32_t dims, uint64_t n)
{
    if (type > PINK_B200_F16 || dims == 0 || dims > kMaxRow || n == 0 || n > 0x7FFFFFFFull) return 0;
    uint64_t most = 0;
    for (int residual = 0; residual < 2; ++residual)
        for (int whole = 0; whole < 2; ++whole) {
            const NormGradPlan p = plan_norm_grad(type, dims, n, residual != 0, whole != 0);
            most = std::max(most, 2 * sums_bytes(p, dims) + means_bytes(p, n));
        }
    return most;
}

int pink_b200_op_layer_norm_backward(uint32_t type, uint32_t dims, uint64_t n, const void* dev_dy, uint64_t ld_dy, const void* dev_x, uint64_t ld_x,
                                     const float* dev_mean, const float* dev_rstd, const float* dev_weight, const void* dev_residual,
                                     uint64_t ld_residual, void* dev_dx, uint64_t ld_dx, float* dev_dweight, float* dev_dbias, void* dev_workspace,
                                     uint64_t workspace_bytes, void* stream)
{
    const int rc = norm_args(type, dims, n);
    if (rc) return rc;
    if (ld_dy < dims || ld_x < dims || (dev_residual && ld_residual < dims) || (dev_dx && ld_dx < dims))
        return report_error(PINK_B200_EINVAL, "leading dimension smaller than the row");
    if (!dev_dweight != !dev_dbias) return report_error(PINK_B200_EINVAL, "the gradients of weight and bias come together");
    if (dev_dx && dev_dx == dev_residual && n > 1 && ld_dx != ld_residual)
        return report_error(PINK_B200_EINVAL, "dx in the residual's place needs its leading dimension");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (n == 0) {
        cudaError_t e = cudaSuccess;
        if (dev_dweight) e = cudaMemsetAsync(dev_dweight, 0, (size_t)dims * 4, st);
        if (e == cudaSuccess && dev_dbias) e = cudaMemsetAsync(dev_dbias, 0, (size_t)dims * 4, st);
        return launch_status(e, "clearing the gradients");
    }
    if (!dev_dy || !dev_x || !dev_mean || !dev_rstd) return report_error(PINK_B200_EINVAL, "null argument");
    const bool dx_whole = alignment_of(RowAlign().add(dev_dx, ld_dx, element_size(type)), element_size(type)) == kSixteen;
    const NormGradPlan plan = plan_norm_grad(type, dims, n, dev_residual != nullptr, dev_dx && dx_whole);
    const uint64_t sums = dev_dweight ? sums_bytes(plan, dims) : 0, need = 2 * sums + means_bytes(plan, n);
    if (need && (!dev_workspace || workspace_bytes < need)) return report_error(PINK_B200_EINVAL, "workspace too small (pink_b200_layer_norm_workspace)");
    if (need && !aligned16(dev_workspace)) return report_error(PINK_B200_EINVAL, "the workspace must be 16-byte aligned");
    if (!dev_dx && !dev_dweight) return PINK_B200_OK;
    uint8_t* ws = static_cast<uint8_t*>(dev_workspace);
    float* dw = dev_dweight ? reinterpret_cast<float*>(ws) : nullptr;
    float* db = dev_dweight ? reinterpret_cast<float*>(ws + sums) : nullptr;
    cudaError_t e = with_type(type, [&](auto t) {
        using T = decltype(t);
        NormGradArgs a{dev_dy, ld_dy, dev_x, ld_x, dev_mean, dev_rstd, dev_weight, dev_residual, ld_residual, dev_dx, ld_dx, dw, db, n, dims, 0, 0};
        a.whole_dx = dx_whole;
        a.whole_w = aligned16(dev_weight);
        const RowAlign al = RowAlign().add(dev_dy, ld_dy, sizeof(T)).add(dev_x, ld_x, sizeof(T)).add(dev_residual, ld_residual, sizeof(T));
        Means* means = reinterpret_cast<Means*>(ws + 2 * sums);
        return run_norm_grad<T>(a, plan, alignment_of(al, sizeof(T)), means, st);
    });
    if (e == cudaSuccess && dev_dweight)
        e = launch_following(norm_columns_kernel, dim3((dims + 31) / 32, 2), 256, 0, st, dw, db, plan.parts, dims, dev_dweight, dev_dbias);
    return launch_status(e, "layer norm gradient");
}

} // extern "C"

#endif // PINK_NORM_TYPE
