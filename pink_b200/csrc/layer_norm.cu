// Layer norm and its gradient (pink_b200_op_layer_norm*).
//
//   m = mean of a row, s = 1 / sqrt(variance + eps), h = (x - m) s, y = h w + b
//   g = dy w,  dx = s (g - mean(g) - h mean(g h)) + r,  dw = column sums of dy h,  db = column sums of dy
//
// Both are bound by memory: a row is read once and kept in registers.  The variance is summed over (x - m)^2, not as a difference of
// sums, and what the rounding of m leaves in every element of a row -- as much as the whole spread where a row lies far from zero -- is
// summed beside it and taken out again: mean(x - m) in the forward pass, mean(h) in the backward pass.
#include "readout.cuh"

#include <algorithm>

namespace pinkb {
namespace {

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

// A row in the registers of LANES lanes (rows of a block side by side) or of a block (LANES 0), CH chunks a thread, chunks of a row dealt in turn.
template <typename T, int LANES, int CH, bool WHOLE>
__global__ void __launch_bounds__(LANES ? 256 : 1024) norm_kernel(const NormArgs a)
{
    constexpr uint32_t V = kChunk<T>;
    __shared__ float scratch[2][32][2];
    const uint32_t threads = LANES ? LANES : blockDim.x, t = LANES ? threadIdx.x % threads : threadIdx.x;
    const uint64_t row = LANES ? (uint64_t)blockIdx.x * (256 / threads) + threadIdx.x / threads : blockIdx.x;
    const bool there = row < a.n;
    const Rows<Raw<T>> x{ static_cast<const Raw<T>*>(a.x), a.ld_x, a.n, a.D };
    Piece<T, WHOLE> in[CH];
    follow();
#pragma unroll
    for (int i = 0; i < CH; ++i)
        if (there && (t + i * threads) * V < a.D) in[i].load(x, row, (t + i * threads) * V);
    float f[CH][V], s1[2] = { 0.0f, 0.0f };
#pragma unroll
    for (int i = 0; i < CH; ++i) {
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) f[i][v] = 0.0f;
        if (there && (t + i * threads) * V < a.D) in[i].floats(f[i]);          // (zeros beyond the row's end)
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) s1[0] += f[i][v];
    }
    row_sums<LANES>(s1, scratch, 0);
    const float mean = s1[0] / (float)a.D;
    float s2[2] = { 0.0f, 0.0f };
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t c = (t + i * threads) * V;
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            f[i][v] = c + v < a.D ? f[i][v] - mean : 0.0f;
            s2[0] += f[i][v];
            s2[1] = fmaf(f[i][v], f[i][v], s2[1]);
        }
    }
    row_sums<LANES>(s2, scratch, 1);
    const float away = s2[0] / (float)a.D;
    const float rstd = 1.0f / sqrtf(fmaxf(s2[1] / (float)a.D - away * away, 0.0f) + a.eps);
    if (!there) return;
    if (t == 0 && a.mean) a.mean[row] = mean + away;
    if (t == 0 && a.rstd) a.rstd[row] = rstd;
    T* y = static_cast<T*>(a.y) + row * a.ld_y;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const uint32_t c = (t + i * threads) * V;
        if (c >= a.D) break;
        float w[V], b[V];
        load_vector<V>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
        load_vector<V>(a.bias, c, a.D - c, a.whole_w, 0.0f, b);
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) f[i][v] = fmaf((f[i][v] - away) * rstd, w[v], b[v]);
        store_chunk(y + c, f[i], a.D - c, a.whole_y);
    }
}

// Rows that do not fit the registers of a block: three passes, of which the second and third find the row in L2.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(1024) norm_long_kernel(const NormArgs a)
{
    constexpr uint32_t V = kChunk<T>;
    __shared__ float scratch[2][32][2];
    const uint64_t row = blockIdx.x;
    const Rows<Raw<T>> x{ static_cast<const Raw<T>*>(a.x), a.ld_x, a.n, a.D };
    follow();
    auto each = [&](auto fn) {
        for (uint32_t c = threadIdx.x * V; c < a.D; c += 1024 * V) {
            Piece<T, WHOLE> in;
            in.load(x, row, c);
            float f[V];
            in.floats(f);
            fn(f, c);
        }
    };
    float s1[2] = { 0.0f, 0.0f }, s2[2] = { 0.0f, 0.0f };
    each([&](float (&f)[V], uint32_t) {
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) s1[0] += f[v];
    });
    block_sums(s1, scratch, 0);
    const float mean = s1[0] / (float)a.D;
    each([&](float (&f)[V], uint32_t c) {
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            const float d = c + v < a.D ? f[v] - mean : 0.0f;
            s2[0] += d;
            s2[1] = fmaf(d, d, s2[1]);
        }
    });
    block_sums(s2, scratch, 1);
    const float away = s2[0] / (float)a.D;
    const float rstd = 1.0f / sqrtf(fmaxf(s2[1] / (float)a.D - away * away, 0.0f) + a.eps);
    if (threadIdx.x == 0 && a.mean) a.mean[row] = mean + away;
    if (threadIdx.x == 0 && a.rstd) a.rstd[row] = rstd;
    T* y = static_cast<T*>(a.y) + row * a.ld_y;
    each([&](float (&f)[V], uint32_t c) {
        float w[V], b[V];
        load_vector<V>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
        load_vector<V>(a.bias, c, a.D - c, a.whole_w, 0.0f, b);
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) f[v] = fmaf(((f[v] - mean) - away) * rstd, w[v], b[v]);
        store_chunk(y + c, f, a.D - c, a.whole_y);
    });
}

// dx of a chunk, given the sums of its row.
template <uint32_t V>
__device__ __forceinline__ void input_gradient(const float (&g)[V], const float (&h)[V], float c1, float c2, float rstd, float (&d)[V])
{
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) d[v] = rstd * fmaf(-h[v], c2, g[v] - c1);
}

// The gradient; a thread keeps its columns from row to row and adds up what they give for weight and bias.  The next row's elements are
// on their way while a row is summed.
template <typename T, int LANES, int CH, bool WHOLE>
__global__ void __launch_bounds__(LANES ? 256 : 1024) norm_grad_kernel(const NormGradArgs a)
{
    constexpr uint32_t V = kChunk<T>, kGroups = LANES ? 256 / LANES : 1;
    __shared__ float scratch[2][32][3];
    __shared__ float meet[LANES ? kGroups : 1][LANES ? LANES * CH * V : 1];
    const uint32_t threads = LANES ? LANES : blockDim.x, t = LANES ? threadIdx.x % threads : threadIdx.x;
    const uint32_t group = LANES ? threadIdx.x / threads : 0;
    const uint64_t step = (uint64_t)gridDim.x * kGroups;
    const Rows<Raw<T>> x{ static_cast<const Raw<T>*>(a.x), a.ld_x, a.n, a.D }, dy{ static_cast<const Raw<T>*>(a.dy), a.ld_dy, a.n, a.D };
    const Rows<Raw<T>> res{ static_cast<const Raw<T>*>(a.residual), a.ld_residual, a.n, a.D };
    float dw[CH][V], db[CH][V];
#pragma unroll
    for (int i = 0; i < CH; ++i)
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) dw[i][v] = db[i][v] = 0.0f;
    Piece<T, WHOLE> px[CH], pd[CH];
    float mean = 0.0f, rstd = 0.0f;
    follow();
    const uint64_t first = (uint64_t)blockIdx.x * kGroups;
    auto fetch = [&](uint64_t r) {
        if (r >= a.n) return;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const uint32_t c = (t + i * threads) * V;
            if (c < a.D) { px[i].load(x, r, c); pd[i].load(dy, r, c); }
        }
        mean = a.mean[r];
        rstd = a.rstd[r];
    };
    fetch(first + group);
    uint32_t turn = 0;
    for (uint64_t r0 = first; r0 < a.n; r0 += step, ++turn) {        // (all groups of a block take as many steps: their lanes meet)
        const uint64_t r = r0 + group;
        const bool there = r < a.n;
        float g[CH][V], h[CH][V], s[3] = { 0.0f, 0.0f, 0.0f };
        const float rs = rstd;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const uint32_t c = (t + i * threads) * V;
            if (there && c < a.D) {
                px[i].floats(h[i]);
                pd[i].floats(g[i]);
#pragma unroll
                for (uint32_t v = 0; v < V; ++v) h[i][v] = c + v < a.D ? (h[i][v] - mean) * rs : 0.0f;
            } else {
#pragma unroll
                for (uint32_t v = 0; v < V; ++v) h[i][v] = g[i][v] = 0.0f;
            }
        }
        fetch(r + step);
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const uint32_t c = (t + i * threads) * V;
            float w[V];
            if (c < a.D) load_vector<V>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
            else
#pragma unroll
                for (uint32_t v = 0; v < V; ++v) w[v] = 0.0f;
#pragma unroll
            for (uint32_t v = 0; v < V; ++v) {
                const float gw = g[i][v] * w[v];
                s[0] += gw;
                s[1] = fmaf(gw, h[i][v], s[1]);
                s[2] += h[i][v];
            }
        }
        row_sums<LANES>(s, scratch, turn);
        const float off = s[2] / (float)a.D, c1 = s[0] / (float)a.D, c2 = s[1] / (float)a.D - c1 * off;
        if (!there) continue;
        T* dx = a.dx ? static_cast<T*>(a.dx) + r * a.ld_dx : nullptr;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            const uint32_t c = (t + i * threads) * V;
            if (c >= a.D) break;
            float w[V], d[V];
            load_vector<V>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
#pragma unroll
            for (uint32_t v = 0; v < V; ++v) {
                h[i][v] -= off;
                dw[i][v] = fmaf(g[i][v], h[i][v], dw[i][v]);
                db[i][v] += g[i][v];
                w[v] *= g[i][v];
            }
            if (!dx) continue;
            input_gradient<V>(w, h[i], c1, c2, rs, d);
            if (a.residual) {
                Piece<T, WHOLE> pr;
                pr.load(res, r, c);
                float add[V];
                pr.floats(add);
#pragma unroll
                for (uint32_t v = 0; v < V; ++v) d[v] += add[v];
            }
            store_chunk(dx + c, d, a.D - c, a.whole_dx);
        }
    }
    if (!a.dweight) return;
    for (int both = 0; both < 2; ++both) {
        float* out = (both ? a.dbias : a.dweight) + (size_t)blockIdx.x * a.D;
        if constexpr (LANES == 0) {
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (uint32_t v = 0; v < V; ++v) {
                    const uint32_t c = (t + i * threads) * V + v;
                    if (c < a.D) out[c] = both ? db[i][v] : dw[i][v];
                }
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < CH; ++i)
#pragma unroll
                for (uint32_t v = 0; v < V; ++v) meet[group][(t + i * threads) * V + v] = both ? db[i][v] : dw[i][v];
            __syncthreads();
            for (uint32_t c = threadIdx.x; c < a.D; c += 256) {
                float s = 0.0f;
#pragma unroll 8
                for (uint32_t q = 0; q < kGroups; ++q) s += meet[q][c];
                out[c] = s;
            }
        }
    }
}

// Rows that do not fit the registers of a block, first half: mean(g), mean(g h) and mean(h) of every row.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(1024) norm_grad_means_kernel(const NormGradArgs a, float* means)
{
    constexpr uint32_t V = kChunk<T>;
    __shared__ float scratch[2][32][3];
    const uint64_t row = blockIdx.x;
    const Rows<Raw<T>> x{ static_cast<const Raw<T>*>(a.x), a.ld_x, a.n, a.D }, dy{ static_cast<const Raw<T>*>(a.dy), a.ld_dy, a.n, a.D };
    follow();
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s[3] = { 0.0f, 0.0f, 0.0f };
#pragma unroll 2
    for (uint32_t c = threadIdx.x * V; c < a.D; c += 1024 * V) {
        Piece<T, WHOLE> px, pd;
        px.load(x, row, c);
        pd.load(dy, row, c);
        float h[V], g[V], w[V];
        px.floats(h);
        pd.floats(g);
        load_vector<V>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            const float hv = c + v < a.D ? (h[v] - mean) * rstd : 0.0f, gw = g[v] * w[v];
            s[0] += gw;
            s[1] = fmaf(gw, hv, s[1]);
            s[2] += hv;
        }
    }
    block_sums(s, scratch, 0);
    if (threadIdx.x == 0) {
        const float off = s[2] / (float)a.D, c1 = s[0] / (float)a.D;
        means[3 * row] = c1;
        means[3 * row + 1] = s[1] / (float)a.D - c1 * off;
        means[3 * row + 2] = off;
    }
}

// Second half: a block takes 256 chunks' columns and every gridDim.y-th row.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(256) norm_grad_long_kernel(const NormGradArgs a, const float* means)
{
    constexpr uint32_t V = kChunk<T>;
    const Rows<Raw<T>> x{ static_cast<const Raw<T>*>(a.x), a.ld_x, a.n, a.D }, dy{ static_cast<const Raw<T>*>(a.dy), a.ld_dy, a.n, a.D };
    const Rows<Raw<T>> res{ static_cast<const Raw<T>*>(a.residual), a.ld_residual, a.n, a.D };
    const uint64_t c64 = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * V;
    follow();
    if (c64 >= a.D) return;
    const uint32_t c = (uint32_t)c64;
    float w[V], dw[V], db[V];
    load_vector<V>(a.weight, c, a.D - c, a.whole_w, 1.0f, w);
#pragma unroll
    for (uint32_t v = 0; v < V; ++v) dw[v] = db[v] = 0.0f;
#pragma unroll 2
    for (uint64_t r = blockIdx.y; r < a.n; r += gridDim.y) {
        Piece<T, WHOLE> px, pd;
        px.load(x, r, c);
        pd.load(dy, r, c);
        const float mean = a.mean[r], rstd = a.rstd[r], c1 = means[3 * r], c2 = means[3 * r + 1], off = means[3 * r + 2];
        float h[V], g[V], d[V];
        px.floats(h);
        pd.floats(g);
#pragma unroll
        for (uint32_t v = 0; v < V; ++v) {
            h[v] = (h[v] - mean) * rstd - off;
            dw[v] = fmaf(g[v], h[v], dw[v]);
            db[v] += g[v];
            g[v] *= w[v];
        }
        if (!a.dx) continue;
        input_gradient<V>(g, h, c1, c2, rstd, d);
        if (a.residual) {
            Piece<T, WHOLE> pr;
            pr.load(res, r, c);
            float add[V];
            pr.floats(add);
#pragma unroll
            for (uint32_t v = 0; v < V; ++v) d[v] += add[v];
        }
        store_chunk(static_cast<T*>(a.dx) + r * a.ld_dx + c, d, a.D - c, a.whole_dx);
    }
    if (!a.dweight) return;
#pragma unroll
    for (uint32_t v = 0; v < V; ++v)
        if (c + v < a.D) {
            a.dweight[(size_t)blockIdx.y * a.D + c + v] = dw[v];
            a.dbias[(size_t)blockIdx.y * a.D + c + v] = db[v];
        }
}

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

// How a row of D elements of `size` bytes is dealt to threads: lanes of a warp (0: a block of `threads`), chunks a thread.
struct Deal { uint32_t lanes, threads; };

int norm_args(uint32_t type, uint32_t D, uint64_t n)
{
    if (type > PINK_B200_F16) return report_error(PINK_B200_EINVAL, "unknown element type");
    if (D == 0 || D > kMaxRow) return report_error(PINK_B200_EINVAL, "a row must have 1 to 16777216 elements");
    if (n > 0x7FFFFFFFull) return report_error(PINK_B200_EINVAL, "too many rows");
    return PINK_B200_OK;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

uint32_t whole_warps(uint32_t chunks) { return (chunks + 31) / 32 * 32; }

template <typename T, bool WHOLE>
cudaError_t run_norm(const NormArgs& a, cudaStream_t st)
{
    const uint32_t chunks = (a.D + kChunk<T> - 1) / kChunk<T>;
    auto lanes = [&](auto kernel, uint32_t per_row) {
        const uint64_t rows = 256 / per_row;
        return launch_following(kernel, dim3((unsigned)((a.n + rows - 1) / rows)), 256, 0, st, a);
    };
    constexpr int kFour = 32 / kChunk<T>;                // chunks of 32 elements
    if (chunks <= 8) return lanes(norm_kernel<T, 8, 1, WHOLE>, 8);
    if (chunks <= 32) return lanes(norm_kernel<T, 32, 1, WHOLE>, 32);
    if (a.D <= 1024) return lanes(norm_kernel<T, 32, kFour, WHOLE>, 32);
    if (a.D <= 16384) return launch_following(norm_kernel<T, 0, kFour / 2, WHOLE>, dim3((unsigned)a.n), whole_warps((chunks + kFour / 2 - 1) / (kFour / 2)), 0, st, a);
    return launch_following(norm_long_kernel<T, WHOLE>, dim3((unsigned)a.n), 1024, 0, st, a);
}

int norm_sms()
{
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms > 0 ? sms : 148;
}

// Blocks (rows of partial sums) of the gradient.
struct NormGradPlan { uint32_t lanes, threads, parts; bool is_long; };

NormGradPlan plan_norm_grad(uint32_t type, uint32_t D, uint64_t n)
{
    const uint32_t V = 16 / (uint32_t)element_size(type), chunks = (D + V - 1) / V, sms = (uint32_t)norm_sms();
    NormGradPlan p{};
    if (chunks <= 8) p.lanes = 8;
    else if (chunks <= 32) p.lanes = 32;
    if (p.lanes) {
        p.threads = 256;
        const uint64_t rows = 256 / p.lanes;
        p.parts = (uint32_t)std::min<uint64_t>((n + rows - 1) / rows, 4 * sms);
    } else if (D <= 8192) {
        p.threads = whole_warps((D + 7) / 8);
        p.parts = (uint32_t)std::min<uint64_t>(n, (uint64_t)sms * (1024 / p.threads));
    } else {
        p.is_long = true;
        p.threads = 256;
        const uint64_t columns = (chunks + 255) / 256;
        p.parts = (uint32_t)std::min<uint64_t>((n + 7) / 8, std::max<uint64_t>(1, 8 * sms / columns));
    }
    return p;
}

template <typename T, bool WHOLE>
cudaError_t run_norm_grad(const NormGradArgs& a, const NormGradPlan& p, float* means, cudaStream_t st)
{
    if (p.lanes == 8) return launch_following(norm_grad_kernel<T, 8, 1, WHOLE>, dim3(p.parts), p.threads, 0, st, a);
    if (p.lanes == 32) return launch_following(norm_grad_kernel<T, 32, 1, WHOLE>, dim3(p.parts), p.threads, 0, st, a);
    if (!p.is_long) return launch_following(norm_grad_kernel<T, 0, 8 / kChunk<T>, WHOLE>, dim3(p.parts), p.threads, 0, st, a);
    const cudaError_t e = launch_following(norm_grad_means_kernel<T, WHOLE>, dim3((unsigned)a.n), 1024, 0, st, a, means);
    if (e != cudaSuccess) return e;
    const uint64_t chunks = (a.D + kChunk<T> - 1) / kChunk<T>;
    return launch_following(norm_grad_long_kernel<T, WHOLE>, dim3((unsigned)((chunks + 255) / 256), p.parts), p.threads, 0, st, a, means);
}

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
        const bool whole = RowAlign().add(dev_x, ld_x, sizeof(T)).elements(sizeof(T), kChunk<T>) == kChunk<T>;
        cudaStream_t st = static_cast<cudaStream_t>(stream);
        return whole ? run_norm<T, true>(a, st) : run_norm<T, false>(a, st);
    }), "layer norm");
}

int pink_b200_op_layer_norm_backward(uint32_t type, uint32_t dims, uint64_t n, const void* dev_dy, uint64_t ld_dy, const void* dev_x, uint64_t ld_x,
                                     const float* dev_mean, const float* dev_rstd, const float* dev_weight, const void* dev_residual,
                                     uint64_t ld_residual, void* dev_dx, uint64_t ld_dx, float* dev_dweight, float* dev_dbias, void* dev_workspace,
                                     uint64_t* workspace_bytes, uint32_t size_only, void* stream)
{
    const int rc = norm_args(type, dims, n);
    if (rc) return rc;
    if (ld_dy < dims || ld_x < dims || (dev_residual && ld_residual < dims) || (dev_dx && ld_dx < dims))
        return report_error(PINK_B200_EINVAL, "leading dimension smaller than the row");
    if (!dev_dweight != !dev_dbias) return report_error(PINK_B200_EINVAL, "the gradients of weight and bias come together");
    if (size_only && !workspace_bytes) return report_error(PINK_B200_EINVAL, "null argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (n == 0) {
        if (size_only) { *workspace_bytes = 0; return PINK_B200_OK; }
        cudaError_t e = cudaSuccess;
        if (dev_dweight) e = cudaMemsetAsync(dev_dweight, 0, (size_t)dims * 4, st);
        if (e == cudaSuccess && dev_dbias) e = cudaMemsetAsync(dev_dbias, 0, (size_t)dims * 4, st);
        return launch_status(e, "clearing the gradients");
    }
    const NormGradPlan plan = plan_norm_grad(type, dims, n);
    const uint64_t sums = dev_dweight ? ((uint64_t)plan.parts * dims * 4 + 255) / 256 * 256 : 0;
    const uint64_t need = 2 * sums + (plan.is_long ? n * 12 : 0);
    if (size_only) { *workspace_bytes = need; return PINK_B200_OK; }
    if (!dev_dy || !dev_x || !dev_mean || !dev_rstd) return report_error(PINK_B200_EINVAL, "null argument");
    if (need && (!dev_workspace || !workspace_bytes || *workspace_bytes < need)) return report_error(PINK_B200_EINVAL, "workspace too small (ask with size_only)");
    if (need && !aligned16(dev_workspace)) return report_error(PINK_B200_EINVAL, "the workspace must be 16-byte aligned");
    if (!dev_dx && !dev_dweight) return PINK_B200_OK;
    uint8_t* ws = static_cast<uint8_t*>(dev_workspace);
    float* dw = dev_dweight ? reinterpret_cast<float*>(ws) : nullptr;
    float* db = dev_dweight ? reinterpret_cast<float*>(ws + sums) : nullptr;
    cudaError_t e = with_type(type, [&](auto t) {
        using T = decltype(t);
        NormGradArgs a{dev_dy, ld_dy, dev_x, ld_x, dev_mean, dev_rstd, dev_weight, dev_residual, ld_residual, dev_dx, ld_dx, dw, db, n, dims, 0, 0};
        a.whole_dx = RowAlign().add(dev_dx, ld_dx, sizeof(T)).elements(sizeof(T), kChunk<T>) == kChunk<T>;
        a.whole_w = aligned16(dev_weight);
        const bool whole = RowAlign().add(dev_dy, ld_dy, sizeof(T)).add(dev_x, ld_x, sizeof(T)).add(dev_residual, ld_residual, sizeof(T))
                               .elements(sizeof(T), kChunk<T>) == kChunk<T>;
        float* means = reinterpret_cast<float*>(ws + 2 * sums);
        return whole ? run_norm_grad<T, true>(a, plan, means, st) : run_norm_grad<T, false>(a, plan, means, st);
    });
    if (e == cudaSuccess && dev_dweight)
        e = launch_following(norm_columns_kernel, dim3((dims + 31) / 32, 2), 256, 0, st, dw, db, plan.parts, dims, dev_dweight, dev_dbias);
    return launch_status(e, "layer norm gradient");
}

} // extern "C"
