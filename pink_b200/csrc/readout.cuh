// Shared pieces of the read-out operators and of those that train a head (route.cu, read_out.cu, product.cu, gated.cu, layer_norm.cu, distill.cu): element types,
// rows at any alignment, reductions, launches.
#pragma once
#include "../../include/pink_b200.h"
#include "kernels.cuh"
#include "ptx.cuh"

#include <cfloat>
#include <cstdio>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace pinkb {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// VEC consecutive elements, loaded and stored as one word of VEC * sizeof(T) bytes (the caller has checked the alignment), and held
// packed: an array of 16-bit elements would be loaded one by one.
template <int BYTES> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

template <typename T> struct TwoOf;                      // two 16-bit elements in a register, to and from float
template <> struct TwoOf<__nv_bfloat16>
{
    static __device__ __forceinline__ float2 floats(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
    static __device__ __forceinline__ uint32_t packed(float a, float b)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <> struct TwoOf<__half>
{
    static __device__ __forceinline__ float2 floats(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
    static __device__ __forceinline__ uint32_t packed(float a, float b)
    {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};

template <typename T, int VEC>
struct Pack
{
    using W = typename Word<sizeof(T) * VEC>::type;
    W w;
    static __device__ __forceinline__ Pack load(const T* p) { return Pack{ *reinterpret_cast<const W*>(p) }; }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<W*>(p) = w; }
    __device__ __forceinline__ void floats(float (&f)[VEC]) const
    {
        if constexpr (sizeof(T) * VEC == 2) {
            f[0] = to_float(*reinterpret_cast<const T*>(&w));
        } else {
            const uint32_t* q = reinterpret_cast<const uint32_t*>(&w);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if constexpr (sizeof(T) == 4) {
                    f[v] = __uint_as_float(q[v]);
                } else if (v % 2 == 0) {
                    const float2 two = TwoOf<T>::floats(q[v / 2]);
                    f[v] = two.x;
                    f[v + 1] = two.y;
                }
            }
        }
    }
    static __device__ __forceinline__ Pack of(const float (&f)[VEC])
    {
        Pack p;
        if constexpr (sizeof(T) * VEC == 2) {
            const T h = from_float<T>(f[0]);
            p.w = *reinterpret_cast<const uint16_t*>(&h);
        } else {
            uint32_t* q = reinterpret_cast<uint32_t*>(&p.w);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                if constexpr (sizeof(T) == 4) q[v] = __float_as_uint(f[v]);
                else if (v % 2 == 0) q[v / 2] = TwoOf<T>::packed(f[v], f[v + 1]);
            }
        }
        return p;
    }
};

// A matrix in memory, for reads at any alignment.
template <typename E> struct Rows { const E* p; uint64_t ld; uint64_t rows; uint32_t cols; };

// The 16 bytes of elements that start at col of a row (zero beyond its end).  Rows may start on any element, so two aligned words that cover
// them are loaded and shifted together later: loads of several chunks are then in flight at once.  Where a word would reach beyond the
// matrix, the elements are read one by one.
struct Chunk { uint4 a, b; uint32_t off; };              // off: bytes into `a`

template <typename E>
__device__ __forceinline__ Chunk load_chunk(const Rows<E>& m, uint64_t row, uint32_t col)
{
    constexpr uint32_t kEach = 16 / sizeof(E), kPerWord = 4 / sizeof(E);
    const E* src = m.p + row * m.ld + col;
    const uint32_t off = (uint32_t)reinterpret_cast<uintptr_t>(src) & 15u;
    const E* lo = src - off / sizeof(E);
    if (col + kEach <= m.cols && lo >= m.p && lo + 2 * kEach <= m.p + (m.rows - 1) * m.ld + m.cols)
        return { *reinterpret_cast<const uint4*>(lo), *(reinterpret_cast<const uint4*>(lo) + 1), off };
    uint32_t w[4] = { 0, 0, 0, 0 };
#pragma unroll
    for (uint32_t q = 0; q < kEach; ++q)
        if (col + q < m.cols) w[q / kPerWord] |= (uint32_t)src[q] << (q % kPerWord) * 16;
    return { make_uint4(w[0], w[1], w[2], w[3]), make_uint4(0, 0, 0, 0), 0u };
}

__device__ __forceinline__ uint4 joined(const Chunk& e)
{
    uint32_t w[8] = { e.a.x, e.a.y, e.a.z, e.a.w, e.b.x, e.b.y, e.b.z, e.b.w };
    if (e.off & 8u)
#pragma unroll
        for (int q = 0; q < 6; ++q) w[q] = w[q + 2];
    if (e.off & 4u)
#pragma unroll
        for (int q = 0; q < 5; ++q) w[q] = w[q + 1];
    const uint32_t bits = (e.off & 2u) * 8u;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits), __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

inline size_t element_size(uint32_t type) { return type == PINK_B200_F32 ? 4 : 2; }

// Calls fn with a value of the element type that `type` names.
template <typename Fn>
cudaError_t with_type(uint32_t type, Fn fn)
{
    if (type == PINK_B200_F32) return fn(float());
    if (type == PINK_B200_BF16) return fn(__nv_bfloat16());
    return fn(__half());
}

// Largest power of two of elements (at most `most`) that every listed row start is aligned to.
struct RowAlign
{
    uint64_t bits = 0;
    RowAlign& add(const void* p, uint64_t ld, size_t size)
    {
        if (p) bits |= reinterpret_cast<uintptr_t>(p) | ld * size;
        return *this;
    }
    uint32_t elements(size_t size, uint32_t most) const
    {
        uint32_t v = most;
        while (v > 1 && bits % (v * size)) v >>= 1;
        return v;
    }
};

// Maximum and sum over a warp; every lane gets the result.  The sum's order is fixed.
__device__ __forceinline__ float warp_max(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    return v;
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

// Elements of a 16-byte chunk, and the unsigned word an element is loaded as.
template <typename T> constexpr uint32_t kChunk = 16 / sizeof(T);
template <typename T> using Raw = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;

// ---- rows in registers -------------------------------------------------------------------------------------------------------
// Kernels that keep a row in registers are bound by instructions before they are bound by memory: a row's alignment is looked at once, its
// 16-bit elements stay packed, and arithmetic goes two elements at a time.

// Two floats in a register pair, which one instruction adds or multiplies.  (Held as one word of 64 bits: taken apart and put together again between
// instructions they cost more moves than the pairs save.)
struct F2
{
    unsigned long long w;
    __device__ __forceinline__ float lo() const { float2 f = both(); return f.x; }
    __device__ __forceinline__ float hi() const { float2 f = both(); return f.y; }
    __device__ __forceinline__ float2 both() const
    {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(w));
        return f;
    }
};
__device__ __forceinline__ F2 two(float a, float b)
{
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r.w) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ F2 two(float v) { return two(v, v); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w)); return r; }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.w) : "l"(a.w), "l"(b.w)); return r; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.w) : "l"(a.w), "l"(b.w), "l"(c.w)); return r; }

// Pairs of a chunk, to and from its four words.
template <typename T> constexpr int kPairs = kChunk<T> / 2;
template <typename T> __device__ __forceinline__ uint32_t word_of(const uint4& c, int i) { return i == 0 ? c.x : i == 1 ? c.y : i == 2 ? c.z : c.w; }
template <typename T>
__device__ __forceinline__ F2 pair_of(const uint4& c, int i)
{
    if constexpr (sizeof(T) == 4) {
        return i == 0 ? two(__uint_as_float(c.x), __uint_as_float(c.y)) : two(__uint_as_float(c.z), __uint_as_float(c.w));
    } else {
        const float2 f = TwoOf<T>::floats(word_of<T>(c, i));
        return two(f.x, f.y);
    }
}

// Stores the first `left` elements of a chunk; `whole`: the place is a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void store_pairs(T* p, const F2 (&f)[kPairs<T>], uint32_t left, bool whole)
{
    uint4 c;
    if constexpr (sizeof(T) == 4) c = make_uint4(__float_as_uint(f[0].lo()), __float_as_uint(f[0].hi()), __float_as_uint(f[1].lo()), __float_as_uint(f[1].hi()));
    else c = make_uint4(TwoOf<T>::packed(f[0].lo(), f[0].hi()), TwoOf<T>::packed(f[1].lo(), f[1].hi()), TwoOf<T>::packed(f[2].lo(), f[2].hi()), TwoOf<T>::packed(f[3].lo(), f[3].hi()));
    if (whole && left >= kChunk<T>) {
        *reinterpret_cast<uint4*>(p) = c;
        return;
    }
    // (a loop that stays one: unrolled, its instructions would be issued, without effect, behind every whole chunk)
    Raw<T>* r = reinterpret_cast<Raw<T>*>(p);
#pragma unroll 1
    for (uint32_t i = 0; i < kChunk<T> && i < left; ++i) {
        r[i] = (Raw<T>)c.x;
        constexpr uint32_t kBits = sizeof(T) * 8;
        if constexpr (kBits == 32) c = make_uint4(c.y, c.z, c.w, 0);
        else c = make_uint4(__funnelshift_r(c.x, c.y, kBits), __funnelshift_r(c.y, c.z, kBits), __funnelshift_r(c.z, c.w, kBits), c.w >> kBits);
    }
}

// How rows are aligned: all on 16-byte boundaries, all on 8-byte boundaries, or on any element.
enum : int { kAny = 0, kEight = 8, kSixteen = 16 };

inline int alignment_of(const RowAlign& al, size_t size)
{
    const uint32_t v = al.elements(size, 16 / (uint32_t)size) * (uint32_t)size;
    return v >= 16 ? kSixteen : v >= 8 ? kEight : kAny;
}

// Calls fn with the alignment as a constant.
template <typename Fn>
cudaError_t with_alignment(int align, Fn fn)
{
    if (align == kSixteen) return fn(std::integral_constant<int, kSixteen>());
    if (align == kEight) return fn(std::integral_constant<int, kEight>());
    return fn(std::integral_constant<int, kAny>());
}

// A row, and a chunk of it on its way.  16-bit rows at any alignment: three words of eight bytes cover a chunk and are shifted together
// by all() (two of sixteen would take five instructions more); float32: element by element, in order.
template <typename T, int ALIGN>
struct RowOf
{
    static constexpr bool kShift = ALIGN == kAny && sizeof(T) == 2;
    const Raw<T>* p;
    uint32_t cols, off;              // off: bytes from the 8-byte boundary below
    bool inner;                      // words around the row's ends lie inside the matrix

    __device__ __forceinline__ RowOf(const void* base, uint64_t ld, uint64_t row, uint64_t rows, uint32_t n)
        : p(static_cast<const Raw<T>*>(base) + row * ld), cols(n), off(0), inner(row >= 8 && row + 12 < rows)
    {
        if constexpr (kShift) off = (uint32_t)reinterpret_cast<uintptr_t>(p) & 7u;
    }

    struct Words { uint2 a, b, c; };
    using Chunk = std::conditional_t<kShift, Words, uint4>;

    __device__ __forceinline__ uint4 one_by_one(uint32_t col) const
    {
        if constexpr (sizeof(T) == 4) {
            uint32_t w[4];
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) w[q] = col + q < cols ? p[col + q] : 0;
            return make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            uint32_t w[4] = { 0, 0, 0, 0 };
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q)             // (all on their way at once)
                if (col + q < cols) w[q / 2] |= (uint32_t)p[col + q] << (q & 1) * 16;
            return make_uint4(w[0], w[1], w[2], w[3]);
        }
    }

    // The chunk from col on, zero beyond the row's end; col < cols.
    __device__ __forceinline__ Chunk load(uint32_t col) const
    {
        const bool whole = col + kChunk<T> <= cols;
        if constexpr (ALIGN == kSixteen) {
            return whole ? *reinterpret_cast<const uint4*>(p + col) : one_by_one(col);
        } else if constexpr (ALIGN == kEight) {
            if (!whole) return one_by_one(col);
            const uint2 a = *reinterpret_cast<const uint2*>(p + col), b = *(reinterpret_cast<const uint2*>(p + col) + 1);
            return make_uint4(a.x, a.y, b.x, b.y);
        } else if constexpr (!kShift) {
            return one_by_one(col);
        } else {
            // (a row beside the matrix's ends: its first and last chunks may have words that reach beyond)
            if (whole && (inner || (col >= 8 && col + 16 <= cols))) {
                const uint2* lo = reinterpret_cast<const uint2*>(reinterpret_cast<const char*>(p + col) - off);
                return { lo[0], lo[1], lo[2] };
            }
            const uint4 c = one_by_one(col);
            const uint64_t l = c.x | (uint64_t)c.y << 32, h = c.z | (uint64_t)c.w << 32;
            const uint32_t up = off * 8;
            const uint64_t x = l << up, y = up ? h << up | l >> (64 - up) : h, z = up ? h >> (64 - up) : 0;
            return { make_uint2((uint32_t)x, (uint32_t)(x >> 32)), make_uint2((uint32_t)y, (uint32_t)(y >> 32)), make_uint2((uint32_t)z, (uint32_t)(z >> 32)) };
        }
    }

    __device__ __forceinline__ uint4 all(const Chunk& c) const
    {
        if constexpr (!kShift) {
            return c;
        } else {
            const bool far = off & 4u;
            const uint32_t bits = (off & 2u) * 8u;
            const uint32_t w0 = far ? c.a.y : c.a.x, w1 = far ? c.b.x : c.a.y, w2 = far ? c.b.y : c.b.x, w3 = far ? c.c.x : c.b.y, w4 = far ? c.c.y : c.c.x;
            return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits), __funnelshift_r(w3, w4, bits));
        }
    }
};

// Sums of N numbers over the threads of a block (whole warps), for all of them, in a fixed order.  `scratch` holds [2][32][N]; turn alternates from
// one sum to the next, so that one barrier suffices.
template <int N>
__device__ __forceinline__ void block_sums(float (&v)[N], float (*scratch)[32][N], uint32_t turn)
{
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(v[i]);
    if (warps == 1) {
        __syncwarp();                                    // (orders memory as the barrier does)
        return;
    }
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) scratch[turn & 1][warp][i] = v[i];
    __syncthreads();
    if (warps <= 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = scratch[turn & 1][0][i];
            for (uint32_t w = 1; w < warps; ++w) v[i] += scratch[turn & 1][w][i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = warp_sum(lane < warps ? scratch[turn & 1][lane][i] : 0.0f);
}

constexpr uint32_t kNoNeuron = 0xFFFFFFFFu;

inline int launch_status(cudaError_t e, const char* what)
{
    if (e == cudaSuccess) return PINK_B200_OK;
    cudaGetLastError();
    char msg[256];
    std::snprintf(msg, sizeof(msg), "%s: %s", what, cudaGetErrorString(e));
    return report_error(PINK_B200_ECUDA, msg);
}

// Opts a kernel into `most` bytes of dynamic shared memory where a call may need more than the 48 KB that every launch has, in which the
// kernel's own arrays (of less than 8 KB) count.  The limit is the kernel's, for all threads of the process, so every call asks for the
// same, the largest that any needs: asking for its own it could take away, between another thread's request and launch, what that one has
// asked for.
template <typename... P>
cudaError_t allow_shared(void (*kernel)(P...), size_t bytes, size_t most)
{
    if (bytes <= 40 * 1024) return cudaSuccess;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most);
}

// A launch whose blocks may be set up while the kernel before it in the stream still runs: the kernel starts with follow() (or waits
// later, before it touches global memory), which returns when that one is complete.
template <typename... P, typename... A>
cudaError_t launch_following(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const A&... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

__device__ __forceinline__ void follow()
{
    griddep_launch();                                    // the next kernel's blocks may be set up from now on
    griddep_wait();
}

} // namespace pinkb
