// Shared pieces of the read-out operators (route.cu, read_out.cu, product.cu): element types, argument checks, reductions.
#pragma once
#include "../../include/pink_b200.h"
#include "kernels.cuh"
#include "ptx.cuh"

#include <cfloat>
#include <cstdio>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

} // namespace pinkb
