// Rows that pass through shared memory (layer_norm.cu, distill.cu).  Every source that includes this has its own of all of it.
#pragma once
#include "readout.cuh"

#include <algorithm>

namespace pinkb {
namespace {

// A block takes a row at a time and keeps what belongs to its columns in registers, CH chunks a thread.  Rows arrive in a ring of kRing stages by
// asynchronous copies of 16 bytes, so that three are on their way while one is summed; a row keeps its place relative to 16-byte
// boundaries, whatever its alignment.  The barrier of a row's sums also says that the next row has arrived and that the one before has been read:
// one barrier a row.
constexpr uint32_t kRing = 4, kRingSmem = 216 * 1024;         // (beside up to 8 KB of a kernel's own arrays)

// Bytes of a stage for one matrix: the granules that a row touches, and what a thread may read behind its last chunk.
__host__ __device__ inline uint32_t staged_bytes(uint32_t D, uint32_t size) { return (D * size + 31) / 16 * 16 + 16; }

// Copies the first or last row of a matrix: the granules from low to high as they are, the row's elements before and behind these one by one.  (A call,
// so that the rows between do not hold registers for it.)
template <typename T>
__device__ __noinline__ void copy_at_end(const char* src, uint32_t to, uint32_t off, uint32_t end, uint32_t pitch, uint32_t low, uint32_t high)
{
    for (uint32_t g = threadIdx.x * 16; g < high; g += pitch)
        if (g >= low) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to + g), "l"(src + g) : "memory");
    auto element = [&](uint32_t e) {
        const Raw<T> v = *reinterpret_cast<const Raw<T>*>(src + e);
        if constexpr (sizeof(T) == 4) asm volatile("st.shared.b32 [%0], %1;" :: "r"(to + e), "r"(v) : "memory");
        else asm volatile("st.shared.b16 [%0], %1;" :: "r"(to + e), "h"(v) : "memory");
    };
    if (threadIdx.x >= kChunk<T>) return;
    const uint32_t e = threadIdx.x * (uint32_t)sizeof(T);
    if (low && e >= off && e < end) element(e);
    if (high < end && high + e >= off && high + e < end) element(high + e);
}

// A matrix whose rows r, r + step, ... pass through the ring: `next` is the next row to copy, `phase` belongs to the next to read.
template <typename T, int CH>
struct Staged
{
    uint64_t next, pace;             // byte address of a row, and from row to row
    uint32_t dst, bytes;             // its place in a stage (shared-memory address in stage 0), bytes of a row
    uint32_t phase, phase_pace;      // place of a row behind a 16-byte boundary
    uint32_t threads;                // that copy

    __device__ __forceinline__ Staged(const void* base, uint64_t ld, uint32_t row, uint32_t step, uint32_t D, uint32_t smem, uint32_t n_threads)
        : next(reinterpret_cast<uint64_t>(base) + row * ld * sizeof(T)), pace(step * ld * sizeof(T)), dst(smem), bytes(D * sizeof(T)),
          phase((uint32_t)next & 15u), phase_pace((uint32_t)pace & 15u), threads(n_threads) {}

    // Copies the next row, whose stage begins `at` bytes behind stage 0.  before, behind: the matrix goes on for 16 bytes at least before and behind the row, so
    // that the granules at its ends lie inside it; otherwise the row's elements in them are copied one by one.
    __device__ __forceinline__ void copy(uint32_t at, bool before, bool behind)
    {
        const uint32_t off = (uint32_t)next & 15u, end = off + bytes, mine = threadIdx.x * 16, to = dst + at + mine, pitch = threads * 16;
        const char* src = reinterpret_cast<const char*>(next - off) + mine;
        if (__builtin_expect(before && behind, 1)) {
#pragma unroll
            for (int j = 0; j < CH; ++j)
                if (j + 1 < CH || mine + j * pitch < end)    // (all slots of a row but the last are whole)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to + j * pitch), "l"(src + j * pitch) : "memory");
            if (threadIdx.x < 2 && CH * pitch + mine < end)  // (two more granules at most: what lies before the first boundary and behind the last)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to + CH * pitch), "l"(src + CH * pitch) : "memory");
        } else {
            copy_at_end<T>(reinterpret_cast<const char*>(next - off), dst + at, off, end, pitch, before || off == 0 ? 0 : 16, behind ? end : end & ~15u);
        }
        next += pace;
    }

    __device__ __forceinline__ uint32_t place(uint32_t at) const { return dst + at + phase; }      // of the row to read
    __device__ __forceinline__ void advance() { phase = (phase + phase_pace) & 15u; }
};

__device__ __forceinline__ uint2 ld_shared8(uint32_t p)
{
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
    return v;
}

// The chunk at byte p of shared memory; what is beyond the row's end is not zero.
template <typename T, int ALIGN>
__device__ __forceinline__ uint4 staged_chunk(uint32_t p)
{
    uint4 v;
    if constexpr (ALIGN == kSixteen) {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
    } else if constexpr (ALIGN == kEight) {
        const uint2 a = ld_shared8(p), b = ld_shared8(p + 8);
        v = make_uint4(a.x, a.y, b.x, b.y);
    } else if constexpr (sizeof(T) == 4) {
        asm volatile("ld.shared.b32 %0, [%4];\n ld.shared.b32 %1, [%4 + 4];\n ld.shared.b32 %2, [%4 + 8];\n ld.shared.b32 %3, [%4 + 12];"
                     : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w) : "r"(p) : "memory");
    } else {
        const uint32_t at = p & 7u, bits = (at & 2u) * 8u;
        const bool far = at & 4u;
        const uint2 a = ld_shared8(p - at), b = ld_shared8(p - at + 8), c = ld_shared8(p - at + 16);
        const uint32_t w0 = far ? a.y : a.x, w1 = far ? b.x : a.y, w2 = far ? b.y : b.x, w3 = far ? c.x : b.y, w4 = far ? c.y : c.x;
        v = make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits), __funnelshift_r(w3, w4, bits));
    }
    return v;
}

template <typename T>
__device__ __forceinline__ float staged_element(uint32_t p)
{
    if constexpr (sizeof(T) == 4) {
        float v;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(p) : "memory");
        return v;
    } else {
        uint16_t v;
        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(p) : "memory");
        return to_float(*reinterpret_cast<const T*>(&v));
    }
}

__device__ __forceinline__ void copies_committed() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <uint32_t PENDING> __device__ __forceinline__ void copies_waited() { asm volatile("cp.async.wait_group %0;" :: "n"(PENDING) : "memory"); }

// ---- host side -------------------------------------------------------------------------------------------------------------

inline uint32_t whole_warps(uint32_t threads) { return (threads + 31) / 32 * 32; }

inline int sm_count()
{
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms > 0 ? sms : 148;
}

// Threads of a block that deals whole chunks out, `per` a thread, so that no slot but the last is partly empty: (per - 1) threads <= chunks.  0: there is
// no such block of at most 512.
inline uint32_t ring_threads(uint32_t chunks, uint32_t per)
{
    const uint32_t threads = std::max(32u, whole_warps((chunks + per - 1) / per));
    return threads <= 512 && (per - 1) * threads <= chunks ? threads : 0;
}

// As many blocks as the device holds at once, at most one a row.
template <typename... P, typename... A>
cudaError_t launch_ring(void (*kernel)(P...), uint64_t rows, uint32_t threads, uint32_t smem, cudaStream_t st, const A&... args)
{
    cudaError_t e = allow_shared(kernel, smem, kRingSmem);
    int blocks = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, kernel, (int)threads, smem);
    if (e != cudaSuccess) return e;
    return launch_following(kernel, dim3((unsigned)std::min<uint64_t>(rows, (uint64_t)sm_count() * std::max(1, blocks))), threads, smem, st, args...);
}

} // namespace
} // namespace pinkb
