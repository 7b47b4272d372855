// kv_attend.cuh — what the attention kernels over the paged cache share (kv_attend.cu for few rows,
// kv_attend_tc.cu for chunks).
#pragma once
#include "kv.cuh"
#include "tcgen05.cuh"

namespace cpg {

struct AttendArgs {
    KvRows b;
    KvView c;
    const void *q;
    void *out;
    size_t q_stride, out_stride;
    int H;
    float scale2;                    // scale · log2(e)
    int window, box;                 // box: positions of one tensor TMA load
    float *part;                     // 2 slots per block
    int *counters;                   // zero between calls
};

constexpr int KV_MAX_GRID = 512;      // blocks of a launch, at most

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// Weights that go into f16 operands are lifted by 2^14 (kv_attend_tc.cu, which lets them grow to 2^8 before
// it rescales: by 2^7): f16 has nothing below 2^-25, and of a long cache thousands of weights of 2^-26 of
// the largest one count. l and o carry the factor, which cancels in o / l. So that it can be taken off the
// maximum exactly, an f16 cache's running maxima are rounded up to whole numbers (in powers of two).
template <bool HALF> __device__ __forceinline__ float kv_top(float top) { return HALF ? ceilf(top) : top; }
template <bool HALF> constexpr float kv_lift(float by) { return HALF ? by : 0.0f; }

// (x, y) as N terms of two 16-bit halves each, largest first. f16: rounded, 22 bits from two terms.
// bf16: one term rounded; three terms cut off, which leaves nothing of an f32.
template <bool HALF, int N>
__device__ __forceinline__ void split_pair(float x, float y, uint32_t (&t)[N]) {
    if constexpr (HALF) {
        const __half2 h = __floats2half2_rn(x, y);
        t[0] = *reinterpret_cast<const uint32_t *>(&h);
        if constexpr (N == 2) {
            const float2 f = __half22float2(h);
            const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
            t[1] = *reinterpret_cast<const uint32_t *>(&l);
        }
    } else if constexpr (N == 1) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        t[0] = *reinterpret_cast<const uint32_t *>(&h);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
            t[i] = __byte_perm(a, b, 0x7632);
            x -= __uint_as_float(a & 0xffff0000u);
            y -= __uint_as_float(b & 0xffff0000u);
        }
    }
}

// a / b of non-negative numbers; nearly always both have 32 bits, which divide in a fifth of the time.
__device__ __forceinline__ long kv_div(long a, long b) {
    return ((a | b) >> 32) == 0 ? (long)((uint32_t)a / (uint32_t)b) : a / b;
}
// Units 0..U-1 over NB blocks: block b has [start(b), start(b + 1)), the first U % NB one more.
struct KvCut {
    long each, more;
    KvCut() = default;
    __device__ __forceinline__ KvCut(long U, long NB) : each(kv_div(U, NB)), more(U - each * NB) {}
    __device__ __forceinline__ long start(long b) const { return b * each + min(b, more); }
    __device__ __forceinline__ int owner(long u) const {
        const long big = more * (each + 1);
        return (int)(u < big ? kv_div(u, each + 1) : more + kv_div(u - big, each));
    }
};

// Adds 1 to a counter of parts: what the block wrote before (its barrier passed) is seen by whoever
// counts after it, and the other way round.
__device__ __forceinline__ int kv_arrive(int *counter) {
    int old;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
    return old;
}

}  // namespace cpg
