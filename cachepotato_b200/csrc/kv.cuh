// kv.cuh — the paged key/value cache as its kernels see it (kv.cu, kv_attend.cu).
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include "common.cuh"

namespace cpg {

// The pools. Element (page, place, head, e) of either lies at page·sp + place·st + head·sh + e.
struct KvView {
    void *k, *v;
    size_t sp, st, sh;
    int P, n_pages, KV, type;
    int *status;
};

// The rows of one call (cpg_kv_batch). Everything behind the three pointers is only known on the
// device, so every index taken from there is checked where it is used.
struct KvRows {
    int n, T;
    const int *q_start, *pos0, *pages;
    int table_stride, max_pages;
};

// Tensor maps of the two pools: axes (element, place, head, page), a box of 128 bytes by `box`
// positions, which lie in one page wherever they start at a multiple of box; 128-byte swizzle.
struct KvMaps {
    CUtensorMap m[2];
    int box;
};

// Status bits a kernel leaves in KvView::status (reported and cleared by cpg_kv_check).
enum : int { KV_BAD_PAGE = 1, KV_BAD_POS = 2, KV_TIMEOUT = 4 };

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32(float v) { return v; }
template <> __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements as f32 (16-byte loads where N allows) and back, each rounded once.
template <typename T, int N>
__device__ __forceinline__ void load_vec(const T *p, float (&v)[N]) {
    constexpr int B = N * (int)sizeof(T);
    static_assert(B == 8 || B % 16 == 0, "vector width");
    if constexpr (B == 8) {
        const uint2 w = *reinterpret_cast<const uint2 *>(p);
        const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = to_f32(e[i]);
    } else {
#pragma unroll
        for (int b = 0; b < B / 16; ++b) {
            const uint4 w = *reinterpret_cast<const uint4 *>(reinterpret_cast<const char *>(p) + 16 * b);
            const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int i = 0; i < 16 / (int)sizeof(T); ++i) v[b * (16 / sizeof(T)) + i] = to_f32(e[i]);
        }
    }
}
template <typename T, int N>
__device__ __forceinline__ void store_vec(T *p, const float (&v)[N]) {
    constexpr int B = N * (int)sizeof(T);
    static_assert(B == 8 || B % 16 == 0, "vector width");
    if constexpr (B == 8) {
        uint2 w;
        T *e = reinterpret_cast<T *>(&w);
#pragma unroll
        for (int i = 0; i < N; ++i) e[i] = from_f32<T>(v[i]);
        *reinterpret_cast<uint2 *>(p) = w;
    } else {
#pragma unroll
        for (int b = 0; b < B / 16; ++b) {
            uint4 w;
            T *e = reinterpret_cast<T *>(&w);
#pragma unroll
            for (int i = 0; i < 16 / (int)sizeof(T); ++i) e[i] = from_f32<T>(v[b * (16 / sizeof(T)) + i]);
            *reinterpret_cast<uint4 *>(reinterpret_cast<char *>(p) + 16 * b) = w;
        }
    }
}

// The number of entries of q_start[1..n] that are <= t: the sequence row t belongs to where the
// starts ascend (and t < q_start[n]). Warp-wide, every lane gets it; 32 probes a step.
__device__ __forceinline__ int kv_find_seq(const int *__restrict__ q_start, int n, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = n;                                   // the answer lies in [lo, hi]
    while (hi - lo > 32) {
        const int step = (hi - lo + 33) / 33;            // 33 parts cover [lo, hi]
        const int at = lo + (lane + 1) * step;            // entry number at, 1-based
        const unsigned le = __ballot_sync(0xffffffffu, at <= hi && q_start[at] <= t);
        const int c = __popc(le);
        hi = min(hi, lo + (c + 1) * step - 1);
        lo += c * step;
    }
    const unsigned le = __ballot_sync(0xffffffffu, lo + lane + 1 <= hi && q_start[lo + lane + 1] <= t);
    return lo + __popc(le);
}

// Sequence i's rows [r0, r0 + len) and the position of its first one, made safe: rows inside
// [0, T), positions inside the table (rows past it are cut off). bad: something had to be cut.
struct KvSeq {
    int r0, len, p0;
    bool bad;
};
__device__ __forceinline__ KvSeq kv_seq(const KvRows &b, int P, int i) {
    KvSeq s;
    const int a = b.q_start[i], e = b.q_start[i + 1];
    s.p0 = b.pos0[i];
    s.r0 = max(a, 0);
    s.len = max(0, min(e, b.T) - s.r0);
    s.bad = a < 0 || e < a || e > b.T || s.p0 < 0;
    const long cap = (long)b.max_pages * P;
    if (s.p0 < 0) s.len = 0;
    if ((long)s.p0 + s.len > cap) {
        s.len = (int)max(0l, cap - s.p0);
        s.bad = true;
    }
    return s;
}

}  // namespace cpg
