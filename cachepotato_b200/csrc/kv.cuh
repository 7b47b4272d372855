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
    int table_stride;
    int cap;                         // positions a sequence may have: the table's, and what 32 bits count
};

// Tensor maps of the two pools: axes (element, place, head, page), a box of 128 bytes by `box`
// positions, which lie in one page wherever they start at a multiple of box; 128-byte swizzle.
struct KvMaps {
    CUtensorMap m[2];
    int box;
};

// Status bits a kernel leaves in KvView::status (reported and cleared by cpg_kv_check).
enum : int { KV_BAD_PAGE = 1, KV_BAD_POS = 2, KV_TIMEOUT = 4 };

// Four consecutive elements as f32, and back, each rounded once.
__device__ __forceinline__ void load4(const float *p, float *v) {
    const float4 w = *reinterpret_cast<const float4 *>(p);
    v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w;
}
__device__ __forceinline__ void load4(const __half *p, float *v) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&w.y));
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
}
__device__ __forceinline__ void load4(const __nv_bfloat16 *p, float *v) {
    const uint2 w = *reinterpret_cast<const uint2 *>(p);
    v[0] = __uint_as_float(w.x << 16); v[1] = __uint_as_float(w.x & 0xffff0000u);
    v[2] = __uint_as_float(w.y << 16); v[3] = __uint_as_float(w.y & 0xffff0000u);
}
__device__ __forceinline__ void store4(float *p, const float *v) {
    *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__half *p, const float *v) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ void store4(__nv_bfloat16 *p, const float *v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
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
// [0, T), positions inside the table (rows past either are cut off, and a sequence whose start or
// first position is negative, or that ends before it starts, has none). bad: something of it was cut.
struct KvSeq {
    int r0, len, p0;
    bool bad;
};
__device__ __forceinline__ KvSeq kv_seq(const KvRows &b, int i) {
    KvSeq s;
    const int a = b.q_start[i], e = b.q_start[i + 1];
    s.r0 = a;
    s.p0 = b.pos0[i];
    s.len = 0;
    s.bad = a < 0 || e < a || e > b.T || (e > a && s.p0 < 0);    // (no rows: pos0 may be anything)
    if (a >= 0 && s.p0 >= 0 && min(e, b.T) > a) {
        const int n = min(e, b.T) - a;
        s.len = min(n, max(0, b.cap - s.p0));
        s.bad = s.bad || s.len < n;
    }
    return s;
}

}  // namespace cpg
