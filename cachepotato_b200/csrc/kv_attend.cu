// kv_attend.cu — attention of new rows over the paged key/value cache (qwen3_moe.c:135-155 per
// head, for many sequences at once).
//
// Row t of sequence i stands at position p = pos0[i] + t - q_start[i] and sees the cached positions
// j <= p (and j > p - window). For each query head h over its cached head kh = h / (H / KV):
//   out = sum_j e^(scale q.k_j - m) v_j / sum_j e^(scale q.k_j - m),   m = max_j scale q.k_j
#include <math.h>

#include "kv.cuh"

namespace cpg {

struct AttendArgs {
    KvRows b;
    KvView c;
    const void *q;
    void *out;
    size_t q_stride, out_stride;
    int H;
    float scale;                     // times log2(e)
    int window;
};

// One warp per (row, head): a key at a time, lane l holding elements l·HD/32.., the running maximum
// and sum of the softmax in every lane.
template <typename TI, typename TC, int HD>
__global__ void __launch_bounds__(256) k_kv_attend_row(const __grid_constant__ AttendArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int N = HD / 32;
    const int t = blockIdx.x, lane = threadIdx.x & 31, h = blockIdx.y * 8 + (threadIdx.x >> 5);
    const int i = kv_find_seq(a.b.q_start, a.b.n, t);
    if (i >= a.b.n || h >= a.H) return;
    const KvSeq sq = kv_seq(a.b, a.c.P, i);
    if (sq.bad && lane == 0) atomicOr(a.c.status, KV_BAD_POS);
    if (t < sq.r0 || t >= sq.r0 + sq.len) return;
    const int p = sq.p0 + (t - sq.r0);
    const size_t head = (size_t)(h / (a.H / a.c.KV)) * a.c.sh;
    float q[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < N; ++e) {
        q[e] = to_f32(((const TI *)a.q)[(size_t)t * a.q_stride + (size_t)h * HD + lane * N + e]);
        o[e] = 0.0f;
    }
    for (int j = a.window ? max(0, p - a.window + 1) : 0; j <= p; ++j) {
        const int page = a.b.pages[(size_t)i * a.b.table_stride + j / a.c.P];
        if (page < 0 || page >= a.c.n_pages) {
            if (lane == 0) atomicOr(a.c.status, KV_BAD_PAGE);
            continue;
        }
        const size_t at = (size_t)page * a.c.sp + (size_t)(j % a.c.P) * a.c.st + head + lane * N;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) s = fmaf(q[e], to_f32(((const TC *)a.c.k)[at + e]), s);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        s *= a.scale;
        const float mn = fmaxf(m, s), r = m == -INFINITY ? 0.0f : exp2f(m - mn);
        const float w = mn == -INFINITY ? 0.0f : exp2f(s - mn);
        l = fmaf(l, r, w);
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = fmaf(w, to_f32(((const TC *)a.c.v)[at + e]), o[e] * r);
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
        ((TI *)a.out)[(size_t)t * a.out_stride + (size_t)h * HD + lane * N + e] = from_f32<TI>(l == 0.0f ? 0.0f : o[e] / l);
}

template <typename TI, typename TC>
static cudaError_t launch_row(int hd, const AttendArgs &a, cudaStream_t s) {
    const dim3 grid(a.b.T, (a.H + 7) / 8);
    return hd == 128 ? launch_pdl(k_kv_attend_row<TI, TC, 128>, grid, dim3(256), 0, s, a)
                     : launch_pdl(k_kv_attend_row<TI, TC, 64>, grid, dim3(256), 0, s, a);
}

size_t kv_attend_ws_bytes(int hd, int type) { return 256; }

int kv_attend_launch(const KvView &c, int hd, const KvRows &b, const void *q, size_t q_stride, void *out,
                     size_t out_stride, int type, int n_heads, float scale, int window, int max_new, void *ws,
                     cudaStream_t s) {
    const AttendArgs a{b, c, q, out, q_stride, out_stride, n_heads, scale * 1.4426950408889634f, window};
    cudaError_t ce;
    if (type == CPG_T_F32)
        ce = c.type == CPG_T_F32   ? launch_row<float, float>(hd, a, s)
             : c.type == CPG_T_F16 ? launch_row<float, __half>(hd, a, s)
                                   : launch_row<float, __nv_bfloat16>(hd, a, s);
    else
        ce = type == CPG_T_F16 ? launch_row<__half, __half>(hd, a, s) : launch_row<__nv_bfloat16, __nv_bfloat16>(hd, a, s);
    return ce == cudaSuccess ? CPG_OK : cuda_fail(ce, "cpg_kv_attend");
}

}  // namespace cpg
