// kv.cu — the paged key/value cache: the handle, its checks, and appending rows to it.
//
// The reference keeps one contiguous f32 cache per sequence (qwen3_moe.h:40-70); here the
// positions of many sequences share pools of fixed-size pages, found through a table per sequence.
#include <math.h>

#include <new>

#include "kv.cuh"

struct cpg_kv {
    cpg::KvView v;
    cpg::KvMaps maps;
    int hd, device, rope_dim, rope_f32;
    float theta;
    double freq[64];                 // theta^(-2j/R) / pi: a position's angle in half turns is p·freq
};

namespace cpg {

// ------------------------------------------------------------------------------ append
// One block per row (and per group of heads, for few rows). For every query and key head x:
// y = x / sqrt(mean x² + eps) · g (head_rmsnorm, qwen3_moe.c:44-49; only with a gain), then the
// rotation of (y_j, y_{j+R/2}) by p·theta^(-2j/R) (rope_apply_from, kernels.c:425-447). Queries go
// to q_out, keys and values to the row's place in the pools, each value rounded once.
//
// A far position's angle needs more than 32 bits (at position 10^6 an f32 product is off by up to
// 0.06): the product with freq is taken in 64 bits in half turns, where dropping whole turns is
// exact, and the rest in [-1, 1] goes to sincospif. With rope_f32 it is the reference's arithmetic
// instead: an f32 frequency, an f32 product.
//
// A thread holds 16 bytes of a head; lanes of a head exchange rotation partners by shuffle (R/2 is
// a multiple of a thread's elements). The row's R/2 sines are computed once per block while the
// first heads' loads are in flight.
struct AppendArgs {
    KvRows b;
    KvView c;
    const void *q, *k, *v;
    void *q_out;
    size_t q_stride, k_stride, v_stride, qo_stride;
    const float *q_norm, *k_norm;
    float eps, theta;
    int H, R, rope_f32;
    double freq[64];
};

constexpr int AP_U = 4;              // heads of a lane group in flight

template <typename TI, typename TC, int HD>
__global__ void __launch_bounds__(512) k_kv_append(const __grid_constant__ AppendArgs a) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int N = 16 / (int)sizeof(TI);               // elements per thread
    constexpr int LPH = HD / N, HPW = 32 / LPH;           // lanes per head, heads per warp
    __shared__ float2 s_cs[64];
    __shared__ int s_where[3];                            // position, page, live
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    const int KV = a.c.KV, nh = a.H + 2 * KV;             // heads q, then k, then v
    const int sub = lane % LPH, e0 = sub * N;
    const int groups = (blockDim.x >> 5) * HPW;           // heads of the block in flight
    const int per = (nh + gridDim.y - 1) / gridDim.y;     // this block's heads
    const int h0 = blockIdx.y * per, h1 = min(nh, h0 + per);
    const int first = h0 + (tid >> 5) * HPW + lane / LPH;

    float x[AP_U][N];
    auto load = [&](int base) {
#pragma unroll
        for (int u = 0; u < AP_U; ++u) {
            const int h = base + u * groups;
            if (h >= h1) continue;
            const TI *src = h < a.H ? (const TI *)a.q + (size_t)t * a.q_stride + (size_t)h * HD
                            : h < a.H + KV ? (const TI *)a.k + (size_t)t * a.k_stride + (size_t)(h - a.H) * HD
                                           : (const TI *)a.v + (size_t)t * a.v_stride + (size_t)(h - a.H - KV) * HD;
            load_vec<TI, N>(src + e0, x[u]);
        }
    };
    load(first);

    if (tid < 32) {
        const int i = kv_find_seq(a.b.q_start, a.b.n, t);
        int pos = 0, page = -1, live = 0;
        if (i < a.b.n) {
            const int a0 = a.b.q_start[i], p0 = a.b.pos0[i];
            if (t >= a0 && p0 >= 0) {
                live = 1;
                const long p = (long)p0 + (t - a0);
                pos = (int)min(p, 0x7fffffffl);
                const long at = p / a.c.P;
                if (at < a.b.max_pages) page = a.b.pages[(size_t)i * a.b.table_stride + at];
                if (page < 0 || page >= a.c.n_pages) {
                    page = -1;
                    if (lane == 0) atomicOr(a.c.status, at < a.b.max_pages ? KV_BAD_PAGE : KV_BAD_POS);
                }
            } else if (lane == 0 && p0 < 0) {
                atomicOr(a.c.status, KV_BAD_POS);
            }
        }
        if (lane == 0) {
            s_where[0] = pos;
            s_where[1] = page;
            s_where[2] = live;
        }
    }
    __syncthreads();
    if (!s_where[2]) return;                              // a row of no sequence
    const int pos = s_where[0], page = s_where[1], R = a.R;
    for (int j = tid; j < R / 2; j += blockDim.x) {
        float sn, cs;
        if (a.rope_f32) {
            const float ang = __fmul_rn((float)pos, powf(a.theta, __fdiv_rn(-2.0f * (float)j, (float)R)));
            cs = cosf(ang);
            sn = sinf(ang);
        } else {
            const double turn = (double)pos * a.freq[j];
            sincospif((float)(turn - 2.0 * rint(0.5 * turn)), &sn, &cs);
        }
        s_cs[j] = make_float2(cs, sn);
    }
    __syncthreads();
    const size_t place = page < 0 ? 0 : (size_t)page * a.c.sp + (size_t)(pos % a.c.P) * a.c.st + e0;

    for (int base = first; base < h1; base += AP_U * groups) {
        if (base != first) load(base);
#pragma unroll
        for (int u = 0; u < AP_U; ++u) {
            const int h = base + u * groups;
            // the shuffles below are among the lanes of one head, which agree on h
            const unsigned mask = LPH == 32 ? 0xffffffffu : (((1u << (LPH & 31)) - 1u) << (lane / LPH * LPH));
            if (h >= h1) continue;
            float(&y)[N] = x[u];
            if (h < a.H + KV) {
                const float *gain = h < a.H ? a.q_norm : a.k_norm;
                if (gain) {
                    float ss = 0.0f;
#pragma unroll
                    for (int i = 0; i < N; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
                    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
                    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(ss, (float)HD) + a.eps));
                    float g[N];
                    load_vec<float, N>(gain + e0, g);
#pragma unroll
                    for (int i = 0; i < N; ++i) y[i] = __fmul_rn(__fmul_rn(y[i], inv), g[i]);
                }
                if (R) {
                    const int half = R / 2, d = half / N;                // lanes to the partner
                    const bool low = e0 < half, in = e0 < R;
                    const int from = in ? (low ? lane + d : lane - d) : lane;
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        const float other = __shfl_sync(mask, y[i], from);
                        if (in) {
                            const float2 cs = s_cs[(low ? e0 : e0 - half) + i];
                            y[i] = low ? __fsub_rn(__fmul_rn(y[i], cs.x), __fmul_rn(other, cs.y))
                                       : __fadd_rn(__fmul_rn(y[i], cs.x), __fmul_rn(other, cs.y));
                        }
                    }
                }
            }
            if (h < a.H)
                store_vec<TI, N>((TI *)a.q_out + (size_t)t * a.qo_stride + (size_t)h * HD + e0, y);
            else if (page >= 0) {
                const bool isk = h < a.H + KV;
                TC *dst = (TC *)(isk ? a.c.k : a.c.v) + place + (size_t)(h - a.H - (isk ? 0 : KV)) * a.c.sh;
                store_vec<TC, N>(dst, y);
            }
        }
    }
}

template <typename TI, typename TC>
static cudaError_t launch_append(int hd, const AppendArgs &a, dim3 grid, dim3 block, cudaStream_t s) {
    return hd == 128 ? launch_pdl(k_kv_append<TI, TC, 128>, grid, block, 0, s, a)
                     : launch_pdl(k_kv_append<TI, TC, 64>, grid, block, 0, s, a);
}

int kv_attend_launch(const KvView &c, const KvMaps &maps, int hd, const KvRows &b, const void *q, size_t q_stride,
                     void *out, size_t out_stride, int type, int n_heads, float scale, int window, int max_new, void *ws,
                     cudaStream_t s);
int tensor_map(CUtensorMap *map, int type, int rank, const void *base, const uint64_t *dims, const uint64_t *strides,
               const uint32_t *box);
size_t kv_attend_ws_bytes(int hd, int type);

static size_t type_bytes(int type) { return type == CPG_T_F32 ? 4 : 2; }
static bool type_ok(int type) { return type == CPG_T_F32 || type == CPG_T_F16 || type == CPG_T_BF16; }

}  // namespace cpg

using namespace cpg;

extern "C" int cpg_kv_create(const cpg_kv_desc *d, cpg_kv **out) {
    CPG_REQUIRE(d && out, "cpg_kv_create: null argument");
    *out = nullptr;
    CPG_REQUIRE(d->head_dim == 64 || d->head_dim == 128, "cpg_kv_create: head_dim %d (64 or 128)", d->head_dim);
    CPG_REQUIRE(d->n_kv >= 1 && d->n_kv <= 1024, "cpg_kv_create: n_kv %d (1..1024)", d->n_kv);
    CPG_REQUIRE(d->page_size >= 8 && d->page_size <= 65536 && d->page_size % 8 == 0,
                "cpg_kv_create: page_size %d (a multiple of 8, at most 65536)", d->page_size);
    CPG_REQUIRE(d->n_pages >= 1, "cpg_kv_create: n_pages %d", d->n_pages);
    CPG_REQUIRE(type_ok(d->type), "cpg_kv_create: element type %d", d->type);
    CPG_REQUIRE(d->k && d->v, "cpg_kv_create: null pool");
    const size_t es = type_bytes(d->type), hd = d->head_dim;
    CPG_REQUIRE(((uintptr_t)d->k | (uintptr_t)d->v) % 16 == 0, "cpg_kv_create: pools must be 16-byte aligned");
    const long st[3] = {d->page_stride, d->pos_stride, d->head_stride};
    const long n[3] = {d->n_pages, d->page_size, d->n_kv};
    for (int i = 0; i < 3; ++i)
        CPG_REQUIRE(n[i] == 1 || (st[i] >= (long)hd && st[i] * es % 16 == 0 && st[i] < (1l << 36)),
                    "cpg_kv_create: stride %ld (at least head_dim, a multiple of 16 bytes)", st[i]);
    // no two (page, place, head) may share memory: in order of stride, each passes the extent below it
    long extent = (long)hd, done = 0;
    for (int r = 0; r < 3; ++r) {
        int at = -1;
        for (int i = 0; i < 3; ++i)
            if (!(done >> i & 1) && n[i] > 1 && (at < 0 || st[i] < st[at])) at = i;
        if (at < 0) break;
        CPG_REQUIRE(st[at] >= extent, "cpg_kv_create: strides %ld, %ld, %ld make positions overlap", st[0], st[1], st[2]);
        extent += (n[at] - 1) * st[at];
        done |= 1l << at;
    }
    CPG_REQUIRE(d->rope_dim >= 0 && d->rope_dim <= d->head_dim && d->rope_dim % 16 == 0,
                "cpg_kv_create: rope_dim %d (a multiple of 16, at most head_dim)", d->rope_dim);
    CPG_REQUIRE(d->rope_dim == 0 || (d->rope_theta > 0.0f && isfinite(d->rope_theta)), "cpg_kv_create: rope_theta %g",
                (double)d->rope_theta);
    cpg_kv *kv = new (std::nothrow) cpg_kv();
    if (!kv) {
        set_error("cpg_kv_create: host allocation failed");
        return CPG_ENOMEM;
    }
    kv->v = KvView{d->k, d->v, (size_t)d->page_stride, (size_t)d->pos_stride, (size_t)d->head_stride,
                   d->page_size, d->n_pages, d->n_kv, d->type, nullptr};
    kv->hd = d->head_dim;
    kv->rope_dim = d->rope_dim;
    kv->rope_f32 = d->rope_f32 != 0;
    kv->theta = d->rope_theta;
    for (int j = 0; j < d->rope_dim / 2; ++j)
        kv->freq[j] = pow((double)d->rope_theta, -2.0 * j / d->rope_dim) / 3.14159265358979323846;
    kv->maps.box = 8;
    while (kv->maps.box < 64 && d->page_size % (2 * kv->maps.box) == 0) kv->maps.box *= 2;
    const uint64_t dims[4] = {hd, (uint64_t)d->page_size, (uint64_t)d->n_kv, (uint64_t)d->n_pages};
    uint64_t ts[3];                                       // an axis of one entry has no stride of its own
    for (int i = 0; i < 3; ++i) ts[i] = (n[(i + 1) % 3] > 1 ? st[(i + 1) % 3] : (long)hd) * es;
    const uint32_t box[4] = {(uint32_t)(128 / es), (uint32_t)kv->maps.box, 1, 1};
    for (int i = 0; i < 2; ++i) {
        const int rc = tensor_map(&kv->maps.m[i], d->type, 4, i ? d->v : d->k, dims, ts, box);
        if (rc) {
            delete kv;
            return rc;
        }
    }
    cudaError_t ce = cudaGetDevice(&kv->device);
    if (ce == cudaSuccess) ce = cudaMalloc(&kv->v.status, sizeof(int));
    if (ce == cudaSuccess) ce = cudaMemset(kv->v.status, 0, sizeof(int));
    if (ce != cudaSuccess) {
        cudaFree(kv->v.status);
        delete kv;
        return cuda_fail(ce, "cpg_kv_create");
    }
    *out = kv;
    return CPG_OK;
}

extern "C" void cpg_kv_destroy(cpg_kv *kv) {
    if (!kv) return;
    cudaFree(kv->v.status);
    delete kv;
}

// The checks append and attend share.
static int kv_rows(const cpg_kv *kv, const cpg_kv_batch *b, const char *fn, KvRows *r) {
    CPG_REQUIRE(kv && b, "%s: null argument", fn);
    CPG_REQUIRE(b->n_seqs >= 0 && b->rows >= 0, "%s: %d sequences, %d rows", fn, b->n_seqs, b->rows);
    CPG_REQUIRE(b->n_seqs == 0 || (b->q_start && b->pos0 && b->pages), "%s: null batch array", fn);
    CPG_REQUIRE(b->n_seqs == 0 || (b->max_pages >= 1 && b->table_stride >= b->max_pages),
                "%s: table of %d pages, row stride %d", fn, b->max_pages, b->table_stride);
    int dev = -1;
    CPG_CUDA(cudaGetDevice(&dev));
    CPG_REQUIRE(dev == kv->device, "%s: the cache is on device %d, the current device is %d", fn, kv->device, dev);
    *r = KvRows{b->n_seqs, b->rows, b->q_start, b->pos0, b->pages, b->table_stride, b->max_pages};
    return CPG_OK;
}

static int rows_ok(const char *fn, const char *what, const void *p, long stride, int heads, int hd, int type) {
    CPG_REQUIRE(p && (uintptr_t)p % 16 == 0, "%s: %s must be a 16-byte aligned device pointer", fn, what);
    CPG_REQUIRE(stride >= (long)heads * hd && stride * (long)type_bytes(type) % 16 == 0,
                "%s: %s row stride %ld (at least %d x %d, a multiple of 16 bytes)", fn, what, stride, heads, hd);
    return CPG_OK;
}

extern "C" int cpg_kv_append(const cpg_kv *kv, const cpg_kv_batch *b, int type, int n_heads, const void *q,
                             long q_stride, const void *k, long k_stride, const void *v, long v_stride,
                             const float *q_norm, const float *k_norm, float eps, void *q_out, long q_out_stride,
                             void *stream) {
    const char *fn = "cpg_kv_append";
    AppendArgs a{};
    int rc = kv_rows(kv, b, fn, &a.b);
    if (rc) return rc;
    CPG_REQUIRE(type == CPG_T_F32 || type == kv->v.type, "%s: rows of type %d over a cache of type %d (f32 or the cache's)",
                fn, type, kv->v.type);
    CPG_REQUIRE(n_heads >= 0 && n_heads <= 4096, "%s: n_heads %d", fn, n_heads);
    CPG_REQUIRE(eps >= 0.0f && isfinite(eps), "%s: eps %g", fn, (double)eps);
    CPG_REQUIRE(((uintptr_t)q_norm | (uintptr_t)k_norm) % 16 == 0, "%s: gains must be 16-byte aligned", fn);
    if (a.b.T == 0 || a.b.n == 0) return CPG_OK;
    rc = rows_ok(fn, "k", k, k_stride, kv->v.KV, kv->hd, type);
    if (!rc) rc = rows_ok(fn, "v", v, v_stride, kv->v.KV, kv->hd, type);
    if (!rc && n_heads) rc = rows_ok(fn, "q", q, q_stride, n_heads, kv->hd, type);
    if (!rc && n_heads) rc = rows_ok(fn, "q_out", q_out, q_out_stride, n_heads, kv->hd, type);
    if (rc) return rc;
    a.c = kv->v;
    a.q = q; a.k = k; a.v = v; a.q_out = q_out;
    a.q_stride = q_stride; a.k_stride = k_stride; a.v_stride = v_stride; a.qo_stride = q_out_stride;
    a.q_norm = q_norm; a.k_norm = k_norm;
    a.eps = eps; a.theta = kv->theta;
    a.H = n_heads; a.R = kv->rope_dim; a.rope_f32 = kv->rope_f32;
    for (int j = 0; j < a.R / 2; ++j) a.freq[j] = kv->freq[j];
    // heads in flight per warp: 16 bytes a lane; warps for all heads of a row at AP_U each, and a
    // row over several blocks while the rows alone leave SMs idle
    const int per_warp = 32 * (16 / (int)type_bytes(type)) / kv->hd;
    const int nh = n_heads + 2 * kv->v.KV;
    int split = 1;
    while (split < 8 && (long)a.b.T * split < sm_count() && nh / (split * 2) >= per_warp) split *= 2;
    const int per = (nh + split - 1) / split;
    int warps = (per + per_warp * AP_U - 1) / (per_warp * AP_U);
    if (split > 1) warps = (per + per_warp - 1) / per_warp;
    warps = warps < 2 ? 2 : warps > 16 ? 16 : warps;
    const dim3 grid(a.b.T, split), block(32 * warps);
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t ce;
    if (type == CPG_T_F32)
        ce = kv->v.type == CPG_T_F32   ? launch_append<float, float>(kv->hd, a, grid, block, s)
             : kv->v.type == CPG_T_F16 ? launch_append<float, __half>(kv->hd, a, grid, block, s)
                                       : launch_append<float, __nv_bfloat16>(kv->hd, a, grid, block, s);
    else
        ce = type == CPG_T_F16 ? launch_append<__half, __half>(kv->hd, a, grid, block, s)
                               : launch_append<__nv_bfloat16, __nv_bfloat16>(kv->hd, a, grid, block, s);
    return ce == cudaSuccess ? CPG_OK : cuda_fail(ce, fn);
}

extern "C" size_t cpg_kv_attend_workspace_bytes(const cpg_kv *kv, int n_heads) {
    if (!kv || n_heads < 1 || n_heads % kv->v.KV) {
        set_error("cpg_kv_attend_workspace_bytes: bad argument");
        return 0;
    }
    return kv_attend_ws_bytes(kv->hd, kv->v.type);
}

extern "C" int cpg_kv_attend(const cpg_kv *kv, const cpg_kv_batch *b, int type, int n_heads, const void *q,
                             long q_stride, void *out, long out_stride, float scale, int window, void *ws,
                             size_t ws_bytes, void *stream) {
    const char *fn = "cpg_kv_attend";
    KvRows r;
    int rc = kv_rows(kv, b, fn, &r);
    if (rc) return rc;
    CPG_REQUIRE(type == CPG_T_F32 || type == kv->v.type, "%s: rows of type %d over a cache of type %d (f32 or the cache's)",
                fn, type, kv->v.type);
    CPG_REQUIRE(n_heads >= 1 && n_heads <= 4096 && n_heads % kv->v.KV == 0, "%s: %d heads over %d cached heads", fn,
                n_heads, kv->v.KV);
    CPG_REQUIRE(scale > 0.0f && isfinite(scale), "%s: scale %g must be positive", fn, (double)scale);
    CPG_REQUIRE(window >= 0, "%s: window %d", fn, window);
    if (r.T == 0 || r.n == 0) return CPG_OK;
    rc = rows_ok(fn, "q", q, q_stride, n_heads, kv->hd, type);
    if (!rc) rc = rows_ok(fn, "out", out, out_stride, n_heads, kv->hd, type);
    if (rc) return rc;
    const size_t need = kv_attend_ws_bytes(kv->hd, kv->v.type);
    CPG_REQUIRE(ws && (uintptr_t)ws % 256 == 0 && ws_bytes >= need, "%s: workspace of %zu bytes at a 256-byte boundary needed, got %zu",
                fn, need, ws ? ws_bytes : (size_t)0);
    return kv_attend_launch(kv->v, kv->maps, kv->hd, r, q, q_stride, out, out_stride, type, n_heads, scale, window, b->max_new, ws,
                            (cudaStream_t)stream);
}

extern "C" int cpg_kv_check(const cpg_kv *kv, void *stream) {
    CPG_REQUIRE(kv, "cpg_kv_check: null argument");
    int st = 0;
    cudaStream_t s = (cudaStream_t)stream;
    CPG_CUDA(cudaMemcpyAsync(&st, kv->v.status, sizeof(int), cudaMemcpyDeviceToHost, s));
    CPG_CUDA(cudaMemsetAsync(kv->v.status, 0, sizeof(int), s));
    CPG_CUDA(cudaStreamSynchronize(s));
    if (st & KV_TIMEOUT) {
        set_error("cpg_kv_check: a bounded device wait gave up");
        return CPG_ETIMEOUT;
    }
    CPG_REQUIRE(!(st & KV_BAD_POS), "cpg_kv_check: a sequence's rows or positions lay outside its rows or its table");
    CPG_REQUIRE(!(st & KV_BAD_PAGE), "cpg_kv_check: a page id lay outside the pool");
    return CPG_OK;
}
