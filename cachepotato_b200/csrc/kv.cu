// kv.cu — the paged key/value cache: the handle, its checks, and appending rows to it.
//
// The reference keeps one contiguous f32 cache per sequence (qwen3_moe.h:40-70); here the
// positions of many sequences share pools of fixed-size pages, found through a table per sequence.
#include <math.h>
#include <stddef.h>

#include <algorithm>
#include <new>

#include "kv.cuh"

struct cpg_kv {
    cpg::KvView v;
    cpg::KvMaps maps;
    int hd, device, rope_dim, rope_f32;
    float theta;
    bool owns;                       // the device block is this handle's (kv_create_like shares it)
};

// The handle's device memory: the status word, and theta^(-2j/R) / pi (a position's angle in half
// turns is p times that). Device memory, not a launch argument: lanes that index the constant bank
// with different j are served one after another.
struct KvDevice {
    int status, pad[31];
    double freq[64];
};

namespace cpg {

// ------------------------------------------------------------------------------ append
// One block per run of rows, or for few rows one per row and group of heads. For every query and key head x:
// y = x / sqrt(mean x² + eps) · g (head_rmsnorm, qwen3_moe.c:44-49; only with a gain), then the
// rotation of (y_j, y_{j+R/2}) by p·theta^(-2j/R) (rope_apply_from, kernels.c:425-447). Queries go
// to q_out, keys and values to the row's place in the pools, each value rounded once.
//
// A far position's angle needs more than 32 bits (at position 10^6 an f32 product is off by up to
// 0.06): the product with freq is taken in 64 bits in half turns, where dropping whole turns is
// exact, and the rest in [-1, 1] goes to sincospif. With rope_f32 it is the reference's arithmetic
// instead: an f32 frequency, an f32 product.
//
// A thread holds two runs of E elements of a head that are rotation partners, 16 bytes of a row each
// (elements Ec.. and R/2 + Ec.., c < R / 2E; the rest in neighbouring runs), so nothing crosses lanes
// but the sum of squares, and a row's sines are the same registers for all of a thread's heads. The
// rows' places (a search over q_start, then the table) and sines are found once per block, while the
// first row's loads are in flight.
//
// Bound by memory: each value is read and written once. What counts is the bytes in flight, so a
// thread asks for the next row's heads, unconverted, before it works on this one's, and a run is as
// long as one wave of blocks needs to take all rows. Measured: 16384 rows of 32 + 2·4 heads in bf16
// (336 MB) 75 us, 4.5 TB/s (8 bytes a load 85 us; without asking ahead as well 111), in f32 (671 MB)
// 117 us, 5.7 TB/s (32 bytes a load 162: registers for three blocks instead of four); in a captured graph
// one row 3.6 us, 64 rows 4.1 us.
struct AppendArgs {
    KvRows b;
    KvView c;
    const void *q, *k, *v;
    void *q_out;
    size_t q_stride, k_stride, v_stride, qo_stride;
    const float *q_norm, *k_norm;
    float eps, theta;
    int H, R, rope_f32, rows;
    const double *freq;
};

constexpr int AP_MAX_ROWS = 32, AP_BLOCKS = 4;            // rows of a block; blocks per SM

// N elements, four at a time, and a store of all of them at once (8 or 16 bytes).
template <int N, typename T>
__device__ __forceinline__ void get(const T *p, float *y) {
#pragma unroll
    for (int i = 0; i < N; i += 4) load4(p + i, y + i);
}
template <int N, typename T>
__device__ __forceinline__ void put(T *p, const float *y) {
    struct alignas(N * sizeof(T) < 16 ? 8 : 16) Run { T v[N]; } o;
#pragma unroll
    for (int i = 0; i < N; i += 4) store4(o.v + i, y + i);
    *reinterpret_cast<Run *>(p) = o;
}

template <typename TI, typename TC, int HD>
__global__ void __launch_bounds__(128, AP_BLOCKS) k_kv_append(const __grid_constant__ AppendArgs a) {
    using Raw = uint4;                                    // as it lies in memory
    pdl_wait();
    pdl_launch_dependents();
    constexpr int E = sizeof(Raw) / sizeof(TI);           // elements of a load
    constexpr int TPH = HD / (2 * E), HPW = 32 / TPH;     // threads per head, heads per warp
    constexpr int AP_U = 16 / E;                          // query heads of a lane group in flight
    extern __shared__ float4 s_cs[];                      // a row's R / 4: pairs Ec + 2i, Ec + 2i + 1 at i·R/2E + c
    __shared__ int s_pos[AP_MAX_ROWS], s_page[AP_MAX_ROWS];   // position, -1: no sequence's row; page, -1: none
    const int t0 = blockIdx.x * a.rows, rows = min(a.rows, a.b.T - t0);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int KV = a.c.KV, R = a.R;
    const int sub = lane % TPH;
    const bool turns = sub < R / (2 * E);
    const int ea = turns ? E * sub : 2 * E * sub, eb = ea + (turns ? R / 2 : E);   // 2E·sub = R + 2E·(sub - R/2E)
    // lane groups of a row, over all its blocks: group `grp` takes the heads grp, grp + groups, ...
    const int groups = gridDim.y * (blockDim.x >> 5) * HPW;
    const int grp = (blockIdx.y * (blockDim.x >> 5) + warp) * HPW + lane / TPH;
    // keys and values change sides with every row: they are fewer than the lane groups
    auto kv_grp = [&](int t) { return t & 1 ? (grp < groups / 2 ? grp + groups - groups / 2 : grp - groups / 2) : grp; };

    // a row's query heads from h, and its key or value head h
    auto load_q = [&](Raw (&x)[AP_U][2], int t, int h) {
        const TI *src = (const TI *)a.q + (size_t)t * a.q_stride + h * HD;
#pragma unroll
        for (int u = 0; u < AP_U; ++u)
            if (h + u * groups < a.H) {
                x[u][0] = *reinterpret_cast<const Raw *>(src + u * groups * HD + ea);
                x[u][1] = *reinterpret_cast<const Raw *>(src + u * groups * HD + eb);
            }
    };
    auto load_kv = [&](Raw (&x)[2], int t, int h) {
        if (h >= 2 * KV) return;
        const TI *src = (h < KV ? (const TI *)a.k + (size_t)t * a.k_stride : (const TI *)a.v + (size_t)t * a.v_stride) +
                        (h < KV ? h : h - KV) * HD;
        x[0] = *reinterpret_cast<const Raw *>(src + ea);
        x[1] = *reinterpret_cast<const Raw *>(src + eb);
    };
    Raw nq[AP_U][2], nkv[2];                              // the next row's
    load_q(nq, t0, grp);
    load_kv(nkv, t0, kv_grp(t0));

    for (int r = warp; r < rows; r += blockDim.x >> 5) {
        const int t = t0 + r, i = kv_find_seq(a.b.q_start, a.b.n, t);
        int pos = -1, page = -1;
        if (i < a.b.n) {
            const KvSeq q = kv_seq(a.b, i);
            if (q.r0 >= 0 && t >= q.r0 && q.p0 >= 0) {
                pos = (int)min((long)q.p0 + (t - q.r0), 0x7fffffffl);
                if (t - q.r0 < q.len) {                   // (its place is in the table)
                    page = a.b.pages[(size_t)i * a.b.table_stride + pos / a.c.P];
                    if (page < 0 || page >= a.c.n_pages) {
                        page = -1;
                        if (lane == 0) atomicOr(a.c.status, KV_BAD_PAGE);
                    }
                }
            }
        }
        if (lane == 0) {
            s_pos[r] = pos;
            s_page[r] = page;
        }
    }
    // every sequence is looked at once, whether a row leads to it or not; the last warps first, which
    // have no row to find where there are few
    const size_t all = (size_t)gridDim.x * gridDim.y * blockDim.x;
    for (size_t i = ((size_t)blockIdx.y * gridDim.x + blockIdx.x + 1) * blockDim.x - 1 - tid; i < a.b.n; i += all)
        if (kv_seq(a.b, (int)i).bad) atomicOr(a.c.status, KV_BAD_POS);
    float gq[2 * E];
    auto gains = [&](const float *g, float *to) {
        get<E>(g + ea, to);
        get<E>(g + eb, to + E);
    };
    if (a.q_norm) gains(a.q_norm, gq);
    __syncthreads();
    for (int z = tid; z < rows * (R / 2); z += blockDim.x) {
        const int r = z / (R / 2), j = z - r * (R / 2), pos = s_pos[r];
        float sn, cs;
        if (a.rope_f32) {
            const float ang = __fmul_rn((float)pos, powf(a.theta, __fdiv_rn(-2.0f * (float)j, (float)R)));
            cs = cosf(ang);
            sn = sinf(ang);
        } else {
            const double turn = (double)pos * __ldg(a.freq + j);
            sincospif((float)(turn - 2.0 * rint(0.5 * turn)), &sn, &cs);
        }
        reinterpret_cast<float2 *>(s_cs)[r * (R / 2) + 2 * (j % E / 2 * (R / (2 * E)) + j / E) + (j & 1)] = make_float2(cs, sn);
    }
    __syncthreads();
    // the sums below are among the threads of one head, which agree on everything that branches
    const unsigned mask = ((1u << TPH) - 1u) << (lane / TPH * TPH);

    auto norm = [&](float (&y)[2 * E], const float (&g)[2 * E]) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * E; ++i) ss = fmaf(y[i], y[i], ss);
#pragma unroll
        for (int o = TPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        const float inv = rsqrtf(fmaf(ss, 1.0f / HD, a.eps));
#pragma unroll
        for (int i = 0; i < 2 * E; ++i) y[i] *= inv * g[i];
    };
    for (int r = 0; r < rows; ++r) {
        const int t = t0 + r, pos = s_pos[r], page = s_page[r];
        Raw xq[AP_U][2], xkv[2];
#pragma unroll
        for (int u = 0; u < AP_U; ++u) {
            xq[u][0] = nq[u][0];
            xq[u][1] = nq[u][1];
        }
        xkv[0] = nkv[0];
        xkv[1] = nkv[1];
        if (r + 1 < rows) {
            load_q(nq, t + 1, grp);
            load_kv(nkv, t + 1, kv_grp(t + 1));
        }
        if (pos < 0) continue;                            // a row of no sequence
        float4 cs[E / 2] = {};
        if (turns) {
#pragma unroll
            for (int i = 0; i < E / 2; ++i) cs[i] = s_cs[r * (R / 4) + i * (R / (2 * E)) + sub];
        }
        auto turn = [&](float (&y)[2 * E]) {
            if (!turns) return;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float c = i & 1 ? cs[i / 2].z : cs[i / 2].x, sn = i & 1 ? cs[i / 2].w : cs[i / 2].y;
                const float lo = y[i], hi = y[E + i];
                y[i] = fmaf(lo, c, -(hi * sn));
                y[E + i] = fmaf(hi, c, lo * sn);
            }
        };
        for (int h = grp;;) {
            TI *dst = (TI *)a.q_out + (size_t)t * a.qo_stride + h * HD;
#pragma unroll
            for (int u = 0; u < AP_U; ++u)
                if (h + u * groups < a.H) {
                    float y[2 * E];
                    get<E>(reinterpret_cast<const TI *>(&xq[u][0]), y);
                    get<E>(reinterpret_cast<const TI *>(&xq[u][1]), y + E);
                    if (a.q_norm) norm(y, gq);
                    turn(y);
                    put<E>(dst + u * groups * HD + ea, y);
                    put<E>(dst + u * groups * HD + eb, y + E);
                }
            h += AP_U * groups;
            if (h >= a.H) break;
            load_q(xq, t, h);
        }
        if (page < 0) continue;
        const size_t place = (size_t)page * a.c.sp + (size_t)(pos % a.c.P) * a.c.st;
        for (int h = kv_grp(t); h < 2 * KV;) {                  // keys, then values
            const bool isk = h < KV;
            float y[2 * E];
            get<E>(reinterpret_cast<const TI *>(&xkv[0]), y);
            get<E>(reinterpret_cast<const TI *>(&xkv[1]), y + E);
            if (isk) {
                if (a.k_norm) {
                    float gk[2 * E];
                    gains(a.k_norm, gk);
                    norm(y, gk);
                }
                turn(y);
            }
            TC *to = (TC *)(isk ? a.c.k : a.c.v) + place + (size_t)(isk ? h : h - KV) * a.c.sh;
            put<E>(to + ea, y);
            put<E>(to + eb, y + E);
            h += groups;
            load_kv(xkv, t, h);
        }
    }
}

template <typename TI, typename TC>
static cudaError_t launch_append(int hd, const AppendArgs &a, dim3 grid, dim3 block, cudaStream_t s) {
    const size_t smem = (size_t)a.rows * (a.R / 2) * sizeof(float2);
    return hd == 128 ? launch_pdl(k_kv_append<TI, TC, 128>, grid, block, smem, s, a)
                     : launch_pdl(k_kv_append<TI, TC, 64>, grid, block, smem, s, a);
}

int kv_attend_launch(const KvView &c, const KvMaps &maps, int hd, const KvRows &b, const void *q, size_t q_stride,
                     void *out, size_t out_stride, int type, int n_heads, float scale, int window, int max_new, void *ws,
                     cudaStream_t s);
int tensor_map(CUtensorMap *map, int type, int rank, const void *base, const uint64_t *dims, const uint64_t *strides,
               const uint32_t *box);
size_t kv_attend_ws_bytes(int hd);

static size_t type_bytes(int type) { return type == CPG_T_F32 ? 4 : 2; }
static bool type_ok(int type) { return type == CPG_T_F32 || type == CPG_T_F16 || type == CPG_T_BF16; }

}  // namespace cpg

using namespace cpg;

// A handle of `d`; with `like`, one that shares the device block (status word, frequencies) of a
// handle with the same rotation: the layers of a model report through one word.
static int kv_create(const cpg_kv_desc *d, const cpg_kv *like, cpg_kv **out) {
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
    KvDevice dev{};
    for (int j = 0; j < d->rope_dim / 2; ++j)
        dev.freq[j] = pow((double)d->rope_theta, -2.0 * j / d->rope_dim) / 3.14159265358979323846;
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
    kv->owns = !like;
    if (like) kv->v.status = like->v.status;
    if (ce == cudaSuccess && !like) ce = cudaMalloc(&kv->v.status, sizeof(KvDevice));
    if (ce == cudaSuccess && !like) ce = cudaMemcpy(kv->v.status, &dev, sizeof(KvDevice), cudaMemcpyHostToDevice);
    // (the copy out of pageable memory may return before it has landed; the caller's stream need not wait for it)
    if (ce == cudaSuccess && !like) ce = cudaStreamSynchronize(cudaStreamLegacy);
    if (ce != cudaSuccess) {
        if (kv->owns) cudaFree(kv->v.status);
        delete kv;
        cudaGetLastError();                              // reported; the next launch's check does not see it
        return cuda_fail(ce, "cpg_kv_create");
    }
    *out = kv;
    return CPG_OK;
}

extern "C" int cpg_kv_create(const cpg_kv_desc *d, cpg_kv **out) { return kv_create(d, nullptr, out); }
namespace cpg {
int kv_create_like(const cpg_kv_desc *d, const cpg_kv *like, cpg_kv **out) { return kv_create(d, like, out); }
}  // namespace cpg

extern "C" void cpg_kv_destroy(cpg_kv *kv) {
    if (!kv) return;
    if (kv->owns) cudaFree(kv->v.status);
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
    // positions and the ends of their tiles stay in 32 bits, and so do a row tile's tiles over all cached heads
    const long cap = std::min({(long)b->max_pages * kv->v.P, 0x7fff0000l, (1l << 36) / kv->v.KV});
    *r = KvRows{b->n_seqs, b->rows, b->q_start, b->pos0, b->pages, b->table_stride, (int)cap};
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
    a.freq = (const double *)((const char *)kv->v.status + offsetof(KvDevice, freq));
    // Many rows: runs that one wave of blocks takes, four warps each. Few rows: one a
    // block, and a row over several blocks while the rows alone leave SMs idle.
    const int per_warp = (type == CPG_T_F32 ? 256 : 512) / kv->hd, heads = std::max(n_heads, 2 * kv->v.KV), sms = sm_count();
    a.rows = std::min(AP_MAX_ROWS, (a.b.T + sms * AP_BLOCKS - 1) / (sms * AP_BLOCKS));
    int split = 1;
    while (split < 8 && (long)a.b.T * split < sms && heads > split * 4 * per_warp) split *= 2;
    const int warps = std::min(4, (heads + per_warp - 1) / per_warp);
    const dim3 grid((a.b.T + a.rows - 1) / a.rows, split), block(32 * warps);
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
    return kv_attend_ws_bytes(kv->hd);
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
    // (the kernels take it in powers of two)
    CPG_REQUIRE(scale > 0.0f && isfinite(scale * 1.4426950408889634f), "%s: scale %g must be positive, below 2.3e38", fn, (double)scale);
    CPG_REQUIRE(window >= 0, "%s: window %d", fn, window);
    CPG_REQUIRE((long)r.T * n_heads <= 0x7fff0000l, "%s: %d rows of %d heads", fn, r.T, n_heads);
    if (r.T == 0 || r.n == 0) return CPG_OK;
    if (window >= r.cap) window = 0;                      // hides nothing; the kernels' p - window - j stays in 32 bits
    rc = rows_ok(fn, "q", q, q_stride, n_heads, kv->hd, type);
    if (!rc) rc = rows_ok(fn, "out", out, out_stride, n_heads, kv->hd, type);
    if (rc) return rc;
    const size_t need = kv_attend_ws_bytes(kv->hd);
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
