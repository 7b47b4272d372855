// kv_attend.cu — attention of new rows over the paged key/value cache (qwen3_moe.c:135-155 per
// head, for many sequences at once).
//
// Row t of sequence i stands at position p = pos0[i] + t - q_start[i] and sees the cached positions
// j <= p (and j > p - window). For each query head h over its cached head kh = h / (H / KV):
//   out = sum_j e^(scale q.k_j - m) v_j / sum_j e^(scale q.k_j - m),   m = max_j scale q.k_j
//
// k_kv_attend: single rows (and any other shape). Bound by reading the cache once: 2 · HD · elements
// per position and cached head against 4 G flops each, G = H / KV.
//   work    A sequence's rows are G·len (row, head) pairs per cached head, in tiles of 16: the A
//           operand of one mma.m16n8k16. An item is (sequence, row tile, cached head), its units
//           are tiles of 64 positions. The units of all items, in order, are cut into equal ranges,
//           one per block: every block has the same number whatever the lengths, and a single long
//           sequence is spread over the whole GPU. Nothing about lengths is read on the host.
//   block   Four warps; warp w takes positions 16w..16w+15 of each tile through a ring of its own in
//           shared memory (16-byte cp.async, NU units of K or V in flight), so no warp waits for
//           another inside an item and the ring runs on across items. One pass: running maximum and
//           sum per row in registers, the scores' fragment is the A operand of P·V as it stands.
//           At an item's end the four warps' (m, l, o) are added in a fixed order.
//   join    A block's part of an item that others share goes to the workspace. Parts are joined in
//           groups of about the root of their number, each by the block that finishes its group last,
//           and the groups by the one that finishes last of all: two short steps where one block
//           reading up to 296 parts took longer than the attention itself. The order of additions
//           is that of the parts, so results do not depend on which block came last.
//   types   16-bit rows: one product per step, P rounded to the cache's type (its rounding is as
//           large as the result's own). f32 rows keep about 22 bits: over an f16 cache q (scaled by
//           a power of two per row) and P are split into two f16 terms; over a bf16 cache into three
//           bf16 terms; over an f32 cache K and V are split as well (three bf16 terms by truncation,
//           exact) and the six products of weight 2^-16 and more are kept. All sums are f32.
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv.cuh"

namespace cpg {

struct AttendArgs {
    KvRows b;
    KvView c;
    const void *q;
    void *out;
    size_t q_stride, out_stride;
    int H;
    float scale2;                    // scale · log2(e)
    int window;
    float *part;                     // 2 slots per block
    int *counters;                   // 2 per block (groups, by slot), then 1 per block (items)
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 16 bytes, or zeros where !ok (src is then not read).
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void *src, bool ok) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}

// d += a·b, m16n8k16, of f16 (HALF) or bf16 operands.
template <bool HALF>
__device__ __forceinline__ void mma_acc(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

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

constexpr int KD_WARPS = 4, KD_KEYS = 16, KD_TILE = KD_WARPS * KD_KEYS, KD_ROWS = 16;
constexpr int KD_RING = 24 * 1024;                       // bytes in a warp's ring
constexpr int KD_MAX_GRID = 512;
template <int HD> constexpr int kd_slot() { return 2 * KD_ROWS + HD / 2 * 32; }   // floats: m, l, o in fragment order
template <int HD> constexpr int kd_smem() { return KD_WARPS * KD_RING + 2 * kd_slot<HD>() * 4; }

// Sequence i's units: KV · row tiles · position tiles (the same for each of its items).
struct KdSeq {
    KvSeq s;
    int rt, nt, lo_t;
    long units;
};
__device__ __forceinline__ KdSeq kd_seq(const AttendArgs &a, int G, int i) {
    KdSeq q;
    q.s = kv_seq(a.b, a.c.P, i);
    q.rt = (int)(((long)q.s.len * G + KD_ROWS - 1) / KD_ROWS);
    q.lo_t = a.window ? max(0, q.s.p0 - a.window + 1) / KD_TILE : 0;
    q.nt = q.s.len ? (q.s.p0 + q.s.len + KD_TILE - 1) / KD_TILE - q.lo_t : 0;
    q.units = (long)a.c.KV * q.rt * q.nt;
    return q;
}

// A place in the order of units: item (seq, row tile, cached head), position tile.
struct KdCursor {
    int seq, sub, kt;                // sub = row tile · KV + cached head; kt from 0
    KdSeq q;
    int r0, nr, lo, hi;              // the row tile: first (row, head) pair, their number, positions seen
    __device__ __forceinline__ void item(const AttendArgs &a, int G) {
        r0 = sub / a.c.KV * KD_ROWS;
        nr = min(KD_ROWS, q.s.len * G - r0);
        lo = a.window ? max(0, q.s.p0 + r0 / G - a.window + 1) : 0;
        hi = q.s.p0 + (r0 + nr - 1) / G + 1;
    }
    __device__ __forceinline__ void next(const AttendArgs &a, int G) {
        if (++kt < q.nt) return;
        kt = 0;
        if (++sub < q.rt * a.c.KV) {
            item(a, G);
            return;
        }
        sub = 0;
        do {
            if (++seq >= a.b.n) return;
            q = kd_seq(a, G, seq);
        } while (q.units == 0);
        item(a, G);
    }
    __device__ __forceinline__ int head(const AttendArgs &a) const { return sub % a.c.KV; }
};

// Two states of a row pair joined: m, l (rows g and g + 8 of the lane) and NR registers of o.
template <int NR>
__device__ __forceinline__ void kd_join(float (&m)[2], float (&l)[2], float (&o)[NR][4], const float (&m2)[2],
                                        const float (&l2)[2], const float *o2, int stride) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const float mn = fmaxf(m[r], m2[r]), base = mn == -INFINITY ? 0.0f : mn;
        const float c1 = ex2(m[r] - base), c2 = ex2(m2[r] - base);
        l[r] = l[r] * c1 + l2[r] * c2;
        m[r] = mn;
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) o[i][2 * r + e] = o[i][2 * r + e] * c1 + o2[(4 * i + 2 * r + e) * stride] * c2;
    }
}

template <typename TI, typename TC, int HD>
__global__ void __launch_bounds__(KD_WARPS * 32, 2) k_kv_attend(const __grid_constant__ AttendArgs a) {
    constexpr bool F32C = std::is_same<TC, float>::value, F32I = std::is_same<TI, float>::value;
    constexpr bool HALF = std::is_same<TC, __half>::value;
    constexpr int NQ = !F32I ? 1 : HALF ? 2 : 3, NK = F32C ? 3 : 1;
    constexpr int ES = (int)sizeof(TC), ROWB = HD * ES, UNIT = KD_KEYS * ROWB;   // bytes of a key row, of a ring unit
    constexpr int NU = KD_RING / UNIT;
    constexpr int CPR = ROWB / 16, RPI = 32 / CPR;        // 16-byte chunks per row, rows per warp-wide copy
    constexpr int KS = HD / 16, NT = HD / 8;              // k steps of q·k, n tiles of p·v
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ long s_scan[KD_WARPS], s_off;
    __shared__ int s_seq, s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int G = a.H / a.c.KV;
    pdl_wait();
    pdl_launch_dependents();

    // ---- this block's range of units, and the item it starts in
    KdSeq mine{};
    long sum = 0;
    for (int i = tid; i < a.b.n; i += KD_WARPS * 32) {
        mine = kd_seq(a, G, i);
        sum += mine.units;
        if (mine.s.bad && blockIdx.x == 0) atomicOr(a.c.status, KV_BAD_POS);
    }
    const long own_sum = sum;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_scan[warp] = sum;
    __syncthreads();
    long U = 0;
#pragma unroll
    for (int w = 0; w < KD_WARPS; ++w) U += s_scan[w];
    const int NB = (int)min((long)gridDim.x, U);
    const int blk = blockIdx.x;
    if (blk >= NB) return;
    const long u0 = U * blk / NB, u1 = U * (blk + 1) / NB;
    long before = 0;
    for (int c0 = 0;; c0 += KD_WARPS * 32) {              // a chunk of sequences at a time; U > u0, so it ends
        long x = own_sum;
        if (a.b.n > KD_WARPS * 32) x = c0 + tid < a.b.n ? kd_seq(a, G, c0 + tid).units : 0;
        long inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        __syncthreads();
        if (lane == 31) s_scan[warp] = inc;
        __syncthreads();
        long base = before, all = 0;
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) {
            if (w < warp) base += s_scan[w];
            all += s_scan[w];
        }
        if (u0 >= base + inc - x && u0 < base + inc) {
            s_seq = c0 + tid;
            s_off = u0 - (base + inc - x);
        }
        before += all;
        if (u0 < before) break;
    }
    __syncthreads();
    KdCursor cur;
    cur.seq = s_seq;
    cur.q = kd_seq(a, G, cur.seq);
    cur.sub = (int)(s_off / cur.q.nt);
    cur.kt = (int)(s_off - (long)cur.sub * cur.q.nt);
    cur.item(a, G);
    KdCursor ld = cur;
    long ul = u0;                                         // unit pair (K, V) the loader is at
    bool ld_v = false;

    const uint32_t ring = smem_u32(smem) + warp * KD_RING;
    float *const s_o = reinterpret_cast<float *>(smem + KD_WARPS * KD_RING);
    size_t off[2] = {0, 0};
    bool ok[2] = {false, false};
    int vis_lo = 0, vis_hi = 0, slot_ld = 0;
    // one ring unit: this warp's 16 keys of the loader's tile, K first, then V
    auto load_unit = [&]() {
        if (ul < u1) {
            const int j0 = (ld.q.lo_t + ld.kt) * KD_TILE + warp * KD_KEYS;
            if (!ld_v) {
                vis_lo = ld.lo - j0;
                vis_hi = ld.hi - j0;
#pragma unroll
                for (int x = 0; x < 2; ++x) {             // pages hold multiples of 8 positions
                    ok[x] = 8 * x < vis_hi && 8 * x + 8 > vis_lo;
                    if (ok[x]) {
                        const int pg = (j0 + 8 * x) / a.c.P;
                        const int page = a.b.pages[(size_t)ld.seq * a.b.table_stride + pg];
                        ok[x] = page >= 0 && page < a.c.n_pages;
                        if (!ok[x] && lane == 0) atomicOr(a.c.status, KV_BAD_PAGE);
                        off[x] = ok[x] ? (size_t)page * a.c.sp + (size_t)(j0 + 8 * x - pg * a.c.P) * a.c.st +
                                             (size_t)ld.head(a) * a.c.sh : 0;
                    }
                }
            }
            if (vis_hi > 0 && vis_lo < KD_KEYS) {
                const TC *base = (const TC *)(ld_v ? a.c.v : a.c.k);
                const int c = lane % CPR;
#pragma unroll
                for (int i = 0; i < KD_KEYS / RPI; ++i) {
                    const int r = i * RPI + lane / CPR;
                    const int sw = !F32C ? (r & 7) : ld_v ? ((r >> 1) & 3) * 2 : (r & 1) * 4;
                    const bool in = ok[r >> 3] && r < vis_hi && r >= vis_lo;
                    const TC *src = in ? base + off[r >> 3] + (size_t)(r & 7) * a.c.st + c * (16 / ES) : base;
                    cp_async16_or_zero(ring + slot_ld * UNIT + r * ROWB + ((c ^ sw) << 4), src, in);
                }
            }
            if (ld_v) {
                if (++ul < u1) ld.next(a, G);
            }
            ld_v = !ld_v;
        }
        cp_async_commit();
        slot_ld = slot_ld + 1 == NU ? 0 : slot_ld + 1;
    };
#pragma unroll 1
    for (int i = 0; i < NU - 1; ++i) load_unit();

    uint32_t qa[NQ][KS][4];
    float o[NT][4], m[2], l[2], sc[2];
    int p_row[2];
    bool fresh = true;
    int slot = 0;
    for (long u = u0; u < u1; ++u) {
        if (fresh) {                                      // a new item: its rows of q, empty sums
            fresh = false;
            const int kh = cur.head(a);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int rr = cur.r0 + g + 8 * r;
                const bool live = g + 8 * r < cur.nr;
                const int tok = rr / G;
                p_row[r] = live ? cur.q.s.p0 + tok : cur.hi - 1;
                const TI *src = (const TI *)a.q + (size_t)(cur.q.s.r0 + tok) * a.q_stride + (size_t)(kh * G + rr - tok * G) * HD;
                sc[r] = a.scale2;
                if constexpr (!F32I) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            qa[0][ks][r + 2 * x] = live ? *reinterpret_cast<const uint32_t *>(src + 16 * ks + 8 * x + 2 * t) : 0u;
                } else {
                    float f[KS][4];
                    float mx = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        // f32 cache: K is read four elements a lane, so step ks of lane t is elements
                        // 4t..4t+3 of the 16; otherwise 2t, 2t+1 and 8 further
                        if constexpr (F32C) {
                            const float4 v = live ? *reinterpret_cast<const float4 *>(src + 16 * ks + 4 * t) : make_float4(0.f, 0.f, 0.f, 0.f);
                            f[ks][0] = v.x; f[ks][1] = v.y; f[ks][2] = v.z; f[ks][3] = v.w;
                        } else {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const float2 v = live ? *reinterpret_cast<const float2 *>(src + 16 * ks + 8 * x + 2 * t) : make_float2(0.f, 0.f);
                                f[ks][2 * x] = v.x;
                                f[ks][2 * x + 1] = v.y;
                            }
                        }
                        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(f[ks][0]), fabsf(f[ks][1])), fmaxf(fabsf(f[ks][2]), fabsf(f[ks][3]))));
                    }
                    float s = 1.0f;
                    if constexpr (HALF) {                 // the row into f16's range by a power of two
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const int eb = min(max((int)(__float_as_uint(mx) >> 23), 1), 253);
                        s = __uint_as_float((uint32_t)(254 - eb) << 23);
                        sc[r] = a.scale2 * __uint_as_float((uint32_t)eb << 23);
                    }
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            uint32_t tm[NQ];
                            split_pair<HALF, NQ>(f[ks][2 * x] * s, f[ks][2 * x + 1] * s, tm);
#pragma unroll
                            for (int n = 0; n < NQ; ++n) qa[n][ks][r + 2 * x] = tm[n];
                        }
                }
                m[r] = -INFINITY;
                l[r] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        }
        const int j0 = (cur.q.lo_t + cur.kt) * KD_TILE + warp * KD_KEYS;
        const bool active = j0 < cur.hi && j0 + KD_KEYS > cur.lo;
        float s[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {            // K, then V
            load_unit();
            cp_async_wait_group<NU - 1>();
            __syncwarp();
            const uint32_t at = ring + slot * UNIT;
            if (active && half == 0) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
                    if constexpr (!F32C) {
                        const int r = 8 * n + (lane & 7);
#pragma unroll
                        for (int k2 = 0; k2 < KS / 2; ++k2) {
                            uint32_t b[4];
                            ldsm4(b, at + r * ROWB + (((4 * k2 + (lane >> 3)) ^ (r & 7)) << 4));
#pragma unroll
                            for (int q = NQ - 1; q >= 0; --q) {
                                mma_acc<HALF>(s[n], qa[q][2 * k2], b[0], b[1]);
                                mma_acc<HALF>(s[n], qa[q][2 * k2 + 1], b[2], b[3]);
                            }
                        }
                    } else {
                        const int r = 8 * n + g;
#pragma unroll
                        for (int ks = 0; ks < KS; ++ks) {
                            float4 v;
                            asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                                         : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                                         : "r"(at + r * ROWB + (((4 * ks + t) ^ ((r & 1) * 4)) << 4)));
                            uint32_t b0[NK], b1[NK];
                            split_pair<HALF, NK>(v.x, v.y, b0);
                            split_pair<HALF, NK>(v.z, v.w, b1);
#pragma unroll
                            for (int d = NK - 1; d >= 0; --d)          // terms of weight 2^-8d
#pragma unroll
                                for (int k = 0; k <= d; ++k) mma_acc<HALF>(s[n], qa[d - k][ks], b0[k], b1[k]);
                        }
                    }
                }
                const int span = (cur.nr - 1) / G + 1;      // positions between the tile's rows, at most
                const bool cut = j0 + KD_KEYS > cur.hi - span || (a.window && j0 < cur.lo + span);
                if (cut) {                                // some row of the tile does not see all 16
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = j0 + 8 * n + 2 * t + (e & 1), p = p_row[e >> 1];
                            if (j > p || (a.window && j <= p - a.window)) s[n][e] = -INFINITY;
                        }
                }
                float c[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float mx = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                    const float mn = fmaxf(m[r], mx * sc[r]), base = mn == -INFINITY ? 0.0f : mn;
                    c[r] = ex2(m[r] - base);
                    m[r] = mn;
                    float add = 0.0f;
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 2 * r; e < 2 * r + 2; ++e) {
                            s[n][e] = ex2(fmaf(s[n][e], sc[r], -base));
                            add += s[n][e];
                        }
                    l[r] = fmaf(l[r], c[r], add);
                }
                if (__any_sync(0xffffffffu, c[0] != 1.0f || c[1] != 1.0f)) {
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        o[i][0] *= c[0]; o[i][1] *= c[0];
                        o[i][2] *= c[1]; o[i][3] *= c[1];
                    }
                }
            } else if (active) {
                uint32_t pa[NQ][4];
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        uint32_t tm[NQ];
                        split_pair<HALF, NQ>(s[n][2 * r], s[n][2 * r + 1], tm);
#pragma unroll
                        for (int q = 0; q < NQ; ++q) pa[q][r + 2 * n] = tm[q];
                    }
                if constexpr (!F32C) {
                    const int r = lane & 15;
#pragma unroll
                    for (int n2 = 0; n2 < NT / 2; ++n2) {
                        uint32_t b[4];
                        ldsm4t(b, at + r * ROWB + (((2 * n2 + (lane >> 4)) ^ (r & 7)) << 4));
#pragma unroll
                        for (int q = NQ - 1; q >= 0; --q) {
                            mma_acc<HALF>(o[2 * n2], pa[q], b[0], b[1]);
                            mma_acc<HALF>(o[2 * n2 + 1], pa[q], b[2], b[3]);
                        }
                    }
                } else {
                    // lane (g, t) reads columns 32cb + 4g.. of keys 2t, 2t+1, 2t+8, 2t+9: n tile 4cb + x
                    // is the columns 32cb + 4n + x
#pragma unroll
                    for (int cb = 0; cb < HD / 32; ++cb) {
                        float v[4][4];
#pragma unroll
                        for (int y = 0; y < 4; ++y) {
                            const int r = 2 * t + (y & 1) + 8 * (y >> 1);
                            asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];"
                                         : "=f"(v[y][0]), "=f"(v[y][1]), "=f"(v[y][2]), "=f"(v[y][3])
                                         : "r"(at + r * ROWB + (((8 * cb + g) ^ (((r >> 1) & 3) * 2)) << 4)));
                        }
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            uint32_t b0[NK], b1[NK];
                            split_pair<HALF, NK>(v[0][x], v[1][x], b0);
                            split_pair<HALF, NK>(v[2][x], v[3][x], b1);
#pragma unroll
                            for (int d = NK - 1; d >= 0; --d)
#pragma unroll
                                for (int k = 0; k <= d; ++k) mma_acc<HALF>(o[4 * cb + x], pa[d - k], b0[k], b1[k]);
                        }
                    }
                }
            }
            __syncwarp();
            slot = slot + 1 == NU ? 0 : slot + 1;
        }
        const bool item_ends = cur.kt + 1 == cur.q.nt;
        if (!item_ends && u + 1 < u1) {
            cur.next(a, G);
            continue;
        }

        // ---- the item, or this block's part of it, is done: join the four warps
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
        auto put = [&](float *to) {                       // m, l and o in fragment order
            if (t == 0) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    to[g + 8 * r] = m[r];
                    to[KD_ROWS + g + 8 * r] = l[r];
                }
            }
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) to[2 * KD_ROWS + (4 * i + e) * 32 + lane] = o[i][e];
        };
        auto add = [&](const float *from) {
            const float m2[2] = {from[g], from[g + 8]}, l2[2] = {from[KD_ROWS + g], from[KD_ROWS + g + 8]};
            kd_join<NT>(m, l, o, m2, l2, from + 2 * KD_ROWS + lane, 32);
        };
        if (warp >= 2) put(s_o + (warp - 2) * kd_slot<HD>());
        __syncthreads();
        if (warp < 2) add(s_o + warp * kd_slot<HD>());
        __syncthreads();
        if (warp == 1) put(s_o);
        __syncthreads();
        if (warp == 0) add(s_o);

        // ---- who else has a part of it: unit range [ua, ue) of the item, owners b0..b1
        const long ua = u - cur.kt, ue = ua + cur.q.nt;
        const int b0 = (int)(((ua + 1) * NB - 1) / U), b1 = (int)((ue * NB - 1) / U);
        bool write = b0 == b1;
        if (!write) {
            const int np = b1 - b0 + 1, p = blk - b0;
            int gs = 1;
            while (gs * gs < np) ++gs;
            if (np <= 8) gs = np;
            const int ng = (np + gs - 1) / gs, gi = p / gs, n_in = min(gs, np - gi * gs);
            auto slot_of = [&](int part) { return (size_t)(part == 0 ? 2 * b0 + 1 : 2 * (b0 + part)); };
            if (warp == 0) put(a.part + slot_of(p) * kd_slot<HD>());
            // parts first, first + step, ... (n of them) joined by this block if it is the last of `want`
            auto join = [&](int *counter, int want, int first, int step, int n) -> bool {
                if (warp == 0) {
                    __threadfence();
                    __syncwarp();
                    int last = 0;
                    if (lane == 0) {
                        last = atomicAdd(counter, 1) == want - 1;
                        if (last) *counter = 0;           // ready for the next call
                        __threadfence();
                    }
                    if (lane == 0) s_last = last;
                }
                __syncthreads();
                const bool last = s_last != 0;
                __syncthreads();
                if (!last) return false;
                // warp w: a quarter of the registers of o, for the rows that hold something
                float mm[2] = {-INFINITY, -INFINITY}, ll[2] = {0.0f, 0.0f};
                const bool both = cur.nr > 8;
                for (int k = 0; k < n; ++k) {
                    const float *src = a.part + slot_of(first + k * step) * kd_slot<HD>();
                    mm[0] = fmaxf(mm[0], __ldcg(src + g));
                    if (both) mm[1] = fmaxf(mm[1], __ldcg(src + g + 8));
                }
                float oo[NT / 4][4] = {};
                const float base[2] = {mm[0] == -INFINITY ? 0.0f : mm[0], mm[1] == -INFINITY ? 0.0f : mm[1]};
#pragma unroll 4
                for (int k = 0; k < n; ++k) {
                    const float *src = a.part + slot_of(first + k * step) * kd_slot<HD>();
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        if (r && !both) break;
                        const float w = ex2(__ldcg(src + g + 8 * r) - base[r]);
                        ll[r] = fmaf(w, __ldcg(src + KD_ROWS + g + 8 * r), ll[r]);
#pragma unroll
                        for (int i = 0; i < NT / 4; ++i)
#pragma unroll
                            for (int e = 2 * r; e < 2 * r + 2; ++e)
                                oo[i][e] = fmaf(w, __ldcg(src + 2 * KD_ROWS + (4 * (warp * (NT / 4) + i) + e) * 32 + lane), oo[i][e]);
                    }
                }
                // back together in warp 0
                float *to = s_o;
                if (warp == 0 && t == 0) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        to[g + 8 * r] = mm[r];
                        to[KD_ROWS + g + 8 * r] = ll[r];
                    }
                }
#pragma unroll
                for (int i = 0; i < NT / 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[2 * KD_ROWS + (4 * (warp * (NT / 4) + i) + e) * 32 + lane] = oo[i][e];
                __syncthreads();
                if (warp == 0) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        m[r] = to[g + 8 * r];
                        l[r] = to[KD_ROWS + g + 8 * r];
                    }
#pragma unroll
                    for (int i = 0; i < NT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][e] = to[2 * KD_ROWS + (4 * i + e) * 32 + lane];
                }
                return true;
            };
            int *const groups = a.counters, *const items = a.counters + 2 * KD_MAX_GRID;
            if (join(groups + slot_of(gi * gs), n_in, gi * gs, 1, n_in)) {
                if (ng == 1) write = true;
                else {
                    if (warp == 0) put(a.part + slot_of(gi * gs) * kd_slot<HD>());
                    write = join(items + b0, ng, 0, gs, ng);
                }
            }
        }
        if (write && warp == 0) {
            const int kh = cur.head(a);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                if (g + 8 * r >= cur.nr) continue;
                const int rr = cur.r0 + g + 8 * r, tok = rr / G;
                TI *dst = (TI *)a.out + (size_t)(cur.q.s.r0 + tok) * a.out_stride + (size_t)(kh * G + rr - tok * G) * HD;
                const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
                if constexpr (!F32C) {
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        const float v[2] = {o[i][2 * r] * inv, o[i][2 * r + 1] * inv};
                        if constexpr (F32I) *reinterpret_cast<float2 *>(dst + 8 * i + 2 * t) = make_float2(v[0], v[1]);
                        else {
                            uint32_t w[1];
                            split_pair<HALF, 1>(v[0], v[1], w);
                            *reinterpret_cast<uint32_t *>(dst + 8 * i + 2 * t) = w[0];
                        }
                    }
                } else {
#pragma unroll
                    for (int cb = 0; cb < HD / 32; ++cb)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            *reinterpret_cast<float4 *>(dst + 32 * cb + 8 * t + 4 * e) =
                                make_float4(o[4 * cb][2 * r + e] * inv, o[4 * cb + 1][2 * r + e] * inv,
                                            o[4 * cb + 2][2 * r + e] * inv, o[4 * cb + 3][2 * r + e] * inv);
                }
            }
        }
        __syncthreads();                                  // s_o and s_last are free again
        fresh = true;
        if (u + 1 < u1) cur.next(a, G);
    }
    cp_async_wait_all();
}

// Workspace: counters, then the parts.
constexpr size_t KD_COUNTERS = (3 * KD_MAX_GRID * sizeof(int) + 255) / 256 * 256;

size_t kv_attend_ws_bytes(int hd, int type) {
    const size_t slot = (hd == 128 ? kd_slot<128>() : kd_slot<64>()) * sizeof(float);
    return KD_COUNTERS + 2 * (size_t)KD_MAX_GRID * slot;
}

template <typename TI, typename TC, int HD>
static int launch_kd(const AttendArgs &a, cudaStream_t s) {
    static std::atomic<bool> set[64];                    // once per device
    int dev = 0;
    CPG_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
        const int rc = allow_max_smem((const void *)k_kv_attend<TI, TC, HD>);
        if (rc) return rc;
        if (dev < 64) set[dev].store(true, std::memory_order_release);
    }
    const int grid = std::min(KD_MAX_GRID, 2 * sm_count());
    const cudaError_t ce = launch_pdl(k_kv_attend<TI, TC, HD>, dim3(grid), dim3(KD_WARPS * 32), (size_t)kd_smem<HD>(), s, a);
    return ce == cudaSuccess ? CPG_OK : cuda_fail(ce, "cpg_kv_attend");
}
template <typename TI, typename TC>
static int launch_hd(int hd, const AttendArgs &a, cudaStream_t s) {
    return hd == 128 ? launch_kd<TI, TC, 128>(a, s) : launch_kd<TI, TC, 64>(a, s);
}

int kv_attend_launch(const KvView &c, int hd, const KvRows &b, const void *q, size_t q_stride, void *out,
                     size_t out_stride, int type, int n_heads, float scale, int window, int max_new, void *ws,
                     cudaStream_t s) {
    const AttendArgs a{b, c, q, out, q_stride, out_stride, n_heads, scale * 1.4426950408889634f, window,
                       (float *)((uint8_t *)ws + KD_COUNTERS), (int *)ws};
    if (type == CPG_T_F32)
        return c.type == CPG_T_F32   ? launch_hd<float, float>(hd, a, s)
               : c.type == CPG_T_F16 ? launch_hd<float, __half>(hd, a, s)
                                     : launch_hd<float, __nv_bfloat16>(hd, a, s);
    return type == CPG_T_F16 ? launch_hd<__half, __half>(hd, a, s) : launch_hd<__nv_bfloat16, __nv_bfloat16>(hd, a, s);
}

}  // namespace cpg
