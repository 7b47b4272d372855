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
//   block   One producer warp, four consumer warps. The producer walks the block's units and keeps a
//           ring of K and V tiles of 64 positions full by tensor TMA: a box is as many positions as
//           lie in one page (the largest power of two dividing the page size, at most 64) by 128
//           bytes, swizzled; a box without a page reads zeros from outside the pool. Consumer warp
//           w takes positions 16w..16w+15 of every tile; it waits for tiles only, never for another
//           consumer inside an item, and the ring runs on across items. One pass: running maximum
//           and sum per row in registers, the scores' fragment is the A operand of P·V as it
//           stands. At an item's end the four warps' (m, l, o) are added in a fixed order.
//           Places of a page behind what is cached, or in front of the window, may hold anything: scores
//           there are replaced, and so are the values' fragments (a weight of zero does not silence a NaN).
//   join    A block's part of an item that others share goes to the workspace. Parts are joined in
//           groups of about the root of their number, each by the block that finishes its group last,
//           and the groups by the one that finishes last of all: two short steps where one block
//           reading up to 296 parts took longer than the attention itself. The order of additions
//           is that of the parts, so results do not depend on which block came last.
//           What counts the parts is one acquire-release addition: a sequentially consistent fence waits
//           for the tiles in flight, 15 us where a block ends an item in the middle of its range.
//   measured  (on the device, calls in a captured graph) 128 bf16 rows over 1000-8000 positions (1.14 GB):
//           187 us, 0.93 of the copy bandwidth; 64 f32 rows over f16, 128-4096 positions (294 MB): 56 us,
//           0.80 (59 from call to call), over bf16 60 us, over f32 (586 MB) 113 us, 0.80; one bf16
//           row over 128K positions (268 MB): 59 us, 0.70 (4.5 us until the first tile, 41 of tiles at the
//           copy bandwidth, the rest the joins of 74 parts); one f32 row over 512 positions: 11 us.
//   types   16-bit rows: one product per step, P rounded to the cache's type (its rounding is as
//           large as the result's own). f32 rows keep about 22 bits: over an f16 cache q (scaled by
//           a power of two per row, as far up as f16 goes: the small elements of a row with a large one
//           keep their bits) and P are split into two f16 terms; over a bf16 cache into three
//           bf16 terms; over an f32 cache K and V are split as well (three bf16 terms by truncation,
//           exact) and the six products of weight 2^-16 and more are kept. The tensor core cuts
//           off what it adds to an accumulator instead of rounding, so for f32 rows an accumulator
//           takes few steps, the smallest products first, and is added to the running sum by a
//           rounded f32 addition (errors 2.9e-6 without that, 3e-7 with it). Where a tile has at most 8
//           rows the other 8 of the operand hold the second term of the same rows, and one product
//           does the work of two (PACK).
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_attend.cuh"

namespace cpg {

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// d = a·b
template <bool HALF>
__device__ __forceinline__ void mma_new(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (HALF)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ float4 lds4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
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

// The terms of a pair of elements as fragment register `at` of the operands, one operand a term. Packed:
// rows 8.. of the first operand hold the second term of rows 0..7.
template <bool PACK, int NP, int NQ>
__device__ __forceinline__ void place_terms(uint32_t (&w)[NP][4], const uint32_t (&tm)[NQ], int at) {
    if constexpr (PACK) {
        w[0][at] = tm[0];
        w[0][at + 1] = tm[1];
        if constexpr (NP > 1) {
            w[1][at] = tm[2];
            w[1][at + 1] = 0u;
        }
    } else {
#pragma unroll
        for (int n = 0; n < NQ; ++n) w[n][at] = tm[n];
    }
}

constexpr int KD_WARPS = 4, KD_KEYS = 16, KD_TILE = KD_WARPS * KD_KEYS, KD_ROWS = 16;
constexpr int KD_THREADS = (KD_WARPS + 1) * 32;
constexpr int KD_RING = 96 * 1024;
template <int HD> constexpr int kd_slot() { return 2 * KD_ROWS + HD / 2 * 32; }   // floats: m, l, o in fragment order
constexpr int KD_JOIN = 24;                              // parts of one join, at most (root of KV_MAX_GRID)
// behind the ring: q's terms (f32 rows) and later three quarters of half the warps' sums, both
// 3 · HD / 16 · 512 bytes; the maxima and sums of what is joined
template <int HD> constexpr int kd_buf() { return 3 * HD / 16 * 512; }
template <int HD> constexpr int kd_smem() { return 1008 + KD_RING + kd_buf<HD>() + KD_JOIN * 2 * KD_ROWS * 4; }

// Sequence i's units: for each row tile, KV · (KD_FIXED + the position tiles its rows see).
// Beginning and ending an item takes a block as long as some four tiles (5 us against 1.4 us for 64
// bf16 positions), so an item counts for KD_FIXED tiles more than it has: without them the blocks
// that end one item and begin the next finish last (64 f32 rows over f16 70 us against 61, 128K
// positions and one row 63 against 59).
constexpr int KD_FIXED = 4;
struct KdSeq {
    KvSeq s;
    int rt;                          // row tiles
    long units;
};
// Row tile r of a sequence: its (row, head) pairs from r0, nr of them, and the positions they see.
template <int ROWS>
struct KdRows {
    int r0, nr, lo, hi, lo_t, nt;
    __device__ __forceinline__ KdRows() {}
    __device__ __forceinline__ KdRows(const AttendArgs &a, int G, const KvSeq &s, int r) {
        r0 = r * ROWS;
        nr = min(ROWS, s.len * G - r0);
        lo = a.window ? max(0, s.p0 + r0 / G - a.window + 1) : 0;
        hi = s.p0 + (r0 + nr - 1) / G + 1;
        lo_t = lo / KD_TILE;
        nt = (hi + KD_TILE - 1) / KD_TILE - lo_t;
    }
};
template <int ROWS>
__device__ __forceinline__ KdSeq kd_seq(const AttendArgs &a, int G, int i) {
    KdSeq q;
    q.s = kv_seq(a.b, i);
    q.rt = (int)(((long)q.s.len * G + ROWS - 1) / ROWS);
    long tiles = 0;
    for (int r = 0; r < q.rt; ++r) tiles += KD_FIXED + KdRows<ROWS>(a, G, q.s, r).nt;
    q.units = a.c.KV * tiles;
    return q;
}

// A place in the order of units: item (seq, row tile, cached head), position tile.
template <int ROWS>
struct KdCursor {
    int seq, rt, kh, kt;             // kt from -KD_FIXED
    KvSeq s;
    int n_rt;
    KdRows<ROWS> r;
    __device__ __forceinline__ void next_item(const AttendArgs &a, int G) {
        kt = -KD_FIXED;
        if (++kh < a.c.KV) return;
        kh = 0;
        if (++rt == n_rt) {
            rt = 0;
            do {
                if (++seq >= a.b.n) return;
                s = kv_seq(a.b, seq);
            } while (s.len == 0);
            n_rt = (int)(((long)s.len * G + ROWS - 1) / ROWS);
        }
        r = KdRows<ROWS>(a, G, s, rt);
    }
};

template <typename TI, typename TC, int HD, bool PACK>
__global__ void __launch_bounds__(KD_THREADS, 2) k_kv_attend(const __grid_constant__ AttendArgs a,
                                                             const __grid_constant__ CUtensorMap tm_k,
                                                             const __grid_constant__ CUtensorMap tm_v) {
    constexpr bool F32C = std::is_same<TC, float>::value, F32I = std::is_same<TI, float>::value;
    constexpr bool HALF = std::is_same<TC, __half>::value;
    constexpr int NQ = !F32I ? 1 : HALF ? 2 : 3, NK = F32C ? 3 : 1;
    constexpr int NP = PACK ? NQ - 1 : NQ;                // operands that hold the terms of q or P
    constexpr int ROWS = PACK ? 8 : KD_ROWS, RL = ROWS / 8;               // rows of a tile; of a lane
    constexpr int ES = (int)sizeof(TC), PARTS = HD * ES / 128, UNIT = KD_TILE * HD * ES;  // 128-byte columns; ring unit
    constexpr int NU = KD_RING / UNIT;
    constexpr int KS = HD / 16, NT = HD / 8;              // k steps of q·k, n tiles of p·v
    constexpr int KU = F32C ? 1 : KS / 2;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t *const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t full[NU], empty[NU];
    __shared__ long s_scan[KD_WARPS + 1], s_off;
    __shared__ KdCursor<ROWS> s_cur;
    __shared__ int s_last, s_abort;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int G = a.H / a.c.KV;
    if (tid == 0) {
        for (int i = 0; i < NU; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], KD_WARPS);
        }
        fence_mbar_init();
        s_abort = 0;
    }
    if (tid == KD_WARPS * 32) {
        prefetch_map(&tm_k);
        prefetch_map(&tm_v);
    }
    pdl_wait();
    pdl_launch_dependents();

    // ---- this block's range of units, and the item it starts in
    const int n = a.b.n;
    KdSeq mine{};
    long U = 0, before = 0, u0 = 0, u1 = 0;
    int NB = 0;
    const int blk = blockIdx.x;
    KvCut cut(0, 1);
    auto range = [&](long total) {                        // false: nothing for this block
        U = total;
        NB = (int)min((long)gridDim.x, U);
        if (blk >= NB) return false;
        cut = KvCut(U, NB);
        u0 = cut.start(blk);
        u1 = cut.start(blk + 1);
        return true;
    };
    if (n > KD_THREADS) {                                 // more sequences than threads: their sum first
        long sum = 0;
        for (int i = tid; i < n; i += KD_THREADS) {
            const KdSeq q = kd_seq<ROWS>(a, G, i);
            sum += q.units;
            if (q.s.bad && blk == 0) atomicOr(a.c.status, KV_BAD_POS);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) s_scan[warp] = sum;
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int w = 0; w <= KD_WARPS; ++w) sum += s_scan[w];
        if (!range(sum)) return;
        __syncthreads();
    }
    for (int c0 = 0; c0 < n; c0 += KD_THREADS) {          // THREADS sequences at a time
        long inc = 0;
        if (c0 + tid < n) {
            mine = kd_seq<ROWS>(a, G, c0 + tid);
            inc = mine.units;
            // (of more, all have been looked at above: this loop ends at the block's own)
            if (n <= KD_THREADS && mine.s.bad && blk == 0) atomicOr(a.c.status, KV_BAD_POS);
        }
        const long x = inc;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) s_scan[warp] = inc;
        __syncthreads();
        long base = before, all = 0;
#pragma unroll
        for (int w = 0; w <= KD_WARPS; ++w) {
            if (w < warp) base += s_scan[w];
            all += s_scan[w];
        }
        if (n <= KD_THREADS && !range(all)) return;
        if (c0 + tid < n && u0 >= base + inc - x && u0 < base + inc) {
            KdCursor<ROWS> c;
            c.seq = c0 + tid;
            c.s = mine.s;
            c.n_rt = mine.rt;
            s_off = u0 - (base + inc - x);
            s_cur = c;
        }
        before += all;
        __syncthreads();
        if (u0 < before) break;
    }
    if (u0 >= u1) return;                                 // no sequences at all
    if (warp == 0) {                                      // the row tile that holds unit s_off, 32 at a time
        KdCursor<ROWS> c = s_cur;
        long off = s_off;
        for (int r0 = 0; r0 < c.n_rt; r0 += 32) {
            const int r = r0 + lane;
            int each = 0;
            if (r < c.n_rt) {
                c.r = KdRows<ROWS>(a, G, c.s, r);
                each = KD_FIXED + c.r.nt;
            }
            long inc = (long)each * a.c.KV;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const long y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            const long all = __shfl_sync(0xffffffffu, inc, 31), from = inc - (long)each * a.c.KV;
            if (off < all) {
                if (off >= from && off < inc) {
                    c.rt = r;
                    c.kh = (int)(off - from) / each;
                    c.kt = (int)(off - from) - c.kh * each - KD_FIXED;
                    s_cur = c;
                }
                break;
            }
            off -= all;
        }
    }
    __syncthreads();
    KdCursor<ROWS> cur = s_cur;
    volatile int *const abort_flag = &s_abort;

    if (warp == KD_WARPS) {
        // ---- producer: lane b loads box b of every unit (box = position group · PARTS + column, at
        // most 8 groups of 4)
        const int boxes = KD_TILE / a.box * PARTS;
        const uint32_t ring = smem_u32(smem);
        int slot = 0, turn = 0;
        bool stop = false;
        for (long u = u0; u < u1 && !stop;) {
            if (cur.kt < 0) {                             // nothing to load
                u -= cur.kt;
                cur.kt = 0;
                if (u >= u1) break;
            }
            const int n_here = (int)min((long)(cur.r.nt - cur.kt), u1 - u);
            // page and place of this lane's box of tile i; the next tile's is asked for ahead
            auto find = [&](int i, int &page, int &place) {
                const int j = (cur.r.lo_t + cur.kt + i) * KD_TILE + lane / PARTS * a.box;
                place = -1;                               // nothing of it is seen
                if (lane < boxes && i < n_here && j < cur.r.hi && j + a.box > cur.r.lo) {
                    const int pg = j / a.c.P;
                    page = a.b.pages[(size_t)cur.seq * a.b.table_stride + pg];
                    place = j - pg * a.c.P;
                }
            };
            int next_page = 0, next_place;
            find(0, next_page, next_place);
            for (int i = 0; i < n_here && !stop; ++i) {
                const bool inside = next_place >= 0 && next_page >= 0 && next_page < a.c.n_pages;
                if (next_place >= 0 && !inside) atomicOr(a.c.status, KV_BAD_PAGE);
                const int page = inside ? next_page : a.c.n_pages, place = max(next_place, 0);   // outside the pool: zeros
                find(i + 1, next_page, next_place);
#pragma unroll
                for (int half = 0; half < 2; ++half) {    // K, then V
                    const bool ok = !turn || *abort_flag || mbar_wait(&empty[slot], (uint32_t)(turn - 1) & 1u);
                    if (!ok) {
                        *abort_flag = 1;
                        atomicOr(a.c.status, KV_TIMEOUT);
                    }
                    stop = __any_sync(0xffffffffu, !ok || *abort_flag);
                    if (stop) break;
                    if (lane == 0) mbar_arrive_expect_tx(&full[slot], UNIT);
                    __syncwarp();
                    if (lane < boxes)
                        tma_load_4d(ring + slot * UNIT + lane % PARTS * (KD_TILE * 128) + lane / PARTS * a.box * 128, half ? &tm_v : &tm_k,
                                    lane % PARTS * (128 / ES), place, cur.kh, page, &full[slot]);
                    if (++slot == NU) {
                        slot = 0;
                        ++turn;
                    }
                }
            }
            u += n_here;
            if (u < u1 && !stop) cur.next_item(a, G);
        }
        if (stop) {                                       // copies in flight land before the block may end
            for (int i = 0; i < NU; ++i) {
                const int n = turn + (i < slot);          // fills of slot i
                if (n) mbar_wait(&full[i], (uint32_t)(n - 1) & 1u);
            }
        }
        return;
    }

    // ---- consumers
    const uint32_t ring = smem_u32(smem);
    float *const s_o = reinterpret_cast<float *>(smem + KD_RING);
    uint4 *const s_q = reinterpret_cast<uint4 *>(s_o);    // f32 rows: q's terms in fragment order
    uint32_t qa[NQ == 1 ? KS : 1][4];
    float o[NT][4], m[2], l[2], sc[2];
    int p_row[2];
    int slot = 0;
    uint32_t phase = 0;
    for (long u = u0; u < u1;) {
        if (cur.kt < 0) {
            u -= cur.kt;
            cur.kt = 0;
            if (u >= u1) break;                           // its first tile is the next block's
        }
        {                                                 // an item: its rows of q, empty sums
            const int kh = cur.kh;
            float f[2][F32I ? KS : 1][4];
            float up[2];
            m[1] = -INFINITY;                             // (packed: no rows of these)
            l[1] = 0.0f;
#pragma unroll
            for (int r = 0; r < RL; ++r) {
                const int rr = cur.r.r0 + g + 8 * r;
                const bool live = g + 8 * r < cur.r.nr;
                const int tok = rr / G;
                p_row[r] = live ? cur.s.p0 + tok : cur.r.hi - 1;
                const TI *src = (const TI *)a.q + (size_t)(cur.s.r0 + tok) * a.q_stride + (size_t)(kh * G + rr - tok * G) * HD;
                sc[r] = a.scale2;
                up[r] = 1.0f;
                if constexpr (!F32I) {
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            qa[ks][r + 2 * x] = live ? *reinterpret_cast<const uint32_t *>(src + 16 * ks + 8 * x + 2 * t) : 0u;
                } else {
                    float mx = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) {
                        // f32 cache: K is read four elements a lane; step 2i + b of lane t is elements
                        // 32i + 8t + 4b.. (conflict-free); otherwise 16ks + 2t, + 1 and 8 further
                        if constexpr (F32C) {
                            const float4 v = live ? *reinterpret_cast<const float4 *>(src + 32 * (ks / 2) + 8 * t + 4 * (ks & 1))
                                                  : make_float4(0.f, 0.f, 0.f, 0.f);
                            f[r][ks][0] = v.x; f[r][ks][1] = v.y; f[r][ks][2] = v.z; f[r][ks][3] = v.w;
                        } else {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const float2 v = live ? *reinterpret_cast<const float2 *>(src + 16 * ks + 8 * x + 2 * t) : make_float2(0.f, 0.f);
                                f[r][ks][2 * x] = v.x;
                                f[r][ks][2 * x + 1] = v.y;
                            }
                        }
                        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(f[r][ks][0]), fabsf(f[r][ks][1])), fmaxf(fabsf(f[r][ks][2]), fabsf(f[r][ks][3]))));
                    }
                    if constexpr (HALF) {                 // the row by a power of two so that its largest is in [2^14, 2^15)
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const int eb = min(max((int)(__float_as_uint(mx) >> 23), 15), 254);
                        up[r] = __uint_as_float((uint32_t)(268 - eb) << 23);
                        sc[r] = fmaxf(a.scale2 * __uint_as_float((uint32_t)(eb - 14) << 23), 0x1p-126f);   // (a zero would make hidden scores NaN)
                    }
                }
                m[r] = -INFINITY;
                l[r] = 0.0f;
            }
            if constexpr (F32I) {                         // warp w writes the steps w, w + 4, ... of all terms
#pragma unroll
                for (int k4 = 0; k4 < KS / 4; ++k4) {
                    uint32_t w[NP][4];
#pragma unroll
                    for (int r = 0; r < RL; ++r)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            uint32_t tm[NQ];
                            float lo = 0.0f, hi = 0.0f;
#pragma unroll
                            for (int y = 0; y < 4; ++y)
                                if (warp == y) {
                                    lo = f[r][4 * k4 + y][2 * x];
                                    hi = f[r][4 * k4 + y][2 * x + 1];
                                }
                            split_pair<HALF, NQ>(lo * up[r], hi * up[r], tm);
                            place_terms<PACK>(w, tm, r + 2 * x);
                        }
#pragma unroll
                    for (int n = 0; n < NP; ++n)
                        s_q[(n * KS + 4 * k4 + warp) * 32 + lane] = make_uint4(w[n][0], w[n][1], w[n][2], w[n][3]);
                }
                named_bar_sync(1, KD_WARPS * 32);
            }
#pragma unroll
            for (int i = 0; i < NT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        }
        const int n_here = (int)min((long)(cur.r.nt - cur.kt), u1 - u);          // this block's tiles of it
        int j0 = (cur.r.lo_t + cur.kt) * KD_TILE + warp * KD_KEYS;
#pragma unroll 1
        for (int left = n_here; left > 0; --left, j0 += KD_TILE) {
            const bool active = j0 < cur.r.hi && j0 + KD_KEYS > cur.r.lo;
            float s[2][4], c[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {            // K, then V
                if (!*abort_flag && !mbar_wait(&full[slot], phase)) {
                    *abort_flag = 1;                          // from here on nothing waits; results are void
                    atomicOr(a.c.status, KV_TIMEOUT);
                }
                const uint32_t at = ring + slot * UNIT + warp * (KD_KEYS * 128);
                if (active && half == 0) {
                    float big[2][2][4] = {}, low[2][4] = {};  // f32 rows: large products in two chains, small ones
#pragma unroll
                    for (int n = 0; n < 2; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.0f;
                    // f32 cache: not unrolled, for a short step's time is in fetching its code
#pragma unroll KU
                    for (int k2 = 0; k2 < KS / 2; ++k2) {     // 32 elements
                        uint32_t q2[NP][2][4];
#pragma unroll
                        for (int q = 0; q < NP; ++q)
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                if constexpr (NQ == 1) {
#pragma unroll
                                    for (int e = 0; e < 4; ++e) q2[q][b][e] = qa[2 * k2 + b][e];
                                } else {
                                    const uint4 v = s_q[(q * KS + 2 * k2 + b) * 32 + lane];
                                    q2[q][b][0] = v.x; q2[q][b][1] = v.y; q2[q][b][2] = v.z; q2[q][b][3] = v.w;
                                }
                            }
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            if constexpr (!F32C) {
                                const int r = 8 * n + (lane & 7), ch = 4 * k2 + (lane >> 3);
                                uint32_t b[4];
                                ldsm4(b, at + ch / 8 * (KD_TILE * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                                if constexpr (NQ == 1) {
                                    mma_acc<HALF>(s[n], q2[0][0], b[0], b[1]);
                                    mma_acc<HALF>(s[n], q2[0][1], b[2], b[3]);
                                } else {
                                    mma_acc<HALF>(big[n][0], q2[0][0], b[0], b[1]);
                                    mma_acc<HALF>(big[n][1], q2[0][1], b[2], b[3]);
#pragma unroll
                                    for (int q = NP - 1; q >= 1; --q) {
                                        mma_acc<HALF>(low[n], q2[q][0], b[0], b[1]);
                                        mma_acc<HALF>(low[n], q2[q][1], b[2], b[3]);
                                    }
                                }
                            } else {
                                const int r = 8 * n + g;
#pragma unroll
                                for (int b = 0; b < 2; ++b) {
                                    const float4 v = lds4(at + k2 * (KD_TILE * 128) + r * 128 + (((2 * t + b) ^ (r & 7)) << 4));
                                    uint32_t b0[NK], b1[NK];
                                    split_pair<HALF, NK>(v.x, v.y, b0);
                                    split_pair<HALF, NK>(v.z, v.w, b1);
                                    mma_acc<HALF>(big[n][b], q2[0][b], b0[0], b1[0]);
                                    if constexpr (PACK) {
                                        mma_acc<HALF>(low[n], q2[0][b], b0[2], b1[2]);
                                        mma_acc<HALF>(low[n], q2[1][b], b0[0], b1[0]);
                                        mma_acc<HALF>(low[n], q2[0][b], b0[1], b1[1]);
                                    } else {
#pragma unroll
                                        for (int d = NK - 1; d >= 1; --d)  // terms of weight 2^-8d
#pragma unroll
                                            for (int k = 0; k <= d; ++k) mma_acc<HALF>(low[n], q2[d - k][b], b0[k], b1[k]);
                                    }
                                }
                            }
                        }
                    }
                    if constexpr (NQ > 1) {
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int e = 0; e < 2 * RL; ++e) {
                                float small = low[n][e];
                                if constexpr (PACK) small += (low[n][e + 2] + big[n][0][e + 2]) + big[n][1][e + 2];
                                s[n][e] = (big[n][0][e] + big[n][1][e]) + small;
                            }
                    }
                    const int span = (cur.r.nr - 1) / G + 1;    // positions between the tile's rows, at most
                    if (j0 + KD_KEYS > cur.r.hi - span || (a.window && j0 < cur.r.lo + span)) {
                        // some row of the tile does not see all 16
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int e = 0; e < 2 * RL; ++e) {
                                const int j = j0 + 8 * n + 2 * t + (e & 1), p = p_row[e >> 1];
                                if (j > p || (a.window && j <= p - a.window)) s[n][e] = -INFINITY;
                            }
                    }
#pragma unroll
                    for (int r = 0; r < RL; ++r) {
                        float mx = fmaxf(fmaxf(s[0][2 * r], s[0][2 * r + 1]), fmaxf(s[1][2 * r], s[1][2 * r + 1]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        const float mn = fmaxf(m[r], kv_top<HALF>(mx * sc[r])), base = mn == -INFINITY ? 0.0f : mn;
                        const float minus = kv_lift<HALF>(14.0f) - base;
                        c[r] = ex2(m[r] - base);
                        m[r] = mn;
                        float add = 0.0f;
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int e = 2 * r; e < 2 * r + 2; ++e) {
                                s[n][e] = ex2(fmaf(s[n][e], sc[r], minus));
                                add += s[n][e];
                            }
                        l[r] = fmaf(l[r], c[r], add);
                    }
                    if constexpr (NQ == 1) {
                        if (__any_sync(0xffffffffu, c[0] != 1.0f || c[1] != 1.0f)) {
#pragma unroll
                            for (int i = 0; i < NT; ++i) {
                                o[i][0] *= c[0]; o[i][1] *= c[0];
                                o[i][2] *= c[1]; o[i][3] *= c[1];
                            }
                        }
                    }
                } else if (active) {
                    uint32_t pa[NP][4];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int r = 0; r < RL; ++r) {
                            uint32_t tm[NQ];
                            split_pair<HALF, NQ>(s[n][2 * r], s[n][2 * r + 1], tm);
                            place_terms<PACK>(pa, tm, r + 2 * n);
                        }
                    // keys 2t, 2t+1, 2t+8, 2t+9 of this lane's fragments that nobody sees
                    bool hide[4];
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const int j = j0 + 2 * t + (y & 1) + 8 * (y >> 1);
                        hide[y] = j >= cur.r.hi || j < cur.r.lo;
                    }
                    const bool any = j0 + KD_KEYS > cur.r.hi || j0 < cur.r.lo;
                    // f32 rows: o = o·c + sum, rounded
                    auto add_to = [&](float (&to)[4], const float (&sum)[4]) {
#pragma unroll
                        for (int e = 0; e < 2 * RL; ++e) to[e] = fmaf(to[e], c[e >> 1], PACK ? sum[e] + sum[e + 2 & 3] : sum[e]);
                    };
                    if constexpr (!F32C) {
                        const uint32_t k0 = (hide[0] ? 0u : 0xffffu) | (hide[1] ? 0u : 0xffff0000u);
                        const uint32_t k1 = (hide[2] ? 0u : 0xffffu) | (hide[3] ? 0u : 0xffff0000u);
                        const int r = lane & 15;
#pragma unroll
                        for (int n2 = 0; n2 < NT / 2; ++n2) {
                            const int ch = 2 * n2 + (lane >> 4);
                            uint32_t b[4];
                            ldsm4t(b, at + ch / 8 * (KD_TILE * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4));
                            if (any) {
                                b[0] &= k0; b[1] &= k1;
                                b[2] &= k0; b[3] &= k1;
                            }
                            if constexpr (NQ == 1) {
                                mma_acc<HALF>(o[2 * n2], pa[0], b[0], b[1]);
                                mma_acc<HALF>(o[2 * n2 + 1], pa[0], b[2], b[3]);
                            } else {
#pragma unroll
                                for (int x = 0; x < 2; ++x) {
                                    float sum[4];
                                    mma_new<HALF>(sum, pa[NP - 1], b[2 * x], b[2 * x + 1]);
#pragma unroll
                                    for (int q = NP - 2; q >= 0; --q) mma_acc<HALF>(sum, pa[q], b[2 * x], b[2 * x + 1]);
                                    add_to(o[2 * n2 + x], sum);
                                }
                            }
                        }
                    } else {
                        // lane (g, t) reads columns 32cb + 4g.. of its four keys: n tile 4cb + x is the
                        // columns 32cb + 4n + x
#pragma unroll
                        for (int cb = 0; cb < HD / 32; ++cb) {
                            float v[4][4];
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                const int r = 2 * t + (y & 1) + 8 * (y >> 1);
                                const float4 w = lds4(at + cb * (KD_TILE * 128) + r * 128 + ((g ^ (r & 7)) << 4));
                                v[y][0] = w.x; v[y][1] = w.y; v[y][2] = w.z; v[y][3] = w.w;
                                if (any && hide[y]) v[y][0] = v[y][1] = v[y][2] = v[y][3] = 0.0f;
                            }
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                uint32_t b0[NK], b1[NK];
                                split_pair<HALF, NK>(v[0][x], v[1][x], b0);
                                split_pair<HALF, NK>(v[2][x], v[3][x], b1);
                                float sum[4];
                                mma_new<HALF>(sum, pa[NP - 1], b0[0], b1[0]);          // smallest products first
                                if constexpr (PACK) {
#pragma unroll
                                    for (int k = NK - 1; k >= 0; --k) mma_acc<HALF>(sum, pa[0], b0[k], b1[k]);
                                } else {
#pragma unroll
                                    for (int d = NK - 1; d >= 0; --d)
#pragma unroll
                                        for (int k = d == NK - 1; k <= d; ++k) mma_acc<HALF>(sum, pa[d - k], b0[k], b1[k]);
                                }
                                add_to(o[4 * cb + x], sum);
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[slot]);
                if (++slot == NU) {
                    slot = 0;
                    phase ^= 1;
                }
            }
        }

        // ---- the item, or this block's part of it, is done. The warps' sums are brought to the
        // common maximum and added so that each warp ends with a quarter of the columns: half the
        // n tiles of every quarter at a time, through shared memory
        constexpr int NQT = NT / 4;                       // n tiles of a quarter
        float *const s_m = s_o + kd_buf<HD>() / 4, *const s_l = s_m + KD_JOIN * KD_ROWS;
#pragma unroll
        for (int r = 0; r < RL; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (t == 0) {
                s_m[warp * KD_ROWS + g + 8 * r] = m[r];
                s_l[warp * KD_ROWS + g + 8 * r] = l[r];
            }
        }
        // the largest maximum of n states in s_m, and the sum of s_l for it
        auto common = [&](int n_states) {
#pragma unroll
            for (int r = 0; r < RL; ++r) {
                m[r] = -INFINITY;
                l[r] = 0.0f;
                for (int k = 0; k < n_states; ++k) m[r] = fmaxf(m[r], s_m[k * KD_ROWS + g + 8 * r]);
                const float base = m[r] == -INFINITY ? 0.0f : m[r];
                for (int k = 0; k < n_states; ++k)
                    l[r] = fmaf(ex2(s_m[k * KD_ROWS + g + 8 * r] - base), s_l[k * KD_ROWS + g + 8 * r], l[r]);
            }
        };
        {
            const float own[2] = {m[0], m[1]};
            named_bar_sync(1, KD_WARPS * 32);             // and q's terms are no longer read
            common(KD_WARPS);
#pragma unroll
            for (int r = 0; r < RL; ++r) {
                const float f = m[r] == -INFINITY ? 0.0f : ex2(own[r] - m[r]);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    o[i][2 * r] *= f;
                    o[i][2 * r + 1] *= f;
                }
            }
        }
        float oq[NQT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int w = 0; w < KD_WARPS; ++w)
                if (w != warp) {
#pragma unroll
                    for (int i = 0; i < NQT / 2; ++i)
#pragma unroll
                        for (int e = 0; e < 2 * RL; ++e)
                            s_o[((w * 3 + (warp < w ? warp : warp - 1)) * (NQT / 2 * 4) + 4 * i + e) * 32 + lane] = o[w * NQT + h * (NQT / 2) + i][e];
                }
            named_bar_sync(1, KD_WARPS * 32);
#pragma unroll
            for (int i = 0; i < NQT / 2; ++i)
#pragma unroll
                for (int e = 0; e < 2 * RL; ++e) {
                    float sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < KD_WARPS; ++w) {
                        float v = 0.0f;
                        if (w != warp) v = s_o[((warp * 3 + (w < warp ? w : w - 1)) * (NQT / 2 * 4) + 4 * i + e) * 32 + lane];
                        else {
#pragma unroll
                            for (int x = 0; x < KD_WARPS; ++x)
                                if (x == warp) v = o[x * NQT + h * (NQT / 2) + i][e];
                        }
                        sum += v;
                    }
                    oq[h * (NQT / 2) + i][e] = sum;
                }
            named_bar_sync(1, KD_WARPS * 32);
        }

        // ---- who else has a part of it: the item's tiles are units [ua, ue), blocks b0..b1
        const long ua = u - cur.kt, ue = ua + cur.r.nt;
        u += n_here;
        const int b0 = cut.owner(ua), b1 = cut.owner(ue - 1);
        bool write = b0 == b1;
        if (!write) {
            const int np = b1 - b0 + 1, p = blk - b0;
            int gs = np;
            if (np > 16)
                for (gs = 4; gs * gs < np;) ++gs;
            const int ng = (np + gs - 1) / gs, gi = p / gs, n_in = min(gs, np - gi * gs);
            auto part = [&](int k) { return a.part + (size_t)(k == 0 ? 2 * b0 + 1 : 2 * (b0 + k)) * kd_slot<HD>(); };
            auto put = [&](float *to) {                   // m, l and o in fragment order, a quarter a warp
                if (warp == 0 && t == 0) {
#pragma unroll
                    for (int r = 0; r < RL; ++r) {
                        to[g + 8 * r] = m[r];
                        to[KD_ROWS + g + 8 * r] = l[r];
                    }
                }
                to += 2 * KD_ROWS + warp * NQT * 128 + lane;
#pragma unroll
                for (int i = 0; i < NQT; ++i)
#pragma unroll
                    for (int e = 0; e < 2 * RL; ++e) __stcg(to + (4 * i + e) * 32, oq[i][e]);
            };
            // parts first, first + step, ... (count of them): joined by the last of their blocks
            auto join = [&](int *counter, int first, int step, int count) -> bool {
                named_bar_sync(1, KD_WARPS * 32);
                if (tid == 0) {
                    const int last = kv_arrive(counter) == count - 1;
                    if (last) *counter = 0;               // ready for the next call
                    s_last = last;
                }
                named_bar_sync(1, KD_WARPS * 32);
                if (!s_last) return false;
#pragma unroll
                for (int x = 0; x < KD_JOIN / 8; ++x) {
                    const int k = tid / KD_ROWS + 8 * x, row = tid % KD_ROWS;
                    if (k < count) {
                        s_m[k * KD_ROWS + row] = __ldcg(part(first + k * step) + row);
                        s_l[k * KD_ROWS + row] = __ldcg(part(first + k * step) + KD_ROWS + row);
                    }
                }
                constexpr int F = 4;                      // parts in flight
#pragma unroll
                for (int i = 0; i < NQT; ++i) oq[i][0] = oq[i][1] = oq[i][2] = oq[i][3] = 0.0f;
                for (int k0 = 0; k0 < count; k0 += F) {
                    float v[F][NQT][2 * RL];
#pragma unroll
                    for (int x = 0; x < F; ++x) {
                        const float *src = part(first + min(k0 + x, count - 1) * step) + 2 * KD_ROWS + warp * NQT * 128 + lane;
#pragma unroll
                        for (int i = 0; i < NQT; ++i)
#pragma unroll
                            for (int e = 0; e < 2 * RL; ++e) v[x][i][e] = e < 2 || cur.r.nr > 8 ? __ldcg(src + (4 * i + e) * 32) : 0.0f;
                    }
                    if (k0 == 0) {
                        named_bar_sync(1, KD_WARPS * 32);
                        common(count);
                    }
#pragma unroll
                    for (int x = 0; x < F; ++x) {
                        if (k0 + x >= count) break;
#pragma unroll
                        for (int r = 0; r < RL; ++r) {
                            const float w = m[r] == -INFINITY ? 0.0f : ex2(s_m[(k0 + x) * KD_ROWS + g + 8 * r] - m[r]);
#pragma unroll
                            for (int i = 0; i < NQT; ++i)
#pragma unroll
                                for (int e = 2 * r; e < 2 * r + 2; ++e) oq[i][e] = fmaf(w, v[x][i][e], oq[i][e]);
                        }
                    }
                }
                return true;
            };
            put(part(p));
            // (a group of one is joined as it stands)
            write = n_in == 1 || join(a.counters + (gi == 0 ? 2 * b0 + 1 : 2 * (b0 + gi * gs)), gi * gs, 1, n_in);
            if (write && ng > 1) {
                if (n_in > 1) put(part(gi * gs));
                write = join(a.counters + 2 * KV_MAX_GRID + b0, 0, gs, ng);
            }
        }
        if (write) {
            const int kh = cur.kh;
#pragma unroll
            for (int r = 0; r < RL; ++r) {
                if (g + 8 * r >= cur.r.nr) continue;
                const int rr = cur.r.r0 + g + 8 * r, tok = rr / G;
                TI *dst = (TI *)a.out + (size_t)(cur.s.r0 + tok) * a.out_stride + (size_t)(kh * G + rr - tok * G) * HD;
                const float inv = l[r] == 0.0f ? 0.0f : 1.0f / l[r];
                if constexpr (!F32C) {
#pragma unroll
                    for (int i = 0; i < NQT; ++i) {
                        const float v[2] = {oq[i][2 * r] * inv, oq[i][2 * r + 1] * inv};
                        TI *to = dst + 8 * (warp * NQT + i) + 2 * t;
                        if constexpr (F32I) *reinterpret_cast<float2 *>(to) = make_float2(v[0], v[1]);
                        else {
                            uint32_t w[1];
                            split_pair<HALF, 1>(v[0], v[1], w);
                            *reinterpret_cast<uint32_t *>(to) = w[0];
                        }
                    }
                } else {                                  // n tile 4cb + x, column n: 32cb + 4n + x
                    const int n0 = warp * NQT;
#pragma unroll
                    for (int i = 0; i < NQT; i += 2)
#pragma unroll
                        for (int e = 0; e < 2; ++e)
                            *reinterpret_cast<float2 *>(dst + 32 * ((n0 + i) / 4) + 8 * t + 4 * e + (n0 + i) % 4) =
                                make_float2(oq[i][2 * r + e] * inv, oq[i + 1][2 * r + e] * inv);
                }
            }
        }
        named_bar_sync(1, KD_WARPS * 32);                 // the joining buffers are free again
        if (u < u1) cur.next_item(a, G);
    }
}

int kv_attend_tc_launch(const AttendArgs &a, const CUtensorMap *maps, int hd, cudaStream_t s);
int kv_attend_tcf_launch(const AttendArgs &a, const CUtensorMap *maps, int hd, cudaStream_t s);
size_t kv_attend_tc_part_bytes(int hd);

// Workspace: counters (of this kernel, then of the chunk kernel's), then the parts. The counters
// lie at fixed places and are zero between calls, so calls of any shape may follow one another.
constexpr size_t KD_COUNTERS = 3 * KV_MAX_GRID, KT_COUNTERS = 6 * KV_MAX_GRID;
constexpr size_t KV_PARTS_AT = (KD_COUNTERS + KT_COUNTERS) * sizeof(int);
static_assert(KV_PARTS_AT % 256 == 0, "parts start at a 256-byte boundary");

size_t kv_attend_ws_bytes(int hd) {
    const size_t slot = (hd == 128 ? kd_slot<128>() : kd_slot<64>()) * sizeof(float);
    const size_t parts = 2 * (size_t)KV_MAX_GRID * slot;
    return KV_PARTS_AT + std::max(parts, kv_attend_tc_part_bytes(hd));
}

template <typename TI, typename TC, int HD, bool PACK>
static int launch_kd(const AttendArgs &a, const CUtensorMap *maps, cudaStream_t s) {
    static std::atomic<bool> set[64];                    // once per device
    int dev = 0;
    CPG_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
        const int rc = allow_max_smem((const void *)k_kv_attend<TI, TC, HD, PACK>);
        if (rc) return rc;
        if (dev < 64) set[dev].store(true, std::memory_order_release);
    }
    const int grid = std::min(KV_MAX_GRID, 2 * sm_count());
    const cudaError_t ce = launch_pdl(k_kv_attend<TI, TC, HD, PACK>, dim3(grid), dim3(KD_THREADS), (size_t)kd_smem<HD>(), s, a,
                                      maps[0], maps[1]);
    return ce == cudaSuccess ? CPG_OK : cuda_fail(ce, "cpg_kv_attend");
}
template <typename TI, typename TC>
static int launch_hd(int hd, bool pack, const AttendArgs &a, const CUtensorMap *maps, cudaStream_t s) {
    if constexpr (std::is_same<TI, float>::value)
        if (pack) return hd == 128 ? launch_kd<TI, TC, 128, true>(a, maps, s) : launch_kd<TI, TC, 64, true>(a, maps, s);
    return hd == 128 ? launch_kd<TI, TC, 128, false>(a, maps, s) : launch_kd<TI, TC, 64, false>(a, maps, s);
}

int kv_attend_launch(const KvView &c, const KvMaps &maps, int hd, const KvRows &b, const void *q, size_t q_stride,
                     void *out, size_t out_stride, int type, int n_heads, float scale, int window, int max_new, void *ws,
                     cudaStream_t s) {
    AttendArgs a{b, c, q, out, q_stride, out_stride, n_heads, scale * 1.4426950408889634f, window, maps.box,
                 (float *)((uint8_t *)ws + KV_PARTS_AT), (int *)ws};
    const CUtensorMap *m = maps.m;
    // Past two row tiles of this file's kernel per sequence and cached head, and four in all, the chunk
    // kernels take over: their 128 or 256 rows share each tile of K and V that is read, but beginning and
    // joining cost them more. Measured (us, few / chunk, 4 cached heads of 128): 64 rows of one sequence
    // over 4096 positions 18 / 36 in bf16, 19 / 34 in f32 over f16, 28 / 36 in f32; 128 rows 22 / 36,
    // 29 / 38, 54 / 39; of 64 sequences over 1000 positions 24 rows 53 / 43, 64 rows 94 / 43 in bf16.
    // Of single rows (up to eight per cached head) f32 ones are packed: 64 rows over f16 56 us instead
    // of 61, one row over 512 f32 positions 11.2 instead of 13.5.
    const int G = n_heads / c.KV;
    const long most = max_new > 0 ? std::min(max_new, b.T) : b.T;
    if (G <= 128 && most * G > 2 * KD_ROWS && (long)b.T * G > 4 * KD_ROWS) {
        a.counters += KD_COUNTERS;
        return type == CPG_T_F32 ? kv_attend_tcf_launch(a, m, hd, s) : kv_attend_tc_launch(a, m, hd, s);
    }
    const bool pack = most * G <= KD_ROWS / 2;
    a.box = std::min(maps.box, KD_TILE);
    if (type == CPG_T_F32)
        return c.type == CPG_T_F32   ? launch_hd<float, float>(hd, pack, a, m, s)
               : c.type == CPG_T_F16 ? launch_hd<float, __half>(hd, pack, a, m, s)
                                     : launch_hd<float, __nv_bfloat16>(hd, pack, a, m, s);
    return type == CPG_T_F16 ? launch_hd<__half, __half>(hd, pack, a, m, s) : launch_hd<__nv_bfloat16, __nv_bfloat16>(hd, pack, a, m, s);
}

}  // namespace cpg
