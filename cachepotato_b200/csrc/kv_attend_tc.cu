// kv_attend_tc.cu — attention of chunks of new rows over the paged cache on the 5th-generation
// tensor cores (the formula and the meaning of the arguments: kv_attend.cu).
//
// 16-bit rows over a cache of their type. Bound by the tensor cores (4 · HD flops per row and
// position) and, nearly as much, by the exponential unit: a 128 x 128 tile of scores takes 1024
// cycles of both q·k and p·v at HD = 128, and 1024 cycles for its 16384 exponentials.
//   work    A sequence's rows are (token, head) pairs per cached head. An item is (sequence, cached
//           head, pair of row tiles): two tiles of 128/G tokens x G heads, M = 128 rows each, that
//           share every K and V tile read from L2. Its units are tiles of 64 positions; the units of
//           all items are cut into equal ranges, one per SM (as in kv_attend.cu: causal items of all
//           lengths, one long one or hundreds of short ones fill the GPU the same way).
//   block   warps 0-3, 4-7  softmax of row tile 0 and 1, one thread per row: S out of TMEM, running
//                           maximum and sum, P (16-bit) back over S; at an item's end O out of TMEM.
//                           O is rescaled in place, and only when a row's maximum has grown by more
//                           than 2^8 since the last time: the scale cancels in O / l, and f32 and the
//                           cache's types hold weights up to 2^8 as well as up to 1.
//           warps 8, 10     producers of q and the K tiles, and of the V tiles: tensor TMA into a ring
//           warps 9, 11     tcgen05.mma of row tile 0 and 1: S = q·K^T (both operands in shared memory),
//                           O += P·V (P from TMEM). One thread for both row tiles was the limit: its
//                           waits for tiles that are there take 100 to 250 cycles each.
//           TMEM: two S of 64 columns for each row tile | O0 O1 of 128; P lies over its S.
//   order   With two S a row tile's next q·k runs while the softmax works on this one, so neither waits
//           for the other unless it is the slower (one S of 128 columns, q·k behind p·v: 3900 cycles
//           for two row tiles and 128 positions, of which the tensor core worked half). The tensor core
//           runs what one thread issues in order, so q·k may overwrite P of the tile before last.
//   join    Parts of an item that several blocks share, as in kv_attend.cu.
//   measured  4096 new bf16 rows of 32 heads over 12288 positions and themselves (962 GFLOP): 865 us while
//           the GPU is cool, 985 us (980 TFLOP/s) once it is held at its power limit; the tensor pipe and
//           the exponential unit are each at work in half of the active cycles, so half are lost at any
//           clock: two softmax warps a scheduler, each with its steps in order. 47 single rows and a chunk
//           of 2001 over 500-8000 positions (285 GFLOP, 478 MB): 376 us, 425 at the power limit; chunks
//           with a window of 1000, 14 heads of 64 in f16 (14.6 GFLOP): 50 us.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "kv_attend_tc.cuh"

namespace cpg {

constexpr int KT_TILE = 64, KT_FIXED = 4;                 // positions of an MMA tile; units an item's begin and end are worth
template <int HD> constexpr int kt_unit() { return KT_TILE * HD * 2; }
template <int HD> constexpr int kt_units() { return HD == 128 ? 10 : 16; }
template <int HD> constexpr int kt_smem() { return 1024 + 2 * KT_ROWS * HD * 2 + kt_units<HD>() * kt_unit<HD>(); }

// Row tile x of an item: tokens [t0, t1) of the sequence and the positions its rows see between them.
struct KtRows {
    int t0, t1, lo, hi;
    __device__ __forceinline__ KtRows(const AttendArgs &a, const KtCursor<KT_TILE, KT_FIXED> &c, int Q, int x) {
        t0 = c.pair * Q + x * (Q / 2);
        t1 = min(c.s.len, t0 + Q / 2);
        lo = c.lo_of(a, t0);
        hi = t1 > t0 ? c.s.p0 + t1 : 0;
    }
    __device__ __forceinline__ bool sees(int j0) const { return j0 < hi && j0 + KT_TILE > lo; }
};

template <bool HALF, int HD>
__global__ void __launch_bounds__(KT_THREADS, 1) k_kv_attend_tc(const __grid_constant__ AttendArgs a,
                                                               const __grid_constant__ CUtensorMap tm_q,
                                                               const __grid_constant__ CUtensorMap tm_k,
                                                               const __grid_constant__ CUtensorMap tm_v) {
    constexpr int PARTS = HD / 64;                        // 128-byte columns of a row
    constexpr int COL = KT_TILE * 128, QCOL = KT_ROWS * 128;   // bytes of one in a K or V tile, in a row tile
    constexpr int UNIT = kt_unit<HD>(), NU = kt_units<HD>(), QT = KT_ROWS * HD * 2;
    constexpr uint32_t FMT = HALF ? 0u : UMMA_BF16;
    constexpr uint32_t ID_QK = umma_idesc_f16(128, KT_TILE) | FMT, ID_PV = umma_idesc_f16(128, HD) | FMT | UMMA_B_MN;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t *const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t full[NU], empty[NU], q_full, q_empty, fixed[NU], s_full[2][2], p_full[2][2],
        o_done[2][2], drain[2];
    __shared__ KtShared<KT_TILE, KT_FIXED> sh;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_last[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.H / a.c.KV, TT = KT_ROWS / G, Q = 2 * TT;             // tokens of a row tile, of a pair
    if (tid == 0) {
        for (int i = 0; i < NU; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 2);
            mbar_init(&fixed[i], 1);
        }
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 2);
        for (int x = 0; x < 2; ++x) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(&s_full[x][b], 1);
                mbar_init(&p_full[x][b], 4);
                mbar_init(&o_done[x][b], 1);
            }
        }
        mbar_init(&drain[0], 1);
        mbar_init(&drain[1], 1);
        fence_mbar_init();
        s_abort = 0;
        prefetch_map(&tm_q);
        prefetch_map(&tm_k);
        prefetch_map(&tm_v);
    }
    pdl_wait();
    pdl_launch_dependents();

    long u0, u1;                                          // this block's range of units
    if (!kt_begin<KT_TILE, KT_FIXED>(a, Q, sh, u0, u1)) return;
    if (warp == KT_MMA) {                                 // all of TMEM
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    volatile int *const abort_flag = &s_abort;
    int *const status = a.c.status;
    const uint32_t sq = smem_u32(smem), ring = sq + 2 * QT;
    KtCursor<KT_TILE, KT_FIXED> cur = sh.cur;
    // skips an item's fixed share: false if nothing of the item itself is this block's
    auto begin = [&](long &u) {
        if (cur.kt < 0) {
            u -= cur.kt;
            cur.kt = 0;
        }
        return u < u1;
    };

    if (warp >= 8) {
        if (warp == KT_LOAD_K || warp == KT_LOAD_V) {
            // ---------------- producers: K tiles (and q) in the ring's even slots, V tiles in the odd
            // ones. Lane b loads box b of a tile: issuing small boxes (16 positions: 2 KB) takes a warp
            // some 50 cycles each, so one warp for both was the limit.
            const bool is_v = warp == KT_LOAD_V;
            const CUtensorMap *const map = is_v ? &tm_v : &tm_k;
            const int boxes = KT_TILE / a.box * PARTS;
            int slot = is_v, turn = 0, items = 0;
            bool ok = true;
            for (long u = u0; u < u1 && ok;) {
                if (!begin(u)) break;
                const KtRows r0(a, cur, Q, 0), r1(a, cur, Q, 1);
                if (!is_v) {
                    ok = !items || kt_wait_warp(&q_empty, (uint32_t)(items - 1) & 1u, abort_flag, status);
                    if (!ok) break;
                    const bool two = r1.t1 > r1.t0;
                    if (lane == 0) mbar_arrive_expect_tx(&q_full, (two ? 2u : 1u) * (uint32_t)(TT * G * 128 * PARTS));
                    __syncwarp();
                    if (lane < 2 * PARTS && (two || lane < PARTS)) {
                        const int x = lane / PARTS, part = lane % PARTS;
                        tma_load_3d(sq + x * QT + part * QCOL, &tm_q, part * 64, cur.kh * G, cur.s.r0 + (x ? r1.t0 : r0.t0), &q_full);
                    }
                    ++items;
                }
                const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u);
                const int lo = r0.lo;
                // page and place of this lane's box of tile i; the next tile's is asked for ahead
                auto find = [&](int i, int &page, int &place) {
                    const int j = (cur.lo_t + cur.kt + i) * KT_TILE + lane / PARTS * a.box;
                    place = -1;                           // nothing of it is seen
                    if (lane < boxes && i < n_here && j < cur.hi && j + a.box > lo) {
                        const int pg = j / a.c.P;
                        page = a.b.pages[(size_t)cur.seq * a.b.table_stride + pg];
                        place = j - pg * a.c.P;
                    }
                };
                int next_page = 0, next_place;
                find(0, next_page, next_place);
                for (int i = 0; i < n_here; ++i) {
                    const bool inside = next_place >= 0 && next_page >= 0 && next_page < a.c.n_pages;
                    if (next_place >= 0 && !inside) atomicOr(status, KV_BAD_PAGE);
                    const int page = inside ? next_page : a.c.n_pages, place = max(next_place, 0);   // outside the pool: zeros
                    find(i + 1, next_page, next_place);
                    ok = !turn || kt_wait_warp(&empty[slot], (uint32_t)(turn - 1) & 1u, abort_flag, status);
                    if (!ok) break;
                    if (lane == 0) mbar_arrive_expect_tx(&full[slot], UNIT);
                    __syncwarp();
                    if (lane < boxes)
                        tma_load_4d(ring + slot * UNIT + lane % PARTS * COL + lane / PARTS * a.box * 128, map, lane % PARTS * 64,
                                    place, cur.kh, page, &full[slot]);
                    // places of a V tile that no row of the item sees, in a box some row sees
                    const int j0 = (cur.lo_t + cur.kt + i) * KT_TILE;
                    if (is_v && kt_fix(a, KT_TILE, lo, cur.hi, j0)) {
                        ok = kt_wait_warp(&full[slot], (uint32_t)turn & 1u, abort_flag, status);
                        if (!ok) break;
                        kt_clear<KT_TILE, PARTS>(a, smem + 2 * QT + slot * UNIT, lo, cur.hi, j0, lane);
                        if (lane == 0) mbar_arrive(&fixed[slot]);
                    }
                    slot += 2;
                    if (slot >= NU) {
                        slot -= NU;
                        ++turn;
                    }
                }
                if (!ok) break;
                u += n_here;
                if (u < u1) cur.next_item(a, Q);
            }
            if (!ok) {                                    // copies in flight land before the block may end
                for (int i = is_v; i < NU; i += 2) {
                    const int fills = turn + (i < slot);
                    if (fills) mbar_wait(&full[i], (uint32_t)(fills - 1) & 1u);
                }
                if (items) mbar_wait(&q_full, (uint32_t)(items - 1) & 1u);
            }
        } else {
            // ---------------- tensor core, row tile x: one elected lane waits and issues
            const int x = warp == KT_MMA ? 0 : 1;
            if (elect_one()) {
                int ks = 0, vs = 1;                       // ring slots of the next K and V
                uint32_t kp = 0, vp = 0, pp = 0, qp = 0, fp = 0;           // parities; pp, fp: a bit per P, per slot
                uint32_t qb = 0, pb = 0;                  // the S of the next q·k, the P of the next p·v
                auto step2 = [&](int &s, uint32_t &ph) {
                    s += 2;
                    if (s >= NU) {
                        s -= NU;
                        ph ^= 1;
                    }
                };
                auto wait = [&](uint64_t *bar, uint32_t parity) { return kt_wait(bar, parity, abort_flag, status); };
                const uint64_t dq = umma_desc_sw128(sq + x * QT);
                const uint32_t tS = tmem + x * 128, tO = tmem + 256 + x * 128;
                // S = q · K^T from the next K (if the row tile sees it), which is then let go
                auto qk = [&](bool sees, bool last) {
                    if (!wait(&full[ks], kp)) return false;
                    tc_fence_after();
                    if (sees) {
                        const uint64_t dk = umma_desc_sw128(ring + ks * UNIT);
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k)
                            umma_f16(tS + qb * KT_TILE, dq + ((k / 4 * QCOL + k % 4 * 32) >> 4), dk + ((k / 4 * COL + k % 4 * 32) >> 4),
                                     ID_QK, k ? 1u : 0u);
                        umma_commit(&s_full[x][qb]);
                        qb ^= 1;
                    }
                    umma_commit(&empty[ks]);
                    if (last) umma_commit(&q_empty);
                    step2(ks, kp);
                    return true;
                };
                bool ok = true;
                for (long u = u0; u < u1 && ok;) {
                    if (!begin(u)) break;
                    const KtRows rt(a, cur, Q, x);
                    const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u);
                    const int first = (cur.lo_t + cur.kt) * KT_TILE, lo = cur.lo_of(a, cur.pair * Q);
                    if (!wait(&q_full, qp)) break;
                    qp ^= 1;
                    bool begun = false;
                    ok = qk(rt.sees(first), n_here == 1);
                    for (int i = 0; i < n_here && ok; ++i) {
                        const int j0 = first + i * KT_TILE;
                        if (i + 1 < n_here) ok = qk(rt.sees(j0 + KT_TILE), i + 2 == n_here);
                        ok = ok && wait(&full[vs], vp);
                        if (ok && kt_fix(a, KT_TILE, lo, cur.hi, j0)) {
                            ok = wait(&fixed[vs], fp >> vs & 1u);
                            fp ^= 1u << vs;
                        }
                        if (ok && rt.sees(j0)) {          // O += P · V
                            ok = wait(&p_full[x][pb], pp >> pb & 1u);
                            if (!ok) break;
                            pp ^= 1u << pb;
                            tc_fence_after();
                            const uint64_t dv = umma_desc_sw128_mn(ring + vs * UNIT, COL);
#pragma unroll
                            for (int k = 0; k < KT_TILE / 16; ++k)
                                umma_f16_ts(tO, tS + pb * KT_TILE + k * 8, dv + (k * 2048 >> 4), ID_PV, begun || k ? 1u : 0u);
                            umma_commit(&o_done[x][pb]);
                            pb ^= 1;
                            begun = true;
                        }
                        if (!ok) break;
                        umma_commit(&empty[vs]);
                        step2(vs, vp);
                    }
                    u += n_here;
                    if (u < u1) cur.next_item(a, Q);
                }
                // every MMA issued has finished before the block ends
                umma_commit(&drain[x]);
                mbar_wait(&drain[x], 0);
            }
            __syncwarp();
        }
    } else {
        // ---------------- softmax and output of row tile x, one thread per row
        const int x = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lanes + x * 128, tO = tmem + lanes + 256 + x * 128;
        const int tok = row / G, g = row - tok * G;
        uint32_t given = 0;                               // P handed over so far: P number n lies over S n % 2
        // P number n has been multiplied. A barrier for each of the two P, and each is waited for before
        // its next P is written: a parity tells two phases apart, and the softmax may be two P ahead of
        // the products when V tiles come late (one barrier let it read O too early then).
        auto done = [&](uint32_t n) { kt_wait(&o_done[x][n & 1], n >> 1 & 1u, abort_flag, status); };
        for (long u = u0; u < u1;) {
            if (!begin(u)) break;
            const KtRows rt(a, cur, Q, x);
            const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u);
            const int first = (cur.lo_t + cur.kt) * KT_TILE;
            const bool live = tok < rt.t1 - rt.t0 && row < TT * G;
            const int p0 = cur.s.p0 + rt.t0, p = live ? p0 + tok : rt.hi - 1;             // the tile's first, this row's position
            float m = -INFINITY, l = 0.0f;
            bool begun = false;
            for (int i = 0; i < n_here; ++i) {
                const int j0 = first + i * KT_TILE;
                if (!rt.sees(j0)) continue;
                const uint32_t buf = given & 1, tP = tS + buf * KT_TILE;
                kt_wait(&s_full[x][buf], given >> 1 & 1u, abort_flag, status);
                if (given >= 2) done(given - 2);          // has come with this S; see above
                tc_fence_after();
                uint32_t s[KT_TILE];
                tmem_ld32_nowait(tP, s);
                tmem_ld32_nowait(tP + 32, s + 32);
                tmem_wait_ld();
                settle32(s);
                settle32(s + 32);
                if (j0 + KT_TILE > p0 + 1 || (a.window && j0 < rt.hi - a.window)) {
                    // some row of the tile does not see all 64
                    const int top = min(p - j0, 63), bottom = a.window ? max(p - a.window - j0, -1) : -1;
                    const uint64_t seen = top < 0 ? 0ull : (~0ull >> (63 - top)) & (bottom >= 63 ? 0ull : ~0ull << (bottom + 1));
#pragma unroll
                    for (int e = 0; e < KT_TILE; ++e)
                        if (!(seen >> e & 1)) s[e] = 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < KT_TILE; e += 2)
                    mx[e / 2 & 3] = fmaxf(mx[e / 2 & 3], fmaxf(__uint_as_float(s[e]), __uint_as_float(s[e + 1])));
                const float top = kv_top<HALF>(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2);
                const bool grow = top > m + 8.0f;
                if (__any_sync(0xffffffffu, grow)) {      // O and l to the scale of a larger maximum
                    const float f = grow ? ex2(m - top) : 1.0f;
                    if (grow) {
                        m = top;
                        l *= f;
                    }
                    if (begun) {                          // once its last product has finished
                        done(given - 1);
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tmem_ld32_nowait(tO + c, o);
                            tmem_wait_ld();
                            settle32(o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st32(tO + c, o);
                        }
                    }
                }
                begun = true;
                const float off = kv_lift<HALF>(7.0f) - (m == -INFINITY ? 0.0f : m);
                const f32x2 minus = pack2(off, off), scale22 = pack2(a.scale2, a.scale2);
                f32x2 add[2] = {0, 0};
#pragma unroll
                for (int e = 0; e < KT_TILE / 2; ++e) {   // the weights, packed into the registers behind
                    float e0, e1;
                    unpack2(fma2(pack2(__uint_as_float(s[2 * e]), __uint_as_float(s[2 * e + 1])), scale22, minus), e0, e1);
                    e0 = ex2(e0);
                    e1 = ex2(e1);
                    add[e & 1] = add2(add[e & 1], pack2(e0, e1));
                    uint32_t w[1];
                    split_pair<HALF, 1>(e0, e1, w);
                    s[e] = w[0];
                }
                tmem_st32(tP, s);
                float a0, a1;
                unpack2(add2(add[0], add[1]), a0, a1);
                l += a0 + a1;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[x][buf]);
                ++given;
            }
            if (begun) {
                done(given - 1);
                tc_fence_after();
            }

            // ---- the item, or this block's part of it, is done: its tiles are units [ua, ue), blocks b0..b1
            const long ua = u - cur.kt, ue = ua + cur.nt;
            u += n_here;
            const int b0 = sh.cut.owner(ua), b1 = sh.cut.owner(ue - 1);
            const size_t cell = (size_t)(cur.s.r0 + rt.t0 + tok);
            uint16_t *const dst = (uint16_t *)a.out + cell * a.out_stride + (size_t)(cur.kh * G + g) * HD;
            // 16 columns from c of the row, times f, to out
            auto write16 = [&](int c, const float *v, float f) {
                if (!live) return;
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    uint32_t t1[1];
                    split_pair<HALF, 1>(v[2 * e] * f, v[2 * e + 1] * f, t1);
                    w[e] = t1[0];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    *reinterpret_cast<uint4 *>(dst + c + 8 * e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
            };
            auto load16 = [&](int c, float *v) {          // O's columns; nothing has been added to it: zeros
                uint32_t o[16];
                if (begun) {
                    tmem_ld16_nowait(tO + c, o);
                    tmem_wait_ld();
                    settle16(o);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) v[e] = begun ? __uint_as_float(o[e]) : 0.0f;
            };
            if (rt.t1 <= rt.t0) {
                // the second tile of a short pair
            } else if (b0 == b1) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 2
                for (int c = 0; c < HD; c += 16) {
                    float v[16];
                    load16(c, v);
                    write16(c, v, inv);
                }
            } else {
                const int np = b1 - b0 + 1, pi = (int)blockIdx.x - b0;
                int gs = np;
                if (np > 4)
                    for (gs = 2; gs * gs < np;) ++gs;
                const int ng = (np + gs - 1) / gs, gi = pi / gs, n_in = min(gs, np - gi * gs);
                const KtParts<HD> parts{a.part, x, row, b0, live};
                float *to = parts.at(pi);
                __stcg(to + row, m);
                __stcg(to + KT_ROWS + row, l);
#pragma unroll 2
                for (int c = 0; c < HD; c += 16) {
                    float v[16];
                    load16(c, v);
                    parts.put16(to, c, v);
                }
                if ((n_in == 1 || parts.join(a.counters + parts.slot_of(gi * gs) * 2 + x, &s_last[x], gi * gs, 1, n_in, ng == 1, write16)) && ng > 1)
                    parts.join(a.counters + 4 * KV_MAX_GRID + b0 * 2 + x, &s_last[x], 0, gs, ng, true, write16);
            }
            tc_fence_before();
            if (u < u1) cur.next_item(a, Q);
        }
    }
    // all roles leave here (a timeout anywhere raised the abort flag, every wait is bounded)
    tc_fence_before();
    __syncthreads();
    if (warp == KT_MMA) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

size_t kv_attend_tc_part_bytes(int hd) {
    return 4 * (size_t)sm_count() * (hd == 128 ? kt_part<128>() : kt_part<64>()) * sizeof(float);
}

int tensor_map(CUtensorMap *map, int type, int rank, const void *base, const uint64_t *dims, const uint64_t *strides,
               const uint32_t *box);

template <bool HALF, int HD>
static int launch_kt(const AttendArgs &a, const CUtensorMap &q, const CUtensorMap *maps, cudaStream_t s) {
    static std::atomic<bool> set[64];                    // once per device
    int dev = 0;
    CPG_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
        const int rc = allow_max_smem((const void *)k_kv_attend_tc<HALF, HD>);
        if (rc) return rc;
        if (dev < 64) set[dev].store(true, std::memory_order_release);
    }
    const int grid = std::min(KV_MAX_GRID, sm_count());
    const cudaError_t ce = launch_pdl(k_kv_attend_tc<HALF, HD>, dim3(grid), dim3(KT_THREADS), (size_t)kt_smem<HD>(), s, a, q,
                                      maps[0], maps[1]);
    return ce == cudaSuccess ? CPG_OK : cuda_fail(ce, "cpg_kv_attend");
}

int kv_attend_tc_launch(const AttendArgs &a, const CUtensorMap *maps, int hd, cudaStream_t s) {
    const int G = a.H / a.c.KV;
    const uint64_t dims[3] = {(uint64_t)hd, (uint64_t)a.H, (uint64_t)a.b.T};
    const uint64_t strides[2] = {(uint64_t)hd * 2, (uint64_t)(a.b.T > 1 ? a.q_stride : (size_t)a.H * hd) * 2};
    const uint32_t box[3] = {64, (uint32_t)G, (uint32_t)(KT_ROWS / G)};
    CUtensorMap q;
    const int rc = tensor_map(&q, a.c.type, 3, a.q, dims, strides, box);
    if (rc) return rc;
    if (a.c.type == CPG_T_F16) return hd == 128 ? launch_kt<true, 128>(a, q, maps, s) : launch_kt<true, 64>(a, q, maps, s);
    return hd == 128 ? launch_kt<false, 128>(a, q, maps, s) : launch_kt<false, 64>(a, q, maps, s);
}

}  // namespace cpg
