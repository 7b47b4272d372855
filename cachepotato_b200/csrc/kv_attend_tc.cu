// kv_attend_tc.cu — attention of chunks of new rows over the paged cache on the 5th-generation
// tensor cores (the formula and the meaning of the arguments: kv_attend.cu).
//
// 16-bit rows over a cache of their type. Bound by the tensor cores (4 · HD flops per row and
// position) and, nearly as much, by the exponential unit: a 128 x 128 tile of scores takes 1024
// cycles of both q·k and p·v at HD = 128, and 1024 cycles for its 16384 exponentials.
//   work    A sequence's rows are (token, head) pairs per cached head. An item is (sequence, cached
//           head, pair of row tiles): two tiles of 128/G tokens x G heads, M = 128 rows each, that
//           share every K and V tile read from L2. Its units are tiles of 128 positions; the units of
//           all items are cut into equal ranges, one per SM (as in kv_attend.cu: causal items of all
//           lengths, one long one or hundreds of short ones fill the GPU the same way).
//   block   warps 0-3, 4-7  softmax of row tile 0 and 1, one thread per row: S out of TMEM, running
//                           maximum and sum, P (16-bit) back over S; at an item's end O out of TMEM.
//                           O is rescaled in place, and only when a row's maximum has grown by more
//                           than 2^8 since the last time: the scale cancels in O / l, and f32 and the
//                           cache's types hold weights up to 2^8 as well as up to 1. So a tile's
//                           weights are taken with the maximum at hand, in one pass over S, and only
//                           if it proves too small are they taken again. (An item's first tile is
//                           gone over for the maximum first.)
//           warp 8          producer: q tiles and the ring of K and V tiles, tensor TMA
//           warp 9          tcgen05.mma: S = q·K^T (both operands in shared memory), O += P·V (P from
//                           TMEM). While one row tile is in its softmax the other's products run.
//           warp 10         clears the places of an item's last V tile that lie in its last page behind
//                           the last position (they may hold anything, and 0 · NaN is NaN)
//           TMEM: S0 S1 | O0 O1, 128 columns each; P lies over its S.
//   order   The tensor core runs what one thread issues in order, so q·k of the next tile may be
//           issued behind the p·v that still reads P from the same columns, and a finished q·k says
//           that the p·v before it has finished: between then and its own P the softmax owns O.
//   join    Parts of an item that several blocks share, as in kv_attend.cu.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "kv_attend_tc.cuh"

namespace cpg {

constexpr int KT_TILE = 128;                              // positions of an MMA tile
template <int HD> constexpr int kt_unit() { return KT_TILE * HD * 2; }
template <int HD> constexpr int kt_units() { return HD == 128 ? 5 : 8; }
template <int HD> constexpr int kt_smem() { return 1024 + 2 * KT_ROWS * HD * 2 + kt_units<HD>() * kt_unit<HD>(); }

// Row tile x of an item: tokens [t0, t1) of the sequence and the positions its rows see between them.
struct KtRows {
    int t0, t1, lo, hi;
    __device__ __forceinline__ KtRows(const AttendArgs &a, const KtCursor<KT_TILE> &c, int Q, int x) {
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
    constexpr int PARTS = HD / 64, COL = KT_TILE * 128;   // 128-byte columns of a tile, bytes of one
    constexpr int UNIT = kt_unit<HD>(), NU = kt_units<HD>(), QT = KT_ROWS * HD * 2;
    constexpr uint32_t FMT = HALF ? 0u : UMMA_BF16;
    constexpr uint32_t ID_QK = umma_idesc_f16(128, KT_TILE) | FMT, ID_PV = umma_idesc_f16(128, HD) | FMT | UMMA_B_MN;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t *const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t full[NU], empty[NU], q_full, q_empty, asked[NU], fixed[NU], s_full[2], p_full[2], o_full[2], drain;
    __shared__ KtShared<KT_TILE> sh;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_last[2], s_ask[NU][3];     // a V tile to clear: ring slot, its fill's parity, first place
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.H / a.c.KV, TT = KT_ROWS / G, Q = 2 * TT;             // tokens of a row tile, of a pair
    if (tid == 0) {
        for (int i = 0; i < NU; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
            mbar_init(&asked[i], 1);
            mbar_init(&fixed[i], 1);
        }
        mbar_init(&q_full, 1);
        mbar_init(&q_empty, 1);
        for (int x = 0; x < 2; ++x) {
            mbar_init(&s_full[x], 1);
            mbar_init(&p_full[x], 4);
            mbar_init(&o_full[x], 1);
        }
        mbar_init(&drain, 1);
        fence_mbar_init();
        s_abort = 0;
        prefetch_map(&tm_q);
        prefetch_map(&tm_k);
        prefetch_map(&tm_v);
    }
    pdl_wait();
    pdl_launch_dependents();

    long u0, u1;                                          // this block's range of units
    if (!kt_begin<KT_TILE>(a, Q, sh, u0, u1)) return;
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
    KtCursor<KT_TILE> cur = sh.cur;
    // skips an item's fixed share: false if nothing of the item itself is this block's
    auto begin = [&](long &u) {
        if (cur.kt < 0) {
            u -= cur.kt;
            cur.kt = 0;
        }
        return u < u1;
    };

    if (warp >= 8) {
        if (warp == KT_PRODUCER) {
            // ---------------- producer: lane b loads box b of every unit
            const int groups = KT_TILE / a.box, boxes = groups * PARTS;
            int slot = 0, turn = 0, items = 0, asks = 0;
            bool ok = true;
            for (long u = u0; u < u1 && ok;) {
                if (!begin(u)) break;
                if (items && !kt_wait_warp(&q_empty, (uint32_t)(items - 1) & 1u, abort_flag, status)) break;
                const KtRows r0(a, cur, Q, 0), r1(a, cur, Q, 1);
                const bool two = r1.t1 > r1.t0;
                if (lane == 0) mbar_arrive_expect_tx(&q_full, (two ? 2u : 1u) * (uint32_t)(TT * G * 128 * PARTS));
                __syncwarp();
                if (lane < 2 * PARTS && (two || lane < PARTS)) {
                    const int x = lane / PARTS, part = lane % PARTS;
                    tma_load_3d(sq + x * QT + part * COL, &tm_q, part * 64, cur.kh * G, cur.s.r0 + (x ? r1.t0 : r0.t0), &q_full);
                }
                ++items;
                const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u);
                const int lo = r0.lo;
                for (int i = 0; i < n_here; ++i) {
                    const int j0 = (cur.lo_t + cur.kt + i) * KT_TILE;
                    int page = a.c.n_pages, place = 0;    // outside the pool: zeros
                    const int j = j0 + lane / PARTS * a.box;
                    if (lane < boxes && j < cur.hi && j + a.box > lo) {
                        const int pg = j / a.c.P;
                        const int id = a.b.pages[(size_t)cur.seq * a.b.table_stride + pg];
                        if (id >= 0 && id < a.c.n_pages) page = id;
                        else atomicOr(status, KV_BAD_PAGE);
                        place = j - pg * a.c.P;
                    }
#pragma unroll
                    for (int half = 0; half < 2; ++half) {                // K, then V
                        ok = !turn || kt_wait_warp(&empty[slot], (uint32_t)(turn - 1) & 1u, abort_flag, status);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&full[slot], UNIT);
                        __syncwarp();
                        if (lane < boxes)
                            tma_load_4d(ring + slot * UNIT + lane % PARTS * COL + lane / PARTS * a.box * 128, half ? &tm_v : &tm_k,
                                        lane % PARTS * 64, place, cur.kh, page, &full[slot]);
                        if (half && kt_fix(a, KT_TILE, cur.hi - j0)) {
                            if (lane == 0) {
                                s_ask[asks % NU][0] = slot;
                                s_ask[asks % NU][1] = turn & 1;
                                s_ask[asks % NU][2] = cur.hi - j0;
                                mbar_arrive(&asked[asks % NU]);
                            }
                            ++asks;
                        }
                        if (++slot == NU) {
                            slot = 0;
                            ++turn;
                        }
                    }
                    if (!ok) break;
                }
                u += n_here;
                if (u < u1) cur.next_item(a, Q);
            }
            if (*abort_flag) {                            // copies in flight land before the block may end
                for (int i = 0; i < NU; ++i) {
                    const int fills = turn + (i < slot);
                    if (fills) mbar_wait(&full[i], (uint32_t)(fills - 1) & 1u);
                }
                if (items) mbar_wait(&q_full, (uint32_t)(items - 1) & 1u);
            }
        } else if (warp == KT_MMA) {
            // ---------------- tensor core: one elected lane waits and issues
            if (elect_one()) {
                int ks = 0, vs = 1;                       // ring slots of the next K and V
                uint32_t kp = 0, vp = 0, pp0 = 0, pp1 = 0, qp = 0, fp = 0;               // fp: a bit per slot
                auto step2 = [&](int &s, uint32_t &ph) {
                    s += 2;
                    if (s >= NU) {
                        s -= NU;
                        ph ^= 1;
                    }
                };
                auto wait = [&](uint64_t *bar, uint32_t parity) { return kt_wait(bar, parity, abort_flag, status); };
                bool ok = true;
                for (long u = u0; u < u1 && ok;) {
                    if (!begin(u)) break;
                    const KtRows r0(a, cur, Q, 0), r1(a, cur, Q, 1);
                    const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u);
                    const int first = (cur.lo_t + cur.kt) * KT_TILE;
                    if (!wait(&q_full, qp)) break;
                    qp ^= 1;
                    bool begun0 = false, begun1 = false;
                    // S_x = q_x · K^T from ring slot ks, O_x += P_x · V from slot vs; x = 0, 1
                    auto qk = [&](int x) {
                        const uint64_t dq = umma_desc_sw128(sq + x * QT), dk = umma_desc_sw128(ring + ks * UNIT);
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k) {
                            const uint32_t at = (k / 4 * COL + k % 4 * 32) >> 4;       // of the descriptor's start
                            umma_f16(tmem + x * 128, dq + at, dk + at, ID_QK, k ? 1u : 0u);
                        }
                        umma_commit(&s_full[x]);
                    };
                    auto pv = [&](int x, bool begun) {
                        const uint64_t dv = umma_desc_sw128_mn(ring + vs * UNIT, COL);
#pragma unroll
                        for (int k = 0; k < KT_TILE / 16; ++k)
                            umma_f16_ts(tmem + 256 + x * 128, tmem + x * 128 + k * 8, dv + (k * 2048 >> 4), ID_PV, begun || k ? 1u : 0u);
                    };
                    if (!wait(&full[ks], kp)) break;
                    tc_fence_after();
                    bool s0 = r0.sees(first), s1 = r1.sees(first);         // whether the row tiles see this unit
                    if (s0) qk(0);
                    if (s1) qk(1);
                    umma_commit(&empty[ks]);
                    if (n_here == 1) umma_commit(&q_empty);
                    step2(ks, kp);
                    for (int i = 0; i < n_here; ++i) {
                        const int j0 = first + i * KT_TILE;
                        const bool more = i + 1 < n_here;
                        const bool n0 = more && r0.sees(j0 + KT_TILE), n1 = more && r1.sees(j0 + KT_TILE);
                        ok = wait(&full[vs], vp) && (!more || wait(&full[ks], kp));
                        if (ok && kt_fix(a, KT_TILE, cur.hi - j0)) {
                            ok = wait(&fixed[vs], fp >> vs & 1u);
                            fp ^= 1u << vs;
                        }
                        if (!ok) break;
                        if (s0) {
                            ok = wait(&p_full[0], pp0);
                            if (!ok) break;
                            pp0 ^= 1;
                            tc_fence_after();
                            pv(0, begun0);
                            begun0 = true;
                            if (!n0) umma_commit(&o_full[0]);
                        }
                        if (n0) qk(0);
                        if (s1) {
                            ok = wait(&p_full[1], pp1);
                            if (!ok) break;
                            pp1 ^= 1;
                            tc_fence_after();
                            pv(1, begun1);
                            begun1 = true;
                            if (!n1) umma_commit(&o_full[1]);
                        }
                        umma_commit(&empty[vs]);
                        if (n1) qk(1);
                        if (more) umma_commit(&empty[ks]);
                        if (i + 2 == n_here) umma_commit(&q_empty);
                        step2(vs, vp);
                        if (more) step2(ks, kp);
                        s0 = n0;
                        s1 = n1;
                    }
                    u += n_here;
                    if (u < u1) cur.next_item(a, Q);
                }
                // every MMA issued has finished before the block ends
                umma_commit(&drain);
                mbar_wait(&drain, 0);
            }
            __syncwarp();
        } else if (warp == KT_FIXER) {
            // the V tiles the producer asks for, in its order. A slot asked for is not filled again before
            // it is cleared, so its barriers are never more than one phase from what is waited for.
            int asks = 0;
            for (long u = u0; u < u1;) {
                if (!begin(u)) break;
                const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u);
                if (kt_fix(a, KT_TILE, cur.hi - (cur.lo_t + cur.kt + n_here - 1) * KT_TILE)) {
                    const int at = asks % NU;
                    if (!kt_wait_warp(&asked[at], (uint32_t)(asks / NU) & 1u, abort_flag, status)) break;
                    const int slot = s_ask[at][0], end = s_ask[at][2];
                    if (!kt_wait_warp(&full[slot], (uint32_t)s_ask[at][1], abort_flag, status)) break;
                    const int rows_z = (end + a.box - 1) / a.box * a.box - end;
                    for (int z = lane; z < rows_z * 8 * PARTS; z += 32) {
                        const int row = end + z / (8 * PARTS), c = z % (8 * PARTS);
                        *reinterpret_cast<uint4 *>(smem + 2 * QT + slot * UNIT + c / 8 * COL + row * 128 + c % 8 * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&fixed[slot]);
                    ++asks;
                }
                u += n_here;
                if (u < u1) cur.next_item(a, Q);
            }
        }
    } else {
        // ---------------- softmax and output of row tile x, one thread per row
        const int x = warp >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lanes + x * 128, tO = tmem + lanes + 256 + x * 128;
        const int tok = row / G, g = row - tok * G;
        uint32_t sp = 0, op = 0;
        for (long u = u0; u < u1;) {
            if (!begin(u)) break;
            const KtRows rt(a, cur, Q, x);
            const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u);
            const int first = (cur.lo_t + cur.kt) * KT_TILE;
            const bool live = tok < rt.t1 - rt.t0 && row < TT * G;
            const int p = live ? cur.s.p0 + rt.t0 + tok : rt.hi - 1;      // this row's position
            float m = -INFINITY, l = 0.0f;
            bool begun = false;
            for (int i = 0; i < n_here; ++i) {
                const int j0 = first + i * KT_TILE;
                if (!rt.sees(j0)) continue;
                kt_wait(&s_full[x], sp, abort_flag, status);
                sp ^= 1;
                tc_fence_after();
                // some row of the tile does not see all 128
                const bool edge = j0 + KT_TILE > cur.s.p0 + rt.t0 + 1 || (a.window && j0 < rt.hi - a.window);
                const int top_j = p - j0, bottom_j = a.window ? top_j - a.window : -1;
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                // scores of 16 columns from c that the row does not see
                auto hide = [&](uint32_t *v, int c) {
                    const int up = min(max(top_j + 1 - c, 0), 16), dn = min(max(bottom_j + 1 - c, 0), 16);
                    const uint32_t seen = ((1u << up) - 1u) & ~((1u << dn) - 1u);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (!(seen >> e & 1u)) v[e] = 0xff800000u;
                };
                // weights of 16 scores -> 8 packed pairs; their sum added to `add`
                const f32x2 scale22 = pack2(a.scale2, a.scale2);
                auto weigh = [&](const uint32_t *v, f32x2 minus, uint32_t *pk, f32x2 (&add)[2]) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const f32x2 x = fma2(pack2(__uint_as_float(v[2 * e]), __uint_as_float(v[2 * e + 1])), scale22, minus);
                        float e0, e1;
                        unpack2(x, e0, e1);
                        e0 = ex2(e0);
                        e1 = ex2(e1);
                        add[e & 1] = add2(add[e & 1], pack2(e0, e1));
                        uint32_t w[1];
                        split_pair<HALF, 1>(e0, e1, w);
                        pk[e] = w[0];
                    }
                };
                auto largest = [&](const uint32_t *v) {
#pragma unroll
                    for (int e = 0; e < 16; e += 2)
                        mx[e / 2 & 3] = fmaxf(mx[e / 2 & 3], fmaxf(__uint_as_float(v[e]), __uint_as_float(v[e + 1])));
                };
                // O and l to the scale of a larger maximum
                auto raise = [&](float top) {
                    const bool grow = top > m + 8.0f;
                    if (!__any_sync(0xffffffffu, grow)) return false;
                    const float f = grow ? ex2(m - top) : 1.0f;
                    if (grow) {
                        m = top;
                        l *= f;
                    }
                    if (begun) {                          // O holds sums (an item's first product sets it)
#pragma unroll 1
                        for (int c = 0; c < HD; c += 16) {
                            uint32_t o[16];
                            tmem_ld16_nowait(tO + c, o);
                            tmem_wait_ld();
                            settle16(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tmem_st16(tO + c, o);
                        }
                    }
                    return true;
                };
                auto top_of = [&]() { return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale2; };
                if (!begun) {                             // nothing is known of the maximum yet
                    uint32_t s[2][32];
                    tmem_ld32_nowait(tS, s[0]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t *const v = s[c & 1];
                        tmem_wait_ld();
                        settle32(v);
                        if (c < 3) tmem_ld32_nowait(tS + 32 * (c + 1), s[(c + 1) & 1]);
                        if (edge) {
                            hide(v, 32 * c);
                            hide(v + 16, 32 * c + 16);
                        }
                        largest(v);
                        largest(v + 16);
                    }
                    raise(top_of());
                }
                f32x2 add[2] = {0, 0};
                uint32_t pk[64];                          // kept until m has proved large enough
                {
                    const float base = m == -INFINITY ? 0.0f : m;
                    const f32x2 minus = pack2(-base, -base);
                    uint32_t s[2][16];
                    tmem_ld16_nowait(tS, s[0]);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {         // 16 columns while the next 16 are on their way
                        uint32_t *const v = s[c & 1];
                        tmem_wait_ld();
                        settle16(v);
                        if (c < 7) tmem_ld16_nowait(tS + 16 * (c + 1), s[(c + 1) & 1]);
                        if (edge) hide(v, 16 * c);
                        largest(v);
                        weigh(v, minus, pk + 8 * c, add);
                    }
                }
                if (!raise(top_of())) {
                    tmem_st32(tS, pk);
                    tmem_st32(tS + 32, pk + 32);
                } else {                                  // rarely: the weights again, with the new maximum
                    const float base = m == -INFINITY ? 0.0f : m;
                    const f32x2 minus = pack2(-base, -base);
                    add[0] = add[1] = 0;
#pragma unroll 1
                    for (int c = 0; c < 128; c += 16) {   // P's columns lie behind those of S still to be read
                        uint32_t v[16], w[8];
                        tmem_ld16_nowait(tS + c, v);
                        tmem_wait_ld();
                        settle16(v);
                        if (edge) hide(v, c);
                        weigh(v, minus, w, add);
                        tmem_st8(tS + c / 2, w);
                    }
                }
                begun = true;
                float a0, a1;
                unpack2(add2(add[0], add[1]), a0, a1);
                l += a0 + a1;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[x]);
            }
            if (begun) {
                kt_wait(&o_full[x], op, abort_flag, status);
                op ^= 1;
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
                if (parts.join(a.counters + parts.slot_of(gi * gs) * 2 + x, &s_last[x], gi * gs, 1, n_in, ng == 1, write16) && ng > 1)
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
