// kv_attend_tcf.cu — attention of chunks of f32 rows over the paged cache on the 5th-generation tensor
// cores, at f32 accuracy (the formula and the meaning of the arguments: kv_attend.cu).
//
// Operands are split as in kv_attend.cu: q and the weights into two f16 terms over an f16 cache, into
// three bf16 terms otherwise, an f32 cache's keys and values into three bf16 terms; the products whose
// weight is 2^-16 and more are kept, smallest first. The tensor core cuts off what it adds to an
// accumulator, so nothing is accumulated there for longer than one tile of 64 positions: each p·v is
// added, rounded, to a row's sums in registers. Bound by the tensor cores over an f32 cache (six
// products), by the softmax's registers and instructions over a 16-bit one.
//   work    Items are (sequence, cached head, row tile): 128/G tokens x G heads = 128 rows; units are
//           tiles of 64 positions, shared out as in kv_attend_tc.cu.
//   block   warps 0-3   one thread per row: q's terms into TMEM; per tile the softmax (exact running
//                       maximum, since rescaling costs nothing: it is the factor of the addition), P's
//                       terms over S, and the last tile's p·v from TMEM into 128 registers of sums
//           warps 4-7   f32 cache: the tile that TMA brought into three bf16 planes, 128-byte swizzle;
//                       places behind the last position become zeros
//           warps 8, 10 producers (tensor TMA), as in kv_attend_tc.cu
//           warp 9      tcgen05.mma: S = q·K^T with q from TMEM, into one of two S while the softmax
//                       works on the other; p·v
//           TMEM: q's terms at 0, S at 192 and 256, P's first two terms over its S, the third at 320,
//           p·v at 352.
//   join    Parts of an item that several blocks share, as in kv_attend_tc.cu.
//   measured  512 f32 rows of 32 heads over themselves, f32 cache (2.1 GFLOP, six times that in bf16
//           products): 40 us: 2.5 us to the block's range, 4 us for q's terms, 3.3 us a tile (softmax,
//           p·v and its collection wait for one another), 3.5 us to end an item; over f16 35 us, bf16 31 us.
//           2048 rows behind 4096 positions (172 GFLOP): 1186 us over f32, 461 over f16, 537 over bf16.
//           Heads of 128 spill 128 to 172 bytes a thread.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "kv_attend_tc.cuh"

namespace cpg {

constexpr int KF_TILE = 64, KF_FIXED = 2;                 // positions of an MMA tile; units an item's begin and end are worth
constexpr int KF_S = 192, KF_P3 = 320, KF_O = 352;        // TMEM columns
template <bool F32C, int HD> constexpr int kf_plane() { return KF_TILE * HD * 2; }                    // one 16-bit plane of a tile
template <bool F32C, int HD> constexpr int kf_unit() { return KF_TILE * HD * (F32C ? 4 : 2); }        // what TMA brings
template <bool F32C, int HD> constexpr int kf_units() { return (F32C ? 96 : 128) * 1024 / kf_unit<F32C, HD>(); }
template <bool F32C, int HD> constexpr int kf_smem() {
    return 1024 + kf_units<F32C, HD>() * kf_unit<F32C, HD>() + (F32C ? 6 * kf_plane<F32C, HD>() : 0);
}

template <bool HALF, bool F32C, int HD>
__global__ void __launch_bounds__(KT_THREADS, 1) k_kv_attend_tcf(const __grid_constant__ AttendArgs a,
                                                                const __grid_constant__ CUtensorMap tm_k,
                                                                const __grid_constant__ CUtensorMap tm_v) {
    constexpr int NQ = HALF ? 2 : 3, NK = F32C ? 3 : 1;
    constexpr int ES = F32C ? 4 : 2, PARTS = HD * ES / 128, COL = KF_TILE * 128;       // 128-byte columns of a tile
    constexpr int UNIT = kf_unit<F32C, HD>(), NU = kf_units<F32C, HD>(), PLANE = kf_plane<F32C, HD>();
    constexpr uint32_t FMT = HALF ? 0u : UMMA_BF16;
    constexpr uint32_t ID_QK = umma_idesc_f16(128, KF_TILE) | FMT, ID_PV = umma_idesc_f16(128, HD) | FMT | UMMA_B_MN;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t *const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t full[NU], empty[NU], fixed[NU], k_full, k_empty, v_full, v_empty, q_full, s_full[2], p_full,
        o_full, drain;
    __shared__ KtShared<KF_TILE, KF_FIXED> sh;
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort, s_last;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.H / a.c.KV, TT = KT_ROWS / G;         // tokens of a row tile
    if (tid == 0) {
        for (int i = 0; i < NU; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], F32C ? 4 : 1);
            mbar_init(&fixed[i], 1);
        }
        mbar_init(&k_full, 4);
        mbar_init(&v_full, 4);
        mbar_init(&k_empty, 1);
        mbar_init(&v_empty, 1);
        mbar_init(&q_full, 4);
        mbar_init(&s_full[0], 1);
        mbar_init(&s_full[1], 1);
        mbar_init(&p_full, 4);
        mbar_init(&o_full, 1);
        mbar_init(&drain, 1);
        fence_mbar_init();
        s_abort = 0;
        prefetch_map(&tm_k);
        prefetch_map(&tm_v);
    }
    pdl_wait();
    pdl_launch_dependents();

    long u0, u1;                                          // this block's range of units
    if (!kt_begin<KF_TILE, KF_FIXED>(a, TT, sh, u0, u1)) return;
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
    uint8_t *const planes = smem + NU * UNIT;             // K's three, then V's
    const uint32_t ring = smem_u32(smem);
    KtCursor<KF_TILE, KF_FIXED> cur = sh.cur;
    // skips an item's fixed share: false if nothing of the item itself is this block's
    auto begin = [&](long &u) {
        if (cur.kt < 0) {
            u -= cur.kt;
            cur.kt = 0;
        }
        return u < u1;
    };

    // registers: the block starts with 384 x 168; 128 threads take 232, 128 keep 168, 128 go down to 104
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp == KT_LOAD_K || warp == KT_LOAD_V) {
            // ---------------- producers of the K and of the V tiles, in turn through the ring (an f32
            // cache's three slots serve both: one warp loads them). Lane b loads box b of a tile.
            const int first_half = !F32C && warp == KT_LOAD_V, halves = F32C ? 2 : 1;
            const int boxes = KF_TILE / a.box * PARTS;
            int slot = first_half, turn = 0;
            bool ok = !F32C || warp == KT_LOAD_K;
            const bool mine = ok;
            for (long u = u0; u < u1 && ok;) {
                if (!begin(u)) break;
                const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u), lo = cur.lo_of(a, cur.pair * TT);
                // page and place of this lane's box of tile i; the next tile's is asked for ahead
                auto find = [&](int i, int &page, int &place) {
                    const int j = (cur.lo_t + cur.kt + i) * KF_TILE + lane / PARTS * a.box;
                    place = -1;                           // nothing of it is seen
                    if (lane < boxes && i < n_here && j < cur.hi && j + a.box > lo) {
                        const int pg = j / a.c.P;
                        page = a.b.pages[(size_t)cur.seq * a.b.table_stride + pg];
                        place = j - pg * a.c.P;
                    }
                };
                int next_page = 0, next_place;
                find(0, next_page, next_place);
                for (int i = 0; i < n_here && ok; ++i) {
                    const bool inside = next_place >= 0 && next_page >= 0 && next_page < a.c.n_pages;
                    if (next_place >= 0 && !inside) atomicOr(status, KV_BAD_PAGE);
                    const int page = inside ? next_page : a.c.n_pages, place = max(next_place, 0);   // outside the pool: zeros
                    find(i + 1, next_page, next_place);
                    for (int half = first_half; half < first_half + halves; ++half) {     // K, then V
                        ok = !turn || kt_wait_warp(&empty[slot], (uint32_t)(turn - 1) & 1u, abort_flag, status);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(&full[slot], UNIT);
                        __syncwarp();
                        if (lane < boxes)
                            tma_load_4d(ring + slot * UNIT + lane % PARTS * COL + lane / PARTS * a.box * 128, half ? &tm_v : &tm_k,
                                        lane % PARTS * (128 / ES), place, cur.kh, page, &full[slot]);
                        // 16-bit cache: places that no row of the item sees, in a box some row sees
                        const int j0 = (cur.lo_t + cur.kt + i) * KF_TILE;
                        if (!F32C && half && kt_fix(a, KF_TILE, lo, cur.hi, j0)) {
                            ok = kt_wait_warp(&full[slot], (uint32_t)turn & 1u, abort_flag, status);
                            if (!ok) break;
                            kt_clear<KF_TILE, PARTS>(a, smem + slot * UNIT, lo, cur.hi, j0, lane);
                            if (lane == 0) mbar_arrive(&fixed[slot]);
                        }
                        slot += 3 - halves;
                        if (slot >= NU) {
                            slot -= NU;
                            ++turn;
                        }
                    }
                }
                u += n_here;
                if (u < u1) cur.next_item(a, TT);
            }
            if (mine && !ok) {                            // copies in flight land before the block may end
                for (int i = first_half; i < NU; i += 3 - halves) {
                    const int fills = turn + (i < slot);
                    if (fills) mbar_wait(&full[i], (uint32_t)(fills - 1) & 1u);
                }
            }
        } else if (warp == KT_MMA) {
            // ---------------- tensor core: one elected lane waits and issues
            if (elect_one()) {
                int ks = 0, vs = 1;                       // 16-bit cache: ring slots of the next K and V
                uint32_t kp = 0, vp = 0, fp = 0, pp = 0, qp = 0, b = 0;   // parities; b: the S of the next q·k
                auto step2 = [&](int &s, uint32_t &ph) {
                    s += 2;
                    if (s >= NU) {
                        s -= NU;
                        ph ^= 1;
                    }
                };
                auto wait = [&](uint64_t *bar, uint32_t parity) { return kt_wait(bar, parity, abort_flag, status); };
                const uint32_t kplanes = smem_u32(planes), vplanes = kplanes + 3 * PLANE;
                auto qk = [&]() {
                    if (!wait(F32C ? &k_full : &full[ks], kp)) return false;
                    tc_fence_after();
                    const uint64_t dk = umma_desc_sw128(F32C ? kplanes : ring + ks * UNIT);
                    uint32_t more = 0;
#pragma unroll
                    for (int d = NQ - 1; d >= 0; --d)     // terms of weight 2^-8d (2^-11d)
#pragma unroll
                        for (int j = 0; j <= d && j < NK; ++j)
#pragma unroll
                            for (int k = 0; k < HD / 16; ++k) {
                                umma_f16_ts(tmem + KF_S + b * KF_TILE, tmem + (d - j) * (HD / 2) + k * 8,
                                            dk + ((j * PLANE + k / 4 * COL + k % 4 * 32) >> 4), ID_QK, more);
                                more = 1;
                            }
                    umma_commit(&s_full[b]);
                    umma_commit(F32C ? &k_empty : &empty[ks]);
                    b ^= 1;
                    if (F32C) kp ^= 1;
                    else step2(ks, kp);
                    return true;
                };
                bool ok = true;
                for (long u = u0; u < u1 && ok;) {
                    if (!begin(u)) break;
                    const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u);
                    const int first = (cur.lo_t + cur.kt) * KF_TILE, lo = cur.lo_of(a, cur.pair * TT);
                    if (!wait(&q_full, qp)) break;
                    qp ^= 1;
                    tc_fence_after();
                    ok = qk();
                    for (int i = 0; i < n_here && ok; ++i) {
                        const uint32_t s = tmem + KF_S + (b ^ 1) * KF_TILE;           // of this tile
                        if (i + 1 < n_here) ok = qk();
                        ok = ok && wait(&p_full, pp);
                        pp ^= 1;
                        ok = ok && wait(F32C ? &v_full : &full[vs], vp);
                        if (ok && !F32C && kt_fix(a, KF_TILE, lo, cur.hi, first + i * KF_TILE)) {
                            ok = wait(&fixed[vs], fp >> vs & 1u);
                            fp ^= 1u << vs;
                        }
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t dv = umma_desc_sw128_mn(F32C ? vplanes : ring + vs * UNIT, COL);
                        uint32_t more = 0;
#pragma unroll
                        for (int d = NQ - 1; d >= 0; --d)
#pragma unroll
                            for (int j = 0; j <= d && j < NK; ++j)
#pragma unroll
                                for (int k = 0; k < KF_TILE / 16; ++k) {
                                    umma_f16_ts(tmem + KF_O, (d - j < 2 ? s + (d - j) * 32 : tmem + KF_P3) + k * 8,
                                                dv + ((j * PLANE + k * 2048) >> 4), ID_PV, more);
                                    more = 1;
                                }
                        umma_commit(&o_full);
                        umma_commit(F32C ? &v_empty : &empty[vs]);
                        if (F32C) vp ^= 1;
                        else step2(vs, vp);
                    }
                    u += n_here;
                    if (u < u1) cur.next_item(a, TT);
                }
                // every MMA issued has finished before the block ends
                umma_commit(&drain);
                mbar_wait(&drain, 0);
            }
            __syncwarp();
        }
    } else if (warp >= 4) {
        if constexpr (F32C) {
            // ---------------- an f32 tile into three bf16 planes
            int slot = 0, n = 0;
            uint32_t phase = 0;
            for (long u = u0; u < u1;) {
                if (!begin(u)) break;
                const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u), lo = cur.lo_of(a, cur.pair * TT);
                for (int i = 0; i < n_here; ++i, ++n) {
                    const int j0 = (cur.lo_t + cur.kt + i) * KF_TILE;
#pragma unroll 1
                    for (int half = 0; half < 2; ++half) {                // K, then V
                        kt_wait(&full[slot], phase, abort_flag, status);
                        if (n) kt_wait(half ? &v_empty : &k_empty, (uint32_t)(n - 1) & 1u, abort_flag, status);
                        const uint8_t *const src = smem + slot * UNIT;
                        uint8_t *const dst = planes + half * 3 * PLANE;
#pragma unroll 2
                        for (int it = 0; it < KF_TILE * HD / 8 / 128; ++it) {
                            // eight elements of a place; eight lanes take eight places, so neither side
                            // has bank conflicts
                            const int idx = it * 128 + tid - 128, r = (idx & 7) | (idx >> 5 & 7) << 3, gr = (idx >> 3 & 3) | idx >> 8 << 2;
                            const uint8_t *at = src + gr / 4 * COL + r * 128;
                            float4 x = *reinterpret_cast<const float4 *>(at + (((gr * 2 & 7) ^ (r & 7)) << 4));
                            float4 y = *reinterpret_cast<const float4 *>(at + (((gr * 2 + 1 & 7) ^ (r & 7)) << 4));
                            if (half && (j0 + r >= cur.hi || j0 + r < lo)) x = y = make_float4(0.f, 0.f, 0.f, 0.f);
                            uint32_t t[4][3];
                            split_pair<false, 3>(x.x, x.y, t[0]);
                            split_pair<false, 3>(x.z, x.w, t[1]);
                            split_pair<false, 3>(y.x, y.y, t[2]);
                            split_pair<false, 3>(y.z, y.w, t[3]);
#pragma unroll
                            for (int p = 0; p < 3; ++p)
                                *reinterpret_cast<uint4 *>(dst + p * PLANE + gr / 8 * COL + r * 128 + (((gr & 7) ^ (r & 7)) << 4)) =
                                    make_uint4(t[0][p], t[1][p], t[2][p], t[3][p]);
                        }
                        fence_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(half ? &v_full : &k_full);
                            mbar_arrive(&empty[slot]);    // only now: TMA refills it
                        }
                        if (++slot == NU) {
                            slot = 0;
                            phase ^= 1;
                        }
                    }
                }
                u += n_here;
                if (u < u1) cur.next_item(a, TT);
            }
        }
    } else {
        // ---------------- softmax, sums and output, one thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int row = tid;
        const uint32_t tq = tmem + ((uint32_t)(warp * 32) << 16);
        const int tok = row / G, g = row - tok * G;
        uint32_t sp = 0, op = 0, b = 0;                   // sp: a parity bit for each S
        for (long u = u0; u < u1;) {
            if (!begin(u)) break;
            const int n_here = (int)min((long)(cur.nt - cur.kt), u1 - u);
            const int first = (cur.lo_t + cur.kt) * KF_TILE;
            const int t0 = cur.pair * TT, nt = min(cur.s.len - t0, TT);
            const bool live = tok < nt && row < TT * G;
            const int p0 = cur.s.p0 + t0, p = live ? p0 + tok : cur.hi - 1;           // the tile's first, this row's position
            const size_t cell = (size_t)(cur.s.r0 + t0 + tok);
            float sc = a.scale2;
            {                                             // q's terms
                const float4 *const src = (const float4 *)((const float *)a.q + cell * a.q_stride + (size_t)(cur.kh * G + g) * HD);
                float up = 1.0f;
                if constexpr (HALF) {                     // the row by a power of two so that its largest is in [2^14, 2^15)
                    float mx = 0.0f;
                    if (live) {
#pragma unroll 8
                        for (int e = 0; e < HD / 4; ++e) {
                            const float4 v = src[e];
                            mx = fmaxf(mx, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                        }
                    }
                    const int eb = min(max((int)(__float_as_uint(mx) >> 23), 15), 254);
                    up = __uint_as_float((uint32_t)(268 - eb) << 23);
                    sc = fmaxf(a.scale2 * __uint_as_float((uint32_t)(eb - 14) << 23), 0x1p-126f);   // (a zero would make hidden scores NaN)
                }
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    uint32_t w[NQ][16];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float4 v = live ? src[c / 4 + e] : make_float4(0.f, 0.f, 0.f, 0.f);
                        uint32_t t1[NQ], t2[NQ];
                        split_pair<HALF, NQ>(v.x * up, v.y * up, t1);
                        split_pair<HALF, NQ>(v.z * up, v.w * up, t2);
#pragma unroll
                        for (int q = 0; q < NQ; ++q) {
                            w[q][2 * e] = t1[q];
                            w[q][2 * e + 1] = t2[q];
                        }
                    }
#pragma unroll
                    for (int q = 0; q < NQ; ++q) tmem_st16(tq + q * (HD / 2) + c / 2, w[q]);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&q_full);
            }
            float m = -INFINITY, l = 0.0f, f = 0.0f;      // f: from the sums' scale to that of the p·v in flight
            float o[HD];
#pragma unroll
            for (int e = 0; e < HD; ++e) o[e] = 0.0f;
            auto collect = [&]() {                        // o = o·f + p·v
                kt_wait(&o_full, op, abort_flag, status);
                op ^= 1;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < HD; c += 32) {
                    uint32_t v[32];
                    tmem_ld32_nowait(tq + KF_O + c, v);
                    tmem_wait_ld();
                    settle32(v);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[c + e] = fmaf(o[c + e], f, __uint_as_float(v[e]));
                }
            };
#pragma unroll 1
            for (int i = 0; i < n_here; ++i) {
                if (i) collect();
                const uint32_t tS = tq + KF_S + b * KF_TILE;
                kt_wait(&s_full[b], sp >> b & 1u, abort_flag, status);
                sp ^= 1u << b;
                b ^= 1;
                tc_fence_after();
                uint32_t s[64];
                tmem_ld32_nowait(tS, s);
                tmem_ld32_nowait(tS + 32, s + 32);
                tmem_wait_ld();
                settle32(s);
                settle32(s + 32);
                const int j0 = first + i * KF_TILE;
                if (j0 + KF_TILE > p0 + 1 || (a.window && j0 < cur.hi - a.window)) {
                    // some row of the tile does not see all 64
                    const int top = min(p - j0, 63), bottom = a.window ? max(p - a.window - j0, -1) : -1;
                    const uint64_t seen = top < 0 ? 0ull : (~0ull >> (63 - top)) & (bottom < 0 ? ~0ull : bottom >= 63 ? 0ull : ~0ull << (bottom + 1));
#pragma unroll
                    for (int e = 0; e < 64; ++e)
                        if (!(seen >> e & 1)) s[e] = 0xff800000u;
                }
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 64; e += 2) mx[e / 2 & 3] = fmaxf(mx[e / 2 & 3], fmaxf(__uint_as_float(s[e]), __uint_as_float(s[e + 1])));
                const float mn = fmaxf(m, kv_top<HALF>(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * sc));
                const float base = mn == -INFINITY ? 0.0f : mn, minus = kv_lift<HALF>(14.0f) - base;
                f = ex2(m - base);
                m = mn;
                float add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < 4; ++c) {             // 16 weights, their terms
                    uint32_t w[NQ][8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float e0 = ex2(fmaf(__uint_as_float(s[16 * c + 2 * e]), sc, minus));
                        const float e1 = ex2(fmaf(__uint_as_float(s[16 * c + 2 * e + 1]), sc, minus));
                        add[e & 1] += e0;
                        add[2 + (e & 1)] += e1;
                        uint32_t t[NQ];
                        split_pair<HALF, NQ>(e0, e1, t);
#pragma unroll
                        for (int q = 0; q < NQ; ++q) w[q][e] = t[q];
                    }
                    tmem_st8(tS + 8 * c, w[0]);
                    tmem_st8(tS + 32 + 8 * c, w[1]);
                    if constexpr (NQ == 3) tmem_st8(tq + KF_P3 + 8 * c, w[2]);
                }
                l = fmaf(l, f, (add[0] + add[1]) + (add[2] + add[3]));
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full);
            }
            collect();

            // ---- the item, or this block's part of it, is done: its tiles are units [ua, ue), blocks b0..b1
            const long ua = u - cur.kt, ue = ua + cur.nt;
            u += n_here;
            const int b0 = sh.cut.owner(ua), b1 = sh.cut.owner(ue - 1);
            float *const dst = (float *)a.out + cell * a.out_stride + (size_t)(cur.kh * G + g) * HD;
            auto write16 = [&](int c, const float *v, float inv) {       // 16 columns from c of the row
                if (!live) return;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<float4 *>(dst + c + 4 * e) = make_float4(v[4 * e] * inv, v[4 * e + 1] * inv, v[4 * e + 2] * inv, v[4 * e + 3] * inv);
            };
            if (b0 == b1) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                for (int c = 0; c < HD; c += 16) write16(c, o + c, inv);
            } else {
                const int np = b1 - b0 + 1, pi = (int)blockIdx.x - b0;
                int gs = np;
                if (np > 4)
                    for (gs = 2; gs * gs < np;) ++gs;
                const int ng = (np + gs - 1) / gs, gi = pi / gs, n_in = min(gs, np - gi * gs);
                const KtParts<HD> parts{a.part, 0, row, b0, live};
                float *to = parts.at(pi);
                __stcg(to + row, m);
                __stcg(to + KT_ROWS + row, l);
#pragma unroll
                for (int c = 0; c < HD; c += 16) parts.put16(to, c, o + c);
                if ((n_in == 1 || parts.join(a.counters + parts.slot_of(gi * gs) * 2, &s_last, gi * gs, 1, n_in, ng == 1, write16)) && ng > 1)
                    parts.join(a.counters + 4 * KV_MAX_GRID + b0 * 2, &s_last, 0, gs, ng, true, write16);
            }
            if (u < u1) cur.next_item(a, TT);
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

template <bool HALF, bool F32C, int HD>
static int launch_kf(const AttendArgs &a, const CUtensorMap *maps, cudaStream_t s) {
    static std::atomic<bool> set[64];                    // once per device
    int dev = 0;
    CPG_CUDA(cudaGetDevice(&dev));
    if (dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
        const int rc = allow_max_smem((const void *)k_kv_attend_tcf<HALF, F32C, HD>);
        if (rc) return rc;
        if (dev < 64) set[dev].store(true, std::memory_order_release);
    }
    const int grid = std::min(KV_MAX_GRID, sm_count());
    const cudaError_t ce = launch_pdl(k_kv_attend_tcf<HALF, F32C, HD>, dim3(grid), dim3(KT_THREADS), (size_t)kf_smem<F32C, HD>(),
                                      s, a, maps[0], maps[1]);
    return ce == cudaSuccess ? CPG_OK : cuda_fail(ce, "cpg_kv_attend");
}

int kv_attend_tcf_launch(const AttendArgs &a, const CUtensorMap *maps, int hd, cudaStream_t s) {
    if (a.c.type == CPG_T_F32) return hd == 128 ? launch_kf<false, true, 128>(a, maps, s) : launch_kf<false, true, 64>(a, maps, s);
    if (a.c.type == CPG_T_F16) return hd == 128 ? launch_kf<true, false, 128>(a, maps, s) : launch_kf<true, false, 64>(a, maps, s);
    return hd == 128 ? launch_kf<false, false, 128>(a, maps, s) : launch_kf<false, false, 64>(a, maps, s);
}

}  // namespace cpg
