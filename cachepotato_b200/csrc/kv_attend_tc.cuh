// kv_attend_tc.cuh — what the tcgen05 attention kernels share (kv_attend_tc.cu for 16-bit rows,
// kv_attend_tcf.cu for f32 rows): the units of chunks, a block's share of them, bounded waits, and the
// joining of an item's parts.
#pragma once
#include <algorithm>

#include "kv_attend.cuh"

namespace cpg {

constexpr int KT_ROWS = 128;                              // rows of an MMA tile
constexpr int KT_THREADS = 384, KT_LOAD_K = 8, KT_MMA = 9, KT_LOAD_V = 10;
template <int HD> constexpr int kt_part() { return (2 + HD) * KT_ROWS; }       // floats of a row tile's part: m, l, o (four columns of a row together)

// Sequence i in units. Group p of its rows (one row tile or a pair) holds tokens [p·Q, min(len, p·Q + Q)).
struct KtSeq {
    KvSeq s;
    int pairs;
    long head_units;                                      // of one cached head
};
// tiles of TILE positions of pair p; with a window, from the first token's on
template <int TILE>
__device__ __forceinline__ int kt_tiles(const AttendArgs &a, int Q, const KvSeq &s, int p) {
    const int lo = a.window ? max(0, s.p0 + p * Q - a.window + 1) : 0;
    return (s.p0 + min(s.len, p * Q + Q) - 1) / TILE + 1 - lo / TILE;
}
template <int TILE, int FIXED>
__device__ __forceinline__ KtSeq kt_seq(const AttendArgs &a, int Q, int i) {
    KtSeq q;
    q.s = kv_seq(a.b, i);
    q.pairs = (q.s.len + Q - 1) / Q;
    q.head_units = 0;
    // a handful of instructions a pair; a closed form took longer than summing thousands of pairs
    for (int p = 0; p < q.pairs; ++p) q.head_units += FIXED + kt_tiles<TILE>(a, Q, q.s, p);
    return q;
}

// A place in the order of units: sequence, cached head, pair, position tile (kt from -FIXED: an item's
// begin and end are worth FIXED units, see KD_FIXED).
template <int TILE, int FIXED>
struct KtCursor {
    int seq, kh, pair, kt;
    KvSeq s;
    int pairs;
    int lo_t, nt, hi;                                     // the item's position tiles; one past its last position
    __device__ __forceinline__ int lo_of(const AttendArgs &a, int tok) const {
        return a.window ? max(0, s.p0 + tok - a.window + 1) : 0;
    }
    __device__ __forceinline__ void item(const AttendArgs &a, int Q) {
        hi = s.p0 + min(s.len, (pair + 1) * Q);
        lo_t = lo_of(a, pair * Q) / TILE;
        nt = kt_tiles<TILE>(a, Q, s, pair);
    }
    __device__ __forceinline__ void next_item(const AttendArgs &a, int Q) {
        kt = -FIXED;
        if (++pair < pairs) {
            item(a, Q);
            return;
        }
        pair = 0;
        if (++kh == a.c.KV) {
            kh = 0;
            do {
                if (++seq >= a.b.n) return;
                s = kv_seq(a.b, seq);
            } while (s.len == 0);
            pairs = (s.len + Q - 1) / Q;
        }
        item(a, Q);
    }
};

// What a block keeps in shared memory of its share.
template <int TILE, int FIXED>
struct KtShared {
    long scan[KT_THREADS / 32], off;
    KvCut cut;
    KtCursor<TILE, FIXED> cur;
};
// This block's range [u0, u1) of all items' units, and in sh.cur the place it starts at, for which the
// caller's next __syncthreads makes sh ready. false: it has nothing to do (the whole block agrees).
template <int TILE, int FIXED>
__device__ __forceinline__ bool kt_begin(const AttendArgs &a, int Q, KtShared<TILE, FIXED> &sh, long &u0, long &u1) {
    u0 = u1 = 0;
    const int n = a.b.n, blk = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    long before = 0;
    KvCut cut;
    auto range = [&](long total) {                        // false: nothing for this block
        const int NB = (int)min((long)gridDim.x, total);
        if (blk >= NB) return false;
        cut = KvCut(total, NB);
        u0 = cut.start(blk);
        u1 = cut.start(blk + 1);
        return true;
    };
    if (n > KT_THREADS) {                                 // more sequences than threads: their sum first
        long sum = 0;
        for (int i = tid; i < n; i += KT_THREADS) {
            const KtSeq q = kt_seq<TILE, FIXED>(a, Q, i);
            sum += q.head_units * a.c.KV;
            if (q.s.bad && blk == 0) atomicOr(a.c.status, KV_BAD_POS);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) sh.scan[warp] = sum;
        __syncthreads();
        sum = 0;
        for (int w = 0; w < KT_THREADS / 32; ++w) sum += sh.scan[w];
        if (!range(sum)) return false;
        __syncthreads();
    }
    for (int c0 = 0; c0 < n; c0 += KT_THREADS) {          // THREADS sequences at a time
        KtSeq mine{};
        if (c0 + tid < n) {
            mine = kt_seq<TILE, FIXED>(a, Q, c0 + tid);
            // (of more, all have been looked at above: this loop ends at the block's own)
            if (n <= KT_THREADS && mine.s.bad && blk == 0) atomicOr(a.c.status, KV_BAD_POS);
        }
        const long x = mine.head_units * a.c.KV;
        long inc = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) sh.scan[warp] = inc;
        __syncthreads();
        long base = before, all = 0;
        for (int w = 0; w < KT_THREADS / 32; ++w) {
            if (w < warp) base += sh.scan[w];
            all += sh.scan[w];
        }
        if (n <= KT_THREADS && !range(all)) return false;
        const long at = u0 - (base + inc - x);
        if (at >= 0 && at < x) {
            KtCursor<TILE, FIXED> c;
            c.seq = c0 + tid;
            c.s = mine.s;
            c.pairs = mine.pairs;
            c.kh = (int)kv_div(at, mine.head_units);
            sh.off = at - c.kh * mine.head_units;
            sh.cur = c;
        }
        before += all;
        __syncthreads();
        if (u0 < before) break;
    }
    if (u0 >= u1) return false;                           // no sequences at all
    if (tid == 0) sh.cut = cut;
    if (warp == 0) {                                      // the pair that holds unit sh.off, 32 pairs at a time
        KtCursor<TILE, FIXED> c = sh.cur;
        long off = sh.off;
        for (int p0 = 0; p0 < c.pairs; p0 += 32) {
            const int p = p0 + lane, mine = p < c.pairs ? FIXED + kt_tiles<TILE>(a, Q, c.s, p) : 0;
            int inc = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            const int all = __shfl_sync(0xffffffffu, inc, 31);
            if (off < all) {
                if (off >= inc - mine && off < inc) {
                    c.pair = p;
                    c.kt = (int)off - (inc - mine) - FIXED;
                    c.item(a, Q);
                    sh.cur = c;
                }
                break;
            }
            off -= all;
        }
    }
    return true;
}

__device__ __forceinline__ bool kt_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int *status) {
    if (mbar_try_wait(smem_u32(bar), parity)) return true;
    if (*abort_flag) return false;
    if (mbar_wait(bar, parity)) return true;
    *abort_flag = 1;
    atomicOr(status, KV_TIMEOUT);
    return false;
}

// The same for a whole warp, which goes on or leaves together.
__device__ __forceinline__ bool kt_wait_warp(uint64_t *bar, uint32_t parity, volatile int *abort_flag, int *status) {
    return __all_sync(0xffffffffu, kt_wait(bar, parity, abort_flag, status));
}

// Whether the V tile at position j0 of an item that sees [lo, hi) has places outside that range in the
// boxes of its first or last position: what they hold is nobody's, and a weight of zero does not silence
// a NaN, so they are cleared (kt_clear) before the tile is multiplied. (box is a power of two.)
__device__ __forceinline__ bool kt_fix(const AttendArgs &a, int tile, int lo, int hi, int j0) {
    return (lo > j0 && (lo - j0) & (a.box - 1)) || (hi < j0 + tile && (hi - j0) & (a.box - 1));
}
// Those places become zeros, by one warp, in a tile of PARTS columns of 128 bytes a place.
template <int TILE, int PARTS>
__device__ __forceinline__ void kt_clear(const AttendArgs &a, uint8_t *at, int lo, int hi, int j0, int lane) {
    auto clear = [&](int from, int to) {                  // places [from, to) of the tile
        for (int z = lane; z < (to - from) * 8 * PARTS; z += 32) {
            const int row = from + z / (8 * PARTS), c = z % (8 * PARTS);
            *reinterpret_cast<uint4 *>(at + c / 8 * (TILE * 128) + row * 128 + c % 8 * 16) = make_uint4(0, 0, 0, 0);
        }
    };
    const int front = lo - j0, end = hi - j0;
    if (front > 0) clear(front & -a.box, front);
    if (end < TILE) clear(end, (end + a.box - 1) & -a.box);
    fence_async_smem();
    __syncwarp();
}

// Two f32 in one 64-bit register, worked on by one instruction (sm_100).
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(f32x2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Nothing that uses r may be moved before this point (the wait for the loads that fill it).
__device__ __forceinline__ void settle16(uint32_t *r) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                      "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}
__device__ __forceinline__ void settle32(uint32_t *r) {
    settle16(r);
    settle16(r + 16);
}

// The parts of one item for row tile x of its group, among the blocks from b0 on: block b0 leaves its
// part in the second of its two slots (the item is its last), the others in their first. 128 threads
// (named barrier 1 + x), one per row.
template <int HD>
struct KtParts {
    float *base;
    int x, row, b0;
    bool live;                                            // rows that hold nothing are neither left nor read
    __device__ __forceinline__ int slot_of(int k) const { return k == 0 ? 2 * b0 + 1 : 2 * (b0 + k); }
    __device__ __forceinline__ float *at(int k) const { return base + ((size_t)slot_of(k) * 2 + x) * kt_part<HD>(); }
    __device__ __forceinline__ void put16(float *to, int c, const float *v) const {
        if (!live) return;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            __stcg(reinterpret_cast<float4 *>(to + 2 * KT_ROWS) + (c / 4 + e) * KT_ROWS + row,
                   make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]));
    }
    // parts first, first + step, ... (count of them), joined by the last of their blocks: into the first
    // one's place, or (last) through write(column, 16 sums, 1 / l); false for the blocks that were not last
    template <typename Write>
    __device__ __forceinline__ bool join(int *counter, int *s_last, int first, int step, int count, bool last, Write write) const {
        named_bar_sync(1 + x, 128);
        if (row == 0) {
            const int mine = kv_arrive(counter) == count - 1;
            if (mine) *counter = 0;                       // ready for the next call
            *s_last = mine;
        }
        named_bar_sync(1 + x, 128);
        const bool mine = *s_last != 0;
        named_bar_sync(1 + x, 128);
        if (!mine) return false;
        if (!live) return true;
        float M = -INFINITY, L = 0.0f;
#pragma unroll 4
        for (int k = 0; k < count; ++k) M = fmaxf(M, __ldcg(at(first + k * step) + row));
        const float bs = M == -INFINITY ? 0.0f : M;
#pragma unroll 4
        for (int k = 0; k < count; ++k)
            L = fmaf(ex2(__ldcg(at(first + k * step) + row) - bs), __ldcg(at(first + k * step) + KT_ROWS + row), L);
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        float *to = at(first);
#pragma unroll 1
        for (int c = 0; c < HD; c += 32) {
            float v[32];
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = 0.0f;
            for (int k = 0; k < count; k += 2) {          // two parts' columns in flight
                float4 y[2][8];
                float w[2];
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const float *src = at(first + min(k + z, count - 1) * step);
                    w[z] = __ldcg(src + row);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        y[z][e] = __ldcg(reinterpret_cast<const float4 *>(src + 2 * KT_ROWS) + (c / 4 + e) * KT_ROWS + row);
                }
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    const float f = k + z < count ? ex2(w[z] - bs) : 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[4 * e] = fmaf(f, y[z][e].x, v[4 * e]);
                        v[4 * e + 1] = fmaf(f, y[z][e].y, v[4 * e + 1]);
                        v[4 * e + 2] = fmaf(f, y[z][e].z, v[4 * e + 2]);
                        v[4 * e + 3] = fmaf(f, y[z][e].w, v[4 * e + 3]);
                    }
                }
            }
            if (last) {
                write(c, v, inv);
                write(c + 16, v + 16, inv);
            } else {
                put16(to, c, v);
                put16(to, c + 16, v + 16);
            }
        }
        if (!last) {
            __stcg(to + row, M);
            __stcg(to + KT_ROWS + row, L);
        }
        return true;
    }
};

}  // namespace cpg
