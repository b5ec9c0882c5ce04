// Attention, forward (attention.h): o = softmax(t) v over the visible keys, and the logarithm of the softmax's sum.
// attn_fwd_kernel: a workgroup owns 128 queries of one head, a wave 32 of them; tiles of 64 keys pass through the LDS once, double-buffered by LDS-DMA, with
//   the running maximum and sum of every query in its lane.  The accumulators are rescaled only when a maximum grows by more than 2^8 since they were last
//   (at every growth: 4096 x 16 heads x 64 88 us instead of 84, in one run).  Measured, without a mask, 4096 x 16 heads, medians of 60 launches: x 128 bfloat16
//   143 us = 0.96 PFLOP/s (a large matrix product of the library: 1.20), x 64 float16 92 us = 0.75 PFLOP/s.  The matrix pipe is busy for half of the time;
//   the exponentials, maxima and roundings between the two products share the issue slots with it, two waves a SIMD taking turns, and bound it, most of all
//   at 64 channels.
// attn_token_kernel: few queries over many keys.  The rows of a wave are (query, head) pairs that share a key head, so a key is read once for all of
//   them; every wave walks its own tiles of 32 keys through its own LDS (no barriers), the keys are split over `splits` workgroups, and
//   attn_combine_kernel joins their (maximum, sum, accumulator).  Measured: 16 single tokens of 32 heads on 8 over caches of up to 16384 keys x 128, 802 MB:
//   149 + 6 us, 5.4 TB/s (a large copy: 4.9): bound by memory.
#include "attention.h"

// Lowest and highest document of every ATTN_TILE tokens.  Tokens of no document do not count (none at all: an empty range that meets no other), but a tile
// that holds some of them must not pass for one of a single document: its range gets one document more.
__global__ __launch_bounds__(256) void attn_ranges_kernel(const int* __restrict__ doc, int64_t stride, int L, int tiles, int2* __restrict__ out) {
    const int groups = (tiles + 3) / 4, b = blockIdx.x / groups, t = (blockIdx.x - b * groups) * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= tiles) return;
    const int j = t * ATTN_TILE + lane;
    const int d = doc[b * stride + (j < L ? j : L - 1)];
    int lo = d < 0 ? 0x7fffffff : d, hi = d < 0 ? -1 : d;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
    }
    if (__ballot(d < 0) && lo == hi) --lo;
    if (lane == 0) out[(int64_t)b * tiles + t] = make_int2(lo, hi);
}

// Row blocks of 128 queries by how many tiles of keys they walk, the longest first: one workgroup a sequence counts and ranks them, 1024 / blocks threads to
// a block.  In their own order the last long blocks of a packed row start late and the chip waits for them: 16384 tokens of 12 documents, 16 heads x 64,
// four rounds of workgroups, 195 -> 168 us with this kernel; two rounds (2 x 4096, 16 heads) gain nothing, hence the third round in attn_ranges.
static constexpr int ATTN_ORDER_TILES = 1024, ATTN_ORDER_BLOCKS = 512;
__global__ __launch_bounds__(1024) void attn_order_kernel(AttnParams p, int* __restrict__ order) {
    __shared__ int2 tiles[ATTN_ORDER_TILES];
    __shared__ int counts[ATTN_ORDER_BLOCKS], ranks[ATTN_ORDER_BLOCKS];
    const int b = blockIdx.x, n = attn_keys(p, b), prefix = attn_prefix(p, b);
    const int log = max(6, 32 - __builtin_clz(p.row_blocks - 1 | 1)), i = threadIdx.x & ((1 << log) - 1), seg = threadIdx.x >> log, segs = 1024 >> log;
    const bool mine = i < p.row_blocks;
    int lo = 1, hi = 0, end = 0;
    if (mine) {
        const int2* r = p.qtiles + (int64_t)b * p.nqt + 2 * i;
        const int2 r0 = r[0], r1 = 2 * i + 1 < p.nqt ? r[1] : r[0];
        lo = max(min(r0.x, r1.x), 0);
        hi = max(r0.y, r1.y);
        end = min(attn_limit(p, min(i * 128 + 127, p.Lq - 1), n, prefix) / ATTN_TILE + 1, p.nkt);
        if (seg == 0) counts[i] = ranks[i] = 0;
    }
    for (int t = threadIdx.x; t < p.nkt; t += 1024) tiles[t] = p.ktiles[(int64_t)b * p.nkt + t];
    __syncthreads();
    int count = 0;
#pragma unroll 4
    for (int t = seg; t < end; t += segs) {
        const int2 of = tiles[t];
        count += (of.y >= lo) & (of.x <= hi);
    }
    if (mine) atomicAdd(counts + i, count);
    __syncthreads();
    if (mine) {
        const int own = counts[i];
        int rank = 0;
#pragma unroll 4
        for (int j = seg; j < p.row_blocks; j += segs) rank += (counts[j] > own) | ((counts[j] == own) & (j > i));
        atomicAdd(ranks + i, rank);
    }
    __syncthreads();
    if (mine && seg == 0) order[b * p.row_blocks + ranks[i]] = i;
}

// One wave's softmax step over the 32 queries of its lanes: S (raw products of KB blocks of 32 keys) -> P as second operands; rescales acc, sum and m.
// MASK: not every key of the tile is visible to every query.
template <typename T, int KB, int DB, int MODE, bool MASK>
__device__ __forceinline__ void attn_softmax_form(f32x16 (&S)[KB], typename AttnVec<T>::x8 (&P)[KB][2], f32x16 (&acc)[DB], float& m, float& sum, const AttnScore& f,
                                                  int lim, int at, int j0, int half, const int* docs, int qdoc) {
    if constexpr (MODE != ATTN_PLAIN) {
        const float dist = (float)(at - j0 - 4 * half);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                S[kb][r] = MODE == ATTN_BIAS ? S[kb][r] * f.mul : f.capped(f.cap_r(S[kb][r]), 0.f);
                if constexpr (MODE != ATTN_CAP) S[kb][r] -= f.slope * fabsf(dist - (float)(32 * kb + 8 * (r >> 2) + (r & 3)));
            }
    }
    if constexpr (MASK) {
        const int last = lim - j0 - 4 * half;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) S[kb][r] = 32 * kb + 8 * (r >> 2) + (r & 3) <= last ? S[kb][r] : -INFINITY;
        if (docs)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const int4 d = *reinterpret_cast<const int4*>(docs + 32 * kb + 8 * a + 4 * half);
                    S[kb][4 * a] = d.x == qdoc ? S[kb][4 * a] : -INFINITY;
                    S[kb][4 * a + 1] = d.y == qdoc ? S[kb][4 * a + 1] : -INFINITY;
                    S[kb][4 * a + 2] = d.z == qdoc ? S[kb][4 * a + 2] : -INFINITY;
                    S[kb][4 * a + 3] = d.w == qdoc ? S[kb][4 * a + 3] : -INFINITY;
                    if (a & 1) __builtin_amdgcn_sched_barrier(0);     // (two loads at a time: registers)
                }
    }
    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) tops[r & 3] = fmaxf(tops[r & 3], S[kb][r]);
    const float mul = MODE == ATTN_PLAIN ? f.mul : 1.f;
    const float top = attn_half_max(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]))) * mul;          // (mul > 0; -inf stays -inf)
    if (__ballot((top > m + 8.f) | ((m == -INFINITY) & (top > m)))) {
        const float now = fmaxf(m, top);
        const float shrink = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        sum *= shrink;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[db][r] *= shrink;
    }
    const float sub = m == -INFINITY ? 0.f : m;
    float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            S[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[kb][r], mul, -sub));
            add[r & 3] += S[kb][r];
        }
        // weights to 16 bits (half a step of the inputs' own type, each on its own: their sum above is of the unrounded ones)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int e = 0; e < 8; ++e) P[kb][c][e] = (T)S[kb][8 * c + e];
    }
    sum += (add[0] + add[1]) + (add[2] + add[3]);
}
template <typename T, int KB, int DB, int MODE>
__device__ __forceinline__ void attn_softmax_step(f32x16 (&S)[KB], typename AttnVec<T>::x8 (&P)[KB][2], f32x16 (&acc)[DB], float& m, float& sum, const AttnScore& f,
                                                  bool full, int lim, int at, int j0, int half, const int* docs, int qdoc) {
    if (full) attn_softmax_form<T, KB, DB, MODE, false>(S, P, acc, m, sum, f, lim, at, j0, half, docs, qdoc);
    else attn_softmax_form<T, KB, DB, MODE, true>(S, P, acc, m, sum, f, lim, at, j0, half, docs, qdoc);
}

// The sums of one wave's 32 rows (query i and head h are the lane's own) over the keys [first, end), 32 at a time, `step` apart
template <int DB> struct AttnSums {
    f32x16 acc[DB];
    float m, sum;
};
template <typename T, int DB>
__device__ __forceinline__ void attn_fwd_store(const AttnParams& p, const f32x16 (&acc)[DB], float m, float sum, int b, int i, int h, int split, int half, bool row_ok) {
    if (p.splits > 1) {
        const int hk = h / p.G;
        const int64_t at = (((int64_t)(b * p.Hk + hk) * p.Lq + i) * p.G + h - hk * p.G) * p.splits + split;
        attn_store_part<DB>(p.part + at * p.D, acc, 1.f, half, p.D, row_ok);
        if (row_ok && half == 0) {
            p.part[p.part_ml + 2 * at] = m;
            p.part[p.part_ml + 2 * at + 1] = sum;
        }
    } else {
        const float by = sum == 0.f ? 0.f : 1.f / sum;
        const int64_t row_at = ((int64_t)(b * (int64_t)p.Lq + i) * p.Hq + h) * p.D;
        attn_store_row<T, DB>((T*)p.out + row_at, acc, by, half, p.D, row_ok);
        if (p.rest) attn_store_row<T, DB, true>((T*)p.rest + row_at, acc, by, half, p.D, row_ok);
        if (p.lse && row_ok && half == 0) p.lse[((int64_t)b * p.Hq + h) * p.Lq + i] = sum == 0.f ? -INFINITY : (m + __builtin_amdgcn_logf(sum)) * ATTN_LN2;
    }
}
#ifdef __HIP_DEVICE_COMPILE__
template <typename T, int DB>
static __device__ __forceinline__ AttnSums<DB> attn_sums_again(attn_args args, int b, int i, int h, bool row_ok, int first, int end, int step, uint32_t lds, bool fine) {
    constexpr int ROW = DB > 2 ? 128 : 64, KEYS = 32, BYTES = KEYS * ROW * 2;
    const AttnParams p = *args;
    const int lane = threadIdx.x & 63, half = lane >> 5, hk = attn_uniform(h / p.G);
    const int n = attn_keys(p, b), at = i + n - p.Lq;
    const int qdoc = p.kdoc && row_ok ? p.qdoc[b * p.qdoc_stride + i] : 0;
    const int lim = !row_ok || qdoc < 0 ? -1 : attn_limit(p, i, n, attn_prefix(p, b));
    const T* q = row_ok ? (const T*)p.q + b * p.qs[0] + i * p.qs[1] + h * p.qs[2] : nullptr;
    const uint64_t k = attn_addr((const T*)p.k + b * p.ks[0] + hk * p.ks[2]), v = attn_addr((const T*)p.v + b * p.vs[0] + hk * p.vs[2]);
    const AttnScore f(p, row_ok ? h : 0);
    AttnStage<ROW, KEYS, 1> sk, sv;
    sk.setup(0, lane, p.ks[1], p.D);
    sv.setup(0, lane, p.vs[1], p.D);
    const AttnLane<ROW> at_lane(lane);
    AttnSums<DB> s;
    AttnMarks<DB> plus, minus;
#pragma unroll 1
    for (int walk = 0; walk < 3; ++walk) {
        const int kind = walk == 0 ? ATTN_PLUS : walk == 1 ? ATTN_MINUS : ATTN_FINITE;
#pragma unroll
        for (int db = 0; db < DB; ++db) s.acc[db] = f32x16{};
        s.m = -INFINITY;
        s.sum = 0.f;
#pragma unroll 1
        for (int j0 = first; j0 < end; j0 += step) {
            uint32_t seen = 0;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int j = j0 + 4 * half + 8 * (r >> 2) + (r & 3);
                if (j <= lim && (!p.kdoc || p.kdoc[b * p.kdoc_stride + j] == qdoc)) seen |= 1u << r;
            }
            if (!__ballot(seen != 0)) continue;
            attn_landed();                                              // (the LDS reads of the tile before)
            sk.issue(k, j0 / KEYS, n, (int)p.ks[1], p.D, lds, 0);
            sv.issue(v, j0 / KEYS, n, (int)p.vs[1], p.D, lds + BYTES, 0);
            attn_landed();
            attn_change<T, BYTES>(lds + BYTES, lane, kind);
            attn_landed();
            const uint32_t k_lds = at_lane.rows(lds), v_lds = at_lane.cols(lds + BYTES);
            f32x16 S = {};
            typename AttnVec<T>::x8 P[2];
            if (kind == ATTN_FINITE) {
#pragma unroll
                for (int c = 0; c < 2 * DB; ++c) S = attn_mfma(attn_row_frag<T, ROW>(k_lds, 0, c), attn_lane_frag<T>(q, 2 * c + half, p.D), S);
                float top = -INFINITY;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    S[r] = seen >> r & 1 ? attn_score(f, S[r], (float)(at - (j0 + 4 * half + 8 * (r >> 2) + (r & 3)))) : -INFINITY;
                    top = fmaxf(top, S[r]);
                }
                const float now = fmaxf(s.m, attn_half_max(top)), shrink = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(s.m - now);
                s.m = now;
                s.sum *= shrink;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s.acc[db][r] *= shrink;
                const float sub = now == -INFINITY ? 0.f : now;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    S[r] = __builtin_amdgcn_exp2f(S[r] - sub);
                    s.sum += S[r];
                }
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e) P[c][e] = (T)S[8 * c + e];
            } else {
                attn_ones<T>(seen, P);
            }
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const auto vf = attn_col_frag<T, ROW>(v_lds, c, db);
                    s.acc[db] = attn_mfma(vf, P[c], s.acc[db]);
                    if (fine && kind == ATTN_FINITE) s.acc[db] = attn_mfma(vf, attn_left_over<T>(S, P[c], c), s.acc[db]);
                }
        }
        if (walk == 0) plus.take(s.acc);
        if (walk == 1) minus.take(s.acc);
    }
    plus.add(s.acc, INFINITY);
    minus.add(s.acc, -INFINITY);
    s.sum = attn_half_sum(s.sum);
    return s;
}
template <typename T, int DB>
static __device__ __attribute__((noinline)) AttnSums<DB> attn_out_again(attn_args args, int b, int i, int h, bool row_ok, int first, int end, int step, uint32_t lds) {
    return attn_sums_again<T, DB>(args, b, i, h, row_ok, first, end, step, lds, true);
}
template <typename T, int DB>
static __device__ __attribute__((noinline)) void attn_rows_again(attn_args args, int b, int i, int h, bool row_ok, int split, int first, int end, uint32_t lds, bool fine) {
    const AttnSums<DB> s = attn_sums_again<T, DB>(args, b, i, h, row_ok, first, end, 32, lds, fine);
    const AttnParams p = *args;
    attn_fwd_store<T, DB>(p, s.acc, s.m, s.sum, b, i, h, split, (threadIdx.x & 63) >> 5, row_ok);
}
#endif

template <typename T, int DB, int MODE, bool DOCS>
__global__ __launch_bounds__(256, DB < 3 ? 3 : 2) void attn_fwd_kernel(AttnParams p) {
#ifdef __HIP_DEVICE_COMPILE__                            // (hipcc drops the launch stub of a template whose body its host pass cannot read)
    constexpr int ROW = DB > 2 ? 128 : 64, TILE_BYTES = ATTN_TILE * ROW * 2;
    __shared__ __align__(1024) char smem[4 * TILE_BYTES];                 // [buffer][k, v]
    __shared__ __align__(16) int sdoc[2][ATTN_TILE];
    __shared__ uint32_t said[4];
    const int wave = attn_uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
    // consecutive workgroups go to different XCDs: give each XCD whole heads, so that its L2 serves their keys, and the longest rows of a head first
    // (p.splits > 1: the keys in that many runs of whole tiles, joined by attn_combine_kernel)
    const int total = p.B * p.Hq * p.row_blocks * p.splits, per = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || id >= total) return;
    const int split = id % p.splits, pos = id / p.splits % p.row_blocks, bh = id / p.splits / p.row_blocks, h = bh % p.Hq, b = bh / p.Hq, hk = h / p.G;
    const int blk = DOCS && p.order ? p.order[b * p.row_blocks + pos] : p.row_blocks - 1 - pos;
    const int n = attn_keys(p, b), prefix = attn_prefix(p, b), q0 = blk * 128;
    const int i = q0 + 32 * wave + l31;
    const bool row_ok = i < p.Lq;
    const int qdoc = DOCS && row_ok ? p.qdoc[b * p.qdoc_stride + i] : 0;
    const int lim = !row_ok || qdoc < 0 ? -1 : attn_limit(p, i, n, prefix);
    const int lim_last = attn_limit(p, min(q0 + 32 * wave + 31, p.Lq - 1), n, prefix);
    const int key_end = attn_limit(p, min(q0 + 127, p.Lq - 1), n, prefix) + 1;
    int dlo = 0, dhi = 0;
    bool one = true;                                                            // one document, and every query in it
    if constexpr (DOCS) {                                                       // documents of this workgroup's queries: two ranges of ATTN_TILE queries
        const int2* r = p.qtiles + (int64_t)b * p.nqt + 2 * blk;
        const int2 r0 = r[0], r1 = 2 * blk + 1 < p.nqt ? r[1] : r[0];
        dlo = min(r0.x, r1.x);
        dhi = max(r0.y, r1.y);
        one = r0.x == r0.y && r1.x == r1.y && r0.x == r1.x;
    }
    AttnTiles<DOCS> tiles;
    const int run = (p.nkt + p.splits - 1) / p.splits, run_first = split * run, run_end = min((key_end + ATTN_TILE - 1) / ATTN_TILE, run_first + run);
    tiles.start(DOCS ? p.ktiles + (int64_t)b * p.nkt : nullptr, run_first, run_end, max(dlo, 0), dhi);

    typename AttnVec<T>::x8 qf[2 * DB];
    const T* q = row_ok ? (const T*)p.q + b * p.qs[0] + i * p.qs[1] + h * p.qs[2] : nullptr;
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c) qf[c] = attn_lane_frag<T>(q, 2 * c + half, p.D);
    const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[2];
    const T* v = (const T*)p.v + b * p.vs[0] + hk * p.vs[2];
    const int* kdoc = DOCS ? p.kdoc + b * p.kdoc_stride : nullptr;
    const AttnScore f(p, h);
    AttnStage<ROW, ATTN_TILE, 4> sk, sv;
    sk.setup(wave, lane, p.ks[1], p.D);
    sv.setup(wave, lane, p.vs[1], p.D);

    f32x16 acc[DB] = {};
    float m = -INFINITY, sum = 0.f;
    int doc_next = 0;                                                   // of the tile being staged: loaded ahead of its pieces, written behind the products
    const uint64_t k_at = attn_addr(k), v_at = attn_addr(v);
    const int k_row = (int)p.ks[1], v_row = (int)p.vs[1];
    const AttnLane<ROW> at_lane(lane);
    const uint32_t lds = attn_lds(smem);
    auto stage = [&](int t, int buf) {
        if (DOCS && wave == 0) doc_next = kdoc[min(t * ATTN_TILE + lane, p.Lk - 1)];
        sk.issue(k_at, t, n, k_row, p.D, lds + buf * 2 * TILE_BYTES, wave);
        sv.issue(v_at, t, n, v_row, p.D, lds + buf * 2 * TILE_BYTES + TILE_BYTES, wave);
    };
    int t = tiles.next(lane), buf = 0;
    const bool fine = tiles.few(lane);
    if (t >= 0) stage(t, 0);
    if (DOCS && wave == 0) sdoc[0][lane] = doc_next;
    // every key of tile t visible to every query of the workgroup
    const int full_end = DOCS && !one ? 0 : attn_limit(p, q0, n, prefix) + 1;
    auto full = [&] { return !fine && (t + 1) * ATTN_TILE <= full_end && (!DOCS || ((tiles.low == dlo) & (tiles.high == dlo))); };
    auto visit = [&](auto mask) {
        const int j0 = t * ATTN_TILE, now = buf;
        attn_sync();
        t = tiles.next(lane);
        buf ^= 1;
        if (t >= 0) stage(t, buf);
        if (!mask.value || j0 <= lim_last) {
            const uint32_t k_lds = at_lane.rows(lds + now * 2 * TILE_BYTES), v_lds = at_lane.cols(lds + now * 2 * TILE_BYTES + TILE_BYTES);
            // every fragment is on its way before the first product that needs one: keys ahead of the scores, values ahead of the softmax
            typename AttnVec<T>::x8 kf[2][2 * DB], vf[DB][2][2], P[2][2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int c = 0; c < 2 * DB; ++c) kf[kb][c] = attn_row_frag<T, ROW>(k_lds, kb, c);
            __builtin_amdgcn_sched_barrier(0);
            f32x16 S[2] = {};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int c = 0; c < 2 * DB; ++c) S[kb] = attn_mfma(kf[kb][c], qf[c], S[kb]);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int c = 0; c < 2; ++c) vf[db][kb][c] = attn_col_frag<T, ROW>(v_lds, 2 * kb + c, db);
            __builtin_amdgcn_sched_barrier(0);
            attn_softmax_form<T, 2, DB, MODE, mask.value>(S, P, acc, m, sum, f, lim, i + n - p.Lq, j0, half, DOCS ? sdoc[now] : nullptr, qdoc);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int db = 0; db < DB; ++db) acc[db] = attn_mfma(vf[db][kb][c], P[kb][c], acc[db]);
            if constexpr (mask.value)
                if (fine) {                                             // (attn_left_over)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const typename AttnVec<T>::x8 left = attn_left_over<T>(S[kb], P[kb][c], c);
#pragma unroll
                            for (int db = 0; db < DB; ++db) acc[db] = attn_mfma(vf[db][kb][c], left, acc[db]);
                        }
                }
        }
        if (DOCS && wave == 0) sdoc[buf][lane] = doc_next;
    };
    // (two loops, not one with a branch inside: the accumulators keep their registers)
    while (t >= 0) {
        while (t >= 0 && full()) visit(std::false_type());
        while (t >= 0 && !full()) visit(std::true_type());
    }
    sum = attn_half_sum(sum);
    bool store = row_ok;
    if (attn_any(attn_has_nan(acc) && sum == sum && row_ok, wave, said)) {
        attn_rows_again<T, DB>(attn_kernel_args(), b, i, h, row_ok, split, run_first * ATTN_TILE, min(key_end, run_end * ATTN_TILE), lds + wave * TILE_BYTES, fine);
        attn_clear(acc);                                                // (stored there; a return would keep the sums across the call)
        store = false;
    }
    attn_fwd_store<T, DB>(p, acc, m, sum, b, i, h, split, half, store);
#endif
}

// ---- few queries: rows r = query * G + head of the group, 32 a workgroup
template <typename T, int DB, int MODE>
__global__ __launch_bounds__(256, DB < 3 ? 3 : 2) void attn_token_kernel(AttnParams p) {
#ifdef __HIP_DEVICE_COMPILE__                            // (hipcc drops the launch stub of a template whose body its host pass cannot read)
    constexpr int ROW = DB > 2 ? 128 : 64, KEYS = 32, TILE_BYTES = KEYS * ROW * 2, WAVES = 4;
    extern __shared__ __align__(1024) char smem[];                        // [wave][buffer][k, v], then the waves' results
    __shared__ float sm[WAVES][32], ssum[WAVES][32];
    __shared__ __align__(16) int sdoc[WAVES][2][KEYS];
    const int wave = attn_uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
    const int split = blockIdx.x % p.splits, blk = blockIdx.x / p.splits % p.row_blocks, bh = blockIdx.x / (p.splits * p.row_blocks);
    const int hk = bh % p.Hk, b = bh / p.Hk, rows = p.Lq * p.G;
    const int n = attn_keys(p, b), prefix = attn_prefix(p, b);
    const int r = blk * 32 + l31, i = r / p.G, h = hk * p.G + r - i * p.G;
    const bool row_ok = r < rows;
    const int qdoc = p.kdoc && row_ok ? p.qdoc[b * p.qdoc_stride + i] : 0;
    const int lim = !row_ok || qdoc < 0 ? -1 : attn_limit(p, i, n, prefix);
    const int lim_first = attn_limit(p, blk * 32 / p.G, n, prefix), lim_last = attn_limit(p, min(blk * 32 + 31, rows - 1) / p.G, n, prefix);
    // this workgroup's share of the keys, in whole rounds of the four waves' tiles
    const int rounds = (lim_last + WAVES * KEYS) / (WAVES * KEYS), per = (rounds + p.splits - 1) / p.splits;
    const int k0 = split * per * WAVES * KEYS, k1 = min(lim_last + 1, (split + 1) * per * WAVES * KEYS);
    typename AttnVec<T>::x8 qf[2 * DB];
    const T* q = row_ok ? (const T*)p.q + b * p.qs[0] + i * p.qs[1] + h * p.qs[2] : nullptr;
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c) qf[c] = attn_lane_frag<T>(q, 2 * c + half, p.D);
    const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[2];
    const T* v = (const T*)p.v + b * p.vs[0] + hk * p.vs[2];
    const int* kdoc = p.kdoc ? p.kdoc + b * p.kdoc_stride : nullptr;
    AttnScore f(p, row_ok ? h : hk * p.G);
    AttnStage<ROW, KEYS, 1> sk, sv;
    sk.setup(0, lane, p.ks[1], p.D);
    sv.setup(0, lane, p.vs[1], p.D);
    char* mine = smem + wave * 4 * TILE_BYTES;
    const uint64_t k_at = attn_addr(k), v_at = attn_addr(v);
    const int k_row = (int)p.ks[1], v_row = (int)p.vs[1];
    const AttnLane<ROW> at_lane(lane);
    const uint32_t lds = attn_lds(mine);
    int doc_next = 0;
    auto stage = [&](int j0, int buf) {
        if (kdoc && lane < KEYS) doc_next = kdoc[min(j0 + lane, p.Lk - 1)];
        sk.issue(k_at, j0 / KEYS, n, k_row, p.D, lds + buf * 2 * TILE_BYTES, 0);
        sv.issue(v_at, j0 / KEYS, n, v_row, p.D, lds + buf * 2 * TILE_BYTES + TILE_BYTES, 0);
    };
    f32x16 acc[DB] = {};
    float m = -INFINITY, sum = 0.f;
    int j0 = k0 + wave * KEYS;
    if (j0 < k1) stage(j0, 0);
    if (kdoc && lane < KEYS) sdoc[wave][0][lane] = doc_next;
    for (int buf = 0; j0 < k1; buf ^= 1, j0 += WAVES * KEYS) {
        asm volatile("" ::: "memory");
        attn_landed();                                                  // the wave's own pieces: no other wave touches this LDS
        if (j0 + WAVES * KEYS < k1) stage(j0 + WAVES * KEYS, buf ^ 1);
        const uint32_t k_lds = at_lane.rows(lds + buf * 2 * TILE_BYTES), v_lds = at_lane.cols(lds + buf * 2 * TILE_BYTES + TILE_BYTES);
        f32x16 S[1] = {};
#pragma unroll
        for (int c = 0; c < 2 * DB; ++c) S[0] = attn_mfma(attn_row_frag<T, ROW>(k_lds, 0, c), qf[c], S[0]);
        const bool full = j0 + KEYS - 1 <= lim_first && !kdoc;
        typename AttnVec<T>::x8 P[1][2];
        attn_softmax_step<T, 1, DB, MODE>(S, P, acc, m, sum, f, full, lim, i + n - p.Lq, j0, half, kdoc ? sdoc[wave][buf] : nullptr, qdoc);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int c = 0; c < 2; ++c) acc[db] = attn_mfma(attn_col_frag<T, ROW>(v_lds, c, db), P[0][c], acc[db]);
        // what rounding the weights left over, in a second product (attn_left_over): free here, where the keys' bytes bound the call (the one above 154 us with
        // it and without, errors of the norm 1.66e-3, the output's own rounding, instead of 2.34e-3)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const typename AttnVec<T>::x8 left = attn_left_over<T>(S[0], P[0][c], c);
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] = attn_mfma(attn_col_frag<T, ROW>(v_lds, c, db), left, acc[db]);
        }
        if (kdoc && lane < KEYS) sdoc[wave][buf ^ 1][lane] = doc_next;
    }
    // join the four waves: common maximum, then the accumulators through the LDS, one [32 rows][32 * DB + 1] float image a wave
    constexpr int PITCH = 32 * DB + 1;
    __shared__ uint32_t said[WAVES];
    sum = attn_half_sum(sum);
    if (attn_any(attn_has_nan(acc) && sum == sum && row_ok, wave, said)) {
        const AttnSums<DB> s = attn_out_again<T, DB>(attn_kernel_args(), b, i, h, row_ok, k0 + wave * KEYS, k1, WAVES * KEYS, lds);
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = s.acc[db];
        m = s.m;
        sum = s.sum;
    }
    if (half == 0) {
        sm[wave][l31] = m;
        ssum[wave][l31] = sum;
    }
    __syncthreads();                                                    // (also: every wave is done with its tiles)
    float top = -INFINITY, all = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, sm[w][l31]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all += ssum[w][l31] == 0.f ? 0.f : ssum[w][l31] * __builtin_amdgcn_exp2f(sm[w][l31] - top);
    const float shrink = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    float* img = reinterpret_cast<float*>(smem) + wave * 32 * PITCH;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int rr = 0; rr < 16; ++rr) img[l31 * PITCH + 32 * db + 8 * (rr >> 2) + 4 * half + (rr & 3)] = m == -INFINITY ? 0.f : acc[db][rr] * shrink;
    __syncthreads();
    const bool direct = p.splits == 1;
    for (int e = wave * 8; e < wave * 8 + 8; ++e) {                     // eight rows a wave
        const int re = blk * 32 + e;
        if (re >= rows) break;
        const int ie = re / p.G, he = hk * p.G + re - ie * p.G;
        const float te = __shfl(top, e), ae = __shfl(all, e);
        float x[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 2; ++c)
            if (lane + 64 * c < 32 * DB)
#pragma unroll
                for (int w = 0; w < WAVES; ++w) x[c] += reinterpret_cast<float*>(smem)[(w * 32 + e) * PITCH + lane + 64 * c];
        if (direct) {
            attn_store_pair<T>(p, ((int64_t)(b * (int64_t)p.Lq + ie) * p.Hq + he) * p.D, x, ae == 0.f ? 0.f : 1.f / ae, lane);
            if (p.lse && lane == 0) p.lse[((int64_t)b * p.Hq + he) * p.Lq + ie] = ae == 0.f ? -INFINITY : (te + __builtin_amdgcn_logf(ae)) * ATTN_LN2;
        } else {
            const int64_t at = (int64_t)(bh * (int64_t)rows + re) * p.splits + split;
            if (lane < p.D) p.part[at * p.D + lane] = x[0];
            if (lane + 64 < p.D) p.part[at * p.D + lane + 64] = x[1];
            if (lane == 0) {
                p.part[p.part_ml + 2 * at] = te;
                p.part[p.part_ml + 2 * at + 1] = ae;
            }
        }
    }
#endif
}

// the splits' accumulators, in order: four channels a lane, 32 lanes a row (16 up to 64 channels), no lane waits for another
__device__ __host__ __forceinline__ int attn_combine_lanes(int D) { return D > 64 ? 32 : 16; }
template <typename T>
__global__ __launch_bounds__(256) void attn_combine_kernel(AttnParams p) {
    const int rows = p.Lq * p.G, lanes = attn_combine_lanes(p.D), d = 4 * (threadIdx.x & (lanes - 1));
    const int64_t w = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    if (w >= (int64_t)p.B * p.Hk * rows || d >= p.D) return;
    const int r = (int)(w % rows), bh = (int)(w / rows), hk = bh % p.Hk, b = bh / p.Hk, i = r / p.G, h = hk * p.G + r - i * p.G;
    const float2* ml = reinterpret_cast<const float2*>(p.part + p.part_ml) + w * p.splits;
    const float* a = p.part + w * p.splits * p.D + d;
    float top = -INFINITY;
#pragma unroll 8
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, ml[s].x);
    float all = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < p.splits; ++s) {
        const float2 st = ml[s];
        const float4 v = *reinterpret_cast<const float4*>(a + (int64_t)s * p.D);
        const float by = st.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(st.x - top);      // (0: nothing visible in this share, whose accumulator is zero)
        all += by * st.y;
        x[0] += by * v.x; x[1] += by * v.y; x[2] += by * v.z; x[3] += by * v.w;
    }
    const float scale = all == 0.f ? 0.f : 1.f / all;
    const int64_t at = ((int64_t)(b * (int64_t)p.Lq + i) * p.Hq + h) * p.D + d;
    typename AttnVec<T>::x4 o, rest;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        o[e] = (T)(x[e] * scale);
        rest[e] = (T)(x[e] * scale - (float)(T)(x[e] * scale));
    }
    *reinterpret_cast<typename AttnVec<T>::x4*>((T*)p.out + at) = o;
    if (p.rest) *reinterpret_cast<typename AttnVec<T>::x4*>((T*)p.rest + at) = rest;
    if (p.lse && d == 0) p.lse[((int64_t)b * p.Hq + h) * p.Lq + i] = all == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(all)) * ATTN_LN2;
}

void attn_ranges(AttnParams& p, void* workspace, hipStream_t stream) {
    if (!p.kdoc) return;
    int2* kt = (int2*)workspace;
    int2* qt = kt + (int64_t)p.B * p.nkt;
    if (p.nkt) hipLaunchKernelGGL(attn_ranges_kernel, dim3(cdiv(p.nkt, 4) * p.B), dim3(256), 0, stream, p.kdoc, p.kdoc_stride, p.Lk, p.nkt, kt);
    if (p.qdoc == p.kdoc && p.qdoc_stride == p.kdoc_stride && p.Lq == p.Lk) qt = kt;
    else hipLaunchKernelGGL(attn_ranges_kernel, dim3(cdiv(p.nqt, 4) * p.B), dim3(256), 0, stream, p.qdoc, p.qdoc_stride, p.Lq, p.nqt, qt);
    p.ktiles = kt;
    p.qtiles = qt;
    p.row_blocks = cdiv(p.Lq, 128);
    if (p.nkt > ATTN_ORDER_TILES || p.row_blocks > ATTN_ORDER_BLOCKS || (int64_t)p.B * p.Hq * p.row_blocks <= 1024 || !n3d_grid_fits(p.B, 1024)) return;
    int* order = (int*)(kt + (int64_t)p.B * (p.nkt + p.nqt));
    hipLaunchKernelGGL(attn_order_kernel, dim3(p.B), dim3(1024), 0, stream, p, order);
    p.order = order;
}

// The token kernel up to 24 queries, or where its rows (queries x heads of a group) fill two 32-row blocks at most; its keys go to enough workgroups to fill
// the chip twice.  (Single tokens aside, against the kernel of 128 queries: 5 queries x 16 heads a group over 8192 keys 34 us against 60, 16 x 16 over 4096
// 134 / 203, 24 x 8 over 2048 97 / 111; but 32 x 16 over 8192 39 / 37, 32 x 3 over 512 14 / 10, 100 x 1 over 4096 23 / 16.  512 workgroups: the call above
// 153 us, with 256 156, with 1024 157.  256 keys a workgroup: one token of 8 heads over 4096 12.4 us, with 128 12.6, with 1024 19.2.)
static bool attn_plan(AttnParams& p) {
    const int64_t rows = (int64_t)p.Lq * p.G;
    if (rows > 64 && p.Lq > 24) {
        p.row_blocks = cdiv(p.Lq, 128);
        p.splits = attn_room((int64_t)p.B * p.Hq * p.row_blocks, p.nkt);
        return false;
    }
    p.row_blocks = (int)cdiv64(rows, 32);
    const int64_t groups = (int64_t)p.B * p.Hk * p.row_blocks;
    int64_t s = 512 / groups, most = cdiv64(p.Lk, 256);                 // (256 keys: two rounds of the four waves)
    if (s > most) s = most;
    p.splits = s < 1 ? 1 : s > 64 ? 64 : (int)s;
    return true;
}

template <typename T, int DB, int MODE, bool DOCS>
static hipError_t attn_fwd_launch(AttnParams& p, bool token, hipStream_t stream) {
    if (token) {
        constexpr int lds = 4 * 4 * 32 * (DB > 2 ? 128 : 64) * 2;
        const hipError_t e = hipFuncSetAttribute((const void*)attn_token_kernel<T, DB, MODE>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL((attn_token_kernel<T, DB, MODE>), dim3(p.B * p.Hk * p.row_blocks * p.splits), dim3(256), lds, stream, p);
    } else {
        hipLaunchKernelGGL((attn_fwd_kernel<T, DB, MODE, DOCS>), dim3((unsigned)attn_even((int64_t)p.B * p.Hq * p.splits * p.row_blocks)), dim3(256), 0, stream, p);
    }
    if (p.splits > 1) hipLaunchKernelGGL((attn_combine_kernel<T>), dim3((unsigned)cdiv64((int64_t)p.B * p.Lq * p.Hq, 256 / attn_combine_lanes(p.D))), dim3(256), 0, stream, p);
    return hipSuccess;
}

// floats of the workspace; parts_at: where the splits' parts lie in it (behind the document ranges)
static int64_t attn_fwd_floats(AttnParams& p, bool& token, int64_t& parts_at) {
    parts_at = (attn_range_floats(p) + 3) / 4 * 4;
    token = attn_plan(p);
    if (p.splits == 1) return attn_range_floats(p);
    const int64_t parts = (int64_t)p.B * p.Hq * p.Lq * p.splits;
    p.part_ml = parts * p.D;
    return parts_at + parts * (p.D + 2);
}

static bool attn_fwd_fits(const AttnParams& p, bool token) {
    const int64_t groups = (int64_t)p.B * p.row_blocks * p.splits;
    return token ? n3d_grid_fits(groups * p.Hk, 256) : n3d_grid_fits(attn_even(groups * p.Hq), 256) && attn_ranges_fit(p);
}

extern "C" int64_t n3d_attention_workspace(const n3d_attention_desc* d) {
    AttnParams p;
    const char* bad = attn_params(d, p);
    N3D_CHECK(!bad, "attention: %s", bad);
    if (p.B == 0 || p.Lq == 0) return 0;
    bool token;
    int64_t parts_at;
    const int64_t need = 4 * attn_fwd_floats(p, token, parts_at);
    N3D_CHECK(attn_fwd_fits(p, token), "attention: too many rows for one launch");
    return need;
}

extern "C" int n3d_attention(const n3d_attention_desc* d, n3d_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    AttnParams p;
    const char* bad = attn_params(d, p);
    N3D_CHECK(!bad, "attention: %s", bad);
    if (p.B == 0 || p.Lq == 0) return 0;
    bool token;
    int64_t parts_at;
    const int64_t need = 4 * attn_fwd_floats(p, token, parts_at);
    N3D_CHECK(attn_fwd_fits(p, token), "attention: too many rows for one launch");
    N3D_CHECK(need == 0 || (d->workspace && d->workspace_bytes >= need && (uintptr_t)d->workspace % 16 == 0), "attention: a workspace of %lld bytes is needed (16-byte aligned)",
              (long long)need);
    const double pairs = (double)p.B * p.Hq * p.Lq * p.Lk * p.D;
    N3dProfScope prof(N3D_K_ATTENTION, stream, 4.0 * pairs, 4.0 * ((double)p.B * p.Lq * p.Hq * p.D + (double)p.B * p.Lk * p.Hk * p.D));
    if (!token) attn_ranges(p, d->workspace, stream);
    p.part = (float*)d->workspace + parts_at;
    hipError_t e = hipSuccess;
    if (d->dtype == N3D_F16) attn_forms(p, [&](auto db, auto mode, auto docs) { e = attn_fwd_launch<_Float16, db.value, mode.value, docs.value>(p, token, stream); });
    else attn_forms(p, [&](auto db, auto mode, auto docs) { e = attn_fwd_launch<__bf16, db.value, mode.value, docs.value>(p, token, stream); });
    N3D_CHECK(e == hipSuccess, "attention: %s", hipGetErrorString(e));
    N3D_LAUNCH_CHECK();
    return 0;
}
