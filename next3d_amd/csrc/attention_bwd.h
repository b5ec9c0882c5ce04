// Attention, backward (attention.h):  P = exp2(u - lse),  dP = do v^T,  delta = sum(do o),  dt = P (dP - delta),  ds = dt (1 - tanh^2),
//   dq = scale ds k,   dk = scale ds^T q,   dv = P^T do,   dk and dv summed over the query heads of a key head.
// attn_prep_kernel: delta.
// attn_dq_kernel: a workgroup owns 128 queries of a head and walks the keys;  attn_dkv_kernel: a workgroup owns 128 keys of a key head and walks the
// queries of all its heads.  Scores are computed in both (7 products for 5) so that every sum has one owner: no atomics, the same bits every time.
// Measured, 4096 x 16 heads x 128 bfloat16 without a mask, medians of 60 launches: prep 10 us, dq 188 us (1.10 PFLOP/s of its three products), dk / dv 301 us
// (0.91 of its four); x 64 float16: 7 us and 314 us for both.  The matrix pipe is busy for 58 % (dq) and 42 % (dk / dv, whose waves also trade weights and
// wait for each other twice a tile); the rest is the same vector work as in the forward pass, here without a running maximum.
#pragma once
#include "attention.h"

// float16 has 5 exponent bits, and P ~ 1 / length and ds ~ P do v leave its range on long rows or with small gradients (bfloat16 has float32's exponents).
// The dk / dv kernel therefore uses P 2^12, and both kernels ds 2^e with an e of the lane's own — a query's in dq, a key's in dk / dv — found like the running
// maximum of a softmax: e begins high, and where a visible ds 2^e reaches 2 it is lowered until the largest is 1/4 to 1/2, and the accumulators with it.  So
// dscores of any size are rounded by half a step of their own, or, below 2^-12 of the lane's largest, by 2^-23 of that; what a lane does not see has no say.
template <typename T> static constexpr float ATTN_P_SHIFT = std::is_same<T, _Float16>::value ? 12.f : 0.f;
static constexpr int ATTN_DS_EXP = 64;                        // (|P dP| < 2^41 in float16: 2^64 of it is a float32)

template <typename T>
__global__ __launch_bounds__(256) void attn_prep_kernel(AttnParams p) {
    // 16 lanes a row, 8 channels a lane
    const int lane16 = threadIdx.x & 15, D = p.D;
    const uint32_t rows = (uint32_t)p.B * p.Lq * p.Hq;                    // (below 2^31: n3d_attention_bwd)
    for (uint32_t w = blockIdx.x * 16 + (threadIdx.x >> 4); w < rows; w += gridDim.x * 16) {
        const uint32_t bi = w / p.Hq;
        const int h = w - bi * p.Hq, b = bi / p.Lq, i = bi - b * p.Lq;
        float s = 0.f;
        if (lane16 * 8 < D) {
            const auto x = *reinterpret_cast<const typename AttnVec<T>::x8*>((const T*)p.dout + b * p.ds[0] + i * p.ds[1] + h * p.ds[2] + lane16 * 8);
            const auto y = *reinterpret_cast<const typename AttnVec<T>::x8*>((const T*)p.o + (int64_t)w * D + lane16 * 8);
            typename AttnVec<T>::x8 z = {};
            if (p.rest) z = *reinterpret_cast<const typename AttnVec<T>::x8*>((const T*)p.rest + (int64_t)w * D + lane16 * 8);
#pragma unroll
            for (int e = 0; e < 8; ++e) s += (float)x[e] * ((float)y[e] + (float)z[e]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (lane16 == 0) p.delta[((int64_t)b * p.Hq + h) * p.Lq + i] = s;
    }
}

template <typename T>
__device__ __forceinline__ void attn_pack(const f32x16& x, typename AttnVec<T>::x8 (&out)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) out[c][e] = (T)x[8 * c + e];
}

// This wave's 32 x 32 block of ds 2^e, to be rounded to float16: where a column's largest reaches 2, e falls, and the block and the column's accumulators with
// it.  (Infinities and NaN pass: the result is one of them.)  2 is the number from which on the first bit of a float's exponent is set: a block without such a
// column pays for eight or's and a ballot.  (Against one exponent for the whole call, training steps of 2 x 4096 causal, 16 heads on 4 x 32, 64, 128: 409 ->
// 415, 513 -> 511, 781 -> 791 us; looking at the 16 maxima instead: 449, 523, 799.)
template <int NB>
__device__ __forceinline__ void attn_fit(f32x16& ds, int& e, f32x16 (&acc)[NB]) {
    uint32_t bits = 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) bits |= __builtin_bit_cast(uint32_t, (float)ds[r]);
    if (__ballot((bits & 0x40000000u) != 0)) {
        float top = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(ds[r]));
        top = attn_half_max(top);                                         // (a column's queries or keys are in both halves)
        const int by = top >= 2.f && top < INFINITY ? ilogbf(top) + 2 : 0;
        const float shrink = ldexpf(1.f, -by);
        e -= by;
#pragma unroll
        for (int r = 0; r < 16; ++r) ds[r] *= shrink;
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][r] *= shrink;
    }
}

// Raw score and dP of one element -> P 2^shift (in lse2) and, times ds_by, ds (SCALED false: ds_by is 1)
template <int MODE, bool SCALED>
__device__ __forceinline__ void attn_ds(f32x16& S, f32x16& dP, int r, const AttnScore& f, float ds_by, float lse2, float delta, float dist) {
    float u, d = dP[r] - delta;
    if constexpr (MODE == ATTN_CAP || MODE == ATTN_CAP_BIAS) {
        const float x = f.cap_r(S[r]);
        u = f.capped(x, lse2);
        d *= __builtin_fmaf(-x, x, x);                       // a quarter of 1 - tanh^2: attn_ds_unit
    } else {
        u = __builtin_fmaf(S[r], f.mul, -lse2);
    }
    if constexpr (MODE == ATTN_BIAS || MODE == ATTN_CAP_BIAS) u -= f.slope * fabsf(dist);
    S[r] = __builtin_amdgcn_exp2f(u);
    if constexpr (SCALED) d *= ds_by;
    dP[r] = S[r] * d;
}
template <int MODE> static constexpr float attn_ds_unit() { return MODE == ATTN_CAP || MODE == ATTN_CAP_BIAS ? 4.f : 1.f; }

__device__ __forceinline__ float attn_lse2(float lse) { return lse == -INFINITY ? INFINITY : lse * ATTN_LOG2E; }       // (a row that sees nothing: every weight 0)

template <int DB> static constexpr bool attn_dkv_pair() { return DB > 3; }      // (see attn_dkv)
// waves a SIMD that the registers of these kernels, and of what they call, leave room for (256 threads; pairs: one workgroup of 512 a CU)
template <int DB, bool DOCS> static constexpr int attn_dq_waves() { return DB < 2 || (DB < 3 && !DOCS) ? 3 : 2; }
template <int DB> static constexpr int attn_dkv_waves() { return DB < 2 ? 3 : 2; }
// what both kinds of workgroups keep in the LDS
template <int DB> static constexpr int attn_row() { return DB > 2 ? 128 : 64; }
template <int DB> static constexpr int attn_lds_bytes() { return 4 * ATTN_TILE * attn_row<DB>() * 2; }
struct AttnRows {
    float lse[2][ATTN_TILE], delta[2][ATTN_TILE];
};

#ifdef __HIP_DEVICE_COMPILE__                            // (hipcc drops the launch stub of a template whose body its host pass cannot read)
// P 2^shift (in lse2) and ds 2^e / scale (in ds_by) of one pair from its raw products, in any form of the scores
__device__ __forceinline__ void attn_pair(const AttnScore& f, float s, float dp, float lse2, float delta, float ds_by, float dist, float& w, float& ds) {
    const float x = f.cap_out > 0.f ? f.cap_r(s) : 0.5f;
    w = __builtin_amdgcn_exp2f(attn_score(f, s, dist) - lse2);
    ds = w * ((dp - delta) * ds_by * 4.f * __builtin_fmaf(-x, x, x));
}
template <typename T, int DB>
__device__ __forceinline__ void attn_dq_store(const AttnParams& p, const f32x16 (&acc)[DB], float unit, int ds_exp, int b, int i, int h, int split, int half, bool row_ok) {
    const float by = ldexpf(p.scale * unit, -ds_exp);
    const int64_t row_at = ((int64_t)(b * (int64_t)p.Lq + i) * p.Hq + h) * p.D, all = (int64_t)p.B * p.Lq * p.Hq * p.D;
    if (p.splits > 1) attn_store_part<DB>(p.part + split * all + row_at, acc, by, half, p.D, row_ok);
    else attn_store_row<T, DB>((T*)p.dq + row_at, acc, by, half, p.D, row_ok);
}
// NB blocks of channels from 64 part on
template <typename T, int NB>
__device__ __forceinline__ void attn_dkv_store(const AttnParams& p, const f32x16 (&dk)[NB], const f32x16 (&dv)[NB], float unit, int ds_exp, int b, int j, int hk, int split, int part, int half, bool store) {
    const float k_by = ldexpf(p.scale * unit, -ds_exp), v_by = ldexpf(1.f, -(int)ATTN_P_SHIFT<T>);
    const int64_t row = ((int64_t)b * p.Lk + j) * p.Hk + hk, all = (int64_t)p.B * p.Lk * p.Hk;
    if (p.k_splits > 1) {
        float* pk = p.k_part + (2 * split * all + row) * p.D;
        float* pv = p.k_part + ((2 * split + 1) * all + row) * p.D;
        attn_store_part<NB>(pk + 64 * part, dk, k_by, half, p.D - 64 * part, store);
        attn_store_part<NB>(pv + 64 * part, dv, v_by, half, p.D - 64 * part, store);
    } else {
        attn_store_row<T, NB>((T*)p.dk + row * p.D + 64 * part, dk, k_by, half, p.D - 64 * part, store);
        attn_store_row<T, NB>((T*)p.dv + row * p.D + 64 * part, dv, v_by, half, p.D - 64 * part, store);
    }
}
// A wave's sums once more (attention.h: infinities and NaN).  WAVES (a SIMD's) keeps the copies of kernels with different registers apart.
// dq of 32 queries over the keys [first, end)
template <typename T, int DB, int WAVES>
static __device__ __attribute__((noinline)) void attn_dq_again(attn_args args, int b, int i, int h, bool row_ok, int split, int first, int end, uint32_t lds) {
    constexpr int ROW = attn_row<DB>(), KEYS = 32, BYTES = KEYS * ROW * 2;
    constexpr bool FIT = ATTN_P_SHIFT<T> != 0.f;
    const AttnParams p = *args;
    const int lane = threadIdx.x & 63, half = lane >> 5, hk = attn_uniform(h / p.G);
    const int n = attn_keys(p, b), at = i + n - p.Lq;
    const int qdoc = p.kdoc && row_ok ? p.qdoc[b * p.qdoc_stride + i] : 0;
    const int lim = !row_ok || qdoc < 0 ? -1 : attn_limit(p, i, n, attn_prefix(p, b));
    const T* q = row_ok ? (const T*)p.q + b * p.qs[0] + i * p.qs[1] + h * p.qs[2] : nullptr;
    const T* dout = row_ok ? (const T*)p.dout + b * p.ds[0] + i * p.ds[1] + h * p.ds[2] : nullptr;
    const int64_t stat = ((int64_t)b * p.Hq + h) * p.Lq + i;
    const float lse2 = row_ok ? attn_lse2(p.lse[stat]) : INFINITY, delta = row_ok ? p.delta[stat] : 0.f;
    const uint64_t k = attn_addr((const T*)p.k + b * p.ks[0] + hk * p.ks[2]), v = attn_addr((const T*)p.v + b * p.vs[0] + hk * p.vs[2]);
    const AttnScore f(p, h);
    AttnStage<ROW, KEYS, 1> sk, sv;
    sk.setup(0, lane, p.ks[1], p.D);
    sv.setup(0, lane, p.vs[1], p.D);
    const AttnLane<ROW> at_lane(lane);
    struct {
        f32x16 dk[DB];
        int ds_exp;
    } g;
    AttnMarks<DB> either;                                               // (an infinity of a key too: its pair's score is not finite then, and ds 0 or NaN)
#pragma unroll 1
    for (int walk = 0; walk < 2; ++walk) {
        const int kind = walk == 0 ? ATTN_EITHER : ATTN_FINITE;
#pragma unroll
        for (int db = 0; db < DB; ++db) g.dk[db] = f32x16{};
        g.ds_exp = FIT ? ATTN_DS_EXP : 0;
#pragma unroll 1
        for (int j0 = first; j0 < end; j0 += KEYS) {
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
            typename AttnVec<T>::x8 d[2];
            if (kind == ATTN_FINITE) {
                const uint32_t k_lds = at_lane.rows(lds), v_lds = at_lane.rows(lds + BYTES);
                f32x16 S = {}, dP = {};
#pragma unroll
                for (int c = 0; c < 2 * DB; ++c) S = attn_mfma(attn_row_frag<T, ROW>(k_lds, 0, c), attn_lane_frag<T>(q, 2 * c + half, p.D), S);
#pragma unroll
                for (int c = 0; c < 2 * DB; ++c) dP = attn_mfma(attn_row_frag<T, ROW>(v_lds, 0, c), attn_lane_frag<T>(dout, 2 * c + half, p.D), dP);
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float w, ds;
                    attn_pair(f, S[r], dP[r], lse2 - (float)g.ds_exp, delta, 1.f, (float)(at - (j0 + 4 * half + 8 * (r >> 2) + (r & 3))), w, ds);
                    dP[r] = seen >> r & 1 ? ds : 0.f;
                }
                if constexpr (FIT) attn_fit(dP, g.ds_exp, g.dk);
                attn_pack<T>(dP, d);
            } else {
                attn_ones<T>(seen, d);
            }
            attn_landed();
            attn_change<T, BYTES>(lds, lane, kind);
            attn_landed();
            const uint32_t kc_lds = at_lane.cols(lds);
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int c = 0; c < 2; ++c) g.dk[db] = attn_mfma(attn_col_frag<T, ROW>(kc_lds, c, db), d[c], g.dk[db]);
        }
        if (walk == 0) either.take(g.dk);
    }
    either.add(g.dk, NAN);
    attn_dq_store<T, DB>(p, g.dk, 1.f, g.ds_exp, b, i, h, split, half, row_ok);
}
// dk and dv of 32 keys, NB blocks of channels from 32 NB part on, over the queries [first, end) of the heads [g0, g1) of their group
template <typename T, int DB, int NB, int WAVES>
static __device__ __attribute__((noinline)) void attn_dkv_again(attn_args args, int b, int hk, int j, int kdoc, int split, int g0, int g1, int first, int end, int part, uint32_t lds) {
    constexpr int ROW = attn_row<DB>(), ROWS = 32, BYTES = ROWS * ROW * 2;
    constexpr float SHIFT = ATTN_P_SHIFT<T>;
    constexpr bool FIT = SHIFT != 0.f;
    const AttnParams p = *args;
    const int lane = threadIdx.x & 63, half = lane >> 5, n = attn_keys(p, b), off = n - p.Lq;
    const bool key_ok = j < n && kdoc >= 0;
    const int qmin = !key_ok ? 0x7fffffff : !p.causal || j < attn_prefix(p, b) ? 0 : max(j - off, 0);
    const T* k = j < n ? (const T*)p.k + b * p.ks[0] + j * p.ks[1] + hk * p.ks[2] : nullptr;
    const T* v = j < n ? (const T*)p.v + b * p.vs[0] + j * p.vs[1] + hk * p.vs[2] : nullptr;
    AttnStage<ROW, ROWS, 1> sq, sd;
    sq.setup(0, lane, p.qs[1], p.D);
    sd.setup(0, lane, p.ds[1], p.D);
    const AttnLane<ROW> at_lane(lane);
    struct {
        f32x16 dk[NB], dv[NB];
        int ds_exp;
    } g;
    AttnMarks<NB> either, plus, minus;                                  // (an infinity of a query: as a key's in attn_dq_again)
#pragma unroll 1
    for (int walk = 0; walk < 3; ++walk) {
        const int kind = walk == 0 ? ATTN_PLUS : walk == 1 ? ATTN_MINUS : ATTN_FINITE;
#pragma unroll
        for (int db = 0; db < NB; ++db) g.dk[db] = g.dv[db] = f32x16{};
        g.ds_exp = FIT ? ATTN_DS_EXP : 0;
#pragma unroll 1
        for (int gh = g0; gh < g1; ++gh) {
            const int h = hk * p.G + gh;
            const AttnScore f(p, h);
            const uint64_t q = attn_addr((const T*)p.q + b * p.qs[0] + h * p.qs[2]), dout = attn_addr((const T*)p.dout + b * p.ds[0] + h * p.ds[2]);
            const int64_t stat = ((int64_t)b * p.Hq + h) * p.Lq;
#pragma unroll 1
            for (int i0 = first; i0 < end; i0 += ROWS) {
                uint32_t seen = 0;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int i = i0 + 4 * half + 8 * (r >> 2) + (r & 3);
                    if (i >= qmin && i < p.Lq && (!p.kdoc || p.qdoc[b * p.qdoc_stride + i] == kdoc)) seen |= 1u << r;
                }
                if (!__ballot(seen != 0)) continue;
                attn_landed();                                          // (the LDS reads of the tile before)
                sq.issue(q, i0 / ROWS, p.Lq, (int)p.qs[1], p.D, lds, 0);
                sd.issue(dout, i0 / ROWS, p.Lq, (int)p.ds[1], p.D, lds + BYTES, 0);
                attn_landed();
                typename AttnVec<T>::x8 w[2], d[2];
                if (kind == ATTN_FINITE) {
                    const uint32_t q_lds = at_lane.rows(lds), d_lds = at_lane.rows(lds + BYTES);
                    f32x16 S = {}, dP = {};
#pragma unroll
                    for (int c = 0; c < 2 * DB; ++c) S = attn_mfma(attn_row_frag<T, ROW>(q_lds, 0, c), attn_lane_frag<T>(k, 2 * c + half, p.D), S);
#pragma unroll
                    for (int c = 0; c < 2 * DB; ++c) dP = attn_mfma(attn_row_frag<T, ROW>(d_lds, 0, c), attn_lane_frag<T>(v, 2 * c + half, p.D), dP);
                    const float ds_by = FIT ? ldexpf(1.f, g.ds_exp - (int)SHIFT) : 1.f;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int i = i0 + 4 * half + 8 * (r >> 2) + (r & 3), row = min(i, p.Lq - 1);
                        float weight, ds;
                        attn_pair(f, S[r], dP[r], attn_lse2(p.lse[stat + row]) - SHIFT, p.delta[stat + row], ds_by, (float)(i + off - j), weight, ds);
                        S[r] = seen >> r & 1 ? weight : 0.f;
                        dP[r] = seen >> r & 1 ? ds : 0.f;
                    }
                    if constexpr (FIT) attn_fit(dP, g.ds_exp, g.dk);
                    attn_pack<T>(S, w);
                    attn_pack<T>(dP, d);
                } else {
                    attn_ones<T>(seen, w);
                    attn_ones<T>(seen, d);
                }
                attn_landed();
                attn_change<T, BYTES>(lds, lane, kind == ATTN_FINITE ? ATTN_FINITE : ATTN_EITHER);
                attn_change<T, BYTES>(lds + BYTES, lane, kind);
                attn_landed();
                const uint32_t qc_lds = at_lane.cols(lds) ^ (part << 7), dc_lds = at_lane.cols(lds + BYTES) ^ (part << 7);
#pragma unroll
                for (int db = 0; db < NB; ++db)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        g.dv[db] = attn_mfma(attn_col_frag<T, ROW>(dc_lds, c, db), w[c], g.dv[db]);
                        g.dk[db] = attn_mfma(attn_col_frag<T, ROW>(qc_lds, c, db), d[c], g.dk[db]);
                    }
            }
        }
        if (walk == 0) {
            either.take(g.dk);
            plus.take(g.dv);
        }
        if (walk == 1) minus.take(g.dv);
    }
    either.add(g.dk, NAN);
    plus.add(g.dv, INFINITY);
    minus.add(g.dv, -INFINITY);
    attn_dkv_store<T, NB>(p, g.dk, g.dv, 1.f, g.ds_exp, b, j, hk, split, part, half, j < p.Lk);
}

template <typename T, int DB, int MODE, bool DOCS, int WAVES>
__device__ __forceinline__ void attn_dq(const AttnParams& p, int group, char* smem, int (*sdoc)[ATTN_TILE], uint32_t (&said)[4]) {
    constexpr int ROW = attn_row<DB>(), TILE_BYTES = ATTN_TILE * ROW * 2;
    const int wave = attn_uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
    // p.splits > 1: the keys in that many runs of whole tiles, float32 parts that attn_parts_kernel adds in order
    const int total = p.B * p.Hq * p.row_blocks * p.splits, per = (total + 7) / 8;
    const int id = (group & 7) * per + (group >> 3);
    if (group >> 3 >= per || id >= total) return;
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
    bool one = true;
    if constexpr (DOCS) {
        const int2* r = p.qtiles + (int64_t)b * p.nqt + 2 * blk;
        const int2 r0 = r[0], r1 = 2 * blk + 1 < p.nqt ? r[1] : r[0];
        dlo = min(r0.x, r1.x);
        dhi = max(r0.y, r1.y);
        one = r0.x == r0.y && r1.x == r1.y && r0.x == r1.x;
    }
    AttnTiles<DOCS> tiles;
    const int run = (p.nkt + p.splits - 1) / p.splits, run_first = split * run, run_end = min((key_end + ATTN_TILE - 1) / ATTN_TILE, run_first + run);
    tiles.start(DOCS ? p.ktiles + (int64_t)b * p.nkt : nullptr, run_first, run_end, max(dlo, 0), dhi);
    typename AttnVec<T>::x8 qf[2 * DB], df[2 * DB];
    const T* q = row_ok ? (const T*)p.q + b * p.qs[0] + i * p.qs[1] + h * p.qs[2] : nullptr;
    const T* dout = row_ok ? (const T*)p.dout + b * p.ds[0] + i * p.ds[1] + h * p.ds[2] : nullptr;
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c) {
        qf[c] = attn_lane_frag<T>(q, 2 * c + half, p.D);
        df[c] = attn_lane_frag<T>(dout, 2 * c + half, p.D);
    }
    const int64_t stat = ((int64_t)b * p.Hq + h) * p.Lq + i;
    const float lse2 = row_ok ? attn_lse2(p.lse[stat]) : INFINITY, delta = row_ok ? p.delta[stat] : 0.f;
    const T* k = (const T*)p.k + b * p.ks[0] + hk * p.ks[2];
    const T* v = (const T*)p.v + b * p.vs[0] + hk * p.vs[2];
    const int* kdoc = DOCS ? p.kdoc + b * p.kdoc_stride : nullptr;
    const AttnScore f(p, h);
    constexpr bool FIT = ATTN_P_SHIFT<T> != 0.f;
    int ds_exp = FIT ? ATTN_DS_EXP : 0;                                 // (2^e in the weights: a lane's column is one query)
    AttnStage<ROW, ATTN_TILE, 4> sk, sv;
    sk.setup(wave, lane, p.ks[1], p.D);
    sv.setup(wave, lane, p.vs[1], p.D);
    f32x16 acc[DB] = {};
    const uint64_t k_at = attn_addr(k), v_at = attn_addr(v);
    const int k_row = (int)p.ks[1], v_row = (int)p.vs[1];
    const AttnLane<ROW> at_lane(lane);
    const uint32_t lds = attn_lds(smem);
    int doc_next = 0;                                                   // of the tile being staged: loaded ahead of its pieces, written behind the products
    auto stage = [&](int t, int buf) {
        const uint32_t at = lds + buf * 2 * TILE_BYTES;
        if (DOCS && wave == 0) doc_next = kdoc[min(t * ATTN_TILE + lane, p.Lk - 1)];
        sk.issue(k_at, t, n, k_row, p.D, at, wave);
        sv.issue(v_at, t, n, v_row, p.D, at + TILE_BYTES, wave);
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
            const uint32_t k_lds = at_lane.rows(lds + now * 2 * TILE_BYTES), v_lds = at_lane.rows(lds + now * 2 * TILE_BYTES + TILE_BYTES);
            const uint32_t kc_lds = at_lane.cols(lds + now * 2 * TILE_BYTES);
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                typename AttnVec<T>::x8 kf[2 * DB], vf[2 * DB], cf[DB][2], d[2];
#pragma unroll
                for (int c = 0; c < 2 * DB; ++c) kf[c] = attn_row_frag<T, ROW>(k_lds, kb, c);
                // (values behind the first products where registers are short: half of the keys' are free again by then.  Training step of 2 x 4096 x 16
                // heads on 4 x 128, causal with caps: 929 us, with all ahead 939; documents 506 / 520)
                constexpr int FIRST = DB > 2 ? DB : 0;
                f32x16 S = {}, dP = {};
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < FIRST; ++c) S = attn_mfma(kf[c], qf[c], S);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = 0; c < 2 * DB; ++c) vf[c] = attn_row_frag<T, ROW>(v_lds, kb, c);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int c = FIRST; c < 2 * DB; ++c) S = attn_mfma(kf[c], qf[c], S);
#pragma unroll
                for (int c = 0; c < 2 * DB; ++c) dP = attn_mfma(vf[c], df[c], dP);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int c = 0; c < 2; ++c) cf[db][c] = attn_col_frag<T, ROW>(kc_lds, 2 * kb + c, db);
                __builtin_amdgcn_sched_barrier(0);
                const int jb = j0 + 32 * kb + 4 * half;
                const float dist = (float)(i + n - p.Lq - jb), less = FIT ? lse2 - (float)ds_exp : lse2;
#pragma unroll
                for (int r = 0; r < 16; ++r) attn_ds<MODE, false>(S, dP, r, f, 1.f, less, delta, dist - (float)(8 * (r >> 2) + (r & 3)));
                if constexpr (mask.value) {
                    const int last = lim - jb;
#pragma unroll
                    for (int r = 0; r < 16; ++r) dP[r] = 8 * (r >> 2) + (r & 3) <= last ? dP[r] : 0.f;
                    if constexpr (DOCS)
#pragma unroll
                        for (int a = 0; a < 4; ++a) {
                            const int4 o = *reinterpret_cast<const int4*>(&sdoc[now][32 * kb + 8 * a + 4 * half]);
                            dP[4 * a] = o.x == qdoc ? dP[4 * a] : 0.f;
                            dP[4 * a + 1] = o.y == qdoc ? dP[4 * a + 1] : 0.f;
                            dP[4 * a + 2] = o.z == qdoc ? dP[4 * a + 2] : 0.f;
                            dP[4 * a + 3] = o.w == qdoc ? dP[4 * a + 3] : 0.f;
                        }
                }
                if constexpr (FIT) attn_fit(dP, ds_exp, acc);
                attn_pack<T>(dP, d);
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int db = 0; db < DB; ++db) acc[db] = attn_mfma(cf[db][c], d[c], acc[db]);
                if (mask.value && fine)                                 // (attn_left_over)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const typename AttnVec<T>::x8 left = attn_left_over<T>(dP, d[c], c);
#pragma unroll
                        for (int db = 0; db < DB; ++db) acc[db] = attn_mfma(cf[db][c], left, acc[db]);
                    }
            }
        }
        if (DOCS && wave == 0) sdoc[buf][lane] = doc_next;
    };
    while (t >= 0) {
        while (t >= 0 && full()) visit(std::false_type());
        while (t >= 0 && !full()) visit(std::true_type());
    }
    bool store = row_ok;
    if (attn_any(attn_has_nan(acc) && row_ok && lse2 == lse2, wave, said)) {
        attn_dq_again<T, DB, WAVES>(attn_kernel_args(), b, i, h, row_ok, split, run_first * ATTN_TILE, min(key_end, run_end * ATTN_TILE), lds + wave * TILE_BYTES);
        attn_clear(acc);                                                // (stored there; a return would keep the sums across the call)
        store = false;
    }
    attn_dq_store<T, DB>(p, acc, attn_ds_unit<MODE>(), ds_exp, b, i, h, split, half, store);
}

// A wave owns 32 keys: their K and V as operands and their dk and dv as accumulators.  Beyond 96 channels that is more than half of a SIMD's registers, so
// one wave a SIMD, whose vector work and products would wait for each other (537 us at 2 x 4096 x 16 heads x 128, causal with caps; two loops interleaved by
// hand: 555).  There two waves share 32 keys (attn_dkv_pair): each takes the scores of half of a tile's queries, they trade the 16-bit weights through the
// LDS, and each adds up half of the channels over all of the queries.
template <typename T, int DB, int MODE, bool DOCS, int WAVES>
__device__ __forceinline__ void attn_dkv(const AttnParams& p, int group, char* smem, AttnRows& rows, int (*sdoc)[ATTN_TILE], uint32_t (&said)[attn_dkv_pair<DB>() ? 8 : 4],
                                         char* traded, int (*exps)[64]) {
    constexpr int ROW = attn_row<DB>(), TILE_BYTES = ATTN_TILE * ROW * 2;
    constexpr float SHIFT = ATTN_P_SHIFT<T>;
    constexpr bool PAIR = attn_dkv_pair<DB>(), FIT = SHIFT != 0.f;
    constexpr int NB = PAIR ? DB / 2 : DB;                              // blocks of 32 channels a wave adds up
    typedef typename AttnVec<T>::x8 frag;
    // smem: [buffer][q, do];  traded (pairs): [key group][half of the queries][w, w, d, d][lane] fragments;  exps: [key group][half][lane], their ds_exp
    const int wave = attn_uniform(threadIdx.x >> 6), keys = PAIR ? wave & 3 : wave, part = PAIR ? wave >> 2 : 0, lane = threadIdx.x & 63, l31 = lane & 31, half = lane >> 5;
    // p.k_splits: 1 (a workgroup adds up all heads of the group), or float32 parts that attn_parts_kernel adds in order: the heads of the group in
    // p.k_splits / p.chunks equal runs, the queries in p.chunks runs of whole tiles
    const int total = p.B * p.Hk * p.k_splits * p.k_blocks, per = (total + 7) / 8;
    const int id = (group & 7) * per + (group >> 3);
    if (group >> 3 >= per || id >= total) return;
    const int blk = id % p.k_blocks, split = id / p.k_blocks % p.k_splits, bh = id / p.k_blocks / p.k_splits, hk = bh % p.Hk, b = bh / p.Hk;
    const int heads = p.G * p.chunks / p.k_splits, g0 = split / p.chunks * heads, g1 = g0 + heads;
    const int n = attn_keys(p, b), prefix = attn_prefix(p, b), k0 = blk * 128, off = n - p.Lq;
    const int j = k0 + 32 * keys + l31;
    const int kdoc = DOCS && j < p.Lk ? p.kdoc[b * p.kdoc_stride + j] : 0;
    const bool key_ok = j < n && kdoc >= 0;
    // first query that sees key x
    auto first_query = [&](int x) { return !p.causal || x < prefix ? 0 : max(x - off, 0); };
    const int qmin = key_ok ? first_query(j) : 0x7fffffff;
    const int wave_first = first_query(k0 + 32 * keys);
    const bool wave_on = k0 + 32 * keys < n;
    int dlo = 0, dhi = 0;
    bool one = true;
    if constexpr (DOCS) {
        const int2* r = p.ktiles + (int64_t)b * p.nkt + 2 * blk;
        const int2 r0 = r[0], r1 = 2 * blk + 1 < p.nkt ? r[1] : r[0];
        dlo = min(r0.x, r1.x);
        dhi = max(r0.y, r1.y);
        one = r0.x == r0.y && r1.x == r1.y && r0.x == r1.x;
    }
    const int2* ranges = DOCS ? p.qtiles + (int64_t)b * p.nqt : nullptr;
    const int run = (p.nqt + p.chunks - 1) / p.chunks, run_first = split % p.chunks * run, run_end = min(p.nqt, run_first + run);
    const int t_first = max(first_query(k0) / ATTN_TILE, run_first), t_end = k0 < n ? run_end : 0;
    AttnTiles<DOCS> tiles;
    int g = g0;
    tiles.start(ranges, t_first, t_end, max(dlo, 0), dhi);
    auto next = [&](int& gn) {
        int t = tiles.next(lane);
        while (t < 0 && gn + 1 < g1) {
            ++gn;
            tiles.start(ranges, t_first, t_end, max(dlo, 0), dhi);
            t = tiles.next(lane);
        }
        return t;
    };
    frag kf[2 * DB], vf[2 * DB];
    const T* k = j < n ? (const T*)p.k + b * p.ks[0] + j * p.ks[1] + hk * p.ks[2] : nullptr;
    const T* v = j < n ? (const T*)p.v + b * p.vs[0] + j * p.vs[1] + hk * p.vs[2] : nullptr;
#pragma unroll
    for (int c = 0; c < 2 * DB; ++c) {
        kf[c] = attn_lane_frag<T>(k, 2 * c + half, p.D);
        vf[c] = attn_lane_frag<T>(v, 2 * c + half, p.D);
    }
    AttnStage<ROW, ATTN_TILE, PAIR ? 8 : 4> sq, sd;
    sq.setup(wave, lane, p.qs[1], p.D);
    sd.setup(wave, lane, p.ds[1], p.D);
    int ds_exp = FIT ? ATTN_DS_EXP : 0;                                 // (a lane's column is one key; the two waves of a pair keep theirs alike)
    const AttnLane<ROW> at_lane(lane);
    const uint32_t lds = attn_lds(smem);
    float row_next = 0.f;
    auto stage = [&](int t, int gt, int buf) {
        const int h = hk * p.G + gt, i0 = t * ATTN_TILE;
        const uint32_t at = lds + buf * 2 * TILE_BYTES;
        // the rows' statistics: loaded ahead of the pieces (one of the three a wave), written to the LDS behind the products of the tile before
        const int i = i0 + lane;
        const int64_t stat = ((int64_t)b * p.Hq + h) * p.Lq + i;
        if (wave == 0) row_next = i < p.Lq ? attn_lse2(p.lse[stat]) - SHIFT : INFINITY;            // (queries behind the last: every weight 0)
        if (wave == 1) row_next = i < p.Lq ? p.delta[stat] : 0.f;
        if (DOCS && wave == 2) row_next = __builtin_bit_cast(float, i < p.Lq ? p.qdoc[b * p.qdoc_stride + i] : -1);
        sq.issue(attn_addr((const T*)p.q + b * p.qs[0] + h * p.qs[2]), t, p.Lq, (int)p.qs[1], p.D, at, wave);
        sd.issue(attn_addr((const T*)p.dout + b * p.ds[0] + h * p.ds[2]), t, p.Lq, (int)p.ds[1], p.D, at + TILE_BYTES, wave);
    };
    auto commit = [&](int buf) {
        if (wave == 0) rows.lse[buf][lane] = row_next;
        if (wave == 1) rows.delta[buf][lane] = row_next;
        if (DOCS && wave == 2) sdoc[buf][lane] = __builtin_bit_cast(int, row_next);
    };
    f32x16 dk[NB] = {}, dv[NB] = {};
    AttnScore f(p, hk * p.G);
    int t = next(g), buf = 0;
    const bool fine = tiles.few(lane);
    if (t >= 0) stage(t, g, 0);
    commit(0);
    // every query of tile t sees every key of the workgroup (but those behind the last, whose lanes are not stored)
    const int full_first = DOCS && !one ? 0x7fffffff : first_query(min(k0 + 127, n - 1));
    auto full = [&] { return !fine && t * ATTN_TILE >= full_first && (!DOCS || ((tiles.low == dlo) & (tiles.high == dlo))); };
    auto visit = [&](auto mask) {
        const int i0 = t * ATTN_TILE, now = buf;
        const float slope = MODE != ATTN_PLAIN && p.slopes ? p.slopes[hk * p.G + g] * ATTN_LOG2E : 0.f;
        attn_sync();
        t = next(g);
        buf ^= 1;
        if (t >= 0) stage(t, g, buf);
        const bool on = wave_on && (!mask.value || i0 + ATTN_TILE - 1 >= wave_first);
        f.slope = slope;
        constexpr int BLOCK = 32 * ROW * 2;                             // bytes of half a tile
        const uint32_t tile = lds + now * 2 * TILE_BYTES;
        // first operands of half a tile, this wave's channels
        auto columns = [&](int qb, frag (&qc)[NB][2], frag (&dc)[NB][2]) {
            const uint32_t qc_lds = at_lane.cols(tile + qb * BLOCK) ^ (part << 7), dc_lds = at_lane.cols(tile + TILE_BYTES + qb * BLOCK) ^ (part << 7);
#pragma unroll
            for (int db = 0; db < NB; ++db)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    dc[db][c] = attn_col_frag<T, ROW>(dc_lds, c, db);
                    qc[db][c] = attn_col_frag<T, ROW>(qc_lds, c, db);
                }
        };
        // weights and dscores of the 32 queries of half a tile as second operands
        auto weights = [&](int qb, frag (&w)[2], frag (&d)[2], frag (&w_left)[2], frag (&d_left)[2], auto&& ahead) {
            const uint32_t q_lds = at_lane.rows(tile + qb * BLOCK), d_lds = at_lane.rows(tile + TILE_BYTES + qb * BLOCK);
            frag qf[2 * DB], df[2 * DB];
            constexpr int FIRST = DB > 2 ? DB : 0;                      // (as in attn_dq_kernel)
            f32x16 S = {}, dP = {};
#pragma unroll
            for (int c = 0; c < 2 * DB; ++c) qf[c] = attn_row_frag<T, ROW>(q_lds, 0, c);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < FIRST; ++c) S = attn_mfma(qf[c], kf[c], S);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = 0; c < 2 * DB; ++c) df[c] = attn_row_frag<T, ROW>(d_lds, 0, c);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int c = FIRST; c < 2 * DB; ++c) S = attn_mfma(qf[c], kf[c], S);
#pragma unroll
            for (int c = 0; c < 2 * DB; ++c) dP = attn_mfma(df[c], vf[c], dP);
            __builtin_amdgcn_sched_barrier(0);
            ahead();
            __builtin_amdgcn_sched_barrier(0);
            const int ib = 32 * qb + 4 * half;
            const float dist = (float)(i0 + ib + off - j), ds_by = FIT ? ldexpf(1.f, ds_exp - (int)SHIFT) : 1.f;
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const float4 l4 = *reinterpret_cast<const float4*>(&rows.lse[now][ib + 8 * a]), e4 = *reinterpret_cast<const float4*>(&rows.delta[now][ib + 8 * a]);
                const float l[4] = {l4.x, l4.y, l4.z, l4.w}, de[4] = {e4.x, e4.y, e4.z, e4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) attn_ds<MODE, FIT>(S, dP, 4 * a + e, f, ds_by, l[e], de[e], dist + (float)(8 * a + e));
            }
            if constexpr (mask.value) {
                const int first = qmin - i0 - ib;
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const bool see = 8 * (r >> 2) + (r & 3) >= first;
                    S[r] = see ? S[r] : 0.f;
                    dP[r] = see ? dP[r] : 0.f;
                }
                if constexpr (DOCS)
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const int4 o4 = *reinterpret_cast<const int4*>(&sdoc[now][ib + 8 * a]);
                        const int o[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const bool see = o[e] == kdoc;
                            S[4 * a + e] = see ? S[4 * a + e] : 0.f;
                            dP[4 * a + e] = see ? dP[4 * a + e] : 0.f;
                        }
                    }
            }
            if constexpr (FIT) attn_fit(dP, ds_exp, dk);
            attn_pack<T>(S, w);
            attn_pack<T>(dP, d);
            if (mask.value && fine)                                     // (attn_left_over)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    w_left[c] = attn_left_over<T>(S, w[c], c);
                    d_left[c] = attn_left_over<T>(dP, d[c], c);
                }
        };
        auto products = [&](const frag (&w)[2], const frag (&d)[2], const frag (&qc)[NB][2], const frag (&dc)[NB][2]) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int db = 0; db < NB; ++db) {
                    dv[db] = attn_mfma(dc[db][c], w[c], dv[db]);
                    dk[db] = attn_mfma(qc[db][c], d[c], dk[db]);
                }
        };
        if constexpr (PAIR) {
            frag w[2], d[2], w_left[2], d_left[2], qc[NB][2], dc[NB][2];
            frag* mine = reinterpret_cast<frag*>(traded) + (keys * 2 + part) * 4 * 64 + lane;
            const frag* theirs = reinterpret_cast<const frag*>(traded) + (keys * 2 + (part ^ 1)) * 4 * 64 + lane;
            if (on) {
                // (the products' fragments are on their way during the vector work, and the other half's during the wait: 932 -> 911 us for a training step of
                // 2 x 4096 x 16 heads on 4 x 128, causal with caps.  The unpaired form lets two workgroups overlap instead: 458 us at x 64, with this 473)
                weights(part, w, d, w_left, d_left, [&] { columns(part, qc, dc); });
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    mine[c * 64] = w[c];
                    mine[(2 + c) * 64] = d[c];
                }
                if constexpr (FIT) exps[keys * 2 + part][lane] = ds_exp;
                products(w, d, qc, dc);
                if (mask.value && fine) products(w_left, d_left, qc, dc);
                columns(part ^ 1, qc, dc);
            }
            attn_traded();
            if (on) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    w[c] = theirs[c * 64];
                    d[c] = theirs[(2 + c) * 64];
                }
                if constexpr (FIT) {                                    // the lower of the two exponents for both
                    const int other = exps[keys * 2 + (part ^ 1)][lane], low = min(ds_exp, other);
                    if (__ballot(other != ds_exp)) {
                        const float by = ldexpf(1.f, low - ds_exp), their = ldexpf(1.f, low - other);
                        ds_exp = low;
#pragma unroll
                        for (int db = 0; db < NB; ++db)
#pragma unroll
                            for (int r = 0; r < 16; ++r) dk[db][r] *= by;
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                d[c][e] = (T)((float)d[c][e] * their);
                                if (mask.value && fine) d_left[c][e] = (T)((float)d_left[c][e] * by);
                            }
                    }
                }
                products(w, d, qc, dc);
            }
            if (mask.value && fine) {                                   // (the same for all waves of the workgroup)
                attn_traded();
                if (on) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        mine[c * 64] = w_left[c];
                        mine[(2 + c) * 64] = d_left[c];
                    }
                }
                attn_traded();
                if (on) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        w[c] = theirs[c * 64];
                        d[c] = theirs[(2 + c) * 64];
                    }
                    products(w, d, qc, dc);
                }
            }
        } else if (on) {
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
                frag w[2], d[2], w_left[2], d_left[2], qc[NB][2], dc[NB][2];
                weights(qb, w, d, w_left, d_left, [] {});
                columns(qb, qc, dc);
                products(w, d, qc, dc);
                if (mask.value && fine) products(w_left, d_left, qc, dc);
            }
        }
        commit(buf);
    };
    while (t >= 0) {
        while (t >= 0 && full()) visit(std::false_type());
        while (t >= 0 && !full()) visit(std::true_type());
    }
    bool store = j < p.Lk;
    if (attn_any((attn_has_nan(dk) || attn_has_nan(dv)) && key_ok, wave, said)) {
        const int first = max(first_query(k0) / ATTN_TILE, run_first) * ATTN_TILE, end = min(t_end * ATTN_TILE, p.Lq);
#pragma unroll 1
        for (int turn = 0; turn < (PAIR ? 2 : 1); ++turn) {             // (two waves of a pair share their half of a buffer: one after the other)
            if (turn == part) attn_dkv_again<T, DB, NB, WAVES>(attn_kernel_args(), b, hk, j, kdoc, split, g0, g1, first, end, part, lds + keys * TILE_BYTES);
            if (PAIR) __syncthreads();
        }
        attn_clear(dk);
        attn_clear(dv);
        store = false;
    }
    if (!key_ok)                                                        // keys that nobody sees (their lanes held something else)
#pragma unroll
        for (int db = 0; db < NB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) dk[db][r] = dv[db][r] = 0.f;
    attn_dkv_store<T, NB>(p, dk, dv, attn_ds_unit<MODE>(), ds_exp, b, j, hk, split, part, half, store);
}
#endif

template <typename T, int DB, int MODE, bool DOCS>
__global__ __launch_bounds__(256, (attn_dq_waves<DB, DOCS>())) void attn_dq_kernel(AttnParams p) {
#ifdef __HIP_DEVICE_COMPILE__
    __shared__ __align__(1024) char smem[attn_lds_bytes<DB>()];
    __shared__ __align__(16) int sdoc[2][ATTN_TILE];
    __shared__ uint32_t said[4];
    attn_dq<T, DB, MODE, DOCS, attn_dq_waves<DB, DOCS>()>(p, blockIdx.x, smem, sdoc, said);
#endif
}
template <typename T, int DB, int MODE, bool DOCS>
__global__ __launch_bounds__(attn_dkv_pair<DB>() ? 512 : 256, attn_dkv_waves<DB>()) void attn_dkv_kernel(AttnParams p) {
#ifdef __HIP_DEVICE_COMPILE__
    __shared__ __align__(1024) char smem[attn_lds_bytes<DB>()];
    __shared__ __align__(16) AttnRows rows;
    __shared__ __align__(16) int sdoc[2][ATTN_TILE];
    __shared__ __align__(16) char traded[attn_dkv_pair<DB>() ? 4 * 2 * 4 * 1024 : 16];
    __shared__ int exps[attn_dkv_pair<DB>() && ATTN_P_SHIFT<T> != 0.f ? 8 : 1][64];
    __shared__ uint32_t said[attn_dkv_pair<DB>() ? 8 : 4];
    attn_dkv<T, DB, MODE, DOCS, attn_dkv_waves<DB>()>(p, blockIdx.x, smem, rows, sdoc, said, traded, exps);
#endif
}
// Both in one launch where that is two rounds of the chip at most (1024 workgroups): small calls wait for single workgroups, and so for both kinds at once.
// Training step of 3 x 1021 x 6 heads x 72, documents: 105 -> 91 us, 2 x 1200 x 8 heads on 2 x 72, causal with caps: 125 -> 100, 4096 x 16 x 64: 425 -> 424.
// (Larger ones keep two launches: the dq workgroups alone need fewer registers, and more of them share a CU.)
template <typename T, int DB, int MODE, bool DOCS>
__global__ __launch_bounds__(256, attn_dkv_waves<DB>()) void attn_grads_kernel(AttnParams p) {
#ifdef __HIP_DEVICE_COMPILE__
    static_assert(!attn_dkv_pair<DB>(), "256 threads each");
    __shared__ __align__(1024) char smem[attn_lds_bytes<DB>()];
    __shared__ __align__(16) AttnRows rows;
    __shared__ __align__(16) int sdoc[2][ATTN_TILE];
    __shared__ uint32_t said[4];
    if ((int)blockIdx.x < p.first_k) attn_dq<T, DB, MODE, DOCS, attn_dkv_waves<DB>()>(p, blockIdx.x, smem, sdoc, said);
    else attn_dkv<T, DB, MODE, DOCS, attn_dkv_waves<DB>()>(p, blockIdx.x - p.first_k, smem, rows, sdoc, said, nullptr, nullptr);
#endif
}

// part [split][output][elements] -> the outputs (one or two: gridDim.y), the splits in order; eight elements a thread
template <typename T>
__global__ __launch_bounds__(256) void attn_parts_kernel(const float* __restrict__ part, int splits, int64_t all, T* __restrict__ out0, T* __restrict__ out1) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (at >= all) return;
    float x[8] = {};
    for (int s = 0; s < splits; ++s) {
        const float4* a = reinterpret_cast<const float4*>(part + (s * (int64_t)gridDim.y + blockIdx.y) * all + at);
        const float4 u = a[0], w = a[1];
        x[0] += u.x; x[1] += u.y; x[2] += u.z; x[3] += u.w;
        x[4] += w.x; x[5] += w.y; x[6] += w.z; x[7] += w.w;
    }
    typename AttnVec<T>::x8 o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = (T)x[e];
    *reinterpret_cast<typename AttnVec<T>::x8*>((blockIdx.y ? out1 : out0) + at) = o;
}

template <typename T, int DB, int MODE, bool DOCS>
static void attn_bwd_launch(AttnParams& p, hipStream_t stream) {
    const int64_t q_rows = (int64_t)p.B * p.Lq * p.Hq, k_rows = (int64_t)p.B * p.Lk * p.Hk;
    hipLaunchKernelGGL((attn_prep_kernel<T>), dim3((unsigned)(cdiv64(q_rows, 16) < 2048 ? cdiv64(q_rows, 16) : 2048)), dim3(256), 0, stream, p);
    auto add = [&](const float* part, int count, int64_t all, void* a, void* b) {
        if (count > 1) hipLaunchKernelGGL((attn_parts_kernel<T>), dim3((unsigned)cdiv64(all, 2048), b ? 2 : 1), dim3(256), 0, stream, part, count, all, (T*)a, (T*)b);
    };
    const unsigned dq = p.dq ? attn_even((int64_t)p.B * p.Hq * p.splits * p.row_blocks) : 0;
    const unsigned dkv = p.dk && p.Lk > 0 ? attn_even((int64_t)p.B * p.Hk * p.k_splits * p.k_blocks) : 0;
    bool both = false;
    if constexpr (!attn_dkv_pair<DB>()) {
        if ((both = dq && dkv && dq + dkv <= 1024)) {
            p.first_k = dq;
            hipLaunchKernelGGL((attn_grads_kernel<T, DB, MODE, DOCS>), dim3(dq + dkv), dim3(256), 0, stream, p);
        }
    }
    if (dq) {
        if (!both) hipLaunchKernelGGL((attn_dq_kernel<T, DB, MODE, DOCS>), dim3(dq), dim3(256), 0, stream, p);
        add(p.part, p.splits, q_rows * p.D, p.dq, nullptr);
    }
    if (dkv) {
        if (!both) hipLaunchKernelGGL((attn_dkv_kernel<T, DB, MODE, DOCS>), dim3(dkv), dim3(attn_dkv_pair<DB>() ? 512 : 256), 0, stream, p);
        add(p.k_part, p.k_splits, k_rows * p.D, p.dk, p.dv);
    }
}

// the kernels of one element type, each in a file of its own (they take two minutes to compile)
template <typename T>
static void attn_bwd_typed(AttnParams& p, hipStream_t stream) {
    attn_forms(p, [&](auto db, auto mode, auto docs) { attn_bwd_launch<T, db.value, mode.value, docs.value>(p, stream); });
}
