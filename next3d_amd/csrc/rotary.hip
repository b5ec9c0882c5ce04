// Rotary positions with several axes (time, height, width) for gfx950: every pair p of channels (x0, x1) of a token turns by the angle
//   theta = position[token][axis(p)] * base^(-e(p)),        (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos)
// with e(p) = 2 i / s for pair i of an axis section of s channels (ladder 'axis'), or p / P for pair p of all P (ladder 'shared').
// The gradient is the same kernel with -sin.  HBM-bound: q and k of a token are one launch, read once and written once; the cosines and sines of a
// workgroup's tokens are computed once into the LDS and serve every head of q and k.  The angle is taken in 64 bits and reduced to a fraction of a
// turn there — in 32 bits the angle of position 100000 is off by 0.004 — and the cosine and sine of that fraction are float32.
// Measured (medians of 60 launches): q and k of 32768 tokens x 16 heads x 128 channels each, bfloat16, 116 us (4.6 TB/s; a large copy reaches 4.9); a single
// token of 8 sequences 4.0 us.
#include "token_vec.h"

static constexpr int ROT_THREADS = 256, ROT_MAX_AXES = 4, ROT_MAX_TABLE = 2048;

// x / d for x < 2^31 by multiplication (d > 0)
struct RotDiv {
    uint32_t d, mul, shift;
};
static RotDiv rot_div(uint32_t d) {
    RotDiv r = {d, 0, 0};
    while ((1ull << r.shift) < d) ++r.shift;
    r.mul = (uint32_t)(((1ull << 32) * ((1ull << r.shift) - d)) / d + 1);
    return r;
}
__device__ __forceinline__ uint32_t rot_quot(uint32_t x, const RotDiv& r) { return (__umulhi(x, r.mul) + x) >> r.shift; }

struct RotParams {
    const void* x[2];             // q and k (k may be absent: heads 0)
    void* y[2];
    const void* pos;
    int64_t sb[2], sl[2], sh[2];  // element strides of batch, token and head
    int64_t pos_sb, pos_sl;       // element strides of the positions' batch (0: shared) and token
    int64_t tokens;               // B * L
    int L, heads[2], D, P, axes, pos_type, shared, tpb, sign;
    int first[ROT_MAX_AXES + 1];  // first pair of every axis
    double log2_base;
    RotDiv by_unit, by_heads, by_len;
};

// the axis of pair p
__device__ __forceinline__ int rot_axis(const RotParams& r, int p) {
    int a = 0;
#pragma unroll
    for (int i = 1; i < ROT_MAX_AXES; ++i) a += (i < r.axes && p >= r.first[i]) ? 1 : 0;
    return a;
}

// W pairs a unit: two runs of W channels (halves) or one of 2 W (interleaved).  The channels behind the last pair pass through in units of the same width.
template <typename T, int W, bool INTER>
__global__ __launch_bounds__(ROT_THREADS) void rotary_kernel(RotParams r) {
    extern __shared__ float2 table[];                      // [tpb][P]
    constexpr int RUN = INTER ? 2 * W : W;
    const int64_t t0 = (int64_t)blockIdx.x * r.tpb;
    const int nt = (int)(r.tokens - t0 < r.tpb ? r.tokens - t0 : r.tpb);
    for (int i = threadIdx.x; i < nt * r.P; i += ROT_THREADS) {
        const int t = i / r.P, p = i - t * r.P;
        const int64_t b = rot_quot((uint32_t)(t0 + t), r.by_len), l = t0 + t - b * r.L;
        const int a = rot_axis(r, p);
        const int64_t at = b * r.pos_sb + l * r.pos_sl + a;
        const double pos = r.pos_type == 0 ? (double)((const float*)r.pos)[at]
                                           : r.pos_type == 1 ? (double)((const int*)r.pos)[at] : (double)((const long long*)r.pos)[at];
        const double e = r.shared ? (double)p / r.P : (double)(p - r.first[a]) / (r.first[a + 1] - r.first[a]);
        const double quarters = pos * exp2(-e * r.log2_base) * 0.63661977236758134308;      // 2 / pi
        const double whole = rint(quarters);
        float s, c;
        sincospif(0.5f * (float)(quarters - whole), &s, &c);                               // within an eighth of a turn: the rounding to float is 5e-8 at most
        const int k = (int)(long long)whole;
        if (k & 1) {
            const float t1 = c;
            c = -s;
            s = t1;
        }
        if (k & 2) {
            c = -c;
            s = -s;
        }
        table[i] = make_float2(c, r.sign < 0 ? -s : s);
    }
    __syncthreads();
    const int units = (int)r.by_unit.d, heads = r.heads[0] + r.heads[1], rot_units = r.P / W;
    const int work = nt * heads * units;
    for (int i = threadIdx.x; i < work; i += ROT_THREADS) {
        const int hu = (int)rot_quot(i, r.by_unit), u = i - hu * units;
        const int t = (int)rot_quot(hu, r.by_heads);
        int h = hu - t * heads;
        const int which = h >= r.heads[0];
        if (which) h -= r.heads[0];
        const int64_t tok = t0 + t;
        const int64_t b = rot_quot((uint32_t)tok, r.by_len), l = tok - b * r.L;
        const T* x = (const T*)r.x[which] + b * r.sb[which] + l * r.sl[which] + h * r.sh[which];
        T* y = (T*)r.y[which] + (tok * r.heads[which] + h) * r.D;
        if (u < rot_units) {
            const int p = u * W;
            const float2* cs = table + t * r.P + p;
            if constexpr (INTER) {
                float v[2 * W];
                token_load<T, 2 * W>(x + 2 * p, v);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const float x0 = v[2 * e], x1 = v[2 * e + 1];
                    v[2 * e] = x0 * cs[e].x - x1 * cs[e].y;
                    v[2 * e + 1] = x0 * cs[e].y + x1 * cs[e].x;
                }
                token_store<T, 2 * W>(y + 2 * p, v);
            } else {
                int lo, gap;
                if (r.shared) {
                    lo = p;
                    gap = r.P;
                } else {
                    const int a = rot_axis(r, p);
                    lo = p + r.first[a];                   // 2 * first + (p - first)
                    gap = r.first[a + 1] - r.first[a];
                }
                float v0[W], v1[W];
                token_load<T, W>(x + lo, v0);
                token_load<T, W>(x + lo + gap, v1);
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    const float x0 = v0[e], x1 = v1[e];
                    v0[e] = x0 * cs[e].x - x1 * cs[e].y;
                    v1[e] = x0 * cs[e].y + x1 * cs[e].x;
                }
                token_store<T, W>(y + lo, v0);
                token_store<T, W>(y + lo + gap, v1);
            }
        } else {
            const int c = 2 * r.P + (u - rot_units) * RUN;
            if (c + RUN <= r.D) {
                float v[RUN];
                token_load<T, RUN>(x + c, v);
                token_store<T, RUN>(y + c, v);
            } else {
                for (int i = c; i < r.D; ++i) y[i] = x[i];
            }
        }
    }
}

template <typename T, int W, bool INTER>
static void rotary_launch(const RotParams& r, hipStream_t stream) {
    const dim3 grid((unsigned)cdiv64(r.tokens, r.tpb));
    hipLaunchKernelGGL((rotary_kernel<T, W, INTER>), grid, dim3(ROT_THREADS), (size_t)r.tpb * r.P * sizeof(float2), stream, r);
}

extern "C" int n3d_rotary(const n3d_rotary_desc* d, n3d_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    N3D_CHECK(d, "rotary: null descriptor");
    N3D_CHECK(d->B >= 0 && d->L >= 0 && d->heads_q >= 0 && d->heads_k >= 0, "rotary: negative sizes");
    const int64_t tokens = (int64_t)d->B * d->L;
    const int heads = d->heads_q + d->heads_k;
    if (tokens == 0 || heads == 0) return 0;
    N3D_CHECK(tokens < 0x7fffffff, "rotary: too many tokens");
    N3D_CHECK(d->D >= 2 && d->D <= 1024 && heads <= 4096, "rotary: 2 to 1024 channels, 4096 heads at most");
    N3D_CHECK(d->axes >= 1 && d->axes <= ROT_MAX_AXES, "rotary: 1 to %d axes", ROT_MAX_AXES);
    N3D_CHECK(d->dtype == N3D_F32 || d->dtype == N3D_F16 || d->dtype == N3D_BF16, "rotary: unsupported dtype %d", d->dtype);
    N3D_CHECK(d->pos_type >= 0 && d->pos_type <= 2 && d->positions, "rotary: bad positions");
    N3D_CHECK(d->base > 0.0, "rotary: base must be positive");
    N3D_CHECK((d->heads_q == 0 || (d->q && d->out_q)) && (d->heads_k == 0 || (d->k && d->out_k)), "rotary: null tensor");
    RotParams r = {};
    r.x[0] = d->q; r.x[1] = d->k; r.y[0] = d->out_q; r.y[1] = d->out_k; r.pos = d->positions;
    for (int i = 0; i < 2; ++i) {
        const int64_t* st = i ? d->k_strides : d->q_strides;
        r.sb[i] = st[0]; r.sl[i] = st[1]; r.sh[i] = st[2];
    }
    r.pos_sb = d->pos_batch_stride; r.pos_sl = d->pos_token_stride;
    r.tokens = tokens; r.L = d->L; r.heads[0] = d->heads_q; r.heads[1] = d->heads_k; r.D = d->D;
    r.axes = d->axes; r.pos_type = d->pos_type; r.shared = d->shared_ladder != 0; r.sign = d->inverse ? -1 : 1;
    r.log2_base = log2(d->base);
    for (int a = 0; a < d->axes; ++a) {
        N3D_CHECK(d->sections[a] >= 0 && d->sections[a] % 2 == 0 && d->sections[a] <= d->D, "rotary: sections are even numbers of channels");
        r.first[a + 1] = r.first[a] + d->sections[a] / 2;
    }
    for (int a = d->axes; a < ROT_MAX_AXES; ++a) r.first[a + 1] = r.first[d->axes];
    r.P = r.first[d->axes];
    N3D_CHECK(r.P > 0 && 2 * r.P <= d->D, "rotary: the sections add up to %d of %d channels", 2 * r.P, d->D);
    // the widest unit (16 bytes a load at most) that neither a half of a section nor the end of the rotated channels cuts
    const int rest = d->D - 2 * r.P;
    int w = d->dtype == N3D_F32 ? 4 : 8;
    if (d->interleaved) w /= 2;
    for (; w > 1; w >>= 1) {
        bool ok = r.P % w == 0;
        if (!d->interleaved && !r.shared)
            for (int a = 0; a < d->axes; ++a) ok = ok && (r.first[a + 1] - r.first[a]) % w == 0;
        if (ok) break;
    }
    const int units = r.P / w + cdiv(rest, d->interleaved ? 2 * w : w);
    r.by_unit = rot_div(units); r.by_heads = rot_div(heads); r.by_len = rot_div(d->L);
    // tokens a workgroup: four rounds of its threads over the channels and a full round over the angles, as long as 1024 workgroups remain (16 rounds: 121 us
    // instead of 113 for the call above, in one run; one round, or 256 to 4096 workgroups, are as fast where many tokens come, but then a workgroup's angles fill no round)
    int64_t tpb = cdiv64(4 * ROT_THREADS, (int64_t)heads * units);
    if (tpb < cdiv(ROT_THREADS, r.P)) tpb = cdiv(ROT_THREADS, r.P);
    if (tpb > tokens / 1024) tpb = tokens / 1024;
    if (tpb > ROT_MAX_TABLE / r.P) tpb = ROT_MAX_TABLE / r.P;
    r.tpb = tpb < 1 ? 1 : (int)tpb;
    N3D_CHECK(n3d_grid_fits(cdiv64(tokens, r.tpb), ROT_THREADS), "rotary: too many tokens for one launch");
    const double esize = d->dtype == N3D_F32 ? 4.0 : 2.0;
    N3dProfScope prof(N3D_K_ROTARY, stream, 3.0 * tokens * heads * d->D, 2.0 * esize * tokens * heads * d->D);
    token_dispatch(d->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        constexpr int MAX = 16 / sizeof(T);
        if (d->interleaved) {
            if (w == MAX / 2) rotary_launch<T, MAX / 2, true>(r, stream);
            else if (w == 2) rotary_launch<T, 2, true>(r, stream);
            else rotary_launch<T, 1, true>(r, stream);
        } else {
            if (w == MAX) rotary_launch<T, MAX, false>(r, stream);
            else if (w == 4) rotary_launch<T, 4, false>(r, stream);
            else if (w == 2) rotary_launch<T, 2, false>(r, stream);
            else rotary_launch<T, 1, false>(r, stream);
        }
    });
    N3D_LAUNCH_CHECK();
    return 0;
}
