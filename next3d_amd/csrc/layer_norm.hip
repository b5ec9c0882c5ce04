// layer_norm for gfx950: y = (x - mean) * rstd * w + b over the last dimension, and its gradients.
//   forward   m = sum(x) / C,  d = x - m,  c = sum(d) / C,  mean = m + c,  var = sum(d^2) / C - c^2,  rstd = 1 / sqrt(var + eps),  (x - mean) = d - c
//             (c is what the rounding of the first sum left over: with it a row of equal values gives zeros, whatever the value)
//   backward  g = dy * w,  xh = (x - mean) * rstd:   dx = rstd * (g - mean(g) - xh * mean(g * xh)),  dw = sum_rows dy * xh,  db = sum_rows dy
// HBM-bound: a row is read once into registers (LPR lanes hold it, K vectors of 16 bytes each), both statistics are taken from the registers — the
// variance from centred values, so a large common offset costs no digits — and the result is written once.  All sums are float32.
// Measured (medians of 60 launches): 16384 x 4096 bfloat16 forward 56 us (4.8 TB/s; a large copy reaches 4.9), backward 90 + 7 us for the parts' sum (4.5);
// 786432 x 32 float16 20 (5.0) and 28 + 4 us (5.4); 5003 x 1001 float32 12 and 15 + 4.4 us; 112 x 512 float32 3.4 us.  Bound by memory, below some 20 MB by
// the launches.
// dw / db: a thread keeps the same columns for every row it visits and adds them up in registers; the workgroup's sums go to `ws` as one row and a
// second launch adds the rows in index order.  No atomics: the same call gives the same bits.
#include "token_vec.h"

// threads of a workgroup whose rows are held by `lpr` lanes each
static constexpr int ln_threads(int lpr) { return lpr > 256 ? lpr : 256; }
static constexpr int LN_BIG_THREADS = 1024;

// v[i] <- the sum over the LPR lanes of a row (N <= 2)
template <int LPR, int N>
__device__ __forceinline__ void ln_sum(float (&v)[N], float* red, int& slot) {
#pragma unroll
    for (int o = (LPR < 64 ? LPR : 64) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], o);
    if constexpr (LPR > 64) {
        // two slots in turn: a slot is written again only behind the barrier of the call in between, which every reader of it has reached
        constexpr int W = LPR / 64;
        float* r = red + slot * 2 * W;
        slot ^= 1;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) r[i * W + (threadIdx.x >> 6)] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v[i] += r[i * W + w];
        }
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void ln_load(const T* __restrict__ p, int64_t c, int64_t C, float (&f)[VEC]) {
    if (c + VEC <= C) {
        token_load<T, VEC>(p + c, f);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = c + e < C ? (float)p[c + e] : 0.f;
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void ln_store(T* __restrict__ p, int64_t c, int64_t C, const float (&f)[VEC]) {
    if (c + VEC <= C) {
        token_store<T, VEC>(p + c, f);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (c + e < C) p[c + e] = (T)f[e];
    }
}

// weight / bias: float32, or the type of x; absent: `none`
template <typename T, int VEC>
__device__ __forceinline__ void ln_affine(const void* w, int w32, int64_t c, int64_t C, float none, float (&f)[VEC]) {
    if (!w) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = none;
    } else if (w32) {
        ln_load<float, VEC>((const float*)w, c, C, f);
    } else {
        ln_load<T, VEC>((const T*)w, c, C, f);
    }
}

struct LnParams {
    const void *x, *w, *b, *dy;
    void *y, *dx;
    float *mean, *rstd, *ws;
    int64_t rows, x_stride, dy_stride;
    int C, w32;
    float eps;
};

template <typename T, int LPR, int K>
__global__ __launch_bounds__(ln_threads(LPR)) void ln_fwd_kernel(LnParams p) {
    constexpr int VEC = 16 / sizeof(T), THREADS = ln_threads(LPR), RPB = THREADS / LPR;
    __shared__ float red[2 * 2 * (LPR > 64 ? LPR / 64 : 1)];
    const int lane = threadIdx.x % LPR, C = p.C;
    const float n = (float)C;
    int slot = 0;
    float w[K][VEC], b[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        ln_affine<T, VEC>(p.w, p.w32, (k * LPR + lane) * VEC, C, 1.f, w[k]);
        ln_affine<T, VEC>(p.b, p.w32, (k * LPR + lane) * VEC, C, 0.f, b[k]);
    }
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR; row < p.rows; row += (int64_t)gridDim.x * RPB) {
        const T* x = (const T*)p.x + row * p.x_stride;
        T* y = (T*)p.y + row * C;
        float v[K][VEC];
        float s[1] = {0.f}, q[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            ln_load<T, VEC>(x, (k * LPR + lane) * VEC, C, v[k]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[0] += v[k][e];
        }
        ln_sum<LPR>(s, red, slot);
        const float m = s[0] / n;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * LPR + lane) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[k][e] = c + e < C ? v[k][e] - m : 0.f;
                q[0] += v[k][e] * v[k][e];
                q[1] += v[k][e];
            }
        }
        ln_sum<LPR>(q, red, slot);
        const float rest = q[1] / n, mean = m + rest, rstd = 1.f / sqrtf(fmaxf(q[0] / n - rest * rest, 0.f) + p.eps);
        if (lane == 0 && p.mean) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float o[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) o[e] = (v[k][e] - rest) * rstd * w[k][e] + b[k][e];
            ln_store<T, VEC>(y, (k * LPR + lane) * VEC, C, o);
        }
    }
}

// rows longer than the registers of a workgroup: the row is read again for each step (out of the L2, which holds it)
template <typename T>
__global__ __launch_bounds__(LN_BIG_THREADS) void ln_fwd_big_kernel(LnParams p) {
    constexpr int VEC = 16 / sizeof(T), STEP = LN_BIG_THREADS * VEC;
    __shared__ float red[2 * 2 * (LN_BIG_THREADS / 64)];
    const int C = p.C;
    const float n = (float)C;
    int slot = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.x_stride;
        T* y = (T*)p.y + row * C;
        float s[1] = {0.f}, q[2] = {0.f, 0.f};
        for (int64_t c = threadIdx.x * VEC; c < C; c += STEP) {
            float v[VEC];
            ln_load<T, VEC>(x, c, C, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) s[0] += v[e];
        }
        ln_sum<LN_BIG_THREADS>(s, red, slot);
        const float m = s[0] / n;
        for (int64_t c = threadIdx.x * VEC; c < C; c += STEP) {
            float v[VEC];
            ln_load<T, VEC>(x, c, C, v);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = c + e < C ? v[e] - m : 0.f;
                q[0] += d * d;
                q[1] += d;
            }
        }
        ln_sum<LN_BIG_THREADS>(q, red, slot);
        const float rest = q[1] / n, mean = m + rest, rstd = 1.f / sqrtf(fmaxf(q[0] / n - rest * rest, 0.f) + p.eps);
        if (threadIdx.x == 0 && p.mean) {
            p.mean[row] = mean;
            p.rstd[row] = rstd;
        }
        for (int64_t c = threadIdx.x * VEC; c < C; c += STEP) {
            float v[VEC], w[VEC], b[VEC];
            ln_load<T, VEC>(x, c, C, v);
            ln_affine<T, VEC>(p.w, p.w32, c, C, 1.f, w);
            ln_affine<T, VEC>(p.b, p.w32, c, C, 0.f, b);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = (v[e] - m - rest) * rstd * w[e] + b[e];
            ln_store<T, VEC>(y, c, C, v);
        }
    }
}

template <typename T, int LPR, int K>
__global__ __launch_bounds__(ln_threads(LPR)) void ln_bwd_kernel(LnParams p) {
    constexpr int VEC = 16 / sizeof(T), THREADS = ln_threads(LPR), RPB = THREADS / LPR, COLS = (LPR < 64 ? LPR : 64) * K * VEC;
    __shared__ float red[2 * 2 * (LPR > 64 ? LPR / 64 : 1)];
    const int lane = threadIdx.x % LPR, C = p.C;
    const float n = (float)C;
    int slot = 0;
    float w[K][VEC], dw[K][VEC], db[K][VEC];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        ln_affine<T, VEC>(p.w, p.w32, (k * LPR + lane) * VEC, C, 1.f, w[k]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) dw[k][e] = db[k][e] = 0.f;
    }
    for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR; row < p.rows; row += (int64_t)gridDim.x * RPB) {
        const T* x = (const T*)p.x + row * p.x_stride;
        const T* dy = (const T*)p.dy + row * p.dy_stride;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float xh[K][VEC], g[K][VEC];
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * LPR + lane) * VEC;
            ln_load<T, VEC>(x, c, C, xh[k]);
            ln_load<T, VEC>(dy, c, C, g[k]);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * LPR + lane) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                xh[k][e] = c + e < C ? (xh[k][e] - mean) * rstd : 0.f;
                dw[k][e] += g[k][e] * xh[k][e];
                db[k][e] += g[k][e];
                g[k][e] *= w[k][e];
                s[0] += g[k][e];
                s[1] += g[k][e] * xh[k][e];
            }
        }
        if (p.dx) {
            ln_sum<LPR>(s, red, slot);
            s[0] /= n;
            s[1] /= n;
            T* dx = (T*)p.dx + row * C;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float o[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) o[e] = rstd * (g[k][e] - s[0] - xh[k][e] * s[1]);
                ln_store<T, VEC>(dx, (k * LPR + lane) * VEC, C, o);
            }
        }
    }
    if (!p.ws) return;
    float* out = p.ws + (int64_t)blockIdx.x * 2 * C;
    if constexpr (LPR > 64) {                               // one row at a time: every column has one owner
#pragma unroll
        for (int k = 0; k < K; ++k) {
            ln_store<float, VEC>(out, (k * LPR + lane) * VEC, C, dw[k]);
            ln_store<float, VEC>(out + C, (k * LPR + lane) * VEC, C, db[k]);
        }
    } else {                                                // the wave's row groups by shuffles, the four waves one after the other through the LDS
        __shared__ float acc[2][COLS];
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e)
#pragma unroll
                for (int o = LPR; o < 64; o <<= 1) {
                    dw[k][e] += __shfl_xor(dw[k][e], o);
                    db[k][e] += __shfl_xor(db[k][e], o);
                }
        for (int wv = 0; wv < THREADS / 64; ++wv) {
            if ((int)(threadIdx.x >> 6) == wv && (threadIdx.x & 63) < LPR) {
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const int c = (k * LPR + lane) * VEC + e;
                        acc[0][c] = (wv ? acc[0][c] : 0.f) + dw[k][e];
                        acc[1][c] = (wv ? acc[1][c] : 0.f) + db[k][e];
                    }
            }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < C; c += THREADS) {
            out[c] = acc[0][c];
            out[C + c] = acc[1][c];
        }
    }
}

template <typename T>
__global__ __launch_bounds__(LN_BIG_THREADS) void ln_bwd_big_kernel(LnParams p) {
    constexpr int VEC = 16 / sizeof(T), STEP = LN_BIG_THREADS * VEC;
    __shared__ float red[2 * 2 * (LN_BIG_THREADS / 64)];
    const int C = p.C;
    const float n = (float)C;
    int slot = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.x_stride;
        const T* dy = (const T*)p.dy + row * p.dy_stride;
        T* dx = (T*)p.dx + row * C;
        const float mean = p.mean[row], rstd = p.rstd[row];
        float s[2] = {0.f, 0.f};
        for (int64_t c = threadIdx.x * VEC; c < C; c += STEP) {
            float v[VEC], g[VEC], w[VEC];
            ln_load<T, VEC>(x, c, C, v);
            ln_load<T, VEC>(dy, c, C, g);
            ln_affine<T, VEC>(p.w, p.w32, c, C, 1.f, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {                 // (dy beyond the row is 0)
                s[0] += g[e] * w[e];
                s[1] += g[e] * w[e] * ((v[e] - mean) * rstd);
            }
        }
        ln_sum<LN_BIG_THREADS>(s, red, slot);
        s[0] /= n;
        s[1] /= n;
        for (int64_t c = threadIdx.x * VEC; c < C; c += STEP) {
            float v[VEC], g[VEC], w[VEC];
            ln_load<T, VEC>(x, c, C, v);
            ln_load<T, VEC>(dy, c, C, g);
            ln_affine<T, VEC>(p.w, p.w32, c, C, 1.f, w);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = rstd * (g[e] * w[e] - s[0] - (v[e] - mean) * rstd * s[1]);
            ln_store<T, VEC>(dx, c, C, v);
        }
    }
}

// column sums of the long rows: blockIdx.x owns 256 vectors of columns, blockIdx.y every gridDim.y-th row
template <typename T>
__global__ __launch_bounds__(256) void ln_cols_big_kernel(LnParams p) {
    constexpr int VEC = 16 / sizeof(T);
    const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC, C = p.C;
    if (c >= C) return;
    float dw[VEC] = {}, db[VEC] = {};
    for (int64_t row = blockIdx.y; row < p.rows; row += gridDim.y) {
        const float mean = p.mean[row], rstd = p.rstd[row];
        float v[VEC], g[VEC];
        ln_load<T, VEC>((const T*)p.x + row * p.x_stride, c, C, v);
        ln_load<T, VEC>((const T*)p.dy + row * p.dy_stride, c, C, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            dw[e] += g[e] * ((v[e] - mean) * rstd);
            db[e] += g[e];
        }
    }
    float* out = p.ws + (int64_t)blockIdx.y * 2 * C;
    ln_store<float, VEC>(out, c, C, dw);
    ln_store<float, VEC>(out + C, c, C, db);
}

// ws [parts][2 C] -> dw, db.  32 columns x 32 row groups a workgroup, the groups added in index order.
template <typename TW>
__global__ __launch_bounds__(1024) void ln_reduce_kernel(const float* __restrict__ ws, int parts, int64_t C, TW* __restrict__ dw, TW* __restrict__ db) {
    __shared__ float acc[32][33];
    const int g = threadIdx.x >> 5;
    for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < 2 * C; c0 += (int64_t)gridDim.x * 32) {
        const int64_t c = c0 + (threadIdx.x & 31);
        float s = 0.f;
        if (c < 2 * C) {
#pragma unroll 8
            for (int r = g; r < parts; r += 32) s += ws[(int64_t)r * 2 * C + c];
        }
        acc[g][threadIdx.x & 31] = s;
        __syncthreads();
        if (g == 0 && c < 2 * C) {
            float t = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i) t += acc[i][threadIdx.x & 31];
            TW* d = c < C ? dw : db;
            if (d) d[c < C ? c : c - C] = (TW)t;
        }
        __syncthreads();
    }
}

// Lanes per row and vectors per lane of a row of `nv` 16-byte vectors; f(LPR, K) as integral constants; false: a long row.
// Two vectors a lane halve the shuffles, but a wave is kept to one row, or a workgroup of 256 to one, as long as its loads are enough.  Training step of
// bfloat16 rows, against half / twice the lanes: 64 channels 247 us (4 x 2: 271), 256: 234 (32 x 1: 245), 512: 234 (64 x 1: 245), 1024: 228 (256 x 1: 411),
// 2048: 247 (64 x 4: 333), 4096: 243 (512 x 1: 268), each of 1.2e8 elements.
template <typename F>
static bool ln_plan(int64_t nv, F&& f) {
#define LN_CASE(limit, lpr, k) \
    if (nv <= (limit)) { f(std::integral_constant<int, lpr>(), std::integral_constant<int, k>()); return true; }
    LN_CASE(4, 4, 1)
    LN_CASE(8, 8, 1)
    LN_CASE(16, 8, 2)
    LN_CASE(32, 16, 2)
    LN_CASE(64, 32, 2)
    LN_CASE(128, 64, 2)
    LN_CASE(256, 256, 1)
    LN_CASE(512, 256, 2)
    LN_CASE(1024, 512, 2)
    LN_CASE(2048, 1024, 2)
#undef LN_CASE
    return false;
}

// Workgroups of the backward pass, and rows of its partial column sums: 262144 threads in all.  16384 x 4096 bfloat16: 142 us with 1024 workgroups of 256, 183
// with half and 157 with twice as many (a part is written and read again for every workgroup); 4000 x 8192: 101 with 512 of 512, 112 with 1024.
static int ln_parts(int64_t rows, int64_t C, int dtype) {
    const int64_t nv = cdiv64(C, dtype == N3D_F32 ? 4 : 8);
    int64_t n = 0;
    int64_t most = 0;
    if (ln_plan(nv, [&](auto lpr, auto) {
            n = cdiv64(rows, ln_threads(lpr.value) / lpr.value);
            most = 1024 * 256 / ln_threads(lpr.value);
        }))
        return (int)(n < most ? n : most);
    return (int)(rows < 64 ? rows : 64);
}

static const char* ln_check(const LnParams& p, int dtype, int w_dtype) {
    if (dtype != N3D_F32 && dtype != N3D_F16 && dtype != N3D_BF16) return "unsupported dtype";
    if (w_dtype != N3D_F32 && w_dtype != dtype) return "weight and bias are float32 or have the type of x";
    if (p.rows < 0 || p.rows > 0x7fffffff || p.C < 1) return "bad sizes";
    if (!p.x) return "null tensor";
    return nullptr;
}

extern "C" int n3d_layer_norm(const void* x, const void* w, const void* b, void* y, float* mean, float* rstd, int64_t rows, int C, int64_t x_stride, int dtype,
                              int w_dtype, float eps, n3d_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    LnParams p = {x, w, b, nullptr, y, nullptr, mean, rstd, nullptr, rows, x_stride, 0, C, w_dtype == N3D_F32, eps};
    if (rows == 0) return 0;
    const char* bad = ln_check(p, dtype, w_dtype);
    N3D_CHECK(!bad, "layer_norm: %s", bad);
    N3D_CHECK(y && (!mean) == (!rstd), "layer_norm: null tensor");
    N3D_CHECK(eps >= 0.f, "layer_norm: eps must not be negative");
    const double esize = dtype == N3D_F32 ? 4.0 : 2.0;
    N3dProfScope prof(N3D_K_LAYER_NORM, stream, 8.0 * rows * C, 2.0 * esize * rows * C);
    token_dispatch(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool ok = ln_plan(cdiv64(C, 16 / sizeof(T)), [&](auto lpr, auto k) {
            const int64_t want = cdiv64(rows, ln_threads(lpr.value) / lpr.value);
            hipLaunchKernelGGL((ln_fwd_kernel<T, lpr.value, k.value>), dim3((unsigned)(want < 4096 ? want : 4096)), dim3(ln_threads(lpr.value)), 0, stream, p);
        });
        if (!ok) hipLaunchKernelGGL((ln_fwd_big_kernel<T>), dim3((unsigned)(rows < 1024 ? rows : 1024)), dim3(LN_BIG_THREADS), 0, stream, p);
    });
    N3D_LAUNCH_CHECK();
    return 0;
}

extern "C" int64_t n3d_layer_norm_bwd_workspace(int64_t rows, int C, int dtype) {
    if (rows <= 0 || C < 1) return 0;
    return (int64_t)ln_parts(rows, C, dtype) * 2 * C;
}

extern "C" int n3d_layer_norm_bwd(const void* dy, const void* x, const void* w, const float* mean, const float* rstd, void* dx, void* dw, void* db, float* workspace,
                                  int64_t rows, int C, int64_t x_stride, int64_t dy_stride, int dtype, int w_dtype, n3d_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    const bool cols = dw || db;
    LnParams p = {x, w, nullptr, dy, nullptr, dx, (float*)mean, (float*)rstd, cols ? workspace : nullptr, rows, x_stride, dy_stride, C, w_dtype == N3D_F32, 0.f};
    N3D_CHECK(rows > 0, "layer_norm_bwd: no rows");
    const char* bad = ln_check(p, dtype, w_dtype);
    N3D_CHECK(!bad, "layer_norm_bwd: %s", bad);
    N3D_CHECK(dy && mean && rstd && (!cols || workspace), "layer_norm_bwd: null tensor");
    if (!dx && !cols) return 0;
    const double esize = dtype == N3D_F32 ? 4.0 : 2.0;
    N3dProfScope prof(N3D_K_LAYER_NORM, stream, 14.0 * rows * C, 3.0 * esize * rows * C);
    const int parts = ln_parts(rows, C, dtype);
    token_dispatch(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const bool ok = ln_plan(cdiv64(C, 16 / sizeof(T)), [&](auto lpr, auto k) {
            hipLaunchKernelGGL((ln_bwd_kernel<T, lpr.value, k.value>), dim3(parts), dim3(ln_threads(lpr.value)), 0, stream, p);
        });
        if (!ok) {
            if (dx) hipLaunchKernelGGL((ln_bwd_big_kernel<T>), dim3((unsigned)(rows < 1024 ? rows : 1024)), dim3(LN_BIG_THREADS), 0, stream, p);
            if (cols) hipLaunchKernelGGL((ln_cols_big_kernel<T>), dim3((unsigned)cdiv64(C, 256 * (16 / sizeof(T))), parts), dim3(256), 0, stream, p);
        }
    });
    N3D_LAUNCH_CHECK();
    if (cols) {
        const int64_t blocks = cdiv64(2 * (int64_t)C, 32), most = 1 << 20;          // (2^32 threads are more than a launch can have)
        token_dispatch(w_dtype, [&](auto* t) {
            using TW = std::remove_pointer_t<decltype(t)>;
            hipLaunchKernelGGL((ln_reduce_kernel<TW>), dim3((unsigned)(blocks < most ? blocks : most)), dim3(1024), 0, stream, workspace, parts, (int64_t)C, (TW*)dw, (TW*)db);
        });
        N3D_LAUNCH_CHECK();
    }
    return 0;
}
