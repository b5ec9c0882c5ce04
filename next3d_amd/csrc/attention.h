// What the attention kernels share (attention_fwd.hip, attention_bwd.hip): parameters, the visibility rule, matrix fragments and tile staging.
//
// Score of query i (of Lq) and key j (of the n in use) of one head:   t = scale * q.k;   t = cap tanh(t / cap);   t -= slope |i + n - Lq - j|
// visible:  j < n,  and (not causal, or j <= i + n - Lq, or j < prefix),  and (no documents, or doc(i) == doc(j) >= 0).
// Scores are kept in base 2 (t log2 e), softmax statistics and every accumulator in float32.
//
// Matrix layout (v_mfma_f32_32x32x16: operand element e of lane (l31, half) is row / column l31, k = 8 half + e; accumulator register r is row
// 8 (r / 4) + 4 half + r % 4, column l31).  Products are arranged so that a lane owns ONE column — a query in the forward and dq kernels, a key in the
// dk / dv kernel — and the 16 scores a lane holds are, in register order, the second operand of the next product: k is only a name for "which row", so
// that product's first operand is read with the same naming (two transposed LDS reads of four rows each).  Scores never leave their lane.
#pragma once
#include "common.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void attn_lds_void;

static constexpr float ATTN_LOG2E = 1.4426950408889634f, ATTN_LN2 = 0.6931471805599453f;
static constexpr int ATTN_TILE = 64;                 // keys (queries in the dk / dv kernel) of an LDS tile, and of a document range

struct AttnParams {
    const void *q, *k, *v, *o, *dout;
    void *out, *rest, *dq, *dk, *dv;
    float* lse;
    int64_t qs[3], ks[3], vs[3], ds[3];              // element strides (batch, token, head) of q, k, v, dout; out / dq / dk / dv are dense
    const int *prefix, *lengths, *qdoc, *kdoc;
    int64_t qdoc_stride, kdoc_stride;
    const float* slopes;
    const int2 *ktiles, *qtiles;                     // lowest and highest document of every ATTN_TILE keys / queries, [B][nkt] / [B][nqt] (attn_ranges_kernel)
    float* delta;                                    // [B][Hq][Lq]
    float* part;                                     // partial results of split kernels
    int64_t part_ml;                                 // offset of their statistics in `part`
    int B, Lq, Lk, Hq, Hk, G, D, nkt, nqt, causal, row_blocks;
    const int* order;                                // [B, row blocks of queries], the longest first, or null: the last first
    int splits;                                      // workgroups a row block's work is split over
    // the dk / dv kernel's own: blocks of keys, workgroups a block's work is split over, of them over the queries of a head; its parts
    int k_blocks, k_splits, chunks, first_k;         // (first_k: where its workgroups begin in a launch of both kinds)
    float* k_part;
    float scale, softcap;
};

template <typename T> struct AttnVec;
template <> struct AttnVec<_Float16> { typedef _Float16 x8 __attribute__((ext_vector_type(8))); typedef _Float16 x4 __attribute__((ext_vector_type(4))); };
template <> struct AttnVec<__bf16> { typedef __bf16 x8 __attribute__((ext_vector_type(8))); typedef __bf16 x4 __attribute__((ext_vector_type(4))); };

__device__ __forceinline__ f32x16 attn_mfma(AttnVec<_Float16>::x8 a, AttnVec<_Float16>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 attn_mfma(AttnVec<__bf16>::x8 a, AttnVec<__bf16>::x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// the other half's value (lane ^ 32) folded in
__device__ __forceinline__ void attn_halves(float x, float& lower, float& upper) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t a = r[0], b = r[1];                       // (a bit cast straight from r[1] reads r[0])
    lower = __builtin_bit_cast(float, a);
    upper = __builtin_bit_cast(float, b);
}
__device__ __forceinline__ float attn_half_max(float x) {
    float a, b;
    attn_halves(x, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float attn_half_sum(float x) {
    float a, b;
    attn_halves(x, a, b);
    return a + b;
}
__device__ __forceinline__ int attn_uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// keys in use / last visible key of query i without documents (-1: none)
__device__ __forceinline__ int attn_keys(const AttnParams& p, int b) {
    const int n = p.lengths ? p.lengths[b] : p.Lk;
    return n < 0 ? 0 : n < p.Lk ? n : p.Lk;
}
__device__ __forceinline__ int attn_prefix(const AttnParams& p, int b) { return p.prefix ? max(p.prefix[b], 0) : 0; }
__device__ __forceinline__ int attn_limit(const AttnParams& p, int i, int n, int prefix) {
    int lim = n - 1;
    if (p.causal) {
        int c = i + n - p.Lq;
        c = c > prefix - 1 ? c : prefix - 1;
        lim = c < lim ? c : lim;
    }
    return lim < -1 ? -1 : lim;
}

// base-2 score of a raw product, and the factor d t / d (scale q.k) of the cap
struct AttnScore {
    float mul, cap_in, cap_out, slope;               // mul: scale log2 e;  cap_in: 2 scale log2 e / cap;  cap_out: cap log2 e;  slope: slope log2 e
    __device__ AttnScore(const AttnParams& p, int head) {
        mul = p.scale * ATTN_LOG2E;
        cap_in = p.softcap > 0.f ? fminf(fmaxf(2.f * ATTN_LOG2E * p.scale / p.softcap, -3e38f), 3e38f) : 0.f;      // (finite: a zero stays a zero)
        cap_out = p.softcap > 0.f ? p.softcap * ATTN_LOG2E : 0.f;
        slope = p.slopes ? p.slopes[head] * ATTN_LOG2E : 0.f;
    }
    // tanh x = 1 - 2 r with r = 1 / (1 + e^2x), off by some 2^-23 absolutely, 2^-23 cap of a score;  1 - tanh^2 = 4 (r - r^2)
    __device__ __forceinline__ float cap_r(float s) const { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * cap_in)); }
    // the capped score less `sub`
    __device__ __forceinline__ float capped(float r, float sub) const { return __builtin_fmaf(-2.f * cap_out, r, cap_out - sub); }
};

// ---- LDS tiles: ROW channels of 16 bits a row (64 or 128; channels beyond D are zero), rows of 16-byte chunks.  Chunk c of row r sits at c ^ swizzle(r):
// 16 rows of one chunk, and 4 rows of 4 neighbouring chunks (a transposed read), each touch every bank once.
template <int ROW>
__device__ __forceinline__ int attn_swizzle(int row) {
    if constexpr (ROW == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// One piece: 16 bytes a lane from voff of the buffer to lds + 16 lane (zeros beyond the range).  In asm because the compiler, which sees LDS behind the
// builtin, would wait for every piece in flight before the next LDS read of any buffer.  It has no register result; attn_sync / attn_landed wait for it, and
// the compiler's own vmcnt waits, which do not count it, can only be longer than needed (loads return in order).  Nor does it keep, in asm, the five wait states between a
// vector instruction that writes a scalar register (a readfirstlane, the reload of a spilled descriptor) and a memory instruction that reads it: the move and
// the s_nop are five.  (m0, which the compiler reserves and a clobber list may not name, has no other use in these kernels.)
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void attn_piece(i32x4 rsrc, int voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" : : "s"(lds), "v"(voff), "s"(rsrc) : "memory");
}

// Staging by LDS-DMA: a piece is 1 KB = 64 lanes x 16 bytes; wave w of W takes pieces w, w + W, ...  Rows behind the last and channels behind D are beyond
// the descriptor's range and arrive as zeros.
template <int ROW, int ROWS, int WAVES>
struct AttnStage {
    static constexpr int CHUNKS = ROW / 8, RPP = 64 / CHUNKS, PIECES = ROWS / RPP / WAVES;
    static_assert(PIECES >= 1, "a wave stages whole pieces");
    int voff[PIECES];
    __device__ __forceinline__ void setup(int wave, int lane, int64_t stride, int D) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int row = (wave + i * WAVES) * RPP + lane / CHUNKS, c = (lane % CHUNKS) ^ attn_swizzle<ROW>(row);
            voff[i] = c * 8 < D ? row * (int)stride * 2 + c * 16 : (int)0x80000000;
        }
    }
    // rows [t ROWS, ...) of the `rows` rows at `base` -> lds (t ROWS < rows)
    __device__ __forceinline__ void issue(uint64_t base, int t, int rows, int stride, int D, uint32_t lds, int wave) const {
        const int left = rows - t * ROWS;
        const uint64_t a = base + (uint64_t)(uint32_t)t * (uint32_t)(ROWS * 2 * stride);
        const int n = ((left < ROWS ? left : ROWS) - 1) * stride * 2 + D * 2;
        const i32x4 r = {attn_uniform((int)a), attn_uniform((int)(a >> 32)), attn_uniform(n), 0x00020000};
#pragma unroll
        for (int i = 0; i < PIECES; ++i) attn_piece(r, voff[i], attn_uniform(lds + (wave + i * WAVES) * 1024));
    }
};
__device__ __forceinline__ uint32_t attn_lds(const void* p) { return (uint32_t)(uintptr_t)(attn_lds_void*)p; }
__device__ __forceinline__ uint64_t attn_addr(const void* p) { return (uint64_t)p & 0xffffffffffffull; }       // (48 bits: the descriptor's upper 16 are 0)

// Where a lane reads its fragments of a tile at LDS address `tile` (a multiple of 256).  The compiler would keep every fragment's address in a register of its own across the
// loop; the empty asm makes the two bases new in each iteration, and an exclusive or (chunks) and the instruction's offset (rows) give the rest.
template <int ROW>
struct AttnLane {
    uint32_t row0, col0;
    __device__ __forceinline__ AttnLane(int lane) {
        const int l31 = lane & 31, half = lane >> 5, l16 = lane & 15, r = 4 * half + (l16 >> 2);
        row0 = l31 * (ROW * 2) + ((half ^ attn_swizzle<ROW>(l31)) << 4);
        col0 = r * (ROW * 2) + (((((lane >> 4) & 1) * 2 + ((l16 & 3) >> 1)) ^ attn_swizzle<ROW>(r)) << 4) + (l16 & 1) * 8;
    }
    __device__ __forceinline__ uint32_t rows(uint32_t tile) const {
        uint32_t a = row0 + tile;
        asm volatile("" : "+v"(a));
        return a;
    }
    __device__ __forceinline__ uint32_t cols(uint32_t tile) const {
        uint32_t a = col0 + tile;
        asm volatile("" : "+v"(a));
        return a;
    }
};
// first operand, rows = tile rows 32 block + l31, k = channels 16 c + 8 half + 0..7
template <typename T, int ROW>
__device__ __forceinline__ typename AttnVec<T>::x8 attn_row_frag(uint32_t rows, int block, int c) {
    typedef __attribute__((address_space(3))) const typename AttnVec<T>::x8* ptr;
    return *(ptr)(uintptr_t)((rows ^ (c << 5)) + block * 32 * ROW * 2);
}
// first operand, rows = channels 32 db + l31, k = tile rows 16 block + {4 half + 0..3, 8 + 4 half + 0..3}; eight rows on, bit 1 of the swizzle differs
template <typename T, int ROW>
__device__ __forceinline__ typename AttnVec<T>::x8 attn_col_frag(uint32_t cols, int block, int db) {
    typedef __attribute__((address_space(3))) s16x4* ptr;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)((cols ^ (db << 6)) + block * 16 * ROW * 2));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ptr)(uintptr_t)((cols ^ (db << 6) ^ 32) + block * 16 * ROW * 2 + 8 * ROW * 2));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const s16x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(typename AttnVec<T>::x8, v);
}
// second operand from global memory: column = this lane's row of `p` (null: zeros), k = channels 16 c + 8 half + 0..7
template <typename T>
__device__ __forceinline__ typename AttnVec<T>::x8 attn_lane_frag(const T* p, int chunk, int D) {
    typename AttnVec<T>::x8 z = {};
    return p && chunk * 8 < D ? *reinterpret_cast<const typename AttnVec<T>::x8*>(p + chunk * 8) : z;
}

// Eight values of x that `rounded` holds in 16 bits: what the rounding left over.  The single-token kernel, and workgroups of the others that walk ATTN_FEW
// tiles or fewer, take a second product with it, of the weights and of the dscores, whether or not gradients are wanted (the same call gives the same bits in
// both): rows of a few keys have nothing to average the roundings out (22 causal queries: float16 dq / dk off by 3.4e-4 of their norm without it, 2.0e-4 with
// it, plain float32 arithmetic 2.0e-4).  Such workgroups take every tile as one with a mask, which the code of the others is spared.  In every masked tile of
// long documents it would cost 26 % of the forward pass (2 x 4096 x 16 heads x 64: 73 -> 92 us) and gain little.
static constexpr int ATTN_FEW = 4;
template <typename T>
__device__ __forceinline__ typename AttnVec<T>::x8 attn_left_over(const f32x16& x, typename AttnVec<T>::x8 rounded, int c) {
    typename AttnVec<T>::x8 left;
#pragma unroll
    for (int e = 0; e < 8; ++e) left[e] = (T)(x[8 * c + e] - (float)rounded[e]);
    return left;
}

// this wave's pieces have landed and its LDS accesses are done (the asm for the hardware, the builtin for the compiler's own book-keeping)
__device__ __forceinline__ void attn_landed() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);
}
// ... and every other wave's: a tile buffer changes hands
__device__ __forceinline__ void attn_sync() {
    attn_landed();
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}

// LDS stores of all waves are visible; pieces stay in flight
__device__ __forceinline__ void attn_traded() {
    asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
}

// ---- which tiles to visit: [t, end) in order; with documents only those whose range [lowest, highest] meets [lo, hi] (64 ranges looked at together)
template <bool DOCS>
struct AttnTiles {
    const int2* ranges;
    int t, end, lo, hi, base, low = 0, high = 0;             // low, high: documents of the tile last returned
    uint64_t bits;
    int2 mine;
    __device__ __forceinline__ void start(const int2* r, int first, int stop, int dlo, int dhi) {
        ranges = r; t = first; end = stop; lo = dlo; hi = dhi; bits = 0; base = first - 64;
    }
    // behind the first next(): ATTN_FEW tiles at most (with documents: of the first 128 ranges from where the first such tile lies)
    __device__ __forceinline__ bool few(int lane) const {
        if constexpr (!DOCS) return end - t < ATTN_FEW;
        int more = __popcll(bits);
        if (more < ATTN_FEW && base + 64 < end) {
            const int i = base + 64 + lane;
            const int2 r = i < end ? ranges[i] : make_int2(1, 0);
            more += __popcll(__ballot((i < end) & (r.y >= lo) & (r.x <= hi)));
        }
        return more < ATTN_FEW;
    }
    // the next tile or -1
    __device__ __forceinline__ int next(int lane) {
        if constexpr (!DOCS) return t < end ? t++ : -1;
        while (bits == 0) {
            base += 64;
            if (base >= end) return -1;
            const int i = base + lane;
            mine = i < end ? ranges[i] : make_int2(1, 0);
            bits = __ballot((i < end) & (mine.y >= lo) & (mine.x <= hi));
        }
        const int n = __builtin_ctzll(bits);
        bits &= bits - 1;
        low = __builtin_amdgcn_readlane(mine.x, n);
        high = __builtin_amdgcn_readlane(mine.y, n);
        return attn_uniform(base + n);
    }
};

// base-2 score of raw product s at distance `dist`, in any form
__device__ __forceinline__ float attn_score(const AttnScore& f, float s, float dist) {
    const float u = f.cap_out > 0.f ? f.capped(f.cap_r(s), 0.f) : s * f.mul;
    return u - f.slope * fabsf(dist);
}

// ---- infinities and NaN.  A masked weight is zero, but zero times them is NaN in a matrix product.  Where an accumulator ends as NaN, the workgroup's waves
// take their sums again, each its own 32 columns through its own LDS (attn_out_again, attn_dq_again, attn_dkv_again).  They walk three times, with the products'
// first operands changed in the LDS: ones where a tile holds NaN or infinities of one sign, and ones for the visible pairs as second operands, say what reaches
// a sum; then zeros in their places.  The functions are not inlined (inside the kernels they cost these their registers) and serve every form of the scores;
// a call pays one barrier for them; a training step of 4096 x 4 heads on 2, causal, in which one key of v is NaN takes 9 (64 channels) to 19 (128) times as long.
enum { ATTN_FINITE = 0, ATTN_PLUS = 1, ATTN_MINUS = -1, ATTN_EITHER = 2 };      // what is left of a tile: finite values; ones at NaN and +inf, -inf, both
template <typename T> struct AttnBits;
template <> struct AttnBits<_Float16> { static constexpr short INF = 0x7c00, ONE = 0x3c00; };
template <> struct AttnBits<__bf16> { static constexpr short INF = 0x7f80, ONE = 0x3f80; };
typedef short attn_s16x8 __attribute__((ext_vector_type(8)));
template <typename T, int BYTES>
__device__ __forceinline__ void attn_change(uint32_t tile, int lane, int kind) {
    typedef __attribute__((address_space(3))) attn_s16x8* ptr;
#pragma unroll 1
    for (int at = lane * 16; at < BYTES; at += 1024) {
        attn_s16x8 v = *(ptr)(uintptr_t)(tile + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int size = v[e] & 0x7fff;
            const bool hit = size > AttnBits<T>::INF || (size == AttnBits<T>::INF && (kind == ATTN_EITHER || (v[e] < 0) == (kind == ATTN_MINUS)));
            if (kind == ATTN_FINITE) v[e] = size >= AttnBits<T>::INF ? (short)0 : v[e];
            else v[e] = hit ? AttnBits<T>::ONE : (short)0;
        }
        *(ptr)(uintptr_t)(tile + at) = v;
    }
}
// ones at the registers of `seen`
template <typename T>
__device__ __forceinline__ void attn_ones(uint32_t seen, typename AttnVec<T>::x8 (&out)[2]) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        attn_s16x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = seen >> (8 * c + e) & 1 ? AttnBits<T>::ONE : (short)0;
        out[c] = __builtin_bit_cast(typename AttnVec<T>::x8, v);
    }
}
// a bit for every accumulator that counted something, and what that adds to the sums of another walk
template <int N> struct AttnMarks {
    uint32_t bits[(N + 1) / 2];
    __device__ __forceinline__ void take(const f32x16 (&count)[N]) {
#pragma unroll
        for (int i = 0; i < (N + 1) / 2; ++i) bits[i] = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) bits[i >> 1] |= count[i][r] > 0.f ? 1u << ((i & 1) * 16 + r) : 0u;
    }
    __device__ __forceinline__ void add(f32x16 (&acc)[N], float x) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][r] += bits[i >> 1] >> ((i & 1) * 16 + r) & 1 ? x : 0.f;
    }
};
// the parameters of the running kernel, where a function that is not inlined finds them (a copy on the stack would be scratch memory of every lane)
typedef const __attribute__((address_space(4))) AttnParams* attn_args;
__device__ __forceinline__ attn_args attn_kernel_args() { return (attn_args)__builtin_amdgcn_kernarg_segment_ptr(); }
template <int N>
__device__ __forceinline__ void attn_clear(f32x16 (&acc)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = f32x16{};
}
// does any wave of the workgroup say yes?  (`said`: one word a wave; all of them are behind their last tile then)
template <int WAVES>
__device__ __forceinline__ bool attn_any(bool yes, int wave, uint32_t (&said)[WAVES]) {
    const uint64_t mine = __ballot(yes);
    if ((threadIdx.x & 63) == 0) said[wave] = mine != 0;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all |= said[w];
    return __builtin_expect(attn_uniform(all) != 0, 0);
}
template <int N>
__device__ __forceinline__ bool attn_has_nan(const f32x16 (&acc)[N]) {
    bool nan = false;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) nan = nan || acc[i][r] != acc[i][r];
    return nan;
}

// a row's 32 * DB channels spread over lanes l31 and l31 + 32 -> 16-byte stores (the halves trade their 8-byte runs).  REST: what the rounding left over
template <typename T, int DB, bool REST = false>
__device__ __forceinline__ void attn_store_row(T* row, const f32x16 (&acc)[DB], float by, int half, int D, bool on) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int a = 0; a < 4; a += 2) {
            typename AttnVec<T>::x4 x, y;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float u = acc[db][4 * a + e] * by, w = acc[db][4 * a + 4 + e] * by;
                x[e] = REST ? (T)(u - (float)(T)u) : (T)u;
                y[e] = REST ? (T)(w - (float)(T)w) : (T)w;
            }
            uint2 u = __builtin_bit_cast(uint2, x), w = __builtin_bit_cast(uint2, y);
            const auto r0 = __builtin_amdgcn_permlane32_swap(u.x, w.x, false, false);
            const auto r1 = __builtin_amdgcn_permlane32_swap(u.y, w.y, false, false);
            const int d = 32 * db + 8 * a + 8 * half;
            if (on && d < D) *reinterpret_cast<uint4*>(row + d) = make_uint4(r0[0], r1[0], r0[1], r1[1]);
        }
}
// ... as float32
template <int DB>
__device__ __forceinline__ void attn_store_part(float* row, const f32x16 (&acc)[DB], float by, int half, int D, bool on) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int d = 32 * db + 8 * a + 4 * half;
            if (on && d < D) *reinterpret_cast<float4*>(row + d) = make_float4(acc[db][4 * a] * by, acc[db][4 * a + 1] * by, acc[db][4 * a + 2] * by, acc[db][4 * a + 3] * by);
        }
}
// channels lane and lane + 64 of a finished row -> out (and rest)
template <typename T>
__device__ __forceinline__ void attn_store_pair(const AttnParams& p, int64_t at, const float (&x)[2], float by, int lane) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int d = lane + 64 * c;
        if (d >= p.D) continue;
        const T t = (T)(x[c] * by);
        ((T*)p.out)[at + d] = t;
        if (p.rest) ((T*)p.rest)[at + d] = (T)(x[c] * by - (float)t);
    }
}

// ---- host: a checked descriptor as kernel parameters
// Workgroups that share a row block's walk of `tiles` tiles, where there are `groups` row blocks of all heads: parts cost a round trip through memory and a
// launch, so only as far as the chip has room (two workgroups a CU), in runs of eight tiles at least and from 24 tiles on.
// (Training step of 4096 x 2 heads x 64: 234 -> 121 us, 2 x 1500 x 4 x 64: 95 -> 83; 1100 x 1 x 64, 18 tiles: 77 -> 82 from the launches, hence 24.)
static inline int attn_room(int64_t groups, int tiles) {
    const int64_t s = 512 / groups;
    return groups >= 256 || tiles < 24 ? 1 : (int)(s < tiles / 8 ? s : tiles / 8);
}
// workgroups of the kernels whose workgroups share the XCDs evenly (attn_fwd_kernel)
static inline int64_t attn_even(int64_t workgroups) { return cdiv64(workgroups, 8) * 8; }
static inline const char* attn_params(const n3d_attention_desc* d, AttnParams& p) {
    if (!d) return "null descriptor";
    if (d->B < 0 || d->Lq < 0 || d->Lk < 0) return "negative sizes";
    if (d->dtype != N3D_F16 && d->dtype != N3D_BF16) return "float16 or bfloat16 only";
    if (d->heads_k < 1 || d->heads_q < 1 || d->heads_q % d->heads_k) return "the query heads must be a multiple of the key heads";
    if (d->D < 8 || d->D > 128 || d->D % 8) return "head sizes are multiples of 8 from 8 to 128";
    if ((int64_t)d->B * d->heads_q * ((d->Lq > d->Lk ? d->Lq : d->Lk) / 32 + 1) >= (1 << 28) || d->Lq > (1 << 30) || d->Lk > (1 << 30)) return "too many rows for one launch";
    // (a capped score is off by 2^-22 of the cap: beyond 4096 that is more than the weights' own rounding)
    if (!(fabsf(d->scale) <= 0x1p100f) || !(d->softcap == 0.f || (d->softcap >= 0x1p-100f && d->softcap <= 4096.f))) return "scale within 2^100, softcap 0 or 2^-100 to 4096";
    if (d->prefix && !d->causal) return "a prefix needs causal";
    if ((!d->q_documents) != (!d->k_documents)) return "documents of the queries and of the keys, or neither";
    const bool some = d->B > 0 && d->Lq > 0;
    if (some && (!d->q || !d->out)) return "null tensor";
    if (some && d->Lk > 0 && (!d->k || !d->v)) return "null tensor";
    const int64_t* strides[3] = {d->q_strides, d->k_strides, d->v_strides};
    for (const int64_t* s : strides)
        for (int i = 0; i < 3; ++i)
            if (s[i] % 8 || s[i] < 0 || (i == 1 && s[i] > (1 << 23))) return "strides must be multiples of 8 elements, of tokens 2^23 at most";
    if (((uintptr_t)d->q | (uintptr_t)d->k | (uintptr_t)d->v | (uintptr_t)d->out | (uintptr_t)d->out_rest) % 16) return "tensors must be 16-byte aligned";
    p = AttnParams{};
    p.q = d->q; p.k = d->k; p.v = d->v; p.out = d->out; p.o = d->out; p.rest = d->out_rest; p.lse = d->lse;
    for (int i = 0; i < 3; ++i) {
        p.qs[i] = d->q_strides[i]; p.ks[i] = d->k_strides[i]; p.vs[i] = d->v_strides[i]; p.ds[i] = d->dout_strides[i];
    }
    p.prefix = d->prefix; p.lengths = d->lengths; p.qdoc = d->q_documents; p.kdoc = d->k_documents;
    p.qdoc_stride = d->q_doc_stride; p.kdoc_stride = d->k_doc_stride; p.slopes = d->slopes;
    p.B = d->B; p.Lq = d->Lq; p.Lk = d->Lk; p.Hq = d->heads_q; p.Hk = d->heads_k; p.G = d->heads_q / d->heads_k; p.D = d->D;
    p.nkt = cdiv(d->Lk, ATTN_TILE); p.nqt = cdiv(d->Lq, ATTN_TILE);
    p.causal = d->causal != 0; p.scale = d->scale; p.softcap = d->softcap;
    p.splits = p.k_splits = p.chunks = 1;
    return nullptr;
}

// How a score comes out of the raw product: a positive multiple of it; any multiple and a distance; a cap; a cap and a distance.  Each is straight code of
// its own in the kernels: values that pass through a branch in place cost a register copy each, and no product is scheduled across it.
enum { ATTN_PLAIN = 0, ATTN_BIAS = 1, ATTN_CAP = 2, ATTN_CAP_BIAS = 3 };
// f(32-channel blocks, mode, documents), as integral constants
template <typename F>
static inline void attn_forms(const AttnParams& p, F&& f) {
    auto doc = [&](auto db, auto mode) {
        if (p.kdoc) f(db, mode, std::true_type());
        else f(db, mode, std::false_type());
    };
    auto form = [&](auto db) {
        if (p.softcap > 0.f) {
            if (p.slopes) doc(db, std::integral_constant<int, ATTN_CAP_BIAS>());
            else doc(db, std::integral_constant<int, ATTN_CAP>());
        } else {
            if (p.slopes || !(p.scale > 0.f)) doc(db, std::integral_constant<int, ATTN_BIAS>());
            else doc(db, std::integral_constant<int, ATTN_PLAIN>());
        }
    };
    switch (cdiv(p.D, 32)) {
        case 1: form(std::integral_constant<int, 1>()); break;
        case 2: form(std::integral_constant<int, 2>()); break;
        case 3: form(std::integral_constant<int, 3>()); break;
        default: form(std::integral_constant<int, 4>()); break;
    }
}

// workspace, in floats: the document ranges come first
// do the launches of attn_ranges fit? (the order of the blocks is left out where its own does not)
static inline bool attn_ranges_fit(const AttnParams& p) { return !p.kdoc || n3d_grid_fits((int64_t)p.B * cdiv(p.nkt > p.nqt ? p.nkt : p.nqt, 4), 256); }
static inline int64_t attn_range_floats(const AttnParams& p) { return p.kdoc ? 2 * (int64_t)p.B * (p.nkt + p.nqt) + (int64_t)p.B * cdiv(p.Lq, 128) : 0; }
void attn_ranges(AttnParams& p, void* workspace, hipStream_t stream);      // attention_fwd.hip
