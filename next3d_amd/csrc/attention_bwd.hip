// Attention, backward: how the work is split, where the workspace's parts lie, and the C entry (the kernels: attention_bwd.h).
#include "attention.h"

void attn_bwd_f16(AttnParams& p, hipStream_t stream);                      // attention_bwd_f16.hip
void attn_bwd_bf16(AttnParams& p, hipStream_t stream);                     // attention_bwd_bf16.hip

// How the gradients' work is split (attn_room)
static void attn_bwd_split(AttnParams& p) {
    p.row_blocks = cdiv(p.Lq, 128);
    p.splits = attn_room((int64_t)p.B * p.Hq * p.row_blocks, p.nkt);
    // dk / dv: a group's heads in as many runs as fill the chip (256 workgroups beyond 96 channels, 512 up to there), or fill it twice where the diagonal
    // or documents leave long and short ones.  Training step of 2 x 4096 x 16 heads on 4: causal x 128, 1024 -> 512 workgroups: 755 -> 727 us (half the parts);
    // causal x 64: 467, at 512 518; no mask x 128, 512 -> 256: 1337 -> 1317; documents x 128: 492, at 256 526; documents x 64: 310, at 512 342.
    p.k_blocks = cdiv(p.Lk, 128);
    const int64_t groups = (int64_t)p.B * p.Hk * (p.Lk ? p.k_blocks : 1), fill = (p.D > 96 ? 256 : 512) * (p.causal || p.kdoc ? 2 : 1);
    int heads = 1;
    while (heads < p.G && (p.G % heads || groups * heads < fill)) ++heads;
    p.chunks = heads < p.G ? 1 : attn_room(groups * heads, p.nqt);
    p.k_splits = heads * p.chunks;
}

// Where the workspace's parts lie, in floats: document ranges and order, delta, parts of dq, parts of dk and dv, the end
struct AttnBwdSpace {
    int64_t delta, part, k_part, end;
};
static AttnBwdSpace attn_bwd_plan(AttnParams& p) {
    attn_bwd_split(p);
    AttnBwdSpace at;
    at.delta = (attn_range_floats(p) + 3) / 4 * 4;
    at.part = at.delta + ((int64_t)p.B * p.Hq * p.Lq + 3) / 4 * 4;
    at.k_part = at.part + (p.splits > 1 ? (int64_t)p.splits * p.B * p.Lq * p.Hq * p.D : 0);
    at.end = at.k_part + (p.k_splits > 1 ? 2 * (int64_t)p.k_splits * p.B * p.Lk * p.Hk * p.D : 0);
    return at;
}

// (pairs of waves in dk / dv beyond 96 channels: 512 threads)
static bool attn_bwd_fits(const AttnParams& p) {
    return n3d_grid_fits(attn_even((int64_t)p.B * p.Hq * p.splits * p.row_blocks), 256) && attn_ranges_fit(p) &&
           n3d_grid_fits(attn_even((int64_t)p.B * p.Hk * p.k_splits * p.k_blocks), p.D > 96 ? 512 : 256);
}

extern "C" int64_t n3d_attention_bwd_workspace(const n3d_attention_desc* d) {
    AttnParams p;
    const char* bad = attn_params(d, p);
    N3D_CHECK(!bad, "attention_bwd: %s", bad);
    if (p.B == 0 || p.Lq == 0) return 0;
    const int64_t need = 4 * attn_bwd_plan(p).end;
    N3D_CHECK(attn_bwd_fits(p), "attention_bwd: too many rows for one launch");
    return need;
}

extern "C" int n3d_attention_bwd(const n3d_attention_desc* d, n3d_stream_t stream_) {
    hipStream_t stream = (hipStream_t)stream_;
    AttnParams p;
    const char* bad = attn_params(d, p);
    N3D_CHECK(!bad, "attention_bwd: %s", bad);
    N3D_CHECK(p.B > 0 && p.Lq > 0, "attention_bwd: no queries");
    N3D_CHECK((int64_t)p.B * p.Lq * p.Hq < (1ll << 31) && (int64_t)p.B * p.Lk * p.Hk < (1ll << 31), "attention_bwd: 2^31 rows or more");
    N3D_CHECK(d->lse && d->dout && (!d->dk) == (!d->dv) && (d->dq || d->dk || p.Lk == 0), "attention_bwd: null tensor");
    for (int i = 0; i < 3; ++i)
        N3D_CHECK(d->dout_strides[i] % 8 == 0 && d->dout_strides[i] >= 0 && (i != 1 || d->dout_strides[i] <= (1 << 23)), "attention_bwd: strides must be multiples of 8 elements, of tokens 2^23 at most");
    N3D_CHECK(((uintptr_t)d->dout | (uintptr_t)d->dq | (uintptr_t)d->dk | (uintptr_t)d->dv) % 16 == 0, "attention_bwd: tensors must be 16-byte aligned");
    const AttnBwdSpace at = attn_bwd_plan(p);
    const int64_t need = 4 * at.end;
    N3D_CHECK(attn_bwd_fits(p), "attention_bwd: too many rows for one launch");
    N3D_CHECK(d->workspace && d->workspace_bytes >= need && (uintptr_t)d->workspace % 16 == 0, "attention_bwd: a workspace of %lld bytes is needed (16-byte aligned)", (long long)need);
    float* ws = (float*)d->workspace;
    p.dout = d->dout; p.dq = d->dq; p.dk = d->dk; p.dv = d->dv;
    p.delta = ws + at.delta;
    p.part = ws + at.part;
    p.k_part = ws + at.k_part;
    const double pairs = (double)p.B * p.Hq * p.Lq * p.Lk * p.D;
    N3dProfScope prof(N3D_K_ATTENTION, stream, 10.0 * pairs, 8.0 * ((double)p.B * p.Lq * p.Hq * p.D + (double)p.B * p.Lk * p.Hk * p.D));
    attn_ranges(p, ws, stream);
    if (d->dtype == N3D_F16) attn_bwd_f16(p, stream);
    else attn_bwd_bf16(p, stream);
    N3D_LAUNCH_CHECK();
    return 0;
}
