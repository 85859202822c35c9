// Whole-sequence attention: argument checks, the rules that split the work, and the entry points.
#include "attn_seq.h"

namespace {

constexpr long long MAX_STRIDE = 1ll << 40;
// A tile's rows are addressed by 31-bit byte offsets from its first: up to 64 positions and the heads of one position
constexpr long long MAX_TILE_BYTES = 1ll << 30;

int head_columns(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256; }

int check_tensor(const char* who, const char* name, const void* p, const int64_t st[3], int heads, int dtype, bool empty) {
    if (empty) return 0;
    MIC_ARG_CHECK(p, "%s: %s is a null pointer", who, name);
    const int e = 16 / (int)mic_dtype_size(dtype);
    MIC_ARG_CHECK(((uintptr_t)p & 15) == 0, "%s: %s is not 16-byte aligned", who, name);
    for (int i = 0; i < 3; ++i)
        MIC_ARG_CHECK(st[i] >= 0 && st[i] < MAX_STRIDE && st[i] % e == 0, "%s: stride %lld of %s is not a multiple of 16 bytes", who, (long long)st[i], name);
    MIC_ARG_CHECK(64 * st[1] * (16 / e) <= MAX_TILE_BYTES && heads * st[2] * (16 / e) <= MAX_TILE_BYTES, "%s: strides %lld, %lld of %s are too large", who, (long long)st[1],
                  (long long)st[2], name);
    return 0;
}

int check_sizes(const char* who, const mic_attn_seq_desc* d) {
    MIC_ARG_CHECK(d, "%s: null descriptor", who);
    MIC_ARG_CHECK(d->dtype == MIC_F32 || d->dtype == MIC_BF16, "%s: bad dtype %d", who, d->dtype);
    MIC_ARG_CHECK(d->B >= 0 && d->Tq >= 0 && d->Tk >= 0 && d->Hq > 0 && d->Hkv > 0 && d->D > 0, "%s: bad sizes B=%d Tq=%d Tk=%d Hq=%d Hkv=%d D=%d", who, d->B, d->Tq,
                  d->Tk, d->Hq, d->Hkv, d->D);
    MIC_ARG_CHECK(d->Hq % d->Hkv == 0, "%s: %d query heads do not share %d key heads evenly", who, d->Hq, d->Hkv);
    MIC_ARG_CHECK(d->D <= 256 && d->D % (16 / (int)mic_dtype_size(d->dtype)) == 0, "%s: heads of %d columns (at most 256, whole 16 bytes)", who, d->D);
    // row and key numbers have 32 bits, and a launch has fewer than 2^32 threads (the short forward four workgroups of 256 to 128 rows)
    const long long lim = 1ll << 30, tiles = 1ll << 22;
    const long long group = d->Hq / d->Hkv, R = d->Tq * group;
    MIC_ARG_CHECK(d->Hq <= 1 << 15 && R < lim && d->Tk < lim && ((R + 127) / 128) * d->Hkv * (long long)d->B < tiles && (((long long)d->Tk + 127) / 128) * d->Hkv * (long long)d->B < tiles,
                  "%s: too many rows (B=%d Tq=%d Tk=%d Hq=%d)", who, d->B, d->Tq, d->Tk, d->Hq);
    return 0;
}

AttnSeqArgs args_of(const mic_attn_seq_desc* d) {
    AttnSeqArgs a = {};
    a.q = d->q; a.k = d->k; a.v = d->v; a.g = d->grad_o;
    a.o = d->o; a.dq = d->dq; a.dk = d->dk; a.dv = d->dv;
    a.lse = d->lse;
    a.mask = d->key_mask; a.mask_sb = d->mask_stride;
    a.q_sb = d->q_stride[0]; a.q_st = d->q_stride[1]; a.q_sh = d->q_stride[2];
    a.k_sb = d->k_stride[0]; a.k_st = d->k_stride[1]; a.k_sh = d->k_stride[2];
    a.v_sb = d->v_stride[0]; a.v_st = d->v_stride[1]; a.v_sh = d->v_stride[2];
    a.o_sb = d->o_stride[0]; a.o_st = d->o_stride[1]; a.o_sh = d->o_stride[2];
    a.g_sb = d->g_stride[0]; a.g_st = d->g_stride[1]; a.g_sh = d->g_stride[2];
    a.B = d->B; a.Tq = d->Tq; a.Tk = d->Tk; a.Hq = d->Hq; a.Hkv = d->Hkv; a.D = d->D;
    a.group = d->Hq / d->Hkv;
    a.R = d->Tq * a.group;
    a.causal = d->causal != 0;
    a.off = d->Tk - d->Tq;
    a.scale = d->scale;
    a.scale_log2 = d->scale * ATTN_LOG2E;
    a.splits = a.dq_splits = 1;
    a.group_magic = a.group > 1 ? (unsigned)(((1ull << 32) + a.group - 1) / a.group) : 0;
    return a;
}

constexpr int SHORT_KEYS = 64;
// One tile of keys: the kernels of attn_seq_short.hip.  Their forward reads the keys again for every 32 rows, the general one for every
// 128, which wins from 128 rows on where there are rows enough to fill the GPU.
bool short_grad(const AttnSeqArgs& a) { return a.Tk > 0 && a.Tk <= SHORT_KEYS; }
bool short_fwd(const AttnSeqArgs& a) { return short_grad(a) && (a.R <= 128 || (long long)a.B * a.Hkv * a.R < 256 * 128); }

// The forward shares the keys of a row tile out over workgroups when row tiles leave a third of the compute units idle: one tile of keys
// per workgroup at least, 512 workgroups at most.
void split_keys(AttnSeqArgs& a, int dtype) {
    const int BK = head_columns(a.D) * (int)mic_dtype_size(dtype) <= 256 ? 64 : 32;
    const long long base = (long long)((a.R + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK) * a.Hkv * a.B;
    const int tiles = (a.Tk + BK - 1) / BK;
    a.splits = 1;
    a.tiles_per_split = tiles;
    if (short_fwd(a) || base == 0 || base >= 160 || tiles < 4) return;
    const int want = (int)((512 + base - 1) / base);  // at most 512: the join's table
    const int s = want < tiles ? want : tiles;
    a.tiles_per_split = (tiles + s - 1) / s;
    a.splits = (tiles + a.tiles_per_split - 1) / a.tiles_per_split;
}
// Row tiles (of 32) that see any key of key tile kt
int row_tiles_of(const AttnSeqArgs& a, int kt) {
    const long long first = a.causal ? ((long long)kt * ATTN_SEQ_BLOCK - a.off > 0 ? ((long long)kt * ATTN_SEQ_BLOCK - a.off) * a.group : 0) : 0;
    return (a.R + 31) / 32 - (int)((first < a.R ? first : a.R) / 32);
}
// The key gradients share the rows out where key tiles alone leave compute units idle: every workgroup takes `tiles_per_split` row tiles
// of a key tile, as many as make 512 workgroups (two to a compute unit), at least four (one with a single tile of keys).  Under
// causality the first keys are seen by the most rows and get the most workgroups: 2 x 4096 queries of 16 heads, a fixed number of
// ranges per key tile took 518 us, ranges of equal length 400 us.  Without it 1024 workgroups: a mask leaves some with little to do
// (9 x 333 queries, 391 keys, 8 heads of 64, padded, fp32: 45 us where 512 took 56; 1024 under causality: the same, and a join of 24 us
// instead of 13).
void split_rows(AttnSeqArgs& a, int dtype) {
    split_keys(a, dtype);  // the query gradients' rule is the forward's, whichever kernel takes the forward
    a.dq_splits = short_grad(a) ? 1 : a.splits;
    const int tiles_k = (a.Tk + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK;
    const long long base = (long long)tiles_k * a.Hkv * a.B;
    const int least = short_grad(a) ? 1 : 4, tiles = (a.R + 31) / 32;
    a.splits = 1;
    a.tiles_per_split = tiles;
    if (base == 0 || base >= 512 || tiles == 0) return;
    long long work = 0;
    int longest = 0;
    for (int kt = 0; kt < tiles_k; ++kt) {
        const int n = short_grad(a) ? tiles : row_tiles_of(a, kt);
        work += n;
        if (n > longest) longest = n;
    }
    work *= (long long)a.Hkv * a.B;
    // every key tile's last range is half empty on average
    const long long room = short_grad(a) ? 512 : (a.causal ? 512 : 1024) - base / 2;
    long long per = (work + room - 1) / room;
    if (per < least) per = least;
    if (per >= longest) return;
    a.splits = (int)((longest + per - 1) / per);
    a.tiles_per_split = a.causal ? (int)per : (longest + a.splits - 1) / a.splits;  // all key tiles alike: even ranges
}

long long up256(long long b) { return (b + 255) / 256 * 256; }
long long fwd_rows(const AttnSeqArgs& a) { return (long long)a.splits * a.B * a.Hkv * a.R; }
long long fwd_bytes(const AttnSeqArgs& a) { return a.splits > 1 ? up256(fwd_rows(a) * a.D * 4) + up256(fwd_rows(a) * 8) : 0; }
long long delta_bytes(const AttnSeqArgs& a) { return up256((long long)a.B * a.Hq * a.Tq * 4); }
// the partial sums of dQ and, after them, of dK and dV lie in the same place
long long grad_bytes(const AttnSeqArgs& a) {
    const long long q = a.dq_splits > 1 ? up256((long long)a.dq_splits * a.B * a.Tq * a.Hq * a.D * 4) : 0;
    const long long kv = a.splits > 1 ? up256(2ll * a.splits * a.B * a.Tk * a.Hkv * a.D * 4) : 0;
    return delta_bytes(a) + (q > kv ? q : kv);
}

}  // namespace

extern "C" int64_t mic_attn_seq_workspace_bytes(const mic_attn_seq_desc* d, int grad) {
    MIC_TRY(check_sizes("mic_attn_seq_workspace_bytes", d));
    AttnSeqArgs a = args_of(d);
    if (grad) {
        split_rows(a, d->dtype);
        return grad_bytes(a);
    }
    split_keys(a, d->dtype);
    return fwd_bytes(a);
}

extern "C" int mic_attn_seq(const mic_attn_seq_desc* d, void* stream) {
    const char* who = "mic_attn_seq";
    MIC_TRY(check_sizes(who, d));
    AttnSeqArgs a = args_of(d);
    const bool no_rows = d->B == 0 || d->Tq == 0, no_keys = d->B == 0 || d->Tk == 0;
    if (no_rows) return 0;
    MIC_TRY(check_tensor(who, "q", d->q, d->q_stride, d->Hq, d->dtype, false));
    MIC_TRY(check_tensor(who, "k", d->k, d->k_stride, d->Hkv, d->dtype, no_keys));
    MIC_TRY(check_tensor(who, "v", d->v, d->v_stride, d->Hkv, d->dtype, no_keys));
    MIC_TRY(check_tensor(who, "o", d->o, d->o_stride, d->Hq, d->dtype, false));
    MIC_ARG_CHECK(d->lse, "%s: lse is a null pointer", who);
    split_keys(a, d->dtype);
    const long long need = fwd_bytes(a);
    MIC_ARG_CHECK(need == 0 || (d->workspace && d->workspace_bytes >= need && ((uintptr_t)d->workspace & 15) == 0), "%s: workspace of %lld bytes, %lld needed", who,
                  (long long)d->workspace_bytes, need);
    if (need) {
        a.part = (float*)d->workspace;
        a.part_ml = (float*)((char*)d->workspace + up256(fwd_rows(a) * a.D * 4));
    }
    if (short_fwd(a)) return mic_attn_seq_short_fwd_launch(a, d->dtype, (hipStream_t)stream);
    return mic_attn_seq_fwd_launch(a, d->dtype, (hipStream_t)stream);
}

extern "C" int mic_attn_seq_grad(const mic_attn_seq_desc* d, void* stream) {
    const char* who = "mic_attn_seq_grad";
    MIC_TRY(check_sizes(who, d));
    AttnSeqArgs a = args_of(d);
    const bool no_rows = d->B == 0 || d->Tq == 0, no_keys = d->B == 0 || d->Tk == 0;
    MIC_TRY(check_tensor(who, "q", d->q, d->q_stride, d->Hq, d->dtype, no_rows));
    MIC_TRY(check_tensor(who, "k", d->k, d->k_stride, d->Hkv, d->dtype, no_keys));
    MIC_TRY(check_tensor(who, "v", d->v, d->v_stride, d->Hkv, d->dtype, no_keys));
    MIC_TRY(check_tensor(who, "o", d->o, d->o_stride, d->Hq, d->dtype, no_rows));
    MIC_TRY(check_tensor(who, "grad_o", d->grad_o, d->g_stride, d->Hq, d->dtype, no_rows));
    MIC_ARG_CHECK(no_rows || (d->lse && d->dq), "%s: lse or dq is a null pointer", who);
    MIC_ARG_CHECK(no_keys || (d->dk && d->dv), "%s: dk or dv is a null pointer", who);
    MIC_ARG_CHECK((((uintptr_t)d->dq | (uintptr_t)d->dk | (uintptr_t)d->dv) & 15) == 0, "%s: a gradient is not 16-byte aligned", who);
    split_rows(a, d->dtype);
    const long long need = grad_bytes(a);
    MIC_ARG_CHECK(need == 0 || (d->workspace && d->workspace_bytes >= need && ((uintptr_t)d->workspace & 15) == 0), "%s: workspace of %lld bytes, %lld needed", who,
                  (long long)d->workspace_bytes, need);
    a.delta = (float*)d->workspace;
    a.part = (float*)((char*)d->workspace + delta_bytes(a));
    if (!no_rows && short_grad(a)) return mic_attn_seq_short_grad_launch(a, d->dtype, (hipStream_t)stream);
    if (!no_rows) MIC_TRY(mic_attn_seq_dq_launch(a, d->dtype, (hipStream_t)stream));
    if (!no_keys) MIC_TRY(mic_attn_seq_dkv_launch(a, d->dtype, (hipStream_t)stream));
    return 0;
}
