// Softmax cross entropy of a linear layer over the vocabulary, without keeping the logits:
//   z = x w^T + bias     lse = log sum_v exp z_v     loss = lse - z_target
//   d = weight * (exp(z - lse) - onehot(target))     dx = d w     dw = d^T x     dbias = column sums of d
// Forward: the logits' tiles end in the statistics (maximum, sum) of their 64 columns; a second launch joins a row's parts.
// Gradient: piece by piece of the vocabulary the logits are computed again, their epilogue turns them into d (rounded to bf16 for
// bf16 operands: both remaining products take it as a matrix-core operand; dbias is summed before the rounding), and two more
// products use the piece.  dw's rows of a piece are complete; dx is summed over the pieces in fp32.
#include "vocab_gemm.h"

namespace {

constexpr int MAX_IGNORE = 4;
struct Targets {
    const void* t;
    int wide, n_ignore, V;
    int ignore[MAX_IGNORE];
};
// the row's target, or -1 where the row does not count
__device__ __forceinline__ int target_of(const Targets& t, int row) {
    const long long v = t.wide ? ((const long long*)t.t)[row] : (long long)((const int*)t.t)[row];
    if (v < 0 || v >= t.V) return -1;
    for (int i = 0; i < t.n_ignore; ++i)
        if (v == t.ignore[i]) return -1;
    return (int)v;
}

// ---- epilogue: statistics of 64 columns of logits per row -------------------------------------------------------------------
struct StatsEpi {
    struct Args {
        const float* bias;
        Targets t;
        float2* part;  // [N][parts]
        float* zt;     // [N] logit of the target
        int N, V, parts;
    };
    __device__ static __forceinline__ void run(const Args& a, f32x16_t (&acc)[2][2], int p0, int q0, int lane, int tp, int, int) {
        const int h = lane >> 5;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = q0 + j * 32 + (lane & 31);
            const int t = row < a.N ? target_of(a.t, row) : -1;
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int v = p0 + i * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
                    float z = acc[i][j][e];
                    if (v < a.V) z += a.bias ? a.bias[v] : 0.f;
                    else z = -INFINITY;
                    if (v == t) a.zt[row] = z;
                    acc[i][j][e] = z;
                    m = fmaxf(m, z);
                }
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const float m_use = m == -INFINITY ? 0.f : m;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f((acc[i][j][e] - m_use) * ATTN_LOG2E);
            s += __shfl_xor(s, 32, 64);
            if (h == 0 && row < a.N) a.part[(long long)row * a.parts + tp] = make_float2(m, s);
        }
    }
};

// one wave per row
__global__ __launch_bounds__(256) void vocab_loss_rows_kernel(const float2* __restrict__ part, const float* __restrict__ zt, Targets t, float* __restrict__ loss,
                                                              float* __restrict__ lse, int N, int parts) {
    const int lane = threadIdx.x & 63, row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= N) return;
    const float2* p = part + (long long)row * parts;
    float m = -INFINITY;
    for (int i = lane; i < parts; i += 64) m = fmaxf(m, p[i].x);
    m = wave_max(m);
    const float m_use = m == -INFINITY ? 0.f : m;
    float s = 0.f;
    for (int i = lane; i < parts; i += 64) s += p[i].y * __builtin_amdgcn_exp2f((p[i].x - m_use) * ATTN_LOG2E);
    s = wave_sum(s);
    if (lane == 0) {
        const float l = m + logf(s);
        lse[row] = l;
        loss[row] = target_of(t, row) >= 0 ? l - zt[row] : 0.f;
    }
}

// ---- epilogue: logits -> d --------------------------------------------------------------------------------------------------
template <typename T> struct GradEpi {
    struct Args {
        const float* bias;
        Targets t;
        const float *lse, *weight;
        T* d;            // [N][ld], columns from v0 on
        float* part_db;  // [parts][Vc] or NULL
        int N, V, Vc, ld, v0;
    };
    __device__ static __forceinline__ void run(const Args& a, f32x16_t (&acc)[2][2], int p0, int q0, int lane, int, int tq, int) {
        const int h = lane >> 5;
        float sum[2][16];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = q0 + j * 32 + (lane & 31);
            const int t = row < a.N ? target_of(a.t, row) : -1;
            const float w = t >= 0 ? a.weight[row] : 0.f, lse2 = t >= 0 ? a.lse[row] * ATTN_LOG2E : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const int c = p0 + i * 32 + 8 * e4 + 4 * h;  // column of the piece
                    float d[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int v = a.v0 + c + e;
                        float z = acc[i][j][4 * e4 + e];
                        if (a.bias && c + e < a.Vc) z += a.bias[v];
                        const float p = __builtin_amdgcn_exp2f(fmaf(z, ATTN_LOG2E, -lse2));
                        d[e] = t >= 0 && c + e < a.Vc ? w * (v == t ? p - 1.0f : p) : 0.f;
                        sum[i][4 * e4 + e] = (j ? sum[i][4 * e4 + e] : 0.f) + d[e];
                    }
                    if (row < a.N && c < a.ld) store4<T>(a.d + (long long)row * a.ld + c, d[0], d[1], d[2], d[3]);
                }
        }
        if (a.part_db == nullptr) return;
        // sums over the 32 lanes of a half: every exchange halves the values a lane carries; value x ends in the lane whose low five bits are x
        float v[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) v[x] = sum[x >> 4][x & 15];
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            const bool up = lane & d;
#pragma unroll
            for (int x = 0; x < d; ++x) {
                const float give = up ? v[x] : v[x + d], keep = up ? v[x + d] : v[x];
                v[x] = keep + __shfl_xor(give, d, 64);
            }
        }
        const int x = lane & 31, c = p0 + (x >> 4) * 32 + 8 * ((x & 15) >> 2) + 4 * h + (x & 3);
        if (c < a.Vc) a.part_db[(long long)tq * a.Vc + c] = v[0];
    }
};

// ---- epilogue: fp32 partial results of a slice, or the rounded result ---------------------------------------------------------
template <typename T> struct OutEpi {
    struct Args {
        T* out;       // [Nq][ld] rounded, used with one slice
        float* part;  // [slices][Nq][Np] fp32 otherwise
        long long ld;
        int Np, Nq;
    };
    __device__ static __forceinline__ void run(const Args& a, f32x16_t (&acc)[2][2], int p0, int q0, int lane, int, int, int slice) {
        const int h = lane >> 5;
        const bool whole = a.Np % 4 == 0 && a.ld % 4 == 0;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int row = q0 + j * 32 + (lane & 31);
            if (row >= a.Nq) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const int c = p0 + i * 32 + 8 * e4 + 4 * h;
                    const float v[4] = {acc[i][j][4 * e4], acc[i][j][4 * e4 + 1], acc[i][j][4 * e4 + 2], acc[i][j][4 * e4 + 3]};
                    if (a.part) {
                        float* o = a.part + ((long long)slice * a.Nq + row) * a.Np + c;
                        if (whole && c < a.Np) store4<float>(o, v[0], v[1], v[2], v[3]);
                        else if (!whole)
                            for (int e = 0; e < 4; ++e)
                                if (c + e < a.Np) o[e] = v[e];
                    } else {
                        T* o = a.out + (long long)row * a.ld + c;
                        if (whole && c < a.Np) store4<T>(o, v[0], v[1], v[2], v[3]);
                        else if (!whole)
                            for (int e = 0; e < 4; ++e)
                                if (c + e < a.Np) o[e] = from_f32<T>(v[e]);
                    }
                }
        }
    }
};

// out = the sum of `parts` fp32 matrices [rows][cols], in order
template <typename T> __global__ __launch_bounds__(256) void vocab_sum_parts_kernel(const float* __restrict__ part, T* __restrict__ out, long long n, int parts) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (n % 4 == 0) {
        if (i * 4 >= n) return;
        float4 s = make_float4(0, 0, 0, 0);
        for (int k = 0; k < parts; ++k) {
            const float4 p = *reinterpret_cast<const float4*>(part + k * n + i * 4);
            s.x += p.x; s.y += p.y; s.z += p.z; s.w += p.w;
        }
        store4<T>(out + i * 4, s.x, s.y, s.z, s.w);
    } else {
        for (long long e = i * 4; e < n && e < i * 4 + 4; ++e) {
            float s = 0.f;
            for (int k = 0; k < parts; ++k) s += part[k * n + e];
            out[e] = from_f32<T>(s);
        }
    }
}

// rows of `cols` elements with any stride -> rows of `padded` elements, zeros behind
template <typename T> __global__ __launch_bounds__(256) void vocab_pad_kernel(const T* __restrict__ in, long long ld, T* __restrict__ out, long long rows, int cols, int padded) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * padded) return;
    const long long r = i / padded;
    const int c = (int)(i - r * padded);
    out[i] = c < cols ? in[r * ld + c] : (T)0.f;
}

// ---- plan ---------------------------------------------------------------------------------------------------------------------
long long up256(long long b) { return (b + 255) / 256 * 256; }
int tiles(long long n) { return (int)((n + VT - 1) / VT); }

struct Plan {
    int Hp, e;              // columns of the operands the products read (H rounded up to whole 16 bytes)
    bool pad;               // x and w are copied to that width first
    int parts;              // forward: column parts per row
    int Vc, pieces, ld;     // gradient: words per piece, row stride of d
    int sx, sw;             // slices of k of dx (per piece) and dw
    long long xpad, wpad, part, zt, d, dx, dw, db, bytes;
};

int slices(long long tiles, long long K, int ks) {
    // k is shared out while there are fewer than 512 workgroups and every one keeps 8 steps of k
    long long s = (512 + tiles - 1) / tiles;
    const long long most = (K + ks - 1) / ks / 8;
    if (s > most) s = most;
    if (s > 32) s = 32;
    return (int)(s < 1 ? 1 : s);
}

Plan make_plan(const mic_vocab_loss_desc* d, bool grad) {
    Plan p = {};
    if (d->N == 0) return p;
    const long long N = d->N, H = d->H, V = d->V, es = (long long)mic_dtype_size(d->dtype);
    p.e = 16 / (int)es;
    p.Hp = (int)((H + p.e - 1) / p.e * p.e);
    p.pad = p.Hp != H || d->ld_x % p.e || d->ld_w % p.e || (((uintptr_t)d->x | (uintptr_t)d->w) & 15);
    long long o = 0;
    p.xpad = o;
    if (p.pad) o += up256(N * p.Hp * es);
    p.wpad = o;
    if (p.pad) o += up256(V * p.Hp * es);
    if (!grad) {
        p.parts = tiles(V) * 2;
        p.part = o; o += up256(N * p.parts * 8);
        p.zt = o; o += up256(N * 4);
    } else {
        // a piece of d takes at most 256 MiB (what the last-level cache holds), at least one tile of words
        long long vc = (256ll << 20) / (es * N) / VT * VT;
        if (vc < VT) vc = VT;
        if (vc > V) vc = V;
        p.pieces = (int)((V + vc - 1) / vc);
        p.Vc = (int)(((V + p.pieces - 1) / p.pieces + VT - 1) / VT * VT);
        if (p.Vc > V) p.Vc = (int)V;
        p.pieces = (int)((V + p.Vc - 1) / p.Vc);
        p.ld = (p.Vc + p.e - 1) / p.e * p.e;
        const int ks = 128 / (int)es;
        p.sx = slices((long long)tiles(N) * tiles(H), p.Vc, ks);
        p.sw = slices((long long)tiles(p.Vc) * tiles(H), N, ks);
        p.d = o; o += up256(N * p.ld * es);
        p.dx = o;
        if (p.sx * p.pieces > 1) o += up256((long long)p.sx * p.pieces * N * H * 4);
        p.dw = o;
        if (p.sw > 1) o += up256((long long)p.sw * p.Vc * H * 4);
        p.db = o;
        if (d->db) o += up256((long long)tiles(N) * 2 * V * 4);
    }
    p.bytes = o;
    return p;
}

int check_desc(const char* who, const mic_vocab_loss_desc* d) {
    MIC_ARG_CHECK(d, "%s: null descriptor", who);
    MIC_ARG_CHECK(d->dtype == MIC_F32 || d->dtype == MIC_BF16, "%s: bad dtype %d", who, d->dtype);
    MIC_ARG_CHECK(d->N >= 0 && d->H > 0 && d->V > 0, "%s: bad sizes N=%d H=%d V=%d", who, d->N, d->H, d->V);
    const long long lim = 1ll << 30;
    MIC_ARG_CHECK(d->N < lim && d->H < lim && d->V < lim && (long long)(tiles(d->N) + 1) * (tiles(d->V) + 1) < lim / 32 && (long long)(tiles(d->N) + 1) * (tiles(d->H) + 1) < lim / 32 &&
                      (long long)(tiles(d->V) + 1) * (tiles(d->H) + 1) < lim / 32,
                  "%s: sizes out of range N=%d H=%d V=%d", who, d->N, d->H, d->V);
    MIC_ARG_CHECK(d->target_bits == 32 || d->target_bits == 64, "%s: targets of %d bits", who, d->target_bits);
    MIC_ARG_CHECK(d->n_ignore >= 0 && d->n_ignore <= MAX_IGNORE, "%s: %d ignored words (at most %d)", who, d->n_ignore, MAX_IGNORE);
    MIC_ARG_CHECK(d->ld_x >= d->H && d->ld_w >= d->H, "%s: row stride below H=%d", who, d->H);
    return 0;
}

Targets targets_of(const mic_vocab_loss_desc* d) {
    Targets t = {};
    t.t = d->targets; t.wide = d->target_bits == 64; t.n_ignore = d->n_ignore; t.V = d->V;
    for (int i = 0; i < d->n_ignore; ++i) t.ignore[i] = d->ignore[i];
    return t;
}

template <typename T, bool PCOL, bool QCOL, typename Epi> int gemm(const Operand& p, const Operand& q, int K, int slices, const typename Epi::Args& ea, hipStream_t s) {
    GemmShape g = {p, q, K, tiles(p.n), tiles(q.n), slices};
    MIC_LAUNCH((vocab_gemm_kernel<T, PCOL, QCOL, Epi>), dim3((unsigned)((long long)g.tiles_p * g.tiles_q * slices)), dim3(256), 0, s, g, ea);
    return 0;
}

// x and w as the products read them: in place, or copied to whole 16-byte rows
template <typename T> int operands(const mic_vocab_loss_desc* d, const Plan& p, char* ws, Operand& x, Operand& w, hipStream_t s) {
    x = {d->x, d->ld_x, d->N};
    w = {d->w, d->ld_w, d->V};
    if (!p.pad) return 0;
    T *xp = (T*)(ws + p.xpad), *wp = (T*)(ws + p.wpad);
    const long long nx = (long long)d->N * p.Hp, nw = (long long)d->V * p.Hp;
    MIC_LAUNCH((vocab_pad_kernel<T>), dim3((unsigned)((nx + 255) / 256)), dim3(256), 0, s, (const T*)d->x, (long long)d->ld_x, xp, (long long)d->N, d->H, p.Hp);
    MIC_LAUNCH((vocab_pad_kernel<T>), dim3((unsigned)((nw + 255) / 256)), dim3(256), 0, s, (const T*)d->w, (long long)d->ld_w, wp, (long long)d->V, d->H, p.Hp);
    x = {xp, p.Hp, d->N};
    w = {wp, p.Hp, d->V};
    return 0;
}

template <typename T> int forward(const mic_vocab_loss_desc* d, const Plan& p, hipStream_t s) {
    char* ws = (char*)d->workspace;
    Operand x, w;
    MIC_TRY(operands<T>(d, p, ws, x, w, s));
    StatsEpi::Args ea = {};
    ea.bias = d->bias; ea.t = targets_of(d);
    ea.part = (float2*)(ws + p.part); ea.zt = (float*)(ws + p.zt);
    ea.N = d->N; ea.V = d->V; ea.parts = p.parts;
    MIC_TRY((gemm<T, false, false, StatsEpi>(w, x, d->H, 1, ea, s)));
    MIC_LAUNCH(vocab_loss_rows_kernel, dim3((d->N + 3) / 4), dim3(256), 0, s, (const float2*)ea.part, (const float*)ea.zt, ea.t, d->loss, d->lse, d->N, p.parts);
    return 0;
}

template <typename T> int sum_parts(const float* part, void* out, long long n, int parts, hipStream_t s) {
    MIC_LAUNCH((vocab_sum_parts_kernel<T>), dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, s, part, (T*)out, n, parts);
    return 0;
}

template <typename T> int gradient(const mic_vocab_loss_desc* d, const Plan& p, hipStream_t s) {
    char* ws = (char*)d->workspace;
    Operand x, w;
    MIC_TRY(operands<T>(d, p, ws, x, w, s));
    const long long N = d->N, H = d->H;
    T* dl = (T*)(ws + p.d);
    float *part_dx = (float*)(ws + p.dx), *part_dw = (float*)(ws + p.dw), *part_db = (float*)(ws + p.db);
    for (int i = 0; i < p.pieces; ++i) {
        const int v0 = i * p.Vc, vc = d->V - v0 < p.Vc ? d->V - v0 : p.Vc;
        const Operand wi = {(const T*)w.p + v0 * w.ld, w.ld, vc};
        typename GradEpi<T>::Args ga = {};
        ga.bias = d->bias; ga.t = targets_of(d); ga.lse = d->lse; ga.weight = d->grad_rows;
        ga.d = dl; ga.part_db = d->db ? part_db : nullptr;
        ga.N = d->N; ga.V = d->V; ga.Vc = vc; ga.ld = p.ld; ga.v0 = v0;
        MIC_TRY((gemm<T, false, false, GradEpi<T>>(wi, x, d->H, 1, ga, s)));
        if (d->db) MIC_TRY(sum_parts<float>(part_db, d->db + v0, vc, tiles(N) * 2, s));
        // dx += d w: k runs over the words of the piece
        typename OutEpi<T>::Args xa = {};
        xa.out = (T*)d->dx; xa.ld = H; xa.Np = d->H; xa.Nq = d->N;
        if (p.sx * p.pieces > 1) xa.part = part_dx + (long long)i * p.sx * N * H;
        const Operand wc = {wi.p, wi.ld, d->H}, dr = {dl, p.ld, d->N};
        MIC_TRY((gemm<T, true, false, OutEpi<T>>(wc, dr, vc, p.sx, xa, s)));
        // dw = d^T x: k runs over the rows
        typename OutEpi<T>::Args wa = {};
        wa.out = (T*)d->dw + v0 * H; wa.ld = H; wa.Np = d->H; wa.Nq = vc;
        if (p.sw > 1) wa.part = part_dw;
        const Operand xc = {x.p, x.ld, d->H}, dc = {dl, p.ld, vc};
        MIC_TRY((gemm<T, true, true, OutEpi<T>>(xc, dc, d->N, p.sw, wa, s)));
        if (p.sw > 1) MIC_TRY(sum_parts<T>(part_dw, wa.out, vc * H, p.sw, s));
    }
    if (p.sx * p.pieces > 1) MIC_TRY(sum_parts<T>(part_dx, d->dx, N * H, p.sx * p.pieces, s));
    return 0;
}

__global__ __launch_bounds__(256) void vocab_clear_kernel(uint16_t* p, long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

}  // namespace

extern "C" int64_t mic_vocab_loss_workspace_bytes(const mic_vocab_loss_desc* d, int grad) {
    MIC_TRY(check_desc("mic_vocab_loss_workspace_bytes", d));
    return make_plan(d, grad != 0).bytes;
}

static int check_call(const char* who, const mic_vocab_loss_desc* d, const Plan& p) {
    MIC_ARG_CHECK(d->N == 0 || (d->x && d->w && d->targets && d->lse), "%s: null pointer", who);
    MIC_ARG_CHECK(p.bytes == 0 || (d->workspace && d->workspace_bytes >= p.bytes && ((uintptr_t)d->workspace & 15) == 0), "%s: workspace of %lld bytes, %lld needed", who,
                  (long long)d->workspace_bytes, p.bytes);
    return 0;
}

extern "C" int mic_vocab_loss(const mic_vocab_loss_desc* d, void* stream) {
    const char* who = "mic_vocab_loss";
    MIC_TRY(check_desc(who, d));
    const Plan p = make_plan(d, false);
    MIC_TRY(check_call(who, d, p));
    if (d->N == 0) return 0;
    MIC_ARG_CHECK(d->loss, "%s: null pointer", who);
    return d->dtype == MIC_BF16 ? forward<bf16_t>(d, p, (hipStream_t)stream) : forward<float>(d, p, (hipStream_t)stream);
}

extern "C" int mic_vocab_loss_grad(const mic_vocab_loss_desc* d, void* stream) {
    const char* who = "mic_vocab_loss_grad";
    MIC_TRY(check_desc(who, d));
    const Plan p = make_plan(d, true);
    MIC_TRY(check_call(who, d, p));
    MIC_ARG_CHECK(d->dw && (d->N == 0 || (d->dx && d->grad_rows)), "%s: null pointer", who);
    MIC_ARG_CHECK((((uintptr_t)d->dx | (uintptr_t)d->dw | (uintptr_t)d->db) & 15) == 0, "%s: a gradient is not 16-byte aligned", who);
    hipStream_t s = (hipStream_t)stream;
    if (d->N == 0) {  // no rows: the sums over them are zero
        const long long n = (long long)d->V * d->H * (long long)mic_dtype_size(d->dtype) / 2;
        MIC_LAUNCH(vocab_clear_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, (uint16_t*)d->dw, n);
        if (d->db) MIC_LAUNCH(vocab_clear_kernel, dim3((unsigned)((2ll * d->V + 255) / 256)), dim3(256), 0, s, (uint16_t*)d->db, 2ll * d->V);
        return 0;
    }
    return d->dtype == MIC_BF16 ? gradient<bf16_t>(d, p, s) : gradient<float>(d, p, s);
}
