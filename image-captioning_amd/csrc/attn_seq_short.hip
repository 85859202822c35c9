// Whole-sequence attention where the keys fit one tile (up to 64: captions, the image tokens of a cross-attention).
//
// With 29 queries and 49 keys there is nothing to pipeline: the time is the memory's latency and its bandwidth, so a workgroup loads
// everything once, the products are a handful of MFMAs, and the four waves share them out: the scores by reduction range and key
// tile (partial tiles are exchanged through LDS in register order, so no layout changes), the outputs by columns.
// The gradient is one launch instead of two: it reads q, k, v and the output's gradient once, takes delta as the sum of P dP (no read
// of o, and no rounding of o in it) and keeps dK and dV in registers while it walks the row tiles.
// 256 captions, two heads of 256 columns, bf16: 29 queries and keys 9 us forward (30 MB, 3.4 TB/s) and 17 us backward (53 MB); 29 queries on
// 49 keys 11 and 24 us (that gradient spills 8 of its 256 registers).  fp32: 16 us forward and 41 us backward, 25 and 69 us; with 256 columns
// and several row tiles the gradient spills 43 of 512.
#include "attn_seq.h"

namespace {

typedef float4 Exchange[4][4][64];  // [unit][quad of registers][lane]

__device__ __forceinline__ void give(Exchange& ex, int unit, int lane, const f32x16_t& x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) ex[unit][e][lane] = make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
}
__device__ __forceinline__ void take(const Exchange& ex, int unit, int lane, f32x16_t& x, bool add) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float4 v = ex[unit][e][lane];
        x[4 * e] = add ? x[4 * e] + v.x : v.x;
        x[4 * e + 1] = add ? x[4 * e + 1] + v.y : v.y;
        x[4 * e + 2] = add ? x[4 * e + 2] + v.z : v.z;
        x[4 * e + 3] = add ? x[4 * e + 3] + v.w : v.w;
    }
}

// ---- forward: a workgroup per 32 rows ---------------------------------------------------------------------------------------
template <typename T, int DP, int KT> __global__ __launch_bounds__(256) void attn_seq_short_fwd_kernel(AttnSeqArgs a) {
    constexpr int NC = DP / 16, ND = DP / 32, PARTS = 4 / KT, NU = (NC + PARTS - 1) / PARTS, NDW = (ND + 3) / 4;
    __shared__ __attribute__((aligned(16))) T sv[KT * 32 * DP];
    __shared__ Exchange ex;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_r = (a.R + 31) / 32, id = blockIdx.x, rt = id % tiles_r, hk = id / tiles_r % a.Hkv, b = id / tiles_r / a.Hkv;
    const int r = rt * 32 + (lane & 31);
    const bool row_ok = r < a.R;
    const int qi = row_ok ? r / a.group : 0, qh = hk * a.group + (row_ok ? r - qi * a.group : 0);
    const T* qrow = row_ok ? (const T*)a.q + b * a.q_sb + qi * a.q_st + qh * a.q_sh : nullptr;
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    const int ukt = wave % KT, upart = wave / KT, ukey = ukt * 32 + (lane & 31);
    {  // this wave's part of the scores of key tile ukt
        const T* krow = key_seen(a, b, ukey) ? kb + (long long)ukey * a.k_st : nullptr;
        Frag8<T> kf[NU], qf[NU];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int c = u * PARTS + upart;  // past the head's columns: zeros
            kf[u] = load_frag<T>(krow, 16 * c + 8 * h, a.D);
            qf[u] = load_frag<T>(qrow, 16 * c + 8 * h, a.D);
        }
        stage<T, DP, KT * 32, 256>(sv, a.D, [&](int x) { return key_seen(a, b, x) ? vb + (long long)x * a.v_st : nullptr; });
        f32x16_t s = f32x16_t{};
#pragma unroll
        for (int u = 0; u < NU; ++u) mma32(kf[u], qf[u], s);
        give(ex, wave, lane, s);
    }
    __syncthreads();
    const int lim = a.causal ? qi + a.off : a.Tk - 1;
    f32x16_t s[KT];
    float m = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int p = 0; p < PARTS; ++p) take(ex, p * KT + kt, lane, s[kt], p > 0);
        const unsigned bits = key_bits(a, b, kt * 32, lane) >> (4 * h);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int j = 8 * (e >> 2) + (e & 3);
            const bool seen = ((bits >> j) & 1) && kt * 32 + 4 * h + j <= lim;
            s[kt][e] = seen ? s[kt][e] * a.scale_log2 : -INFINITY;
            m = fmaxf(m, s[kt][e]);
        }
    }
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const float m_use = m == -INFINITY ? 0.f : m;
    float l = 0.f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            s[kt][e] = __builtin_amdgcn_exp2f(s[kt][e] - m_use);
            l += s[kt][e];
        }
    l += __shfl_xor(l, 32, 64);
    Frag8<T> p[KT][2];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
        for (int j = 0; j < 2; ++j) p[kt][j] = frag_of<T>(s[kt], j);
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    T* o = (T*)a.o + b * a.o_sb + qi * a.o_st + qh * a.o_sh;
#pragma unroll
    for (int n = 0; n < NDW; ++n) {
        const int d = n * 4 + wave;
        if (d >= ND) break;
        f32x16_t acc = f32x16_t{};
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int j = 0; j < 2; ++j) mma32(read_col<DP>(sv, d * 32, kt * 32 + 16 * j, lane), p[kt][j], acc);
        if (row_ok)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = d * 32 + 8 * e + 4 * h;
                if (col < a.D) store4<T>(o + col, acc[4 * e] * inv, acc[4 * e + 1] * inv, acc[4 * e + 2] * inv, acc[4 * e + 3] * inv);
            }
    }
    if (row_ok && wave == 0 && h == 0) a.lse[((long long)b * a.Hq + qh) * a.Tq + qi] = l == 0.f ? -INFINITY : (m + log2f(l)) * ATTN_LN2;
}

// ---- gradient: a workgroup per key head (and range of rows) --------------------------------------------------------------------
// ROWS: 0 = all row tiles, 1 = there is one row tile (its dK and dV are written column tile by column tile and need no registers
// of their own), 2 = a range of row tiles, partial sums.  Two workgroups to a compute unit (256 registers a lane) where LDS and
// registers allow it: one loads while the other computes.
template <typename T, int DP, int KT, int ROWS> struct GradOccupancy {
    static constexpr int value = (KT * 32 + 64) * DP * sizeof(T) <= 65536 && (ROWS == 1 || KT == 1 || (sizeof(T) == 2 && DP <= 128)) ? 2 : 1;
};
template <typename T, int DP, int KT, int ROWS>
__global__ __launch_bounds__(256, (GradOccupancy<T, DP, KT, ROWS>::value)) void attn_seq_short_grad_kernel(AttnSeqArgs a) {
    constexpr int NC = DP / 16, ND = DP / 32, HALVES = 2 / KT, NU = NC / HALVES, NDW = (ND + 3) / 4, KP = KT * 32, NDA = ROWS == 1 ? 1 : NDW;
    constexpr bool SPLIT = ROWS == 2;
    __shared__ __attribute__((aligned(16))) T sk[KP * DP];
    __shared__ __attribute__((aligned(16))) T sq[32 * DP];
    __shared__ __attribute__((aligned(16))) T sg[32 * DP];
    __shared__ Exchange ex;  // later P and dS, [32 rows][KP keys] each
    static_assert(2 * 32 * KP * sizeof(T) <= sizeof(Exchange), "P and dS fit");
    T *sp = reinterpret_cast<T*>(&ex), *sd = sp + 32 * KP;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int id = blockIdx.x;
    const int split = SPLIT ? id % a.splits : 0;
    if (SPLIT) id /= a.splits;
    const int hk = id % a.Hkv, b = id / a.Hkv;
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    // units of the score products: 0, 1 = S, 2, 3 = dP; by halves of the columns (one key tile) or by key tiles (two)
    const int utype = wave >> 1, upart = wave & 1, ukey = (KT == 2 ? upart * 32 : 0) + (lane & 31), c0 = KT == 2 ? 0 : upart * NU;
    const T* urow = key_seen(a, b, ukey) ? (utype ? vb + (long long)ukey * a.v_st : kb + (long long)ukey * a.k_st) : nullptr;
    stage<T, DP, KP, 256>(sk, a.D, [&](int x) { return key_seen(a, b, x) ? kb + (long long)x * a.k_st : nullptr; });
    unsigned bits[KT];
    int first = KP;  // the first key that is seen
#pragma unroll
    for (int kt = KT - 1; kt >= 0; --kt) {
        const unsigned all = key_bits(a, b, kt * 32, lane);
        if (all) first = kt * 32 + __builtin_ctz(all);
        bits[kt] = all >> (4 * h);
    }
    // rows below this see nothing: zeros, whatever q and g hold there
    const int blind = first == KP ? a.R : a.causal ? max(0, first - a.off) * a.group : 0;
    auto store = [&](int d, int kt, const f32x16_t& x, const f32x16_t& y) {
        const int key = kt * 32 + (lane & 31);
        if (key >= a.Tk) return;
        const long long at = (((long long)b * a.Tk + key) * a.Hkv + hk) * a.D, all = (long long)a.B * a.Tk * a.Hkv * a.D;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = d * 32 + 8 * e + 4 * h;
            if (col >= a.D) continue;
            if (SPLIT) {
                float* p = a.part + 2 * split * all + at + col;
                store4<float>(p, x[4 * e] * a.scale, x[4 * e + 1] * a.scale, x[4 * e + 2] * a.scale, x[4 * e + 3] * a.scale);
                store4<float>(p + all, y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
            } else {
                store4<T>((T*)a.dk + at + col, x[4 * e] * a.scale, x[4 * e + 1] * a.scale, x[4 * e + 2] * a.scale, x[4 * e + 3] * a.scale);
                store4<T>((T*)a.dv + at + col, y[4 * e], y[4 * e + 1], y[4 * e + 2], y[4 * e + 3]);
            }
        }
    };
    f32x16_t dk[NDA][KT], dv[NDA][KT];
#pragma unroll
    for (int n = 0; n < NDA; ++n)
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) dk[n][kt] = dv[n][kt] = f32x16_t{};
    int t0 = 0, t1 = (a.R + 31) / 32;
    if (SPLIT) {
        t0 = split * a.tiles_per_split;
        t1 = min(t1, t0 + a.tiles_per_split);
    }
    for (int t = t0; t < t1; ++t) {
        auto row_of = [&](const void* p, long long sb, long long st, long long sh, int x) -> const T* {
            const int r = t * 32 + x;
            if (r < blind || r >= a.R) return nullptr;
            const int qi = r / a.group;
            return (const T*)p + b * sb + qi * st + (hk * a.group + r - qi * a.group) * sh;
        };
        const int r = t * 32 + (lane & 31);
        const bool row_ok = r < a.R;
        const int qi = row_ok ? r / a.group : 0, qh = hk * a.group + (row_ok ? r - qi * a.group : 0);
        constexpr bool UREG = NU * sizeof(T) <= 32;  // else (fp32, 256 columns) the wave's operands are loaded as they are used
        Frag8<T> uf[UREG ? NU : 1];
        if constexpr (UREG)
#pragma unroll
            for (int u = 0; u < NU; ++u) uf[u] = load_frag<T>(urow, 16 * (c0 + u) + 8 * h, a.D);
        float lse2 = INFINITY;
        if (row_ok) {
            const float x = a.lse[((long long)b * a.Hq + qh) * a.Tq + qi];
            lse2 = x == -INFINITY ? INFINITY : x * ATTN_LOG2E;
        }
        if (t > t0) __syncthreads();  // the last tile's columns have been read
        stage<T, DP, 32, 256>(sq, a.D, [&](int x) { return row_of(a.q, a.q_sb, a.q_st, a.q_sh, x); });
        stage<T, DP, 32, 256>(sg, a.D, [&](int x) { return row_of(a.g, a.g_sb, a.g_st, a.g_sh, x); });
        __syncthreads();
        {
            f32x16_t x = f32x16_t{};
            const T* rows = utype ? sg : sq;
            if constexpr (UREG) {
#pragma unroll
                for (int u = 0; u < NU; ++u) mma32(uf[u], read_row<DP>(rows, lane & 31, c0 + u, h), x);
            } else {
#pragma unroll 4
                for (int u = 0; u < NU; ++u) mma32(load_frag<T>(urow, 16 * (c0 + u) + 8 * h, a.D), read_row<DP>(rows, lane & 31, c0 + u, h), x);
            }
            give(ex, wave, lane, x);
        }
        __syncthreads();
        f32x16_t s[KT], dp[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            take(ex, kt, lane, s[kt], false);
            take(ex, 2 + kt, lane, dp[kt], false);
            if (KT == 1) {
                take(ex, 1, lane, s[kt], true);
                take(ex, 3, lane, dp[kt], true);
            }
        }
        const int lim = a.causal ? qi + a.off : a.Tk - 1;
        float delta = 0.f;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = 8 * (e >> 2) + (e & 3);
                const bool seen = ((bits[kt] >> j) & 1) && kt * 32 + 4 * h + j <= lim;
                s[kt][e] = seen ? __builtin_amdgcn_exp2f(fmaf(s[kt][e], a.scale_log2, -lse2)) : 0.f;
                dp[kt][e] = seen ? dp[kt][e] : 0.f;
                delta = fmaf(s[kt][e], dp[kt][e], delta);
            }
        delta += __shfl_xor(delta, 32, 64);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[kt][e] = s[kt][e] * (dp[kt][e] - delta);
        __syncthreads();  // every wave has taken the parts
        if (wave < 2) {
            T* to = wave ? sd : sp;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const f32x16_t& x = wave ? dp[kt] : s[kt];
                    const int key = kt * 32 + 8 * e + 4 * h;
                    store4<T>(to + Tile<T, KP>::at(lane & 31, key / Tile<T, KP>::E) + key % Tile<T, KP>::E, x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
                }
        }
        __syncthreads();
        T* dq = (T*)a.dq + (((long long)b * a.Tq + qi) * a.Hq + qh) * a.D;
#pragma unroll
        for (int n = 0; n < NDW; ++n) {
            const int d = n * 4 + wave;
            if (d >= ND) break;
            f32x16_t acc = f32x16_t{};
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int j = 0; j < 2; ++j) mma32(read_col<DP>(sk, d * 32, kt * 32 + 16 * j, lane), frag_of<T>(dp[kt], j), acc);
            if (row_ok)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int col = d * 32 + 8 * e + 4 * h;
                    if (col < a.D) store4<T>(dq + col, acc[4 * e] * a.scale, acc[4 * e + 1] * a.scale, acc[4 * e + 2] * a.scale, acc[4 * e + 3] * a.scale);
                }
            const int at = ROWS == 1 ? 0 : n;
            if (ROWS == 1)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) dk[0][kt] = dv[0][kt] = f32x16_t{};
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const Frag8<T> g = read_col<DP>(sg, d * 32, 16 * j, lane), q = read_col<DP>(sq, d * 32, 16 * j, lane);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    mma32(g, read_col<KP>(sp, kt * 32, 16 * j, lane), dv[at][kt]);
                    mma32(q, read_col<KP>(sd, kt * 32, 16 * j, lane), dk[at][kt]);
                }
            }
            if (ROWS == 1)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) store(d, kt, dk[0][kt], dv[0][kt]);
        }
    }
    if (ROWS == 1) return;
#pragma unroll
    for (int n = 0; n < NDW; ++n) {
        const int d = n * 4 + wave;
        if (d >= ND) break;
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) store(d, kt, dk[n % NDA][kt], dv[n % NDA][kt]);
    }
}

template <typename T, int DP, int KT> int launch_fwd(const AttnSeqArgs& a, hipStream_t s) {
    MIC_LAUNCH((attn_seq_short_fwd_kernel<T, DP, KT>), dim3((unsigned)((long long)((a.R + 31) / 32) * a.Hkv * a.B)), dim3(256), 0, s, a);
    return 0;
}
template <typename T, int DP, int KT> int launch_grad(const AttnSeqArgs& a, hipStream_t s) {
    const long long blocks = (long long)a.Hkv * a.B;
    if (a.splits > 1) {
        MIC_LAUNCH((attn_seq_short_grad_kernel<T, DP, KT, 2>), dim3((unsigned)(blocks * a.splits)), dim3(256), 0, s, a);
        return mic_attn_seq_dkv_join(a, sizeof(T) == 2 ? MIC_BF16 : MIC_F32, s);
    }
    if (a.R <= 32) MIC_LAUNCH((attn_seq_short_grad_kernel<T, DP, KT, 1>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    else MIC_LAUNCH((attn_seq_short_grad_kernel<T, DP, KT, 0>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    return 0;
}

}  // namespace

#define SHORT_D(FN, T, KT) (a.D <= 32 ? FN<T, 32, KT>(a, s) : a.D <= 64 ? FN<T, 64, KT>(a, s) : a.D <= 128 ? FN<T, 128, KT>(a, s) : FN<T, 256, KT>(a, s))
#define SHORT_T(FN, KT) (dtype == MIC_BF16 ? SHORT_D(FN, bf16_t, KT) : SHORT_D(FN, float, KT))
int mic_attn_seq_short_fwd_launch(const AttnSeqArgs& a, int dtype, hipStream_t s) { return a.Tk <= 32 ? SHORT_T(launch_fwd, 1) : SHORT_T(launch_fwd, 2); }
int mic_attn_seq_short_grad_launch(const AttnSeqArgs& a, int dtype, hipStream_t s) { return a.Tk <= 32 ? SHORT_T(launch_grad, 1) : SHORT_T(launch_grad, 2); }
