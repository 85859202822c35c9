// Whole-sequence attention, gradient of the queries:  P = exp(scale * q k^T - lse) is recomputed tile by tile,
//   delta = g . o   dS = P (g v^T - delta)   dq = scale * dS k
// Split as the forward (attn_seq_fwd.hip): a wave holds 32 rows' q and g as B operands, walks the keys, and dS^T is the B operand
// of dQ^T = K^T dS^T.  Also leaves delta for the key-gradient kernel.
#include "attn_seq.h"

namespace {

template <typename T, int DP, int BK> __global__ __launch_bounds__(256) void attn_seq_dq_kernel(AttnSeqArgs a) {
    constexpr int NC = DP / 16, ND = DP / 32, KT = BK / 32, NR = InRegs<T, DP>::value ? NC : 1;
    __shared__ __attribute__((aligned(16))) T sk[BK * DP];
    __shared__ __attribute__((aligned(16))) T sv[BK * DP];
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_r = (a.R + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK, id = blockIdx.x;
    const int rt = tiles_r - 1 - id % tiles_r, hk = id / tiles_r % a.Hkv, b = id / tiles_r / a.Hkv;
    const int r0 = rt * ATTN_SEQ_BLOCK + wave * 32, r = r0 + (lane & 31);
    const bool row_ok = r < a.R;
    const int qi = row_ok ? r / a.group : 0, qh = hk * a.group + (row_ok ? r - qi * a.group : 0);
    const T* qrow = row_ok ? (const T*)a.q + b * a.q_sb + qi * a.q_st + qh * a.q_sh : nullptr;
    const T* grow = row_ok ? (const T*)a.g + b * a.g_sb + qi * a.g_st + qh * a.g_sh : nullptr;
    const T* orow = row_ok ? (const T*)a.o + b * a.o_sb + qi * a.o_st + qh * a.o_sh : nullptr;
    Frag8<T> qf[NR], gf[NR];
    float delta = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const Frag8<T> g = load_frag<T>(grow, 16 * c + 8 * h, a.D), o = load_frag<T>(orow, 16 * c + 8 * h, a.D);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)g.v[e], (float)o.v[e], delta);
        if constexpr (InRegs<T, DP>::value) {
            gf[c] = g;
            qf[c] = load_frag<T>(qrow, 16 * c + 8 * h, a.D);
        }
    }
    delta += __shfl_xor(delta, 32, 64);
    const long long at = ((long long)b * a.Hq + qh) * a.Tq + qi;
    float lse2 = INFINITY;  // a row that sees nothing, or is none: every probability is zero
    if (row_ok) {
        if (h == 0) a.delta[at] = delta;
        const float x = a.lse[at];
        lse2 = x == -INFINITY ? INFINITY : x * ATTN_LOG2E;
    }
    const int last = min(rt * ATTN_SEQ_BLOCK + ATTN_SEQ_BLOCK, a.R) - 1;
    const int k_end = a.causal ? min(a.Tk, last / a.group + a.off + 1) : a.Tk;
    const int w_last = min(r0 + 31, a.R - 1);
    const int w_end = r0 < a.R ? (a.causal ? min(a.Tk, w_last / a.group + a.off + 1) : a.Tk) : 0;
    const int lim = a.causal ? qi + a.off : a.Tk - 1;
    f32x16_t acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16_t{};
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    for (int k0 = 0; k0 < k_end; k0 += BK) {
        __syncthreads();
        stage<T, DP, BK, 256>(sk, a.D, [&](int x) { return key_seen(a, b, k0 + x) ? kb + (long long)(k0 + x) * a.k_st : nullptr; });
        stage<T, DP, BK, 256>(sv, a.D, [&](int x) { return key_seen(a, b, k0 + x) ? vb + (long long)(k0 + x) * a.v_st : nullptr; });
        __syncthreads();
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            if (k0 + kt * 32 >= w_end) continue;
            f32x16_t s = f32x16_t{}, dp = f32x16_t{};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if constexpr (InRegs<T, DP>::value) {
                    mma32(read_row<DP>(sk, kt * 32 + (lane & 31), c, h), qf[c], s);
                    mma32(read_row<DP>(sv, kt * 32 + (lane & 31), c, h), gf[c], dp);
                } else {
                    mma32(read_row<DP>(sk, kt * 32 + (lane & 31), c, h), load_frag<T>(qrow, 16 * c + 8 * h, a.D), s);
                    mma32(read_row<DP>(sv, kt * 32 + (lane & 31), c, h), load_frag<T>(grow, 16 * c + 8 * h, a.D), dp);
                }
            }
            const unsigned bits = key_bits(a, b, k0 + kt * 32, lane) >> (4 * h);
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int j = 8 * (e >> 2) + (e & 3);
                const bool seen = ((bits >> j) & 1) && k0 + kt * 32 + 4 * h + j <= lim;
                const float p = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, -lse2));
                s[e] = seen ? p * (dp[e] - delta) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const Frag8<T> ds = frag_of<T>(s, j);  // bf16: rounded for the product
#pragma unroll
                for (int d = 0; d < ND; ++d) mma32(read_col<DP>(sk, d * 32, kt * 32 + 16 * j, lane), ds, acc[d]);
            }
        }
    }
    if (!row_ok) return;
    T* dq = (T*)a.dq + (((long long)b * a.Tq + qi) * a.Hq + qh) * a.D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = d * 32 + 8 * e + 4 * h;
            if (col < a.D)
                store4<T>(dq + col, acc[d][4 * e] * a.scale, acc[d][4 * e + 1] * a.scale, acc[d][4 * e + 2] * a.scale, acc[d][4 * e + 3] * a.scale);
        }
}

template <typename T, int DP> int launch(const AttnSeqArgs& a, hipStream_t s) {
    constexpr int BK = KeyTile<T, DP>::value;
    const long long blocks = (long long)((a.R + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK) * a.Hkv * a.B;
    MIC_LAUNCH((attn_seq_dq_kernel<T, DP, BK>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    return 0;
}
template <typename T> int launch_d(const AttnSeqArgs& a, hipStream_t s) {
    return a.D <= 32 ? launch<T, 32>(a, s) : a.D <= 64 ? launch<T, 64>(a, s) : a.D <= 128 ? launch<T, 128>(a, s) : launch<T, 256>(a, s);
}

}  // namespace

int mic_attn_seq_dq_launch(const AttnSeqArgs& a, int dtype, hipStream_t s) {
    return dtype == MIC_BF16 ? launch_d<bf16_t>(a, s) : launch_d<float>(a, s);
}
