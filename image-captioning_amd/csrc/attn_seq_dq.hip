// Whole-sequence attention, gradient of the queries:  P = exp(scale * q k^T - lse) is recomputed tile by tile,
//   delta = g . o   dS = P (g v^T - delta)   dq = scale * dS k
// Split as the forward (attn_seq_fwd.hip): a wave holds 32 rows' q and g as B operands, walks the keys, and dS^T is the B operand
// of dQ^T = K^T dS^T.  Also leaves delta for the key-gradient kernel.
#include "attn_seq.h"

namespace {

template <typename T, int DP, int BK> __global__ __launch_bounds__(256, (DP * sizeof(T) <= 256 ? 2 : 1)) void attn_seq_dq_kernel(AttnSeqArgs a) {
    constexpr int NC = DP / 16, ND = DP / 32, KT = BK / 32, NR = InRegs<T, DP>::value ? NC : 1, ES = sizeof(T);
    __shared__ __attribute__((aligned(16))) T sk[2][BK * DP];
    __shared__ __attribute__((aligned(16))) T sv[2][BK * DP];
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_r = (a.R + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK, heads = a.Hkv * a.B, id = blockIdx.x;
    const int rt = tiles_r - 1 - id / heads, hk = id % heads % a.Hkv, b = id % heads / a.Hkv;
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
    const int w_first = min(r0, a.R - 1), w_last = min(r0 + 31, a.R - 1);
    const int w_end = r0 < a.R ? (a.causal ? min(a.Tk, w_last / a.group + a.off + 1) : a.Tk) : 0;
    const int w_all = a.causal ? w_first / a.group + a.off : a.Tk - 1;
    const int lim = a.causal ? qi + a.off : a.Tk - 1;
    f32x16_t acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16_t{};
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    const unsigned k_row = (unsigned)(a.k_st * ES), v_row = (unsigned)(a.v_st * ES), lds_k = lds_address(sk), lds_v = lds_address(sv);
    auto request = [&](int t, int buf, const unsigned (&seen)[KT]) {
        auto row = [&](unsigned stride) {
            return [&, stride](int x) { return (seen[x >> 5] >> (x & 31)) & 1 ? x * stride : 0x80000000u; };
        };
        request_tile<T, DP, BK>(kb + (long long)t * BK * a.k_st, lds_k + buf * BK * DP * ES, a.D, wave, lane, row(k_row));
        request_tile<T, DP, BK>(vb + (long long)t * BK * a.v_st, lds_v + buf * BK * DP * ES, a.D, wave, lane, row(v_row));
    };
    const int t1 = k_end > 0 ? (k_end + BK - 1) / BK : 0;
    unsigned bits[KT], next[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        bits[kt] = key_bits(a, b, kt * 32, lane);
        next[kt] = key_bits(a, b, BK + kt * 32, lane);
    }
    if (t1 > 0) request(0, 0, bits);
    for (int t = 0; t < t1; ++t) {
        const int k0 = t * BK, cur = t & 1;
        tile_landed();
        if (t + 1 < t1) request(t + 1, cur ^ 1, next);
        bool ok[KT];  // the tile after the next
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) ok[kt] = key_seen(a, b, k0 + 2 * BK + kt * 32 + (lane & 31));
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            if (k0 + kt * 32 >= w_end) continue;
            f32x16_t s = f32x16_t{}, dp = f32x16_t{};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                if constexpr (InRegs<T, DP>::value) {
                    mma32(read_row<DP>(sk[cur], kt * 32 + (lane & 31), c, h), qf[c], s);
                    mma32(read_row<DP>(sv[cur], kt * 32 + (lane & 31), c, h), gf[c], dp);
                } else {
                    mma32(read_row<DP>(sk[cur], kt * 32 + (lane & 31), c, h), load_frag<T>(qrow, 16 * c + 8 * h, a.D), s);
                    mma32(read_row<DP>(sv[cur], kt * 32 + (lane & 31), c, h), load_frag<T>(grow, 16 * c + 8 * h, a.D), dp);
                }
            }
            if (bits[kt] == 0xffffffffu && k0 + kt * 32 + 31 <= w_all) {  // nothing hidden: the common case
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, -lse2)) * (dp[e] - delta);
            } else {
                const unsigned mine = bits[kt] >> (4 * h);
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = 8 * (e >> 2) + (e & 3);
                    const bool seen = ((mine >> j) & 1) && k0 + kt * 32 + 4 * h + j <= lim;
                    const float p = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, -lse2));
                    s[e] = seen ? p * (dp[e] - delta) : 0.f;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const Frag8<T> ds = frag_of<T>(s, j);  // bf16: rounded for the product
#pragma unroll
                for (int d = 0; d < ND; ++d) mma32(read_col<DP>(sk[cur], d * 32, kt * 32 + 16 * j, lane), ds, acc[d]);
            }
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            bits[kt] = next[kt];
            next[kt] = (unsigned)__ballot(ok[kt]);
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
