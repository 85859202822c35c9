// Whole-sequence attention, gradients of the keys and values:
//   dv = P^T g     dk = scale * dS^T q     over all rows (queries of every head of the group) that see the key
// A wave owns 32 keys: their k and v stay in registers as B operands, S = Q K^T and dP = G V^T come out with a lane per key, and P
// and dS are the B operands of dV^T = G^T P and dK^T = Q^T dS.  The workgroup's four waves walk the same tiles of 32 rows.
// With `splits` the rows are shared out over several workgroups, which leave fp32 partial sums that a second launch adds in order.
#include "attn_seq.h"

namespace {

template <typename T, int DP, bool SPLIT> __global__ __launch_bounds__(256) void attn_seq_dkv_kernel(AttnSeqArgs a) {
    constexpr int NC = DP / 16, ND = DP / 32, NR = InRegs<T, DP>::value ? NC : 1;
    __shared__ __attribute__((aligned(16))) T sq[32 * DP];
    __shared__ __attribute__((aligned(16))) T sg[32 * DP];
    __shared__ float s_lse[32], s_delta[32];
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_k = (a.Tk + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK;
    int id = blockIdx.x;
    const int split = SPLIT ? id % a.splits : 0;
    if (SPLIT) id /= a.splits;
    const int kt = id % tiles_k, hk = id / tiles_k % a.Hkv, b = id / tiles_k / a.Hkv;  // the first keys, which the most rows see, first
    const int k0 = kt * ATTN_SEQ_BLOCK + wave * 32, key = k0 + (lane & 31);
    const bool seen = key_seen(a, b, key);
    const T* krow = seen ? (const T*)a.k + b * a.k_sb + hk * a.k_sh + (long long)key * a.k_st : nullptr;
    const T* vrow = seen ? (const T*)a.v + b * a.v_sb + hk * a.v_sh + (long long)key * a.v_st : nullptr;
    Frag8<T> kf[NR], vf[NR];
    if constexpr (InRegs<T, DP>::value) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            kf[c] = load_frag<T>(krow, 16 * c + 8 * h, a.D);
            vf[c] = load_frag<T>(vrow, 16 * c + 8 * h, a.D);
        }
    }
    // rows below `first` see no key of the workgroup (of the wave: w_first)
    const int first = a.causal ? max(0, kt * ATTN_SEQ_BLOCK - a.off) * a.group : 0, w_first = a.causal ? max(0, k0 - a.off) * a.group : 0;
    int t0 = min(first, a.R) / 32, t1 = (a.R + 31) / 32;
    if (SPLIT) {
        t0 = max(t0, split * a.tiles_per_split);
        t1 = min(t1, (split + 1) * a.tiles_per_split);
    }
    f32x16_t dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16_t{};
    for (int t = t0; t < t1; ++t) {
        const int r0 = t * 32;
        auto row_of = [&](const void* p, long long sb, long long st, long long sh, int x) -> const T* {
            const int r = r0 + x;
            if (r >= a.R) return nullptr;
            const int qi = r / a.group;
            return (const T*)p + b * sb + qi * st + (hk * a.group + r - qi * a.group) * sh;
        };
        __syncthreads();
        stage<T, DP, 32, 256>(sq, a.D, [&](int x) { return row_of(a.q, a.q_sb, a.q_st, a.q_sh, x); });
        stage<T, DP, 32, 256>(sg, a.D, [&](int x) { return row_of(a.g, a.g_sb, a.g_st, a.g_sh, x); });
        if (threadIdx.x < 32) {
            const int r = r0 + threadIdx.x;
            float lse2 = INFINITY, delta = 0.f;
            if (r < a.R) {
                const int qi = r / a.group;
                const long long at = ((long long)b * a.Hq + hk * a.group + r - qi * a.group) * a.Tq + qi;
                const float x = a.lse[at];
                lse2 = x == -INFINITY ? INFINITY : x * ATTN_LOG2E;
                delta = a.delta[at];
            }
            s_lse[threadIdx.x] = lse2;
            s_delta[threadIdx.x] = delta;
        }
        __syncthreads();
        if (k0 >= a.Tk || r0 + 31 < w_first) continue;
        f32x16_t s = f32x16_t{}, dp = f32x16_t{};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            if constexpr (InRegs<T, DP>::value) {
                mma32(read_row<DP>(sq, lane & 31, c, h), kf[c], s);
                mma32(read_row<DP>(sg, lane & 31, c, h), vf[c], dp);
            } else {
                mma32(read_row<DP>(sq, lane & 31, c, h), load_frag<T>(krow, 16 * c + 8 * h, a.D), s);
                mma32(read_row<DP>(sg, lane & 31, c, h), load_frag<T>(vrow, 16 * c + 8 * h, a.D), dp);
            }
        }
        // a query sees this lane's key from row (key - off) * group on
        const int from = !seen ? 0x7fffffff : a.causal ? max(0, key - a.off) * a.group : 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int x = 8 * (e >> 2) + 4 * h + (e & 3);
            const bool ok = r0 + x >= from;
            const float p = ok ? __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, -s_lse[x])) : 0.f;
            s[e] = p;
            dp[e] = ok ? p * (dp[e] - s_delta[x]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const Frag8<T> p = frag_of<T>(s, j), ds = frag_of<T>(dp, j);  // bf16: rounded for the products
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                mma32(read_col<DP>(sg, d * 32, 16 * j, lane), p, dv[d]);
                mma32(read_col<DP>(sq, d * 32, 16 * j, lane), ds, dk[d]);
            }
        }
    }
    if (key >= a.Tk) return;
    const long long at = (((long long)b * a.Tk + key) * a.Hkv + hk) * a.D, all = (long long)a.B * a.Tk * a.Hkv * a.D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = d * 32 + 8 * e + 4 * h;
            if (col >= a.D) continue;
            const float x[4] = {dk[d][4 * e] * a.scale, dk[d][4 * e + 1] * a.scale, dk[d][4 * e + 2] * a.scale, dk[d][4 * e + 3] * a.scale};
            if (SPLIT) {
                float* p = a.part + 2 * split * all + at + col;
                store4<float>(p, x[0], x[1], x[2], x[3]);
                store4<float>(p + all, dv[d][4 * e], dv[d][4 * e + 1], dv[d][4 * e + 2], dv[d][4 * e + 3]);
            } else {
                store4<T>((T*)a.dk + at + col, x[0], x[1], x[2], x[3]);
                store4<T>((T*)a.dv + at + col, dv[d][4 * e], dv[d][4 * e + 1], dv[d][4 * e + 2], dv[d][4 * e + 3]);
            }
        }
}

// adds the partial sums of all row ranges, four elements per thread
template <typename T> __global__ __launch_bounds__(256) void attn_seq_dkv_join_kernel(AttnSeqArgs a) {
    const long long all = (long long)a.B * a.Tk * a.Hkv * a.D, i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= 2 * all) return;
    float x[4] = {};
    for (int s = 0; s < a.splits; ++s) {
        const float4 p = *reinterpret_cast<const float4*>(a.part + 2 * s * all + i);
        x[0] += p.x; x[1] += p.y; x[2] += p.z; x[3] += p.w;
    }
    store4<T>(i < all ? (T*)a.dk + i : (T*)a.dv + (i - all), x[0], x[1], x[2], x[3]);
}

template <typename T> int join(const AttnSeqArgs& a, hipStream_t s) {
    const long long quads = (long long)a.B * a.Tk * a.Hkv * a.D / 2;
    MIC_LAUNCH((attn_seq_dkv_join_kernel<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, a);
    return 0;
}

template <typename T, int DP> int launch(const AttnSeqArgs& a, hipStream_t s) {
    const long long blocks = (long long)((a.Tk + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK) * a.Hkv * a.B;
    if (a.splits > 1) {
        MIC_LAUNCH((attn_seq_dkv_kernel<T, DP, true>), dim3((unsigned)(blocks * a.splits)), dim3(256), 0, s, a);
        return join<T>(a, s);
    } else {
        MIC_LAUNCH((attn_seq_dkv_kernel<T, DP, false>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    }
    return 0;
}
template <typename T> int launch_d(const AttnSeqArgs& a, hipStream_t s) {
    return a.D <= 32 ? launch<T, 32>(a, s) : a.D <= 64 ? launch<T, 64>(a, s) : a.D <= 128 ? launch<T, 128>(a, s) : launch<T, 256>(a, s);
}

}  // namespace

int mic_attn_seq_dkv_launch(const AttnSeqArgs& a, int dtype, hipStream_t s) {
    return dtype == MIC_BF16 ? launch_d<bf16_t>(a, s) : launch_d<float>(a, s);
}
int mic_attn_seq_dkv_join(const AttnSeqArgs& a, int dtype, hipStream_t s) { return dtype == MIC_BF16 ? join<bf16_t>(a, s) : join<float>(a, s); }
