// Whole-sequence attention, gradient of the queries:  P = exp(scale * q k^T - lse) is recomputed tile by tile,
//   delta = g . o   dS = P (g v^T - delta)   dq = scale * dS k
// Split as the forward (attn_seq_fwd.hip): a wave holds 32 rows' q and g as B operands, walks the keys, and dS^T is the B operand
// of dQ^T = K^T dS^T.  Also leaves delta for the key-gradient kernel.  Rows of 512 bytes: g of the four waves lies in LDS, the
// registers are full with q and dQ (in fp32 beyond that: 28 to 60 of them spill).  2 x 4096 causal queries of 16 heads of 128 columns,
// bf16: 226 us, 910 TFLOP/s.  With few rows the keys are shared out as in the forward; the partial sums of dQ are added in order.
// delta needs the row's whole output before the first key, so in bf16 it comes from o as rounded (attn_seq_short.hip, which has all keys at
// hand, sums P dP instead): 4096 causal keys, relative error of dQ 0.00238 from the roundings of dS and dQ, 0.00248 with it.
#include "attn_seq.h"

#include <type_traits>

namespace {

template <typename T, int DP, int BK, bool SPLIT> __global__ __launch_bounds__(256, (DP * sizeof(T) <= 256 ? 2 : 1)) void attn_seq_dq_kernel(AttnSeqArgs a) {
    constexpr int NC = DP / 16, ND = DP / 32, KT = BK / 32, ES = sizeof(T);
    constexpr bool GLDS = sizeof(T) == 2 && DP == 256;
    constexpr int TILE = BK * DP * ES, OFF_K = 0, OFF_V = 2 * TILE, OFF_G = 4 * TILE;  // two tiles of k, two of v, the waves' g
    __shared__ __attribute__((aligned(16))) unsigned char smem[4 * TILE + (GLDS ? 4 * 32 * DP * ES : 0)];
    const lds_bytes_t lds = (lds_bytes_t)smem;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_r = (a.R + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK, heads = a.Hkv * a.B;
    int id = blockIdx.x;
    const int split = SPLIT ? id % a.dq_splits : 0;
    if (SPLIT) id /= a.dq_splits;
    const int rt = tiles_r - 1 - id / heads, hk = id % heads % a.Hkv, b = id % heads / a.Hkv;
    const int r0 = rt * ATTN_SEQ_BLOCK + wave * 32, r = r0 + (lane & 31);
    const bool row_ok = r < a.R;
    const int qi = row_ok ? r / a.group : 0, qh = hk * a.group + (row_ok ? r - qi * a.group : 0);
    const T* qrow = row_ok ? (const T*)a.q + b * a.q_sb + qi * a.q_st + qh * a.q_sh : nullptr;
    const T* grow = row_ok ? (const T*)a.g + b * a.g_sb + qi * a.g_st + qh * a.g_sh : nullptr;
    const T* orow = row_ok ? (const T*)a.o + b * a.o_sb + qi * a.o_st + qh * a.o_sh : nullptr;
    Frag8<T> qf[NC], gf[GLDS || !InRegs<T, DP>::value ? 1 : NC];
    TileReader<T, DP> read;
    read.init(lane);
    float delta = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const Frag8<T> g = load_frag<T>(grow, 16 * c + 8 * h, a.D), o = load_frag<T>(orow, 16 * c + 8 * h, a.D);
#pragma unroll
        for (int e = 0; e < 8; ++e) delta = fmaf((float)g.v[e], (float)o.v[e], delta);
        qf[c] = load_frag<T>(qrow, 16 * c + 8 * h, a.D);
        if constexpr (InRegs<T, DP>::value) {
            if constexpr (GLDS) *reinterpret_cast<uint4*>(smem + OFF_G + (wave * 32 * DP + Tile<T, DP>::at(lane & 31, 2 * c + h)) * ES) = __builtin_bit_cast(uint4, g);
            else gf[c] = g;
        }
    }
    delta += __shfl_xor(delta, 32, 64);
    const long long at = ((long long)b * a.Hq + qh) * a.Tq + qi;
    float lse2 = INFINITY;  // a row that sees nothing, or is none: every probability is zero
    if (row_ok) {
        if (h == 0 && split == 0) a.delta[at] = delta;
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
    const unsigned k_row = (unsigned)(a.k_st * ES), v_row = (unsigned)(a.v_st * ES), lds0 = lds_address(smem);
    TileOffsets<T, DP, BK> at_k, at_v;  // of a tile whose keys are all seen
    at_k.set(a.D, wave, lane, [&](int x) { return x * k_row; });
    at_v.set(a.D, wave, lane, [&](int x) { return x * v_row; });
    auto request = [&](int t, int buf, const unsigned (&seen)[KT]) {
        const T *kt0 = kb + (long long)t * BK * a.k_st, *vt0 = vb + (long long)t * BK * a.v_st;
        if ((seen[0] | seen[KT - 1]) == 0) return;  // a tile whose keys are all hidden is passed over
        if ((seen[0] & seen[KT - 1]) == 0xffffffffu) {
            at_k.request(kt0, lds0 + OFF_K + buf * TILE, wave);
            at_v.request(vt0, lds0 + OFF_V + buf * TILE, wave);
            return;
        }
        auto row = [&](unsigned stride) {
            return [&, stride](int x) { return (seen[x >> 5] >> (x & 31)) & 1 ? x * stride : 0x80000000u; };
        };
        request_tile<T, DP, BK>(kt0, lds0 + OFF_K + buf * TILE, a.D, wave, lane, row(k_row));
        request_tile<T, DP, BK>(vt0, lds0 + OFF_V + buf * TILE, a.D, wave, lane, row(v_row));
    };
    int t0 = 0, t1 = k_end > 0 ? (k_end + BK - 1) / BK : 0;
    if (SPLIT) {  // an even share of the tiles that are seen
        t0 = (int)((long long)t1 * split / a.dq_splits);
        t1 = (int)((long long)t1 * (split + 1) / a.dq_splits);
    }
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
    unsigned bits[KT], next[KT];
#pragma unroll
    for (int kt = 0; kt < KT; ++kt) {
        bits[kt] = key_bits(a, b, t0 * BK + kt * 32, lane);
        next[kt] = key_bits(a, b, (t0 + 1) * BK + kt * 32, lane);
    }
    if (t0 < t1) request(t0, 0, bits);
    // one tile out of buffer CUR
    auto step = [&](auto which, int t) {
        constexpr int CUR = decltype(which)::value;
        const int k0 = t * BK;
        tile_landed();
        unsigned ok[KT];  // the tile after the next: loaded now, waited for when this one is done
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) ok[kt] = 1;
        if (mask)
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) ok[kt] = mask[min(k0 + 2 * BK + kt * 32 + (lane & 31), a.Tk - 1)];
        if (t + 1 < t1) request(t + 1, CUR ^ 1, next);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            if (k0 + kt * 32 >= w_end || bits[kt] == 0) continue;
            f32x16_t s = f32x16_t{}, dp = f32x16_t{};
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int at = kt * 32 * DP * ES;
                const Frag8<T> k = read.rows(lds, OFF_K + CUR * TILE + at, c), v = read.rows(lds, OFF_V + CUR * TILE + at, c);
                if constexpr (GLDS) {
                    mma32(k, qf[c], s);
                    mma32(v, read.rows(lds + wave * 32 * DP * ES, OFF_G, c), dp);
                } else if constexpr (InRegs<T, DP>::value) {
                    mma32(k, qf[c], s);
                    mma32(v, gf[c], dp);
                } else {
                    mma32(k, qf[c], s);
                    mma32(v, load_frag<T>(grow, 16 * c + 8 * h, a.D), dp);
                }
            }
            if constexpr (sizeof(T) == 2) reads_ahead<(GLDS ? 3 : 2), 2, NC>();
            __builtin_amdgcn_s_setprio(0);
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
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const Frag8<T> ds = frag_of<T>(s, j);  // bf16: rounded for the product
#pragma unroll
                for (int d = 0; d < ND; ++d) mma32(read.cols(lds, OFF_K + CUR * TILE, d, kt * 32 + 16 * j), ds, acc[d]);
            }
            if constexpr (sizeof(T) == 2) reads_ahead<4, 2, ND>();
            __builtin_amdgcn_s_setprio(0);
        }
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
            bits[kt] = next[kt];
            asm volatile("" : "+v"(ok[kt]));  // (else the comparison, and its wait, moves up to the load)
            next[kt] = (unsigned)__ballot(ok[kt] != 0 && k0 + 2 * BK + kt * 32 + (lane & 31) < a.Tk);
        }
    };
    for (int t = t0; t < t1; t += 2) {
        step(std::integral_constant<int, 0>{}, t);
        if (t + 1 < t1) step(std::integral_constant<int, 1>{}, t + 1);
    }
    if (!row_ok) return;
    const long long place = (((long long)b * a.Tq + qi) * a.Hq + qh) * a.D;
    T* dq = (T*)a.dq + place;
    float* part = a.part + (long long)split * a.B * a.Tq * a.Hq * a.D + place;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = d * 32 + 8 * e + 4 * h;
            if (col >= a.D) continue;
            const float x[4] = {acc[d][4 * e] * a.scale, acc[d][4 * e + 1] * a.scale, acc[d][4 * e + 2] * a.scale, acc[d][4 * e + 3] * a.scale};
            if (SPLIT) store4<float>(part + col, x[0], x[1], x[2], x[3]);
            else store4<T>(dq + col, x[0], x[1], x[2], x[3]);
        }
}

// adds the partial sums of all key ranges, four elements per thread
template <typename T> __global__ __launch_bounds__(256) void attn_seq_dq_join_kernel(AttnSeqArgs a) {
    const long long all = (long long)a.B * a.Tq * a.Hq * a.D, i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= all) return;
    float x[4] = {};
#pragma unroll 8
    for (int s = 0; s < a.dq_splits; ++s) {
        const float4 p = *reinterpret_cast<const float4*>(a.part + s * all + i);
        x[0] += p.x; x[1] += p.y; x[2] += p.z; x[3] += p.w;
    }
    store4<T>((T*)a.dq + i, x[0], x[1], x[2], x[3]);
}

template <typename T, int DP> int launch(const AttnSeqArgs& a, hipStream_t s) {
    constexpr int BK = KeyTile<T, DP>::value;
    const long long blocks = (long long)((a.R + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK) * a.Hkv * a.B;
    if (a.dq_splits > 1) {
        MIC_LAUNCH((attn_seq_dq_kernel<T, DP, BK, true>), dim3((unsigned)(blocks * a.dq_splits)), dim3(256), 0, s, a);
        const long long quads = (long long)a.B * a.Tq * a.Hq * a.D / 4;
        MIC_LAUNCH((attn_seq_dq_join_kernel<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, a);
    } else {
        MIC_LAUNCH((attn_seq_dq_kernel<T, DP, BK, false>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    }
    return 0;
}
template <typename T> int launch_d(const AttnSeqArgs& a, hipStream_t s) {
    return a.D <= 32 ? launch<T, 32>(a, s) : a.D <= 64 ? launch<T, 64>(a, s) : a.D <= 128 ? launch<T, 128>(a, s) : launch<T, 256>(a, s);
}

}  // namespace

int mic_attn_seq_dq_launch(const AttnSeqArgs& a, int dtype, hipStream_t s) {
    return dtype == MIC_BF16 ? launch_d<bf16_t>(a, s) : launch_d<float>(a, s);
}
