// Whole-sequence attention, forward:  o = softmax(scale * q k^T, masked) v  in one pass over the keys with a running maximum and
// sum, and lse = log sum exp of every row for the gradient.  See attn_seq.h for the layouts.
//
// A workgroup of four waves takes 128 rows of one key head; a wave keeps 32 rows' queries as B operands in registers and computes
// S^T = K Q^T, so a lane owns one row (query) and the statistics of a row are 16 registers of one lane and one exchange with
// the lane 32 away.  P^T then is the B operand of O^T = V^T P^T.
//
// 2 x 4096 causal queries of 16 heads (2 key heads) of 128 columns, bf16: 190 us, 720 TFLOP/s; matrix and vector instructions (32 exponentials
// and some 150 others beside 32 products per wave and tile) together fill the time.  One query, 4093 keys, 8 x 8 heads on 2 key
// heads: 9.5 us for 33.5 MB and 3.9 us to join 32 ranges of keys.  9 x 333 queries, 391 padded keys, 8 heads of 64, fp32: 30 us.
// 256 columns take one wave per SIMD: with 256 registers a lane bf16 spills (4 x 1024 causal queries, 8 heads: 132 us, with 512 77 us); fp32 with
// 128 columns is faster with two (148 and 161 us), though its form for shared keys spills 14 registers then, and fp32 with 256 columns 6 to 9.
#include "attn_seq.h"

#include <type_traits>

namespace {

template <typename T, int DP, int BK, bool SPLIT> __global__ __launch_bounds__(256, (DP <= 128 ? 2 : 1)) void attn_seq_fwd_kernel(AttnSeqArgs a) {
    constexpr int NC = DP / 16, ND = DP / 32, KT = BK / 32, ES = sizeof(T);
    constexpr int TILE = BK * DP * ES, OFF_K = 0, OFF_V = 2 * TILE;  // two tiles of k, two of v
    __shared__ __attribute__((aligned(16))) unsigned char smem[4 * TILE];
    const lds_bytes_t lds = (lds_bytes_t)smem;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tiles_r = (a.R + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK, heads = a.Hkv * a.B;
    int id = blockIdx.x;
    const int split = SPLIT ? id % a.splits : 0;
    if (SPLIT) id /= a.splits;
    // the last rows, which see the most keys, first
    const int rt = tiles_r - 1 - id / heads, hk = id % heads % a.Hkv, b = id % heads / a.Hkv;
    const int r0 = rt * ATTN_SEQ_BLOCK + wave * 32, r = r0 + (lane & 31);
    const bool row_ok = r < a.R;
    const int qi = row_ok ? r / a.group : 0, qh = hk * a.group + (row_ok ? r - qi * a.group : 0);
    const T* qrow = row_ok ? (const T*)a.q + b * a.q_sb + qi * a.q_st + qh * a.q_sh : nullptr;
    Frag8<T> qf[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) qf[c] = load_frag<T>(qrow, 16 * c + 8 * h, a.D);

    const int last = min(rt * ATTN_SEQ_BLOCK + ATTN_SEQ_BLOCK, a.R) - 1;
    const int k_end = a.causal ? min(a.Tk, last / a.group + a.off + 1) : a.Tk;  // keys any row of the workgroup may see
    const int w_first = min(r0, a.R - 1), w_last = min(r0 + 31, a.R - 1);
    const int w_end = r0 < a.R ? (a.causal ? min(a.Tk, w_last / a.group + a.off + 1) : a.Tk) : 0;  // any row of the wave
    const int w_all = a.causal ? w_first / a.group + a.off : a.Tk - 1;                             // last key every row of the wave sees
    const int lim = a.causal ? qi + a.off : a.Tk - 1;                                              // last key this lane's row sees
    int t0 = 0, t1 = k_end > 0 ? (k_end + BK - 1) / BK : 0;
    if (SPLIT) {
        t0 = split * a.tiles_per_split;
        t1 = min(t1, t0 + a.tiles_per_split);
    }
    f32x16_t acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16_t{};
    float m = -INFINITY, l = 0.f;
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    const unsigned k_row = (unsigned)(a.k_st * ES), v_row = (unsigned)(a.v_st * ES), lds0 = lds_address(smem);
    TileReader<T, DP> read;
    read.init(lane);
    // rows no query may see are zeros: whatever they hold, infinities and NaN included, stays out of the products
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
        if (k0 < w_end && (bits[0] | bits[KT - 1]) != 0) {
            f32x16_t s[KT];
            float top = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) s[kt] = f32x16_t{};
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int kt = 0; kt < KT; ++kt)
                    mma32(read.rows(lds, OFF_K + CUR * TILE + kt * 32 * DP * ES, c), qf[c], s[kt]);
            if constexpr (sizeof(T) == 2) reads_ahead<KT, KT, NC>();
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
                if (bits[kt] == 0xffffffffu && k0 + kt * 32 + 31 <= w_all) {  // nothing hidden: the common case
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        s[kt][e] *= a.scale_log2;
                        top = fmaxf(top, s[kt][e]);
                    }
                } else {
                    const unsigned mine = bits[kt] >> (4 * h);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int j = 8 * (e >> 2) + (e & 3);
                        const bool seen = ((mine >> j) & 1) && k0 + kt * 32 + 4 * h + j <= lim;
                        s[kt][e] = seen ? s[kt][e] * a.scale_log2 : -INFINITY;
                        top = fmaxf(top, s[kt][e]);
                    }
                }
            }
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float m_new = fmaxf(m, top), m_use = m_new == -INFINITY ? 0.f : m_new;
            float sum = 0.f;
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[kt][e] = __builtin_amdgcn_exp2f(s[kt][e] - m_use);
                    sum += s[kt][e];
                }
            sum += __shfl_xor(sum, 32, 64);
            if (__any(m_new > m)) {  // some row's maximum rose
                const float alpha = __builtin_amdgcn_exp2f(m - m_use);
                l *= alpha;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[d][e] *= alpha;
            }
            m = m_new;
            l += sum;
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int kt = 0; kt < KT; ++kt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const Frag8<T> p = frag_of<T>(s[kt], j);  // bf16: the probabilities are rounded for the product, the sum l is not
#pragma unroll
                    for (int d = 0; d < ND; ++d) mma32(read.cols(lds, OFF_V + CUR * TILE, d, kt * 32 + 16 * j), p, acc[d]);
                }
            if constexpr (sizeof(T) == 2) reads_ahead<4, 2, KT * ND>();
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
    if (SPLIT) {
        const long long at = (((long long)split * a.B + b) * a.Hkv + hk) * a.R + r;
        float* o = a.part + at * a.D;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = d * 32 + 8 * e + 4 * h;
                if (col < a.D) store4<float>(o + col, acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]);
            }
        if (h == 0) {
            a.part_ml[2 * at] = m;
            a.part_ml[2 * at + 1] = l;
        }
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    T* o = (T*)a.o + b * a.o_sb + qi * a.o_st + qh * a.o_sh;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int col = d * 32 + 8 * e + 4 * h;
            if (col < a.D) store4<T>(o + col, acc[d][4 * e] * inv, acc[d][4 * e + 1] * inv, acc[d][4 * e + 2] * inv, acc[d][4 * e + 3] * inv);
        }
    if (h == 0) a.lse[((long long)b * a.Hq + qh) * a.Tq + qi] = l == 0.f ? -INFINITY : (m + log2f(l)) * ATTN_LN2;
}

// Joins the key ranges of a row: a workgroup per row.  The weight of every range first (a lane each), then each wave adds a quarter of the
// ranges, all of whose loads are independent, and the waves' sums are added in order.
template <typename T> __global__ __launch_bounds__(256) void attn_seq_join_kernel(AttnSeqArgs a) {
    __shared__ float weight[512], part[4][256];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long rows = (long long)a.B * a.Hkv * a.R, row = blockIdx.x;
    float m = -INFINITY;  // every wave looks at all ranges
    for (int s = lane; s < a.splits; s += 64) m = fmaxf(m, a.part_ml[2 * (s * rows + row)]);
    m = wave_max(m);
    const float m_use = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = lane; s < a.splits; s += 64) {
        const float w = __builtin_amdgcn_exp2f(a.part_ml[2 * (s * rows + row)] - m_use);
        if (wave == 0) weight[s] = w;
        l += w * a.part_ml[2 * (s * rows + row) + 1];
    }
    l = wave_sum(l);
    __syncthreads();
    const int col = lane * 4, s0 = a.splits * wave / 4, s1 = a.splits * (wave + 1) / 4;
    float acc[4] = {};
    if (col < a.D)
#pragma unroll 8
        for (int s = s0; s < s1; ++s) {
            const float4 x = *reinterpret_cast<const float4*>(a.part + (s * rows + row) * a.D + col);
            const float w = weight[s];
            acc[0] += w * x.x; acc[1] += w * x.y; acc[2] += w * x.z; acc[3] += w * x.w;
        }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[wave][col + e] = acc[e];
    __syncthreads();
    if (wave) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = ((part[0][col + e] + part[1][col + e]) + part[2][col + e] + part[3][col + e]) * inv;
    const int r = (int)(row % a.R), hk = (int)(row / a.R % a.Hkv), qi = r / a.group, qh = hk * a.group + r - qi * a.group;
    const long long b = row / a.R / a.Hkv;
    if (col < a.D) store4<T>((T*)a.o + b * a.o_sb + qi * a.o_st + qh * a.o_sh + col, acc[0], acc[1], acc[2], acc[3]);
    if (lane == 0) a.lse[(b * a.Hq + qh) * a.Tq + qi] = l == 0.f ? -INFINITY : (m + log2f(l)) * ATTN_LN2;
}

template <typename T, int DP> int launch(const AttnSeqArgs& a, hipStream_t s) {
    constexpr int BK = KeyTile<T, DP>::value;
    const long long blocks = (long long)((a.R + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK) * a.Hkv * a.B;
    if (a.splits > 1) {
        MIC_LAUNCH((attn_seq_fwd_kernel<T, DP, BK, true>), dim3((unsigned)(blocks * a.splits)), dim3(256), 0, s, a);
        const long long rows = (long long)a.B * a.Hkv * a.R;
        MIC_LAUNCH((attn_seq_join_kernel<T>), dim3((unsigned)rows), dim3(256), 0, s, a);
    } else {
        MIC_LAUNCH((attn_seq_fwd_kernel<T, DP, BK, false>), dim3((unsigned)blocks), dim3(256), 0, s, a);
    }
    return 0;
}
template <typename T> int launch_d(const AttnSeqArgs& a, hipStream_t s) {
    return a.D <= 32 ? launch<T, 32>(a, s) : a.D <= 64 ? launch<T, 64>(a, s) : a.D <= 128 ? launch<T, 128>(a, s) : launch<T, 256>(a, s);
}

}  // namespace

int mic_attn_seq_fwd_launch(const AttnSeqArgs& a, int dtype, hipStream_t s) {
    return dtype == MIC_BF16 ? launch_d<bf16_t>(a, s) : launch_d<float>(a, s);
}
