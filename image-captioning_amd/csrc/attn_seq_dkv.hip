// Whole-sequence attention, gradients of the keys and values:
//   dv = P^T g     dk = scale * dS^T q     over all rows (queries of every head of the group) that see the key
// A wave owns 32 keys: their k stay in registers as B operands and their v in LDS (the registers are full with dK and dV), S = Q K^T
// and dP = G V^T come out with a lane per key, and P and dS are the B operands of dV^T = G^T P and dK^T = Q^T dS.  The workgroup's
// four waves walk the same tiles of 32 rows.
// 2 x 4096 causal queries of 16 heads on 2 key heads of 128 columns, bf16: 350 us, 790 TFLOP/s, the matrix units 45 % busy: 250 registers a lane
// leave two waves to a SIMD and operands that are read one step ahead (the form without `splits` needs 3 more and spills them; fp32 with
// 256 columns spills 130 at one wave per SIMD).
// With `splits` the rows are shared out over several workgroups, which leave fp32 partial sums that a second launch adds in order.
#include "attn_seq.h"

#include <type_traits>

namespace {

// (a lambda that stays a call has its captures in scratch memory: fp32 with 256 columns 700 bytes a lane instead of 140)
#define INLINE __attribute__((always_inline))

template <typename T, int DP, bool SPLIT> __global__ __launch_bounds__(256, (DP * sizeof(T) <= 256 ? 2 : 1)) void attn_seq_dkv_kernel(AttnSeqArgs a) {
    constexpr int NC = DP / 16, ND = DP / 32, ES = sizeof(T);
    constexpr bool KEEP = InRegs<T, DP>::value;  // else v is read from memory for every tile
    constexpr int TILE = 32 * DP * ES, OFF_Q = 0, OFF_G = 2 * TILE, OFF_V = 4 * TILE;  // two tiles of q, two of g, the four waves' v
    __shared__ __attribute__((aligned(16))) unsigned char smem[4 * TILE + (KEEP ? 4 * TILE : 0)];
    __shared__ __attribute__((aligned(16))) float s_lse[2][32], s_delta[2][32];
    const lds_bytes_t lds = (lds_bytes_t)smem;
    const int lane = threadIdx.x & 63, h = lane >> 5, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int heads = a.Hkv * a.B;
    int id = blockIdx.x;
    const int hk = id % heads % a.Hkv, b = id % heads / a.Hkv;
    id /= heads;
    const int split = SPLIT ? id % a.splits : 0;
    if (SPLIT) id /= a.splits;
    const int kt = id;  // the first keys, which the most rows see, first
    const int k0 = kt * ATTN_SEQ_BLOCK + wave * 32, key = k0 + (lane & 31);
    const bool seen = key_seen(a, b, key);
    const T* krow = seen ? (const T*)a.k + b * a.k_sb + hk * a.k_sh + (long long)key * a.k_st : nullptr;
    const T* vrow = seen ? (const T*)a.v + b * a.v_sb + hk * a.v_sh + (long long)key * a.v_st : nullptr;
    TileReader<T, DP> read;
    read.init(lane);
    Frag8<T> kf[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) kf[c] = load_frag<T>(krow, 16 * c + 8 * h, a.D);
    if constexpr (KEEP) {
        T* sv = reinterpret_cast<T*>(smem + OFF_V) + wave * 32 * DP;  // rows hidden keys would have are zeros
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const Frag8<T> v = load_frag<T>(vrow, 16 * c + 8 * h, a.D);
            constexpr int E = Tile<T, DP>::E;
#pragma unroll
            for (int k = 0; k < 8 / E; ++k) {
                Vec16<T> x;
#pragma unroll
                for (int e = 0; e < E; ++e) x.v[e] = v.v[k * E + e];
                st16(sv + Tile<T, DP>::at(lane & 31, (16 * c + 8 * h) / E + k), x);
            }
        }
    }
    // rows below `first` see no key of the workgroup, below w_first none of the wave; from w_all on they see every key of the wave
    const int first = a.causal ? max(0, kt * ATTN_SEQ_BLOCK - a.off) * a.group : 0, w_first = a.causal ? max(0, k0 - a.off) * a.group : 0;
    const int w_all = a.causal ? max(0, k0 + 31 - a.off) * a.group : 0;
    const unsigned w_seen = (unsigned)__ballot(seen);
    const bool all_seen = w_seen == 0xffffffffu;
    int b_first = 0x7fffffff;  // the first key that is seen, of all the workgroup's
#pragma unroll
    for (int w = 3; w >= 0; --w) {
        const unsigned bits = key_bits(a, b, kt * ATTN_SEQ_BLOCK + w * 32, lane);
        if (bits) b_first = kt * ATTN_SEQ_BLOCK + w * 32 + __builtin_ctz(bits);
    }
    // Rows below this see none of them.  Those that share a tile with rows that do are fetched as zeros, whatever q and g hold there.
    const int blind = a.causal && b_first != 0x7fffffff ? min(max(0, b_first - a.off) * a.group, a.R) : 0;
    // a row sees this lane's key from row (key - off) * group on
    const int from = !seen ? 0x7fffffff : a.causal ? max(0, key - a.off) * a.group : 0;
    int t0 = min(first, a.R) / 32, t1 = (a.R + 31) / 32;
    if (SPLIT) {
        t0 += split * a.tiles_per_split;
        if (split > 0 && t0 >= t1) return;  // this key tile needs fewer workgroups
        t1 = min(t1, t0 + a.tiles_per_split);
    }
    if (b_first == 0x7fffffff) t1 = t0;
    const unsigned q_row = (unsigned)(a.q_st * ES), q_head = (unsigned)(a.q_sh * ES), g_row = (unsigned)(a.g_st * ES), g_head = (unsigned)(a.g_sh * ES);
    const unsigned lds0 = lds_address(smem);
    TileOffsets<T, DP, 32> at_q, at_g;
    const T* qb = (const T*)a.q + b * a.q_sb + hk * a.group * a.q_sh;
    const T* gb = (const T*)a.g + b * a.g_sb + hk * a.group * a.g_sh;
    const bool even = 32 % a.group == 0;  // every tile then begins with a query's first head, and a lane's offsets never change
    const int step_i = even ? 32 / a.group : 0;
    long long at_stats;  // lse and delta of the lane's row: 32 threads, loaded a tile ahead
    // row x of a tile: query (rest + x) / group from the tile's first on, of `rows` that there are, the first `none` of them left out
    auto places = [&](int rest, int rows, int none) INLINE {
        auto row = [&](unsigned per_row, unsigned per_head) {
            return [&, per_row, per_head](int x) {
                const unsigned y = rest + x, i = a.group == 1 ? y : by_group(a, y);
                return x >= none && x < rows ? i * per_row + (y - i * a.group) * per_head : 0x80000000u;
            };
        };
        at_q.set(a.D, wave, lane, row(q_row, q_head));
        at_g.set(a.D, wave, lane, row(g_row, g_head));
        const unsigned y = rest + (lane & 31), i = a.group == 1 ? y : by_group(a, y);
        at_stats = ((long long)b * a.Hq + hk * a.group + (y - i * a.group)) * a.Tq + i;
    };
    if (even) places(0, 32, 0);
    float lse2 = INFINITY, delta = 0.f;
    auto request = [&](int t, int buf) INLINE {
        const int r0 = t * 32, i0 = even ? t * step_i : r0 / a.group;
        // (the tile behind one with such rows takes its offsets anew)
        if (!even || r0 + 32 > a.R || r0 < blind + 32) places(even ? 0 : r0 - i0 * a.group, a.R - r0, blind - r0);
        at_q.request(qb + (long long)i0 * a.q_st, lds0 + OFF_Q + buf * TILE, wave);
        at_g.request(gb + (long long)i0 * a.g_st, lds0 + OFF_G + buf * TILE, wave);
        lse2 = INFINITY;
        delta = 0.f;
        if (threadIdx.x < 32 && r0 + (int)threadIdx.x < a.R) {
            lse2 = a.lse[at_stats + i0];
            delta = a.delta[at_stats + i0];
        }
    };
    auto put_stats = [&](int buf) {
        if (threadIdx.x < 32) {
            s_lse[buf][threadIdx.x] = lse2 == -INFINITY ? INFINITY : lse2 * ATTN_LOG2E;  // no key seen: every probability is zero
            s_delta[buf][threadIdx.x] = delta;
        }
    };
    f32x16_t dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16_t{};
    if (t0 < t1) {
        request(t0, 0);
        put_stats(0);
    }
    // one tile out of buffer CUR
    auto step = [&](auto which, int t) INLINE {
        constexpr int CUR = decltype(which)::value;
        const int r0 = t * 32;
        tile_landed();
        if (t + 1 < t1) request(t + 1, CUR ^ 1);
        if (w_seen != 0 && r0 + 31 >= w_first) {
            f32x16_t s = f32x16_t{}, dp = f32x16_t{};
            if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(read.row));  // recomputed in every step: the registers are needed for reads ahead
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const Frag8<T> q = read.rows(lds, OFF_Q + CUR * TILE, c), g = read.rows(lds, OFF_G + CUR * TILE, c);
                if constexpr (KEEP) {
                    mma32(q, kf[c], s);
                    mma32(g, read.rows(lds + wave * TILE, OFF_V, c), dp);
                } else {
                    mma32(q, kf[c], s);
                    mma32(g, load_frag<T>(vrow, 16 * c + 8 * h, a.D), dp);
                }
            }
            if constexpr (sizeof(T) == 2) reads_ahead<3, 2, NC>();
            __builtin_amdgcn_s_setprio(0);
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const float4 l4 = *reinterpret_cast<const float4*>(&s_lse[CUR][8 * e4 + 4 * h]), d4 = *reinterpret_cast<const float4*>(&s_delta[CUR][8 * e4 + 4 * h]);
                const float ls[4] = {l4.x, l4.y, l4.z, l4.w}, ds[4] = {d4.x, d4.y, d4.z, d4.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int e = 4 * e4 + i;
                    s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2, -ls[i]));
                    dp[e] = s[e] * (dp[e] - ds[i]);
                }
            }
            if (!(all_seen && r0 >= w_all))  // something is hidden
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool ok = r0 + 8 * (e >> 2) + 4 * h + (e & 3) >= from;
                    s[e] = ok ? s[e] : 0.f;
                    dp[e] = ok ? dp[e] : 0.f;
                }
            Frag8<T> p[2], ds[2];  // bf16: rounded for the products
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                p[j] = frag_of<T>(s, j);
                ds[j] = frag_of<T>(dp, j);
            }
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    mma32(read.cols(lds, OFF_G + CUR * TILE, d, 16 * j), p[j], dv[d]);
                    mma32(read.cols(lds, OFF_Q + CUR * TILE, d, 16 * j), ds[j], dk[d]);
                }
            if constexpr (sizeof(T) == 2) reads_ahead<4, 2, 2 * ND>();
        }
        __builtin_amdgcn_s_setprio(0);
        if (t + 1 < t1) put_stats(CUR ^ 1);
    };
    for (int t = t0; t < t1; t += 2) {
        step(std::integral_constant<int, 0>{}, t);
        if (t + 1 < t1) step(std::integral_constant<int, 1>{}, t + 1);
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

// adds the partial sums of all row ranges of a key, four elements per thread
template <typename T> __global__ __launch_bounds__(256) void attn_seq_dkv_join_kernel(AttnSeqArgs a, int general) {
    const long long all = (long long)a.B * a.Tk * a.Hkv * a.D, i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= 2 * all) return;
    int ranges = a.splits;
    if (general && a.causal) {  // as many as the key's tile has
        const int key = (int)((i < all ? i : i - all) / ((long long)a.Hkv * a.D) % a.Tk), kt = key / ATTN_SEQ_BLOCK;
        const int first = max(0, kt * ATTN_SEQ_BLOCK - a.off) * a.group, n = (a.R + 31) / 32 - min(first, a.R) / 32;
        ranges = max(1, (n + a.tiles_per_split - 1) / a.tiles_per_split);
    }
    float x[4] = {};
#pragma unroll 4
    for (int s = 0; s < ranges; ++s) {
        const float4 p = *reinterpret_cast<const float4*>(a.part + 2 * s * all + i);
        x[0] += p.x; x[1] += p.y; x[2] += p.z; x[3] += p.w;
    }
    store4<T>(i < all ? (T*)a.dk + i : (T*)a.dv + (i - all), x[0], x[1], x[2], x[3]);
}

template <typename T> int join(const AttnSeqArgs& a, int general, hipStream_t s) {
    const long long quads = (long long)a.B * a.Tk * a.Hkv * a.D / 2;
    MIC_LAUNCH((attn_seq_dkv_join_kernel<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, s, a, general);
    return 0;
}

template <typename T, int DP> int launch(const AttnSeqArgs& a, hipStream_t s) {
    const long long blocks = (long long)((a.Tk + ATTN_SEQ_BLOCK - 1) / ATTN_SEQ_BLOCK) * a.Hkv * a.B;
    if (a.splits > 1) {
        MIC_LAUNCH((attn_seq_dkv_kernel<T, DP, true>), dim3((unsigned)(blocks * a.splits)), dim3(256), 0, s, a);
        return join<T>(a, 1, s);
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
int mic_attn_seq_dkv_join(const AttnSeqArgs& a, int dtype, hipStream_t s) { return dtype == MIC_BF16 ? join<bf16_t>(a, 0, s) : join<float>(a, 0, s); }
