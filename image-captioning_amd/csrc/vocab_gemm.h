// Tiled matrix product of the vocabulary loss:  out[q][p] = sum_k Q(q, k) P(p, k), tiles of 128 x 128 or 64 x 64 (S = 2, 1), four
// waves of half that edge.
//
// Each operand lies in memory either with k consecutive (a row per index: "row" operand) or with its index consecutive (a row per
// k: "column" operand), and goes to LDS as it lies; a column operand is read from LDS by a transposing read (bf16) or scalar
// reads (fp32).  So logits (x w^T), dx (d w) and dw (d^T x) run on the same tiles without a transposed copy of anything.
// The result tile holds a lane per q and eight-row groups of p in registers: a row of the output (a token's logits) belongs to
// two lanes, whose statistics need one exchange.
// 24 x 512 x 32000, bf16: 10.5 us, 33 MB of w read once at 3.1 TB/s.  1111 x 300 x 10007, fp32: 81 us, 82 TFLOP/s; 4096 x 1024 x 32000: 122.
#pragma once
#include "attn_seq.h"

namespace {

// rows r0 + 8h..8h+7 of column d0 + (lane & 31): the order in which read_row takes k
template <int DP> __device__ __forceinline__ Frag8<bf16_t> read_col_k(const bf16_t* t, int d0, int r0, int lane) {
    const int h = lane >> 5, j = lane & 15, col = d0 + ((lane >> 4) & 1) * 16 + (j & 3) * 4, row = r0 + 8 * h + (j >> 2);
    typedef __attribute__((address_space(3))) v4i16_t* lds_t;
    const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(t + Tile<bf16_t, DP>::at(row, col >> 3) + (col & 7)));
    const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(t + Tile<bf16_t, DP>::at(row + 4, col >> 3) + (col & 7)));
    typedef short v8i16_t __attribute__((ext_vector_type(8)));
    Frag8<bf16_t> f;
    f.v = __builtin_bit_cast(bf16x8_t, (v8i16_t)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    return f;
}
template <int DP> __device__ __forceinline__ Frag8<float> read_col_k(const float* t, int d0, int r0, int lane) {
    const int h = lane >> 5, col = d0 + (lane & 31);
    Frag8<float> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = t[Tile<float, DP>::at(r0 + 8 * h + e, col >> 2) + (col & 3)];
    return f;
}

struct Operand {
    const void* p;
    long long ld;  // elements between rows in memory
    int n;         // how many indices there are
};

// One operand's tile of VT indices x KS steps of k: fetched to registers, later stored to LDS.
template <typename T, bool COL, int VT> struct OperandTile {
    static constexpr int KS = 128 / (int)sizeof(T);
    static constexpr int DP = COL ? VT : KS;
    using L = Tile<T, DP>;
    static constexpr int ROUNDS = VT * KS / L::E / 256;
    uint4 x[ROUNDS];
    __device__ __forceinline__ void fetch(const Operand& o, int i0, int k0, int k_end) {
#pragma unroll
        for (int n = 0; n < ROUNDS; ++n) {
            const int i = threadIdx.x + n * 256, r = i / L::CPR, c = i % L::CPR * L::E;
            const int idx = COL ? i0 + c : i0 + r, k = COL ? k0 + r : k0 + c;
            const T* p = (const T*)o.p + (COL ? k * o.ld + idx : idx * o.ld + k);
            x[n] = idx < o.n && k < k_end ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void put(T* tile) const {
#pragma unroll
        for (int n = 0; n < ROUNDS; ++n) {
            const int i = threadIdx.x + n * 256;
            *reinterpret_cast<uint4*>(tile + L::at(i / L::CPR, i % L::CPR)) = x[n];
        }
    }
    // indices i0..i0+31 of the tile, 16 steps of k from 16 * s
    __device__ static __forceinline__ Frag8<T> frag(const T* tile, int i0, int s, int lane) {
        if constexpr (COL) return read_col_k<DP>(tile, i0, 16 * s, lane);
        else return read_row<DP>(tile, i0 + (lane & 31), s, lane >> 5);
    }
};

struct GemmShape {
    Operand p, q;
    const int* rows;    // NULL, or the number of rows to take, on the device: limits q.n (k for products over the rows)
    const int* slices;  // NULL (one), or the number of ranges of k, on the device
    int rows_are_k;
    int K, tiles_p, tiles_q;
};

// Epi::run(args, acc, p0, q0, lane, part_p, part_q, slice): acc[i][j] = p0 + 32 i.., q0 + 32 j..; parts number the waves' columns and rows
template <typename T, int S> using GemmLds = T[2][64 * S * 128 / (int)sizeof(T)];  // two tiles of an operand
// the tile of workgroup `order` of the product
template <typename T, int S, bool PCOL, bool QCOL, typename Epi> __device__ __forceinline__ void vocab_gemm_tile(GemmShape g, const typename Epi::Args& ea, int order, GemmLds<T, S>& sp, GemmLds<T, S>& sq) {
    constexpr int VT = 64 * S, WAVE = 32 * S;
    using TP = OperandTile<T, PCOL, VT>;
    using TQ = OperandTile<T, QCOL, VT>;
    constexpr int KS = TP::KS;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wp = wave >> 1, wq = wave & 1;
    if (g.rows) {  // the grid is laid out for all rows: what is behind the counted ones ends here
        const int rows = *g.rows;
        if (g.rows_are_k) {
            g.K = min(g.K, rows);
        } else {
            g.q.n = min(g.q.n, rows);
            g.tiles_q = min(g.tiles_q, (rows + VT - 1) / VT);
        }
    }
    const int slices = g.slices ? *g.slices : 1;
    // workgroups b and b + 8 share an XCD and its L2: every XCD takes a contiguous range of the tiles that are left
    int id;
    {
        const int n = g.tiles_p * g.tiles_q * slices, o = order, per = n >> 3, rest = n & 7, xcd = o & 7;
        if (o >= n) return;
        id = (xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per) + (o >> 3);
    }
    const int slice = id % slices;
    id /= slices;
    const int tq = id % g.tiles_q, tp = id / g.tiles_q;
    const int p0 = tp * VT, q0 = tq * VT;
    const int nk = (g.K + KS - 1) / KS, kb = (int)((long long)nk * slice / slices), ke = (int)((long long)nk * (slice + 1) / slices);
    f32x16_t acc[S][S];
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
        for (int j = 0; j < S; ++j) acc[i][j] = f32x16_t{};
    TP fp;
    TQ fq;
    if (kb < ke) {
        fp.fetch(g.p, p0, kb * KS, g.K);
        fq.fetch(g.q, q0, kb * KS, g.K);
        fp.put(sp[0]);
        fq.put(sq[0]);
    }
    for (int t = kb; t < ke; ++t) {
        const int cur = (t - kb) & 1;
        __syncthreads();
        if (t + 1 < ke) {
            fp.fetch(g.p, p0, (t + 1) * KS, g.K);
            fq.fetch(g.q, q0, (t + 1) * KS, g.K);
        }
        // the next step's operands are on their way from LDS while a step's products run
        Frag8<T> a[2][S], b[2][S];
        auto load = [&](int s) {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                a[s & 1][i] = TP::frag(sp[cur], wp * WAVE + i * 32, s, lane);
                b[s & 1][i] = TQ::frag(sq[cur], wq * WAVE + i * 32, s, lane);
            }
        };
        load(0);
#pragma unroll
        for (int s = 0; s < KS / 16; ++s) {
            if (s + 1 < KS / 16) load(s + 1);
            if constexpr (sizeof(T) == 4) {  // the sums in turn: no product waits for the one before
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int i = 0; i < S; ++i)
#pragma unroll
                        for (int j = 0; j < S; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[s & 1][i].v[e], b[s & 1][j].v[e], acc[i][j], 0, 0, 0);
            } else {
#pragma unroll
                for (int i = 0; i < S; ++i)
#pragma unroll
                    for (int j = 0; j < S; ++j) mma32(a[s & 1][i], b[s & 1][j], acc[i][j]);
            }
        }
        if (t + 1 < ke) {
            fp.put(sp[cur ^ 1]);
            fq.put(sq[cur ^ 1]);
        }
    }
    Epi::run(ea, acc, p0 + wp * WAVE, q0 + wq * WAVE, lane, tp * 2 + wp, tq * 2 + wq, slice);
}
template <typename T, int S, typename Epi> __global__ __launch_bounds__(256, 2) void vocab_gemm_kernel(GemmShape g, typename Epi::Args ea) {
    __shared__ __attribute__((aligned(16))) GemmLds<T, S> sp;
    __shared__ __attribute__((aligned(16))) GemmLds<T, S> sq;
    vocab_gemm_tile<T, S, false, false, Epi>(g, ea, blockIdx.x, sp, sq);
}
// Two products in one launch, both of whose P lie with their index consecutive: the second one's workgroups from `first` on (a multiple of
// 8), its Q likewise.
template <typename T, int S, typename Epi>
__global__ __launch_bounds__(256, 2) void vocab_gemm_pair_kernel(GemmShape x, typename Epi::Args xa, GemmShape w, typename Epi::Args wa, int first) {
    __shared__ __attribute__((aligned(16))) GemmLds<T, S> sp;
    __shared__ __attribute__((aligned(16))) GemmLds<T, S> sq;
    if ((int)blockIdx.x < first) vocab_gemm_tile<T, S, true, false, Epi>(x, xa, blockIdx.x, sp, sq);
    else vocab_gemm_tile<T, S, true, true, Epi>(w, wa, (int)blockIdx.x - first, sp, sq);
}

}  // namespace
