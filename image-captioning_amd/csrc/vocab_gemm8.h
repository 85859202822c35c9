// The vocabulary loss's products in bf16 on 256 x 256 tiles:  out[q][p] = sum_k Q(q, k) P(p, k), the main loop of igemm8.hip (see
// there for the phases, the two wave rows half a phase apart and the counted waits) for plain matrices of either orientation.
//
// A workgroup of 8 waves is 2 (q) x 4 (p) waves of 128 x 64.  A K-tile of 64 is four half-tiles of 16 KiB: Q0 = q rows {0..63} of both
// wave rows, Q1 = {64..127}, P0 = p {0..31} of the four wave columns, P1 = {32..63}; two K-tiles are resident.
//  * row operand (k consecutive in memory): two planes of 128 rows x 64 bytes, read with ds_read_b128, as in igemm8.hip;
//  * column operand (index consecutive): 64 rows of k x 256 bytes, read with transposing reads.  16-byte chunk c of row k is stored at
//    chunk c ^ 2f, f = (k & 3) | (k >> 3 & 1) << 2: the 8 rows x 2 chunks that half a wave reads at once are 16 different chunks.
// A workgroup stays and takes every 256th tile: the next tile's first requests are under way while the epilogue of the last one
// computes (epilogues leave LDS alone; what they need of bias and rows is put into a small side buffer beforehand).  With H = 512 a
// tile is 13 us of products, and its start and end used to cost 17 us more.  8192 x 2048 x 65536: 1628 us, 1350 TFLOP/s (the library's
// product of 8192^3 runs at 1408); 7424 x 512 x 3500: 35 us, 750, as 406 tiles are 1.6 rounds of 256.  (The gradient's logits spill 6 registers
// around the epilogue.)
// Requests go straight to LDS through a buffer descriptor whose base is the K-tile's, so a lane's offset never changes and no
// operand is too long; an index outside the operand or a k past the end is bit 31 of the offset, which returns zeros without
// touching memory.
#pragma once
#include "attn_seq.h"
#include "igemm_shared.h"

namespace {

#define VG_BARRIER() asm volatile("s_barrier" ::: "memory")

struct Operand8 {
    const void* p;
    long long ld;  // elements between rows in memory
    int n;         // indices
};
struct Gemm8Shape {
    Operand8 p, q;
    const int* rows;    // the number of rows to take, on the device: limits q.n (k for products over the rows)
    const int* slices;  // the number of ranges of k, on the device
    int rows_are_k;
    int K, tiles_p, tiles_q;
};

constexpr unsigned G8_HALF = 16384, G8_TILE = 4 * G8_HALF, G8_DEAD = 0x80000000u;
constexpr unsigned G8_Q0 = 0, G8_P0 = G8_HALF, G8_P1 = 2 * G8_HALF, G8_Q1 = 3 * G8_HALF;
constexpr int G8_SIDE = 4 * 256;  // per tile: four values for each of its 256 columns or rows

// What one wave requests of an operand.  IS_Q: indices of a half-tile are 2 x 64 (wave rows), else 4 x 32 (wave columns).
template <bool COL, bool IS_Q> struct Request8 {
    unsigned off[2], step;            // byte offset of this lane's first piece of half-tile h; from there to the second piece
    int k_lane, k_step;               // k of the first piece within the K-tile; to the second
    unsigned long long base[2], adv;  // the half-tiles' next K-tile
    int k[2];                         // its first k
    __device__ static __forceinline__ int index(int i0, int h, int l) { return IS_Q ? i0 + (l >> 6) * 128 + h * 64 + (l & 63) : i0 + (l >> 5) * 64 + h * 32 + (l & 31); }
    __device__ __forceinline__ void init(const Operand8& o, int i0, int k0, int wave, int lane) {
        const long long row_bytes = o.ld * 2;
        if constexpr (COL) {
            const int kr = wave * 8 + (lane >> 4), f = ((lane >> 4) & 3) | ((wave & 1) << 2);  // both pieces: rows kr and kr + 4
            const int c = (lane & 15) ^ (2 * f);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = index(i0, h, c * 8);
                off[h] = i < o.n ? (unsigned)(kr * row_bytes + (i - i0) * 2) : G8_DEAD;
            }
            step = (unsigned)(4 * row_bytes);
            k_lane = kr;
            k_step = 4;
            adv = 64 * row_bytes;
            base[0] = base[1] = (unsigned long long)o.p + (unsigned long long)k0 * row_bytes + (unsigned long long)i0 * 2;
        } else {
            const int lr = wave * 16 + (lane >> 2), ch = (lane & 3) ^ (((lr >> 3) & 1) << 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = index(i0, h, lr);
                off[h] = i < o.n ? (unsigned)((i - i0) * row_bytes + ch * 16) : G8_DEAD;
            }
            step = 64;
            k_lane = ch * 8;
            k_step = 32;
            adv = 128;
            base[0] = base[1] = (unsigned long long)o.p + (unsigned long long)i0 * row_bytes + (unsigned long long)k0 * 2;
        }
        k[0] = k[1] = k0;
    }
    __device__ __forceinline__ void issue(int h, unsigned lds, int K) {
        const srd_t srd = make_srd((const void*)base[h]);
        const unsigned d0 = k[h] + k_lane >= K ? G8_DEAD : 0u, d1 = k[h] + k_lane + k_step >= K ? G8_DEAD : 0u;
        request16(off[h] | d0, srd, lds);
        request16((off[h] + step) | d1, srd, lds + (COL ? 1024u : 8192u));
        base[h] += adv;
        k[h] += 64;
    }
    // LDS address of the wave's first piece inside a half-tile
    __device__ static __forceinline__ unsigned piece(int wave) { return COL ? wave * 2048u : wave * 1024u; }
};

// Fragment reads: N tiles of 16 indices of a half-tile, from local index `first` on
template <bool COL, int N> struct Read8 {
    unsigned at[COL ? N : 1];
    __device__ __forceinline__ void init(int first, int lane) {
        if constexpr (COL) {
            const int g = lane >> 4, j = lane & 15, f = (j >> 2) | ((g & 1) << 2);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = first / 8 + 2 * n;
                at[n] = (unsigned)((8 * g + (j >> 2)) * 256 + ((c ^ (2 * f)) + ((j & 3) >> 1)) * 16 + (j & 1) * 8);
            }
        } else {
            at[0] = (unsigned)lds_off(first + (lane & 15), lane >> 4);
        }
    }
    __device__ __forceinline__ uint4 load(const unsigned char* smem, unsigned off, int n, int kp) const {
        if constexpr (COL) {
            typedef short v4i16 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) v4i16* lds_t;
            const unsigned char* p = smem + off + at[n] + kp * 8192;
            const v4i16 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p);
            const v4i16 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(p + 1024));
            typedef short v8i16 __attribute__((ext_vector_type(8)));
            return __builtin_bit_cast(uint4, (v8i16)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            return *reinterpret_cast<const uint4*>(smem + off + kp * 8192 + n * 1024 + at[0]);
        }
    }
};

// Epi::side(args, p0, q0, thread, side) fills the side buffer; Epi::run(args, acc, p0, q0, lane, wave, tile_p, tile_q, slice, side):
// acc[j][i] = p0 + 64 (wave & 3) + 16 j.., q0 + 128 (wave >> 2) + 16 i..
// The tiles of a product from `order` on, gridDim.x apart; returns how many there are.  COUNTED, SLICED: whether the shape has rows and slices
// (what it has not costs scalar registers).
template <bool PCOL, bool QCOL, bool COUNTED, bool SLICED, typename Epi>
__device__ __forceinline__ int vocab_gemm8_tiles(const Gemm8Shape& shape, const typename Epi::Args& ea, int order, unsigned char (&smem)[2 * G8_TILE], float (&side)[2][G8_SIDE]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wq = wave >> 2, wp = wave & 3;
    const Operand8 &gp = shape.p;
    Operand8 gq = shape.q;
    int K = shape.K, tiles_q = shape.tiles_q;
    const int tiles_p = shape.tiles_p;
    if (COUNTED) {  // the grid is laid out for all rows: what is behind the counted ones ends here
        const int rows = __builtin_amdgcn_readfirstlane(*shape.rows);
        if (shape.rows_are_k) {
            K = min(K, rows);
        } else {
            gq.n = min(gq.n, rows);
            tiles_q = min(tiles_q, (rows + 255) / 256);
        }
    }
    const int slices = SLICED ? __builtin_amdgcn_readfirstlane(*shape.slices) : 1, total = tiles_p * tiles_q * slices, nk = (K + 63) / 64;
    if (order >= total) return total;

    struct Place {
        int tp, tq, slice, t_begin, t_end;
    };
    auto place = [&](int o) {
        // tiles o and o + 8 share an XCD and its L2: every XCD takes a contiguous range
        const int per = total >> 3, rest = total & 7, xcd = o & 7;
        int id = (xcd < rest ? xcd * (per + 1) : rest * (per + 1) + (xcd - rest) * per) + (o >> 3);
        Place x;
        x.slice = 0;
        if (SLICED) {
            x.slice = id % slices;
            id /= slices;
        }
        // 4 q tiles side by side walk the p tiles, so what runs at once on an XCD is a block of both and shares its operands in L2
        const int band = id / (4 * tiles_p), left = min(4, tiles_q - band * 4), in = id - band * 4 * tiles_p;
        x.tq = band * 4 + in % left;
        x.tp = in / left;
        x.t_begin = SLICED ? (int)((long long)x.slice * nk / slices) : 0;
        x.t_end = SLICED ? (int)((long long)(x.slice + 1) * nk / slices) : nk;
        // the same in every lane, computed in vector registers: the buffers' bases are built from them
        x.tp = __builtin_amdgcn_readfirstlane(x.tp);
        x.tq = __builtin_amdgcn_readfirstlane(x.tq);
        x.slice = __builtin_amdgcn_readfirstlane(x.slice);
        x.t_begin = __builtin_amdgcn_readfirstlane(x.t_begin);
        x.t_end = __builtin_amdgcn_readfirstlane(x.t_end);
        return x;
    };

    Request8<QCOL, true> rq;
    Request8<PCOL, false> rp;
    Read8<QCOL, 4> fq;
    Read8<PCOL, 2> fp;
    fq.init(wq * 64, lane);
    fp.init(wp * 32, lane);
    const unsigned lds0 = (unsigned)(uintptr_t)(lptr_t)smem;
    const unsigned piece_q = __builtin_amdgcn_readfirstlane(lds0 + Request8<QCOL, true>::piece(wave));
    const unsigned piece_p = __builtin_amdgcn_readfirstlane(lds0 + Request8<PCOL, false>::piece(wave));
    // a tile's side buffer, its first K-tile and three half-tiles of the second
    auto begin = [&](const Place& x, int parity) {
        Epi::side(ea, x.tp * 256, x.tq * 256, threadIdx.x, side[parity]);
        if (x.t_begin >= x.t_end) return;
        rq.init(gq, x.tq * 256, x.t_begin * 64, wave, lane);
        rp.init(gp, x.tp * 256, x.t_begin * 64, wave, lane);
        rq.issue(0, piece_q + G8_Q0, K);
        rp.issue(0, piece_p + G8_P0, K);
        rp.issue(1, piece_p + G8_P1, K);
        rq.issue(1, piece_q + G8_Q1, K);
        rq.issue(0, piece_q + G8_TILE + G8_Q0, K);
        rp.issue(0, piece_p + G8_TILE + G8_P0, K);
        rp.issue(1, piece_p + G8_TILE + G8_P1, K);
    };

    f32x4_t acc[4][8];
    uint4 xa[4][2] = {}, wb0[2][2] = {}, wb1[2][2] = {};
    auto ldq = [&](unsigned off) {
#pragma unroll
        for (int kp = 0; kp < 2; ++kp)
#pragma unroll
            for (int i = 0; i < 4; ++i) xa[i][kp] = fq.load(smem, off, i, kp);
    };
    auto ldp = [&](uint4 (&wb)[2][2], unsigned off) {
#pragma unroll
        for (int kp = 0; kp < 2; ++kp)
#pragma unroll
            for (int j = 0; j < 2; ++j) wb[j][kp] = fp.load(smem, off, j, kp);
    };
    auto quadrant = [&](const uint4 (&wb)[2][2], int hq, int hp) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kp = 0; kp < 2; ++kp)
#pragma unroll
            for (int jj = 0; jj < 2; ++jj)
#pragma unroll
                for (int ii = 0; ii < 4; ++ii) Mma<bf16_t>::run(wb[jj][kp], xa[ii][kp], acc[hp * 2 + jj][hq * 4 + ii]);
        __builtin_amdgcn_s_setprio(0);
        __builtin_amdgcn_sched_barrier(0);
        VG_BARRIER();
    };
    // one K-tile out of the buffer at `cur`; `oth` is the other buffer
    auto tile = [&](unsigned cur, unsigned oth) {
        ldp(wb0, cur + G8_P0);
        __builtin_amdgcn_sched_barrier(0);
        ldq(cur + G8_Q0);
        rq.issue(1, piece_q + oth + G8_Q1, K);
        __builtin_amdgcn_sched_barrier(0);
        // the P0 reads, issued first, have returned: its half-tile is requested again two barriers on
        if constexpr (QCOL) asm volatile("s_waitcnt lgkmcnt(15)" ::: "memory");  // at most 15 of the 16 reads of Q0 outstanding
        else asm volatile("s_waitcnt lgkmcnt(8)" ::: "memory");
        VG_BARRIER();
        quadrant(wb0, 0, 0);
        ldp(wb1, cur + G8_P1);
        rp.issue(0, piece_p + cur + G8_P0, K);
        __builtin_amdgcn_sched_barrier(0);
        VG_BARRIER();
        quadrant(wb1, 0, 1);
        ldq(cur + G8_Q1);
        rq.issue(0, piece_q + cur + G8_Q0, K);
        __builtin_amdgcn_sched_barrier(0);
        VG_BARRIER();
        quadrant(wb1, 1, 1);
        rp.issue(1, piece_p + cur + G8_P1, K);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_waitcnt vmcnt(6)" ::: "memory");  // all but the last three half-tiles: the next K-tile has landed
        VG_BARRIER();
        quadrant(wb0, 1, 0);
    };

    Place at = place(order);
    begin(at, 0);
    for (int parity = 0;; parity ^= 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[j][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (at.t_begin < at.t_end) {
            // all but the last three half-tiles (an epilogue's stores, issued since, only make the wait longer)
            asm volatile("s_waitcnt vmcnt(6)" ::: "memory");
            VG_BARRIER();
            if (wq == 1) VG_BARRIER();
            unsigned cur = 0;
            for (int t = at.t_begin; t < at.t_end; ++t) {
                tile(cur, G8_TILE - cur);
                cur = G8_TILE - cur;
            }
            if (wq == 0) VG_BARRIER();
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // requests past the end are still landing
        }
        __syncthreads();  // nobody reads the tile any more, the side buffer is whole
        const Place done = at;
        order += gridDim.x;
        if (order < total) {
            at = place(order);
            begin(at, parity ^ 1);
        }
        Epi::run(ea, acc, done.tp * 256, done.tq * 256, lane, wave, done.tp, done.tq, done.slice, side[parity]);
        if (order >= total) return total;
    }
}
template <typename Epi> __global__ __launch_bounds__(512) void vocab_gemm8_kernel(Gemm8Shape g, typename Epi::Args ea) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * G8_TILE];
    __shared__ __attribute__((aligned(16))) float side[2][G8_SIDE];
    vocab_gemm8_tiles<false, false, Epi::COUNTED, false, Epi>(g, ea, blockIdx.x, smem, side);
}
// Two products in one launch, both of whose P lie with their index consecutive, and the second one's Q: their tiles are dealt out in turn,
// the second one's from the next multiple of 8 on.  An epilogue without a side buffer leaves LDS alone, so a workgroup goes from
// one product to the other like from tile to tile.
template <typename Epi> __global__ __launch_bounds__(512) void vocab_gemm8_pair_kernel(Gemm8Shape x, typename Epi::Args xa, Gemm8Shape w, typename Epi::Args wa) {
    __shared__ __attribute__((aligned(16))) unsigned char smem[2 * G8_TILE];
    __shared__ __attribute__((aligned(16))) float side[2][G8_SIDE];
    const int n = (vocab_gemm8_tiles<true, false, true, true, Epi>(x, xa, blockIdx.x, smem, side) + 7) & ~7, grid = gridDim.x, block = blockIdx.x;
    vocab_gemm8_tiles<true, true, true, true, Epi>(w, wa, block >= n ? block - n : (n - block + grid - 1) / grid * grid + block - n, smem, side);
}

}  // namespace
