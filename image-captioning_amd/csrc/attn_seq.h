// Pieces shared by the whole-sequence attention kernels (attn_seq_fwd.hip, attn_seq_dq.hip, attn_seq_dkv.hip): arguments, the
// LDS tile image, MFMA fragments and tile staging.
//
// Query heads that share a key head are packed: a "row" r of key head hk is query i = r / group of query head
// hk * group + r % group, so one pass over the keys serves the whole group, and the gradients of a shared key head are sums over
// its rows.
//
// All products run on 32x32 MFMA tiles.  Lane l, half h = l >> 5: operand A holds row l & 31, B column l & 31, both the eight
// reduction indices 8h..8h+7 of a step of 16; the result holds column l & 31 and rows 8*(r >> 2) + 4h + (r & 3) of register r.
// Eight consecutive result registers therefore are one B operand of the next product if its reduction index is taken in the
// order 4h..4h+3, 8+4h..8+4h+3: the probabilities go from one product into the next without leaving their lanes, and the
// other operand is read from LDS in that order (a transposing read in bf16, eight scalar reads in fp32).
#pragma once
#include "mic_common.h"

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct AttnSeqArgs {
    const void *q, *k, *v, *g;      // g: gradient of the output
    void *o, *dq, *dk, *dv;
    float *lse, *delta, *part, *part_ml;
    const unsigned char* mask;      // [B][Tk], non-zero = the key may be seen, or NULL
    long long mask_sb;
    long long q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, o_sb, o_st, o_sh, g_sb, g_st, g_sh;  // element strides
    int B, Tq, Tk, Hq, Hkv, D, group, R;  // R = Tq * group rows per key head
    int causal, off;                // query i sees keys up to i + off
    float scale, scale_log2;
    int splits, tiles_per_split;
    int dq_splits;                  // key ranges of the query gradients
    unsigned group_magic;           // ceil(2^32 / group), group > 1: x / group is the high half of x times it while x * group < 2^32
};

namespace {

constexpr float ATTN_LOG2E = 1.4426950408889634f, ATTN_LN2 = 0.6931471805599453f;

template <typename T> struct Frag8;
template <> struct Frag8<bf16_t> {
    bf16x8_t v;
};
template <> struct Frag8<float> {
    float v[8];
};

__device__ __forceinline__ void mma32(const Frag8<bf16_t>& a, const Frag8<bf16_t>& b, f32x16_t& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0);
}
// 32x32x2 takes one reduction index per half: step e pairs indices e of both halves, as the bf16 fragment lays them out
__device__ __forceinline__ void mma32(const Frag8<float>& a, const Frag8<float>& b, f32x16_t& c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
}

template <typename T> __device__ __forceinline__ Frag8<T> frag_zero() {
    Frag8<T> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = (T)0.f;
    return f;
}
// registers 8j..8j+7 of a result tile as the B operand of the next product
template <typename T> __device__ __forceinline__ Frag8<T> frag_of(const f32x16_t& p, int j) {
    Frag8<T> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = (T)p[8 * j + e];
    return f;
}

// LDS image of a tile of rows of DP elements: 16-byte chunk c of row r is stored at chunk c ^ tile_swizzle(r).  Both kinds of
// read then spread over all 64 banks: the same chunk of 16 consecutive rows (row operands), and 32 columns of the 4 rows a
// transposing read takes together.
template <typename T, int DP> struct Tile {
    static constexpr int E = 16 / (int)sizeof(T);     // elements per chunk
    static constexpr int CPR = DP / E;                // chunks per row
    __device__ static __forceinline__ int swizzle(int r) {
        if constexpr (CPR == 4) return (r >> 2) & 3;
        else if constexpr (CPR == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        else return ((r & 3) << 2) | ((r >> 2) & 3);
    }
    __device__ static __forceinline__ int at(int r, int c) { return r * DP + ((c ^ swizzle(r)) * E); }
};

// row operand: row r, reduction step c (16 columns)
template <int DP> __device__ __forceinline__ Frag8<bf16_t> read_row(const bf16_t* t, int r, int c, int h) {
    Frag8<bf16_t> f;
    f.v = *reinterpret_cast<const bf16x8_t*>(t + Tile<bf16_t, DP>::at(r, 2 * c + h));
    return f;
}
template <int DP> __device__ __forceinline__ Frag8<float> read_row(const float* t, int r, int c, int h) {
    Frag8<float> f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float4 x = *reinterpret_cast<const float4*>(t + Tile<float, DP>::at(r, 4 * c + 2 * h + k));
        f.v[4 * k] = x.x; f.v[4 * k + 1] = x.y; f.v[4 * k + 2] = x.z; f.v[4 * k + 3] = x.w;
    }
    return f;
}
// column operand: column d0 + (lane & 31), rows r0 + {4h..4h+3, 8+4h..8+4h+3}
typedef short v4i16_t __attribute__((ext_vector_type(4)));
template <int DP> __device__ __forceinline__ Frag8<bf16_t> read_col(const bf16_t* t, int d0, int r0, int lane) {
    // every 16 lanes exchange a 4 x 16 block: lane j reads row j / 4, columns 4 (j mod 4)..+3 and receives column j of the four rows
    const int h = lane >> 5, j = lane & 15, col = d0 + ((lane >> 4) & 1) * 16 + (j & 3) * 4, row = r0 + 4 * h + (j >> 2);
    typedef __attribute__((address_space(3))) v4i16_t* lds_t;
    const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(t + Tile<bf16_t, DP>::at(row, col >> 3) + (col & 7)));
    const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)(t + Tile<bf16_t, DP>::at(row + 8, col >> 3) + (col & 7)));
    typedef short v8i16_t __attribute__((ext_vector_type(8)));
    Frag8<bf16_t> f;
    f.v = __builtin_bit_cast(bf16x8_t, (v8i16_t)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    return f;
}
template <int DP> __device__ __forceinline__ Frag8<float> read_col(const float* t, int d0, int r0, int lane) {
    const int h = lane >> 5, col = d0 + (lane & 31);
    Frag8<float> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = t[Tile<float, DP>::at(r0 + 4 * h + (e & 3) + (e >> 2) * 8, col >> 2) + (col & 3)];
    return f;
}

// The same reads with a lane's addresses computed once.  The swizzle mixes a few low bits of the chunk number with bits of the row
// that depend on the lane alone, so a handful of registers serve every step, column tile and row tile: what differs otherwise is
// a constant, which the instruction carries.  `tile` is the tile's byte offset in `smem`, a constant too.
typedef __attribute__((address_space(3))) const unsigned char* lds_bytes_t;
template <typename T, int DP> struct TileReader;
template <int DP> struct TileReader<bf16_t, DP> {
    static constexpr int NR = DP / 16 < 8 ? DP / 16 : 8, NCOL = DP / 32 < 4 ? DP / 32 : 4;
    unsigned row, col[NCOL][2];  // the chunk number enters a row's address by exclusive or: one address, and a constant per step
    __device__ __forceinline__ void init(int lane) {
        const int h = lane >> 5, j = lane & 15;
        row = (unsigned)Tile<bf16_t, DP>::at(lane & 31, h) * 2u;
#pragma unroll
        for (int d = 0; d < NCOL; ++d)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int c = d * 32 + ((lane >> 4) & 1) * 16 + (j & 3) * 4;
                col[d][s] = (unsigned)(Tile<bf16_t, DP>::at(4 * h + (j >> 2) + 8 * s, c >> 3) + (c & 7)) * 2u;
            }
    }
    __device__ __forceinline__ Frag8<bf16_t> rows(lds_bytes_t smem, int tile, int c) const {
        typedef __attribute__((address_space(3))) const bf16x8_t* p_t;
        Frag8<bf16_t> f;
        f.v = *(p_t)(smem + (row ^ (unsigned)(c % NR * 32)) + (tile + c / NR * 256));
        return f;
    }
    __device__ __forceinline__ Frag8<bf16_t> cols(lds_bytes_t smem, int tile, int d, int r0) const {
        typedef __attribute__((address_space(3))) v4i16_t* p_t;
        const int k = tile + r0 * DP * 2 + d / NCOL * 256;
        const v4i16_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p_t)(smem + col[d % NCOL][0] + k));
        const v4i16_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((p_t)(smem + col[d % NCOL][1] + k));
        typedef short v8i16_t __attribute__((ext_vector_type(8)));
        Frag8<bf16_t> f;
        f.v = __builtin_bit_cast(bf16x8_t, (v8i16_t)__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        return f;
    }
};
template <int DP> struct TileReader<float, DP> {
    static constexpr int NR = DP / 16 < 4 ? DP / 16 : 4, NCOL = DP / 32 < 2 ? DP / 32 : 2;
    unsigned row[NR][2], col[NCOL][8];
    __device__ __forceinline__ void init(int lane) {
        const int h = lane >> 5;
#pragma unroll
        for (int c = 0; c < NR; ++c)
#pragma unroll
            for (int k = 0; k < 2; ++k) row[c][k] = (unsigned)Tile<float, DP>::at(lane & 31, 4 * c + 2 * h + k) * 4u;
#pragma unroll
        for (int d = 0; d < NCOL; ++d)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int c = d * 32 + (lane & 31);
                col[d][e] = (unsigned)(Tile<float, DP>::at(4 * h + (e & 3) + (e >> 2) * 8, c >> 2) + (c & 3)) * 4u;
            }
    }
    __device__ __forceinline__ Frag8<float> rows(lds_bytes_t smem, int tile, int c) const {
        Frag8<float> f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const f32x4_t x = *(__attribute__((address_space(3))) const f32x4_t*)(smem + row[c % NR][k] + (tile + c / NR * 256));
            f.v[4 * k] = x[0]; f.v[4 * k + 1] = x[1]; f.v[4 * k + 2] = x[2]; f.v[4 * k + 3] = x[3];
        }
        return f;
    }
    __device__ __forceinline__ Frag8<float> cols(lds_bytes_t smem, int tile, int d, int r0) const {
        typedef __attribute__((address_space(3))) const float* p_t;
        Frag8<float> f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f.v[e] = *(p_t)(smem + col[d % NCOL][e] + (tile + r0 * DP * 4 + d / NCOL * 256));
        return f;
    }
};

// fp32 with more than 128 columns: the second of a wave's own operands in the gradients (g, v) does not fit the registers next to the first
// and the sums, it is read again for every tile (4 x 1024 causal queries, 8 heads of 256: 1165 us, with both read again 1355).  What is left
// still spills: 130 registers in the key gradients, 28 to 60 in the query gradients.
template <typename T, int DP> struct InRegs {
    static constexpr bool value = sizeof(T) == 2 || DP <= 128;
};

// eight consecutive elements of a row in memory, zero past the head's D columns
template <typename T> __device__ __forceinline__ Frag8<T> load_frag(const T* row, int col, int D) {
    Frag8<T> f = frag_zero<T>();
    if constexpr (sizeof(T) == 2) {
        if (row && col < D) f.v = *reinterpret_cast<const bf16x8_t*>(row + col);
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (row && col + 4 * k < D) {
                const float4 x = *reinterpret_cast<const float4*>(row + col + 4 * k);
                f.v[4 * k] = x.x; f.v[4 * k + 1] = x.y; f.v[4 * k + 2] = x.z; f.v[4 * k + 3] = x.w;
            }
    }
    return f;
}

// ROWS rows into a tile; row_ptr(r) is the row's address or NULL for a row of zeros
template <typename T, int DP, int ROWS, int THREADS, typename P> __device__ __forceinline__ void stage(T* tile, int D, P row_ptr) {
    using L = Tile<T, DP>;
    constexpr int ALL = ROWS * L::CPR, N = (ALL + THREADS - 1) / THREADS;
    constexpr int G = N < 8 ? N : 8;  // loads in flight per thread
    static_assert(N % G == 0 && (N == 1 || ALL % THREADS == 0), "whole rounds");
#pragma unroll
    for (int n0 = 0; n0 < N; n0 += G) {
        uint4 x[G];
#pragma unroll
        for (int n = 0; n < G; ++n) {
            const int i = threadIdx.x + (n0 + n) * THREADS, r = i / L::CPR, c = i % L::CPR;
            const T* p = ALL >= THREADS || i < ALL ? row_ptr(r) : nullptr;
            x[n] = p && c * L::E < D ? *reinterpret_cast<const uint4*>(p + c * L::E) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int n = 0; n < G; ++n) {
            const int i = threadIdx.x + (n0 + n) * THREADS, r = i / L::CPR, c = i % L::CPR;
            if (ALL >= THREADS || i < ALL) *reinterpret_cast<uint4*>(tile + L::at(r, c)) = x[n];
        }
    }
}

// ---- tiles straight to LDS -----------------------------------------------------------------------------------------------------
// One buffer load per 1 KiB of a tile: a wave's 64 lanes fetch 16 bytes each from their own offsets and the result lands linearly in
// LDS, so the tile image's swizzle is applied to the chunk a lane fetches.  The buffer's base is the tile's, its length 2 GiB: an
// offset with bit 31 set (a row that is hidden or does not exist, a chunk past the head's columns) returns zeros without touching
// memory.  The loads are inline assembly because the compiler would drain the memory counter before the next LDS read if it saw
// them; the kernels wait for it themselves (s_waitcnt vmcnt(0), then a barrier, before a tile is read).
typedef unsigned srd_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ srd_t make_srd(const void* p) {
    const unsigned long long a = (unsigned long long)p;
    // the same in every lane, but perhaps computed in vector registers
    return srd_t{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)a), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)) & 0xffffu, 0x80000000u, 0x00020000u};
}
__device__ __forceinline__ void request16(unsigned voff, const srd_t& srd, unsigned lds) {
    unsigned keep;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %3, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep)
                 : "v"(voff), "s"(__builtin_amdgcn_readfirstlane((int)lds)), "s"(srd)
                 : "memory");
}
typedef __attribute__((address_space(3))) void* lds_ptr_t;
__device__ __forceinline__ unsigned lds_address(const void* p) { return __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(lds_ptr_t)p); }
// every request of this wave has landed and every wave is here: the tile requested last may be read, the other one written
__device__ __forceinline__ void tile_landed() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// ROWS rows of a tile by four waves; offset(row) is the row's byte offset from the base, or bit 31
template <typename T, int DP, int ROWS, typename F> __device__ __forceinline__ void request_tile(const T* base, unsigned lds, int D, int wave, int lane, F offset) {
    using L = Tile<T, DP>;
    constexpr int ROWB = DP * (int)sizeof(T), PIECES = ROWS * ROWB / 1024, PER = (PIECES + 3) / 4;
    const srd_t srd = make_srd(base);
#pragma unroll
    for (int n = 0; n < PER; ++n) {
        const int piece = n * 4 + wave;
        if (PIECES % 4 != 0 && piece >= PIECES) break;
        const int at = piece * 1024 + lane * 16, row = at / ROWB, c = (at % ROWB / 16) ^ L::swizzle(row);
        const unsigned off = c * L::E < D ? offset(row) + c * 16u : 0x80000000u;
        request16(off, srd, lds + piece * 1024);
    }
}

// The same with a lane's offsets computed once, for tiles whose rows lie alike
template <typename T, int DP, int ROWS> struct TileOffsets {
    static constexpr int PIECES = ROWS * DP * (int)sizeof(T) / 1024, PER = (PIECES + 3) / 4;
    unsigned off[PER];
    template <typename F> __device__ __forceinline__ void set(int D, int wave, int lane, F offset) {
        using L = Tile<T, DP>;
        constexpr int ROWB = DP * (int)sizeof(T);
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int at = (n * 4 + wave) * 1024 + lane * 16, row = at / ROWB, c = (at % ROWB / 16) ^ L::swizzle(row);
            off[n] = c * L::E < D ? offset(row) + c * 16u : 0x80000000u;
        }
    }
    __device__ __forceinline__ void request(const T* base, unsigned lds, int wave) const {
        const srd_t srd = make_srd(base);
#pragma unroll
        for (int n = 0; n < PER; ++n) {
            const int piece = n * 4 + wave;
            if (PIECES % 4 != 0 && piece >= PIECES) break;
            request16(off[n], srd, lds + piece * 1024);
        }
    }
};

// The order of a product's loop: the LDS reads of a step are issued before the matrix instructions of the step before it.  Left to itself
// the compiler reads an operand right before its use and waits for it: key gradients of 2 x 4096 queries of 16 heads of 128 columns,
// 400 us that way and 350 us in this order.
template <int READS, int MFMAS, int STEPS> __device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
    for (int i = 1; i < STEPS; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
        __builtin_amdgcn_sched_group_barrier(0x8, MFMAS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, MFMAS, 0);
}

// four consecutive columns of a result, rounded once
template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 2) {
        typedef bf16_t v4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<v4*>(p) = v4{(bf16_t)a, (bf16_t)b, (bf16_t)c, (bf16_t)d};
    } else {
        *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
    }
}

// bit j: key k0 + j exists and may be seen (causality aside); the same word in every lane
__device__ __forceinline__ unsigned key_bits(const AttnSeqArgs& a, int b, int k0, int lane) {
    const int key = k0 + (lane & 31);
    bool ok = key < a.Tk;
    if (ok && a.mask) ok = a.mask[b * a.mask_sb + key] != 0;
    return (unsigned)__ballot(ok);
}
// x / group for group > 1, x < group + 64
__device__ __forceinline__ unsigned by_group(const AttnSeqArgs& a, unsigned x) { return __umulhi(x, a.group_magic); }
__device__ __forceinline__ bool key_seen(const AttnSeqArgs& a, int b, int key) { return key < a.Tk && (!a.mask || a.mask[b * a.mask_sb + key] != 0); }

}  // namespace

// rows of a workgroup of the forward and query-gradient kernels, keys of one of the key-gradient kernel
#define ATTN_SEQ_BLOCK 128

// keys per tile of the forward and query-gradient kernels
template <typename T, int DP> struct KeyTile {
    static constexpr int value = DP * sizeof(T) <= 256 ? 64 : 32;
};

int mic_attn_seq_fwd_launch(const AttnSeqArgs& a, int dtype, hipStream_t s);
int mic_attn_seq_dq_launch(const AttnSeqArgs& a, int dtype, hipStream_t s);
int mic_attn_seq_dkv_launch(const AttnSeqArgs& a, int dtype, hipStream_t s);
int mic_attn_seq_dkv_join(const AttnSeqArgs& a, int dtype, hipStream_t s);  // adds the partial dK and dV of `splits` row ranges
// up to 64 keys
int mic_attn_seq_short_fwd_launch(const AttnSeqArgs& a, int dtype, hipStream_t s);
int mic_attn_seq_short_grad_launch(const AttnSeqArgs& a, int dtype, hipStream_t s);
