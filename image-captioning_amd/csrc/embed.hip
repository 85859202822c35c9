// Embedding of whole token sequences and its gradient.
//
//   out[n, :]    = scale * table[id(n), :] + pos[n mod T, :]
//   d_table[v,:] = scale * sum over { n : id(n) = v } of g[n, :]          d_pos[t, :] = sum over b of g[b*T + t, :]
//
// Both directions are bound by memory: the lookup reads a row and writes one; the gradient has to read g once and write every
// row of d_table once (zeros for the words that did not occur).
//
// The gradient of the table is summed without atomics, so the same inputs give the same bits.  The tokens are sorted by word
// (stable radix sort on the word's bits, 9 bits at most to a pass), and the SORTED list, not the vocabulary, is cut into equal
// chunks: captions are half padding and words follow Zipf's law, so a split by word would give one workgroup half of the sum.  A
// run of one word inside a chunk is summed in registers and written once; a run that crosses chunks leaves one fp32 partial row
// per chunk, which the join adds in the order of the chunks.
#include "mic_common.h"

namespace {

constexpr int SORT_THREADS = 1024;
constexpr int SORT_WAVES = SORT_THREADS / 64;
constexpr int MAX_DIGITS = 512;
constexpr int MAX_SORT_BLOCKS = 64;

__device__ __forceinline__ int load_id(const void* ids, int wide, long long i, int vocab) {
    const long long v = wide ? ((const long long*)ids)[i] : (long long)((const int*)ids)[i];
    return v < 0 ? 0 : (v >= vocab ? vocab - 1 : (int)v);  // never index outside the table
}

// VEC consecutive elements as fp32: one 16-byte access (two for 8 floats) where VEC > 1
template <typename T, int VEC> __device__ __forceinline__ void load_vec(const T* p, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = to_f32<T>(*p);
    } else {
        constexpr int E = Vec16<T>::N;
#pragma unroll
        for (int c = 0; c < VEC / E; ++c) {
            const Vec16<T> x = ld16(p + c * E);
#pragma unroll
            for (int e = 0; e < E; ++e) v[c * E + e] = to_f32<T>(x.v[e]);
        }
    }
}
template <typename T, int VEC> __device__ __forceinline__ void store_vec(T* p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        *p = from_f32<T>(v[0]);
    } else {
        constexpr int E = Vec16<T>::N;
#pragma unroll
        for (int c = 0; c < VEC / E; ++c) {
            Vec16<T> x;
#pragma unroll
            for (int e = 0; e < E; ++e) x.v[e] = from_f32<T>(v[c * E + e]);
            st16(p + c * E, x);
        }
    }
}

// ---- lookup: one thread per VEC columns of a row -------------------------------------------------------------------------
template <typename TT, typename TO, int VEC>
__global__ __launch_bounds__(256) void embed_rows_kernel(const void* __restrict__ ids, int wide, const TT* __restrict__ table, long long ld_table,
                                                         const TT* __restrict__ pos, long long ld_pos, TO* __restrict__ out, float scale,
                                                         long long n, int T, int H, int vocab) {
    const int per_row = H / VEC;
    const long long total = n * per_row, stride = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        const long long r = i / per_row;
        const int c = (int)(i - r * per_row) * VEC;
        float v[VEC];
        load_vec<TT, VEC>(table + load_id(ids, wide, r, vocab) * ld_table + c, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= scale;
        if (pos) {
            float p[VEC];
            load_vec<TT, VEC>(pos + (r % T) * ld_pos + c, p);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] += p[e];
        }
        store_vec<TO, VEC>(out + r * H + c, v);
    }
}

// ---- stable radix sort of (word, token index) ----------------------------------------------------------------------------
struct SortArgs {
    const void* ids;           // first pass: the caller's tokens
    int wide, vocab;
    const int *key_in, *idx_in;  // later passes
    int *key_out, *idx_out;
    unsigned* hist;            // [blocks][MAX_DIGITS]
    long long n;
    int per_block, shift, bits;
};

__device__ __forceinline__ int sort_key(const SortArgs& a, long long i) { return a.ids ? load_id(a.ids, a.wide, i, a.vocab) : a.key_in[i]; }

__global__ __launch_bounds__(SORT_THREADS) void embed_hist_kernel(SortArgs a) {
    __shared__ unsigned h[MAX_DIGITS];
    if (threadIdx.x < MAX_DIGITS) h[threadIdx.x] = 0;
    __syncthreads();
    const long long lo = (long long)blockIdx.x * a.per_block, hi = lo + a.per_block < a.n ? lo + a.per_block : a.n;
    const int mask = (1 << a.bits) - 1;
    for (long long i = lo + threadIdx.x; i < hi; i += SORT_THREADS) atomicAdd(&h[(sort_key(a, i) >> a.shift) & mask], 1u);
    __syncthreads();
    if (threadIdx.x < MAX_DIGITS) a.hist[blockIdx.x * MAX_DIGITS + threadIdx.x] = h[threadIdx.x];
}

__global__ __launch_bounds__(SORT_THREADS) void embed_scatter_kernel(SortArgs a) {
    __shared__ unsigned next[MAX_DIGITS];                 // where the next key of a digit goes
    __shared__ unsigned wc[SORT_WAVES][MAX_DIGITS];       // keys of a digit in a wave, then the wave's first place
    __shared__ unsigned scan[8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // first place of every digit for this block: digits below it anywhere, then this digit in the blocks before
    unsigned before = 0, total = 0;
    if (tid < MAX_DIGITS) {
        for (int b = 0; b < (int)gridDim.x; ++b) {
            const unsigned c = a.hist[b * MAX_DIGITS + tid];
            total += c;
            if (b < (int)blockIdx.x) before += c;
        }
    }
    unsigned inc = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_up(inc, d, 64);
        if (lane >= d) inc += o;
    }
    if (tid < MAX_DIGITS && lane == 63) scan[wave] = inc;
    __syncthreads();
    if (tid < MAX_DIGITS) {
        unsigned base = 0;
        for (int w = 0; w < wave; ++w) base += scan[w];
        next[tid] = base + inc - total + before;
    }
    const long long lo = (long long)blockIdx.x * a.per_block, hi = lo + a.per_block < a.n ? lo + a.per_block : a.n;
    const int mask = (1 << a.bits) - 1;
    for (long long r = lo; r < hi; r += SORT_THREADS) {  // the same number of rounds for every thread
#pragma unroll
        for (int k = 0; k < SORT_WAVES * MAX_DIGITS / SORT_THREADS; ++k) (&wc[0][0])[tid + k * SORT_THREADS] = 0;
        __syncthreads();
        const long long i = r + tid;
        const bool ok = i < hi;
        const int key = ok ? sort_key(a, i) : 0;
        const int idx = ok ? (a.ids ? (int)i : a.idx_in[i]) : 0;
        const int dig = (key >> a.shift) & mask;
        unsigned long long same = __ballot(ok);  // lanes of this wave with the same digit
        for (int b = 0; b < a.bits; ++b) {
            const unsigned long long one = __ballot((dig >> b) & 1);
            same &= ((dig >> b) & 1) ? one : ~one;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1ull));
        if (ok && rank == 0) wc[wave][dig] = (unsigned)__popcll(same);
        __syncthreads();
        if (tid < MAX_DIGITS) {
            unsigned at = next[tid];
#pragma unroll
            for (int w = 0; w < SORT_WAVES; ++w) {
                const unsigned c = wc[w][tid];
                wc[w][tid] = at;
                at += c;
            }
            next[tid] = at;
        }
        __syncthreads();
        if (ok) {
            const unsigned p = wc[wave][dig] + (unsigned)rank;
            a.key_out[p] = key;
            a.idx_out[p] = idx;
        }
        __syncthreads();
    }
}

// ---- sums over the sorted list ---------------------------------------------------------------------------------------------
struct SumArgs {
    const int *key, *idx;   // sorted words and the tokens they stand for
    const void* g;
    void* d_table;
    float *head, *tail;     // [chunks][H] partial rows of runs that began before the chunk / go on after it
    long long n;
    int H, vocab, chunk, chunks, slabs;
    float scale;
};

// first position of the sorted list whose word is not below v
__device__ __forceinline__ int lower_bound_key(const int* key, int n, int v) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int mid = (int)(((unsigned)lo + (unsigned)hi) >> 1);
        if (key[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// A wave takes one chunk of the sorted list and one slab of 64*VEC columns; the waves behind those clear the rows of words that
// do not occur, 64 rows each.
template <typename TG, typename TO, int VEC> __global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs a) {
    const int lane = threadIdx.x & 63;
    const long long unit = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sums = (long long)a.chunks * a.slabs;
    const TG* g = (const TG*)a.g;
    TO* dt = (TO*)a.d_table;
    if (unit >= sums) {
        const long long v0 = (unit - sums) * 64;
        if (v0 >= a.vocab) return;
        const int v = (int)v0 + lane;
        bool absent = false;
        if (v < a.vocab) {
            const int p = lower_bound_key(a.key, (int)a.n, v);
            absent = p >= (int)a.n || a.key[p] != v;
        }
        unsigned long long todo = __ballot(absent);
        const float zero[VEC] = {};
        while (todo) {
            const int r = __ffsll((unsigned long long)todo) - 1;
            todo &= todo - 1;
            for (int c = lane * VEC; c < a.H; c += 64 * VEC) store_vec<TO, VEC>(dt + (v0 + r) * a.H + c, zero);
        }
        return;
    }
    const int chunk = (int)(unit / a.slabs), slab = (int)(unit - (long long)chunk * a.slabs);
    const int col = (slab * 64 + lane) * VEC;
    const bool live = col < a.H;
    const int i0 = chunk * a.chunk, i1 = i0 + a.chunk < (int)a.n ? i0 + a.chunk : (int)a.n;
    const bool cont_in = i0 > 0 && a.key[i0 - 1] == a.key[i0];
    const bool cont_out = i1 < (int)a.n && a.key[i1] == a.key[i1 - 1];
    float acc[VEC] = {};
    bool first = true;  // still in the run the chunk began with
    int word = a.key[i0];
    constexpr int U = 8;  // rows in flight
    for (int i = i0; i < i1; i += U) {
        float v[U][VEC];
        int w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = i + u < i1 ? i + u : i1 - 1;
            w[u] = a.key[j];
            const long long row = a.idx[j];
            if (live) load_vec<TG, VEC>(g + row * a.H + col, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= i1) break;
            if (w[u] != word) {  // the run ended: the same branch for the whole wave
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = first && cont_in ? acc[e] : acc[e] * a.scale;
                if (live) {
                    if (first && cont_in) store_vec<float, VEC>(a.head + (long long)chunk * a.H + col, acc);
                    else store_vec<TO, VEC>(dt + (long long)word * a.H + col, acc);
                }
                first = false;
                word = w[u];
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += live ? v[u][e] : 0.f;
        }
    }
    if (!live) return;
    if (first && cont_in) {
        store_vec<float, VEC>(a.head + (long long)chunk * a.H + col, acc);
    } else if (cont_out) {
        store_vec<float, VEC>(a.tail + (long long)chunk * a.H + col, acc);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= a.scale;
        store_vec<TO, VEC>(dt + (long long)word * a.H + col, acc);
    }
}

// One workgroup per chunk whose last run begins in it and goes on: adds that run's partial rows in chunk order.
template <typename TO, int VEC> __global__ __launch_bounds__(256) void embed_join_kernel(SumArgs a) {
    __shared__ float part[4][64 * VEC];
    __shared__ int last_chunk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int chunk = blockIdx.x, slab = blockIdx.y;
    const int i0 = chunk * a.chunk, i1 = i0 + a.chunk;
    if (i1 >= (int)a.n) return;
    const int word = a.key[i1 - 1];
    if (a.key[i1] != word) return;
    if (i0 > 0 && a.key[i0] == word && a.key[i0 - 1] == word) return;  // began in an earlier chunk
    if (threadIdx.x == 0) last_chunk = (lower_bound_key(a.key, (int)a.n, word + 1) - 1) / a.chunk;
    __syncthreads();
    const int m = last_chunk - chunk + 1;  // the tail of this chunk, then the heads of the following ones
    const int col = (slab * 64 + lane) * VEC;
    const bool live = col < a.H;
    const int lo = (int)((long long)m * wave / 4), hi = (int)((long long)m * (wave + 1) / 4);
    float acc[VEC] = {};
    constexpr int U = 4;
    for (int k = lo; k < hi; k += U) {
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = k + u < hi ? k + u : hi - 1;
            if (live) load_vec<float, VEC>((j == 0 ? a.tail : a.head) + (long long)(chunk + j) * a.H + col, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += live && k + u < hi ? v[u][e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[wave][lane * VEC + e] = acc[e];
    __syncthreads();
    if (wave == 0 && live) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            float s = part[0][lane * VEC + e];
#pragma unroll
            for (int w = 1; w < 4; ++w) s += part[w][lane * VEC + e];
            acc[e] = s * a.scale;
        }
        store_vec<TO, VEC>((TO*)a.d_table + (long long)word * a.H + col, acc);
    }
}

// ---- sum over sequences: columns of a [B][W] matrix, W = T*H; `slices` of the rows leave fp32 partial rows when there are several
template <typename TG, typename TO, int VEC>
__global__ __launch_bounds__(256) void embed_colsum_kernel(const TG* __restrict__ g, TO* __restrict__ out, float* __restrict__ part_out, int B,
                                                           long long W, int slices) {
    __shared__ float part[4][64 * VEC];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, slice = blockIdx.y;
    const long long col = ((long long)blockIdx.x * 64 + lane) * VEC;
    const bool live = col < W;
    const int b0 = (int)((long long)B * slice / slices), b1 = (int)((long long)B * (slice + 1) / slices), rows = b1 - b0;
    const int lo = b0 + (int)((long long)rows * wave / 4), hi = b0 + (int)((long long)rows * (wave + 1) / 4);
    float acc[VEC] = {};
    constexpr int U = 4;
    for (int b = lo; b < hi; b += U) {
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = b + u < hi ? b + u : hi - 1;
            if (live) load_vec<TG, VEC>(g + j * W + col, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += live && b + u < hi ? v[u][e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < VEC; ++e) part[wave][lane * VEC + e] = acc[e];
    __syncthreads();
    if (wave == 0 && live) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            float s = part[0][lane * VEC + e];
#pragma unroll
            for (int w = 1; w < 4; ++w) s += part[w][lane * VEC + e];
            acc[e] = s;
        }
        if (slices == 1) store_vec<TO, VEC>(out + col, acc);
        else store_vec<float, VEC>(part_out + slice * W + col, acc);
    }
}

// ---- the gradient's plan: everything that depends on the sizes alone -------------------------------------------------------
struct GradPlan {
    int sort_blocks, per_block, passes, bits;
    int chunk, chunks, slices;
    long long key[2], idx[2], hist, head, tail, pos, bytes;  // byte offsets into the workspace
};

long long up256(long long b) { return (b + 255) / 256 * 256; }

GradPlan grad_plan(long long n, int T, int H, int vocab, bool want_pos) {
    GradPlan p = {};
    int blocks = (int)((n + SORT_THREADS - 1) / SORT_THREADS);
    blocks = blocks < 1 ? 1 : blocks > MAX_SORT_BLOCKS ? MAX_SORT_BLOCKS : blocks;
    p.per_block = (int)(((n + blocks - 1) / blocks + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS);
    if (p.per_block < SORT_THREADS) p.per_block = SORT_THREADS;
    p.sort_blocks = (int)((n + p.per_block - 1) / p.per_block);
    int nb = 1;
    while (nb < 31 && (1ll << nb) < vocab) ++nb;
    p.passes = (nb + 8) / 9;
    p.bits = (nb + p.passes - 1) / p.passes;
    // a wave per chunk and 512 columns: about 4,096 of them, 8 to 64 rows each
    const int slabs = (H + 511) / 512;
    long long c = n * slabs / 4096;
    p.chunk = (int)(c < 8 ? 8 : c > 64 ? 64 : c);
    p.chunks = (int)((n + p.chunk - 1) / p.chunk);
    long long o = 0;
    for (int i = 0; i < 2; ++i) {
        p.key[i] = o; o += up256(n * 4);
        p.idx[i] = o; o += up256(n * 4);
    }
    p.hist = o; o += up256((long long)p.sort_blocks * MAX_DIGITS * 4);
    p.head = o; o += up256((long long)p.chunks * H * 4);
    p.tail = o; o += up256((long long)p.chunks * H * 4);
    p.slices = 1;
    if (want_pos) {
        // about 1,024 workgroups over the columns of [B][T*H], at least 32 sequences to a slice
        const long long B = n / T, groups = ((long long)T * H + 511) / 512;
        long long s = 1024 / (groups < 1 ? 1 : groups);
        if (s > B / 32) s = B / 32;
        p.slices = (int)(s < 1 ? 1 : s > 512 ? 512 : s);
        p.pos = o;
        if (p.slices > 1) o += up256((long long)p.slices * T * H * 4);
    }
    p.bytes = o;
    return p;
}

bool ok_dtype(int d) { return d == MIC_F32 || d == MIC_BF16; }

template <typename TG, typename TO, int VEC>
int launch_grad(const GradPlan& p, const void* ids, int wide, const void* g, void* d_table, void* d_pos, float scale, long long n, int T, int H, int vocab,
                char* ws, hipStream_t s) {
    SortArgs a = {};
    a.wide = wide; a.vocab = vocab; a.n = n; a.per_block = p.per_block; a.bits = p.bits;
    a.hist = (unsigned*)(ws + p.hist);
    for (int i = 0; i < p.passes && n > 0; ++i) {
        a.ids = i == 0 ? ids : nullptr;
        a.key_in = (const int*)(ws + p.key[(i + 1) & 1]);
        a.idx_in = (const int*)(ws + p.idx[(i + 1) & 1]);
        a.key_out = (int*)(ws + p.key[i & 1]);
        a.idx_out = (int*)(ws + p.idx[i & 1]);
        a.shift = i * p.bits;
        MIC_LAUNCH(embed_hist_kernel, dim3(p.sort_blocks), dim3(SORT_THREADS), 0, s, a);
        MIC_LAUNCH(embed_scatter_kernel, dim3(p.sort_blocks), dim3(SORT_THREADS), 0, s, a);
    }
    SumArgs m = {};
    m.key = (const int*)(ws + p.key[(p.passes - 1) & 1]);
    m.idx = (const int*)(ws + p.idx[(p.passes - 1) & 1]);
    m.g = g; m.d_table = d_table;
    m.head = (float*)(ws + p.head); m.tail = (float*)(ws + p.tail);
    m.n = n; m.H = H; m.vocab = vocab; m.chunk = p.chunk; m.chunks = p.chunks; m.scale = scale;
    m.slabs = (H + 64 * VEC - 1) / (64 * VEC);
    const long long units = (long long)p.chunks * m.slabs + (vocab + 63) / 64;
    MIC_LAUNCH((embed_sum_kernel<TG, TO, VEC>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, s, m);
    if (p.chunks > 1) MIC_LAUNCH((embed_join_kernel<TO, VEC>), dim3(p.chunks, m.slabs), dim3(256), 0, s, m);
    if (d_pos) {
        const long long W = (long long)T * H;
        const unsigned groups = (unsigned)((W + 64 * VEC - 1) / (64 * VEC));
        float* part = (float*)(ws + p.pos);
        MIC_LAUNCH((embed_colsum_kernel<TG, TO, VEC>), dim3(groups, p.slices), dim3(256), 0, s, (const TG*)g, (TO*)d_pos, part, (int)(n / T), W, p.slices);
        if (p.slices > 1)
            MIC_LAUNCH((embed_colsum_kernel<float, TO, VEC>), dim3(groups, 1), dim3(256), 0, s, (const float*)part, (TO*)d_pos, (float*)nullptr, p.slices, W, 1);
    }
    return 0;
}

}  // namespace

extern "C" int mic_embed_rows(const void* ids, int ids_bits, const void* table, int64_t ld_table, const void* pos, int64_t ld_pos, void* out,
                              int table_dtype, int out_dtype, float scale, int64_t n, int T, int H, int vocab, void* stream) {
    MIC_ARG_CHECK(n >= 0 && n < (1ll << 31) && T > 0 && H > 0 && vocab > 0, "mic_embed_rows: bad sizes n=%lld T=%d H=%d vocab=%d", (long long)n, T, H, vocab);
    MIC_ARG_CHECK(ids_bits == 32 || ids_bits == 64, "mic_embed_rows: token ids of %d bits", ids_bits);
    MIC_ARG_CHECK(ok_dtype(table_dtype) && ok_dtype(out_dtype), "mic_embed_rows: bad dtype %d / %d", table_dtype, out_dtype);
    MIC_ARG_CHECK(ld_table >= H && (!pos || ld_pos >= H), "mic_embed_rows: row stride below H=%d", H);
    if (n == 0) return 0;
    MIC_ARG_CHECK(ids && table && out, "mic_embed_rows: null pointer");
    hipStream_t s = (hipStream_t)stream;
    const bool vec = H % 8 == 0 && ld_table % 8 == 0 && (!pos || ld_pos % 8 == 0) && (((uintptr_t)table | (uintptr_t)out | (uintptr_t)pos) & 15) == 0;
    const long long work = n * (vec ? H / 8 : H);
    const long long blocks = (work + 255) / 256;
    const dim3 grid((unsigned)(blocks > 65536 ? 65536 : blocks));
#define GO(TT, TO, VEC)                                                                                                                   \
    MIC_LAUNCH((embed_rows_kernel<TT, TO, VEC>), grid, dim3(256), 0, s, ids, ids_bits == 64, (const TT*)table, (long long)ld_table, (const TT*)pos, \
               (long long)ld_pos, (TO*)out, scale, (long long)n, T, H, vocab)
#define GO_VEC(TT, TO)             \
    do {                           \
        if (vec) GO(TT, TO, 8);    \
        else GO(TT, TO, 1);        \
    } while (0)
    if (table_dtype == MIC_F32 && out_dtype == MIC_F32) GO_VEC(float, float);
    else if (table_dtype == MIC_F32) GO_VEC(float, bf16_t);
    else if (out_dtype == MIC_F32) GO_VEC(bf16_t, float);
    else GO_VEC(bf16_t, bf16_t);
#undef GO
#undef GO_VEC
    return 0;
}

extern "C" int64_t mic_embed_grad_workspace_bytes(int64_t n, int T, int H, int vocab, int want_pos) {
    if (n < 0 || n >= (1ll << 30) || T <= 0 || H <= 0 || vocab <= 0 || (want_pos && n % T != 0)) return MIC_ERR_ARG;
    return grad_plan(n, T, H, vocab, want_pos != 0).bytes;
}

extern "C" int mic_embed_grad(const void* ids, int ids_bits, const void* g, void* d_table, void* d_pos, int g_dtype, int out_dtype, float scale,
                              int64_t n, int T, int H, int vocab, void* workspace, int64_t workspace_bytes, void* stream) {
    MIC_ARG_CHECK(n >= 0 && n < (1ll << 30) && T > 0 && H > 0 && vocab > 0, "mic_embed_grad: bad sizes n=%lld T=%d H=%d vocab=%d", (long long)n, T, H, vocab);
    MIC_ARG_CHECK(ids_bits == 32 || ids_bits == 64, "mic_embed_grad: token ids of %d bits", ids_bits);
    MIC_ARG_CHECK(ok_dtype(g_dtype) && ok_dtype(out_dtype), "mic_embed_grad: bad dtype %d / %d", g_dtype, out_dtype);
    MIC_ARG_CHECK(!d_pos || n % T == 0, "mic_embed_grad: %lld tokens are not whole sequences of %d", (long long)n, T);
    MIC_ARG_CHECK(d_table && (n == 0 || (ids && g)), "mic_embed_grad: null pointer");
    const GradPlan p = grad_plan(n, T, H, vocab, d_pos != nullptr);
    MIC_ARG_CHECK(workspace_bytes >= p.bytes && (p.bytes == 0 || workspace), "mic_embed_grad: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, p.bytes);
    MIC_ARG_CHECK(((uintptr_t)workspace & 15) == 0, "mic_embed_grad: workspace is not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const bool vec = H % 8 == 0 && (((uintptr_t)g | (uintptr_t)d_table | (uintptr_t)d_pos) & 15) == 0;
#define GO(TG, TO, VEC) return launch_grad<TG, TO, VEC>(p, ids, ids_bits == 64, g, d_table, d_pos, scale, n, T, H, vocab, (char*)workspace, s)
#define GO_VEC(TG, TO)             \
    do {                           \
        if (vec) GO(TG, TO, 8);    \
        else GO(TG, TO, 1);        \
    } while (0)
    if (g_dtype == MIC_F32 && out_dtype == MIC_F32) GO_VEC(float, float);
    else if (g_dtype == MIC_F32) GO_VEC(float, bf16_t);
    else if (out_dtype == MIC_F32) GO_VEC(bf16_t, float);
    else GO_VEC(bf16_t, bf16_t);
#undef GO
#undef GO_VEC
}
