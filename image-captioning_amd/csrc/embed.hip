// Embedding of whole token sequences and its gradient.
//
//   out[n, :]    = scale * table[id(n), :] + pos[n mod T, :]
//   d_table[v,:] = scale * sum over { n : id(n) = v } of g[n, :]          d_pos[t, :] = sum over b of g[b*T + t, :]
//
// Both directions are bound by memory: the lookup reads a row and writes one; the gradient has to read g once and write every
// row of d_table once (zeros for the words that did not occur).
//
// The gradient of the table is summed without atomics, so the same inputs give the same bits.  The tokens are sorted by word
// (up to 8,192 tokens: every token counts the tokens before it, in one launch; more: stable radix sort on the word's bits, 9 bits at
// most to a pass), and the SORTED list, not the vocabulary, is cut into equal
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

// Eight columns at a time, whatever H and the alignment are: A = rows are whole 16-byte pieces on 16-byte boundaries; else only the first n of
// the eight belong to the row, and the vector access takes any address (HSA devices run with unaligned access on).
constexpr int VEC = 8;
template <typename T, bool A> __device__ __forceinline__ void load8(const T* p, int n, float (&v)[VEC]) {
    if (A || n >= VEC) {
        T x[VEC];
        if constexpr (A) {
#pragma unroll
            for (int c = 0; c < VEC / Vec16<T>::N; ++c) {
                const Vec16<T> y = ld16(p + c * Vec16<T>::N);
#pragma unroll
                for (int e = 0; e < Vec16<T>::N; ++e) x[c * Vec16<T>::N + e] = y.v[e];
            }
        } else {
            __builtin_memcpy(x, p, sizeof(x));
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = to_f32<T>(x[e]);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = e < n ? to_f32<T>(p[e]) : 0.f;
    }
}
// The same from a row of a matrix that ends at `end`: what follows the row is the next one, so the vector access is safe for all but
// the last columns of the matrix, and the columns past n are never stored.
template <typename T, bool A> __device__ __forceinline__ void load8_before(const T* p, const T* end, int n, float (&v)[VEC]) {
    load8<T, A>(p, A || p + VEC <= end ? VEC : n, v);
}
// OUT: a result, which is written once, goes past the caches where a lane's eight columns are one access (bf16), so that the rows read again
// stay in them: 126,821 tokens of 1,024 columns, the table's gradient 102 -> 84 us, lookups repeated on one table 91 -> 55 us.  Eight floats
// are two accesses 32 bytes apart, which took twice the time that way.
template <typename T, bool A, bool OUT> __device__ __forceinline__ void store8(T* p, int n, const float (&v)[VEC]) {
    if constexpr (A && OUT && sizeof(T) == 2) {
        typedef unsigned words_t __attribute__((ext_vector_type(4)));
        Vec16<T> y;
#pragma unroll
        for (int e = 0; e < VEC; ++e) y.v[e] = from_f32<T>(v[e]);
        __builtin_nontemporal_store(__builtin_bit_cast(words_t, y), reinterpret_cast<words_t*>(p));
    } else if constexpr (A) {
#pragma unroll
        for (int c = 0; c < VEC / Vec16<T>::N; ++c) {
            Vec16<T> y;
#pragma unroll
            for (int e = 0; e < Vec16<T>::N; ++e) y.v[e] = from_f32<T>(v[c * Vec16<T>::N + e]);
            st16(p + c * Vec16<T>::N, y);
        }
    } else if (n >= VEC) {
        T x[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = from_f32<T>(v[e]);
        __builtin_memcpy(p, x, sizeof(x));
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (e < n) p[e] = from_f32<T>(v[e]);
    }
}

// A wave clears a row that may begin anywhere: whole 16-byte pieces, one to a lane, whatever the row's alignment.  The gradient of 420 tokens
// for 26,692 rows of 977 floats 31 us, of 100,000 rows of 512 40 us (5.1 TB/s); by eight columns to a lane 54 and 49 us, past the
// caches 37 and 48.
template <typename T> __device__ __forceinline__ void clear_row(T* row, int n, int lane) {
    constexpr int E = Vec16<T>::N;
    typedef unsigned words_t __attribute__((ext_vector_type(4)));
    const int head = min(n, (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T)), body = (n - head) / E * E;
    if (lane < head) row[lane] = (T)0.f;
    for (int c = lane * E; c < body; c += 64 * E) {
        *reinterpret_cast<words_t*>(row + head + c) = words_t{0, 0, 0, 0};
    }
    if (head + body + lane < n) row[head + body + lane] = (T)0.f;
}

// ---- lookup: one thread per eight columns of a row ---------------------------------------------------------------------------
// 126,821 tokens of 1,024 bf16 columns, words by Zipf's law: 84 us, 3.1 TB/s of results written and as much read, in part from the caches.
// 768 tokens of 512: 2.8 us, which is the launch.
template <typename TT, typename TO, bool A, typename I>
__global__ __launch_bounds__(256) void embed_rows_kernel(const void* __restrict__ ids, int wide, const TT* __restrict__ table, long long ld_table,
                                                         const TT* __restrict__ pos, long long ld_pos, TO* __restrict__ out, float scale,
                                                         long long n, int T, int H, int vocab) {
    const I per_row = (H + VEC - 1) / VEC, total = (I)n * per_row, stride = (I)gridDim.x * 256;
    const TT *table_end = table + (vocab - 1) * ld_table + H, *pos_end = pos ? pos + (T - 1) * ld_pos + H : nullptr;
    for (I i = (I)blockIdx.x * 256 + threadIdx.x; i < total; i += stride) {
        const I r = i / per_row;
        const int c = (int)(i - r * per_row) * VEC, m = H - c;
        float v[VEC];
        load8_before<TT, A>(table + load_id(ids, wide, r, vocab) * ld_table + c, table_end, m, v);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] *= scale;
        if (pos) {
            float p[VEC];
            load8_before<TT, A>(pos + (long long)(r % (I)T) * ld_pos + c, pos_end, m, p);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] += p[e];
        }
        store8<TO, A, true>(out + (long long)r * H + c, m, v);
    }
}

// ---- stable radix sort of (word, token index) ----------------------------------------------------------------------------
// Two launches a pass instead of one with a look-back: at most 64 workgroups, none waits for another.  126,821 tokens: 4.7 and 10.5 us a pass,
// the latency of 2 x 1024 keys per workgroup one after another, beside 84 us of sums.
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
    {
        constexpr int PARTS = SORT_THREADS / MAX_DIGITS;
        const int dig = tid & (MAX_DIGITS - 1), blocks = gridDim.x;
#pragma unroll 8
        for (int b = tid / MAX_DIGITS; b < blocks; b += PARTS) {
            const unsigned c = a.hist[b * MAX_DIGITS + dig];
            total += c;
            before += b < (int)blockIdx.x ? c : 0u;
        }
        if (tid >= MAX_DIGITS) {
            wc[tid / MAX_DIGITS][dig] = total;
            wc[SORT_WAVES / 2 + tid / MAX_DIGITS][dig] = before;
        }
        __syncthreads();
        if (tid < MAX_DIGITS)
#pragma unroll
            for (int p = 1; p < PARTS; ++p) {
                total += wc[p][tid];
                before += wc[SORT_WAVES / 2 + p][tid];
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
    float *head, *tail;     // [chunks][Hs] partial rows of runs that began before the chunk / go on after it
    long long n;
    int H, Hs, vocab, chunk, chunks, slabs;  // Hs: H rounded up to eight columns
    int cleared;            // the rows of words that do not occur are cleared already
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

// Bound by memory: 126,821 rows of 1,024 bf16 columns read, 65,537 written: 84 us, 4.7 TB/s.  7,680 rows of 512 (480 waves): 8 us, the latency of
// words, then rows, then results.
// A wave takes one chunk of the sorted list and one slab of 64*VEC columns; the waves behind those clear the rows of words that
// do not occur, 64 rows each.
template <typename TG, typename TO, bool A> __global__ __launch_bounds__(256) void embed_sum_kernel(SumArgs a) {
    const int lane = threadIdx.x & 63;
    const long long unit = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sums = (long long)a.chunks * a.slabs;
    const TG *g = (const TG*)a.g, *g_end = g + a.n * a.H;
    TO* dt = (TO*)a.d_table;
    if (unit >= sums) {
        const long long v0 = (unit - sums) * 64;
        if (a.cleared || v0 >= a.vocab) return;
        const int v = (int)v0 + lane;
        bool absent = false;
        if (v < a.vocab) {
            const int p = lower_bound_key(a.key, (int)a.n, v);
            absent = p >= (int)a.n || a.key[p] != v;
        }
        unsigned long long todo = __ballot(absent);
        while (todo) {
            const int r = __ffsll((unsigned long long)todo) - 1;
            todo &= todo - 1;
            clear_row(dt + (v0 + r) * a.H, a.H, lane);
        }
        return;
    }
    const int chunk = (int)(unit / a.slabs), slab = (int)(unit - (long long)chunk * a.slabs);
    const int col = (slab * 64 + lane) * VEC, m = a.H - col;
    const bool live = m > 0;
    const int i0 = chunk * a.chunk, i1 = i0 + a.chunk < (int)a.n ? i0 + a.chunk : (int)a.n;
    const bool cont_in = i0 > 0 && a.key[i0 - 1] == a.key[i0];
    const bool cont_out = i1 < (int)a.n && a.key[i1] == a.key[i1 - 1];
    // a chunk is at most 64 rows: lane i holds the i-th word and token
    const int my = i0 + lane < i1 ? i0 + lane : i1 - 1, my_key = a.key[my], my_idx = a.idx[my];
    float acc[VEC] = {};
    bool first = true;  // still in the run the chunk began with
    int word = __builtin_amdgcn_readlane(my_key, 0);
    constexpr int U = 8;  // rows in flight
    const int rows = i1 - i0;
    for (int i = 0; i < rows; i += U) {
        float v[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = i + u < rows ? i + u : rows - 1;
            const long long row = __builtin_amdgcn_readlane(my_idx, j);
            if (live) load8_before<TG, A>(g + row * a.H + col, g_end, m, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u >= rows) break;
            const int w = __builtin_amdgcn_readlane(my_key, i + u);
            if (w != word) {  // the run ended: the same branch for the whole wave
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = first && cont_in ? acc[e] : acc[e] * a.scale;
                if (live) {
                    if (first && cont_in) store8<float, true, false>(a.head + (long long)chunk * a.Hs + col, m, acc);
                    else store8<TO, A, true>(dt + (long long)word * a.H + col, m, acc);
                }
                first = false;
                word = w;
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] += live ? v[u][e] : 0.f;
        }
    }
    if (!live) return;
    if (first && cont_in) {
        store8<float, true, false>(a.head + (long long)chunk * a.Hs + col, m, acc);
    } else if (cont_out) {
        store8<float, true, false>(a.tail + (long long)chunk * a.Hs + col, m, acc);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= a.scale;
        store8<TO, A, true>(dt + (long long)word * a.H + col, m, acc);
    }
}

// Joins the partial rows of a run that crosses chunks, in the order of the chunks: the tail of the chunk it begins in (the owner),
// then the heads of the following chunks, all of which begin with its word.  Most such runs cross one border and a wave each does
// them; a run over more than JOIN_LONG chunks takes a workgroup of 16 waves, found by the one chunk number in JOIN_LONG that is a
// multiple of it and the first such in the run.  10.8 us at 126,821 tokens, 5 us at 7,680 of which half are one word.
constexpr int JOIN_LONG = 32;

// W columns of a lane (8, or 1 where a run is long)
template <int W> __device__ __forceinline__ void add_partials(const SumArgs& a, int owner, int lo, int hi, int col, bool live, float (&acc)[W]) {
    constexpr int U = W == 1 ? 16 : 8;
    for (int k = lo; k < hi; k += U) {
        float v[U][W];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = k + u < hi ? k + u : hi - 1;
            if (!live) continue;
            const float* p = (j == 0 ? a.tail : a.head) + (long long)(owner + j) * a.Hs + col;
            if constexpr (W == 1) v[u][0] = *p;
            else load8<float, true>(p, W, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < W; ++e) acc[e] += live && k + u < hi ? v[u][e] : 0.f;
    }
}

template <typename TO, bool A> __global__ __launch_bounds__(1024) void embed_join_kernel(SumArgs a, int long_blocks) {
    __shared__ float part[16][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TO* dt = (TO*)a.d_table;
    float acc[VEC] = {};
    if ((int)blockIdx.x >= long_blocks) {  // a wave per chunk and slab
        const long long unit = (long long)(blockIdx.x - long_blocks) * 16 + wave;
        const int chunk = (int)(unit / a.slabs), slab = (int)(unit - (long long)chunk * a.slabs);
        if (chunk >= a.chunks - 1) return;
        const int i0 = chunk * a.chunk, i1 = i0 + a.chunk, word = a.key[i1 - 1];
        if (a.key[i1] != word) return;
        if (i0 > 0 && a.key[i0] == word && a.key[i0 - 1] == word) return;  // began in an earlier chunk
        const int next = chunk + 1 + lane;
        const unsigned long long same = __ballot(next < a.chunks && a.key[(long long)(next < a.chunks ? next : chunk) * a.chunk] == word);
        const int m = 1 + __popcll(same);
        if (m > JOIN_LONG) return;
        const int col = (slab * 64 + lane) * VEC;
        const bool live = col < a.H;
        add_partials<VEC>(a, chunk, 0, m, col, live, acc);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] *= a.scale;
        if (live) store8<TO, A, true>(dt + (long long)word * a.H + col, a.H - col, acc);
        return;
    }
    // 64 columns each, so that a run's partial rows are read by several compute units
    const int slabs = (a.H + 63) / 64, at = (blockIdx.x / slabs + 1) * JOIN_LONG, slab = blockIdx.x % slabs;  // at < chunks
    const int word = a.key[(long long)at * a.chunk];
    {  // most runs are short: the chunks at - 32 .. at + 31 tell
        const int near = at - 32 + lane;
        const unsigned long long same = __ballot(near < a.chunks && a.key[(long long)(near < a.chunks ? near : at) * a.chunk] == word);
        if (__popcll(same) < JOIN_LONG - 1) return;  // the same for every wave
    }
    int before = 0, after = 0;  // chunks before `at`, and from `at` on, that begin with the word
    for (int c = at - 1;; c -= 1024) {
        const int mine = c - (int)threadIdx.x;
        const int more = __syncthreads_count(mine >= 0 && a.key[(long long)(mine >= 0 ? mine : 0) * a.chunk] == word);
        before += more;
        if (more < 1024) break;
    }
    for (int c = at;; c += 1024) {
        const int mine = c + (int)threadIdx.x;
        const int more = __syncthreads_count(mine < a.chunks && a.key[(long long)(mine < a.chunks ? mine : at) * a.chunk] == word);
        after += more;
        if (more < 1024) break;
    }
    const int begin = at - before;  // the first chunk that begins with the word; the run may begin before it
    const int owner = begin > 0 && a.key[(long long)begin * a.chunk - 1] == word ? begin - 1 : begin;
    const int m = at + after - owner;
    if (m <= JOIN_LONG || at <= owner || at - JOIN_LONG > owner) return;
    const int col = slab * 64 + lane;
    float sum[1] = {};
    add_partials<1>(a, owner, (int)((long long)m * wave / 16), (int)((long long)m * (wave + 1) / 16), col, col < a.H, sum);
    part[wave][lane] = sum[0];
    __syncthreads();
    if (wave == 0 && col < a.H) {
        float t = part[0][lane];
#pragma unroll
        for (int w = 1; w < 16; ++w) t += part[w][lane];
        dt[(long long)word * a.H + col] = from_f32<TO>(t * a.scale);
    }
}

// ---- sum over sequences: columns of a [B][W] matrix, W = T*H; `slices` of the rows leave fp32 partial rows when there are several
// A workgroup takes L * N columns, N to a lane; its 1024 / L groups of L lanes share the rows.  With L = 16 and N = 8 a batch of 256 captions
// of 30 x 512 columns is 120 workgroups with one round of loads each, two to a compute unit: the first launch of the gradient takes 11 us, with L = 64
// and one workgroup to a compute unit it took 5 us more.
template <typename TG, typename TO, int L, int N, bool A>
__device__ __forceinline__ void colsum(float* lds, const TG* __restrict__ g, TO* __restrict__ out, float* __restrict__ part_out, int B, long long W, int slices,
                                       long long group, int slice) {
    constexpr int C = L * N, SHARES = 1024 / L, PARTS = 1024 / C, U = 4;
    static_assert(SHARES % PARTS == 0, "whole shares");
    const int lane = threadIdx.x % L, share = threadIdx.x / L;
    const long long col = group * C + lane * N;
    const bool live = col < W;
    const int m = W - col < N ? (int)(W - col) : N;
    const int b0 = (int)((long long)B * slice / slices), b1 = (int)((long long)B * (slice + 1) / slices), rows = b1 - b0;
    const int lo = b0 + (int)((long long)rows * share / SHARES), hi = b0 + (int)((long long)rows * (share + 1) / SHARES);
    float acc[N] = {};
    for (int b = lo; b < hi; b += U) {
        float v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = b + u < hi ? b + u : hi - 1;
            if (!live) continue;
            if constexpr (N == 1) v[u][0] = to_f32<TG>(g[j * W + col]);
            else load8<TG, A>(g + j * W + col, m, v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] += live && b + u < hi ? v[u][e] : 0.f;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) lds[share * C + lane * N + e] = acc[e];
    __syncthreads();
    // the shares of a column in order: PARTS threads take some each, one adds what they leave
    const int c = threadIdx.x % C, part = threadIdx.x / C;
    float t = lds[part * (SHARES / PARTS) * C + c];
#pragma unroll
    for (int k = 1; k < SHARES / PARTS; ++k) t += lds[(part * (SHARES / PARTS) + k) * C + c];
    __syncthreads();
    lds[threadIdx.x] = t;
    __syncthreads();
    const long long at = group * C + c;
    if (part > 0 || at >= W) return;
#pragma unroll
    for (int k = 1; k < PARTS; ++k) t += lds[k * C + c];
    if (slices == 1) out[at] = from_f32<TO>(t);
    else part_out[slice * W + at] = t;
}
template <typename TO> __global__ __launch_bounds__(1024) void embed_colsum_join_kernel(const float* __restrict__ part_in, TO* __restrict__ out, int parts, long long W) {
    __shared__ float lds[1024];
    colsum<float, TO, 64, 1, true>(lds, part_in, out, nullptr, parts, W, 1, blockIdx.x, 0);
}

// ---- the first launch of the gradient: three jobs that need nothing from each other, by block number -------------------------
//  1. sorting: up to 8,192 tokens every token's place by counting the tokens that come before it; else the first histogram
//  2. up to 8,192 tokens: the rows of words that do not occur are cleared (with more, embed_sum_kernel does it by searching)
//  3. the sums over sequences
struct FirstArgs {
    SortArgs sort;
    const void* g;
    void *d_table, *d_pos;
    float* pos_part;
    long long W;
    int H, B, slices, rank_blocks, zero_blocks, sum_blocks;
    long long groups;
};
constexpr int SUM_COLUMNS = 16 * VEC;
constexpr int RANK_MAX = 8192, RANK_TOKENS = 32, ZERO_ROWS = 128;
constexpr int RANK_MAX_VOCAB = 1 << 18;  // word and token number share 31 bits

template <typename TG, typename TO, bool A> __global__ __launch_bounds__(1024, 8) void embed_first_kernel(FirstArgs f) {  // two workgroups to a compute unit
    __shared__ __attribute__((aligned(16))) unsigned lds[RANK_MAX + 1024];  // 36 KiB, also the column sums' 1024 x VEC floats
    static_assert(1024 * VEC <= RANK_MAX + 1024, "column sums fit");
    const SortArgs& a = f.sort;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int block = blockIdx.x;
    if (block < f.rank_blocks) {
        // the place of token i is the number of (word, token) pairs below its own
        const int n = (int)a.n, n4 = (n + 127) / 128 * 128;
#pragma unroll 8
        for (int i = tid; i < n4; i += 1024) lds[i] = i < n ? ((unsigned)load_id(a.ids, a.wide, i, a.vocab) << 13) | (unsigned)i : 0xffffffffu;
        __syncthreads();
        // 32 tokens to a workgroup (240 of them for 7,680 tokens), a half wave per thirty-second of the list
        const int i = block * RANK_TOKENS + (lane & 31), part = tid >> 5;
        const unsigned mine = lds[i < n ? i : n - 1];
        unsigned count = 0;
        const int per = n4 / 32;
        const uint4* p = reinterpret_cast<const uint4*>(lds + part * per);
#pragma unroll 4
        for (int k = 0; k < per / 4; ++k) {
            const uint4 c = p[k];
            count += (c.x < mine) + (c.y < mine) + (c.z < mine) + (c.w < mine);
        }
        unsigned* counts = lds + RANK_MAX;
        counts[tid] = count;
        __syncthreads();
        if (tid < RANK_TOKENS && i < n) {
            unsigned at = 0;
#pragma unroll
            for (int w = 0; w < 32; ++w) at += counts[w * 32 + tid];
            a.key_out[at] = (int)(mine >> 13);
            a.idx_out[at] = i;
        }
        return;
    }
    block -= f.rank_blocks;
    if (block < f.zero_blocks) {
        const int v0 = block * ZERO_ROWS, n = (int)a.n;
        if (tid < ZERO_ROWS) lds[tid] = 0;
        __syncthreads();
#pragma unroll 8
        for (int i = tid; i < n; i += 1024) {
            const int v = load_id(a.ids, a.wide, i, a.vocab) - v0;
            if (v >= 0 && v < ZERO_ROWS) lds[v] = 1;
        }
        __syncthreads();
        for (int r = wave; r < ZERO_ROWS && v0 + r < a.vocab; r += 16)
            if (!lds[r]) clear_row((TO*)f.d_table + (long long)(v0 + r) * f.H, f.H, lane);
        return;
    }
    for (long long i = block - f.zero_blocks; i < f.groups * f.slices; i += f.sum_blocks) {
        colsum<TG, TO, 16, VEC, A>(reinterpret_cast<float*>(lds), (const TG*)f.g, (TO*)f.d_pos, f.pos_part, f.B, f.W, f.slices, i % f.groups, (int)(i / f.groups));
        __syncthreads();
    }
}

// ---- the gradient's plan: everything that depends on the sizes alone -------------------------------------------------------
struct GradPlan {
    bool rank;              // few tokens: places by counting
    int sort_blocks, per_block, passes, bits;
    int chunk, chunks, slices;
    long long key[2], idx[2], hist, head, tail, pos, bytes;  // byte offsets into the workspace
};

long long up256(long long b) { return (b + 255) / 256 * 256; }

GradPlan grad_plan(long long n, int T, int H, int vocab, bool want_pos) {
    GradPlan p = {};
    p.rank = n > 0 && n <= RANK_MAX && vocab <= RANK_MAX_VOCAB;
    int blocks = (int)((n + SORT_THREADS - 1) / SORT_THREADS);
    blocks = blocks < 1 ? 1 : blocks > MAX_SORT_BLOCKS ? MAX_SORT_BLOCKS : blocks;
    p.per_block = (int)(((n + blocks - 1) / blocks + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS);
    if (p.per_block < SORT_THREADS) p.per_block = SORT_THREADS;
    p.sort_blocks = (int)((n + p.per_block - 1) / p.per_block);
    int nb = 1;
    while (nb < 31 && (1ll << nb) < vocab) ++nb;
    p.passes = (nb + 8) / 9;
    p.bits = (nb + p.passes - 1) / p.passes;
    // a wave per chunk and 512 columns: about 4,096 of them, 16 to 64 rows each
    const int slabs = (H + 511) / 512;
    long long c = n * slabs / 4096;
    p.chunk = (int)(c < 16 ? 16 : c > 64 ? 64 : c);  // at most the 64 lanes that hold a chunk's words
    p.chunks = (int)((n + p.chunk - 1) / p.chunk);
    long long o = 0;
    for (int i = 0; i < 2; ++i) {
        p.key[i] = o; o += up256(n * 4);
        p.idx[i] = o; o += up256(n * 4);
    }
    p.hist = o; o += up256((long long)p.sort_blocks * MAX_DIGITS * 4);
    const long long row = (H + VEC - 1) / VEC * VEC * 4;
    p.head = o; o += up256(p.chunks * row);
    p.tail = o; o += up256(p.chunks * row);
    p.slices = 1;
    if (want_pos) {
        // up to 256 workgroups over the columns of [B][T*H], at least 256 sequences (a round of loads) to a slice
        const long long B = n / T, groups = ((long long)T * H + SUM_COLUMNS - 1) / SUM_COLUMNS;
        long long s = 256 / (groups < 1 ? 1 : groups);
        if (s > B / 256) s = B / 256;
        p.slices = (int)(s < 1 ? 1 : s > 512 ? 512 : s);
        p.pos = o;
        if (p.slices > 1) o += up256((long long)p.slices * T * H * 4);
    }
    p.bytes = o;
    return p;
}

// columns of a row, and elements of d_pos
constexpr int MAX_H = 1 << 20;
constexpr long long MAX_POS = 1ll << 31;

bool ok_dtype(int d) { return d == MIC_F32 || d == MIC_BF16; }

template <typename TG, typename TO, bool A>
int launch_grad(const GradPlan& p, const void* ids, int wide, const void* g, void* d_table, void* d_pos, float scale, long long n, int T, int H, int vocab,
                char* ws, hipStream_t s) {
    SortArgs a = {};
    a.wide = wide; a.vocab = vocab; a.n = n; a.per_block = p.per_block; a.bits = p.bits;
    a.hist = (unsigned*)(ws + p.hist);
    a.ids = ids;
    a.key_out = (int*)(ws + p.key[0]);
    a.idx_out = (int*)(ws + p.idx[0]);
    FirstArgs f = {};
    f.sort = a;
    f.g = g; f.d_table = d_table; f.d_pos = d_pos; f.H = H;
    f.pos_part = (float*)(ws + p.pos);
    if (p.rank) {
        f.rank_blocks = (int)((n + RANK_TOKENS - 1) / RANK_TOKENS);
        f.zero_blocks = (vocab + ZERO_ROWS - 1) / ZERO_ROWS;
    }
    if (d_pos) {
        f.B = (int)(n / T);
        f.W = (long long)T * H;
        f.slices = p.slices;
        f.groups = (f.W + SUM_COLUMNS - 1) / SUM_COLUMNS;
        const long long sums = f.groups * f.slices;
        f.sum_blocks = (int)(sums < 1 << 20 ? sums : 1 << 20);  // a launch has fewer than 2^32 threads
    }
    const long long first = f.rank_blocks + f.zero_blocks + f.sum_blocks;
    if (first > 0) MIC_LAUNCH((embed_first_kernel<TG, TO, A>), dim3((unsigned)first), dim3(1024), 0, s, f);
    if (d_pos && p.slices > 1)
        MIC_LAUNCH((embed_colsum_join_kernel<TO>), dim3((unsigned)((f.W + 63) / 64)), dim3(1024), 0, s, (const float*)f.pos_part, (TO*)d_pos, p.slices, f.W);
    const int passes = p.rank ? 1 : p.passes;
    for (int i = 0; i < passes && !p.rank && n > 0; ++i) {
        a.ids = i == 0 ? ids : nullptr;
        a.key_in = (const int*)(ws + p.key[(i + 1) & 1]);
        a.idx_in = (const int*)(ws + p.idx[(i + 1) & 1]);
        a.key_out = (int*)(ws + p.key[i & 1]);
        a.idx_out = (int*)(ws + p.idx[i & 1]);
        a.shift = i * p.bits;
        MIC_LAUNCH(embed_hist_kernel, dim3(p.sort_blocks), dim3(SORT_THREADS), 0, s, a);
        MIC_LAUNCH(embed_scatter_kernel, dim3(p.sort_blocks), dim3(SORT_THREADS), 0, s, a);
    }
    SumArgs m = {};  // (no tokens: no chunks, and every row is one of a word that does not occur)
    m.key = (const int*)(ws + p.key[(passes - 1) & 1]);
    m.idx = (const int*)(ws + p.idx[(passes - 1) & 1]);
    m.g = g; m.d_table = d_table;
    m.head = (float*)(ws + p.head); m.tail = (float*)(ws + p.tail);
    m.n = n; m.H = H; m.Hs = (H + VEC - 1) / VEC * VEC; m.vocab = vocab; m.chunk = p.chunk; m.chunks = p.chunks; m.scale = scale; m.cleared = p.rank;
    m.slabs = (H + 64 * VEC - 1) / (64 * VEC);
    const long long units = (long long)p.chunks * m.slabs + (p.rank ? 0 : ((long long)vocab + 63) / 64);
    MIC_LAUNCH((embed_sum_kernel<TG, TO, A>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, s, m);
    if (p.chunks > 1) {
        const int long_blocks = (p.chunks - 1) / JOIN_LONG * ((H + 63) / 64);
        const long long waves = (long long)(p.chunks - 1) * m.slabs;
        MIC_LAUNCH((embed_join_kernel<TO, A>), dim3((unsigned)(long_blocks + (waves + 15) / 16)), dim3(1024), 0, s, m, long_blocks);
    }
    return 0;
}

}  // namespace

extern "C" int mic_embed_rows(const void* ids, int ids_bits, const void* table, int64_t ld_table, const void* pos, int64_t ld_pos, void* out,
                              int table_dtype, int out_dtype, float scale, int64_t n, int T, int H, int vocab, void* stream) {
    MIC_ARG_CHECK(n >= 0 && n < (1ll << 31) && T > 0 && H > 0 && H <= MAX_H && vocab > 0, "mic_embed_rows: bad sizes n=%lld T=%d H=%d vocab=%d", (long long)n, T, H, vocab);
    MIC_ARG_CHECK(ids_bits == 32 || ids_bits == 64, "mic_embed_rows: token ids of %d bits", ids_bits);
    MIC_ARG_CHECK(ok_dtype(table_dtype) && ok_dtype(out_dtype), "mic_embed_rows: bad dtype %d / %d", table_dtype, out_dtype);
    MIC_ARG_CHECK(ld_table >= H && (!pos || ld_pos >= H), "mic_embed_rows: row stride below H=%d", H);
    if (n == 0) return 0;
    MIC_ARG_CHECK(ids && table && out, "mic_embed_rows: null pointer");
    hipStream_t s = (hipStream_t)stream;
    const bool vec = H % 8 == 0 && ld_table % 8 == 0 && (!pos || ld_pos % 8 == 0) && (((uintptr_t)table | (uintptr_t)out | (uintptr_t)pos) & 15) == 0;
    const long long work = n * ((H + VEC - 1) / VEC);
    const long long blocks = (work + 255) / 256;
    const dim3 grid((unsigned)(blocks > 1048576 ? 1048576 : blocks));
    const bool small = work < (1ll << 31);  // 32-bit index arithmetic: a 64-bit division costs as much as the rest of the thread
#define GO_I(TT, TO, A, I)                                                                                                                     \
    MIC_LAUNCH((embed_rows_kernel<TT, TO, A, I>), grid, dim3(256), 0, s, ids, ids_bits == 64, (const TT*)table, (long long)ld_table, (const TT*)pos, \
               (long long)ld_pos, (TO*)out, scale, (long long)n, T, H, vocab)
#define GO(TT, TO, A)                       \
    do {                                    \
        if (small) GO_I(TT, TO, A, unsigned); \
        else GO_I(TT, TO, A, long long);    \
    } while (0)
#define GO_VEC(TT, TO)             \
    do {                           \
        if (vec) GO(TT, TO, true);    \
        else GO(TT, TO, false);        \
    } while (0)
    if (table_dtype == MIC_F32 && out_dtype == MIC_F32) GO_VEC(float, float);
    else if (table_dtype == MIC_F32) GO_VEC(float, bf16_t);
    else if (out_dtype == MIC_F32) GO_VEC(bf16_t, float);
    else GO_VEC(bf16_t, bf16_t);
#undef GO_I
#undef GO
#undef GO_VEC
    return 0;
}

extern "C" int64_t mic_embed_grad_workspace_bytes(int64_t n, int T, int H, int vocab, int want_pos) {
    if (n < 0 || n >= (1ll << 30) || T <= 0 || H <= 0 || H > MAX_H || vocab <= 0 || (want_pos && (n % T != 0 || (long long)T * H >= MAX_POS))) return MIC_ERR_ARG;
    return grad_plan(n, T, H, vocab, want_pos != 0).bytes;
}

extern "C" int mic_embed_grad(const void* ids, int ids_bits, const void* g, void* d_table, void* d_pos, int g_dtype, int out_dtype, float scale,
                              int64_t n, int T, int H, int vocab, void* workspace, int64_t workspace_bytes, void* stream) {
    MIC_ARG_CHECK(n >= 0 && n < (1ll << 30) && T > 0 && H > 0 && H <= MAX_H && vocab > 0 && (!d_pos || (long long)T * H < MAX_POS),
                  "mic_embed_grad: bad sizes n=%lld T=%d H=%d vocab=%d", (long long)n, T, H, vocab);
    MIC_ARG_CHECK(ids_bits == 32 || ids_bits == 64, "mic_embed_grad: token ids of %d bits", ids_bits);
    MIC_ARG_CHECK(ok_dtype(g_dtype) && ok_dtype(out_dtype), "mic_embed_grad: bad dtype %d / %d", g_dtype, out_dtype);
    MIC_ARG_CHECK(!d_pos || n % T == 0, "mic_embed_grad: %lld tokens are not whole sequences of %d", (long long)n, T);
    MIC_ARG_CHECK(d_table && (n == 0 || (ids && g)), "mic_embed_grad: null pointer");
    const GradPlan p = grad_plan(n, T, H, vocab, d_pos != nullptr);
    MIC_ARG_CHECK(workspace_bytes >= p.bytes && (p.bytes == 0 || workspace), "mic_embed_grad: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, p.bytes);
    MIC_ARG_CHECK(((uintptr_t)workspace & 15) == 0, "mic_embed_grad: workspace is not 16-byte aligned");
    hipStream_t s = (hipStream_t)stream;
    const bool vec = H % 8 == 0 && (((uintptr_t)g | (uintptr_t)d_table | (uintptr_t)d_pos) & 15) == 0;
#define GO(TG, TO, A) return launch_grad<TG, TO, A>(p, ids, ids_bits == 64, g, d_table, d_pos, scale, n, T, H, vocab, (char*)workspace, s)
#define GO_VEC(TG, TO)             \
    do {                           \
        if (vec) GO(TG, TO, true);    \
        else GO(TG, TO, false);        \
    } while (0)
    if (g_dtype == MIC_F32 && out_dtype == MIC_F32) GO_VEC(float, float);
    else if (g_dtype == MIC_F32) GO_VEC(float, bf16_t);
    else if (out_dtype == MIC_F32) GO_VEC(bf16_t, float);
    else GO_VEC(bf16_t, bf16_t);
#undef GO
#undef GO_VEC
}
