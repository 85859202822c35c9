// Softmax cross entropy of a linear layer over the vocabulary, without keeping the logits:
//   z = x w^T + bias     lse = log sum_v exp z_v     loss = lse - z_target
//   d = weight * (exp(z - lse) - onehot(target))     dx = d w     dw = d^T x     dbias = column sums of d
// Forward: a wave's part of a logits' tile ends in the statistics (maximum, sum) of its columns (64, 32 on the smallest tiles); a second
// launch joins a row's parts.
// Gradient: piece by piece of the vocabulary the logits are computed again, their epilogue turns them into d (rounded to bf16 for
// bf16 operands: both remaining products take it as a matrix-core operand; dbias is summed before the rounding), and two more
// products use the piece.  dw's rows of a piece are complete; dx is summed over the pieces in fp32.
// Rows that do not count (padding: half of a batch of captions) have no gradient, so the gradient's products run over the counted
// rows alone, whatever the others hold: they are gathered first, their number stays on the device, and workgroups behind the last one
// end at once.
//
// Two kernels: 256 x 256 tiles for bf16 (vocab_gemm8.h), 128 x 128 and 64 x 64 tiles for fp32 and for products too small to fill the
// larger ones (vocab_gemm.h).
#include "vocab_gemm.h"
#include "vocab_gemm8.h"

namespace {

constexpr int MAX_IGNORE = 4;
struct Targets {
    const void* t;
    int wide, n_ignore, V;
    int ignore[MAX_IGNORE];
};
// the row's target, or -1 where the row does not count
__device__ __forceinline__ int target_of(const Targets& t, int row) {
    const long long v = t.wide ? ((const long long*)t.t)[row] : (long long)((const int*)t.t)[row];
    if (v < 0 || v >= t.V) return -1;
    for (int i = 0; i < t.n_ignore; ++i)
        if (v == t.ignore[i]) return -1;
    return (int)v;
}

// ---- epilogue: statistics of a wave's columns of logits (half a tile) per row -------------------------------------------------
struct StatsEpi {
    struct Args {
        const float* bias;
        Targets t;
        float2* part;  // [parts][N]
        float* zt;     // [N] logit of the target
        int N, V, parts;
    };
    template <int S> __device__ static __forceinline__ void run(const Args& a, f32x16_t (&acc)[S][S], int p0, int q0, int lane, int tp, int, int) {
        const int h = lane >> 5;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int row = q0 + j * 32 + (lane & 31);
            const int t = row < a.N ? target_of(a.t, row) : -1;
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int v = p0 + i * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
                    float z = acc[i][j][e];
                    if (v < a.V) z += a.bias ? a.bias[v] : 0.f;
                    else z = -INFINITY;
                    if (v == t) a.zt[row] = z;
                    acc[i][j][e] = z;
                    m = fmaxf(m, z);
                }
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            const float m_use = m == -INFINITY ? 0.f : m;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f((acc[i][j][e] - m_use) * ATTN_LOG2E);
            s += __shfl_xor(s, 32, 64);
            if (h == 0 && row < a.N) a.part[(long long)tp * a.N + row] = make_float2(m, s);
        }
    }
};

// joins the parts of a row: 16 rows to a workgroup, 64 threads share a row's parts
__global__ __launch_bounds__(1024) void vocab_loss_rows_kernel(const float2* __restrict__ part, const float* __restrict__ zt, Targets t, float* __restrict__ loss,
                                                               float* __restrict__ lse, int N, int parts) {
    __shared__ float2 sum[64][16];
    const int lane = threadIdx.x & 15, share = threadIdx.x >> 4, row = blockIdx.x * 16 + lane;
    float m = -INFINITY, s = 0.f;
    if (row < N)
#pragma unroll 4
        for (int i = share; i < parts; i += 64) {
            const float2 p = part[(long long)i * N + row];
            const float top = fmaxf(m, p.x), use = top == -INFINITY ? 0.f : top;
            s = s * __builtin_amdgcn_exp2f((m - use) * ATTN_LOG2E) + p.y * __builtin_amdgcn_exp2f((p.x - use) * ATTN_LOG2E);
            m = top;
        }
    sum[share][lane] = make_float2(m, s);
    for (int d = 32; d > 0; d >>= 1) {
        __syncthreads();
        if (share < d) {
            const float2 o = sum[share + d][lane];
            const float top = fmaxf(m, o.x), use = top == -INFINITY ? 0.f : top;
            s = s * __builtin_amdgcn_exp2f((m - use) * ATTN_LOG2E) + o.y * __builtin_amdgcn_exp2f((o.x - use) * ATTN_LOG2E);
            m = top;
            sum[share][lane] = make_float2(m, s);
        }
    }
    if (share == 0 && row < N) {
        const float l = m + logf(s);
        lse[row] = l;
        loss[row] = target_of(t, row) >= 0 ? l - zt[row] : 0.f;
    }
}

// ---- epilogue: logits -> d --------------------------------------------------------------------------------------------------
// What a row of the gradient needs, in the order of the gathered rows
struct RowInfo {
    const int* target;
    const float *lse, *weight;
};
template <typename T> struct GradEpi {
    struct Args {
        const float* bias;
        RowInfo r;
        T* d;            // [N][ld], columns from v0 on
        float* part_db;  // [parts][Vc] or NULL
        const int* count;  // the rows there are
        int Vc, ld, v0;
    };
    template <int S> __device__ static __forceinline__ void run(const Args& a, f32x16_t (&acc)[S][S], int p0, int q0, int lane, int, int tq, int) {
        const int n = *a.count;
        const int h = lane >> 5;
        float sum[S][16];
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int row = q0 + j * 32 + (lane & 31);
            const int t = row < n ? a.r.target[row] : -1;
            const float w = t >= 0 ? a.r.weight[row] : 0.f, lse2 = t >= 0 ? a.r.lse[row] * ATTN_LOG2E : 0.f;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const int c = p0 + i * 32 + 8 * e4 + 4 * h;  // column of the piece
                    float d[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int v = a.v0 + c + e;
                        float z = acc[i][j][4 * e4 + e];
                        if (a.bias && c + e < a.Vc) z += a.bias[v];
                        const float p = __builtin_amdgcn_exp2f(fmaf(z, ATTN_LOG2E, -lse2));
                        d[e] = t >= 0 && c + e < a.Vc ? w * (v == t ? p - 1.0f : p) : 0.f;
                        sum[i][4 * e4 + e] = (j ? sum[i][4 * e4 + e] : 0.f) + d[e];
                    }
                    if (row < n && c < a.ld) store4<T>(a.d + (long long)row * a.ld + c, d[0], d[1], d[2], d[3]);
                }
        }
        if (a.part_db == nullptr) return;
        // sums over the 32 lanes of a half: every exchange halves the values a lane carries; value x ends in the lanes whose low bits are x
        constexpr int N = 16 * S;
        float v[N];
#pragma unroll
        for (int x = 0; x < N; ++x) v[x] = sum[x >> 4][x & 15];
#pragma unroll
        for (int d = N / 2; d > 0; d >>= 1) {
            const bool up = lane & d;
#pragma unroll
            for (int x = 0; x < d; ++x) {
                const float give = up ? v[x] : v[x + d], keep = up ? v[x + d] : v[x];
                v[x] = keep + __shfl_xor(give, d, 64);
            }
        }
        if (S == 1) v[0] += __shfl_xor(v[0], 16, 64);
        const int x = lane & (N - 1), c = p0 + (x >> 4) * 32 + 8 * ((x & 15) >> 2) + 4 * h + (x & 3);
        if (c < a.Vc) a.part_db[(long long)tq * a.Vc + c] = v[0];
    }
};

// ---- epilogue: fp32 partial results of a slice, or the rounded result ---------------------------------------------------------
template <typename T> struct OutEpi {
    struct Args {
        T* out;        // [Nq][Np] rounded, taken where there is one slice; or NULL
        float* part;   // fp32 [Nq][Np] per slice otherwise, each slice before the last; without `out` one after the other, of *count rows
        const int* count;  // on the device: with `out` the slices, without it the rows there are
        int Np, Nq;
    };
    // the rows to write, and the slice's partial matrix (NULL: write the result)
    __device__ static __forceinline__ int rows(const Args& a) { return a.out ? a.Nq : __builtin_amdgcn_readfirstlane(*a.count); }
    __device__ static __forceinline__ float* part(const Args& a, int slice) {
        if (a.out) return a.part && __builtin_amdgcn_readfirstlane(*a.count) != 1 ? a.part - (long long)slice * a.Nq * a.Np : nullptr;
        return a.part + (long long)slice * rows(a) * a.Np;
    }
    template <int S> __device__ static __forceinline__ void run(const Args& a, f32x16_t (&acc)[S][S], int p0, int q0, int lane, int, int, int slice) {
        const int h = lane >> 5, nq = rows(a);
        float* to = part(a, slice);
        const bool whole = a.Np % 4 == 0;
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const int row = q0 + j * 32 + (lane & 31);
            if (row >= nq) continue;
#pragma unroll
            for (int i = 0; i < S; ++i)
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const int c = p0 + i * 32 + 8 * e4 + 4 * h;
                    const float v[4] = {acc[i][j][4 * e4], acc[i][j][4 * e4 + 1], acc[i][j][4 * e4 + 2], acc[i][j][4 * e4 + 3]};
                    if (to) {
                        float* o = to + (long long)row * a.Np + c;
                        if (whole && c < a.Np) store4<float>(o, v[0], v[1], v[2], v[3]);
                        else if (!whole)
                            for (int e = 0; e < 4; ++e)
                                if (c + e < a.Np) o[e] = v[e];
                    } else {
                        T* o = a.out + (long long)row * a.Np + c;
                        if (whole && c < a.Np) store4<T>(o, v[0], v[1], v[2], v[3]);
                        else if (!whole)
                            for (int e = 0; e < 4; ++e)
                                if (c + e < a.Np) o[e] = from_f32<T>(v[e]);
                    }
                }
        }
    }
};

// ---- the same epilogues on the 256 x 256 tiles: a lane holds 4 consecutive p of 4 tiles for 8 rows --------------------------------
// side buffer: [0] bias of the tile's 256 columns (-infinity past the last word), [1] targets of its 256 rows, [2] weights, [3] lse
struct StatsEpi8 {
    typedef StatsEpi::Args Args;
    static constexpr bool COUNTED = false;
    __device__ static __forceinline__ void side(const Args& a, int p0, int q0, int tid, float* side) {
        const int i = tid & 255;
        if (tid < 256) {
            side[i] = p0 + i < a.V ? (a.bias ? a.bias[p0 + i] : 0.f) : -INFINITY;
        } else {
            reinterpret_cast<int*>(side)[256 + i] = q0 + i < a.N ? target_of(a.t, q0 + i) : -1;
        }
    }
    __device__ static __forceinline__ void run(const Args& a, f32x4_t (&acc)[4][8], int p0, int q0, int lane, int wave, int tp, int, int, const float* side) {
        const int pl = 64 * (wave & 3) + 4 * (lane >> 4), ql = 128 * (wave >> 2) + (lane & 15);
        if (p0 + 64 * (wave & 3) >= a.V) return;  // its parts are not looked at
        float m[8], s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) m[i] = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const f32x4_t b = *reinterpret_cast<const f32x4_t*>(side + pl + 16 * j);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[j][i] += b;
                m[i] = fmaxf(m[i], fmaxf(fmaxf(acc[j][i][0], acc[j][i][1]), fmaxf(acc[j][i][2], acc[j][i][3])));
            }
        }
        bool far = false;
        // the four lanes of a row, all rows at once: an exchange's latency is paid four times, not 32
#pragma unroll
        for (int d = 16; d < 64; d <<= 1) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __shfl_xor(m[i], d, 64);
#pragma unroll
            for (int i = 0; i < 8; ++i) m[i] = fmaxf(m[i], o[i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int tc = reinterpret_cast<const int*>(side)[256 + ql + 16 * i] - p0 - pl;  // the target's column, from the lane's first
            const float m2 = (m[i] == -INFINITY ? 0.f : m[i]) * ATTN_LOG2E;
            s[i] = 0.f;
            if ((unsigned)tc < 64u && (tc & 12) == 0) {  // in this lane's columns
                float z = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) z = tc == 16 * j + e ? acc[j][i][e] : z;
                a.zt[q0 + ql + 16 * i] = z;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[i] += __builtin_amdgcn_exp2f(fmaf(acc[j][i][e], ATTN_LOG2E, -m2));
            far |= fabsf(m2) == INFINITY;
        }
        if (__any(far))  // all hidden by the type's lowest value, the exponent's maximum is not a number of 32 bits: by differences
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float top = m[i] == -INFINITY ? 0.f : m[i];
                s[i] = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[i] += __builtin_amdgcn_exp2f((acc[j][i][e] - top) * ATTN_LOG2E);
            }
#pragma unroll
        for (int d = 16; d < 64; d <<= 1) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = __shfl_xor(s[i], d, 64);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += o[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = q0 + ql + 16 * i;
            if (lane < 16 && row < a.N) a.part[(long long)(tp * 4 + (wave & 3)) * a.N + row] = make_float2(m[i], s[i]);
        }
    }
};

struct GradEpi8 {
    typedef GradEpi<bf16_t>::Args Args;
    static constexpr bool COUNTED = true;
    __device__ static __forceinline__ int rows(const Args& a) { return *a.count; }
    __device__ static __forceinline__ void side(const Args& a, int p0, int q0, int tid, float* side) {
        const int i = tid & 255;
        if (tid < 256) {
            side[i] = p0 + i < a.Vc ? (a.bias ? a.bias[a.v0 + p0 + i] * ATTN_LOG2E : 0.f) : -INFINITY;  // beyond the piece: probability zero
        } else {
            const int row = q0 + i;
            const int t = row < rows(a) ? a.r.target[row] : -1;
            reinterpret_cast<int*>(side)[256 + i] = t < 0 ? -(1 << 30) : t - a.v0 - p0;  // column of the tile, anything outside it for none
            side[512 + i] = t < 0 ? 0.f : a.r.weight[row];
            side[768 + i] = t < 0 ? 0.f : a.r.lse[row] * ATTN_LOG2E;
        }
    }
    __device__ static __forceinline__ void run(const Args& a, f32x4_t (&acc)[4][8], int p0, int q0, int lane, int wave, int, int tq, int, const float* side) {
        const int pl = 64 * (wave & 3) + 4 * (lane >> 4), ql = 128 * (wave >> 2) + (lane & 15), n = rows(a);
        f32x4_t b[4];
        float sum[16];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            b[j] = *reinterpret_cast<const f32x4_t*>(side + pl + 16 * j);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[4 * j + e] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = q0 + ql + 16 * i;
            const int tc = reinterpret_cast<const int*>(side)[256 + ql + 16 * i] - pl;
            const float w = side[512 + ql + 16 * i], lse2 = side[768 + ql + 16 * i];
            const bool counts = tc > -(1 << 29);
            bf16_t* out = a.d + (long long)row * a.ld + p0 + pl;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float d[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float p = __builtin_amdgcn_exp2f(fmaf(acc[j][i][e], ATTN_LOG2E, b[j][e] - lse2));
                    d[e] = counts ? w * (tc == 16 * j + e ? p - 1.0f : p) : 0.f;  // a row that does not count stays zero whatever its logits are
                    sum[4 * j + e] += d[e];
                }
                if (row < n && p0 + pl + 16 * j < a.ld) store4<bf16_t>(out + 16 * j, d[0], d[1], d[2], d[3]);
            }
        }
        if (a.part_db == nullptr) return;
        // sums over 16 lanes, halving the values at every exchange: value x ends in the lane whose low four bits are x
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) {
            const bool up = lane & d;
#pragma unroll
            for (int x = 0; x < d; ++x) {
                const float give = up ? sum[x] : sum[x + d], keep = up ? sum[x + d] : sum[x];
                sum[x] = keep + __shfl_xor(give, d, 64);
            }
        }
        const int x = lane & 15, c = p0 + pl + 16 * (x >> 2) + (x & 3);
        if (c < a.Vc) a.part_db[(long long)(tq * 2 + (wave >> 2)) * a.Vc + c] = sum[0];
    }
};

struct OutEpi8 {
    typedef OutEpi<bf16_t>::Args Args;
    __device__ static __forceinline__ void side(const Args&, int, int, int, float*) {}
    __device__ static __forceinline__ void run(const Args& a, f32x4_t (&acc)[4][8], int p0, int q0, int lane, int wave, int, int, int slice, const float*) {
        const int pw = p0 + 64 * (wave & 3) + 4 * (lane >> 4), qw = q0 + 128 * (wave >> 2) + (lane & 15), nq = OutEpi<bf16_t>::rows(a);
        float* to = OutEpi<bf16_t>::part(a, slice);
        const bool whole = a.Np % 4 == 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = qw + 16 * i;
            if (row >= nq) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = pw + 16 * j;
                const f32x4_t& v = acc[j][i];
                if (to) {
                    float* o = to + (long long)row * a.Np + c;
                    if (whole && c < a.Np) store4<float>(o, v[0], v[1], v[2], v[3]);
                    else if (!whole)
                        for (int e = 0; e < 4; ++e)
                            if (c + e < a.Np) o[e] = v[e];
                } else {
                    bf16_t* o = a.out + (long long)row * a.Np + c;
                    if (whole && c < a.Np) store4<bf16_t>(o, v[0], v[1], v[2], v[3]);
                    else if (!whole)
                        for (int e = 0; e < 4; ++e)
                            if (c + e < a.Np) o[e] = (bf16_t)v[e];
                }
            }
        }
    }
};

// ---- the sums of partial results, by block number in one launch ---------------------------------------------------------------------
// out[row] = the sum of fp32 rows at[row] (negative: zeros) of the partial matrices, in order: `pieces` groups of *slices matrices (the
// last: *slices_last), `room` elements apart, of *counted rows each.  Without `at`: row `row` of *slices_last matrices `stride` elements
// apart, where there are several (one is the result already).
struct SumParts {
    const float* part;
    void* out;
    const int *at, *slices, *slices_last, *counted;
    long long stride, room;
    int rows, cols, pieces;
    unsigned blocks;  // 0: nothing to do
};
template <typename T> __device__ __forceinline__ void sum_parts(const SumParts& a, unsigned block) {
    const int quads = (a.cols + 3) / 4;
    const long long i = (long long)block * 256 + threadIdx.x;
    const int row = (int)(i / quads), c = (int)(i - (long long)row * quads) * 4;
    const int whole = *a.slices, last = *a.slices_last;
    if (row >= a.rows || (!a.at && last == 1)) return;
    const int src = a.at ? a.at[row] : row;
    const long long stride = a.at ? (long long)*a.counted * a.cols : a.stride;
    float s[4] = {};
    if (src >= 0) {
        for (int g = 0; g < a.pieces; ++g) {
            const float* p = a.part + g * a.room + (long long)src * a.cols + c;
            const int parts = g == a.pieces - 1 ? last : whole;
            if (a.cols % 4 == 0) {
#pragma unroll 8
                for (int k = 0; k < parts; ++k) {
                    const float4 x = *reinterpret_cast<const float4*>(p + k * stride);
                    s[0] += x.x; s[1] += x.y; s[2] += x.z; s[3] += x.w;
                }
            } else {
                for (int e = 0; e < 4 && c + e < a.cols; ++e)
                    for (int k = 0; k < parts; ++k) s[e] += p[k * stride + e];
            }
        }
    }
    T* o = (T*)a.out + (long long)row * a.cols + c;
    if (a.cols % 4 == 0) store4<T>(o, s[0], s[1], s[2], s[3]);
    else
        for (int e = 0; e < 4 && c + e < a.cols; ++e) o[e] = from_f32<T>(s[e]);
}
// column sums of a [parts][n] matrix: 16 columns to a workgroup, 16 groups of threads share the rows, added in order
struct ColSum {
    const float* part;
    float* out;
    const int* rows;  // the gathered rows there are: parts of row_tile rows beyond them were not written
    int n, parts, row_tile;
    unsigned blocks;
};
__device__ __forceinline__ void column_sums(const ColSum& a, unsigned block) {
    __shared__ float sum[16][17];
    const int lane = threadIdx.x & 15, group = threadIdx.x >> 4, c = block * 16 + lane;
    const int parts = min(a.parts, (*a.rows + a.row_tile - 1) / a.row_tile);
    const int lo = (int)((long long)parts * group / 16), hi = (int)((long long)parts * (group + 1) / 16);
    float s = 0.f;
#pragma unroll 8
    for (int k = lo; k < hi; ++k) s += c < a.n ? a.part[(long long)k * a.n + c] : 0.f;
    sum[group][lane] = s;
    __syncthreads();
    if (group == 0 && c < a.n) {
        s = sum[0][lane];
#pragma unroll
        for (int w = 1; w < 16; ++w) s += sum[w][lane];
        a.out[c] = s;
    }
}
template <typename T> __global__ __launch_bounds__(256) void vocab_finish_kernel(SumParts x, SumParts y, ColSum b) {
    unsigned block = blockIdx.x;
    if (block < b.blocks) return column_sums(b, block);
    block -= b.blocks;
    if (block < x.blocks) return sum_parts<T>(x, block);
    sum_parts<T>(y, block - x.blocks);
}

// ---- the rows of the gradient ------------------------------------------------------------------------------------------------------
// Target, weight and lse of the counted rows, in their order: `at` tells where a row went (-1: it does not count), *count how many there
// are.  A block counts the rows before its own again (at most 64 blocks) instead of waiting for others.
//
// The last block also decides into how many ranges of k the products dx and dw are cut (of a whole piece and of the last one), now that the
// rows are known.
struct SplitRule {
    float capacity;         // workgroups resident at once
    float fixed, traffic;   // in steps of k: what a workgroup costs beside its steps; what the partial tiles of a full GPU cost
};
struct Split {
    int tiles, nk, most;    // tiles of the result (dx: per tile of rows), steps of k (dw: 0, by the rows), ranges allowed
    long long elements;     // of one partial matrix (dx: per row)
};
// 1 to 10, 12, 16, 24, 32, 48, 64 ranges (i < 16)
constexpr int MAX_SLICES = 64;
__device__ __forceinline__ int slices_at(int i) { return i < 10 ? i + 1 : (i & 1 ? 16 : 12) << ((i - 10) >> 1); }
// The pair of numbers that costs least: a lane looks at one number for x and four for w.  Both products are one launch, whose
// tiles are dealt out in turn: the first workgroups have one tile of x more, or the ones behind them one of w.
// The partial matrices of both have to fit `room` elements; one of x alone does.
__device__ __forceinline__ int2 choose_slices(const SplitRule& r, int tiles_x, int nk_x, int most_x, long long elements_x, int tiles_w, int nk_w, int most_w, long long elements_w,
                                              long long room, int lane) {
    const int sx = slices_at(lane & 15);
    const float all_x = (float)(tiles_x * sx) / r.capacity, some = floorf(all_x), up = ceilf(all_x), kx = ceilf((float)nk_x / sx) + r.fixed;
    float best = INFINITY;
    int at = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int sw = slices_at((lane >> 4) * 4 + i);
        const float all_w = (float)(tiles_w * sw) / r.capacity, rounds = ceilf(all_x + all_w), kw = ceilf((float)nk_w / sw) + r.fixed;
        float cost = fmaxf(up * kx + (rounds - up) * kw, some * kx + (rounds - some) * kw) + (all_x + (sw > 1 ? all_w : 0.f)) * r.traffic;
        if (sx > most_x || sw > most_w || sx * elements_x + (sw > 1 ? sw * elements_w : 0) > room) cost = INFINITY;
        if (cost < best) {
            best = cost;
            at = sw * 128 + sx;
        }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const float c = __shfl_xor(best, d, 64);
        const int o = __shfl_xor(at, d, 64);
        if (c < best || (c == best && o < at)) {
            best = c;
            at = o;
        }
    }
    return make_int2(at & 127, at >> 7);
}
enum { COUNT, SX, SX_LAST, SW, SW_LAST, DECISIONS };  // what `count` points to
struct RowsArgs {
    Targets t;
    const float *weight, *lse;
    int *target_out, *at, *count;
    float *weight_out, *lse_out;
    int N, per_block;
    SplitRule rule;
    Split dx[2], dw[2];     // whole pieces, the last one
    long long room;         // elements for the partial matrices of a piece
    int edge, ks;
};
__global__ __launch_bounds__(1024) void vocab_rows_kernel(RowsArgs a) {
    __shared__ int wave_sum[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int lo = blockIdx.x * a.per_block, hi = min(a.N, lo + a.per_block);
    int base = 0, mine = 0;
#pragma unroll 4
    for (int i = tid; i < lo; i += 1024) mine += target_of(a.t, i) >= 0;
    for (int d = 32; d > 0; d >>= 1) mine += __shfl_xor(mine, d, 64);
    if (lane == 0) wave_sum[wave] = mine;
    __syncthreads();
    for (int w = 0; w < 16; ++w) base += wave_sum[w];
    __syncthreads();
    for (int r = lo; r < hi; r += 1024) {
        const int i = r + tid, t = i < hi ? target_of(a.t, i) : -1;
        const unsigned long long in = __ballot(t >= 0);
        if (lane == 0) wave_sum[wave] = __popcll(in);
        __syncthreads();
        int to = base + __popcll(in & ((1ull << lane) - 1ull)), all = 0;
        for (int w = 0; w < 16; ++w) {
            if (w < wave) to += wave_sum[w];
            all += wave_sum[w];
        }
        base += all;
        __syncthreads();
        if (i < hi) a.at[i] = t >= 0 ? to : -1;
        if (t >= 0) {
            a.target_out[to] = t;
            a.weight_out[to] = a.weight[i];
            a.lse_out[to] = a.lse[i];
        }
    }
    if (blockIdx.x == gridDim.x - 1 && wave < 2) {  // whole pieces, the last one
        const int rows = base, i = wave;
        const int2 n = choose_slices(a.rule, a.dx[i].tiles * ((rows + a.edge - 1) / a.edge), a.dx[i].nk, a.dx[i].most, rows * a.dx[i].elements, a.dw[i].tiles,
                                     (rows + a.ks - 1) / a.ks, a.dw[i].most, a.dw[i].elements, a.room, lane);
        if (lane == 0) {
            a.count[i ? SX_LAST : SX] = n.x;
            a.count[i ? SW_LAST : SW] = n.y;
            if (i == 0) a.count[COUNT] = rows;
        }
    }
}

// rows of `cols` elements with any stride -> rows of `padded` elements (whole 16 bytes), zeros behind; row r goes to at[r] (NULL: r;
// negative: nowhere)
template <typename T> __global__ __launch_bounds__(256) void vocab_pad_kernel(const T* __restrict__ in, long long ld, T* __restrict__ out, const int* __restrict__ at, long long rows,
                                                                              int cols, int padded) {
    constexpr int E = Vec16<T>::N;
    const int per = padded / E;
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x, r = i / per;
    if (r >= rows) return;
    const int c = (int)(i - r * per) * E;
    const long long to = at ? at[r] : r;
    if (to < 0) return;
    const T* p = in + r * ld + c;
    Vec16<T> v;
    if (c + E <= cols && ((uintptr_t)p & 15) == 0) {
        v = ld16(p);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v.v[e] = c + e < cols ? p[e] : (T)0.f;
    }
    st16(out + to * padded + c, v);
}

// ---- plan ---------------------------------------------------------------------------------------------------------------------
long long up256(long long b) { return (b + 255) / 256 * 256; }

int edge_tiles(long long n, int edge) { return (int)((n + edge - 1) / edge); }

// the share of the rounds of `slots` workgroups that `tiles` keep busy
double filled(long long tiles, int slots) { return (double)tiles / ((tiles + slots - 1) / slots * slots); }

struct Plan {
    int Hp, e;              // columns of the operands the products read (H rounded up to whole 16 bytes)
    bool pad;               // x and w are copied to that width first
    bool big;               // 256 x 256 tiles
    bool copy_x;            // x is copied: to that width, or (gradient) its counted rows alone
    int edge;               // tile edge
    int parts;              // forward: column parts per row
    int Vc, pieces, ld;     // gradient: words per piece, row stride of d
    int sx, sw;             // at most so many slices of k of dx (per piece) and dw
    long long room;         // elements for the partial sums of a piece: dx from the front, dw from the end
    long long xpad, wpad, part, zt, d, sums, db, rows, bytes;
};


// The most ranges k may be cut into: every one keeps four steps of k.  How many are used is decided when the rows are known.
int most_slices(long long K, int ks) {
    const long long s = (K + ks - 1) / ks / 4;
    return (int)(s < 1 ? 1 : s > MAX_SLICES ? MAX_SLICES : s);
}

// Rows kernel: the gathered targets, lse, weights, places and the count
long long rows_bytes(long long N) { return up256(N * 4) * 4 + 256; }  // (the decisions take five words of the last 256 bytes)

Plan make_plan(const mic_vocab_loss_desc* d, bool grad) {
    Plan p = {};
    if (d->N == 0) return p;
    const long long N = d->N, H = d->H, V = d->V, es = (long long)mic_dtype_size(d->dtype);
    p.e = 16 / (int)es;
    p.Hp = (int)((H + p.e - 1) / p.e * p.e);
    p.pad = p.Hp != H || d->ld_x % p.e || d->ld_w % p.e || (((uintptr_t)d->x | (uintptr_t)d->w) & 15);
    // The large tiles from 128 rows and as many logits as 96 full tiles on.  Forward + gradient on large and on small ones, all rows counted:
    //   2,400 rows x 3500   H = 64: 18+50 18+42   128: 18+51 25+54   512: 22+74 36+84   1024: 32+102 52+132   2048: 50+158 82+219
    //   1,800 rows x 3500           17+51 18+38        17+52 18+45        22+70 24+73         31+94  37+116         49+130 61+196
    //   1,200 rows x 3500           17+46 18+35        17+49 18+41        22+66 22+60         31+86  30+88          49+114 52+147
    //   512 rows x 16000            19+51 17+39        18+52 19+47        23+74 27+92         33+113 43+142         53+169 72+243
    // and 100 rows x 70000 with H = 1024 273 and 217 in all.  So the border fits H of some hundred columns; with H <= 128 the small tiles'
    // gradient would be better up to about 250 tiles, from H = 1024 on the large ones are from 64.  They address 256 rows (64 of k) with 31 bits.
    p.big = d->dtype == MIC_BF16 && N >= 128 && N * V >= 96ll << 16 && H >= 64 && H < (1 << 21) && d->ld_x < (1 << 21) && d->ld_w < (1 << 21);
    // 64 x 64 tiles where 128 x 128 ones would leave compute units idle, half of each tile (H = 64: 20,000 x 3500 forward and gradient 533
    // us, on the larger 746), and in fp32 also the last round of them: a small tile costs 8 % more there (4096 x 512 x 16384: 2663 and
    // 2443 us), 1111 x 300 x 10007 is 1.4 rounds of large tiles and 2.8 of small ones (266 and 302 us)
    const long long large = (long long)edge_tiles(N, 128) * edge_tiles(V, 128), small = (long long)edge_tiles(N, 64) * edge_tiles(V, 64);
    // (from 2^24 of the small ones on the larger alone: a tile is a workgroup of 256 threads, and a launch has fewer than 2^32)
    const bool fine = small < 1 << 24 && (large < 512 || H <= 64 || N <= 64 || (d->dtype == MIC_F32 && 1.08 * filled(large, 512) < filled(small, 1024)));
    p.edge = p.big ? 256 : fine ? 64 : 128;
    p.copy_x = p.pad || grad;
    long long o = 0;
    p.xpad = o;
    if (p.copy_x) o += up256(N * p.Hp * es);
    p.wpad = o;
    if (p.pad) o += up256(V * p.Hp * es);
    if (!grad) {
        p.parts = p.big ? (int)((V + 63) / 64) : edge_tiles(V, p.edge) * 2;
        p.part = o; o += up256(N * p.parts * 8);
        p.zt = o; o += up256(N * 4);
    } else {
        // a piece of d takes at most 256 MiB (what the last-level cache holds), but with many rows it is that wide that d and the
        // partial sums of dx, N * H * 4 bytes per piece, take the same space: es * Vc = 4 H V / Vc (and 31 bits address 256 of its rows)
        long long vc = (256ll << 20) / (es * N), even = (long long)sqrt(4.0 * H * V / es);
        if (even > 1 << 20) even = 1 << 20;
        vc = (vc > even ? vc : even) / p.edge * p.edge;
        if (vc < p.edge) vc = p.edge;
        if (vc > V) vc = V;
        p.pieces = (int)((V + vc - 1) / vc);
        p.Vc = (int)(((V + p.pieces - 1) / p.pieces + p.edge - 1) / p.edge * p.edge);
        if (p.Vc > V) p.Vc = (int)V;
        p.pieces = (int)((V + p.Vc - 1) / p.Vc);
        p.ld = (p.Vc + p.e - 1) / p.e * p.e;
        const int ks = 128 / (int)es;
        p.sx = most_slices(p.Vc, ks);
        p.sw = most_slices(N, ks);
        // never more partial tiles than would fill the GPU twice
        const long long wide = p.big ? 512 : p.edge == 128 ? 1024 : 2048, tx = (long long)edge_tiles(N, p.edge) * edge_tiles(H, p.edge), tw = (long long)edge_tiles(p.Vc, p.edge) * edge_tiles(H, p.edge);
        while (p.sx > 1 && p.sx * tx > 2 * wide) --p.sx;
        while (p.sw > 1 && p.sw * tw > wide) --p.sw;
        p.rows = o; o += rows_bytes(N);
        p.d = o; o += up256(N * p.ld * es);
        // One copy of dx (its pieces are added at the end) and the partial tiles of one round of workgroups, if that many can be: the rule that
        // chooses the slices keeps to it, and the copies of dx have the counted rows alone.  7424 x 512 x 3500 in bf16, half counted: the rule
        // without a limit chooses 4 and 4 slices, 56 MB of the 82.
        const long long round = (p.big ? 256ll : p.edge == 128 ? 512 : 1024) * p.edge * p.edge, most = (p.sx * N + (p.sw > 1 ? p.sw * (long long)p.Vc : 0)) * H;
        p.room = ((N * H + round < most ? N * H + round : most) + 63) / 64 * 64;
        p.sums = o; o += p.pieces * p.room * 4;
        p.db = o;
        if (d->db) o += up256((long long)edge_tiles(N, p.edge) * 2 * p.Vc * 4);
    }
    p.bytes = o;
    return p;
}

int check_desc(const char* who, const mic_vocab_loss_desc* d) {
    MIC_ARG_CHECK(d, "%s: null descriptor", who);
    MIC_ARG_CHECK(d->dtype == MIC_F32 || d->dtype == MIC_BF16, "%s: bad dtype %d", who, d->dtype);
    MIC_ARG_CHECK(d->N >= 0 && d->H > 0 && d->V > 0, "%s: bad sizes N=%d H=%d V=%d", who, d->N, d->H, d->V);
    // tile numbers have 32 bits: at most 2^37 logits (2^23 tiles of 128 x 128), 2^33 elements of x or w
    const long long N = d->N / 64 + 2ll, H = d->H / 64 + 2ll, V = d->V / 64 + 2ll;
    MIC_ARG_CHECK(N <= 1 << 19 && H <= 1 << 21 && V <= 1 << 21 && N * V < 1 << 25 && N * H < 1 << 21 && V * H < 1 << 21, "%s: sizes out of range N=%d H=%d V=%d", who, d->N,
                  d->H, d->V);
    MIC_ARG_CHECK(d->target_bits == 32 || d->target_bits == 64, "%s: targets of %d bits", who, d->target_bits);
    MIC_ARG_CHECK(d->n_ignore >= 0 && d->n_ignore <= MAX_IGNORE, "%s: %d ignored words (at most %d)", who, d->n_ignore, MAX_IGNORE);
    MIC_ARG_CHECK(d->ld_x >= d->H && d->ld_w >= d->H, "%s: row stride below H=%d", who, d->H);
    return 0;
}

Targets targets_of(const mic_vocab_loss_desc* d) {
    Targets t = {};
    t.t = d->targets; t.wide = d->target_bits == 64; t.n_ignore = d->n_ignore; t.V = d->V;
    for (int i = 0; i < d->n_ignore; ++i) t.ignore[i] = d->ignore[i];
    return t;
}

struct Rows {
    const int* count;   // NULL: all
    int are_k;
    const int* slices;  // NULL: one
    int most;           // slices the grid is laid out for
};
int grid_tiles(const GemmShape& g, int most) { return g.tiles_p * g.tiles_q * most; }
template <typename T, int S> GemmShape shape_of(const Operand& p, const Operand& q, const Rows& r, int K) {
    return {p, q, r.count, r.slices, r.are_k, K, edge_tiles(p.n, 64 * S), edge_tiles(q.n, 64 * S)};
}
Gemm8Shape shape8_of(const Operand& p, const Operand& q, const Rows& r, int K) {
    return {{p.p, p.ld, p.n}, {q.p, q.ld, q.n}, r.count, r.slices, r.are_k, K, edge_tiles(p.n, 256), edge_tiles(q.n, 256)};
}
// bf16 on the tiles of the plan, fp32 on the small ones
template <typename T, typename Epi, typename Epi8> int product(const Plan& pl, const Operand& p, const Operand& q, const Rows& r, int K, const typename Epi::Args& ea, hipStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (pl.big) {
            const Gemm8Shape g = shape8_of(p, q, r, K);
            const long long all = (long long)g.tiles_p * g.tiles_q;
            MIC_LAUNCH((vocab_gemm8_kernel<Epi8>), dim3((unsigned)(all < 256 ? all : 256)), dim3(512), 0, s, g, ea);  // one to a compute unit
            return 0;
        }
    if (pl.edge == 64) {
        const GemmShape g = shape_of<T, 1>(p, q, r, K);
        MIC_LAUNCH((vocab_gemm_kernel<T, 1, Epi>), dim3((unsigned)grid_tiles(g, 1)), dim3(256), 0, s, g, ea);
    } else {
        const GemmShape g = shape_of<T, 2>(p, q, r, K);
        MIC_LAUNCH((vocab_gemm_kernel<T, 2, Epi>), dim3((unsigned)grid_tiles(g, 1)), dim3(256), 0, s, g, ea);
    }
    return 0;
}
struct OutProduct {
    Operand p, q;
    Rows r;
    int K;
};
template <typename T, int S> int pair_of(const OutProduct& x, const typename OutEpi<T>::Args& xa, const OutProduct& w, const typename OutEpi<T>::Args& wa, hipStream_t s) {
    const GemmShape gx = shape_of<T, S>(x.p, x.q, x.r, x.K), gw = shape_of<T, S>(w.p, w.q, w.r, w.K);
    const int first = (grid_tiles(gx, x.r.most) + 7) / 8 * 8;
    MIC_LAUNCH((vocab_gemm_pair_kernel<T, S, OutEpi<T>>), dim3((unsigned)(first + grid_tiles(gw, w.r.most))), dim3(256), 0, s, gx, xa, gw, wa, first);
    return 0;
}
// dx and dw of a piece in one launch: 7424 x 512 x 3500 in bf16 is 30 and 28 tiles, which filled the GPU only in 5 ranges of k each; together
// they take 41 us where two launches took 58, and leave fewer partial sums (the last launch 12 instead of 16 us)
template <typename T> int products(const Plan& pl, const OutProduct& x, const typename OutEpi<T>::Args& xa, const OutProduct& w, const typename OutEpi<T>::Args& wa, hipStream_t s) {
    if constexpr (sizeof(T) == 2)
        if (pl.big) {
            MIC_LAUNCH((vocab_gemm8_pair_kernel<OutEpi8>), dim3(256), dim3(512), 0, s, shape8_of(x.p, x.q, x.r, x.K), xa, shape8_of(w.p, w.q, w.r, w.K), wa);
            return 0;
        }
    return pl.edge == 64 ? pair_of<T, 1>(x, xa, w, wa, s) : pair_of<T, 2>(x, xa, w, wa, s);
}

template <typename T> int copy_rows(const void* in, long long ld, void* out, const int* at, long long rows, int cols, int padded, hipStream_t s) {
    const long long n = rows * (padded / Vec16<T>::N);
    MIC_LAUNCH((vocab_pad_kernel<T>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, (const T*)in, ld, (T*)out, at, rows, cols, padded);
    return 0;
}
// x and w as the products read them: in place, or copied to whole 16-byte rows (x: and gathered)
template <typename T> int operands(const mic_vocab_loss_desc* d, const Plan& p, char* ws, const int* at, Operand& x, Operand& w, hipStream_t s) {
    x = {d->x, d->ld_x, d->N};
    w = {d->w, d->ld_w, d->V};
    if (p.copy_x) {
        MIC_TRY(copy_rows<T>(d->x, d->ld_x, ws + p.xpad, at, d->N, d->H, p.Hp, s));
        x = {ws + p.xpad, p.Hp, d->N};
    }
    if (p.pad) {
        MIC_TRY(copy_rows<T>(d->w, d->ld_w, ws + p.wpad, nullptr, d->V, d->H, p.Hp, s));
        w = {ws + p.wpad, p.Hp, d->V};
    }
    return 0;
}

template <typename T> int forward(const mic_vocab_loss_desc* d, const Plan& p, hipStream_t s) {
    char* ws = (char*)d->workspace;
    Operand x, w;
    MIC_TRY(operands<T>(d, p, ws, nullptr, x, w, s));
    StatsEpi::Args ea = {};
    ea.bias = d->bias; ea.t = targets_of(d);
    ea.part = (float2*)(ws + p.part); ea.zt = (float*)(ws + p.zt);
    ea.N = d->N; ea.V = d->V; ea.parts = p.parts;
    MIC_TRY((product<T, StatsEpi, StatsEpi8>(p, w, x, Rows{}, d->H, ea, s)));
    MIC_LAUNCH(vocab_loss_rows_kernel, dim3((d->N + 15) / 16), dim3(1024), 0, s, (const float2*)ea.part, (const float*)ea.zt, ea.t, d->loss, d->lse, d->N, p.parts);
    return 0;
}

template <typename T> int gradient(const mic_vocab_loss_desc* d, const Plan& p, hipStream_t s) {
    char* ws = (char*)d->workspace;
    const long long N = d->N, H = d->H, step = up256(N * 4);
    RowsArgs ra = {};
    ra.t = targets_of(d);
    ra.weight = d->grad_rows; ra.lse = d->lse;
    ra.target_out = (int*)(ws + p.rows);
    ra.lse_out = (float*)(ws + p.rows + step);
    ra.weight_out = (float*)(ws + p.rows + 2 * step);
    ra.at = (int*)(ws + p.rows + 3 * step);
    ra.count = (int*)(ws + p.rows + 4 * step);
    ra.N = d->N;
    const long long share = (N + 63) / 64;
    ra.per_block = (int)((share + 1023) / 1024 * 1024);
    // measured on 256 x 256 tiles: a step of 64 k is 1.7 us, a workgroup's start and end 4 steps, writing and reading again the partial
    // tiles of all compute units 16; on 128 x 128 tiles (two workgroups to a compute unit) 2 and 7
    ra.rule = p.big ? SplitRule{256.f, 4.f, 16.f} : p.edge == 128 ? SplitRule{512.f, 2.f, 7.f} : SplitRule{1024.f, 3.f, 7.f};
    ra.edge = p.edge;
    ra.ks = 128 / (int)sizeof(T);
    const int last = d->V - (p.pieces - 1) * p.Vc, th = edge_tiles(H, p.edge);
    ra.dx[0] = {th, (p.Vc + ra.ks - 1) / ra.ks, p.sx, H};
    ra.dx[1] = {th, (last + ra.ks - 1) / ra.ks, p.sx, H};
    ra.dw[0] = {th * edge_tiles(p.Vc, p.edge), 0, p.sw, p.Vc * H};
    ra.dw[1] = {th * edge_tiles(last, p.edge), 0, p.sw, last * H};
    ra.room = p.room;
    MIC_LAUNCH(vocab_rows_kernel, dim3((unsigned)((N + ra.per_block - 1) / ra.per_block)), dim3(1024), 0, s, ra);
    const int *at = ra.at, *count = ra.count;
    Operand x, w;
    MIC_TRY(operands<T>(d, p, ws, at, x, w, s));
    T* dl = (T*)(ws + p.d);
    float *sums = (float*)(ws + p.sums), *part_db = (float*)(ws + p.db);
    auto parts_of = [&](const float* part, T* out, const int* where, int rows, long long stride, int pieces, int whole, int end) {
        const long long quads = (long long)rows * ((H + 3) / 4);
        return SumParts{part, out, where, ra.count + whole, ra.count + end, count, stride, p.room, rows, d->H, pieces, (unsigned)((quads + 255) / 256)};
    };
    auto finish = [&](const SumParts& x1, const SumParts& x2, const ColSum& c) -> int {
        const unsigned blocks = x1.blocks + x2.blocks + c.blocks;
        if (blocks) MIC_LAUNCH((vocab_finish_kernel<T>), dim3(blocks), dim3(256), 0, s, x1, x2, c);
        return 0;
    };
    for (int i = 0; i < p.pieces; ++i) {
        const bool end = i == p.pieces - 1;
        const int v0 = i * p.Vc, vc = end ? last : p.Vc;
        const Operand wi = {(const T*)w.p + v0 * w.ld, w.ld, vc};
        typename GradEpi<T>::Args ga = {};
        ga.bias = d->bias; ga.r = {ra.target_out, ra.lse_out, ra.weight_out};
        ga.d = dl; ga.part_db = d->db ? part_db : nullptr;
        ga.Vc = vc; ga.ld = p.ld; ga.v0 = v0;
        ga.count = count;
        MIC_TRY((product<T, GradEpi<T>, GradEpi8>(p, wi, x, Rows{count, 0, nullptr, 1}, d->H, ga, s)));
        // dx += d w: k runs over the words of the piece
        typename OutEpi<T>::Args xa = {};
        xa.Np = d->H; xa.Nq = d->N;
        xa.part = sums + i * p.room; xa.count = count;  // rows of the gathered order
        const Operand wc = {wi.p, wi.ld, d->H}, dr = {dl, p.ld, d->N};
        const Rows rx = {count, 0, ra.count + (end ? SX_LAST : SX), p.sx};
        // dw = d^T x: k runs over the rows
        typename OutEpi<T>::Args wa = {};
        wa.out = (T*)d->dw + v0 * H; wa.Np = d->H; wa.Nq = vc;
        if (p.sw > 1) wa.part = sums + (i + 1) * p.room - vc * H;
        const Operand xc = {x.p, x.ld, d->H}, dc = {dl, p.ld, vc};
        const Rows rw = {count, 1, ra.count + (end ? SW_LAST : SW), p.sw};
        wa.count = rw.slices;
        MIC_TRY((products<T>(p, {wc, dr, rx, vc}, xa, {xc, dc, rw, d->N}, wa, s)));
        SumParts sw = {}, sx = {};
        ColSum sb = {};
        if (p.sw > 1) sw = parts_of(wa.part, wa.out, nullptr, vc, -(vc * H), 1, SW, end ? SW_LAST : SW);
        if (d->db) sb = {part_db, d->db + v0, count, vc, edge_tiles(N, p.edge) * 2, p.edge / 2, (unsigned)((vc + 15) / 16)};
        if (end) sx = parts_of(sums, (T*)d->dx, at, d->N, 0, p.pieces, SX, SX_LAST);
        MIC_TRY(finish(sx, sw, sb));
    }
    return 0;
}

__global__ __launch_bounds__(256) void vocab_clear_kernel(uint16_t* p, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) p[i] = 0;
}

}  // namespace

extern "C" int64_t mic_vocab_loss_workspace_bytes(const mic_vocab_loss_desc* d, int grad) {
    MIC_TRY(check_desc("mic_vocab_loss_workspace_bytes", d));
    return make_plan(d, grad != 0).bytes;
}

static int check_call(const char* who, const mic_vocab_loss_desc* d, const Plan& p) {
    MIC_ARG_CHECK(d->N == 0 || (d->x && d->w && d->targets && d->lse), "%s: null pointer", who);
    MIC_ARG_CHECK(p.bytes == 0 || (d->workspace && d->workspace_bytes >= p.bytes && ((uintptr_t)d->workspace & 15) == 0), "%s: workspace of %lld bytes, %lld needed", who,
                  (long long)d->workspace_bytes, p.bytes);
    return 0;
}

extern "C" int mic_vocab_loss(const mic_vocab_loss_desc* d, void* stream) {
    const char* who = "mic_vocab_loss";
    MIC_TRY(check_desc(who, d));
    const Plan p = make_plan(d, false);
    MIC_TRY(check_call(who, d, p));
    if (d->N == 0) return 0;
    MIC_ARG_CHECK(d->loss, "%s: null pointer", who);
    return d->dtype == MIC_BF16 ? forward<bf16_t>(d, p, (hipStream_t)stream) : forward<float>(d, p, (hipStream_t)stream);
}

extern "C" int mic_vocab_loss_grad(const mic_vocab_loss_desc* d, void* stream) {
    const char* who = "mic_vocab_loss_grad";
    MIC_TRY(check_desc(who, d));
    const Plan p = make_plan(d, true);
    MIC_TRY(check_call(who, d, p));
    MIC_ARG_CHECK(d->dw && (d->N == 0 || (d->dx && d->grad_rows)), "%s: null pointer", who);
    MIC_ARG_CHECK((((uintptr_t)d->dx | (uintptr_t)d->dw | (uintptr_t)d->db) & 15) == 0, "%s: a gradient is not 16-byte aligned", who);
    hipStream_t s = (hipStream_t)stream;
    if (d->N == 0) {  // no rows: the sums over them are zero
        const long long n = (long long)d->V * d->H * (long long)mic_dtype_size(d->dtype) / 2;
        auto clear = [&](void* p, long long halves) -> int {
            const long long blocks = (halves + 255) / 256;
            MIC_LAUNCH(vocab_clear_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, s, (uint16_t*)p, halves);
            return 0;
        };
        MIC_TRY(clear(d->dw, n));
        if (d->db) MIC_TRY(clear(d->db, 2ll * d->V));
        return 0;
    }
    return d->dtype == MIC_BF16 ? gradient<bf16_t>(d, p, s) : gradient<float>(d, p, s);
}
