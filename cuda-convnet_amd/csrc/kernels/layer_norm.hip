// Layer norm over the features of each case, forward and backward, for (numFeatures, numCases) matrices with the cases contiguous:
//   y[f,n] = gain[f] (x[f,n] - mean[n]) r[n] + bias[f],  r = 1 / sqrt(var + eps)
//   dx = r (h - mean_f(h) - xh mean_f(h xh)),  h = gain g,  xh = (x - mean) r;  dgain[f] = sum_n g xh;  dbias[f] = sum_n g.
// The sums over the features run down a column, so threads lie along the columns (16-byte accesses where numCases allows) and a
// block's row lanes are joined in LDS.  All of it waits for memory, or, where the matrices are small, for its launches.  Variances are joined as (count, mean, sum of squared deviations) -- Chan, Golub, LeVeque
// 1983 -- and never formed as a difference of large sums.  All orders are fixed by the shape: results repeat bit for bit.
#include <algorithm>
#include "common.h"

// Every product is rounded before it is added, as in the formulas written out operation by operation: with two or three features the
// gradient is a difference of nearly equal numbers, and a product left unrounded on one side of it shows.  (All kernels here wait for
// memory: no time is lost.)
#pragma clang fp contract(off)

namespace {

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int T_SPLIT = 256, T_WHOLE = 256;  // threads of a block
constexpr int JOIN = 4, AHEAD = 4;           // split: partial sums a lane joins; rows it has asked for by then
constexpr int CUS = 256;

// VW neighbouring columns of one row; at the right edge of the matrix only `cnt` of them exist.  Rows start at any multiple of four
// bytes: the hardware takes 16-byte accesses at such addresses.
template <int VW>
struct Cols {
    float v[VW];
};
template <int VW>
__device__ __forceinline__ Cols<VW> load_cols(const float* p, int cnt) {
    Cols<VW> r = {};
    if constexpr (VW == 4) {
        if (cnt == 4) {
            const f32x4u t = *reinterpret_cast<const f32x4u*>(p);
#pragma unroll
            for (int j = 0; j < 4; j++) r.v[j] = t[j];
            return r;
        }
    }
#pragma unroll
    for (int j = 0; j < VW; j++)
        if (j < cnt) r.v[j] = p[j];
    return r;
}
template <int VW>
__device__ __forceinline__ void store_cols(float* p, const Cols<VW>& r, int cnt) {
    if constexpr (VW == 4) {
        if (cnt == 4) {
            f32x4u t;
#pragma unroll
            for (int j = 0; j < 4; j++) t[j] = r.v[j];
            *reinterpret_cast<f32x4u*>(p) = t;
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < VW; j++)
        if (j < cnt) p[j] = r.v[j];
}

__device__ __forceinline__ void join(float& n, float& mean, float& m2, float n2, float mean2, float m22) {
    const float t = n + n2;
    if (t > 0.f) {
        const float d = mean2 - mean, w = n2 / t;
        mean += d * w;
        m2 += m22 + d * d * n * w;
    }
    n = t;
}

// Where a thread of a T-thread block stands: columns col .. col + cnt - 1, rows rl, rl + rowLanes, ...
template <int VW, int T>
struct Place {
    int cl, rl, rowLanes, col, cnt;
    __device__ __forceinline__ Place(int tile, int logLanes, int N) {
        const int lanes = 1 << logLanes;
        cl = threadIdx.x & (lanes - 1);
        rl = threadIdx.x >> logLanes;
        rowLanes = T >> logLanes;
        col = (tile * lanes + cl) * VW;
        cnt = max(0, min(VW, N - col));
    }
};
// Sums of NV values a thread over the row lanes of its columns; every thread gets them.  Lanes of a wave, then the waves, in a fixed order.
template <int NV, int T>
__device__ __forceinline__ void sum_rows(float (&v)[NV], int cl, int logLanes, float (*sh)[64][NV]) {
    for (int o = 1 << logLanes; o < 64; o <<= 1)
#pragma unroll
        for (int k = 0; k < NV; k++) v[k] += __shfl_xor(v[k], o, 64);
    if constexpr (T > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((int)(threadIdx.x & 63) < (1 << logLanes))
#pragma unroll
            for (int k = 0; k < NV; k++) sh[wave][cl][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; k++) v[k] = 0.f;
#pragma unroll
        for (int w = 0; w < T / 64; w++)
#pragma unroll
            for (int k = 0; k < NV; k++) v[k] += sh[w][cl][k];
    }
}

// ---- forward, a block holds all rows of its columns in registers (R a thread): one read, the variance from exact deviations.
// 512 x 1: 2.8 us, 512 x 128: 5.3 us, 1024 x 16384: 22.9 us (134 MB in all, the input from the last-level cache).
template <int VW, int R>
__global__ __launch_bounds__(T_WHOLE) void k_ln_whole(const float* x, const float* __restrict__ gain, const float* __restrict__ bias, float* y,
                                                      float* __restrict__ caseStats, float eps, int F, int N, int logLanes, int tiles) {
    constexpr int T = T_WHOLE;
    __shared__ float sh[T / 64][64][VW];
    int grp, sub;
    mcn_xcd_group(blockIdx.x, 8, gridDim.x / 8, grp, sub);  // eight neighbouring tiles on one XCD: they share cache lines (the grid is a multiple of eight)
    const int tile = grp * 8 + sub;
    if (tile >= tiles) return;
    const Place<VW, T> p(tile, logLanes, N);
    Cols<VW> v[R];
    const size_t first = (size_t)p.rl * N + p.col, step = (size_t)p.rowLanes * N;
    const float* xp = x + first;
#pragma unroll
    for (int i = 0; i < R; i++, xp += step) v[i] = p.rl + i * p.rowLanes < F ? load_cols<VW>(xp, p.cnt) : Cols<VW>{};
    float mean[VW] = {}, m2[VW] = {};
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < VW; j++) mean[j] += v[i].v[j];
    sum_rows<VW, T>(mean, p.cl, logLanes, sh);
#pragma unroll
    for (int j = 0; j < VW; j++) mean[j] /= (float)F;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const bool in = p.rl + i * p.rowLanes < F;
#pragma unroll
        for (int j = 0; j < VW; j++) {
            v[i].v[j] -= mean[j];
            m2[j] += in ? v[i].v[j] * v[i].v[j] : 0.f;
        }
    }
    sum_rows<VW, T>(m2, p.cl, logLanes, sh);
    Cols<VW> mu, rs;
#pragma unroll
    for (int j = 0; j < VW; j++) {
        mu.v[j] = mean[j];
        rs.v[j] = 1.f / sqrtf(m2[j] / (float)F + eps);
    }
    if (caseStats && p.rl == 0) {
        store_cols<VW>(caseStats + p.col, mu, p.cnt);
        store_cols<VW>(caseStats + N + p.col, rs, p.cnt);
    }
    float* yp = y + first;
#pragma unroll
    for (int i = 0; i < R; i++, yp += step) {
        const int r = p.rl + i * p.rowLanes;
        if (r >= F) break;
        const float g = gain ? gain[r] : 1.f, b = bias ? bias[r] : 0.f;
#pragma unroll
        for (int j = 0; j < VW; j++) v[i].v[j] = g * (v[i].v[j] * rs.v[j]) + b;
        store_cols<VW>(yp, v[i], p.cnt);
    }
}

// ---- gains' and biases' gradients of a small matrix, by blocks of their own in the same launch: groups of 1 << logLanes lanes take a
// row each and read it from the caches the other blocks fill.  (Partial sums per tile of columns, and a launch that joins them, for the
// larger ones: reading those twice would cost more.)
struct RowSums {
    float *gainGrad, *biasGrad;
    float gainTargets, gainOutput, biasTargets, biasOutput;
    int first;     // first block of this kind
    int logLanes;
};
__device__ __forceinline__ void row_sums_block(const float* g, const float* x, const float* __restrict__ caseStats, int F, int N, const RowSums& q) {
    const int lanes = 1 << q.logLanes, l = threadIdx.x & (lanes - 1);
    const int r = (blockIdx.x - q.first) * (T_WHOLE >> q.logLanes) + (threadIdx.x >> q.logLanes);
    float sg = 0.f, sb = 0.f;
    if (r < F) {
        const float *gp = g + (size_t)r * N, *xp = x + (size_t)r * N;
#pragma unroll 4
        for (int c = l * 4; c < N; c += lanes * 4) {
            const int cnt = min(4, N - c);
            const Cols<4> gv = load_cols<4>(gp + c, cnt), xv = load_cols<4>(xp + c, cnt), mu = load_cols<4>(caseStats + c, cnt),
                          rs = load_cols<4>(caseStats + N + c, cnt);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                sg += gv.v[j] * ((xv.v[j] - mu.v[j]) * rs.v[j]);
                sb += gv.v[j];
            }
        }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) {
        sg += __shfl_xor(sg, o, 64);
        sb += __shfl_xor(sb, o, 64);
    }
    if (l == 0 && r < F) {
        if (q.gainGrad) q.gainGrad[r] = (q.gainTargets != 0.f ? q.gainTargets * q.gainGrad[r] : 0.f) + q.gainOutput * sg;
        if (q.biasGrad) q.biasGrad[r] = (q.biasTargets != 0.f ? q.biasTargets * q.biasGrad[r] : 0.f) + q.biasOutput * sb;
    }
}

// ---- backward, the same way: both matrices in registers.  A block goes through its tiles one after the other with its rows fixed, so
// the row sums for gains and biases stay in registers too and leave once per block: rowPart[block][2][F].  512 x 128: 4.7 us.
template <int VW, int R>
__global__ __launch_bounds__(T_WHOLE) void k_ln_undo_whole(const float* g, const float* x, const float* __restrict__ gain,
                                                     const float* __restrict__ caseStats, float* target, float* __restrict__ rowPart,
                                                     float scaleTargets, float scaleOutput, int F, int N, int logLanes, int tiles, RowSums q) {
    if ((int)blockIdx.x >= q.first) {
        row_sums_block(g, x, caseStats, F, N, q);
        return;
    }
    constexpr int T = T_WHOLE;
    __shared__ float sh[T / 64][64][2 * VW];
    int grp, sub;
    mcn_xcd_group(blockIdx.x, 8, q.first / 8, grp, sub);  // (the blocks of this kind are a multiple of eight)
    const int block = grp * 8 + sub, rowLanes = T >> logLanes, rl = threadIdx.x >> logLanes;
    float sg[R] = {}, sb[R] = {};
    const float invF = 1.f / (float)F;
    const size_t step = (size_t)rowLanes * N;
    for (int tile = block; tile < tiles; tile += q.first) {
        const Place<VW, T> p(tile, logLanes, N);
        const size_t first = (size_t)rl * N + p.col;
        Cols<VW> gv[R], xv[R];
        const float *gp = g + first, *xp = x + first;
#pragma unroll
        for (int i = 0; i < R; i++, gp += step, xp += step) {
            const bool in = rl + i * rowLanes < F;
            gv[i] = in ? load_cols<VW>(gp, p.cnt) : Cols<VW>{};
            xv[i] = in ? load_cols<VW>(xp, p.cnt) : Cols<VW>{};
        }
        const Cols<VW> mu = load_cols<VW>(caseStats + p.col, p.cnt), rs = load_cols<VW>(caseStats + N + p.col, p.cnt);
        float s[2 * VW] = {};
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int r = rl + i * rowLanes;
            const float ga = gain && r < F ? gain[r] : 1.f;
#pragma unroll
            for (int j = 0; j < VW; j++) {
                const float xh = (xv[i].v[j] - mu.v[j]) * rs.v[j];
                sg[i] += gv[i].v[j] * xh;
                sb[i] += gv[i].v[j];
                const float h = ga * gv[i].v[j];
                s[j] += h;
                s[VW + j] += h * xh;
                xv[i].v[j] = xh;
                gv[i].v[j] = h;
            }
        }
        if (!target) continue;
        sum_rows<2 * VW, T>(s, p.cl, logLanes, sh);
#pragma unroll
        for (int j = 0; j < 2 * VW; j++) s[j] *= invF;
        float* tp = target + first;
#pragma unroll
        for (int i = 0; i < R; i++, tp += step) {
            if (rl + i * rowLanes >= F) break;
            Cols<VW> o;
#pragma unroll
            for (int j = 0; j < VW; j++) o.v[j] = scaleOutput * (rs.v[j] * (gv[i].v[j] - s[j] - xv[i].v[j] * s[VW + j]));
            if (scaleTargets != 0.f) {
                const Cols<VW> t = load_cols<VW>(tp, p.cnt);
#pragma unroll
                for (int j = 0; j < VW; j++) o.v[j] += scaleTargets * t.v[j];
            }
            store_cols<VW>(tp, o, p.cnt);
        }
    }
    if (!rowPart) return;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int r = rl + i * rowLanes;
        for (int o = (1 << logLanes) >> 1; o > 0; o >>= 1) {
            sg[i] += __shfl_xor(sg[i], o, 64);
            sb[i] += __shfl_xor(sb[i], o, 64);
        }
        if ((threadIdx.x & ((1 << logLanes) - 1)) == 0 && r < F) {
            float* out = rowPart + (size_t)block * 2 * F + r;
            out[0] = sg[i];
            out[F] = sb[i];
        }
    }
}

// ---- more rows than a block's registers hold: ranges of rows, joined by a second launch that reads the matrices again.
// 4096 x 16384 (268 MB a matrix): sums 67 us (4.0 TB/s), apply 89 us (6.0 TB/s, part of it from the last-level cache); backward 137 us (3.9
// TB/s) and 146 us (5.5 TB/s).  A copy reaches 5.2 TB/s.  4213 x 509: 4.7 + 8.2 and 7.4 + 8.5 us; the apply launches' 512 blocks each read the
// partial sums of all 64 ranges, 16.8 MB a launch, as much as the matrix there.
struct Split {
    int F, N, logLanes, colTiles, splits, rowsPerSplit;
};

template <int VW>
__global__ __launch_bounds__(T_SPLIT) void k_ln_split_stats(const float* __restrict__ x, float* __restrict__ part, Split s) {
    constexpr int T = T_SPLIT, R = 8;
    __shared__ float sh[T / 64][64][VW];
    const Place<VW, T> p(blockIdx.x, s.logLanes, s.N);
    const int r0 = blockIdx.y * s.rowsPerSplit, r1 = min(s.F, r0 + s.rowsPerSplit);
    // a thread: R rows at a time, their mean and deviations exactly, then joined to what it has
    float n = 0.f, mean[VW] = {}, m2[VW] = {};
    for (int c = r0 + p.rl; c < r1; c += R * p.rowLanes) {
        Cols<VW> v[R];
        const int have = min(R, (r1 - c + p.rowLanes - 1) / p.rowLanes);
#pragma unroll
        for (int i = 0; i < R; i++) v[i] = i < have ? load_cols<VW>(x + (size_t)(c + i * p.rowLanes) * s.N + p.col, p.cnt) : Cols<VW>{};
        const float rows = (float)have, inv = 1.f / rows;
        float t = n;
#pragma unroll
        for (int j = 0; j < VW; j++) {
            float a = 0.f, b = 0.f;
#pragma unroll
            for (int i = 0; i < R; i++) a += v[i].v[j];
            a *= inv;
#pragma unroll
            for (int i = 0; i < R; i++) {
                const float d = v[i].v[j] - a;
                b += i < have ? d * d : 0.f;
            }
            t = n;
            join(t, mean[j], m2[j], rows, a, b);
        }
        n = t;
    }
    // then the row lanes: the mean of all, and the deviations about it
    const float invAll = 1.f / (float)(r1 - r0);
    float all[VW];
#pragma unroll
    for (int j = 0; j < VW; j++) all[j] = n * mean[j];
    sum_rows<VW, T>(all, p.cl, s.logLanes, sh);
#pragma unroll
    for (int j = 0; j < VW; j++) {
        all[j] *= invAll;
        const float d = mean[j] - all[j];
        m2[j] += n * d * d;
        mean[j] = all[j];
    }
    sum_rows<VW, T>(m2, p.cl, s.logLanes, sh);
    if (p.rl == 0) {
        Cols<VW> a, b;
#pragma unroll
        for (int j = 0; j < VW; j++) { a.v[j] = mean[j]; b.v[j] = m2[j]; }
        float* out = part + (size_t)blockIdx.y * 2 * s.N + p.col;
        store_cols<VW>(out, a, p.cnt);
        store_cols<VW>(out + s.N, b, p.cnt);
    }
}

// joins the ranges and writes y; the blocks of the first range also leave the case statistics
template <int VW>
__global__ __launch_bounds__(T_SPLIT) void k_ln_split_apply(const float* x, const float* __restrict__ gain, const float* __restrict__ bias,
                                                            float* y, float* __restrict__ caseStats, const float* __restrict__ part, float eps,
                                                            Split s) {
    const Place<VW, T_SPLIT> p(blockIdx.x, s.logLanes, s.N);
    __shared__ float sh[T_SPLIT / 64][64][VW];
    const int r0 = blockIdx.y * s.rowsPerSplit, r1 = min(s.F, r0 + s.rowsPerSplit);
    // everything this thread will need first, before the sums make it wait: one trip to memory instead of three
    Cols<VW> a[JOIN], b[JOIN], v[AHEAD];
#pragma unroll
    for (int i = 0; i < JOIN; i++) {
        const int k = p.rl + i * p.rowLanes;
        a[i] = k < s.splits ? load_cols<VW>(part + (size_t)k * 2 * s.N + p.col, p.cnt) : Cols<VW>{};
        b[i] = k < s.splits ? load_cols<VW>(part + ((size_t)k * 2 + 1) * s.N + p.col, p.cnt) : Cols<VW>{};
    }
#pragma unroll
    for (int i = 0; i < AHEAD; i++) {
        const int r = r0 + p.rl + i * p.rowLanes;
        v[i] = r < r1 ? load_cols<VW>(x + (size_t)r * s.N + p.col, p.cnt) : Cols<VW>{};
    }
    auto rowsOf = [&](int i) {
        const int k = p.rl + i * p.rowLanes;
        return k < s.splits ? (float)(min(s.F, (k + 1) * s.rowsPerSplit) - k * s.rowsPerSplit) : 0.f;
    };
    float mean[VW] = {}, m2[VW] = {};
#pragma unroll
    for (int i = 0; i < JOIN; i++)
#pragma unroll
        for (int j = 0; j < VW; j++) mean[j] += rowsOf(i) * a[i].v[j];
    sum_rows<VW, T_SPLIT>(mean, p.cl, s.logLanes, sh);
#pragma unroll
    for (int j = 0; j < VW; j++) mean[j] /= (float)s.F;
#pragma unroll
    for (int i = 0; i < JOIN; i++)
#pragma unroll
        for (int j = 0; j < VW; j++) {
            const float d = a[i].v[j] - mean[j];
            m2[j] += b[i].v[j] + rowsOf(i) * d * d;
        }
    sum_rows<VW, T_SPLIT>(m2, p.cl, s.logLanes, sh);
    Cols<VW> mu, rs;
#pragma unroll
    for (int j = 0; j < VW; j++) {
        mu.v[j] = mean[j];
        rs.v[j] = 1.f / sqrtf(m2[j] / (float)s.F + eps);
    }
    if (caseStats && blockIdx.y == 0 && p.rl == 0) {
        store_cols<VW>(caseStats + p.col, mu, p.cnt);
        store_cols<VW>(caseStats + s.N + p.col, rs, p.cnt);
    }
    for (int c = r0 + p.rl; c < r1; c += AHEAD * p.rowLanes) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int r = c + i * p.rowLanes;
            if (r >= r1) break;
            const float g = gain ? gain[r] : 1.f, t = bias ? bias[r] : 0.f;
#pragma unroll
            for (int j = 0; j < VW; j++) v[i].v[j] = g * ((v[i].v[j] - mu.v[j]) * rs.v[j]) + t;
            store_cols<VW>(y + (size_t)r * s.N + p.col, v[i], p.cnt);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int r = c + (i + AHEAD) * p.rowLanes;
            if (r < r1) v[i] = load_cols<VW>(x + (size_t)r * s.N + p.col, p.cnt);
        }
    }
}

// backward: per range the column sums of h and h xh (colPart[split][2][N]), per tile of columns the row sums of g xh and g
// (rowPart[tile][2][F])
template <int VW>
__global__ __launch_bounds__(T_SPLIT) void k_ln_undo_split_sums(const float* __restrict__ g, const float* __restrict__ x,
                                                                const float* __restrict__ gain, const float* __restrict__ caseStats,
                                                                float* __restrict__ colPart, float* __restrict__ rowPart, Split s, RowSums q) {
    if ((int)blockIdx.x >= q.first) {
        row_sums_block(g, x, caseStats, s.F, s.N, q);
        return;
    }
    __shared__ float sh[T_SPLIT / 64][64][2 * VW];
    const int tile = blockIdx.x % s.colTiles, split = blockIdx.x / s.colTiles;
    const Place<VW, T_SPLIT> p(tile, s.logLanes, s.N);
    const int r0 = split * s.rowsPerSplit, r1 = min(s.F, r0 + s.rowsPerSplit);
    const Cols<VW> mu = load_cols<VW>(caseStats + p.col, p.cnt), rs = load_cols<VW>(caseStats + s.N + p.col, p.cnt);
    float v[2 * VW] = {};
    const int steps = (max(r1 - r0, 0) + p.rowLanes - 1) / p.rowLanes;  // the same for every lane: the shuffles below need whole groups
    for (int i = 0; i < steps; i++) {
        const int r = r0 + p.rl + i * p.rowLanes;
        float sg = 0.f, sb = 0.f;
        if (r < r1) {
            const Cols<VW> gv = load_cols<VW>(g + (size_t)r * s.N + p.col, p.cnt), xv = load_cols<VW>(x + (size_t)r * s.N + p.col, p.cnt);
            const float ga = gain ? gain[r] : 1.f;
#pragma unroll
            for (int j = 0; j < VW; j++) {
                const float xh = (xv.v[j] - mu.v[j]) * rs.v[j], gx = gv.v[j] * xh;
                v[j] += ga * gv.v[j];
                v[VW + j] += ga * gx;
                sg += gx;
                sb += gv.v[j];
            }
        }
        if (rowPart) {
            for (int o = (1 << s.logLanes) >> 1; o > 0; o >>= 1) {
                sg += __shfl_xor(sg, o, 64);
                sb += __shfl_xor(sb, o, 64);
            }
            if (p.cl == 0 && r < r1) {
                float* out = rowPart + (size_t)tile * 2 * s.F + r;
                out[0] = sg;
                out[s.F] = sb;
            }
        }
    }
    sum_rows<2 * VW, T_SPLIT>(v, p.cl, s.logLanes, sh);
    if (p.rl == 0) {
        Cols<VW> a, b;
#pragma unroll
        for (int j = 0; j < VW; j++) { a.v[j] = v[j]; b.v[j] = v[VW + j]; }
        float* out = colPart + (size_t)split * 2 * s.N + p.col;
        store_cols<VW>(out, a, p.cnt);
        store_cols<VW>(out + s.N, b, p.cnt);
    }
}

template <int VW>
__global__ __launch_bounds__(T_SPLIT) void k_ln_undo_split_apply(const float* __restrict__ g, const float* __restrict__ x,
                                                                 const float* __restrict__ gain, const float* __restrict__ caseStats,
                                                                 const float* __restrict__ colPart, float* target, float scaleTargets,
                                                                 float scaleOutput, Split s) {
    const Place<VW, T_SPLIT> p(blockIdx.x, s.logLanes, s.N);
    const Cols<VW> mu = load_cols<VW>(caseStats + p.col, p.cnt), rs = load_cols<VW>(caseStats + s.N + p.col, p.cnt);
    __shared__ float sh[T_SPLIT / 64][64][2 * VW];
    const int r0 = blockIdx.y * s.rowsPerSplit, r1 = min(s.F, r0 + s.rowsPerSplit);
    Cols<VW> gv[AHEAD], xv[AHEAD];  // (as in the forward kernel: asked for ahead of the sums)
    auto ask = [&](int c) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int r = c + i * p.rowLanes;
            if (r < r1) {
                gv[i] = load_cols<VW>(g + (size_t)r * s.N + p.col, p.cnt);
                xv[i] = load_cols<VW>(x + (size_t)r * s.N + p.col, p.cnt);
            }
        }
    };
    float sums[2 * VW] = {};
    {
        Cols<VW> a[JOIN], b[JOIN];
#pragma unroll
        for (int i = 0; i < JOIN; i++) {
            const int k = p.rl + i * p.rowLanes;
            a[i] = k < s.splits ? load_cols<VW>(colPart + (size_t)k * 2 * s.N + p.col, p.cnt) : Cols<VW>{};
            b[i] = k < s.splits ? load_cols<VW>(colPart + ((size_t)k * 2 + 1) * s.N + p.col, p.cnt) : Cols<VW>{};
        }
        ask(r0 + p.rl);
#pragma unroll
        for (int i = 0; i < JOIN; i++)
#pragma unroll
            for (int j = 0; j < VW; j++) { sums[j] += a[i].v[j]; sums[VW + j] += b[i].v[j]; }
    }
    sum_rows<2 * VW, T_SPLIT>(sums, p.cl, s.logLanes, sh);
    const float invF = 1.f / (float)s.F;
    float s1[VW], s2[VW];
#pragma unroll
    for (int j = 0; j < VW; j++) { s1[j] = sums[j] * invF; s2[j] = sums[VW + j] * invF; }
    for (int c = r0 + p.rl; c < r1; c += AHEAD * p.rowLanes) {
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int r = c + i * p.rowLanes;
            if (r >= r1) break;
            const float ga = gain ? gain[r] : 1.f;
            Cols<VW> o;
#pragma unroll
            for (int j = 0; j < VW; j++) {
                const float xh = (xv[i].v[j] - mu.v[j]) * rs.v[j];
                o.v[j] = scaleOutput * (rs.v[j] * (ga * gv[i].v[j] - s1[j] - xh * s2[j]));
            }
            float* to = target + (size_t)r * s.N + p.col;
            if (scaleTargets != 0.f) {
                const Cols<VW> t = load_cols<VW>(to, p.cnt);
#pragma unroll
                for (int j = 0; j < VW; j++) o.v[j] += scaleTargets * t.v[j];
            }
            store_cols<VW>(to, o, p.cnt);
        }
        ask(c + AHEAD * p.rowLanes);
    }
}

// ---- gains' and biases' gradients from the partial row sums: 32 of the 2 F sums x 16 lanes over the partials per block
__global__ __launch_bounds__(512) void k_ln_undo_rows(const float* __restrict__ rowPart, float* gainGrad, float* biasGrad, float gainTargets,
                                                      float gainOutput, float biasTargets, float biasOutput, int F, int parts) {
    __shared__ float sh[16][33];
    const int c = threadIdx.x & 31, l = threadIdx.x >> 5, i = blockIdx.x * 32 + c;
    float v = 0.f;
    if (i < 2 * F) {
#pragma unroll 4
        for (int t = l; t < parts; t += 16) v += rowPart[(size_t)t * 2 * F + i];
    }
    sh[l][c] = v;
    __syncthreads();
    if (l != 0 || i >= 2 * F) return;
    for (int k = 1; k < 16; k++) v += sh[k][c];
    const bool isBias = i >= F;
    float* out = isBias ? biasGrad : gainGrad;
    if (!out) return;
    const float sT = isBias ? biasTargets : gainTargets, sO = isBias ? biasOutput : gainOutput;
    const int f = isBias ? i - F : i;
    out[f] = (sT != 0.f ? sT * out[f] : 0.f) + sO * v;
}

// How a shape is laid out.
struct Plan {
    bool whole;
    int vw, logLanes, tiles;  // whole
    int blocks;               // backward, whole
    Split split;
};
constexpr size_t CACHED_BYTES = (size_t)128 << 20;  // a matrix that stays in the last-level cache
// Both matrices of a backward pass, and the cases of a row: up to these the rows are summed by blocks of their own in the same launch, as
// their second read comes from the caches, with at most 16 steps of a wave along a row (forward and backward, so / with partial sums and a
// launch that joins them: 16 x 512 13.7 / 16.5 us, 128 x 4096 14.4 / 16.6, 512 x 4096 19.6 / 18.9, 2 x 8192 20.3 / 16.4, 128 x 8192 22.2 /
// 16.0, 16 x 32768 71 / 27, 16 x 262144 583 / 113, 2 x 2000000 4050 / 770).  Longer rows of one wave would also be one long chain of sums.
constexpr size_t SMALL_BYTES = (size_t)32 << 20;
constexpr int SMALL_CASES = 4096;
constexpr int FWD_ROWS = 16, BWD_ROWS = 8;       // rows a thread of the whole kernels holds
// rows: FWD_ROWS or BWD_ROWS
Plan ln_plan(int F, int N, int rows) {
    Plan p = {};
    p.vw = N >= 4 ? 4 : 1;
    const int lanes = divup(N, p.vw), most = T_WHOLE * rows;
    // whole: four column lanes (64 bytes of a row) are the fastest where there are tiles for every CU and the rows fit, fewer else
    int lg = p.vw == 1 ? (N == 1 ? 0 : N == 2 ? 1 : 2) : 2;
    while (p.vw == 4 && lg > 0 && (divup(lanes, 1 << lg) < CUS || ((size_t)F << lg) > (size_t)most)) lg--;
    p.logLanes = lg;
    p.tiles = divup(lanes, 1 << lg);
    // Two lanes a row (32 bytes) read every cache line from several tiles, which pays while the cache holds the matrix (forward, whole /
    // split: 2048 x 8192, 67 MB, 27 / 37 us; 2048 x 32768, 268 MB, 223 / 164 us), one lane only where it is small.
    p.whole = ((size_t)F << lg) <= (size_t)most && (lg > 1 || (lg == 1 ? (size_t)F * N * 4 <= CACHED_BYTES : p.tiles <= CUS));
    p.blocks = std::min(divup(p.tiles, 8) * 8, 4 * CUS);
    Split& s = p.split;
    s.F = F;
    s.N = N;
    s.logLanes = 0;
    while ((1 << s.logLanes) < lanes && s.logLanes < 4) s.logLanes++;
    // split: 256 bytes of a row (16 lanes), fewer while that leaves CUs without a block (9075 x 128 forward: 11.6 -> 9.7 us; 100000 x 64:
    // 75 -> 28 us), and up to 16 blocks a CU (4096 x 16384, both passes: 4 a CU 457 us, 16 438 us)
    for (;; s.logLanes--) {
        s.colTiles = divup(lanes, 1 << s.logLanes);
        const int rowLanes = T_SPLIT >> s.logLanes;
        s.splits = std::max(1, std::min({JOIN * rowLanes, divup(16 * CUS, s.colTiles), divup(F, 4 * rowLanes)}));
        if (s.logLanes <= 2 || s.colTiles * s.splits >= CUS) break;
    }
    s.rowsPerSplit = divup(F, s.splits);
    s.splits = divup(F, s.rowsPerSplit);
    return p;
}

inline bool al16(const void* p) { return ((uintptr_t)p % 16) == 0; }

bool ln_sizes_ok(int F, int N) { return F > 0 && N > 0 && F <= (1 << 26) && N <= (1 << 26); }  // (every grid: below 2^32 threads)

int ln_require_workspace(const void* ws, size_t have, size_t need, const char* what) {
    if (need > 0 && (!ws || have < need)) {
        mcn_set_error("%s: workspace %zu < %zu bytes", what, ws ? have : (size_t)0, need);
        return MCN_EWORKSPACE;
    }
    MCN_REQUIRE(al16(ws), "%s: the workspace is not 16-byte aligned", what);
    return MCN_OK;
}

}  // namespace

MCN_API size_t mcn_layer_norm_workspace_bytes(int numFeatures, int numCases) {
    if (!ln_sizes_ok(numFeatures, numCases)) return 0;
    const Plan p = ln_plan(numFeatures, numCases, FWD_ROWS);
    return p.whole ? 0 : (size_t)p.split.splits * 2 * numCases * sizeof(float);
}

MCN_API int mcn_layer_norm(const float* inputs, const float* gains, const float* biases, float* target, float* caseStats, int numFeatures,
                           int numCases, float eps, void* workspace, size_t workspaceBytes, void* stream) {
    MCN_REQUIRE(inputs && target && ln_sizes_ok(numFeatures, numCases), "layerNorm: bad argument");
    const size_t n = (size_t)numFeatures * numCases;
    MCN_REQUIRE(target == inputs || !mcn_overlap(target, n, inputs, n), "layerNorm: target overlaps inputs in part");
    const size_t f = numFeatures, stats = (size_t)2 * numCases;
    if (int rc = mcn_refuse_overlaps("layerNorm", {{"target", target, n}}, {{"gains", gains, f}, {"biases", biases, f}})) return rc;
    if (int rc = mcn_refuse_overlaps("layerNorm", {{"caseStats", caseStats, stats}},
                                     {{"target", target, n}, {"inputs", inputs, n}, {"gains", gains, f}, {"biases", biases, f}})) return rc;
    MCN_REQUIRE(eps > 0.f, "layerNorm: eps %g is not positive", (double)eps);
    if (int rc = ln_require_workspace(workspace, workspaceBytes, mcn_layer_norm_workspace_bytes(numFeatures, numCases), "layerNorm")) return rc;
    hipStream_t st = (hipStream_t)stream;
    const int F = numFeatures, N = numCases;
    const Plan p = ln_plan(F, N, FWD_ROWS);
    if (p.whole) {
        const dim3 grid(divup(p.tiles, 8) * 8);
#define WHOLE(VW, R) MCN_LAUNCH((k_ln_whole<VW, R>), grid, dim3(T_WHOLE), 0, st, inputs, gains, biases, target, caseStats, eps, F, N, p.logLanes, p.tiles)
        // (few rows a thread: 160 x 4096 5.3 -> 4.6 us, 512 x 128 5.3 -> 4.8 us)
        const bool few = ((size_t)F << p.logLanes) <= T_WHOLE * 4;
        if (p.vw == 4 && few) WHOLE(4, 4);
        else if (p.vw == 4) WHOLE(4, FWD_ROWS);
        else if (few) WHOLE(1, 4);
        else WHOLE(1, FWD_ROWS);
#undef WHOLE
    } else {
        const Split& s = p.split;
        const dim3 grid(s.colTiles, s.splits);
        float* part = (float*)workspace;
        if (p.vw == 4) {
            MCN_LAUNCH(k_ln_split_stats<4>, grid, dim3(T_SPLIT), 0, st, inputs, part, s);
            MCN_LAUNCH(k_ln_split_apply<4>, grid, dim3(T_SPLIT), 0, st, inputs, gains, biases, target, caseStats, part, eps, s);
        } else {
            MCN_LAUNCH(k_ln_split_stats<1>, grid, dim3(T_SPLIT), 0, st, inputs, part, s);
            MCN_LAUNCH(k_ln_split_apply<1>, grid, dim3(T_SPLIT), 0, st, inputs, gains, biases, target, caseStats, part, eps, s);
        }
    }
    return MCN_LAUNCH_CHECK("layerNorm");
}

MCN_API size_t mcn_layer_norm_undo_workspace_bytes(int numFeatures, int numCases) {
    if (!ln_sizes_ok(numFeatures, numCases)) return 0;
    const Plan p = ln_plan(numFeatures, numCases, BWD_ROWS);
    const size_t parts = p.whole ? p.blocks : p.split.colTiles;  // (of a small matrix the row sums need none: kept simple)
    return (parts * 2 * numFeatures + (p.whole ? 0 : (size_t)p.split.splits * 2 * numCases)) * sizeof(float);
}

MCN_API int mcn_layer_norm_undo(const float* outGrads, const float* inputs, const float* gains, const float* caseStats, float* target,
                                float* gainGrads, float* biasGrads, int numFeatures, int numCases, float scaleTargets, float scaleOutput,
                                float scaleGainTargets, float scaleGainOutput, float scaleBiasTargets, float scaleBiasOutput,
                                void* workspace, size_t workspaceBytes, void* stream) {
    MCN_REQUIRE(outGrads && inputs && caseStats && ln_sizes_ok(numFeatures, numCases), "layerNormUndo: bad argument");
    MCN_REQUIRE(target || gainGrads || biasGrads, "layerNormUndo: nothing to compute");
    const size_t n = (size_t)numFeatures * numCases;
    const size_t f = numFeatures;
    if (int rc = mcn_refuse_overlaps("layerNormUndo", {{"target", target, n}, {"gainGrads", gainGrads, f}, {"biasGrads", biasGrads, f}},
                                     {{"outGrads", outGrads, n}, {"inputs", inputs, n}, {"gains", gains, f}, {"caseStats", caseStats, (size_t)2 * numCases}})) return rc;
    if (int rc = ln_require_workspace(workspace, workspaceBytes, mcn_layer_norm_undo_workspace_bytes(numFeatures, numCases), "layerNormUndo")) return rc;
    hipStream_t st = (hipStream_t)stream;
    const int F = numFeatures, N = numCases;
    const Plan p = ln_plan(F, N, BWD_ROWS);
    const bool rows = gainGrads || biasGrads, small = N <= SMALL_CASES && (size_t)F * N * 8 <= SMALL_BYTES;
    float* rowPart = rows && !small ? (float*)workspace : nullptr;
    const Split& sp = p.split;
    RowSums q = {gainGrads, biasGrads, scaleGainTargets, scaleGainOutput, scaleBiasTargets, scaleBiasOutput, 0, 0};
    while (q.logLanes < 6 && (4 << q.logLanes) < N) q.logLanes++;
    const int rowBlocks = rows && small ? divup(F, T_WHOLE >> q.logLanes) : 0;
    int parts;
    if (p.whole) {
        parts = p.blocks;
        q.first = target || rowPart ? p.blocks : 0;
        const dim3 grid(q.first + rowBlocks);
#define WHOLE(VW, R) MCN_LAUNCH((k_ln_undo_whole<VW, R>), grid, dim3(T_WHOLE), 0, st, outGrads, inputs, gains, caseStats, target, \
                                rowPart, scaleTargets, scaleOutput, F, N, p.logLanes, p.tiles, q)
        if (p.vw == 4) WHOLE(4, BWD_ROWS);
        else WHOLE(1, BWD_ROWS);
#undef WHOLE
    } else {
        parts = sp.colTiles;
        q.first = target || rowPart ? sp.colTiles * sp.splits : 0;
        const dim3 sums(q.first + rowBlocks), grid(sp.colTiles, sp.splits);
        float* colPart = (float*)workspace + (size_t)parts * 2 * F;
        if (p.vw == 4) {
            MCN_LAUNCH(k_ln_undo_split_sums<4>, sums, dim3(T_SPLIT), 0, st, outGrads, inputs, gains, caseStats, colPart, rowPart, sp, q);
            if (target) MCN_LAUNCH(k_ln_undo_split_apply<4>, grid, dim3(T_SPLIT), 0, st, outGrads, inputs, gains, caseStats, colPart, target, scaleTargets, scaleOutput, sp);
        } else {
            MCN_LAUNCH(k_ln_undo_split_sums<1>, sums, dim3(T_SPLIT), 0, st, outGrads, inputs, gains, caseStats, colPart, rowPart, sp, q);
            if (target) MCN_LAUNCH(k_ln_undo_split_apply<1>, grid, dim3(T_SPLIT), 0, st, outGrads, inputs, gains, caseStats, colPart, target, scaleTargets, scaleOutput, sp);
        }
    }
    if (rowPart)
        MCN_LAUNCH(k_ln_undo_rows, dim3((unsigned)divup_sz((size_t)2 * F, 32)), dim3(512), 0, st, rowPart, gainGrads, biasGrads, scaleGainTargets,
                   scaleGainOutput, scaleBiasTargets, scaleBiasOutput, F, parts);
    return MCN_LAUNCH_CHECK("layerNormUndo");
}
