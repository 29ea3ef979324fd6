// Layer norm over the features of each case, forward and backward, for (numFeatures, numCases) matrices with the cases contiguous:
//   y[f,n] = gain[f] (x[f,n] - mean[n]) r[n] + bias[f],  r = 1 / sqrt(var + eps)
//   dx = r (h - mean_f(h) - xh mean_f(h xh)),  h = gain g,  xh = (x - mean) r;  dgain[f] = sum_n g xh;  dbias[f] = sum_n g.
// The sums over the features run down a column, so threads lie along the columns (16-byte accesses where numCases allows) and a
// block's row lanes are joined in LDS.  Variances are joined as (count, mean, sum of squared deviations) -- Chan, Golub, LeVeque
// 1983 -- and never formed as a difference of large sums.  All orders are fixed by the shape: results repeat bit for bit.
#include <algorithm>
#include "common.h"

namespace {

constexpr int T = 256;       // threads of a block
constexpr int MAX_SPLIT = 64;

// Shape of one launch: a block covers colLanes * VW columns and one range of rows; rowLanes = T / colLanes.
struct LnShape {
    int F, N;
    int logColLanes;      // colLanes = 1 << logColLanes
    int colTiles, splits, rowsPerSplit;
};

LnShape ln_shape(int F, int N, int vw) {
    LnShape s;
    s.F = F;
    s.N = N;
    const int lanes = divup(N, vw);
    s.logColLanes = 0;
    while ((1 << s.logColLanes) < lanes && (1 << s.logColLanes) < 64 / vw) s.logColLanes++;
    const int colLanes = 1 << s.logColLanes, rowLanes = T / colLanes;
    s.colTiles = divup(lanes, colLanes);
    // enough blocks for the chip, at least four rows a lane in each
    s.splits = std::max(1, std::min({MAX_SPLIT, divup(1024, s.colTiles), divup(F, 4 * rowLanes)}));
    s.rowsPerSplit = divup(F, s.splits);
    s.splits = divup(F, s.rowsPerSplit);
    return s;
}

template <int VW>
struct Vec {
    float v[VW];
};
template <int VW>
__device__ __forceinline__ Vec<VW> load_cols(const float* __restrict__ p) {
    Vec<VW> r;
    if constexpr (VW == 4) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(p);
        for (int j = 0; j < 4; j++) r.v[j] = t[j];
    } else {
        r.v[0] = *p;
    }
    return r;
}
template <int VW>
__device__ __forceinline__ void store_cols(float* __restrict__ p, const Vec<VW>& r) {
    if constexpr (VW == 4) {
        f32x4 t;
        for (int j = 0; j < 4; j++) t[j] = r.v[j];
        *reinterpret_cast<f32x4*>(p) = t;
    } else {
        *p = r.v[0];
    }
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

// Stage 1: mean and sum of squared deviations of one range of rows, into part[split][2][N].
template <int VW>
__global__ __launch_bounds__(T) void k_ln_stats(const float* __restrict__ x, float* __restrict__ part, LnShape s) {
    __shared__ float sh[2][T][VW];
    const int colLanes = 1 << s.logColLanes, rowLanes = T >> s.logColLanes;
    const int cl = threadIdx.x & (colLanes - 1), rl = threadIdx.x >> s.logColLanes;
    const int col = (blockIdx.x * colLanes + cl) * VW;
    const int r0 = blockIdx.y * s.rowsPerSplit, r1 = min(s.F, r0 + s.rowsPerSplit);
    const bool live = col < s.N;
    float mean[VW] = {}, m2[VW] = {}, cnt = 0.f;
    if (live)
        for (int r = r0 + rl; r < r1; r += rowLanes) {
            const Vec<VW> v = load_cols<VW>(x + (size_t)r * s.N + col);
            const float w = 1.f / (cnt + 1.f);
#pragma unroll
            for (int j = 0; j < VW; j++) {
                const float d = v.v[j] - mean[j];
                mean[j] += d * w;
                m2[j] += d * (v.v[j] - mean[j]);
            }
            cnt += 1.f;
        }
#pragma unroll
    for (int j = 0; j < VW; j++) {
        sh[0][threadIdx.x][j] = mean[j];
        sh[1][threadIdx.x][j] = m2[j];
    }
    __syncthreads();
    const int rows = r1 - r0;
    for (int half = rowLanes >> 1; half > 0; half >>= 1) {
        if (rl < half) {
            const int o = threadIdx.x + (half << s.logColLanes);
            // rows held by row lanes rl, rl + half, ... so far: every lane's share of the range follows from its index
            float na = 0.f, nb = 0.f;
            for (int k = rl; k < rowLanes; k += 2 * half) na += (float)(k < rows ? (rows - k + rowLanes - 1) / rowLanes : 0);
            for (int k = rl + half; k < rowLanes; k += 2 * half) nb += (float)(k < rows ? (rows - k + rowLanes - 1) / rowLanes : 0);
#pragma unroll
            for (int j = 0; j < VW; j++) {
                float n = na, a = sh[0][threadIdx.x][j], b = sh[1][threadIdx.x][j];
                join(n, a, b, nb, sh[0][o][j], sh[1][o][j]);
                sh[0][threadIdx.x][j] = a;
                sh[1][threadIdx.x][j] = b;
            }
        }
        __syncthreads();
    }
    if (rl == 0 && live) {
        Vec<VW> a, b;
        for (int j = 0; j < VW; j++) { a.v[j] = sh[0][threadIdx.x][j]; b.v[j] = sh[1][threadIdx.x][j]; }
        float* p = part + (size_t)blockIdx.y * 2 * s.N + col;
        store_cols<VW>(p, a);
        store_cols<VW>(p + s.N, b);
    }
}

// Stage 2: joins the ranges and writes y; the blocks of the first range also leave the case statistics.
template <int VW>
__global__ __launch_bounds__(T) void k_ln_apply(const float* x, const float* __restrict__ gain, const float* __restrict__ bias, float* y,
                                                float* __restrict__ caseStats, const float* __restrict__ part, float eps, LnShape s) {
    const int colLanes = 1 << s.logColLanes, rowLanes = T >> s.logColLanes;
    const int cl = threadIdx.x & (colLanes - 1), rl = threadIdx.x >> s.logColLanes;
    const int col = (blockIdx.x * colLanes + cl) * VW;
    if (col >= s.N) return;
    float mean[VW] = {}, m2[VW] = {}, cnt = 0.f;
    for (int k = 0; k < s.splits; k++) {
        const float rows = (float)(min(s.F, (k + 1) * s.rowsPerSplit) - k * s.rowsPerSplit);
        const Vec<VW> a = load_cols<VW>(part + (size_t)k * 2 * s.N + col), b = load_cols<VW>(part + ((size_t)k * 2 + 1) * s.N + col);
        float n = 0.f;
#pragma unroll
        for (int j = 0; j < VW; j++) {
            n = cnt;
            join(n, mean[j], m2[j], rows, a.v[j], b.v[j]);
        }
        cnt = n;
    }
    Vec<VW> mu, rs;
#pragma unroll
    for (int j = 0; j < VW; j++) {
        mu.v[j] = mean[j];
        rs.v[j] = 1.f / sqrtf(m2[j] / (float)s.F + eps);
    }
    if (caseStats && blockIdx.y == 0 && rl == 0) {
        store_cols<VW>(caseStats + col, mu);
        store_cols<VW>(caseStats + s.N + col, rs);
    }
    const int r0 = blockIdx.y * s.rowsPerSplit, r1 = min(s.F, r0 + s.rowsPerSplit);
    for (int r = r0 + rl; r < r1; r += rowLanes) {
        Vec<VW> v = load_cols<VW>(x + (size_t)r * s.N + col);
        const float g = gain ? gain[r] : 1.f, b = bias ? bias[r] : 0.f;
#pragma unroll
        for (int j = 0; j < VW; j++) v.v[j] = g * ((v.v[j] - mu.v[j]) * rs.v[j]) + b;
        store_cols<VW>(y + (size_t)r * s.N + col, v);
    }
}

// Backward, stage 1: per range of rows the column sums of h and h xh (colPart[split][2][N]), and per tile of columns the row sums of
// g xh and g (rowPart[tile][2][F]).
template <int VW>
__global__ __launch_bounds__(T) void k_ln_undo_sums(const float* __restrict__ g, const float* __restrict__ x, const float* __restrict__ gain,
                                                    const float* __restrict__ caseStats, float* __restrict__ colPart,
                                                    float* __restrict__ rowPart, LnShape s) {
    __shared__ float sh[2][T][VW];
    const int colLanes = 1 << s.logColLanes, rowLanes = T >> s.logColLanes;
    const int cl = threadIdx.x & (colLanes - 1), rl = threadIdx.x >> s.logColLanes;
    const int col = (blockIdx.x * colLanes + cl) * VW;
    const int r0 = blockIdx.y * s.rowsPerSplit, r1 = min(s.F, r0 + s.rowsPerSplit);
    const bool live = col < s.N;
    Vec<VW> mu = {}, rs = {};
    if (live) {
        mu = load_cols<VW>(caseStats + col);
        rs = load_cols<VW>(caseStats + s.N + col);
    }
    float s1[VW] = {}, s2[VW] = {};
    const int steps = (max(r1 - r0, 0) + rowLanes - 1) / rowLanes;  // the same for every lane: the shuffles below need whole groups
    for (int i = 0; i < steps; i++) {
        const int r = r0 + rl + i * rowLanes;
        float sg = 0.f, sb = 0.f;
        if (live && r < r1) {
            const Vec<VW> gv = load_cols<VW>(g + (size_t)r * s.N + col), xv = load_cols<VW>(x + (size_t)r * s.N + col);
            const float ga = gain ? gain[r] : 1.f;
#pragma unroll
            for (int j = 0; j < VW; j++) {
                const float xh = (xv.v[j] - mu.v[j]) * rs.v[j], gx = gv.v[j] * xh;
                s1[j] += ga * gv.v[j];
                s2[j] += ga * gx;
                sg += gx;
                sb += gv.v[j];
            }
        }
        if (rowPart) {
            for (int o = colLanes >> 1; o > 0; o >>= 1) {
                sg += __shfl_xor(sg, o, 64);
                sb += __shfl_xor(sb, o, 64);
            }
            if (cl == 0 && r < r1) {
                float* p = rowPart + (size_t)blockIdx.x * 2 * s.F + r;
                p[0] = sg;
                p[s.F] = sb;
            }
        }
    }
#pragma unroll
    for (int j = 0; j < VW; j++) {
        sh[0][threadIdx.x][j] = s1[j];
        sh[1][threadIdx.x][j] = s2[j];
    }
    __syncthreads();
    for (int half = rowLanes >> 1; half > 0; half >>= 1) {
        if (rl < half) {
            const int o = threadIdx.x + (half << s.logColLanes);
#pragma unroll
            for (int j = 0; j < VW; j++) {
                sh[0][threadIdx.x][j] += sh[0][o][j];
                sh[1][threadIdx.x][j] += sh[1][o][j];
            }
        }
        __syncthreads();
    }
    if (rl == 0 && live) {
        Vec<VW> a, b;
        for (int j = 0; j < VW; j++) { a.v[j] = sh[0][threadIdx.x][j]; b.v[j] = sh[1][threadIdx.x][j]; }
        float* p = colPart + (size_t)blockIdx.y * 2 * s.N + col;
        store_cols<VW>(p, a);
        store_cols<VW>(p + s.N, b);
    }
}

// Backward, stage 2: dx.
template <int VW>
__global__ __launch_bounds__(T) void k_ln_undo_apply(const float* __restrict__ g, const float* __restrict__ x, const float* __restrict__ gain,
                                                     const float* __restrict__ caseStats, const float* __restrict__ colPart, float* target,
                                                     float scaleTargets, float scaleOutput, LnShape s) {
    const int colLanes = 1 << s.logColLanes, rowLanes = T >> s.logColLanes;
    const int cl = threadIdx.x & (colLanes - 1), rl = threadIdx.x >> s.logColLanes;
    const int col = (blockIdx.x * colLanes + cl) * VW;
    if (col >= s.N) return;
    const Vec<VW> mu = load_cols<VW>(caseStats + col), rs = load_cols<VW>(caseStats + s.N + col);
    float s1[VW] = {}, s2[VW] = {};
    for (int k = 0; k < s.splits; k++) {
        const Vec<VW> a = load_cols<VW>(colPart + (size_t)k * 2 * s.N + col), b = load_cols<VW>(colPart + ((size_t)k * 2 + 1) * s.N + col);
#pragma unroll
        for (int j = 0; j < VW; j++) { s1[j] += a.v[j]; s2[j] += b.v[j]; }
    }
    const float invF = 1.f / (float)s.F;
#pragma unroll
    for (int j = 0; j < VW; j++) { s1[j] *= invF; s2[j] *= invF; }
    const int r0 = blockIdx.y * s.rowsPerSplit, r1 = min(s.F, r0 + s.rowsPerSplit);
    for (int r = r0 + rl; r < r1; r += rowLanes) {
        const size_t at = (size_t)r * s.N + col;
        const Vec<VW> gv = load_cols<VW>(g + at), xv = load_cols<VW>(x + at);
        const float ga = gain ? gain[r] : 1.f;
        Vec<VW> o;
#pragma unroll
        for (int j = 0; j < VW; j++) {
            const float xh = (xv.v[j] - mu.v[j]) * rs.v[j];
            o.v[j] = scaleOutput * (rs.v[j] * (ga * gv.v[j] - s1[j] - xh * s2[j]));
        }
        if (scaleTargets != 0.f) {
            const Vec<VW> t = load_cols<VW>(target + at);
#pragma unroll
            for (int j = 0; j < VW; j++) o.v[j] += scaleTargets * t.v[j];
        }
        store_cols<VW>(target + at, o);
    }
}

// Backward, stage 3: the gains' and biases' gradients from the tiles' row sums.
__global__ __launch_bounds__(T) void k_ln_undo_rows(const float* __restrict__ rowPart, float* gainGrad, float* biasGrad, float gainTargets,
                                                    float gainOutput, float biasTargets, float biasOutput, int F, int tiles) {
    const int i = blockIdx.x * T + threadIdx.x;
    if (i >= 2 * F) return;
    const bool isBias = i >= F;
    float* out = isBias ? biasGrad : gainGrad;
    if (!out) return;
    float v = 0.f;
    for (int t = 0; t < tiles; t++) v += rowPart[(size_t)t * 2 * F + i];
    const float sT = isBias ? biasTargets : gainTargets, sO = isBias ? biasOutput : gainOutput;
    const int f = isBias ? i - F : i;
    out[f] = (sT != 0.f ? sT * out[f] : 0.f) + sO * v;
}

inline bool al16(const void* p) { return ((uintptr_t)p % 16) == 0; }

bool ln_sizes_ok(int F, int N) { return F > 0 && N > 0 && F <= (1 << 28) && N <= (1 << 28); }

int ln_require_workspace(const void* ws, size_t have, size_t need, const char* what) {
    if (need > 0 && (!ws || have < need)) {
        mcn_set_error("%s: workspace %zu < %zu bytes", what, ws ? have : (size_t)0, need);
        return MCN_EWORKSPACE;
    }
    MCN_REQUIRE(al16(ws), "%s: the workspace is not 16-byte aligned", what);
    return MCN_OK;
}

size_t al4(size_t n) { return (n + 3) / 4 * 4; }

}  // namespace

// The workspace does not depend on the pointers' alignment: the larger of the two forms.
MCN_API size_t mcn_layer_norm_workspace_bytes(int numFeatures, int numCases) {
    if (!ln_sizes_ok(numFeatures, numCases)) return 0;
    size_t b = 0;
    for (int vw = 1; vw <= 4; vw += 3) b = std::max(b, (size_t)ln_shape(numFeatures, numCases, vw).splits * 2 * numCases * sizeof(float));
    return b;
}

MCN_API int mcn_layer_norm(const float* inputs, const float* gains, const float* biases, float* target, float* caseStats, int numFeatures,
                           int numCases, float eps, void* workspace, size_t workspaceBytes, void* stream) {
    MCN_REQUIRE(inputs && target && ln_sizes_ok(numFeatures, numCases), "layerNorm: bad argument");
    MCN_REQUIRE(eps > 0.f, "layerNorm: eps %g is not positive", (double)eps);
    if (int rc = ln_require_workspace(workspace, workspaceBytes, mcn_layer_norm_workspace_bytes(numFeatures, numCases), "layerNorm")) return rc;
    hipStream_t st = (hipStream_t)stream;
    float* part = (float*)workspace;
    const bool vec = numCases % 4 == 0 && al16(inputs) && al16(target) && al16(caseStats);
    const LnShape s = ln_shape(numFeatures, numCases, vec ? 4 : 1);
    const dim3 grid(s.colTiles, s.splits);
    if (vec) {
        MCN_LAUNCH(k_ln_stats<4>, grid, dim3(T), 0, st, inputs, part, s);
        MCN_LAUNCH(k_ln_apply<4>, grid, dim3(T), 0, st, inputs, gains, biases, target, caseStats, part, eps, s);
    } else {
        MCN_LAUNCH(k_ln_stats<1>, grid, dim3(T), 0, st, inputs, part, s);
        MCN_LAUNCH(k_ln_apply<1>, grid, dim3(T), 0, st, inputs, gains, biases, target, caseStats, part, eps, s);
    }
    return MCN_LAUNCH_CHECK("layerNorm");
}

MCN_API size_t mcn_layer_norm_undo_workspace_bytes(int numFeatures, int numCases) {
    if (!ln_sizes_ok(numFeatures, numCases)) return 0;
    size_t b = 0;
    for (int vw = 1; vw <= 4; vw += 3) {
        const LnShape s = ln_shape(numFeatures, numCases, vw);
        b = std::max(b, (al4((size_t)s.splits * 2 * numCases) + (size_t)s.colTiles * 2 * numFeatures) * sizeof(float));
    }
    return b;
}

MCN_API int mcn_layer_norm_undo(const float* outGrads, const float* inputs, const float* gains, const float* caseStats, float* target,
                                float* gainGrads, float* biasGrads, int numFeatures, int numCases, float scaleTargets, float scaleOutput,
                                float scaleGainTargets, float scaleGainOutput, float scaleBiasTargets, float scaleBiasOutput,
                                void* workspace, size_t workspaceBytes, void* stream) {
    MCN_REQUIRE(outGrads && inputs && caseStats && ln_sizes_ok(numFeatures, numCases), "layerNormUndo: bad argument");
    MCN_REQUIRE(target || gainGrads || biasGrads, "layerNormUndo: nothing to compute");
    MCN_REQUIRE(target != outGrads && target != inputs, "layerNormUndo: the target is one of the operands");
    if (int rc = ln_require_workspace(workspace, workspaceBytes, mcn_layer_norm_undo_workspace_bytes(numFeatures, numCases), "layerNormUndo")) return rc;
    hipStream_t st = (hipStream_t)stream;
    const bool vec = numCases % 4 == 0 && al16(outGrads) && al16(inputs) && al16(caseStats) && al16(target);
    const LnShape s = ln_shape(numFeatures, numCases, vec ? 4 : 1);
    float* colPart = (float*)workspace;
    const bool rows = gainGrads || biasGrads;
    float* rowPart = rows ? colPart + al4((size_t)s.splits * 2 * numCases) : nullptr;
    const dim3 grid(s.colTiles, s.splits);
    if (vec)
        MCN_LAUNCH(k_ln_undo_sums<4>, grid, dim3(T), 0, st, outGrads, inputs, gains, caseStats, colPart, rowPart, s);
    else
        MCN_LAUNCH(k_ln_undo_sums<1>, grid, dim3(T), 0, st, outGrads, inputs, gains, caseStats, colPart, rowPart, s);
    if (target) {
        if (vec)
            MCN_LAUNCH(k_ln_undo_apply<4>, grid, dim3(T), 0, st, outGrads, inputs, gains, caseStats, colPart, target, scaleTargets, scaleOutput, s);
        else
            MCN_LAUNCH(k_ln_undo_apply<1>, grid, dim3(T), 0, st, outGrads, inputs, gains, caseStats, colPart, target, scaleTargets, scaleOutput, s);
    }
    if (rows)
        MCN_LAUNCH(k_ln_undo_rows, dim3((unsigned)divup_sz((size_t)2 * numFeatures, T)), dim3(T), 0, st, rowPart, gainGrads, biasGrads, scaleGainTargets,
                   scaleGainOutput, scaleBiasTargets, scaleBiasOutput, numFeatures, s.colTiles);
    return MCN_LAUNCH_CHECK("layerNormUndo");
}
