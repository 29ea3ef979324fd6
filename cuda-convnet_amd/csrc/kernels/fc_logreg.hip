// A fully connected classifier layer, its softmax and the logistic-regression cost in one operator that never holds the
// (numOutputs, numCases) matrix of logits:
//   z = W x + b;  M = max_v z, S = sum_v exp(z - M) per case;  log p[label] = z[label] - M - log S
//   dz = coeff ((v == label) - exp(z - M) / S);  dx (+)= W^T dz,  dW = dz x^T,  db = sum_n dz.
// Forward: tiles of z leave (max, sum of exp(z - max), entries at the max) per case, a second launch joins the tiles.  Backward:
// the classes are taken in pieces whose dz fits a bounded workspace; a piece's z is computed again.
#include <math.h>
#include <algorithm>
#include "common.h"

namespace {

constexpr int BV = 64, BN = 64, BK = 32;  // tile of z: classes x cases, features per step
constexpr size_t PIECE_ELEMS = (size_t)1 << 24;

struct FclArgs {
    const float *W, *X, *bias, *labels;
    int D, V, N;
    int v0, vRows;        // the piece: classes [v0, v0 + vRows)
    int nTiles;
    float* part;          // forward: [vTiles][3][N]
    float* labelLogits;   // forward: [N]
    const float* stats;   // backward: [2][N]
    float* dz;            // backward: [vRows][N]
    float coeff;
};

__device__ __forceinline__ bool label_of(float l, int V, int& label) {
    const bool ok = l >= 0.f && l < (float)V;  // (false for a NaN)
    label = ok ? (int)l : -1;
    return ok;
}

template <bool BWD>
__global__ __launch_bounds__(256) void k_fcl_tile(FclArgs p) {
    __shared__ float As[BV][BK + 4];
    __shared__ float Bs[BK][BN + 4];
    __shared__ float red[3][4][BN];
    const int tn = blockIdx.x % p.nTiles, tv = blockIdx.x / p.nTiles;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int vBase = tv * BV, nBase = tn * BN;
    f32x4 acc[4] = {};
    for (int k0 = 0; k0 < p.D; k0 += BK) {
#pragma unroll
        for (int u = 0; u < BV * BK / 256; u++) {
            const int e = tid + 256 * u, r = e / BK, k = e % BK;
            const bool in = vBase + r < p.vRows && k0 + k < p.D;
            As[r][k] = in ? p.W[(size_t)(p.v0 + vBase + r) * p.D + k0 + k] : 0.f;
        }
#pragma unroll
        for (int u = 0; u < BK * BN / 256; u++) {
            const int e = tid + 256 * u, k = e / BN, c = e % BN;
            const bool in = nBase + c < p.N && k0 + k < p.D;
            Bs[k][c] = in ? p.X[(size_t)(k0 + k) * p.N + nBase + c] : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < BK; k += 4) {
            const float a = As[wave * 16 + (lane & 15)][k + (lane >> 4)];
#pragma unroll
            for (int t = 0; t < 4; t++) acc[t] = mfma16(a, Bs[k + (lane >> 4)][t * 16 + (lane & 15)], acc[t]);
        }
        __syncthreads();
    }
    const int rowInPiece = vBase + wave * 16 + (lane >> 4) * 4;
    float bv[4];
    bool live[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        live[r] = rowInPiece + r < p.vRows;
        bv[r] = live[r] && p.bias ? p.bias[p.v0 + rowInPiece + r] : 0.f;
    }
#pragma unroll
    for (int t = 0; t < 4; t++) {
        const int c = t * 16 + (lane & 15), n = nBase + c;
        int label = -1;
        if (n < p.N) label_of(p.labels[n], p.V, label);
        float z[4];
#pragma unroll
        for (int r = 0; r < 4; r++) z[r] = acc[t][r] + bv[r];
        if (BWD) {
            if (n < p.N) {
                const float M = p.stats[n], S = p.stats[p.N + n];
                const float inv = label >= 0 && S != 0.f ? 1.f / S : 0.f;
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (live[r]) {
                        const float prob = inv != 0.f ? expf(z[r] - M) * inv : 0.f;
                        const float hot = label == p.v0 + rowInPiece + r ? 1.f : 0.f;
                        p.dz[(size_t)(rowInPiece + r) * p.N + n] = label >= 0 && S != 0.f ? p.coeff * (hot - prob) : 0.f;
                    }
            }
            continue;
        }
        float m = -INFINITY;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (live[r] && z[r] > m) m = z[r];
            if (live[r] && label == p.v0 + rowInPiece + r && n < p.N) p.labelLogits[n] = z[r];
        }
        for (int o = 16; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        float s = 0.f, cnt = 0.f;
#pragma unroll
        for (int r = 0; r < 4; r++)
            if (live[r] && z[r] != -INFINITY) {  // (a masked class adds nothing; a NaN comes through)
                s += expf(z[r] - m);
                cnt += z[r] == m ? 1.f : 0.f;
            }
        for (int o = 16; o < 64; o <<= 1) {
            s += __shfl_xor(s, o, 64);
            cnt += __shfl_xor(cnt, o, 64);
        }
        if (lane < 16) {
            red[0][wave][c] = m;
            red[1][wave][c] = s;
            red[2][wave][c] = cnt;
        }
    }
    if (BWD) return;
    __syncthreads();
    if (tid < BN && nBase + tid < p.N) {
        float m = -INFINITY;
        for (int w = 0; w < 4; w++) m = fmaxf(m, red[0][w][tid]);
        float s = 0.f, cnt = 0.f;
        for (int w = 0; w < 4; w++) {
            const float mw = red[0][w][tid];
            // (a wave without a finite logit has sum 0 -- or NaN, if one was NaN)
            s += mw == -INFINITY ? red[1][w][tid] : red[1][w][tid] * expf(mw - m);
            cnt += mw == m ? red[2][w][tid] : 0.f;
        }
        float* out = p.part + (size_t)tv * 3 * p.N + nBase + tid;
        out[0] = m;
        out[p.N] = s;
        out[2 * (size_t)p.N] = cnt;
    }
}

// Joins the tiles of every case: 16 cases x 16 tile lanes per block, tiles in a fixed order.
__global__ __launch_bounds__(256) void k_fcl_join(const float* __restrict__ part, const float* __restrict__ labelLogits,
                                                  const float* __restrict__ labels, float* __restrict__ caseStats, float* __restrict__ logProbs,
                                                  float* __restrict__ correct, int V, int N, int tiles) {
    __shared__ float sh[3][16][17];
    const int c = threadIdx.x & 15, l = threadIdx.x >> 4, n = blockIdx.x * 16 + c;
    float m = -INFINITY, s = 0.f, cnt = 0.f;
    if (n < N)
        for (int t = l; t < tiles; t += 16) {
            const float* q = part + (size_t)t * 3 * N + n;
            const float mt = q[0], st = q[N], ct = q[2 * (size_t)N];
            if (mt > m) {
                s = (m == -INFINITY ? s : s * expf(m - mt)) + st;
                cnt = ct;
                m = mt;
            } else {
                s += mt == -INFINITY ? st : st * expf(mt - m);
                if (mt == m) cnt += ct;
            }
        }
    sh[0][l][c] = m;
    sh[1][l][c] = s;
    sh[2][l][c] = cnt;
    __syncthreads();
    if (l != 0 || n >= N) return;
    for (int k = 0; k < 16; k++) m = fmaxf(m, sh[0][k][c]);
    s = cnt = 0.f;
    for (int k = 0; k < 16; k++) {
        const float mk = sh[0][k][c];
        s += mk == -INFINITY ? sh[1][k][c] : sh[1][k][c] * expf(mk - m);
        cnt += mk == m ? sh[2][k][c] : 0.f;
    }
    caseStats[n] = m;
    caseStats[N + n] = s;
    int label;
    float lp = 0.f, hit = 0.f;
    if (label_of(labels[n], V, label)) {
        const float z = labelLogits[n];
        lp = s == 0.f ? -INFINITY : z - m - logf(s);
        hit = z == m && cnt > 0.f ? 1.f / cnt : 0.f;
    }
    logProbs[n] = lp;
    correct[n] = hit;
}

// costOut[0] += -sum(log p[label]), costOut[1] += cases that count - sum(correct); one block, fixed order.
__global__ __launch_bounds__(256) void k_fcl_cost(const float* __restrict__ labels, const float* __restrict__ logProbs,
                                                  const float* __restrict__ correct, int V, int N, double* costOut) {
    __shared__ double sh[2][256];
    double a = 0, b = 0;
    for (int n = threadIdx.x; n < N; n += 256) {
        int label;
        if (label_of(labels[n], V, label)) {
            a -= logProbs[n];
            b += 1.0 - correct[n];
        }
    }
    sh[0][threadIdx.x] = a;
    sh[1][threadIdx.x] = b;
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) {
        if ((int)threadIdx.x < h) {
            sh[0][threadIdx.x] += sh[0][threadIdx.x + h];
            sh[1][threadIdx.x] += sh[1][threadIdx.x + h];
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        costOut[0] += sh[0][0];
        costOut[1] += sh[1][0];
    }
}

bool fcl_sizes_ok(int D, int V, int N) { return D > 0 && V > 0 && N > 0 && V <= (1 << 24) && D <= (1 << 20) && N <= (1 << 20); }

int fcl_piece_rows(int V, int D, int N) {
    const size_t rows = std::min<size_t>(PIECE_ELEMS / (size_t)std::max(N, D), (size_t)1 << 19) / BV * BV;
    return (int)std::min<size_t>((size_t)V, std::max<size_t>(rows, BV));
}

size_t al16b(size_t b) { return (b + 15) / 16 * 16; }

size_t fcl_cost_bytes(int D, int V, int N) { return al16b((size_t)divup(V, BV) * 3 * N * sizeof(float)) + al16b((size_t)N * sizeof(float)); }
size_t fcl_inner_bytes(int rows, int D, int N) {
    return al16b(std::max({mcn_gemm_workspace_bytes(rows, D, N, 0, 1), mcn_gemm_workspace_bytes(D, N, rows, 1, 0), mcn_add_sum_workspace_bytes(rows, N, 1)}));
}
size_t fcl_grad_bytes(int D, int V, int N) {
    const int rows = fcl_piece_rows(V, D, N), rest = V % rows;
    return al16b((size_t)rows * N * sizeof(float)) + std::max(fcl_inner_bytes(rows, D, N), rest ? fcl_inner_bytes(rest, D, N) : 0);
}

int fcl_check(const char* what, const void* ws, size_t have, size_t need) {
    if (!ws || have < need) {
        mcn_set_error("%s: workspace %zu < %zu bytes", what, ws ? have : (size_t)0, need);
        return MCN_EWORKSPACE;
    }
    MCN_REQUIRE(((uintptr_t)ws & 15) == 0, "%s: the workspace is not 16-byte aligned", what);
    return MCN_OK;
}

}  // namespace

MCN_API size_t mcn_fc_logreg_workspace_bytes(int numInputs, int numOutputs, int numCases, int backward) {
    if (!fcl_sizes_ok(numInputs, numOutputs, numCases)) return 0;
    const size_t fwd = fcl_cost_bytes(numInputs, numOutputs, numCases);
    return backward ? std::max(fwd, fcl_grad_bytes(numInputs, numOutputs, numCases)) : fwd;
}

MCN_API int mcn_fc_logreg_cost(const float* weights, const float* inputs, const float* biases, const float* labels, float* caseStats,
                               float* labelLogProbs, float* correctProbs, int numInputs, int numOutputs, int numCases, double* costOut,
                               void* workspace, size_t workspaceBytes, void* stream) {
    MCN_REQUIRE(weights && inputs && labels && caseStats && labelLogProbs && correctProbs, "fcLogregCost: null pointer");
    MCN_REQUIRE(fcl_sizes_ok(numInputs, numOutputs, numCases), "fcLogregCost: %d inputs, %d outputs, %d cases", numInputs, numOutputs, numCases);
    if (int rc = fcl_check("fcLogregCost", workspace, workspaceBytes, fcl_cost_bytes(numInputs, numOutputs, numCases))) return rc;
    hipStream_t s = (hipStream_t)stream;
    const int tiles = divup(numOutputs, BV);
    FclArgs p = {weights, inputs, biases, labels, numInputs, numOutputs, numCases, 0, numOutputs, divup(numCases, BN)};
    p.part = (float*)workspace;
    p.labelLogits = (float*)((char*)workspace + al16b((size_t)tiles * 3 * numCases * sizeof(float)));
    MCN_REQUIRE((size_t)tiles * p.nTiles < ((size_t)1 << 31), "fcLogregCost: too many tiles");
    MCN_LAUNCH(k_fcl_tile<false>, dim3(tiles * p.nTiles), dim3(256), 0, s, p);
    MCN_LAUNCH(k_fcl_join, dim3(divup(numCases, 16)), dim3(256), 0, s, p.part, p.labelLogits, labels, caseStats, labelLogProbs, correctProbs,
               numOutputs, numCases, tiles);
    if (costOut) MCN_LAUNCH(k_fcl_cost, dim3(1), dim3(256), 0, s, labels, labelLogProbs, correctProbs, numOutputs, numCases, costOut);
    return MCN_LAUNCH_CHECK("fcLogregCost");
}

MCN_API int mcn_fc_logreg_grad(const float* weights, const float* inputs, const float* biases, const float* labels, const float* caseStats,
                               float* inputGrads, float* weightGrads, float* biasGrads, int numInputs, int numOutputs, int numCases,
                               float coeff, float scaleInputTargets, float scaleWeightTargets, float scaleWeightOutput,
                               float scaleBiasTargets, float scaleBiasOutput, void* workspace, size_t workspaceBytes, void* stream) {
    MCN_REQUIRE(weights && inputs && labels && caseStats, "fcLogregGrad: null pointer");
    MCN_REQUIRE(inputGrads || weightGrads || biasGrads, "fcLogregGrad: nothing to compute");
    MCN_REQUIRE(inputGrads != inputs && weightGrads != weights, "fcLogregGrad: a gradient is written over its operand");
    MCN_REQUIRE(fcl_sizes_ok(numInputs, numOutputs, numCases), "fcLogregGrad: %d inputs, %d outputs, %d cases", numInputs, numOutputs, numCases);
    if (int rc = fcl_check("fcLogregGrad", workspace, workspaceBytes, fcl_grad_bytes(numInputs, numOutputs, numCases))) return rc;
    hipStream_t s = (hipStream_t)stream;
    const int D = numInputs, N = numCases, piece = fcl_piece_rows(numOutputs, D, N);
    float* dz = (float*)workspace;
    void* ws = (char*)workspace + al16b((size_t)piece * N * sizeof(float));
    const size_t wsBytes = workspaceBytes - al16b((size_t)piece * N * sizeof(float));
    for (int v0 = 0; v0 < numOutputs; v0 += piece) {
        const int rows = std::min(piece, numOutputs - v0);
        FclArgs p = {weights, inputs, biases, labels, D, numOutputs, N, v0, rows, divup(N, BN)};
        p.stats = caseStats;
        p.dz = dz;
        p.coeff = coeff;
        MCN_LAUNCH(k_fcl_tile<true>, dim3(divup(rows, BV) * p.nTiles), dim3(256), 0, s, p);
        if (int rc = MCN_LAUNCH_CHECK("fcLogregGrad")) return rc;
        if (weightGrads)
            if (int rc = mcn_gemm(dz, inputs, weightGrads + (size_t)v0 * D, rows, D, N, 0, 1, scaleWeightOutput, scaleWeightTargets, ws, wsBytes, stream)) return rc;
        if (biasGrads)
            if (int rc = mcn_add_sum(biasGrads + v0, dz, rows, N, 1, scaleBiasTargets, scaleBiasOutput, ws, wsBytes, stream)) return rc;
        if (inputGrads)
            if (int rc = mcn_gemm(weights + (size_t)v0 * D, dz, inputGrads, D, N, rows, 1, 0, 1.f, v0 ? 1.f : scaleInputTargets, ws, wsBytes, stream)) return rc;
    }
    return MCN_OK;
}
