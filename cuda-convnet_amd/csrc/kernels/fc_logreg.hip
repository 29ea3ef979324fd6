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

constexpr int BV = 64, BN = 64, BK = 32;  // k_fcl_tile: classes x cases, features per step
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

// Statistics of a set of logits: the max, the entries at the max, and the sum of exp(z - max) over the OTHER entries.  The three are
// kept apart because log S = log(count) + log1p(rest / count) is exact where a case is all but certain (S = 1 + a small rest).
struct Stat {
    float m, rest, cnt;
};
__device__ __forceinline__ void stat_join(Stat& a, float m, float rest, float cnt) {
    if (m > a.m) {
        a.rest = (a.rest + a.cnt) * (a.m == -INFINITY ? 1.f : expf(a.m - m)) + rest;  // (nothing there: sum 0, or NaN, which stays)
        a.cnt = cnt;
        a.m = m;
    } else if (m == a.m) {
        a.rest += rest;
        a.cnt += cnt;
    } else {
        a.rest += (rest + cnt) * (m == -INFINITY ? 1.f : expf(m - a.m));
    }
}

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
                const bool top = z[r] == m && m < INFINITY;
                s += top ? 0.f : expf(z[r] - m);
                cnt += top ? 1.f : 0.f;
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
        Stat a = {-INFINITY, 0.f, 0.f};
        for (int w = 0; w < 4; w++) stat_join(a, red[0][w][tid], red[1][w][tid], red[2][w][tid]);
        float* out = p.part + (size_t)tv * 3 * p.N + nBase + tid;
        out[0] = a.m;
        out[p.N] = a.rest;
        out[2 * (size_t)p.N] = a.cnt;
    }
}

// Joins the tiles of every case: 16 cases x 64 tile lanes per block; first the max, then the sums, so that no exponential waits for
// another (running joins of 782 tiles took 32 us for 1024 cases).
__global__ __launch_bounds__(1024) void k_fcl_join(const float* __restrict__ part, const float* __restrict__ labelLogits,
                                                   const float* __restrict__ labels, float* __restrict__ caseStats, float* __restrict__ logProbs,
                                                   float* __restrict__ correct, int V, int N, int tiles) {
    __shared__ float sh[2][64][17];
    const int c = threadIdx.x & 15, l = threadIdx.x >> 4, n = blockIdx.x * 16 + c;
    float m = -INFINITY;
    if (n < N) {
#pragma unroll 8
        for (int t = l; t < tiles; t += 64) m = fmaxf(m, part[(size_t)t * 3 * N + n]);
    }
    sh[0][l][c] = m;
    __syncthreads();
    for (int k = 0; k < 64; k++) m = fmaxf(m, sh[0][k][c]);
    __syncthreads();
    float rest = 0.f, cnt = 0.f;
    if (n < N) {
#pragma unroll 8
        for (int t = l; t < tiles; t += 64) {
            const float* q = part + (size_t)t * 3 * N + n;
            const bool top = q[0] == m;
            // (a tile without a finite logit holds 0, or a NaN, which stays)
            rest += top ? q[N] : (q[N] + q[2 * (size_t)N]) * (q[0] == -INFINITY ? 1.f : expf(q[0] - m));
            cnt += top ? q[2 * (size_t)N] : 0.f;
        }
    }
    sh[0][l][c] = rest;
    sh[1][l][c] = cnt;
    __syncthreads();
    if (l != 0 || n >= N) return;
    for (int k = 1; k < 64; k++) {
        rest += sh[0][k][c];
        cnt += sh[1][k][c];
    }
    const float s = cnt + rest;
    caseStats[n] = m;
    caseStats[N + n] = s;
    int label;
    float lp = 0.f, hit = 0.f;
    if (label_of(labels[n], V, label)) {
        const float z = labelLogits[n];
        lp = s == 0.f ? -INFINITY : cnt > 0.f ? (z - m) - (logf(cnt) + log1pf(rest / cnt)) : z - m - logf(s);
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

// ---------------------------------------------------------------------------------------------------------------------------
// Many cases: the three products on 16-bit matrix instructions with fp32 accuracy.  fp32 matrix instructions reach 157 TFLOP/s, 16-bit
// ones 2500: an fp32 operand is split into 16-bit pieces whose products are exact in fp32, and the products that matter are added up.
//   fp16 x 2 (logits, weight gradient): after scaling by a power of two (max of a row in [2^14, 2^15)) y = hi + 2^-11 lo with 11 bits
//     each; hi hi, hi lo and lo hi are kept (3 instructions), the cross terms in an accumulator of their own, so that lo keeps its
//     bits: relative error 2^-22 of a product, for entries down to 2^-28 of their row's max; an entry further down is off by 2^-50 of
//     that max.  Rows are scaled along the dimension that is NOT summed over, so one large row never costs another its bits.
//   bf16 x 3 (input gradient): y = h + m + l with 8 bits each, hh + hm + mh + hl + lh + mm kept (6 instructions): relative error about
//     2^-24, with fp32's own range.  Its sum runs over the classes, whose weights have no common scale.
// Operands are split ONCE by a pack launch into fragments, the 64 lanes x 16 bytes that one 16 x 16 x 32 instruction reads:
//   fragment (rowBlock, kBlock, piece): lane l holds row l & 15, entries k = 8 (l >> 4) .. + 7 of the block's 32,
// stored one after the other (1 KB each, the pieces of one block together), zero-padded to whole tiles.  A product kernel copies
// fragments to LDS (global_load_lds, 16 bytes a lane, no registers, no swizzle: lanes read them back in order, conflict-free).
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int FRAG = 1024;      // bytes of a fragment
constexpr int TILE = 128;       // rows and columns of a product's tile
constexpr float LO = 2048.f;    // scale of the low fp16 piece

struct Split16 { f16x8 hi, lo; };
__device__ __forceinline__ Split16 split16(const float (&y)[8]) {
    Split16 s;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        s.hi[j] = (_Float16)y[j];
        s.lo[j] = (_Float16)((y[j] - (float)s.hi[j]) * LO);
    }
    return s;
}
struct Split24 { bf16x8 p[3]; };
__device__ __forceinline__ Split24 split24(const float (&y)[8]) {
    Split24 s;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        float r = y[j];
#pragma unroll
        for (int q = 0; q < 3; q++) {
            s.p[q][j] = (__bf16)r;
            r -= (float)s.p[q][j];
        }
    }
    return s;
}
// the power of two that brings a row of largest magnitude m to [2^14, 2^15); a row of zeros, infinities or NaNs stays as it is
__device__ __forceinline__ int scale_exp(float m) { return m > 0.f && m < INFINITY ? 14 - ilogbf(m) : 0; }

// C tile of 128 x 128 by four waves, 64 x 64 each: acc[hi/cross][mb][nb].  P = 2: fp16 pieces, P = 3: bf16 pieces.  A, B: first fragment
// of the tile's first row block; aRow, bRow: bytes between row blocks; k blocks [k0, k1).  LDS: two stages.  One barrier a step: it
// says that a stage has landed (the copies are waited for in front of it) and that everyone has read the other one.
template <int P>
struct Acc {
    f32x4 c[P == 2 ? 2 : 1][4][4];
};
template <int P>
__device__ __forceinline__ void product_tile(const char* A, size_t aRow, const char* B, size_t bRow, int k0, int k1, char* lds, Acc<P>& acc) {
    constexpr int FRAGS = 16 * P, STAGE = FRAGS * FRAG;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
#pragma unroll
    for (int h = 0; h < (P == 2 ? 2 : 1); h++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc.c[h][i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    if (k0 >= k1) return;
    auto copy = [&](int kb, char* stage) {
#pragma unroll
        for (int i = 0; i < FRAGS / 4; i++) {
            const int f = wave * (FRAGS / 4) + i, blk = f / P, q = f % P;
            const char* src = (blk < 8 ? A + (size_t)blk * aRow : B + (size_t)(blk - 8) * bRow) + ((size_t)kb * P + q) * FRAG + lane * 16;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                             (__attribute__((address_space(3))) void*)(stage + f * FRAG), 16, 0, 0);
        }
    };
    copy(k0, lds);
    for (int kb = k0; kb < k1; kb++) {
        const char* cur = lds + ((kb - k0) & 1) * STAGE;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if constexpr (P == 2) {
            f16x8 a[4][2], b[4][2];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    a[i][q] = *reinterpret_cast<const f16x8*>(cur + ((wm * 4 + i) * P + q) * FRAG + lane * 16);
                    b[i][q] = *reinterpret_cast<const f16x8*>(cur + ((8 + wn * 4 + i) * P + q) * FRAG + lane * 16);
                }
            if (kb + 1 < k1) copy(kb + 1, lds + ((kb + 1 - k0) & 1) * STAGE);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    acc.c[0][i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i][0], b[j][0], acc.c[0][i][j], 0, 0, 0);
                    acc.c[1][i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i][0], b[j][1], acc.c[1][i][j], 0, 0, 0);
                    acc.c[1][i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[i][1], b[j][0], acc.c[1][i][j], 0, 0, 0);
                }
        } else {
            bf16x8 a[4][3], b[4][3];
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int q = 0; q < 3; q++) {
                    a[i][q] = *reinterpret_cast<const bf16x8*>(cur + ((wm * 4 + i) * P + q) * FRAG + lane * 16);
                    b[i][q] = *reinterpret_cast<const bf16x8*>(cur + ((8 + wn * 4 + i) * P + q) * FRAG + lane * 16);
                }
            if (kb + 1 < k1) copy(kb + 1, lds + ((kb + 1 - k0) & 1) * STAGE);
#pragma unroll
            for (int s = 2; s >= 0; s--)  // small products first
#pragma unroll
                for (int q = 0; q <= s; q++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            acc.c[0][i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i][q], b[j][s - q], acc.c[0][i][j], 0, 0, 0);
        }
    }
}
__device__ __forceinline__ float acc_value(const Acc<2>& a, int i, int j, int r) { return a.c[0][i][j][r] + a.c[1][i][j][r] * (1.f / LO); }

// ---- packing
__device__ __forceinline__ float max_or_nan(float m, float v) { return v > m || v != v ? v : m; }
__device__ __forceinline__ void store_split16(char* out, int lane, const float (&y)[8]) {
    const Split16 s = split16(y);
    *reinterpret_cast<f16x8*>(out + lane * 16) = s.hi;
    *reinterpret_cast<f16x8*>(out + FRAG + lane * 16) = s.lo;
}

// Fragments of x (D, N).  The first caseBlocks blocks take 16 cases each: (rows = cases, k = features) for the logits; the others 16
// features each: (rows = features, k = cases) for the weight gradient, in which a case without a label is zero, whatever it holds.
// Each block finds its rows' largest magnitudes first; what it reads then comes from its caches.
__global__ __launch_bounds__(512) void k_fcl_pack_x(const float* __restrict__ X, const float* __restrict__ labels, int* __restrict__ caseExp,
                                                    int* __restrict__ featExp, char* __restrict__ byCase, char* __restrict__ byFeat, int D,
                                                    int V, int N, int Kd, int Kn, int caseBlocks) {
    __shared__ float sh[8][16];
    __shared__ int exps[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    float m = 0.f;
    if ((int)blockIdx.x < caseBlocks) {
        const int n = blockIdx.x * 16 + c;
        if (n < N) {
#pragma unroll 8
            for (int d = threadIdx.x >> 4; d < D; d += 32) m = max_or_nan(m, fabsf(X[(size_t)d * N + n]));
        }
        m = max_or_nan(m, __shfl_xor(m, 16, 64));
        m = max_or_nan(m, __shfl_xor(m, 32, 64));
        sh[wave][c] = m;
        __syncthreads();
        if (threadIdx.x < 16) {
            for (int w = 1; w < 8; w++) m = max_or_nan(m, sh[w][c]);
            caseExp[n] = exps[c] = scale_exp(m);
        }
        __syncthreads();
        const int e = exps[c];
        for (int kb = wave; kb < Kd; kb += 8) {
            const int d0 = kb * 32 + g * 8;
            float y[8];
#pragma unroll
            for (int j = 0; j < 8; j++) y[j] = n < N && d0 + j < D ? ldexpf(X[(size_t)(d0 + j) * N + n], e) : 0.f;
            store_split16(byCase + ((size_t)blockIdx.x * Kd + kb) * 2 * FRAG, lane, y);
        }
        return;
    }
    const int d0 = (blockIdx.x - caseBlocks) * 16, r = threadIdx.x >> 5;
    if (d0 + r < D) {
#pragma unroll 4
        for (int n = threadIdx.x & 31; n < N; n += 32) {
            int label;
            const bool counts = label_of(labels[n], V, label);
            const float v = fabsf(X[(size_t)(d0 + r) * N + n]);
            m = counts ? max_or_nan(m, v) : m;
        }
    }
    for (int o = 1; o < 32; o <<= 1) m = max_or_nan(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 31) == 0) featExp[d0 + r] = exps[r] = scale_exp(m);
    __syncthreads();
    const int d = d0 + c, e = exps[c];
    for (int kb = wave; kb < Kn; kb += 8) {
        const int n0 = kb * 32 + g * 8;
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            int label;
            y[j] = d < D && n0 + j < N && label_of(labels[n0 + j], V, label) ? ldexpf(X[(size_t)d * N + n0 + j], e) : 0.f;
        }
        store_split16(byFeat + ((size_t)(d0 / 16) * Kn + kb) * 2 * FRAG, lane, y);
    }
}

// Fragments of a piece of W, 32 classes per block: (rows = classes, k = features, fp16) for the logits and, TRANS, (rows = features,
// k = classes, bf16) for the input gradient.  k order of the latter: entry 8 g + j of a block of 32 is class 4 g + j (j < 4) or
// 16 + 4 g + j - 4, which is how the lanes of the logits' tile hold them.  512 features at a time go through registers (all of a
// thread's loads in flight at once) and LDS; rows of at most 512 features are read once, longer ones a second time for their max.
constexpr int CW = 512, CW_LD = CW + 4;
template <bool TRANS>
__global__ __launch_bounds__(512) void k_fcl_pack_w(const float* __restrict__ W, int* __restrict__ rowExp, char* __restrict__ byClass,
                                                    char* __restrict__ byFeat, int D, int rows, int Kd, int Kv, int Dp) {
    extern __shared__ __attribute__((aligned(16))) float tile[];  // [32][CW_LD], then 32 exponents
    int* exps = reinterpret_cast<int*>(tile + 32 * CW_LD);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, v0 = blockIdx.x * 32, c = lane & 15, g = lane >> 4;
    f32x4 t[4][2];
    auto load = [&](int d0) {  // a wave: rows 4 wave .. + 3, a lane: features d0 + 4 lane .. and 256 further on
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int v = v0 + wave * 4 + r, d = d0 + h * 256 + lane * 4;
                const float* src = W + (size_t)v * D + d;
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
                if (v < rows) {
                    if (d + 4 <= D) {
                        const f32x4u u = *reinterpret_cast<const f32x4u*>(src);
                        x = (f32x4){u[0], u[1], u[2], u[3]};
                    } else {
#pragma unroll
                        for (int j = 0; j < 3; j++)
                            if (d + j < D) x[j] = src[j];
                    }
                }
                t[r][h] = x;
            }
    };
    float m[4] = {};
    for (int d0 = 0; d0 < D; d0 += CW) {
        load(d0);
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < 4; j++) m[r] = max_or_nan(m[r], fabsf(t[r][h][j]));
    }
#pragma unroll
    for (int r = 0; r < 4; r++) {
        for (int o = 1; o < 64; o <<= 1) m[r] = max_or_nan(m[r], __shfl_xor(m[r], o, 64));
        if (lane == 0) rowExp[v0 + wave * 4 + r] = exps[wave * 4 + r] = scale_exp(m[r]);
    }
    const int Dt = TRANS ? Dp : Kd * 32;
    for (int d0 = 0; d0 < Dt; d0 += CW) {
        if (D > CW) load(d0);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int h = 0; h < 2; h++) *reinterpret_cast<f32x4*>(tile + (wave * 4 + r) * CW_LD + h * 256 + lane * 4) = t[r][h];
        __syncthreads();
        for (int f = wave; f < 2 * CW / 32; f += 8) {
            const int rb = f & 1, kb = d0 / 32 + (f >> 1), r = rb * 16 + c;
            if (kb >= Kd) break;
            const f32x4* src = reinterpret_cast<const f32x4*>(tile + r * CW_LD + (f >> 1) * 32 + g * 8);
            const f32x4 lo = src[0], hi = src[1];
            const int e = exps[r];
            float y[8];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                y[j] = ldexpf(lo[j], e);
                y[4 + j] = ldexpf(hi[j], e);
            }
            store_split16(byClass + (((size_t)blockIdx.x * 2 + rb) * Kd + kb) * 2 * FRAG, lane, y);
        }
        if (TRANS)
            for (int f = wave; f < CW / 16 && d0 + f * 16 < Dp; f += 8) {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) y[j] = tile[((j < 4 ? 0 : 12) + g * 4 + j) * CW_LD + f * 16 + c];
                const Split24 s = split24(y);
                char* out = byFeat + ((size_t)(d0 / 16 + f) * Kv + blockIdx.x) * 3 * FRAG + lane * 16;
#pragma unroll
                for (int q = 0; q < 3; q++) *reinterpret_cast<bf16x8*>(out + q * FRAG) = s.p[q];
            }
    }
}
constexpr int PACK_LDS = (32 * CW_LD + 32) * 4;

// ---- logits of a piece
struct WideArgs {
    const char *wByClass, *xByCase;
    const int *rowExp, *caseExp;
    const float *bias, *labels, *stats;
    int V, N, v0, rows, Kd, vTiles, nTiles;
    float *part, *labelLogits;  // forward: part + the piece's first tile
    char *dzByCase, *dzByClass; // backward: (rows = cases, k = classes, bf16) and (rows = classes, k = cases, fp16), of dz / coeff
    float* dbPart;              // backward: [nTiles][V], row sums of dz / coeff
    int Kv, Kn;
};

constexpr int DZ_EXP = 14;                 // |dz / coeff| <= 1
constexpr int DZ_LD = TILE + 4;
constexpr int LOGIT_LDS = TILE * DZ_LD * 4;  // the dz tile; the product's two stages take 64 KB of it

template <bool BWD>
__global__ __launch_bounds__(256, 2) void k_fcl_logits(WideArgs p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // the tiles of one block of classes on one XCD: they read the same rows of W
    int tv, tn;
    mcn_xcd_group(blockIdx.x, p.nTiles, p.vTiles, tv, tn);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    const int c = lane & 15, g = lane >> 4;
    const size_t row = (size_t)p.Kd * 2 * FRAG;
    Acc<2> acc;
    product_tile<2>(p.wByClass + (size_t)tv * 8 * row, row, p.xByCase + (size_t)tn * 8 * row, row, 0, p.Kd, lds, acc);
    const int vBase = tv * TILE + wm * 64, nBase = tn * TILE + wn * 64;
    // z in place of the first accumulator; a class behind the last one gets -inf
#pragma unroll
    for (int i = 0; i < 4; i++) {
        int fw[4];
        float bv[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int v = vBase + i * 16 + g * 4 + r;
            fw[r] = p.rowExp[v];
            bv[r] = v < p.rows ? (p.bias ? p.bias[p.v0 + v] : 0.f) : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int e = p.caseExp[nBase + j * 16 + c];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float z = ldexpf(acc_value(acc, i, j, r), -(fw[r] + e));
                acc.c[0][i][j][r] = bv[r] == -INFINITY && z == z ? -INFINITY : z + bv[r];
            }
        }
    }
    if constexpr (!BWD) {
        __syncthreads();
        float(*red)[3][64] = reinterpret_cast<float(*)[3][64]>(lds);  // [wave][max, rest, count][64 cases]
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = nBase + j * 16 + c;
            int label = -1;
            if (n < p.N) label_of(p.labels[n], p.V, label);
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float z = acc.c[0][i][j][r];
                    m = z > m ? z : m;
                    const int v = vBase + i * 16 + g * 4 + r;
                    if (label == p.v0 + v && v < p.rows) p.labelLogits[n] = z;
                }
            for (int o = 16; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
            float rest = 0.f, cnt = 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float z = acc.c[0][i][j][r];
                    const bool top = z == m && m < INFINITY;
                    if (z != -INFINITY) {
                        rest += top ? 0.f : expf(z - m);
                        cnt += top ? 1.f : 0.f;
                    }
                }
            for (int o = 16; o < 64; o <<= 1) {
                rest += __shfl_xor(rest, o, 64);
                cnt += __shfl_xor(cnt, o, 64);
            }
            if (g == 0) {
                red[wave][0][j * 16 + c] = m;
                red[wave][1][j * 16 + c] = rest;
                red[wave][2][j * 16 + c] = cnt;
            }
        }
        __syncthreads();
        const int t = threadIdx.x, n = tn * TILE + t;
        if (t < TILE && n < p.N) {
            Stat a = {-INFINITY, 0.f, 0.f};
            for (int m = 0; m < 2; m++) {
                const int w = m * 2 + (t >> 6);
                stat_join(a, red[w][0][t & 63], red[w][1][t & 63], red[w][2][t & 63]);
            }
            float* out = p.part + (size_t)tv * 3 * p.N + n;
            out[0] = a.m;
            out[p.N] = a.rest;
            out[2 * (size_t)p.N] = a.cnt;
        }
        return;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = nBase + j * 16 + c;
            int label = -1;
            float M = 0.f, S = 0.f;
            if (n < p.N && label_of(p.labels[n], p.V, label)) {
                M = p.stats[n];
                S = p.stats[p.N + n];
            }
            const bool counts = S != 0.f;  // (no label, or no class left: nothing; a NaN goes on)
            const float inv = counts ? 1.f / S : 0.f;
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float z = acc.c[0][i][j][r];
                    const float hot = label == p.v0 + vBase + i * 16 + g * 4 + r ? 1.f : 0.f;
                    acc.c[0][i][j][r] = counts ? hot - (z == -INFINITY ? 0.f : expf(z - M) * inv) : 0.f;
                }
            if (p.dzByCase) {
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    float y[8];
#pragma unroll
                    for (int k = 0; k < 8; k++) y[k] = acc.c[0][2 * q + (k >> 2)][j][k & 3];
                    const Split24 s = split24(y);
                    char* out = p.dzByCase + ((size_t)(nBase / 16 + j) * p.Kv + vBase / 32 + q) * 3 * FRAG + lane * 16;
#pragma unroll
                    for (int k = 0; k < 3; k++) *reinterpret_cast<bf16x8*>(out + k * FRAG) = s.p[k];
                }
            }
        }
        // turned over in LDS for the weight gradient, whose sum runs over the cases; the row sums on the way
        __syncthreads();
        float* T = reinterpret_cast<float*>(lds);
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int r = 0; r < 4; r++) T[(wm * 64 + i * 16 + g * 4 + r) * DZ_LD + wn * 64 + j * 16 + c] = acc.c[0][i][j][r];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int vb = wave * 2 + u;
            float sum = 0.f;
#pragma unroll
            for (int kb = 0; kb < 4; kb++) {
                const f32x4* src = reinterpret_cast<const f32x4*>(T + (vb * 16 + c) * DZ_LD + kb * 32 + g * 8);
                const f32x4 lo = src[0], hi = src[1];
                float y[8];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    y[k] = lo[k] * (float)(1 << DZ_EXP);
                    y[4 + k] = hi[k] * (float)(1 << DZ_EXP);
                }
                sum += ((lo[0] + lo[1]) + (lo[2] + lo[3])) + ((hi[0] + hi[1]) + (hi[2] + hi[3]));
                if (p.dzByClass) {
                    const Split16 s = split16(y);
                    char* out = p.dzByClass + ((size_t)(tv * 8 + vb) * p.Kn + tn * 4 + kb) * 2 * FRAG + lane * 16;
                    *reinterpret_cast<f16x8*>(out) = s.hi;
                    *reinterpret_cast<f16x8*>(out + FRAG) = s.lo;
                }
            }
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            const int v = tv * TILE + vb * 16 + c;
            if (p.dbPart && g == 0 && v < p.rows) p.dbPart[(size_t)tn * p.V + p.v0 + v] = sum;
        }
    }
}

// ---- weight gradient of a piece: (features x classes) tiles, so that a lane's four rows are four neighbours of one row of W
__global__ __launch_bounds__(256, 2) void k_fcl_wgrad(const char* xByFeat, const char* dzByClass, const int* __restrict__ featExp,
                                                      float* __restrict__ dW, int D, int rows, int Kn, int dTiles, int vTiles, float scaleTargets,
                                                      float scaleOutput) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int tv, td;
    mcn_xcd_group(blockIdx.x, dTiles, vTiles, tv, td);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    const int c = lane & 15, g = lane >> 4;
    const size_t row = (size_t)Kn * 2 * FRAG;
    Acc<2> acc;
    product_tile<2>(xByFeat + (size_t)td * 8 * row, row, dzByClass + (size_t)tv * 8 * row, row, 0, Kn, lds, acc);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = td * TILE + wm * 64 + i * 16 + g * 4;
        int e[4];
#pragma unroll
        for (int r = 0; r < 4; r++) e[r] = -(featExp[d + r] + DZ_EXP);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int v = tv * TILE + wn * 64 + j * 16 + c;
            if (v >= rows) continue;
            float* out = dW + (size_t)v * D + d;
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = scaleOutput * ldexpf(acc_value(acc, i, j, r), e[r]);
            if (d + 4 <= D) {
                f32x4u t = {y[0], y[1], y[2], y[3]};
                if (scaleTargets != 0.f) {
                    const f32x4u old = *reinterpret_cast<const f32x4u*>(out);
#pragma unroll
                    for (int r = 0; r < 4; r++) t[r] += scaleTargets * old[r];
                }
                *reinterpret_cast<f32x4u*>(out) = t;
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (d + r < D) out[r] = (scaleTargets != 0.f ? scaleTargets * out[r] : 0.f) + y[r];
            }
        }
    }
}

// ---- input gradient: the sum over the classes is split; slab s of (Dp, Np) adds up its share of every piece, in order
__global__ __launch_bounds__(256, 1) void k_fcl_igrad(const char* dzByCase, const char* wByFeat, float* __restrict__ slabs, int Np, int Dp,
                                                      int Kv, int kPerSplit, int nTiles, int dTiles, int first) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int tiles = nTiles * dTiles, s = blockIdx.x / tiles, t = blockIdx.x % tiles, td = t / nTiles, tn = t % nTiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    const int c = lane & 15, g = lane >> 4;
    const size_t row = (size_t)Kv * 3 * FRAG;
    Acc<3> acc;
    product_tile<3>(dzByCase + (size_t)tn * 8 * row, row, wByFeat + (size_t)td * 8 * row, row, s * kPerSplit, min(Kv, (s + 1) * kPerSplit), lds, acc);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int d = td * TILE + wn * 64 + j * 16 + c, n = tn * TILE + wm * 64 + i * 16 + g * 4;
            f32x4* out = reinterpret_cast<f32x4*>(slabs + ((size_t)s * Dp + d) * Np + n);
            *out = first ? acc.c[0][i][j] : *out + acc.c[0][i][j];
        }
}

// ---- the end: input gradients from the slabs (blocks below dxBlocks), bias gradients from the tiles' row sums
__global__ __launch_bounds__(256) void k_fcl_finish(const float* __restrict__ slabs, const float* __restrict__ dbPart, float* dX, float* dB,
                                                    int D, int V, int N, int Np, int Dp, int splits, int nTiles, int dxBlocks, float coeff,
                                                    float scaleInputTargets, float scaleBiasTargets, float scaleBiasOutput) {
    if ((int)blockIdx.x < dxBlocks) {
        const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
        if (i >= (size_t)D * N) return;
        const size_t d = i / N, n = i % N;
        float v = 0.f;
#pragma unroll 8
        for (int s = 0; s < splits; s++) v += slabs[((size_t)s * Dp + d) * Np + n];
        dX[i] = (scaleInputTargets != 0.f ? scaleInputTargets * dX[i] : 0.f) + coeff * v;
        return;
    }
    const int v = (blockIdx.x - dxBlocks) * 256 + threadIdx.x;
    if (v >= V) return;
    float s = 0.f;
#pragma unroll 8
    for (int t = 0; t < nTiles; t++) s += dbPart[(size_t)t * V + v];
    dB[v] = (scaleBiasTargets != 0.f ? scaleBiasTargets * dB[v] : 0.f) + scaleBiasOutput * coeff * s;
}

// Sizes and workspace of the wide path: a function of the shape alone.
struct WidePlan {
    int Np, Dp, Kd, Kn, nTiles, dTiles;
    int rows, pieces;        // classes per piece (a multiple of TILE), pieces
    int splits, kPerSplit;   // input gradient
    size_t rowExp, caseExp, featExp, xByCase, xByFeat, wByClass, wByFeat, dzByCase, dzByClass, dbPart, slabs, part, labelLogits, total;
};

bool wide_usable(int D, int V, int N) { return N > 48; }

size_t al256(size_t b) { return (b + 255) / 256 * 256; }

WidePlan wide_plan(int D, int V, int N, bool bwd) {
    WidePlan p = {};
    p.nTiles = divup(N, TILE);
    p.dTiles = divup(D, TILE);
    p.Np = p.nTiles * TILE;
    p.Dp = p.dTiles * TILE;
    p.Kd = divup(D, 32);
    p.Kn = p.Np / 32;
    // a piece's fragments should stay in the 256 MB last-level cache between the launches that write and read them
    const size_t perRow = (size_t)p.Kd * 128 + (bwd ? (size_t)p.Dp * 6 + (size_t)p.Np * 10 : 0);
    const int most = (int)std::max<size_t>(1, std::min<size_t>(((size_t)128 << 20) / perRow / TILE, (size_t)1 << 16));
    p.pieces = divup(divup(V, TILE), most);
    p.rows = divup(divup(V, TILE), p.pieces) * TILE;
    p.pieces = divup(V, p.rows);
    const int Kv = p.rows / 32;
    p.splits = std::max(1, std::min(Kv / 8, 256 / (p.nTiles * p.dTiles)));
    p.kPerSplit = divup(Kv, p.splits);
    p.splits = divup(Kv, p.kPerSplit);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += al256(bytes); return o; };
    p.rowExp = take((size_t)p.rows * 4);
    p.caseExp = take((size_t)p.Np * 4);
    p.featExp = take((size_t)p.Dp * 4);
    p.xByCase = take((size_t)p.Np / 16 * p.Kd * 2 * FRAG);
    p.wByClass = take((size_t)p.rows / 16 * p.Kd * 2 * FRAG);
    if (bwd) {
        p.xByFeat = take((size_t)p.Dp / 16 * p.Kn * 2 * FRAG);
        p.wByFeat = take((size_t)p.Dp / 16 * Kv * 3 * FRAG);
        p.dzByCase = take((size_t)p.Np / 16 * Kv * 3 * FRAG);
        p.dzByClass = take((size_t)p.rows / 16 * p.Kn * 2 * FRAG);
        p.dbPart = take((size_t)p.nTiles * V * 4);
        p.slabs = take((size_t)p.splits * p.Dp * p.Np * 4);
    } else {
        p.part = take((size_t)p.pieces * (p.rows / TILE) * 3 * N * 4);
        p.labelLogits = take((size_t)N * 4);
    }
    p.total = at;
    return p;
}

int wide_cost(const float* W, const float* X, const float* bias, const float* labels, float* stats, float* logp, float* correct, int D, int V,
              int N, char* ws, hipStream_t s) {
    const WidePlan q = wide_plan(D, V, N, false);
    WideArgs a = {};
    a.wByClass = ws + q.wByClass;
    a.xByCase = ws + q.xByCase;
    a.rowExp = (const int*)(ws + q.rowExp);
    a.caseExp = (const int*)(ws + q.caseExp);
    a.bias = bias; a.labels = labels; a.V = V; a.N = N; a.Kd = q.Kd; a.nTiles = q.nTiles;
    a.labelLogits = (float*)(ws + q.labelLogits);
    MCN_LAUNCH(k_fcl_pack_x, dim3(q.Np / 16), dim3(512), 0, s, X, labels, (int*)(ws + q.caseExp), (int*)nullptr, ws + q.xByCase, (char*)nullptr,
               D, V, N, q.Kd, q.Kn, q.Np / 16);
    int tiles = 0;
    for (int v0 = 0; v0 < V; v0 += q.rows) {
        const int rows = std::min(q.rows, V - v0), vTiles = divup(rows, TILE);
        MCN_LAUNCH(k_fcl_pack_w<false>, dim3(vTiles * (TILE / 32)), dim3(512), PACK_LDS, s, W + (size_t)v0 * D, (int*)(ws + q.rowExp), ws + q.wByClass,
                   (char*)nullptr, D, rows, q.Kd, vTiles * (TILE / 32), q.Dp);
        a.v0 = v0;
        a.rows = rows;
        a.vTiles = vTiles;
        a.part = (float*)(ws + q.part) + (size_t)tiles * 3 * N;
        MCN_LAUNCH(k_fcl_logits<false>, dim3(vTiles * q.nTiles), dim3(256), LOGIT_LDS, s, a);
        tiles += vTiles;
        if (int rc = MCN_LAUNCH_CHECK("fcLogregCost")) return rc;
    }
    MCN_LAUNCH(k_fcl_join, dim3(divup(N, 16)), dim3(1024), 0, s, (const float*)(ws + q.part), a.labelLogits, labels, stats, logp, correct, V, N, tiles);
    return MCN_LAUNCH_CHECK("fcLogregCost");
}

int wide_grad(const float* W, const float* X, const float* bias, const float* labels, const float* stats, float* dX, float* dW, float* dB, int D,
              int V, int N, float coeff, float scaleInputTargets, float scaleWeightTargets, float scaleWeightOutput, float scaleBiasTargets,
              float scaleBiasOutput, char* ws, hipStream_t s) {
    const WidePlan q = wide_plan(D, V, N, true);
    WideArgs a = {};
    a.wByClass = ws + q.wByClass;
    a.xByCase = ws + q.xByCase;
    a.rowExp = (const int*)(ws + q.rowExp);
    a.caseExp = (const int*)(ws + q.caseExp);
    a.bias = bias; a.labels = labels; a.stats = stats; a.V = V; a.N = N; a.Kd = q.Kd; a.nTiles = q.nTiles; a.Kn = q.Kn;
    a.dzByCase = dX ? ws + q.dzByCase : nullptr;
    a.dzByClass = dW ? ws + q.dzByClass : nullptr;
    a.dbPart = dB ? (float*)(ws + q.dbPart) : nullptr;
    MCN_LAUNCH(k_fcl_pack_x, dim3(q.Np / 16 + (dW ? q.Dp / 16 : 0)), dim3(512), 0, s, X, labels, (int*)(ws + q.caseExp), (int*)(ws + q.featExp),
               ws + q.xByCase, ws + q.xByFeat, D, V, N, q.Kd, q.Kn, q.Np / 16);
    for (int v0 = 0; v0 < V; v0 += q.rows) {
        const int rows = std::min(q.rows, V - v0), vTiles = divup(rows, TILE), Kv = vTiles * (TILE / 32);
        if (dX)
            MCN_LAUNCH(k_fcl_pack_w<true>, dim3(Kv), dim3(512), PACK_LDS, s, W + (size_t)v0 * D, (int*)(ws + q.rowExp), ws + q.wByClass,
                       ws + q.wByFeat, D, rows, q.Kd, Kv, q.Dp);
        else
            MCN_LAUNCH(k_fcl_pack_w<false>, dim3(Kv), dim3(512), PACK_LDS, s, W + (size_t)v0 * D, (int*)(ws + q.rowExp), ws + q.wByClass,
                       ws + q.wByFeat, D, rows, q.Kd, Kv, q.Dp);
        a.v0 = v0;
        a.rows = rows;
        a.vTiles = vTiles;
        a.Kv = Kv;
        MCN_LAUNCH(k_fcl_logits<true>, dim3(vTiles * q.nTiles), dim3(256), LOGIT_LDS, s, a);
        if (dW)
            MCN_LAUNCH(k_fcl_wgrad, dim3(vTiles * q.dTiles), dim3(256), 2 * 32 * FRAG, s, ws + q.xByFeat, a.dzByClass, (const int*)(ws + q.featExp),
                       dW + (size_t)v0 * D, D, rows, q.Kn, q.dTiles, vTiles, scaleWeightTargets, scaleWeightOutput * coeff);
        if (dX)
            MCN_LAUNCH(k_fcl_igrad, dim3(q.splits * q.nTiles * q.dTiles), dim3(256), 2 * 48 * FRAG, s, a.dzByCase, ws + q.wByFeat,
                       (float*)(ws + q.slabs), q.Np, q.Dp, Kv, q.kPerSplit, q.nTiles, q.dTiles, v0 == 0);
        if (int rc = MCN_LAUNCH_CHECK("fcLogregGrad")) return rc;
    }
    if (dX || dB) {
        const int dxBlocks = dX ? (int)divup_sz((size_t)D * N, 256) : 0;
        MCN_LAUNCH(k_fcl_finish, dim3(dxBlocks + (dB ? divup(V, 256) : 0)), dim3(256), 0, s, (const float*)(ws + q.slabs), (const float*)(ws + q.dbPart),
                   dX, dB, D, V, N, q.Np, q.Dp, q.splits, q.nTiles, dxBlocks, coeff, scaleInputTargets, scaleBiasTargets, scaleBiasOutput);
    }
    return MCN_LAUNCH_CHECK("fcLogregGrad");
}

bool fcl_sizes_ok(int D, int V, int N) { return D > 0 && V > 0 && N > 0 && V <= (1 << 24) && D <= (1 << 20) && N <= (1 << 20); }

int fcl_piece_rows(int V, int D, int N) {
    const size_t rows = std::min<size_t>(PIECE_ELEMS / (size_t)std::max(N, D), (size_t)1 << 19) / BV * BV;
    return (int)std::min<size_t>((size_t)V, std::max<size_t>(rows, BV));
}

size_t al16b(size_t b) { return (b + 15) / 16 * 16; }

size_t fcl_cost_bytes(int D, int V, int N) {
    if (wide_usable(D, V, N)) return wide_plan(D, V, N, false).total;
    return al16b((size_t)divup(V, BV) * 3 * N * sizeof(float)) + al16b((size_t)N * sizeof(float));
}
size_t fcl_inner_bytes(int rows, int D, int N) {
    return al16b(std::max({mcn_gemm_workspace_bytes(rows, D, N, 0, 1), mcn_gemm_workspace_bytes(D, N, rows, 1, 0), mcn_add_sum_workspace_bytes(rows, N, 1)}));
}
size_t fcl_grad_bytes(int D, int V, int N) {
    if (wide_usable(D, V, N)) return wide_plan(D, V, N, true).total;
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
    if (wide_usable(numInputs, numOutputs, numCases)) {
        if (int rc = wide_cost(weights, inputs, biases, labels, caseStats, labelLogProbs, correctProbs, numInputs, numOutputs, numCases, (char*)workspace, s)) return rc;
    } else {
        const int tiles = divup(numOutputs, BV);
        FclArgs p = {weights, inputs, biases, labels, numInputs, numOutputs, numCases, 0, numOutputs, divup(numCases, BN)};
        p.part = (float*)workspace;
        p.labelLogits = (float*)((char*)workspace + al16b((size_t)tiles * 3 * numCases * sizeof(float)));
        MCN_LAUNCH(k_fcl_tile<false>, dim3(tiles * p.nTiles), dim3(256), 0, s, p);
        MCN_LAUNCH(k_fcl_join, dim3(divup(numCases, 16)), dim3(1024), 0, s, p.part, p.labelLogits, labels, caseStats, labelLogProbs, correctProbs,
                   numOutputs, numCases, tiles);
    }
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
    if (wide_usable(numInputs, numOutputs, numCases))
        return wide_grad(weights, inputs, biases, labels, caseStats, inputGrads, weightGrads, biasGrads, numInputs, numOutputs, numCases, coeff,
                         scaleInputTargets, scaleWeightTargets, scaleWeightOutput, scaleBiasTargets, scaleBiasOutput, (char*)workspace, s);
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
