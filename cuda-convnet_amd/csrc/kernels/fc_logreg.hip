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

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // (16-byte accesses at any multiple of four bytes)

constexpr int NARROW = 64;  // k_fcl_narrow: most cases
// Fragments of a piece, the most MB.  Both calls at 96 / 128 / 160 / 192 / 256 MB, ms: 512 x 100000 x 1024 1.51 / 1.52 / 1.52 / 1.44 / 1.49,
// 1024 x 50000 x 1024 1.51 / 1.46 / 1.42 / 1.39 / 1.41, 160 x 300000 x 512 1.49 / 1.51 / 1.46 / 1.44 / 1.46, 512 x 60000 x 2048 1.84 / 1.65 /
// 1.60 / 1.60 / 1.65, 512 x 200000 x 512 1.90 / 1.71 / 1.74 / 1.69 / 1.66; 2048 x 60000 x 256 alone would have 256: 1.65 / 1.50 / 1.60 / 1.50 / 1.37.
constexpr int PIECE_MB = 192;

struct NarrowArgs {
    const float *W, *X, *bias, *labels;
    int D, V, N;
    int v0, rows;        // the piece: classes [v0, v0 + rows)
    float* part;         // forward: [tiles][3][N]
    float* labelLogits;  // forward: [N]
    const float* stats;  // backward
    char* dz;            // backward: dz / coeff, split into fragments of (rows = cases, k = classes) as the wide path's
    size_t near;         // and once more, this far behind it, without the levels
    unsigned char* levels;
    int* anyLevel;
    float* dbPart;       // backward: [V], row sums of dz / coeff
    int Kv;
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

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __fp16 fp16x4 __attribute__((__vector_size__(4 * sizeof(__fp16))));  // (the type the transposing read is declared with)

constexpr int FRAG = 1024, PAIR = 2 * FRAG;  // bytes of a fragment, of its two pieces
constexpr int TILE = 128;                    // columns of a product's tile
constexpr float LO = 2048.f;                 // scale of the low piece
constexpr int DZ_EXP = 14;                   // |dz / coeff| <= 1
// dz / coeff of a class that is far from 64 cases, all of it below 2^-28, is stored times a further 2^28, below 2^-56 2^56 and below 2^-84
// 2^74 (a level, one byte for every class and 64 cases): so what a class's weight gradient sums has its 22 bits down to 2^-102, and fewer down
// to 2^-124.  (At one scale for all, 2^14, an entry of 2^-36 is off by 6e-5 of itself, one of 2^-48 by 0.2, and below 2^-50 nothing is left.)
constexpr float FAR = 1.f / (1 << 28);
__device__ __forceinline__ int level_of(float most) { return most == 0.f || !(most < FAR) ? 0 : most >= FAR * FAR ? 1 : most >= FAR * FAR * FAR ? 2 : 3; }
__device__ __forceinline__ int level_exp(int level) { return min(28 * level, 74); }
__device__ __forceinline__ float level_scale(int level) { return ldexpf(1.f, DZ_EXP + level_exp(level)); }
// the largest of the 16 lanes of a row; a NaN is larger than anything
__device__ __forceinline__ float row_max(float v) {
    unsigned m = __float_as_uint(v);
#define ROTATED(n) (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x120 + n, 0xf, 0xf, false)
    m = max(m, ROTATED(8));
    m = max(m, ROTATED(4));
    m = max(m, ROTATED(2));
    m = max(m, ROTATED(1));
#undef ROTATED
    return __uint_as_float(m);
}
constexpr int EXP_ZERO = 1 << 20;            // a group of zeros: any scale will do
// The exponents of the cases and of the groups of 32 classes are kept with a flag: whether the group holds an infinity or NaN.
__device__ __forceinline__ int exp_odd(int e, bool odd) { return e * 2 + (odd ? 1 : 0); }
__device__ __forceinline__ int exp_of(int eo) { return eo >> 1; }
__device__ __forceinline__ bool is_odd(int eo) { return eo & 1; }

__device__ __forceinline__ bool label_of(float l, int V, int& label) {
    const bool ok = l >= 0.f && l < (float)V;  // (false for a NaN)
    label = ok ? (int)l : -1;
    return ok;
}

// exp(x) for x <= 0, to about one unit in the last place: 2^(x log2 e) with the product's rounding error carried along.  Below -104 the
// result is no normal number, and 0 will do; a NaN comes through.
__device__ __forceinline__ float exp_neg(float x) {
    constexpr float L = 1.44269504f, L_LOW = 1.925963033500e-8f, LN2 = 0.693147181f;  // log2 e = L + L_LOW
    x = x < -104.f ? -104.f : x;
    const float h = x * L, l = fmaf(x, L_LOW, fmaf(x, L, -h));
    const float e = __builtin_amdgcn_exp2f(h);
    return fmaf(e * LN2, l, e);
}

// Few cases (at most 16 NB): bound by reading W once, so fp32 matrix instructions do, straight from the operands' own layouts.  A block
// takes 16 RG classes, its four waves a quarter of the features each (16 at a time: a lane reads 16 bytes of its class's row, and the
// four matrix instructions that follow take one feature of every lane's four); their sums are joined in LDS.  RG = 1 while the classes
// do not fill the chip, 4 beyond, where it keeps the number of tiles to join down.  160 x 4213, one case: 4.4 us and 5.2 us to join, bound
// by two launches; 512 x 100000, 16 cases: 42 us (4.9 TB/s) and 14 us to join.
// Backward, the logits are computed again in the same way, and so to the same bits: where a case is all but certain, 1 - p of its label
// is a difference that other roundings of z would drown.
template <bool BWD, int NB, int RG>
__global__ __launch_bounds__(256) void k_fcl_narrow(NarrowArgs p) {
    __shared__ f32x4 red[4][RG][NB][64];
    __shared__ float rowSum[4][16 * RG], rowMax[4][16 * RG];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int vBase = blockIdx.x * 16 * RG;
    const float* rowPtr[RG];
#pragma unroll
    for (int q = 0; q < RG; q++) rowPtr[q] = p.W + (size_t)(p.v0 + min(vBase + q * 16 + c, p.rows - 1)) * p.D;  // (a class behind the last one: read and not used)
    f32x4 acc[RG][NB] = {};
    const int steps = (p.D + 15) / 16;
    for (int t = wave; t < steps; t += 4) {
        const int k = t * 16 + g * 4;
        f32x4 a[RG];
        float b[NB][4];
        const bool whole = k + 4 <= p.D;
#pragma unroll
        for (int q = 0; q < RG; q++) {
            if (whole) {
                const f32x4u u = *reinterpret_cast<const f32x4u*>(rowPtr[q] + k);
                a[q] = (f32x4){u[0], u[1], u[2], u[3]};
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) a[q][j] = k + j < p.D ? rowPtr[q][k + j] : 0.f;
            }
        }
#pragma unroll
        for (int n = 0; n < NB; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) b[n][j] = n * 16 + c < p.N && k + j < p.D ? p.X[(size_t)(k + j) * p.N + n * 16 + c] : 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int q = 0; q < RG; q++)
#pragma unroll
                for (int n = 0; n < NB; n++) acc[q][n] = mfma16(a[q][j], b[n][j], acc[q][n]);
    }
#pragma unroll
    for (int q = 0; q < RG; q++)
#pragma unroll
        for (int n = 0; n < NB; n++) red[wave][q][n][lane] = acc[q][n];
    __syncthreads();
    float z[RG][4], m = -INFINITY;
    const int n = wave * 16 + c;  // a wave: 16 cases
    int label = -1;
    if (wave < NB) {
        if (n < p.N) label_of(p.labels[n], p.V, label);
#pragma unroll
        for (int q = 0; q < RG; q++) {
            const f32x4 s = (red[0][q][wave][lane] + red[1][q][wave][lane]) + (red[2][q][wave][lane] + red[3][q][wave][lane]);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int v = vBase + q * 16 + g * 4 + r;
                const float bv = v < p.rows ? (p.bias ? p.bias[p.v0 + v] : 0.f) : -INFINITY;
                z[q][r] = bv == -INFINITY ? -INFINITY : s[r] + bv;  // (a class that is taken out, whatever its weights hold)
                m = fmaxf(z[q][r], m);
            }
        }
    }
    if constexpr (BWD) {
        float M = 0.f, S = 0.f;
        if (label >= 0) {
            M = p.stats[n];
            S = p.stats[p.N + n];
        }
        const bool counts = S != 0.f;  // (no label, or no class left: nothing; a NaN goes on)
        const float inv = counts ? 1.f / S : 0.f;
        char* out = p.dz + ((size_t)wave * p.Kv + vBase / 32) * PAIR + lane * 8;
        char* rest = out + (size_t)4 * p.Kv * PAIR;  // cases 64 .. 127 of the tile: there are none
        auto place = [&](int q) { return ((vBase / 16 + q) & 1) * 512 + (((vBase & 16) + q * 16) >> 5) * PAIR; };
        auto store = [&](char* to, const float (&t)[4], const float (&scale)[4]) {
            f16x4 hi, lo;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float y = t[r] * scale[r];
                hi[r] = (_Float16)y;
                lo[r] = (_Float16)((y - (float)hi[r]) * LO);
            }
            *reinterpret_cast<f16x4*>(to) = hi;
            *reinterpret_cast<f16x4*>(to + FRAG) = lo;
        };
#pragma unroll
        for (int q = 0; q < RG; q++) {
            const float one = (float)(1 << DZ_EXP);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                float t = 0.f;
                if (wave < NB && counts) t = (label == p.v0 + vBase + q * 16 + g * 4 + r ? 1.f : 0.f) - exp_neg(z[q][r] - M) * inv;
                z[q][r] = t;
                const float most = row_max(fabsf(t));
                for (int o = 1; o < 16; o <<= 1) t += __shfl_xor(t, o, 64);
                if (c == 0) {
                    rowSum[wave][q * 16 + g * 4 + r] = t;
                    rowMax[wave][q * 16 + g * 4 + r] = most;
                }
            }
            store(out + p.near + place(q), z[q], {one, one, one, one});
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < RG; q++) {
            float scale[4];
            unsigned levels = 0;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int v = q * 16 + g * 4 + r;
                const int level = level_of(fmaxf(fmaxf(rowMax[0][v], rowMax[1][v]), fmaxf(rowMax[2][v], rowMax[3][v])));
                scale[r] = level_scale(level);
                levels |= level << 8 * r;
            }
            store(out + place(q), z[q], scale);
            *reinterpret_cast<f16x4*>(rest + place(q)) = (f16x4){};
            *reinterpret_cast<f16x4*>(rest + place(q) + FRAG) = (f16x4){};
            if (c == 0 && wave == 0 && levels) {  // (of cases 64 .. 127 there are none)
                *reinterpret_cast<unsigned*>(p.levels + vBase + q * 16 + g * 4) = levels;
                *p.anyLevel = 1;
            }
        }
        if (p.dbPart && tid < 16 * RG && vBase + tid < p.rows)
            p.dbPart[p.v0 + vBase + tid] = (rowSum[0][tid] + rowSum[1][tid]) + (rowSum[2][tid] + rowSum[3][tid]);
        return;
    }
    if (wave >= NB) return;
    for (int o = 16; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const float from = m == -INFINITY ? 0.f : m;
    float rest = 0.f, cnt = 0.f;
#pragma unroll
    for (int q = 0; q < RG; q++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float x = z[q][r] - from;
            const bool top = x == 0.f && m != -INFINITY;
            rest += top ? 0.f : exp_neg(x);
            cnt += top ? 1.f : 0.f;
            if (label >= 0 && label == vBase + q * 16 + g * 4 + r) p.labelLogits[n] = z[q][r];
        }
    for (int o = 16; o < 64; o <<= 1) {
        rest += __shfl_xor(rest, o, 64);
        cnt += __shfl_xor(cnt, o, 64);
    }
    if (g == 0 && n < p.N) {
        float* out = p.part + (size_t)blockIdx.x * 3 * p.N + n;
        out[0] = m;
        out[p.N] = rest;
        out[2 * (size_t)p.N] = cnt;
    }
}

// Joins the tiles of every case: 16 cases x 64 tile lanes per block; first the max, then the sums, so that no exponential waits for
// another.  A lane asks for all of its first eight tiles at once and keeps them (up to 512 tiles: one trip to memory, 5.2-6.3 us; 100000
// classes x 1024 cases, 800 tiles: 12.6 us).
__global__ __launch_bounds__(1024) void k_fcl_join(const float* __restrict__ part, const float* __restrict__ labelLogits,
                                                   const float* __restrict__ labels, float* __restrict__ caseStats, float* __restrict__ logProbs,
                                                   float* __restrict__ correct, int V, int N, int tiles) {
    constexpr int KEPT = 8;
    __shared__ float sh[2][64][17];
    const int c = threadIdx.x & 15, l = threadIdx.x >> 4, n = blockIdx.x * 16 + c;
    const float* at = part + (size_t)l * 3 * N + n;
    const size_t step = (size_t)64 * 3 * N;
    float km[KEPT], kr[KEPT], kc[KEPT];
#pragma unroll
    for (int i = 0; i < KEPT; i++) {
        const bool in = n < N && l + 64 * i < tiles;
        km[i] = in ? at[i * step] : -INFINITY;
        kr[i] = in ? at[i * step + N] : 0.f;
        kc[i] = in ? at[i * step + 2 * (size_t)N] : 0.f;
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < KEPT; i++) m = fmaxf(m, km[i]);
    if (n < N) {
#pragma unroll 8
        for (int t = l + 64 * KEPT; t < tiles; t += 64) m = fmaxf(m, part[(size_t)t * 3 * N + n]);
    }
    sh[0][l][c] = m;
    __syncthreads();
    for (int k = 0; k < 64; k++) m = fmaxf(m, sh[0][k][c]);
    __syncthreads();
    float rest = 0.f, cnt = 0.f;
    auto add = [&](float tm, float tr, float tc) {
        const bool top = tm == m;
        // (a tile without a finite logit holds 0, or a NaN, which stays)
        rest += top ? tr : (tr + tc) * (tm == -INFINITY ? 1.f : expf(tm - m));
        cnt += top ? tc : 0.f;
    };
#pragma unroll
    for (int i = 0; i < KEPT; i++) add(km[i], kr[i], kc[i]);
    if (n < N) {
#pragma unroll 8
        for (int t = l + 64 * KEPT; t < tiles; t += 64) {
            const float* q = part + (size_t)t * 3 * N + n;
            add(q[0], q[N], q[2 * (size_t)N]);
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
// Many cases: the three products on fp16 matrix instructions with fp32 accuracy.  fp32 matrix instructions reach 157 TFLOP/s, fp16 ones
// 2500: an fp32 operand, scaled by a power of two, is split into y = hi + 2^-11 lo with 11 bits each; the products of pieces are exact in
// fp32, and hi hi, hi lo and lo hi are summed (3 instructions), the cross terms in an accumulator of their own, so that lo keeps its
// bits.  With the largest magnitude of a scaled group below 2^15 the relative error of a product is at most 2^-21 (2^-23 of either operand and
// lo lo, which is left out, 2^-22; 2^-24 in the mean square) for entries down to 2^-21 of the group's largest, and an entry further down is off
// by at most 2^-43 of it.  The groups: a case's features for the
// logits, a feature's cases for the weight gradient, 32 classes' weights, and for dz / coeff a class over 64 cases in the weight gradient
// (levels, above) and all of it in the input gradient, where the label's entry, 1 - p, is off by 2^-25 anyway.  Along the summed dimension
// a group is either whole or its scale is carried along (CarryScale, CarryLevels), so a row of large weights takes no bits from the
// other groups, nor one case that is sure of a class from the class's other cases.
//
// Operands are split ONCE by a pack launch into fragments of 16 rows x 32 k entries and two pieces, 1 KB each:
//   entry (row c, k = 16 h + 4 g + j) of a piece lies at byte 512 h + 128 g + 8 c + 2 j, zero-padded to whole tiles.
// A product copies fragments to LDS as they are (global_load_lds, 16 bytes a lane: no registers, no swizzle).  As the first operand,
// and with k along its own k, a lane (c, g) of a 16 x 16 x 32 instruction reads two 8-byte entries, h = 0 and 1; as the operand whose k
// is the fragments' ROW, a transposing LDS read (ds_read_b64_tr_b16) gives lane (k = 16 h + c, g) rows 4 g .. 4 g + 3 of two fragments.
// Both read 512 contiguous bytes a wave, without conflicts, and in both a lane's eight entries are 4 g + j and 16 + 4 g + j of the step's
// 32, so that every pairing sums the same terms.  So W and dz are each stored once, and serve two products.

// the power of two that brings a group of largest finite magnitude m to [2^14, 2^15)
__device__ __forceinline__ int scale_exp(float m) { return m > 0.f ? 14 - ilogbf(m) : 0; }
__device__ __forceinline__ void max_finite(float& m, bool& odd, float v) {
    const bool finite = v < INFINITY;  // (v >= 0; false for a NaN)
    m = fmaxf(m, finite ? v : 0.f);
    odd |= !finite;
}

// An infinity's pieces are infinite and NaN, and so are its products: right for the gradients, where a finite dz (0, or below 1 in size)
// meets it, but not for the logits (odd_logits).
// entries k = 16 h + 4 g + j (y[4 h + j]) of row c into a fragment pair, lane = 16 g + c
__device__ __forceinline__ void store_pair(char* out, int lane, const float (&y)[8]) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        f16x4 hi, lo;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            hi[j] = (_Float16)y[4 * h + j];
            lo[j] = (_Float16)((y[4 * h + j] - (float)hi[j]) * LO);
        }
        *reinterpret_cast<f16x4*>(out + h * 512 + lane * 8) = hi;
        *reinterpret_cast<f16x4*>(out + FRAG + h * 512 + lane * 8) = lo;
    }
}

// ---- one product tile: (32 MB) x 128 by four waves, 2 x 2, each (16 MB) x 64.
template <int MB>
struct Acc {
    f32x4 c[2][MB][4];  // hi hi; cross terms, still times LO
    __device__ __forceinline__ float value(int i, int j, int r) const { return c[0][i][j][r] + c[1][i][j][r] * (1.f / LO); }
};
template <int MB>
struct Frags {
    f16x8 a[MB][2], b[4][2];
};
// LDS stages of a block that has its CU to itself: as many as 144 KB hold.  A 64 x 128 tile spends 384 matrix cycles on a step of 24 KB,
// and needs five stages in flight for it.
constexpr int tile_stages(int mb) { return mb == 4 ? 4 : 6; }
constexpr int tile_units(int mb) { return 2 * mb + 8; }
constexpr int tile_lds(int mb) { return tile_stages(mb) * tile_units(mb) * PAIR; }

// All but the N youngest copies of this wave have landed, its LDS reads are done, and everyone is here.
template <int N>
__device__ __forceinline__ void wait_copies_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0), by the builtin: the compiler then knows that the reads are done
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// The two pieces of a pair (2 KB) from global memory to LDS; the instruction's offset counts on both sides.  The compiler would drain
// every such copy in front of the next LDS read if it knew of it; here the waits are wait_copies_and_meet's.  No register but m0 is written.
__device__ __forceinline__ void copy_pair_half(const char* src, unsigned lds, unsigned laneOff, int piece) {
    if (piece == 0) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(laneOff), "s"(src) : "m0", "memory");
    else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:1024" ::"s"(lds), "v"(laneOff), "s"(src) : "m0", "memory");
}
__device__ __forceinline__ f16x8 read_frag(const char* p) {
    const f16x4 a = *reinterpret_cast<const f16x4*>(p), b = *reinterpret_cast<const f16x4*>(p + 512);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ f16x8 read_frag_turned(const char* p, const char* q) {
    const f16x4 a = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)p));
    const f16x4 b = __builtin_bit_cast(f16x4, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) fp16x4*)q));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

struct NoScale {
    template <int MB>
    __device__ __forceinline__ void operator()(int, Acc<MB>&) const {}
    __device__ __forceinline__ bool moves(int) const { return false; }
    __device__ __forceinline__ size_t move(int) const { return 0; }
};

// A: pair (row block 0 of the tile, k block 0); aRow: bytes between its row blocks.  B: the same, or, TURNED, pair (row block 0, k block 0
// of the tile's columns) of fragments whose rows are this product's k.  scale(step, acc) runs in front of a step's products,
// where scale.moves(step), scale.move(step) is added to where this wave copies from, from that step on.
//
// Step t multiplies what step t - 1 read, reads stage t + 1 and asks for stage t + STAGES, whose buffer everyone has read by then.  One
// wave a SIMD: whatever is not a matrix instruction has to be issued while one runs (16 cycles), so the reads and copies stand between
// them, a few after every third, and the steps have no branches: behind the end, the last stage is copied again.
template <int MB, bool TURNED, class Scale>
__device__ __forceinline__ void product_tile(const char* A, size_t aRow, const char* B, size_t bRow, int k0, int k1, char* lds, Acc<MB>& acc,
                                             const Scale& scale) {
    constexpr int UNITS = tile_units(MB), STAGES = tile_stages(MB), STAGE = UNITS * PAIR, MINE = UNITS / 4, COPIES = MINE * 2;
    constexpr int READS = 8 + 2 * MB, OPS = READS + COPIES, SLOTS = 4 * MB;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc.c[h][i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    int n = k1 - k0;
    if (n <= 0) return;
    // this wave's units: where they are read from, and how far that moves in a step
    const char* src[MINE];
    size_t adv[MINE];
#pragma unroll
    for (int i = 0; i < MINE; i++) {
        const int u = wave * MINE + i, w = u - 2 * MB;
        const bool isA = u < 2 * MB;
        src[i] = isA      ? A + (size_t)u * aRow + (size_t)k0 * PAIR
                 : TURNED ? B + (size_t)(2 * k0 + (w >> 2)) * bRow + (size_t)(w & 3) * PAIR
                          : B + (size_t)w * bRow + (size_t)k0 * PAIR;
        adv[i] = isA || !TURNED ? (size_t)PAIR : 2 * bRow;
        asm volatile("" : "+s"(src[i]), "+s"(adv[i]));  // (kept in registers, not computed again from the arguments in every step)
    }
    asm volatile("" : "+s"(n));
    const unsigned ldsBase = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)lds) + wave * MINE * PAIR;
    const unsigned laneOff = lane * 16;
    const int offA = wm * MB * PAIR + lane * 8;
    const int offB = (2 * MB + (TURNED ? wn * 2 : wn * 4)) * PAIR + (TURNED ? (lane & 3) * 128 + ((lane >> 4) * 4 + ((lane & 15) >> 2)) * 8 : lane * 8);
    auto read = [&](Frags<MB>& f, const char* s, int r) {  // the r-th of READS
        if (r < 8) {
            const int j = r & 3, q = r >> 2;
            if constexpr (TURNED) {
                const char* p = s + offB + (j >> 1) * PAIR + q * FRAG + (j & 1) * 512;
                f.b[j][q] = read_frag_turned(p, p + 4 * PAIR);
            } else {
                f.b[j][q] = read_frag(s + offB + j * PAIR + q * FRAG);
            }
        } else {
            const int i = (r - 8) >> 1, q = (r - 8) & 1;
            f.a[i][q] = read_frag(s + offA + i * PAIR + q * FRAG);
        }
    };
    int at = 0;                   // the stage that src points at
    auto move_source = [&] {
        if (__builtin_expect(scale.moves(at), 0)) {
            const size_t by = scale.move(at);
#pragma unroll
            for (int i = 0; i < MINE; i++) src[i] += by;
        }
    };
    move_source();
    unsigned fill = 0, take = 0;  // byte offsets of the buffers that are copied to, and read
    auto next_stage = [&] {
        const bool more = at < n - 1;
        at += more ? 1 : 0;
#pragma unroll
        for (int i = 0; i < MINE; i++) src[i] += more ? adv[i] : 0;
        if (more) move_source();
        fill = fill == (STAGES - 1) * STAGE ? 0 : fill + STAGE;
    };
    auto step = [&](int t, Frags<MB>& now, Frags<MB>& next) {
        wait_copies_and_meet<(STAGES - 2) * COPIES>();  // stage t + 1 has landed
        take = take == (STAGES - 1) * STAGE ? 0 : take + STAGE;
        const char* from = lds + take;
        scale(t, acc);
#pragma unroll
        for (int m = 0; m < 12 * MB; m++) {
            const int i = m / 12, k = m % 12 / 4, j = m % 4;
            f32x4& to = acc.c[k ? 1 : 0][i][j];
            to = __builtin_amdgcn_mfma_f32_16x16x32_f16(now.a[i][k == 2], now.b[j][k == 1], to, 0, 0, 0);
            if (m % 3 == 2) {
                const int slot = m / 3;
#pragma unroll
                for (int o = slot * OPS / SLOTS; o < (slot + 1) * OPS / SLOTS; o++) {
                    if (o < READS) read(next, from, o);
                    else copy_pair_half(src[(o - READS) >> 1], ldsBase + fill + ((o - READS) >> 1) * PAIR, laneOff, (o - READS) & 1);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        next_stage();
    };
#pragma unroll
    for (int t = 0; t < STAGES; t++) {
#pragma unroll
        for (int o = 0; o < COPIES; o++) copy_pair_half(src[o >> 1], ldsBase + fill + (o >> 1) * PAIR, laneOff, o & 1);
        next_stage();
    }
    wait_copies_and_meet<(STAGES - 1) * COPIES>();
    Frags<MB> f0, f1;
#pragma unroll
    for (int r = 0; r < READS; r++) read(f0, lds, r);
    int t = 0;
    for (; t + 1 < n; t += 2) {
        step(t, f0, f1);
        step(t + 1, f1, f0);
    }
    if (t < n) step(t, f0, f1);
    wait_copies_and_meet<0>();  // the buffers are free again
}

// The same product on 128 x 128 tiles with two blocks per CU: half the registers, so a stage's fragments are read in the step that
// multiplies them, and two stages of LDS.  For the logits, whose epilogue (an exponential per entry) takes as long as their products:
// one block's epilogue runs next to the other's products.
constexpr int SHARED_LDS = 2 * tile_units(4) * PAIR;
template <bool TURNED, class Scale>
__device__ __forceinline__ void product_tile_shared(const char* A, size_t aRow, const char* B, size_t bRow, int k0, int k1, char* lds, Acc<4>& acc,
                                                    const Scale& scale) {
    constexpr int UNITS = tile_units(4), STAGE = UNITS * PAIR, MINE = UNITS / 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
#pragma unroll
    for (int h = 0; h < 2; h++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc.c[h][i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    int n = k1 - k0;
    if (n <= 0) return;
    const char* src[MINE];
    size_t adv = wave < 2 || !TURNED ? (size_t)PAIR : 2 * bRow;  // (two waves copy A's units, two B's)
#pragma unroll
    for (int i = 0; i < MINE; i++) {
        const int u = wave * MINE + i, w = u - 8;
        src[i] = u < 8    ? A + (size_t)u * aRow + (size_t)k0 * PAIR
                 : TURNED ? B + (size_t)(2 * k0 + (w >> 2)) * bRow + (size_t)(w & 3) * PAIR
                          : B + (size_t)w * bRow + (size_t)k0 * PAIR;
        asm volatile("" : "+s"(src[i]));
    }
    asm volatile("" : "+s"(adv));
    asm volatile("" : "+s"(n));
    const unsigned ldsBase = __builtin_amdgcn_readfirstlane((unsigned)(unsigned long long)(__attribute__((address_space(3))) char*)lds) + wave * MINE * PAIR;
    const unsigned laneOff = lane * 16;
    const int offA = wm * 4 * PAIR + lane * 8;
    const int offB = (8 + (TURNED ? wn * 2 : wn * 4)) * PAIR + (TURNED ? (lane & 3) * 128 + ((lane >> 4) * 4 + ((lane & 15) >> 2)) * 8 : lane * 8);
    unsigned fill = 0, take = 0;
    auto move_source = [&](int t) {
        if (__builtin_expect(scale.moves(t), 0)) {
            const size_t by = scale.move(t);
#pragma unroll
            for (int i = 0; i < MINE; i++) src[i] += by;
        }
    };
    auto copy = [&](int t) {
        move_source(t);
#pragma unroll
        for (int o = 0; o < 2 * MINE; o++) copy_pair_half(src[o >> 1], ldsBase + fill + (o >> 1) * PAIR, laneOff, o & 1);
#pragma unroll
        for (int i = 0; i < MINE; i++) src[i] += adv;
        fill ^= STAGE;
    };
    copy(0);
    for (int t = 0; t < n; t++) {
        wait_copies_and_meet<0>();  // stage t has landed, and everyone has read the other buffer
        if (t + 1 < n) copy(t + 1);
        Frags<4> f;
        const char* s = lds + take;
        take ^= STAGE;
        auto readB = [&](int j, int q) {
            if constexpr (TURNED) {
                const char* p = s + offB + (j >> 1) * PAIR + q * FRAG + (j & 1) * 512;
                f.b[j][q] = read_frag_turned(p, p + 4 * PAIR);
            } else {
                f.b[j][q] = read_frag(s + offB + j * PAIR + q * FRAG);
            }
        };
        auto readA = [&](int i, int q) { f.a[i][q] = read_frag(s + offA + i * PAIR + q * FRAG); };
        readA(0, 0);
#pragma unroll
        for (int j = 0; j < 4; j++) readB(j, 0);
        readA(0, 1);
#pragma unroll
        for (int j = 0; j < 4; j++) readB(j, 1);
#pragma unroll
        for (int i = 1; i < 4; i++) {
            readA(i, 0);
            readA(i, 1);
        }
        scale(t, acc);
        // The wave that has its fragments goes before the other block's, which then reads under these products (512 x 100000 x 1024, both
        // calls, with the copies asked for before the reads and the reads in the products' order: 1.56 -> 1.50 ms).
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int m = 0; m < 48; m++) {
            const int i = m / 12, k = m % 12 / 4, j = m % 4;
            f32x4& to = acc.c[k ? 1 : 0][i][j];
            to = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.a[i][k == 2], f.b[j][k == 1], to, 0, 0, 0);
        }
        __builtin_amdgcn_s_setprio(0);
    }
    wait_copies_and_meet<0>();
}

// ---- packing
// What a pack launch makes, 512 threads a block: blocks below caseBlocks, 16 cases of x each (rows = cases, k = features) for the logits;
// the next featBlocks, 16 features of x each (rows = features, k = cases) for the weight gradient, in which a case without a label, or
// without a class left, is zero, whatever it holds; the others, 32 classes of the piece each (rows = classes, k = features).
struct PackArgs {
    const float *X, *labels, *stats;  // stats: for the features' blocks
    int *caseExp, *featExp;
    char *xByCase, *xByFeat;
    int D, V, N, Kd, Kn, caseBlocks, featBlocks;
    const float *W, *bias;  // of the piece
    int* classExp;
    char* wByClass;
    unsigned char* levels;  // backward: cleared by the classes' blocks
    int* anyLevel;
    int rows, Kv;
};

// Bound by memory: W is read once and written once, as two pieces of 16 bits (10575 x 512: 12.4 us, 3.5 TB/s; 100000 x 512, one call: 89 us,
// 4.6 TB/s).  Each block finds its rows' largest magnitudes first; what it reads then comes from its caches.
__device__ __forceinline__ void pack_cases(const PackArgs& p, int block, float* sh, int* exps) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4, n = block * 16 + c;
    float m = 0.f;
    bool odd = false;
    if (n < p.N) {
#pragma unroll 8
        for (int d = threadIdx.x >> 4; d < p.D; d += 32) max_finite(m, odd, fabsf(p.X[(size_t)d * p.N + n]));
    }
    float any = odd ? 1.f : 0.f;
    for (int o = 16; o < 64; o <<= 1) {
        m = fmaxf(m, __shfl_xor(m, o, 64));
        any = fmaxf(any, __shfl_xor(any, o, 64));
    }
    sh[wave * 16 + c] = m;
    sh[128 + wave * 16 + c] = any;
    __syncthreads();
    if (threadIdx.x < 16) {
        for (int w = 1; w < 8; w++) {
            m = fmaxf(m, sh[w * 16 + c]);
            any = fmaxf(any, sh[128 + w * 16 + c]);
        }
        exps[c] = scale_exp(m);
        p.caseExp[n] = exp_odd(exps[c], any != 0.f);
    }
    __syncthreads();
    const int e = exps[c];
    for (int kb = wave; kb < p.Kd; kb += 8) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int d = kb * 32 + (j >> 2) * 16 + g * 4 + (j & 3);
            y[j] = n < p.N && d < p.D ? ldexpf(p.X[(size_t)d * p.N + n], e) : 0.f;
        }
        store_pair(p.xByCase + ((size_t)block * p.Kd + kb) * PAIR, lane, y);
    }
}

// (not without a label, and not without a class left)
__device__ __forceinline__ bool has_gradient(const PackArgs& p, int n) {
    int label;
    return label_of(p.labels[n], p.V, label) && p.stats[p.N + n] != 0.f;
}
__device__ __forceinline__ void pack_feats(const PackArgs& p, int block, int* exps) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4, d0 = block * 16, r = threadIdx.x >> 5;
    float m = 0.f;
    bool odd = false;
    if (d0 + r < p.D) {
#pragma unroll 4
        for (int n = threadIdx.x & 31; n < p.N; n += 32) {
            const float v = fabsf(p.X[(size_t)(d0 + r) * p.N + n]);
            if (has_gradient(p, n)) max_finite(m, odd, v);
        }
    }
    for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    if ((threadIdx.x & 31) == 0) p.featExp[d0 + r] = exps[r] = scale_exp(m);
    __syncthreads();
    const int d = d0 + c, e = exps[c];
    for (int kb = wave; kb < p.Kn; kb += 8) {
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int n = kb * 32 + (j >> 2) * 16 + g * 4 + (j & 3);
            y[j] = d < p.D && n < p.N && has_gradient(p, n) ? ldexpf(p.X[(size_t)d * p.N + n], e) : 0.f;
        }
        store_pair(p.xByFeat + ((size_t)block * p.Kn + kb) * PAIR, lane, y);
    }
}

// 32 classes with one scale, a power of 2^8: their largest magnitude comes to [2^7, 2^15), and neighbouring groups mostly share it
// (CarryScale).  A class that a bias of -inf takes out is zero, whatever its weights hold.  512 features at a time go through registers
// (all of a thread's loads in flight at once) and LDS; rows of at most 512 features are read once, longer ones a second time for their
// max.
constexpr int CW = 512, CW_LD = CW + 4;
constexpr int PACK_LDS = (32 * CW_LD + 16) * 4;
__device__ __forceinline__ void pack_classes(const PackArgs& p, int block, float* tile) {
    float* maxima = tile + 32 * CW_LD;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, v0 = block * 32, c = lane & 15, g = lane >> 4, D = p.D;
    bool live[4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
        const int v = v0 + wave * 4 + r;
        live[r] = v < p.rows && (!p.bias || p.bias[v] != -INFINITY);
    }
    f32x4 t[4][2];
    auto load = [&](int d0) {  // a wave: rows 4 wave .. + 3, a lane: features d0 + 4 lane .. and 256 further on
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int d = d0 + h * 256 + lane * 4;
                const float* src = p.W + (size_t)(v0 + wave * 4 + r) * D + d;
                f32x4 x = {0.f, 0.f, 0.f, 0.f};
                if (live[r]) {
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
    float m = 0.f, zero = 0.f;  // zero: a NaN once an infinity or NaN has been met
    for (int d0 = 0; d0 < D; d0 += CW) {
        load(d0);
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    m = fmaxf(m, fabsf(t[r][h][j]));
                    zero = fmaf(t[r][h][j], 0.f, zero);
                }
    }
    for (int o = 1; o < 64; o <<= 1) {
        m = fmaxf(m, __shfl_xor(m, o, 64));
        zero += __shfl_xor(zero, o, 64);
    }
    if (lane == 0) {
        maxima[wave] = m;
        maxima[8 + wave] = zero;
    }
    int e = 0;
    for (int d0 = 0; d0 < p.Kd * 32; d0 += CW) {
        if (D > CW) load(d0);
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int h = 0; h < 2; h++) *reinterpret_cast<f32x4*>(tile + (wave * 4 + r) * CW_LD + h * 256 + lane * 4) = t[r][h];
        if (d0 == 0) {
            for (int w = 0; w < 8; w++) {  // (every wave: the barrier above covers the maxima)
                m = fmaxf(m, maxima[w]);
                zero += maxima[8 + w];
            }
            const bool odd = zero != zero;  // the same for all threads
            if (odd) {                      // the finite ones' maximum; the first features are in the tile already
                m = 0.f;
                bool met = false;
                for (int d = 0; d < D; d += CW) {
                    load(d);
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int j = 0; j < 4; j++) max_finite(m, met, fabsf(t[r][h][j]));
                }
                for (int o = 1; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
                __syncthreads();
                if (lane == 0) maxima[wave] = m;
                __syncthreads();
                for (int w = 0; w < 8; w++) m = fmaxf(m, maxima[w]);
            }
            e = scale_exp(m) & ~7;
            if (threadIdx.x == 0) p.classExp[block] = exp_odd(m == 0.f ? EXP_ZERO : e, odd);
        }
        __syncthreads();
        for (int f = wave; f < 2 * CW / 32; f += 8) {
            const int rb = f & 1, kb = d0 / 32 + (f >> 1), r = rb * 16 + c;
            if (kb >= p.Kd) break;
            float y[8];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(tile + r * CW_LD + (f >> 1) * 32 + h * 16 + g * 4);
#pragma unroll
                for (int j = 0; j < 4; j++) y[4 * h + j] = ldexpf(x[j], e);
            }
            store_pair(p.wByClass + (((size_t)block * 2 + rb) * p.Kd + kb) * PAIR, lane, y);
        }
    }
}

__global__ __launch_bounds__(512) void k_fcl_pack(PackArgs p) {
    extern __shared__ __attribute__((aligned(16))) float tile[];  // [32][CW_LD], then the waves' maxima
    __shared__ int exps[16];
    const int b = blockIdx.x;
    if (b < p.caseBlocks) pack_cases(p, b, tile, exps);
    else if (b < p.caseBlocks + p.featBlocks) pack_feats(p, b - p.caseBlocks, exps);
    else {
        const int block = b - p.caseBlocks - p.featBlocks;
        if (p.levels) {
            for (int i = threadIdx.x; i < p.Kn / 2 * 8; i += 512) reinterpret_cast<unsigned*>(p.levels + ((size_t)(i >> 3) * p.Kv + block) * 32)[i & 7] = 0;
            if (block == 0 && threadIdx.x == 0) *p.anyLevel = 0;
        }
        pack_classes(p, block, tile);
    }
}

// ---- logits of a piece
struct WideArgs {
    const char *wByClass, *xByCase;
    const int *classExp, *caseExp;
    const float *bias, *labels, *stats;
    int V, N, v0, rows, Kd, kSteps, vTiles, nTiles;
    float *part, *labelLogits;  // forward: part + the piece's first tile
    char* dz;                   // backward: dz / coeff, (rows = cases, k = classes)
    float* dbPart;              // backward: [nTiles][V], row sums of dz / coeff
    int Kv;
    size_t near;                // backward: dz of 32 classes x 64 cases with a level is there once more, this far behind, without
    unsigned char* levels;      // backward: [Np / 64][32 Kv], zeros
    int* anyLevel;              // backward: whether there are any, zero
    const float *W, *X;
    int D;
};

// Logits whose weights or inputs hold an infinity or NaN: the products of pieces make a NaN of any of them, where the formula has the sum
// of the terms that are not finite (all of one sign: that infinity).  Where an infinite input meets the zeros of a class that is taken
// out, too.  Rare: a lane's entries lie in LDS, 256 floats apart; a lane looks for such operands at one of 64 features, and the features that
// have some are gone through one by one.
typedef const __attribute__((address_space(4))) WideArgs* LateArgs;
template <int MB>
__device__ __forceinline__ void odd_logits(LateArgs p, float* z, int vBase, int nBase, int lane) {
    constexpr unsigned NOTHING_YET = 0x7FC0BEEFu;  // (a NaN, which it stays if no term turns up)
    const int vFirst = vBase + (lane >> 4) * 4, nFirst = nBase + (lane & 15), D = p->D, N = p->N, rows = p->rows;
    const float *W = p->W + (size_t)p->v0 * D, *X = p->X, *bias = p->bias ? p->bias + p->v0 : nullptr;
    auto class_of = [&](int e) { return vFirst + (e >> 4) * 16 + (e & 3); };
    auto case_of = [&](int e) { return nFirst + ((e >> 2) & 3) * 16; };
    auto bias_of = [&](int v) { return v < rows ? (bias ? bias[v] : 0.f) : -INFINITY; };
#pragma unroll 1
    for (int e = 0; e < 16 * MB; e++) {
        const float was = z[e * 256];
        if (bias_of(class_of(e)) == -INFINITY) z[e * 256] = -INFINITY;
        else if (case_of(e) < N && was != was) z[e * 256] = __uint_as_float(NOTHING_YET);
    }
#pragma unroll 1
    for (int d0 = 0; d0 < D; d0 += 64) {
        float none = 0.f;  // a NaN once there is one
        if (d0 + lane < D) {
#pragma unroll 8
            for (int v = vBase; v < min(rows, vBase + 16 * MB); v++) none = fmaf(W[(size_t)v * D + d0 + lane], 0.f, none);
#pragma unroll 8
            for (int n = nBase; n < min(N, nBase + 64); n++) none = fmaf(X[(size_t)(d0 + lane) * N + n], 0.f, none);
        }
        unsigned long long odd = __ballot(none != 0.f);
        for (; odd; odd &= odd - 1) {
            const int d = d0 + __builtin_ctzll(odd);
            bool open = false;  // whether a further term can change anything: not where there is a NaN
#pragma unroll 1
            for (int e = 0; e < 16 * MB; e++) {
                const int v = class_of(e), n = case_of(e);
                const float b = bias_of(v);
                if (n >= N || b == -INFINITY) continue;
                const float w = W[(size_t)v * D + d], x = X[(size_t)d * N + n];
                float sum = z[e * 256];
                if (!(fabsf(w) < INFINITY && fabsf(x) < INFINITY)) {
                    sum = __float_as_uint(sum) == NOTHING_YET ? w * x + b : sum + w * x;
                    z[e * 256] = sum;
                }
                open |= __float_as_uint(sum) == NOTHING_YET || fabsf(sum) == INFINITY;
            }
            if (!__any(open)) return;
        }
    }
}

// SHARED: two blocks per CU (MB = 4).  512 x 100000 x 1024: forward 328 us, 959 TFLOP/s of fp16 products, backward, which writes dz,
// 387 us, 813; a large library product of fp16 operands reaches 1126.
template <int MB, bool BWD, bool SHARED>
__global__ __launch_bounds__(256, SHARED ? 2 : 1) void k_fcl_logits(WideArgs p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    // the tiles of one block of classes on one XCD: they read the same rows of W
    int tv, tn;
    mcn_xcd_group(blockIdx.x, p.nTiles, p.vTiles, tv, tn);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    const int c = lane & 15, g = lane >> 4;
    const size_t row = (size_t)p.Kd * PAIR;
    Acc<MB> acc;
    if constexpr (SHARED)
        product_tile_shared<false>(p.wByClass + (size_t)tv * 2 * MB * row, row, p.xByCase + (size_t)tn * 8 * row, row, 0, p.kSteps, lds, acc, NoScale());
    else
        product_tile<MB, false>(p.wByClass + (size_t)tv * 2 * MB * row, row, p.xByCase + (size_t)tn * 8 * row, row, 0, p.kSteps, lds, acc, NoScale());
    const int vBase = tv * 32 * MB + wm * 16 * MB, nBase = tn * TILE + wn * 64;
    // z in place of the first accumulator.  A class behind the last one, or taken out by its bias, has fragments of zeros: -inf.
    int ex[4], label[4];
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int n = nBase + j * 16 + c;
        const int eo = p.caseExp[n];
        ex[j] = exp_of(eo);
        odd |= is_odd(eo);
        label[j] = -1;
        if (n < p.N) label_of(p.labels[n], p.V, label[j]);
    }
#pragma unroll
    for (int i = 0; i < MB; i++) {
        const int eo = p.classExp[(vBase + i * 16) / 32], we = exp_of(eo), ew = we == EXP_ZERO ? 0 : we;
        odd |= is_odd(eo);
        float bv[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int v = vBase + i * 16 + g * 4 + r;
            bv[r] = v < p.rows ? (p.bias ? p.bias[p.v0 + v] : 0.f) : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) acc.c[0][i][j][r] = ldexpf(acc.value(i, j, r), -(ew + ex[j])) + bv[r];
    }
    if (__builtin_expect(__any(odd), 0)) {  // (the stages' LDS is free)
        static_assert(16 * MB * 256 * 4 <= (SHARED ? SHARED_LDS : tile_lds(MB)), "the tile's logits in the stages' LDS");
        float* mine = reinterpret_cast<float*>(lds) + threadIdx.x;
#pragma unroll
        for (int k = 0; k < 16 * MB; k++) mine[k * 256] = acc.c[0][k >> 4][(k >> 2) & 3][k & 3];
        // arguments that only this branch needs are loaded in it: with their loads moved to the front 512 x 10575, 509 cases, took 28.5 us for 24.1
        LateArgs late = (LateArgs)__builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(late));
        odd_logits<MB>(late, mine, vBase, nBase, lane);
#pragma unroll
        for (int k = 0; k < 16 * MB; k++) acc.c[0][k >> 4][(k >> 2) & 3][k & 3] = mine[k * 256];
    }
    // where the label's entry lies among a lane's 4 MB rows, if it does: row 16 i + r from here
    int at[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        at[j] = label[j] - (p.v0 + vBase + g * 4);
        if (label[j] < 0 || at[j] < 0 || at[j] >= 16 * MB || (at[j] & 15) > 3) at[j] = -1;
    }
    if constexpr (!BWD) {
        __syncthreads();
        float(*red)[3][64] = reinterpret_cast<float(*)[3][64]>(lds);  // [wave][max, rest, count][64 cases]
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int r = 0; r < 4; r += 2) m = fmaxf(fmaxf(acc.c[0][i][j][r], acc.c[0][i][j][r + 1]), m);
            if (__any(at[j] >= 0)) {
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
                        if (at[j] == i * 16 + r) p.labelLogits[nBase + j * 16 + c] = acc.c[0][i][j][r];
            }
            for (int o = 16; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
            const float from = m == -INFINITY ? 0.f : m;
            float rest = 0.f;
            int tops = 0;
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float x = acc.c[0][i][j][r] - from;
                    const bool top = x == 0.f && m != -INFINITY;
                    const float e = exp_neg(x);
                    rest += top ? 0.f : e;
                    tops += top ? 1 : 0;
                }
            float cnt = (float)tops;
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
        float sums[MB][4] = {};
        auto largest = [&](int i, int r) {
            return fmaxf(fmaxf(fmaxf(fabsf(acc.c[0][i][0][r]), fabsf(acc.c[0][i][1][r])), fabsf(acc.c[0][i][2][r])), fabsf(acc.c[0][i][3][r]));
        };
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int n = nBase + j * 16 + c;
            float M = 0.f, S = 0.f;
            if (label[j] >= 0) {
                M = p.stats[n];
                S = p.stats[p.N + n];
            }
            const bool counts = S != 0.f;  // (no label, or no class left: nothing; a NaN goes on)
            const float inv = counts ? 1.f / S : 0.f;
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float t = -exp_neg(acc.c[0][i][j][r] - M) * inv;
                    acc.c[0][i][j][r] = counts ? t : 0.f;
                }
            if (__any(at[j] >= 0 && counts)) {
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc.c[0][i][j][r] += counts && at[j] == i * 16 + r ? 1.f : 0.f;
            }
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) sums[i][r] += acc.c[0][i][j][r];
        }
        auto store = [&](char* to, int i, int j, auto scale) {  // rows 16 i .. + 15, cases 16 j .. + 15
            f16x4 hi, lo;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float y = acc.c[0][i][j][r] * scale(r);
                hi[r] = (_Float16)y;
                lo[r] = (_Float16)((y - (float)hi[r]) * LO);
            }
            *reinterpret_cast<f16x4*>(to + (i >> 1) * PAIR + (i & 1) * 512) = hi;
            *reinterpret_cast<f16x4*>(to + (i >> 1) * PAIR + FRAG + (i & 1) * 512) = lo;
        };
        auto plain = [](int) { return (float)(1 << DZ_EXP); };
        // The classes that are far from this wave's cases are looked for where the sum of what a lane holds of one is small.  Its entries are
        // -p, or 1 - p, which is no number between 0 and 2^-24: the sum is below 0 then, and a zero is no sign of it.
        unsigned least = ~0u;
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) least = min(least, __float_as_uint(sums[i][r]) - 0x80000001u);
        if (__builtin_expect(__any(least < __float_as_uint(4 * FAR) - 1), 0)) {
            LateArgs late = (LateArgs)__builtin_amdgcn_kernarg_segment_ptr();
            asm volatile("" : "+s"(late));
            unsigned char* levels = late->levels + (size_t)(nBase / 64) * late->Kv * 32 + vBase + g * 4;
#pragma unroll
            for (int q = 0; q < MB / 2; q++) {
                unsigned packed[2] = {};
                float scale[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int level = level_of(row_max(largest(2 * q + h, r)));
                        packed[h] |= level << 8 * r;
                        scale[h][r] = level_scale(level);
                    }
                const bool any = __any(packed[0] | packed[1]);
                if (any) {
                    if (c < 2) *reinterpret_cast<unsigned*>(levels + (2 * q + c) * 16) = c == 0 ? packed[0] : packed[1];
                    if (lane == 0) *late->anyLevel = 1;
                }
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    char* out = late->dz + ((size_t)(nBase / 16 + j) * late->Kv + vBase / 32) * PAIR + lane * 8;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        store(out, 2 * q + h, j, [&](int r) { return scale[h][r]; });
                        if (any) store(out + late->near, 2 * q + h, j, plain);
                    }
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                char* out = p.dz + ((size_t)(nBase / 16 + j) * p.Kv + vBase / 32) * PAIR + lane * 8;
#pragma unroll
                for (int i = 0; i < MB; i++) store(out, i, j, plain);
            }
        }
        if (p.dbPart) {  // row sums: over the lanes of a row, then the two waves of 64 cases
            __syncthreads();
            float(*rowSum)[32 * MB] = reinterpret_cast<float(*)[32 * MB]>(lds);
#pragma unroll
            for (int i = 0; i < MB; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    float t = sums[i][r];
                    for (int o = 1; o < 16; o <<= 1) t += __shfl_xor(t, o, 64);
                    if (c == 0) rowSum[wn][wm * 16 * MB + i * 16 + g * 4 + r] = t;
                }
            __syncthreads();
            const int t = threadIdx.x, v = tv * 32 * MB + t;
            if (t < 32 * MB && v < p.rows) p.dbPart[(size_t)tn * p.V + p.v0 + v] = rowSum[0][t] + rowSum[1][t];
        }
    }
}

struct GradArgs {
    const char *xByFeat, *dz, *wByClass;
    const int *featExp, *classExp;
    float *dW, *slabs;
    int D, rows, Kn, Kv, Kd, Np, Dp, nTiles, dTiles, kPerSplit, first;
    int inputBlocks;  // blocks of the input gradient, then those of the weight gradient
    float scaleTargets, scaleOutput;
    const unsigned char* levels;
    const int* anyLevel;
    size_t near;
    int allNear;  // few cases: all of dz is there twice
};

template <bool SHARED, class Scale>
__device__ __forceinline__ void turned_tile(const char* A, size_t aRow, const char* B, size_t bRow, int k0, int k1, char* lds, Acc<4>& acc,
                                            const Scale& scale) {
    if constexpr (SHARED) product_tile_shared<true>(A, aRow, B, bRow, k0, k1, lds, acc, scale);
    else product_tile<4, true>(A, aRow, B, bRow, k0, k1, lds, acc, scale);
}

// The weight gradient's accumulators are in units of 2^-(14 + level_exp) of the class they add for: where its level changes from 64 cases to
// the next they are brought to it, exactly.  |sum| < 2^49 at any level, so 2^74 takes none out of range.
struct CarryLevels {
    const unsigned char* levels;  // of this wave's 64 classes
    size_t row;
    int halves;
    mutable int next;              // the step that has something to do: a change, or 64 x 64 cases further on
    mutable unsigned long long far;  // a bit for each 64 cases: whether any class has a level
    mutable unsigned cur;          // a byte for each of a lane's four classes
    __device__ __forceinline__ CarryLevels(const unsigned char* l, size_t r, int n, bool any) : levels(l), row(r), halves(n), next(any ? 0 : -1), far(0), cur(0) {}
    __device__ __forceinline__ bool moves(int) const { return false; }
    __device__ __forceinline__ size_t move(int) const { return 0; }
    template <int MB>
    __device__ __forceinline__ void operator()(int t, Acc<MB>& acc) const {
        if (__builtin_expect(t != next, 1)) return;
        const int h = t >> 1, b = h & 63;
        if (b == 0) {
            const int i = h + (int)(threadIdx.x & 63);
            unsigned any = 0;
            if (i < halves) {
                const uint4* p = reinterpret_cast<const uint4*>(levels + i * row);
                const uint4 q = p[0], r = p[1], s = p[2], u = p[3];
                any = q.x | q.y | q.z | q.w | r.x | r.y | r.z | r.w | s.x | s.y | s.z | s.w | u.x | u.y | u.z | u.w;
            }
            far = __ballot(any != 0);
        }
        unsigned now = 0;
        if (far >> b & 1) {
#pragma unroll
            for (int j = 0; j < 4; j++) now |= (unsigned)levels[h * row + j * 16 + (threadIdx.x & 15)] << 8 * j;
        }
        bring(now, acc);
        const unsigned long long later = b == 63 ? 0 : ((far | far << 1) >> (b + 1)) << (b + 1);  // cases with levels, and the ones behind them
        next = 2 * (later ? h - b + __builtin_ctzll(later) : h - b + 64);
    }
    template <int MB>
    __device__ __forceinline__ void bring(unsigned now, Acc<MB>& acc) const {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int up = level_exp(now >> 8 * j & 255) - level_exp(cur >> 8 * j & 255);
            if (!__any(up != 0)) continue;
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) acc.c[k][i][j][r] = ldexpf(acc.c[k][i][j][r], up);
        }
        cur = now;
    }
    template <int MB>
    __device__ __forceinline__ void end(Acc<MB>& acc) const {  // no level
        if (__builtin_expect(__any(cur != 0), 0)) bring(0, acc);
    }
};

// weight gradient: (features x classes) tiles, so that a lane's four rows are four neighbours of one row of W
template <bool SHARED>
__device__ __forceinline__ void weight_tile(const GradArgs& p, int L, char* lds) {
    int tv, td;
    mcn_xcd_group(L, p.dTiles, p.Kv / 4, tv, td);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    const int c = lane & 15, g = lane >> 4;
    const size_t row = (size_t)p.Kn * PAIR;
    Acc<4> acc;
    const CarryLevels carry(p.levels + tv * TILE + wn * 64, (size_t)p.Kv * 32, p.Kn / 2, __builtin_amdgcn_readfirstlane(*p.anyLevel) != 0);
    turned_tile<SHARED>(p.xByFeat + (size_t)td * 8 * row, row, p.dz + (size_t)tv * 4 * PAIR, (size_t)p.Kv * PAIR, 0, p.Kn, lds, acc, carry);
    carry.end(acc);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int d = td * TILE + wm * 64 + i * 16 + g * 4;
        int e[4];
#pragma unroll
        for (int r = 0; r < 4; r++) e[r] = -(p.featExp[d + r] + DZ_EXP);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int v = tv * TILE + wn * 64 + j * 16 + c;
            if (v >= p.rows) continue;
            float* out = p.dW + (size_t)v * p.D + d;
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = p.scaleOutput * ldexpf(acc.value(i, j, r), e[r]);
            if (d + 4 <= p.D) {
                f32x4u t = {y[0], y[1], y[2], y[3]};
                if (p.scaleTargets != 0.f) {
                    const f32x4u old = *reinterpret_cast<const f32x4u*>(out);
#pragma unroll
                    for (int r = 0; r < 4; r++) t[r] += p.scaleTargets * old[r];
                }
                *reinterpret_cast<f32x4u*>(out) = t;
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (d + r < p.D) out[r] = (p.scaleTargets != 0.f ? p.scaleTargets * out[r] : 0.f) + y[r];
            }
        }
    }
}

// The accumulators are in units of 2^-(exponent of the group they last added): when the next 32 classes have another scale, they are
// brought to it, exactly, by a power of two.  A group of zeros has none.  |sum| < 2^30 in the units of its largest weights (the dz / coeff
// of a case add up to 2 at most); where a group's are more than 2^80 times smaller, or larger, the sum goes to the slab and begins anew, so
// that it stays in range whatever the weights.  Exponents come 64 at a time into a register of the lanes.
// Here every class's dz is wanted at the one scale: the waves that copy it take 32 classes with levels from behind.
struct CarryScale {
    f32x4* out;       // of the slab: this lane's four cases of row block 0 and column block 0
    size_t column;    // entries from one feature to the next
    mutable bool fresh;  // there is nothing in the slab yet
    const int* exps;  // of the product's k blocks, from k0 on
    int count;
    const unsigned char* levels;  // of the 64 cases that this wave copies, or NULL
    size_t near;
    mutable int held, cur, low;      // low: the smallest since the sum began
    mutable int next;                // the step from which it copies from the other place, or 64 further on
    mutable unsigned long long far;  // a bit for each k block
    mutable bool there;
    __device__ __forceinline__ CarryScale(float* o, size_t c, bool f, const int* e, int n, const unsigned char* l, size_t d)
        : out(reinterpret_cast<f32x4*>(o)), column(c / 4), fresh(f), exps(e), count(n), levels(l), near(d), held(load(0)), cur(EXP_ZERO), low(0),
          next(l ? 0 : -1), far(0), there(false) {}
    template <int MB>
    __device__ __forceinline__ void put(const Acc<MB>& acc) const {
        const int e = cur == EXP_ZERO ? 0 : -(cur + DZ_EXP);
#pragma unroll
        for (int i = 0; i < MB; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                f32x4* to = out + j * 16 * column + i * 4;
                f32x4 y;
#pragma unroll
                for (int r = 0; r < 4; r++) y[r] = ldexpf(acc.value(i, j, r), e);
                *to = fresh ? y : *to + y;
            }
        fresh = false;
    }
    __device__ __forceinline__ bool moves(int t) const { return t == next; }
    __device__ __forceinline__ size_t move(int t) const {
        const int b = t & 63;
        if (b == 0) {
            const int i = t + (int)(threadIdx.x & 63);
            unsigned any = 0;
            if (i < count) {
                const uint4* p = reinterpret_cast<const uint4*>(levels + (size_t)i * 32);
                const uint4 q = p[0], r = p[1];
                any = q.x | q.y | q.z | q.w | r.x | r.y | r.z | r.w;
            }
            far = __ballot(any != 0);
        }
        const bool now = far >> b & 1, was = there;
        there = now;
        const unsigned long long later = (now ? ~far : far) >> b;  // (its lowest bit is not set)
        next = later ? t + __builtin_ctzll(later) : t - b + 64;
        return (now ? near : 0) - (was ? near : 0);
    }
    __device__ __forceinline__ int load(int t) const {
        const int i = t + (int)(threadIdx.x & 63);
        return i < count ? exp_of(exps[i]) : EXP_ZERO;
    }
    template <int MB>
    __device__ __forceinline__ void operator()(int t, Acc<MB>& acc) const {
        if (t > 0 && (t & 63) == 0) held = load(t);
        const int e = __builtin_amdgcn_readlane(held, t & 63);
        if (e == EXP_ZERO || e == cur) return;
        if (cur == EXP_ZERO) {
            low = e;
        } else {
            const bool anew = e - low > 80 || e - cur < -80;
            if (__builtin_expect(anew, 0)) put(acc);
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < MB; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++) acc.c[h][i][j][r] = anew ? 0.f : ldexpf(acc.c[h][i][j][r], e - cur);
            low = anew ? e : min(low, e);
        }
        cur = e;
    }
};

// input gradient: the sum over the classes is split; slab s of (Dp, Np) adds up its share of every piece, in order
template <bool SHARED>
__device__ __forceinline__ void input_tile(const GradArgs& p, int L, char* lds) {
    // the tiles of one split on one XCD: they read the same classes of dz and W
    int s, t;
    mcn_xcd_group(L, p.nTiles * p.dTiles, p.inputBlocks / (p.nTiles * p.dTiles), s, t);
    const int td = t / p.nTiles, tn = t % p.nTiles;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
    const int c = lane & 15, g = lane >> 4;
    const size_t row = (size_t)p.Kv * PAIR;
    const int k0 = s * p.kPerSplit, k1 = min(p.Kv, k0 + p.kPerSplit);
    Acc<4> acc;
    const unsigned char* levels = wave < 2 && !p.allNear && __builtin_amdgcn_readfirstlane(*p.anyLevel) ? p.levels + ((size_t)(tn * 2 + wave) * p.Kv + k0) * 32 : nullptr;
    float* out = p.slabs + ((size_t)s * p.Dp + td * TILE + wn * 64 + c) * p.Np + tn * TILE + wm * 64 + g * 4;
    const CarryScale carry(out, p.Np, p.first, p.classExp + k0, k1 - k0, levels, p.near);
    turned_tile<SHARED>(p.dz + (p.allNear ? p.near : 0) + (size_t)tn * 8 * row, row, p.wByClass + (size_t)td * 4 * PAIR, (size_t)p.Kd * PAIR, k0, k1, lds, acc, carry);
    carry.put(acc);
}

// ---- both gradients of a piece in one launch: they wait for the same logits and not for each other.  512 x 100000 x 1024: 568 us, 1108
// TFLOP/s of fp16 products; 512 x 10575 x 128: 16.3 us.
template <bool SHARED>
__global__ __launch_bounds__(256, SHARED ? 2 : 1) void k_fcl_grads(GradArgs p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if ((int)blockIdx.x < p.inputBlocks) input_tile<SHARED>(p, blockIdx.x, lds);
    else weight_tile<SHARED>(p, blockIdx.x - p.inputBlocks, lds);
}

// ---- the end: input gradients from the slabs (blocks below dxBlocks), bias gradients from the tiles' row sums.  A case that does not count,
// or has no class left, gets zero whatever the weights hold (its dz is zero, but 0 times an infinity or NaN is not).  The packed weights of
// a class that its bias takes out are zero; a case that has such a class for its label, and others left, still has the formula's
// weights[label] * 1, and gets it here.
struct FinishArgs {
    const float *slabs, *dbPart, *W, *bias, *labels, *stats;
    float *dX, *dB;
    int D, V, N, Np, Dp, splits, nTiles, dxBlocks;
    float coeff, scaleInputTargets, scaleBiasTargets, scaleBiasOutput;
};
__global__ __launch_bounds__(256) void k_fcl_finish(FinishArgs p) {
    if ((int)blockIdx.x < p.dxBlocks) {
        for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < (size_t)p.D * p.N; i += (size_t)p.dxBlocks * 256) {
            const size_t d = i / p.N, n = i % p.N;
            float v = 0.f;
#pragma unroll 8
            for (int s = 0; s < p.splits; s++) v += p.slabs[((size_t)s * p.Dp + d) * p.Np + n];
            int label;
            if (!label_of(p.labels[n], p.V, label) || p.stats[p.N + n] == 0.f) v = 0.f;
            else if (p.bias && p.bias[label] == -INFINITY) v += p.W[(size_t)label * p.D + d];
            p.dX[i] = (p.scaleInputTargets != 0.f ? p.scaleInputTargets * p.dX[i] : 0.f) + p.coeff * v;
        }
        return;
    }
    const int v = (blockIdx.x - p.dxBlocks) * 256 + threadIdx.x;
    if (v >= p.V) return;
    float s = 0.f;
#pragma unroll 8
    for (int t = 0; t < p.nTiles; t++) s += p.dbPart[(size_t)t * p.V + v];
    p.dB[v] = (p.scaleBiasTargets != 0.f ? p.scaleBiasTargets * p.dB[v] : 0.f) + p.scaleBiasOutput * p.coeff * s;
}

// Which tile a product takes: SHARED 128 x 128, two blocks per CU; WHOLE 128 x 128 or HALF 64 x 128, one block per CU with its stages
// further ahead.  A launch runs in rounds of 512 or 256 blocks, and a tile costs its rows / 32 (twice that for two sharing a CU) and a
// fixed part, the fill of its stages and its epilogue, of about one more.  512 x 100000 x 1024: SHARED logits 330 us, WHOLE tiles of
// twice the rows 390 us; 512 x 10575 x 128, 83 row tiles: logits HALF 13 us, SHARED 25 us.
enum TileKind { SHARED, WHOLE, HALF };
TileKind tile_choice(int rows32, int colTiles) {
    const long whole = (long)divup(rows32, 4) * colTiles, half = (long)divup(rows32, 2) * colTiles;
    const long cost[3] = {(whole + 511) / 512 * 9, (whole + 255) / 256 * 5, (half + 255) / 256 * 3};
    return cost[HALF] < cost[WHOLE] && cost[HALF] < cost[SHARED] ? HALF : cost[WHOLE] < cost[SHARED] ? WHOLE : SHARED;
}
int tile_rows32(TileKind k) { return k == HALF ? 2 : 4; }
int tile_bytes(TileKind k) { return k == SHARED ? SHARED_LDS : tile_lds(tile_rows32(k)); }

// Sizes and workspace of the wide path: a function of the shape alone.
struct WidePlan {
    int Np, Dp, Kd, kSteps, Kn, nTiles, dTiles;  // Kd: k blocks of W's and x's fragments, padded; kSteps: those that hold anything
    int rows, last;                              // classes per piece, and of the last one, which takes a short rest with it
    int Kv;                                      // k blocks of the first piece, padded
    int kPerSplit, splits;                       // input gradient: every split of a whole piece holds something, so that the first piece
                                                 // writes every slab
    size_t classExp, caseExp, featExp, xByCase, xByFeat, wByClass, dz, dzNear, levels, anyLevel, dbPart, slabs, part, labelLogits, total;
};
// When the packed operands pay for the logits (us of a whole cost call, narrow / wide).  512 x 10575: 16 cases 16 / 34, 64 cases 26 / 35;
// 512 x 100000: 56 / 145, 121 / 147.  Both calls go by the number of cases alone: the gradients' logits are the cost's, to the bit.
// The other products of the gradients always take them (512 x 10575: one case 50 us, 16 cases 43 us, 64 cases 51 us).
bool wide_cost_usable(int N) { return N > NARROW; }

size_t al256(size_t b) { return (b + 255) / 256 * 256; }

WidePlan wide_plan(int D, int V, int N, bool bwd) {
    WidePlan p = {};
    p.nTiles = divup(N, TILE);
    p.dTiles = divup(D, TILE);
    p.kSteps = divup(D, 32);
    p.Kd = p.dTiles * 4;
    p.Np = p.nTiles * TILE;
    p.Dp = p.dTiles * TILE;
    p.Kn = p.Np / 32;
    // a piece's fragments should stay in the 256 MB last-level cache between the launches that write and read them; whole rounds of
    // shared tiles where the classes fill some; a rest of at most a quarter goes with the last piece (with it / a piece of its own, ms:
    // 512 x 100000 x 1024 1.44 / 1.46, 160 x 100000 x 1024 0.81 / 0.82, cost of 2048 x 100000 x 256 0.80 / 0.83, 512 x 100000 x 512 0.88 / 0.87)
    const size_t perRow = (size_t)p.Kd * 128 + (bwd ? (size_t)p.Np * 4 : 0);
    const int most = (int)std::max<size_t>(TILE, std::min<size_t>(((size_t)PIECE_MB << 20) / perRow / TILE * TILE, (size_t)1 << 17));
    const int round = std::max(1, 512 / p.nTiles) * TILE;
    p.rows = std::min(V, most > round ? most / round * round : most);
    const int rest = V % p.rows;
    p.last = rest == 0 ? p.rows : rest <= p.rows / 4 ? p.rows + rest : rest;
    p.rows = std::min(V, V <= p.last ? p.last : p.rows);
    p.Kv = divup(p.rows, TILE) * 4;
    const size_t mostKv = (size_t)divup(std::max(p.rows, p.last), TILE) * 4;
    p.kPerSplit = divup(p.Kv, std::max(1, std::min(p.Kv / 8, 512 / (p.nTiles * p.dTiles))));
    p.splits = divup(p.Kv, p.kPerSplit);
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t o = at; at += al256(bytes); return o; };
    p.classExp = take(mostKv * 4);
    p.caseExp = take((size_t)p.Np * 4);
    p.xByCase = take((size_t)p.Np / 16 * p.Kd * PAIR);
    p.wByClass = take(mostKv * 2 * p.Kd * PAIR);
    if (bwd) {
        p.featExp = take((size_t)p.Dp * 4);
        p.xByFeat = take((size_t)p.Dp / 16 * p.Kn * PAIR);
        p.dz = take((size_t)p.Np / 16 * mostKv * PAIR);
        p.dzNear = take((size_t)p.Np / 16 * mostKv * PAIR);
        p.levels = take((size_t)p.Np / 64 * mostKv * 32);
        p.anyLevel = take(4);
        p.dbPart = take((size_t)p.nTiles * V * 4);
        p.slabs = take((size_t)p.splits * p.Dp * p.Np * 4);
    } else {
        p.part = take((size_t)(divup(V, 64) + divup(V, p.rows) * 2) * 3 * N * 4);
        p.labelLogits = take((size_t)N * 4);
    }
    p.total = at;
    return p;
}

// RG of k_fcl_narrow.  Forward, 1 / 4 (us of a cost call, 512 features, 16 cases): 10575 classes 16 / 18, 20000 24 / 22, 100000 86 / 53.
// Backward nothing is joined, and only the reads of x are fewer (gradients, 64 cases): 10575 classes 50 / 56, 20000 81 / 85, 40000 158 / 160,
// 100000 411 / 397.
int narrow_groups(int rows, bool bwd) { return rows > (bwd ? 32 : 16) * 1024 ? 4 : 1; }
int narrow_tiles(int rows) { return divup(rows, 16 * narrow_groups(rows, false)); }
// blocks: narrow_tiles(rows) forward, all of the piece's packed classes backward
template <bool BWD>
void launch_narrow(const NarrowArgs& p, int blocks, hipStream_t s) {
#define NARROW_LAUNCH(NB)                                                                                                    \
    if (narrow_groups(p.rows, BWD) == 1) MCN_LAUNCH((k_fcl_narrow<BWD, NB, 1>), dim3(blocks), dim3(256), 0, s, p); \
    else MCN_LAUNCH((k_fcl_narrow<BWD, NB, 4>), dim3(blocks), dim3(256), 0, s, p)
    switch (divup(p.N, 16)) {
        case 1: NARROW_LAUNCH(1); break;
        case 2: NARROW_LAUNCH(2); break;
        case 3: NARROW_LAUNCH(3); break;
        default: NARROW_LAUNCH(4); break;
    }
#undef NARROW_LAUNCH
}

template <bool BWD>
void launch_logits(TileKind kind, const WideArgs& a, hipStream_t s) {
    const dim3 grid(a.vTiles * a.nTiles), block(256);
    if (kind == SHARED) MCN_LAUNCH((k_fcl_logits<4, BWD, true>), grid, block, tile_bytes(SHARED), s, a);
    else if (kind == WHOLE) MCN_LAUNCH((k_fcl_logits<4, BWD, false>), grid, block, tile_bytes(WHOLE), s, a);
    else MCN_LAUNCH((k_fcl_logits<2, BWD, false>), grid, block, tile_bytes(HALF), s, a);
}

WideArgs wide_args(const WidePlan& q, const float* W, const float* X, const float* bias, const float* labels, int D, int V, int N, char* ws) {
    WideArgs a = {};
    a.W = W;
    a.X = X;
    a.D = D;
    a.wByClass = ws + q.wByClass;
    a.xByCase = ws + q.xByCase;
    a.classExp = (const int*)(ws + q.classExp);
    a.caseExp = (const int*)(ws + q.caseExp);
    a.bias = bias;
    a.labels = labels;
    a.V = V;
    a.N = N;
    a.Kd = q.Kd;
    a.kSteps = q.kSteps;
    return a;
}
// the classes of the piece that begins at v0
int piece_rows(const WidePlan& q, int V, int v0) { return V - v0 <= q.last ? V - v0 : q.rows; }
// one piece: its packed rows, tiles and k blocks; with the first one, x
TileKind wide_piece(const WidePlan& q, WideArgs& a, PackArgs& k, const float* W, int D, int v0, hipStream_t s) {
    a.v0 = v0;
    a.rows = k.rows = piece_rows(q, a.V, v0);
    a.nTiles = q.nTiles;
    a.Kv = k.Kv = divup(a.rows, TILE) * 4;
    const TileKind kind = tile_choice(a.Kv, q.nTiles);
    a.vTiles = a.Kv / tile_rows32(kind);
    k.W = W + (size_t)v0 * D;
    k.bias = a.bias ? a.bias + v0 : nullptr;
    MCN_LAUNCH(k_fcl_pack, dim3(k.caseBlocks + k.featBlocks + a.Kv), dim3(512), PACK_LDS, s, k);
    k.caseBlocks = k.featBlocks = 0;
    return kind;
}
PackArgs pack_args(const WidePlan& q, const float* X, const float* labels, const float* stats, int D, int V, int N, bool feats, char* ws) {
    PackArgs k = {};
    k.X = X; k.labels = labels; k.stats = stats;
    k.caseExp = (int*)(ws + q.caseExp); k.featExp = (int*)(ws + q.featExp);
    k.xByCase = ws + q.xByCase; k.xByFeat = ws + q.xByFeat;
    k.D = D; k.V = V; k.N = N; k.Kd = q.Kd; k.Kn = q.Kn;
    k.caseBlocks = q.Np / 16; k.featBlocks = feats ? q.Dp / 16 : 0;
    k.classExp = (int*)(ws + q.classExp); k.wByClass = ws + q.wByClass;
    return k;
}

// k blocks of a share of a piece's input gradient: the last piece has no more shares than there are slabs, and a short one fewer, not
// shorter ones
int piece_share(const WidePlan& q, int Kv) { return Kv == q.Kv ? q.kPerSplit : std::max(8, divup(Kv, q.splits)); }
// two blocks a CU once there is more than one for each; one with its stages further ahead / two: 512 x 4213 x 128, all gradients,
// 39.9 / 41.5 us; 512 x 10575 x 128 53 / 50 us
bool grads_shared(int blocks) { return blocks > 256; }

int wide_cost(const float* W, const float* X, const float* bias, const float* labels, float* stats, float* logp, float* correct, int D, int V,
              int N, char* ws, hipStream_t s) {
    const WidePlan q = wide_plan(D, V, N, false);
    WideArgs a = wide_args(q, W, X, bias, labels, D, V, N, ws);
    a.labelLogits = (float*)(ws + q.labelLogits);
    PackArgs pack = pack_args(q, X, labels, nullptr, D, V, N, false, ws);
    int tiles = 0;
    for (int v0 = 0; v0 < V; v0 += a.rows) {
        const TileKind kind = wide_piece(q, a, pack, W, D, v0, s);
        a.part = (float*)(ws + q.part) + (size_t)tiles * 3 * N;
        launch_logits<false>(kind, a, s);
        tiles += a.vTiles;
        if (int rc = MCN_LAUNCH_CHECK("fcLogregCost")) return rc;
    }
    MCN_LAUNCH(k_fcl_join, dim3(divup(N, 16)), dim3(1024), 0, s, (const float*)(ws + q.part), a.labelLogits, labels, stats, logp, correct, V, N, tiles);
    return MCN_LAUNCH_CHECK("fcLogregCost");
}

int wide_grad(const float* W, const float* X, const float* bias, const float* labels, const float* stats, float* dX, float* dW, float* dB, int D,
              int V, int N, float coeff, float scaleInputTargets, float scaleWeightTargets, float scaleWeightOutput, float scaleBiasTargets,
              float scaleBiasOutput, char* ws, hipStream_t s) {
    const WidePlan q = wide_plan(D, V, N, true);
    WideArgs a = wide_args(q, W, X, bias, labels, D, V, N, ws);
    a.stats = stats;
    a.dz = ws + q.dz;
    a.near = q.dzNear - q.dz;
    a.levels = (unsigned char*)ws + q.levels;
    a.anyLevel = (int*)(ws + q.anyLevel);
    a.dbPart = dB ? (float*)(ws + q.dbPart) : nullptr;
    float* slabs = (float*)(ws + q.slabs);
    const bool narrow = !wide_cost_usable(N);  // (the forward call's logits, to the bit)
    PackArgs pack = pack_args(q, X, labels, stats, D, V, N, dW != nullptr, ws);
    if (narrow) pack.caseBlocks = 0;
    pack.levels = a.levels;
    pack.anyLevel = a.anyLevel;
    NarrowArgs few = {W, X, bias, labels, D, V, N};
    few.stats = stats; few.dz = a.dz; few.near = a.near; few.levels = a.levels; few.anyLevel = a.anyLevel; few.dbPart = a.dbPart;
    GradArgs t = {};
    t.xByFeat = ws + q.xByFeat; t.dz = ws + q.dz; t.wByClass = ws + q.wByClass;
    t.levels = a.levels; t.anyLevel = a.anyLevel; t.near = a.near; t.allNear = narrow;
    t.featExp = (const int*)(ws + q.featExp); t.classExp = (const int*)(ws + q.classExp);
    t.slabs = slabs;
    t.D = D; t.Kn = q.Kn; t.Kd = q.Kd; t.Np = q.Np; t.Dp = q.Dp; t.nTiles = q.nTiles; t.dTiles = q.dTiles;
    t.scaleTargets = scaleWeightTargets;
    t.scaleOutput = scaleWeightOutput * coeff;
    for (int v0 = 0; v0 < V; v0 += a.rows) {
        const TileKind kind = wide_piece(q, a, pack, W, D, v0, s);
        if (narrow) {
            few.v0 = v0;
            few.rows = a.rows;
            few.Kv = a.Kv;
            launch_narrow<true>(few, a.Kv * 2 / narrow_groups(a.rows, true), s);
        } else {
            launch_logits<true>(kind, a, s);
        }
        t.kPerSplit = piece_share(q, a.Kv);
        t.inputBlocks = dX ? divup(a.Kv, t.kPerSplit) * q.nTiles * q.dTiles : 0;
        t.dW = dW ? dW + (size_t)v0 * D : nullptr;
        t.rows = a.rows;
        t.Kv = a.Kv;
        t.first = v0 == 0;
        const int blocks = t.inputBlocks + (dW ? a.Kv / 4 * q.dTiles : 0);
        if (grads_shared(blocks)) MCN_LAUNCH(k_fcl_grads<true>, dim3(blocks), dim3(256), tile_bytes(SHARED), s, t);
        else if (blocks > 0) MCN_LAUNCH(k_fcl_grads<false>, dim3(blocks), dim3(256), tile_bytes(WHOLE), s, t);
        if (int rc = MCN_LAUNCH_CHECK("fcLogregGrad")) return rc;
    }
    if (dX || dB) {
        const int dxBlocks = dX ? (int)std::min<size_t>(divup_sz((size_t)D * N, 256), 1 << 16) : 0;
        const FinishArgs f = {slabs, (const float*)(ws + q.dbPart), W, bias, labels, stats, dX, dB, D, V, N, q.Np, q.Dp, q.splits, q.nTiles,
                              dxBlocks, coeff, scaleInputTargets, scaleBiasTargets, scaleBiasOutput};
        MCN_LAUNCH(k_fcl_finish, dim3(dxBlocks + (dB ? divup(V, 256) : 0)), dim3(256), 0, s, f);
    }
    return MCN_LAUNCH_CHECK("fcLogregGrad");
}

bool fcl_sizes_ok(int D, int V, int N) {
    return D > 0 && V > 0 && N > 0 && V <= (1 << 24) && D <= (1 << 20) && N <= (1 << 20) && (size_t)D * N <= (size_t)1 << 34;
}

size_t al16b(size_t b) { return (b + 15) / 16 * 16; }
size_t fcl_cost_bytes(int D, int V, int N) {
    if (wide_cost_usable(N)) return wide_plan(D, V, N, false).total;
    return al16b((size_t)narrow_tiles(V) * 3 * N * sizeof(float)) + al16b((size_t)N * sizeof(float));
}
size_t fcl_grad_bytes(int D, int V, int N) { return wide_plan(D, V, N, true).total; }

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
    const size_t n = (size_t)numCases;
    if (int rc = mcn_refuse_overlaps("fcLogregCost",
                                     {{"caseStats", caseStats, 2 * n}, {"labelLogProbs", labelLogProbs, n}, {"correctProbs", correctProbs, n}, {"costOut", (const float*)costOut, 4}},
                                     {{"weights", weights, (size_t)numOutputs * numInputs}, {"inputs", inputs, (size_t)numInputs * numCases},
                                      {"biases", biases, (size_t)numOutputs}, {"labels", labels, n}}))
        return rc;
    if (int rc = fcl_check("fcLogregCost", workspace, workspaceBytes, fcl_cost_bytes(numInputs, numOutputs, numCases))) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (wide_cost_usable(numCases)) {
        if (int rc = wide_cost(weights, inputs, biases, labels, caseStats, labelLogProbs, correctProbs, numInputs, numOutputs, numCases, (char*)workspace, s)) return rc;
    } else {
        const int tiles = narrow_tiles(numOutputs);
        NarrowArgs p = {weights, inputs, biases, labels, numInputs, numOutputs, numCases, 0, numOutputs};
        p.part = (float*)workspace;
        p.labelLogits = (float*)((char*)workspace + al16b((size_t)tiles * 3 * numCases * sizeof(float)));
        launch_narrow<false>(p, tiles, s);
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
    MCN_REQUIRE(fcl_sizes_ok(numInputs, numOutputs, numCases), "fcLogregGrad: %d inputs, %d outputs, %d cases", numInputs, numOutputs, numCases);
    const size_t nX = (size_t)numInputs * numCases, nW = (size_t)numOutputs * numInputs, nB = (size_t)numOutputs, n = (size_t)numCases;
    if (int rc = mcn_refuse_overlaps("fcLogregGrad", {{"inputGrads", inputGrads, nX}, {"weightGrads", weightGrads, nW}, {"biasGrads", biasGrads, nB}},
                                     {{"weights", weights, nW}, {"inputs", inputs, nX}, {"biases", biases, nB}, {"labels", labels, n}, {"caseStats", caseStats, 2 * n}}))
        return rc;
    if (int rc = fcl_check("fcLogregGrad", workspace, workspaceBytes, fcl_grad_bytes(numInputs, numOutputs, numCases))) return rc;
    return wide_grad(weights, inputs, biases, labels, caseStats, inputGrads, weightGrads, biasGrads, numInputs, numOutputs, numCases, coeff,
                     scaleInputTargets, scaleWeightTargets, scaleWeightOutput, scaleBiasTargets, scaleBiasOutput, (char*)workspace,
                     (hipStream_t)stream);
}

#ifdef MCN_TEST_HOOKS
// What the pieces of a call take, so that a test knows which forms it runs: five numbers for each of the first `most` pieces (classes, tiles
// of the logits as in TileKind, or 3 for few cases, k blocks of a share of the input gradient, shares, 1 where all gradients' tiles go
// two to a CU).  The number of pieces.
MCN_API int mcn_fc_logreg_test_forms(int numInputs, int numOutputs, int numCases, int backward, int* out, int most) {
    if (!fcl_sizes_ok(numInputs, numOutputs, numCases)) return 0;
    const WidePlan q = wide_plan(numInputs, numOutputs, numCases, backward != 0);
    int pieces = 0;
    for (int v0 = 0, rows; v0 < numOutputs; v0 += rows, pieces++) {
        rows = piece_rows(q, numOutputs, v0);
        const int Kv = divup(rows, TILE) * 4, share = piece_share(q, Kv), shares = divup(Kv, share);
        if (pieces >= most) continue;
        int* o = out + 5 * pieces;
        o[0] = rows;
        o[1] = wide_cost_usable(numCases) ? (int)tile_choice(Kv, q.nTiles) : 3;
        o[2] = share;
        o[3] = shares;
        o[4] = grads_shared(shares * q.nTiles * q.dTiles + Kv / 4 * q.dTiles);
    }
    return pieces;
}
#endif
