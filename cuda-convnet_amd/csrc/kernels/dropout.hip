// Dropout with a counter-based generator: the mask is a function of (seed, step, element), so it is never stored -- the
// backward pass draws it again from the same numbers (mcn_dropout on the gradient).
//
// Generator: Philox-4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011):
// counter (element / 4, step), 64 bits each, key = seed; element e takes word e % 4 of the four.
//
// Bound by memory: ten rounds are 20 multiplications for 32 bytes moved.  8192 x 16384: 210 us, 5.1 TB/s, a copy's rate; small matrices: the
// launch.
#include <math.h>
#include "common.h"

static __device__ __forceinline__ void philox4x32(uint64_t quad, uint64_t step, uint64_t seed, uint32_t (&w)[4]) {
    uint32_t c0 = (uint32_t)quad, c1 = (uint32_t)(quad >> 32), c2 = (uint32_t)step, c3 = (uint32_t)(step >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; r++) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// One thread per four elements (one generator call).  VEC: both matrices 16-byte aligned, one 16-byte access each.
// A dropped element is selected away, not multiplied by zero: an infinity or NaN in it does not come through.
template <bool VEC, bool ADD>
__global__ __launch_bounds__(256) void k_dropout(const float* inputs, float* target, size_t n, uint32_t threshold, float keepScale,
                                                 float scaleTargets, uint64_t seed, uint64_t step, const uint64_t* deviceStep) {
    if (deviceStep) step += *deviceStep;
    const size_t quads = (n + 3) / 4;
    for (size_t q = (size_t)blockIdx.x * blockDim.x + threadIdx.x; q < quads; q += (size_t)gridDim.x * blockDim.x) {
        uint32_t w[4];
        philox4x32(q, step, seed, w);
        if (VEC && q * 4 + 4 <= n) {
            const f32x4 x = reinterpret_cast<const f32x4*>(inputs)[q];
            f32x4 y;
#pragma unroll
            for (int j = 0; j < 4; j++) y[j] = w[j] >= threshold ? x[j] * keepScale : 0.f;
            if (ADD) {
                const f32x4 t = reinterpret_cast<const f32x4*>(target)[q];
#pragma unroll
                for (int j = 0; j < 4; j++) y[j] = scaleTargets * t[j] + y[j];
            }
            reinterpret_cast<f32x4*>(target)[q] = y;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const size_t e = q * 4 + j;
                if (e < n) {
                    const float y = w[j] >= threshold ? inputs[e] * keepScale : 0.f;
                    target[e] = ADD ? scaleTargets * target[e] + y : y;
                }
            }
        }
    }
}

MCN_API int mcn_dropout(const float* inputs, float* target, size_t numElements, float dropProb, uint64_t seed, uint64_t step,
                        const uint64_t* deviceStep, float scaleTargets, float scaleOutput, void* stream) {
    MCN_REQUIRE(inputs && target, "dropout: null pointer");
    MCN_REQUIRE(dropProb >= 0.f && dropProb < 1.f, "dropout: probability %g is not in [0, 1)", (double)dropProb);  // (refuses a NaN too)
    MCN_REQUIRE(numElements <= (size_t)1 << 40, "dropout: %zu elements", numElements);
    MCN_REQUIRE(target == inputs || !mcn_overlap(target, numElements, inputs, numElements), "dropout: target overlaps inputs in part");
    if (numElements == 0) return MCN_OK;
    const uint32_t threshold = (uint32_t)((double)dropProb * 4294967296.0);  // (a float below 1 is at most 1 - 2^-24: fits)
    const float keepScale = (float)((double)scaleOutput / (1.0 - (double)dropProb));
    const size_t quads = divup_sz(numElements, 4);
    const size_t blocks = divup_sz(quads, 256);
    const dim3 grid((unsigned)(blocks < 4096 ? blocks : 4096)), block(256);
    const bool vec = (((uintptr_t)inputs | (uintptr_t)target) & 15) == 0;
    hipStream_t s = (hipStream_t)stream;
#define LAUNCH(V, A) MCN_LAUNCH((k_dropout<V, A>), grid, block, 0, s, inputs, target, numElements, threshold, keepScale, scaleTargets, seed, step, deviceStep)
    if (vec) {
        if (scaleTargets != 0.f) LAUNCH(true, true); else LAUNCH(true, false);
    } else {
        if (scaleTargets != 0.f) LAUNCH(false, true); else LAUNCH(false, false);
    }
#undef LAUNCH
    return MCN_LAUNCH_CHECK("dropout");
}

__global__ void k_counter_add(uint64_t* counter, uint64_t by) { *counter += by; }

MCN_API int mcn_counter_add(uint64_t* counter, uint64_t by, void* stream) {
    MCN_REQUIRE(counter, "counterAdd: null pointer");
    MCN_LAUNCH(k_counter_add, dim3(1), dim3(1), 0, (hipStream_t)stream, counter, by);
    return MCN_LAUNCH_CHECK("counterAdd");
}
