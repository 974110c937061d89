// What the products share: matrix instructions, activations, tiles of operands in LDS.
#pragma once
#include "bs_embed.hpp"

namespace bse {

template <typename T>
struct Mma;
template <>
struct Mma<f16> {
    __device__ static f32x16 go(Vec<f16, 8> a, Vec<f16, 8> b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Mma<bf16> {
    __device__ static f32x16 go(Vec<bf16, 8> a, Vec<bf16, 8> b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

template <typename T>
struct Mma16;
template <>
struct Mma16<f16> {
    __device__ static f32x4 go(Vec<f16, 8> a, Vec<f16, 8> b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Mma16<bf16> {
    __device__ static f32x4 go(Vec<bf16, 8> a, Vec<bf16, 8> b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

constexpr float LOG2E = 1.4426950408889634f;

// z (1 + erf(z / sqrt 2)) / 2 in the form of formula 7.1.26 of Abramowitz and Stegun's handbook: with x = |z| / sqrt 2 and t = 1 /
// (1 + p |z|), erfc(x) / 2 = t P(t) exp(-x^2).  Its five coefficients are off by 1.5e-7 of 1, which is 7e-4 of the result at
// z = -4.2 and 3e-2 at -12, several roundings of a 16-bit type.  Those here are of degree 6, the least squares over |z| <= 13.5
// reweighted until the largest of the errors against 7e-8 exp(x^2) and 4e-6 of erfc(x) is least: off by 2.8e-6 of itself and by
// 1.6e-7, float32 roundings included (the five: 2.4e-7), beside the rounding of the exponent, 1.5 z^2 units of 2^-24 of a result
// below 0.  Past z = -13.2, where exp(-x^2) is below float32's normal range, the result may be 0.  8191 x 1024 -> 4096:
// 87 us, 84 with five coefficients (another card: 92, and 102 with the library's erff).
__device__ inline float gelu_part(float z, float e) {  // (1 + erf(z / sqrt 2)) / 2 for e = exp(-z^2 / 2)
    const float t = __builtin_amdgcn_rcpf(fmaf(0.348f, fabsf(z), 1.0f));
    float q = fmaf(t, 0.044490628f, -0.18701635f);
    q = fmaf(t, fmaf(t, fmaf(t, q, 0.22043395f), 0.0022022785f), 0.14531076f);
    const float rest = t * fmaf(t, fmaf(t, q, 0.13556218f), 0.13901654f) * e;  // erfc(x) / 2
    return z < 0.0f ? rest : 1.0f - rest;
}
__device__ inline float gelu(float z) { return z * gelu_part(z, __builtin_amdgcn_exp2f(z * z * (-0.5f * LOG2E))); }

// one branch for all values: the branches are the call's, not the lanes'
template <int N>
__device__ inline void activate(float (&z)[N], int act) {
    if (act == BS_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = z[j] < 0.0f ? 0.0f : z[j];
    } else if (act == BS_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = gelu(z[j]);
    } else if (act == BS_ACT_GELU_TANH) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
            const float u = 0.79788456080286536f * fmaf(0.044715f * z[j] * z[j], z[j], z[j]);
            z[j] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-2.0f * LOG2E * u));
        }
    } else if (act == BS_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] *= __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-LOG2E * z[j]));
    }
}

// Meets the workgroup's other waves once all but this wave's N youngest moves to LDS are done.  Products
// written before it stay before it, and with them the waits for the LDS reads that feed them; reads that
// are still on their way at the meeting are of a step that nobody overwrites yet.
template <int N>
__device__ inline void meet() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4 | 15 << 8);  // vmcnt(N)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
}

// Tiles of BM rows of x by BN rows of w; WM x WN waves; inner steps of BK; NS steps in LDS.
template <int BM_, int BN_, int WM_, int WN_, int BK_, int NS_, int PER_CU_>
struct Tile {
    static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, BK = BK_, NS = NS_, PER_CU = PER_CU_;
    static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
    static constexpr int TM = BM / WM / 32, TN = BN / WN / 32;  // 32 x 32 results of a wave
    static constexpr int CH = BK / 8;                           // 16-byte chunks of a row
    static constexpr int STEP = (BM + BN) * BK;                 // elements of a step: rows of x, then of w
    static constexpr int MOVES = (BM + BN) * CH / THREADS;      // 16-byte moves of a thread per step
    static constexpr int JOIN = 32 * (TN * 32 + 4) * 4;         // bytes in which a wave turns 32 rows of results
    static constexpr int LDS = NS * STEP * 2 > WAVES * JOIN ? NS * STEP * 2 : WAVES * JOIN;
    // the 16 lanes of a quarter wave read one chunk of 16 rows: spread over the 256 bytes of all banks
    __device__ static int swizzle(int r, int c) { return BK == 64 ? c ^ ((r >> 1) & 7) : c ^ ((r >> 2) & 3); }
    __device__ static int place(int r, int c) { return r * BK + swizzle(r, c) * 8; }
};

// chunk c of 16 bytes in row r of an LDS tile of S bytes per row (64, 128, 256 or 512).  16 rows read at one
// chunk (a quarter wave's operand of K) lie in 16 different chunks of the 256 bytes that all banks span,
// and the 4 rows x 64 bytes of a transposed read of V in 4 different quarters of them.
template <int S>
__device__ inline int place(int r, int c) {
    const int f = S >= 256 ? ((r & 3) << 2 | ((r >> 2) & 3)) : S == 128 ? (((r >> 1) & 1) << 2 | ((r >> 2) & 3)) : ((r >> 2) & 3);
    return r * S + ((c ^ f) << 4);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// For code that counts its moves to LDS by itself: the compiler takes every transposing read for one that may read what a move
// writes, and puts a wait for all of the wave's moves before it, unless the read's pointer is known to have no alias.
__device__ __forceinline__ s16x4 read_transposed(const char* __restrict p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

}  // namespace bse
