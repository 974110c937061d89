// Products with bias, activation and residual in the epilogue (include/bs_embed.h).
//
// out = act(x w^T + b) + r.  Both operands are rows of the inner dimension, so tiles of both go to LDS
// as they lie and the matrix instructions read 16 bytes (8 inner elements) per lane.  The weight is the
// instruction's first operand: a lane of the result then holds one row of out and groups of four
// adjacent columns.
#include "bs_embed.hpp"

#include <algorithm>
#include <type_traits>

namespace {
using namespace bse;

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

struct Params {
    const void *x, *w, *bias, *residual;
    void* out;
    int64_t xs, ws, rs, os;
    uint32_t rows, inner, cols;
    int act;
    uint32_t splits;  // pieces of the inner dimension; > 1: their sums go to `parts`, splits x rows x cols
    float* parts;
};

constexpr float LOG2E = 1.4426950408889634f;

// z (1 + erf(z / sqrt 2)) / 2 by formula 7.1.26 of Abramowitz and Stegun's handbook: with x = |z| / sqrt 2,
// t = 1 / (1 + p x), erfc(x) = t (a1 + t (a2 + .. )) exp(-x^2), off by 1.5e-7 at most, so by 1.3 units of 2^-24
// |z| here; the halves and roots are in the constants.  That is absolute: a result far below 1 is off by 7e-4 of itself at
// z = -4.2 and 3e-3 at -5.7, which float32 results show (1 + erf in float32 is off by 2e-3 and loses all of it there).
// 8191 x 1024 -> 4096: 92 us, 102 us with the library's erff.
__device__ inline float gelu(float z) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.23164189f, fabsf(z), 1.0f));
    const float q = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5307027145f, -0.7265760135f), 0.7107068705f), -0.142248368f), 0.127414796f);
    const float rest = q * __builtin_amdgcn_exp2f(z * z * (-0.5f * LOG2E));  // erfc(x) / 2
    return z * (z < 0.0f ? rest : 1.0f - rest);
}

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

// N adjacent columns of one row, those inside
template <typename T, typename O, int N>
__device__ inline void finish(const Params& p, uint32_t row, uint32_t col, float (&z)[N]) {
    const int n = static_cast<int>(p.cols - col);
    if (p.bias) {
        const Vec<T, N> b = load_some<T, N>(static_cast<const T*>(p.bias) + col, n);
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] += static_cast<float>(b[j]);
    }
    activate(z, p.act);
    if (p.residual) {
        const Vec<O, N> r = load_some<O, N>(static_cast<const O*>(p.residual) + static_cast<int64_t>(row) * p.rs + col, n);
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] += static_cast<float>(r[j]);
    }
    Vec<O, N> o;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = static_cast<O>(z[j]);
    store_some<O, N>(static_cast<O*>(p.out) + static_cast<int64_t>(row) * p.os + col, o, n);
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

// Direct: rows are 16-byte aligned, whole steps go from memory to LDS without registers
template <typename T, typename O, typename C, bool Direct>
__global__ __launch_bounds__(C::THREADS, C::PER_CU * C::WAVES / 4) void linear_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    T* buf = reinterpret_cast<T*>(lds);
    const T* x = static_cast<const T*>(p.x);
    const T* w = static_cast<const T*>(p.w);
    // Workgroup b runs on XCD b mod 8: each XCD takes a contiguous run of tiles, 8 tile rows high, so that
    // the tiles in flight on it share operands in its L2.
    const uint32_t mt = (p.rows + C::BM - 1) / C::BM, nt = (p.cols + C::BN - 1) / C::BN, total = mt * nt;
    const uint32_t xcd = blockIdx.x & 7, q8 = total >> 3, r8 = total & 7;
    const uint32_t id = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3);
    const uint32_t band = id / (8 * nt), high = mt - band * 8 < 8 ? mt - band * 8 : 8, in = id - band * 8 * nt;
    const uint32_t m0 = (band * 8 + in % high) * C::BM, n0 = in / high * C::BN;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 31, h = lane >> 5;
    const int wm = wave / C::WN * C::TM * 32, wn = wave % C::WN * C::TN * 32;

    // this thread's moves: 16 bytes each, to LDS positions that are linear over the workgroup
    const T* from[C::MOVES];
    int chunk[C::MOVES];
#pragma unroll
    for (int i = 0; i < C::MOVES; ++i) {
        const int at = i * C::THREADS + threadIdx.x, r = at / C::CH;
        chunk[i] = C::swizzle(r, at % C::CH);
        // rows past the end repeat the last one: their products are not stored
        if (r < C::BM) {
            const uint32_t m = m0 + r < p.rows ? m0 + r : p.rows - 1;
            from[i] = x + static_cast<int64_t>(m) * p.xs + chunk[i] * 8;
        } else {
            const uint32_t n = n0 + r - C::BM < p.cols ? n0 + r - C::BM : p.cols - 1;
            from[i] = w + static_cast<int64_t>(n) * p.ws + chunk[i] * 8;
        }
    }
    // this workgroup's piece: whole steps [begin, whole), and for the last piece what is left after them
    const uint32_t allsteps = (p.inner + C::BK - 1) / C::BK, piece = (allsteps + p.splits - 1) / p.splits;
    const uint32_t begin = blockIdx.y * piece, steps = min(begin + piece, allsteps), whole = min(steps, p.inner / C::BK);
    auto move = [&](uint32_t t, int slot, int first = 0, int n = C::MOVES) {  // Direct
#pragma unroll
        for (int i = first; i < first + n; ++i)
            __builtin_amdgcn_global_load_lds((global_ptr)(from[i] + static_cast<size_t>(t) * C::BK),
                                             (lds_ptr)(buf + slot * C::STEP + (i * C::THREADS + wave * 64) * 8), 16, 0, 0);
    };
    auto fetch = [&](uint32_t t, Vec<T, 8> (&v)[C::MOVES]) {
#pragma unroll
        for (int i = 0; i < C::MOVES; ++i) {
            const int left = static_cast<int>(p.inner) - static_cast<int>(t * C::BK) - chunk[i] * 8;
            v[i] = left > 0 ? load_some<T, 8>(from[i] + static_cast<size_t>(t) * C::BK, left) : Vec<T, 8>{};
        }
    };
    auto put = [&](int slot, const Vec<T, 8> (&v)[C::MOVES]) {
#pragma unroll
        for (int i = 0; i < C::MOVES; ++i)
            *reinterpret_cast<Vec<T, 8>*>(buf + slot * C::STEP + (i * C::THREADS + threadIdx.x) * 8) = v[i];
    };
    f32x16 acc[C::TN][C::TM] = {};
    struct Parts {
        Vec<T, 8> a[C::TN], b[C::TM];
    };
    auto read = [&](int slot, int s, Parts& f) {  // 16 inner elements
        const T* tx = buf + slot * C::STEP;
        const T* tw = tx + C::BM * C::BK;
#pragma unroll
        for (int i = 0; i < C::TN; ++i) f.a[i] = *reinterpret_cast<const Vec<T, 8>*>(tw + C::place(wn + i * 32 + l, s * 2 + h));
#pragma unroll
        for (int j = 0; j < C::TM; ++j) f.b[j] = *reinterpret_cast<const Vec<T, 8>*>(tx + C::place(wm + j * 32 + l, s * 2 + h));
    };
    auto product = [&](const Parts& f, int from_, int to) {
#pragma unroll
        for (int i = from_; i < to; ++i)
#pragma unroll
            for (int j = 0; j < C::TM; ++j) acc[i][j] = Mma<T>::go(f.a[i], f.b[j], acc[i][j]);
    };
    auto multiply = [&](int slot) {
        Parts f;
#pragma unroll
        for (int s = 0; s < C::BK / 16; ++s) {
            read(slot, s, f);
            product(f, 0, C::TN);
        }
    };
    if (Direct) {
        // At meeting t steps t and t + 1 are in LDS and nobody reads step t - 1 any more, whose place step
        // t + NS - 1 gets.  Operands are read one part (16 inner elements) ahead of their products, across the
        // meeting too.  A move past the last step repeats the last one, so that every wait counts the same.
        const uint32_t last = whole ? whole - 1 : 0;
        if (whole > begin) {
            Parts f[2];
#pragma unroll
            for (int i = 0; i < C::NS - 1; ++i) move(min(begin + i, last), i);
            meet<(C::NS - 2) * C::MOVES>();
            read(0, 0, f[0]);
            int slot = 0;
            for (uint32_t t = begin; t < whole; ++t) {
                meet<(C::NS - 3) * C::MOVES>();
                move(min(t + C::NS - 1, last), slot == 0 ? C::NS - 1 : slot - 1);
                const int next = slot == C::NS - 1 ? 0 : slot + 1;
#pragma unroll
                for (int s = 0; s < C::BK / 16; ++s) {
                    product(f[s & 1], 0, C::TN / 2);
                    __builtin_amdgcn_sched_barrier(0);
                    if (s + 1 < C::BK / 16)
                        read(slot, s + 1, f[(s + 1) & 1]);
                    else
                        read(next, 0, f[(s + 1) & 1]);
                    __builtin_amdgcn_sched_barrier(0);
                    product(f[s & 1], C::TN / 2, C::TN);
                    __builtin_amdgcn_sched_barrier(0);
                }
                slot = next;
            }
        }
        meet<0>();
        __syncthreads();
        if (steps > whole) {
            Vec<T, 8> v[C::MOVES];
            fetch(whole, v);
            put(0, v);
            __syncthreads();
            multiply(0);
            __syncthreads();
        }
    } else {
        Vec<T, 8> v[C::MOVES];
        fetch(begin, v);
        put(begin & 1, v);
        for (uint32_t t = begin; t < steps; ++t) {
            __syncthreads();
            if (t + 1 < steps) fetch(t + 1, v);
            multiply(t & 1);
            if (t + 1 < steps) put(~t & 1, v);
        }
        __syncthreads();
    }
    // a wave turns 32 rows of its results at a time: a lane then has 8 adjacent columns
    constexpr int W = C::TN * 32, PITCH = W + 4, LANES = W / 8;
    float* turn = reinterpret_cast<float*>(lds + wave * C::JOIN);
    auto spread = [&](auto J) {
        constexpr int j = decltype(J)::value;
        if constexpr (j < C::TM) {
#pragma unroll
            for (int i = 0; i < C::TN; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<f32x4*>(turn + l * PITCH + i * 32 + q * 8 + h * 4) =
                        f32x4{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
        }
    };
    static_assert(C::TM <= 4, "cases below");
#pragma unroll 1
    for (int j = 0; j < C::TM; ++j) {  // not unrolled: the epilogue's code stays in the instruction cache
        switch (j) {
            case 0: spread(std::integral_constant<int, 0>()); break;
            case 1: spread(std::integral_constant<int, 1>()); break;
            case 2: spread(std::integral_constant<int, 2>()); break;
            default: spread(std::integral_constant<int, 3>()); break;
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int k = 0; k < 32 * LANES / 64; ++k) {
            const int r = k * (64 / LANES) + lane / LANES, c = lane % LANES * 8;
            const uint32_t row = m0 + wm + j * 32 + r, col = n0 + wn + c;
            float z[8];
            const f32x4 z0 = *reinterpret_cast<const f32x4*>(turn + r * PITCH + c), z1 = *reinterpret_cast<const f32x4*>(turn + r * PITCH + c + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = z0[e], z[4 + e] = z1[e];
            if (row >= p.rows || col >= p.cols) continue;
            if (p.splits > 1) {
                float* part = p.parts + (static_cast<size_t>(blockIdx.y) * p.rows + row) * p.cols + col;
                store_some<float, 4>(part, z0, static_cast<int>(p.cols - col));
                if (p.cols - col > 4) store_some<float, 4>(part + 4, z1, static_cast<int>(p.cols - col) - 4);
            } else {
                finish<T, O>(p, row, col, z);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// the pieces' sums in order, and the epilogue: a thread takes four adjacent columns of a row
template <typename T, typename O>
__global__ __launch_bounds__(256) void linear_join_kernel(Params p) {
    const uint32_t across = (p.cols + 3) / 4;
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint32_t row = static_cast<uint32_t>(at / across), col = static_cast<uint32_t>(at % across) * 4;
    if (row >= p.rows) return;
    const int n = static_cast<int>(p.cols - col);
    const float* part = p.parts + static_cast<size_t>(row) * p.cols + col;
    f32x4 s = load_some<float, 4>(part, n);
    for (uint32_t i = 1; i < p.splits; ++i) s += load_some<float, 4>(part + static_cast<size_t>(i) * p.rows * p.cols, n);
    float z[4] = {s[0], s[1], s[2], s[3]};
    finish<T, O>(p, row, col, z);
}

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

// Few rows: the weight is read once, from memory to registers, and bounds the time.  A workgroup has NT x 16 of
// its rows, its eight waves a contiguous piece each of the inner dimension, so that 16 columns are enough work
// for a compute unit and nothing is joined across workgroups; x (MT x 16 rows) comes from the L2.  17 x 4096 -> 4096
// in bf16: 10.6 us among other calls, 3.2 TB/s; 1 x 1024 -> 128 4.2 us, a chain of four loads and a launch.
template <typename T, typename O, int MT, int NT>
__global__ __launch_bounds__(512) void linear_few_kernel(Params p) {
    __shared__ f32x4 join[8][NT * MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * (NT * 16);
    // rows past the end repeat the last one: their products are not stored
    const T *wp[NT], *xp[MT];
#pragma unroll
    for (int i = 0; i < NT; ++i) wp[i] = static_cast<const T*>(p.w) + static_cast<int64_t>(min(n0 + i * 16 + l, p.cols - 1)) * p.ws + g * 8;
#pragma unroll
    for (int i = 0; i < MT; ++i)
        xp[i] = static_cast<const T*>(p.x) + static_cast<int64_t>(min(static_cast<uint32_t>(i * 16 + l), p.rows - 1)) * p.xs + g * 8;
    f32x4 acc[NT][MT] = {};
    const uint32_t steps = (p.inner + 31) / 32, piece = (steps + 7) / 8, begin = wave * piece;
    const uint32_t end = min(begin + piece, steps), whole = min(end, p.inner / 32);
    constexpr int U = 8;  // steps in flight
    uint32_t t = begin;
    for (; t + U <= whole; t += U) {
        Vec<T, 8> a[U][NT], b[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < NT; ++i) a[u][i] = load_any<T, 8>(wp[i] + (t + u) * 32);
#pragma unroll
            for (int i = 0; i < MT; ++i) b[u][i] = load_any<T, 8>(xp[i] + (t + u) * 32);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j) acc[i][j] = Mma16<T>::go(a[u][i], b[u][j], acc[i][j]);
    }
    for (; t < end; ++t) {
        const int left = static_cast<int>(p.inner - t * 32) - g * 8;
        Vec<T, 8> a[NT], b[MT];
#pragma unroll
        for (int i = 0; i < NT; ++i) a[i] = left > 0 ? load_some<T, 8>(wp[i] + t * 32, left) : Vec<T, 8>{};
#pragma unroll
        for (int i = 0; i < MT; ++i) b[i] = left > 0 ? load_some<T, 8>(xp[i] + t * 32, left) : Vec<T, 8>{};
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[i][j] = Mma16<T>::go(a[i], b[j], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) join[wave][i * MT + j][lane] = acc[i][j];
    __syncthreads();
    if (wave >= NT * MT) return;
    // wave i MT + j: rows 16 j + l, columns 16 i + 4 g to + 3; the waves' sums in order
    f32x4 s = join[0][wave][lane];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += join[k][wave][lane];
    const uint32_t row = wave % MT * 16 + l, col = n0 + wave / MT * 16 + g * 4;
    float z[4] = {s[0], s[1], s[2], s[3]};
    if (row < p.rows && col < p.cols) finish<T, O>(p, row, col, z);
}

// Tall: one workgroup of 8 waves per compute unit, three steps of 64; 2048 x 4096 -> 4096 takes 73 us (945 TFLOP/s).  The
// wait for the oldest step at every meeting bounds it.  Four waves of 128 x 64 take 76 us, tiles of 128 x 256 74.
// Mid: two workgroups per compute unit, four steps of 32; the same takes 90 us: operands in 64-byte rows cost twice
// the requests.  Steps of 64, which leave one workgroup of 128 x 128 per compute unit, take 96.
// Small: 1024 x 1024 -> 1024 takes 8 us, the latency of its 16 steps.
using Tall = Tile<256, 128, 4, 2, 64, 3, 1>;
using Mid = Tile<128, 128, 2, 2, 32, 4, 2>;
using Small = Tile<64, 64, 2, 2, 64, 4, 2>;

// Large products: tiles of 256 x 256 by 8 waves of 128 (rows of x) x 64 (rows of w), inner steps of 64.
//
// A step's operands take 64 KB of LDS and two steps fit, so that the way from memory to LDS would have one
// step's time.  It has one and a half: a step is four phases, and the quarters of its operands (x0, x1: the
// first and second 64 rows of every wave; w0, w1: the first and second 32) are read into registers a phase
// before their products, whereupon the moves of step t + 2 into that quarter start.
//   phase 0: read w1(t)              products w0 x0
//   phase 1: read x1(t)              products w1 x0    move x0, w0 (t + 2)
//   phase 2:                         products w0 x1    move w1 (t + 2)
//   phase 3: read x0, w0 (t + 1)     products w1 x1    move x1 (t + 2)
// A workgroup per CU goes through its tiles without a break: the moves of the next tile's first steps are
// under way while a tile's results are written.  A tile that would pass an edge is shifted back inside and
// does not write what its neighbour writes.
//
// 16384 x 4096 -> 4096 with bias and residual takes 474 us (1160 TFLOP/s; the library reaches 1348 without either at
// 8192 x 8192 x 8192), the matrix pipe busy for 0.59 of the time at 1.83 GHz: the meetings bound it, four a step.
// Inner steps of 32 took 625 us, reads and moves in a row before the products 562, moves later in the phase 583.
// 8191 x 1024 -> 4096 with gelu takes 84 us: 8 us of epilogue after every 16 steps, which nothing overlaps.
template <typename T, typename O>
__global__ __launch_bounds__(512, 2) void linear_big_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int STEP = 512 * 64;  // elements: 256 rows of x, then 256 of w
    T* buf = reinterpret_cast<T*>(lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 31, h = lane >> 5;
    float* turn = reinterpret_cast<float*>(lds + 2 * STEP * 2) + wave * 1024;
    const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
    auto swizzle = [](int r, int c) { return c ^ ((r >> 1) & 7); };

    const uint32_t mt = (p.rows + 255) / 256, nt = (p.cols + 255) / 256, total = mt * nt;
    // Workgroup b runs on XCD b mod 8: each XCD takes a contiguous run of tiles, 8 tile rows high, so that
    // the tiles in flight on it share operands in its L2.
    const uint32_t xcd = blockIdx.x & 7, q8 = total >> 3, r8 = total & 7;
    const uint32_t run = xcd * q8 + (xcd < r8 ? xcd : r8), end = run + q8 + (xcd < r8 ? 1 : 0), stride = gridDim.x >> 3;
    uint32_t id = run + (blockIdx.x >> 3);
    if (id >= end) return;
    auto origin = [&](uint32_t i, uint32_t& m, uint32_t& n) {
        const uint32_t band = i / (8 * nt), high = min(mt - band * 8, 8u), in = i - band * 8 * nt;
        m = (band * 8 + in % high) * 256;
        n = in / high * 256;
    };

    // this thread's part of a move of 64 rows; those of w are 32 rows of each of two waves' 64
    const int r = threadIdx.x >> 3, c = swizzle(r, threadIdx.x & 7), rw = (r & 31) + (r >> 5) * 64;
    const uint32_t vx = static_cast<uint32_t>(r) * static_cast<uint32_t>(p.xs) * 2 + c * 16;
    const uint32_t vw = static_cast<uint32_t>(rw) * static_cast<uint32_t>(p.ws) * 2 + c * 16;
    const int rows8 = wave * 8, rows8w = (rows8 & 31) + (rows8 >> 5) * 64;
    struct Source {
        const char *x, *w;  // the tile's first rows, at the step to be moved
    };
    const uint64_t xhop = static_cast<uint64_t>(p.xs) * 2, whop = static_cast<uint64_t>(p.ws) * 2;
    auto move_x = [&](const Source& f, int slot, int g, int i) {
        move16(f.x + (i * 128 + g * 64) * xhop, vx, buf + slot * STEP + (i * 128 + g * 64 + rows8) * 64);
    };
    auto move_w = [&](const Source& f, int slot, int g, int i) {
        move16(f.w + (i * 128 + g * 32) * whop, vw, buf + slot * STEP + (256 + i * 128 + g * 32 + rows8w) * 64);
    };
    Vec<T, 8> fx[4][4], fw[2][4];
    // a lane's place in a row of LDS: rows of operands differ by multiples of 32, so the swizzle is the lane's
    int at[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) at[s] = l * 64 + swizzle(l, s * 2 + h) * 8;
    auto read_x = [&](int slot, int j, int s) {
        fx[j][s] = *reinterpret_cast<const Vec<T, 8>*>(buf + slot * STEP + (wm + j * 32) * 64 + at[s]);
    };
    auto read_w = [&](int slot, int i, int s) {
        fw[i][s] = *reinterpret_cast<const Vec<T, 8>*>(buf + slot * STEP + (256 + wn + i * 32) * 64 + at[s]);
    };
    f32x16 acc[2][4];
    // Eight matrix instructions; `between` puts the phase's reads and moves between them, one or two at a time:
    // issued in a row they would keep the wave from its products until the memory pipes have taken them all.
    auto product = [&](int i, int j, auto between) {
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            acc[i][j + (n & 1)] = Mma<T>::go(fw[i][n >> 1], fx[j + (n & 1)][n >> 1], acc[i][j + (n & 1)]);
            __builtin_amdgcn_sched_barrier(0);
            between(n);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    const uint32_t steps = p.inner / 64;
    uint32_t m0, n0;
    origin(id, m0, n0);
    auto source = [&](uint32_t m, uint32_t n) {
        return Source{static_cast<const char*>(p.x) + min(m, p.rows - 256) * xhop, static_cast<const char*>(p.w) + min(n, p.cols - 256) * whop};
    };
    Source from = source(m0, n0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) move_x(from, t, 0, i), move_w(from, t, 0, i);
#pragma unroll
        for (int i = 0; i < 2; ++i) move_w(from, t, 1, i);
#pragma unroll
        for (int i = 0; i < 2; ++i) move_x(from, t, 1, i);
        from.x += 128;
        from.w += 128;
    }
    meet<12>();
    int slot = 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) read_x(0, 0, n), read_x(0, 1, n), read_w(0, 0, n);
    while (true) {
        const uint32_t next = id + stride;
        uint32_t mn = m0, nn = n0;
        if (next < end) origin(next, mn, nn);  // else the moves past the end repeat this tile's, unread
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = f32x16{};
        for (uint32_t t = 0; t < steps; ++t) {
            if (t + 2 == steps) from = source(mn, nn);
            // the moves in flight at a meeting, from the oldest: the quarter that the phase reads is the first of them
            meet<10>();
            product(0, 0, [&](int n) {
                if (n < 4) read_w(slot, 1, n);
            });
            meet<8>();
            product(1, 0, [&](int n) {
                read_x(slot, 2 + (n & 1), n >> 1);
                if (n & 1) (n & 2) ? move_w(from, slot, 0, n >> 2) : move_x(from, slot, 0, n >> 2);
            });
            meet<12>();
            product(0, 2, [&](int n) {
                if ((n & 3) == 1) move_w(from, slot, 1, n >> 2);
            });
            meet<10>();
            product(1, 2, [&](int n) {
                if (n < 4) {
                    read_w(slot ^ 1, 0, n);
                    read_x(slot ^ 1, 0, n);
                } else {
                    read_x(slot ^ 1, 1, n - 4);
                    if (n & 1) move_x(from, slot, 1, (n - 4) >> 1);
                }
            });
            from.x += 128;
            from.w += 128;
            slot ^= 1;
        }
        // results: 16 rows at a time through the wave's 4 KB, then 8 adjacent columns a lane, the same for all rows:
        // bias once, residuals 16 rows ahead
        const uint32_t ms = min(m0, p.rows - 256), ns = min(n0, p.cols - 256);
        const uint32_t col = ns + wn + (lane & 7) * 8, top = ms + wm + (lane >> 3);
        Vec<T, 8> bias = {};
        if (p.bias) bias = load_any<T, 8>(static_cast<const T*>(p.bias) + col);
        Vec<O, 8> res[2] = {};
        auto residual = [&](int g, int k) {
            return load_any<O, 8>(static_cast<const O*>(p.residual) + static_cast<int64_t>(top + g * 16 + k * 8) * p.rs + col);
        };
        if (p.residual) {
#pragma unroll
            for (int k = 0; k < 2; ++k) res[k] = residual(0, k);
        }
        auto put = [&](auto J, int half) {
            constexpr int j = decltype(J)::value;
            if ((l >> 4) == half) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<f32x4*>(turn + (l & 15) * 64 + ((i * 8 + q * 2 + h) ^ (l & 15)) * 4) =
                            f32x4{acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
            }
        };
#pragma unroll 1
        for (int g = 0; g < 8; ++g) {  // not unrolled: the epilogue's code stays in the instruction cache
            const int half = g & 1;
            switch (g >> 1) {
                case 0: put(std::integral_constant<int, 0>(), half); break;
                case 1: put(std::integral_constant<int, 1>(), half); break;
                case 2: put(std::integral_constant<int, 2>(), half); break;
                default: put(std::integral_constant<int, 3>(), half); break;
            }
            Vec<O, 8> soon[2] = {};
            if (p.residual && g < 7) {
#pragma unroll
                for (int k = 0; k < 2; ++k) soon[k] = residual(g + 1, k);
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int rr = k * 8 + (lane >> 3), cc = (lane & 7) * 2;
                const f32x4 z0 = *reinterpret_cast<const f32x4*>(turn + rr * 64 + (cc ^ rr) * 4);
                const f32x4 z1 = *reinterpret_cast<const f32x4*>(turn + rr * 64 + ((cc + 1) ^ rr) * 4);
                float z[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = (e < 4 ? z0[e] : z1[e - 4]) + static_cast<float>(bias[e]);
                activate(z, p.act);
                Vec<O, 8> o;
#pragma unroll
                for (int e = 0; e < 8; ++e) o[e] = static_cast<O>(z[e] + static_cast<float>(res[k][e]));
                const uint32_t row = top + g * 16 + k * 8;
                if (row < m0) continue;
                O* out = static_cast<O*>(p.out) + static_cast<int64_t>(row) * p.os + col;
                if (col >= n0) {
                    store_any<O, 8>(out, o);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (col + e >= n0) out[e] = o[e];
                }
            }
            res[0] = soon[0];
            res[1] = soon[1];
            __builtin_amdgcn_wave_barrier();
        }
        if (next >= end) break;
        id = next;
        m0 = mn;
        n0 = nn;
    }
    __builtin_amdgcn_s_waitcnt(0);  // moves into this workgroup's LDS end before it does
}

// Rows up to which the weight is streamed: 17 x 4096 -> 4096 12 us, 40 with the tiles of 64; 48 and 64 rows would take
// 18.3 and 20.7, against 15.0 and 14.8.
constexpr uint32_t FEW = 32;

uint64_t tiles_of(uint64_t rows, uint32_t cols, uint32_t high, uint32_t wide) { return (rows + high - 1) / high * ((cols + wide - 1) / wide); }
uint64_t tiles_of(uint64_t rows, uint32_t cols, uint32_t size) { return tiles_of(rows, cols, size, size); }

// Pieces of the inner dimension for tiles of 64, where they leave compute units idle: three at least, of 1024 elements
// at least, to be worth the second launch.  With and without: 64 x 8192 -> 1024 12.2 and 31.6 us, 64 x 4096 -> 4096 12.2
// and 17.7, but two pieces of 512 x 2048 -> 768 12.0 and 10.8, of 700 x 4096 -> 1000 18.5 and 18.1.  (Pieces of 512
// elements: 14.5 us for the first, 14.3 for the second.)  Where rows cannot be 16-byte aligned a step takes twice the
// time and two are enough: 64 x 2500 -> 1024 16.4 and 25.0.
uint32_t splits_of(uint64_t rows, uint32_t inner, uint32_t cols) {
    if (rows <= FEW) return 1;
    const uint64_t tiles = tiles_of(rows, cols, 64);
    const uint32_t want = static_cast<uint32_t>(std::min<uint64_t>(2 * CUS / tiles, inner / 1024));
    if (want < (inner % 8 ? 2 : 3)) return 1;
    const uint32_t steps = (inner + 63) / 64, piece = (steps + want - 1) / want;
    return (steps + piece - 1) / piece;
}

template <typename T, typename O, typename C, bool Direct>
int start(const Params& p, hipStream_t s) {
    auto* k = linear_kernel<T, O, C, Direct>;
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_lds(reinterpret_cast<const void*>(k), C::LDS, done)) return rc;
    const uint32_t tiles = (p.cols + C::BN - 1) / C::BN * ((p.rows + C::BM - 1) / C::BM);
    k<<<dim3(tiles, p.splits), C::THREADS, C::LDS, s>>>(p);
    if (p.splits > 1) {
        const uint64_t quads = static_cast<uint64_t>(p.rows) * ((p.cols + 3) / 4);
        linear_join_kernel<T, O><<<static_cast<uint32_t>((quads + 255) / 256), 256, 0, s>>>(p);
    }
    return BS_OK;
}
template <typename T, typename O>
int start_big(const Params& p, hipStream_t s) {
    constexpr int LDS = 160 * 1024;
    auto* k = linear_big_kernel<T, O>;
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_lds(reinterpret_cast<const void*>(k), LDS, done)) return rc;
    const uint32_t tiles = (p.cols + 255) / 256 * ((p.rows + 255) / 256);
    k<<<tiles < CUS ? (tiles + 7) / 8 * 8 : CUS, 512, LDS, s>>>(p);
    return BS_OK;
}
template <typename T, typename O, int MT>
int start_few(const Params& p, hipStream_t s) {
    // 32 columns a workgroup, half the reads of x, where that leaves a workgroup for every compute unit:
    // 17 x 8192 -> 8192 takes 35 us instead of 46
    if (p.cols >= 32 * CUS)
        linear_few_kernel<T, O, MT, 2><<<(p.cols + 31) / 32, 512, 0, s>>>(p);
    else
        linear_few_kernel<T, O, MT, 1><<<(p.cols + 15) / 16, 512, 0, s>>>(p);
    return BS_OK;
}

template <typename T, typename O>
int launch(const Params& p, hipStream_t s) {
    if (p.rows <= FEW) return p.rows <= 16 ? start_few<T, O, 1>(p, s) : start_few<T, O, 2>(p, s);
    const bool direct = aligned16(p.x) && aligned16(p.w) && p.xs % 8 == 0 && p.ws % 8 == 0;
    // Tiles of 256 where they fill the compute units' rounds to 0.55 at least.  Big and Mid: 4096 x 4096 -> 4096 (1.0)
    // 113 and 163 us, -> 3584 (0.88) 102 and 149, 3000 x 1024 -> 4096 (0.75) 33.6 and 38, 2304 x 4096 -> 4096 (0.56) 88
    // and 110, but 4096 x 1024 -> 4352 (0.53) 62 and 55, 2048 x 4096 -> 4096 (0.5) 86 and 81.
    auto fill = [](uint64_t tiles) { return static_cast<float>(tiles) / static_cast<float>((tiles + CUS - 1) / CUS * CUS); };
    if (fill(tiles_of(p.rows, p.cols, 256)) >= 0.55f && direct && p.rows >= 256 && p.cols >= 256 && p.inner % 64 == 0 && p.inner >= 128 &&
        p.xs < (1 << 22) && p.ws < (1 << 22))
        return start_big<T, O>(p, s);
    // Tall and Mid: 2048 x 4096 -> 4096 (1.0) 73 and 90 us, 8192 x 1024 -> 1024 (1.0) 24 and 27, 3000 x 2048 -> 2048 (0.75)
    // 35 and 40, but 2048 x 1024 -> 2048 (0.5) 20 and 16
    if (fill(tiles_of(p.rows, p.cols, 256, 128)) >= 0.75f && direct) return start<T, O, Tall, true>(p, s);
    // Mid and Small: 2048 x 4096 -> 2048 (256 tiles of 128) 42 and 53 us, 1024 x 4096 -> 2048 (128) 38 and 28
    if (tiles_of(p.rows, p.cols, 128) >= CUS) return direct ? start<T, O, Mid, true>(p, s) : start<T, O, Mid, false>(p, s);
    return direct ? start<T, O, Small, true>(p, s) : start<T, O, Small, false>(p, s);
}

int check(const char* what, uint64_t rows, uint32_t inner, uint32_t cols) {
    const std::string w = what;
    if (rows > 0x7FFFFFFFull) return refuse(w + ": rows must be < 2^31");
    if (inner == 0 || inner > (1u << 24) || cols == 0 || cols > (1u << 24)) return refuse(w + ": inner and cols must be in 1..2^24");
    // A grid of 2^32 threads is cut short without an error.  Tiles of 256 x 128 by 512 threads and of 128 x 128 by 256 have the
    // most; smaller ones run where those are few.
    if ((rows + 255) / 256 * 512 * ((cols + 127) / 128) > 0xFFFFFFFFull) return refuse(w + ": rows x cols is too large for one launch");
    return BS_OK;
}

}  // namespace

extern "C" int bs_linear_workspace(uint64_t rows, uint32_t inner, uint32_t cols, uint64_t* bytes) try {
    if (!bytes) return refuse("bs_linear_workspace: bytes is null");
    if (const int rc = check("bs_linear_workspace", rows, inner, cols)) return rc;
    const uint32_t splits = splits_of(rows, inner, cols);
    *bytes = splits > 1 ? splits * rows * cols * sizeof(float) : 0;
    return BS_OK;
} catch (...) {
    return bs_internal_exception();
}

extern "C" int bs_linear(const void* x, int64_t x_stride, const void* w, int64_t w_stride, const void* bias, const void* residual,
                         int64_t residual_stride, void* out, int64_t out_stride, uint64_t rows, uint32_t inner, uint32_t cols,
                         int type, int out_type, int activation, void* workspace, uint64_t workspace_bytes, void* stream) try {
    if (const int rc = check("bs_linear", rows, inner, cols)) return rc;
    if (type != BS_F16 && type != BS_BF16) return refuse("bs_linear: type must be BS_F16 or BS_BF16");
    if (out_type != type && out_type != BS_F32) return refuse("bs_linear: out_type must be type or BS_F32");
    if (activation < BS_ACT_NONE || activation > BS_ACT_SILU) return refuse("bs_linear: unknown activation " + std::to_string(activation));
    if (rows == 0) return BS_OK;
    if (!x || !w || !out) return refuse("bs_linear: x, w and out must be given");
    if (x_stride < inner || w_stride < inner || out_stride < cols || (residual && residual_stride < cols))
        return refuse("bs_linear: rows overlap (a stride is shorter than its row)");
    if (x_stride >= (1 << 24) || w_stride >= (1 << 24) || out_stride >= (1 << 24) || (residual && residual_stride >= (1 << 24)))
        return refuse("bs_linear: strides must be < 2^24");
    const uint32_t splits = splits_of(rows, inner, cols);
    if (splits > 1) {
        const uint64_t need = splits * rows * cols * sizeof(float);
        if (!workspace || workspace_bytes < need) return refuse("bs_linear: the workspace must hold " + std::to_string(need) + " bytes");
        if (!aligned16(workspace)) return refuse("bs_linear: the workspace must be 16-byte aligned");
    }
    const Params p{x, w, bias, residual, out, x_stride, w_stride, residual_stride, out_stride, static_cast<uint32_t>(rows), inner, cols, activation,
                   splits, static_cast<float*>(workspace)};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int rc = type == BS_F16 ? (out_type == BS_F32 ? launch<f16, float>(p, s) : launch<f16, f16>(p, s))
                                  : (out_type == BS_F32 ? launch<bf16, float>(p, s) : launch<bf16, bf16>(p, s));
    return rc ? rc : launched("bs_linear");
} catch (...) {
    return bs_internal_exception();
}
