// Gated products and their gradients (include/bs_embed.h).
//
//   h  = act(g) u,  g = x wg^T,  u = x wu^T
//   dg = dh u act'(g),  du = dh act(g):  rows of d = (dg | du), in the workspace
//   dx = dg wg + du wu,  dwg = dg^T x,  dwu = du^T x
//
// Three kinds of products, all of an operand X, whose rows are the result's rows, and an operand W, whose rows are its
// columns:
//   GATED    X = x (rows x inner), W = 32 rows of wg, 32 of wu, and so on, so that a wave has g and u of the same results
//   INPUT    X = d (rows x 2 cols), W = the columns of wg over those of wu
//   WEIGHTS  X = the columns of d, W = the columns of x: the inner dimension is the rows
// Where an operand's rows are columns in memory, its tile lies in LDS as in memory, an inner element per row, and is read
// by transposing LDS reads.
#include "bs_product.hpp"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace {
using namespace bse;

enum { GATED = 0, INPUT = 1, WEIGHTS = 2 };

struct Params {
    const void *x, *wg, *wu;
    int64_t xs, wgs, wus;
    void *h, *gate, *up;  // GATED; gate and up may be null
    int64_t hs;
    const void *dh, *g, *u;
    int64_t dhs, gs, us;
    void *dx, *dwg, *dwu;
    char* d;      // rows_up x 2 cols, rows past the last are 0
    char* tail;   // the last rows % 64 rows of x, then zeros: 64 x inner
    uint32_t rows, inner, cols;
    int act;
    uint32_t input_splits, weight_splits;  // pieces of the gradients' inner dimensions; > 1: their sums go to
    float *input_parts, *weight_parts;     // splits x the result
};

// ------------------------------------------------------------------------------------------------ d

// 1 / (1 + e) and e / (1 + e) for e = 2^v, neither by a difference; 0 and 1 past 2^126, for a 1 / (1 + e) that stopped at 2^-126
// would give far gates values and slopes that grow with them
__device__ inline void halves_of_one(float v, float& s, float& rest) {
    const float e = __builtin_amdgcn_exp2f(fminf(v, 126.0f));
    s = __builtin_amdgcn_rcpf(1.0f + e);
    rest = e * s;
    s = v > 126.0f ? 0.0f : s;
}
// An activation and its slope.  An infinite gate, a finite product past the type's range (65504 in float16) that the forward call
// took as it was, has their limits: factors that vanish there are not multiplied by it.
__device__ inline void act_and_slope(float z, int act, float& a, float& slope) {
    if (act == BS_ACT_RELU) {
        a = z < 0.0f ? 0.0f : z;
        slope = z > 0.0f ? 1.0f : z <= 0.0f ? 0.0f : z;  // NaN as it is
    } else if (act == BS_ACT_GELU) {  // P = (1 + erf(z / sqrt 2)) / 2: slope P + z exp(-z^2 / 2) / sqrt(2 pi)
        const float e = __builtin_amdgcn_exp2f(z * z * (-0.5f * LOG2E)), part = gelu_part(z, e);
        a = part == 0.0f ? 0.0f : z * part;
        slope = e == 0.0f ? part : fmaf(z * 0.3989422804014327f, e, part);
    } else if (act == BS_ACT_GELU_TANH) {  // z s, s = 1 / (1 + exp(-2 v)): slope s + z s (1 - s) 2 v'
        const float q = z * z;
        float s, rest;
        halves_of_one(-2.0f * LOG2E * 0.79788456080286536f * fmaf(0.044715f * q, z, z), s, rest);
        a = s == 0.0f ? 0.0f : z * s;
        const float bend = s * rest;
        slope = bend == 0.0f ? s : fmaf(z * bend, 2.0f * 0.79788456080286536f * fmaf(3.0f * 0.044715f, q, 1.0f), s);
    } else if (act == BS_ACT_SILU) {  // z s, s = 1 / (1 + exp(-z)): slope s + z s (1 - s)
        float s, rest;
        halves_of_one(-LOG2E * z, s, rest);
        a = s == 0.0f ? 0.0f : z * s;
        const float bend = s * rest;
        slope = bend == 0.0f ? s : fmaf(z, bend, s);
    } else {
        a = z;
        slope = 1.0f;
    }
}

// d, 8 columns a thread; the rows past the last are 0 and so are those of x's tail.  dg and du are rounded to the inputs' type
// for their products, as every operand of a matrix product is: off by half a unit each, at random, which gives a sum of n of
// them the error that the same sum of rounded inputs has.  Memory bounds it: 8191 x 4096 takes 52 us, 335 MB at 6.5 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void gated_slopes_kernel(Params p, uint32_t rows_up, uint32_t tail_rows, Divisor by_across) {
    const uint32_t across = (p.cols + 7) / 8, wide = (p.inner + 7) / 8;
    const uint64_t all = static_cast<uint64_t>(rows_up) * across, more = static_cast<uint64_t>(tail_rows) * wide;
    T* d = reinterpret_cast<T*>(p.d);
    for (uint64_t i = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; i < all + more; i += static_cast<uint64_t>(gridDim.x) * 256) {
        if (i >= all) {
            const uint32_t r = static_cast<uint32_t>((i - all) / wide), c = static_cast<uint32_t>((i - all) % wide) * 8, row = rows_up - tail_rows + r;
            const int n = static_cast<int>(p.inner - c);
            Vec<T, 8> v = {};
            if (row < p.rows) v = load_some<T, 8>(static_cast<const T*>(p.x) + static_cast<int64_t>(row) * p.xs + c, n);
            store_some<T, 8>(reinterpret_cast<T*>(p.tail) + static_cast<size_t>(r) * p.inner + c, v, n);
            continue;
        }
        const uint32_t row = all >> 31 ? static_cast<uint32_t>(i / across) : by_across.quotient(static_cast<uint32_t>(i)), c = static_cast<uint32_t>(i - static_cast<uint64_t>(row) * across) * 8;
        const int n = static_cast<int>(p.cols - c);
        Vec<T, 8> dg = {}, du = {};
        if (row < p.rows) {
            const Vec<T, 8> h = load_some<T, 8>(static_cast<const T*>(p.dh) + static_cast<int64_t>(row) * p.dhs + c, n);
            const Vec<T, 8> g = load_some<T, 8>(static_cast<const T*>(p.g) + static_cast<int64_t>(row) * p.gs + c, n);
            const Vec<T, 8> u = load_some<T, 8>(static_cast<const T*>(p.u) + static_cast<int64_t>(row) * p.us + c, n);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float a, slope;
                act_and_slope(static_cast<float>(g[j]), p.act, a, slope);
                dg[j] = static_cast<T>(static_cast<float>(h[j]) * static_cast<float>(u[j]) * slope);
                du[j] = static_cast<T>(static_cast<float>(h[j]) * a);
            }
        }
        store_some<T, 8>(d + static_cast<size_t>(row) * 2 * p.cols + c, dg, n);
        store_some<T, 8>(d + static_cast<size_t>(row) * 2 * p.cols + p.cols + c, du, n);
    }
}

// ------------------------------------------------------------------------------------------------ results

// the sizes of a product: rows and columns of its result, inner elements
template <int FORM>
__device__ __host__ inline uint32_t rows_of(const Params& p) { return FORM == WEIGHTS ? 2 * p.cols : p.rows; }
template <int FORM>
__device__ __host__ inline uint32_t cols_of(const Params& p) { return FORM == GATED ? p.cols : p.inner; }
template <int FORM>
__device__ __host__ inline uint32_t inner_of(const Params& p) { return FORM == GATED ? p.inner : FORM == INPUT ? 2 * p.cols : p.rows; }

// a row of the result, and N adjacent ones of it, those inside
template <typename T, int FORM>
__device__ inline T* row_of(const Params& p, uint32_t row) {
    if (FORM == INPUT) return static_cast<T*>(p.dx) + static_cast<size_t>(row) * p.inner;
    return row < p.cols ? static_cast<T*>(p.dwg) + static_cast<size_t>(row) * p.inner : static_cast<T*>(p.dwu) + static_cast<size_t>(row - p.cols) * p.inner;
}
template <typename T, int FORM, int N>
__device__ inline void write(const Params& p, uint32_t row, uint32_t col, const float (&z)[N]) {
    Vec<T, N> o;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = static_cast<T>(z[j]);
    store_some<T, N>(row_of<T, FORM>(p, row) + col, o, static_cast<int>(p.inner - col));
}
template <typename T, int N>
__device__ inline void write_gated(const Params& p, uint32_t row, uint32_t col, float (&g)[N], const float (&u)[N]) {
    const int n = static_cast<int>(p.cols - col);
    Vec<T, N> o;
    if (p.gate) {
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = static_cast<T>(g[j]);
        store_some<T, N>(static_cast<T*>(p.gate) + static_cast<size_t>(row) * p.cols + col, o, n);
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = static_cast<T>(u[j]);
        store_some<T, N>(static_cast<T*>(p.up) + static_cast<size_t>(row) * p.cols + col, o, n);
    }
    activate(g, p.act);
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] = static_cast<T>(g[j] * u[j]);
    store_some<T, N>(static_cast<T*>(p.h) + static_cast<int64_t>(row) * p.hs + col, o, n);
}

// ------------------------------------------------------------------------------------------------ tiles

// 8 inner elements of a lane's row of an operand whose inner elements are rows of S bytes in LDS: lanes 16 g .. 16 g + 15 read
// 4 rows x 16 columns and get a column's 4 rows each
template <typename T, int S>
__device__ inline Vec<T, 8> read_across(const char* tile, int inner, int column, int lane) {
    const int k = inner + (lane >> 5) * 8 + ((lane & 15) >> 2), e = column + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    const s16x4 lo = read_transposed(tile + place<S>(k, e >> 3) + (e & 7) * 2);
    const s16x4 hi = read_transposed(tile + place<S>(k + 4, e >> 3) + (e & 7) * 2);
    return __builtin_bit_cast(Vec<T, 8>, Vec<short, 8>{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
}

// Tiles of any size and alignment, two workgroups per compute unit.  1000 x 1024 -> 4096 takes 24 us (700 TFLOP/s), 300 x 768 ->
// 2048 8.7, most of it the latency of its 12 steps and a launch.  Direct: operands are 16-byte aligned, whole steps go from
// memory to LDS without registers.  Tile `b` of the product; of its inner dimension piece y of `splits`, whose sums go to `parts`
// if there are several.
template <typename T, int FORM, typename C, bool Direct>
__device__ inline void one_tile(const Params& p, char* lds, uint32_t b, uint32_t y, uint32_t splits, float* parts) {
    constexpr bool XT = FORM == WEIGHTS, WT = FORM != GATED;  // the operand's rows are columns in memory
    constexpr int OUT = FORM == GATED ? C::BN / 2 : C::BN;    // columns of the result in a tile
    T* buf = reinterpret_cast<T*>(lds);
    const uint32_t rows = rows_of<FORM>(p), cols = cols_of<FORM>(p), inner = inner_of<FORM>(p);
    // Workgroup b runs on XCD b mod 8: each XCD takes a contiguous run of tiles, 8 tile rows high, so that
    // the tiles in flight on it share operands in its L2.
    const uint32_t mt = (rows + C::BM - 1) / C::BM, nt = (cols + OUT - 1) / OUT, total = mt * nt;
    const uint32_t xcd = b & 7, q8 = total >> 3, r8 = total & 7;
    const uint32_t id = xcd * q8 + (xcd < r8 ? xcd : r8) + (b >> 3);
    const uint32_t band = id / (8 * nt), high = mt - band * 8 < 8 ? mt - band * 8 : 8, in = id - band * 8 * nt;
    const uint32_t m0 = (band * 8 + in % high) * C::BM, n0 = in / high * OUT;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 31, h = lane >> 5;
    const int wm = wave / C::WN * C::TM * 32, wn = wave % C::WN * C::TN * 32;
    constexpr int XMOVES = C::BM * C::BK / 8 / C::THREADS;

    // A thread's moves: 16 bytes each, to LDS positions that are linear over the workgroup.  Of an operand that lies in LDS as
    // rows of the result: row `line` of it, inner elements `at` on; of one that lies there as rows of inner elements: inner
    // element `line`, results `at` on.
    auto spot = [&](int i, int& line, int& at) {
        const int k = i * C::THREADS + static_cast<int>(threadIdx.x);
        if (i < XMOVES ? XT : WT) {
            const int w = i < XMOVES ? C::BM : C::BN, j = i < XMOVES ? k : k - C::BM * C::BK / 8;
            line = j / (w / 8);
            const int c = j % (w / 8);
            at = (w == 64 ? (place<128>(line, c) - line * 128) : w == 128 ? (place<256>(line, c) - line * 256) : (place<512>(line, c) - line * 512)) / 2;
        } else {
            line = (k / C::CH) - (i < XMOVES ? 0 : C::BM);
            at = C::swizzle(k / C::CH, k % C::CH) * 8;
        }
    };
    // where the 8 elements of a move come from, at inner element k0 of the product, and how many of them there are
    auto source = [&](int i, uint32_t k0, int& n) -> const T* {
        int line, at;
        spot(i, line, at);
        if (i < XMOVES) {
            if (XT) {
                const uint32_t k = k0 + line, m = m0 + at;
                n = k < inner && m < rows ? static_cast<int>(rows - m) : 0;
                return reinterpret_cast<const T*>(p.d) + static_cast<size_t>(k) * 2 * p.cols + m;
            }
            const uint32_t m = min(m0 + line, rows - 1), k = k0 + at;  // rows past the end repeat the last one: their products are not stored
            n = static_cast<int>(inner) - static_cast<int>(k);
            return FORM == GATED ? static_cast<const T*>(p.x) + static_cast<int64_t>(m) * p.xs + k : reinterpret_cast<const T*>(p.d) + static_cast<size_t>(m) * 2 * p.cols + k;
        }
        if (WT) {
            const uint32_t k = k0 + line, c = n0 + at;
            n = k < inner && c < cols ? static_cast<int>(cols - c) : 0;
            if (FORM == WEIGHTS) return static_cast<const T*>(p.x) + static_cast<int64_t>(k) * p.xs + c;
            return k < p.cols ? static_cast<const T*>(p.wg) + static_cast<int64_t>(k) * p.wgs + c : static_cast<const T*>(p.wu) + static_cast<int64_t>(k - p.cols) * p.wus + c;
        }
        const uint32_t c = min(n0 + (line >> 6) * 32 + (line & 31), cols - 1), k = k0 + at;
        n = static_cast<int>(inner) - static_cast<int>(k);
        return line & 32 ? static_cast<const T*>(p.wu) + static_cast<int64_t>(c) * p.wus + k : static_cast<const T*>(p.wg) + static_cast<int64_t>(c) * p.wgs + k;
    };
    // this workgroup's piece: whole steps [begin, whole), and for the last piece what is left after them
    const uint32_t allsteps = (inner + C::BK - 1) / C::BK, piece = (allsteps + splits - 1) / splits;
    const uint32_t begin = y * piece, steps = min(begin + piece, allsteps), whole = min(steps, inner / C::BK);
    auto fetch = [&](uint32_t t, Vec<T, 8> (&v)[C::MOVES]) {
#pragma unroll
        for (int i = 0; i < C::MOVES; ++i) {
            int n;
            const T* from = source(i, t * C::BK, n);
            v[i] = n > 0 ? load_some<T, 8>(from, n) : Vec<T, 8>{};
        }
    };
    auto put = [&](int slot, const Vec<T, 8> (&v)[C::MOVES]) {
#pragma unroll
        for (int i = 0; i < C::MOVES; ++i) *reinterpret_cast<Vec<T, 8>*>(buf + slot * C::STEP + (i * C::THREADS + threadIdx.x) * 8) = v[i];
    };
    f32x16 acc[C::TN][C::TM] = {};
    struct Parts {
        Vec<T, 8> a[C::TN], b[C::TM];
    };
    auto read = [&](int slot, int s, Parts& f) {  // 16 inner elements
        const T* tx = buf + slot * C::STEP;
        const T* tw = tx + C::BM * C::BK;
#pragma unroll
        for (int i = 0; i < C::TN; ++i)
            f.a[i] = WT ? read_across<T, C::BN * 2>(reinterpret_cast<const char*>(tw), s * 16, wn + i * 32, lane)
                        : *reinterpret_cast<const Vec<T, 8>*>(tw + C::place(wn + i * 32 + l, s * 2 + h));
#pragma unroll
        for (int j = 0; j < C::TM; ++j)
            f.b[j] = XT ? read_across<T, C::BM * 2>(reinterpret_cast<const char*>(tx), s * 16, wm + j * 32, lane)
                        : *reinterpret_cast<const Vec<T, 8>*>(tx + C::place(wm + j * 32 + l, s * 2 + h));
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
        // whole steps: no inner element is past the end; results past it repeat the last 8, and are not stored
        const T* from[C::MOVES];
#pragma unroll
        for (int i = 0; i < C::MOVES; ++i) {
            int line, at, n;
            spot(i, line, at);
            from[i] = source(i, 0, n);
            if (i < XMOVES) {
                if (XT) from[i] = reinterpret_cast<const T*>(p.d) + static_cast<size_t>(line) * 2 * p.cols + min(m0 + at, rows - 8);
            } else if (WT) {
                const uint32_t c = min(n0 + at, cols - 8);
                from[i] = FORM == WEIGHTS ? static_cast<const T*>(p.x) + static_cast<int64_t>(line) * p.xs + c : static_cast<const T*>(p.wg) + static_cast<int64_t>(line) * p.wgs + c;
            }
        }
        auto move = [&](uint32_t t, int slot) {
            const size_t k = static_cast<size_t>(t) * C::BK;
            // elements from step 0 to step t of an operand
            const int64_t xhop = XT ? static_cast<int64_t>(k) * 2 * p.cols : static_cast<int64_t>(k);
            int64_t whop = static_cast<int64_t>(k);
            if (FORM == WEIGHTS) whop *= p.xs;
            if (FORM == INPUT)  // cols is a multiple of the step; strides of both weights are alike
                whop = k < p.cols ? whop * p.wgs : (static_cast<const T*>(p.wu) - static_cast<const T*>(p.wg)) + (whop - p.cols) * p.wgs;
#pragma unroll
            for (int i = 0; i < C::MOVES; ++i)
                __builtin_amdgcn_global_load_lds((global_ptr)(from[i] + (i < XMOVES ? xhop : whop)),
                                                 (lds_ptr)(buf + slot * C::STEP + (i * C::THREADS + wave * 64) * 8), 16, 0, 0);
        };
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
        if (steps > whole && begin <= whole) {
            Vec<T, 8> v[C::MOVES];
            fetch(whole, v);
            put(0, v);
            __syncthreads();
            multiply(0);
            __syncthreads();
        }
    } else {
        Vec<T, 8> v[C::MOVES];
        if (steps > begin) {
            fetch(begin, v);
            put(begin & 1, v);
        }
        for (uint32_t t = begin; t < steps; ++t) {
            __syncthreads();
            if (t + 1 < steps) fetch(t + 1, v);
            multiply(t & 1);
            if (t + 1 < steps) put(~t & 1, v);
        }
        __syncthreads();
    }
    // a wave turns 32 rows of its results at a time: a lane then has 8 adjacent columns (GATED: of both products)
    static_assert(FORM != GATED || C::TN == 2, "a wave has 32 columns of both products");
    constexpr int W = C::TN * 32, PITCH = W + 4, LANES = FORM == GATED ? 4 : W / 8;
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
    static_assert(C::TM <= 2, "cases below");
#pragma unroll 1
    for (int j = 0; j < C::TM; ++j) {  // not unrolled: the epilogue's code stays in the instruction cache
        if (j == 0)
            spread(std::integral_constant<int, 0>());
        else
            spread(std::integral_constant<int, 1>());
        __builtin_amdgcn_wave_barrier();
#pragma unroll 1
        for (int k = 0; k < 32 * LANES / 64; ++k) {
            const int r = k * (64 / LANES) + lane / LANES, c = lane % LANES * 8;
            const uint32_t row = m0 + wm + j * 32 + r, col = n0 + (FORM == GATED ? wn / 2 : wn) + c;
            float z[8], u[8];
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const f32x4 z4 = *reinterpret_cast<const f32x4*>(turn + r * PITCH + c + e);
#pragma unroll
                for (int x = 0; x < 4; ++x) z[e + x] = z4[x];
                if (FORM == GATED) {
                    const f32x4 u4 = *reinterpret_cast<const f32x4*>(turn + r * PITCH + 32 + c + e);
#pragma unroll
                    for (int x = 0; x < 4; ++x) u[e + x] = u4[x];
                }
            }
            if (row >= rows || col >= cols) continue;
            if constexpr (FORM == GATED) {
                write_gated<T, 8>(p, row, col, z, u);
            } else if (splits > 1) {
                float* part = parts + (static_cast<size_t>(y) * rows + row) * cols + col;
                store_some<float, 4>(part, f32x4{z[0], z[1], z[2], z[3]}, static_cast<int>(cols - col));
                if (cols - col > 4) store_some<float, 4>(part + 4, f32x4{z[4], z[5], z[6], z[7]}, static_cast<int>(cols - col) - 4);
            } else {
                write<T, FORM, 8>(p, row, col, z);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <typename T, typename C, bool Direct>
__global__ __launch_bounds__(C::THREADS, C::PER_CU * C::WAVES / 4) void gated_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    one_tile<T, GATED, C, Direct>(p, lds, blockIdx.x, 0, 1, nullptr);
}
// Both products of the gradients in one launch, `inputs` workgroups of dx first.
template <typename T, typename CI, typename CW, bool Direct>
__global__ __launch_bounds__(256, 2) void gated_backward_kernel(Params p, uint32_t input_tiles, uint32_t inputs, uint32_t weight_tiles) {
    static_assert(CI::THREADS == 256 && CW::THREADS == 256 && CI::PER_CU == 2 && CW::PER_CU == 2, "of one launch");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    if (blockIdx.x < inputs) {
        one_tile<T, INPUT, CI, Direct>(p, lds, blockIdx.x % input_tiles, blockIdx.x / input_tiles, p.input_splits, p.input_parts);
    } else {
        const uint32_t b = blockIdx.x - inputs;
        one_tile<T, WEIGHTS, CW, Direct>(p, lds, b % weight_tiles, b / weight_tiles, p.weight_splits, p.weight_parts);
    }
}

// the pieces' sums in order: a thread takes four adjacent columns of a row
template <typename T, int FORM>
__global__ __launch_bounds__(256) void gated_join_kernel(Params p) {
    const uint32_t rows = rows_of<FORM>(p), cols = cols_of<FORM>(p), across = (cols + 3) / 4;
    const uint64_t at = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x;
    const uint32_t row = static_cast<uint32_t>(at / across), col = static_cast<uint32_t>(at % across) * 4;
    if (row >= rows) return;
    const int n = static_cast<int>(cols - col);
    const uint32_t splits = FORM == INPUT ? p.input_splits : p.weight_splits;
    const float* part = (FORM == INPUT ? p.input_parts : p.weight_parts) + static_cast<size_t>(row) * cols + col;
    f32x4 s = load_some<float, 4>(part, n);
    for (uint32_t i = 1; i < splits; ++i) s += load_some<float, 4>(part + static_cast<size_t>(i) * rows * cols, n);
    const float z[4] = {s[0], s[1], s[2], s[3]};
    write<T, FORM, 4>(p, row, col, z);
}

// Few rows: both weights are read once, from memory to registers, and bound the time.  A workgroup has P x 16 rows of each, its
// eight waves a contiguous piece each of the inner dimension; x (MT x 16 rows) comes from the L2, as often as there are
// workgroups.  One row of 4096 -> 8192 takes 27.5 us (4.9 TB/s), 17 rows 30.7; 8 more steps' loads ahead spill (106 us).
template <typename T, int MT, int P>
__global__ __launch_bounds__(512) void gated_few_kernel(Params p) {
    constexpr int NT = 2 * P;  // tiles of 16 rows: of wg, wu, wg, ..
    __shared__ f32x4 join[8][NT * MT][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
    const uint32_t n0 = blockIdx.x * (P * 16);
    // rows past the end repeat the last one: their products are not stored
    const T *wp[NT], *xp[MT];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const uint32_t n = min(n0 + i * 16 + l, p.cols - 1);
        wp[2 * i] = static_cast<const T*>(p.wg) + static_cast<int64_t>(n) * p.wgs + g * 8;
        wp[2 * i + 1] = static_cast<const T*>(p.wu) + static_cast<int64_t>(n) * p.wus + g * 8;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) xp[i] = static_cast<const T*>(p.x) + static_cast<int64_t>(min(static_cast<uint32_t>(i * 16 + l), p.rows - 1)) * p.xs + g * 8;
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
    if (wave >= P * MT) return;
    // wave i MT + j: rows 16 j + l, columns 16 i + 4 g to + 3; the waves' sums in order
    const int gate = wave / MT * 2 * MT + wave % MT, up = gate + MT;
    f32x4 s = join[0][gate][lane], r = join[0][up][lane];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += join[k][gate][lane], r += join[k][up][lane];
    const uint32_t row = wave % MT * 16 + l, col = n0 + wave / MT * 16 + g * 4;
    float z[4] = {s[0], s[1], s[2], s[3]};
    const float u[4] = {r[0], r[1], r[2], r[3]};
    if (row < p.rows && col < p.cols) write_gated<T, 4>(p, row, col, z, u);
}

// ------------------------------------------------------------------------------------------------ large tiles

// Tiles of 256 rows of X x 256 rows of W by 8 waves of 128 x 64, inner steps of 64, two of them in LDS.  A step is four phases,
// and the quarters of its operands (x0, x1: the first and second 64 rows of every wave; w0, w1: the first and second 32) are
// read into registers a phase before their products, whereupon the moves of step t + 2 into that quarter start.
//   phase 0: read w1(t)              products w0 x0
//   phase 1: read x1(t)              products w1 x0    move x0, w0 (t + 2)
//   phase 2:                         products w0 x1    move w1 (t + 2)
//   phase 3: read x0, w0 (t + 1)     products w1 x1    move x1 (t + 2)
// GATED: w0 is of wg and w1 of wu.  Where an operand's rows are columns in memory, its quarters are its first and second 128
// rows, so that a line of a move is 256 bytes (of 64 bytes in w and 128 in x, as the waves' rows follow each other, the
// weights' gradients of 8192 x 4096 -> 4096 took 726 us), and lie in LDS as 64 inner elements x 128 rows.  A workgroup goes through its tiles without a break: the moves of the next tile's first steps are under way
// while a tile's results are written.  A tile that would pass an edge is shifted back inside and does not write what its
// neighbour writes.
//
// 8192 x 4096 -> 8192 takes 820-850 us by box (1290-1340 TFLOP/s; the library reaches 1407 at 8192 x 8192 x 8192), the matrix
// pipe busy for 0.75 of the time.  A step takes 3250 cycles, 2048 of them matrix instructions and as many LDS traffic (196 KB
// read, 64 KB moved, 128 bytes a cycle); with half as many meetings it takes as long.  A tile's first step takes 2500 more, behind
// its predecessor's writes, and its results 4800 cycles, with gelu 10800, with gate and up written too 14200: a fifth of the time
// at 1024 inner elements (8191 x 1024 -> 4096: 150-155 us).  Waiting for the next tile's moves before those writes, or counting
// the writes apart, did not pay (168 and 163 against 151-155).  Gradients of 8192 x 4096 -> 4096: 870 us with the pass for d, 1270
// TFLOP/s.
//
// The tiles run .. run + count - 1 of the product, 8 tile rows high; this workgroup's are those from `first` on, `stride` apart.
template <typename T, int FORM>
__device__ inline void big_tiles(const Params& p, char* lds, uint32_t run, uint32_t first, uint32_t count, uint32_t stride) {
    constexpr bool XT = FORM == WEIGHTS, WT = FORM != GATED;
    constexpr uint32_t OUT = FORM == GATED ? 128 : 256;  // columns of the result in a tile
    constexpr int STEP = 512 * 64;                       // elements: 256 rows of X, then 256 of W
    if (first >= count) return;
    T* buf = reinterpret_cast<T*>(lds);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane & 31, h = lane >> 5;
    char* turn = lds + 2 * STEP * 2 + wave * 4096;
    const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
    auto swizzle = [](int r, int c) { return c ^ ((r >> 1) & 7); };
    const uint32_t rows = rows_of<FORM>(p), cols = cols_of<FORM>(p);
    const uint32_t steps = FORM == GATED ? p.inner / 64 : FORM == INPUT ? p.cols / 32 : (p.rows + 63) / 64;
    const uint32_t mt = (rows + 255) / 256, nt = (cols + OUT - 1) / OUT;
    auto origin = [&](uint32_t i, uint32_t& m, uint32_t& n) {
        const uint32_t id = run + i, band = id / (8 * nt), high = min(mt - band * 8, 8u), in = id - band * 8 * nt;
        m = (band * 8 + in % high) * 256;
        n = in / high * OUT;
    };

    // bytes between the lines of an operand in memory, and this thread's part of a move: 64 lines of 64 inner elements, or 32
    // inner elements of 128 rows of the operand
    const uint64_t xhop = FORM == GATED ? static_cast<uint64_t>(p.xs) * 2 : static_cast<uint64_t>(p.cols) * 4;
    const uint64_t whop = FORM == WEIGHTS ? static_cast<uint64_t>(p.xs) * 2 : static_cast<uint64_t>(p.wgs) * 2;
    const int r = threadIdx.x >> 3, c = swizzle(r, threadIdx.x & 7);
    const int k = threadIdx.x >> 4, kc = (threadIdx.x & 15) ^ ((k & 3) << 2 | ((k >> 2) & 3));
    const uint32_t vx = XT ? k * static_cast<uint32_t>(xhop) + kc * 16 : r * static_cast<uint32_t>(xhop) + c * 16;
    const uint32_t vw = WT ? k * static_cast<uint32_t>(whop) + kc * 16 : r * static_cast<uint32_t>(whop) + c * 16;
    const uint32_t vtail = k * p.inner * 2 + kc * 16;  // WEIGHTS: in x's tail
    const int rows8 = wave * 8, rows8w = (rows8 & 31) + (rows8 >> 5) * 64;
    struct Source {
        const char *x, *w0, *w1;  // the tile's first lines at the step to be moved
        uint64_t whop;
        bool tail;
    } from;
    // the sources of step t of the tile at m, n
    auto point = [&](uint32_t m, uint32_t n, uint32_t t) {
        const uint64_t ms = min(m, rows - 256), ns = min(n, cols - OUT);
        from.whop = whop;
        from.tail = false;
        if (FORM == GATED) {
            from.x = static_cast<const char*>(p.x) + ms * xhop + t * 128ull;
            from.w0 = static_cast<const char*>(p.wg) + ns * whop + t * 128ull;
            from.w1 = static_cast<const char*>(p.wu) + ns * whop + t * 128ull;
        } else if (FORM == INPUT) {
            from.x = p.d + ms * xhop + t * 128ull;
            const uint32_t at = t * 64;
            from.w0 = (at < p.cols ? static_cast<const char*>(p.wg) + at * whop : static_cast<const char*>(p.wu) + (at - p.cols) * whop) + ns * 2;
            from.w1 = from.w0 + 256;
        } else {
            from.x = p.d + t * 64ull * xhop + ms * 2;
            from.tail = t * 64 + 64 > p.rows;
            from.whop = from.tail ? p.inner * 2ull : whop;
            from.w0 = (from.tail ? p.tail : static_cast<const char*>(p.x) + t * 64ull * whop) + ns * 2;
            from.w1 = from.w0 + 256;
        }
    };
    auto move_x = [&](int slot, int g, int i) {
        if (XT)
            move16(from.x + i * 32 * xhop + g * 256, vx, buf + slot * STEP + g * 8192 + i * 4096 + wave * 512);
        else
            move16(from.x + (i * 128 + g * 64) * xhop, vx, buf + slot * STEP + (i * 128 + g * 64 + rows8) * 64);
    };
    auto move_w = [&](int slot, int g, int i) {
        const char* w = g ? from.w1 : from.w0;
        if (WT)
            move16(w + i * 32 * from.whop, FORM == WEIGHTS && from.tail ? vtail : vw, buf + slot * STEP + 256 * 64 + g * 8192 + i * 4096 + wave * 512);
        else
            move16(w + i * 64 * whop, vw, buf + slot * STEP + (256 + i * 128 + g * 32 + rows8w) * 64);
    };
    Vec<T, 8> fx[4][4], fw[2][4];
    // a lane's places in LDS: of 16 inner elements in a row (rows of operands differ by multiples of 32, so the swizzle is the
    // lane's), or of 4 inner elements and the next 4 in a column
    int at[4], ax[2][2], aw[2];
#pragma unroll
    for (int s = 0; s < 4; ++s) at[s] = l * 64 + swizzle(l, s * 2 + h) * 8;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int kk = h * 8 + ((lane & 15) >> 2) + half * 4, e = ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
#pragma unroll
        for (int j = 0; j < 2; ++j) ax[j][half] = place<256>(kk, ((wave >> 2) * 64 + j * 32 + e) >> 3) + (e & 7) * 2;
        aw[half] = place<256>(kk, ((wave & 3) * 32 + e) >> 3) + (e & 7) * 2;
    }
    auto pair = [&](const T* base, int lo, int hi) {
        const s16x4 a = read_transposed(reinterpret_cast<const char*>(base) + lo), b = read_transposed(reinterpret_cast<const char*>(base) + hi);
        return __builtin_bit_cast(Vec<T, 8>, Vec<short, 8>{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
    };
    auto read_x = [&](int slot, int j, int s) {
        fx[j][s] = XT ? pair(buf + slot * STEP + (j >> 1) * 8192 + s * 2048, ax[j & 1][0], ax[j & 1][1])
                      : *reinterpret_cast<const Vec<T, 8>*>(buf + slot * STEP + (wm + j * 32) * 64 + at[s]);
    };
    auto read_w = [&](int slot, int i, int s) {
        fw[i][s] = WT ? pair(buf + slot * STEP + 256 * 64 + i * 8192 + s * 2048, aw[0], aw[1])
                      : *reinterpret_cast<const Vec<T, 8>*>(buf + slot * STEP + (256 + wn + i * 32) * 64 + at[s]);
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

    uint32_t m0, n0, id = first;
    origin(id, m0, n0);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        point(m0, n0, t);
#pragma unroll
        for (int i = 0; i < 2; ++i) move_x(t, 0, i), move_w(t, 0, i);
#pragma unroll
        for (int i = 0; i < 2; ++i) move_w(t, 1, i);
#pragma unroll
        for (int i = 0; i < 2; ++i) move_x(t, 1, i);
    }
    meet<12>();
    int slot = 0;
#pragma unroll
    for (int n = 0; n < 4; ++n) read_x(0, 0, n), read_x(0, 1, n), read_w(0, 0, n);
    while (true) {
        const uint32_t next = id + stride;
        uint32_t mn = m0, nn = n0;
        if (next < count) origin(next, mn, nn);  // else the moves past the end repeat this tile's, unread
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = f32x16{};
        for (uint32_t t = 0; t < steps; ++t) {
            if (t + 2 < steps)
                point(m0, n0, t + 2);
            else
                point(mn, nn, t + 2 - steps);
            // the moves in flight at a meeting, from the oldest: the quarter that the phase reads is the first of them
            meet<10>();
            product(0, 0, [&](int n) {
                if (n < 4) read_w(slot, 1, n);
            });
            meet<8>();
            product(1, 0, [&](int n) {
                read_x(slot, 2 + (n & 1), n >> 1);
                if (n & 1) (n & 2) ? move_w(slot, 0, n >> 2) : move_x(slot, 0, n >> 2);
            });
            meet<12>();
            product(0, 2, [&](int n) {
                if ((n & 3) == 1) move_w(slot, 1, n >> 2);
            });
            meet<10>();
            product(1, 2, [&](int n) {
                if (n < 4) {
                    read_w(slot ^ 1, 0, n);
                    read_x(slot ^ 1, 0, n);
                } else {
                    read_x(slot ^ 1, 1, n - 4);
                    if (n & 1) move_x(slot, 1, (n - 4) >> 1);
                }
            });
            slot ^= 1;
        }
        // Results, rounded, 32 x 32 at a time through the wave's 4 KB, of which each takes half: a lane that has 4 adjacent
        // columns of one row eight columns apart then has 8 of two rows.  A row's chunks of 16 bytes are spread over the banks.
        const uint32_t ms = min(m0, rows - 256), ns = min(n0, cols - OUT);
        const int rr = lane >> 2, cc = lane & 3;
        auto put = [&](int half, const f32x16& z) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<Vec<T, 4>*>(turn + half * 2048 + l * 64 + ((q ^ ((l >> 2) & 3)) << 4) + h * 8) =
                    Vec<T, 4>{static_cast<T>(z[q * 4]), static_cast<T>(z[q * 4 + 1]), static_cast<T>(z[q * 4 + 2]), static_cast<T>(z[q * 4 + 3])};
        };
        struct Two {
            Vec<T, 8> of[2];
        };
        auto take = [&](int half) {
            Two v;
#pragma unroll
            for (int k = 0; k < 2; ++k) v.of[k] = *reinterpret_cast<const Vec<T, 8>*>(turn + half * 2048 + (k * 16 + rr) * 64 + ((cc ^ ((rr >> 2) & 3)) << 4));
            return v;
        };
        auto give = [&](auto row_at, uint32_t row, uint32_t col, const Two& v) {  // rows row and row + 16; what lies from m0 and n0 on
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (row + k * 16 < m0) continue;
                T* to = row_at(row + k * 16);
                if (col >= n0) {
                    store_any<T, 8>(to + col, v.of[k]);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (col + e >= n0) to[col + e] = v.of[k][e];
                }
            }
        };
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {  // not unrolled: the epilogue's code stays in the instruction cache
            f32x16 z, u;
            switch (j) {
                case 0: z = acc[0][0], u = acc[1][0]; break;
                case 1: z = acc[0][1], u = acc[1][1]; break;
                case 2: z = acc[0][2], u = acc[1][2]; break;
                default: z = acc[0][3], u = acc[1][3]; break;
            }
            const uint32_t row = ms + (XT ? (j >> 1) * 128 + (wave >> 2) * 64 + (j & 1) * 32 : wm + j * 32) + rr;
            if constexpr (FORM == GATED) {
                const uint32_t col = ns + wn / 2 + cc * 8;
                if (p.gate) {
                    put(0, z);
                    put(1, u);
                    __builtin_amdgcn_wave_barrier();
                    const Two a = take(0), b = take(1);
                    give([&](uint32_t r) { return static_cast<T*>(p.gate) + static_cast<size_t>(r) * p.cols; }, row, col, a);
                    give([&](uint32_t r) { return static_cast<T*>(p.up) + static_cast<size_t>(r) * p.cols; }, row, col, b);
                    __builtin_amdgcn_wave_barrier();
                }
                float g[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) g[e] = z[e];
                activate(g, p.act);
#pragma unroll
                for (int e = 0; e < 16; ++e) z[e] = g[e] * u[e];
                put(0, z);
                __builtin_amdgcn_wave_barrier();
                give([&](uint32_t r) { return static_cast<T*>(p.h) + static_cast<int64_t>(r) * p.hs; }, row, col, take(0));
            } else {
                const uint32_t col = ns + (wave & 3) * 32 + cc * 8;
                put(0, z);
                put(1, u);
                __builtin_amdgcn_wave_barrier();
                const Two a = take(0), b = take(1);
                auto at = [&](uint32_t r) { return row_of<T, FORM>(p, r); };
                give(at, row, col, a);
                give(at, row, col + 128, b);
            }
            __builtin_amdgcn_wave_barrier();
        }
        if (next >= count) break;
        id = next;
        m0 = mn;
        n0 = nn;
    }
    __builtin_amdgcn_s_waitcnt(0);  // moves into this workgroup's LDS end before it does
}

// Workgroup b runs on XCD b mod 8: each XCD takes a contiguous run of tiles, so that the tiles in flight on it share operands
// in its L2.
struct Share {
    uint32_t run, count;
};
__device__ inline Share share_of(uint32_t tiles) {
    const uint32_t xcd = blockIdx.x & 7, q8 = tiles >> 3, r8 = tiles & 7;
    return Share{xcd * q8 + (xcd < r8 ? xcd : r8), q8 + (xcd < r8 ? 1 : 0)};
}
template <typename T>
__global__ __launch_bounds__(512, 2) void gated_big_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const Share s = share_of((p.rows + 255) / 256 * ((p.cols + 127) / 128));
    big_tiles<T, GATED>(p, lds, s.run, blockIdx.x >> 3, s.count, gridDim.x >> 3);
}
// Both products of the gradients in one launch, so that the tiles of both fill the compute units.
template <typename T>
__global__ __launch_bounds__(512, 2) void gated_big_backward_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const uint32_t nt = (p.inner + 255) / 256, stride = gridDim.x >> 3;
    const Share a = share_of(p.dx ? (p.rows + 255) / 256 * nt : 0), b = share_of(p.dwg ? (2 * p.cols + 255) / 256 * nt : 0);
    uint32_t first = blockIdx.x >> 3;
    big_tiles<T, INPUT>(p, lds, a.run, first, a.count, stride);
    __syncthreads();
    if (first < a.count) first += (a.count - first + stride - 1) / stride * stride;
    big_tiles<T, WEIGHTS>(p, lds, b.run, first - a.count, b.count, stride);
}

// Mid and Small: two workgroups per compute unit.  Flat and Narrow: GATED's waves have 64 rows of W; Narrow has a workgroup for
// every tile of 64 x 32 results, where tiles of Flat (64 x 64) leave compute units idle: 64 x 4096 -> 8192 34 and 56 us, 128 x
// 4096 -> 4096 21.8 and 36.3, 200 x 2048 -> 4096 16.5 and 20.1, but 300 x 4096 -> 4096 (320 tiles of 64) 47 and 37.
using Mid = Tile<128, 128, 2, 2, 32, 4, 2>;
using Small = Tile<64, 64, 2, 2, 64, 4, 2>;
using Narrow = Tile<64, 64, 2, 1, 64, 4, 2>;
using Flat = Tile<64, 128, 2, 2, 64, 3, 2>;

constexpr uint32_t FEW = 32;

uint64_t tiles_of(uint64_t rows, uint64_t cols, uint32_t high, uint32_t wide) { return (rows + high - 1) / high * ((cols + wide - 1) / wide); }

template <typename T, typename C, bool Direct>
int start(const Params& p, hipStream_t s) {
    auto* k = gated_kernel<T, C, Direct>;
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_lds(reinterpret_cast<const void*>(k), C::LDS, done)) return rc;
    k<<<static_cast<uint32_t>(tiles_of(p.rows, p.cols, C::BM, C::BN / 2)), C::THREADS, C::LDS, s>>>(p);
    return BS_OK;
}

bool rows16(const void* p, int64_t stride) { return aligned16(p) && stride % 8 == 0; }

template <typename T>
int start_big(const Params& p, bool backward, uint64_t tiles, hipStream_t s) {
    constexpr int LDS = 160 * 1024;
    auto* k = backward ? gated_big_backward_kernel<T> : gated_big_kernel<T>;
    static std::atomic<uint64_t> done[2];
    if (const int rc = allow_lds(reinterpret_cast<const void*>(k), LDS, done[backward])) return rc;
    k<<<tiles < CUS ? static_cast<uint32_t>(tiles + 7) / 8 * 8 : CUS, 512, LDS, s>>>(p);
    return BS_OK;
}

template <typename T>
int launch_forward(Params p, hipStream_t s) {
    if (p.rows <= FEW) {
        // Up to 32 rows: with 64, 64 x 4096 -> 8192 would take 39 us, 34 with tiles; 48 x 1024 -> 4096 8.5 either way.  32
        // columns a workgroup, half the reads of x, where that leaves a workgroup for every compute unit: 17 x 4096 -> 8192
        // takes 30.6 us, 35.7 with 16.
        if (p.rows <= 16)
            gated_few_kernel<T, 1, 1><<<(p.cols + 15) / 16, 512, 0, s>>>(p);
        else if (p.cols >= 32 * CUS)
            gated_few_kernel<T, 2, 2><<<(p.cols + 31) / 32, 512, 0, s>>>(p);
        else
            gated_few_kernel<T, 2, 1><<<(p.cols + 15) / 16, 512, 0, s>>>(p);
        return BS_OK;
    }
    const bool direct = rows16(p.x, p.xs) && rows16(p.wg, p.wgs) && rows16(p.wu, p.wus);
    // Tiles of 256 where they take fewer rounds of workgroups than tiles of 128, of which two share a compute unit.  256 and
    // 128: 2560 x 4096 -> 1792 (140 and 560 tiles) 73 and 104 us, 4096 x 1024 -> 1280 25.4 and 32.0, 4200 x 1024 -> 2048 (272
    // and 1056) 53 and 56, 5000 x 4096 -> 2048 169 and 202, but 2048 x 4096 -> 1792 (112 and 448) 73 and 70, 1500 x 2048 ->
    // 2048 39.6 and 35.7.  128 and 64: 1500 x 2048 -> 2048 (384 tiles of 128) 35.7 and 40.6, but 2048 x 1024 -> 1024 (256)
    // 14.6 and 13.4.
    const uint64_t big = tiles_of(p.rows, p.cols, 256, 128), mid = tiles_of(p.rows, p.cols, 128, 64);
    if (direct && (big + CUS - 1) / CUS < (mid + 2 * CUS - 1) / (2 * CUS) && p.rows >= 256 && p.cols >= 128 && p.inner % 64 == 0 &&
        p.inner >= 128 && p.xs < (1 << 22) && p.wgs < (1 << 22) && p.wgs == p.wus)
        return start_big<T>(p, false, big, s);
    if (mid > CUS) return direct ? start<T, Mid, true>(p, s) : start<T, Mid, false>(p, s);
    if (tiles_of(p.rows, p.cols, 64, 64) <= CUS) return direct ? start<T, Narrow, true>(p, s) : start<T, Narrow, false>(p, s);
    return direct ? start<T, Flat, true>(p, s) : start<T, Flat, false>(p, s);
}
// How the gradients' two products are cut: tiles of 256 (big), 128 or 64, and with the latter pieces of the inner dimensions.
struct Plan {
    bool big, input_mid, weight_mid;
    uint32_t input_splits, weight_splits;
    uint64_t input_tiles, weight_tiles;
};
// `dx`, `dw`: which are wanted; `big`: whether the operands' alignment and strides allow tiles of 256
Plan plan_of(uint64_t rows, uint32_t inner, uint32_t cols, bool dx, bool dw, bool big) {
    auto cut = [&](uint32_t size) {
        Plan n{};
        n.input_tiles = dx ? tiles_of(rows, inner, size, size) : 0;
        n.weight_tiles = dw ? tiles_of(2ull * cols, inner, size, size) : 0;
        n.input_splits = n.weight_splits = 1;
        return n;
    };
    Plan n = cut(256);
    if (big && rows >= 256 && cols >= 128 && cols % 64 == 0 && inner >= 256 && inner % 8 == 0) {
        // A workgroup per compute unit takes its share of the tiles one after the other, dx's first.  Worth it where they are
        // at work for 0.55 of the time, which they are not where one product has few long tiles: 20000 x 256 -> 256 takes 340 us
        // with them (2 tiles of 313 steps beside 79 of 8), 43 with smaller ones.
        const uint64_t most = (n.input_tiles + n.weight_tiles + CUS - 1) / CUS, input_steps = cols / 32, weight_steps = (rows + 63) / 64;
        // the workgroups with the most and with the fewest tiles of dx
        const uint64_t more = std::min((n.input_tiles + CUS - 1) / CUS, most), less = n.weight_tiles ? n.input_tiles / CUS : more;
        const uint64_t time = std::max(more * input_steps + (most - more) * weight_steps, less * input_steps + (most - less) * weight_steps);
        const uint64_t work = n.input_tiles * input_steps + n.weight_tiles * weight_steps;
        if (static_cast<double>(work) >= 0.55 * static_cast<double>(time * CUS)) {
            n.big = true;
            return n;
        }
    }
    // Two workgroups per compute unit, in one launch, of tiles of 64 or 128 for either product, and pieces of an inner dimension
    // about as long as their share of all work, of 1024 elements at least: what takes the least time, by the microseconds of a
    // workgroup's start and of 64 inner elements, and of the launch that joins pieces and its bytes.  Against tiles of 64 alone
    // below a tile of 128 for every compute unit: 300 x 768 -> 2048 20.9 and 23.6 us, 1000 x 1024 -> 2048 34.8 and 37.4, 2000 x
    // 256 -> 1024 21.2 and 24.5, but 256 x 2048 -> 2048 28.9 and 26.8.
    constexpr double START = 2.5, SMALL = 0.45, MID = 1.4, JOIN = 4.0, BYTES = 4e6;
    const uint64_t input_steps = (2ull * cols + 63) / 64, weight_steps = (rows + 63) / 64;
    double best = 0.0;
    for (int way = 0; way < 16; ++way) {
        Plan c{};
        c.input_mid = way & 1;
        c.weight_mid = way >> 1 & 1;
        c.input_tiles = dx ? tiles_of(rows, inner, c.input_mid ? 128 : 64, c.input_mid ? 128 : 64) : 0;
        c.weight_tiles = dw ? tiles_of(2ull * cols, inner, c.weight_mid ? 128 : 64, c.weight_mid ? 128 : 64) : 0;
        const double a = c.input_mid ? MID : SMALL, b = c.weight_mid ? MID : SMALL;
        const double work = static_cast<double>(c.input_tiles * input_steps) * a + static_cast<double>(c.weight_tiles * weight_steps) * b;
        const auto splits = [&](bool cut, uint64_t steps, double step) {
            const uint64_t share = std::max<uint64_t>(16, static_cast<uint64_t>(work / (2 * CUS) / step));
            return cut && steps > share ? static_cast<uint32_t>((steps + share - 1) / share) : 1u;
        };
        c.input_splits = splits(dx && (way & 4), input_steps, a);
        c.weight_splits = splits(dw && (way & 8), weight_steps, b);
        const double longest = std::max(dx ? a * static_cast<double>(input_steps) / c.input_splits : 0.0, dw ? b * static_cast<double>(weight_steps) / c.weight_splits : 0.0);
        const double groups = static_cast<double>(c.input_tiles * c.input_splits + c.weight_tiles * c.weight_splits);
        double time = std::max((work + START * groups) / (2 * CUS), longest + START);
        if (c.input_splits > 1) time += JOIN + 8.0 * static_cast<double>(rows * inner) * c.input_splits / BYTES;
        if (c.weight_splits > 1) time += JOIN + 16.0 * static_cast<double>(static_cast<uint64_t>(cols) * inner) * c.weight_splits / BYTES;
        if (way && time >= best) continue;
        best = time;
        n = c;
    }
    return n;
}
uint64_t up16(uint64_t n) { return (n + 15) / 16 * 16; }
// the workspace of the gradients: d, then x's tail or the pieces' sums of both products
struct Space {
    uint64_t d, input_parts, weight_parts;
    uint64_t bytes() const { return d + std::max<uint64_t>(input_parts + weight_parts, tail); }
    uint64_t tail;
};
Space space_of(const Plan& n, uint64_t rows, uint32_t inner, uint32_t cols) {
    Space s{};
    s.d = up16((rows + 63) / 64 * 64 * 2 * cols * 2);
    s.input_parts = n.input_splits > 1 ? up16(n.input_splits * rows * inner * 4) : 0;
    s.weight_parts = n.weight_splits > 1 ? up16(n.weight_splits * 2ull * cols * inner * 4) : 0;
    s.tail = n.big ? 128ull * inner : 0;
    return s;
}
// Whether tiles of 256 are taken depends on more than the sizes: the larger of both.
uint64_t space_for(uint64_t rows, uint32_t inner, uint32_t cols, bool dx, bool dw) {
    return std::max(space_of(plan_of(rows, inner, cols, dx, dw, true), rows, inner, cols).bytes(),
                    space_of(plan_of(rows, inner, cols, dx, dw, false), rows, inner, cols).bytes());
}

template <typename T, typename CI, typename CW, bool Direct>
int start_backward(const Params& p, const Plan& n, hipStream_t s) {
    constexpr int LDS = std::max(CI::LDS, CW::LDS);
    auto* k = gated_backward_kernel<T, CI, CW, Direct>;
    static std::atomic<uint64_t> done{0};
    if (const int rc = allow_lds(reinterpret_cast<const void*>(k), LDS, done)) return rc;
    const uint64_t inputs = n.input_tiles * n.input_splits, all = inputs + n.weight_tiles * n.weight_splits;
    k<<<static_cast<uint32_t>(all), 256, LDS, s>>>(p, static_cast<uint32_t>(std::max<uint64_t>(n.input_tiles, 1)), static_cast<uint32_t>(inputs),
                                                            static_cast<uint32_t>(std::max<uint64_t>(n.weight_tiles, 1)));
    auto join = [&](auto* kernel, uint64_t rows) { kernel<<<static_cast<uint32_t>((rows * ((p.inner + 3) / 4) + 255) / 256), 256, 0, s>>>(p); };
    if (n.input_splits > 1) join(gated_join_kernel<T, INPUT>, p.rows);
    if (n.weight_splits > 1) join(gated_join_kernel<T, WEIGHTS>, 2ull * p.cols);
    return BS_OK;
}
template <typename T>
int launch_backward(Params p, char* workspace, hipStream_t s) {
    const bool aligned = rows16(p.x, p.xs) && rows16(p.wg, p.wgs) && rows16(p.wu, p.wus) && p.wgs == p.wus;
    const bool near = p.xs < (1 << 22) && p.wgs < (1 << 22) && p.cols < (1 << 21);
    const Plan n = plan_of(p.rows, p.inner, p.cols, p.dx, p.dwg, aligned && near);
    const Space space = space_of(n, p.rows, p.inner, p.cols);
    p.d = workspace;
    p.tail = workspace + space.d;
    p.input_parts = reinterpret_cast<float*>(workspace + space.d);
    p.weight_parts = reinterpret_cast<float*>(workspace + space.d + space.input_parts);
    p.input_splits = n.input_splits;
    p.weight_splits = n.weight_splits;
    const uint32_t rows_up = (p.rows + 63) / 64 * 64, tail_rows = n.big && p.rows % 64 ? 64 : 0;
    if (p.rows) {
        const uint64_t chunks = static_cast<uint64_t>(rows_up) * ((p.cols + 7) / 8) + static_cast<uint64_t>(tail_rows) * ((p.inner + 7) / 8);
        gated_slopes_kernel<T><<<static_cast<uint32_t>(std::min<uint64_t>((chunks + 255) / 256, 1u << 22)), 256, 0, s>>>(p, rows_up, tail_rows, Divisor((p.cols + 7) / 8));
    }
    if (n.big) return start_big<T>(p, true, n.input_tiles + n.weight_tiles, s);
    // a step of dx's inner dimension lies in one weight
    const bool direct = aligned && p.cols % 64 == 0 && p.inner % 8 == 0;
    if (n.input_mid)
        return n.weight_mid ? direct ? start_backward<T, Mid, Mid, true>(p, n, s) : start_backward<T, Mid, Mid, false>(p, n, s)
                            : direct ? start_backward<T, Mid, Small, true>(p, n, s) : start_backward<T, Mid, Small, false>(p, n, s);
    return n.weight_mid ? direct ? start_backward<T, Small, Mid, true>(p, n, s) : start_backward<T, Small, Mid, false>(p, n, s)
                        : direct ? start_backward<T, Small, Small, true>(p, n, s) : start_backward<T, Small, Small, false>(p, n, s);
}

int check(const std::string& what, uint64_t rows, uint32_t inner, uint32_t cols) {
    if (rows > 0x7FFFFFFFull) return refuse(what + ": rows must be < 2^31");
    if (inner == 0 || inner > (1u << 24) || cols == 0 || cols > (1u << 23)) return refuse(what + ": inner must be in 1..2^24, cols in 1..2^23");
    // A grid of 2^32 threads is cut short without an error.  Tiles of 64 x 64 results by 256 threads are the most.
    if ((tiles_of(rows, std::max(inner, cols), 64, 64) + tiles_of(2ull * cols, inner, 64, 64)) * 256 > 0xFFFFFFFFull)
        return refuse(what + ": the sizes are too large for one launch");
    return BS_OK;
}
int check_rows(const std::string& what, const char* name, const void* p, int64_t stride, uint32_t row) {
    if (!p) return refuse(what + ": " + name + " must be given");
    if (stride < row) return refuse(what + ": rows of " + name + " overlap (a stride is shorter than its row)");
    if (stride >= (1 << 24)) return refuse(what + ": strides must be < 2^24");
    return BS_OK;
}

}  // namespace

extern "C" int bs_gated(const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride, const void* w_up, int64_t w_up_stride, void* out,
                        int64_t out_stride, void* gate, void* up, uint64_t rows, uint32_t inner, uint32_t cols, int type, int activation, void* stream) try {
    const std::string what = "bs_gated";
    if (const int rc = check(what, rows, inner, cols)) return rc;
    if (type != BS_F16 && type != BS_BF16) return refuse(what + ": type must be BS_F16 or BS_BF16");
    if (activation < BS_ACT_NONE || activation > BS_ACT_SILU) return refuse(what + ": unknown activation " + std::to_string(activation));
    if (!gate != !up) return refuse(what + ": gate and up must be given together");
    if (rows == 0) return BS_OK;
    if (const int rc = check_rows(what, "x", x, x_stride, inner)) return rc;
    if (const int rc = check_rows(what, "w_gate", w_gate, w_gate_stride, inner)) return rc;
    if (const int rc = check_rows(what, "w_up", w_up, w_up_stride, inner)) return rc;
    if (const int rc = check_rows(what, "out", out, out_stride, cols)) return rc;
    Params p{};
    p.x = x, p.wg = w_gate, p.wu = w_up, p.h = out, p.gate = gate, p.up = up;
    p.xs = x_stride, p.wgs = w_gate_stride, p.wus = w_up_stride, p.hs = out_stride;
    p.rows = static_cast<uint32_t>(rows), p.inner = inner, p.cols = cols, p.act = activation;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    const int rc = type == BS_F16 ? launch_forward<f16>(p, s) : launch_forward<bf16>(p, s);
    return rc ? rc : launched("bs_gated");
} catch (...) {
    return bs_internal_exception();
}

extern "C" int bs_gated_backward_workspace(uint64_t rows, uint32_t inner, uint32_t cols, uint64_t* bytes) try {
    if (!bytes) return refuse("bs_gated_backward_workspace: bytes is null");
    if (const int rc = check("bs_gated_backward_workspace", rows, inner, cols)) return rc;
    // whichever gradients are asked for
    *bytes = rows ? std::max({space_for(rows, inner, cols, true, true), space_for(rows, inner, cols, true, false), space_for(rows, inner, cols, false, true)}) : 0;
    return BS_OK;
} catch (...) {
    return bs_internal_exception();
}

extern "C" int bs_gated_backward(const void* dh, int64_t dh_stride, const void* x, int64_t x_stride, const void* w_gate, int64_t w_gate_stride,
                                 const void* w_up, int64_t w_up_stride, const void* gate, int64_t gate_stride, const void* up, int64_t up_stride,
                                 void* dx, void* dw_gate, void* dw_up, uint64_t rows, uint32_t inner, uint32_t cols, int type, int activation,
                                 void* workspace, uint64_t workspace_bytes, void* stream) try {
    const std::string what = "bs_gated_backward";
    if (const int rc = check(what, rows, inner, cols)) return rc;
    if (type != BS_F16 && type != BS_BF16) return refuse(what + ": type must be BS_F16 or BS_BF16");
    if (activation < BS_ACT_NONE || activation > BS_ACT_SILU) return refuse(what + ": unknown activation " + std::to_string(activation));
    if (!dw_gate != !dw_up) return refuse(what + ": dw_gate and dw_up must be given together");
    if (!dx && !dw_gate) return BS_OK;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    Params p{};
    p.x = x, p.wg = w_gate, p.wu = w_up, p.dh = dh, p.g = gate, p.u = up, p.dx = dx, p.dwg = dw_gate, p.dwu = dw_up;
    p.xs = x_stride, p.wgs = w_gate_stride, p.wus = w_up_stride, p.dhs = dh_stride, p.gs = gate_stride, p.us = up_stride;
    p.rows = static_cast<uint32_t>(rows), p.inner = inner, p.cols = cols, p.act = activation;
    if (rows) {
        if (const int rc = check_rows(what, "dh", dh, dh_stride, cols)) return rc;
        if (const int rc = check_rows(what, "x", x, x_stride, inner)) return rc;
        if (const int rc = check_rows(what, "w_gate", w_gate, w_gate_stride, inner)) return rc;
        if (const int rc = check_rows(what, "w_up", w_up, w_up_stride, inner)) return rc;
        if (const int rc = check_rows(what, "gate", gate, gate_stride, cols)) return rc;
        if (const int rc = check_rows(what, "up", up, up_stride, cols)) return rc;
        const uint64_t need = space_for(rows, inner, cols, dx, dw_gate);
        if (!workspace || workspace_bytes < need) return refuse(what + ": the workspace must hold " + std::to_string(need) + " bytes");
        if (!aligned16(workspace)) return refuse(what + ": the workspace must be 16-byte aligned");
    } else if (!dw_gate) {
        return BS_OK;
    }
    // without rows the weights' gradients are 0, sums of no steps
    const int rc = type == BS_F16 ? launch_backward<f16>(p, static_cast<char*>(workspace), s) : launch_backward<bf16>(p, static_cast<char*>(workspace), s);
    return rc ? rc : launched("bs_gated_backward");
} catch (...) {
    return bs_internal_exception();
}
