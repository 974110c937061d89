// Norm of every head of queries and keys with the rotation by their positions, and its gradients (include/bs_embed.h).
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = M(pos) (x r w),  M: pairs turned by the angles pos f, times the magnitude
//   d = M^T dy,  dw = sum of d x r over tokens and heads,  dx = r (d w - x r^2 mean(d w x))
//
// A workgroup has queries or keys of a few tokens: first their angles, each once, to LDS, then their heads.  A head
// belongs to a few lanes, each with 2 N elements in two accesses of N: the two halves of N pairs (elements i and i +
// rotary / 2) or 2 N neighbours, so that both partners of a pair are the lane's.
//
// Memory bounds both directions.  32768 tokens of 32 + 8 heads of 128 in bf16, columns of a product 48 heads wide: 156 us, 4.3
// TB/s (a copy reaches 5.0); the gradients of 16384 with float32 weights: 122 us, 4.1 TB/s.  Weights in LDS instead of
// registers and queries and keys in workgroups of their own took the first from 198 us to 176, the second from 182 to 151.
#include "bs_embed.hpp"

#include <algorithm>
#include <cmath>

namespace {
using namespace bse;

constexpr uint32_t THREADS = 256, WAVES = THREADS / 64;
// Workgroups of the gradients: 16384 tokens of 32 + 8 heads of 128 in bf16 take 151 us with 2 per compute unit, 132 with 4,
// 124 with 8, 130 with 16, each of which has its part of the weights' gradients.
constexpr uint32_t MOST_PARTS = 8 * CUS;

// the queries' heads or the keys'
struct Side {
    const void *x, *grad, *weight;
    void *out, *weight_grad;
    int64_t x_stride, x_head, grad_stride, grad_head, out_stride, out_head;
    uint32_t heads;
    Divisor by_heads;
    uint32_t block, blocks;  // tokens of a workgroup's turn, and such turns
    uint32_t groups;         // workgroups
    float* parts;            // of the weight's gradient: groups x head_dim
};
struct Params {
    Side side[2];
    const int32_t* positions;
    const double* frequencies;
    uint32_t tokens, head_dim, rotary, rotated, units;  // accesses of a head in pairs of N: those with pairs to turn come first
    uint32_t lanes, shift;                              // of a head: 2^shift
    Divisor by_half;
    int interleaved, norm, wtype;
    float eps, magnitude;
};

// N elements from two places of a head, K times
template <int N, int K>
struct Unit {
    float a[K][N], b[K][N];
};
template <typename T, int N, int K>
struct Raw {  // as they lie in memory: on their way until they are taken
    Vec<T, N> a[K], b[K];
};
struct Places {
    uint32_t a, b;  // first elements
    bool turned, live;
};
template <int N>
__device__ inline Places places_of(const Params& p, uint32_t u) {
    Places x;
    x.live = u < p.units;
    x.turned = u < p.rotated;
    if (!x.turned) {
        x.a = p.rotary + (u - p.rotated) * 2 * N;
        x.b = x.a + N;
    } else if (p.interleaved) {
        x.a = u * 2 * N;
        x.b = x.a + N;
    } else {
        x.a = u * N;
        x.b = p.rotary / 2 + u * N;
    }
    return x;
}
// Read once: they leave the caches to the results, which attention reads next (32768 tokens of 32 + 8 heads of 128 in bf16: 176
// us otherwise, 162 so)
template <typename T, int N, int K>
__device__ inline void load(const T* head, const Places (&at)[K], bool live, Raw<T, N, K>& x) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        x.a[k] = x.b[k] = Vec<T, N>{};
        if (live && at[k].live) {
            x.a[k] = load_once<T, N>(head + at[k].a);
            x.b[k] = load_once<T, N>(head + at[k].b);
        }
    }
}
template <typename T, int N, int K>
__device__ inline void take(const Raw<T, N, K>& from, Unit<N, K>& x) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) x.a[k][i] = static_cast<float>(from.a[k][i]), x.b[k][i] = static_cast<float>(from.b[k][i]);
}
template <typename T, int N, int K>
__device__ inline void store(T* head, const Places (&at)[K], bool live, const Unit<N, K>& x) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        Vec<T, N> a, b;
#pragma unroll
        for (int i = 0; i < N; ++i) a[i] = static_cast<T>(x.a[k][i]), b[i] = static_cast<T>(x.b[k][i]);
        if (live && at[k].live) {
            store_any<T, N>(head + at[k].a, a);
            store_any<T, N>(head + at[k].b, b);
        }
    }
}
// the weight, or 1, to LDS in float32: in registers it would cost a wave or two of every SIMD
template <typename T>
__device__ inline void weights(const Params& p, const Side& a, float* to) {
    for (uint32_t i = threadIdx.x; i < p.head_dim; i += THREADS)
        to[i] = !a.weight ? 1.0f : p.wtype == BS_F32 ? static_cast<const float*>(a.weight)[i] : static_cast<float>(static_cast<const T*>(a.weight)[i]);
}
template <int N, int K>
__device__ inline void read_weight(const float* w, const Places (&at)[K], Unit<N, K>& x) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        Vec<float, N> a = {}, b = {};
        if (at[k].live) {  // places are multiples of N elements
            a = *reinterpret_cast<const Vec<float, N>*>(w + at[k].a);
            b = *reinterpret_cast<const Vec<float, N>*>(w + at[k].b);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) x.a[k][i] = a[i], x.b[k][i] = b[i];
    }
}

// sin and cos of a quarter turn times r in -1/2 .. 1/2, by their series at 0: what is left out is below 2^-29 of sin and
// 2^-33 at an eighth of a turn
__device__ inline void eighth(float r, float& s, float& c) {
    const float x = r * 1.57079632679489662f, q = x * x;
    s = x * fmaf(q, fmaf(q, fmaf(q, fmaf(q, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
    c = fmaf(q, fmaf(q, fmaf(q, fmaf(q, fmaf(q, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
}
// The angles of tokens t0 .. t0 + n - 1, each once: rotary / 2 cosines, then as many sines, a token.  Turns are counted in
// float64 (the angle of a far position has no bits left after the point in float32), what is left of a turn in float32.
__device__ inline void angles(const Params& p, float* table, uint32_t t0, uint32_t n) {
    const uint32_t half = p.rotary / 2;
    for (uint32_t i = threadIdx.x; i < n * half; i += THREADS) {
        const uint32_t tok = p.by_half.quotient(i), j = i - tok * half;
        const double pos = p.positions ? static_cast<double>(p.positions[t0 + tok]) : static_cast<double>(t0 + tok);
        double turns = pos * (p.frequencies[j] * 0.15915494309189533577);
        turns = (turns - rint(turns)) * 4.0;
        const double quarters = rint(turns);
        float s, c;
        eighth(static_cast<float>(turns - quarters), s, c);
        const int q = static_cast<int>(quarters);
        const float cs = q & 1 ? s : c, sn = q & 1 ? c : s;
        table[tok * p.rotary + j] = ((q + 1) & 2 ? -cs : cs) * p.magnitude;
        table[tok * p.rotary + half + j] = (q & 2 ? -sn : sn) * p.magnitude;
    }
}
// turns the pairs by the table's angles, back if Back
template <bool Back, int N, int K>
__device__ inline void turn(const Params& p, const float* table, const Places (&at)[K], uint32_t lane, Unit<N, K>& x) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (!at[k].turned) continue;
        const float* t = table + (lane + k * p.lanes) * N;
        // multiples of N elements on both sides, so they are aligned
        const Vec<float, N> c = *reinterpret_cast<const Vec<float, N>*>(t), up = *reinterpret_cast<const Vec<float, N>*>(t + p.rotary / 2);
        const Vec<float, N> s = Back ? -up : up;
        auto pair = [&](float& a, float& b, int i) {
            const float u = a;
            a = fmaf(u, c[i], -(b * s[i]));
            b = fmaf(b, c[i], u * s[i]);
        };
        if (N == 1 || !p.interleaved) {
#pragma unroll
            for (int i = 0; i < N; ++i) pair(x.a[k][i], x.b[k][i], i);
        } else {
#pragma unroll
            for (int i = 0; i + 1 < N; i += 2) {
                pair(x.a[k][i], x.a[k][i + 1], i / 2);
                pair(x.b[k][i], x.b[k][i + 1], N / 2 + i / 2);
            }
        }
    }
}
// Sum over a head's lanes, the same bits in all of them.  Exchanges within 16 lanes are operands of the additions (by 4 and 8: a
// mirror of 8 and 16 lanes, whose halves hold one value each by then); with all of them through LDS the gradients of 16384
// tokens take 124 us instead of 122.
template <int Control>
__device__ inline float from_lane(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), Control, 0xF, 0xF, true));
}
__device__ inline float head_sum(float v, uint32_t lanes) {
    if (lanes >= 2) v += from_lane<0xB1>(v);    // quad_perm 1 0 3 2
    if (lanes >= 4) v += from_lane<0x4E>(v);    // quad_perm 2 3 0 1
    if (lanes >= 8) v += from_lane<0x141>(v);   // row_half_mirror
    if (lanes >= 16) v += from_lane<0x140>(v);  // row_mirror
    if (lanes >= 32) v += __shfl_xor(v, 16);
    if (lanes >= 64) v += __shfl_xor(v, 32);
    return v;
}
template <int N, int K>
__device__ inline float dot(const Unit<N, K>& x, const Unit<N, K>& y) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(x.a[k][i], y.a[k][i], fmaf(x.b[k][i], y.b[k][i], s));
    return s;
}
// 1 / sqrt(v): the instruction's result, off by a unit, and a step of Newton's method
__device__ inline float inverse_root(float v) {
    const float r = __builtin_amdgcn_rsqf(v);
    const float e = fmaf(-v * r, r, 1.0f);
    return fabsf(e) < 1.0f ? fmaf(0.5f * r, e, r) : r;  // zero, infinity and NaN as they are
}

// A workgroup's turn: the heads of its tokens follow each other, 64 / lanes in a wave's pass.
struct Turn {
    uint32_t t0, n, heads, passes;
    __device__ Turn(const Params& p, const Side& a, uint32_t block) : t0(block * a.block), n(min(a.block, p.tokens - t0)), heads(n * a.heads) {
        const uint32_t slots = 64u >> p.shift;
        passes = (heads + slots - 1) / slots;
    }
};
struct Row {
    uint32_t tok, head;  // tok in the turn
    bool live;
    __device__ Row() {}
    __device__ Row(const Params& p, const Side& a, const Turn& t, uint32_t pass) {
        const uint32_t i = pass * (64u >> p.shift) + ((threadIdx.x & 63) >> p.shift);
        live = i < t.heads;
        tok = live ? a.by_heads.quotient(i) : 0;
        head = live ? i - tok * a.heads : 0;
    }
    __device__ int64_t at(const Turn& t, int64_t stride, int64_t head_stride) const {
        return static_cast<int64_t>(t.t0 + tok) * stride + static_cast<int64_t>(head) * head_stride;
    }
};

template <typename T, int N, int K>
__global__ __launch_bounds__(THREADS) void rotate_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const bool key = blockIdx.x >= p.side[0].groups;
    const Side& a = p.side[key];
    float *w = lds, *table = lds + p.head_dim;
    const uint32_t lane = threadIdx.x & (p.lanes - 1), wave = uniform(threadIdx.x >> 6);
    Places at[K];
#pragma unroll
    for (int k = 0; k < K; ++k) at[k] = places_of<N>(p, lane + k * p.lanes);
    if (p.norm) weights<T>(p, a, w);
    const float over = 1.0f / static_cast<float>(p.head_dim);
    for (uint32_t b = key ? blockIdx.x - p.side[0].groups : blockIdx.x; b < a.blocks; b += a.groups) {
        const Turn t(p, a, b);
        auto fetch = [&](uint32_t pass, Row& r, Raw<T, N, K>& x) {
            r = Row(p, a, t, pass);
            load(static_cast<const T*>(a.x) + r.at(t, a.x_stride, a.x_head), at, r.live, x);
        };
        Row next;
        Raw<T, N, K> soon;
        if (wave < t.passes) fetch(wave, next, soon);
        __syncthreads();  // nobody reads the last turn's angles any more
        angles(p, table, t.t0, t.n);
        __syncthreads();
        for (uint32_t pass = wave; pass < t.passes; pass += WAVES) {
            const Row r = next;
            Unit<N, K> x;
            take(soon, x);
            if (pass + WAVES < t.passes) fetch(pass + WAVES, next, soon);
            if (p.norm) {
                const float rstd = inverse_root(fmaf(head_sum(dot(x, x), p.lanes), over, p.eps));
                Unit<N, K> g;
                read_weight<N, K>(w, at, g);
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        x.a[k][i] = x.a[k][i] * rstd * g.a[k][i];
                        x.b[k][i] = x.b[k][i] * rstd * g.b[k][i];
                    }
            }
            turn<false>(p, table + r.tok * p.rotary, at, lane, x);
            store<T, N, K>(static_cast<T*>(a.out) + r.at(t, a.out_stride, a.out_head), at, r.live, x);
        }
    }
}

template <typename T, int N, int K>
__global__ __launch_bounds__(THREADS, 4) void rotate_backward_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) float lds[];
    const bool key = blockIdx.x >= p.side[0].groups;
    const Side& a = p.side[key];
    float *w = lds, *table = lds + p.head_dim;
    const uint32_t group = key ? blockIdx.x - p.side[0].groups : blockIdx.x;
    const uint32_t lane = threadIdx.x & (p.lanes - 1), wave = uniform(threadIdx.x >> 6);
    Places at[K];
#pragma unroll
    for (int k = 0; k < K; ++k) at[k] = places_of<N>(p, lane + k * p.lanes);
    if (p.norm) weights<T>(p, a, w);
    Unit<N, K> dw = {};
    const float over = 1.0f / static_cast<float>(p.head_dim);
    for (uint32_t b = group; b < a.blocks; b += a.groups) {
        const Turn t(p, a, b);
        auto fetch = [&](uint32_t pass, Row& r, Raw<T, N, K>& d, Raw<T, N, K>& x) {
            r = Row(p, a, t, pass);
            load(static_cast<const T*>(a.grad) + r.at(t, a.grad_stride, a.grad_head), at, r.live, d);
            if (p.norm) load(static_cast<const T*>(a.x) + r.at(t, a.x_stride, a.x_head), at, r.live, x);
        };
        Row next;
        Raw<T, N, K> soon_d, soon_x;
        if (wave < t.passes) fetch(wave, next, soon_d, soon_x);
        __syncthreads();  // nobody reads the last turn's angles any more
        angles(p, table, t.t0, t.n);
        __syncthreads();
        for (uint32_t pass = wave; pass < t.passes; pass += WAVES) {
            const Row r = next;
            Unit<N, K> x, d;
            take(soon_d, d);
            if (p.norm) take(soon_x, x);
            if (pass + WAVES < t.passes) fetch(pass + WAVES, next, soon_d, soon_x);
            turn<true>(p, table + r.tok * p.rotary, at, lane, d);
            if (p.norm) {
                const float rstd = inverse_root(fmaf(head_sum(dot(x, x), p.lanes), over, p.eps));
                Unit<N, K> g;
                read_weight<N, K>(w, at, g);
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        x.a[k][i] *= rstd;
                        x.b[k][i] *= rstd;
                        if (r.live) {
                            dw.a[k][i] = fmaf(d.a[k][i], x.a[k][i], dw.a[k][i]);
                            dw.b[k][i] = fmaf(d.b[k][i], x.b[k][i], dw.b[k][i]);
                        }
                        d.a[k][i] *= g.a[k][i];
                        d.b[k][i] *= g.b[k][i];
                    }
                const float along = head_sum(dot(d, x), p.lanes) * over;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        d.a[k][i] = rstd * fmaf(-along, x.a[k][i], d.a[k][i]);
                        d.b[k][i] = rstd * fmaf(-along, x.b[k][i], d.b[k][i]);
                    }
            }
            store<T, N, K>(static_cast<T*>(a.out) + r.at(t, a.out_stride, a.out_head), at, r.live, d);
        }
    }
    if (!a.parts) return;
    // the workgroup's sums: over the wave's heads by exchanges, over the waves through LDS, in a fixed order
    __shared__ float sums[WAVES][256];
    auto add = [&](float v) {
        for (uint32_t m = p.lanes; m < 64; m <<= 1) v += __shfl_xor(v, m);
        return v;
    };
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float sa = add(dw.a[k][i]), sb = add(dw.b[k][i]);
            if ((threadIdx.x & 63) < p.lanes && at[k].live) {
                sums[wave][at[k].a + i] = sa;
                sums[wave][at[k].b + i] = sb;
            }
        }
    __syncthreads();
    if (threadIdx.x < p.head_dim) {
        float s = 0.0f;
#pragma unroll
        for (uint32_t v = 0; v < WAVES; ++v) s += sums[v][threadIdx.x];
        a.parts[static_cast<size_t>(group) * p.head_dim + threadIdx.x] = s;
    }
}

// the workgroups' parts of the weights' gradients: 16 columns a workgroup, 64 runs of parts each, in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void rotate_parts_kernel(Params p) {
    __shared__ float sums[64][17];
    const Side& a = p.side[blockIdx.y];
    const uint32_t x = threadIdx.x & 15, y = threadIdx.x >> 4, c = blockIdx.x * 16 + x;
    if (!a.weight_grad) return;
    float s = 0.0f;
    if (c < p.head_dim) {
#pragma unroll 8
        for (uint32_t i = y; i < a.groups; i += 64) s += a.parts[static_cast<size_t>(i) * p.head_dim + c];
    }
    sums[y][x] = s;
    __syncthreads();
    for (uint32_t m = 32; m; m >>= 1) {
        if (y < m) sums[y][x] += sums[y + m][x];
        __syncthreads();
    }
    if (y || c >= p.head_dim) return;
    if (p.wtype == BS_F32)
        static_cast<float*>(a.weight_grad)[c] = sums[0][x];
    else
        static_cast<T*>(a.weight_grad)[c] = static_cast<T>(sums[0][x]);
}

// How heads are laid over lanes: accesses of `wide` elements, or of 2, or of 1, whichever the halves and the rest allow
uint32_t access_of(const bs_head_norm_rotary_args& a) {
    const uint32_t half = a.rotary / 2, rest = a.head_dim - a.rotary;
    for (uint32_t n : {a.type == BS_F32 ? 4u : 8u, 2u})
        if (half % n == 0 && rest % (2 * n) == 0) return n;
    return 1;
}
uint32_t ceil_div(uint64_t a, uint64_t b) { return static_cast<uint32_t>((a + b - 1) / b); }

Params plan(const bs_head_norm_rotary_args& a, uint32_t access, bool backward) {
    Params p{};
    p.side[0] = Side{a.q, a.q_grad, a.q_weight, a.q_out, a.q_weight_grad, a.q_stride, a.q_head_stride, a.q_grad_stride, a.q_grad_head_stride, a.q_out_stride, a.q_out_head_stride, a.heads, Divisor(a.heads), 0, 0, 0, nullptr};
    p.side[1] = Side{a.k, a.k_grad, a.k_weight, a.k_out, a.k_weight_grad, a.k_stride, a.k_head_stride, a.k_grad_stride, a.k_grad_head_stride, a.k_out_stride, a.k_out_head_stride, a.kv_heads, Divisor(std::max(a.kv_heads, 1u)), 0, 0, 0, nullptr};
    p.positions = a.positions;
    p.frequencies = a.frequencies;
    p.tokens = a.tokens;
    p.head_dim = a.head_dim;
    p.rotary = a.rotary;
    p.rotated = a.rotary / 2 / access;
    p.units = a.head_dim / 2 / access;
    p.by_half = Divisor(a.rotary ? a.rotary / 2 : 1);
    p.interleaved = a.interleaved;
    p.norm = a.norm;
    p.wtype = a.wtype;
    p.eps = a.eps;
    p.magnitude = a.magnitude;
    const uint32_t held = access == 1 ? ceil_div(p.units, 2) : p.units;  // lanes that a head needs
    while ((1u << p.shift) < held) ++p.shift;
    p.lanes = 1u << p.shift;
    for (Side& side : p.side) {
        if (!side.heads || !a.tokens) continue;
        // tokens of a turn: two passes a wave (156 us in the case above, 159 with one, 162 with four), less where that leaves
        // compute units without work, and angles within 16 KB
        uint32_t block = std::max(1u, 2 * WAVES * (64 >> p.shift) / side.heads);
        block = std::min(block, ceil_div(a.tokens, 4 * CUS));
        if (a.rotary) block = std::min(block, 16384 / (4 * a.rotary));
        side.block = std::max(1u, block);
        side.blocks = ceil_div(a.tokens, side.block);
        side.groups = std::min(side.blocks, backward ? std::max(1u, MOST_PARTS * side.heads / (a.heads + a.kv_heads)) : 1u << 22);
    }
    return p;
}

template <typename T, int N, int K>
int start(const Params& p, bool backward, hipStream_t s) {
    const uint32_t lds = (std::max(p.side[0].block, p.side[1].block) * p.rotary + p.head_dim) * 4, groups = p.side[0].groups + p.side[1].groups;
    if (!backward) {
        rotate_kernel<T, N, K><<<groups, THREADS, lds, s>>>(p);
        return BS_OK;
    }
    rotate_backward_kernel<T, N, K><<<groups, THREADS, lds, s>>>(p);
    if (p.side[0].parts) rotate_parts_kernel<T><<<dim3(ceil_div(p.head_dim, 16), 2), 1024, 0, s>>>(p);
    return BS_OK;
}
template <typename T>
int launch(const Params& p, uint32_t access, bool backward, hipStream_t s) {
    return access > 2 ? start<T, VN<T>, 1>(p, backward, s) : access == 2 ? start<T, 2, 1>(p, backward, s) : start<T, 1, 2>(p, backward, s);
}

int check(const std::string& what, const bs_head_norm_rotary_args* args) {
    if (!args) return refuse(what + ": args is null");
    const bs_head_norm_rotary_args& a = *args;
    if (a.type != BS_F32 && a.type != BS_F16 && a.type != BS_BF16) return refuse(what + ": type must be BS_F32, BS_F16 or BS_BF16");
    if (a.wtype != BS_F32 && a.wtype != a.type) return refuse(what + ": wtype must be type or BS_F32");
    if (a.head_dim < 2 || a.head_dim > 256 || a.head_dim % 2) return refuse(what + ": head_dim must be even, in 2..256");
    if (a.rotary > a.head_dim || a.rotary % 2) return refuse(what + ": rotary must be even, at most head_dim");
    if (a.heads == 0 || a.heads > 1024 || a.kv_heads > 1024) return refuse(what + ": heads must be in 1..1024, kv_heads in 0..1024");
    if (a.tokens > 0x7FFFFFFFu) return refuse(what + ": tokens must be < 2^31");
    if (a.norm && !(a.eps >= 0.0f && a.eps < INFINITY)) return refuse(what + ": eps must be finite and not negative");
    if (!(std::abs(a.magnitude) < INFINITY)) return refuse(what + ": magnitude must be finite");
    if (!a.norm && (a.q_weight || a.k_weight || a.q_weight_grad || a.k_weight_grad)) return refuse(what + ": weights belong to the norm");
    if (a.rotary && !a.frequencies) return refuse(what + ": frequencies must be given");
    return BS_OK;
}
// heads of tokens that lie apart; those that are written do not overlap each other either
int check_rows(const std::string& what, const char* name, const void* p, int64_t s, int64_t hs, uint32_t tokens, uint32_t heads, uint32_t dim, bool written) {
    if (!p) return refuse(what + ": " + name + " must be given");
    const int64_t t = tokens, h = heads, d = dim;
    if ((t > 1 && s < d) || (h > 1 && hs < d) || s > (int64_t{1} << 40) || hs > (int64_t{1} << 40)) return refuse(what + ": heads of " + name + " overlap (a stride is shorter than head_dim) or lie too far apart");
    if (written && t > 1 && h > 1 && s < (h - 1) * hs + d && hs < (t - 1) * s + d) return refuse(what + ": heads of " + name + " overlap");
    return BS_OK;
}
uint64_t workspace_of(const Params& p) { return static_cast<uint64_t>(p.side[0].groups + p.side[1].groups) * p.head_dim * sizeof(float); }

int run(const std::string& what, const bs_head_norm_rotary_args* args, bool backward, void* workspace, uint64_t bytes, void* stream) {
    if (const int rc = check(what, args)) return rc;
    const bs_head_norm_rotary_args& a = *args;
    const bool sums = backward && (a.q_weight_grad || a.k_weight_grad);
    if (a.tokens == 0 && !sums) return BS_OK;
    for (int key = 0; a.tokens && key < (a.kv_heads ? 2 : 1); ++key) {
        const uint32_t heads = key ? a.kv_heads : a.heads;
        if (!backward || a.norm)
            if (const int rc = check_rows(what, key ? "k" : "q", key ? a.k : a.q, key ? a.k_stride : a.q_stride, key ? a.k_head_stride : a.q_head_stride, a.tokens, heads, a.head_dim, false)) return rc;
        if (backward)
            if (const int rc = check_rows(what, key ? "k_grad" : "q_grad", key ? a.k_grad : a.q_grad, key ? a.k_grad_stride : a.q_grad_stride, key ? a.k_grad_head_stride : a.q_grad_head_stride, a.tokens, heads, a.head_dim, false)) return rc;
        if (const int rc = check_rows(what, key ? "k_out" : "q_out", key ? a.k_out : a.q_out, key ? a.k_out_stride : a.q_out_stride, key ? a.k_out_head_stride : a.q_out_head_stride, a.tokens, heads, a.head_dim, true)) return rc;
    }
    const uint32_t access = access_of(a);
    Params p = plan(a, access, backward);
    if (sums) {
        const uint64_t need = workspace_of(p);
        if (need && (!workspace || bytes < need)) return refuse(what + ": the workspace must hold " + std::to_string(need) + " bytes");
        if (!aligned16(workspace)) return refuse(what + ": the workspace must be 16-byte aligned");
        p.side[0].parts = static_cast<float*>(workspace);
        p.side[1].parts = p.side[0].parts + static_cast<size_t>(p.side[0].groups) * a.head_dim;
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.tokens == 0) {  // no parts: zeros
        if (a.type == BS_F16)
            rotate_parts_kernel<f16><<<dim3(ceil_div(a.head_dim, 16), 2), 1024, 0, s>>>(p);
        else
            rotate_parts_kernel<bf16><<<dim3(ceil_div(a.head_dim, 16), 2), 1024, 0, s>>>(p);  // of BS_F32: wtype is too
        return launched(what.c_str());
    }
    const int rc = a.type == BS_F32 ? launch<float>(p, access, backward, s) : a.type == BS_F16 ? launch<f16>(p, access, backward, s) : launch<bf16>(p, access, backward, s);
    return rc ? rc : launched(what.c_str());
}

}  // namespace

extern "C" int bs_head_norm_rotary(const bs_head_norm_rotary_args* args, void* stream) try {
    return run("bs_head_norm_rotary", args, false, nullptr, 0, stream);
} catch (...) {
    return bs_internal_exception();
}

extern "C" int bs_head_norm_rotary_backward(const bs_head_norm_rotary_args* args, void* workspace, uint64_t workspace_bytes, void* stream) try {
    return run("bs_head_norm_rotary_backward", args, true, workspace, workspace_bytes, stream);
} catch (...) {
    return bs_internal_exception();
}

extern "C" int bs_head_norm_rotary_backward_workspace(const bs_head_norm_rotary_args* args, uint64_t* bytes) try {
    if (!bytes) return refuse("bs_head_norm_rotary_backward_workspace: bytes is null");
    bs_head_norm_rotary_args a{};
    if (args) a = *args;
    a.frequencies = reinterpret_cast<const double*>(16);  // pointers are not looked at
    if (const int rc = check("bs_head_norm_rotary_backward_workspace", args ? &a : nullptr)) return rc;
    *bytes = a.norm ? workspace_of(plan(a, access_of(a), true)) : 0;
    return BS_OK;
} catch (...) {
    return bs_internal_exception();
}
