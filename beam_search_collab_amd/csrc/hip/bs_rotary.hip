// Norm of every head of queries and keys with the rotation by their positions, and its gradients (include/bs_embed.h).
//
//   r = 1 / sqrt(mean(x^2) + eps),  y = M(pos) (x r w),  M: pairs turned by the angles pos f, times the magnitude
//   d = M^T dy,  dw = sum of d x r over tokens and heads,  dx = r (d w - x r^2 mean(d w x))
//
// A workgroup takes a few tokens: first their angles, each once, to LDS, then their heads, one after another.  A head
// belongs to a few lanes, each with 2 N elements in two accesses of N: the two halves of N pairs (elements i and i +
// rotary / 2) or 2 N neighbours, so that both partners of a pair are the lane's.
#include "bs_embed.hpp"

#include <algorithm>
#include <cmath>

namespace {
using namespace bse;

constexpr uint32_t THREADS = 256, WAVES = THREADS / 64;
constexpr uint32_t MOST_PARTS = 2 * CUS;  // workgroups of the gradients

struct Params {
    bs_head_norm_rotary_args a;
    uint32_t block, blocks;   // tokens of a workgroup's turn, and such turns
    uint32_t lanes, shift;    // of a head: 2^shift
    uint32_t rotated, units;  // accesses of a head in pairs of N: those with pairs to turn come first
    Divisor by_heads, by_kv, by_half;
    float* parts;             // of the weights' gradients: workgroups x 2 x head_dim
};

// N elements from two places of a head, K times
template <int N, int K>
struct Unit {
    float a[K][N], b[K][N];
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
        x.a = p.a.rotary + (u - p.rotated) * 2 * N;
        x.b = x.a + N;
    } else if (p.a.interleaved) {
        x.a = u * 2 * N;
        x.b = x.a + N;
    } else {
        x.a = u * N;
        x.b = p.a.rotary / 2 + u * N;
    }
    return x;
}
template <typename S, int N>
__device__ inline void take(const S* p, float (&out)[N]) {
    const Vec<S, N> v = load_any<S, N>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = static_cast<float>(v[i]);
}
template <typename T, int N, int K>
__device__ inline void load(const T* head, const Places (&at)[K], bool live, Unit<N, K>& x) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int i = 0; i < N; ++i) x.a[k][i] = x.b[k][i] = 0.0f;
        if (live && at[k].live) {
            take<T, N>(head + at[k].a, x.a[k]);
            take<T, N>(head + at[k].b, x.b[k]);
        }
    }
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
// a weight of `wtype`, or 1
template <typename T, int N, int K>
__device__ inline void load_weight(const void* w, int wtype, const Places (&at)[K], Unit<N, K>& x) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) x.a[k][i] = x.b[k][i] = 1.0f;
    if (!w) return;
    if (wtype == BS_F32)
        load<float, N, K>(static_cast<const float*>(w), at, true, x);
    else
        load<T, N, K>(static_cast<const T*>(w), at, true, x);
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
    const uint32_t half = p.a.rotary / 2;
    for (uint32_t i = threadIdx.x; i < n * half; i += THREADS) {
        const uint32_t tok = p.by_half.quotient(i), j = i - tok * half;
        const double pos = p.a.positions ? static_cast<double>(p.a.positions[t0 + tok]) : static_cast<double>(t0 + tok);
        double turns = pos * (p.a.frequencies[j] * 0.15915494309189533577);
        turns = (turns - rint(turns)) * 4.0;
        const double quarters = rint(turns);
        float s, c;
        eighth(static_cast<float>(turns - quarters), s, c);
        const int q = static_cast<int>(quarters);
        const float cs = q & 1 ? s : c, sn = q & 1 ? c : s;
        table[tok * p.a.rotary + j] = ((q + 1) & 2 ? -cs : cs) * p.a.magnitude;
        table[tok * p.a.rotary + half + j] = (q & 2 ? -sn : sn) * p.a.magnitude;
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
        const Vec<float, N> c = *reinterpret_cast<const Vec<float, N>*>(t), up = *reinterpret_cast<const Vec<float, N>*>(t + p.a.rotary / 2);
        const Vec<float, N> s = Back ? -up : up;
        auto pair = [&](float& a, float& b, int i) {
            const float u = a;
            a = fmaf(u, c[i], -(b * s[i]));
            b = fmaf(b, c[i], u * s[i]);
        };
        if (N == 1 || !p.a.interleaved) {
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
// sum over a head's lanes
__device__ inline float head_sum(float v, uint32_t lanes) {
    for (uint32_t m = 1; m < lanes; m <<= 1) v += __shfl_xor(v, m);
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

// a head of a workgroup's tokens: pass by pass, first those of the queries
struct Row {
    uint32_t tok, head;  // tok in the workgroup's turn
    bool key, live;
};
struct Turn {
    uint32_t t0, n, queries, keys, passes, query_passes;
    __device__ Turn(const Params& p, uint32_t block) : t0(block * p.block), n(min(p.block, p.a.tokens - t0)) {
        const uint32_t slots = 64u >> p.shift;
        queries = n * p.a.heads;
        keys = n * p.a.kv_heads;
        query_passes = (queries + slots - 1) / slots;
        passes = query_passes + (keys + slots - 1) / slots;
    }
    __device__ Row row(const Params& p, uint32_t pass) const {
        Row r;
        r.key = pass >= query_passes;
        const uint32_t i = (r.key ? pass - query_passes : pass) * (64u >> p.shift) + ((threadIdx.x & 63) >> p.shift);
        r.live = i < (r.key ? keys : queries);
        r.tok = r.key ? p.by_kv.quotient(i) : p.by_heads.quotient(i);
        r.head = i - r.tok * (r.key ? p.a.kv_heads : p.a.heads);
        return r;
    }
};
template <typename T>
__device__ inline T* head_of(const void* base, int64_t stride, int64_t head_stride, uint32_t t0, const Row& r) {
    return const_cast<T*>(static_cast<const T*>(base)) + static_cast<int64_t>(t0 + r.tok) * stride + static_cast<int64_t>(r.head) * head_stride;
}

template <typename T, int N, int K>
__global__ __launch_bounds__(THREADS) void rotate_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) float table[];
    const bs_head_norm_rotary_args& a = p.a;
    const uint32_t lane = threadIdx.x & (p.lanes - 1), wave = uniform(threadIdx.x >> 6);
    Places at[K];
#pragma unroll
    for (int k = 0; k < K; ++k) at[k] = places_of<N>(p, lane + k * p.lanes);
    Unit<N, K> wq, wk;
    load_weight<T, N, K>(a.q_weight, a.wtype, at, wq);
    load_weight<T, N, K>(a.k_weight, a.wtype, at, wk);
    const float over = 1.0f / static_cast<float>(a.head_dim);
    for (uint32_t b = blockIdx.x; b < p.blocks; b += gridDim.x) {
        const Turn turn_(p, b);
        auto fetch = [&](uint32_t pass, Row& r, Unit<N, K>& x) {
            r = turn_.row(p, pass);
            load<T, N, K>(r.key ? head_of<T>(a.k, a.k_stride, a.k_head_stride, turn_.t0, r) : head_of<T>(a.q, a.q_stride, a.q_head_stride, turn_.t0, r),
                          at, r.live, x);
        };
        Row r, next;
        Unit<N, K> x, y;
        if (wave < turn_.passes) fetch(wave, r, x);
        __syncthreads();  // nobody reads the last turn's angles any more
        angles(p, table, turn_.t0, turn_.n);
        __syncthreads();
        for (uint32_t pass = wave; pass < turn_.passes; pass += WAVES) {
            if (pass + WAVES < turn_.passes) fetch(pass + WAVES, next, y);
            if (a.norm) {
                const float rstd = inverse_root(fmaf(head_sum(dot(x, x), p.lanes), over, a.eps));
                const Unit<N, K>& w = r.key ? wk : wq;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        x.a[k][i] = x.a[k][i] * rstd * w.a[k][i];
                        x.b[k][i] = x.b[k][i] * rstd * w.b[k][i];
                    }
            }
            turn<false>(p, table + (r.live ? r.tok : 0) * a.rotary, at, lane, x);
            store<T, N, K>(r.key ? head_of<T>(a.k_out, a.k_out_stride, a.k_out_head_stride, turn_.t0, r)
                                 : head_of<T>(a.q_out, a.q_out_stride, a.q_out_head_stride, turn_.t0, r),
                           at, r.live, x);
            r = next;
            x = y;
        }
    }
}

template <typename T, int N, int K>
__global__ __launch_bounds__(THREADS) void rotate_backward_kernel(Params p) {
    extern __shared__ __attribute__((aligned(16))) float table[];
    const bs_head_norm_rotary_args& a = p.a;
    const uint32_t lane = threadIdx.x & (p.lanes - 1), wave = uniform(threadIdx.x >> 6);
    Places at[K];
#pragma unroll
    for (int k = 0; k < K; ++k) at[k] = places_of<N>(p, lane + k * p.lanes);
    Unit<N, K> wq, wk, dwq = {}, dwk = {};
    load_weight<T, N, K>(a.q_weight, a.wtype, at, wq);
    load_weight<T, N, K>(a.k_weight, a.wtype, at, wk);
    const float over = 1.0f / static_cast<float>(a.head_dim);
    for (uint32_t b = blockIdx.x; b < p.blocks; b += gridDim.x) {
        const Turn turn_(p, b);
        __syncthreads();
        angles(p, table, turn_.t0, turn_.n);
        __syncthreads();
        for (uint32_t pass = wave; pass < turn_.passes; pass += WAVES) {
            const Row r = turn_.row(p, pass);
            Unit<N, K> x, d;
            load<T, N, K>(r.key ? head_of<T>(a.k_grad, a.k_grad_stride, a.k_grad_head_stride, turn_.t0, r)
                                : head_of<T>(a.q_grad, a.q_grad_stride, a.q_grad_head_stride, turn_.t0, r),
                          at, r.live, d);
            if (a.norm)
                load<T, N, K>(r.key ? head_of<T>(a.k, a.k_stride, a.k_head_stride, turn_.t0, r) : head_of<T>(a.q, a.q_stride, a.q_head_stride, turn_.t0, r),
                              at, r.live, x);
            turn<true>(p, table + (r.live ? r.tok : 0) * a.rotary, at, lane, d);
            if (a.norm) {
                const float rstd = inverse_root(fmaf(head_sum(dot(x, x), p.lanes), over, a.eps));
                auto side = [&](const Unit<N, K>& w, Unit<N, K>& dw) {
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
                            d.a[k][i] *= w.a[k][i];
                            d.b[k][i] *= w.b[k][i];
                        }
                };
                if (r.key)
                    side(wk, dwk);
                else
                    side(wq, dwq);
                const float along = head_sum(dot(d, x), p.lanes) * over;
#pragma unroll
                for (int k = 0; k < K; ++k)
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        d.a[k][i] = rstd * fmaf(-along, x.a[k][i], d.a[k][i]);
                        d.b[k][i] = rstd * fmaf(-along, x.b[k][i], d.b[k][i]);
                    }
            }
            store<T, N, K>(r.key ? head_of<T>(a.k_out, a.k_out_stride, a.k_out_head_stride, turn_.t0, r)
                                 : head_of<T>(a.q_out, a.q_out_stride, a.q_out_head_stride, turn_.t0, r),
                           at, r.live, d);
        }
    }
    if (!p.parts) return;
    // the workgroup's sums: over the wave's heads by exchanges, over the waves through LDS, in a fixed order
    __shared__ float sums[WAVES][2][256];
    auto add = [&](float v) {
        for (uint32_t m = p.lanes; m < 64; m <<= 1) v += __shfl_xor(v, m);
        return v;
    };
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float qa = add(dwq.a[k][i]), qb = add(dwq.b[k][i]), ka = add(dwk.a[k][i]), kb = add(dwk.b[k][i]);
            if ((threadIdx.x & 63) < p.lanes && at[k].live) {
                sums[wave][0][at[k].a + i] = qa;
                sums[wave][0][at[k].b + i] = qb;
                sums[wave][1][at[k].a + i] = ka;
                sums[wave][1][at[k].b + i] = kb;
            }
        }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < 2 * a.head_dim; i += THREADS) {
        const uint32_t side = i >= a.head_dim, c = i - side * a.head_dim;
        float s = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) s += sums[w][side][c];
        p.parts[static_cast<size_t>(blockIdx.x) * 2 * a.head_dim + i] = s;
    }
}

// the workgroups' parts of the weights' gradients: 16 columns a workgroup, 64 runs of parts each, in a fixed order
template <typename T>
__global__ __launch_bounds__(1024) void rotate_parts_kernel(Params p, uint32_t parts) {
    __shared__ float sums[64][17];
    const bs_head_norm_rotary_args& a = p.a;
    const uint32_t x = threadIdx.x & 15, y = threadIdx.x >> 4, c = blockIdx.x * 16 + x, wide = 2 * a.head_dim;
    float s = 0.0f;
    if (c < wide) {
#pragma unroll 4
        for (uint32_t i = y; i < parts; i += 64) s += p.parts[static_cast<size_t>(i) * wide + c];
    }
    sums[y][x] = s;
    __syncthreads();
    for (uint32_t m = 32; m; m >>= 1) {
        if (y < m) sums[y][x] += sums[y + m][x];
        __syncthreads();
    }
    if (y || c >= wide) return;
    const bool key = c >= a.head_dim;
    void* out = key ? a.k_weight_grad : a.q_weight_grad;
    const uint32_t i = key ? c - a.head_dim : c;
    if (!out) return;
    if (a.wtype == BS_F32)
        static_cast<float*>(out)[i] = sums[0][x];
    else
        static_cast<T*>(out)[i] = static_cast<T>(sums[0][x]);
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
    p.a = a;
    p.rotated = a.rotary / 2 / access;
    p.units = a.head_dim / 2 / access;
    const uint32_t held = access == 1 ? ceil_div(p.units, 2) : p.units;  // lanes that a head needs
    while ((1u << p.shift) < held) ++p.shift;
    p.lanes = 1u << p.shift;
    const uint32_t slots = 64 >> p.shift, heads = a.heads + a.kv_heads;
    // tokens of a turn: four passes a wave, less where that leaves compute units without work, and angles within 16 KB
    uint32_t block = std::max(1u, 4 * WAVES * slots / heads);
    block = std::min(block, ceil_div(a.tokens, 4 * CUS));
    if (a.rotary) block = std::min(block, 16384 / (4 * a.rotary));
    p.block = std::max(1u, block);
    p.blocks = ceil_div(a.tokens, p.block);
    p.by_heads = Divisor(a.heads);
    p.by_kv = Divisor(a.kv_heads ? a.kv_heads : 1);
    p.by_half = Divisor(a.rotary ? a.rotary / 2 : 1);
    return p;
}

uint32_t parts_of(const Params& p) { return std::min(p.blocks, MOST_PARTS); }

template <typename T, int N, int K>
int start(const Params& p, bool backward, hipStream_t s) {
    const uint32_t lds = p.block * p.a.rotary * 4;
    if (!backward) {
        rotate_kernel<T, N, K><<<std::min(p.blocks, 1u << 23), THREADS, lds, s>>>(p);
        return BS_OK;
    }
    const uint32_t parts = parts_of(p);
    rotate_backward_kernel<T, N, K><<<p.parts ? parts : std::min(p.blocks, 1u << 23), THREADS, lds, s>>>(p);
    if (p.parts) rotate_parts_kernel<T><<<ceil_div(2 * p.a.head_dim, 16), 1024, 0, s>>>(p, parts);
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
uint64_t workspace_of(const Params& p) { return static_cast<uint64_t>(parts_of(p)) * 2 * p.a.head_dim * sizeof(float); }

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
        p.parts = static_cast<float*>(workspace);
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (a.tokens == 0) {  // no parts: zeros
        if (a.type == BS_F16)
            rotate_parts_kernel<f16><<<ceil_div(2 * a.head_dim, 16), 1024, 0, s>>>(p, 0);
        else
            rotate_parts_kernel<bf16><<<ceil_div(2 * a.head_dim, 16), 1024, 0, s>>>(p, 0);  // of BS_F32: wtype is too
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
