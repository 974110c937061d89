// Products with bias, activation and residual in the epilogue (include/bs_embed.h).
//
// out = act(x w^T + b) + r.  Both operands are rows of the inner dimension, so tiles of both go to LDS
// as they lie and the matrix instructions read 16 bytes (8 inner elements) per lane.  The weight is the
// instruction's first operand: a lane of the result then holds one row of out and groups of four
// adjacent columns.
#include "bs_embed.hpp"

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
};

__device__ inline float activate(float z, int act) {
    switch (act) {
        case BS_ACT_RELU: return z < 0.0f ? 0.0f : z;
        case BS_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case BS_ACT_GELU_TANH: {
            // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
            const float u = 0.79788456080286536f * fmaf(0.044715f * z * z, z, z);
            return z / (1.0f + __expf(-2.0f * u));
        }
        case BS_ACT_SILU: return z / (1.0f + __expf(-z));
        default: return z;
    }
}

// four adjacent columns of one row: n of them are inside
template <typename T, typename O>
__device__ inline void finish(const Params& p, uint32_t row, uint32_t col, f32x4 z) {
    if (row >= p.rows || col >= p.cols) return;
    const int n = static_cast<int>(p.cols - col);
    if (p.bias) {
        const Vec<T, 4> b = load_some<T, 4>(static_cast<const T*>(p.bias) + col, n);
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] += static_cast<float>(b[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) z[j] = activate(z[j], p.act);
    if (p.residual) {
        const Vec<O, 4> r = load_some<O, 4>(static_cast<const O*>(p.residual) + static_cast<int64_t>(row) * p.rs + col, n);
#pragma unroll
        for (int j = 0; j < 4; ++j) z[j] += static_cast<float>(r[j]);
    }
    Vec<O, 4> o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = static_cast<O>(z[j]);
    store_some<O, 4>(static_cast<O*>(p.out) + static_cast<int64_t>(row) * p.os + col, o, n);
}

// 16-byte chunk c (0..7) of tile row r (64 inner elements = 128 bytes): the 16 lanes of a quarter wave
// read one chunk of 16 rows, which this spreads over all banks
__device__ inline int place(int r, int c) { return r * 64 + ((c ^ ((r >> 1) & 7)) << 3); }

// Any sizes, strides and alignments: tiles of 128 x 128, inner steps of 64, through registers.
template <typename T, typename O>
__global__ __launch_bounds__(256) void linear_kernel(Params p) {
    __shared__ __attribute__((aligned(16))) T tx[128 * 64], tw[128 * 64];
    const T* x = static_cast<const T*>(p.x);
    const T* w = static_cast<const T*>(p.w);
    const uint32_t across = (p.cols + 127) / 128, m0 = blockIdx.x / across * 128, n0 = blockIdx.x % across * 128;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 31, h = lane >> 5;
    const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
    f32x16 acc[2][2] = {};
    for (uint32_t k0 = 0; k0 < p.inner; k0 += 64) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = i * 256 + threadIdx.x, r = at >> 3, c = at & 7;
            const uint32_t k = k0 + c * 8;
            const int n = static_cast<int>(p.inner) - static_cast<int>(k);
            // rows past the end repeat the last one: their products are not stored
            const uint32_t m = m0 + r < p.rows ? m0 + r : p.rows - 1, v = n0 + r < p.cols ? n0 + r : p.cols - 1;
            Vec<T, 8> a = {}, b = {};
            if (n > 0) {
                a = load_some<T, 8>(x + static_cast<int64_t>(m) * p.xs + k, n);
                b = load_some<T, 8>(w + static_cast<int64_t>(v) * p.ws + k, n);
            }
            *reinterpret_cast<Vec<T, 8>*>(tx + place(r, c)) = a;
            *reinterpret_cast<Vec<T, 8>*>(tw + place(r, c)) = b;
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            Vec<T, 8> a[2], b[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                a[i] = *reinterpret_cast<const Vec<T, 8>*>(tw + place(wn + i * 32 + l, s * 2 + h));
                b[i] = *reinterpret_cast<const Vec<T, 8>*>(tx + place(wm + i * 32 + l, s * 2 + h));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = Mma<T>::go(a[i], b[j], acc[i][j]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 z = {acc[i][j][q * 4], acc[i][j][q * 4 + 1], acc[i][j][q * 4 + 2], acc[i][j][q * 4 + 3]};
                finish<T, O>(p, m0 + wm + j * 32 + l, n0 + wn + i * 32 + q * 8 + h * 4, z);
            }
}

template <typename T, typename O>
void launch(const Params& p, hipStream_t s) {
    linear_kernel<T, O><<<(p.cols + 127) / 128 * ((p.rows + 127) / 128), 256, 0, s>>>(p);
}

int check(const char* what, uint64_t rows, uint32_t inner, uint32_t cols) {
    const std::string w = what;
    if (rows > 0x7FFFFFFFull) return refuse(w + ": rows must be < 2^31");
    if (inner == 0 || inner > (1u << 24) || cols == 0 || cols > (1u << 24)) return refuse(w + ": inner and cols must be in 1..2^24");
    if (((rows + 127) >> 7) * ((cols + 127) >> 7) > 0x7FFFFFFFull) return refuse(w + ": rows x cols is too large for one launch");
    return BS_OK;
}

}  // namespace

extern "C" int bs_linear_workspace(uint64_t rows, uint32_t inner, uint32_t cols, uint64_t* bytes) try {
    if (!bytes) return refuse("bs_linear_workspace: bytes is null");
    if (const int rc = check("bs_linear_workspace", rows, inner, cols)) return rc;
    *bytes = 0;
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
    const Params p{x, w, bias, residual, out, x_stride, w_stride, residual_stride, out_stride, static_cast<uint32_t>(rows), inner, cols, activation};
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == BS_F16)
        out_type == BS_F32 ? launch<f16, float>(p, s) : launch<f16, f16>(p, s);
    else
        out_type == BS_F32 ? launch<bf16, float>(p, s) : launch<bf16, bf16>(p, s);
    return launched("bs_linear");
} catch (...) {
    return bs_internal_exception();
}
