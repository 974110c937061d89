// Layer norm and its gradients (include/bs_embed.h).
//
//   y  = (x - mean) rstd w + b,  rstd = 1 / sqrt(var + eps),  xh = (x - mean) rstd
//   dx = rstd (dy w - avg(dy w) - xh avg(dy w xh)),  dw = sum of dy xh and db = sum of dy over the rows
//
// Both directions read each row once and keep it in registers: a row belongs to W wavefronts, a lane to the
// same 8, 16 or 32 columns of every row, so weights are loaded once per wavefront and the gradients of the
// weights grow in registers.  Memory bounds both: 65536 x 1024 in bf16 takes 47 us forward (5.7 TB/s; a copy
// reaches 5.1), 32768 x 4096 takes 147 us backward with 4-byte weights (5.5 TB/s).  Short calls are bounded by
// the latency of their dependent steps: 24 x 768 takes 4.0 us, 1000 x 960 in f32 backward 7.0 + 6.2 us.
#include "bs_embed.hpp"

namespace {
using namespace bse;

constexpr uint32_t MAX_COLS = 16384;

// W waves per row; NV accesses of 16 bytes per lane and row
template <typename T, int NV, int W>
struct Cols {
    static constexpr int N = VN<T>;
    static constexpr int E = N * NV;                    // elements per lane
    static constexpr int THREADS = W == 1 ? 256 : 64 * W;
    static constexpr int ROWS = W == 1 ? 4 : 1;         // rows per workgroup at a time
    __device__ static int lane() { return W == 1 ? (threadIdx.x & 63) : threadIdx.x; }
    __device__ static int col(int i) { return (i * 64 * W + lane()) * N; }
    // columns of the row that wave w holds
    __device__ static int held(int w, int cols) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int left = cols - (i * W + w) * 64 * N;
            n += left <= 0 ? 0 : left < 64 * N ? left : 64 * N;
        }
        return n;
    }
};

template <typename T, int NV, int W, typename S>
__device__ inline void load_cols(const S* p, int cols, float (&out)[Cols<T, NV, W>::E]) {
    using C = Cols<T, NV, W>;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = C::col(i);
        Vec<S, C::N> v = {};
        if (c < cols) v = load_some<S, C::N>(p + c, cols - c);
#pragma unroll
        for (int j = 0; j < C::N; ++j) out[i * C::N + j] = static_cast<float>(v[j]);
    }
}
template <typename T, int NV, int W, typename S>
__device__ inline void store_cols(S* p, int cols, const float (&in)[Cols<T, NV, W>::E]) {
    using C = Cols<T, NV, W>;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = C::col(i);
        Vec<S, C::N> v;
#pragma unroll
        for (int j = 0; j < C::N; ++j) v[j] = static_cast<S>(in[i * C::N + j]);
        if (c < cols) store_some<S, C::N>(p + c, v, cols - c);
    }
}

// The sums of two values over the wave at the price of one: the lower half of the lanes adds up the first, the upper half the
// second, as the first exchange leaves them.
__device__ inline void both_sums(float& a, float& b) {
    const bool low = (threadIdx.x & 63) < 32;
    float v = (low ? a : b) + __shfl_xor(low ? b : a, 32);
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) v += __shfl_xor(v, m);
    a = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 0));
    b = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 32));
}

// Statistics of a row, whose values become their differences from a mean of the wave's own columns.  That mean is off by
// the roundings of a sum of large values where the row lies far from zero; the mean c of the differences corrects it:
// mean = m + c, M2 = sum of d^2 - n c^2.  So neither the variance nor what is normalised, d - off, loses more than the
// roundings of differences, however far the mean lies from zero.  (At 1000 +- 0.001 and 512 columns the first mean alone is
// off by 0.05 deviations.)  Waves' parts are joined about the first one's mean, M2 = sum(M2_w + n_w (mean_w - mean)^2).
struct Stats {
    float mean, off, m2;
};
template <typename T, int NV, int W>
__device__ inline Stats row_stats(int cols, float4* part, float (&x)[Cols<T, NV, W>::E]) {
    using C = Cols<T, NV, W>;
    const int wave = W == 1 ? 0 : threadIdx.x >> 6;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < C::E; ++i) s += x[i];  // 0 past the row
    s = wave_sum(s);
    const int mine = C::held(wave, cols);
    const float over = mine > 0 ? 1.0f / static_cast<float>(mine) : 0.0f, m = s * over;  // the same for all rows
    float q = 0.0f, e = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = C::col(i);
#pragma unroll
        for (int j = 0; j < C::N; ++j) {
            const float d = c + j < cols ? x[i * C::N + j] - m : 0.0f;
            x[i * C::N + j] = d;
            e += d;
            q = fmaf(d, d, q);
        }
    }
    both_sums(e, q);
    const bool fine = fabsf(e) < INFINITY;  // else m, which is not finite either, is the mean
    const float c = fine ? e * over : 0.0f, m2 = fine ? fmaf(-e, c, q) : q;
    Stats r{m + c, c, m2 < 0.0f ? 0.0f : m2};
    if (W > 1) {
        if ((threadIdx.x & 63) == 0) part[wave] = make_float4(m, c, r.m2, 0.0f);
        __syncthreads();
        const float m0 = part[0].x;
        float t = 0.0f;
        for (int w = 0; w < W; ++w) t = fmaf(static_cast<float>(C::held(w, cols)), (part[w].x - m0) + part[w].y, t);
        t /= static_cast<float>(cols);
        r = Stats{m0 + t, t - (m - m0), 0.0f};
        for (int w = 0; w < W; ++w) {
            const int k = C::held(w, cols);
            const float d = k > 0 ? ((part[w].x - m0) + part[w].y) - t : 0.0f;
            r.m2 += fmaf(static_cast<float>(k) * d, d, part[w].z);
        }
        if (!(fabsf(t) < INFINITY)) {  // some wave's mean is not finite
            r.mean = 0.0f;
            for (int w = 0; w < W; ++w) r.mean += C::held(w, cols) > 0 ? part[w].x : 0.0f;
        }
    }
    return r;
}

template <typename T, typename WT, int NV, int W>
__global__ __launch_bounds__((Cols<T, NV, W>::THREADS)) void norm_kernel(const T* x, int64_t xs, const WT* weight, const WT* bias,
                                                                        float eps, T* y, int64_t ys, float* mean_out,
                                                                        float* rstd_out, uint64_t rows, int cols) {
    using C = Cols<T, NV, W>;
    __shared__ float4 part[2][W];
    float w[C::E], b[C::E], v[C::E];
    if (weight) {
        load_cols<T, NV, W>(weight, cols, w);
    } else {
#pragma unroll
        for (int i = 0; i < C::E; ++i) w[i] = 1.0f;
    }
    if (bias) {
        load_cols<T, NV, W>(bias, cols, b);
    } else {
#pragma unroll
        for (int i = 0; i < C::E; ++i) b[i] = 0.0f;
    }
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * C::ROWS;
    int turn = 0;
    for (uint64_t r = static_cast<uint64_t>(blockIdx.x) * C::ROWS + (C::ROWS > 1 ? threadIdx.x >> 6 : 0); r < rows; r += step, turn ^= 1) {
        load_cols<T, NV, W>(x + static_cast<int64_t>(r) * xs, cols, v);
        const Stats st = row_stats<T, NV, W>(cols, part[turn], v);
        const float rstd = 1.0f / sqrtf(st.m2 / static_cast<float>(cols) + eps);
#pragma unroll
        for (int i = 0; i < C::E; ++i) v[i] = fmaf(fmaf(v[i], rstd, -st.off * rstd), w[i], b[i]);
        store_cols<T, NV, W>(y + static_cast<int64_t>(r) * ys, cols, v);
        if (C::lane() == 0) {
            if (mean_out) mean_out[r] = st.mean;
            if (rstd_out) rstd_out[r] = rstd;
        }
    }
}

// dx, and per workgroup the sums over its rows: part[2][cols] (dweight, then dbias)
template <typename T, typename WT, int NV, int W>
__global__ __launch_bounds__((Cols<T, NV, W>::THREADS)) void norm_backward_kernel(
    const T* dy, int64_t dys, const T* x, int64_t xs, const float* mean_in, const float* rstd_in, const WT* weight, T* dx,
    int64_t dxs, float* parts, uint64_t rows, int cols) {
    using C = Cols<T, NV, W>;
    __shared__ float2 part[2][W];
    float w[C::E], dw[C::E], db[C::E];
    if (weight) {
        load_cols<T, NV, W>(weight, cols, w);
    } else {
#pragma unroll
        for (int i = 0; i < C::E; ++i) w[i] = 1.0f;
    }
#pragma unroll
    for (int i = 0; i < C::E; ++i) dw[i] = db[i] = 0.0f;
    const uint64_t step = static_cast<uint64_t>(gridDim.x) * C::ROWS;
    const float over = 1.0f / static_cast<float>(cols);
    int turn = 0;
    for (uint64_t r = static_cast<uint64_t>(blockIdx.x) * C::ROWS + (C::ROWS > 1 ? threadIdx.x >> 6 : 0); r < rows; r += step, turn ^= 1) {
        float g[C::E], h[C::E];
        load_cols<T, NV, W>(dy + static_cast<int64_t>(r) * dys, cols, g);
        load_cols<T, NV, W>(x + static_cast<int64_t>(r) * xs, cols, h);
        const float mean = mean_in[r], rstd = rstd_in[r];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < C::E; ++i) {
            const float xh = (h[i] - mean) * rstd;
            h[i] = xh;
            dw[i] = fmaf(g[i], xh, dw[i]);  // g is 0 past the row
            db[i] += g[i];
            g[i] *= w[i];
            s1 += g[i];
            s2 = fmaf(g[i], xh, s2);
        }
        if (!dx) continue;
        s1 = wave_sum(s1);
        s2 = wave_sum(s2);
        if (W > 1) {
            if ((threadIdx.x & 63) == 0) part[turn][threadIdx.x >> 6] = make_float2(s1, s2);
            __syncthreads();
            s1 = s2 = 0.0f;
            for (int i = 0; i < W; ++i) {
                s1 += part[turn][i].x;
                s2 += part[turn][i].y;
            }
        }
        s1 *= over;
        s2 *= over;
#pragma unroll
        for (int i = 0; i < C::E; ++i) g[i] = rstd * (g[i] - s1 - h[i] * s2);
        store_cols<T, NV, W>(dx + static_cast<int64_t>(r) * dxs, cols, g);
    }
    if (!parts) return;
    float* mine = parts + static_cast<size_t>(blockIdx.x) * 2 * cols;
    if (C::ROWS == 1) {
        store_cols<T, NV, W>(mine, cols, dw);
        store_cols<T, NV, W>(mine + cols, cols, db);
    } else {  // the four waves hold the same columns: joined in wave order
        constexpr int LW = C::ROWS == 1 ? 1 : 64 * C::E;
        __shared__ float join[2][LW];
        const int wave = threadIdx.x >> 6;
        for (int k = 0; k < C::ROWS; ++k) {
            if (wave == k) {
#pragma unroll
                for (int i = 0; i < C::E; ++i) {
                    float* a = &join[0][i * 64 + C::lane()];
                    float* c = &join[1][i * 64 + C::lane()];
                    *a = k ? *a + dw[i] : dw[i];
                    *c = k ? *c + db[i] : db[i];
                }
            }
            __syncthreads();
        }
        if (wave < 2) {
            float v[C::E];
#pragma unroll
            for (int i = 0; i < C::E; ++i) v[i] = join[wave][i * 64 + C::lane()];
            store_cols<T, NV, W>(mine + static_cast<size_t>(wave) * cols, cols, v);
        }
    }
}

// Sums of the workgroups' parts, in order: a workgroup takes 64 columns, wave i the parts i, i + 16, ..  A wave's loads
// wait for memory, so 16 are on their way at a time: 1024 parts of 2 x 4096 take 6.9 us, 18 with one at a time.  What is left of
// n past a multiple of 256 is loaded one at a time, so fewer parts can take longer: 250 of 2 x 960 6.4 us.
template <typename WT>
__global__ __launch_bounds__(1024) void norm_parts_kernel(const float* parts, uint32_t n, int cols, WT* dweight, WT* dbias) {
    __shared__ float join[16][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t c = blockIdx.x * 64 + lane, all = 2u * cols;
    float s = 0.0f;
    if (c < all) {
        constexpr int U = 16;  // loads in flight; the sum stays in order
        uint32_t i = wave;
        for (; i + 16 * (U - 1) < n; i += 16 * U) {
            float v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = parts[static_cast<size_t>(i + 16 * u) * all + c];
#pragma unroll
            for (int u = 0; u < U; ++u) s += v[u];
        }
        for (; i < n; i += 16) s += parts[static_cast<size_t>(i) * all + c];
    }
    join[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < all) {
        for (int i = 1; i < 16; ++i) s += join[i][lane];
        if (c < static_cast<uint32_t>(cols))
            dweight[c] = static_cast<WT>(s);
        else
            dbias[c - cols] = static_cast<WT>(s);
    }
}

// Workgroups of a backward call.  Each writes its sums once, so that fewer are better until loads run short of
// waves: in us at 256 / 512 / 1024 workgroups, 65536 x 768: 107 / 65 / 59; 30000 x 2048: 171 / 95 / 74; 32768 x 4096:
// 240 / 148 / 164; 16384 x 8192: 196 / 161 / 171; 8192 x 16384: 159 / 173 / 200.
uint32_t backward_groups(uint64_t rows, uint32_t cols) {
    const uint32_t per = cols <= 1024 ? 4 : 1;
    const uint64_t want = (rows + per - 1) / per;
    const uint64_t most = CUS * (cols <= 2048 ? 4 : cols <= 8192 ? 2 : 1);
    return static_cast<uint32_t>(want < most ? want : most);
}

struct Forward {
    const void *x, *weight, *bias;
    int64_t xs, ys;
    float eps;
    void* y;
    float *mean, *rstd;
    uint64_t rows;
    int cols;
    hipStream_t s;
    // Few waves meet seldom: 30000 x 2048 takes 43 us with two waves a row and 59 with four, 60000 x 1024 45 with one
    // and 101 with four, 16000 x 8192 97 with four (32 columns a lane) and 109 with eight (16).
    template <typename T, typename WT>
    void pick() const {
        if (cols <= 512)
            go<T, WT, 8 / VN<T>, 1>();
        else if (cols <= 1024)
            go<T, WT, 16 / VN<T>, 1>();
        else if (cols <= 2048)
            go<T, WT, 16 / VN<T>, 2>();
        else if (cols <= 4096)
            go<T, WT, 32 / VN<T>, 2>();
        else if (cols <= 8192)
            go<T, WT, 32 / VN<T>, 4>();
        else
            go<T, WT, 32 / VN<T>, 8>();
    }
    template <typename T, typename WT, int NV, int W>
    void go() const {
        using C = Cols<T, NV, W>;
        // weights are loaded once per workgroup, so they stay for many rows; 2 / 4 / 8 / 16 per compute unit:
        // 65536 x 768: 57 / 39 / 40 / 42 us, 32768 x 4096: 144 / 103 / 104 / 104, 8192 x 16384: 129 / 131 / 139 / 147.
        // Six where six fit at a time (by registers, 16 columns of 16 bits a lane), so that all have the same number of rows:
        // 65536 x 1024 47.3 us, with four 47.6, with eight 51.2; 65536 x 768 in another run 39.8, with eight 43.1
        const uint64_t want = (rows + C::ROWS - 1) / C::ROWS, most = CUS * (W == 8 ? 4 : W == 1 && C::E == 16 && sizeof(T) == 2 ? 6 : 8);
        norm_kernel<T, WT, NV, W><<<static_cast<uint32_t>(want < most ? want : most), C::THREADS, 0, s>>>(
            static_cast<const T*>(x), xs, static_cast<const WT*>(weight), static_cast<const WT*>(bias), eps, static_cast<T*>(y), ys,
            mean, rstd, rows, cols);
    }
};
struct Backward {
    const void *dy, *x, *weight;
    int64_t dys, xs, dxs;
    const float *mean, *rstd;
    void* dx;
    float* parts;
    uint32_t groups;
    uint64_t rows;
    int cols;
    hipStream_t s;
    // A lane holds five values per column here, so a row has more waves than forward: 60000 x 1024 takes 78 us with one
    // wave a row and 98 with four, 30000 x 2048 74 with four and 75 with two, 16000 x 3000 61 and 65, 16000 x 8192 156
    // with four and 154 with eight.  8 columns a lane where they are enough: 60000 x 512 37 us, with 16 39; 60000 x 2048
    // 139 and 143.
    template <typename T, typename WT>
    void pick() const {
        if (cols <= 512)
            go<T, WT, 8 / VN<T>, 1>();
        else if (cols <= 1024)
            go<T, WT, 16 / VN<T>, 1>();
        else if (cols <= 2048)
            go<T, WT, 8 / VN<T>, 4>();
        else if (cols <= 4096)
            go<T, WT, 16 / VN<T>, 4>();
        else if (cols <= 8192)
            go<T, WT, 32 / VN<T>, 4>();
        else
            go<T, WT, 32 / VN<T>, 8>();
    }
    template <typename T, typename WT, int NV, int W>
    void go() const {
        norm_backward_kernel<T, WT, NV, W><<<groups, Cols<T, NV, W>::THREADS, 0, s>>>(
            static_cast<const T*>(dy), dys, static_cast<const T*>(x), xs, mean, rstd, static_cast<const WT*>(weight),
            static_cast<T*>(dx), dxs, parts, rows, cols);
    }
};

template <typename F>
void by_type(const F& f, int type, int wtype) {
    if (type == BS_F32)
        f.template pick<float, float>();
    else if (type == BS_F16)
        wtype == BS_F32 ? f.template pick<f16, float>() : f.template pick<f16, f16>();
    else
        wtype == BS_F32 ? f.template pick<bf16, float>() : f.template pick<bf16, bf16>();
}

int check(const char* what, uint64_t rows, uint32_t cols, int type, int wtype) {
    const std::string w = what;
    if (type < BS_F32 || type > BS_BF16) return refuse(w + ": type must be BS_F32, BS_F16 or BS_BF16");
    if (wtype != type && wtype != BS_F32) return refuse(w + ": wtype must be the rows' type or BS_F32");
    if (cols == 0 || cols > MAX_COLS) return refuse(w + ": cols must be in 1.." + std::to_string(MAX_COLS));
    if (rows > 0x7FFFFFFFull) return refuse(w + ": rows must be < 2^31");
    return BS_OK;
}

}  // namespace

extern "C" int bs_layer_norm(const void* x, int64_t x_stride, const void* weight, const void* bias, int wtype, float eps, void* y,
                             int64_t y_stride, float* mean, float* rstd, uint64_t rows, uint32_t cols, int type,
                             void* stream) try {
    if (const int rc = check("bs_layer_norm", rows, cols, type, wtype)) return rc;
    if (!(eps >= 0.0f)) return refuse("bs_layer_norm: eps must be >= 0");
    if (rows == 0) return BS_OK;
    if (!x || !y) return refuse("bs_layer_norm: x and y must be given");
    if (x_stride < cols || y_stride < cols) return refuse("bs_layer_norm: rows overlap (stride < cols)");
    by_type(Forward{x, weight, bias, x_stride, y_stride, eps, y, mean, rstd, rows, static_cast<int>(cols),
                    static_cast<hipStream_t>(stream)},
            type, wtype);
    return launched("bs_layer_norm");
} catch (...) {
    return bs_internal_exception();
}

extern "C" int bs_layer_norm_backward_workspace(uint64_t rows, uint32_t cols, int type, uint64_t* bytes) try {
    if (!bytes) return refuse("bs_layer_norm_backward_workspace: bytes is null");
    if (const int rc = check("bs_layer_norm_backward_workspace", rows, cols, type, type)) return rc;
    *bytes = static_cast<uint64_t>(backward_groups(rows, cols)) * 2 * cols * sizeof(float);
    return BS_OK;
} catch (...) {
    return bs_internal_exception();
}

extern "C" int bs_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const float* mean,
                                      const float* rstd, const void* weight, int wtype, void* dx, int64_t dx_stride,
                                      void* dweight, void* dbias, uint64_t rows, uint32_t cols, int type, void* workspace,
                                      uint64_t workspace_bytes, void* stream) try {
    if (const int rc = check("bs_layer_norm_backward", rows, cols, type, wtype)) return rc;
    if (!dweight != !dbias) return refuse("bs_layer_norm_backward: dweight and dbias must be given together");
    if (rows && (!dy || !x || !mean || !rstd)) return refuse("bs_layer_norm_backward: dy, x, mean and rstd must be given");
    if (rows && (dy_stride < cols || x_stride < cols || (dx && dx_stride < cols)))
        return refuse("bs_layer_norm_backward: rows overlap (stride < cols)");
    const uint32_t groups = backward_groups(rows, cols);
    if (dweight && groups) {
        const uint64_t need = static_cast<uint64_t>(groups) * 2 * cols * sizeof(float);
        if (!workspace || workspace_bytes < need)
            return refuse("bs_layer_norm_backward: the workspace must hold " + std::to_string(need) + " bytes");
        if (!aligned16(workspace)) return refuse("bs_layer_norm_backward: the workspace must be 16-byte aligned");
    }
    const hipStream_t s = static_cast<hipStream_t>(stream);
    float* parts = dweight ? static_cast<float*>(workspace) : nullptr;
    if (groups && (dx || dweight))
        by_type(Backward{dy, x, weight, dy_stride, x_stride, dx_stride, mean, rstd, dx, parts, groups, rows,
                         static_cast<int>(cols), s},
                type, wtype);
    if (dweight) {  // also without rows: the sums are then 0
        const uint32_t blocks = (2 * cols + 63) / 64;
        if (wtype == BS_F32)
            norm_parts_kernel<float><<<blocks, 1024, 0, s>>>(parts, groups, cols, static_cast<float*>(dweight), static_cast<float*>(dbias));
        else if (wtype == BS_F16)
            norm_parts_kernel<f16><<<blocks, 1024, 0, s>>>(parts, groups, cols, static_cast<f16*>(dweight), static_cast<f16*>(dbias));
        else
            norm_parts_kernel<bf16><<<blocks, 1024, 0, s>>>(parts, groups, cols, static_cast<bf16*>(dweight), static_cast<bf16*>(dbias));
    }
    return launched("bs_layer_norm_backward");
} catch (...) {
    return bs_internal_exception();
}
