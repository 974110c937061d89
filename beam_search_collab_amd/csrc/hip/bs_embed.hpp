// What the encoder operators share: element types, 16-byte accesses at any element alignment,
// wave sums, argument checks.  Declarations of the entry points: include/bs_embed.h.
#pragma once
#include "bs_embed.h"
#include "bs_hip.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

void bs_internal_set_error(const std::string& msg);
int bs_internal_exception();

namespace bse {

using f16 = _Float16;
using bf16 = __bf16;

constexpr uint32_t CUS = 256;  // of the MI355X; sizes grids, results do not depend on it

inline int refuse(const std::string& msg) {
    bs_internal_set_error(msg);
    return BS_EINVAL;
}
inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return BS_OK;
    bs_internal_set_error(std::string(what) + " launch failed: " + hipGetErrorString(e));
    return BS_EHIP;
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <typename T>
constexpr int VN = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte access
template <typename T, int N>
using Vec = T __attribute__((ext_vector_type(N)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// N elements from any element boundary: gfx950 takes 16-byte accesses at every address, and one
// that crosses a cache line costs one more line access, not a second instruction
template <typename T, int N>
__device__ inline Vec<T, N> load_any(const T* p) {
    Vec<T, N> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <typename T, int N>
__device__ inline void store_any(T* p, Vec<T, N> v) {
    __builtin_memcpy(p, &v, sizeof(v));
}
// the first n (0..N) of N elements, 0 past them
template <typename T, int N>
__device__ inline Vec<T, N> load_some(const T* p, int n) {
    if (n >= N) return load_any<T, N>(p);
    Vec<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? p[i] : static_cast<T>(0.0f);
    return v;
}
template <typename T, int N>
__device__ inline void store_some(T* p, Vec<T, N> v, int n) {
    if (n >= N) {
        store_any<T, N>(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < n) p[i] = v[i];
}

// sum over the 64 lanes, the same bits in every lane
__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

}  // namespace bse
