// What the encoder operators share: element types, 16-byte accesses at any element alignment,
// wave sums, argument checks.  Declarations of the entry points: include/bs_embed.h.
#pragma once
#include "bs_embed.h"
#include "bs_hip.h"

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>
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
// Lets a kernel use more than 64 KB of dynamic LDS: once per device and kernel (`done`: a bit per device)
inline int allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e == hipSuccess && (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1))) {
        e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == hipSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    if (e == hipSuccess) return BS_OK;
    bs_internal_set_error(std::string("hipFuncSetAttribute failed: ") + hipGetErrorString(e));
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
// the same for elements that the kernel reads once: they do not displace others from the caches
template <typename T, int N>
__device__ inline Vec<T, N> load_once(const T* p) {
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    return __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
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

typedef __attribute__((address_space(1))) const void* global_ptr;
typedef __attribute__((address_space(3))) void* lds_ptr;

// a value that all lanes share, to scalar registers
__device__ inline uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline uint64_t uniform(uint64_t v) {
    return static_cast<uint64_t>(uniform(static_cast<uint32_t>(v >> 32))) << 32 | uniform(static_cast<uint32_t>(v));
}

// 16 bytes a lane from base + offset to LDS, where the wave's lanes follow each other from `to` on.  The base stays
// in scalar registers: the compiler would otherwise carry a 64-bit address per lane and move, and a wave that
// computes addresses issues nothing else (attention spent 1100 of 4300 cycles per tile on eight moves so).
__device__ inline void move16(const char* base, uint32_t offset, void* to) {
    uint64_t b = uniform(reinterpret_cast<uint64_t>(base));
    asm volatile("" : "+s"(b), "+v"(offset));
    __builtin_amdgcn_global_load_lds((global_ptr)(reinterpret_cast<const char*>(b) + offset), (lds_ptr)to, 16, 0, 0);
}

// n / d for n < 2^31 and one d: floor(n m / 2^(31 + s)) with s = ceil(log2 d), m = ceil(2^(31 + s) / d) < 2^32.  (m d -
// 2^(31 + s) < d <= 2^s, so the quotient is off by less than n / 2^31 / d and never reaches the next integer.)
struct Divisor {
    uint32_t m, s;
    Divisor(uint32_t d = 1) : m(0), s(0) {
        while ((1ull << s) < d) ++s;
        m = static_cast<uint32_t>(((1ull << (31 + s)) + d - 1) / d);
    }
    __device__ uint32_t quotient(uint32_t n) const { return __umulhi(n << 1, m) >> s; }
};

// sum over the 64 lanes, the same bits in every lane
__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

}  // namespace bse
