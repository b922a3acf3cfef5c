// Element types of the transformer-block operators (fp32, bf16, fp16): conversions, vector loads / stores, dispatch on the C ABI's dtype code.
#pragma once
#include "common.h"

namespace suhpe {

using bf16 = __bf16;
using f16 = _Float16;

template <typename T, int N> struct Vec { typedef T type __attribute__((ext_vector_type(N))); };
template <typename T> struct Vec<T, 1> { typedef T type; };

// N consecutive elements as floats; the address is aligned to N * sizeof(T) bytes (N a power of two, at most 16 bytes)
template <typename T, int N> __device__ __forceinline__ void load_n(const T* p, float* v) {
    if constexpr (N == 1) {
        v[0] = (float)*p;
    } else {
        const typename Vec<T, N>::type t = *reinterpret_cast<const typename Vec<T, N>::type*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)t[i];
    }
}
// one rounding to T (round to nearest even)
template <typename T, int N> __device__ __forceinline__ void store_n(T* p, const float* v) {
    if constexpr (N == 1) {
        *p = (T)v[0];
    } else {
        typename Vec<T, N>::type t;
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = (T)v[i];
        *reinterpret_cast<typename Vec<T, N>::type*>(p) = t;
    }
}

inline int dtype_size(int dtype) { return dtype == SUHPE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == SUHPE_F32 || dtype == SUHPE_BF16 || dtype == SUHPE_F16; }
inline bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// no byte of an output in another output or in an input (outputs first; a null pointer is no range): products of one launch write side by side
struct Range { const void* p; int64_t bytes; };
inline bool apart(const Range* r, int outputs, int count) {
    for (int i = 0; i < outputs; ++i)
        for (int j = i + 1; j < count; ++j) {
            const uintptr_t a = reinterpret_cast<uintptr_t>(r[i].p), b = reinterpret_cast<uintptr_t>(r[j].p);
            if (a && b && a < b + r[j].bytes && b < a + r[i].bytes) return false;
        }
    return true;
}

// Philox4x32-10, the generator of suhpe_dropout_mask: the four words of call number `ctr` under key `seed`
__device__ __forceinline__ void philox_words(uint64_t seed, uint64_t ctr, uint32_t (&w)[4]) {
    uint32_t c0 = (uint32_t)ctr, c1 = (uint32_t)(ctr >> 32), c2 = 0x5355u, c3 = 0x4850u;
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c1 = (uint32_t)p1; c3 = (uint32_t)p0; c0 = n0; c2 = n2;
        k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
    }
    w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

}  // namespace suhpe
