// Device helpers of the sequence operators (gfx950).
//
// Tensors are read in chunks of 8 channels: 16 bytes of bf16 or 32 of f32. A
// chunk that cannot be read whole (odd width, odd stride, odd base address)
// is read one element at a time by the same code.
#pragma once

#include "common.hpp"
#include "params.hpp"

#define SEQ_CH 8

// Pointers that the compiler cannot trace back to the launch, named as what
// they are: loads and stores through them are global, not generic.
template <typename T>
using gmem = __attribute__((address_space(1))) T*;
typedef __attribute__((ext_vector_type(4))) int i32x4;

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, float (&v)[SEQ_CH]) {
    if constexpr (VEC) {
        Chunk16 c[SEQ_CH * sizeof(T) / 16];
#pragma unroll
        for (int i = 0; i < (int)(SEQ_CH * sizeof(T) / 16); ++i) c[i] = ((const Chunk16*)p)[i];
        const T* e = (const T*)c;
#pragma unroll
        for (int j = 0; j < SEQ_CH; ++j) v[j] = to_f32(e[j]);
    } else {
#pragma unroll
        for (int j = 0; j < SEQ_CH; ++j) v[j] = j < n ? to_f32(p[j]) : 0.f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, const float (&v)[SEQ_CH]) {
    if constexpr (VEC) {
        Chunk16 c[SEQ_CH * sizeof(T) / 16];
        T* e = (T*)c;
#pragma unroll
        for (int j = 0; j < SEQ_CH; ++j) e[j] = from_f32<T>(v[j]);
#pragma unroll
        for (int i = 0; i < (int)(SEQ_CH * sizeof(T) / 16); ++i) ((Chunk16*)p)[i] = c[i];
    } else {
#pragma unroll
        for (int j = 0; j < SEQ_CH; ++j)
            if (j < n) p[j] = from_f32<T>(v[j]);
    }
}

__device__ __forceinline__ void zero8(float (&v)[SEQ_CH]) {
#pragma unroll
    for (int j = 0; j < SEQ_CH; ++j) v[j] = 0.f;
}

// Valid length of sequence b, held inside [0, L].
__device__ __forceinline__ int seq_len(const void* lens, int is64, int b, int L) {
    if (!lens) return L;
    const long n = is64 ? ((gmem<const long>)lens)[b] : (long)((gmem<const int>)lens)[b];
    return n < 0 ? 0 : n > L ? L : (int)n;
}

// log(1 + e^x) without overflow; the tail keeps full relative accuracy.
__device__ __forceinline__ float softplus_f(float x) {
    return fmaxf(x, 0.f) + log1pf(__expf(-fabsf(x)));
}

// 16 bytes as they are in memory, two bf16 to a register: kept so while they
// wait, or each of them would take a register of its own.
template <typename T>
struct Pack {
    static constexpr int E = 16 / sizeof(T);
    i32x4 w;

    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) return __int_as_float(w[j]);
        else return __int_as_float(j & 1 ? w[j >> 1] & 0xffff0000 : w[j >> 1] << 16);
    }
    // n of the E elements are there; VEC: all, and aligned
    template <bool VEC>
    __device__ __forceinline__ void load(const T* p, int n) {
        if constexpr (VEC) {
            w = *(const i32x4*)p;
        } else {
            T v[E];
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = j < n ? p[j] : (T)0.f;
            __builtin_memcpy(&w, v, 16);
        }
    }
};

static inline int pow2_ceil(long n) {
    int p = 1;
    while (p < n) p <<= 1;
    return p;
}
