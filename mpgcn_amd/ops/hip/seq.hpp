// Device helpers of the sequence operators (gfx950).
//
// Tensors move in pieces of 16 bytes at any element's address: the hardware
// takes wide accesses that are not aligned, so odd widths, strides and base
// addresses run through the same code. Only a row's last piece may be partial.
#pragma once

#include "common.hpp"
#include "params.hpp"

#define SEQ_CH 8

// Pointers that the compiler cannot trace back to the launch, named as what
// they are: loads and stores through them are global, not generic.
template <typename T>
using gmem = __attribute__((address_space(1))) T*;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(2))) int i32x2;
typedef i32x4 __attribute__((aligned(2))) any16;  // 16, 8, 4 bytes at any bf16's address
typedef i32x2 __attribute__((aligned(2))) any8;
typedef int __attribute__((aligned(2))) any4;

// A piece of E elements as it is in memory, two bf16 to a register: kept so
// while it waits, or each of them would take a register of its own. `n` of the
// elements are there; where that is neither all nor none it is `rem`, the same
// for every thread: what a row's width leaves over.
template <typename T, int E_ = 16 / sizeof(T)>
struct Pack {
    static constexpr int E = E_, W = E * sizeof(T) / 4;      // elements, registers
    static constexpr int WORD = 4 / sizeof(T), HALF = E / 2;  // elements of 4 bytes, of half of 16
    __attribute__((ext_vector_type(W))) int w;

    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) return __int_as_float(w[j]);
        else return __int_as_float(j & 1 ? w[j >> 1] & 0xffff0000 : w[j >> 1] << 16);
    }
    __device__ __forceinline__ void set(const float (&v)[E]) {
        T t[E];
#pragma unroll
        for (int j = 0; j < E; ++j) t[j] = from_f32<T>(v[j]);
        __builtin_memcpy(&w, t, sizeof(w));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = 0;
    }
    __device__ __forceinline__ void load(const T* from, int n, int rem) {
        const auto p = (gmem<const T>)from;
        if (n >= E) {
            if constexpr (W == 4) w = *(gmem<const any16>)p;
            else w = *(gmem<const any8>)p;
            return;
        }
        clear();
        if (rem == 0 || n <= 0) return;
        // halves, words and single bf16 of what is left, each at its own place
        const bool h = W == 4 && (rem & HALF), q = rem & WORD, o = WORD == 2 && (rem & 1);
        i32x2 vh = {0, 0};
        int vq = 0, vo = 0;
        if (h) vh = *(gmem<const any8>)p;
        if (q) vq = *(gmem<const any4>)(p + (h ? HALF : 0));
        if (o) vo = *(gmem<const unsigned short>)(p + (h ? HALF : 0) + (q ? WORD : 0));
        const int a = q ? vq : vo, b = q ? vo : 0;
        w[0] = h ? vh[0] : a;
        w[1] = h ? vh[1] : b;
        if constexpr (W == 4) {
            w[2] = h ? a : 0;
            w[3] = h ? b : 0;
        }
    }
    __device__ __forceinline__ void store(T* to, int n, int rem) const {
        const auto p = (gmem<T>)to;
        if (n >= E) {
            if constexpr (W == 4) *(gmem<any16>)p = w;
            else *(gmem<any8>)p = w;
            return;
        }
        if (rem == 0 || n <= 0) return;
        const bool h = W == 4 && (rem & HALF), q = rem & WORD, o = WORD == 2 && (rem & 1);
        const int a = h ? w[W == 4 ? 2 : 0] : w[0], b = h ? w[W == 4 ? 3 : 1] : w[1];
        if (h) *(gmem<any8>)p = i32x2{w[0], w[1]};
        if (q) *(gmem<any4>)(p + (h ? HALF : 0)) = a;
        if (o) *(gmem<unsigned short>)(p + (h ? HALF : 0) + (q ? WORD : 0)) = (unsigned short)(q ? b : a);
    }
};

// Eight channels as f32; n of them are there, D the row's width.
template <typename T>
struct Raw8 {
    static constexpr int E = Pack<T>::E;
    Pack<T> w[SEQ_CH / E];
    __device__ __forceinline__ float get(int j) const { return w[j / E].get(j % E); }
    // what was formed from it is forgotten
    __device__ __forceinline__ void fresh() {
#pragma unroll
        for (int i = 0; i < SEQ_CH / E; ++i) asm volatile("" : "+v"(w[i].w));
    }
    __device__ __forceinline__ void load(const T* p, int n, int D) {
#pragma unroll
        for (int i = 0; i < SEQ_CH / E; ++i) w[i].load(p + i * E, n - i * E, D % E);
    }
};
template <typename T>
__device__ __forceinline__ void load8(const T* p, int n, int D, float (&v)[SEQ_CH]) {
    Raw8<T> r;
    r.load(p, n, D);
#pragma unroll
    for (int j = 0; j < SEQ_CH; ++j) v[j] = r.get(j);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int n, int D, const float (&v)[SEQ_CH]) {
    constexpr int E = Pack<T>::E;
#pragma unroll
    for (int i = 0; i < SEQ_CH / E; ++i) {
        float t[E];
#pragma unroll
        for (int j = 0; j < E; ++j) t[j] = v[i * E + j];
        Pack<T> k;
        k.set(t);
        k.store(p + i * E, n - i * E, D % E);
    }
}

// Valid length of sequence b, held inside [0, L].
__device__ __forceinline__ int seq_len(const void* lens, int is64, int b, int L) {
    if (!lens) return L;
    const long n = is64 ? ((gmem<const long>)lens)[b] : (long)((gmem<const int>)lens)[b];
    return n < 0 ? 0 : n > L ? L : (int)n;
}

// A grid of `blocks`, and a block's number in it. One dimension of a grid holds
// fewer than 2^32 threads; a launch of more is cut short without an error.
static inline dim3 grid_of(long blocks) {
    const long x = blocks < 1L << 21 ? blocks : 1L << 21;
    return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}
__device__ __forceinline__ long block_id() { return (long)blockIdx.y * gridDim.x + blockIdx.x; }

static inline int pow2_ceil(long n) {
    int p = 1;
    while (p < n) p <<= 1;
    return p;
}
