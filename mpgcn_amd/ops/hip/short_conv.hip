// Short causal convolution over time, one filter of K taps per channel
// (gfx950):  s[t] = bias + sum_k w[k] x[t - K + 1 + k],  y[t] = silu(s[t]).
//
// Bound by memory: 2K flops against one element read and one written. A thread
// owns 8 channels (16 bytes of bf16) and walks the time axis with the last
// K - 1 inputs in registers, so an input is read once per tile and again only
// by the K - 1 outputs that the next tile shares with it.
#include "seq.hpp"

#define CONV_TT 8    // outputs a thread computes in one tile, forward
#define CONV_BT 16   // the same, backward (each tile recomputes K - 1 gradients)

namespace {

__device__ __forceinline__ float silu_f(float s) { return s * fast_sigmoid(s); }

// Input t of sequence b: the carried state before the first, zero before that.
template <typename T, int K, bool VEC>
__device__ __forceinline__ void input8(const ShortConvParams& p, const T* x, const T* s0, int t,
                                       int len, int n, float (&v)[SEQ_CH]) {
    if (t >= 0 && t < len)
        load8<T, VEC>(x + t * p.x_t, n, v);
    else if (t < 0 && t >= -(K - 1) && s0)
        load8<T, VEC>(s0 + (long)(t + K - 1) * p.D, n, v);
    else
        zero8(v);
}

template <int K>
__device__ __forceinline__ void taps8(const ShortConvParams& p, int c0, int n, float (&w)[K][SEQ_CH],
                                      float (&bias)[SEQ_CH]) {
#pragma unroll
    for (int j = 0; j < SEQ_CH; ++j) {
        bias[j] = (p.bias && j < n) ? p.bias[c0 + j] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][j] = j < n ? p.w[(long)(c0 + j) * K + k] : 0.f;
    }
}

template <typename T, int K, bool VEC>
__launch_bounds__(256) __global__ void short_conv_fwd_kernel(ShortConvParams p, long items, int dv,
                                                             int tiles) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const int c0 = (int)(i % dv) * SEQ_CH;
    const long r = i / dv;
    const int tile = (int)(r % tiles), b = (int)(r / tiles);
    const int n = p.D - c0 < SEQ_CH ? p.D - c0 : SEQ_CH;
    const int len = seq_len(p.lens, p.lens64, b, p.L);
    const T* x = (const T*)p.x + b * p.x_b + c0;
    const T* s0 = p.s0 ? (const T*)p.s0 + (long)b * (K - 1) * p.D + c0 : nullptr;
    T* y = (T*)p.y + (long)b * p.L * p.D + c0;

    const int t0 = tile * CONV_TT;
    const int t1 = t0 + CONV_TT < p.L ? t0 + CONV_TT : p.L;
    float w[K][SEQ_CH], bias[SEQ_CH], in[CONV_TT + K - 1][SEQ_CH];
    // every load of the tile is in flight before the first is used
#pragma unroll
    for (int j = 0; j < CONV_TT + K - 1; ++j)
        input8<T, K, VEC>(p, x, s0, t0 + j - (K - 1), len, n, in[j]);
    taps8<K>(p, c0, n, w, bias);
#pragma unroll
    for (int j = 0; j < CONV_TT; ++j) {
        if (t0 + j >= t1) break;
        float o[SEQ_CH];
#pragma unroll
        for (int c = 0; c < SEQ_CH; ++c) {
            float s = bias[c];
#pragma unroll
            for (int k = 0; k < K; ++k) s = fmaf(w[k][c], in[j + k][c], s);
            o[c] = t0 + j < len ? (p.silu ? silu_f(s) : s) : 0.f;
        }
        store8<T, VEC>(y + (long)(t0 + j) * p.D, n, o);
    }
    if (p.s1 && tile == 0) {
        T* s1 = (T*)p.s1 + (long)b * (K - 1) * p.D + c0;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            float v[SEQ_CH];
            input8<T, K, VEC>(p, x, s0, len - (K - 1) + j, len, n, v);
            store8<T, VEC>(s1 + (long)j * p.D, n, v);
        }
    }
}

// Backward: ds[t] = dy[t] silu'(s[t]) with s recomputed, dx[t] = sum_k w[k]
// ds[t + K - 1 - k], dw[k] = sum ds[t] x[t - K + 1 + k]. A thread streams one
// tile in time order holding the last K inputs and the last K values of ds;
// filter gradients stay in registers over all of its tiles, are joined per
// block and written once, then summed in a fixed order (no atomics).
template <typename T, int K, bool VEC>
__launch_bounds__(256) __global__ void short_conv_bwd_kernel(ShortConvParams p, int dv, int cw,
                                                             int tiles) {
    extern __shared__ float lds[];  // [256][SEQ_CH * (K + 1)]
    const int rt = threadIdx.x / cw, nrt = 256 / cw;
    const int cv = blockIdx.y * cw + threadIdx.x % cw;
    const int c0 = cv * SEQ_CH;
    const bool live = cv < dv;
    const int n = p.D - c0 < SEQ_CH ? p.D - c0 : SEQ_CH;
    float dw[K][SEQ_CH] = {}, db[SEQ_CH] = {};
    if (live) {
        float w[K][SEQ_CH], bias[SEQ_CH];
        taps8<K>(p, c0, n, w, bias);
        const long items = (long)p.B * tiles;
        for (long i = (long)blockIdx.x * nrt + rt; i < items; i += (long)p.slots * nrt) {
            const int tile = (int)(i % tiles), b = (int)(i / tiles);
            const int len = seq_len(p.lens, p.lens64, b, p.L);
            const T* x = (const T*)p.x + b * p.x_b + c0;
            const T* s0 = p.s0 ? (const T*)p.s0 + (long)b * (K - 1) * p.D + c0 : nullptr;
            const T* ds1 = p.ds1 ? (const T*)p.ds1 + (long)b * (K - 1) * p.D + c0 : nullptr;
            const T* dy = (const T*)p.dy + (long)b * p.L * p.D + c0;
            T* dx = (T*)p.dx + (long)b * p.L * p.D + c0;
            T* ds0 = p.ds0 ? (T*)p.ds0 + (long)b * (K - 1) * p.D + c0 : nullptr;
            const int t0 = tile * CONV_BT;
            const int t1 = t0 + CONV_BT < p.L ? t0 + CONV_BT : p.L;
            float xw[K][SEQ_CH], gw[K][SEQ_CH];
#pragma unroll
            for (int k = 0; k < K; ++k) {
                zero8(gw[k]);
                if (k) input8<T, K, VEC>(p, x, s0, t0 - K + k, len, n, xw[k]);
                else zero8(xw[0]);
            }
            // t runs K - 1 past the tile: those gradients reach back into it.
            // The first tile starts with the outputs whose window holds the
            // carried state, so it emits that state's gradient as it goes.
            for (int t = t0; t < t1 + K - 1; ++t) {
                float g[SEQ_CH];
#pragma unroll
                for (int k = 0; k < K - 1; ++k)
#pragma unroll
                    for (int c = 0; c < SEQ_CH; ++c) {
                        xw[k][c] = xw[k + 1][c];
                        gw[k][c] = gw[k + 1][c];
                    }
                input8<T, K, VEC>(p, x, s0, t, len, n, xw[K - 1]);
                if (t < len) load8<T, VEC>(dy + (long)t * p.D, n, g);
                else zero8(g);
#pragma unroll
                for (int c = 0; c < SEQ_CH; ++c) {
                    float s = bias[c];
#pragma unroll
                    for (int k = 0; k < K; ++k) s = fmaf(w[k][c], xw[k][c], s);
                    if (p.silu) {
                        const float sg = fast_sigmoid(s);
                        g[c] *= sg * (1.f + s * (1.f - sg));
                    }
                    g[c] = t < len ? g[c] : 0.f;
                    gw[K - 1][c] = g[c];
                    if (t < t1) {
                        db[c] += g[c];
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][c] = fmaf(g[c], xw[k][c], dw[k][c]);
                    }
                }
                // ds[t - K + 1 .. t] are in gw: input t - K + 1 is complete
                const int ti = t - (K - 1);
                if (ti < t0 && (tile || !ds0)) continue;
                float o[SEQ_CH];
                zero8(o);
                const int tail = ti - (len - (K - 1));
                if (ds1 && tail >= 0 && tail < K - 1)
                    load8<T, VEC>(ds1 + (long)tail * p.D, n, o);
#pragma unroll
                for (int c = 0; c < SEQ_CH; ++c)
#pragma unroll
                    for (int k = 0; k < K; ++k) o[c] = fmaf(w[K - 1 - k][c], gw[k][c], o[c]);
                if (ti >= 0) {
                    if (ti < t1) store8<T, VEC>(dx + (long)ti * p.D, n, o);
                } else {
                    store8<T, VEC>(ds0 + (long)(ti + K - 1) * p.D, n, o);
                }
            }
        }
    }
    constexpr int W = SEQ_CH * (K + 1);
    float* mine = lds + threadIdx.x * W;
#pragma unroll
    for (int c = 0; c < SEQ_CH; ++c) {
#pragma unroll
        for (int k = 0; k < K; ++k) mine[c * K + k] = dw[k][c];
        mine[SEQ_CH * K + c] = db[c];
    }
    __syncthreads();
    float* ws = p.ws + (long)blockIdx.x * p.D * (K + 1);
    for (int i = threadIdx.x; i < cw * W; i += 256) {
        const int v = i / W, e = i % W;
        const int c = (blockIdx.y * cw + v) * SEQ_CH;
        float s = 0.f;
        for (int r = 0; r < nrt; ++r) s += lds[(r * cw + v) * W + e];
        if (e < SEQ_CH * K) {
            if (c + e / K < p.D) ws[(long)c * K + e] = s;
        } else if (c + e - SEQ_CH * K < p.D) {
            ws[(long)p.D * K + c + e - SEQ_CH * K] = s;
        }
    }
}

// One new token: the state shifts by one input. A thread owns its 8 channels
// of the state alone and reads them all before it writes, so the new state may
// overwrite the old.
template <typename T, int K, bool VEC>
__launch_bounds__(256) __global__ void short_conv_step_kernel(
    const T* __restrict__ x, long x_b, const T* s_in, T* s_out, const float* __restrict__ w,
    const float* __restrict__ bias, T* __restrict__ y, long items, int dv, int D, int silu) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const int c0 = (int)(i % dv) * SEQ_CH;
    const long b = i / dv;
    const int n = D - c0 < SEQ_CH ? D - c0 : SEQ_CH;
    float in[K][SEQ_CH], o[SEQ_CH];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) load8<T, VEC>(s_in + (b * (K - 1) + k) * D + c0, n, in[k]);
    load8<T, VEC>(x + b * x_b + c0, n, in[K - 1]);
#pragma unroll
    for (int c = 0; c < SEQ_CH; ++c) {
        float s = (bias && c < n) ? bias[c0 + c] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) s = fmaf(c < n ? w[(long)(c0 + c) * K + k] : 0.f, in[k][c], s);
        o[c] = silu ? silu_f(s) : s;
    }
    store8<T, VEC>(y + b * D + c0, n, o);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store8<T, VEC>(s_out + (b * (K - 1) + k) * D + c0, n, in[k + 1]);
}

template <typename F>
void by_type(int K, int is_f32, int vec, F f) {
    auto with_k = [&](auto t, auto v) {
        using T = decltype(t);
        constexpr bool V = decltype(v)::value;
        if (K == 2) f.template operator()<T, 2, V>();
        else if (K == 3) f.template operator()<T, 3, V>();
        else f.template operator()<T, 4, V>();
    };
    auto with_t = [&](auto t) {
        if (vec) with_k(t, std::true_type{});
        else with_k(t, std::false_type{});
    };
    if (is_f32) with_t(float{});
    else with_t(__bf16{});
}

struct Fwd {
    const ShortConvParams& p;
    hipStream_t s;
    template <typename T, int K, bool V>
    void operator()() const {
        const int dv = (p.D + SEQ_CH - 1) / SEQ_CH;
        const int tiles = p.L ? (p.L + CONV_TT - 1) / CONV_TT : 1;
        const long items = (long)p.B * tiles * dv;
        hipLaunchKernelGGL((short_conv_fwd_kernel<T, K, V>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s,
            p, items, dv, tiles);
    }
};

struct Bwd {
    const ShortConvParams& p;
    hipStream_t s;
    template <typename T, int K, bool V>
    void operator()() const {
        const int dv = (p.D + SEQ_CH - 1) / SEQ_CH;
        const int cw = pow2_ceil(dv) < 64 ? pow2_ceil(dv) : 64;
        const int tiles = p.L ? (p.L + CONV_BT - 1) / CONV_BT : 1;
        const size_t smem = 256 * SEQ_CH * (K + 1) * sizeof(float);
        hipLaunchKernelGGL((short_conv_bwd_kernel<T, K, V>), dim3(p.slots, (dv + cw - 1) / cw), dim3(256), smem, s,
            p, dv, cw, tiles);
    }
};

struct Step {
    const void* x; long x_b; const void* s_in; void* s_out; const float* w; const float* bias;
    void* y; long B; int D, silu; hipStream_t s;
    template <typename T, int K, bool V>
    void operator()() const {
        const int dv = (D + SEQ_CH - 1) / SEQ_CH;
        const long items = B * dv;
        hipLaunchKernelGGL((short_conv_step_kernel<T, K, V>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s,
            (const T*)x, x_b, (const T*)s_in, (T*)s_out, w, bias, (T*)y, items, dv, D, silu);
    }
};

}  // namespace

extern "C" void short_conv_fwd_launch(const ShortConvParams& p, int K, int is_f32, int vec,
                                      hipStream_t s) {
    by_type(K, is_f32, vec, Fwd{p, s});
}

// Blocks per channel group in the backward: enough to fill 256 CUs a few times
// over, no more than there are row threads with work.
extern "C" int short_conv_bwd_slots(long B, long L, long D) {
    const long dv = (D + SEQ_CH - 1) / SEQ_CH;
    const long cw = pow2_ceil(dv) < 64 ? pow2_ceil(dv) : 64;
    const long groups = (dv + cw - 1) / cw;
    const long items = B * (L ? (L + CONV_BT - 1) / CONV_BT : 1);
    const long want = (items + 256 / cw - 1) / (256 / cw);
    const long cap = (1024 + groups - 1) / groups;
    return (int)(want < cap ? want : cap);
}

extern "C" void short_conv_bwd_launch(const ShortConvParams& p, int K, int is_f32, int vec,
                                      hipStream_t s) {
    by_type(K, is_f32, vec, Bwd{p, s});
}

extern "C" void short_conv_step_launch(const void* x, long x_b, const void* s_in, void* s_out,
                                       const float* w, const float* bias, void* y, long B, int D,
                                       int K, int silu, int is_f32, int vec, hipStream_t s) {
    by_type(K, is_f32, vec, Step{x, x_b, s_in, s_out, w, bias, y, B, D, silu, s});
}

// Column sums of a (nb, E) float workspace in a fixed order: 16 row threads a
// column, joined in LDS.
__launch_bounds__(1024) __global__ void seq_colsum_kernel(const float* __restrict__ ws,
                                                          float* __restrict__ out, long nb, long E) {
    __shared__ float part[16][65];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const long e = (long)blockIdx.x * 64 + c;
    float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
    if (e < E) {
        long b = r;
        for (; b + 48 < nb; b += 64) {
            s0 += ws[b * E + e];
            s1 += ws[(b + 16) * E + e];
            s2 += ws[(b + 32) * E + e];
            s3 += ws[(b + 48) * E + e];
        }
        for (; b < nb; b += 16) s0 += ws[b * E + e];
    }
    part[r][c] = (s0 + s1) + (s2 + s3);
    __syncthreads();
    if (r == 0 && e < E) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += part[i][c];
        out[e] = s;
    }
}

extern "C" void seq_colsum_launch(const float* ws, float* out, long nb, long E, hipStream_t s) {
    hipLaunchKernelGGL(seq_colsum_kernel, dim3((unsigned)((E + 63) / 64)), dim3(1024), 0, s,
            ws, out, nb, E);
}
