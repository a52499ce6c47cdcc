// Short causal convolution over time, one filter of K taps per channel
// (gfx950):  s[t] = bias + sum_k w[k] x[t - K + 1 + k],  y[t] = silu(s[t]).
//
// Bound by memory: 2K flops against one element read and one written. A thread
// owns 16 bytes of channels and walks a tile of the time axis with the last
// K - 1 inputs in registers; a block of steps is loaded while the block before
// is worked on. Tiles are as long as keeps the card full: each reads K - 1
// inputs of its neighbour again. 16384 x 4096 bf16: 71 us, 3.8 TB/s; forward and
// backward of 70688 x 7 x 32 f32: 23 + 43 us, 4.8 TB/s of what both move.
#include "seq.hpp"

namespace {

template <typename T>
constexpr int conv_e() { return 16 / sizeof(T); }  // channels a thread, forward
#define CONV_BE 4  // backward: with 8 of bf16 its windows and sums would take all registers and some more

__device__ __forceinline__ float silu_f(float s) { return s * fast_sigmoid(s); }

// A thread's E channels at one step; n of them are there, D in a row.
template <typename T, int E>
__device__ __forceinline__ Pack<T, E> row_at(const T* p, int n, int D) {
    Pack<T, E> r;
    r.load(p, n, D % E);
    return r;
}
template <typename T, int E>
__device__ __forceinline__ void put_row(T* p, int n, int D, const float (&v)[E]) {
    Pack<T, E> r;
    r.set(v);
    r.store(p, n, D % E);
}
template <typename T, int E>
__device__ __forceinline__ Pack<T, E> no_row() {
    Pack<T, E> r;
    r.clear();
    return r;
}

// Input t of a sequence: the carried state before the first, zero before that
// and past the end.
template <typename T, int E, int K>
__device__ __forceinline__ Pack<T, E> input_row(const ShortConvParams& p, const T* x, const T* s0, int t, int len, int n,
                                                int width) {
    if (t >= 0 && t < len) return row_at<T, E>(x + t * p.x_t, n, width);
    if (t < 0 && t >= -(K - 1) && s0) return row_at<T, E>(s0 + (long)(t + K - 1) * p.D, n, width);
    return no_row<T, E>();
}

template <int K, int E>
__device__ __forceinline__ void taps(const float* w, const float* bias, int c0, int n, float (&wv)[K][E], float (&bv)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j) {
        const int c = j < n ? c0 + j : c0;
        bv[j] = bias ? bias[c] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) wv[k][j] = w[(long)c * K + k];
    }
}

// WHOLE: every thread has all of its channels, and no code for fewer.
template <typename T, int K, bool WHOLE>
__launch_bounds__(256) __global__ void short_conv_fwd_kernel(ShortConvParams p, long items, int dv, int tiles) {
    constexpr int E = conv_e<T>(), NB = 4;
    const long i = block_id() * 256 + threadIdx.x;
    if (i >= items) return;
    const int c0 = (int)(i % dv) * E;
    const long r = i / dv;
    const int tile = (int)(r % tiles), b = (int)(r / tiles);
    const int n = WHOLE || p.D - c0 >= E ? E : p.D - c0, width = WHOLE ? E : p.D;
    const int len = seq_len(p.lens, p.lens64, b, p.L);
    const T* x = (const T*)p.x + b * p.x_b + c0;
    const T* s0 = p.s0 ? (const T*)p.s0 + (long)b * (K - 1) * p.D + c0 : nullptr;
    const int t0 = tile * p.tile, t1 = t0 + p.tile < p.L ? t0 + p.tile : p.L;
    T* y = (T*)p.y + ((long)b * p.L + t0) * p.D + c0;

    Pack<T, E> raw[NB];
    float w[K][E], bias[E], win[K][E];
    auto read = [&](int t) {
        const T* s = x + t * p.x_t;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            raw[j] = t + j < len ? row_at<T, E>(s, n, width) : no_row<T, E>();
            s += p.x_t;
        }
    };
    Pack<T, E> edge[K - 1];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) edge[k] = input_row<T, E, K>(p, x, s0, t0 - (K - 1) + k, len, n, width);
    read(t0);
    taps<K, E>(p.w, p.bias, c0, n, w, bias);
#pragma unroll
    for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int c = 0; c < E; ++c) win[k + 1][c] = edge[k].get(c);
    for (int t = t0; t < t1; t += NB) {
        Pack<T, E> cur[NB];
#pragma unroll
        for (int j = 0; j < NB; ++j) cur[j] = raw[j];
        if (t + NB < t1) read(t + NB);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            float o[E];
#pragma unroll
            for (int c = 0; c < E; ++c) {
#pragma unroll
                for (int k = 0; k < K - 1; ++k) win[k][c] = win[k + 1][c];
                win[K - 1][c] = cur[j].get(c);
                float s = bias[c];
#pragma unroll
                for (int k = 0; k < K; ++k) s = fmaf(w[k][c], win[k][c], s);
                o[c] = t + j < len ? (p.silu ? silu_f(s) : s) : 0.f;
            }
            if (t + j < t1) put_row<T, E>(y, n, width, o);
            y += p.D;
        }
    }
    if (p.s1 && tile == 0) {
        T* s1 = (T*)p.s1 + (long)b * (K - 1) * p.D + c0;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            const Pack<T, E> v = input_row<T, E, K>(p, x, s0, len - (K - 1) + j, len, n, width);
            float o[E];
#pragma unroll
            for (int c = 0; c < E; ++c) o[c] = v.get(c);
            put_row<T, E>(s1 + (long)j * p.D, n, width, o);
        }
    }
}

// Backward: ds[t] = dy[t] silu'(s[t]) with s recomputed, dx[t] = sum_k w[k]
// ds[t + K - 1 - k], dw[k] = sum ds[t] x[t - K + 1 + k]. A thread streams one
// tile in time order, K - 1 steps past its end, holding the last K inputs and
// the last K values of ds; filter gradients stay in registers over all of its
// tiles, are joined per block and written once, then summed in a fixed order
// (no atomics).
template <typename T, int K, bool WHOLE>
__launch_bounds__(256) __global__ void short_conv_bwd_kernel(ShortConvParams p, int dv, int cw, int tiles) {
    constexpr int E = CONV_BE, NB = 4;
    constexpr int W = E * (K + 1);
    extern __shared__ float lds[];  // [256][W]
    const int rt = threadIdx.x / cw, nrt = 256 / cw;
    // blocks of one channel group after those of another
    const int group = blockIdx.x / p.slots, slot = blockIdx.x - group * p.slots;
    const int cv = group * cw + threadIdx.x % cw;
    const int c0 = cv * E;
    const int n = WHOLE || p.D - c0 >= E ? E : p.D - c0, width = WHOLE ? E : p.D;
    float dw[K][E] = {}, db[E] = {};
    if (cv < dv) {
        float w[K][E], bias[E];
        taps<K, E>(p.w, p.bias, c0, n, w, bias);
        const long items = (long)p.B * tiles;
        for (long i = (long)slot * nrt + rt; i < items; i += (long)p.slots * nrt) {
            const int tile = (int)(i % tiles), b = (int)(i / tiles);
            const int len = seq_len(p.lens, p.lens64, b, p.L);
            const int t0 = tile * p.tile, t1 = t0 + p.tile < p.L ? t0 + p.tile : p.L;
            const T* x = (const T*)p.x + b * p.x_b + c0;
            const T* s0 = p.s0 ? (const T*)p.s0 + (long)b * (K - 1) * p.D + c0 : nullptr;
            const T* ds1 = p.ds1 ? (const T*)p.ds1 + (long)b * (K - 1) * p.D + c0 : nullptr;
            const T* dy = (const T*)p.dy + (long)b * p.L * p.D + c0;
            T* dx = (T*)p.dx + (long)b * p.L * p.D + c0;
            T* ds0 = p.ds0 ? (T*)p.ds0 + (long)b * (K - 1) * p.D + c0 : nullptr;
            Pack<T, E> xr[NB], yr[NB], edge[K - 1];
            auto read = [&](int t) {
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    const bool on = t + j < len;
                    xr[j] = on ? row_at<T, E>(x + (t + j) * p.x_t, n, width) : no_row<T, E>();
                    yr[j] = on ? row_at<T, E>(dy + (long)(t + j) * p.D, n, width) : no_row<T, E>();
                }
            };
#pragma unroll
            for (int k = 0; k < K - 1; ++k) edge[k] = input_row<T, E, K>(p, x, s0, t0 - (K - 1) + k, len, n, width);
            read(t0);
            float xw[K][E], gw[K][E];
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int c = 0; c < E; ++c) {
                    gw[k][c] = 0.f;
                    xw[k][c] = k ? edge[k ? k - 1 : 0].get(c) : 0.f;
                }
            // The first tile starts with the outputs whose window holds the
            // carried state, so it emits that state's gradient as it goes.
            for (int tb = t0; tb < t1 + K - 1; tb += NB) {
                Pack<T, E> xc[NB], yc[NB];
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    xc[j] = xr[j];
                    yc[j] = yr[j];
                }
                if (tb + NB < t1 + K - 1) read(tb + NB);
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    const int t = tb + j;
                    if (t >= t1 + K - 1) break;
#pragma unroll
                    for (int c = 0; c < E; ++c) {
#pragma unroll
                        for (int k = 0; k < K - 1; ++k) {
                            xw[k][c] = xw[k + 1][c];
                            gw[k][c] = gw[k + 1][c];
                        }
                        xw[K - 1][c] = xc[j].get(c);
                        float s = bias[c], g = yc[j].get(c);
#pragma unroll
                        for (int k = 0; k < K; ++k) s = fmaf(w[k][c], xw[k][c], s);
                        if (p.silu) {
                            const float sg = fast_sigmoid(s);
                            g *= sg * (1.f + s * (1.f - sg));
                        }
                        g = t < len ? g : 0.f;
                        gw[K - 1][c] = g;
                        g = t < t1 ? g : 0.f;  // past the tile it is another's
                        db[c] += g;
#pragma unroll
                        for (int k = 0; k < K; ++k) dw[k][c] = fmaf(g, xw[k][c], dw[k][c]);
                    }
                    // ds[t - K + 1 .. t] are in gw: input t - K + 1 is complete
                    const int ti = t - (K - 1);
                    if (ti >= t1 || (ti < t0 && (tile || !ds0))) continue;
                    float o[E];
#pragma unroll
                    for (int c = 0; c < E; ++c) o[c] = 0.f;
                    const int tail = ti - (len - (K - 1));
                    if (ds1 && tail >= 0 && tail < K - 1) {
                        const Pack<T, E> v = row_at<T, E>(ds1 + (long)tail * p.D, n, width);
#pragma unroll
                        for (int c = 0; c < E; ++c) o[c] = v.get(c);
                    }
#pragma unroll
                    for (int c = 0; c < E; ++c)
#pragma unroll
                        for (int k = 0; k < K; ++k) o[c] = fmaf(w[K - 1 - k][c], gw[k][c], o[c]);
                    if (ti >= 0) put_row<T, E>(dx + (long)ti * p.D, n, width, o);
                    else put_row<T, E>(ds0 + (long)(ti + K - 1) * p.D, n, width, o);
                }
            }
        }
    }
    float* mine = lds + threadIdx.x * W;
#pragma unroll
    for (int c = 0; c < E; ++c) {
#pragma unroll
        for (int k = 0; k < K; ++k) mine[c * K + k] = dw[k][c];
        mine[E * K + c] = db[c];
    }
    __syncthreads();
    float* ws = p.ws + (long)slot * p.D * (K + 1);
    for (int i = threadIdx.x; i < cw * W; i += 256) {
        const int v = i / W, e = i % W;
        const int c = (group * cw + v) * E;
        float s = 0.f;
        for (int r = 0; r < nrt; ++r) s += lds[(r * cw + v) * W + e];
        if (e < E * K) {
            if (c + e / K < p.D) ws[(long)c * K + e] = s;
        } else if (c + e - E * K < p.D) {
            ws[(long)p.D * K + c + e - E * K] = s;
        }
    }
}

// One new token: the state shifts by one input. A thread owns its 8 channels
// of the state alone and reads them all before it writes, so the new state may
// overwrite the old. 1 x 1024: 5.5 us, a launch and one dependent load.
template <typename T, int K>
__launch_bounds__(256) __global__ void short_conv_step_kernel(
    const T* __restrict__ x, long x_b, const T* s_in, T* s_out, const float* __restrict__ w,
    const float* __restrict__ bias, T* __restrict__ y, long items, int dv, int D, int silu) {
    const long i = block_id() * 256 + threadIdx.x;
    if (i >= items) return;
    const int c0 = (int)(i % dv) * SEQ_CH;
    const long b = i / dv;
    const int n = D - c0 < SEQ_CH ? D - c0 : SEQ_CH;
    float in[K][SEQ_CH], o[SEQ_CH];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) load8<T>(s_in + (b * (K - 1) + k) * D + c0, n, D, in[k]);
    load8<T>(x + b * x_b + c0, n, D, in[K - 1]);
#pragma unroll
    for (int c = 0; c < SEQ_CH; ++c) {
        float s = (bias && c < n) ? bias[c0 + c] : 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) s = fmaf(c < n ? w[(long)(c0 + c) * K + k] : 0.f, in[k][c], s);
        o[c] = silu ? silu_f(s) : s;
    }
    store8<T>(y + b * D + c0, n, D, o);
#pragma unroll
    for (int k = 0; k < K - 1; ++k) store8<T>(s_out + (b * (K - 1) + k) * D + c0, n, D, in[k + 1]);
}

// Threads of a block side by side in the channels.
inline int conv_cw(long dv) { return pow2_ceil(dv) < 64 ? pow2_ceil(dv) : 64; }

// Steps of a tile, a multiple of 8: whole sequences if that leaves enough
// threads, else as few as `threads` of them need.
inline int conv_tile(long B, long L, long dv, long threads) {
    long tiles = threads / (B * dv > 0 ? B * dv : 1);
    tiles = tiles < 1 ? 1 : tiles;
    const long t = ((L + tiles - 1) / tiles + 7) / 8 * 8;
    return (int)(t < 16 ? (L <= 8 ? 8 : 16) : t);
}

template <typename F>
void by_type(int K, int is_f32, F f) {
    auto with = [&](auto t) {
        using T = decltype(t);
        if (K == 2) f.template operator()<T, 2>();
        else if (K == 3) f.template operator()<T, 3>();
        else f.template operator()<T, 4>();
    };
    if (is_f32) with(float{});
    else with(__bf16{});
}

struct Fwd {
    const ShortConvParams& p;
    hipStream_t s;
    template <typename T, int K>
    void operator()() const {
        const int dv = (p.D + conv_e<T>() - 1) / conv_e<T>();
        const int tiles = p.L ? (p.L + p.tile - 1) / p.tile : 1;
        const long items = (long)p.B * tiles * dv;
        const dim3 grid = grid_of((items + 255) / 256);
        if (p.D % conv_e<T>() == 0)
            hipLaunchKernelGGL((short_conv_fwd_kernel<T, K, true>), grid, dim3(256), 0, s, p, items, dv, tiles);
        if (p.D % conv_e<T>() != 0)
            hipLaunchKernelGGL((short_conv_fwd_kernel<T, K, false>), grid, dim3(256), 0, s, p, items, dv, tiles);
    }
};

struct Bwd {
    const ShortConvParams& p;
    hipStream_t s;
    template <typename T, int K>
    void operator()() const {
        const int dv = (p.D + CONV_BE - 1) / CONV_BE;
        const int cw = conv_cw(dv);
        const int tiles = p.L ? (p.L + p.tile - 1) / p.tile : 1;
        const size_t smem = 256 * CONV_BE * (K + 1) * sizeof(float);
        const dim3 grid((unsigned)p.slots * ((dv + cw - 1) / cw));
        if (p.D % CONV_BE == 0)
            hipLaunchKernelGGL((short_conv_bwd_kernel<T, K, true>), grid, dim3(256), smem, s, p, dv, cw, tiles);
        if (p.D % CONV_BE != 0)
            hipLaunchKernelGGL((short_conv_bwd_kernel<T, K, false>), grid, dim3(256), smem, s, p, dv, cw, tiles);
    }
};

struct Step {
    const void* x; long x_b; const void* s_in; void* s_out; const float* w; const float* bias;
    void* y; long B; int D, silu; hipStream_t s;
    template <typename T, int K>
    void operator()() const {
        const int dv = (D + SEQ_CH - 1) / SEQ_CH;
        const long items = B * dv;
        hipLaunchKernelGGL((short_conv_step_kernel<T, K>), grid_of((items + 255) / 256), dim3(256), 0, s,
            (const T*)x, x_b, (const T*)s_in, (T*)s_out, w, bias, (T*)y, items, dv, D, silu);
    }
};

}  // namespace

// The tile of p and, for the backward, the blocks that share a channel group:
// each writes a row of filter gradients.
extern "C" void short_conv_plan(ShortConvParams* p, int is_f32, int back) {
    const long e = back ? CONV_BE : is_f32 ? 4 : 8, dv = (p->D + e - 1) / e;
    // Tiles for 16 waves a CU forward, 8 backward. The registers allow 8 to 20 by
    // type and taps: 12 for whole rows of bf16 and 4 taps, so that of the 1024
    // blocks of 16384 x 4096 768 run at once; 8 to 16 backward.
    p->tile = conv_tile(p->B, p->L, dv, back ? 256L * 8 * 64 : 256L * 16 * 64);
    const long cw = conv_cw(dv), groups = (dv + cw - 1) / cw, rows = 256 / cw;
    const long items = p->B * (p->L ? ((long)p->L + p->tile - 1) / p->tile : 1);
    const long want = (items + rows - 1) / rows, cap = (512 + groups - 1) / groups;
    p->slots = (int)(want < cap ? want : cap);
}

extern "C" void short_conv_fwd_launch(const ShortConvParams& p, int K, int is_f32, hipStream_t s) {
    by_type(K, is_f32, Fwd{p, s});
}

extern "C" void short_conv_bwd_launch(const ShortConvParams& p, int K, int is_f32, hipStream_t s) {
    by_type(K, is_f32, Bwd{p, s});
}

extern "C" void short_conv_step_launch(const void* x, long x_b, const void* s_in, void* s_out,
                                       const float* w, const float* bias, void* y, long B, int D,
                                       int K, int silu, int is_f32, hipStream_t s) {
    by_type(K, is_f32, Step{x, x_b, s_in, s_out, w, bias, y, B, D, silu, s});
}

// Column sums of a (nb, E) float workspace in a fixed order: 16 row threads a
// column, joined in LDS.
__launch_bounds__(1024) __global__ void seq_colsum_kernel(const float* __restrict__ ws,
                                                          float* __restrict__ out, long nb, long E) {
    __shared__ float part[16][65];
    const int c = threadIdx.x & 63, r = threadIdx.x >> 6;
    const long e = block_id() * 64 + c;
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
    hipLaunchKernelGGL(seq_colsum_kernel, grid_of((E + 63) / 64), dim3(1024), 0, s,
            ws, out, nb, E);
}
