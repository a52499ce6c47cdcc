// The norms around a block with its gate and residual scale, one pass (gfx950).
// Per row of D channels, each part optional:
//   p = x silu(gate)
//   p = p inv1 post,              inv1 = rsqrt(mean(p^2) + eps)
//   h = residual + scale p
//   y = h inv2 pre,               inv2 = rsqrt(mean(h^2) + eps)
//
// Bound by memory: every tensor is read once and written once. A row lives in
// the registers of TPR threads (8 channels a chunk, VPT chunks a thread), both
// norms are taken from there in f32, and h feeds the second norm unrounded.
// 8192 x 2560 with an f32 residual: 57 us forward, 92 us backward (4.4 and 4.1
// TB/s); 1835008 x 32 with a gate: 193 us both, at a copy's rate. Both passes of
// wide rows, f32 residual: 4096 x 5120 135 us, 2048 x 8192 160 us, 1024 x 16384
// 332 us (4.6, 3.1, 1.5 TB/s): the backward of four chunks a thread with a
// residual spills 259 to 559 registers.
#include "seq.hpp"

namespace {

// Sum over the TPR threads of a row; for more than a wave through LDS, where
// `slot` alternates so that one barrier a sum is enough.
__device__ __forceinline__ float row_sum(float v, int tpr, float* lds, int& slot) {
    if (tpr <= 64) {
        for (int m = 1; m < tpr; m <<= 1) v += __shfl_xor(v, m);
        return v;
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    const int nw = tpr / 64, wave = threadIdx.x / 64;
    float* buf = lds + slot * 16;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) buf[wave] = v;
    __syncthreads();
    const int w0 = wave / nw * nw;
    float s = 0.f;
    for (int i = 0; i < nw; ++i) s += buf[w0 + i];
    return s;
}

// Eight weights of a row's chunk; ones where there is no such weight.
__device__ __forceinline__ void param8(const float* w, int c, int D, float (&v)[SEQ_CH]) {
#pragma unroll
    for (int j = 0; j < SEQ_CH; ++j) v[j] = 1.f;
    if (w && c < D) load8(w + c, D - c, D, v);
}

// The weights of a thread's columns: kept over its rows where it has one chunk,
// else read where they are used, to leave the registers to the row.
template <int VPT, bool RES>
struct Weights {
    static constexpr bool KEEP = VPT == 1;
    float w[KEEP ? 3 : 1][SEQ_CH];

    __device__ __forceinline__ Weights(const BlockNormParams& p, int c) {
        if (!KEEP) return;
        param8(p.post, c, p.D, w[0]);
        if (RES) param8(p.scale, c, p.D, w[KEEP ? 1 : 0]);
        if (RES) param8(p.pre, c, p.D, w[KEEP ? 2 : 0]);
    }
    // which: 0 post, 1 scale, 2 pre
    template <int WHICH>
    __device__ __forceinline__ void get(const float* from, int c, int D, float (&v)[SEQ_CH]) const {
        if (KEEP) {
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) v[j] = w[KEEP ? WHICH : 0][j];
        } else {
            param8(from, c, D, v);
        }
    }
};

// The same for the backward, whose registers hold the column gradients: in LDS
// where a thread has one chunk. Each thread reads back only what it put there.
template <int VPT, bool RES>
struct WeightsBack {
    static constexpr bool KEEP = VPT == 1;
    f32x4* mine;  // [3][2][blockDim]

    __device__ __forceinline__ WeightsBack(const BlockNormParams& p, int c, float* lds) {
        mine = (f32x4*)lds + threadIdx.x;
        if (!KEEP) return;
        keep(p.post, c, p.D, 0);
        if (RES) keep(p.scale, c, p.D, 1);
        if (RES) keep(p.pre, c, p.D, 2);
    }
    __device__ __forceinline__ void keep(const float* from, int c, int D, int which) {
        float v[SEQ_CH];
        param8(from, c, D, v);
        mine[(which * 2) * blockDim.x] = f32x4{v[0], v[1], v[2], v[3]};
        mine[(which * 2 + 1) * blockDim.x] = f32x4{v[4], v[5], v[6], v[7]};
    }
    template <int WHICH>
    __device__ __forceinline__ void get(const float* from, int c, int D, float (&v)[SEQ_CH]) const {
        if (KEEP) {
            unsigned at = WHICH * 2 * blockDim.x;
            asm volatile("" : "+v"(at));  // read here, not kept over the rows
            const f32x4 a = mine[at], b = mine[at + blockDim.x];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[j] = a[j];
                v[4 + j] = b[j];
            }
        } else {
            if (VPT > 2) asm volatile("" : "+v"(c));  // not kept between the walks
            param8(from, c, D, v);
        }
    }
};

// A thread keeps its columns and takes one row after another; with one chunk a
// thread a row's loads are in flight while the row before is worked on.
// WHOLE: every piece is whole or absent, and there is no code for a partial one.
// MOST: threads of a block; more than 512 leave a thread fewer registers.
template <typename T, typename TR, int VPT, bool RES, bool WHOLE, int MOST>
__launch_bounds__(MOST) __global__ void block_norm_fwd_kernel(BlockNormParams p, int tpr) {
    __shared__ float lds[32];
    int slot = 0;
    const int rpb = blockDim.x / tpr, lane = threadIdx.x % tpr;
    const int width = WHOLE ? SEQ_CH : p.D;
    const float rd = 1.f / (float)p.D;
    const long stride = (long)gridDim.x * rpb, rounds = (p.R + stride - 1) / stride;
    long r = (long)blockIdx.x * rpb + threadIdx.x / tpr;

    const Weights<VPT, RES> wt(p, lane * SEQ_CH);
    constexpr bool AHEAD = VPT == 1;
    Raw8<T> xr[VPT], gr[VPT];
    Raw8<TR> rr[VPT];
    auto read = [&](long row) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            const int n = row < p.R ? p.D - c : 0;
            xr[i].load((const T*)p.x + row * p.x_r + c, n, width);
            if (p.gate) gr[i].load((const T*)p.gate + row * p.g_r + c, n, width);
            if (RES) rr[i].load((const TR*)p.res + row * p.r_r + c, n, width);
        }
    };
    if (AHEAD) read(r);
    for (long k = 0; k < rounds; ++k, r += stride) {
        const bool live = r < p.R;
        float v[VPT][SEQ_CH], hv[VPT][SEQ_CH];
        float ss = 0.f;
        if (!AHEAD) read(r);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) {
                v[i][j] = xr[i].get(j);
                if (p.gate) {
                    const float g = gr[i].get(j);
                    v[i][j] *= g * fast_sigmoid(g);
                }
                if (RES) hv[i][j] = rr[i].get(j);
                ss = fmaf(v[i][j], v[i][j], ss);
            }
        if (AHEAD && k + 1 < rounds) read(r + stride);
        if (p.post) {
            const float inv = 1.f / sqrtf(row_sum(ss, tpr, lds, slot) * rd + p.eps);
            if (live && lane == 0 && p.inv1) p.inv1[r] = inv;
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                float w1[SEQ_CH];
                wt.template get<0>(p.post, (i * tpr + lane) * SEQ_CH, p.D, w1);
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) v[i][j] *= inv * w1[j];
            }
        }
        if (!RES) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int c = (i * tpr + lane) * SEQ_CH;
                if (live && c < p.D) store8<T>((T*)p.y + r * p.D + c, p.D - c, width, v[i]);
            }
            continue;
        }
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            float ws[SEQ_CH];
            wt.template get<1>(p.scale, c, p.D, ws);
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) {
                hv[i][j] = fmaf(ws[j], v[i][j], hv[i][j]);  // zeros past the row's end
                ss = fmaf(hv[i][j], hv[i][j], ss);
            }
            if (live && c < p.D) store8<TR>((TR*)p.h + r * p.D + c, p.D - c, width, hv[i]);
        }
        if (p.pre) {
            const float inv = 1.f / sqrtf(row_sum(ss, tpr, lds, slot) * rd + p.eps);
            if (live && lane == 0 && p.inv2) p.inv2[r] = inv;
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int c = (i * tpr + lane) * SEQ_CH;
                float w2[SEQ_CH];
                wt.template get<2>(p.pre, c, p.D, w2);
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) hv[i][j] *= inv * w2[j];
                if (live && c < p.D) store8<T>((T*)p.y + r * p.D + c, p.D - c, width, hv[i]);
            }
        }
    }
}

// Backward, h recomputed from the inputs (unrounded, and no more bytes than
// reading it back):
//   dh += inv2 (t - h inv2^2 mean(t h)),  t = dy pre
//   dresidual = dh;  q = dh scale post;  n1 = p0 inv1
//   dp0 = inv1 (q - n1 mean(q n1));  dx, dgate by the product and silu'
// Column gradients stay in registers over a thread's rows, are joined in LDS
// over the block's row groups and written once per block.
template <typename T, typename TR, int VPT, bool RES, bool GATE, bool WHOLE, int MOST>
__launch_bounds__(MOST) __global__ void block_norm_bwd_kernel(BlockNormParams p, int tpr) {
    // the weights, then [rpb][VPT * tpr * SEQ_CH] to join the column gradients
    extern __shared__ __attribute__((aligned(16))) float dyn[];
    __shared__ float lds[32];
    int slot = 0;
    const int rpb = blockDim.x / tpr, lane = threadIdx.x % tpr, rg = threadIdx.x / tpr;
    const int width = WHOLE ? SEQ_CH : p.D;
    const float rd = 1.f / (float)p.D;
    const long stride = (long)gridDim.x * rpb, rounds = (p.R + stride - 1) / stride;
    long r = (long)blockIdx.x * rpb + rg;

    const WeightsBack<VPT, RES> wt(p, lane * SEQ_CH, dyn);
    constexpr bool AHEAD = VPT == 1;
    float dpost[VPT][SEQ_CH] = {}, dscale[VPT][SEQ_CH] = {}, dpre[VPT][SEQ_CH] = {};
    Raw8<T> xr[VPT], gr[VPT], yr[VPT];
    Raw8<TR> rr[VPT], hr[VPT];
    float i1 = 1.f, i2 = 1.f;
    // absent gradients count as zeros: n is 0 for them
    auto read = [&](long row) {
        const bool there = row < p.R;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            const int n = there ? p.D - c : 0;
            xr[i].load((const T*)p.x + row * p.x_r + c, n, width);
            if (GATE) gr[i].load((const T*)p.gate + row * p.g_r + c, n, width);
            if (!RES || p.pre) yr[i].load((const T*)p.dy + row * p.D + c, p.dy ? n : 0, width);
            if (RES && p.pre) rr[i].load((const TR*)p.res + row * p.r_r + c, n, width);
            if (RES) hr[i].load((const TR*)p.dh + row * p.D + c, p.dh ? n : 0, width);
        }
        if (p.post && there) i1 = p.inv1[row];
        if (RES && p.pre && there) i2 = p.inv2[row];
    };
    if (AHEAD) read(r);
    for (long k = 0; k < rounds; ++k, r += stride) {
        const bool live = r < p.R;
        if (!AHEAD) read(r);
        const float inv1 = i1, inv2 = i2;
        Raw8<T> xk[VPT], gk[VPT], yk[VPT];
        Raw8<TR> rk[VPT], hk[VPT];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            xk[i] = xr[i];
            gk[i] = gr[i];
            yk[i] = yr[i];
            rk[i] = rr[i];
            hk[i] = hr[i];
        }
        if (AHEAD && k + 1 < rounds) read(r + stride);
        // With four chunks the row waits as it came, and what follows from it is
        // formed anew by each of the three walks over it: kept it would spill.
        auto anew = [&](auto& raw) {
            if (VPT > 2) raw.fresh();
        };
        auto apart = [&] {  // one chunk's weights at a time
            if (VPT > 2) __builtin_amdgcn_sched_barrier(0);
        };
        // the normed row without its weight; the one after the residual, y / pre
        auto normed = [&](int i, float (&v)[SEQ_CH]) {
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) {
                const float g = GATE ? gk[i].get(j) : 0.f;
                v[j] = xk[i].get(j) * (GATE ? g * fast_sigmoid(g) : 1.f) * inv1;
            }
        };
        auto stream = [&](int i, const float (&v)[SEQ_CH], const float (&w1)[SEQ_CH], const float (&ws)[SEQ_CH],
                          float (&h)[SEQ_CH]) {
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) h[j] = fmaf(ws[j] * w1[j], v[j], rk[i].get(j)) * inv2;
        };
        float m = 0.f;
        if (RES && p.pre) {
            float sum2 = 0.f;
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int c = (i * tpr + lane) * SEQ_CH;
                float w1[SEQ_CH], ws[SEQ_CH], w2[SEQ_CH], v[SEQ_CH], h[SEQ_CH];
                wt.template get<0>(p.post, c, p.D, w1);
                wt.template get<1>(p.scale, c, p.D, ws);
                wt.template get<2>(p.pre, c, p.D, w2);
                normed(i, v);
                stream(i, v, w1, ws, h);
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) {
                    const float t = yk[i].get(j);
                    dpre[i][j] = fmaf(t, h[j], dpre[i][j]);
                    sum2 = fmaf(t * w2[j], h[j], sum2);
                }
                apart();
            }
            m = row_sum(sum2, tpr, lds, slot) * rd * inv2;
        }
        float sum1 = 0.f, d[VPT][SEQ_CH];  // d: the gradient on its way down
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            float w1[SEQ_CH], ws[SEQ_CH], v[SEQ_CH];
            anew(xk[i]);
            if (GATE) anew(gk[i]);
            wt.template get<0>(p.post, c, p.D, w1);
            if (RES) wt.template get<1>(p.scale, c, p.D, ws);
            normed(i, v);
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) d[i][j] = RES ? hk[i].get(j) : yk[i].get(j);
            if (RES && p.pre) {
                float w2[SEQ_CH], h[SEQ_CH];
                anew(rk[i]);
                anew(yk[i]);
                wt.template get<2>(p.pre, c, p.D, w2);
                stream(i, v, w1, ws, h);
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) d[i][j] = fmaf(-m, h[j], fmaf(inv2, yk[i].get(j) * w2[j], d[i][j]));
            }
            if (RES && live && c < p.D) store8<TR>((TR*)p.dres + r * p.D + c, p.D - c, width, d[i]);
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) {
                if (RES) {
                    dscale[i][j] = fmaf(d[i][j], v[j] * w1[j], dscale[i][j]);
                    d[i][j] *= ws[j];
                }
                dpost[i][j] = fmaf(d[i][j], v[j], dpost[i][j]);
                d[i][j] *= w1[j];
                sum1 = fmaf(d[i][j], v[j], sum1);
            }
            apart();
        }
        const float m1 = p.post ? row_sum(sum1, tpr, lds, slot) * rd : 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            float v[SEQ_CH], o[SEQ_CH], og[SEQ_CH];
            anew(xk[i]);
            if (GATE) anew(gk[i]);
            normed(i, v);
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) {
                const float dp = inv1 * fmaf(-m1, v[j], d[i][j]);
                o[j] = dp;
                if (GATE) {
                    const float g = gk[i].get(j), sg = fast_sigmoid(g), si = g * sg;
                    o[j] = dp * si;
                    og[j] = dp * xk[i].get(j) * (sg + si * (1.f - sg));
                }
            }
            if (live && c < p.D) {
                store8<T>((T*)p.dx + r * p.D + c, p.D - c, width, o);
                if (GATE) store8<T>((T*)p.dgate + r * p.D + c, p.D - c, width, og);
            }
            apart();
        }
    }
    // column gradients of the weights there are, in the order post | scale | pre
    const int W = VPT * tpr * SEQ_CH;
    float* out = p.ws + (long)blockIdx.x * ((p.post != nullptr) + (p.scale != nullptr) + (p.pre != nullptr)) * p.D;
#pragma unroll
    for (int a = 0; a < 3; ++a) {
        if (!(a == 0 ? p.post : a == 1 ? p.scale : p.pre)) continue;
        auto& acc = a == 0 ? dpost : a == 1 ? dscale : dpre;
        if (rpb > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j)
                    dyn[rg * W + (i * tpr + lane) * SEQ_CH + j] = acc[i][j];
            __syncthreads();
            for (int c = threadIdx.x; c < p.D; c += blockDim.x) {
                float s = 0.f;
                for (int g = 0; g < rpb; ++g) s += dyn[g * W + c];
                out[c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) {
                    const int c = (i * tpr + lane) * SEQ_CH + j;
                    if (c < p.D) out[c] = acc[i][j];
                }
        }
        out += p.D;
    }
}

// Threads a row, chunks a thread: a part of a wave while that holds the row,
// then whole waves with one chunk a thread (to D = 6144), two, four. One chunk
// leaves registers for the next row's loads: 4096 x 5120 takes 135 us with one on
// 640 threads, 231 us with two on 320. Widths just past a power of two of chunks,
// or past whole waves of them, leave threads idle: 264 channels use 33 lanes of
// 64, 520 use 65 threads of 128.
inline void row_shape(long D, int* tpr, int* vpt) {
    const long chunks = (D + SEQ_CH - 1) / SEQ_CH;
    *vpt = chunks <= 768 ? 1 : chunks <= 1024 ? 2 : 4;
    *tpr = chunks <= 64 ? pow2_ceil(chunks) : (int)((chunks + 64 * *vpt - 1) / (64 * *vpt)) * 64;
}

// Whole rows in a block of about 256 threads.
inline int block_threads(int tpr) { return tpr >= 256 ? tpr : 256 / tpr * tpr; }

// Blocks that take the rows in turn: as many as 256 CUs hold at once, given the
// waves that a CU is taken to have registers for. More would leave a second,
// emptier round, fewer an idle place: the counts below are those of the common
// kernels of each kind, not of every one.
inline long row_blocks(long R, int tpr, int waves) {
    const int block = block_threads(tpr), per_cu = waves / (block / 64);
    const long want = (R + block / tpr - 1) / (block / tpr), cap = 256L * (per_cu ? per_cu : 1);
    return want < cap ? want : cap;
}

struct NormFwd {
    const BlockNormParams& p;
    hipStream_t s;
    template <typename T, typename TR, int VPT, bool RES, bool WHOLE, int MOST>
    void operator()(int tpr) const {
        // 20 waves: what one chunk with a residual allows, but for f32 with an f32
        // residual (16); without a residual 32 would fit, several chunks allow fewer
        hipLaunchKernelGGL((block_norm_fwd_kernel<T, TR, VPT, RES, WHOLE, MOST>),
                           dim3((unsigned)row_blocks(p.R, tpr, 20)), dim3(block_threads(tpr)), 0, s, p, tpr);
    }
};

struct NormBwd {
    const BlockNormParams& p;
    hipStream_t s;
    template <typename T, typename TR, int VPT, bool RES, bool WHOLE, int MOST>
    void operator()(int tpr) const {
        const int block = block_threads(tpr);
        const size_t smem = (size_t)block * SEQ_CH * sizeof(float) * (VPT > 1 ? VPT : RES ? 3 : 1);
        if (p.gate)
            hipLaunchKernelGGL((block_norm_bwd_kernel<T, TR, VPT, RES, true, WHOLE, MOST>), dim3(p.slots), dim3(block),
                               smem, s, p, tpr);
        if (!p.gate)
            hipLaunchKernelGGL((block_norm_bwd_kernel<T, TR, VPT, RES, false, WHOLE, MOST>), dim3(p.slots), dim3(block),
                               smem, s, p, tpr);
    }
};

template <typename T, typename TR, bool RES, typename F>
void by_shape(const BlockNormParams& p, F f) {
    int tpr, vpt;
    row_shape(p.D, &tpr, &vpt);
    if (tpr > 512) f.template operator()<T, TR, 1, RES, false, 768>(tpr);
    else if (vpt == 1 && p.D % SEQ_CH == 0) f.template operator()<T, TR, 1, RES, true, 512>(tpr);
    else if (vpt == 1) f.template operator()<T, TR, 1, RES, false, 512>(tpr);
    else if (vpt == 2) f.template operator()<T, TR, 2, RES, false, 512>(tpr);
    else f.template operator()<T, TR, 4, RES, false, 512>(tpr);
}

template <typename F>
void by_type(const BlockNormParams& p, int is_f32, int res_f32, F f) {
    if (!p.res) {
        if (is_f32) by_shape<float, float, false>(p, f);
        else by_shape<__bf16, __bf16, false>(p, f);
    } else if (is_f32) {
        if (res_f32) by_shape<float, float, true>(p, f);
        else by_shape<float, __bf16, true>(p, f);
    } else {
        if (res_f32) by_shape<__bf16, float, true>(p, f);
        else by_shape<__bf16, __bf16, true>(p, f);
    }
}

}  // namespace

// Blocks of the backward, each with its own row of column gradients.
extern "C" int block_norm_slots(long R, long D, int res, int gate) {
    int tpr, vpt;
    row_shape(D, &tpr, &vpt);
    // a gate beside a residual: 8, though bf16 throughout has registers for 12
    return (int)row_blocks(R, tpr, vpt > 1 ? 8 : !res ? 16 : gate ? 8 : 12);
}

extern "C" void block_norm_fwd_launch(const BlockNormParams& p, int is_f32, int res_f32, hipStream_t s) {
    by_type(p, is_f32, res_f32, NormFwd{p, s});
}

extern "C" void block_norm_bwd_launch(const BlockNormParams& p, int is_f32, int res_f32, hipStream_t s) {
    by_type(p, is_f32, res_f32, NormBwd{p, s});
}
