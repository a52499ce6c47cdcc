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

__device__ __forceinline__ void param8(const float* w, int c, int n, float (&v)[SEQ_CH]) {
#pragma unroll
    for (int j = 0; j < SEQ_CH; ++j) v[j] = (w && j < n) ? w[c + j] : 1.f;
}

template <typename T, typename TR, int VPT, bool VEC>
__launch_bounds__(512) __global__ void block_norm_fwd_kernel(BlockNormParams p, int tpr) {
    __shared__ float lds[32];
    int slot = 0;
    const int rpb = blockDim.x / tpr, lane = threadIdx.x % tpr;
    const float rd = 1.f / (float)p.D;
    const long rounds = (p.R + (long)gridDim.x * rpb - 1) / ((long)gridDim.x * rpb);
    for (long k = 0; k < rounds; ++k) {
        const long r = (k * gridDim.x + blockIdx.x) * rpb + threadIdx.x / tpr;
        const bool live = r < p.R;
        float v[VPT][SEQ_CH], hv[VPT][SEQ_CH];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            const int n = live ? p.D - c : 0;
            zero8(v[i]);
            zero8(hv[i]);
            if (n <= 0) continue;
            load8<T, VEC>((const T*)p.x + r * p.x_r + c, n, v[i]);
            if (p.res) load8<TR, VEC>((const TR*)p.res + r * p.r_r + c, n, hv[i]);
            if (p.gate) {
                float g[SEQ_CH];
                load8<T, VEC>((const T*)p.gate + r * p.g_r + c, n, g);
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) v[i][j] *= g[j] * fast_sigmoid(g[j]);
            }
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) ss = fmaf(v[i][j], v[i][j], ss);
        }
        if (p.post) {
            const float inv = 1.f / sqrtf(row_sum(ss, tpr, lds, slot) * rd + p.eps);
            if (live && lane == 0 && p.inv1) p.inv1[r] = inv;
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int c = (i * tpr + lane) * SEQ_CH;
                if (c >= p.D) continue;
                float w[SEQ_CH];
                param8(p.post, c, p.D - c, w);
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) v[i][j] *= inv * w[j];
            }
        }
        if (!p.res) {
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int c = (i * tpr + lane) * SEQ_CH;
                if (live && c < p.D) store8<T, VEC>((T*)p.y + r * p.D + c, p.D - c, v[i]);
            }
            continue;
        }
        ss = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            if (!live || c >= p.D) continue;
            float w[SEQ_CH];
            param8(p.scale, c, p.D - c, w);
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) {
                hv[i][j] = fmaf(w[j], v[i][j], hv[i][j]);
                if (VEC || c + j < p.D) ss = fmaf(hv[i][j], hv[i][j], ss);
            }
            store8<TR, VEC>((TR*)p.h + r * p.D + c, p.D - c, hv[i]);
        }
        if (p.pre) {
            const float inv = 1.f / sqrtf(row_sum(ss, tpr, lds, slot) * rd + p.eps);
            if (live && lane == 0 && p.inv2) p.inv2[r] = inv;
#pragma unroll
            for (int i = 0; i < VPT; ++i) {
                const int c = (i * tpr + lane) * SEQ_CH;
                if (!live || c >= p.D) continue;
                float w[SEQ_CH];
                param8(p.pre, c, p.D - c, w);
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) hv[i][j] *= inv * w[j];
                store8<T, VEC>((T*)p.y + r * p.D + c, p.D - c, hv[i]);
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
template <typename T, typename TR, int VPT, bool VEC>
__launch_bounds__(512) __global__ void block_norm_bwd_kernel(BlockNormParams p, int tpr) {
    extern __shared__ float dyn[];  // [rpb][VPT * tpr * SEQ_CH] when rpb > 1
    __shared__ float lds[32];
    int slot = 0;
    const int rpb = blockDim.x / tpr, lane = threadIdx.x % tpr, rg = threadIdx.x / tpr;
    const float rd = 1.f / (float)p.D;
    float dpost[VPT][SEQ_CH] = {}, dscale[VPT][SEQ_CH] = {}, dpre[VPT][SEQ_CH] = {};
    const long rounds = (p.R + (long)gridDim.x * rpb - 1) / ((long)gridDim.x * rpb);
    for (long k = 0; k < rounds; ++k) {
        const long r = (k * gridDim.x + blockIdx.x) * rpb + rg;
        const bool live = r < p.R;
        float v[VPT][SEQ_CH], hv[VPT][SEQ_CH], d[VPT][SEQ_CH], gt[VPT][SEQ_CH], xv[VPT][SEQ_CH];
        const float inv1 = (p.post && live) ? p.inv1[r] : 1.f;
        const float inv2 = (p.pre && live) ? p.inv2[r] : 1.f;
        float sum2 = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            const int n = live ? p.D - c : 0;
            zero8(xv[i]);
            zero8(gt[i]);
            zero8(v[i]);
            zero8(hv[i]);
            zero8(d[i]);
            if (n <= 0) continue;
            load8<T, VEC>((const T*)p.x + r * p.x_r + c, n, xv[i]);
            if (p.gate) load8<T, VEC>((const T*)p.gate + r * p.g_r + c, n, gt[i]);
            if (p.res) {
                if (p.pre) load8<TR, VEC>((const TR*)p.res + r * p.r_r + c, n, hv[i]);
                if (p.dh) load8<TR, VEC>((const TR*)p.dh + r * p.D + c, n, d[i]);
            } else if (p.dy) {
                load8<T, VEC>((const T*)p.dy + r * p.D + c, n, d[i]);
            }
            // v: the normed row without its weight, n1
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) {
                const float sg = p.gate ? gt[i][j] * fast_sigmoid(gt[i][j]) : 1.f;
                v[i][j] = xv[i][j] * sg * inv1;
            }
            if (p.pre) {
                float wp[SEQ_CH], ws[SEQ_CH], w2[SEQ_CH], t[SEQ_CH];
                zero8(t);
                param8(p.post, c, n, wp);
                param8(p.scale, c, n, ws);
                param8(p.pre, c, n, w2);
                if (p.dy) load8<T, VEC>((const T*)p.dy + r * p.D + c, n, t);
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) {
                    hv[i][j] = fmaf(ws[j] * wp[j], v[i][j], hv[i][j]) * inv2;  // y / pre
                    dpre[i][j] = fmaf(t[j], hv[i][j], dpre[i][j]);
                    t[j] *= w2[j];
                    sum2 = fmaf(t[j], hv[i][j], sum2);
                    d[i][j] = fmaf(inv2, t[j], d[i][j]);
                }
            }
        }
        if (p.pre) {
            const float m = row_sum(sum2, tpr, lds, slot) * rd * inv2;
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) d[i][j] = fmaf(-m, hv[i][j], d[i][j]);
        }
        float sum1 = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            if (!live || c >= p.D) continue;
            const int n = p.D - c;
            float wp[SEQ_CH], ws[SEQ_CH];
            if (p.res) store8<TR, VEC>((TR*)p.dres + r * p.D + c, n, d[i]);
            param8(p.post, c, n, wp);
            param8(p.scale, c, n, ws);
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) {
                dscale[i][j] = fmaf(d[i][j], v[i][j] * wp[j], dscale[i][j]);
                d[i][j] *= ws[j];
                dpost[i][j] = fmaf(d[i][j], v[i][j], dpost[i][j]);
                d[i][j] *= wp[j];
                sum1 = fmaf(d[i][j], v[i][j], sum1);
            }
        }
        const float m1 = p.post ? row_sum(sum1, tpr, lds, slot) * rd : 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int c = (i * tpr + lane) * SEQ_CH;
            if (!live || c >= p.D) continue;
            const int n = p.D - c;
            float o[SEQ_CH], og[SEQ_CH];
#pragma unroll
            for (int j = 0; j < SEQ_CH; ++j) {
                const float dp = inv1 * fmaf(-m1, v[i][j], d[i][j]);
                if (p.gate) {
                    const float sg = fast_sigmoid(gt[i][j]);
                    const float si = gt[i][j] * sg;
                    o[j] = dp * si;
                    og[j] = dp * xv[i][j] * (sg + si * (1.f - sg));
                } else {
                    o[j] = dp;
                    og[j] = 0.f;
                }
            }
            store8<T, VEC>((T*)p.dx + r * p.D + c, n, o);
            if (p.gate) store8<T, VEC>((T*)p.dgate + r * p.D + c, n, og);
        }
    }
    // column gradients of the weights there are, in the order post | scale | pre
    const int W = VPT * tpr * SEQ_CH;
    float* ws = p.ws + (long)blockIdx.x * ((p.post != nullptr) + (p.scale != nullptr) + (p.pre != nullptr)) * p.D;
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
                ws[c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VPT; ++i)
#pragma unroll
                for (int j = 0; j < SEQ_CH; ++j) {
                    const int c = (i * tpr + lane) * SEQ_CH + j;
                    if (c < p.D) ws[c] = acc[i][j];
                }
        }
        ws += p.D;
    }
}

// Threads a row, chunks a thread: one chunk each while a wave holds the row,
// then two in as many whole waves as the row needs (to D = 8192), then four.
inline void row_shape(long D, int* tpr, int* vpt) {
    const long chunks = (D + SEQ_CH - 1) / SEQ_CH;
    *vpt = chunks <= 64 ? 1 : chunks <= 1024 ? 2 : 4;
    *tpr = chunks <= 64 ? pow2_ceil(chunks) : (int)((chunks + 64 * *vpt - 1) / (64 * *vpt)) * 64;
}

// Whole rows in a block of about 256 threads.
inline int block_threads(int tpr) { return tpr >= 256 ? tpr : 256 / tpr * tpr; }

struct NormFwd {
    const BlockNormParams& p;
    hipStream_t s;
    template <typename T, typename TR, int VPT, bool V>
    void operator()(int tpr) const {
        const int block = block_threads(tpr);
        const long want = (p.R + block / tpr - 1) / (block / tpr);
        hipLaunchKernelGGL((block_norm_fwd_kernel<T, TR, VPT, V>), dim3((unsigned)(want < 65536 ? want : 65536)), dim3(block), 0, s,
            p, tpr);
    }
};

struct NormBwd {
    const BlockNormParams& p;
    hipStream_t s;
    template <typename T, typename TR, int VPT, bool V>
    void operator()(int tpr) const {
        const int block = block_threads(tpr);
        const size_t smem = block > tpr ? (size_t)block * VPT * SEQ_CH * sizeof(float) : 0;
        hipLaunchKernelGGL((block_norm_bwd_kernel<T, TR, VPT, V>), dim3(p.slots), dim3(block), smem, s,
            p, tpr);
    }
};

template <typename T, typename TR, typename F>
void by_shape(const BlockNormParams& p, F f) {
    int tpr, vpt;
    row_shape(p.D, &tpr, &vpt);
    auto with = [&](auto v) {
        constexpr bool V = decltype(v)::value;
        if (vpt == 1) f.template operator()<T, TR, 1, V>(tpr);
        else if (vpt == 2) f.template operator()<T, TR, 2, V>(tpr);
        else f.template operator()<T, TR, 4, V>(tpr);
    };
    if (p.vec) with(std::true_type{});
    else with(std::false_type{});
}

template <typename F>
void by_type(const BlockNormParams& p, int is_f32, int res_f32, F f) {
    if (is_f32 && res_f32) by_shape<float, float>(p, f);
    else if (is_f32) by_shape<float, __bf16>(p, f);
    else if (res_f32) by_shape<__bf16, float>(p, f);
    else by_shape<__bf16, __bf16>(p, f);
}

}  // namespace

extern "C" int block_norm_slots(long R, long D) {
    int tpr, vpt;
    row_shape(D, &tpr, &vpt);
    const int block = block_threads(tpr);
    const long want = (R + block / tpr - 1) / (block / tpr);
    const long cap = 1024;
    return (int)(want < cap ? want : cap);
}

extern "C" void block_norm_fwd_launch(const BlockNormParams& p, int is_f32, int res_f32, hipStream_t s) {
    by_type(p, is_f32, res_f32, NormFwd{p, s});
}

extern "C" void block_norm_bwd_launch(const BlockNormParams& p, int is_f32, int res_f32, hipStream_t s) {
    by_type(p, is_f32, res_f32, NormBwd{p, s});
}
