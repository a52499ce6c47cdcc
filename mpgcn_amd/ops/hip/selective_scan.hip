// Selective state space scan (gfx950). Per sequence b and channel d, with N
// states and the per-token B, C shared by the D/G channels of a group:
//   dt_t = softplus(delta_t + dbias)
//   h_t[n] = exp(dt_t A[n]) h_{t-1}[n] + dt_t u_t B_t[n]
//   y_t    = sum_n C_t[n] h_t[n] + skip u_t
//
// States, sums and step sizes are f32 throughout; only what is stored as bf16
// is rounded. A lane owns NS states of one channel (LPC lanes share a channel
// when N > 16), so the sum over states stays in the lane; the 64 lanes of a
// wave are CW channels x RW sequences x LPC. exp is v_exp_f32 of
// dt * (A log2 e). What is past a sequence's valid length has dt = 0 and reads
// no B or C: the state passes it unchanged.
#include "seq.hpp"

#define SCAN_CH 8  // steps whose states the backward holds in registers

namespace {

constexpr float LOG2E = 1.4426950408889634f;

struct Lanes {
    int cw;  // channels a wave covers, a power of two
    int rw;  // sequences a wave covers
    int cb;  // channel blocks per group
};

inline int scan_ns(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : 16; }
inline int scan_lpc(int N) { return N <= 16 ? 1 : N <= 32 ? 2 : 4; }

inline Lanes scan_lanes(long D, long G, long N) {
    const int lpc = scan_lpc((int)N);
    const long per = D / G;
    Lanes l;
    l.cw = pow2_ceil(per) < 64 / lpc ? pow2_ceil(per) : 64 / lpc;
    l.rw = 64 / (l.cw * lpc);
    l.cb = (int)((per + l.cw - 1) / l.cw);
    return l;
}

// NS entries of a row of B or C from state n0; zero past N.
template <typename T, int NS>
__device__ __forceinline__ void state_row(const T* __restrict__ p, int n0, int N, int vec, bool ok,
                                          float (&v)[NS]) {
    if (vec && n0 + NS <= N) {
        if (ok) {
            constexpr int C = NS * sizeof(T) / 16 ? NS * sizeof(T) / 16 : 1;
            if constexpr (NS * sizeof(T) >= 16) {
                Chunk16 c[C];
#pragma unroll
                for (int i = 0; i < C; ++i) c[i] = ((const Chunk16*)(p + n0))[i];
#pragma unroll
                for (int i = 0; i < NS; ++i) v[i] = to_f32(((const T*)c)[i]);
                return;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < NS; ++i) v[i] = (ok && n0 + i < N) ? to_f32(p[n0 + i]) : 0.f;
}

struct Place {
    int b, g, d, n0;  // this lane's sequence, group, channel, first state
    bool ok;          // false: the lane has no work and must store nothing
};

template <int LPC, int NS>
__device__ __forceinline__ Place place_of(const ScanParams& p, int cw, int lane, int g, int cblk, long b0) {
    Place q;
    const int per = p.D / p.G;
    const int rest = lane & (64 / cw - 1);
    const long b = b0 + rest / LPC;
    const int c = cblk * cw + lane / (64 / cw);
    q.ok = b < p.B && c < per;
    q.b = q.ok ? (int)b : 0;
    q.g = g;
    q.d = g * per + (q.ok ? c : 0);
    q.n0 = (lane & (LPC - 1)) * NS;
    return q;
}

template <typename T, int NS, int LPC>
__launch_bounds__(256) __global__ void scan_fwd_kernel(ScanParams p, Lanes l, long waves) {
    const int lane = threadIdx.x & 63;
    long w = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= waves) return;
    const int cblk = (int)(w % l.cb);
    w /= l.cb;
    const int g = (int)(w % p.G);
    const Place q = place_of<LPC, NS>(p, l.cw, lane, g, cblk, (w / p.G) * l.rw);
    const int N = p.N, D = p.D;
    const int len = q.ok ? seq_len(p.lens, p.lens64, q.b, p.L) : 0;

    float A2[NS], h[NS];
    const float* h0 = p.h0 ? p.h0 + ((long)q.b * D + q.d) * N : nullptr;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const bool on = q.n0 + i < N;
        A2[i] = on ? p.A[(long)q.d * N + q.n0 + i] * LOG2E : 0.f;
        h[i] = (on && h0 && q.ok) ? h0[q.n0 + i] : 0.f;
    }
    const float skip = p.skip ? p.skip[q.d] : 0.f;
    const float dbias = p.dbias ? p.dbias[q.d] : 0.f;
    const T* u = (const T*)p.u + q.b * p.u_b + q.d;
    const T* de = (const T*)p.delta + q.b * p.d_b + q.d;
    const T* Bm = (const T*)p.Bm + q.b * p.B_b + q.g * p.B_g;
    const T* Cm = (const T*)p.Cm + q.b * p.C_b + q.g * p.C_g;
    T* y = (T*)p.y + (long)q.b * p.L * D + q.d;
    const long chunks = (p.L + SCAN_CH - 1) / SCAN_CH;

    for (int t0 = 0; t0 < p.L; t0 += SCAN_CH) {
        if (p.ckpt && q.ok) {
            float* ck = p.ckpt + (((long)q.b * chunks + t0 / SCAN_CH) * D + q.d) * N;
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (q.n0 + i < N) ck[q.n0 + i] = h[i];
        }
        float uv[SCAN_CH], dv[SCAN_CH];
#pragma unroll
        for (int j = 0; j < SCAN_CH; ++j) {
            const bool on = t0 + j < len;
            uv[j] = on ? to_f32(u[(t0 + j) * p.u_t]) : 0.f;
            dv[j] = on ? to_f32(de[(t0 + j) * p.d_t]) + dbias : 0.f;
        }
#pragma unroll
        for (int j = 0; j < SCAN_CH; ++j) {
            const int t = t0 + j;
            if (t >= p.L) break;
            const bool on = t < len;
            const float dt = on ? (p.softplus ? softplus_f(dv[j]) : dv[j]) : 0.f;
            const float du = dt * uv[j];
            float Bv[NS], Cv[NS];
            state_row<T, NS>(Bm + t * p.B_t, q.n0, N, p.bvec, on, Bv);
            state_row<T, NS>(Cm + t * p.C_t, q.n0, N, p.bvec, on, Cv);
            float acc = 0.f;
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                h[i] = fmaf(__builtin_amdgcn_exp2f(dt * A2[i]), h[i], du * Bv[i]);
                acc = fmaf(Cv[i], h[i], acc);
            }
#pragma unroll
            for (int m = 1; m < LPC; m <<= 1) acc += __shfl_xor(acc, m);
            if (q.ok && q.n0 == 0) y[(long)t * D] = from_f32<T>(on ? fmaf(skip, uv[j], acc) : 0.f);
        }
    }
    if (p.h1 && q.ok) {
        float* h1 = p.h1 + ((long)q.b * D + q.d) * N;
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (q.n0 + i < N) h1[q.n0 + i] = h[i];
    }
}

// Sum V values over a wave's channels (the high bits of the lane, down to the
// bit `lo`). While a lane carries more than one value each step halves them:
// partners keep one half each and exchange the other. A lane ends with the
// values idx, idx + 1, .. of the V in v[0], v[1], ..
template <int V>
__device__ __forceinline__ void reduce_channels(float (&v)[V], int lo, int lane, int* idx) {
    int at = 0;
#pragma unroll
    for (int s = 0; s < 6; ++s) {
        const int m = 32 >> s;
        if (m < lo) break;
        const int left = V >> (s + 1);
        if (left > 0) {
            const bool up = lane & m;
#pragma unroll
            for (int i = 0; i < left; ++i) {
                const float keep = up ? v[i + left] : v[i];
                const float send = up ? v[i] : v[i + left];
                v[i] = keep + __shfl_xor(send, m);
            }
            at += up ? left : 0;
        } else {
            v[0] += __shfl_xor(v[0], m);
        }
    }
    *idx = at;
}

// Backward, from the adjoint recurrence of the state
//   g_t = C_t dy_t + exp(dt_{t+1} A) g_{t+1}:
//   dC_t = sum_d dy_t h_t            dB_t = sum_d g_t dt_t u_t
//   du_t = skip dy_t + dt_t sum_n g_t B_t
//   ddt_t = u_t sum_n g_t B_t + sum_n g_t A exp(dt_t A) h_{t-1}
//   dA = sum g_t dt_t exp(dt_t A) h_{t-1}
// Walked chunk by chunk from the end: the states of a chunk are recomputed from
// the one saved at its start and held in registers.
template <typename T, int NS, int LPC>
__launch_bounds__(256) __global__ void scan_bwd_kernel(ScanParams p, Lanes l) {
    const int lane = threadIdx.x & 63;
    int w = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int cblk = w % l.cb;
    w /= l.cb;
    const int g = w % p.G;
    const int slot = w / p.G;
    if (slot >= p.slots) return;
    const int N = p.N, D = p.D;
    const long chunks = (p.L + SCAN_CH - 1) / SCAN_CH;
    const long groups = (p.B + l.rw - 1) / l.rw;

    float A2[NS], dA[NS];
    float dskip = 0.f, ddb = 0.f;
    const Place q0 = place_of<LPC, NS>(p, l.cw, lane, g, cblk, 0);
    const int chl = lane / (64 / l.cw);
    const bool has_c = cblk * l.cw + chl < D / p.G;
    const int d = has_c ? g * (D / p.G) + cblk * l.cw + chl : q0.d;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        A2[i] = q0.n0 + i < N ? p.A[(long)d * N + q0.n0 + i] * LOG2E : 0.f;
        dA[i] = 0.f;
    }
    const float skip = p.skip ? p.skip[d] : 0.f;
    const float dbias = p.dbias ? p.dbias[d] : 0.f;

    for (long it = slot; it < groups; it += p.slots) {
        const Place q = place_of<LPC, NS>(p, l.cw, lane, g, cblk, it * l.rw);
        const int len = q.ok ? seq_len(p.lens, p.lens64, q.b, p.L) : 0;
        const T* u = (const T*)p.u + q.b * p.u_b + q.d;
        const T* de = (const T*)p.delta + q.b * p.d_b + q.d;
        const T* Bm = (const T*)p.Bm + q.b * p.B_b + q.g * p.B_g;
        const T* Cm = (const T*)p.Cm + q.b * p.C_b + q.g * p.C_g;
        const long at = (long)q.b * p.L * D + q.d;
        const T* dy = p.dy ? (const T*)p.dy + at : nullptr;
        T* du = (T*)p.du + at;
        T* dde = (T*)p.ddelta + at;

        float gs[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i)
            gs[i] = (p.dh1 && q.ok && q.n0 + i < N) ? p.dh1[((long)q.b * D + q.d) * N + q.n0 + i] : 0.f;

        for (long ck = chunks - 1; ck >= 0; --ck) {
            const int t0 = (int)ck * SCAN_CH;
            float h[NS], hist[SCAN_CH][NS], uv[SCAN_CH], xv[SCAN_CH], dyv[SCAN_CH];
            const float* hs = p.ckpt ? p.ckpt + (((long)q.b * chunks + ck) * D + q.d) * N
                              : p.h0 ? p.h0 + ((long)q.b * D + q.d) * N : nullptr;
#pragma unroll
            for (int i = 0; i < NS; ++i) h[i] = (hs && q.ok && q.n0 + i < N) ? hs[q.n0 + i] : 0.f;
#pragma unroll
            for (int j = 0; j < SCAN_CH; ++j) {
                const bool on = t0 + j < len;
                uv[j] = on ? to_f32(u[(t0 + j) * p.u_t]) : 0.f;
                xv[j] = on ? to_f32(de[(t0 + j) * p.d_t]) + dbias : 0.f;
                dyv[j] = (on && dy) ? to_f32(dy[(long)(t0 + j) * D]) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < SCAN_CH; ++j) {
                const bool on = t0 + j < len;
                const float dt = on ? (p.softplus ? softplus_f(xv[j]) : xv[j]) : 0.f;
                float Bv[NS];
                state_row<T, NS>(Bm + (t0 + j) * p.B_t, q.n0, N, p.bvec, on, Bv);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    hist[j][i] = h[i];
                    h[i] = fmaf(__builtin_amdgcn_exp2f(dt * A2[i]), h[i], dt * uv[j] * Bv[i]);
                }
            }
#pragma unroll
            for (int j = SCAN_CH - 1; j >= 0; --j) {
                const int t = t0 + j;
                if (t >= p.L) continue;
                const bool on = t < len;
                const float dt = on ? (p.softplus ? softplus_f(xv[j]) : xv[j]) : 0.f;
                float Bv[NS], Cv[NS], bc[2 * NS];
                state_row<T, NS>(Bm + t * p.B_t, q.n0, N, p.bvec, on, Bv);
                state_row<T, NS>(Cm + t * p.C_t, q.n0, N, p.bvec, on, Cv);
                float into = 0.f, dec = 0.f;
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    const float a = __builtin_amdgcn_exp2f(dt * A2[i]);
                    const float back = a * hist[j][i];
                    const float now = fmaf(dt * uv[j], Bv[i], back);
                    gs[i] = fmaf(Cv[i], dyv[j], gs[i]);
                    bc[i] = gs[i] * (dt * uv[j]);
                    bc[NS + i] = dyv[j] * now;
                    into = fmaf(gs[i], Bv[i], into);
                    const float gb = gs[i] * back;
                    dec = fmaf(gb, A2[i], dec);
                    dA[i] = fmaf(gb, dt, dA[i]);
                    gs[i] *= a;
                }
#pragma unroll
                for (int m = 1; m < LPC; m <<= 1) {
                    into += __shfl_xor(into, m);
                    dec += __shfl_xor(dec, m);
                }
                float dx = fmaf(uv[j], into, dec * (1.f / LOG2E));
                if (p.softplus) dx *= fast_sigmoid(xv[j]);
                dx = on ? dx : 0.f;
                const bool first = q.n0 == 0;
                if (q.ok && first) {
                    du[(long)t * D] = from_f32<T>(on ? fmaf(skip, dyv[j], dt * into) : 0.f);
                    dde[(long)t * D] = from_f32<T>(dx);
                }
                ddb += dx;
                dskip = fmaf(dyv[j], uv[j], dskip);
                int idx;
                reduce_channels<2 * NS>(bc, 64 / l.cw, lane, &idx);
                // the lane holds `width` values; where there are more channels
                // than values, `spare` lanes hold the same one
                const int width = l.cw < 2 * NS ? 2 * NS / l.cw : 1;
                const int spare = l.cw > 2 * NS ? l.cw / (2 * NS) : 1;
                const long bb = it * l.rw + (lane & (64 / l.cw - 1)) / LPC;
                if (bb < p.B && (chl & (spare - 1)) == 0) {
                    float* o = p.dbc + ((((long)cblk * p.B + bb) * p.L + t) * p.G + g) * 2 * N;
#pragma unroll
                    for (int i = 0; i < 2 * NS; ++i) {
                        if (i >= width) break;
                        const int n = q0.n0 + ((idx + i) & (NS - 1));
                        if (n < N) o[(idx + i >= NS ? N : 0) + n] = bc[i];
                    }
                }
            }
        }
        if (p.dh0 && q.ok) {
#pragma unroll
            for (int i = 0; i < NS; ++i)
                if (q.n0 + i < N) p.dh0[((long)q.b * D + q.d) * N + q.n0 + i] = gs[i];
        }
    }
    // the wave's sequences share their channels: join them, then one row per slot
    for (int m = LPC; m < 64 / l.cw; m <<= 1) {
#pragma unroll
        for (int i = 0; i < NS; ++i) dA[i] += __shfl_xor(dA[i], m);
        dskip += __shfl_xor(dskip, m);
        ddb += __shfl_xor(ddb, m);
    }
    if ((lane & (64 / l.cw - 1)) < LPC && has_c) {
        float* ws = p.ws + (long)slot * D * (N + 2);
#pragma unroll
        for (int i = 0; i < NS; ++i)
            if (q0.n0 + i < N) ws[(long)d * N + q0.n0 + i] = dA[i];
        if (q0.n0 == 0) {
            ws[(long)D * N + d] = dskip;
            ws[(long)D * N + D + d] = ddb;
        }
    }
}

// dB and dC: the channel blocks' partial sums in ascending order.
template <typename T>
__launch_bounds__(256) __global__ void scan_bc_reduce_kernel(const float* __restrict__ dbc,
                                                             T* __restrict__ dB, T* __restrict__ dC,
                                                             long cblocks, long rows, int N) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * 2 * N) return;
    float s = 0.f;
    for (long c = 0; c < cblocks; ++c) s += dbc[c * rows * 2 * N + i];
    const long row = i / (2 * N);
    const int n = (int)(i % (2 * N));
    (n < N ? dB : dC)[row * N + (n < N ? n : n - N)] = from_f32<T>(s);
}

// One new token. Bound by the state, read and written once: 4 states (16
// bytes) a lane, `gp` lanes a channel, joined by lane exchanges for y. Every
// lane reads its own states before it writes them: h_out may be h.
template <typename T, bool VEC>
__launch_bounds__(256) __global__ void scan_step_kernel(ScanStepParams p, int gp, long items) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    const bool ok = i < items;
    const long r = ok ? i / gp : 0;
    const int n0 = ok ? (int)(i % gp) * 4 : p.N;
    const int d = (int)(r % p.D);
    const long b = r / p.D;
    const int g = d / (p.D / p.G);
    const int N = p.N;
    const float uv = to_f32(((const T*)p.u)[b * p.u_b + d]);
    float dt = to_f32(((const T*)p.delta)[b * p.d_b + d]) + (p.dbias ? p.dbias[d] : 0.f);
    if (p.softplus) dt = softplus_f(dt);
    const T* Bm = (const T*)p.Bm + b * p.B_b + g * p.B_g;
    const T* Cm = (const T*)p.Cm + b * p.C_b + g * p.C_g;
    const float* h = p.h + r * N;
    const float* A = p.A + (long)d * N;
    float hv[4], Av[4], Bv[4], Cv[4];
    if (VEC && n0 < N) {
        *(f32x4*)hv = *(const f32x4*)(h + n0);
        *(f32x4*)Av = *(const f32x4*)(A + n0);
        T tb[4], tc[4];
        if constexpr (sizeof(T) == 2) {
            *(long*)tb = *(const long*)(Bm + n0);
            *(long*)tc = *(const long*)(Cm + n0);
        } else {
            *(f32x4*)tb = *(const f32x4*)(Bm + n0);
            *(f32x4*)tc = *(const f32x4*)(Cm + n0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            Bv[j] = to_f32(tb[j]);
            Cv[j] = to_f32(tc[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool on = n0 + j < N;
            hv[j] = on ? h[n0 + j] : 0.f;
            Av[j] = on ? A[n0 + j] : 0.f;
            Bv[j] = on ? to_f32(Bm[n0 + j]) : 0.f;
            Cv[j] = on ? to_f32(Cm[n0 + j]) : 0.f;
        }
    }
    float acc = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        hv[j] = fmaf(__builtin_amdgcn_exp2f(dt * (Av[j] * LOG2E)), hv[j], dt * uv * Bv[j]);
        acc = fmaf(Cv[j], hv[j], acc);
    }
    for (int m = 1; m < gp; m <<= 1) acc += __shfl_xor(acc, m);
    if (!ok) return;
    float* ho = p.h_out + r * N;
    if (VEC && n0 < N) {
        *(f32x4*)(ho + n0) = *(const f32x4*)hv;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < N) ho[n0 + j] = hv[j];
    }
    if (n0 == 0) ((T*)p.y)[b * p.D + d] = from_f32<T>(p.skip ? fmaf(p.skip[d], uv, acc) : acc);
}

template <typename T, typename F>
void by_states(int N, F f) {
    if (N <= 4) f.template operator()<T, 4, 1>();
    else if (N <= 8) f.template operator()<T, 8, 1>();
    else if (N <= 16) f.template operator()<T, 16, 1>();
    else if (N <= 32) f.template operator()<T, 16, 2>();
    else f.template operator()<T, 16, 4>();
}

struct ScanFwd {
    const ScanParams& p;
    hipStream_t s;
    template <typename T, int NS, int LPC>
    void operator()() const {
        const Lanes l = scan_lanes(p.D, p.G, p.N);
        const long waves = (long)((p.B + l.rw - 1) / l.rw) * p.G * l.cb;
        hipLaunchKernelGGL((scan_fwd_kernel<T, NS, LPC>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, s,
            p, l, waves);
    }
};

struct ScanBwd {
    const ScanParams& p;
    hipStream_t s;
    template <typename T, int NS, int LPC>
    void operator()() const {
        const Lanes l = scan_lanes(p.D, p.G, p.N);
        const long waves = (long)p.slots * p.G * l.cb;
        hipLaunchKernelGGL((scan_bwd_kernel<T, NS, LPC>), dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, s,
            p, l);
    }
};

}  // namespace

extern "C" int scan_chunk() { return SCAN_CH; }

extern "C" int scan_cblocks(long D, long G, long N) { return scan_lanes(D, G, N).cb; }

// Waves that share the same channels in the backward, each with its own row of
// parameter gradients: about 4096 waves in all.
extern "C" int scan_bwd_slots(long B, long D, long G, long N) {
    const Lanes l = scan_lanes(D, G, N);
    const long groups = (B + l.rw - 1) / l.rw;
    const long cap = (4096 + G * l.cb - 1) / (G * l.cb);
    return (int)(groups < cap ? groups : cap);
}

extern "C" void scan_fwd_launch(const ScanParams& p, int is_f32, hipStream_t s) {
    if (is_f32) by_states<float>(p.N, ScanFwd{p, s});
    else by_states<__bf16>(p.N, ScanFwd{p, s});
}

extern "C" void scan_bwd_launch(const ScanParams& p, int is_f32, hipStream_t s) {
    if (is_f32) by_states<float>(p.N, ScanBwd{p, s});
    else by_states<__bf16>(p.N, ScanBwd{p, s});
}

extern "C" void scan_bc_reduce_launch(const float* dbc, void* dB, void* dC, long cblocks, long rows,
                                      int N, int is_f32, hipStream_t s) {
    const dim3 grid((unsigned)((rows * 2 * N + 255) / 256));
    if (is_f32)
        hipLaunchKernelGGL((scan_bc_reduce_kernel<float>), grid, dim3(256), 0, s,
            dbc, (float*)dB, (float*)dC, cblocks, rows, N);
    else
        hipLaunchKernelGGL((scan_bc_reduce_kernel<__bf16>), grid, dim3(256), 0, s,
            dbc, (__bf16*)dB, (__bf16*)dC, cblocks, rows, N);
}

extern "C" void scan_step_launch(const ScanStepParams& p, int is_f32, hipStream_t s) {
    const int gp = pow2_ceil((p.N + 3) / 4);
    const long items = (long)p.B * p.D * gp;
    const dim3 grid((unsigned)((items + 255) / 256));
    if (is_f32) {
        if (p.bvec) hipLaunchKernelGGL((scan_step_kernel<float, true>), grid, dim3(256), 0, s,
            p, gp, items);
        else hipLaunchKernelGGL((scan_step_kernel<float, false>), grid, dim3(256), 0, s,
            p, gp, items);
    } else {
        if (p.bvec) hipLaunchKernelGGL((scan_step_kernel<__bf16, true>), grid, dim3(256), 0, s,
            p, gp, items);
        else hipLaunchKernelGGL((scan_step_kernel<__bf16, false>), grid, dim3(256), 0, s,
            p, gp, items);
    }
}
