// Selective state space scan (gfx950). Per sequence b and channel d, with N
// states and the per-token B, C shared by the D/G channels of a group:
//   dt_t = softplus(delta_t + dbias)
//   h_t[n] = exp(dt_t A[n]) h_{t-1}[n] + dt_t u_t B_t[n]
//   y_t    = sum_n C_t[n] h_t[n] + skip u_t
//
// States, sums and step sizes are f32 throughout; only what is stored as bf16
// is rounded. Bound by vector arithmetic: an exp (two issue slots) and four
// more operations per state and step against 6 bytes per channel and step.
//
// Layout. Four lanes share four channels: each owns NQ of the states of all
// four, so a row of B or C costs a lane NQ values for 4 NQ states, and loads
// and stores one of the channels itself. Step sizes go round the four lanes by
// DPP, sums over states come back the same way. For N > 16 a channel's states
// spread over KQ such quads. A wave is RW sequences x CW channels x KQ.
//
// Where the sequences are too few to fill the card the time axis is cut into
// segments: one pass finds each segment's end state from zero and its summed
// step size (the segment's decay is exp(A sum dt)), a small one carries the
// states across, and the main pass runs all segments at once from there.
//
// Addresses are a wave-uniform 64-bit base and a 32-bit lane offset; where the
// sequences of a wave lie too far apart for that a wave takes one sequence.
#include "seq.hpp"

#define SCAN_CH 8  // steps of a chunk: the backward holds their states
#define SCAN_PF 4  // steps that loads run ahead in the forward

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// ---- lane exchanges (whole wave active) -------------------------------------

template <int CTRL, int BANK = 0xf>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, BANK, true));
}

template <int M>
__device__ __forceinline__ float from_xor(float v) {
    if constexpr (M == 1) return dpp<0xB1>(v);       // quad_perm [1,0,3,2]
    else if constexpr (M == 2) return dpp<0x4E>(v);  // quad_perm [2,3,0,1]
    else if constexpr (M == 4)                       // row_shl:4 for the low, row_shr:4 for the high
        return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(dpp<0x104>(v)), __float_as_int(v), 0x114, 0xf,
                                                          0xA, false));
    else return dpp<0x128>(v);                       // row_ror:8
}

// Lanes without the bit M keep a + its partner's a, those with it b + its partner's b.
template <int M>
__device__ __forceinline__ float fold(float a, float b, int lane) {
    if constexpr (M == 16) {
        auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(a), __float_as_int(b), false, false);
        return __int_as_float(r[0]) + __int_as_float(r[1]);
    } else if constexpr (M == 32) {
        auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(a), __float_as_int(b), false, false);
        return __int_as_float(r[0]) + __int_as_float(r[1]);
    } else {
        const bool up = lane & M;
        return (up ? b : a) + from_xor<M>(up ? a : b);
    }
}

// v[c] of the quad's lanes summed; the lane with index c in its quad gets v[c].
__device__ __forceinline__ float quad_sum(const float (&v)[4], int lane) {
    return fold<1>(fold<2>(v[0], v[2], lane), fold<2>(v[1], v[3], lane), lane);
}

template <int KQ>
__device__ __forceinline__ float states_sum(const float (&v)[4], int lane) {
    float s = quad_sum(v, lane);
    if constexpr (KQ >= 2) s += from_xor<4>(s);
    if constexpr (KQ >= 4) s += from_xor<8>(s);
    return s;
}

__device__ __forceinline__ void quad_spread(float v, float (&o)[4]) {
    o[0] = dpp<0x00>(v);
    o[1] = dpp<0x55>(v);
    o[2] = dpp<0xAA>(v);
    o[3] = dpp<0xFF>(v);
}

// Sum V values over the quads of a sequence: lane bits from M up to below
// `span`. While a lane carries more than one value each step halves them.
template <int M, int LEFT, int V>
__device__ __forceinline__ void reduce_quads(float (&v)[V], int span, int lane) {
    if constexpr (M <= 32) {
        if (M >= span) return;
        if constexpr (LEFT > 1) {
#pragma unroll
            for (int i = 0; i < LEFT / 2; ++i) v[i] = fold<M>(v[i], v[i + LEFT / 2], lane);
        } else {
            v[0] = fold<M>(v[0], v[0], lane);
        }
        reduce_quads<M * 2, (LEFT > 1 ? LEFT / 2 : 1), V>(v, span, lane);
    }
}

// Where that leaves a lane: `left` values from number `idx`; lanes that differ
// in the bits of `dup` hold the same.
template <int V, int M0>
__device__ __forceinline__ void reduced_place(int span, int lane, int& idx, int& dup, int& left) {
    idx = 0; dup = 0; left = V;
    for (int m = M0; m < span; m <<= 1) {
        if (left > 1) {
            left >>= 1;
            idx += (lane & m) ? left : 0;
        } else {
            dup |= m;
        }
    }
}

// ---- a lane's place ---------------------------------------------------------

template <typename T, int NQ, int KQ>
struct Place {
    int lane, rs, b, d, n0;   // sequence in the wave, sequence, own channel, first state
    int d4, nd;               // the quad's first channel, how many of its four there are
    bool okb, ok, own;        // the sequence exists; and the channel; and this lane stores it
    int slen, len;            // valid steps of the sequence, of the own channel (0: no such channel)

    __device__ __forceinline__ Place(const ScanParams& p, const ScanPlan& l, int lane_, int g, int cblk, long b0) {
        lane = lane_;
        const int per = p.D / p.G;
        const int quad = (lane / (4 * KQ)) & (l.cw / 4 - 1);
        const int kq = (lane >> 2) & (KQ - 1);
        rs = lane / (l.cw * KQ);
        okb = b0 + rs < p.B;
        rs = okb ? rs : 0;
        b = (int)b0 + rs;
        const int c4 = cblk * l.cw + quad * 4, c = c4 + (lane & 3);
        nd = per - c4 < 0 ? 0 : per - c4 > 4 ? 4 : per - c4;
        const bool okc = c < per;
        d = g * per + (okc ? c : 0);
        d4 = g * per + (nd ? c4 : 0);
        n0 = (kq * 4 + (lane & 3)) * NQ;
        ok = okb && okc;
        own = ok && kq == 0;
        slen = okb ? seq_len(p.lens, p.lens64, b, p.L) : 0;
        len = ok ? slen : 0;
    }
    __device__ __forceinline__ bool state(const ScanParams& p, int c, int i) const { return c < nd && n0 + i < p.N; }
};

// A uniform base and a lane's bytes from there. The offset is kept from being
// widened outside the loops: the load then adds the two by itself.
__device__ __forceinline__ unsigned here(unsigned off) {
    asm volatile("" : "+v"(off));
    return off;
}
template <typename T>
__device__ __forceinline__ T at(const T* base, unsigned off) { return *(const T*)((const char*)base + here(off)); }
template <typename T>
__device__ __forceinline__ void put(T* base, unsigned off, T v) { *(T*)((char*)base + here(off)) = v; }

template <typename T, int NQ>
struct alignas(NQ * sizeof(T) < 16 ? NQ * sizeof(T) : 16) Row { T v[NQ]; };

// NQ entries of a row of B or C; VB: all rows whole and aligned.
template <typename T, int NQ, bool VB>
__device__ __forceinline__ Row<T, NQ> row_at(const T* base, unsigned off, int n) {
    if constexpr (VB) {
        return *(const Row<T, NQ>*)((const char*)base + here(off));
    } else {
        Row<T, NQ> r;
#pragma unroll
        for (int i = 0; i < NQ; ++i) r.v[i] = i < n ? ((const T*)((const char*)base + off))[i] : (T)0.f;
        return r;
    }
}

// to f32; zeros where the step is past the sequence's end
template <typename T, int NQ>
__device__ __forceinline__ void widen(const Row<T, NQ>& r, bool on, float (&v)[NQ]) {
    if constexpr (sizeof(r) >= 4) {
        int w[sizeof(r) / 4];
        __builtin_memcpy(w, &r, sizeof(r));
#pragma unroll
        for (int i = 0; i < (int)(sizeof(r) / 4); ++i) w[i] = on ? w[i] : 0;
        Row<T, NQ> z;
        __builtin_memcpy(&z, w, sizeof(r));
#pragma unroll
        for (int i = 0; i < NQ; ++i) v[i] = to_f32(z.v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < NQ; ++i) v[i] = on ? to_f32(r.v[i]) : 0.f;
    }
}

// log(1 + e^x). e^-|x| with the argument's rounding put right, the logarithm of
// 1 + e with that sum's: a few 2^-24 of the result over the whole range.
__device__ __forceinline__ float softplus_s(float x) {
    const float a = -fabsf(x), hi = a * LOG2E, lo = fmaf(a, LOG2E, -hi);
    float e = __builtin_amdgcn_exp2f(hi);
    e = fmaf(e * lo, LN2, e);
    const float s = 1.f + e;
    return fmaxf(x, 0.f) + fmaf(__builtin_amdgcn_logf(s), LN2, e - (s - 1.f));
}

// s[i] where ok, else 0: read without a branch
__device__ __forceinline__ float pick(const float* __restrict__ s, bool ok, long i) {
    const float v = s[ok ? i : 0];
    return ok ? v : 0.f;
}

template <int NQ, int KQ, typename P>
__device__ __forceinline__ void load_decay(const ScanParams& p, const P& q, f32x4 (&A2)[NQ]) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < NQ; ++i)
            A2[i][c] = pick(p.A, q.state(p, c, i), (long)(q.d4 + c) * p.N + q.n0 + i) * LOG2E;
}

// (B, D, N) states of the lane, or zeros
template <int NQ, typename P>
__device__ __forceinline__ void load_states(const ScanParams& p, const P& q, const float* s, f32x4 (&h)[NQ]) {
    const bool some = s != nullptr && q.okb;
    s = s ? s : p.A;  // anything that can be read
    // addresses and masks are formed here, not kept over the loop around
    int d4 = q.d4, nd = q.nd, n0 = q.n0;
    asm volatile("" : "+v"(d4), "+v"(nd), "+v"(n0));
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < NQ; ++i)
            h[i][c] = pick(s, some && c < nd && n0 + i < p.N, ((long)q.b * p.D + d4 + c) * p.N + n0 + i);
}
template <int NQ, typename P>
__device__ __forceinline__ void store_states(const ScanParams& p, const P& q, float* s, const f32x4 (&h)[NQ]) {
    int d4 = q.d4, nd = q.nd, n0 = q.n0;
    asm volatile("" : "+v"(d4), "+v"(nd), "+v"(n0));
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < NQ; ++i)
            if (q.okb && c < nd && n0 + i < p.N) s[((long)q.b * p.D + d4 + c) * p.N + n0 + i] = h[i][c];
}
// the same in the order of a wave's lanes: 16 bytes a lane, NQ rows of them
template <int NQ>
__device__ __forceinline__ void load_lanes(const float* s, long slot, int lane, f32x4 (&h)[NQ]) {
    const f32x4* v = (const f32x4*)s + slot * NQ * 64 + lane;
#pragma unroll
    for (int i = 0; i < NQ; ++i) h[i] = v[i * 64];
}
template <int NQ>
__device__ __forceinline__ void store_lanes(float* s, long slot, int lane, const f32x4 (&h)[NQ]) {
    f32x4* v = (f32x4*)s + slot * NQ * 64 + lane;
#pragma unroll
    for (int i = 0; i < NQ; ++i) v[i * 64] = h[i];
}


__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// One step's inputs as they are in memory.
template <typename T, int NQ>
struct Step { T u, de, dy; Row<T, NQ> B, C; };

// Walks the inputs step by step: uniform pointers that stop at the ends of the
// sequence, so that a step past them reads what is there and counts as nothing.
template <typename T, int NQ, int KQ, bool VB>
struct Walk {
    const T *u, *de, *Bm, *Cm, *dy;
    unsigned ou, od, oB, oC, oy;  // this lane's bytes from there
    int nB;                       // entries of a row this lane may read
    int t;

    template <typename P>
    __device__ __forceinline__ Walk(const ScanParams& p, const P& q, int g, long b0, int t0) {
        t = t0 < p.L ? t0 : p.L - 1;
        u = (const T*)p.u + b0 * p.u_b + (long)t * p.u_t;
        de = (const T*)p.delta + b0 * p.d_b + (long)t * p.d_t;
        Bm = (const T*)p.Bm + b0 * p.B_b + g * p.B_g + (long)t * p.B_t;
        Cm = (const T*)p.Cm + b0 * p.C_b + g * p.C_g + (long)t * p.C_t;
        dy = (const T*)p.dy + (b0 * p.L + t) * p.D;
        ou = (unsigned)((q.rs * p.u_b + q.d) * sizeof(T));
        od = (unsigned)((q.rs * p.d_b + q.d) * sizeof(T));
        nB = p.N - q.n0 < 0 ? 0 : p.N - q.n0;
        const int n0 = nB ? q.n0 : 0;
        oB = (unsigned)((q.rs * p.B_b + n0) * sizeof(T));
        oC = (unsigned)((q.rs * p.C_b + n0) * sizeof(T));
        oy = (unsigned)(((long)q.rs * p.L * p.D + q.d) * sizeof(T));
    }
    template <bool U, bool DY, bool B, bool C>
    __device__ __forceinline__ Step<T, NQ> read() const {
        Step<T, NQ> s;
        s.de = at(de, od);
        if (U) s.u = at(u, ou);
        if (DY) s.dy = at(dy, oy);
        if (B) s.B = row_at<T, NQ, VB>(Bm, oB, nB);
        if (C) s.C = row_at<T, NQ, VB>(Cm, oC, nB);
        return s;
    }
    __device__ __forceinline__ void forth(const ScanParams& p) {
        const bool go = t + 1 < p.L;
        t += go ? 1 : 0;
        u += go ? p.u_t : 0;
        de += go ? p.d_t : 0;
        Bm += go ? p.B_t : 0;
        Cm += go ? p.C_t : 0;
        dy += go ? p.D : 0;
    }
    __device__ __forceinline__ void back(const ScanParams& p, int from) {  // from step `from` to the one before
        const bool go = from < p.L && from > 0;
        u -= go ? p.u_t : 0;
        de -= go ? p.d_t : 0;
        Bm -= go ? p.B_t : 0;
        Cm -= go ? p.C_t : 0;
        dy -= go ? p.D : 0;
    }
};

__device__ __forceinline__ float step_size(const ScanParams& p, bool on, float x) {
    float s = softplus_s(x);
    asm volatile("" : "+v"(s));  // no branch around it: the steps stay one block
    s = p.softplus ? s : x;
    return on ? s : 0.f;
}

// ---- forward ----------------------------------------------------------------

// MAIN: outputs, chunk states, final state. Otherwise the end state of a
// segment from zero and its summed step size. A wave keeps its channels and
// takes one (sequences, segment) after another.
template <typename T, int NQ, int KQ, bool VB, bool MAIN>
__launch_bounds__(256) __global__ void scan_fwd_kernel(ScanParams p, ScanPlan l) {
    const int lane = threadIdx.x & 63;
    const int w = blockIdx.x * 4 + wave_id();
    const int cblk = w % l.cb, g = w / l.cb % p.G, slot = w / l.cb / p.G;
    if (slot >= l.fslots) return;
    const Place<T, NQ, KQ> q0(p, l, lane, g, cblk, 0);
    f32x4 A2[NQ];
    load_decay<NQ, KQ>(p, q0, A2);
    const float skip = p.skip ? p.skip[q0.d] : 0.f;
    const float dbias = p.dbias ? p.dbias[q0.d] : 0.f;

    const int nseg = MAIN ? l.nseg : l.nseg - 1;  // the last segment's end is no start
    const int items = (int)(l.groups * nseg);
    for (int it = slot; it < items; it += l.fslots) {
        const int seg = it % nseg, grp = it / nseg;
        const long b0 = (long)grp * l.rw;
        const long id = ((long)grp * p.G + g) * l.cb + cblk;
        const Place<T, NQ, KQ> q(p, l, lane, g, cblk, b0);
        f32x4 h[NQ];
        load_states<NQ>(p, q, MAIN && l.nseg == 1 ? p.h0 : nullptr, h);
        if (MAIN && l.nseg > 1) load_lanes<NQ>(p.seg_h, id * l.nseg + seg, lane, h);
        float total = 0.f;
        const int t0 = seg * l.seg_chunks * SCAN_CH;
        const int t1 = t0 + l.seg_chunks * SCAN_CH < p.L ? t0 + l.seg_chunks * SCAN_CH : p.L;
        if (t0 < t1) {
            Walk<T, NQ, KQ, VB> in(p, q, g, b0, t0);
            T* y = (T*)p.y + (b0 * p.L + t0) * p.D;
            // SCAN_PF steps ahead of the arithmetic
            Step<T, NQ> ring[SCAN_PF];
#pragma unroll
            for (int j = 0; j < SCAN_PF; ++j) {
                ring[j] = in.template read<true, false, true, MAIN>();
                in.forth(p);
            }
            for (int tc = t0; tc < t1; tc += SCAN_CH) {
                if (MAIN && p.ckpt) store_lanes<NQ>(p.ckpt, id * l.chunks + tc / SCAN_CH, lane, h);
#pragma unroll
                for (int j = 0; j < SCAN_CH; ++j) {
                    const int t = tc + j;
                    if (t >= t1) break;
                    const Step<T, NQ> cur = ring[j % SCAN_PF];
                    const bool on = t < q.len;
                    const float x = to_f32(cur.de) + dbias, uv = on ? to_f32(cur.u) : 0.f;
                    float dts[4], dus[4], Bv[NQ], Cv[NQ], acc[4] = {};
                    widen<T, NQ>(cur.B, t < q.slen, Bv);
                    if (MAIN) widen<T, NQ>(cur.C, t < q.slen, Cv);
                    ring[j % SCAN_PF] = in.template read<true, false, true, MAIN>();
                    in.forth(p);
                    const float dt = step_size(p, on, x);
                    quad_spread(dt, dts);
                    quad_spread(dt * uv, dus);
                    if (!MAIN) total += dt;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
#pragma unroll
                        for (int i = 0; i < NQ; ++i) {
                            h[i][c] = fmaf(__builtin_amdgcn_exp2f(dts[c] * A2[i][c]), h[i][c], dus[c] * Bv[i]);
                            if (MAIN) acc[c] = fmaf(Cv[i], h[i][c], acc[c]);
                        }
                    if (MAIN) {
                        const float s = states_sum<KQ>(acc, lane);
                        if (q.own) put(y, in.oy, from_f32<T>(on ? fmaf(skip, uv, s) : 0.f));
                        y += p.D;
                    }
                }
            }
        }
        if (!MAIN) {
            store_lanes<NQ>(p.seg_h, id * l.nseg + seg, lane, h);
            p.seg_s[(id * l.nseg + seg) * 64 + lane] = total;
        } else if (p.h1 && seg == l.nseg - 1) {
            store_states<NQ>(p, q, p.h1, h);
        }
    }
}

// Turns each segment's own end state into the state it starts from (forward),
// or its own adjoint at the start into the one at its end (backward). One
// thread per four states; all loads of 16 segments are in flight together.
template <int NQ, int KQ, bool BACK>
__launch_bounds__(256) __global__ void scan_carry_kernel(ScanParams p, ScanPlan l, long waves) {
    const int lane = threadIdx.x & 63;
    const long w = (long)blockIdx.x * 4 + wave_id();
    if (w >= waves) return;
    const int i = (int)(w % NQ);
    const long id = w / NQ;
    const Place<float, NQ, KQ> q(p, l, lane, (int)(id / l.cb % p.G), (int)(id % l.cb), id / l.cb / p.G * l.rw);
    const float* first = BACK ? p.dh1 : p.h0;
    f32x4 A2, carry;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const bool on = q.state(p, c, i);
        A2[c] = pick(p.A, on, (long)(q.d4 + c) * p.N + q.n0 + i) * LOG2E;
        carry[c] = first ? pick(first, on && q.okb, ((long)q.b * p.D + q.d4 + c) * p.N + q.n0 + i) : 0.f;
    }
    f32x4* seg_h = (f32x4*)p.seg_h + (id * l.nseg * NQ + i) * 64 + lane;
    const float* seg_s = p.seg_s + id * l.nseg * 64 + lane;
    constexpr int U = 16;
    for (int s0 = 0; s0 < l.nseg; s0 += U) {
        f32x4 own[U];
        float sum[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            // the last one in order has no successor: nothing was stored for it
            const int s = s0 + j < l.nseg - 1 ? s0 + j : 0;
            const long at = BACK ? l.nseg - 1 - s : s;
            own[j] = seg_h[at * NQ * 64];
            sum[j] = seg_s[at * 64];
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int s = s0 + j;
            const long at = BACK ? l.nseg - 1 - s : s;
            if (s < l.nseg) seg_h[at * NQ * 64] = carry;
            float ss[4];
            quad_spread(sum[j], ss);
#pragma unroll
            for (int c = 0; c < 4; ++c) carry[c] = fmaf(__builtin_amdgcn_exp2f(ss[c] * A2[c]), carry[c], own[j][c]);
        }
    }
}

// ---- backward ---------------------------------------------------------------
//
// From the adjoint recurrence of the state
//   g_t = C_t dy_t + exp(dt_{t+1} A) g_{t+1}:
//   dC_t = sum_d dy_t h_t            dB_t = sum_d g_t dt_t u_t
//   du_t = skip dy_t + dt_t sum_n g_t B_t
//   ddt_t = u_t sum_n g_t B_t + sum_n g_t A exp(dt_t A) h_{t-1}
//   dA = sum g_t dt_t exp(dt_t A) h_{t-1}
// Walked chunk by chunk from the end: a chunk's states are recomputed from the
// one the forward kept at its start and held in registers.

// The adjoint that a segment hands to the one before it, from zero at its end.
template <typename T, int NQ, int KQ, bool VB>
__launch_bounds__(256) __global__ void scan_adjoint_kernel(ScanParams p, ScanPlan l) {
    const int lane = threadIdx.x & 63;
    const int w = blockIdx.x * 4 + wave_id();
    const int cblk = w % l.cb, g = w / l.cb % p.G, slot = w / l.cb / p.G;
    if (slot >= l.fslots) return;
    const Place<T, NQ, KQ> q0(p, l, lane, g, cblk, 0);
    f32x4 A2[NQ];
    load_decay<NQ, KQ>(p, q0, A2);
    const float dbias = p.dbias ? p.dbias[q0.d] : 0.f;
    const int items = (int)(l.groups * (l.nseg - 1));
    for (int it = slot; it < items; it += l.fslots) {
        const int seg = it % (l.nseg - 1) + 1, grp = it / (l.nseg - 1);
        const long b0 = (long)grp * l.rw;
        const long id = ((long)grp * p.G + g) * l.cb + cblk;
        const Place<T, NQ, KQ> q(p, l, lane, g, cblk, b0);
        f32x4 gs[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i) gs[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        float total = 0.f;
        const int t0 = seg * l.seg_chunks * SCAN_CH;
        const int t1 = t0 + l.seg_chunks * SCAN_CH < p.L ? t0 + l.seg_chunks * SCAN_CH : p.L;
        Walk<T, NQ, KQ, VB> in(p, q, g, b0, t1 - 1);
        Step<T, NQ> ring[SCAN_PF];
#pragma unroll
        for (int j = 0; j < SCAN_PF; ++j) {
            ring[j] = in.template read<false, true, false, true>();
            in.back(p, t1 - 1 - j);
        }
        for (int tc = t1 - 1; tc >= t0; tc -= SCAN_PF) {
#pragma unroll
            for (int j = 0; j < SCAN_PF; ++j) {
                const int t = tc - j;
                if (t < t0) break;
                const Step<T, NQ> cur = ring[j];
                const bool on = t < q.len;
                const float x = to_f32(cur.de) + dbias, dyv = on ? to_f32(cur.dy) : 0.f;
                float dts[4], dys[4], Cv[NQ];
                widen<T, NQ>(cur.C, t < q.slen, Cv);
                ring[j] = in.template read<false, true, false, true>();
                in.back(p, t - SCAN_PF);
                const float dt = step_size(p, on, x);
                quad_spread(dt, dts);
                quad_spread(dyv, dys);
                total += dt;
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < NQ; ++i)
                        gs[i][c] = fmaf(Cv[i], dys[c], gs[i][c]) * __builtin_amdgcn_exp2f(dts[c] * A2[i][c]);
            }
        }
        store_lanes<NQ>(p.seg_h, id * l.nseg + seg, lane, gs);
        p.seg_s[(id * l.nseg + seg) * 64 + lane] = total;
    }
}

template <typename T, int NQ, int KQ, bool VB>
__launch_bounds__(256, 2) __global__ void scan_bwd_kernel(ScanParams p, ScanPlan l) {
    const int lane = threadIdx.x & 63;
    const int w = blockIdx.x * 4 + wave_id();
    const int cblk = w % l.cb, g = w / l.cb % p.G, slot = w / l.cb / p.G;
    if (slot >= l.slots) return;
    const int N = p.N, D = p.D;
    const Place<T, NQ, KQ> q0(p, l, lane, g, cblk, 0);

    f32x4 A2[NQ], dA[NQ];
    float dskip = 0.f, ddb = 0.f;
    load_decay<NQ, KQ>(p, q0, A2);
#pragma unroll
    for (int i = 0; i < NQ; ++i) dA[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float skip = p.skip ? p.skip[q0.d] : 0.f;
    const float dbias = p.dbias ? p.dbias[q0.d] : 0.f;
    int idx, dup, left;  // one value a lane is left, or two and no duplicates
    reduced_place<2 * NQ, 4 * KQ>(l.cw * KQ, lane, idx, dup, left);
    const int n1 = q0.n0 + (idx & (NQ - 1));  // the first state whose dB or dC this lane stores

    const int items = (int)(l.groups * l.nseg);
    for (int it = slot; it < items; it += l.slots) {
        const int seg = it % l.nseg, grp = it / l.nseg;
        const long b0 = (long)grp * l.rw;
        const long id = ((long)grp * p.G + g) * l.cb + cblk;
        const Place<T, NQ, KQ> q(p, l, lane, g, cblk, b0);
        const bool keeps = q.okb && !(lane & dup) && n1 < N, keeps2 = q.okb && n1 + 1 < N;
        const unsigned obc = (unsigned)(((long)q.rs * p.L * p.G * 2 * N + (idx >= NQ ? N : 0) + n1) * sizeof(float));

        f32x4 gs[NQ];
        load_states<NQ>(p, q, l.nseg == 1 ? p.dh1 : nullptr, gs);
        if (l.nseg > 1) load_lanes<NQ>(p.seg_h, id * l.nseg + seg, lane, gs);

        const int c0 = seg * l.seg_chunks;
        const int c1 = c0 + l.seg_chunks < l.chunks ? c0 + l.seg_chunks : l.chunks;
        for (int ck = c1 - 1; ck >= c0; --ck) {
            const int t0 = ck * SCAN_CH;
            f32x4 hist[SCAN_CH + 1][NQ];
            if (p.ckpt) load_lanes<NQ>(p.ckpt, id * l.chunks + ck, lane, hist[0]);
            else load_states<NQ>(p, q, p.h0, hist[0]);
            Walk<T, NQ, KQ, VB> in(p, q, g, b0, t0);
            Step<T, NQ> next = in.template read<true, false, true, false>();
#pragma unroll
            for (int j = 0; j < SCAN_CH; ++j) {
                const Step<T, NQ> cur = next;
                if (j + 1 < SCAN_CH) {
                    in.forth(p);
                    next = in.template read<true, false, true, false>();
                }
                const bool on = t0 + j < q.len;
                const float dt = step_size(p, on, to_f32(cur.de) + dbias);
                float dts[4], dus[4], Bv[NQ];
                quad_spread(dt, dts);
                quad_spread(on ? dt * to_f32(cur.u) : 0.f, dus);
                widen<T, NQ>(cur.B, t0 + j < q.slen, Bv);
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < NQ; ++i)
                        hist[j + 1][i][c] =
                            fmaf(__builtin_amdgcn_exp2f(dts[c] * A2[i][c]), hist[j][i][c], dus[c] * Bv[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
            // The walk back reads its inputs anew: held from the walk forward they
            // would take the registers of the states.
            asm volatile("" : "+v"(in.ou), "+v"(in.od), "+v"(in.oB));
            next = in.template read<true, true, true, true>();
            T* du = (T*)p.du + (b0 * p.L + t0 + SCAN_CH - 1) * D;
            T* dde = (T*)p.ddelta + (b0 * p.L + t0 + SCAN_CH - 1) * D;
            float* o = p.dbc + ((((long)cblk * p.B + b0) * p.L + t0 + SCAN_CH - 1) * p.G + g) * 2 * N;
#pragma unroll
            for (int j = SCAN_CH - 1; j >= 0; --j) {
                const int t = t0 + j;
                const bool on = t < q.len;
                const Step<T, NQ> cur = next;
                if (j) {
                    in.back(p, t);
                    next = in.template read<true, true, true, true>();
                }
                const float x = to_f32(cur.de) + dbias;
                const float dt = step_size(p, on, x);
                const float uv = on ? to_f32(cur.u) : 0.f, dyv = on ? to_f32(cur.dy) : 0.f;
                float dts[4], dus[4], dys[4], Bv[NQ], Cv[NQ], bc[2 * NQ] = {}, into[4] = {}, dec[4] = {};
                quad_spread(dt, dts);
                quad_spread(dt * uv, dus);
                quad_spread(dyv, dys);
                widen<T, NQ>(cur.B, t < q.slen, Bv);
                widen<T, NQ>(cur.C, t < q.slen, Cv);
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < NQ; ++i) {
                        const float a = __builtin_amdgcn_exp2f(dts[c] * A2[i][c]);
                        const float back = a * hist[j][i][c];
                        gs[i][c] = fmaf(Cv[i], dys[c], gs[i][c]);
                        bc[i] = fmaf(gs[i][c], dus[c], bc[i]);
                        bc[NQ + i] = fmaf(dys[c], hist[j + 1][i][c], bc[NQ + i]);
                        into[c] = fmaf(gs[i][c], Bv[i], into[c]);
                        const float gb = gs[i][c] * back;
                        dec[c] = fmaf(gb, A2[i][c], dec[c]);
                        dA[i][c] = fmaf(gb, dts[c], dA[i][c]);
                        gs[i][c] *= a;
                    }
                const float in_n = states_sum<KQ>(into, lane);
                float dx = fmaf(uv, in_n, states_sum<KQ>(dec, lane) * LN2);
                if (p.softplus) dx *= fast_sigmoid(x);
                dx = on ? dx : 0.f;
                ddb += dx;
                dskip = fmaf(dyv, uv, dskip);
                reduce_quads<4 * KQ, 2 * NQ>(bc, l.cw * KQ, lane);
                if (t < p.L) {
                    if (q.own) {
                        put(du, in.oy, from_f32<T>(on ? fmaf(skip, dyv, dt * in_n) : 0.f));
                        put(dde, in.oy, from_f32<T>(dx));
                    }
                    if (keeps) put(o, obc, bc[0]);
                    if (left > 1 && keeps2) put(o + 1, obc, bc[1]);
                }
                du -= D;
                dde -= D;
                o -= (long)p.G * 2 * N;
                __builtin_amdgcn_sched_barrier(0);  // one step at a time: no registers for more
            }
        }
        if (p.dh0 && seg == 0) store_states<NQ>(p, q, p.dh0, gs);
    }
    // the wave's sequences share their channels: join them, then one row per slot
    for (int m = l.cw * KQ; m < 64; m <<= 1) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < NQ; ++i) dA[i][c] += __shfl_xor(dA[i][c], m);
        dskip += __shfl_xor(dskip, m);
        ddb += __shfl_xor(ddb, m);
    }
    if (lane < l.cw * KQ) {
        float* ws = p.ws + (long)slot * D * (N + 2);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < NQ; ++i)
                if (q0.state(p, c, i)) ws[(long)(q0.d4 + c) * N + q0.n0 + i] = dA[i][c];
        if (q0.own) {
            ws[(long)D * N + q0.d] = dskip;
            ws[(long)D * N + D + q0.d] = ddb;
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
    if (p.softplus) dt = softplus_s(dt);
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

template <typename F>
void by_states(int N, F f) {
    if (N <= 4) f.template operator()<1, 1>();
    else if (N <= 8) f.template operator()<2, 1>();
    else if (N <= 16) f.template operator()<4, 1>();
    else if (N <= 32) f.template operator()<4, 2>();
    else f.template operator()<4, 4>();
}

template <typename F>
struct Typed {
    F f;
    int is_f32, bvec;
    template <int NQ, int KQ>
    void operator()() const {
        const bool vb = bvec && f.p.N == 4 * NQ * KQ;
        if (is_f32) {
            if (vb) f.template run<float, NQ, KQ, true>();
            else f.template run<float, NQ, KQ, false>();
        } else {
            if (vb) f.template run<__bf16, NQ, KQ, true>();
            else f.template run<__bf16, NQ, KQ, false>();
        }
    }
};

inline dim3 wave_blocks(long waves) { return dim3((unsigned)((waves + 3) / 4)); }

struct ScanFwd {
    const ScanParams& p;
    const ScanPlan& l;
    hipStream_t s;
    template <typename T, int NQ, int KQ, bool VB>
    void run() const {
        const long tasks = l.groups * p.G * l.cb;
        if (l.nseg > 1) {
            hipLaunchKernelGGL((scan_fwd_kernel<T, NQ, KQ, VB, false>), wave_blocks((long)l.fslots * p.G * l.cb), dim3(256),
                               0, s, p, l);
            hipLaunchKernelGGL((scan_carry_kernel<NQ, KQ, false>), wave_blocks(tasks * NQ), dim3(256), 0, s, p, l,
                               tasks * NQ);
        }
        hipLaunchKernelGGL((scan_fwd_kernel<T, NQ, KQ, VB, true>), wave_blocks((long)l.fslots * p.G * l.cb), dim3(256), 0,
                           s, p, l);
    }
};

struct ScanBwd {
    const ScanParams& p;
    const ScanPlan& l;
    hipStream_t s;
    template <typename T, int NQ, int KQ, bool VB>
    void run() const {
        const long tasks = l.groups * p.G * l.cb;
        if (l.nseg > 1) {
            hipLaunchKernelGGL((scan_adjoint_kernel<T, NQ, KQ, VB>), wave_blocks((long)l.fslots * p.G * l.cb), dim3(256), 0, s,
                               p, l);
            hipLaunchKernelGGL((scan_carry_kernel<NQ, KQ, true>), wave_blocks(tasks * NQ), dim3(256), 0, s, p, l,
                               tasks * NQ);
        }
        hipLaunchKernelGGL((scan_bwd_kernel<T, NQ, KQ, VB>), wave_blocks((long)l.slots * p.G * l.cb), dim3(256), 0, s, p,
                           l);
    }
};

}  // namespace

// The lane layout and the cut of the time axis for these sizes and strides.
extern "C" ScanPlan scan_plan(const ScanParams& p, int is_f32) {
    const int kq = p.N <= 16 ? 1 : p.N <= 32 ? 2 : 4, nq = p.N <= 4 ? 1 : p.N <= 8 ? 2 : 4;
    const long es = is_f32 ? 4 : 2, per = p.D / p.G;
    ScanPlan l{};
    // All lanes, or the half of them that leaves the backward's sums over
    // channels one value a lane: two sequences a wave where a group has 32
    // channels or fewer and their lane offsets fit 32 bits.
    l.cw = 64 / kq;
    if (kq == 1 && per <= 32) {
        long far = (long)p.L * p.D, bc = (long)p.L * p.G * 2 * p.N * 4;
        for (long s : {p.u_b, p.d_b, p.B_b, p.C_b}) far = s > far ? s : far;
        if ((far + p.D + 64L) * es <= 0xffffffffL && bc + 1024 <= 0xffffffffL) l.cw = 32;
    }
    l.rw = 64 / (l.cw * kq);
    l.cb = (int)((per + l.cw - 1) / l.cw);
    l.groups = (p.B + l.rw - 1) / l.rw;
    l.chunks = (p.L + SCAN_CH - 1) / SCAN_CH;
    l.state = 64 * 4 * nq;
    // Segments of at least 4 chunks where that brings the waves towards four per
    // SIMD: they cost a second pass over the recurrence, so fewer than 3 do not pay.
    const long tasks = l.groups * p.G * l.cb, same = (long)p.G * l.cb;
    long nseg = tasks ? 4096 / tasks : 1;
    if (nseg > l.chunks / 4) nseg = l.chunks / 4;
    if (nseg < 3) nseg = 1;
    l.seg_chunks = (int)(l.chunks ? (l.chunks + nseg - 1) / nseg : 1);
    l.nseg = l.chunks ? (l.chunks + l.seg_chunks - 1) / l.seg_chunks : 1;
    // Waves that share channels and take their items in turn: four per SIMD in
    // all in the forward, two in the backward (what the registers allow).
    const long items = l.groups * l.nseg;
    const long f = (4096 + same - 1) / same, b = (2048 + same - 1) / same;
    l.fslots = (int)(items < f ? items : f);
    l.slots = (int)(items < b ? items : b);
    return l;
}

extern "C" void scan_fwd_launch(const ScanParams& p, const ScanPlan& l, int is_f32, hipStream_t s) {
    by_states(p.N, Typed<ScanFwd>{ScanFwd{p, l, s}, is_f32, p.bvec});
}

extern "C" void scan_bwd_launch(const ScanParams& p, const ScanPlan& l, int is_f32, hipStream_t s) {
    by_states(p.N, Typed<ScanBwd>{ScanBwd{p, l, s}, is_f32, p.bvec});
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
