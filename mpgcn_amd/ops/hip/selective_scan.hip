// Selective state space scan (gfx950). Per sequence b and channel d, with N
// states and the per-token B, C shared by the D/G channels of a group:
//   dt_t = softplus(delta_t + dbias)
//   h_t[n] = exp(dt_t A[n]) h_{t-1}[n] + dt_t u_t B_t[n]
//   y_t    = sum_n C_t[n] h_t[n] + skip u_t
//
// States, sums and step sizes are f32 throughout; only what is stored as bf16
// is rounded. Bound by vector arithmetic: an exp (two issue slots) and four
// more operations per state and step against 6 bytes per channel and step.
// With 16 states, bf16: 16384 x 2048 in 263 us (a state pass and the main one),
// forward and backward of 262144 x 7 x 32 in 1155 us: the vector pipes are busy
// throughout the one and for 93 % of the other.
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
#include <cfloat>

#include "seq.hpp"

#define SCAN_CH 8  // steps of a chunk: staged together, their states held by the backward

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

// Lane l of a quad holds its channels in the order l, l^1, l^2, l^3: then what a
// lane has for another's channel stands at the same index as in that lane what
// it has for this one's, and the exchanges need no selects.

// Each lane's channel summed over the quad.
__device__ __forceinline__ float quad_sum(const float (&v)[4]) {
    return (v[0] + dpp<0xB1>(v[1])) + (dpp<0x4E>(v[2]) + dpp<0x1B>(v[3]));
}

template <int KQ>
__device__ __forceinline__ float states_sum(const float (&v)[4]) {
    float s = quad_sum(v);
    if constexpr (KQ >= 2) s += from_xor<4>(s);
    if constexpr (KQ >= 4) s += from_xor<8>(s);
    return s;
}

// The quad's values of v in a lane's order.
__device__ __forceinline__ void quad_spread(float v, float (&o)[4]) {
    o[0] = v;
    o[1] = dpp<0xB1>(v);
    o[2] = dpp<0x4E>(v);
    o[3] = dpp<0x1B>(v);
}

// Sum V values over the quads of a sequence: lane bits from below `span` down to
// M0. While a lane carries more than one value each step halves them; the high
// bits go first, whose exchange needs no selects.
template <int M, int M0, int LEFT, int V>
__device__ __forceinline__ void reduce_quads(float (&v)[V], int span, int lane) {
    if constexpr (M >= M0) {
        constexpr int NEXT = LEFT > 1 ? LEFT / 2 : 1;
        if (M < span) {
#pragma unroll
            for (int i = 0; i < NEXT; ++i) v[i] = fold<M>(v[i], v[LEFT > 1 ? i + NEXT : i], lane);
            reduce_quads<M / 2, M0, NEXT>(v, span, lane);
        } else {
            reduce_quads<M / 2, M0, LEFT>(v, span, lane);
        }
    }
}

// Where that leaves a lane: `left` values from number `idx`; lanes that differ
// in the bits of `dup` hold the same.
template <int V, int M0>
__device__ __forceinline__ void reduced_place(int span, int lane, int& idx, int& dup, int& left) {
    idx = 0; dup = 0; left = V;
    for (int m = span / 2; m >= M0; m >>= 1) {
        if (left > 1) {
            left >>= 1;
            idx += (lane & m) ? left : 0;
        } else {
            dup |= m;
        }
    }
}

// ---- a lane's place ---------------------------------------------------------

// Where a lane stands in its wave: its sequence, the channel it loads and
// stores, the four channels and NQ states it computes.
template <int NQ, int KQ>
struct Place {
    static constexpr int CH = 64 / KQ;       // channels of a wave, over its sequences
    static constexpr int NP = 4 * NQ * KQ;   // states, padded
    int rs, col, d, n0, d4, nd, sub;
    bool okc;

    __device__ __forceinline__ Place(const ScanParams& p, const ScanPlan& l, int lane, int g, int cblk) {
        const int per = p.D / p.G;
        const int quad = (lane / (4 * KQ)) & (l.cw / 4 - 1);
        const int kq = (lane >> 2) & (KQ - 1);
        rs = lane / (l.cw * KQ);
        const int c4 = cblk * l.cw + quad * 4, c = c4 + (lane & 3);
        col = rs * l.cw + quad * 4 + (lane & 3);
        sub = lane & 3;
        nd = per - c4 < 0 ? 0 : per - c4 > 4 ? 4 : per - c4;
        okc = c < per;
        d = g * per + (okc ? c : 0);
        d4 = g * per + (nd ? c4 : 0);
        n0 = (kq * 4 + (lane & 3)) * NQ;
    }
    // the channel at index c, and whether there are it and its state i
    __device__ __forceinline__ int ch(int c) const { return d4 + (c ^ sub); }
    __device__ __forceinline__ bool state(const ScanParams& p, int c, int i) const { return (c ^ sub) < nd && n0 + i < p.N; }
};

// log(1 + e^x) and its slope. e^-|x| with the rounding of the argument's product
// put right, the logarithm of 1 + e with that sum's: within 4 + |x| / 4 times
// 2^-24 of the result, where the second part is log2(e)'s own rounding and
// counts for x < 0 alone. Past the exponent's range the remainder is infinite or
// NaN and e is 0: the bound keeps their product 0.
__device__ __forceinline__ float softplus_s(float x, float& slope) {
    const float a = -fabsf(x), hi = a * LOG2E, lo = fminf(fmaf(a, LOG2E, -hi), 1.f);
    float e = __builtin_amdgcn_exp2f(hi);
    e = fmaf(e * lo, LN2, e);
    const float s = 1.f + e, r = __builtin_amdgcn_rcpf(s);
    slope = x < 0.f ? e * r : r;
    return fmaxf(x, 0.f) + fmaf(__builtin_amdgcn_logf(s), LN2, e - (s - 1.f));
}

// the step size, 0 past the sequence's end, and its slope in delta
__device__ __forceinline__ float step_size(bool softplus, bool on, float x, float& slope) {
    float s = softplus_s(x, slope);
    asm volatile("" : "+v"(s));  // no branch around it: the steps stay one block
    s = softplus ? s : x;
    slope = softplus ? slope : 1.f;
    return on ? s : 0.f;
}

// s[i] where ok, else 0: read without a branch
__device__ __forceinline__ float pick(const float* __restrict__ s, bool ok, long i) {
    const float v = ((gmem<const float>)s)[ok ? i : 0];
    return ok ? v : 0.f;
}

// The decay of a state that there is not. Its state is zero as long as its
// inputs' product with zero is: this keeps exp(dt A) finite up to an infinite
// step, where that of 0 would be NaN, and 1 for every finite one.
constexpr float NO_DECAY = -2 * FLT_MIN;  // half of it is a number, too

// log2(e) times the decay of state n0 + i of the lane's channel at index c
template <int NQ, int KQ>
__device__ __forceinline__ float decay(const ScanParams& p, const Place<NQ, KQ>& q, int c, int i) {
    const bool ok = q.state(p, c, i);
    const float v = pick(p.A, ok, (long)q.ch(c) * p.N + q.n0 + i) * LOG2E;
    return ok ? v : NO_DECAY;
}

template <int NQ, int KQ>
__device__ __forceinline__ void load_decay(const ScanParams& p, const Place<NQ, KQ>& q, f32x4 (&A2)[NQ]) {
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < NQ; ++i)
            A2[i][c] = decay(p, q, c, i);
}

// The lane's states in a (B, D, N) tensor, or zeros, for a wave whose first
// sequence is b0.
template <int NQ, int KQ>
__device__ __forceinline__ void load_states(const ScanParams& p, const Place<NQ, KQ>& q, const float* s, long b0,
                                            f32x4 (&h)[NQ]) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) h[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (!s) return;
    const long b = b0 + q.rs;
    // addresses and masks are formed here, not kept over the loop around
    int d4 = q.d4, nd = q.nd, n0 = q.n0, sub = q.sub;
    asm volatile("" : "+v"(d4), "+v"(nd), "+v"(n0), "+v"(sub));
    nd = b < p.B ? nd : 0;
    if (NQ == 4 && p.N == Place<NQ, KQ>::NP && p.D / p.G % 4 == 0) {
        // Unmasked, so that nothing waits for the loads here. All four channels
        // are there or none, and those that are not read the first sequence's of
        // the wave: states that meet only zeros and are not stored.
        s += ((b < p.B ? b : b0) * p.D + d4) * p.N + n0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const i32x4 v = *(gmem<const any16>)(s + (long)(c ^ sub) * p.N);
#pragma unroll
            for (int i = 0; i < NQ; ++i) h[i][c] = __int_as_float(v[i & 3]);
        }
    } else if (NQ == 4) {
        s += b < p.B ? (b * p.D + d4) * p.N + (n0 < p.N ? n0 : 0) : 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            Pack<float> v;
            v.load(s + (long)(c ^ sub) * p.N, (c ^ sub) < nd ? p.N - n0 : 0, p.N % 4);
#pragma unroll
            for (int i = 0; i < NQ; ++i) h[i][c] = v.get(i & 3);
        }
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < NQ; ++i) h[i][c] = pick(s, (c ^ sub) < nd && n0 + i < p.N, (b * p.D + d4 + (c ^ sub)) * p.N + n0 + i);
    }
}
template <int NQ, int KQ>
__device__ __forceinline__ void store_states(const ScanParams& p, const Place<NQ, KQ>& q, float* s, long b0,
                                             const f32x4 (&h)[NQ]) {
    const long b = b0 + q.rs;
    int d4 = q.d4, nd = q.nd, n0 = q.n0, sub = q.sub;
    asm volatile("" : "+v"(d4), "+v"(nd), "+v"(n0), "+v"(sub));
    if (b >= p.B) return;
    s += (b * p.D + d4) * p.N + n0;
    if (NQ == 4) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            Pack<float> v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v.w[i] = __float_as_int(h[i & (NQ - 1)][c]);
            v.store(s + (long)(c ^ sub) * p.N, (c ^ sub) < nd ? p.N - n0 : 0, p.N % 4);
        }
    } else {
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < NQ; ++i)
                if ((c ^ sub) < nd && n0 + i < p.N) ((gmem<float>)s)[(long)(c ^ sub) * p.N + i] = h[i][c];
    }
}
// the same in the order of a wave's lanes: 16 bytes a lane, NQ rows of them
template <int NQ>
__device__ __forceinline__ void load_lanes(const float* s, long slot, int lane, f32x4 (&h)[NQ]) {
    const auto v = (gmem<const f32x4>)s + slot * NQ * 64 + lane;
#pragma unroll
    for (int i = 0; i < NQ; ++i) h[i] = v[i * 64];
}
template <int NQ>
__device__ __forceinline__ void store_lanes(float* s, long slot, int lane, const f32x4 (&h)[NQ]) {
    const auto v = (gmem<f32x4>)s + slot * NQ * 64 + lane;
#pragma unroll
    for (int i = 0; i < NQ; ++i) v[i * 64] = h[i];
}

struct ScanArgs {
    ScanParams p;
    ScanPlan l;
};

// The kernel's arguments read anew from where the launch put them: kept over
// the loops they would not fit the scalar registers.
__device__ __forceinline__ ScanArgs args() {
    auto k = (const __attribute__((address_space(4))) int*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(k));
    int w[sizeof(ScanArgs) / 4];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(ScanArgs) / 4); ++i) w[i] = k[i];
    ScanArgs a;
    __builtin_memcpy(&a, w, sizeof(a));
    return a;
}

// The lane, so that what follows from it is worked out where it is used and
// not kept over the loops.
__device__ __forceinline__ int fresh_lane() {
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));
    return lane;
}

__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

// ---- a chunk's inputs, by way of LDS ----------------------------------------
//
// A wave reads a chunk of 8 steps in 16-byte pieces, one or two a lane and
// tensor, into registers while it works on the chunk before, and puts them into
// LDS of its own when it gets there. B and C are widened to f32 on the way;
// what is past a sequence's end goes in as zeros, whatever it holds. Outputs
// take the same way back over the inputs' place. LDS operations of one wave
// run in order, so no barrier is needed, only that the compiler keeps them so.

template <typename T, int NQ, int KQ>
struct Tile {
    static constexpr int CH = 64 / KQ, NP = 4 * NQ * KQ, RW = KQ == 1 ? 2 : 1;
    T u[SCAN_CH][CH], de[SCAN_CH][CH];
    float bc[SCAN_CH][RW][2][NP];
};
template <typename T, int NQ, int KQ>
struct TileBack : Tile<T, NQ, KQ> {
    using B = Tile<T, NQ, KQ>;
    T dy[SCAN_CH][B::CH];
    float step[SCAN_CH][64][2];  // step size and its slope
    float dbc[B::RW][SCAN_CH][2][B::NP];
    f32x4 A2[NQ][64];            // the decays of the lanes, out of their registers
};

__device__ __forceinline__ void lds_order() {
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// One (8 steps) x (the wave's channels) tensor.
template <typename T, int KQ>
struct Rows {
    static constexpr int CH = 64 / KQ, E = Pack<T>::E, PR = CH / E, P = SCAN_CH * PR;
    static constexpr int K = (P + 63) / 64;  // pieces a lane
    struct Raw { Pack<T> v[K]; };

    // piece k of the lane: its step, sequence, first channel of the tensor, elements there
    static __device__ __forceinline__ void piece(const ScanParams& p, const ScanPlan& l, int lane, int g, int cblk, int k,
                                                 int& row, int& rs, int& d, int& n) {
        const int i = k * 64 + lane;
        row = i / PR;
        const int col = i % PR * E;
        rs = col >= l.cw ? 1 : 0;
        const int per = p.D / p.G, c = cblk * l.cw + col - rs * l.cw;
        n = (P % 64 == 0 || i < P) && c < per ? per - c : 0;
        d = g * per + (n ? c : 0);
    }
    // base: the wave's first sequence at the chunk's first step; last: the last step there is from it
    static __device__ __forceinline__ void read(const ScanParams& p, const ScanPlan& l, int lane, int g, int cblk,
                                                const T* base, long b_stride, int t_stride, int last, bool two, Raw& r) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            int row, rs, d, n;
            piece(p, l, lane, g, cblk, k, row, rs, d, n);
            row = row < last ? row : last;
            const unsigned off =
                ((rs && two ? (unsigned)b_stride : 0u) + (unsigned)row * (unsigned)t_stride + (unsigned)d) * (unsigned)sizeof(T);
            r.v[k].load((const T*)((const char*)base + off), n, p.D / p.G % E);
        }
    }
    static __device__ __forceinline__ void stage(int cw, int lane, const Raw& r, int live0, int live1, T (*tile)[CH]) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = k * 64 + lane, row = i / PR;
            const bool on = row < (i % PR * E >= cw ? live1 : live0);
            i32x4 c;
#pragma unroll
            for (int j = 0; j < 4; ++j) c[j] = on ? r.v[k].w[j] : 0;
            if (P % 64 == 0 || i < P) *(i32x4*)((T*)tile + i * E) = c;
        }
    }
    // back out: rows below `rows`, of a contiguous (B, L, D) tensor
    static __device__ __forceinline__ void write(const ScanParams& p, const ScanPlan& l, int lane, int g, int cblk, T* base,
                                                 int rows, bool two, const T (*tile)[CH]) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            int row, rs, d, n;
            piece(p, l, lane, g, cblk, k, row, rs, d, n);
            if (n == 0 || row >= rows || (rs && !two)) continue;
            const i32x4 c = *(const i32x4*)((const T*)tile + (k * 64 + lane) * E);
            const Pack<T> v{c};
            v.store(base + ((rs ? (long)p.L : 0) + row) * p.D + d, n, p.D / p.G % E);
        }
    }
};

// The chunk's rows of B or of C, to f32.
template <typename T, int NQ, int KQ>
struct States {
    static constexpr int NP = 4 * NQ * KQ, RW = KQ == 1 ? 2 : 1;
    static constexpr int E = NP * sizeof(T) < 16 ? NP : 16 / sizeof(T), PR = NP / E, P = SCAN_CH * RW * PR;
    static constexpr int K = (P + 63) / 64;
    struct Raw { Pack<T, E> v[K]; };

    static __device__ __forceinline__ void read(const ScanParams& p, int lane, const T* base, long b_stride, int t_stride,
                                                int last, bool two, Raw& r) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = k * 64 + lane, e0 = i % PR * E;
            const int rs = RW == 2 && two ? i / PR % RW : 0;
            int row = i / (PR * RW);
            row = row < last ? row : last;
            const int n = p.N > e0 ? p.N - e0 : 0;
            const unsigned off = ((rs ? (unsigned)b_stride : 0u) + (unsigned)row * (unsigned)t_stride +
                                  (unsigned)(n ? e0 : 0)) * (unsigned)sizeof(T);
            r.v[k].load((const T*)((const char*)base + off), n, p.N % E);
        }
    }
    static __device__ __forceinline__ void stage(int lane, const Raw& r, int which, int live0, int live1,
                                                 float (*tile)[RW][2][NP]) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int i = k * 64 + lane, e0 = i % PR * E, rs = i / PR % RW, row = i / (PR * RW);
            const bool on = row < (rs ? live1 : live0);
            if (P % 64 == 0 || i < P) {
#pragma unroll
                for (int e = 0; e < E; e += 4) {
                    f32x4 v;
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[j] = on ? r.v[k].get(e + j) : 0.f;
                    *(f32x4*)&tile[row][rs][which][e0 + e] = v;
                }
            }
        }
    }
};

// What a wave works on: its channels, and one item after another of sequences
// and a segment of their time. Uniform.
struct Work {
    int cblk, g, slot;
    __device__ __forceinline__ explicit Work(const ScanArgs& a) {
        const int w = blockIdx.x * 4 + wave_id();
        cblk = w % a.l.cb;
        g = w / a.l.cb % a.p.G;
        slot = w / a.l.cb / a.p.G;
    }
};
struct Item {
    int seg, c0, c1;  // its chunks
    long b0, id;      // first sequence, task
    int len0, len1;   // valid lengths of the sequences; 0 for one that there is not
    bool two;

    // nseg segments from number `from` on
    __device__ __forceinline__ Item(const ScanArgs& a, const Work& w, int it, int nseg, int from) {
        const int grp = nseg == 1 ? it : it / nseg;
        seg = from + (nseg == 1 ? 0 : it - grp * nseg);
        b0 = (long)grp * a.l.rw;
        id = (long)(grp * a.p.G + w.g) * a.l.cb + w.cblk;
        c0 = seg * a.l.seg_chunks;
        c1 = c0 + a.l.seg_chunks < a.l.chunks ? c0 + a.l.seg_chunks : a.l.chunks;
        two = a.l.rw == 2 && b0 + 1 < a.p.B;
        len0 = seq_len(a.p.lens, a.p.lens64, (int)b0, a.p.L);
        len1 = two ? seq_len(a.p.lens, a.p.lens64, (int)b0 + 1, a.p.L) : 0;
    }
};

// A chunk's inputs on their way: of u, delta, dy, B and C those asked for.
// LEAN: lane offsets are worked out anew for every chunk.
template <typename T, int NQ, int KQ, bool LEAN, bool U, bool DY, bool B, bool C>
struct Inputs {
    using RowsT = Rows<T, KQ>;
    using StatesT = States<T, NQ, KQ>;
    typename RowsT::Raw u, de, dy;
    typename StatesT::Raw Br, Cr;

    __device__ __forceinline__ void read(const Work& w, const Item& m, int ck) {
        const ScanArgs a = args();
        const ScanParams& p = a.p;
        const int lane = LEAN ? fresh_lane() : threadIdx.x & 63;
        const long t0 = (long)ck * SCAN_CH;
        const int last = (int)(p.L - 1 - t0);
        if (U)
            RowsT::read(p, a.l, lane, w.g, w.cblk, (const T*)p.u + m.b0 * p.u_b + t0 * p.u_t, p.u_b, p.u_t, last, m.two, u);
        RowsT::read(p, a.l, lane, w.g, w.cblk, (const T*)p.delta + m.b0 * p.d_b + t0 * p.d_t, p.d_b, p.d_t, last, m.two, de);
        if (DY)
            RowsT::read(p, a.l, lane, w.g, w.cblk, (const T*)p.dy + (m.b0 * p.L + t0) * p.D, (long)p.L * p.D, p.D, last,
                        m.two, dy);
        if (B)
            StatesT::read(p, lane, (const T*)p.Bm + m.b0 * p.B_b + w.g * p.B_g + t0 * p.B_t, p.B_b, p.B_t, last, m.two, Br);
        if (C)
            StatesT::read(p, lane, (const T*)p.Cm + m.b0 * p.C_b + w.g * p.C_g + t0 * p.C_t, p.C_b, p.C_t, last, m.two, Cr);
    }
    // dyt: where dy goes
    template <typename Tl>
    __device__ __forceinline__ void stage(const Item& m, int ck, int cw, Tl& tile, T (*dyt)[RowsT::CH]) {
        const int lane = LEAN ? fresh_lane() : threadIdx.x & 63, t0 = ck * SCAN_CH;
        lds_order();
        if (U) RowsT::stage(cw, lane, u, m.len0 - t0, m.len1 - t0, tile.u);
        RowsT::stage(cw, lane, de, m.len0 - t0, m.len1 - t0, tile.de);
        if (DY) RowsT::stage(cw, lane, dy, m.len0 - t0, m.len1 - t0, dyt);
        if (B) StatesT::stage(lane, Br, 0, m.len0 - t0, m.len1 - t0, tile.bc);
        if (C) StatesT::stage(lane, Cr, 1, m.len0 - t0, m.len1 - t0, tile.bc);
        lds_order();
    }
};

// ---- forward ----------------------------------------------------------------

// MAIN: outputs, chunk states, final state. Otherwise the end state of a
// segment from zero and its summed step size.
template <typename T, int NQ, int KQ, bool MAIN>
__launch_bounds__(256) __global__ void scan_fwd_kernel(ScanArgs) {
    __shared__ Tile<T, NQ, KQ> tiles[4];
    Tile<T, NQ, KQ>& tile = tiles[wave_id()];
    const int lane = threadIdx.x & 63;
    f32x4 A2[NQ];
    float skip, dbias;
    int items, nseg, step, L, cw;
    bool softplus, keep;
    const ScanArgs a0 = args();
    const Work w(a0);
    const Place<NQ, KQ> q(a0.p, a0.l, lane, w.g, w.cblk);
    {
        nseg = MAIN ? a0.l.nseg : a0.l.nseg - 1;  // the last segment's end is no start
        items = (int)(a0.l.groups * nseg);
        step = a0.l.fslots;
        if (w.slot >= step || w.slot >= items) return;
        L = a0.p.L;
        cw = a0.l.cw;
        softplus = a0.p.softplus;
        keep = MAIN && a0.p.ckpt;
        load_decay(a0.p, q, A2);
        skip = a0.p.skip ? ((gmem<const float>)a0.p.skip)[q.d] : 0.f;
        dbias = a0.p.dbias ? ((gmem<const float>)a0.p.dbias)[q.d] : 0.f;
    }
    Inputs<T, NQ, KQ, false, true, false, true, MAIN> in;
    Item m(a0, w, w.slot, nseg, 0);
    if (m.c0 < m.c1) in.read(w, m, m.c0);
    for (int it = w.slot; it < items; it += step) {
        const int len = q.okc ? (q.rs ? m.len1 : m.len0) : 0;
        f32x4 h[NQ];
        {
            const ScanArgs a = args();
            if (MAIN && nseg > 1) load_lanes<NQ>(a.p.seg_h, m.id * nseg + m.seg, lane, h);
            else load_states(a.p, q, MAIN ? a.p.h0 : nullptr, m.b0, h);
        }
        float total = 0.f;
        for (int ck = m.c0; ck < m.c1; ++ck) {
            const int t0 = ck * SCAN_CH;
            in.stage(m, ck, cw, tile, tile.u);
            if (ck + 1 < m.c1) in.read(w, m, ck + 1);
            else if (it + step < items) {
                const Item n(args(), w, it + step, nseg, 0);
                in.read(w, n, n.c0);
            }
            if (keep) {
                const ScanArgs a = args();
                store_lanes<NQ>(a.p.ckpt, m.id * a.l.chunks + ck, lane, h);
            }
#pragma unroll
            for (int j = 0; j < SCAN_CH; ++j) {
                if ((j == 1 || j == 4) && t0 + j >= L) break;  // at every step the steps would not overlap
                const bool on = t0 + j < len;
                const float uv = to_f32(tile.u[j][q.col]);
                float slope, dts[4], dus[4], acc[4] = {};
                const float dt = step_size(softplus, on, to_f32(tile.de[j][q.col]) + dbias, slope);
                quad_spread(dt, dts);
                quad_spread(dt * uv, dus);
                if (!MAIN) total += dt;
                const float* Bv = &tile.bc[j][q.rs][0][q.n0];
                const float* Cv = &tile.bc[j][q.rs][1][q.n0];
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    const float Bi = Bv[i], Ci = MAIN ? Cv[i] : 0.f;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        h[i][c] = fmaf(__builtin_amdgcn_exp2f(dts[c] * A2[i][c]), h[i][c], dus[c] * Bi);
                        if (MAIN) acc[c] = fmaf(Ci, h[i][c], acc[c]);
                    }
                }
                if (MAIN) {
                    const float s = states_sum<KQ>(acc);
                    tile.u[j][q.col] = from_f32<T>(on ? fmaf(skip, uv, s) : 0.f);
                }
            }
            if (MAIN) {
                const ScanArgs a = args();
                lds_order();
                Rows<T, KQ>::write(a.p, a.l, lane, w.g, w.cblk, (T*)a.p.y + (m.b0 * L + t0) * a.p.D, L - t0,
                                      m.two, tile.u);
            }
        }
        const ScanArgs a = args();
        if (!MAIN) {
            store_lanes<NQ>(a.p.seg_h, m.id * a.l.nseg + m.seg, lane, h);
            ((gmem<float>)a.p.seg_s)[(m.id * a.l.nseg + m.seg) * 64 + lane] = total;
        } else if (a.p.h1 && m.seg == a.l.nseg - 1) {
            store_states(a.p, q, a.p.h1, m.b0, h);
        }
        if (it + step < items) m = Item(a, w, it + step, nseg, 0);
    }
}

// A state behind steps of size dt in all, with what they add on their way; A2h
// is half of the decay. It goes on in two halves: between them the value lies
// between the old and the new, so only one out of range itself leaves it. The
// bound keeps a state of zero at zero where steps grow past the range. (Where a
// step's decay is NaN, what it adds is.)
__device__ __forceinline__ float carried(float state, float dt, float A2h, float added) {
    const float half = fminf(__builtin_amdgcn_exp2f(dt * A2h), FLT_MAX);
    return fmaf(state * half, half, added);
}

// Turns each segment's own end state into the state it starts from (forward),
// or its own adjoint at the start into the one at its end (backward). A block
// takes four states of a task's lanes; its waves share the segments: each runs
// through its part from zero, the parts are joined in LDS, and each runs
// through again from where the parts before it end. The loads of 16 segments
// are in flight together.
template <int NQ, int KQ, bool BACK>
__launch_bounds__(1024) __global__ void scan_carry_kernel(ScanParams p, ScanPlan l) {
    __shared__ f32x4 end[16][64];
    __shared__ float sums[16][64];
    const int lane = threadIdx.x & 63, wave = wave_id(), waves = blockDim.x / 64;
    const int i = (int)(blockIdx.x % NQ);
    const long id = blockIdx.x / NQ;
    const Place<NQ, KQ> q(p, l, lane, (int)(id / l.cb % p.G), (int)(id % l.cb));
    const long b = id / l.cb / p.G * l.rw + q.rs;
    const float* first = BACK ? p.dh1 : p.h0;
    f32x4 A2h, carry = {0.f, 0.f, 0.f, 0.f}, start;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const bool on = q.state(p, c, i);
        A2h[c] = 0.5f * decay(p, q, c, i);
        start[c] = first ? pick(first, on && b < p.B, (b * p.D + q.ch(c)) * p.N + q.n0 + i) : 0.f;
    }
    f32x4* seg_h = (f32x4*)p.seg_h + (id * l.nseg * NQ + i) * 64 + lane;
    const float* seg_s = p.seg_s + id * l.nseg * 64 + lane;
    const int part = (l.nseg + waves - 1) / waves, s_lo = wave * part;
    const int s_hi = s_lo + part < l.nseg ? s_lo + part : l.nseg;
    constexpr int U = 16;
    auto run = [&](bool out, float& total) {
        for (int s0 = s_lo; s0 < s_hi; s0 += U) {
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
                const bool on = s < s_hi;
                const long at = BACK ? l.nseg - 1 - s : s;
                if (out && on) seg_h[at * NQ * 64] = carry;
                float ss[4];
                const float sj = on ? sum[j] : 0.f;
                quad_spread(sj, ss);
                total += sj;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    carry[c] = carried(carry[c], ss[c], A2h[c], on ? own[j][c] : 0.f);
            }
        }
    };
    float total = 0.f;
    if (waves > 1) {
        run(false, total);
        end[wave][lane] = carry;
        sums[wave][lane] = total;
        __syncthreads();
        carry = start;
        for (int v = 0; v < wave; ++v) {
            float ss[4];
            quad_spread(sums[v][lane], ss);
#pragma unroll
            for (int c = 0; c < 4; ++c) carry[c] = carried(carry[c], ss[c], A2h[c], end[v][lane][c]);
        }
    } else {
        carry = start;
    }
    run(true, total);
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
template <typename T, int NQ, int KQ>
__launch_bounds__(256) __global__ void scan_adjoint_kernel(ScanArgs) {
    __shared__ Tile<T, NQ, KQ> tiles[4];
    Tile<T, NQ, KQ>& tile = tiles[wave_id()];
    const int lane = threadIdx.x & 63;
    const ScanArgs a0 = args();
    const Work w(a0);
    const Place<NQ, KQ> q(a0.p, a0.l, lane, w.g, w.cblk);
    const int nseg = a0.l.nseg - 1, items = (int)(a0.l.groups * nseg), step = a0.l.fslots, cw = a0.l.cw;
    const bool softplus = a0.p.softplus;
    if (w.slot >= step || w.slot >= items) return;
    f32x4 A2[NQ];
    load_decay(a0.p, q, A2);
    const float dbias = a0.p.dbias ? ((gmem<const float>)a0.p.dbias)[q.d] : 0.f;

    Inputs<T, NQ, KQ, false, false, true, false, true> in;
    Item m(a0, w, w.slot, nseg, 1);
    in.read(w, m, m.c1 - 1);
    for (int it = w.slot; it < items; it += step) {
        const int len = q.okc ? (q.rs ? m.len1 : m.len0) : 0;
        f32x4 gs[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i) gs[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        float total = 0.f;
        for (int ck = m.c1 - 1; ck >= m.c0; --ck) {
            const int t0 = ck * SCAN_CH;
            in.stage(m, ck, cw, tile, tile.u);
            if (ck > m.c0) in.read(w, m, ck - 1);
            else if (it + step < items) {
                const Item n(args(), w, it + step, nseg, 1);
                in.read(w, n, n.c1 - 1);
            }
#pragma unroll
            for (int j = SCAN_CH - 1; j >= 0; --j) {
                float slope, dts[4], dys[4];
                const float dt = step_size(softplus, t0 + j < len, to_f32(tile.de[j][q.col]) + dbias, slope);
                quad_spread(dt, dts);
                quad_spread(to_f32(tile.u[j][q.col]), dys);
                total += dt;
                const float* Cv = &tile.bc[j][q.rs][1][q.n0];
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    const float Ci = Cv[i];
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        gs[i][c] = fmaf(Ci, dys[c], gs[i][c]) * __builtin_amdgcn_exp2f(dts[c] * A2[i][c]);
                }
            }
        }
        const ScanArgs a = args();
        store_lanes<NQ>(a.p.seg_h, m.id * a.l.nseg + m.seg, lane, gs);
        ((gmem<float>)a.p.seg_s)[(m.id * a.l.nseg + m.seg) * 64 + lane] = total;
        if (it + step < items) m = Item(a, w, it + step, nseg, 1);
    }
}

// A chunk's dB and dC where one channel block has all of their terms.
template <typename T, int NQ, int KQ>
__device__ __forceinline__ void write_bc(const ScanParams& p, int lane, int g, long b0, int t0, bool two,
                                         const TileBack<T, NQ, KQ>& tile) {
    using TileT = typename TileBack<T, NQ, KQ>::B;
    constexpr int NP = TileT::NP, PR = NP / 4, P = TileT::RW * SCAN_CH * 2 * PR;  // four states a piece
#pragma unroll
    for (int k = 0; k < (P + 63) / 64; ++k) {
        const int i = k * 64 + lane;
        const int n0 = i % PR * 4, which = i / PR % 2, j = i / (PR * 2) % SCAN_CH, rs = i / (PR * 2 * SCAN_CH);
        if ((P % 64 && i >= P) || t0 + j >= p.L || (rs && !two)) continue;
        const f32x4 v = ((const f32x4*)tile.dbc)[i];
        const float f[4] = {v[0], v[1], v[2], v[3]};
        Pack<T, 4> o;
        o.set(f);
        o.store((T*)(which ? p.dC : p.dB) + (((b0 + rs) * p.L + t0 + j) * p.G + g) * p.N + (n0 < p.N ? n0 : 0),
                n0 < p.N ? p.N - n0 : 0, p.N % 4);
    }
}

template <typename T, int NQ, int KQ>
__launch_bounds__(256, 2) __global__ void scan_bwd_kernel(ScanArgs) {
    using RowsT = Rows<T, KQ>;
    using TileT = TileBack<T, NQ, KQ>;
    constexpr int NP = TileT::B::NP;
    __shared__ TileT tiles[4];
    TileT& tile = tiles[wave_id()];
    const int lane = threadIdx.x & 63;
    const ScanArgs a0 = args();
    const Work w(a0);
    const Place<NQ, KQ> q(a0.p, a0.l, lane, w.g, w.cblk);
    const int items = (int)(a0.l.groups * a0.l.nseg), nseg = a0.l.nseg, step = a0.l.slots, L = a0.p.L, cw = a0.l.cw;
    const bool softplus = a0.p.softplus;
    if (w.slot >= step) return;

    f32x4 dA[NQ];
    float dskip = 0.f, ddb = 0.f;
    {
        f32x4 A2[NQ];
        load_decay(a0.p, q, A2);
#pragma unroll
        for (int i = 0; i < NQ; ++i) tile.A2[i][lane] = A2[i];
    }
#pragma unroll
    for (int i = 0; i < NQ; ++i) dA[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float skip = a0.p.skip ? ((gmem<const float>)a0.p.skip)[q.d] : 0.f;
    const float dbias = a0.p.dbias ? ((gmem<const float>)a0.p.dbias)[q.d] : 0.f;
    int idx, dup, keeps;  // where the sums over channels end up: one value a lane, or two
    reduced_place<2 * NQ, 4 * KQ>(cw * KQ, lane, idx, dup, keeps);
    const int obc = q.rs * (SCAN_CH * 2 * NP) + (idx >= NQ ? NP : 0) + q.n0 + (idx & (NQ - 1));

    // what the next chunk starts from: its inputs and the state before it
    Inputs<T, NQ, KQ, true, true, true, true, true> in;
    f32x4 next_h[NQ];
    auto read_h = [&](const Item& m, int ck) {
        const ScanArgs a = args();
        if (a.p.ckpt) load_lanes<NQ>(a.p.ckpt, m.id * a.l.chunks + ck, lane, next_h);
        else load_states(a.p, q, a.p.h0, m.b0, next_h);
    };
    Item m(a0, w, w.slot, nseg, 0);
    if (m.c0 < m.c1) {
        in.read(w, m, m.c1 - 1);
        read_h(m, m.c1 - 1);
    }
    for (int it = w.slot; it < items; it += step) {
        const int len = q.okc ? (q.rs ? m.len1 : m.len0) : 0;
        f32x4 gs[NQ];  // needed only after the first chunk's walk forward
        {
            const ScanArgs a = args();
            if (nseg > 1) load_lanes<NQ>(a.p.seg_h, m.id * nseg + m.seg, lane, gs);
            else load_states(a.p, q, a.p.dh1, m.b0, gs);
        }
        for (int ck = m.c1 - 1; ck >= m.c0; --ck) {
            const int t0 = ck * SCAN_CH;
            f32x4 hist[SCAN_CH][NQ];  // before every step; the state after it follows from its decay again
#pragma unroll
            for (int i = 0; i < NQ; ++i) hist[0][i] = next_h[i];
            in.stage(m, ck, cw, tile, tile.dy);
#pragma unroll
            for (int j = 0; j < SCAN_CH; ++j) {
                float slope, dts[4], dus[4];
                const float dt = step_size(softplus, t0 + j < len, to_f32(tile.de[j][q.col]) + dbias, slope);
                tile.step[j][lane][0] = dt;
                tile.step[j][lane][1] = slope;
                if (j + 1 == SCAN_CH) continue;
                quad_spread(dt, dts);
                quad_spread(dt * to_f32(tile.u[j][q.col]), dus);
                const float* Bv = &tile.bc[j][q.rs][0][q.n0];
                const int ln = fresh_lane();
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    const float Bi = Bv[i];
                    const f32x4 A2 = tile.A2[i][ln];
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        hist[(j + 1) % SCAN_CH][i][c] =
                            fmaf(__builtin_amdgcn_exp2f(dts[c] * A2[c]), hist[j][i][c], dus[c] * Bi);
                }
                __builtin_amdgcn_sched_barrier(260);  // one step at a time: no registers for more
            }
            lds_order();
#pragma unroll
            for (int j = SCAN_CH - 1; j >= 0; --j) {
                if (t0 + j >= L) continue;
                const bool on = t0 + j < len;
                const float dt = tile.step[j][lane][0], slope = tile.step[j][lane][1];
                const float uv = to_f32(tile.u[j][q.col]), dyv = to_f32(tile.dy[j][q.col]);
                float dts[4], dus[4], dys[4], bc[2 * NQ] = {}, into[4] = {}, dec[4] = {};
                quad_spread(dt, dts);
                quad_spread(dt * uv, dus);
                quad_spread(dyv, dys);
                const float* Bv = &tile.bc[j][q.rs][0][q.n0];
                const float* Cv = &tile.bc[j][q.rs][1][q.n0];
                const int ln = fresh_lane();
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    const float Bi = Bv[i], Ci = Cv[i];
                    const f32x4 A2 = tile.A2[i][ln];
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float a = __builtin_amdgcn_exp2f(dts[c] * A2[c]);
                        const float back = a * hist[j][i][c];
                        gs[i][c] = fmaf(Ci, dys[c], gs[i][c]);
                        bc[i] = fmaf(gs[i][c], dus[c], bc[i]);
                        const float h = fmaf(dus[c], Bi, back);  // formed again: kept it would spill
                        bc[NQ + i] = fmaf(dys[c], h, bc[NQ + i]);
                        into[c] = fmaf(gs[i][c], Bi, into[c]);
                        const float gb = gs[i][c] * back;
                        dec[c] = fmaf(gb, A2[c], dec[c]);
                        dA[i][c] = fmaf(gb, dts[c], dA[i][c]);
                        gs[i][c] *= a;
                    }
                }
                const float in_n = states_sum<KQ>(into);
                float dx = fmaf(uv, in_n, states_sum<KQ>(dec) * LN2) * slope;
                dx = on ? dx : 0.f;
                ddb += dx;
                dskip = fmaf(dyv, uv, dskip);
                tile.u[j][q.col] = from_f32<T>(on ? fmaf(skip, dyv, dt * in_n) : 0.f);
                tile.de[j][q.col] = from_f32<T>(dx);
                reduce_quads<32, 4 * KQ, 2 * NQ>(bc, cw * KQ, lane);
                float* o = &tile.dbc[0][j][0][0] + obc;
                o[0] = bc[0];
                if (keeps > 1) o[1] = bc[1];
                __builtin_amdgcn_sched_barrier(260);
            }
            // the next chunk's inputs are on their way while this one's outputs leave
            if (ck > m.c0) {
                in.read(w, m, ck - 1);
                read_h(m, ck - 1);
            } else if (it + step < items) {
                const Item n(args(), w, it + step, nseg, 0);
                in.read(w, n, n.c1 - 1);
                read_h(n, n.c1 - 1);
            }
            lds_order();
            const ScanArgs a = args();
            const int ln = fresh_lane();
            RowsT::write(a.p, a.l, ln, w.g, w.cblk, (T*)a.p.du + (m.b0 * L + t0) * a.p.D, L - t0, m.two, tile.u);
            RowsT::write(a.p, a.l, ln, w.g, w.cblk, (T*)a.p.ddelta + (m.b0 * L + t0) * a.p.D, L - t0, m.two, tile.de);
            if (!a.p.dbc) {
                write_bc<T, NQ, KQ>(a.p, ln, w.g, m.b0, t0, m.two, tile);
                continue;
            }
            const long row = (((long)w.cblk * a.p.B + m.b0) * a.p.G + w.g) * a.l.chunks + ck;
            constexpr int PC = SCAN_CH * 2 * NP / 4;  // 16-byte pieces of a chunk
#pragma unroll
            for (int r = 0; r < TileT::B::RW; ++r) {
                if (r && !m.two) break;
                const auto o = (gmem<f32x4>)a.p.dbc + (row + (long)r * a.p.G * a.l.chunks) * PC;
#pragma unroll
                for (int i = 0; i < (PC + 63) / 64; ++i)
                    if (PC % 64 == 0 || i * 64 + ln < PC) o[i * 64 + ln] = ((const f32x4*)tile.dbc[r])[i * 64 + ln];
            }
        }
        const ScanArgs a = args();
        if (a.p.dh0 && m.seg == 0) store_states(a.p, q, a.p.dh0, m.b0, gs);
        if (it + step < items) m = Item(a, w, it + step, nseg, 0);
    }
    const ScanArgs a1 = args();
    const ScanParams& p = a1.p;
    const ScanPlan& l = a1.l;
    const int N = p.N, D = p.D, slot = w.slot;
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
        const auto ws = (gmem<float>)p.ws + (long)slot * D * (N + 2);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < NQ; ++i)
                if (q.state(p, c, i)) ws[(long)q.ch(c) * N + q.n0 + i] = dA[i][c];
        if (q.okc) {
            ws[(long)D * N + q.d] = dskip;
            ws[(long)D * N + D + q.d] = ddb;
        }
    }
}

// dB and dC: the channel blocks' partial sums in ascending order.
template <typename T>
__launch_bounds__(256) __global__ void scan_bc_reduce_kernel(const float* __restrict__ dbc, T* __restrict__ dB,
                                                             T* __restrict__ dC, int cblocks, long rows, int B, int L,
                                                             int G, int N, int NP) {
    // a thread: four padded states of one row, of dB and dC in turn
    const int pr = 2 * NP / 4;
    const long Lp = (L + SCAN_CH - 1) / SCAN_CH * SCAN_CH;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < rows * pr; i += (long)gridDim.x * 256) {
        const long row = i / pr;
        const int k = (int)(i % pr) * 4, which = k >= NP, n0 = which ? k - NP : k;
        const int g = (int)(row % G);
        const long bt = row / G, b = bt / L, t = bt % L;
        const f32x4* src = (const f32x4*)dbc + ((b * G + g) * Lp + t) * pr + k / 4;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        for (int c = 0; c < cblocks; ++c) s += src[(long)c * B * G * Lp * pr];
        T* o = (which ? dC : dB) + row * N + n0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < N) o[j] = from_f32<T>(s[j]);
    }
}

// One new token. Bound by the state, read and written once: 4 states (16
// bytes) a lane, `gp` lanes a channel, joined by lane exchanges for y. A thread
// keeps its channel and takes one sequence after another. Every lane reads its
// own states before it writes them: h_out may be h. 256 x 4096 x 16: 28.6 us,
// 4.9 TB/s.
template <typename T>
__launch_bounds__(256) __global__ void scan_step_kernel(ScanStepParams p, int gp) {
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    const bool ok = i / gp < p.D;
    const int d = ok ? (int)(i / gp) : 0, N = p.N;
    const int n0 = ok ? (int)(i % gp) * 4 : N;
    const int n = n0 < N ? N - n0 : 0, at = n ? n0 : 0;
    const int g = d / (p.D / p.G);
    Pack<float> Ap;
    Ap.load(p.A + (long)d * N + at, n, N % 4);
    float A2[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) A2[j] = Ap.get(j) * LOG2E;
    const float dbias = p.dbias ? p.dbias[d] : 0.f, skip = p.skip ? p.skip[d] : 0.f;
    for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
        const long r = (long)b * p.D + d;
        Pack<float> hp;
        Pack<T, 4> Bp, Cp;
        hp.load(p.h + r * N + at, n, N % 4);
        Bp.load((const T*)p.Bm + b * p.B_b + g * p.B_g + at, n, N % 4);
        Cp.load((const T*)p.Cm + b * p.C_b + g * p.C_g + at, n, N % 4);
        const float uv = to_f32(((const T*)p.u)[b * p.u_b + d]);
        const float x = to_f32(((const T*)p.delta)[b * p.d_b + d]) + dbias;
        float slope;
        const float dt = p.softplus ? softplus_s(x, slope) : x, du = dt * uv;
        float acc = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float v = fmaf(__builtin_amdgcn_exp2f(dt * A2[j]), hp.get(j), du * Bp.get(j));
            hp.w[j] = __float_as_int(v);
            acc = j < n ? fmaf(Cp.get(j), v, acc) : acc;  // v is NaN past the last state where du is infinite
        }
        for (int m = 1; m < gp; m <<= 1) acc += __shfl_xor(acc, m);
        hp.store(p.h_out + r * N + at, n, N % 4);
        if (ok && n0 == 0) ((T*)p.y)[r] = from_f32<T>(fmaf(skip, uv, acc));
    }
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
    int is_f32;
    template <int NQ, int KQ>
    void operator()() const {
        if (is_f32) f.template run<float, NQ, KQ>();
        else f.template run<__bf16, NQ, KQ>();
    }
};

inline dim3 wave_blocks(long waves) { return dim3((unsigned)((waves + 3) / 4)); }

// About 16 segments a wave of the carry.
inline dim3 carry_threads(const ScanPlan& l) {
    const int waves = (l.nseg + 15) / 16;
    return dim3(64 * (waves < 16 ? waves : 16));
}

struct ScanFwd {
    const ScanParams& p;
    const ScanPlan& l;
    hipStream_t s;
    template <typename T, int NQ, int KQ>
    void run() const {
        const long tasks = l.groups * p.G * l.cb;
        if (l.nseg > 1) {
            hipLaunchKernelGGL((scan_fwd_kernel<T, NQ, KQ, false>), wave_blocks((long)l.fslots * p.G * l.cb), dim3(256),
                               0, s, ScanArgs{p, l});
            hipLaunchKernelGGL((scan_carry_kernel<NQ, KQ, false>), dim3((unsigned)(tasks * NQ)), carry_threads(l), 0, s, p, l);
        }
        hipLaunchKernelGGL((scan_fwd_kernel<T, NQ, KQ, true>), wave_blocks((long)l.fslots * p.G * l.cb), dim3(256), 0,
                           s, ScanArgs{p, l});
    }
};

struct ScanBwd {
    const ScanParams& p;
    const ScanPlan& l;
    hipStream_t s;
    template <typename T, int NQ, int KQ>
    void run() const {
        const long tasks = l.groups * p.G * l.cb;
        if (l.nseg > 1) {
            hipLaunchKernelGGL((scan_adjoint_kernel<T, NQ, KQ>), wave_blocks((long)l.fslots * p.G * l.cb), dim3(256), 0, s,
                               ScanArgs{p, l});
            hipLaunchKernelGGL((scan_carry_kernel<NQ, KQ, true>), dim3((unsigned)(tasks * NQ)), carry_threads(l), 0, s, p, l);
        }
        hipLaunchKernelGGL((scan_bwd_kernel<T, NQ, KQ>), wave_blocks((long)l.slots * p.G * l.cb), dim3(256), 0, s,
                           ScanArgs{p, l});
    }
};

}  // namespace

// The lane layout and the cut of the time axis for these sizes and strides.
extern "C" ScanPlan scan_plan(const ScanParams& p, int is_f32, int back) {
    const int kq = p.N <= 16 ? 1 : p.N <= 32 ? 2 : 4, nq = p.N <= 4 ? 1 : p.N <= 8 ? 2 : 4;
    const long es = is_f32 ? 4 : 2, per = p.D / p.G;
    ScanPlan l{};
    // Two sequences a wave where a group has 32 channels or fewer and their
    // lane offsets fit 32 bits.
    l.cw = 64 / kq;
    if (kq == 1 && per <= 32) {
        long far = 0;
        for (long s : {(long)p.L * p.D, p.u_b, p.d_b, p.B_b, p.C_b}) far = s > far ? s : far;
        for (long s : {(long)p.D, (long)p.u_t, (long)p.d_t, (long)p.B_t, (long)p.C_t})
            if ((far + 7 * s + p.D + 64) * es > 0xffffffffL) far = 0xffffffffL;
        if (far < 0xffffffffL) l.cw = 32;
    }
    l.rw = 64 / (l.cw * kq);
    l.cb = (int)((per + l.cw - 1) / l.cw);
    l.groups = (p.B + l.rw - 1) / l.rw;
    l.chunks = (p.L + SCAN_CH - 1) / SCAN_CH;
    l.state = 64 * 4 * nq;
    // Segments of at least 4 chunks where that brings the waves towards four per
    // SIMD, in the backward two: what the kernels of 9 states and more have
    // registers for (those of 8 and fewer have some for more: up to 8 forward, 4
    // backward, which is not used). They cost a second pass over the recurrence,
    // so fewer than 3 do not pay. Measured, forward and backward of 8192 x 1536:
    // 378 us against 397 with four in the backward too; prompt of 16384 x 2048:
    // 262 us against 290 with two.
    const long tasks = l.groups * p.G * l.cb, same = (long)p.G * l.cb;
    long nseg = tasks ? (back ? 2048 : 4096) / tasks : 1;
    // Two chunks where four would leave less than two waves a SIMD: 2 x 1024 x
    // 1536 forward and backward 150 us against 154, the one size it was measured
    // at. Whole rounds of waves are not looked at: that call's 1536 backward
    // waves fill 2048 places by three quarters.
    const long least = tasks * (l.chunks / 4) < 2048 ? 2 : 4;
    if (nseg > l.chunks / least) nseg = l.chunks / least;
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
    by_states(p.N, Typed<ScanFwd>{ScanFwd{p, l, s}, is_f32});
}

extern "C" void scan_bwd_launch(const ScanParams& p, const ScanPlan& l, int is_f32, hipStream_t s) {
    by_states(p.N, Typed<ScanBwd>{ScanBwd{p, l, s}, is_f32});
}

extern "C" void scan_bc_reduce_launch(const ScanParams& p, const ScanPlan& l, int is_f32,
                                      hipStream_t s) {
    const int NP = l.state / (4 * l.cw * l.rw) * 4;
    const long rows = (long)p.B * p.L * p.G;
    const long blocks = (rows * (2 * NP / 4) + 255) / 256;
    const dim3 grid((unsigned)(blocks < 1 << 20 ? blocks : 1 << 20));
    if (is_f32) {
        hipLaunchKernelGGL((scan_bc_reduce_kernel<float>), grid, dim3(256), 0, s, p.dbc, (float*)p.dB, (float*)p.dC, l.cb, rows,
                           p.B, p.L, p.G, p.N, NP);
    } else {
        hipLaunchKernelGGL((scan_bc_reduce_kernel<__bf16>), grid, dim3(256), 0, s, p.dbc, (__bf16*)p.dB, (__bf16*)p.dC, l.cb,
                           rows, p.B, p.L, p.G, p.N, NP);
    }
}

extern "C" void scan_step_launch(const ScanStepParams& p, int is_f32, hipStream_t s) {
    const int gp = pow2_ceil((p.N + 3) / 4);
    const long across = ((long)p.D * gp + 255) / 256;
    long down = 8192 / across;  // some rounds of full occupancy
    down = down < 1 ? 1 : down > 65535 ? 65535 : down;
    const dim3 grid((unsigned)across, (unsigned)(p.B < down ? p.B : down));
    if (is_f32) {
        hipLaunchKernelGGL((scan_step_kernel<float>), grid, dim3(256), 0, s, p, gp);
    } else {
        hipLaunchKernelGGL((scan_step_kernel<__bf16>), grid, dim3(256), 0, s, p, gp);
    }
}
