// Torch bindings of the sequence operators: short causal convolution, selective
// scan, norms around a block. mpgcn_amd/ops/sequence.py checks the arguments
// for its users; what the kernels rely on for their bounds is checked here too.
#include <torch/extension.h>
#include <cfloat>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPException.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "params.hpp"

namespace {

using torch::Tensor;
using Opt = c10::optional<Tensor>;

bool has(const Opt& t) { return t.has_value() && t->defined(); }
void* ptr(const Opt& t) { return has(t) ? t->data_ptr() : nullptr; }
const float* fptr(const Opt& t) { return has(t) ? t->data_ptr<float>() : nullptr; }

int f32(const Tensor& t) { return t.scalar_type() == torch::kFloat ? 1 : 0; }

hipStream_t stream() { return c10::hip::getCurrentHIPStream().stream(); }

void check_data(const Tensor& t, const Tensor& like, at::IntArrayRef shape, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device());
    TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must be ", like.scalar_type());
    TORCH_CHECK(t.sizes() == shape, name, " must have shape ", shape, ", got ", t.sizes());
    TORCH_CHECK(t.numel() == 0 || t.size(-1) == 1 || t.stride(-1) == 1, name, " must be contiguous in its last axis");
}

void check_like(const Opt& t, const Tensor& like, at::IntArrayRef shape, const char* name) {
    if (!has(t)) return;
    check_data(*t, like, shape, name);
    TORCH_CHECK(t->is_contiguous(), name, " must be contiguous");
}

void check_f32(const Opt& t, const Tensor& like, at::IntArrayRef shape, const char* name) {
    if (!has(t)) return;
    TORCH_CHECK(t->is_cuda() && t->device() == like.device(), name, " must be on ", like.device());
    TORCH_CHECK(t->scalar_type() == torch::kFloat, name, " must be f32");
    TORCH_CHECK(t->sizes() == shape && t->is_contiguous(), name, " must be contiguous with shape ", shape);
}

int check_lens(const Opt& t, const Tensor& like, long B) {
    if (!has(t)) return 0;
    TORCH_CHECK(t->is_cuda() && t->device() == like.device(), "lengths must be on ", like.device());
    TORCH_CHECK(t->scalar_type() == torch::kInt || t->scalar_type() == torch::kLong,
                "lengths must be int32 or int64");
    TORCH_CHECK(t->dim() == 1 && t->size(0) == B && t->is_contiguous(), "lengths must have shape (B,)");
    return t->scalar_type() == torch::kLong ? 1 : 0;
}

void check_main(const Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be on GPU");
    TORCH_CHECK(t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat, name,
                " must be bf16 or f32");
    for (long s : t.sizes()) TORCH_CHECK(s <= INT_MAX / 2, name, ": extent too large");
}

// A kernel is about to write t: graphs that saved it must not use it any more.
// Tensors made in inference mode have no version, and no graph may save them.
void will_write(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor empty_f32(const Tensor& like, at::IntArrayRef shape) {
    return torch::empty(shape, like.options().dtype(torch::kFloat));
}

// ---- short convolution ------------------------------------------------------

ShortConvParams conv_params(const Tensor& x, const Tensor& w, const Opt& bias, const Opt& s0,
                            const Opt& lens, bool silu) {
    check_main(x, "x");
    TORCH_CHECK(x.dim() == 3, "x must be (B, L, D)");
    const long B = x.size(0), L = x.size(1), D = x.size(2);
    TORCH_CHECK(w.dim() == 2 && w.size(0) == D && w.size(1) >= 2 && w.size(1) <= 4, "weight must be (D, K), K in 2..4");
    const long K = w.size(1);
    check_data(x, x, x.sizes(), "x");
    check_f32(w, x, {D, K}, "weight");
    check_f32(bias, x, {D}, "bias");
    check_like(s0, x, {B, K - 1, D}, "state");
    ShortConvParams p{};
    p.lens64 = check_lens(lens, x, B);
    p.x = x.data_ptr();
    p.w = w.data_ptr<float>();
    p.bias = fptr(bias);
    p.s0 = ptr(s0);
    p.lens = ptr(lens);
    p.x_b = x.stride(0);
    p.x_t = x.stride(1);
    p.B = (int)B;
    p.L = (int)L;
    p.D = (int)D;
    p.silu = silu ? 1 : 0;
    return p;
}

// p: conv_params of these arguments
std::vector<Tensor> short_conv_fwd(ShortConvParams p, const Tensor& x, long K, bool want_state) {
    at::DeviceGuard guard(x.device());
    auto y = torch::empty({p.B, p.L, p.D}, x.options());
    auto s1 = want_state ? torch::empty({p.B, K - 1, p.D}, x.options()) : Tensor();
    if (p.B && p.D && (p.L || want_state)) {
        p.y = y.data_ptr();
        p.s1 = want_state ? s1.data_ptr() : nullptr;
        short_conv_plan(&p, f32(x), 0);
        short_conv_fwd_launch(p, (int)K, f32(x), stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return {y, s1};
}

// {dx, dw (D, K), db (D,), dstate or undefined}
std::vector<Tensor> short_conv_bwd(Tensor dy, Opt ds1, Tensor x, Tensor w, Opt bias, Opt s0, Opt lens, bool silu,
                                   bool want_state) {
    at::DeviceGuard guard(x.device());
    auto p = conv_params(x, w, bias, s0, lens, silu);
    const long K = w.size(1), D = p.D;
    check_like(dy, x, {p.B, p.L, p.D}, "dy");
    check_like(ds1, x, {p.B, K - 1, p.D}, "dstate");
    auto dx = torch::empty({p.B, p.L, p.D}, x.options());
    auto ds0 = want_state ? torch::empty({p.B, K - 1, p.D}, x.options()) : Tensor();
    if (!p.B || !p.D) {
        auto z = torch::zeros({D * (K + 1)}, w.options());
        return {dx, z.narrow(0, 0, D * K).view({D, K}), z.narrow(0, D * K, D), ds0};
    }
    short_conv_plan(&p, f32(x), 1);
    auto ws = empty_f32(x, {p.slots, D * (K + 1)});
    auto sums = empty_f32(x, {D * (K + 1)});
    p.dy = dy.data_ptr();
    p.ds1 = ptr(ds1);
    p.dx = dx.data_ptr();
    p.ds0 = want_state ? ds0.data_ptr() : nullptr;
    p.ws = ws.data_ptr<float>();
    short_conv_bwd_launch(p, (int)K, f32(x), stream());
    seq_colsum_launch(p.ws, sums.data_ptr<float>(), p.slots, D * (K + 1), stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return {dx, sums.narrow(0, 0, D * K).view({D, K}), sums.narrow(0, D * K, D), ds0};
}

void check_conv_step(const Tensor& x, const Tensor& state, const Tensor& state_out, const Tensor& w, const Opt& bias) {
    check_main(x, "x");
    TORCH_CHECK(x.dim() == 2, "x must be (B, D)");
    const long B = x.size(0), D = x.size(1);
    TORCH_CHECK(w.dim() == 2 && w.size(1) >= 2 && w.size(1) <= 4, "weight must be (D, K), K in 2..4");
    const long K = w.size(1);
    check_data(x, x, x.sizes(), "x");
    check_f32(w, x, {D, K}, "weight");
    check_f32(bias, x, {D}, "bias");
    check_like(state, x, {B, K - 1, D}, "state");
    check_like(state_out, x, {B, K - 1, D}, "state_out");
}

// after check_conv_step
Tensor run_conv_step(const Tensor& x, const Tensor& state, const Tensor& state_out, const Tensor& w, const Opt& bias,
                     bool silu) {
    at::DeviceGuard guard(x.device());
    const long B = x.size(0), D = x.size(1), K = w.size(1);
    auto y = torch::empty({B, D}, x.options());
    if (B && D) {
        will_write(state_out);
        short_conv_step_launch(x.data_ptr(), x.stride(0), state.data_ptr(), state_out.data_ptr(),
                               w.data_ptr<float>(), fptr(bias), y.data_ptr(), B, (int)D, (int)K, silu,
                               f32(x), stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return y;
}

Tensor short_conv_step(Tensor x, Tensor state, Tensor state_out, Tensor w, Opt bias, bool silu) {
    check_conv_step(x, state, state_out, w, bias);
    return run_conv_step(x, state, state_out, w, bias, silu);
}

// ---- selective scan ---------------------------------------------------------

// At most a wave each in one launch, four to a block of 256.
void check_channels(long D) { TORCH_CHECK(D <= (1L << 26) - 4, "at most 2^26 - 4 channels"); }

ScanParams scan_params(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                       const Opt& skip, const Opt& dbias, const Opt& h0, const Opt& lens, bool softplus) {
    check_main(u, "u");
    TORCH_CHECK(u.dim() == 3, "u must be (B, L, D)");
    const long B = u.size(0), L = u.size(1), D = u.size(2);
    TORCH_CHECK(A.dim() == 2 && A.size(1) >= 1 && A.size(1) <= 64, "A must be (D, N), N in 1..64");
    const long N = A.size(1);
    TORCH_CHECK(Bm.dim() == 4 && Bm.size(2) >= 1 && D % Bm.size(2) == 0, "B must be (B, L, G, N), G a divisor of D");
    const long G = Bm.size(2);
    check_channels(D);
    check_data(u, u, u.sizes(), "u");
    check_data(delta, u, {B, L, D}, "delta");
    check_data(Bm, u, {B, L, G, N}, "B");
    check_data(Cm, u, {B, L, G, N}, "C");
    check_f32(A, u, {D, N}, "A");
    check_f32(skip, u, {D}, "skip");
    check_f32(dbias, u, {D}, "delta_bias");
    check_f32(h0, u, {B, D, N}, "state");
    ScanParams p{};
    p.lens64 = check_lens(lens, u, B);
    p.u = u.data_ptr();
    p.delta = delta.data_ptr();
    p.Bm = Bm.data_ptr();
    p.Cm = Cm.data_ptr();
    p.A = A.data_ptr<float>();
    p.skip = fptr(skip);
    p.dbias = fptr(dbias);
    p.h0 = fptr(h0);
    p.lens = ptr(lens);
    auto step = [](const Tensor& t) {
        if (t.size(1) < 2) return 0;
        TORCH_CHECK(t.stride(1) < (1L << 26), "the stride between tokens must be below 2^26 elements");
        return (int)t.stride(1);
    };
    p.u_b = u.stride(0); p.u_t = step(u);
    p.d_b = delta.stride(0); p.d_t = step(delta);
    p.B_b = Bm.stride(0); p.B_t = step(Bm); p.B_g = Bm.stride(2);
    p.C_b = Cm.stride(0); p.C_t = step(Cm); p.C_g = Cm.stride(2);
    p.B = (int)B; p.L = (int)L; p.D = (int)D; p.N = (int)N; p.G = (int)G;
    p.softplus = softplus ? 1 : 0;
    return p;
}

// {y, final state, states entering every chunk or undefined}; p: scan_params of these arguments
std::vector<Tensor> selective_scan_fwd(ScanParams p, const Tensor& u, bool want_state, bool train) {
    at::DeviceGuard guard(u.device());
    auto y = torch::empty({p.B, p.L, p.D}, u.options());
    auto h1 = want_state ? empty_f32(u, {p.B, p.D, p.N}) : Tensor();
    Tensor ck, seg_h, seg_s;
    if (p.B && p.D && (p.L || want_state)) {
        const ScanPlan l = scan_plan(p, f32(u), 0);
        const long tasks = l.groups * p.G * l.cb;
        // one chunk starts from the state given: nothing to keep
        if (train && l.chunks > 1) ck = empty_f32(u, {tasks, l.chunks, l.state});
        if (l.nseg > 1) {
            seg_h = empty_f32(u, {tasks, l.nseg, l.state});
            seg_s = empty_f32(u, {tasks, l.nseg, 64});
            p.seg_h = seg_h.data_ptr<float>();
            p.seg_s = seg_s.data_ptr<float>();
        }
        p.y = y.data_ptr();
        p.h1 = want_state ? h1.data_ptr<float>() : nullptr;
        p.ckpt = ck.defined() ? ck.data_ptr<float>() : nullptr;
        scan_fwd_launch(p, l, f32(u), stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return {y, h1, ck};
}

// {du, ddelta, dA, dB, dC, dskip, ddelta_bias, dstate or undefined}
std::vector<Tensor> selective_scan_bwd(Opt dy, Opt dh1, Tensor u, Tensor delta, Tensor A, Tensor Bm, Tensor Cm,
                                       Opt skip, Opt dbias, Opt h0, Opt lens, Opt ck, bool softplus,
                                       bool want_state) {
    at::DeviceGuard guard(u.device());
    auto p = scan_params(u, delta, A, Bm, Cm, skip, dbias, h0, lens, softplus);
    const long B = p.B, L = p.L, D = p.D, N = p.N, G = p.G;
    check_like(dy, u, {B, L, D}, "dy");
    check_f32(dh1, u, {B, D, N}, "dstate");
    auto du = torch::empty({B, L, D}, u.options());
    auto dd = torch::empty({B, L, D}, u.options());
    auto dB = torch::empty({B, L, G, N}, u.options());
    auto dC = torch::empty({B, L, G, N}, u.options());
    auto dh0 = want_state ? empty_f32(u, {B, D, N}) : Tensor();
    auto split = [&](const Tensor& s) {
        return std::vector<Tensor>{du, dd, s.narrow(0, 0, D * N).view({D, N}), dB, dC, s.narrow(0, D * N, D),
                                   s.narrow(0, D * N + D, D), dh0};
    };
    if (!B || !D) {
        dB.zero_();
        dC.zero_();
        return split(torch::zeros({D * (N + 2)}, A.options()));
    }
    const ScanPlan l = scan_plan(p, f32(u), 1);
    const long tasks = l.groups * G * l.cb;
    if (l.chunks > 1) {
        TORCH_CHECK(has(ck), "the forward kept no chunk states");
        check_f32(ck, u, {tasks, l.chunks, l.state}, "chunk states");
    }
    auto ws = empty_f32(u, {l.slots, D * (N + 2)});
    auto sums = empty_f32(u, {D * (N + 2)});
    // one channel block leaves nothing to add up
    Tensor dbc;
    if (l.cb > 1) dbc = empty_f32(u, {l.cb, B, G, l.chunks, 8, 2, l.state / (4 * l.cw * l.rw) * 4});
    Tensor seg_h, seg_s;
    if (l.nseg > 1) {
        seg_h = empty_f32(u, {tasks, l.nseg, l.state});
        seg_s = empty_f32(u, {tasks, l.nseg, 64});
        p.seg_h = seg_h.data_ptr<float>();
        p.seg_s = seg_s.data_ptr<float>();
    }
    const Tensor dyt = has(dy) ? *dy : torch::zeros({B, L, D}, u.options());
    p.dy = dyt.data_ptr();
    p.dh1 = fptr(dh1);
    p.du = du.data_ptr();
    p.ddelta = dd.data_ptr();
    p.ckpt = has(ck) ? ck->data_ptr<float>() : nullptr;
    p.dbc = dbc.defined() ? dbc.data_ptr<float>() : nullptr;
    p.dB = dB.data_ptr();
    p.dC = dC.data_ptr();
    p.ws = ws.data_ptr<float>();
    p.dh0 = want_state ? dh0.data_ptr<float>() : nullptr;
    scan_bwd_launch(p, l, f32(u), stream());
    seq_colsum_launch(p.ws, sums.data_ptr<float>(), l.slots, D * (N + 2), stream());
    if (L && p.dbc) scan_bc_reduce_launch(p, l, f32(u), stream());
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return split(sums);
}

ScanStepParams scan_step_params(const Tensor& u, const Tensor& delta, const Tensor& A, const Tensor& Bm, const Tensor& Cm,
                                const Tensor& state, const Tensor& state_out, const Opt& skip, const Opt& dbias,
                                bool softplus) {
    check_main(u, "u");
    TORCH_CHECK(u.dim() == 2, "u must be (B, D)");
    const long B = u.size(0), D = u.size(1);
    check_channels(D);
    TORCH_CHECK(A.dim() == 2 && A.size(1) >= 1 && A.size(1) <= 64, "A must be (D, N), N in 1..64");
    const long N = A.size(1);
    TORCH_CHECK(Bm.dim() == 2 || Bm.dim() == 3, "B must be (B, N) or (B, G, N)");
    const bool grouped = Bm.dim() == 3;
    const long G = grouped ? Bm.size(1) : 1;
    TORCH_CHECK(G >= 1 && D % G == 0, "the groups must divide the channels");
    check_data(u, u, u.sizes(), "u");
    check_data(delta, u, {B, D}, "delta");
    check_data(Bm, u, grouped ? at::IntArrayRef({B, G, N}) : at::IntArrayRef({B, N}), "B");
    check_data(Cm, u, grouped ? at::IntArrayRef({B, G, N}) : at::IntArrayRef({B, N}), "C");
    check_f32(A, u, {D, N}, "A");
    check_f32(skip, u, {D}, "skip");
    check_f32(dbias, u, {D}, "delta_bias");
    check_f32(state, u, {B, D, N}, "state");
    check_f32(state_out, u, {B, D, N}, "state_out");
    ScanStepParams p{};
    p.u = u.data_ptr(); p.delta = delta.data_ptr(); p.Bm = Bm.data_ptr(); p.Cm = Cm.data_ptr();
    p.A = A.data_ptr<float>(); p.skip = fptr(skip); p.dbias = fptr(dbias);
    p.h = state.data_ptr<float>(); p.h_out = state_out.data_ptr<float>();
    p.u_b = u.stride(0); p.d_b = delta.stride(0);
    p.B_b = Bm.stride(0); p.B_g = grouped ? Bm.stride(1) : 0;
    p.C_b = Cm.stride(0); p.C_g = grouped ? Cm.stride(1) : 0;
    p.B = (int)B; p.D = (int)D; p.N = (int)N; p.G = (int)G;
    p.softplus = softplus ? 1 : 0;
    return p;
}

// p: scan_step_params of u, state_out and the rest
Tensor run_scan_step(ScanStepParams p, const Tensor& u, const Tensor& state_out) {
    at::DeviceGuard guard(u.device());
    auto y = torch::empty({p.B, p.D}, u.options());
    if (p.B && p.D) {
        p.y = y.data_ptr();
        will_write(state_out);
        scan_step_launch(p, f32(u), stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return y;
}

Tensor selective_scan_step(Tensor u, Tensor delta, Tensor A, Tensor Bm, Tensor Cm, Tensor state, Tensor state_out,
                           Opt skip, Opt dbias, bool softplus) {
    return run_scan_step(scan_step_params(u, delta, A, Bm, Cm, state, state_out, skip, dbias, softplus), u, state_out);
}

// ---- norms around a block ---------------------------------------------------

BlockNormParams norm_params(const Tensor& x, const Opt& gate, const Opt& post, const Opt& res, const Opt& scale,
                            const Opt& pre, double eps) {
    check_main(x, "x");
    TORCH_CHECK(x.dim() == 2, "x must be (R, D)");
    const long R = x.size(0), D = x.size(1);
    TORCH_CHECK(D <= 16384, "D must be at most 16384");
    check_data(x, x, x.sizes(), "x");
    if (has(gate)) check_data(*gate, x, {R, D}, "gate");
    if (has(res)) {
        check_main(*res, "residual");
        check_data(*res, *res, {R, D}, "residual");
        TORCH_CHECK(res->device() == x.device(), "residual must be on ", x.device());
    }
    TORCH_CHECK(has(post) || has(pre), "a norm's weight is needed");
    TORCH_CHECK(has(res) || !(has(scale) || has(pre)), "scale and pre need a residual");
    check_f32(post, x, {D}, "post_weight");
    check_f32(scale, x, {D}, "scale");
    check_f32(pre, x, {D}, "pre_weight");
    BlockNormParams p{};
    p.x = x.data_ptr();
    p.gate = ptr(gate);
    p.post = fptr(post);
    p.res = ptr(res);
    p.scale = fptr(scale);
    p.pre = fptr(pre);
    p.x_r = x.stride(0);
    p.g_r = has(gate) ? gate->stride(0) : 0;
    p.r_r = has(res) ? res->stride(0) : 0;
    p.R = R;
    p.D = (int)D;
    p.eps = (float)eps;
    return p;
}

// {y, h, inv1, inv2}, those that there are; p: norm_params of these arguments
std::vector<Tensor> block_norm_fwd(BlockNormParams p, const Tensor& x, const Opt& res, bool train) {
    at::DeviceGuard guard(x.device());
    const long R = p.R, D = p.D;
    auto y = p.pre || !has(res) ? torch::empty({R, D}, x.options()) : Tensor();
    auto h = has(res) ? torch::empty({R, D}, res->options()) : Tensor();
    auto i1 = train && p.post ? empty_f32(x, {R}) : Tensor();
    auto i2 = train && p.pre ? empty_f32(x, {R}) : Tensor();
    if (R && D) {
        p.y = y.defined() ? y.data_ptr() : nullptr;
        p.h = h.defined() ? h.data_ptr() : nullptr;
        p.inv1 = i1.defined() ? i1.data_ptr<float>() : nullptr;
        p.inv2 = i2.defined() ? i2.data_ptr<float>() : nullptr;
        block_norm_fwd_launch(p, f32(x), has(res) ? f32(*res) : f32(x), stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    }
    return {y, h, i1, i2};
}

// {dx, dgate, dpost, dresidual, dscale, dpre}, those that there are
std::vector<Tensor> block_norm_bwd(Opt dy, Opt dh, Tensor x, Opt gate, Opt post, Opt res, Opt scale, Opt pre,
                                   Opt inv1, Opt inv2, double eps) {
    at::DeviceGuard guard(x.device());
    auto p = norm_params(x, gate, post, res, scale, pre, eps);
    const long R = p.R, D = p.D;
    check_like(dy, x, {R, D}, "dy");
    if (has(res)) check_like(dh, *res, {R, D}, "dh");
    check_f32(inv1, x, {R}, "inv1");
    check_f32(inv2, x, {R}, "inv2");
    TORCH_CHECK(has(inv1) == has(post) && has(inv2) == has(pre), "the forward kept no row statistics");
    auto dx = torch::empty({R, D}, x.options());
    auto dg = has(gate) ? torch::empty({R, D}, x.options()) : Tensor();
    auto dr = has(res) ? torch::empty({R, D}, res->options()) : Tensor();
    const long nw = has(post) + has(scale) + has(pre);
    Tensor sums;
    if (R && D) {
        p.slots = block_norm_slots(R, D, has(res), has(gate));
        auto ws = empty_f32(x, {p.slots, nw * D});
        sums = empty_f32(x, {nw, D});
        p.inv1 = (float*)fptr(inv1);
        p.inv2 = (float*)fptr(inv2);
        p.dy = ptr(dy);
        p.dh = has(res) ? ptr(dh) : nullptr;
        p.dx = dx.data_ptr();
        p.dgate = ptr(dg);
        p.dres = ptr(dr);
        p.ws = ws.data_ptr<float>();
        block_norm_bwd_launch(p, f32(x), has(res) ? f32(*res) : f32(x), stream());
        seq_colsum_launch(p.ws, sums.data_ptr<float>(), p.slots, nw * D, stream());
        C10_HIP_KERNEL_LAUNCH_CHECK();
    } else {
        sums = torch::zeros({nw, D}, x.options().dtype(torch::kFloat));
    }
    long at = 0;
    auto next = [&](const Opt& w) { return has(w) ? sums.select(0, at++) : Tensor(); };
    auto dpost = next(post), dscale = next(scale), dpre = next(pre);
    return {dx, dg, dpost, dr, dscale, dpre};
}

// ---- gradients --------------------------------------------------------------

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

Tensor val(const Opt& t) { return has(t) ? *t : Tensor(); }
Opt opt(const Tensor& t) { return t.defined() ? Opt(t) : Opt(); }
Opt rows_of(const Tensor& t) { return t.defined() ? Opt(t.contiguous()) : Opt(); }

// The kernels would drop the tangent of forward mode in silence.
void refuse(const char* name, const Tensor& t) {
    TORCH_CHECK(!c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t.defined() || !t._fw_grad(0).defined(), name,
                " has no forward-mode derivative on a GPU");
}

// Whether any gradient has arrived.
bool any(const variable_list& g, const char* name) {
    bool there = false;
    for (const auto& t : g) {
        refuse(name, t);
        there |= t.defined();
    }
    return there;
}

// The gradients have no gradient of their own: a second derivative raises when
// it is asked for.
variable_list once(variable_list g, const char* name) {
    if (!at::GradMode::is_enabled()) return g;
    for (auto& t : g)
        if (t.defined()) t = t.detach().set_requires_grad(true);
    auto fn = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " has no second derivative",
                                                              (int64_t)g.size());
    return (*fn)(std::move(g));
}

struct ShortConvFn : Function<ShortConvFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opt& bias, const Opt& s0,
                                 const Opt& lens, bool silu, bool want_state) {
        ctx->set_materialize_grads(false);
        auto r = short_conv_fwd(conv_params(x, w, bias, s0, lens, silu), x, w.size(1), want_state);
        ctx->save_for_backward({x, w, val(bias), val(s0), val(lens)});
        ctx->saved_data["silu"] = silu;
        ctx->saved_data["state"] = has(s0) && s0->requires_grad();
        if (!want_state) r.pop_back();
        return r;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list out(7);
        if (any(g, "short_conv")) {
            at::NoGradGuard no_grad;
            auto v = ctx->get_saved_variables();
            const Tensor dy = g[0].defined() ? g[0].contiguous() : torch::zeros(v[0].sizes(), v[0].options());
            auto r = short_conv_bwd(dy, g.size() > 1 ? rows_of(g[1]) : Opt(), v[0], v[1], opt(v[2]), opt(v[3]),
                                    opt(v[4]), ctx->saved_data["silu"].toBool(), ctx->saved_data["state"].toBool());
            out[0] = r[0];
            out[1] = r[1];
            if (v[2].defined()) out[2] = r[2];
            out[3] = r[3];
        }
        return once(out, "short_conv");
    }
};

struct SelectiveScanFn : Function<SelectiveScanFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& delta, const Tensor& A,
                                 const Tensor& Bm, const Tensor& Cm, const Opt& skip, const Opt& dbias, const Opt& h0,
                                 const Opt& lens, bool softplus, bool want_state) {
        ctx->set_materialize_grads(false);
        auto r = selective_scan_fwd(scan_params(u, delta, A, Bm, Cm, skip, dbias, h0, lens, softplus), u, want_state, true);
        ctx->save_for_backward({u, delta, A, Bm, Cm, val(skip), val(dbias), val(h0), val(lens), r[2]});
        ctx->saved_data["softplus"] = softplus;
        ctx->saved_data["state"] = has(h0) && h0->requires_grad();
        r.resize(want_state ? 2 : 1);
        return r;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list out(11);
        if (any(g, "selective_scan")) {
            at::NoGradGuard no_grad;
            auto v = ctx->get_saved_variables();
            auto r = selective_scan_bwd(rows_of(g[0]), g.size() > 1 ? rows_of(g[1]) : Opt(), v[0], v[1], v[2], v[3], v[4],
                                        opt(v[5]), opt(v[6]), opt(v[7]), opt(v[8]), opt(v[9]),
                                        ctx->saved_data["softplus"].toBool(), ctx->saved_data["state"].toBool());
            for (int i = 0; i < 8; ++i) out[i] = r[i];
            if (!v[5].defined()) out[5] = Tensor();
            if (!v[6].defined()) out[6] = Tensor();
        }
        return once(out, "selective_scan");
    }
};

struct BlockNormFn : Function<BlockNormFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const Opt& gate, const Opt& post, const Opt& res,
                                 const Opt& scale, const Opt& pre, double eps) {
        ctx->set_materialize_grads(false);
        auto r = block_norm_fwd(norm_params(x, gate, post, res, scale, pre, eps), x, res, true);
        ctx->save_for_backward({x, val(gate), val(post), val(res), val(scale), val(pre), r[2], r[3]});
        ctx->saved_data["eps"] = eps;
        if (!r[1].defined()) return {r[0]};
        if (!r[0].defined()) return {r[1]};
        return {r[0], r[1]};
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        variable_list out(7);
        if (any(g, "norm_gate_residual")) {
            at::NoGradGuard no_grad;
            auto v = ctx->get_saved_variables();
            const bool y = !v[3].defined() || v[5].defined();
            const Opt dy = y ? rows_of(g[0]) : Opt(), dh = v[3].defined() ? rows_of(g.back()) : Opt();
            auto r = block_norm_bwd(dy, dh, v[0], opt(v[1]), opt(v[2]), opt(v[3]), opt(v[4]), opt(v[5]), opt(v[6]),
                                    opt(v[7]), ctx->saved_data["eps"].toDouble());
            for (int i = 0; i < 6; ++i) out[i] = r[i];
        }
        return once(out, "norm_gate_residual");
    }
};

py::object one_or_pair(const variable_list& r) {
    return r.size() > 1 ? py::object(py::make_tuple(r[0], r[1])) : py::cast(r[0]);
}

// A capture needs the look at live graphs that Python takes first.
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

// ---- calls that need no preparation -----------------------------------------
//
// The operators' common case without Python's share of the time: every argument
// is in the kernels' form. Any other call gives None and goes through the
// checks and conversions of mpgcn_amd/ops/sequence.py, which name what is wrong
// and come back here with `prepared` set.

using Inputs = std::initializer_list<const Tensor*>;

// Nor does a trace see these calls: it would hold their outputs as constants.
void refuse(const char* name, Inputs ts) {
    TORCH_CHECK(!torch::jit::tracer::isTracing(), name, " cannot be traced on a GPU");
    for (const Tensor* t : ts)
        if (t) refuse(name, *t);
}

bool wants_grad(Inputs ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t && t->defined() && t->requires_grad()) return true;
    return false;
}
const Tensor* tp(const Opt& t) { return t.has_value() ? &*t : nullptr; }

// Whether the checks pass. They alone say that a call needs preparation; an
// error of the call itself (memory, a launch) is the caller's to see, since
// running it again could advance a state twice.
template <typename F>
bool fits(bool prepared, F checks) {
    if (prepared) {
        checks();
        return true;
    }
    try {
        checks();
        return true;
    } catch (const c10::Error&) {
        return false;
    }
}

// Two states that a step may read and write: the same memory or none shared.
bool apart(const Tensor& a, const Tensor& b) {
    const char *pa = (const char*)a.data_ptr(), *pb = (const char*)b.data_ptr();
    const long d = pa < pb ? pb - pa : pa - pb;
    return d == 0 || d >= (long)(a.numel() * a.element_size());
}

py::object short_conv_direct(Tensor x, Tensor w, Opt bias, Opt s0, Opt lens, bool silu, bool want_state,
                             bool prepared) {
    if (!x.is_cuda()) return py::none();
    const Inputs ts = {&x, &w, tp(bias), tp(s0)};
    refuse("short_conv", ts);
    const bool train = wants_grad(ts);
    if (train && !prepared && capturing()) return py::none();
    ShortConvParams p;
    if (!fits(prepared, [&] { p = conv_params(x, w, bias, s0, lens, silu); })) return py::none();
    if (train) return one_or_pair(ShortConvFn::apply(x, w, bias, s0, lens, silu, want_state));
    auto r = short_conv_fwd(p, x, w.size(1), want_state);
    if (!want_state) r.pop_back();
    return one_or_pair(r);
}

py::object short_conv_step_direct(Tensor x, Tensor state, Opt state_out, Tensor w, Opt bias, bool silu) {
    if (!x.is_cuda()) return py::none();
    const Tensor out = has(state_out) ? *state_out : state;
    const Inputs ts = {&x, &state, &out, &w, tp(bias)};
    refuse("short_conv_step", ts);
    if (wants_grad(ts) || !apart(state, out) || !fits(false, [&] { check_conv_step(x, state, out, w, bias); }))
        return py::none();
    return py::make_tuple(run_conv_step(x, state, out, w, bias, silu), out);
}

py::object selective_scan_direct(Tensor u, Tensor delta, Tensor A, Tensor Bm, Tensor Cm, Opt skip, Opt dbias, Opt h0,
                                 Opt lens, bool softplus, bool want_state, bool prepared) {
    if (!u.is_cuda()) return py::none();
    const Inputs ts = {&u, &delta, &A, &Bm, &Cm, tp(skip), tp(dbias), tp(h0)};
    refuse("selective_scan", ts);
    const bool train = wants_grad(ts);
    if (train && !prepared && capturing()) return py::none();
    const Tensor B4 = Bm.dim() == 3 ? Bm.unsqueeze(2) : Bm, C4 = Cm.dim() == 3 ? Cm.unsqueeze(2) : Cm;
    ScanParams p;
    if (!fits(prepared, [&] { p = scan_params(u, delta, A, B4, C4, skip, dbias, h0, lens, softplus); }))
        return py::none();
    if (train)
        return one_or_pair(SelectiveScanFn::apply(u, delta, A, B4, C4, skip, dbias, h0, lens, softplus, want_state));
    auto r = selective_scan_fwd(p, u, want_state, false);
    r.resize(want_state ? 2 : 1);
    return one_or_pair(r);
}

py::object selective_scan_step_direct(Tensor u, Tensor delta, Tensor A, Tensor Bm, Tensor Cm, Tensor state,
                                      Opt state_out, Opt skip, Opt dbias, bool softplus) {
    if (!u.is_cuda()) return py::none();
    const Tensor out = has(state_out) ? *state_out : state;
    const Inputs ts = {&u, &delta, &A, &Bm, &Cm, &state, &out, tp(skip), tp(dbias)};
    refuse("selective_scan_step", ts);
    if (wants_grad(ts) || !apart(state, out)) return py::none();
    ScanStepParams p;
    if (!fits(false, [&] { p = scan_step_params(u, delta, A, Bm, Cm, state, out, skip, dbias, softplus); }))
        return py::none();
    return py::make_tuple(run_scan_step(p, u, out), out);
}

py::object block_norm_direct(Tensor x, Opt gate, Opt post, Opt res, Opt scale, Opt pre, double eps, bool prepared) {
    if (!x.is_cuda() || x.dim() < 1 || !(eps >= FLT_MIN)) return py::none();
    const Inputs ts = {&x, tp(gate), tp(post), tp(res), tp(scale), tp(pre)};
    refuse("norm_gate_residual", ts);
    const bool train = wants_grad(ts);
    if (train && !prepared && capturing()) return py::none();
    const auto shape = x.sizes().vec();
    const bool flat = x.dim() == 2;
    if (!fits(prepared, [&] {
            TORCH_CHECK(shape.back() >= 1 && (!has(gate) || gate->sizes() == x.sizes()) &&
                        (!has(res) || res->sizes() == x.sizes()), "gate and residual must have x's shape");
        }))
        return py::none();
    auto rows = [&](const Tensor& t) { return flat ? t : t.reshape({-1, shape.back()}); };  // may copy
    auto opt_rows = [&](const Opt& t) { return has(t) ? Opt(rows(*t)) : Opt(); };
    const Tensor x2 = rows(x);
    const Opt gate2 = opt_rows(gate), res2 = opt_rows(res);
    BlockNormParams p;
    if (!fits(prepared, [&] { p = norm_params(x2, gate2, post, res2, scale, pre, eps); })) return py::none();
    variable_list r;
    if (train) {
        r = BlockNormFn::apply(x2, gate2, post, res2, scale, pre, eps);
    } else {
        for (auto& t : block_norm_fwd(p, x2, res2, false))
            if (t.defined()) r.push_back(t);
    }
    if (!flat)
        for (auto& t : r) t = t.view(shape);
    return one_or_pair(r);
}

}  // namespace

// A leaf whose gradient an eager graph, still alive, accumulates on another
// stream: a backward captured now would wait for that stream and break the capture.
bool accumulates_elsewhere(Tensor leaf) {
    auto acc = torch::autograd::impl::try_get_grad_accumulator(leaf);
    if (!acc) return false;
    const auto s = acc->stream();
    return s.has_value() && *s != c10::impl::VirtualGuardImpl(s->device_type()).getStream(s->device());
}

void bind_sequence(pybind11::module_& m) {
    m.def("accumulates_elsewhere", &accumulates_elsewhere, "leaf has a live accumulator on another stream");
    const auto prepared = py::arg("prepared") = false;
    m.def("short_conv_direct", &short_conv_direct, "short_conv where no preparation is needed, else None", py::arg("x"),
          py::arg("weight"), py::arg("bias"), py::arg("state"), py::arg("lengths"), py::arg("silu"),
          py::arg("return_state"), prepared);
    m.def("short_conv_step", &short_conv_step, "short causal convolution of one new token");
    m.def("selective_scan_step", &selective_scan_step, "selective state space scan of one new token");
    m.def("short_conv_step_direct", &short_conv_step_direct, "short_conv_step, likewise");
    m.def("selective_scan_direct", &selective_scan_direct, "selective_scan, likewise", py::arg("u"), py::arg("delta"),
          py::arg("A"), py::arg("B"), py::arg("C"), py::arg("skip"), py::arg("delta_bias"), py::arg("state"),
          py::arg("lengths"), py::arg("softplus"), py::arg("return_state"), prepared);
    m.def("selective_scan_step_direct", &selective_scan_step_direct, "selective_scan_step, likewise");
    m.def("block_norm_direct", &block_norm_direct, "norm_gate_residual, likewise", py::arg("x"), py::arg("gate"),
          py::arg("post_weight"), py::arg("residual"), py::arg("scale"), py::arg("pre_weight"), py::arg("eps"), prepared);
}
