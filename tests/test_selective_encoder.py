"""The selective temporal encoder, alone and inside the model, the trainer and
the served request path."""

import pytest
import torch

from mpgcn_amd.data import DataGenerator, DataInput
from mpgcn_amd.graph import build_supports
from mpgcn_amd.models import MPGCN, SelectiveEncoder
from mpgcn_amd.train import ModelTrainer


def _model(N=10, H=16, **kw):
    return MPGCN(M=2, K=3, input_dim=1, lstm_hidden_dim=H, lstm_num_layers=1, gcn_hidden_dim=H, gcn_num_layers=3,
                 num_nodes=N, **kw)


def _graphs(N, B, device="cpu"):
    g = torch.Generator().manual_seed(3)
    adj, flow = torch.rand(N, N, generator=g).to(device), torch.rand(B, N, N, generator=g).to(device)
    sup = build_supports(adj.unsqueeze(0), "random_walk_diffusion", 2).squeeze(0)
    return [sup, (build_supports(flow, "random_walk_diffusion", 2),
                  build_supports(flow.transpose(-2, -1), "random_walk_diffusion", 2))]


def _by_hand(enc, x):
    """The block's formulas, step by step, in the encoder's own precision."""
    H, N = enc.hidden_size, enc.state_size
    R, T = x.shape
    uz = x.unsqueeze(-1) * enc.in_proj.weight[:, 0] + enc.in_proj.bias
    u, z = uz[..., :H], uz[..., H:]
    h, past = x.new_zeros(R, H, N), x.new_zeros(R, enc.taps - 1, H)
    full = torch.cat([past, u], 1)
    silu = torch.nn.functional.silu
    for t in range(T):
        v = silu((full[:, t:t + enc.taps] * enc.conv_weight.t()).sum(1) + enc.conv_bias)
        m = v @ enc.x_proj.weight.t()
        dt = torch.nn.functional.softplus(m[:, :H] + enc.delta_bias).unsqueeze(-1)
        h = torch.exp(-dt * torch.exp(enc.A_log)) * h + dt * v.unsqueeze(-1) * m[:, None, H:H + N]
        y = (h * m[:, None, H + N:]).sum(-1) + enc.skip * v

    def rms(a, w):
        return a / torch.sqrt((a * a).mean(-1, keepdim=True) + 1e-5) * w

    o = rms(y * silu(z[:, -1]), enc.gate_norm) @ enc.out_proj.weight.t() + enc.out_proj.bias
    return rms(u[:, -1] + enc.residual_scale * o, enc.out_norm)


def test_encoder_is_its_formulas():
    torch.manual_seed(0)
    enc = SelectiveEncoder(1, 8, state_size=5, taps=3).double()
    x = torch.rand(6, 9, dtype=torch.float64)
    torch.testing.assert_close(enc(x), _by_hand(enc, x), rtol=1e-10, atol=1e-10)
    padded = torch.cat([x, torch.full((6, 7), float("nan"), dtype=x.dtype)], 1)
    torch.testing.assert_close(enc(padded, 9), enc(x), rtol=0, atol=0)


def test_encoder_steps_continue():
    torch.manual_seed(0)
    enc = SelectiveEncoder(1, 8)
    x = torch.rand(5, 12)
    want = [enc(x[:, :t]) for t in (9, 10, 11, 12)]
    h, state = enc.start(x[:, :9])
    got = [h] + [enc.step(x[:, t], state) for t in (9, 10, 11)]
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b.detach(), rtol=0, atol=1e-5)


def test_encoder_refusals():
    for kw in (dict(input_size=2), dict(state_size=0), dict(state_size=65), dict(taps=1), dict(taps=5)):
        with pytest.raises(ValueError):
            SelectiveEncoder(**{"input_size": 1, "hidden_size": 8, **kw})
    with pytest.raises(ValueError):
        _model(temporal="gru")


def test_model_trains_every_parameter_and_round_trips():
    torch.manual_seed(0)
    model = _model(temporal="selective")
    x, y = torch.rand(2, 7, 10, 10, 1), torch.rand(2, 1, 10, 10, 1)
    out = model(x, _graphs(10, 2))
    assert out.shape == (2, 1, 10, 10, 1)
    torch.nn.functional.mse_loss(out, y).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())
    again = _model(temporal="selective")
    again.load_state_dict(model.state_dict())
    assert torch.equal(again(x, _graphs(10, 2)), out)
    assert "branch_models.0.temporal.A_log" in model.state_dict()
    with pytest.raises(RuntimeError):
        _model().load_state_dict(model.state_dict())


def test_trainer_and_forecaster_run_it(tmp_path):
    from mpgcn_amd.serve import Forecaster

    torch.manual_seed(0)
    params = {
        "model": "MPGCN", "device": "cpu", "synthetic_nodes": 12, "synthetic_days": 60, "norm": "none",
        "split_ratio": [6.4, 1.6, 2], "batch_size": 8, "obs_len": 5, "pred_len": 1, "hidden_dim": 8,
        "kernel_type": "random_walk_diffusion", "cheby_order": 2, "loss": "MSE", "optimizer": "Adam",
        "learn_rate": 1e-3, "decay_rate": 0, "num_epochs": 1, "seed": 0, "output_dir": str(tmp_path),
        "temporal": "selective",
    }
    data = DataInput(params).load_data()
    params["N"] = data["OD"].shape[1]
    loaders = DataGenerator(5, 1, params["split_ratio"]).get_data_loader(data, params)
    trainer = ModelTrainer(params, data)
    assert isinstance(trainer.model.branch_models[0]["temporal"], SelectiveEncoder)
    trainer.train(loaders, ["train", "validate"])
    fc = Forecaster({**params, "checkpoint": str(tmp_path / "MPGCN_od.pkl")}, data)
    out = fc.forecast(torch.rand(5, 12, 12), dow=2, horizon=3)
    assert out.shape == (3, 12, 12) and torch.isfinite(out).all()


def test_command_line_names_it():
    import Main

    parser = Main.build_parser()
    assert parser.parse_args([]).temporal == "lstm"
    assert parser.parse_args(["-temporal", "selective"]).temporal == "selective"


# ---- GPU --------------------------------------------------------------------

DEV = "cuda:0"


@pytest.mark.gpu
@pytest.mark.parametrize("H,N,taps,R,T", [(32, 16, 4, 300, 7), (16, 5, 3, 33, 14), (32, 16, 4, 5, 1)])
def test_encoder_on_gpu_f32(H, N, taps, R, T):
    """Outputs and gradients in f32 against the formulas in f64. Every value
    goes through some 100 roundings of 2^-24 on its longest path and the sums
    over R T rows add with them: within 1e-4 of the largest gradient."""
    torch.manual_seed(1)
    enc = SelectiveEncoder(1, H, N, taps)
    x, d = torch.rand(R, T), torch.randn(R, H)
    ref = SelectiveEncoder(1, H, N, taps).double()
    ref.load_state_dict(enc.state_dict())
    hr = _by_hand(ref, x.double())
    hr.backward(d.double())
    enc = enc.to(DEV)
    h = enc(x.to(DEV))
    torch.testing.assert_close(h.detach().cpu().double(), hr.detach(), rtol=1e-4, atol=1e-4)
    h.backward(d.to(DEV))
    for (k, p), q in zip(enc.named_parameters(), ref.parameters()):
        tol = 1e-4 * float(q.grad.abs().max()) + 1e-6
        assert float((p.grad.cpu().double() - q.grad).abs().max()) <= tol, k


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_encoder_steps_on_gpu(dtype):
    torch.manual_seed(2)
    enc = SelectiveEncoder(1, 32).to(DEV)
    x = torch.rand(70, 10, device=DEV).to(dtype)
    with torch.no_grad():
        want = [enc(x[:, :t]) for t in (8, 9, 10)]
    h, state = enc.start(x[:, :8])
    got = [h] + [enc.step(x[:, t], state) for t in (8, 9)]
    # the same kernels' arithmetic in another order of sums: in bf16 a rounding
    # of an intermediate may fall the other way, a step of 2^-7 of its size
    tol = 1e-4 if dtype == torch.float32 else 2.0 ** -5
    for a, b in zip(got, want):
        torch.testing.assert_close(a.float(), b.float(), rtol=tol, atol=tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_model_on_gpu(dtype):
    torch.manual_seed(3)
    N = 32
    model = _model(N, 32, compute_dtype=dtype, temporal="selective").to(DEV)
    opt = torch.optim.Adam(model.parameters(), lr=1e-3)
    x, y = torch.rand(2, 7, N, N, 1, device=DEV), torch.rand(2, 1, N, N, 1, device=DEV)
    graphs = _graphs(N, 2, DEV)
    for _ in range(2):
        opt.zero_grad()
        loss = torch.nn.functional.mse_loss(model(x, graphs), y)
        loss.backward()
        assert all(torch.isfinite(p.grad).all() for p in model.parameters())
        opt.step()
    if dtype == torch.float32:
        ref = _model(N, 32, temporal="selective")
        ref.load_state_dict({k: v.cpu() for k, v in model.state_dict().items()})
        with torch.no_grad():
            torch.testing.assert_close(model(x, graphs).cpu(), ref(x.cpu(), _graphs(N, 2)), rtol=1e-3, atol=1e-3)


@pytest.mark.gpu
def test_served_by_graph_replay(tmp_path):
    from mpgcn_amd.serve import Forecaster

    N = 32
    params = {
        "synthetic_nodes": N, "synthetic_days": 60, "seed": 0, "split_ratio": [7, 1.5, 1.5], "norm": "none",
        "hidden_dim": 32, "kernel_type": "random_walk_diffusion", "cheby_order": 2, "device": DEV,
        "compute_dtype": "bf16", "checkpoint": str(tmp_path / "MPGCN_od.pkl"), "temporal": "selective",
    }
    data = DataInput(params=params).load_data()
    torch.manual_seed(0)
    model = _model(N, 32, compute_dtype=torch.bfloat16, temporal="selective")
    torch.save({"epoch": 1, "state_dict": model.state_dict()}, params["checkpoint"])
    fc = Forecaster(params, data)
    torch.manual_seed(11)
    for dow in (0, 3, 5):
        x = torch.rand(7, N, N)
        got = fc.forecast(x, dow=dow, horizon=3)
        # the same operands without the graph
        graphs = fc._dyn_g_list(torch.tensor([dow], device=DEV))
        cur, want = x[None, ..., None].to(DEV), []
        with torch.no_grad():
            for _ in range(3):
                want.append(fc.model(x_seq=cur, G_list=graphs))
                cur = torch.cat([cur[:, 1:], want[-1]], dim=1)
        assert torch.equal(got, torch.cat(want, dim=1)[0, :, :, :, 0].cpu())
    assert fc._use_graph
