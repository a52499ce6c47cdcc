"""The region-sharded model with selective temporal encoders: two ranks over
gloo against the whole model."""

import os

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from mpgcn_amd.graph import build_supports
from mpgcn_amd.models import MPGCN

N, K, H, B, T = 8, 3, 16, 2, 5
P = 2


def _model():
    torch.manual_seed(1)
    return MPGCN(M=2, K=K, input_dim=1, lstm_hidden_dim=H, lstm_num_layers=1, gcn_hidden_dim=H, gcn_num_layers=3,
                 num_nodes=N, temporal="selective")


def _inputs():
    g = torch.Generator().manual_seed(0)
    x, y, flow = (torch.rand(*s, generator=g) for s in ((B, T, N, N, 1), (B, 1, N, N, 1), (B, N, N)))
    sup = build_supports(torch.rand(1, N, N, generator=g), "random_walk_diffusion", K - 1)[0]
    return x, y, [sup, (build_supports(flow, "random_walk_diffusion", K - 1),
                        build_supports(flow.transpose(-2, -1), "random_walk_diffusion", K - 1))]


def _worker(rank, pg_file, out_file):
    from mpgcn_amd.parallel.region import mpgcn_forward_sharded, shard_dest

    os.environ.update(RANK=str(rank), WORLD_SIZE=str(P), LOCAL_RANK=str(rank))
    dist.init_process_group("gloo", init_method=f"file://{pg_file}", rank=rank, world_size=P)
    model = _model()
    x, y, graphs = _inputs()
    out = mpgcn_forward_sharded(model, shard_dest(x, rank, P), graphs)
    torch.nn.functional.mse_loss(out, shard_dest(y, rank, P)).backward()
    for p in model.parameters():
        dist.all_reduce(p.grad)
        p.grad /= P
    torch.save({"out": out.detach(), "grads": {n: p.grad.clone() for n, p in model.named_parameters()}},
               f"{out_file}.{rank}")
    dist.destroy_process_group()


@pytest.mark.timeout(300)
def test_sharded_selective_model_matches_the_whole(tmp_path):
    ctx = mp.get_context("spawn")
    procs = [ctx.Process(target=_worker, args=(r, str(tmp_path / "pg"), str(tmp_path / "out"))) for r in range(P)]
    for p in procs:
        p.start()
    for p in procs:
        p.join(timeout=240)
        assert p.exitcode == 0
    got = [torch.load(tmp_path / f"out.{r}", weights_only=True) for r in range(P)]
    model = _model()
    x, y, graphs = _inputs()
    ref = model(x, graphs)
    torch.nn.functional.mse_loss(ref, y).backward()
    # the same f32 sums in another order
    torch.testing.assert_close(torch.cat([g["out"] for g in got], dim=-2), ref.detach(), atol=1e-5, rtol=1e-5)
    for n, p in model.named_parameters():
        torch.testing.assert_close(got[0]["grads"][n], p.grad, atol=1e-5, rtol=1e-4, msg=n)
