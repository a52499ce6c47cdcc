"""Inference serving: load a reference-format checkpoint, forecast over HTTP.

The reference stops at the offline test loop (Model_Trainer.py:145-185); this
adds the deployment surface a production user needs: a FastAPI app that holds
the model and the day-of-week correlation graphs resident on one GPU and
answers forecast requests with the same autoregressive rollout protocol as
trainer.test() (dynamic graphs held at the first step's day-of-week, kept for
parity with the reference's scoring path).

    uvicorn "mpgcn_amd.serve:create_app" --factory ...
    # or: python -m mpgcn_amd.serve -ckpt out/MPGCN_od.pkl -synthetic-nodes 64

POST /predict  {"x_seq": [[..]], "dow": 3, "horizon": 7}
    x_seq: (T_obs, N, N) nested lists (or with trailing singleton channel);
    dow:   day-of-week index of the first forecast step (graph key, 0-6);
    horizon: number of autoregressive steps (default 1).
    -> {"forecast": (horizon, N, N) nested lists}
GET  /healthz -> {"status": "ok", "regions": N, "device": "..."}
"""

from __future__ import annotations

import argparse

import torch

from mpgcn_amd.graph import build_supports, get_support_K
from mpgcn_amd.models import MPGCN


class Forecaster:
    """Model + resident graphs; the serving core (framework API, no HTTP)."""

    def __init__(self, params: dict, data: dict):
        self.params = params
        self.device = torch.device(params.get("device", "cpu"))
        cd = str(params.get("compute_dtype", "float32"))
        fp8 = cd == "fp8"  # fp8-forward inference (weights stay fp32 masters)
        compute_dtype = (torch.bfloat16 if cd in ("bf16", "bfloat16", "fp8")
                        else torch.float32)
        K = get_support_K(params["kernel_type"], params["cheby_order"])
        N = data["adj"].shape[-1]
        self.N = N
        self.model = MPGCN(
            M=int(params.get("perspectives", 2)), K=K, input_dim=1,
            lstm_hidden_dim=params["hidden_dim"], lstm_num_layers=1,
            gcn_hidden_dim=params["hidden_dim"], gcn_num_layers=3,
            num_nodes=N, compute_dtype=compute_dtype,
            fusion=params.get("fusion", "mean"),
            fp8_forward=fp8,
            temporal=params.get("temporal", "lstm"),
        ).to(self.device)
        ckpt = torch.load(params["checkpoint"], map_location=self.device,
                          weights_only=False)
        self.model.load_state_dict(ckpt["state_dict"])
        self.model.eval()

        from mpgcn_amd.graph.supports import tag_like

        adj = data["adj"].float().to(self.device)
        sup = build_supports(
            adj.unsqueeze(0), params["kernel_type"], params["cheby_order"]
        )
        self.G_static = tag_like(sup.squeeze(0), sup)
        # (N, N, 7) -> per-dow support stacks, built once at startup
        O_dyn = data["O_dyn_G"].permute(2, 0, 1).float().to(self.device)
        D_dyn = data["D_dyn_G"].permute(2, 0, 1).float().to(self.device)
        self.G_o = build_supports(O_dyn, params["kernel_type"], params["cheby_order"])
        self.G_d = build_supports(D_dyn, params["kernel_type"], params["cheby_order"])
        if int(params.get("perspectives", 2)) == 3:
            # third perspective: supports from the day-of-week-AVERAGED OD
            # correlation graph — the same construction the trainer uses
            # (train/trainer.py _graph_list), so a 3-perspective checkpoint is
            # served with the graphs it was trained on
            corr = data["O_dyn_G"].float().mean(dim=-1).to(self.device)
            csup = build_supports(
                corr.unsqueeze(0), params["kernel_type"], params["cheby_order"]
            )
            self.G_corr = tag_like(csup.squeeze(0), csup)

        # hipGraph capture state: obs_len -> (graph, x_static, y_static, dow)
        self._graphs: dict = {}
        self._use_graph = (self.device.type == "cuda"
                           and bool(params.get("capture_graph", True)))
        # FastAPI serves sync endpoints from a threadpool; replays share the
        # static input/output buffers, so the captured path must serialize
        import threading

        self._graph_lock = threading.Lock()

    # ---- hipGraph-captured request path ------------------------------------
    # A serving forward is launch-dense (hundreds of small kernels for one
    # request) while its shapes are fixed per deployment, so on CUDA the
    # forward is captured ONCE per observed obs_len into a hipGraph and every
    # request replays it: x_seq is copied into a static input buffer and the
    # day-of-week is a device int64 scalar the captured index_select re-reads
    # at each replay (the same i_buf pattern bench.py uses for the train
    # step). Falls back to eager on capture failure or off-CUDA.

    def _dyn_g_list(self, dow_buf: torch.Tensor) -> list:
        from mpgcn_amd.graph.supports import tag_like

        go = tag_like(self.G_o.index_select(0, dow_buf), self.G_o)
        gd = tag_like(self.G_d.index_select(0, dow_buf), self.G_d)
        g_list = [self.G_static, (go, gd)]
        if int(self.params.get("perspectives", 2)) == 3:
            g_list.append(self.G_corr)
        return g_list

    def _captured(self, cur: torch.Tensor):
        key = int(cur.shape[1])
        entry = self._graphs.get(key)
        if entry is None:
            xs = cur.clone()
            dow_buf = torch.zeros(1, dtype=torch.long, device=self.device)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):  # allocator/lazy-state warmup
                for _ in range(2):
                    self.model(x_seq=xs, G_list=self._dyn_g_list(dow_buf))
            torch.cuda.current_stream().wait_stream(side)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                ys = self.model(x_seq=xs, G_list=self._dyn_g_list(dow_buf))
            entry = (graph, xs, ys, dow_buf)
            self._graphs[key] = entry
        return entry

    @torch.no_grad()
    def forecast(self, x_seq: torch.Tensor, dow: int, horizon: int = 1) -> torch.Tensor:
        """x_seq: (T, N, N) or (T, N, N, 1) -> (horizon, N, N)."""
        if x_seq.dim() == 3:
            x_seq = x_seq.unsqueeze(-1)
        cur = x_seq.unsqueeze(0).float().to(self.device)  # (1, T, N, N, 1)
        if self._use_graph:
            try:
                with self._graph_lock:
                    graph, xs, ys, dow_buf = self._captured(cur)
            except Exception:  # capture unsupported here — serve eager
                self._use_graph = False
        preds = []
        if self._use_graph:
            with self._graph_lock:
                xs.copy_(cur)
                dow_buf.fill_(dow % 7)
                for _ in range(horizon):
                    graph.replay()
                    step = ys.clone()  # ys is overwritten by the next replay
                    xs.copy_(torch.cat([xs[:, 1:], step], dim=1))
                    preds.append(step)
                return torch.cat(preds, dim=1)[0, :, :, :, 0].cpu()
        g_list = [self.G_static,
                  (self.G_o[dow % 7:dow % 7 + 1], self.G_d[dow % 7:dow % 7 + 1])]
        if int(self.params.get("perspectives", 2)) == 3:
            g_list.append(self.G_corr)
        for _ in range(horizon):
            step = self.model(x_seq=cur, G_list=g_list)  # (1, 1, N, N, 1)
            cur = torch.cat([cur[:, 1:], step], dim=1)
            preds.append(step)
        return torch.cat(preds, dim=1)[0, :, :, :, 0].cpu()


def create_app(params: dict | None = None, data: dict | None = None):
    """FastAPI app factory; params/data as in ModelTrainer (tests inject both)."""
    from fastapi import FastAPI, HTTPException

    if params is None:
        params, data = _params_from_cli()
    fc = Forecaster(params, data)
    app = FastAPI(title="mpgcn-amd forecast service")

    @app.get("/healthz")
    def healthz():
        return {"status": "ok", "regions": fc.N, "device": str(fc.device)}

    @app.post("/predict")
    def predict(payload: dict):
        try:
            x = torch.tensor(payload["x_seq"], dtype=torch.float32)
            dow = int(payload.get("dow", 0))
            horizon = int(payload.get("horizon", 1))
        except (KeyError, ValueError, TypeError) as e:
            raise HTTPException(status_code=422, detail=str(e))
        if x.dim() not in (3, 4) or x.shape[-2] != fc.N or horizon < 1:
            raise HTTPException(status_code=422, detail="bad x_seq shape/horizon")
        out = fc.forecast(x, dow, horizon)
        return {"forecast": out.tolist()}

    return app


def _params_from_cli():
    from mpgcn_amd.data import DataInput

    ap = argparse.ArgumentParser()
    ap.add_argument("-ckpt", "--checkpoint", required=True)
    ap.add_argument("-in", "--input_dir", default="../data")
    ap.add_argument("-synthetic-nodes", "--synthetic_nodes", type=int, default=0)
    ap.add_argument("-synthetic-days", "--synthetic_days", type=int, default=425)
    ap.add_argument("-device", "--device", default="cuda:0")
    ap.add_argument("-hidden", "--hidden_dim", type=int, default=32)
    ap.add_argument("-kernel", "--kernel_type", default="random_walk_diffusion")
    ap.add_argument("-K", "--cheby_order", type=int, default=2)
    ap.add_argument("-dtype", "--compute_dtype", default="bf16")
    ap.add_argument("-M", "--perspectives", type=int, default=2)
    ap.add_argument("-temporal", "--temporal", choices=["lstm", "selective"],
                    default="lstm")
    ap.add_argument("-split", "--split_ratio", type=float, nargs="+",
                    default=[6.4, 1.6, 2])
    ap.add_argument("-port", "--port", type=int, default=8321)
    args = ap.parse_args()
    params = args.__dict__
    data = DataInput(params=params).load_data()
    return params, data


if __name__ == "__main__":
    import uvicorn

    params, data = _params_from_cli()
    uvicorn.run(create_app(params, data), host="127.0.0.1", port=params["port"])
