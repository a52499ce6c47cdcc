"""More work than the card has places for at once: a wave or a block takes one
item after another, reading the next while it works on the one before."""

import pytest
import torch

import sequence_oracle as oracle
from mpgcn_amd import ops
from test_sequence_gpu import BF, F, check_scan, conv_case, gen, grads, rn, scan_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,B,L,D,N,G", [
    (BF, 20001, 9, 4, 4, 1),     # 10001 pairs of sequences over 4096 waves, backward over 2048
    (F, 9001, 7, 32, 16, 1),     # one chunk: the state given is read again
    (F, 70, 17, 4096, 5, 1),     # 70 sequences over 64 and 32 waves a channel block
    (BF, 600, 12, 330, 24, 2),   # two quads a channel, groups of 165 channels
])
def test_scan_of_more_items_than_waves(dtype, B, L, D, N, G):
    check_scan(*scan_case(B + L, dtype, B, L, D, N, G, True, torch.int32), dtype)


@pytest.mark.parametrize("dtype,B,L,D,N,G,lengths,softplus", [
    (F, 2, 500, 42, 24, 2, torch.int32, True),   # two quads a channel, groups of 21 channels
    (BF, 1, 600, 60, 30, 3, None, False),
    (F, 3, 410, 36, 13, 4, torch.int64, False),
    (BF, 2, 450, 80, 50, 2, torch.int32, True),
])
def test_segments_of_groups(dtype, B, L, D, N, G, lengths, softplus):
    t, n = scan_case(B + L, dtype, B, L, D, N, G, True, lengths)
    if not softplus:  # a step size as it is: positive, as the decay needs
        t["delta"], t["delta_bias"] = t["delta"].abs() * 0.1, t["delta_bias"].abs() * 0.05
    check_scan(t, n, dtype, softplus)


@pytest.mark.parametrize("B,D,N", [(256, 4096, 16), (300, 2048, 33)])
def test_scan_step_of_more_sequences_than_blocks(B, D, N):
    t, _ = scan_case(B + D, BF, B, 1, D, N, 1, True, None)
    ref = oracle.scan(**t)
    one = {k: v if k in ("A", "skip", "delta_bias") else v[:, 0] for k, v in t.items() if k != "state"}
    y, s = ops.selective_scan_step(**one, state=t["state"], delta_softplus=True)
    oracle.within(y.unsqueeze(1), *ref["y"], oracle.scan_roundings(1, N))
    oracle.within(s, *ref["last"], oracle.scan_roundings(1, N))


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("B,L,D,K", [(1500, 5, 520, 4), (120, 60, 1030, 3)])
def test_conv_of_more_items_than_blocks(dtype, B, L, D, K):
    x, w, b, s, n = conv_case(B, dtype, B, L, D, K, True, torch.int32)
    dy = rn(gen(1), B, L, D, dtype=dtype)
    leaves = [t.requires_grad_() for t in (x, w, b, s)]
    y = ops.short_conv(x, w, b, state=s, lengths=n)
    ref = oracle.conv(x, w, b, s, n, True, dy)
    r = oracle.conv_roundings(K)
    oracle.within(y, *ref["y"], r, "y")
    for name, got in zip(("x", "weight", "bias", "state"), grads([y], [dy], leaves)):
        # a sum over all tokens: one thread's part of them in turn, then its block's rows and the blocks'
        oracle.within(got, *ref[name], r + (B * L // 64 + 256 if name in ("weight", "bias") else 0), name)


def check_norm(seed, R, D, dtype, res, gate, m):
    g = gen(seed)
    t = dict(x=rn(g, R, D, dtype=dtype), gate=rn(g, R, D, dtype=dtype) if gate else None,
             post=rn(g, D) if m.get("post") else None,
             residual=None if res is None else rn(g, R, D, dtype=res, scale=2.0),
             scale=rn(g, D) if m.get("scale") else None, pre=rn(g, D) if m.get("pre") else None)
    leaves = {k: v.requires_grad_() for k, v in t.items() if v is not None}
    out = ops.norm_gate_residual(t["x"], gate=t["gate"], post_weight=t["post"], residual=t["residual"],
                                 scale=t["scale"], pre_weight=t["pre"])
    both = res is not None and m.get("pre")
    out = dict(zip(("y", "h"), out)) if both else {"y" if res is None else "h": out}
    d = {k: rn(g, R, D, dtype=v.dtype) for k, v in out.items()}
    ref = oracle.norm(**t, dy=d.get("y"), dh=d.get("h"))
    r = oracle.norm_roundings(D)
    for k, v in out.items():
        oracle.within(v, *ref[k], r, k)
    for k, v in zip(leaves, grads(list(out.values()), list(d.values()), list(leaves.values()))):
        oracle.within(v, *ref[k], r + (min(R, R // 64 + 256) if k in ("post", "scale", "pre") else 0), k)


MODES = [dict(post=True, scale=True, pre=True), dict(pre=True), dict(post=True)]


@pytest.mark.parametrize("dtype,res", [(BF, None), (F, None), (BF, BF), (BF, F), (F, F), (F, BF)])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("R,D", [(2, 6144), (3, 6145), (2, 6152), (300, 7000), (2, 8192), (2, 8193), (300, 12296)])
def test_norm_of_wide_rows(dtype, res, gate, R, D):
    for m in [dict(post=True)] if res is None else MODES:
        check_norm(R + D, R, D, dtype, res, gate, m)


@pytest.mark.parametrize("dtype,res", [(BF, None), (F, None), (BF, F), (F, F)])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("R,D", [(82001, 32), (82001, 21), (5200, 264)])
def test_norm_of_more_rows_than_threads(dtype, res, gate, R, D):
    """The next row is read while a row is worked on."""
    check_norm(R + D, R, D, dtype, res, gate, dict(post=True) if res is None else MODES[0])
