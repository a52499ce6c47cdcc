"""row_gemm with inner widths that are no multiple of the MFMA depth, on LDS
that an earlier kernel left full of NaN."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("K", [1, 5, 16, 24, 40])
def test_row_gemm_tail_reads_no_leftovers(K):
    from mpgcn_amd import ops

    ext = ops.get_ext()
    g = torch.Generator().manual_seed(K)
    bad = torch.full((256, 128), float("nan"), device="cuda:0", dtype=torch.bfloat16)
    X0 = torch.ones(64 * 2048, 256, device="cuda:0", dtype=torch.bfloat16)
    X = torch.randn(64 * 2048, K, generator=g).to(torch.bfloat16).to("cuda:0")
    W = torch.randn(K, 64, generator=g).to(torch.bfloat16).to("cuda:0")
    for _ in range(3):
        ext.row_gemm(X0, bad, None, False)
        out = ext.row_gemm(X, W, None, False)
        ref = X.float() @ W.float()
        # K products and sums in f32, then half a step of bf16
        tol = 2.0 ** -8 * ref.abs() + (K + 1) * 2.0 ** -23 * (X.float().abs() @ W.float().abs())
        assert ((out.float() - ref).abs() <= tol).all()
