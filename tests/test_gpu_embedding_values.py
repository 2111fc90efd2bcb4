"""Token embedding: what NaN and infinity in the table, in the gradient and in
the rows left out reach, and what they do not."""

import pytest
import torch

from ethos_b200 import functional as EF, ops

NAN, INF = float("nan"), float("inf")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [8, 33, 264])
@pytest.mark.parametrize("T", [7, 1000, 5000])
def test_values_stay_in_their_rows(T, d, dtype):
    V = 97
    g = torch.Generator().manual_seed(T + d)
    ids = torch.randint(4, V, (T,), generator=g)
    ids[0], ids[2], ids[3], ids[5] = 0, 1, 2, 3   # rows 0 to 3 have one token each
    W, dy = torch.randn(V, d, generator=g).to(dtype), torch.randn(T, d, generator=g).to(dtype)
    dy[0, 1], dy[2, d - 1], dy[3, 0] = NAN, INF, -INF
    dy[5] = NAN                                   # the padding row's token
    W[0, 0], W[1, 2], W[50] = INF, NAN, NAN
    wg = W.cuda().requires_grad_(True)
    out = EF.embedding(ids.cuda(), wg, scale=2.0, padding_idx=3)
    assert torch.equal(out.detach().cpu().nan_to_num(7.0), (W[ids].float() * 2.0).to(dtype).nan_to_num(7.0))
    dw = torch.autograd.grad(out, wg, dy.cuda())[0].cpu()
    ops.check_device_error("cuda")
    want = torch.zeros(V, d, dtype=torch.bool)    # where the gradient is not finite
    want[0, 1] = want[1, d - 1] = want[2, 0] = True
    assert torch.equal(~torch.isfinite(dw.float()), want)
    assert torch.isnan(dw[0, 1]) and dw[1, d - 1] == INF and dw[2, 0] == -INF and not dw[3].any()


@pytest.mark.gpu
@pytest.mark.parametrize("V,d", [(3, 5), (4096, 64), (5000, 33)])
def test_rows_without_a_token_are_zero_whatever_was_there(V, d, monkeypatch):
    """Every element of dW is written: memory, the workspace's too, that held
    NaN before the call."""
    monkeypatch.setattr(ops, "_bytes", lambda n, dev: torch.full((n,), 255, dtype=torch.uint8, device=dev))
    ids, dy = torch.tensor([1, 1, 2], device="cuda"), torch.ones(3, d, device="cuda")
    for fill in (0, 1):
        junk = [torch.full((V, d), NAN, device="cuda") for _ in range(8)]
        del junk
        dw = ops.embedding_backward(ids, dy, V, 0.5, padding_idx=2 if fill else None)
        want = torch.zeros(V, d, device="cuda")
        want[1] = 1.0
        want[2] = 0.0 if fill else 0.5
        assert torch.equal(dw, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_table_of_one_row_with_any_stride(dtype):
    """The row pitch of a one-row table means nothing; torch keeps what the
    view had, here 1."""
    col = torch.randn(24, 1, device="cuda").to(dtype)
    W = col.t()
    assert W.shape == (1, 24) and W.stride(0) == 1 and W.is_contiguous()
    ids = torch.zeros(5, dtype=torch.int64, device="cuda")
    assert torch.equal(EF.embedding(ids, W), W.expand(5, 24))
    assert torch.equal(ops.embedding_forward(ids, W), W.expand(5, 24))
