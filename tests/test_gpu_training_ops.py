"""The training operators' calls without autograd (ethos_b200.ops) refuse what
the library could only read out of bounds: host tensors, operands that do not
belong together, gradients of another size."""

import pytest
import torch

from ethos_b200 import _lib, functional as EF, ops


@pytest.fixture
def xent():
    g = torch.Generator().manual_seed(1)
    h, W = (torch.randn(n, 24, generator=g).bfloat16().cuda() for n in (10, 40))
    y = torch.randint(0, 40, (10,), generator=g).cuda()
    loss, save = ops.linear_cross_entropy_forward(h, W, y)
    return h, W, torch.ones_like(loss), save


@pytest.mark.gpu
def test_cross_entropy_backward_refuses_operands_that_do_not_belong_together(xent):
    h, W, one, save = xent
    back = ops.linear_cross_entropy_backward
    for wrong in (W.float(), W[:, :16], W[0]):
        with pytest.raises(ValueError, match="weight"):
            back(one, h, wrong, save)
    with pytest.raises(ValueError, match="weight"):
        back(one, h.float(), W, save)
    with pytest.raises(RuntimeError, match="no CPU path"):
        back(one, h, W, save.cpu())
    with pytest.raises(RuntimeError, match="no CPU path"):
        back(one, h, W, None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        back(one.cpu(), h, W, save)
    with pytest.raises(ValueError, match="reduction"):
        back(one, h, W, save, reduction="max")
    for wrong, red in ((torch.ones(9, device="cuda"), "none"), (torch.ones(2, device="cuda"), "sum"),
                       (torch.ones(0, device="cuda"), "mean")):
        with pytest.raises(ValueError, match="grad of"):
            back(wrong, h, W, save, reduction=red)
    dh, dw = back(one, h, W, save)
    assert dh.shape == h.shape and dw.shape == W.shape


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 40, 400])
def test_cross_entropy_backward_with_another_problems_save(T):
    """Sizes that the save buffer shows are refused; labels of a larger table
    (whose size it does not hold) are reported and left out instead of read
    past the smaller one's end; the other tokens keep their label's terms."""
    g = torch.Generator().manual_seed(T)
    h, W = (torch.randn(n, 24, generator=g).bfloat16().cuda() for n in (T, 1 << 20))
    y = torch.full((T,), (1 << 20) - 1).cuda()
    y[0] = 7
    loss, save = ops.linear_cross_entropy_forward(h, W, y, reduction="none")
    one, back = torch.ones(T, device="cuda"), ops.linear_cross_entropy_backward
    for bad_h, bad_grad in ((h[:T - 4].repeat(65, 1), one[:1].expand(65 * (T - 4))), (h.repeat(1, 9), one)):
        with pytest.raises(ValueError, match="save"):
            back(bad_grad, bad_h, W[:, :1].expand(-1, bad_h.shape[1]), save, "none")
    small = W[:100].clone()
    dh, dw = back(one, h, small, save, "none")
    with pytest.raises(_lib.EthosError):
        ops.check_device_error("cuda")
    assert torch.isfinite(dh.float()).all() and torch.isfinite(dw.float()).all()
    want = -small[7].float()  # the other 99 words have next to none of the larger table's probability
    assert (dh[0].float() - want).norm() <= 0.02 * want.norm()


@pytest.mark.gpu
def test_scale_refuses_and_takes_any_float_factor():
    x = torch.arange(8, device="cuda", dtype=torch.float32)
    two = torch.full((), 2.0, device="cuda")
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.scale_(two, x.cpu())
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.scale_(two, x, x.cpu())
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.scale_(two.cpu(), x)
    with pytest.raises(ValueError, match="one value"):
        ops.scale_(torch.ones(0, device="cuda"), x)
    with pytest.raises(ValueError, match="contiguous"):
        ops.scale_(two, x[::2])
    with pytest.raises(ValueError, match="fp32 or bf16"):
        ops.scale_(two, x.half())
    ops.scale_(two.bfloat16(), x)    # read as what it is, not as fp32
    assert torch.equal(x, 2.0 * torch.arange(8, device="cuda"))


@pytest.mark.gpu
def test_balance_backward_refuses():
    w = torch.rand(6, 2, 4, device="cuda")
    ids = torch.zeros(6, 2, 4, dtype=torch.int32, device="cuda")
    loss, _, scratch = ops.balance_forward(w, ids, 5)
    one = torch.ones((), device="cuda")
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.balance_backward(one, scratch.cpu(), (6, 2, 4), 5, torch.float32)
    with pytest.raises(ValueError, match="one value"):
        ops.balance_backward(one[None][:0], scratch, (6, 2, 4), 5, torch.float32)
    with pytest.raises(_lib.EthosError, match="WORKSPACE"):
        ops.balance_backward(one, scratch, (6000, 2, 4), 5, torch.float32)
    assert ops.balance_backward(one, scratch, (6, 2, 4), 5, torch.float32).shape == (6, 2, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("padding", [None, 0, 6, -1, -7])
def test_embedding_backward_takes_padding_rows_as_the_module_does(padding):
    """A negative index counts from the end, in the call without autograd as
    in functional.embedding."""
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, 7, (50,), generator=g).cuda()
    W, dy = (torch.randn(n, 8, generator=g).cuda() for n in (7, 50))
    W.requires_grad_(True)
    want, = torch.autograd.grad(EF.embedding(ids, W, padding_idx=padding), W, dy)
    assert torch.equal(ops.embedding_backward(ids, dy, 7, padding_idx=padding), want)
    assert padding is None or not want[padding].any()


@pytest.mark.gpu
@pytest.mark.parametrize("padding", [7, -8, 1 << 40])
def test_embedding_backward_refuses_padding_rows_outside_the_table(padding):
    ids, dy = torch.zeros(3, dtype=torch.int64, device="cuda"), torch.ones(3, 8, device="cuda")
    with pytest.raises(ValueError, match="padding_idx"):
        ops.embedding_backward(ids, dy, 7, padding_idx=padding)
