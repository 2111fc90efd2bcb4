"""What a caller does to the routing weights and ids that the expert layer
hands out (``return_routing``) does not silently change its gradients."""

import pytest
import torch

from ethos_b200.init import seeded_input
from helpers import rel_err
from test_gpu_training_step import _layer


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("change", ["weights", "weights without grad", "ids"])
def test_a_change_in_place_raises_in_the_backward(change, dtype):
    layer, _ = _layer(dtype, False)
    x = seeded_input(64, 512, seed=2).to("cuda", dtype).view(1, 64, 512).requires_grad_(True)
    y, w, ids = layer(x, return_routing=True)
    if change == "weights":
        w.mul_(0.5)
    elif change == "ids":
        ids.zero_()
    else:
        with torch.no_grad():
            w[:, 0] = 0.0
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_change_of_a_copy_changes_nothing(dtype):
    layer, _ = _layer(dtype, False)
    x = seeded_input(64, 512, seed=2).to("cuda", dtype).view(1, 64, 512)
    grads = []
    for touch in (False, True):
        xg = x.clone().requires_grad_(True)
        y, w, ids = layer(xg, return_routing=True)
        if touch:
            (w * 0.5).add_(1.0)
            ids.long().zero_()
            w.detach().clone().zero_()
        (y.float().sum() + (w * w).sum()).backward()
        grads.append(xg.grad)
    # the order of the layer's split sums is the only difference (one rounding of the output type)
    assert rel_err(grads[1].float(), grads[0].float()) <= (2.0 ** -8 if dtype == torch.bfloat16 else 1e-5)


@pytest.mark.gpu
def test_outputs_without_gradients_may_be_changed():
    layer, _ = _layer(torch.bfloat16, False)
    x = seeded_input(64, 512, seed=2).to("cuda", torch.bfloat16).view(1, 64, 512)
    with torch.no_grad():
        y, w, ids = layer(x, return_routing=True)
        kept = y.clone()
        w.mul_(0.5)
        ids.zero_()
        assert torch.equal(layer(x), kept)
