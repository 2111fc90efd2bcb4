"""The training operators together: EthosDecoder.loss, and the gradient that
reaches the router through the layer's routing weights.

Bars: those of the paths they run in -- 1e-4 for fp32 parameters, 1e-2 for one
bf16 layer (tests/test_gpu_split_backward.py), 3e-2 for the whole bf16 decoder
(tests/test_decoder.py).  The loss itself is an fp32 mean of 96 tokens; in fp32
it differs from the logits' cross entropy by roundings of the logits, 1e-5."""

import pytest
import torch
import torch.nn.functional as F

from ethos_b200 import EthosConfig, EthosExpertLayer, _lib, functional as EF, ops
from ethos_b200.init import seeded_input, seeded_state_dict, tensor_generator
from helpers import dims_of, grad_names, load_golden, oracle_grads, rel_err
from oracle import ethos_oracle as orc
from test_decoder import _decoder

CFG1 = dict(d_model=512, num_experts=4096, top_k=16, num_routing_heads=8, d_latent=128,
            d_intermediate_hypernet=512, d_query=512)


def _layer(dtype, training, seed=3):
    layer = EthosExpertLayer(EthosConfig(**CFG1))
    sd = seeded_state_dict(layer, seed=seed)
    g = torch.Generator().manual_seed(11)
    for k in sd:
        if k.endswith("running_var"):
            sd[k] = 0.5 + torch.rand(sd[k].shape, generator=g)
        elif ".query_norms." in k and k.endswith((".weight", ".bias")):
            sd[k] = (1.0 if k.endswith(".weight") else 0.0) + 0.1 * torch.randn(sd[k].shape, generator=g)
    layer.load_state_dict(sd)
    return layer.to("cuda", dtype).train(training), sd


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [(torch.bfloat16, 1e-2), (torch.float32, 1e-4)])
@pytest.mark.parametrize("training", [False, True])
def test_routing_weights_carry_gradients(dtype, tol, training):
    """A loss on the routing weights alone, and one on the output and the
    weights together, against autograd through the oracle on the same ids."""
    T, H, k = 256, 8, 16
    layer, sd = _layer(dtype, training)
    bf = dtype == torch.bfloat16
    rnd = (lambda t: t.to(torch.bfloat16).float()) if bf else (lambda t: t)
    x = rnd(seeded_input(T, 512, seed=21))
    dw = torch.randn((T, H, k), generator=tensor_generator(7, "dw")) * 0.1
    gy = rnd(torch.randn((T, 512), generator=tensor_generator(5, "gy")))
    for with_y in (False, True):
        xg = x.to("cuda", dtype).view(2, T // 2, 512).requires_grad_(True)
        layer.zero_grad(set_to_none=True)
        y, w, ids = layer(xg, return_routing=True)
        assert y.shape == xg.shape and w.shape == (T, H, k) and w.dtype == torch.float32
        assert ids.dtype == torch.int32 and not ids.requires_grad
        loss = (w * dw.cuda()).sum()
        if with_y:
            loss = loss + (y.view(T, -1) * gy.to("cuda", dtype)).float().sum()
        loss.backward()
        ops.check_device_error("cuda")

        p = orc.params_from_state_dict(sd, dims_of(CFG1), round_bf16=bf)
        p.requires_grad_(True)
        xr = x.clone().requires_grad_(True)
        i64 = ids.cpu().to(torch.int64)
        if with_y:
            yr, wr, _ = orc.layer_forward_given_ids(xr, p, i64, training=training)
            ((wr * dw).sum() + (yr * gy).sum()).backward()
        else:
            wr, _ = orc.router_weights_given_ids(xr, p, i64, training)
            (wr * dw).sum().backward()
        assert rel_err(xg.grad.view(T, -1).float().cpu(), xr.grad) <= tol
        ref, got = oracle_grads(p, H), dict(layer.named_parameters())
        for name in grad_names(H).values():
            if training and "query_projs" in name and name.endswith(".bias"):
                continue  # the batch mean absorbs the bias
            want = ref[name]
            if want is None:  # the experts take no part in the routing weights
                assert not got[name].grad.any(), name
                continue
            assert rel_err(got[name].grad.float().cpu(), want) <= tol, name


@pytest.mark.gpu
def test_routing_outputs_leave_the_layer_as_it_was():
    layer, _ = _layer(torch.bfloat16, False)
    x = seeded_input(64, 512, seed=2).to("cuda", torch.bfloat16).view(1, 64, 512)
    with torch.no_grad():
        y = layer(x)
        y2, w, ids = layer(x, return_routing=True)
        scores, ids64 = layer.router(x.view(64, 512))
    assert torch.equal(y, y2) and torch.equal(ids.long(), ids64)
    assert torch.equal(w.to(torch.bfloat16), scores)
    xg = x.clone().requires_grad_(True)
    layer(xg).sum().backward()
    xr = x.clone().requires_grad_(True)
    layer(xr, return_routing=True)[0].sum().backward()
    assert torch.equal(xg.grad, xr.grad)
    with pytest.raises(ValueError, match="d_weights"):
        out = ops.layer_forward(x.view(64, 512), layer._packed(x.device), False, 1e-5, 0.1, save=True)
        ops.layer_backward(y.view(64, 512), x.view(64, 512), layer._packed(x.device), out, False, 1e-5,
                           d_weights=torch.zeros(63, 8, 16, device="cuda"))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,loss_tol,tol", [(torch.float32, 1e-5, 1e-4), (torch.bfloat16, 1e-2, 3e-2)])
def test_decoder_loss_matches_the_logits_loss(dtype, loss_tol, tol):
    rec = load_golden("decoder")
    model = _decoder(rec).to("cuda", dtype).train()
    ids = rec["input_ids"].cuda()
    labels = torch.roll(ids, -1, 1)
    labels[:, -1] = -100
    labels[0, :10] = -100
    model.zero_grad(set_to_none=True)
    want = F.cross_entropy(model(ids).float().view(-1, rec["model_cfg"]["vocab_size"]), labels.view(-1))
    want.backward()
    grads = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad(set_to_none=True)
    loss, parts = model.loss(ids, labels)
    loss.backward()
    ops.check_device_error("cuda")
    assert abs(loss.item() - want.item()) <= loss_tol * want.item()
    assert parts["cross_entropy"].item() == loss.item() and set(parts) == {"cross_entropy"}
    for n, p in model.named_parameters():
        if grads[n].float().norm() < 1e-6 * max(g.float().norm().item() for g in grads.values()):
            continue  # the projections' biases: the batch mean absorbs them
        assert rel_err(p.grad.float(), grads[n].float()) <= tol, n


@pytest.mark.gpu
def test_decoder_loss_with_balance():
    rec = load_golden("decoder")
    model = _decoder(rec).to("cuda", torch.float32).train()
    ids = rec["input_ids"].cuda()
    labels = torch.roll(ids, -1, 1)
    mask = torch.ones_like(ids, dtype=torch.bool)
    mask[1, 30:] = False
    seen = []
    hook = model.layers[1].post_attention_layernorm.register_forward_hook(lambda m, i, o: seen.append(o.detach()))
    loss, parts = model.loss(ids, labels, balance_coef=0.5, mask=mask)
    hook.remove()
    loss.backward()
    ops.check_device_error("cuda")
    router = model.layers[1].mlp.router
    g_bal = router.sub_keys_1.weight.grad.clone()
    w, eid = router(seen[0].reshape(-1, rec["model_cfg"]["d_model"]))
    want, counts = EF.balance_loss(w, eid, 4096, mask=mask.view(-1))
    assert abs(parts["balance"][0].item() - want.item()) <= 1e-5 * want.item()
    assert torch.equal(parts["expert_counts"][0], counts) and counts.sum().item() == int(mask.sum()) * 128
    assert abs(loss.item() - parts["cross_entropy"].item() - 0.5 * want.item()) <= 1e-5 * loss.item()
    model.zero_grad(set_to_none=True)
    model.loss(ids, labels)[0].backward()
    # the balance term reached the router, and only through it
    assert rel_err(g_bal, router.sub_keys_1.weight.grad) > 1e-3


@pytest.mark.gpu
def test_training_steps_reduce_the_loss():
    from ethos_b200.optim import FusedAdamW
    rec = load_golden("decoder")
    model = _decoder(rec).to("cuda", torch.bfloat16).train()
    opt = FusedAdamW(model.parameters(), lr=1e-3, max_grad_norm=1.0)
    ids = rec["input_ids"].cuda()
    labels = torch.roll(ids, -1, 1)
    losses = []
    for _ in range(8):
        loss, parts = model.loss(ids, labels, balance_coef=0.01)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(parts["cross_entropy"].item())
    ops.check_device_error("cuda")
    assert all(torch.isfinite(torch.tensor(losses))) and losses[-1] < 0.8 * losses[0]


@pytest.mark.gpu
def test_operators_in_a_cuda_graph():
    """Forward and backward of the three operators captured once and replayed
    on new inputs give what the eager calls give."""
    g = torch.Generator().manual_seed(1)
    V, d, T, N = 3000, 256, 700, 4096
    W = torch.randn(V, d, generator=g).mul_(d ** -0.5).bfloat16().cuda().requires_grad_(True)
    ids, labels = (torch.randint(0, V, (T,), generator=g).cuda() for _ in range(2))
    rw = torch.softmax(torch.randn(T, 8, 16, generator=g), -1).cuda().requires_grad_(True)
    rid = torch.randint(0, N, (T, 8, 16), generator=g).cuda()

    def step():
        ce = EF.linear_cross_entropy(EF.embedding(ids, W, scale=16.0), W, labels)
        bal, counts = EF.balance_loss(rw, rid, N)
        dW, drw = torch.autograd.grad(ce + 0.1 * bal, (W, rw))
        return ce.detach(), bal.detach(), counts, dW, drw

    for keep in (True, False):
        old, EF._keeping_pays = EF._keeping_pays, lambda *a: keep  # noqa: B023
        try:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                captured = step()
            for seed in (2, 3):
                g2 = torch.Generator().manual_seed(seed)
                ids.copy_(torch.randint(0, V, (T,), generator=g2))
                labels.copy_(torch.randint(0, V, (T,), generator=g2))
                labels[: 100 * seed] = -100
                rid.copy_(torch.randint(0, N, (T, 8, 16), generator=g2))
                graph.replay()
                for a, b in zip(captured, step()):
                    assert torch.equal(a, b)
        finally:
            EF._keeping_pays = old
    ops.check_device_error("cuda")


@pytest.mark.gpu
def test_a_gradient_cannot_be_differentiated():
    ids = torch.tensor([1, 2, 2], device="cuda")
    W = torch.randn(5, 8, device="cuda", requires_grad=True)
    w3 = torch.rand(3, 1, 1, device="cuda", requires_grad=True)
    h = torch.randn(3, 8, device="cuda", requires_grad=True)
    for out, x in ((EF.embedding(ids, W).sum(), W), (EF.balance_loss(w3, ids.view(3, 1, 1), 5)[0], w3),
                   (EF.linear_cross_entropy(h, W, ids), h)):
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(out, x, create_graph=True, retain_graph=True)
        torch.autograd.grad(out, x)


@pytest.mark.gpu
def test_only_the_gradient_asked_for_is_formed():
    """Both operands require a gradient, one is asked for; and a second pass
    through the same graph gives the first one's values (up to the way)."""
    g = torch.Generator().manual_seed(5)
    h = torch.randn(300, 64, generator=g).cuda().requires_grad_()
    W = torch.randn(1000, 64, generator=g).cuda().requires_grad_()
    y = torch.randint(0, 1000, (300,), generator=g).cuda()
    both = torch.autograd.grad(EF.linear_cross_entropy(h, W, y), (h, W))
    loss = EF.linear_cross_entropy(h, W, y)
    dh, = torch.autograd.grad(loss, h, retain_graph=True)
    dw, = torch.autograd.grad(loss, W)
    assert torch.equal(dh, both[0]) and torch.equal(dw, both[1])


def test_binding_loads_and_reports():
    """The C++ nodes load without a GPU, and their messages hold numbers."""
    nodes = _lib.training()
    with pytest.raises(RuntimeError, match="device 64"):
        nodes.set_error_word(64, 0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        EF.embedding(torch.zeros(3, dtype=torch.long), torch.zeros(5, 8))
