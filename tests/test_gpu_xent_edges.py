"""Cross entropy of the output head where its buffers and its arithmetic can
go wrong: workspaces that hold something else before the call, batches of which
nothing is left, workspaces at every alignment the entry points accept."""

import ctypes

import pytest
import torch

from ethos_b200 import _lib, functional as EF, ops
from test_gpu_xent import _exact, _grad_bound, _inputs, _loss_bound, _rel


@pytest.fixture
def dirty(monkeypatch):
    """Workspaces and save buffers of ops.* calls arrive holding NaN (0xFF in
    every byte, in bf16 and in fp32)."""
    monkeypatch.setattr(ops, "_bytes", lambda n, dev: torch.full((n,), 255, dtype=torch.uint8, device=dev))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,d", [(30, 33), (400, 24), (400, 33), (300, 515), (700, 1031)])
def test_no_token_left_gives_zero_gradients(T, d, dtype, dirty):
    """Every label ignored, widths whose dW goes through padded rows among
    them: zeros, whatever the workspace held."""
    h, W, y = (t.cuda() for t in _inputs(T, 600, d, dtype, seed=2, ignored=2.0))
    for reduction in ("none", "sum", "mean"):
        loss, save = ops.linear_cross_entropy_forward(h, W, y, reduction=reduction)
        grad = torch.ones_like(loss)
        dh, dw = ops.linear_cross_entropy_backward(grad, h, W, save, reduction=reduction)
        assert not dh.any() and not dw.any()
        both = ops.linear_cross_entropy_forward_backward(h, W, y, reduction=reduction)
        assert (both is None) == (dtype == torch.float32 or reduction == "none")
        if both is not None:
            assert not both[2].any() and not both[3].any()
    ops.check_device_error("cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("T,V,d,ignored", [(5, 70, 33, 0.2), (256, 511, 72, 0.5), (300, 777, 515, 0.97),
                                           (700, 2049, 136, 0.6)])
def test_what_the_workspace_held_does_not_matter(T, V, d, ignored, dirty):
    """bf16, both ways: the same bits as with the allocator's memory."""
    h, W, y = (t.cuda() for t in _inputs(T, V, d, torch.bfloat16, seed=T, ignored=ignored))
    y[0] = V - 1
    loss, save = ops.linear_cross_entropy_forward(h, W, y)
    got = (loss, *ops.linear_cross_entropy_backward(torch.ones_like(loss), h, W, save))
    both = ops.linear_cross_entropy_forward_backward(h, W, y)
    for a in (got, (both[0], both[2], both[3])):
        assert all(torch.isfinite(t.float()).all() for t in a)
    want, dh_w, dw_w, q = _exact(h.cpu(), W.cpu(), y.cpu(), "mean")
    for loss, dh, dw in (got, (both[0], both[2], both[3])):
        assert abs(loss.item() - want) <= _loss_bound(q) + 2.0 ** -23 * abs(want)
        assert _rel(dh, dh_w) <= _grad_bound(q, "ch", V / 16, torch.bfloat16)
        assert _rel(dw, dw_w) <= _grad_bound(q, "cw", T / 16, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V,d", [(5, 300, 64), (300, 2049, 136), (40, 777, 33)])
def test_workspaces_at_every_accepted_alignment(T, V, d, dtype, monkeypatch):
    """The entry points take any 16-byte aligned workspace and save buffer (a
    part of a caller's arena): the same bits at 16, 32 and 48 bytes past an
    allocation's start."""
    h, W, y = (t.cuda() for t in _inputs(T, V, d, dtype, seed=T, ignored=0.2))
    y[0] = V - 1
    want = None
    for off in (0, 16, 32, 48):
        def shifted(n, dev, off=off):
            t = torch.empty(n + 64, dtype=torch.uint8, device=dev)[off:off + n]
            assert t.data_ptr() % 64 == off
            return t
        monkeypatch.setattr(ops, "_bytes", shifted)
        loss, save = ops.linear_cross_entropy_forward(h, W, y)
        got = (loss, *ops.linear_cross_entropy_backward(torch.ones_like(loss), h, W, save))
        both = ops.linear_cross_entropy_forward_backward(h, W, y)
        if both is not None:
            got += (both[0], both[2], both[3])
        want = want or got
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    monkeypatch.undo()
    # 8-byte alignment is refused
    L, p = _lib.lib(), ctypes.c_void_p
    save, ws = (ops._bytes(n + 64, h.device) for n in (L.ethos_xent_save_size(T, V, d, 1),
                                                        L.ethos_xent_backward_workspace_size(T, V, d, 1)))
    args = (h.data_ptr(), d, W.data_ptr(), d, 1, 2, T, V, d, loss.data_ptr())
    for a, b in ((0, 8), (8, 0)):
        assert L.ethos_xent_backward(*args, p(save.data_ptr() + a), save.numel() - a, h.data_ptr(), W.data_ptr(),
                                     p(ws.data_ptr() + b), ws.numel() - b, loss.data_ptr(), None) == 3


def _label_only(T, V, d, seed):
    """A problem whose gradients are the label's terms: word 0, a row of
    zeros, has logit 0 and all of the probability, every other word a logit
    of -64 and less, so that with the loss's gradient g
        dh[t] = -g[t] W[y[t]],   dW[v] = -sum over the tokens of label v of g[t] h[t]
    (v > 0) up to e^-60."""
    g = torch.Generator().manual_seed(seed)
    W = torch.randn(V, d, generator=g) * 0.25
    h = torch.randn(T, d, generator=g) * 0.25
    W[:, 0], h[:, 0] = -5.0, 16.0
    W[0] = 0.0
    y = torch.randperm(max(T, V - 1), generator=g)[:T] % (V - 1) + 1
    assert (h @ W[1:].t()).max() < -64
    return h.bfloat16(), W.bfloat16(), y, torch.rand(T, generator=g) + 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("T,V,d", [(40, 300, 64), (256, 600, 33), (300, 700, 136), (700, 2049, 24), (1000, 3000, 515)])
def test_the_labels_terms_are_rounded_once(T, V, d, reduction):
    """bf16, the logits formed again: the label's entry of their gradient,
    g (p - 1), is the largest of a row and reaches both gradients in fp32.
    With one token to a label each result is one product of values of 24 bits
    (p - 1 within 2^-23, one more rounding by g / n and by the product), rounded
    to bf16 once: the rounding of a value within 2^-21 of the exact one."""
    h, W, y, g = _label_only(T, V, d, seed=T)
    ignored = torch.arange(T) % 5 == 3
    y[ignored] = -100
    hc, wc, yc = h.cuda(), W.cuda(), y.cuda()
    loss, save = ops.linear_cross_entropy_forward(hc, wc, yc, reduction=reduction)
    up = g if reduction == "none" else g[0]
    dh, dw = ops.linear_cross_entropy_backward(up.cuda(), hc, wc, save, reduction=reduction)
    coef = {"none": g.double(), "sum": up.double().expand(T),
            "mean": (up.double() / int((~ignored).sum())).expand(T)}[reduction]
    want_h = torch.where(ignored[:, None], 0.0, -coef[:, None] * W.double()[y.clamp(min=0)])
    want_w = torch.zeros(V, d, dtype=torch.float64)
    want_w[y[~ignored]] = -coef[~ignored, None] * h.double()[~ignored]
    rest = torch.ones(V, dtype=torch.bool)
    rest[0] = rest[y[~ignored]] = False
    for got, want in ((dh, want_h), (dw[~rest.cuda()][1:], want_w[~rest][1:])):
        got = got.cpu()
        ok = torch.zeros(got.shape, dtype=torch.bool)
        for f in (1.0 - 2.0 ** -21, 1.0, 1.0 + 2.0 ** -21):
            ok |= got == (want * f).float().to(torch.bfloat16)
        assert ok.all(), f"{int((~ok).sum())} of {ok.numel()}"
    # words that are no token's label: their probabilities, below e^-60 (1e-26)
    assert (dw[rest.cuda()].double().cpu().abs() <= 1e-26 * (coef[:, None] * h.double().abs()).sum(0)).all()
    ops.check_device_error("cuda")


@pytest.mark.gpu
def test_the_labels_terms_over_several_pieces():
    """The same where the vocabulary takes two pieces and labels repeat: sums
    of n fp32 terms, n 2^-24 of their magnitudes, and one rounding to bf16
    (2^-8 of the value at most)."""
    T, V, d = 70000, 20000, 16
    h, W, y, g = (t.cuda() for t in _label_only(T, V, d, seed=1))
    assert ops._size("ethos_xent_backward_workspace_size", T, V, d, 1) < T * V * 2  # not all columns at once
    loss, save = ops.linear_cross_entropy_forward(h, W, y, reduction="none")
    dh, dw = ops.linear_cross_entropy_backward(g, h, W, save, reduction="none")
    want = -g.double()[:, None] * W.double()[y]
    assert ((dh.double() - want).abs() <= (2.0 ** -8 + 2.0 ** -21) * want.abs()).all()
    terms = -g.double()[:, None] * h.double()
    want, mags = (torch.zeros(V, d, dtype=torch.float64, device="cuda").index_add_(0, y, t)
                  for t in (terms, terms.abs()))
    n = torch.bincount(y, minlength=V)[:, None].double()
    bad = (dw.double() - want).abs() > 2.0 ** -8 * want.abs() + (n + 8) * 2.0 ** -24 * mags
    assert not bad[1:].any(), f"{int(bad[1:].sum())} of {bad.numel()}"


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 40, 300])
@pytest.mark.parametrize("gap", [300.0, 30000.0])
def test_a_hopeless_label_leaves_the_other_words_exact(gap, T):
    """fp32: a label whose logit lies far below takes no part in the other
    words' probabilities, so their error is that of their own logits,
    e_l = (d / 16 + 8) 2^-23 A with A from their magnitudes alone: p is within
    2 e_l + 2^-21, and its sums of n terms within n 2^-24 more."""
    V, d = 700, 16
    g = torch.Generator().manual_seed(T)
    h, W = torch.randn(T, d, generator=g), torch.randn(V, d, generator=g)
    W[:, 0], h[:, 0] = 0.0, gap / 10
    W[5] = 0.0
    W[5, 0] = -10.0
    y = torch.full((T,), 5)
    hg, wg = h.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    rest = torch.arange(V) != 5
    others = W[rest][:, 1:].double()
    p = torch.softmax(h[:, 1:].double() @ others.t(), 1)
    e_l = (d / 16 + 8) * 2.0 ** -23 * (h[:, 1:].double().abs() @ others.abs().t()).max().item()
    bound = 2 * e_l + 2.0 ** -21 + max(T, V) * 2.0 ** -24
    for reduction in ("none", "sum"):
        loss = EF.linear_cross_entropy(hg, wg, y.cuda(), reduction=reduction)
        dh, dw = torch.autograd.grad(loss.sum(), (hg, wg))
        mags_h, mags_w = p @ others.abs(), p.t() @ h.double().abs()
        assert ((dh[:, 1:].double().cpu() - p @ others).abs() <= bound * mags_h).all()
        assert ((dw[rest.cuda()].double().cpu() - p.t() @ h.double()).abs() <= bound * mags_w).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("T", [6, 300])
def test_a_second_pass_through_one_graph(T, keep, dtype, monkeypatch):
    """The first pass asks for one gradient, the second, through the same
    graph with another factor, for both: each within the bounds of the formula
    (the factor is one more rounding to bf16)."""
    monkeypatch.setattr(EF, "_keeping_pays", lambda *a: keep)
    h, W, y = _inputs(T, 900, 40, dtype, seed=T, ignored=0.2)
    y[0] = 3
    _, dh_w, dw_w, q = _exact(h, W, y, "mean")
    hg, wg = h.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    loss = EF.linear_cross_entropy(hg, wg, y.cuda())
    first, = torch.autograd.grad(loss, hg, retain_graph=True)
    kept = first.clone()
    dh, dw = torch.autograd.grad(3.0 * loss, (hg, wg), retain_graph=True)
    again, = torch.autograd.grad(loss, wg)
    more = 2.0 ** -9 if dtype == torch.bfloat16 else 2.0 ** -23
    assert _rel(first, dh_w) <= _grad_bound(q, "ch", 900 / 16, dtype) and torch.equal(first, kept)
    assert _rel(dh, 3.0 * dh_w) <= _grad_bound(q, "ch", 900 / 16, dtype) + more
    assert _rel(dw, 3.0 * dw_w) <= _grad_bound(q, "cw", T / 16, dtype) + more
    assert _rel(again, dw_w) <= _grad_bound(q, "cw", T / 16, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [8, 200, 300])
def test_nan_and_infinity_stay_in_their_rows_by_every_way(T, dtype):
    """A token whose state holds NaN or infinity: its loss and its row of dh
    are NaN, every other token's are what they are without it."""
    h, W, y = _inputs(T, 600, 64, dtype, seed=4)
    ok = torch.ones(T, dtype=torch.bool)
    ok[2] = ok[5] = False
    hb = h.clone()
    hb[2, 3], hb[5, 0] = float("nan"), float("inf")
    res = []
    for x in (h, hb):
        loss, save = ops.linear_cross_entropy_forward(x.cuda(), W.cuda(), y.cuda(), reduction="none")
        dh, dw = ops.linear_cross_entropy_backward(torch.ones(T, device="cuda"), x.cuda(), W.cuda(), save, "none")
        both = ops.linear_cross_entropy_forward_backward(x.cuda(), W.cuda(), y.cuda(), reduction="sum")
        res.append((loss, dh) if both is None else (loss, dh, both[2]))
    for clean, bad in zip(*res):
        bad, clean = bad.cpu(), clean.cpu()
        assert torch.equal(bad[ok], clean[ok])
        rows = bad[~ok] if bad.dim() == 1 else bad[~ok].float().isnan().any(1)
        assert rows.isnan().all() if bad.dim() == 1 else rows.all()
