"""Cross entropy of the output head (functional.linear_cross_entropy,
ethos_xent_forward / _backward) against a plain fp64 implementation on the
same operands.

Bounds, from the arithmetic.  A logit is a sum of d products accumulated in
fp32 by the matrix unit, which loses at most one ulp (2^-23) of the running sum
per step of 16; with the six plane products of fp32 operands there are 6 d / 16
steps, of which the d / 16 last ones see the whole sum.  So a logit is within
e_l = (d / 16 + 8) 2^-23 A of exact, A the largest sum of |products| of a row.
The loss is a difference of two values with that error, plus the exponentials
(2^-22 each) and its rounding.  A probability then has relative error 2 e_l +
2^-21.  Gradients compare in the norm: the logits' gradient is rounded to bf16
(2^-9 relative; fp32 operands: 2^-23), summed in fp32 with again up to one ulp
per step, and rounded to the output type; per-element errors relative to the
values add up to
  rel <= 2 e_l + 2^-21 + s 2^-23 C + (bf16: 2 * 2^-9)
where s is the number of steps of the longer contraction and C the cancellation
sum|terms| / |sum| in the norm, computed from the fp64 gradient."""

import ctypes

import pytest
import torch

from ethos_b200 import _lib, functional as EF, ops


def _inputs(T, V, d, dtype, seed, ignored=0.0, sharp=8.0):
    g = torch.Generator().manual_seed(seed)
    W = torch.randn(V, d, generator=g) * d ** -0.5
    y = torch.randint(0, V, (T,), generator=g)
    h = torch.randn(T, d, generator=g) + W[y] * torch.rand(T, 1, generator=g) * sharp
    y[torch.rand(T, generator=g) < ignored] = -100
    return h.to(dtype), W.to(dtype), y


def _exact(h, W, y, reduction, grad=None, ignore=-100):
    """fp64 loss, gradients, and the quantities of the bounds."""
    h, W = h.double(), W.double()
    live = y != ignore
    at = torch.where(live, y, 0)
    l = h @ W.t()
    logp = torch.log_softmax(l, 1)
    rows = torch.where(live, -logp.gather(1, at[:, None])[:, 0], 0.0)
    n = int(live.sum())
    loss = {"none": rows, "sum": rows.sum(), "mean": rows.sum() / n if n else torch.tensor(float("nan"))}[reduction]
    g = {"none": grad.double() if grad is not None else None, "sum": torch.ones(len(y)).double(),
         "mean": torch.full((len(y),), 1.0 / max(n, 1)).double()}[reduction]
    g = torch.where(live, g if g is not None else 0.0, 0.0)
    p = logp.exp()
    p[torch.arange(len(y)), at] -= 1.0
    dl = p * g[:, None]
    mags = (h.abs() @ W.abs().t()).max().item()
    e_l = (h.shape[1] / 16 + 8) * 2.0 ** -23 * mags
    return loss, dl @ W, dl.t() @ h, dict(e_l=e_l, ch=(dl.abs() @ W.abs(), dl @ W), cw=(dl.abs().t() @ h.abs(), dl.t() @ h),
                                          rows=rows)


def _loss_bound(q):
    return 2 * q["e_l"] + 2.0 ** -20 + 2.0 ** -23 * q["rows"].abs().max().item()


def _grad_bound(q, key, steps, dtype):
    mag, val = q[key]
    cancel = (mag.norm() / val.norm()).item() if val.norm() > 0 else 1.0
    # the label's entry p - 1 carries the error of p, relative to 1 - p: in the norm at most that of the others
    rel = (2 * q["e_l"] + 2.0 ** -21 + steps * 2.0 ** -23) * cancel
    return rel + (2 * 2.0 ** -9 if dtype == torch.bfloat16 else 2.0 ** -22)


def _rel(got, want):
    den = want.norm().item()
    return (got.double().cpu() - want).norm().item() / (den if den > 0 else 1.0)


CASES = [
    # T, V, d, ignored: one token and one word; row tiles of one, two, many; columns that end inside a
    # tile; widths that need packing, several K blocks; enough rows for compaction
    (1, 1, 1, 0.0), (1, 300, 64, 0.0), (7, 257, 33, 0.3), (255, 1000, 128, 0.0), (256, 511, 72, 0.5),
    (257, 513, 200, 0.0), (700, 2049, 136, 0.6), (1030, 777, 1031, 0.1), (600, 5003, 320, 0.9),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("T,V,d,ignored", CASES)
def test_loss_and_gradients(T, V, d, ignored, reduction, dtype):
    h, W, y = _inputs(T, V, d, dtype, seed=T + V, ignored=ignored)
    if ignored < 1.0:
        y[0] = V - 1
    g = torch.rand(T, generator=torch.Generator().manual_seed(1)) + 0.5 if reduction == "none" else None
    want, dh_w, dw_w, q = _exact(h, W, y, reduction, g)
    hg, wg = h.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    loss = EF.linear_cross_entropy(hg, wg, y.cuda(), reduction=reduction)
    assert loss.dtype == torch.float32 and loss.shape == want.shape
    scale = T if reduction == "sum" else 1
    assert (loss.detach().double().cpu() - want).abs().max() <= scale * _loss_bound(q) + 2.0 ** -23 * want.abs().max()
    dh, dw = torch.autograd.grad(loss, (hg, wg), None if g is None else g.cuda())
    ops.check_device_error("cuda")
    assert dh.dtype == dtype and dw.dtype == dtype
    if V == 1:  # one word is certain: no gradient
        assert not dh.any() and not dw.any()
        return
    assert _rel(dh, dh_w) <= _grad_bound(q, "ch", min(V, 32 * 64) / 16, dtype)
    assert _rel(dw, dw_w) <= _grad_bound(q, "cw", T / 16, dtype)
    assert not dh[(y == -100).cuda()].any()


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("T,V,d,ignored", CASES)
def test_loss_and_gradients_in_one_call(T, V, d, ignored, reduction):
    """The keeping way at every size (functional.linear_cross_entropy takes it
    for larger problems only), and each gradient alone."""
    h, W, y = _inputs(T, V, d, torch.bfloat16, seed=T + V, ignored=ignored)
    y[0] = V - 1
    want, dh_w, dw_w, q = _exact(h, W, y, reduction)
    args = (h.cuda(), W.cuda(), y.cuda(), -100, reduction)
    loss, _, dh, dw = ops.linear_cross_entropy_forward_backward(*args)
    ops.check_device_error("cuda")
    scale = T if reduction == "sum" else 1
    assert abs(loss.item() - want) <= scale * _loss_bound(q) + 2.0 ** -23 * abs(want)
    assert torch.equal(ops.linear_cross_entropy_forward_backward(*args, need_weight=False)[2], dh)
    assert torch.equal(ops.linear_cross_entropy_forward_backward(*args, need_hidden=False)[3], dw)
    if V == 1:
        assert not dh.any() and not dw.any()
        return
    assert _rel(dh, dh_w) <= _grad_bound(q, "ch", V / 16, torch.bfloat16)
    assert _rel(dw, dw_w) <= _grad_bound(q, "cw", T / 16, torch.bfloat16)
    assert not dh[(y == -100).cuda()].any()


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [5, 30, 400])
def test_every_token_ignored(T, dtype, keep, monkeypatch):
    monkeypatch.setattr(EF, "_keeping_pays", lambda *a: keep)
    h, W, y = _inputs(T, 90, 24, dtype, seed=2, ignored=2.0)
    for reduction in ("mean", "sum", "none"):
        hg, wg = h.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
        loss = EF.linear_cross_entropy(hg, wg, y.cuda(), reduction=reduction)
        if reduction == "mean":
            assert torch.isnan(loss)
        else:
            assert not loss.any()
        dh, dw = torch.autograd.grad(loss.sum(), (hg, wg))
        assert not dh.any() and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pieces_of_the_vocabulary(dtype):
    """More columns than one piece holds: 70 000 tokens x 20 000 words are two
    pieces of bf16.  The gradients of a few rows and words against fp64."""
    T, V, d = (70000, 20000, 16) if dtype == torch.bfloat16 else (24000, 20000, 16)
    h, W, y = _inputs(T, V, d, dtype, seed=3, ignored=0.2)
    hg, wg = h.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    loss = EF.linear_cross_entropy(hg, wg, y.cuda(), reduction="sum")
    dh, dw = torch.autograd.grad(loss, (hg, wg))
    with torch.no_grad():
        h64, w64 = hg.double(), wg.double()
        live = (y != -100).cuda()
        at = torch.where(live, y.cuda(), 0)
        total, dw_w, e_l = 0.0, torch.zeros(V, d, dtype=torch.float64, device="cuda"), 0.0
        for a in range(0, T, 4000):
            l = h64[a:a + 4000] @ w64.t()
            e_l = max(e_l, (h64[a:a + 4000].abs() @ w64.abs().t()).max().item() * 9 * 2.0 ** -23)
            logp = torch.log_softmax(l, 1)
            lv, ab = live[a:a + 4000], at[a:a + 4000]
            total -= (logp.gather(1, ab[:, None])[:, 0] * lv).sum().item()
            p = logp.exp_()
            p.scatter_add_(1, ab[:, None], torch.full((len(ab), 1), -1.0, dtype=torch.float64, device="cuda"))
            p *= lv[:, None]
            bound = 2 * e_l + 2.0 ** -21 + V / 16 * 2.0 ** -23 + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22)
            want = p @ w64
            assert (dh[a:a + 4000].double() - want).norm() <= 4 * bound * want.norm()
            dw_w += p.t() @ h64[a:a + 4000]
    bound = 2 * e_l + 2.0 ** -21 + T / 16 * 2.0 ** -23 + (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -22)
    assert (dw.double() - dw_w).norm() <= 4 * bound * dw_w.norm()
    assert abs(loss.item() - total) <= (2 * e_l + 2.0 ** -20) * T


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 300])
def test_extreme_logits(T):
    """Logits of +-2000 (far outside the exponential's range), rows whose
    label is certain or hopeless, rows of equal logits."""
    V, d = 700, 8
    W = torch.zeros(V, d)
    W[:, 0] = torch.linspace(-1, 1, V)
    W[5, 1] = 1.0
    h = torch.zeros(T, d)
    h[0, 0] = 2000.0
    h[1, 1] = 2000.0
    y = torch.full((T,), 5)
    y[0] = V - 1
    for dtype in (torch.bfloat16, torch.float32):
        hd, wd = h.to(dtype), W.to(dtype)
        want, dh_w, dw_w, q = _exact(hd, wd, y, "none", torch.ones(T))
        hg, wg = hd.cuda().requires_grad_(True), wd.cuda().requires_grad_(True)
        loss = EF.linear_cross_entropy(hg, wg, y.cuda(), reduction="none")
        assert torch.isfinite(loss).all()
        assert (loss.detach().double().cpu() - want).abs().max() <= _loss_bound(q)
        dh, dw = torch.autograd.grad(loss.sum(), (hg, wg))
        assert torch.isfinite(dh.float()).all() and torch.isfinite(dw.float()).all()
        # the rows of equal logits: p = 1 / V everywhere
        assert _rel(dh[2:], dh_w[2:]) <= 2 * 2.0 ** -9
        # a hopeless label the other way round: loss = the whole gap
        y2 = y.clone()
        y2[0] = 0
        loss = EF.linear_cross_entropy(hg, wg, y2.cuda(), reduction="none")
        assert abs(loss[0].item() - _exact(hd, wd, y2, "none", torch.ones(T))[0][0].item()) <= _loss_bound(q)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [6, 300, 900])
def test_hopeless_labels_with_gradients(T):
    """bf16, gradients in the forward call: rows whose largest logit passes
    the label's by hundreds (the exponentials are then taken relative to the
    largest), next to rows that need no such thing, in one row tile and in
    several.  Operand values are exact in bf16, logits whole numbers."""
    V, d = 1100, 16
    W = torch.zeros(V, d)
    W[:, 0] = (torch.arange(V) % 17).float()
    W[:, 1] = (torch.arange(V) % 5).float()
    g = torch.Generator().manual_seed(12)
    h = torch.zeros(T, d)
    h[:, 1] = torch.randint(0, 3, (T,), generator=g).float()
    y = torch.randint(0, V, (T,), generator=g)
    h[1::7, 0] = 40.0      # gaps of up to 640 between logits
    h[3, 0] = 4.0          # 64: just over the range
    y[3] = 17              # logit 0 in column 0 (17 % 17)
    h, W = h.bfloat16(), W.bfloat16()
    for reduction in ("sum", "mean"):
        want, dh_w, dw_w, q = _exact(h, W, y, reduction)
        loss, _, dh, dw = ops.linear_cross_entropy_forward_backward(h.cuda(), W.cuda(), y.cuda(), reduction=reduction)
        scale = T if reduction == "sum" else 1
        assert abs(loss.item() - want) <= scale * _loss_bound(q) + 2.0 ** -23 * abs(want)
        assert _rel(dh, dh_w) <= _grad_bound(q, "ch", V / 16, torch.bfloat16)
        assert _rel(dw, dw_w) <= _grad_bound(q, "cw", T / 16, torch.bfloat16)


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [True, False])
def test_gradient_of_the_loss_scales_and_second_pass(keep, monkeypatch):
    """The loss inside a larger expression, and two passes through its graph
    (the second finds the first's gradients untouched)."""
    monkeypatch.setattr(EF, "_keeping_pays", lambda *a: keep)
    h, W, y = _inputs(400, 900, 64, torch.bfloat16, seed=13, ignored=0.3)
    hg, wg = h.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    _, dh_w, dw_w, q = _exact(h, W, y, "mean")
    loss = EF.linear_cross_entropy(hg, wg, y.cuda())
    a = torch.autograd.grad(0.3 * loss, (hg, wg), retain_graph=True)
    keep = [t.clone() for t in a]
    b = torch.autograd.grad(loss, (hg, wg))
    for got, want, key, steps, f in ((a[0], dh_w, "ch", 900 / 16, 0.3), (a[1], dw_w, "cw", 400 / 16, 0.3),
                                     (b[0], dh_w, "ch", 900 / 16, 1.0), (b[1], dw_w, "cw", 400 / 16, 1.0)):
        # 0.3 is one more rounding to bf16
        assert _rel(got, f * want) <= _grad_bound(q, key, steps, torch.bfloat16) + 2.0 ** -9
    assert all(torch.equal(x, z) for x, z in zip(a, keep))
    with torch.no_grad():
        assert torch.equal(EF.linear_cross_entropy(hg, wg, y.cuda(), reduction="none").sum() > 0,
                           torch.tensor(True, device="cuda"))


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_rows():
    h, W, y = _inputs(300, 600, 32, torch.float32, seed=4)
    h[7, 3], h[9, 0] = float("nan"), float("inf")
    y[11] = -100
    h[11] = float("nan")   # an ignored token's state does not matter
    hg = h.cuda().requires_grad_(True)
    loss = EF.linear_cross_entropy(hg, W.cuda(), y.cuda(), reduction="none")
    bad = torch.zeros(300, dtype=torch.bool)
    bad[7] = bad[9] = True
    assert torch.equal(torch.isnan(loss.detach()).cpu(), bad)
    dh, = torch.autograd.grad(loss.sum(), hg)
    assert torch.equal(torch.isnan(dh).any(1).cpu(), bad) and not dh[11].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [5, 200, 300])
def test_what_an_ignored_token_holds_reaches_no_gradient(T, dtype):
    """NaN, infinity or zeros in the states of ignored tokens: the same loss
    and gradients, by every way."""
    h, W, y = _inputs(T, 515, 72, dtype, seed=T)
    y[1] = y[3] = -100
    for reduction in ("none", "mean"):
        got = []
        for fill in (0.0, float("nan"), float("inf")):
            h[1] = h[3] = fill
            hg, wg = h.cuda().requires_grad_(), W.cuda().requires_grad_()
            loss = EF.linear_cross_entropy(hg, wg, y.cuda(), reduction=reduction)
            got.append((loss.detach(), *torch.autograd.grad(loss.sum(), (hg, wg))))
            if reduction == "mean":
                both = ops.linear_cross_entropy_forward_backward(h.cuda(), W.cuda(), y.cuda())
                if both is not None:
                    got[-1] += (both[0], both[2], both[3])
        assert all(torch.isfinite(t.float()).all() for t in got[0])
        for other in got[1:]:
            assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [2, 9, 300])
def test_nan_in_one_word_reaches_every_token(T, dtype):
    for word in (0, 77, 499):
        h, W, y = _inputs(T, 500, 64, dtype, seed=14)
        y[:] = 5
        W[word, 3] = float("nan")
        assert torch.isnan(EF.linear_cross_entropy(h.cuda(), W.cuda(), y.cuda(), reduction="none")).all()
        if dtype == torch.bfloat16:
            loss, _, dh, _ = ops.linear_cross_entropy_forward_backward(h.cuda(), W.cuda(), y.cuda())
            assert torch.isnan(loss) and torch.isnan(dh).any(1).all()


@pytest.mark.gpu
def test_strides_labels_types_streams_and_repeats():
    h, W, y = _inputs(320, 515, 64, torch.bfloat16, seed=5, ignored=0.2)
    base = EF.linear_cross_entropy(h.cuda(), W.cuda(), y.cuda(), reduction="none")
    # rows inside wider buffers, an odd offset, a transposed copy, int32 labels
    hb = torch.zeros(320, 100, dtype=torch.bfloat16, device="cuda")
    hb[:, 3:67] = h.cuda()
    wb = torch.zeros(515, 77, dtype=torch.bfloat16, device="cuda")
    wb[:, 5:69] = W.cuda()
    yi = torch.stack([y, y], 1).to(torch.int32).cuda()[:, 0]
    assert torch.equal(EF.linear_cross_entropy(hb[:, 3:67], wb[:, 5:69], yi, reduction="none"), base)
    assert torch.equal(EF.linear_cross_entropy(h.cuda().t().contiguous().t(), W.cuda(), y.cuda(), reduction="none"), base)
    # leading dimensions; another stream; the same bits in every run
    assert torch.equal(EF.linear_cross_entropy(h.cuda().view(2, 160, 64), W.cuda(), y.cuda().view(2, 160),
                                               reduction="none"), base.view(2, 160))
    s = torch.cuda.Stream()
    hg, wg = h.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    s.wait_stream(torch.cuda.current_stream())
    grads = []
    with torch.cuda.stream(s):
        for _ in range(3):
            loss = EF.linear_cross_entropy(hg, wg, y.cuda())
            grads.append((loss.detach(), *torch.autograd.grad(loss, (hg, wg))))
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for g in grads[1:]:
        assert all(torch.equal(a, b) for a, b in zip(g, grads[0]))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [40, 300])
def test_gradients_against_differences(T):
    """A central difference of the fp32 loss along random directions.  Its
    truncation error is h^2/6 of the third derivative, which for a softmax is
    at most (largest change of a logit)^3; its rounding error 2 loss bounds
    over 2 h."""
    h, W, y = _inputs(T, 300, 24, torch.float32, seed=6, ignored=0.1)
    g = torch.Generator().manual_seed(7)
    uh, uw = torch.randn(h.shape, generator=g) * 0.1, torch.randn(W.shape, generator=g) * 0.1
    hg, wg = h.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    loss = EF.linear_cross_entropy(hg, wg, y.cuda())
    dh, dw = torch.autograd.grad(loss, (hg, wg))
    q = _exact(h, W, y, "mean")[3]
    step = 2.0 ** -5
    for u, which in ((uh, 0), (uw, 1)):
        vals = []
        for s in (step, -step):
            a = h + s * u if which == 0 else h
            b = W + s * u if which == 1 else W
            vals.append(EF.linear_cross_entropy(a.cuda(), b.cuda(), y.cuda()).item())
        num = (vals[0] - vals[1]) / (2 * step)
        ana = ((dh, dw)[which].double().cpu() * u.double()).sum().item()
        spread = (u.double() @ W.double().t()).abs().max() if which == 0 else (h.double() @ u.double().t()).abs().max()
        assert abs(num - ana) <= step ** 2 / 6 * (2 * spread.item()) ** 3 + _loss_bound(q) / step


@pytest.mark.gpu
def test_labels_out_of_range_are_reported_and_left_out():
    h, W, y = _inputs(280, 100, 16, torch.bfloat16, seed=8)
    for T in (20, 280):
        for bad in (100, -1, 1 << 40):
            yb = y[:T].clone()
            yb[4] = bad
            ok = y[:T].clone()
            ok[4] = -100
            loss = EF.linear_cross_entropy(h[:T].cuda(), W.cuda(), yb.cuda())
            with pytest.raises(_lib.EthosError) as e:
                ops.check_device_error("cuda")
            assert e.value.status == 16
            assert torch.equal(loss, EF.linear_cross_entropy(h[:T].cuda(), W.cuda(), ok.cuda()))
    # another ignore_index, inside the vocabulary
    y2 = torch.where(y == 3, 4, y)
    y2[::7] = 3
    y3 = torch.where(y2 == 3, -100, y2)
    assert torch.equal(EF.linear_cross_entropy(h.cuda(), W.cuda(), y2.cuda(), ignore_index=3),
                       EF.linear_cross_entropy(h.cuda(), W.cuda(), y3.cuda()))
    ops.check_device_error("cuda")


@pytest.mark.gpu
def test_one_gradient_only_and_no_tokens():
    h, W, y = _inputs(300, 200, 40, torch.bfloat16, seed=9)
    hg, wg = h.cuda().requires_grad_(True), W.cuda().requires_grad_(True)
    dh, dw = torch.autograd.grad(EF.linear_cross_entropy(hg, wg, y.cuda()), (hg, wg))
    assert torch.equal(torch.autograd.grad(EF.linear_cross_entropy(hg, W.cuda(), y.cuda()), hg)[0], dh)
    assert torch.equal(torch.autograd.grad(EF.linear_cross_entropy(h.cuda(), wg, y.cuda()), wg)[0], dw)
    # twice through one graph
    loss = EF.linear_cross_entropy(hg, wg, y.cuda())
    a = torch.autograd.grad(loss, hg, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(3.0 * loss, hg)[0].float(), (3.0 * a.float()).to(torch.bfloat16).float()) or \
        _rel(torch.autograd.grad(3.0 * EF.linear_cross_entropy(hg, wg, y.cuda()), hg)[0], 3.0 * a.double().cpu()) <= 2.0 ** -8
    empty = torch.zeros(0, 40, dtype=torch.bfloat16, device="cuda").requires_grad_(True)
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert EF.linear_cross_entropy(empty, wg, none, reduction="none").shape == (0,)
    loss = EF.linear_cross_entropy(empty, wg, none, reduction="sum")
    assert loss.item() == 0.0
    de, dw0 = torch.autograd.grad(loss, (empty, wg))
    assert de.shape == (0, 40) and not dw0.any()
    assert torch.isnan(EF.linear_cross_entropy(empty, wg, none))


@pytest.mark.gpu
def test_backward_in_a_thread_without_a_context():
    """A thread's first CUDA work is the backward, and its memory comes from
    the caching allocator (as in autograd's worker)."""
    import threading
    h, W, y = (t.cuda() for t in _inputs(300, 2000, 64, torch.bfloat16, seed=11, ignored=0.5))
    loss, save = ops.linear_cross_entropy_forward(h, W, y)
    one = torch.ones((), device="cuda")
    want = ops.linear_cross_entropy_backward(one, h, W, save)
    del loss
    again = [t.clone() for t in want]
    del want  # its blocks, and the workspace's, are in the cache now
    got = []
    t = threading.Thread(target=lambda: got.extend(ops.linear_cross_entropy_backward(one, h, W, save)))
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert len(got) == 2 and all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8])
def test_few_tokens(T, dtype):
    """The one-pass forward of up to eight tokens: vocabularies that leave
    shares of one row or none, widths of whole and of partial lane steps, in
    and out of alignment, ignored tokens, and its agreement with nine tokens
    (which take the matrix units)."""
    for V, d in ((1, 8), (31, 256), (3001, 264), (5000, 100), (9001, 515), (700, 1024)):
        h, W, y = _inputs(9, V, d, dtype, seed=V + T, sharp=4.0)
        y[1] = -100
        want, _, _, q = _exact(h[:T], W, y[:T], "none", torch.ones(T))
        got = EF.linear_cross_entropy(h[:T].cuda(), W.cuda(), y[:T].cuda(), reduction="none")
        assert (got.double().cpu() - want).abs().max() <= _loss_bound(q), (V, d)
        wide = torch.zeros(V, d + 5, dtype=dtype, device="cuda")
        wide[:, 2:d + 2] = W.cuda()
        again = EF.linear_cross_entropy(h[:T].cuda(), wide[:, 2:d + 2], y[:T].cuda(), reduction="none")
        assert (again.double().cpu() - want).abs().max() <= _loss_bound(q), (V, d)
        nine = EF.linear_cross_entropy(h.cuda(), W.cuda(), y.cuda(), reduction="none")[:T]
        assert (nine.double().cpu() - want).abs().max() <= _loss_bound(q), (V, d)
    h, W, y = _inputs(T, 400, 64, dtype, seed=T)
    h[0, 0], W[7, 1] = float("inf"), 0.0
    assert torch.isnan(EF.linear_cross_entropy(h.cuda(), W.cuda(), y.cuda(), reduction="none")[0])
    ops.check_device_error("cuda")
    y[0] = 400
    EF.linear_cross_entropy(h.cuda(), W.cuda(), y.cuda())
    with pytest.raises(_lib.EthosError):
        ops.check_device_error("cuda")


@pytest.mark.gpu
def test_refusals():
    h, W, y = (t.cuda() for t in _inputs(10, 20, 8, torch.float32, seed=10))
    with pytest.raises(RuntimeError, match="no CPU path"):
        EF.linear_cross_entropy(h.cpu(), W, y)
    with pytest.raises(RuntimeError, match="no CPU path"):
        EF.linear_cross_entropy(h, W, y.cpu())
    with pytest.raises(ValueError, match="fp32 or bf16"):
        EF.linear_cross_entropy(h.half(), W.half(), y)
    with pytest.raises(ValueError, match="weight"):
        EF.linear_cross_entropy(h, W.bfloat16(), y)
    with pytest.raises(ValueError, match="got"):
        EF.linear_cross_entropy(h, W[:, :4], y)
    with pytest.raises(ValueError, match="belong"):
        EF.linear_cross_entropy(h, W, y[:5])
    with pytest.raises(ValueError, match="reduction"):
        EF.linear_cross_entropy(h, W, y, reduction="max")
    with pytest.raises(ValueError, match="int32 or int64"):
        EF.linear_cross_entropy(h, W, y.float())


def test_entry_point_argument_checks():
    L = _lib.lib()
    v = ctypes.c_void_p(256)
    T, V, d = 300, 1000, 64
    save, fwd, bwd = (f(T, V, d, 1) for f in (L.ethos_xent_save_size, L.ethos_xent_forward_workspace_size,
                                               L.ethos_xent_backward_workspace_size))
    assert save >= 512 * (64 * 2 + 16) and fwd >= 512 * 8 and bwd >= 512 * (1024 * 2 + 64 * 4)
    assert L.ethos_xent_save_size(0, V, d, 1) == 0 and L.ethos_xent_save_size(T, V, d, 5) == 0
    # workspace of the pieces stays bounded: 16 384 x 100 277 logits are 3.3 GB of bf16
    assert L.ethos_xent_backward_workspace_size(16384, 100277, 1024, 1) < 1.2 * 2 ** 30

    def forward(**o):
        a = dict(h=v, ldh=d, w=v, ldw=d, dt=1, y=v, i64=1, ig=-100, red=2, T=T, V=V, d=d, loss=v, save=v, sb=save,
                 ws=v, wb=fwd, err=v, st=None)
        a.update(o)
        return L.ethos_xent_forward(*a.values())

    assert forward(h=None) == 1 and forward(y=None) == 1 and forward(loss=None) == 1 and forward(red=3) == 1
    assert forward(ldh=d - 1) == 1 and forward(T=0) == 1 and forward(dt=2) == 1
    assert forward(V=1 << 25) == 2 and forward(T=1 << 25) == 2
    assert forward(sb=save - 1024) == 4 and forward(ws=None) == 4 and forward(wb=64) == 4
    assert forward(w=ctypes.c_void_p(264)) == 3 and forward(ldw=d + 4) == 3

    def backward(**o):
        a = dict(h=v, ldh=d, w=v, ldw=d, dt=1, red=2, T=T, V=V, d=d, g=v, save=v, sb=save, dh=v, dw=v, ws=v, wb=bwd,
                 err=v, st=None)
        a.update(o)
        return L.ethos_xent_backward(*a.values())

    both = L.ethos_xent_forward_backward_workspace_size(T, V, d, 1)
    assert both >= 512 * 1024 * 2
    assert L.ethos_xent_forward_backward_workspace_size(T, V, d, 0) == 0            # fp32
    assert L.ethos_xent_forward_backward_workspace_size(16384, 100277, 1024, 1) < 4.5 * 2 ** 30
    assert L.ethos_xent_forward_backward_workspace_size(1 << 20, 100277, 1024, 1) == 0

    def fb(**o):
        a = dict(h=v, ldh=d, w=v, ldw=d, dt=1, y=v, i64=1, ig=-100, red=2, T=T, V=V, d=d, loss=v, save=v, sb=save,
                 dh=v, dw=v, ws=v, wb=both, err=v, st=None)
        a.update(o)
        return L.ethos_xent_forward_backward(*a.values())

    assert fb(red=0) == 1 and fb(y=None) == 1 and fb(dt=0) == 2 and fb(wb=64) == 4 and fb(sb=0) == 4
    assert fb(ldw=d + 4) == 3
    assert L.ethos_xent_scale(None, v, 4, None, 0, 1, None) == 1 and L.ethos_xent_scale(v, None, 4, None, 0, 1, None) == 1
    assert L.ethos_xent_scale(v, v, 0, None, 0, 1, None) == 0
    assert backward(g=None) == 1 and backward(save=None) == 4 and backward(wb=64) == 4
    assert backward(dh=None, dw=None) == 0
