"""Balance loss and per-expert counts (functional.balance_loss,
ethos_balance_forward / _backward).

Bounds.  Counts are whole numbers and must be equal.  The loss sums products
rounded to fp32 (2^-24 each) in fp64 and is rounded once: 2^-22 relative, all
terms being positive.  The gradient is one fp32 coefficient times a count: 3
roundings, 2^-22 relative, and 2^-8 for bf16."""

import ctypes

import pytest
import torch

from ethos_b200 import _lib, functional as EF, ops


def _inputs(T, H, k, N, seed, skew=2.0):
    g = torch.Generator().manual_seed(seed)
    ids = (torch.rand(T, H, k, generator=g, dtype=torch.float64) ** skew * N).long().clamp_(max=N - 1)
    w = torch.softmax(torch.randn(T, H, k, generator=g), -1)
    return w, ids


def _reference(w, ids, N, mask):
    """The definition, in fp64: fractions of selections times mean weights."""
    T, H, k = w.shape
    m = torch.ones(T, dtype=torch.bool) if mask is None else mask
    n = int(m.sum())
    flat = ids[m].reshape(-1)
    counts = torch.bincount(flat, minlength=N)
    if n == 0:
        return 0.0, counts, torch.zeros(T, H, k, dtype=torch.float64)
    mass = torch.bincount(flat, weights=w[m].double().reshape(-1), minlength=N)
    f = counts.double() / (n * H * k)
    loss = N * (f * mass / (n * H)).sum()
    return float(loss), counts, f[ids] * (N / (n * H)) * m[:, None, None]


CASES = [(1, 1, 1, 1), (1, 8, 16, 262144), (257, 3, 5, 1001), (2048, 8, 16, 4096), (4097, 8, 16, 262144),
         (33, 1, 4, 7),
         (6001, 8, 16, 120001), (150001, 1, 3, 777)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,itype", [(torch.float32, torch.int32), (torch.bfloat16, torch.int64)])
@pytest.mark.parametrize("masked", [None, 0.4, 1.0])
@pytest.mark.parametrize("T,H,k,N", CASES)
def test_loss_counts_and_gradient(T, H, k, N, masked, dtype, itype):
    w, ids = _inputs(T, H, k, N, seed=T + N)
    w = w.to(dtype)
    mask = None if masked is None else torch.rand(T, generator=torch.Generator().manual_seed(1)) >= masked
    want, counts, grad = _reference(w, ids, N, mask)
    wg = w.cuda().requires_grad_(True)
    loss, c = EF.balance_loss(wg, ids.to(itype).cuda(), N, mask=None if mask is None else mask.cuda())
    assert loss.dtype == torch.float32 and c.dtype == torch.int32 and not c.requires_grad
    assert torch.equal(c.cpu().long(), counts)
    assert abs(loss.item() - want) <= 2.0 ** -22 * abs(want)
    dw, = torch.autograd.grad(0.01 * loss, wg)
    ops.check_device_error("cuda")
    assert dw.dtype == dtype
    grad = grad * float(torch.tensor(0.01))
    bound = (2.0 ** -22 + (2.0 ** -8 if dtype == torch.bfloat16 else 0.0)) * grad.abs()
    assert ((dw.double().cpu() - grad).abs() <= bound).all()


@pytest.mark.gpu
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("T,N,itype", [(65537, 262144, torch.int32), (65537, 262139, torch.int64),
                                       (40009, 40001, torch.int32)])
def test_many_selections_of_one_expert(T, N, itype, masked):
    """Blocks that see one expert more often than a 16-bit counter holds, and
    the pass that adds up the blocks' counters."""
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(0, N, (T, 8, 16), generator=g)
    ids[:, :5] = N - 2
    ids, w = ids.to(itype).cuda(), torch.rand(T, 8, 16, generator=g).cuda().requires_grad_()
    mask = (torch.rand(T, generator=g) >= 0.1).cuda() if masked else None
    m = mask if masked else torch.ones(T, dtype=torch.bool, device="cuda")
    n = int(m.sum())
    want = torch.bincount(ids[m].flatten().long(), minlength=N)
    loss, counts = EF.balance_loss(w, ids, N, mask=mask)
    assert torch.equal(counts.long(), want)
    sel = want.double()[ids.long()] * m[:, None, None] * (N / (n * 8) ** 2 / 16)
    assert abs(loss.item() - float((sel * w.detach().double()).sum())) <= 2.0 ** -22 * loss.item()
    dw, = torch.autograd.grad(loss, w)
    assert ((dw.double() - sel).abs() <= 2.0 ** -22 * sel).all()
    ops.check_device_error("cuda")


@pytest.mark.gpu
def test_even_choice_gives_one():
    N, H, k = 64, 2, 4
    ids = torch.arange(N * 8, device="cuda").remainder(N).view(-1, H, k)
    loss, counts = EF.balance_loss(torch.full(ids.shape, 1.0 / k, device="cuda"), ids, N)
    assert abs(loss.item() - 1.0) <= 2.0 ** -22 and (counts == 8).all()


@pytest.mark.gpu
def test_no_tokens_and_views():
    loss, counts = EF.balance_loss(torch.zeros(0, 2, 4, device="cuda"),
                                   torch.zeros(0, 2, 4, dtype=torch.int64, device="cuda"), 16)
    assert loss.item() == 0.0 and counts.sum().item() == 0
    w, ids = _inputs(50, 4, 8, 99, seed=3)
    wv, iv = w.cuda().transpose(0, 1).contiguous().transpose(0, 1), ids.cuda().flip(0).flip(0)
    assert not wv.is_contiguous()
    want, counts, _ = _reference(w, ids, 99, None)
    loss, c = EF.balance_loss(wv, iv, 99)
    assert abs(loss.item() - want) <= 2.0 ** -22 * want and torch.equal(c.cpu().long(), counts)


@pytest.mark.gpu
def test_weights_of_masked_tokens_do_not_matter():
    for T in (40, 5000):
        w, ids = _inputs(T, 8, 16, 500, seed=9)
        mask = torch.arange(T) % 3 != 0
        bad_w, bad_ids = w.clone(), ids.clone()
        bad_w[~mask] = float("nan")
        bad_ids[~mask] = 1 << 40    # not looked at either
        a = EF.balance_loss(w.cuda(), ids.cuda(), 500, mask=mask.cuda())
        wg = bad_w.cuda().requires_grad_(True)
        b = EF.balance_loss(wg, bad_ids.cuda(), 500, mask=mask.cuda())
        ops.check_device_error("cuda")
        assert torch.equal(a[0], b[0].detach()) and torch.equal(a[1], b[1])
        dw, = torch.autograd.grad(b[0], wg)
        assert torch.isfinite(dw).all() and not dw[~mask.cuda()].any()


@pytest.mark.gpu
def test_same_in_every_run():
    w, ids = _inputs(3000, 8, 16, 4096, seed=4)
    w, ids = w.cuda(), ids.cuda()
    runs = [EF.balance_loss(w, ids, 4096)[0].item() for _ in range(4)]
    assert len(set(runs)) == 1


@pytest.mark.gpu
def test_gradient_against_differences():
    """The loss is linear in the weights for fixed choices, so a central
    difference has no truncation error, only the roundings of the two losses."""
    w, ids = _inputs(64, 2, 4, 50, seed=5)
    u = torch.randn(w.shape, generator=torch.Generator().manual_seed(6)).cuda()
    wg, ids = w.cuda().requires_grad_(True), ids.cuda()
    loss, _ = EF.balance_loss(wg, ids, 50)
    dw, = torch.autograd.grad(loss, wg)
    h = 2.0 ** -3
    with torch.no_grad():
        num = (EF.balance_loss(wg + h * u, ids, 50)[0].double() - EF.balance_loss(wg - h * u, ids, 50)[0].double())
    mags = (dw.double().abs() * (wg.double().abs() + h * u.double().abs())).sum()
    assert abs(num / (2 * h) - (dw.double() * u.double()).sum()) <= 2.0 ** -21 * mags / h


@pytest.mark.gpu
def test_ids_out_of_range_are_reported_and_left_out():
    w, ids = _inputs(20, 2, 4, 30, seed=7)
    bad = ids.clone()
    bad[3, 1, 2], bad[4, 0, 0] = 30, -1
    loss, counts = EF.balance_loss(w.cuda(), bad.cuda(), 30)
    with pytest.raises(_lib.EthosError) as e:
        ops.check_device_error("cuda")
    assert e.value.status == 16
    assert counts.sum().item() == ids.numel() - 2


@pytest.mark.gpu
def test_refusals():
    w, ids = _inputs(4, 2, 4, 30, seed=8)
    w, ids = w.cuda(), ids.cuda()
    with pytest.raises(RuntimeError, match="no CPU path"):
        EF.balance_loss(w.cpu(), ids, 30)
    with pytest.raises(RuntimeError, match="no CPU path"):
        EF.balance_loss(w, ids.cpu(), 30)
    with pytest.raises(ValueError, match="fp32 or bf16"):
        EF.balance_loss(w.half(), ids, 30)
    with pytest.raises(ValueError, match="one shape"):
        EF.balance_loss(w, ids[:, :, :2], 30)
    with pytest.raises(ValueError, match="mask"):
        EF.balance_loss(w, ids, 30, mask=torch.ones(5, dtype=torch.bool, device="cuda"))
    with pytest.raises(_lib.EthosError):
        EF.balance_loss(w, ids, 0)


def test_entry_point_argument_checks():
    L = _lib.lib()
    v = ctypes.c_void_p(256)
    need = L.ethos_balance_scratch_size(4, 2, 4)
    assert need >= 4 * 32 and L.ethos_balance_scratch_size(-1, 2, 4) == 0
    fwd = lambda **o: L.ethos_balance_forward(*[o.get(n, x) for n, x in (  # noqa: E731
        ("ids", v), ("i64", 1), ("w", v), ("dtype", 0), ("mask", None), ("T", 4), ("H", 2), ("k", 4), ("N", 30),
        ("counts", v), ("loss", v), ("scratch", v), ("bytes", need), ("err", v), ("stream", None))])
    assert fwd(ids=None) == 1 and fwd(w=None) == 1 and fwd(counts=None) == 1 and fwd(scratch=None) == 4
    assert fwd(dtype=7) == 1 and fwd(N=0) == 1 and fwd(T=-1) == 1 and fwd(bytes=64) == 4
    assert fwd(T=1 << 29) == 2                                    # selections would pass int32
    assert fwd(scratch=ctypes.c_void_p(260)) == 3
    bwd = lambda **o: L.ethos_balance_backward(*[o.get(n, x) for n, x in (  # noqa: E731
        ("dtype", 0), ("T", 4), ("H", 2), ("k", 4), ("N", 30), ("scratch", v), ("bytes", need), ("grad", v),
        ("dw", v), ("stream", None))])
    assert bwd(T=0) == 0 and bwd(grad=None) == 1 and bwd(dw=None) == 1 and bwd(scratch=None) == 4 and bwd(bytes=8) == 4
