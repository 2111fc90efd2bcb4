"""Token embedding with scaling and its gradient (functional.embedding,
ethos_embedding_forward / _backward).

Bounds.  Forward: one fp32 product rounded once, so bf16 results equal the
rounded fp32 product exactly.  Backward: the fp32 sum of n terms in order is
within n 2^-24 sum|terms| of the exact sum; bf16 adds one rounding, 2^-8 of
the result (half an ulp is 2^-9 relative; doubled where a value sits next to a
power of two)."""

import ctypes

import pytest
import torch

from ethos_b200 import _lib, functional as EF, ops


def _ids(T, V, kind, seed):
    g = torch.Generator().manual_seed(seed)
    if kind == "zipf":
        u = torch.rand(T, generator=g, dtype=torch.float64)
        return (V ** u - 1).long().clamp_(0, V - 1)
    if kind == "one":
        return torch.full((T,), V // 2)
    if kind == "ends":
        return torch.where(torch.rand(T, generator=g) < 0.5, 0, V - 1)
    return torch.randint(0, V, (T,), generator=g)


def _reference(ids, dy, V, scale, padding):
    """fp64 gradient and the bound's sum of magnitudes and term counts."""
    live = torch.ones(ids.numel(), dtype=torch.float64) if padding is None else (ids.reshape(-1) != padding).double()
    d = dy.shape[-1]
    terms = dy.reshape(-1, d).double() * live[:, None] * scale
    want = torch.zeros(V, d, dtype=torch.float64).index_add_(0, ids.reshape(-1), terms)
    mags = torch.zeros(V, d, dtype=torch.float64).index_add_(0, ids.reshape(-1), terms.abs())
    n = torch.bincount(ids.reshape(-1), minlength=V).double()[:, None]
    return want, mags, n


def _check_grad(got, want, mags, n):
    bound = (n + 2) * 2.0 ** -24 * mags
    if got.dtype == torch.bfloat16:
        bound = bound + 2.0 ** -8 * want.abs()
    bad = (got.double().cpu() - want).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} outside the rounding bound"


CASES = [
    # T, V, d, ids: one token, partial chunks, hot rows over many chunks, unaligned widths
    (1, 7, 8, "uniform"), (31, 1000, 64, "uniform"), (33, 40, 1, "zipf"), (257, 50, 1031, "zipf"),
    (1000, 1, 24, "one"), (4099, 32003, 515, "zipf"), (3000, 5000, 128, "one"), (2048, 100277, 256, "ends"),
    (5000, 200001, 12, "zipf"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,V,d,kind", CASES)
def test_embedding_and_gradient(T, V, d, kind, dtype):
    ids = _ids(T, V, kind, seed=T + V)
    g = torch.Generator().manual_seed(1)
    W = torch.randn(V, d, generator=g).to(dtype)
    dy = torch.randn(T, d, generator=g).to(dtype)
    scale = 1.7
    wg = W.cuda().requires_grad_(True)
    out = EF.embedding(ids.cuda(), wg, scale=scale)
    assert torch.equal(out.detach().cpu(), (W[ids].float() * torch.tensor(scale)).to(dtype))
    dW, = torch.autograd.grad(out, wg, dy.cuda())
    ops.check_device_error("cuda")
    assert dW.dtype == dtype
    _check_grad(dW, *_reference(ids, dy, V, float(torch.tensor(scale)), None))


@pytest.mark.gpu
@pytest.mark.parametrize("padding", [0, 19, -1])
def test_padding_row_gets_no_gradient(padding):
    V, d = 20, 16
    ids = torch.randint(0, V, (6, 50), generator=torch.Generator().manual_seed(2))
    ids[0, :25] = padding % V
    W = torch.randn(V, d, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_(True)
    dy = torch.randn(6, 50, d, generator=torch.Generator().manual_seed(4))
    out = EF.embedding(ids.cuda().to(torch.int32), W, padding_idx=padding)
    assert out.shape == (6, 50, d)
    dW, = torch.autograd.grad(out, W, dy.cuda())
    assert torch.equal(dW[padding % V], torch.zeros(d, device="cuda"))
    _check_grad(dW, *_reference(ids, dy, V, 1.0, padding % V))


@pytest.mark.gpu
def test_gradient_is_the_same_in_every_run_and_on_another_stream():
    V, d, T = 3000, 264, 9001
    ids = _ids(T, V, "zipf", 5).cuda()
    dy = torch.randn(T, d, generator=torch.Generator().manual_seed(6)).cuda()
    first = ops.embedding_backward(ids, dy, V, 0.5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = [ops.embedding_backward(ids, dy, V, 0.5) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(s)
    for a in again:
        assert torch.equal(a, first)


@pytest.mark.gpu
def test_empty_batch_strides_and_views():
    W = torch.randn(11, 40, generator=torch.Generator().manual_seed(7)).cuda()
    ids = torch.zeros((0,), dtype=torch.int64, device="cuda")
    assert EF.embedding(ids, W).shape == (0, 40)
    dW = ops.embedding_backward(ids, torch.zeros(0, 40, device="cuda"), 11)
    assert torch.equal(dW, torch.zeros_like(W))
    # a column slice of a wider table (row pitch 40, odd offset), transposed ids
    view = W[:, 3:20]
    ids = torch.arange(10, device="cuda").view(2, 5).t()
    assert torch.equal(EF.embedding(ids, view, scale=2.0), view[ids] * 2.0)
    # an expanded gradient (stride 0)
    w2 = view.clone().requires_grad_(True)
    EF.embedding(ids, w2).sum().backward()
    want = torch.zeros_like(w2)
    want[:10] = 1.0
    assert torch.equal(w2.grad, want)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A table of 2.3 G elements: rows at its far end are looked up and receive
    their gradient, and nothing else does."""
    V, d = 70000, 32776
    W = torch.zeros(V, d, dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 65536, V - 1, 65537, V - 1], device="cuda")
    W[rows] = torch.randn(5, d, device="cuda").bfloat16()
    out = EF.embedding(rows, W)
    assert torch.equal(out, W[rows])
    dy = torch.randn(5, d, generator=torch.Generator().manual_seed(10)).bfloat16().cuda()
    del W
    dW = ops.embedding_backward(rows, dy, V)
    assert torch.equal(dW[0], dy[0]) and torch.equal(dW[65536], dy[1]) and torch.equal(dW[65537], dy[3])
    assert torch.equal(dW[V - 1], (dy[2].float() + dy[4].float()).bfloat16())
    assert torch.count_nonzero(dW.view(torch.int16).any(1)).item() == 4
    ops.check_device_error("cuda")


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of a quadratic of the output, in one direction."""
    V, d, T = 9, 12, 40
    ids = _ids(T, V, "uniform", 8).cuda()
    g = torch.Generator().manual_seed(9)
    W = torch.randn(V, d, generator=g).cuda().requires_grad_(True)
    f = lambda w: EF.embedding(ids, w, scale=0.75).double().square().sum()  # noqa: E731
    dW, = torch.autograd.grad(f(W), W)
    u = torch.randn(V, d, generator=g).cuda()
    h = 2.0 ** -6
    with torch.no_grad():
        num = (f(W + h * u) - f(W - h * u)) / (2 * h)
    # a quadratic has no truncation error; fp32 rounding of the outputs, 2^-24 of f over h
    assert abs(num - (dW.double() * u.double()).sum()) <= 2.0 ** -22 * f(W) / h


@pytest.mark.gpu
def test_ids_out_of_range_are_reported():
    W = torch.ones(5, 8, device="cuda")
    for bad in (5, -1, 1 << 40):
        ids = torch.tensor([1, bad, 2], device="cuda")
        out = EF.embedding(ids, W)
        with pytest.raises(_lib.EthosError) as e:
            ops.check_device_error("cuda")
        assert e.value.status == 16
        assert torch.equal(out[1], torch.zeros(8, device="cuda")) and torch.equal(out[0], W[0])
        dW = ops.embedding_backward(ids, torch.ones(3, 8, device="cuda"), 5)
        with pytest.raises(_lib.EthosError):
            ops.check_device_error("cuda")
        assert torch.equal(dW.sum(1).cpu(), torch.tensor([0.0, 8.0, 8.0, 0.0, 0.0]))
    ops.check_device_error("cuda")


@pytest.mark.gpu
def test_refusals():
    W = torch.ones(5, 8, device="cuda")
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="no CPU path"):
        EF.embedding(ids.cpu(), W)
    with pytest.raises(RuntimeError, match="no CPU path"):
        EF.embedding(ids, W.cpu())
    with pytest.raises(ValueError, match="int32 or int64"):
        EF.embedding(ids.to(torch.int16), W)
    with pytest.raises(ValueError, match="fp32 or bf16"):
        EF.embedding(ids, W.half())
    with pytest.raises(ValueError, match="padding_idx"):
        EF.embedding(ids, W, padding_idx=5)
    with pytest.raises(ValueError, match="belong"):
        ops.embedding_backward(ids, torch.ones(4, 8, device="cuda"), 5)


def test_entry_point_argument_checks():
    L = _lib.lib()
    v = ctypes.c_void_p(256)
    assert L.ethos_embedding_forward(v, 1, v, 8, 1, 0, 5, 8, 1.0, v, v, None) == 0        # nothing to do
    assert L.ethos_embedding_forward(None, 1, v, 8, 1, 3, 5, 8, 1.0, v, v, None) == 1     # no ids
    assert L.ethos_embedding_forward(v, 1, v, 7, 1, 3, 5, 8, 1.0, v, v, None) == 1        # pitch below the width
    assert L.ethos_embedding_forward(v, 1, v, 8, 2, 3, 5, 8, 1.0, v, v, None) == 1        # unknown dtype
    assert L.ethos_embedding_backward_workspace_size(0, 0, 8) == 0
    need = L.ethos_embedding_backward_workspace_size(100, 5, 8)
    assert need >= 4 * (6 + 200) + 4 * 2 * 8 * 4
    args = (v, 1, v, 1, 100, 5, 8, -1, 1.0, v)
    assert L.ethos_embedding_backward(*args, v, 64, v, None) == 4                         # short workspace
    assert L.ethos_embedding_backward(*args, None, need, v, None) == 4
    assert L.ethos_embedding_backward(v, 1, None, 1, 100, 5, 8, -1, 1.0, v, v, need, v, None) == 1
    assert L.ethos_embedding_backward(v, 1, v, 1, 1 << 30, 5, 8, -1, 1.0, v, v, need, v, None) == 2
