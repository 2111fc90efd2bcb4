"""Differentiable training operators around the expert layers, as functions of
tensors: the decoder's token embedding, the balance of the routing, and the
cross entropy of the output head.

All run in ``libethos_b200.so`` on CUDA tensors (there is no CPU path), on the
current stream, and without a host synchronisation: an id outside its range is
recorded in the device error word (``ops.check_device_error``).  The autograd
nodes are C++ (``_training.so``); a gradient cannot be differentiated again
(``create_graph=True`` raises).
"""

from . import ops
from ._lib import training

__all__ = ["embedding", "balance_loss", "linear_cross_entropy"]


_READY = set()


def _nodes(t):
    """The C++ nodes, with the error word of ``t``'s device made known."""
    nodes = training()
    dev = t.device
    if dev not in _READY and t.is_cuda:
        nodes.set_error_word(dev.index, ops.device_error_word(dev).data_ptr())
        _READY.add(dev)
    return nodes


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """``scale * weight[ids]``: rows of the table ``weight [V, d]`` (fp32 or
    bf16) for token ids of any shape, each value rounded once.

    The gradient with respect to ``weight`` is dense, in its dtype: every
    token's ``scale * dy`` summed in fp32 in token order (the same bits in
    every run) and rounded once; rows no token holds are zero.  The row of
    ``padding_idx`` (None: no such row) gets no gradient; a negative index
    counts from the end, as in ``torch.nn.Embedding``."""
    row = -1 if padding_idx is None else ops.padding_row(padding_idx, weight.shape[0])
    return _nodes(weight).embedding(ids, weight, scale, row)


def balance_loss(weights, ids, num_experts, mask=None):
    """Balance loss of the router's choices, and how often each expert was
    chosen: ``(loss, counts)`` from routing ``weights [T, H, k]`` (fp32 or
    bf16) and ``ids [T, H, k]`` (int32 or int64).

    With ``c[e]`` the selections of expert e and n tokens::

        loss = N * sum_e (c[e] / (n H k)) * (sum of e's weights / (n H))

    which is 1 when all N experts are chosen evenly and grows as the choices
    crowd; counts are constants in the gradient.  ``mask`` (bool ``[T]``)
    leaves tokens out; without any token the loss and the gradient are 0.
    ``counts`` is int32 ``[N]``."""
    return _nodes(weights).balance_loss(weights, ids, num_experts, mask)


def _keeping_pays(T, V, d):
    """Whether forming the logits a second time would take longer than the two
    or three launches that keeping their exponentials takes on top (2 to 4 us of
    host time): its time is that of the products (1.2 PFLOP/s, rows in tiles of
    256) or of reading the table (4.5 TB/s).  Loss and gradients, formed again
    against kept, in us: 95 and 99 for 1 token of 32 000 x 64, 104 and 106 for
    256 of 32 000 x 256 (3.6 us by this rule), 147 and 131 for 1000 of 32 000 x
    64 (3.5), 109 and 100 for 1000 of 16 000 x 256 (7), 154 and 133 for 256 of
    32 000 x 1024 (15)."""
    rows = -(-T // 256) * 256
    return max(2.0 * rows * V * d / 1.2e9, 2.0 * V * d / 4.5e6) > 3.0


def linear_cross_entropy(hidden, weight, labels, ignore_index=-100, reduction="mean"):
    """``torch.nn.functional.cross_entropy(hidden @ weight.T, labels)`` without
    the logits: ``hidden [..., d]`` against the vocabulary's rows ``weight [V,
    d]`` (one dtype, fp32 or bf16), ``labels [...]`` int32 or int64.

    The loss is fp32: per token, or summed or averaged over the tokens whose
    label is not ``ignore_index`` (the mean over none is NaN, as torch has
    it).  Ignored tokens take no part in the products; gradients have the
    operands' dtype.

    Where gradients are needed, the loss is one number and the problem is not
    a small one, bf16 operands get them in the forward call, which keeps the
    logits' exponentials (bf16, up to 4 GiB of workspace) for its own
    length; the backward multiplies them by the loss's gradient, which rounds
    them once more unless it is 1 or another power of two.  Otherwise the
    backward forms the logits again, a piece of the vocabulary at a time.
    Neither way keeps anything of size ``T * V`` between the calls."""
    red = ops.XENT_REDUCTION.get(reduction)
    if red is None:
        raise ValueError(f"reduction: none, sum or mean, not {reduction!r}")
    keep = red != 0 and _keeping_pays(labels.numel(), weight.shape[0], weight.shape[-1])
    return _nodes(hidden).cross_entropy(hidden, weight, labels, ignore_index, red, bool(keep))
