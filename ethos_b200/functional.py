"""Differentiable training operators around the expert layers, as functions of
tensors: the decoder's token embedding, the balance of the routing, and the
cross entropy of the output head.

All run in ``libethos_b200.so`` on CUDA tensors (there is no CPU path), on the
current stream, and without a host synchronisation: an id outside its range is
recorded in the device error word (``ops.check_device_error``).
"""

import torch

from . import ops

__all__ = ["embedding", "balance_loss", "linear_cross_entropy"]


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.scale, ctx.padding_idx, ctx.vocab, ctx.dtype = scale, padding_idx, weight.shape[0], weight.dtype
        return ops.embedding_forward(ids, weight, scale)

    @staticmethod
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        return None, ops.embedding_backward(ids, dy, ctx.vocab, ctx.scale, ctx.padding_idx), None, None


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """``scale * weight[ids]``: rows of the table ``weight [V, d]`` (fp32 or
    bf16) for token ids of any shape, each value rounded once.

    The gradient with respect to ``weight`` is dense, in its dtype: every
    token's ``scale * dy`` summed in fp32 in token order (the same bits in
    every run) and rounded once; rows no token holds are zero.  The row of
    ``padding_idx`` (None: no such row) gets no gradient; a negative index
    counts from the end, as in ``torch.nn.Embedding``."""
    if padding_idx is not None:
        V = weight.shape[0]
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx {padding_idx} is not in the table of {V} rows")
        padding_idx = padding_idx % V
    return _Embedding.apply(ids, weight, float(scale), padding_idx)


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weights, ids, num_experts, mask):
        loss, counts, scratch = ops.balance_forward(weights, ids, num_experts, mask)
        ctx.save_for_backward(scratch)
        ctx.shape, ctx.num_experts, ctx.dtype = weights.shape, num_experts, weights.dtype
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)  # no zeros for the counts
        return loss, counts

    @staticmethod
    def backward(ctx, grad, _):
        if grad is None:
            return None, None, None, None
        scratch, = ctx.saved_tensors
        return ops.balance_backward(grad, scratch, ctx.shape, ctx.num_experts, ctx.dtype), None, None, None


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
    return _BalanceLoss.apply(weights, ids, int(num_experts), mask)


def _keeping_pays(T, V, d):
    """Whether forming the logits a second time would take longer than the
    five launches that keeping their exponentials takes on top (about 20 us):
    its time is that of the products (1.2 PFLOP/s, rows in tiles of 256) or of
    reading the table (4.5 TB/s)."""
    rows = -(-T // 256) * 256
    return max(2.0 * rows * V * d / 1.2e9, 2.0 * V * d / 4.5e6) > 20.0


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, labels, ignore_index, reduction, need_hidden, need_weight):
        ctx.grads = None
        ctx.reduction = reduction
        if reduction != "none" and (need_hidden or need_weight) and _keeping_pays(hidden.shape[0], *weight.shape):
            both = ops.linear_cross_entropy_forward_backward(hidden, weight, labels, ignore_index, reduction,
                                                             need_hidden, need_weight)
            if both is not None:
                loss, save, dh, dw = both
                ctx.grads = (dh, dw)
                ctx.save_for_backward(hidden, weight, save)
                return loss
        loss, save = ops.linear_cross_entropy_forward(hidden, weight, labels, ignore_index, reduction)
        ctx.save_for_backward(hidden, weight, save)
        return loss

    @staticmethod
    def backward(ctx, grad):
        hidden, weight, save = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads, ctx.grads = ctx.grads, None
        if grads is not None:
            # the loss's own gradients, scaled where they are
            dh, dw = (g if n else None for g, n in zip(grads, need))
            ops.scale_(grad.to(torch.float32), dh, dw)
        else:  # also a second pass through the graph: the first one's results belong to its caller
            dh, dw = ops.linear_cross_entropy_backward(grad, hidden, weight, save, ctx.reduction, need[0], need[1])
        return dh, dw, None, None, None, None, None


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
    logits' exponentials (bf16, up to 4 GiB of workspace) for its own length;
    the backward multiplies them by the loss's gradient.  Otherwise the backward forms the logits again, a
    piece of the vocabulary at a time.  Neither way keeps anything of size
    ``T * V`` between the calls."""
    if labels.shape != hidden.shape[:-1]:
        raise ValueError(f"labels {tuple(labels.shape)} do not belong to hidden {tuple(hidden.shape)}")
    flat = hidden.reshape(-1, hidden.shape[-1]) if hidden.dim() != 2 else hidden
    grad = torch.is_grad_enabled()
    loss = _LinearCrossEntropy.apply(flat, weight, labels.reshape(-1), ignore_index, reduction,
                                     grad and flat.requires_grad, grad and weight.requires_grad)
    return loss.view(labels.shape) if reduction == "none" else loss
