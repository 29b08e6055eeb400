"""Sums that a test can check to the last term.

``whole(n, width)`` gives gradients that are small whole numbers, none of them zero: every partial sum is
exact in fp32 in any order, so a term that is missing or counted twice shows.  ``norm_weight_grad`` gives
the norm weights' gradient with a bound for sums whose longest chain of additions is known."""
import torch

import operator_oracles as oracle


def whole(n, width, generator, device, dtype=torch.float32):
    size = torch.randint(1, 4, (n, width), generator=generator, device=device)
    sign = torch.randint(0, 2, (n, width), generator=generator, device=device) * 2 - 1
    return (size * sign).to(dtype)


def whole_grad(dy, ids, vocab, scale, padding_idx=None):
    """The embedding gradient of whole numbers: exact."""
    ids, dy = ids.reshape(-1).long(), dy.long().reshape(ids.numel(), -1)
    ok = (ids >= 0) & (ids < vocab)
    if padding_idx is not None:
        ok &= ids != padding_idx
    total = torch.zeros(vocab, dy.shape[1], dtype=torch.int64, device=dy.device).index_add_(0, ids[ok], dy[ok])
    assert total.abs().max().item() < 2 ** 24
    return (total.double() * scale).float()


def norm_weight_grad(x, dy, eps, depth):
    """(sum over rows and heads of dy x r, bound) without rotation for x and dy [rows, heads, d] in 64 bits.

    Each term: r within ``r_error``, two products (2 U); the sum: ``depth`` additions in its longest chain
    and as many roundings, of sum |term| at most each."""
    term = dy * x * (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return term.sum((0, 1)), term.abs().sum((0, 1)) * (oracle.r_error(x.shape[-1]) + (depth + 2) * oracle.U)
