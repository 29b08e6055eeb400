"""The checks of long sums reject a sum that lacks one part (planted here, in the definition)."""
import pytest
import torch

import operator_oracles as oracle
import operator_sums as sums


@pytest.mark.parametrize("n,vocab,width", [(140000, 9, 8), (40000, 2, 16), (9001, 200, 72), (30001, 500, 8)])
def test_embedding_sum_without_one_token(n, vocab, width):
    g = torch.Generator().manual_seed(n)
    ids = torch.randint(0, vocab, (n,), generator=g)
    dy = sums.whole(n, width, g, "cpu")
    want = sums.whole_grad(dy, ids, vocab, 0.5)
    assert torch.equal(torch.zeros(vocab, width).index_add_(0, ids, dy) * 0.5, want)  # in 32 bits, in this order
    for t in (0, n // 2, n - 1):
        rest = torch.arange(n) != t
        less = sums.whole_grad(dy[rest], ids[rest], vocab, 0.5)
        assert (less[ids[t]] != want[ids[t]]).all()


def test_norm_weight_sum_without_one_block():
    rows, heads, d, eps, depth = 20000, 4, 64, 1e-6, 200
    g = torch.Generator().manual_seed(0)
    x = torch.randn(rows, heads, d, generator=g, dtype=torch.float64)
    dy = torch.randn(rows, heads, d, generator=g, dtype=torch.float64).abs() * x.sign()
    want, bound = sums.norm_weight_grad(x, dy, eps, depth)
    in_32 = (dy.float() * x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + eps)).sum((0, 1))
    oracle.within(in_32, want, bound)
    for first, count in ((0, rows // 296), (rows // 2, 8), (rows - 4, 4)):  # a block's rows of 296, a warp's, a few
        keep = torch.ones(rows, dtype=torch.bool)
        keep[first:first + count] = False
        less, _ = sums.norm_weight_grad(x[keep], dy[keep], eps, depth)
        with pytest.raises(AssertionError, match="off by"):
            oracle.within(less, want, bound)
        assert ((less - want).abs() > 1.01 * bound).all()
