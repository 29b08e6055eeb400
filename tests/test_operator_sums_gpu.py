"""Long sums of the embedding and norm-weight gradients, checked to the last term, and the branches that
the other tests pass by: padding and 32-bit ids in few tokens, ids at odd addresses."""
import pytest
import torch

import operator_oracles as oracle
import operator_sums as sums

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ops():
    from revpp import ops

    ops.check_status()
    return ops


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _tokens(kind, n, vocab, g):
    if kind == "uniform":
        return torch.randint(0, vocab, (n,), device="cuda", generator=g)
    if kind == "one":
        return torch.full((n,), vocab - 1, device="cuda")
    u = torch.rand(n, device="cuda", generator=g, dtype=torch.float64)  # "skewed": frequencies as 1 / id
    return (torch.exp(u * torch.tensor(float(vocab), dtype=torch.float64).log().item()).long() - 1).clamp_(0, vocab - 1)


# few tokens, one chunk, runs over many chunks, several segments, clusters of two and of one CTA
CASES = [("uniform", 200, 1, 96), ("one", 256, 3, 130), ("skewed", 255, 40, 1024), ("one", 257, 1, 24), ("one", 1025, 3, 16),
         ("one", 9001, 200, 72), ("skewed", 9999, 257, 515), ("skewed", 40000, 2, 256), ("uniform", 65536, 2, 128),
         ("uniform", 65536, 16, 64), ("one", 140000, 9, 8), ("skewed", 300001, 500, 8), ("skewed", 4097, 30522, 64),
         ("skewed", 140001, 40000, 8), ("skewed", 70000, 70000, 8), ("uniform", 900, 140000, 8), ("skewed", 33000, 140000, 12)]


@pytest.mark.parametrize("kind,n,vocab,width", CASES)
@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_sums_to_the_last_token(kind, n, vocab, width, dtype):
    ops, g = _ops(), _gen(n + vocab)
    ids = _tokens(kind, n, vocab, g)
    dy = sums.whole(n, width, g, "cuda", dtype)
    want = sums.whole_grad(dy, ids, vocab, 0.5)
    dw = torch.full((vocab, width), float("nan"), device="cuda")
    ops.embedding_bwd(dy, ids, dw, scale=0.5, accumulate=False)
    assert torch.equal(dw, want)
    before = sums.whole(vocab, width, g, "cuda")
    dw.copy_(before)
    ops.embedding_bwd(dy, ids, dw, scale=0.5)
    assert torch.equal(dw, before + want)
    assert ops.check_status() == 0


@pytest.mark.parametrize("n", [1, 5, 200, 256, 257, 600, 40000])
@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("padding", [0, 7, -1])
@pytest.mark.parametrize("offset", [0, 1])
def test_padding_types_and_addresses_of_ids(n, id_type, padding, offset):
    ops, g = _ops(), _gen(n)
    vocab, width = 50, 40
    store = torch.randint(0, vocab, (n + offset,), device="cuda", generator=g).to(id_type)
    ids = store[offset:]  # with 1: pairs of ids do not start at their own alignment
    assert ids.data_ptr() % (2 * ids.element_size()) == offset * ids.element_size()
    ids[torch.rand(n, device="cuda", generator=g) < 0.4] = padding % vocab
    dy = sums.whole(n, width, g, "cuda")
    dy[ids == padding % vocab] = float("nan")  # never looked at
    want = sums.whole_grad(torch.nan_to_num(dy), ids, vocab, 1.0, padding % vocab)
    dw = torch.full((vocab, width), float("nan"), device="cuda")
    ops.embedding_bwd(dy, ids, dw, padding_idx=padding, accumulate=False)
    assert torch.equal(dw, want)
    dw.fill_(2.0)
    ops.embedding_bwd(dy, ids, dw, padding_idx=padding)
    assert torch.equal(dw, want + 2)
    y = torch.empty(n, width, device="cuda")
    w = torch.randn(vocab, width, device="cuda", generator=g)
    ops.embedding_fwd(ids, w, y)
    assert torch.equal(y, w[ids.long()])
    assert ops.check_status() == 0


@pytest.mark.parametrize("id_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("n", [200, 3000])
def test_ids_outside_the_table_among_many(id_type, n):
    ops, g = _ops(), _gen(n)
    ids = torch.randint(-20, 70, (n,), device="cuda", generator=g).to(id_type)
    dy = sums.whole(n, 24, g, "cuda")
    dw = torch.full((50, 24), float("nan"), device="cuda")
    ops.embedding_bwd(dy, ids, dw, padding_idx=3, accumulate=False)
    torch.cuda.synchronize()
    assert ops.check_status() == 4
    assert torch.equal(dw, sums.whole_grad(dy, ids, 50, 1.0, 3))


@pytest.mark.parametrize("rows,heads,kv,d,dtype", [(20000, 4, 4, 64, torch.bfloat16), (20000, 4, 4, 64, torch.float32),
                                                   (9001, 12, 6, 72, torch.float32), (30000, 2, 1, 128, torch.float16),
                                                   (40001, 3, 1, 36, torch.bfloat16)])
def test_norm_weight_sums_to_the_last_rows(rows, heads, kv, d, dtype):
    """Terms of one sign.  The longest chain of additions: a lane's rows, a block's sets of heads (64 at
    most for these widths), the partial sums of 8 blocks per SM at most
    (32 slices of them, then the slices)."""
    ops, g = _ops(), _gen(rows)
    width = (heads + 2 * kv) * d
    x = torch.randn(rows, width, device="cuda", generator=g).to(dtype)
    dy = (torch.randn(rows, width, device="cuda", generator=g).abs() * x.float().sign()).to(dtype)
    # at least one block of 8 warps on each of 148 SMs, one head or more per warp: rows per lane
    lane_rows = -(-rows // (148 * 8 // (heads + kv)))
    depth = lane_rows + 64 + 148 * 8 // 32 + 32
    assert depth < 300  # small enough that a block's share of the rows shows
    dx, dwq, dwk = torch.empty_like(x), torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    ops.qk_norm_rope_bwd(dy, x, dx, heads, kv_heads=kv, dwq=dwq, dwk=dwk, eps=1e-6, accumulate=False)
    parts = [t.double().view(rows, -1, d).split([heads, kv, kv], 1) for t in (x, dy)]
    for got, i in ((dwq, 0), (dwk, 1)):
        want, bound = sums.norm_weight_grad(parts[0][i], parts[1][i], 1e-6, depth)
        oracle.within(got, want, bound)
    added = torch.ones(d, device="cuda")
    ops.qk_norm_rope_bwd(dy, x, dx, heads, kv_heads=kv, dwq=added, eps=1e-6)
    assert torch.equal(added, dwq + 1)
