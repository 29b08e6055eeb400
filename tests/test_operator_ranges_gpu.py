"""The token-side operators at the ends of their ranges: row counts and offsets beyond 2^31."""
import pytest
import torch

import operator_oracles as oracle
import operator_sums as sums

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(autouse=True)
def _give_back():
    yield
    torch.cuda.empty_cache()


def test_norm_rotation_of_the_most_rows():
    """2^30 - 1 rows of 2 + 2 x 1 heads of 2: three sets of heads do not divide the lanes, and the lanes
    without a row count on past 2^31 rows."""
    from revpp import ops

    ops.check_status()
    rows, heads, d = 2 ** 30 - 1, 2, 2
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(rows, 8, device="cuda", dtype=torch.float16).normal_(generator=g)
    dy = torch.empty_like(x).normal_(generator=g)
    positions = torch.arange(rows, device="cuda", dtype=torch.int32) % 1000
    cos, sin = oracle.tables(1000, d, "cuda")
    w = 1 + 0.3 * torch.randn(d, device="cuda", generator=g)
    kw = dict(kv_heads=1, wq=w, wk=w, eps=EPS, cos=cos, sin=sin, interleaved=True)
    at = [slice(0, 5000), slice(rows // 2, rows // 2 + 5000), slice(rows - 400000, rows)]
    kept = [(x[s].double().view(-1, 4, d), dy[s].double().view(-1, 4, d)) for s in at]
    dwq = torch.zeros(d, device="cuda")
    ops.qk_norm_rope_bwd(dy, x, dy, heads, dwq=dwq, positions=positions, **kw)
    ops.qk_norm_rope_fwd(x, x, heads, S=1000, **kw)
    torch.cuda.synchronize()
    assert ops.check_status() == 0 and torch.isfinite(dwq).all()
    for s, (xs, dys) in zip(at, kept):
        p = positions[s].long()
        c, n = cos[p], sin[p]
        y, dx = x[s].view(-1, 4, d), dy[s].view(-1, 4, d)
        oracle.within(y[:, :3], oracle.norm_turn(xs[:, :3], w, EPS, c, n, True),
                      oracle.norm_turn_bound(xs[:, :3], w, EPS, c, n, True, x.dtype))
        want, _, bound, _ = oracle.norm_turn_grad(xs[:, :3], w, dys[:, :3], EPS, c, n, True)
        oracle.within(dx[:, :3], want, bound + (want.abs() + bound) * oracle.half_step(x.dtype) + oracle.tiny(x.dtype))
        assert torch.equal(y[:, 3].double(), xs[:, 3]) and torch.equal(dx[:, 3].double(), dys[:, 3])


def test_embedding_gradient_of_a_table_beyond_32_bits():
    """A dW of 2.3 G elements through sort, reduce and join; its last rows lie behind 2^31 elements, and
    one of them is named by tokens of many chunks."""
    from revpp import ops

    ops.check_status()
    vocab, width, n = 70000, 32768, 600
    g = torch.Generator(device="cuda").manual_seed(0)
    ids = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    ids[::3] = 69999
    ids[1:100:3] = 65537
    ids[2:40:3] = 65535
    dy = sums.whole(n, width, g, "cuda", torch.bfloat16)
    rows, at = ids.unique(return_inverse=True)
    want = torch.zeros(len(rows), width, device="cuda").index_add_(0, at, dy.float())
    dw = torch.full((vocab, width), float("nan"), device="cuda")
    ops.embedding_bwd(dy, ids, dw, accumulate=False)
    assert torch.equal(dw[rows], want)
    assert torch.count_nonzero(dw[:, 5]).item() == torch.count_nonzero(want[:, 5]).item()
    assert torch.count_nonzero(dw[:, -1]).item() == torch.count_nonzero(want[:, -1]).item()
    ops.embedding_bwd(dy, ids, dw, scale=2.0)
    assert torch.equal(dw[rows], 3 * want)
    assert ops.check_status() == 0


def test_embedding_of_rows_far_apart():
    """Rows of dy and of the lookup's output 2^23 elements apart: the last ones start behind 2^31 elements."""
    from revpp import ops

    ops.check_status()
    n, vocab, width = 300, 40, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, vocab, (n,), device="cuda", generator=g)
    store = torch.zeros(n, 2 ** 23, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(vocab, width, device="cuda", generator=g).to(torch.bfloat16)
    y = store[:, 8:8 + width]
    ops.embedding_fwd(ids, w, y)
    assert torch.equal(y, w[ids]) and not store[:, :8].any() and not store[:, 8 + width:200].any()
    y.copy_(sums.whole(n, width, g, "cuda", torch.bfloat16))
    for k in (n, 200):  # both kernels
        dw = torch.full((vocab, width), float("nan"), device="cuda")
        ops.embedding_bwd(y[:k], ids[:k], dw, accumulate=False)
        assert torch.equal(dw, sums.whole_grad(y[:k], ids[:k], vocab, 1.0))


def test_norm_rotation_gradient_of_rows_far_apart():
    """Rows 2^20 elements apart, in place and into another buffer."""
    from revpp import ops

    rows, heads, d = 2100, 2, 64
    g = torch.Generator(device="cuda").manual_seed(2)
    width = (heads + 2) * d
    x, dy, dx = (torch.zeros(rows, 2 ** 20, device="cuda", dtype=torch.bfloat16)[:, 8:8 + width] for _ in range(3))
    x.copy_(torch.randn(rows, width, device="cuda", generator=g))
    dy.copy_(torch.randn(rows, width, device="cuda", generator=g))
    cos, sin = oracle.tables(300, d, "cuda")
    at = torch.arange(rows, device="cuda") % 300
    w = 1 + 0.3 * torch.randn(d, device="cuda", generator=g)
    kw = dict(kv_heads=1, wq=w, wk=w, eps=EPS, cos=cos, sin=sin, S=300)
    ops.qk_norm_rope_bwd(dy, x, dx, heads, **kw)
    xs, dys, got = (t.double().view(rows, -1, d) for t in (x.contiguous(), dy.contiguous(), dx.contiguous()))
    want, _, bound, _ = oracle.norm_turn_grad(xs[:, :3], w, dys[:, :3], EPS, cos[at], sin[at], False)
    oracle.within(got[:, :3], want, bound + (want.abs() + bound) * oracle.half_step(x.dtype) + oracle.tiny(x.dtype))
    assert torch.equal(got[:, 3], dys[:, 3])
    ops.qk_norm_rope_bwd(dy, x, dy, heads, **kw)
    assert torch.equal(dy, dx)


def test_clipping_of_a_tensor_beyond_32_bits():
    from revpp import ops

    n = 2 ** 31 + 13
    grad = torch.full((n,), 2.0 ** -10, device="cuda", dtype=torch.bfloat16)
    grad[-1] = 3.0
    norm = ops.clip_grads([grad, torch.zeros(5, device="cuda")], 1.0)
    want = ((n - 1) * 2.0 ** -20 + 9.0) ** 0.5  # the squares and their sum are exact in 64 bits
    assert abs(norm.item() - want) <= want * (oracle.U + 1e-12)
    coef = 1.0 / (want + 1e-6)
    for at, v in ((0, 2.0 ** -10), (n - 2, 2.0 ** -10), (n - 1, 3.0)):
        assert abs(grad[at].item() - v * coef) <= v * coef * (oracle.half_step(grad.dtype) + 2 * oracle.U)
    assert (grad[:-1] == grad[0]).all()
