"""The token-side operators at the ends of their ranges: row counts and offsets beyond 2^31."""
import pytest
import torch

import operator_oracles as oracle

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
