"""Adding the embedding gradient to a table gradient that holds something already."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ops():
    from revpp import ops

    ops.check_status()
    return ops


SMALLEST, NORMAL = 2.0 ** -149, 2.0 ** -126
# zeros, subnormal numbers, numbers just above them, the neighbourhood of 2^-101 and ordinary ones
VALUES = [0.0, -0.0, SMALLEST, -3 * SMALLEST, NORMAL - SMALLEST, -NORMAL / 2, NORMAL, -NORMAL - SMALLEST, 1.5 * NORMAL,
          2.0 ** -102, 2.0 ** -101, -2.0 ** -101, 2.0 ** -101 + 2.0 ** -124, -2.0 ** -102 - 2.0 ** -125, -2.0 ** -100, 1.0, -0.75, 1e30]


@pytest.mark.parametrize("width", [7, 130, 64, 1032])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind", ["few", "many", "runs"])
def test_subnormal_numbers(width, dtype, kind):
    """Each row gets one term that is not zero, so the sum in 32 bits has one rounding and is known exactly.
    Where old value, term or sum is subnormal, each may count as zero: two operands below 2^-126 at most."""
    ops = _ops()
    vocab = {"few": 200, "many": 3000, "runs": 40}[kind]
    g = torch.Generator().manual_seed(width)
    values = torch.tensor(VALUES, dtype=torch.float64)

    def draw(rows):
        return values[torch.randint(0, len(VALUES), (rows, width), generator=g)].float()

    old, term = draw(vocab), draw(vocab).to(dtype)
    want = old + term.float()
    same = torch.randint(0, 4, (vocab, 1), generator=g) == 0  # whole vectors of ordinary size as well
    term = torch.where(same, torch.ones_like(term), term)
    want = torch.where(same, old + 1, want)
    order = torch.randperm(vocab, generator=g)
    if kind == "runs":  # 100 tokens for each row, all but one of them with zeros: within and across warps and chunks
        order = torch.arange(vocab).repeat(100)[torch.randperm(100 * vocab, generator=g)]
        dy = torch.zeros(len(order), width, dtype=dtype)
        for v in range(vocab):
            dy[(order == v).nonzero()[v % 7]] = term[v]
    else:
        dy = term[order]
    dw = old.cuda()
    ops.embedding_bwd(dy.cuda(), order.cuda(), dw)
    term = torch.where(same, torch.ones_like(term), term).float()
    tiny = [(t != 0) & (t.abs() < NORMAL) for t in (old, term, want)]
    tiny = tiny[0] | tiny[1] | tiny[2]
    assert tiny.any() and not tiny.all()
    got = dw.cpu()
    assert torch.equal(got[~tiny], want[~tiny])
    assert (got.double() - want.double())[tiny].abs().max().item() < 2 * NORMAL
    # written, not added: nothing is taken as zero
    ops.embedding_bwd(dy.cuda(), order.cuda(), dw, accumulate=False)
    assert torch.equal(dw.cpu(), term)


def test_not_a_number_and_infinity_stay():
    ops = _ops()
    nan, inf = float("nan"), float("inf")
    for n in (6, 600):
        dw = torch.ones(n, 8, device="cuda")
        dw[1] = nan
        dy = torch.zeros(n, 8, device="cuda")
        dy[2], dy[3], dy[4, 1] = nan, inf, nan
        ops.embedding_bwd(dy, torch.arange(n, device="cuda"), dw)
        assert dw[1:3].isnan().all() and (dw[3] == inf).all() and dw[4, 1].isnan() and (dw[4, 2:] == 1).all()
        assert (dw[0] == 1).all() and (dw[5:] == 1).all()


def test_calls_on_two_streams_add_to_one_table():
    """Whole numbers from two streams at once: nothing is lost."""
    ops = _ops()
    n, vocab, width = 4000, 50, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = [torch.randint(0, vocab, (n,), device="cuda", generator=g) for _ in range(2)]
    dys = [torch.randint(-3, 4, (n, width), device="cuda", generator=g).float() for _ in range(2)]
    dw = torch.zeros(vocab, width, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, i, d in zip(streams, ids, dys):
            with torch.cuda.stream(s):
                ops.embedding_bwd(d, i, dw)
    torch.cuda.synchronize()
    want = torch.zeros(vocab, width, device="cuda", dtype=torch.float64)
    for i, d in zip(ids, dys):
        want.index_add_(0, i, d.double())
    assert torch.equal(dw.double(), 20 * want)
