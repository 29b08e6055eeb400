"""Per-head norm of queries and keys with the rotation against the definition in 64 bits."""
import pytest
import torch

import operator_oracles as oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-6

# rows, heads, kv_heads, d, rot
SHAPES = [(1, 1, 1, 64, 64), (1, 16, 16, 64, 64), (5, 12, 4, 128, 128), (130, 2, 2, 64, 32), (33, 3, 1, 80, 80),
          (64, 4, 2, 96, 24), (7, 1, 1, 256, 256), (9, 2, 1, 255, 254), (50, 5, 5, 20, 6), (17, 1, 1, 1, 0), (40, 3, 3, 13, 2),
          (3, 64, 8, 128, 64), (300, 6, 2, 72, 36), (65, 4, 4, 2, 2), (21, 2, 2, 36, 12), (2000, 2, 1, 16, 16)]


def _ops():
    from revpp import ops

    ops.check_status()
    return ops


def _problem(rows, heads, kv, d, rot, dtype, seed=0, far=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = (heads + 2 * kv) * d
    x = (torch.randn(rows, width, device="cuda", generator=g) * torch.exp(torch.randn(1, width, device="cuda", generator=g))).to(dtype)
    p = {"x": x, "dy": torch.randn(rows, width, device="cuda", generator=g).to(dtype),
         "wq": 1 + 0.3 * torch.randn(d, device="cuda", generator=g), "wk": 1 + 0.3 * torch.randn(d, device="cuda", generator=g),
         "kw": {}, "cos": None, "sin": None}
    if rot:
        cos, sin = oracle.tables(4096, rot, "cuda")
        p["kw"] = {"cos": cos, "sin": sin}
        if far:
            p["kw"]["positions"] = torch.randint(0, 4096, (rows,), device="cuda", generator=g)
            at = p["kw"]["positions"]
        else:
            p["kw"]["S"] = 37
            at = torch.arange(rows, device="cuda") % 37
        p["cos"], p["sin"] = cos[at], sin[at]
    return p


def _heads(t, heads, kv, d):
    return t.double().reshape(t.shape[0], heads + 2 * kv, d).split([heads, kv, kv], 1)


def _check_fwd(y, p, heads, kv, d, wq, wk, interleaved, eps=EPS):
    for got, x, w in zip(_heads(y, heads, kv, d)[:2], _heads(p["x"], heads, kv, d)[:2], (wq, wk)):
        oracle.within(got, oracle.norm_turn(x, w, eps, p["cos"], p["sin"], interleaved),
                      oracle.norm_turn_bound(x, w, eps, p["cos"], p["sin"], interleaved, y.dtype))
    v = (heads + kv) * d
    assert torch.equal(y[:, v:], p["x"][:, v:])


def _check_bwd(dx, dwq, dwk, p, heads, kv, d, wq, wk, interleaved, before=(None, None), eps=EPS):
    dys = _heads(p["dy"], heads, kv, d)
    for got, x, dy, w, dw, old in zip(_heads(dx, heads, kv, d)[:2], _heads(p["x"], heads, kv, d)[:2], dys, (wq, wk),
                                      (dwq, dwk), before):
        want, want_w, bound, bound_w = oracle.norm_turn_grad(x, w, dy, eps, p["cos"], p["sin"], interleaved)
        oracle.within(got, want, bound + (want.abs() + bound) * oracle.half_step(dx.dtype) + oracle.tiny(dx.dtype))
        if dw is not None:
            want_w = want_w if old is None else want_w + old.double()
            oracle.within(dw, want_w, bound_w + want_w.abs() * oracle.U)
    v = (heads + kv) * d
    assert torch.equal(dx[:, v:], p["dy"][:, v:])


@pytest.mark.parametrize("rows,heads,kv,d,rot", SHAPES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_and_backward(rows, heads, kv, d, rot, dtype, interleaved):
    ops = _ops()
    p = _problem(rows, heads, kv, d, rot, dtype, seed=rows + d, far=rows % 2 == 1)
    kw = dict(kv_heads=kv, wq=p["wq"], wk=p["wk"], eps=EPS, interleaved=interleaved, **p["kw"])
    y = torch.full_like(p["x"], float("nan"))
    assert ops.qk_norm_rope_fwd(p["x"], y, heads, **kw) is y
    _check_fwd(y, p, heads, kv, d, p["wq"], p["wk"], interleaved)
    inplace = p["x"].clone()
    ops.qk_norm_rope_fwd(inplace, inplace, heads, **kw)
    assert torch.equal(inplace, y)

    dx = torch.full_like(p["x"], float("nan"))
    dwq, dwk = (torch.full((d,), float("nan"), device="cuda") for _ in range(2))
    ops.qk_norm_rope_bwd(p["dy"], p["x"], dx, heads, dwq=dwq, dwk=dwk, accumulate=False, **kw)
    _check_bwd(dx, dwq, dwk, p, heads, kv, d, p["wq"], p["wk"], interleaved)
    inplace = p["dy"].clone()
    oq, ok = torch.randn(d, device="cuda"), torch.randn(d, device="cuda")
    aq, ak = oq.clone(), ok.clone()
    ops.qk_norm_rope_bwd(inplace, p["x"], inplace, heads, dwq=aq, dwk=ak, **kw)
    assert torch.equal(inplace, dx)
    _check_bwd(inplace, aq, ak, p, heads, kv, d, p["wq"], p["wk"], interleaved, before=(oq, ok))
    assert ops.check_status() == 0


def test_without_weights_or_some_of_the_gradients():
    ops = _ops()
    p = _problem(50, 4, 2, 64, 64, torch.bfloat16)
    y, dx = torch.empty_like(p["x"]), torch.empty_like(p["x"])
    ops.qk_norm_rope_fwd(p["x"], y, 4, kv_heads=2, **p["kw"])
    _check_fwd(y, p, 4, 2, 64, None, None, False)
    dwk = torch.zeros(64, device="cuda")
    ops.qk_norm_rope_bwd(p["dy"], p["x"], dx, 4, kv_heads=2, wk=p["wk"], dwk=dwk, **p["kw"])
    _check_bwd(dx, None, dwk, p, 4, 2, 64, None, p["wk"], False)
    ops.qk_norm_rope_bwd(p["dy"], p["x"], dx.zero_(), 4, kv_heads=2, **p["kw"])
    _check_bwd(dx, None, None, p, 4, 2, 64, None, None, False)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_offsets_and_integer_types(dtype):
    ops = _ops()
    heads, kv, d, rows = 4, 2, 32, 60
    p = _problem(rows, heads, kv, d, 16, dtype)
    width = p["x"].shape[1]
    for off, extra in ((0, 0), (8, 24), (1, 3), (4, 12), (2, 6)):
        store = torch.full((rows, width + extra + off), 3.0, device="cuda", dtype=dtype)
        x, y, g, dx = (store.clone()[:, off:off + width] for _ in range(4))
        x.copy_(p["x"])
        g.copy_(p["dy"])
        kw = dict(kv_heads=kv, wq=p["wq"], wk=p["wk"], eps=EPS, cos=p["kw"]["cos"][:, :8], sin=p["kw"]["sin"][:, :8],
                  positions=p["kw"]["positions"].int())
        ops.qk_norm_rope_fwd(x, y, heads, **kw)
        _check_fwd(y, p, heads, kv, d, p["wq"], p["wk"], False)
        ops.qk_norm_rope_bwd(g, x, dx, heads, **kw)
        _check_bwd(dx, None, None, p, heads, kv, d, p["wq"], p["wk"], False)
        rest = y._base[:, off + width:]
        assert (rest == 3).all() and (y._base[:, :off] == 3).all()  # beside the rows
    # tables inside a wider buffer, at an odd offset
    wide = torch.randn(4096, 40, device="cuda")
    cos, sin = wide[:, 1:9], wide[:, 20:28]
    cos.copy_(p["kw"]["cos"])
    sin.copy_(p["kw"]["sin"])
    y = torch.empty_like(p["x"])
    ops.qk_norm_rope_fwd(p["x"], y, heads, kv_heads=kv, wq=p["wq"], wk=p["wk"], eps=EPS, cos=cos, sin=sin,
                         positions=p["kw"]["positions"])
    _check_fwd(y, p, heads, kv, d, p["wq"], p["wk"], False)


def test_zero_rows_and_values_of_the_types_range():
    ops = _ops()
    x = torch.zeros(4, 3 * 64, device="cuda", dtype=torch.float16)
    x[1] = 60000.0
    x[2] = 2.0 ** -24
    y = torch.empty_like(x)
    p = {"x": x, "cos": None, "sin": None}
    ops.qk_norm_rope_fwd(x, y, 1, eps=EPS)
    _check_fwd(y, p, 1, 1, 64, None, None, False)
    dy = torch.randn(4, 192, device="cuda").half()
    dx = torch.empty_like(x)
    ops.qk_norm_rope_bwd(dy, x, dx, 1, eps=1.0)
    _check_bwd(dx, None, None, dict(p, dy=dy), 1, 1, 64, None, None, False, eps=1.0)
    # an infinity or a NaN stays in its own head and row
    bad = torch.randn(6, 4 * 64, device="cuda")
    bad[2, 5] = float("nan")
    bad[3, 64 + 5] = float("inf")
    out = torch.empty_like(bad)
    ops.qk_norm_rope_fwd(bad, out, 2, kv_heads=1, eps=EPS)
    wrong = ~torch.isfinite(out).view(6, 4, 64).all(-1)
    assert wrong.nonzero().tolist() == [[2, 0], [3, 1]]


def test_positions_outside_the_tables_set_the_status():
    ops = _ops()
    p = _problem(4, 1, 1, 64, 64, torch.float32)
    p["kw"]["positions"] = torch.tensor([0, 4096, -1, 5], device="cuda")
    y = torch.empty_like(p["x"])
    ops.qk_norm_rope_fwd(p["x"], y, 1, eps=EPS, **p["kw"])
    torch.cuda.synchronize()
    assert ops.check_status() == 4
    at = torch.tensor([0, 0, 0, 5], device="cuda")  # row 0 of the tables turns by nothing
    _check_fwd(y, dict(p, cos=p["kw"]["cos"][at], sin=p["kw"]["sin"][at]), 1, 1, 64, None, None, False)
    dx = torch.empty_like(y)
    ops.qk_norm_rope_bwd(p["dy"], p["x"], dx, 1, eps=EPS, **p["kw"])
    torch.cuda.synchronize()
    assert ops.check_status() == 4
    _check_bwd(dx, None, None, dict(p, cos=p["kw"]["cos"][at], sin=p["kw"]["sin"][at]), 1, 1, 64, None, None, False)


def test_empty_batch():
    ops = _ops()
    x = torch.empty(0, 3 * 64, device="cuda")
    ops.qk_norm_rope_fwd(x, torch.empty_like(x), 1)
    dwq = torch.ones(64, device="cuda")
    ops.qk_norm_rope_bwd(x, x, torch.empty_like(x), 1, dwq=dwq)
    assert (dwq == 1).all()
    ops.qk_norm_rope_bwd(x, x, torch.empty_like(x), 1, dwq=dwq, accumulate=False)
    assert not dwq.any()


def test_many_rows_give_the_same_bits_every_time():
    """More rows than one wave of blocks holds; weight gradients over all of them."""
    ops = _ops()
    p = _problem(20000, 4, 4, 64, 64, torch.bfloat16)
    kw = dict(wq=p["wq"], wk=p["wk"], eps=EPS, **p["kw"])
    y = torch.empty_like(p["x"])
    ops.qk_norm_rope_fwd(p["x"], y, 4, **kw)
    _check_fwd(y, p, 4, 4, 64, p["wq"], p["wk"], False)
    got = []
    for _ in range(3):
        dx, dwq, dwk = torch.empty_like(y), torch.empty(64, device="cuda"), torch.empty(64, device="cuda")
        ops.qk_norm_rope_bwd(p["dy"], p["x"], dx, 4, dwq=dwq, dwk=dwk, accumulate=False, **kw)
        got.append((dx, dwq, dwk))
    _check_bwd(*got[0], p, 4, 4, 64, p["wq"], p["wk"], False)
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradient_against_differences(interleaved):
    """<dx, D> against (L(x + h D) - L(x - h D)) / 2h of the kernel's own forward pass, L = <dy, y>."""
    ops = _ops()
    heads, kv, d, h = 2, 2, 64, 2.0 ** -6
    p = _problem(40, heads, kv, d, 32, torch.float32)
    p["x"] = torch.randn(40, (heads + 2 * kv) * d, device="cuda")
    D = torch.randn_like(p["x"])
    kw = dict(wq=p["wq"], wk=p["wk"], eps=EPS, interleaved=interleaved, **p["kw"])
    sides, exact, slack = [], [], 0.0
    for s in (h, -h):
        x = p["x"] + s * D
        y = torch.empty_like(x)
        ops.qk_norm_rope_fwd(x, y, heads, **kw)
        sides.append((y.double() * p["dy"].double()).sum().item())
        at = 0.0
        for i, (xx, w, g) in enumerate(zip(_heads(x, heads, kv, d)[:2], (p["wq"], p["wk"]), _heads(p["dy"], heads, kv, d))):
            at += (oracle.norm_turn(xx, w, EPS, p["cos"], p["sin"], interleaved) * g).sum().item()
            slack += (oracle.norm_turn_bound(xx, w, EPS, p["cos"], p["sin"], interleaved, torch.float32) * g.abs()).sum().item()
        exact.append(at + (_heads(x, heads, kv, d)[2] * _heads(p["dy"], heads, kv, d)[2]).sum().item())
    dx = torch.empty_like(D)
    ops.qk_norm_rope_bwd(p["dy"], p["x"], dx, heads, **kw)
    got = (dx.double() * D.double()).sum().item()
    want = 0.0
    for x, w, dy, u in zip(_heads(p["x"], heads, kv, d)[:2], (p["wq"], p["wk"]), _heads(p["dy"], heads, kv, d), _heads(D, heads, kv, d)):
        gx, _, bound, _ = oracle.norm_turn_grad(x, w, dy, EPS, p["cos"], p["sin"], interleaved)
        want += (gx * u).sum().item()
        slack += ((bound + gx.abs() * oracle.U) * u.abs()).sum().item() * 2 * h
    want += (_heads(p["dy"], heads, kv, d)[2] * _heads(D, heads, kv, d)[2]).sum().item()
    # what the quotient leaves out of the derivative, by the definition in 64 bits
    truncation = abs((exact[0] - exact[1]) / (2 * h) - want)
    assert abs((sides[0] - sides[1]) / (2 * h) - got) <= truncation + slack / (2 * h)


def test_two_graphs_replay_together():
    ops = _ops()
    runs = []
    for k in range(2):
        p = _problem(500 + k, 4, 4, 64, 64, torch.bfloat16, seed=k)
        kw = dict(wq=p["wq"], wk=p["wk"], eps=EPS, **p["kw"])
        y, dx = torch.empty_like(p["x"]), torch.empty_like(p["x"])
        dwq, dwk = torch.zeros(64, device="cuda"), torch.zeros(64, device="cuda")
        ops.qk_norm_rope_fwd(p["x"], y, 4, **kw)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            ops.qk_norm_rope_fwd(p["x"], y, 4, **kw)
            ops.qk_norm_rope_bwd(p["dy"], p["x"], dx, 4, dwq=dwq, dwk=dwk, accumulate=False, **kw)
        runs.append((graph, stream, p, y, dx, dwq, dwk))
    for _, _, p, y, dx, dwq, dwk in runs:
        p["x"].mul_(-0.5)
        for t in (y, dx, dwq, dwk):
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, p, y, dx, dwq, dwk in runs:
        _check_fwd(y, p, 4, 4, 64, p["wq"], p["wk"], False)
        _check_bwd(dx, dwq, dwk, p, 4, 4, 64, p["wq"], p["wk"], False)


def test_offsets_beyond_32_bits():
    """Rows 2^20 elements apart: the last ones start behind 2^31 elements."""
    ops = _ops()
    p = _problem(2100, 1, 1, 64, 64, torch.bfloat16)
    store = torch.empty(2100, 1 << 20, device="cuda", dtype=torch.bfloat16)
    x = store[:, 64:64 + 192]
    x.copy_(p["x"])
    y = torch.empty_like(p["x"])
    ops.qk_norm_rope_fwd(x, y, 1, wq=p["wq"], wk=p["wk"], eps=EPS, **p["kw"])
    _check_fwd(y, p, 1, 1, 64, p["wq"], p["wk"], False)
