"""Global gradient norm and clipping against the definition in 64 bits."""
import pytest
import torch

import operator_oracles as oracle

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _ops():
    from revpp import ops

    return ops


def _grads(sizes, types, seed=0, scale=0.1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, device="cuda", generator=g) * scale).to(types[i % len(types)]) for i, n in enumerate(sizes)]


def _check(norm, outs, grads, max_norm, norm_type):
    flat = torch.cat([g.double().reshape(-1) for g in grads])
    want = flat.square().sum().sqrt() if norm_type == 2.0 else (flat.abs().max() if flat.numel() else flat.sum())
    assert norm.shape == () and norm.dtype == torch.float32
    # 64-bit sums, rounded to fp32 once
    oracle.within(norm, want, want * (oracle.U + 1e-12) + oracle.tiny(torch.float32))
    coef = min(1.0, max_norm / (want.item() + 1e-6))
    for o, g in zip(outs, grads):
        if not g.numel():
            continue
        y = g.double() * coef
        # the factor and the product round to fp32, then to the output type
        oracle.within(o, y, y.abs() * (2 * oracle.U + oracle.half_step(o.dtype)) + oracle.tiny(o.dtype) + oracle.tiny(torch.float32))


@pytest.mark.parametrize("sizes", [[1], [0, 3], [5, 1023, 8192, 8193, 7], [100001], list(range(1, 200)), [3] * 1500,
                                   [2_000_003, 16]])
@pytest.mark.parametrize("types", [[torch.float32], [torch.bfloat16], [torch.float16, torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("max_norm", [0.5, 1e6])
@pytest.mark.parametrize("norm_type", [2.0, float("inf")])
def test_in_place_and_into_other_tensors(sizes, types, max_norm, norm_type):
    ops = _ops()
    if norm_type != 2.0:
        max_norm /= 10
    grads = _grads(sizes, types)
    kept = [g.clone() for g in grads]
    for out_type in TYPES:
        outs = [torch.full(g.shape, float("nan"), device="cuda", dtype=out_type) for g in grads]
        norm = ops.clip_grads(grads, max_norm, out=outs, norm_type=norm_type)
        _check(norm, outs, kept, max_norm, norm_type)
        assert all(torch.equal(a, b) for a, b in zip(grads, kept))
    norm = ops.clip_grads(grads, max_norm, norm_type=norm_type)
    _check(norm, grads, kept, max_norm, norm_type)
    again = [k.clone() for k in kept]
    assert torch.equal(ops.clip_grads(again, max_norm, norm_type=norm_type), norm)
    assert all(torch.equal(a, b) for a, b in zip(again, grads))  # the same bits


def test_matches_the_cpu_form():
    from revpp import optim

    grads = _grads([10, 3000, 77], [torch.float32, torch.bfloat16])
    host = [g.cpu() for g in grads]
    a = optim.clip_grads((g for g in grads), 0.3)
    b = optim.clip_grads(host, 0.3)
    assert abs(a.item() - b.item()) <= 2 * oracle.U * b.item()
    for x, y in zip(grads, host):
        assert (x.cpu().double() - y.double()).abs().max().item() <= y.abs().max().item() * 2 * (oracle.half_step(x.dtype) + 2 * oracle.U)
    assert optim.clip_grads([], 1.0).item() == 0


def test_layouts_and_offsets():
    ops = _ops()
    base = torch.randn(4000, device="cuda")
    grads = [base[1:1000], base[1002:2001], torch.randn(30, 40, device="cuda").t(), torch.randn(2, 3, 4, 5, device="cuda").permute(3, 1, 0, 2),
             torch.randn((), device="cuda"), base[2002:2003].expand(1, 1)]
    kept = [g.clone() for g in grads]
    outside = base[[0, 1000, 1001, 2001, 2003, 3999]].clone()
    outs = [torch.full_like(g, float("nan"), dtype=torch.bfloat16) for g in grads]
    norm = ops.clip_grads(grads, 1.0, out=outs)
    _check(norm, outs, kept, 1.0, 2.0)
    norm = ops.clip_grads(grads, 1.0)
    _check(norm, grads, kept, 1.0, 2.0)
    assert torch.equal(base[[0, 1000, 1001, 2001, 2003, 3999]], outside)
    # the same gradient twice counts twice, into two outputs
    g = torch.randn(100, device="cuda")
    outs = [torch.empty_like(g), torch.empty_like(g)]
    norm = ops.clip_grads([g, g], 0.1, out=outs)
    _check(norm, outs, [g, g], 0.1, 2.0)


@pytest.mark.parametrize("scale", [1e-30, 1e30])
def test_norms_whose_squares_leave_fp32(scale):
    ops = _ops()
    grads = _grads([5000, 33], [torch.float32], scale=scale)
    outs = [torch.empty_like(g) for g in grads]
    _check(ops.clip_grads(grads, scale, out=outs), outs, grads, scale, 2.0)


@pytest.mark.parametrize("norm_type", [2.0, float("inf")])
def test_values_that_are_not_finite(norm_type):
    ops = _ops()
    grads = _grads([5000, 33], [torch.float32, torch.bfloat16])
    grads[1][32] = float("nan")
    outs = [torch.empty_like(g) for g in grads]
    assert ops.clip_grads(grads, 1.0, out=outs, norm_type=norm_type).isnan()
    assert all(o.isnan().all() for o in outs)
    grads[1][32] = -float("inf")
    assert ops.clip_grads(grads, 1.0, out=outs, norm_type=norm_type).item() == float("inf")
    assert not outs[0].any() and outs[1][32].isnan() and not outs[1][:32].any()


def test_refused_on_the_device():
    ops = _ops()
    base = torch.randn(1000, device="cuda")
    with pytest.raises(RuntimeError, match="shares memory"):
        ops.clip_grads([base[:10], base[:10]], 1.0)
    with pytest.raises(RuntimeError, match="shares memory"):
        ops.clip_grads([base[:10], base[5:20]], 1.0)
    with pytest.raises(RuntimeError, match="shares memory"):
        ops.clip_grads([base[:10], base[20:30]], 1.0, out=[base[20:30], base[40:50]])
    with pytest.raises(RuntimeError, match="shares memory"):
        ops.clip_grads([base[:10]], 1.0, out=[base[1:11]])
    with pytest.raises(RuntimeError, match="shares memory"):
        ops.clip_grads([base[:10]], 1.0, out=[base.view(torch.bfloat16)[:10]])
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.clip_grads([base[:10], torch.randn(3)], 1.0, out=[base[20:30], torch.randn(3)])
    with pytest.raises(RuntimeError, match="device"):
        ops.clip_grads([base[:10]], 1.0, out=[torch.randn(10)])


def test_captured_with_new_gradients():
    ops = _ops()
    grads = _grads([700, 9000, 3], [torch.float32, torch.bfloat16])
    outs = [torch.empty_like(g) for g in grads]
    ops.clip_grads(grads, 0.5, out=outs)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads(grads, 0.5, out=outs)
    for g in grads:
        g.mul_(-3)
    graph.replay()
    torch.cuda.synchronize()
    _check(norm, outs, grads, 0.5, 2.0)
