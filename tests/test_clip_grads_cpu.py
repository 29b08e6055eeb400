"""Clipping of separate gradient tensors on the CPU against the definition in 64 bits."""
import pytest
import torch

import operator_oracles as oracle
from revpp import optim


def _coef(grads, max_norm):
    return min(1.0, max_norm / (torch.cat([g.double().reshape(-1) for g in grads]).norm().item() + 1e-6))


def _refused(grads, out=None):
    """Raises, and leaves everything as it was."""
    tensors = list(grads) + list(out or [])
    kept = [t.clone() for t in tensors]
    with pytest.raises(ValueError, match="shares memory"):
        optim.clip_grads(grads, 0.1, out=out)
    assert all(torch.equal(t, k) for t, k in zip(tensors, kept))


def test_outputs_that_share_memory_are_refused():
    g, base = torch.ones(4), torch.arange(1.0, 41.0)
    _refused([g, g])                                        # would be scaled twice
    _refused([g, g.view(2, 2)])
    _refused([base[:2], base[2:4]], out=[base[2:4], base[:2]])  # the second would be read after it was written
    _refused([base[:10], base[5:20]])
    _refused([base[:10]], out=[base[1:11]])
    _refused([base[:10]], out=[base.view(torch.bfloat16)[:10]])
    _refused([g, torch.zeros(4)], out=[base[:4], base[3:7]])
    _refused([base.view(4, 10)[:, :5], base.view(4, 10)[:, 4:6]])
    _refused([base.view(4, 10).t()], out=[base.view(10, 4)])
    _refused([torch.ones(3, 4)], out=[base[:4].expand(3, 4)])
    _refused([base[::2], base[::3]])


def test_tensors_of_one_buffer_that_lie_apart():
    base = torch.randn(24, 10)
    pieces = [base[:, :5], base[:, 5:9], base[::2, 9], base[1::2, 9]]
    kept, before = [p.clone() for p in pieces], base.clone()
    optim.clip_grads(pieces, 0.5)
    oracle.within(base, before.double() * _coef(kept, 0.5), before.double().abs() * 2 * oracle.U)
    # sizes of one leave their strides open
    row = base[:1]
    optim.clip_grads([row], 1e6, out=[row.as_strided((1, 10), (3, 1))])
    # one gradient twice counts twice, into two outputs of one buffer; empty tensors lie nowhere
    g, buf = torch.randn(6), torch.zeros(12)
    optim.clip_grads([g, g, torch.zeros(0)], 0.5, out=[buf[:6], buf[6:], buf[3:3]])
    assert torch.equal(buf[:6], buf[6:])
    oracle.within(buf[:6], g.double() * _coef([g, g], 0.5), g.double().abs() * 2 * oracle.U)


def test_sparse_gradients():
    net = torch.nn.Embedding(6, 3, sparse=True)
    net(torch.tensor([1, 1, 2])).sum().backward()
    dense = net.weight.grad.to_dense()
    norm = optim.clip_grads([net.weight.grad, torch.ones(2)], 0.5)
    assert abs(norm.item() - 17 ** 0.5) <= 2 * oracle.U * 17 ** 0.5  # rows of 2, 2, 2 and 1, 1, 1, and the ones
    oracle.within(net.weight.grad.to_dense(), dense.double() * _coef([dense, torch.ones(2)], 0.5), dense.double() * 4 * oracle.U)
    with pytest.raises(ValueError, match="shares memory"):
        optim.clip_grads([net.weight.grad, net.weight.grad], 0.5)


@pytest.mark.parametrize("max_norm", [0.3, 1e6])
def test_float64_gradients_keep_their_bits(max_norm):
    torch.manual_seed(1)
    grads = [torch.randn(50, dtype=torch.float64), torch.randn(9), torch.randn(7, dtype=torch.float64).to(torch.bfloat16)]
    kept = [g.clone() for g in grads]
    norm = optim.clip_grads(grads, max_norm)
    coef = _coef(kept, max_norm)
    assert norm.dtype == torch.float32
    # norm and factor are computed in 64 bits: about 70 roundings of 2^-53, and the product's
    oracle.within(grads[0], kept[0] * coef, (kept[0] * coef).abs() * 80 * 2.0 ** -53)
    for g, k in zip(grads[1:], kept[1:]):
        y = k.double() * coef
        oracle.within(g, y, y.abs() * (2 * oracle.U + oracle.half_step(g.dtype)))
    if max_norm == 1e6:
        assert all(torch.equal(g, k) for g, k in zip(grads, kept))


def test_float64_gradients_beyond_the_range_of_32_bits():
    for big in (1e60, 1e-60):
        grads = [torch.tensor([3.0, -4.0], dtype=torch.float64) * big, torch.zeros(2)]
        optim.clip_grads(grads, big)
        assert torch.allclose(grads[0], torch.tensor([3.0, -4.0], dtype=torch.float64) * big * (big / (5 * big + 1e-6)), rtol=1e-14, atol=0)
        assert not grads[1].any()


def test_types_without_a_fraction_or_with_an_imaginary_part_are_refused():
    for bad in (torch.tensor([3, 4]), torch.tensor([3 + 4j]), torch.tensor([True])):
        kept = bad.clone()
        with pytest.raises(ValueError, match="gradient 1 must be a floating-point tensor"):
            optim.clip_grads([torch.ones(2), bad], 1.0)
        with pytest.raises(ValueError, match="out 0 must be a floating-point tensor"):
            optim.clip_grads([torch.ones(bad.shape)], 1.0, out=[bad])
        assert torch.equal(bad, kept)


def test_a_missing_gradient_is_named():
    net = torch.nn.Linear(3, 2)
    net.bias.requires_grad_(False)
    net(torch.ones(1, 3)).sum().backward()
    for grads in ([p.grad for p in net.parameters()], [None, torch.ones(2)]):
        at = 1 if grads[0] is not None else 0
        with pytest.raises(TypeError, match=f"gradient {at} is not a tensor: NoneType"):
            optim.clip_grads(grads, 1.0)
    with pytest.raises(TypeError, match="out 0 is not a tensor"):
        optim.clip_grads([torch.ones(2)], 1.0, out=[None])
    # the call for modules with frozen or unused parameters
    norm = optim.clip_grads([p.grad for p in net.parameters() if p.grad is not None], 1.0)
    assert abs(norm.item() - 6 ** 0.5) <= 2 * oracle.U * 6 ** 0.5


def test_tensors_of_several_devices_are_refused():
    a, b = torch.ones(3), torch.ones(3, device="meta")
    for grads, out in (([a, b], None), ([a, a.clone()], [torch.zeros(3), b]), ([a], [b])):
        with pytest.raises(ValueError, match="on one device"):
            optim.clip_grads(grads, 0.1, out=out)
    assert (a == 1).all()


@pytest.mark.gpu
def test_cpu_and_cuda_tensors_in_one_list_are_refused():
    a, b = torch.ones(3), torch.ones(3, device="cuda")
    for grads, out in (([a, b], None), ([a], [b])):
        with pytest.raises(ValueError, match="on one device"):
            optim.clip_grads(grads, 0.1, out=out)
    for grads, out in (([b, a], None), ([b], [a])):
        with pytest.raises(RuntimeError, match="device|CUDA"):
            optim.clip_grads(grads, 0.1, out=out)
    assert (a == 1).all() and (b == 1).all()


def test_tensors_without_memory_pass():
    grads = [torch.ones(3, device="meta"), torch.ones(2, 2, device="meta")]
    assert optim.clip_grads(grads, 1.0).shape == ()
