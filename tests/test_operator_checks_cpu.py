"""Refusals of the embedding, query/key norm and clipping operators (shape and type checks come
before any device is needed), the CPU form of the clipping, and the oracle's own gradient."""
import pytest
import torch

import operator_oracles as oracle


def _ops():
    from revpp import ops

    if not ops.available():
        pytest.skip("extension not built")
    return ops


SHARED = torch.zeros(8, 8)


def _embed(**kw):
    a = dict(ids=torch.zeros(4, dtype=torch.long), w=torch.zeros(5, 8), out=torch.zeros(4, 8))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,message", [
    (dict(ids=torch.zeros(4)), "ids"), (dict(ids=torch.zeros(4, dtype=torch.int16)), "ids"),
    (dict(w=torch.zeros(5, 8, dtype=torch.float64)), "w must be"), (dict(w=torch.zeros(8)), "w must be 2-D"),
    (dict(w=torch.zeros(8, 5).t()), "contiguous along"), (dict(out=torch.zeros(3, 8)), "out must be"),
    (dict(out=torch.zeros(4, 9)), "out must be"), (dict(out=torch.zeros(1, 8).expand(4, 8)), "overlap"),
    (dict(w=torch.zeros(0, 8)), "empty"), (dict(w=SHARED[:5], out=SHARED[4:8]), "must not overlap"), ({}, "CUDA")])
def test_lookup_refuses(kw, message):
    with pytest.raises(RuntimeError, match=message):
        _ops().embedding_fwd(**_embed(**kw))


@pytest.mark.parametrize("kw,error,message", [
    (dict(dw=torch.zeros(5, 8, dtype=torch.bfloat16)), RuntimeError, "float32"),
    (dict(dy=torch.zeros(4, 8, dtype=torch.int32)), RuntimeError, "dy must be"),
    (dict(dy=torch.zeros(5, 8)), RuntimeError, "dy must be"), (dict(dw=torch.zeros(5, 9)), RuntimeError, "dy must be"),
    (dict(dw=torch.zeros(1, 8).expand(5, 8)), RuntimeError, "overlap"),
    (dict(dy=SHARED[:4], dw=SHARED[3:8]), RuntimeError, "must not overlap"), (dict(padding_idx=5), ValueError, "padding_idx"), (dict(padding_idx=-6), ValueError, "padding_idx"),
    ({}, RuntimeError, "CUDA")])
def test_gradient_refuses(kw, error, message):
    a = dict(dy=torch.zeros(4, 8), ids=torch.zeros(4, dtype=torch.int32), dw=torch.zeros(5, 8))
    a.update(kw)
    with pytest.raises(error, match=message):
        _ops().embedding_bwd(**a)


TABLE = torch.zeros(6, 4)


@pytest.mark.parametrize("kw,message", [
    (dict(qkv=torch.zeros(3, 31)), "not a multiple"), (dict(qkv=torch.zeros(3, 4, 8)), "qkv must be"),
    (dict(qkv=torch.zeros(3, 32, dtype=torch.float64)), "qkv must be float32"),
    (dict(qkv=torch.zeros(3, 4 * 257), out=torch.zeros(3, 4 * 257)), "1 to 256"), (dict(heads=0), "heads"), (dict(kv_heads=0), "heads"),
    (dict(out=torch.zeros(3, 33)), "out must be"), (dict(out=torch.zeros(3, 32, dtype=torch.bfloat16)), "type"),
    (dict(out=torch.zeros(1, 32).expand(3, 32)), "overlap"), (dict(wq=torch.zeros(9)), "wq and wk"),
    (dict(wk=torch.zeros(8, dtype=torch.bfloat16)), "wq and wk"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(cos=TABLE), "go together"), (dict(cos=TABLE, sin=TABLE), "positions or S"),
    (dict(cos=TABLE, sin=TABLE, S=3, positions=torch.zeros(3, dtype=torch.long)), "positions or S"),
    (dict(cos=TABLE, sin=TABLE, S=7), "S must be"), (dict(cos=TABLE, sin=TABLE, S=0), "S must be"),
    (dict(cos=torch.zeros(6, 5), sin=torch.zeros(6, 5), S=3), "has room"),
    (dict(cos=TABLE, sin=torch.zeros(6, 3), S=3), "one shape"), (dict(cos=TABLE.double(), sin=TABLE.double(), S=3), "one shape"),
    (dict(cos=torch.zeros(0, 4), sin=torch.zeros(0, 4), positions=torch.zeros(3, dtype=torch.long)), "rows"),
    (dict(cos=TABLE, sin=TABLE, positions=torch.zeros(2, dtype=torch.long)), "one per row"),
    (dict(cos=TABLE, sin=TABLE, positions=torch.zeros(3)), "int64 or int32"), ({}, "CUDA")])
def test_norm_rotation_refuses(kw, message):
    ops = _ops()
    a = dict(qkv=torch.zeros(3, 32), out=torch.zeros(3, 32), heads=2, kv_heads=1)
    a.update(kw)
    with pytest.raises(RuntimeError, match=message):
        ops.qk_norm_rope_fwd(**a)
    if "out" not in kw:
        with pytest.raises(RuntimeError, match=message):
            ops.qk_norm_rope_bwd(torch.zeros(a["qkv"].shape, dtype=a["qkv"].dtype), dqkv=a.pop("out"), **a)


def test_norm_rotation_refuses_shared_memory():
    ops = _ops()
    base = torch.zeros(8, 32)
    with pytest.raises(RuntimeError, match="not overlap"):
        ops.qk_norm_rope_fwd(base[:4], base[1:5], 2, kv_heads=1)
    with pytest.raises(RuntimeError, match="not overlap"):
        ops.qk_norm_rope_fwd(base[::2], base[:4], 2, kv_heads=1)
    with pytest.raises(RuntimeError, match="not overlap"):
        ops.qk_norm_rope_bwd(base[:4], base[4:], base[2:6], 2, kv_heads=1)
    with pytest.raises(RuntimeError, match="overlap qkv"):
        ops.qk_norm_rope_bwd(base[:4], base[4:], base[4:], 2, kv_heads=1)
    w = torch.zeros(12)
    with pytest.raises(RuntimeError, match="dwq and dwk"):
        ops.qk_norm_rope_bwd(base[:4], base[4:], torch.zeros(4, 32), 2, kv_heads=1, dwq=w[:8], dwk=w[4:])


@pytest.mark.parametrize("args,kw,error,message", [
    (([torch.zeros(3)], -1.0), {}, RuntimeError, "max_norm"), (([torch.zeros(3)], float("nan")), {}, RuntimeError, "max_norm"),
    (([], 1.0), {}, RuntimeError, "empty"), (([torch.zeros(3, dtype=torch.int32)], 1.0), {}, RuntimeError, "float32"),
    (([torch.zeros(3).expand(2, 3)], 1.0), {}, RuntimeError, "gaps or repeats"),
    (([torch.zeros(6)[::2]], 1.0), {}, RuntimeError, "gaps or repeats"),
    (([torch.zeros(3)], 1.0), {"out": []}, RuntimeError, "one tensor per gradient"),
    (([torch.zeros(3)], 1.0), {"out": [torch.zeros(4)]}, RuntimeError, "sizes and strides"),
    (([torch.zeros(3, 2)], 1.0), {"out": [torch.zeros(2, 3).t()]}, RuntimeError, "sizes and strides"),
    (([torch.zeros(3)], 1.0), {"norm_type": 1.0}, ValueError, "norm_type"), (([torch.zeros(3)], 1.0), {}, RuntimeError, "CUDA")])
def test_clipping_refuses(args, kw, error, message):
    with pytest.raises(error, match=message):
        _ops().clip_grads(*args, **kw)


def test_clipping_on_the_cpu():
    from revpp import optim

    torch.manual_seed(0)
    for norm_type in (2.0, float("inf")):
        grads = [torch.randn(30, 4), torch.randn(7), torch.zeros(0), torch.randn(3).to(torch.bfloat16)]
        want = torch.linalg.vector_norm(torch.cat([g.double().reshape(-1) for g in grads]), norm_type)
        outs = [torch.empty_like(g, dtype=torch.float32) for g in grads]
        norm = optim.clip_grads(grads, 0.25, out=outs, norm_type=norm_type)
        assert abs(norm.item() - want.item()) <= oracle.U * want.item()
        for o, g in zip(outs, grads):
            if g.numel():
                y = g.double() * (0.25 / (want + 1e-6))
                oracle.within(o, y, y.abs() * 3 * oracle.U)
    grads = [torch.full((4,), 3.0)]
    assert optim.clip_grads(grads, 100.0).item() == 6.0 and (grads[0] == 3).all()
    with pytest.raises(ValueError):
        optim.clip_grads(grads, -1.0)
    with pytest.raises(ValueError):
        optim.clip_grads(grads, 1.0, out=[])
    with pytest.raises(ValueError):
        optim.clip_grads(grads, 1.0, norm_type=3.0)


@pytest.mark.parametrize("rot", [0, 4, 10])
@pytest.mark.parametrize("interleaved", [False, True])
def test_the_oracles_gradient_against_differences(rot, interleaved):
    torch.manual_seed(rot)
    x = torch.randn(5, 3, 10, dtype=torch.float64, requires_grad=True)
    w = torch.randn(10, dtype=torch.float64, requires_grad=True)
    cos, sin = (None, None) if not rot else (t[torch.tensor([0, 3, 90, 3, 7])] for t in oracle.tables(100, rot, "cpu"))

    def f(x, w):
        return oracle.norm_turn(x, w, 1e-3, cos, sin, interleaved)

    assert torch.autograd.gradcheck(f, (x, w))
    dy = torch.randn(5, 3, 10, dtype=torch.float64)
    gx, gw = torch.autograd.grad(f(x, w), (x, w), dy)
    dx, dw, _, _ = oracle.norm_turn_grad(x.detach(), w.detach(), dy, 1e-3, cos, sin, interleaved)
    assert torch.allclose(gx, dx, rtol=1e-12, atol=1e-13) and torch.allclose(gw, dw, rtol=1e-12, atol=1e-13)
