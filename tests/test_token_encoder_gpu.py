"""The token-side operators together, as a training step uses them: lookup, QKV projection, query/key
norm and rotation, attention, their gradients, the embedding's gradient, and clipping; and clipped
gradients of a traced module into the flat buffers that the optimizer steps."""
import pytest
import torch

import operator_oracles as oracle

pytestmark = pytest.mark.gpu

B, S, HEADS, D, VOCAB, SCALE, EPS = 3, 130, 4, 64, 300, 16.0, 1e-6
H = HEADS * D
# The longest way from the inputs to a gradient rounds about 12 times to bf16 (embedding, QKV, norm,
# probabilities, attention output, its gradient, two score gradients, dQKV twice, the input gradient),
# each by at most 2^-8 relative to the value: added up without any cancelling, 12 / 256.
TOLERANCE = 12 * 2.0 ** -8


def _inputs():
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.randint(1, VOCAB, (B, S), device="cuda", generator=g)
    ids[1, 100:] = 0  # a padded sequence
    table = torch.randn(VOCAB, H, device="cuda", generator=g) * 0.05
    w = (torch.randn(3 * H, H, device="cuda", generator=g) * H ** -0.5).to(torch.bfloat16)
    b = (torch.randn(3 * H, device="cuda", generator=g) * 0.1).to(torch.bfloat16)
    wq, wk = (1 + 0.2 * torch.randn(D, device="cuda", generator=g) for _ in range(2))
    do = torch.randn(B * S, H, device="cuda", generator=g).to(torch.bfloat16)
    return ids, table, w, b, wq, wk, do, *oracle.tables(S, D, "cuda")


def _step(ops, inputs, bufs):
    ids, table, w, b, wq, wk, do, cos, sin = inputs
    M = B * S
    ops.embedding_fwd(ids, table, bufs["e"], scale=SCALE)
    ops.linear(bufs["e"], w, bufs["qkv"], bias=b)
    ops.qk_norm_rope_fwd(bufs["qkv"], bufs["rot"], HEADS, wq=wq, wk=wk, eps=EPS, cos=cos, sin=sin, S=S)
    ops.attention_fwd(bufs["rot"], bufs["o"], bufs["lse"], B, S, HEADS)
    ops.attention_bwd(bufs["rot"], bufs["o"], do, bufs["lse"], bufs["drot"], bufs["acc"], bufs["D"], B, S, HEADS)
    ops.qk_norm_rope_bwd(bufs["drot"], bufs["qkv"], bufs["drot"], HEADS, wq=wq, wk=wk, dwq=bufs["dwq"], dwk=bufs["dwk"],
                         eps=EPS, cos=cos, sin=sin, S=S, accumulate=False)
    bufs["dw"].zero_()
    bufs["db"].zero_()
    ops.linear_wgrad(bufs["drot"], bufs["e"], bufs["dw"])
    ops.cast_colsum(bufs["drot"], colsum=bufs["db"])
    ops.linear_dgrad(bufs["drot"], w, bufs["de"])
    ops.embedding_bwd(bufs["de"], ids, bufs["dtable"], scale=SCALE, padding_idx=0, accumulate=False)
    grads = [bufs[k] for k in ("dtable", "dw", "db", "dwq", "dwk")]
    return ops.clip_grads(grads, 0.5, out=bufs["clipped"])


def _buffers():
    M, bf = B * S, torch.bfloat16
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    bufs = dict(e=z(M, H, dtype=bf), qkv=z(M, 3 * H, dtype=bf), rot=z(M, 3 * H, dtype=bf), o=z(M, H, dtype=bf),
                lse=z(B, HEADS, S), drot=z(M, 3 * H, dtype=bf), acc=z(M, H), D=z(B, HEADS, S), dwq=z(D), dwk=z(D),
                dw=z(3 * H, H), db=z(3 * H), de=z(M, H, dtype=bf), dtable=z(VOCAB, H))
    bufs["clipped"] = [torch.zeros_like(bufs[k]) for k in ("dtable", "dw", "db", "dwq", "dwk")]
    return bufs


def _reference(inputs):
    ids, table, w, b, wq, wk, do, cos, sin = inputs
    leaves = [t.double().requires_grad_(True) for t in (table, w, b, wq, wk)]
    table, w, b, wq, wk = leaves
    e = table[ids.reshape(-1)] * SCALE
    x = (e @ w.t() + b).view(B * S, 3 * HEADS, D)
    c, s = cos.repeat(B, 1), sin.repeat(B, 1)
    q, k, v = (oracle.norm_turn(x[:, :HEADS], wq, EPS, c, s, False), oracle.norm_turn(x[:, HEADS:2 * HEADS], wk, EPS, c, s, False),
               x[:, 2 * HEADS:])
    q, k, v = (t.view(B, S, HEADS, D).transpose(1, 2) for t in (q, k, v))
    o = torch.softmax(q @ k.transpose(-1, -2) * D ** -0.5, -1) @ v
    o = o.transpose(1, 2).reshape(B * S, H)
    grads = list(torch.autograd.grad(o, leaves, do.double()))
    grads[0][0] = 0.0  # the padding row
    norm = torch.cat([g.reshape(-1) for g in grads]).norm()
    return o.detach(), grads, norm, min(1.0, 0.5 / (norm.item() + 1e-6))


def _compare(bufs, norm, reference):
    o, grads, want, factor = reference
    assert ((bufs["o"].double() - o).norm() / o.norm()).item() < TOLERANCE
    for got, clipped, g in zip((bufs[k] for k in ("dtable", "dw", "db", "dwq", "dwk")), bufs["clipped"], grads):
        assert ((got.double() - g).norm() / g.norm()).item() < TOLERANCE
        assert ((clipped.double() - g * factor).norm() / (g * factor).norm()).item() < 2 * TOLERANCE  # and the norm's own
    assert abs(norm.item() - want.item()) < TOLERANCE * want.item()


def test_training_step_eager_and_captured():
    from revpp import ops

    ops.check_status()
    inputs, bufs = _inputs(), _buffers()
    norm = _step(ops, inputs, bufs)
    _compare(bufs, norm, _reference(inputs))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        norm = _step(ops, inputs, bufs)
    inputs[0].copy_(torch.roll(inputs[0], 1, dims=0))  # other tokens in the captured batch
    inputs[4].mul_(0.9)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    _compare(bufs, norm, _reference(inputs))
    assert ops.check_status() == 0


def test_traced_modules_gradients_into_the_flat_buffers():
    from revpp import optim
    from revpp.models.params import FlatParams

    torch.manual_seed(0)
    net = torch.nn.Sequential(torch.nn.Embedding(20, 64), torch.nn.Linear(64, 64), torch.nn.Linear(64, 8)).cuda()
    other = torch.nn.Sequential(torch.nn.Embedding(20, 64), torch.nn.Linear(64, 64), torch.nn.Linear(64, 8)).cuda()
    other.load_state_dict(net.state_dict())
    flat = FlatParams(net, "cuda")
    ours = optim.FlatAdamW(flat, lr=1e-3, max_grad_norm=0.0)
    theirs = torch.optim.AdamW(other.parameters(), lr=1e-3, betas=(0.9, 0.999), eps=1e-6, weight_decay=0.01)
    ids = torch.randint(0, 20, (16,), device="cuda")
    for _ in range(3):
        for m in (net, other):
            m.zero_grad(set_to_none=True)
            m(ids).square().sum().backward()
        params = list(net.parameters())
        norm = optim.clip_grads([p.grad for p in params], 0.1, out=[flat.grad_of(p) for p in params])
        want = torch.nn.utils.clip_grad_norm_(other.parameters(), 0.1)
        # fp32 gradients that differ by what the two copies' parameters do
        assert abs(norm.item() - want.item()) <= 1e-4 * want.item()
        ours.step()
        theirs.step()
    for p, q in zip(net.parameters(), other.parameters()):
        # three steps of at most lr each; a gradient's relative error of 1e-4 moves a step by lr * 1e-4
        assert (p - q).abs().max().item() <= 3 * 1e-3 * 1e-2
