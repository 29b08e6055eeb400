"""Cases of the token-embedding, query/key-norm-and-rotation and gradient-clipping operators.

``listed()`` names the measured cases, ``draw(rng)`` gives more of the same ranges,
``prepare`` makes the inputs a training program has in hand, ``run`` makes one pass: the
framework's kernels where ``own`` is true, otherwise the same mathematics in elementary
torch operations.  ``exact`` is the definition in 64 bits and ``work`` the bytes and
operations that a pass cannot do without.

The operators:

* ``embed``       out[t] = scale * table[id[t]]
* ``embed_grad``  dtable[v] = scale * sum of dy[t] over the tokens with id[t] = v != 0 (the
                  padding row), over one or more micro-batches into one gradient buffer
* ``qk``          RMS norm of every query and key head of a packed [rows, (heads + 2 kv_heads) * dim]
                  projection, then the rotation of the first ``rot`` columns by the row's position;
                  value heads are carried over
* ``qk_grad``     its gradients for the projection and for the two norm weights
* ``clip``        global norm over a model's gradient tensors; each one scaled into a flat buffer
"""
import math

import torch

own = False

EPS = 1e-6
ALIGN = 64  # elements: where each tensor starts in a flat buffer


# ---------------------------------------------------------------------------------- cases
def listed():
    return [
        # one sequence of the smallest preset: launch latency
        {"name": "embed_one_sequence", "op": "embed", "tokens": 128, "vocab": 30522, "width": 128, "table": "float32",
         "out": "float32", "scale": 1.0},
        # a 64 x 512 micro-batch on the BERT-Large width, scaled by sqrt(width), bf16 activations
        {"name": "embed_micro_batch", "op": "embed", "tokens": 32768, "vocab": 30522, "width": 1024,
         "table": "float32", "out": "bfloat16", "scale": 32.0},
        # 16 x 512 tokens at the BERT-Base width, bf16 gradients
        {"name": "embed_grad_base", "op": "embed_grad", "tokens": 8192, "vocab": 30522, "width": 768,
         "grad": "bfloat16", "scale": 1.0, "pad": 0.25, "parts": 1},
        # two 64 x 512 micro-batches accumulated into one BERT-Large table gradient
        {"name": "embed_grad_accumulated", "op": "embed_grad", "tokens": 32768, "vocab": 30522, "width": 1024,
         "grad": "float32", "scale": 32.0, "pad": 0.25, "parts": 2},
        # ragged token count and a width that no vector divides; a small vocabulary makes long runs
        {"name": "embed_grad_odd", "op": "embed_grad", "tokens": 9999, "vocab": 257, "width": 515,
         "grad": "float32", "scale": 0.5, "pad": 0.0, "parts": 1},
        # one short sequence of the smallest preset: launch latency
        {"name": "qk_one_sequence", "op": "qk", "rows": 128, "heads": 2, "kv_heads": 2, "dim": 64, "rot": 64,
         "pairs": "halves", "dtype": "bfloat16", "far": False},
        # a 64 x 512 micro-batch of BERT-Large, positions from the row
        {"name": "qk_micro_batch", "op": "qk", "rows": 32768, "heads": 16, "kv_heads": 16, "dim": 64, "rot": 64,
         "pairs": "halves", "dtype": "bfloat16", "far": False},
        # 32 x 577 ViT rows, fewer key heads, half of each head rotated in neighbouring pairs, packed positions
        {"name": "qk_shared_heads", "op": "qk", "rows": 18464, "heads": 16, "kv_heads": 4, "dim": 128, "rot": 64,
         "pairs": "neighbours", "dtype": "float16", "far": True},
        # the backward pass of the BERT-Large micro-batch
        {"name": "qk_grad_micro_batch", "op": "qk_grad", "rows": 32768, "heads": 16, "kv_heads": 16, "dim": 64,
         "rot": 64, "pairs": "halves", "dtype": "bfloat16", "far": False},
        # 9 x 577 rows in 32 bits, a head width that is no power of two, part of it rotated
        {"name": "qk_grad_odd", "op": "qk_grad", "rows": 5193, "heads": 12, "kv_heads": 6, "dim": 72, "rot": 36,
         "pairs": "halves", "dtype": "float32", "far": True},
        # the smallest preset's gradients: launch latency over many small tensors
        {"name": "clip_tiny", "op": "clip", "layers": 4, "width": 128, "vocab": 1000, "dtype": "float32",
         "max_norm": 1.0, "norm": "2"},
        # the BERT-Large gradients
        {"name": "clip_large", "op": "clip", "layers": 24, "width": 1024, "vocab": 30522, "dtype": "float32",
         "max_norm": 1.0, "norm": "2"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_grad", "embed_grad", "qk", "qk_grad", "clip"])
    if op in ("embed", "embed_grad"):
        width = _log(rng, 8, 2048)
        if rng.random() < 0.6:
            width = max(8, width // 8 * 8)
        vocab = min(_log(rng, 2, 131072), 30522 * 1024 // width)
        tokens = min(_log(rng, 1, 65536), 32768 * 1024 // width)
        case = {"op": op, "tokens": tokens, "vocab": vocab, "width": width, "scale": rng.choice([1.0, 0.125, 11.3])}
        types = ["float32", "bfloat16", "float16"]
        if op == "embed":
            case.update(table=rng.choice(types), out=rng.choice(types))
        else:
            case.update(grad=rng.choice(types), pad=rng.choice([0.0, 0.1, 0.5]), parts=rng.choice([1, 1, 2]))
        return case
    if op in ("qk", "qk_grad"):
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 1, 2, 4])
        dim = rng.choice([32, 64, 64, 96, 128, 256, rng.randrange(8, 128) * 2])
        rot = rng.choice([dim // 2 * 2, dim // 4 * 2, 0])
        per_row = (heads + 2 * kv) * dim
        rows = min(_log(rng, 1, 32768), 16384 * 48 * 64 // per_row)
        return {"op": op, "rows": rows, "heads": heads, "kv_heads": kv, "dim": dim, "rot": rot,
                "pairs": rng.choice(["halves", "neighbours"]), "dtype": rng.choice(["bfloat16", "float16", "float32"]),
                "far": rng.random() < 0.5}
    width = _log(rng, 16, 1024)
    return {"op": op, "layers": rng.randrange(1, 25), "width": rng.choice([width, width // 8 * 8]),
            "vocab": _log(rng, 2, 30522), "dtype": rng.choice(["float32", "bfloat16", "mixed"]),
            "max_norm": rng.choice([1.0, 0.002, 1e6]), "norm": rng.choice(["2", "2", "inf"])}


def _dtype(name):
    return getattr(torch, name)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)


# ---------------------------------------------------------------------------------- embedding
def _zipf(case, gen):
    """Token ids with log-uniform frequencies over 1 .. vocab - 1 (0 is the padding id)."""
    n, v = case["tokens"], case["vocab"]
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    ids = torch.exp(u * math.log(v)).long().clamp_(max=v - 1)
    pad = case.get("pad", 0.0)
    if pad:
        ids = torch.where(torch.rand(n, generator=gen, device="cuda") < pad, torch.zeros_like(ids), ids)
    return ids


def _distinct_rows(case):
    """Expected number of distinct ids among the tokens."""
    n, v = case["tokens"] * (1.0 - case.get("pad", 0.0)), case["vocab"]
    if v <= 2:
        return float(min(v - 1, n))
    k = torch.arange(1, v, dtype=torch.float64)
    p = torch.log((k + 1) / k) / math.log(v)
    return float((1 - torch.exp(n * torch.log1p(-p.clamp(max=1 - 1e-12)))).sum())


def _prepare_embed(case, gen):
    n, v, h = case["tokens"], case["vocab"], case["width"]
    s = {"scale": case["scale"]}
    if case["op"] == "embed":
        s["ids"] = _zipf(case, gen)
        s["table"] = (torch.randn(v, h, generator=gen, device="cuda") * 0.02).to(_dtype(case["table"]))
        s["out"] = torch.empty(n, h, device="cuda", dtype=_dtype(case["out"]))
    else:
        s["ids"] = [_zipf(case, gen) for _ in range(case["parts"])]
        s["dy"] = [(torch.randn(n, h, generator=gen, device="cuda") * 0.01).to(_dtype(case["grad"]))
                   for _ in range(case["parts"])]
        s["dtable"] = torch.empty(v, h, device="cuda")
    return s


def _embed(s):
    if own:
        from revpp import ops

        return ops.embedding_fwd(s["ids"], s["table"], s["out"], scale=s["scale"])
    return (s["table"][s["ids"]].float() * s["scale"]).to(s["out"].dtype)


def _embed_grad(s):
    if own:
        from revpp import ops

        for i, (ids, dy) in enumerate(zip(s["ids"], s["dy"])):
            ops.embedding_bwd(dy, ids, s["dtable"], scale=s["scale"], padding_idx=0, accumulate=i > 0)
        return s["dtable"]
    ids, dy = torch.cat(s["ids"]), torch.cat(s["dy"]).float()
    total = torch.zeros_like(s["dtable"])
    total.index_add_(0, ids, dy * (ids != 0).float()[:, None])
    return total * s["scale"]


def _exact_embed(s):
    return s["table"].double().index_select(0, s["ids"]) * s["scale"]


def _exact_embed_grad(s):
    """Differences of running sums over the tokens in the order of their ids."""
    ids, order = torch.sort(torch.cat(s["ids"]), stable=True)
    sums = torch.cat(s["dy"])[order].double().cumsum(0)
    sums = torch.cat([torch.zeros_like(sums[:1]), sums])
    v = s["dtable"].shape[0]
    ends = torch.searchsorted(ids, torch.arange(v + 1, device=ids.device))
    out = (sums[ends[1:]] - sums[ends[:-1]]) * s["scale"]
    out[0] = 0.0
    return out


# ---------------------------------------------------------------------------------- query / key norm and rotation
SEQ = 512  # rows a sequence has where positions follow from the row


def _prepare_qk(case, gen):
    rows, hq, hk, d, rot = (case[k] for k in ("rows", "heads", "kv_heads", "dim", "rot"))
    dt = _dtype(case["dtype"])
    width = (hq + 2 * hk) * d
    gain = torch.exp(torch.randn(hq + 2 * hk, 1, generator=gen, device="cuda")).expand(-1, d).reshape(-1)
    s = {"case": case, "qkv": (torch.randn(rows, width, generator=gen, device="cuda") * gain).to(dt),
         "out": torch.empty(rows, width, device="cuda", dtype=dt),
         "wq": 1 + 0.1 * torch.randn(d, generator=gen, device="cuda"),
         "wk": 1 + 0.1 * torch.randn(d, generator=gen, device="cuda"),
         "cos": None, "sin": None, "positions": None, "S": None}
    if case["op"] == "qk_grad":
        s["dout"] = (torch.randn(rows, width, generator=gen, device="cuda") * 0.01).to(dt)
        s["dwq"], s["dwk"] = torch.empty(d, device="cuda"), torch.empty(d, device="cuda")
    if rot:
        length = 32768 if case["far"] else SEQ
        angle = torch.arange(length, device="cuda", dtype=torch.float64)[:, None] * torch.pow(
            10000.0, -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if case["far"]:
            s["positions"] = torch.randint(0, length, (rows,), generator=gen, device="cuda")
        else:
            s["S"] = SEQ
    return s


def _positions(s):
    rows = s["qkv"].shape[0]
    return s["positions"] if s["positions"] is not None else torch.arange(rows, device="cuda") % s["S"]


def _rotated(s, z, sign):
    rot = s["case"]["rot"]
    if not rot:
        return z
    p = _positions(s)
    c, n = s["cos"][p][:, None, :], s["sin"][p][:, None, :] * sign
    if s["case"]["pairs"] == "halves":
        a, b = z[..., :rot // 2], z[..., rot // 2:rot]
        return torch.cat([a * c - b * n, a * n + b * c, z[..., rot:]], -1)
    a, b = z[..., 0:rot:2], z[..., 1:rot:2]
    return torch.cat([torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2), z[..., rot:]], -1)


def _split(s, packed):
    c = s["case"]
    x = packed.float().view(packed.shape[0], c["heads"] + 2 * c["kv_heads"], c["dim"])
    return x.split([c["heads"], c["kv_heads"], c["kv_heads"]], dim=1)


def _qk(s):
    c = s["case"]
    if own:
        from revpp import ops

        return ops.qk_norm_rope_fwd(s["qkv"], s["out"], c["heads"], kv_heads=c["kv_heads"], wq=s["wq"], wk=s["wk"],
                                    eps=EPS, cos=s["cos"], sin=s["sin"], positions=s["positions"], S=s["S"],
                                    interleaved=c["pairs"] == "neighbours")

    def one(x, w):
        return _rotated(s, x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w, 1.0)

    q, k, v = _split(s, s["qkv"])
    return torch.cat([one(q, s["wq"]), one(k, s["wk"]), v], dim=1).to(s["out"].dtype).view(s["out"].shape)


def _qk_grad(s):
    c = s["case"]
    if own:
        from revpp import ops

        ops.qk_norm_rope_bwd(s["dout"], s["qkv"], s["out"], c["heads"], kv_heads=c["kv_heads"], wq=s["wq"],
                             wk=s["wk"], dwq=s["dwq"], dwk=s["dwk"], eps=EPS, cos=s["cos"], sin=s["sin"],
                             positions=s["positions"], S=s["S"], interleaved=c["pairs"] == "neighbours",
                             accumulate=False)
        return s["out"], s["dwq"], s["dwk"]

    def one(x, w, dy):
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        dz = _rotated(s, dy, -1.0)
        xn = x * r
        g = dz * w
        return r * (g - xn * (g * xn).mean(-1, keepdim=True)), (dz * xn).sum((0, 1))

    q, k, _ = _split(s, s["qkv"])
    dq, dk, dv = _split(s, s["dout"])
    dq, dwq = one(q, s["wq"], dq)
    dk, dwk = one(k, s["wk"], dk)
    return torch.cat([dq, dk, dv], dim=1).to(s["out"].dtype).view(s["out"].shape), dwq, dwk


def _exact_heads(s, x, w):
    """One set of heads, [rows, heads, dim] in 64 bits: the rotation as a product of complex numbers."""
    rot = s["case"]["rot"]
    z = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * w
    if not rot:
        return z
    p = _positions(s)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[p].unsqueeze(1)
    a, rest = z[..., :rot], z[..., rot:]
    if s["case"]["pairs"] == "halves":
        t = torch.complex(a[..., : rot // 2], a[..., rot // 2:]) * turn
        a = torch.cat([t.real, t.imag], -1)
    else:
        t = torch.complex(a[..., 0::2], a[..., 1::2]) * turn
        a = torch.view_as_real(t).flatten(-2)
    return torch.cat([a, rest], -1)


def _exact_qk(s):
    c = s["case"]
    x = s["qkv"].double().view(s["qkv"].shape[0], -1, c["dim"])
    nq, nk = c["heads"], c["kv_heads"]
    y = [_exact_heads(s, x[:, :nq], s["wq"].double()), _exact_heads(s, x[:, nq:nq + nk], s["wk"].double()), x[:, nq + nk:]]
    return torch.cat(y, 1).view(s["qkv"].shape)


def _exact_qk_grad(s):
    """By differentiating the definition, 4096 rows at a time."""
    c = s["case"]
    nq, nk, d = c["heads"], c["kv_heads"], c["dim"]
    parts, dwq, dwk = [], torch.zeros(d, device="cuda", dtype=torch.float64), torch.zeros(d, device="cuda", dtype=torch.float64)
    position = _positions(s) if c["rot"] else None
    for r in range(0, c["rows"], 4096):
        t = dict(s, qkv=s["qkv"][r:r + 4096], positions=None if position is None else position[r:r + 4096])
        x = t["qkv"].double().view(-1, nq + 2 * nk, d).requires_grad_(True)
        wq, wk = s["wq"].double().requires_grad_(True), s["wk"].double().requires_grad_(True)
        y = torch.cat([_exact_heads(t, x[:, :nq], wq), _exact_heads(t, x[:, nq:nq + nk], wk), x[:, nq + nk:]], 1)
        gx, gq, gk = torch.autograd.grad(y, (x, wq, wk), s["dout"][r:r + 4096].double().view(y.shape))
        parts.append(gx.flatten(1))
        dwq, dwk = dwq + gq, dwk + gk
    return torch.cat(parts), dwq, dwk


# ---------------------------------------------------------------------------------- gradient norm and clipping
def _shapes(case):
    """The parameter shapes of a token encoder with a packed QKV projection."""
    w = case["width"]
    layer = [(w,), (w,), (3 * w, w), (3 * w,), (w, w), (w,), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
    return [(case["vocab"], w), (512, w), (2, w), (w,), (w,)] + layer * case["layers"] + [(w,), (w,), (2, w), (2,)]


def _sizes(case):
    return [math.prod(shape) for shape in _shapes(case)]


def _grad_dtype(case, shape):
    if case["dtype"] == "mixed":  # matrices in bf16, vectors in fp32
        return torch.bfloat16 if len(shape) == 2 else torch.float32
    return _dtype(case["dtype"])


def _prepare_clip(case, gen):
    grads = [(torch.randn(shape, generator=gen, device="cuda") * 0.003).to(_grad_dtype(case, shape)) for shape in _shapes(case)]
    room = [-(-n // ALIGN) * ALIGN for n in _sizes(case)]
    flat = torch.zeros(sum(room), device="cuda")
    views, at = [], 0
    for g, n in zip(grads, room):
        views.append(flat[at:at + g.numel()].view(g.shape))
        at += n
    return {"grads": grads, "views": views, "flat": flat, "max_norm": case["max_norm"], "norm": float(case["norm"])}


def _clip(s):
    if own:
        from revpp import optim

        return optim.clip_grads(s["grads"], s["max_norm"], out=s["views"], norm_type=s["norm"]), s["flat"]
    if s["norm"] == 2.0:
        norm = torch.stack([g.float().square().sum() for g in s["grads"]]).sum().sqrt()
    else:
        norm = torch.stack([g.float().abs().max() for g in s["grads"]]).max()
    factor = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    [v.copy_(g.float() * factor) for v, g in zip(s["views"], s["grads"])]
    return norm, s["flat"]


def _exact_clip(s):
    flat = torch.zeros_like(s["flat"], dtype=torch.float64)
    at = 0
    for g in s["grads"]:
        flat[at:at + g.numel()] = g.reshape(-1)
        at += -(-g.numel() // ALIGN) * ALIGN
    norm = torch.linalg.vector_norm(flat, s["norm"])
    return norm, flat * min(1.0, s["max_norm"] / (float(norm) + 1e-6))


# ---------------------------------------------------------------------------------- what is called
def prepare(case, seed):
    gen = _gen(seed)
    if case["op"] in ("embed", "embed_grad"):
        s = _prepare_embed(case, gen)
    elif case["op"] in ("qk", "qk_grad"):
        s = _prepare_qk(case, gen)
    else:
        s = _prepare_clip(case, gen)
    s["op"] = case["op"]
    return s


def run(state):
    return {"embed": _embed, "embed_grad": _embed_grad, "qk": _qk, "qk_grad": _qk_grad, "clip": _clip}[state["op"]](state)


def exact(case, seed):
    state = prepare(case, seed)
    return {"embed": _exact_embed, "embed_grad": _exact_embed_grad, "qk": _exact_qk, "qk_grad": _exact_qk_grad,
            "clip": _exact_clip}[case["op"]](state)


def work(case):
    def size(name):
        return torch.empty(0, dtype=_dtype(name)).element_size()

    if case["op"] == "embed":
        n, h = case["tokens"], case["width"]
        return {"bytes": 8 * n + _distinct_rows(case) * h * size(case["table"]) + n * h * size(case["out"]), "flops": n * h}
    if case["op"] == "embed_grad":
        n, h = case["tokens"] * case["parts"], case["width"]
        return {"bytes": 8 * n + n * (1 - case["pad"]) * h * size(case["grad"]) + case["vocab"] * h * 4,
                "flops": n * (1 - case["pad"]) * h}
    if case["op"] in ("qk", "qk_grad"):
        rows, hq, hk, d, rot = (case[k] for k in ("rows", "heads", "kv_heads", "dim", "rot"))
        qk, all_, e = rows * (hq + hk) * d, rows * (hq + 2 * hk) * d, size(case["dtype"])
        table = rot * 4 * min(rows, 32768 if case["far"] else SEQ) + (8 * rows if case["far"] and rot else 0)
        if case["op"] == "qk":
            return {"bytes": 2 * all_ * e + table, "flops": 4 * qk + 3 * rows * (hq + hk) * rot}
        return {"bytes": (qk + 2 * all_) * e + table, "flops": 11 * qk + 3 * rows * (hq + hk) * rot}
    bytes_in = sum(n * torch.empty(0, dtype=_grad_dtype(case, shape)).element_size() for n, shape in zip(_sizes(case), _shapes(case)))
    return {"bytes": bytes_in + 4 * sum(_sizes(case)), "flops": 3 * sum(_sizes(case))}
