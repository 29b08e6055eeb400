"""Definitions in 64 bits of the embedding, query/key norm and clipping operators, with bounds on
the rounding errors of their fp32 kernels.

``U`` is half a step of fp32 relative to the value and ``half_step(t)`` that of the output type;
results below a type's normal range are rounded to its smallest step, ``tiny(t)`` is half of it.
"""
import torch

U = 2.0 ** -24


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def within(got, want, bound):
    """Elementwise |got - want| <= bound (1 % above it for second-order terms)."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    over = (got - want).abs() - 1.01 * bound
    assert over.max().item() <= 0, f"off by {(got - want).abs().max().item():.3g}, over its bound by {over.max().item():.3g}"


# ---------------------------------------------------------------- embedding
def embed(ids, w, scale):
    ok = (ids >= 0) & (ids < w.shape[0])
    rows = w.double()[torch.where(ok, ids, torch.zeros_like(ids)).long().reshape(-1)] * scale
    return (rows * ok.reshape(-1, 1)).view(*ids.shape, w.shape[1])


def embed_bound(want, out_type):
    # one product in fp32, one rounding to the output type
    return want.abs() * (U + half_step(out_type)) + tiny(out_type)


def embed_grad(dy, ids, vocab, scale, padding_idx=None):
    """(sum, bound): k terms added in fp32 in any order are off by at most (k - 1) U sum |x|, the
    product with the scale adds U."""
    ids, dy = ids.reshape(-1).long(), dy.double().reshape(ids.numel(), -1)
    ok = (ids >= 0) & (ids < vocab)
    if padding_idx is not None:
        ok &= ids != padding_idx
    ids, dy = ids[ok], dy[ok]
    total = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device=dy.device).index_add_(0, ids, dy)
    size = torch.zeros_like(total).index_add_(0, ids, dy.abs())
    terms = torch.zeros(vocab, dtype=torch.float64, device=dy.device).index_add_(0, ids, torch.ones_like(ids, dtype=torch.float64))
    return total * scale, size * abs(scale) * (terms[:, None] + 2) * U


# ---------------------------------------------------------------- query / key norm and rotation
def tables(length, rot, device):
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * torch.pow(
        10000.0, -torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    return angle.cos().float(), angle.sin().float()


def turn(z, cos, sin, interleaved):
    """R z for z [..., heads, d] with cos / sin [rows, rot / 2] (None: z)."""
    if cos is None:
        return z
    h = cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = (z[..., 0:2 * h:2], z[..., 1:2 * h:2]) if interleaved else (z[..., :h], z[..., h:2 * h])
    p, q = a * c - b * s, a * s + b * c
    front = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([front, z[..., 2 * h:]], -1)


def norm_turn(x, w, eps, cos, sin, interleaved):
    """x [rows, heads, d] in 64 bits."""
    z = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return turn(z if w is None else z * w.double(), cos, sin, interleaved)


def _magnitude(z, cos, sin, interleaved):
    """|z1 c| + |z2 s| and |z1 s| + |z2 c| of every pair: what the rotation's rounding scales with."""
    if cos is None:
        return z.abs()
    return turn_abs(z.abs(), cos.abs(), sin.abs(), interleaved)


def turn_abs(z, cos, sin, interleaved):
    h = cos.shape[1]
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = (z[..., 0:2 * h:2], z[..., 1:2 * h:2]) if interleaved else (z[..., :h], z[..., h:2 * h])
    p, q = a * c + b * s, a * s + b * c
    front = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([front, z[..., 2 * h:]], -1)


def r_error(d):
    """Relative error of r: the sum of d squares (d U), its product with 1 / d and the addition of
    eps (3 U) under the root, which halves them, and 2 units in the last place (4 U) of rsqrtf."""
    return (d / 2 + 6) * U


def norm_turn_bound(x, w, eps, cos, sin, interleaved, out_type):
    d = x.shape[-1]
    z = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    z = z if w is None else z * w.double()
    y = turn(z, cos, sin, interleaved)
    # r w and x (r w) round once each, a rotated pair's product and sum once each
    return _magnitude(z, cos, sin, interleaved) * (r_error(d) + 4 * U) + y.abs() * half_step(out_type) + tiny(out_type)


def norm_turn_grad(x, w, dy, eps, cos, sin, interleaved):
    """(dx, dw, bound of dx before its last rounding, bound of dw)."""
    rows, heads, d = x.shape
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    wd = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    back = None if sin is None else -sin
    dz = turn(dy, cos, back, interleaved)
    a = _magnitude(dy, cos, back, interleaved)          # dz rounds to within 2 U a
    xn = x * r
    g = dz * wd
    dx = r * (g - xn * (g * xn).mean(-1, keepdim=True))
    dw = (dz * xn).sum((0, 1))
    e = r_error(d)
    spread = (a * wd.abs() * x.abs()).mean(-1, keepdim=True) * r * r     # at least |mean(g x r) r|
    # the mean: d + 5 roundings and r twice; each product and the difference once
    dx_bound = r * (a * wd.abs() * (e + 6 * U) + x.abs() * spread * (3 * e + (d + 11) * U))
    dw_bound = (a * xn.abs()).sum((0, 1)) * (e + (rows * heads + 5) * U)
    return dx, dw, dx_bound, dw_bound
