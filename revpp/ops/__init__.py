"""Thin Python entry points of the sm_100a kernels (module ``revpp._C``).

Every function here takes CUDA tensors and launches the extension's kernels on the
current stream; there is no PyTorch fallback on the GPU.  CPU execution goes through
``revpp.models.blockmath.TorchMath`` instead.
"""
from __future__ import annotations

import os
from typing import Optional

import torch

from ._ext import available, check_status, ext

EPI_BF16, EPI_GELU, EPI_RESID, EPI_ATOMIC, EPI_DGELU, EPI_F32 = range(6)

_SM_RESERVE = 0


def set_sm_reserve(n: int) -> None:
    """Leave ``n`` SMs free of persistent GEMM CTAs (for concurrent NCCL kernels)."""
    global _SM_RESERVE
    _SM_RESERVE = max(0, int(n))
    if available():
        ext().set_sm_reserve(_SM_RESERVE)


def linear(x: torch.Tensor, w: torch.Tensor, out: torch.Tensor, bias: Optional[torch.Tensor] = None,
           epi: int = EPI_BF16, aux_out: Optional[torch.Tensor] = None, resid: Optional[torch.Tensor] = None,
           sign: float = 1.0) -> torch.Tensor:
    """out[M, N] = epi(x[M, K] @ w[N, K]^T + bias)   (forward GEMM, both operands K-major)."""
    M, K = x.shape
    N = w.shape[0]
    ext().gemm_tc(x, False, w, False, M, N, K, epi, out, bias=bias, aux_out=aux_out, resid=resid, sign=sign)
    return out


def linear_dgrad(dy: torch.Tensor, w: torch.Tensor, out: torch.Tensor, epi: int = EPI_BF16,
                 aux: Optional[torch.Tensor] = None, colsum: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[M, K] = epi(dy[M, N] @ w[N, K])   (input gradient; w read MN-major).  With the
    GELU-backward epilogue, ``colsum`` (fp32 [K]) accumulates the column sums of ``out``."""
    M, N = dy.shape
    K = w.shape[1]
    ext().gemm_tc(dy, False, w, True, M, K, N, epi, out, aux=aux, colsum=colsum)
    return out


def linear_wgrad(dy: torch.Tensor, x: torch.Tensor, dw: torch.Tensor, splits: Optional[int] = None) -> torch.Tensor:
    """dw[N, K] += dy[M, N]^T @ x[M, K]   (weight gradient, fp32 accumulation with atomics)."""
    M, N = dy.shape
    K = x.shape[1]
    C = ext()
    if splits is None:
        splits = C.gemm_suggest_splits(N, K, M)
    C.gemm_tc(dy, True, x, True, N, K, M, EPI_ATOMIC, dw, splits=splits)
    return dw


def layernorm_fwd(x, gamma, beta, eps, y_bf16=None, y_f32=None, y2_f32=None, mean=None, rstd=None):
    ext().layernorm_fwd(x, gamma, beta, eps, y_bf16=y_bf16, y_f32=y_f32, y2_f32=y2_f32, mean=mean, rstd=rstd)


def layernorm_bwd(dy, x, gamma, mean, rstd, dgamma=None, dbeta=None, resid=None, dx_f32=None, dx_bf16=None,
                  colsum=None):
    ext().layernorm_bwd(dy, x, gamma, mean, rstd, dgamma=dgamma, dbeta=dbeta, resid=resid, dx_f32=dx_f32,
                        dx_bf16=dx_bf16, colsum=colsum)


def cast_colsum(inp, out=None, colsum=None):
    ext().cast_colsum(inp, out=out, colsum=colsum)


_ATTN_TC = os.environ.get("REVPP_ATTN_TC", "1") != "0"
_ATTN_FWD = os.environ.get("REVPP_ATTN_FWD", "grid")


def attention_fwd(qkv, out, lse, B, S, heads):
    """Flash attention forward: the tcgen05 kernel with one CTA per query tile, two CTAs per
    SM (REVPP_ATTN_FWD=persistent selects the persistent kernel, measured slower at head
    dim 64; REVPP_ATTN_TC=0 the warp-level mma.sync kernel; both kept as comparison points)."""
    if not _ATTN_TC:
        ext().attn_fwd(qkv, out, lse, B, S, heads)
    elif _ATTN_FWD == "persistent":
        ext().attn_fwd_persistent(qkv, out, lse, B, S, heads)
    else:
        ext().attn_fwd_tc(qkv, out, lse, B, S, heads)


def attention_bwd(qkv, out, dout, lse, dqkv, dq_acc, dbuf, B, S, heads, colsum=None):
    """Flash attention backward (tcgen05; REVPP_ATTN_TC=0 selects the mma.sync kernel).
    ``colsum`` (fp32 [3H]) accumulates the column sums of dqkv (the in-projection bias
    gradient); the tcgen05 path fuses it into its write-out."""
    if _ATTN_TC:
        ext().attn_bwd_tc(qkv, out, dout, lse, dqkv, dq_acc, dbuf, B, S, heads, colsum=colsum)
    else:
        ext().attn_bwd(qkv, out, dout, lse, dqkv, dq_acc, dbuf, B, S, heads)
        if colsum is not None:
            cast_colsum(dqkv, colsum=colsum)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` as [rows, last dimension] without a copy."""
    return t if t.dim() == 2 else t.view(-1, t.shape[-1])


def _ids(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def embedding_fwd(ids: torch.Tensor, w: torch.Tensor, out: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """out[..., :] = scale * w[ids[...]]   (token-embedding lookup).

    ``ids`` int64 / int32 of any shape, ``w`` [V, H] and ``out`` [..., H] each fp32, bf16 or
    fp16, contiguous along H (rows may lie further apart).  An id outside the table sets the
    status word (``check_status``) and gives a row of zeros."""
    ext().embedding_fwd(_ids(ids), w, _rows(out), scale)
    return out


def embedding_bwd(dy: torch.Tensor, ids: torch.Tensor, dw: torch.Tensor, scale: float = 1.0,
                  padding_idx: Optional[int] = None, accumulate: bool = True) -> torch.Tensor:
    """dw[v] (+)= scale * sum of dy[t] over the tokens with ids[t] = v   (gradient of ``embedding_fwd``).

    ``dy`` [..., H] fp32, bf16 or fp16, ``dw`` [V, H] fp32.  The tokens of ``padding_idx`` and ids
    outside the table add nothing.  ``accumulate=False`` writes all of ``dw``, with zeros in the rows
    that no token names.  ``accumulate=True`` adds to the rows that tokens name, and takes subnormal
    numbers (below 2^-126) among the old values, the terms and the sums as zero, like other fp32 atomics.
    The tokens are sorted first and each row's terms are added in an order that their positions in the
    sorted list fix (eight at a time, then across warps and chunks): equal inputs give equal bits,
    unlike the atomics of ``bert_embed_bwd``."""
    V = dw.shape[0]
    if padding_idx is None:
        padding_idx = -1
    elif not -V <= padding_idx < V:
        raise ValueError(f"padding_idx {padding_idx} is outside the table's {V} rows")
    elif padding_idx < 0:
        padding_idx += V
    ext().embedding_bwd(_rows(dy), _ids(ids), dw, scale, padding_idx, accumulate)
    return dw


def qk_norm_rope_fwd(qkv: torch.Tensor, out: torch.Tensor, heads: int, kv_heads: Optional[int] = None,
                     wq: Optional[torch.Tensor] = None, wk: Optional[torch.Tensor] = None, eps: float = 1e-6,
                     cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                     positions: Optional[torch.Tensor] = None, S: Optional[int] = None,
                     interleaved: bool = False) -> torch.Tensor:
    """RMS norm of every query and key head, then the position rotation, on a packed projection.

    ``qkv`` and ``out`` are [M, (heads + 2 * kv_heads) * d] (fp32, bf16 or fp16, d <= 256, rows may
    lie further apart); ``kv_heads`` defaults to ``heads``, which is the layout that
    ``attention_fwd`` reads.  ``out`` may be ``qkv`` itself; otherwise the value heads are copied.
    ``wq`` / ``wk`` are the fp32 [d] norm weights (None: 1).  ``cos`` / ``sin`` (fp32 [P, rot / 2], None:
    no rotation) turn the first ``rot`` columns of a head in pairs (i, i + rot / 2), or (2i, 2i + 1)
    with ``interleaved``; row m takes the angles of ``positions[m]`` (int64 / int32 [M]), or of
    ``m % S``.  A position outside the tables sets the status word and leaves its row unrotated."""
    ext().qk_norm_rope_fwd(qkv, out, heads, heads if kv_heads is None else kv_heads, wq, wk, eps, cos, sin, positions,
                           S, interleaved)
    return out


def qk_norm_rope_bwd(dout: torch.Tensor, qkv: torch.Tensor, dqkv: torch.Tensor, heads: int,
                     kv_heads: Optional[int] = None, wq: Optional[torch.Tensor] = None,
                     wk: Optional[torch.Tensor] = None, dwq: Optional[torch.Tensor] = None,
                     dwk: Optional[torch.Tensor] = None, eps: float = 1e-6, cos: Optional[torch.Tensor] = None,
                     sin: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                     S: Optional[int] = None, interleaved: bool = False, accumulate: bool = True) -> torch.Tensor:
    """Gradient of ``qk_norm_rope_fwd``: ``dqkv`` from ``dout`` and the projection ``qkv`` as it was
    before the norm.  ``dqkv`` may be ``dout`` itself (value heads stay), otherwise the value heads'
    gradient is copied.  ``dwq`` / ``dwk`` (fp32 [d], optional) receive the norm weights' gradients:
    added, or written with ``accumulate=False``; their sums are taken in a fixed order."""
    ext().qk_norm_rope_bwd(dout, qkv, dqkv, heads, heads if kv_heads is None else kv_heads, wq, wk, dwq, dwk, eps, cos,
                           sin, positions, S, interleaved, accumulate)
    return dqkv


def clip_grads(grads, max_norm: float, out=None, norm_type: float = 2.0) -> torch.Tensor:
    """Scale many gradient tensors by min(1, max_norm / (norm + 1e-6)) and return their global norm
    (fp32 scalar on the device, no synchronisation).

    ``grads``: dense fp32 / bf16 / fp16 tensors on one device, of any number and sizes.  ``out``: where
    the scaled gradients go (same sizes and strides, any of the three types), by default the gradients
    themselves.  ``norm_type`` is 2 or inf.  Squares are summed in 64 bits in a fixed order.  A NaN in
    any gradient makes the norm and every output NaN."""
    if norm_type not in (2.0, float("inf")):
        raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")
    return ext().clip_grads(list(grads), max_norm, None if out is None else list(out), norm_type != 2.0)


__all__ = [
    "available", "check_status", "ext", "set_sm_reserve", "linear", "linear_dgrad", "linear_wgrad",
    "layernorm_fwd", "layernorm_bwd", "cast_colsum", "attention_fwd", "attention_bwd",
    "embedding_fwd", "embedding_bwd", "qk_norm_rope_fwd", "qk_norm_rope_bwd", "clip_grads",
    "EPI_BF16", "EPI_GELU", "EPI_RESID", "EPI_ATOMIC", "EPI_DGELU", "EPI_F32",
]
