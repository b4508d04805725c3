"""Operators of the model around the optimizer step: embedding, norm and rotation of queries and keys, cross entropy.

The reference's training script composes them from library calls (reference models/gpt_model.py, train.py); here each is one
pass over its data in hand-written kernels, with its gradient:

  * `embedding` / `embedding_backward`
  * `qk_norm_rope` / `qk_norm_rope_backward`, tables by `rope_tables`
  * `cross_entropy` / `cross_entropy_with_grad`

`embedding`, `qk_norm_rope` and `cross_entropy` take part in autograd, with nodes of the native module (first gradients only, none in
forward mode).
Tensors are bfloat16 or float32 on the GPU (there is no CPU or PyTorch fallback); token ids, targets and positions int64 or
int32.  All work goes to the current stream, nothing waits for the GPU, and the results are the same bits every time.
"""
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}   # DION_AMD_REDUCE_*


# ------------------------------------------------------------------------------------------------------------ embedding
def _padding(padding_idx, num_embeddings):
    if padding_idx is None:
        return -1
    if not -num_embeddings <= padding_idx < num_embeddings:
        raise ValueError(f"padding_idx {padding_idx} is outside the table of {num_embeddings} rows")
    return padding_idx % num_embeddings


def embedding(weight: Tensor, tokens: Tensor, *, scale: float = 1.0, padding_idx: Optional[int] = None,
              out_dtype: Optional[torch.dtype] = None) -> Tensor:
    """`scale * weight[tokens]`, rounded once to `out_dtype` (default: the table's).

    tokens: any shape; a token outside the table gives a row of NaN.  padding_idx: a token whose rows leave no gradient."""
    padding = -1 if padding_idx is None else _padding(padding_idx, weight.size(0))
    return _lib.host().embedding(weight, tokens, scale, padding, out_dtype)


def embedding_backward(grad: Tensor, tokens: Tensor, num_embeddings: int, *, scale: float = 1.0,
                       padding_idx: Optional[int] = None, dtype: Optional[torch.dtype] = None, out: Optional[Tensor] = None,
                       accumulate: bool = False) -> Tensor:
    """The dense gradient of the table: row v is `scale` times the sum of `grad` over the places where `tokens` is v.

    Sums are fp32, rounded once to `dtype` (default: that of `grad`); all tokens together determine their order, so that the last bits
    of a row may change with tokens of other rows.  out: the tensor to write, not over an input; with accumulate=True the gradient is
    added to what is in it, and rows that no token names are not touched."""
    return _lib.host().embedding_grad(grad, tokens, num_embeddings, _padding(padding_idx, num_embeddings), scale, dtype, out,
                                      accumulate)


# ---------------------------------------------------------------------------------------------------------- q / k norms
def rope_tables(length: int, rotary: int, *, base: float = 10000.0, device=None) -> Tuple[Tensor, Tensor]:
    """Cosines and sines (length, rotary / 2) of the angles `position * base ** (-2 i / rotary)`, float32."""
    if rotary < 0 or rotary % 2:
        raise ValueError(f"the number of rotated channels must be even, got {rotary}")
    half = rotary // 2
    speed = base ** (-torch.arange(half, dtype=torch.float64, device=device) / max(half, 1))
    angles = torch.arange(length, dtype=torch.float64, device=device)[:, None] * speed
    return angles.cos().float(), angles.sin().float()


def qk_norm_rope(q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, *, q_gain: Optional[Tensor] = None,
                 k_gain: Optional[Tensor] = None, positions: Optional[Tensor] = None, eps: float = 1e-6,
                 interleaved: bool = False) -> Tuple[Tensor, Tensor]:
    """RMS norm of every head of q and k and the rotation of its first channels by its position, in one pass.

    q: (batch, length, heads, channels), k the same with heads of its own; any strides with contiguous channels, so that both
    may be slices of one projection's output.  The results are contiguous.
    cos, sin: float32 (positions, rotary / 2), see `rope_tables`; constants, refused if a gradient of theirs is wanted.
    The pairs (i, i + rotary / 2) are turned, (u, v) -> (u cos - v sin, v cos + u sin), the pairs (2i, 2i + 1) if `interleaved`;
    channels from `rotary` on are only normed.  A model that turns the other way passes `-sin`.
    q_gain, k_gain: a factor for each channel.  positions: (length) or (batch, length), default 0, 1, 2, ...; a position outside
    the tables gives NaN."""
    return _lib.host().qk_norm_rope(q, k, cos, sin, q_gain, k_gain, positions, eps, interleaved)


def qk_norm_rope_backward(dq: Tensor, dk: Tensor, q: Tensor, k: Tensor, cos: Tensor, sin: Tensor, *,
                          q_gain: Optional[Tensor] = None, k_gain: Optional[Tensor] = None,
                          positions: Optional[Tensor] = None, eps: float = 1e-6, interleaved: bool = False):
    """(dq, dk, dq_gain, dk_gain) from the gradients of `qk_norm_rope`'s results and its arguments; None for absent gains."""
    return _lib.host().qk_norm_rope_grad(q, k, cos, sin, q_gain, k_gain, positions, eps, interleaved, dq, dk)


# -------------------------------------------------------------------------------------------------------- cross entropy
def _reduction(name, allowed=("none", "sum", "mean")):
    if name not in allowed:
        raise ValueError(f"reduction must be one of {allowed}, got {name!r}")
    return _REDUCTIONS[name]


def cross_entropy(logits: Tensor, targets: Tensor, *, ignore_index: int = -100, reduction: str = "mean", softcap: float = 0.0,
                  z_loss: float = 0.0) -> Tensor:
    """Cross entropy over the last dimension, in float32.

    logits: the shape of `targets` and the classes; rows at any pitch, so that padded logits go as `logits[..., :vocab]`.
    softcap: logits are taken as `softcap * tanh(logits / softcap)` (0: as they are; else 1e-30 to 1e30).  z_loss: adds `z_loss * lse ** 2`, lse the
    logarithm of the sum of exponentials.  Targets equal to `ignore_index` have no loss and no gradient, and "mean" is over the
    others (NaN if there are none); any other target outside the classes gives NaN."""
    return _lib.host().cross_entropy(logits, targets, ignore_index, softcap, z_loss, _reduction(reduction))


def cross_entropy_with_grad(logits: Tensor, targets: Tensor, *, ignore_index: int = -100, reduction: str = "mean",
                            softcap: float = 0.0, z_loss: float = 0.0, grad_scale: float = 1.0,
                            inplace: bool = False) -> Tuple[Tensor, Tensor]:
    """(loss, gradient of `grad_scale * loss` with respect to the logits) in one read and one write of the logits.

    For the loss at the end of a model, where the upstream gradient is known beforehand: `logits.backward(dlogits)` then goes on
    from there.  inplace=True writes the gradient over the logits.  reduction: "mean" or "sum"; else as `cross_entropy`."""
    return _lib.host().cross_entropy_with_grad(logits, targets, ignore_index, softcap, z_loss,
                                               _reduction(reduction, ("sum", "mean")), grad_scale, inplace)
