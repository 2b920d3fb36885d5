"""The training operators as differentiable functions.

Thin ``torch.autograd.Function`` wrappers over the forward / backward pairs of ``dax_b200.ops``.  The forward passes keep
their inputs and the row statistics, the backward passes recompute the rest; gradients of inputs that do not need one are
not computed where that saves work (dk and dv of attention together, the parameters of the norms together).  Gradients of
gradients, forward-mode derivatives and ``vmap`` are not available: PyTorch raises.

All of them can be captured into a CUDA graph.  A captured backward pass must not meet an eager autograd graph of the same
leaves that is still alive (PyTorch ties a leaf's accumulation to the stream it was first used on): drop the results of
eager passes before the capture, or take gradients with ``torch.autograd.grad``."""
from __future__ import annotations

from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import ops


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, q_lens, k_lens, sm_scale):
        out, lse = ops.attention_lse(q, k, v, q_lens=q_lens, k_lens=k_lens, sm_scale=sm_scale)
        ctx.save_for_backward(q, k, v, out, lse, q_lens, k_lens)
        ctx.sm_scale = sm_scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, q_lens, k_lens = ctx.saved_tensors
        dq, dk, dv = ops.attention_backward(dout, q, k, v, out, lse, q_lens=q_lens, k_lens=k_lens, sm_scale=ctx.sm_scale,
                                            need_keys=any(ctx.needs_input_grad[1:3]))
        return dq, dk, dv, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, q_lens: Optional[torch.Tensor] = None,
              k_lens: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None) -> torch.Tensor:
    """Differentiable non-causal attention over ``[B, heads, S, 128]`` (bf16 or fp16); arguments as ``ops.attention_lse``.
    Inputs that share memory by broadcasting (``expand``) get the sum of their gradients, as everywhere in autograd."""
    return _Attention.apply(q, k, v, q_lens, k_lens, sm_scale)


class _LayerNormModulate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ln_weight, ln_bias, shift, scale, eps):
        y, mean, rstd = ops.layernorm_modulate(x, eps=eps, ln_weight=ln_weight, ln_bias=ln_bias, shift=shift, scale=scale)
        ctx.save_for_backward(x, mean, rstd, ln_weight, ln_bias, scale)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, mean, rstd, ln_weight, ln_bias, scale = ctx.saved_tensors
        dx, dweight, dbias, dshift, dscale = ops.layernorm_modulate_backward(
            dy, x, mean, rstd, ln_weight=ln_weight, ln_bias=ln_bias, scale=scale, need_params=any(ctx.needs_input_grad[1:5]))
        return dx, dweight, dbias, dshift, dscale, None


def _rows(v: Optional[torch.Tensor], x: torch.Tensor) -> Optional[torch.Tensor]:
    """A modulation vector given as ``[D]``, ``[B, D]`` or ``[B, 1, D]`` (or with one row for all samples) as the kernels want it."""
    if v is None:
        return None
    v = v.float()
    if x.dim() == 2:
        return v.reshape(x.shape[1]).contiguous()
    if v.dim() == 3 and v.shape[1] == 1:
        v = v.squeeze(1)
    return v.expand(x.shape[0], x.shape[2]).contiguous()


def layernorm_modulate(x: torch.Tensor, *, eps: float = 1e-6, ln_weight: Optional[torch.Tensor] = None,
                       ln_bias: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
                       scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Differentiable ``ops.layernorm_modulate``.  Weights and modulation may be of any floating type (they are used, and
    their gradients summed, in fp32); ``shift`` and ``scale`` may be ``[D]``, ``[B, D]`` or ``[B, 1, D]``."""
    w, b = (None if v is None else v.float().contiguous() for v in (ln_weight, ln_bias))
    return _LayerNormModulate.apply(x, w, b, _rows(shift, x), _rows(scale, x), eps)


class _RMSNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, norm_weight, rope_cos, rope_sin, eps):
        y, rstd = ops.rmsnorm_rope(x, norm_weight, eps=eps, rope_cos=rope_cos, rope_sin=rope_sin)
        ctx.save_for_backward(x, rstd, norm_weight, rope_cos, rope_sin)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, rstd, norm_weight, rope_cos, rope_sin = ctx.saved_tensors
        dx, dweight = ops.rmsnorm_rope_backward(dy, x, rstd, norm_weight, rope_cos=rope_cos, rope_sin=rope_sin,
                                                need_params=ctx.needs_input_grad[1])
        return dx, dweight, None, None, None


def rmsnorm_rope(x: torch.Tensor, norm_weight: Optional[torch.Tensor] = None, *, eps: float = 1e-6,
                 rope_cos: Optional[torch.Tensor] = None, rope_sin: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Differentiable ``ops.rmsnorm_rope``; the weight may be of any floating type.  The rotary tables are constants."""
    return _RMSNormRope.apply(x, None if norm_weight is None else norm_weight.float().contiguous(), rope_cos, rope_sin, eps)
