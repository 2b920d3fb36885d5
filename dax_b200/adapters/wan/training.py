"""Differentiable forward of a Wan DiT block: distillation and fine-tuning (LoRA included) of the model that the inference
adapters serve.

``enable_training`` is to training what ``optimize_pipe`` is to inference: it installs an attention processor and binds a
block forward, both built from the operators with gradients (``dax_b200.autograd``): LayerNorm + modulation, RMSNorm +
rotary embedding and attention run as CUDA kernels in both directions, whole batches at a time; the linears stay whatever
modules the model has (their products are library GEMMs), so adapters around them keep working.  The reference has no
training path; the formulas are those of the block that ``dax/adapters/wan/transformer_adapter.py:127-134`` loops over and
of the processor ``dax/adapters/wan/attn_adapter.py:62-304``.

Quantised linears have no gradient, the sequence-parallel exchange has no backward pass here, and the forward that
``optimize_pipe`` binds on the transformer ends in an operator without one: all three are refused."""
from __future__ import annotations

import types
from typing import Optional

import torch

from ... import autograd
from ...parallel import dist as para_dist
from ...quant.nn.dynamic import Linear as QLinear
from .attn_adapter import HEAD_DIM
from .block_adapter import _block_classes
from .transformer_adapter import dit_forward


def _rotary_tables(rotary_emb: torch.Tensor):
    """Complex ``[1, 1, S, 64]`` table -> fp32 cos / sin ``[S, 64]``, made on the current stream for each call: autograd keeps them
    for the backward pass (512 bytes per token and layer), a captured graph makes them again at every replay."""
    r = torch.view_as_real(rotary_emb.reshape(-1, rotary_emb.shape[-1]))
    return r[..., 0].to(torch.float32).contiguous(), r[..., 1].to(torch.float32).contiguous()


class DAXWanTrainingAttnProcessor:
    """Attention processor with a gradient; the call protocol of ``DAXWanAttnProcessor2_0``, and ``context_lens`` (int32
    ``[B]`` on the device): the tokens of each text context that exist, where contexts of different lengths are padded."""

    def __call__(self, attn, hidden_states: torch.Tensor, encoder_hidden_states: Optional[torch.Tensor] = None,
                 attention_mask: Optional[torch.Tensor] = None, rotary_emb: Optional[torch.Tensor] = None,
                 context_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
        if getattr(attn, "add_k_proj", None) is not None:
            raise NotImplementedError("training of the image branch (add_k_proj) is not supported")
        if attention_mask is not None:
            raise NotImplementedError("the attention kernels take lengths (context_lens), not an attention_mask")
        if not hidden_states.is_cuda:
            raise RuntimeError("DAXWanTrainingAttnProcessor runs on CUDA tensors only; there is no CPU fallback")
        if context_lens is not None and encoder_hidden_states is None:
            raise ValueError("context_lens belongs to cross-attention")
        context = hidden_states if encoder_hidden_states is None else encoder_hidden_states
        B, S, D = hidden_states.shape
        if D != attn.heads * HEAD_DIM:
            raise ValueError(f"hidden size {D} != heads {attn.heads} x {HEAD_DIM}")
        cos = sin = None
        if rotary_emb is not None:
            cos, sin = _rotary_tables(rotary_emb)

        def heads(t):
            return t.unflatten(2, (attn.heads, HEAD_DIM)).transpose(1, 2)

        def norm(t, n, rotate):
            if n is None and not rotate:
                return t
            if n is None:
                raise NotImplementedError("rotation without a norm in front of it is not supported in training")
            return autograd.rmsnorm_rope(t, getattr(n, "weight", None), eps=n.eps, rope_cos=cos if rotate else None,
                                         rope_sin=sin if rotate else None)

        rotate = rotary_emb is not None
        q = norm(attn.to_q(hidden_states), attn.norm_q, rotate)
        k = norm(attn.to_k(context), attn.norm_k, rotate)
        out = autograd.attention(heads(q), heads(k), heads(attn.to_v(context)), k_lens=context_lens)
        out = out.transpose(1, 2).flatten(2)
        return attn.to_out[1](attn.to_out[0](out))


def training_block_forward(self, hidden_states, encoder_hidden_states, temb, rotary_emb):
    """Drop-in for ``WanTransformerBlock.forward(hidden_states, encoder_hidden_states, temb, rotary_emb)`` with a gradient."""
    h = hidden_states
    shift_msa, scale_msa, gate_msa, c_shift, c_scale, c_gate = (self.scale_shift_table.float() + temb.float()).unbind(1)
    n = autograd.layernorm_modulate(h, eps=self.norm1.eps, shift=shift_msa, scale=scale_msa)
    h = (h.float() + self.attn1(n, rotary_emb=rotary_emb) * gate_msa[:, None]).type_as(h)
    n = h
    if not isinstance(self.norm2, torch.nn.Identity):
        n = autograd.layernorm_modulate(h, eps=self.norm2.eps, ln_weight=self.norm2.weight, ln_bias=self.norm2.bias)
    h = h + self.attn2(n, encoder_hidden_states=encoder_hidden_states)
    n = autograd.layernorm_modulate(h, eps=self.norm3.eps, shift=c_shift, scale=c_scale)
    return (h.float() + self.ffn(n).float() * c_gate[:, None]).type_as(h)


def enable_training(pipe) -> int:
    """Installs the differentiable processor and block forward on every Wan block of ``pipe.transformer``; returns how many
    blocks were bound."""
    if para_dist.parallel_state.is_enable_sequence_parallel():
        raise NotImplementedError("training under sequence parallelism is not supported: the exchange has no backward pass")
    for name, m in pipe.transformer.named_modules():
        if isinstance(m, QLinear):
            raise NotImplementedError(f"{name} is quantised and has no gradient: enable training before quantising")
    if getattr(getattr(pipe.transformer, "forward", None), "__func__", None) is dit_forward:
        raise NotImplementedError("the transformer has the inference forward of optimize_pipe, which has no gradient: enable training on a pipe "
                                  "that has not been optimised")
    n = 0
    for _, m in pipe.transformer.named_modules():
        if isinstance(m, _block_classes()):
            for attn in (m.attn1, m.attn2):
                attn.set_processor(DAXWanTrainingAttnProcessor())
            m.forward = types.MethodType(training_block_forward, m)
            n += 1
    return n
