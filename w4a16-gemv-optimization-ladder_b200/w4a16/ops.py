"""The library's products as registered torch operators (namespace `w4a16`).

The reference exposes its kernels only through a pybind11 module (kernels/w4a16_kernels.cu:
189-195), invisible to torch's dispatcher.  Registering them lets torch code call
`torch.ops.w4a16.gemv(...)` and trace models that use them (the fake implementations give
output shapes and dtypes without running anything); the implementations call the C ABI
through w4a16.kernels, on the current stream.

    torch.ops.w4a16.gemv(packed, scale, x, group) -> fp32 [rows] or [batch, rows]
    torch.ops.w4a16.gemv_rmsnorm(packed, scale, h, gamma, eps, group) -> fp32 [rows]
    torch.ops.w4a16.gemv_swiglu(packed, scale, gate_up, group) -> fp32 [rows]
    torch.ops.w4a16.dequant(packed, scale, group) -> fp16 [rows, cols]
    torch.ops.w4a16.paged_attention(q, k_pages, v_pages, tables, lengths, seqs, scale) -> [rows, heads, head_dim]
    torch.ops.w4a16.process_logits(logits, tokens, prompt_lens, total_lens, repetition, frequency, presence, bias,
                                   bias_ids, bias_values, mask) -> like logits
"""
from typing import Optional

import torch

from . import kernels as K
from . import logits as _logits
from . import paged as _paged


@torch.library.custom_op("w4a16::gemv", mutates_args=())
def gemv(packed: torch.Tensor, scale: torch.Tensor, x: torch.Tensor, group: int) -> torch.Tensor:
    return K.gemv(packed, scale, x, group=group)


@gemv.register_fake
def _(packed, scale, x, group):
    rows = packed.shape[0]
    shape = (rows,) if x.dim() == 1 else (x.shape[0], rows)
    return packed.new_empty(shape, dtype=torch.float32)


@torch.library.custom_op("w4a16::gemv_rmsnorm", mutates_args=())
def gemv_rmsnorm(packed: torch.Tensor, scale: torch.Tensor, h: torch.Tensor, gamma: torch.Tensor,
                 eps: float, group: int) -> torch.Tensor:
    return K.gemv_rmsnorm(packed, scale, h, gamma, eps, group=group)


@gemv_rmsnorm.register_fake
def _(packed, scale, h, gamma, eps, group):
    return packed.new_empty((packed.shape[0],), dtype=torch.float32)


@torch.library.custom_op("w4a16::gemv_swiglu", mutates_args=())
def gemv_swiglu(packed: torch.Tensor, scale: torch.Tensor, gate_up: torch.Tensor, group: int) -> torch.Tensor:
    return K.gemv_swiglu(packed, scale, gate_up, group=group)


@gemv_swiglu.register_fake
def _(packed, scale, gate_up, group):
    return packed.new_empty((packed.shape[0],), dtype=torch.float32)


@torch.library.custom_op("w4a16::dequant", mutates_args=())
def dequant(packed: torch.Tensor, scale: torch.Tensor, group: int) -> torch.Tensor:
    return K.dequant_int4(packed, scale, group=group)


@dequant.register_fake
def _(packed, scale, group):
    return packed.new_empty((packed.shape[0], packed.shape[1] * 2), dtype=torch.float16)


@torch.library.custom_op("w4a16::paged_attention", mutates_args=())
def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, tables: torch.Tensor,
                    lengths: torch.Tensor, seqs: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    return _paged.paged_attention(q, k_pages, v_pages, tables, lengths, seqs=seqs, scale=scale)


@paged_attention.register_fake
def _(q, k_pages, v_pages, tables, lengths, seqs=None, scale=None):
    return q.new_empty(q.shape)


@torch.library.custom_op("w4a16::process_logits", mutates_args=())
def process_logits(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, prompt_lens: Optional[torch.Tensor] = None,
                   total_lens: Optional[torch.Tensor] = None, repetition: Optional[torch.Tensor] = None,
                   frequency: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, bias_ids: Optional[torch.Tensor] = None,
                   bias_values: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None) -> torch.Tensor:
    return _logits.process_logits(logits, tokens=tokens, prompt_lens=prompt_lens, total_lens=total_lens, repetition=repetition,
                                  frequency=frequency, presence=presence, bias=bias, bias_ids=bias_ids, bias_values=bias_values,
                                  mask=mask)


@process_logits.register_fake
def _(logits, tokens=None, prompt_lens=None, total_lens=None, repetition=None, frequency=None, presence=None, bias=None,
      bias_ids=None, bias_values=None, mask=None):
    return logits.new_empty(logits.shape)
