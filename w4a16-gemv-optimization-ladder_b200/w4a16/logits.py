"""Processing of a step's logits before the next token is chosen: penalties for repeated tokens,
biases and grammar masks, in one launch.  (The reference takes the argmax of the raw logits,
benchmarks/end_to_end.py:33-37.)"""
import ctypes

import torch

from . import _lib
from .kernels import _need, _stream

_LOGIT_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


def process_logits(logits, *, tokens=None, prompt_lens=None, total_lens=None, repetition=None, frequency=None,
                   presence=None, bias=None, bias_ids=None, bias_values=None, mask=None, out=None):
    """Per row b and token v, in fp32, rounded once to the logits' dtype:

        x = logits[b, v]
        v occurs in tokens[b, :total_lens[b]]:  x = x / repetition[b] if x > 0 else x * repetition[b]
        c = occurrences of v in tokens[b, prompt_lens[b]:total_lens[b]]:
                                                x = x - frequency[b] * c - presence[b] * (c > 0)
        x = x + bias[v] + the bias_values of the row's pairs whose bias_ids equal v
        bit v % 32 of mask[b, v // 32] is 0:    x = -inf

    logits       fp32, fp16 or bf16 [rows, vocab] or [vocab], rows contiguous
    tokens       int32 or int64 [rows, history]: prompt, then generated tokens; ids outside the
                 vocabulary (padding) are skipped
    prompt_lens, total_lens  int32 [rows] (default 0 and history; clamped to history)
    repetition, frequency, presence  fp32 [rows], each optional
    bias         fp32 [vocab] or [rows, vocab]
    bias_ids, bias_values  int32 and fp32 [rows, pairs]; an id outside the vocabulary is skipped, the
                 values of an id named twice are added in their order
    mask         int32 [rows, ceil(vocab / 32)] or [ceil(vocab / 32)]: the allowed tokens' bits
    out          where the result goes (default a new tensor; logits itself will do)"""
    _need(isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dtype in _LOGIT_DTYPES and logits.dim() in (1, 2)
          and (logits.stride(-1) == 1 or logits.shape[-1] <= 1),
          "logits must be an fp32, fp16 or bf16 CUDA tensor [rows, vocab] or [vocab] with contiguous rows")
    dev, one = logits.device, logits.dim() == 1
    rows, vocab = (1, logits.shape[0]) if one else logits.shape
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    else:
        _need(isinstance(out, torch.Tensor) and out.device == dev and out.dtype == logits.dtype and out.shape == logits.shape
              and (out.stride(-1) == 1 or vocab <= 1), "out must have the logits' device, dtype and shape, rows contiguous")

    def per_row(t, dtype, name):
        if t is None:
            return None
        _need(isinstance(t, torch.Tensor) and t.device == dev and t.dtype == dtype and t.shape == (rows,) and t.is_contiguous(),
              f"{name} must be a contiguous {dtype} [{rows}] tensor on {dev}")
        return t.data_ptr()

    d = _lib.LogitsDesc()
    d.logits, d.out, d.dtype, d.rows, d.vocab = logits.data_ptr(), out.data_ptr(), _LOGIT_DTYPES[logits.dtype], rows, vocab
    d.stride, d.out_stride = (vocab, vocab) if rows <= 1 else (logits.stride(0), out.stride(0))
    if tokens is not None:
        _need(isinstance(tokens, torch.Tensor) and tokens.device == dev and tokens.dtype in (torch.int32, torch.int64)
              and tokens.dim() == 2 and tokens.shape[0] == rows and (tokens.stride(1) == 1 or tokens.shape[1] <= 1),
              f"tokens must be an int32 or int64 [{rows}, history] tensor on {dev} with contiguous rows")
        d.tokens, d.token_bytes, d.history = tokens.data_ptr(), tokens.element_size(), tokens.shape[1]
        d.token_stride = tokens.stride(0)
    else:
        _need(prompt_lens is None and total_lens is None and repetition is None and frequency is None and presence is None,
              "penalties and lengths need tokens")
    d.prompt_lens = per_row(prompt_lens, torch.int32, "prompt_lens")
    d.total_lens = per_row(total_lens, torch.int32, "total_lens")
    d.repetition = per_row(repetition, torch.float32, "repetition")
    d.frequency = per_row(frequency, torch.float32, "frequency")
    d.presence = per_row(presence, torch.float32, "presence")
    if bias is not None:
        _need(isinstance(bias, torch.Tensor) and bias.device == dev and bias.dtype == torch.float32
              and bias.shape in ((vocab,), (rows, vocab)) and (bias.stride(-1) == 1 or vocab <= 1),
              f"bias must be an fp32 [{vocab}] or [{rows}, {vocab}] tensor on {dev} with contiguous rows")
        d.bias, d.bias_stride = bias.data_ptr(), bias.stride(0) if bias.dim() == 2 and rows > 1 else 0
    _need((bias_ids is None) == (bias_values is None), "bias_ids and bias_values go together")
    if bias_ids is not None:
        _need(isinstance(bias_ids, torch.Tensor) and bias_ids.device == dev and bias_ids.dtype == torch.int32
              and bias_ids.dim() == 2 and bias_ids.shape[0] == rows and bias_ids.is_contiguous(),
              f"bias_ids must be a contiguous int32 [{rows}, pairs] tensor on {dev}")
        _need(isinstance(bias_values, torch.Tensor) and bias_values.device == dev and bias_values.dtype == torch.float32
              and bias_values.shape == bias_ids.shape and bias_values.is_contiguous(),
              "bias_values must be a contiguous fp32 tensor of the shape of bias_ids")
        d.bias_ids, d.bias_values, d.pairs = bias_ids.data_ptr(), bias_values.data_ptr(), bias_ids.shape[1]
    if mask is not None:
        words = -(-vocab // 32)
        _need(isinstance(mask, torch.Tensor) and mask.device == dev and mask.dtype == torch.int32
              and mask.shape in ((words,), (rows, words)) and (mask.stride(-1) == 1 or words <= 1),
              f"mask must be an int32 [{words}] or [{rows}, {words}] tensor on {dev} with contiguous rows")
        d.mask, d.mask_stride = mask.data_ptr(), mask.stride(0) if mask.dim() == 2 and rows > 1 else 0
    if rows == 0 or vocab == 0:
        return out
    with torch.cuda.device(dev):
        status = _lib.lib().w4a16_process_logits(ctypes.byref(d), _stream(dev))
    _lib.check(status, "w4a16_process_logits")
    return out
