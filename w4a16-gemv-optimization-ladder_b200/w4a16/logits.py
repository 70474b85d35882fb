"""Processing of a step's logits before the next token is chosen: penalties for repeated tokens,
biases and grammar masks, in one launch.  (The reference takes the argmax of the raw logits,
benchmarks/end_to_end.py:33-37.)"""
import torch

from . import _lib
from .paged import _call, _refuse

_LOGIT_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}


def _per_row(t, rows, dtype, name, dev):
    if t is None:
        return 0
    if not (isinstance(t, torch.Tensor) and t.dtype is dtype and t.device == dev and t.dim() == 1 and t.shape[0] == rows
            and t.is_contiguous()):
        _refuse(f"{name} must be a contiguous {dtype} [{rows}] tensor on {dev}")
    return t.data_ptr()


def _rows(t, dtypes, shapes, name, dev):
    """A tensor of one of these shapes whose rows are contiguous."""
    if not (isinstance(t, torch.Tensor) and t.device == dev and t.dtype in dtypes and t.shape in shapes
            and (t.stride(-1) == 1 or t.shape[-1] <= 1)):
        _refuse(f"{name} must be a {' or '.join(map(str, dtypes))} tensor {' or '.join(str(list(x)) for x in shapes)} on {dev} with "
                "contiguous rows")
    return t.data_ptr()


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
    repetition, frequency, presence  fp32 [rows], each optional; a repetition lies between 2^-126 and 2^100
    bias         fp32 [vocab] or [rows, vocab]
    bias_ids, bias_values  int32 and fp32 [rows, pairs]; an id outside the vocabulary is skipped, the
                 values of an id named twice are added in their order
    mask         int32 [rows, ceil(vocab / 32)] or [ceil(vocab / 32)]: the allowed tokens' bits
    out          where the result goes (default a new tensor; logits itself will do)"""
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dtype in _LOGIT_DTYPES and logits.dim() in (1, 2)
            and (logits.stride(-1) == 1 or logits.shape[-1] <= 1)):
        _refuse("logits must be an fp32, fp16 or bf16 CUDA tensor [rows, vocab] or [vocab] with contiguous rows")
    dev, shape = logits.device, logits.shape
    rows, vocab = (1, shape[0]) if len(shape) == 1 else shape
    if out is None:
        out = logits.new_empty(*shape)
    else:
        _rows(out, (logits.dtype,), (shape,), "out", dev)
    tp = pl = tl = rp = fp = pp = bp = ip = vp = mp = 0
    token_bytes = history = token_stride = bias_stride = pairs = mask_stride = 0
    if tokens is not None:
        if not (isinstance(tokens, torch.Tensor) and tokens.dim() == 2):
            _refuse(f"tokens must be an int32 or int64 [{rows}, history] tensor")
        history = tokens.shape[1]
        tp = _rows(tokens, (torch.int32, torch.int64), ((rows, history),), "tokens", dev)
        token_bytes, token_stride = tokens.element_size(), tokens.stride(0)
        pl = _per_row(prompt_lens, rows, torch.int32, "prompt_lens", dev)
        tl = _per_row(total_lens, rows, torch.int32, "total_lens", dev)
        rp = _per_row(repetition, rows, torch.float32, "repetition", dev)
        fp = _per_row(frequency, rows, torch.float32, "frequency", dev)
        pp = _per_row(presence, rows, torch.float32, "presence", dev)
    elif not (prompt_lens is total_lens is repetition is frequency is presence is None):
        _refuse("penalties and lengths need tokens")
    if bias is not None:
        bp = _rows(bias, (torch.float32,), ((vocab,), (rows, vocab)), "bias", dev)
        bias_stride = bias.stride(0) if bias.dim() == 2 and rows > 1 else 0
    if bias_ids is not None or bias_values is not None:
        if not (isinstance(bias_ids, torch.Tensor) and bias_ids.dim() == 2 and isinstance(bias_values, torch.Tensor)
                and bias_ids.is_contiguous() and bias_values.is_contiguous()):
            _refuse(f"bias_ids and bias_values must be contiguous [{rows}, pairs] tensors, and go together")
        pairs = bias_ids.shape[1]
        ip = _rows(bias_ids, (torch.int32,), ((rows, pairs),), "bias_ids", dev)
        vp = _rows(bias_values, (torch.float32,), ((rows, pairs),), "bias_values", dev)
    if mask is not None:
        words = -(-vocab // 32)
        mp = _rows(mask, (torch.int32,), ((words,), (rows, words)), "mask", dev)
        mask_stride = mask.stride(0) if mask.dim() == 2 and rows > 1 else 0
    if rows and vocab:
        stride, out_stride = (vocab, vocab) if rows == 1 else (logits.stride(0), out.stride(0))
        d = _lib.pack_logits(logits.data_ptr(), out.data_ptr(), _LOGIT_DTYPES[logits.dtype], rows, vocab, stride, out_stride, tp, token_bytes,
                             history, token_stride, pl, tl, rp, fp, pp, bp, bias_stride, ip, vp, pairs, mp, mask_stride)
        _call("w4a16_process_logits", dev, d)
    return out
