"""process_logits against float64 on the host, row by row: vocabularies around slice edges, types,
histories of no token to many, every part alone and all together, fully masked rows, infinities and
NaN, strides, in place, graphs."""
import pytest
import torch

import w4a16 as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _reference(logits, tokens=None, prompt_lens=None, total_lens=None, repetition=None, frequency=None, presence=None,
               bias=None, bias_ids=None, bias_values=None, mask=None):
    """(result, sum of the sizes of everything added) in float64."""
    x = logits.double().clone()
    rows, vocab = x.shape
    size = torch.zeros_like(x)
    for b in range(rows):
        if tokens is not None:
            h = tokens.shape[1]
            n = min(max(int(total_lens[b]), 0), h) if total_lens is not None else h
            m = min(max(int(prompt_lens[b]), 0), n) if prompt_lens is not None else 0
            all_ids = tokens[b, :n].long()
            seen = torch.unique(all_ids[(all_ids >= 0) & (all_ids < vocab)])
            if repetition is not None:
                r = repetition[b].double()
                x[b, seen] = torch.where(x[b, seen] > 0, x[b, seen] / r, x[b, seen] * r)
            made = tokens[b, m:n].long()
            ids, times = torch.unique(made[(made >= 0) & (made < vocab)], return_counts=True)
            take = torch.zeros(ids.shape, dtype=torch.float64, device=DEV)
            if frequency is not None:
                take = take + frequency[b].double() * times
                size[b, ids] += (frequency[b].double() * times).abs()
            if presence is not None:
                take = take + presence[b].double()
                size[b, ids] += presence[b].double().abs()
            x[b, ids] -= take
        if bias_ids is not None:
            for i, value in zip(bias_ids[b].tolist(), bias_values[b].double()):
                if 0 <= i < vocab:
                    x[b, i] += value
                    size[b, i] += value.abs()
    if bias is not None:
        x = x + bias.double()
        size = size + bias.double().abs()
    if mask is not None:
        at = torch.arange(vocab, device=DEV)
        words = mask if mask.dim() == 2 else mask[None].expand(rows, -1)
        x = x.masked_fill((words[:, at // 32].long() >> (at % 32)) % 2 == 0, float("-inf"))
    return x, size + logits.double().abs()


def _check(out, logits, extra=8, **kw):
    """At most `extra` roundings to fp32 (half a step each) of values no larger than twice the sizes that
    are added (a repetition factor here is below 2), then half a step of the type."""
    ref, size = _reference(logits, **kw)
    u = HALF[logits.dtype]
    assert torch.equal(torch.isnan(out), torch.isnan(ref))
    fine = torch.isfinite(ref) & (ref.abs() <= torch.finfo(logits.dtype).max)
    assert torch.equal(out.double()[~fine & ~torch.isnan(ref)] * 0.5, torch.where(
        ref[~fine & ~torch.isnan(ref)] > 0, float("inf"), float("-inf")).double())
    size = torch.where(torch.isfinite(size), size, 0)
    tol = u * ref.abs() + extra * 2.0 ** -24 * 2 * size + 2.0 ** -25 * (logits.dtype == torch.float16)
    assert ((out.double() - ref).abs()[fine] <= tol[fine]).all()


def _inputs(rows, vocab, history, dtype, seed=0, pairs=20, tok=torch.int32):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def rand(*shape):
        return torch.rand(shape, device=DEV, generator=g)

    logits = (torch.randn(rows, vocab, device=DEV, generator=g) * 5).to(dtype)
    total = (rand(rows) * (history + 1)).int()
    return logits, dict(
        tokens=(rand(rows, history).pow(2) * (vocab + 3) - 1).to(tok), total_lens=total, prompt_lens=total // 2,
        repetition=rand(rows) + 0.7, frequency=rand(rows) - 0.2, presence=rand(rows) - 0.5, bias=rand(vocab) - 0.5,
        bias_ids=(rand(rows, pairs) * (vocab + 4) - 2).int(), bias_values=rand(rows, pairs) * 8 - 4,
        mask=torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), device=DEV, generator=g).int())


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 8191, 8192, 8193, 50257, 128256, 131073, 262147])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_vocabularies(vocab, dtype):
    logits, kw = _inputs(3, vocab, 700, dtype, seed=vocab)
    kept = logits.clone()
    out = K.process_logits(logits, **kw)
    assert torch.equal(logits, kept) and out.dtype == dtype
    _check(out, logits, **kw)
    assert K.process_logits(logits, **kw, out=logits) is logits and torch.equal(logits, out)  # in place


@pytest.mark.parametrize("rows,history,tok", [(1, 1, torch.int32), (1, 20000, torch.int64), (130, 60, torch.int64), (7, 5000, torch.int32), (3, 0, torch.int32)])
def test_histories(rows, history, tok):
    logits, kw = _inputs(rows, 5003, history, torch.float32, seed=rows, tok=tok)
    _check(K.process_logits(logits, **kw), logits, **kw)
    del kw["total_lens"], kw["prompt_lens"]  # the whole history, all of it generated
    _check(K.process_logits(logits, **kw), logits, **kw)


@pytest.mark.parametrize("parts", [(), ("repetition",), ("frequency",), ("presence",), ("bias",), ("bias_ids", "bias_values"), ("mask",),
                                   ("repetition", "mask"), ("frequency", "bias_ids", "bias_values")])
def test_each_part_alone(parts):
    logits, kw = _inputs(4, 3001, 300, torch.float32)
    kw = {n: t for n, t in kw.items() if n in parts or (n in ("tokens", "total_lens", "prompt_lens") and {"repetition", "frequency", "presence"} & set(parts))}
    out = K.process_logits(logits, **kw)
    _check(out, logits, **kw)
    if not parts:
        assert torch.equal(out, logits)


def test_lengths_are_clamped_and_tokens_outside_skipped():
    logits, kw = _inputs(5, 64, 40, torch.float32)
    kw["total_lens"] = torch.tensor([-3, 0, 41, 2 ** 31 - 1, 40], dtype=torch.int32, device=DEV)
    kw["prompt_lens"] = torch.tensor([-1, 5, -2 ** 31, 20, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    kw["tokens"] = torch.tensor([-1, 64, -2 ** 31, 2 ** 31 - 1, 5, 5, 5, 63], dtype=torch.int32, device=DEV).repeat(5, 5)
    _check(K.process_logits(logits, **kw), logits, **kw)
    kw["tokens"] = kw["tokens"].long() + 2 ** 32  # would be inside after a cut to 32 bits
    out = K.process_logits(logits, **kw)
    _check(out, logits, **kw)


def test_infinities_nan_and_masked_rows():
    logits, kw = _inputs(4, 1000, 50, torch.float32)
    kw["mask"][1] = 0        # a grammar that leaves nothing
    kw["mask"][2] = -1       # one that allows all
    logits[0, ::7], logits[2, ::5], logits[2, 1::5], logits[3, ::3] = float("nan"), float("-inf"), float("inf"), torch.finfo(torch.float32).min
    out = K.process_logits(logits, **kw)
    assert (out[1] == float("-inf")).all()
    _check(out, logits, **kw)


def test_strides_and_single_rows():
    big, kw = _inputs(6, 4099, 90, torch.float16)
    logits = big[::2, 1:4097]  # rows apart, odd starts
    kw = {n: (t[:3] if n != "bias" else t[:4096]) for n, t in kw.items()}
    kw["mask"] = kw["mask"][:, :128]
    room = torch.zeros(3, 5000, device=DEV).half()
    out = K.process_logits(logits, **kw, out=room[:, 3:4099])
    _check(out, logits, **kw)
    assert not room[:, :3].any() and not room[:, 4099:].any()
    kw["bias"] = torch.randn(3, 4096, device=DEV)
    kw["mask"] = kw["mask"][0].contiguous()  # one mask for all rows
    _check(K.process_logits(logits, **kw), logits, **kw)
    one = K.process_logits(big[0], bias=torch.ones(4099, device=DEV))
    assert one.shape == (4099,) and torch.equal(one, (big[0].float() + 1).half())


@pytest.mark.parametrize("rows,pairs", [(2, 255), (2, 256), (2, 513), (80, 257), (80, 1500), (2, 5000)])
def test_many_pairs(rows, pairs):
    # more than one round of pairs for a slice of the vocabulary (by 80 rows: of the larger slices); ids
    # named again in the same round and in later ones, one of them by a third of the pairs
    logits, kw = _inputs(rows, 16001, 200, torch.float32, pairs=pairs)
    n = pairs // 3
    kw["bias_ids"][:, n:2 * n] = kw["bias_ids"][:, :n].flip(1)
    kw["bias_ids"][:, 2 * n::2] = 77
    out = K.process_logits(logits, **kw)
    some = [0, rows - 1]
    part = {name: (t if name == "bias" else t[some]) for name, t in kw.items()}
    # a rounding for each value of an id
    _check(out[some], logits[some], extra=8 + max(int(torch.bincount(r[r >= 0]).max()) for r in part["bias_ids"]), **part)
    assert torch.equal(K.process_logits(logits, **kw), out)
    assert torch.equal(K.process_logits(logits, **kw, out=logits), out)


def test_same_bits_every_time_and_in_a_graph():
    logits, kw = _inputs(9, 60001, 3000, torch.float32, pairs=300)
    kw["bias_ids"][:, 100:200] = kw["bias_ids"][:, :100]  # every id twice
    want = K.process_logits(logits, **kw)
    _check(want, logits, extra=24, **kw)
    g, out = torch.cuda.CUDAGraph(), torch.empty_like(logits)
    with torch.cuda.graph(g):
        K.process_logits(logits, **kw, out=out)
    for _ in range(3):
        out.zero_()
        g.replay()
        assert torch.equal(out, want) and torch.equal(K.process_logits(logits, **kw), want)
    kw["total_lens"].zero_()
    g.replay()
    _check(out, logits, extra=24, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(1, 5003), (130, 10007)])
def test_repetition_divides(dtype, rows, vocab):
    """The nearest quotient, but where it lies within 2^-22 of a step of the middle of two neighbours (1 / repetition
    is known to 2^-47): there the other neighbour, which for 16-bit logits rounds to one step of the type at most."""
    g = torch.Generator(device=DEV).manual_seed(vocab)
    logits = (torch.randn(rows, vocab, device=DEV, generator=g) * 5).to(dtype)
    logits[0, :4] = torch.tensor([0.0, -0.0, float("inf"), float("-inf")])
    tokens = torch.arange(vocab, device=DEV, dtype=torch.int32).repeat(rows, 1)
    for scale in (1.0, 2.0 ** -126, 2.0 ** 99):  # the ends of the range
        r = (torch.rand(rows, device=DEV, generator=g) + (0.7 if scale == 1 else 1.0)) * scale
        r[rows // 2] = 1.1 * scale
        out = K.process_logits(logits, tokens=tokens, repetition=r)
        x = logits.float()
        want = torch.where(x > 0, x / r[:, None], x * r[:, None]).to(dtype)
        other = out != want
        assert other.float().mean() <= 4 * 2.0 ** -22 + 1 / other.numel()
        u = 2 * HALF[dtype]
        assert ((out.double() - want.double())[other].abs() <= u * want.double()[other].abs()).all()


def test_refusals_on_the_host():
    logits, kw = _inputs(3, 100, 10, torch.float32)
    t = kw["tokens"]
    bad = [dict(logits=logits.cpu()), dict(logits=logits.double()), dict(logits=logits.t()), dict(logits=logits[None]),
           dict(tokens=t.float()), dict(tokens=t[:2]), dict(tokens=t[0]), dict(tokens=None), dict(repetition=1.2), dict(repetition=kw["repetition"].double()),
           dict(frequency=kw["frequency"][:2]), dict(total_lens=kw["total_lens"].long()), dict(bias=kw["bias"][:99]), dict(bias=kw["bias"].half()),
           dict(bias_ids=None), dict(bias_values=kw["bias_values"][:, :3]), dict(bias_ids=kw["bias_ids"].long()), dict(mask=kw["mask"][:, :3]),
           dict(mask=kw["mask"].bool()), dict(out=logits.half()), dict(out=torch.empty(3, 99, device=DEV)), dict(out=torch.empty(1, 100, device=DEV).expand(3, 100))]
    for change in bad:
        args = dict(kw, logits=logits) | change
        with pytest.raises(RuntimeError):
            K.process_logits(args.pop("logits"), **args)
    flat = torch.zeros(400, device=DEV)
    with pytest.raises(RuntimeError):  # out overlaps logits without being them
        K.process_logits(flat[:300].view(3, 100), out=flat[4:304].view(3, 100))
    assert K.process_logits(logits[:0]).shape == (0, 100) and K.process_logits(logits[:, :0]).shape == (3, 0)
