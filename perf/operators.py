"""The operators of a serving step over a paged key-value cache: their cases, and their plain forms.

Four operators: rotary embedding with the write of new keys and values into cache pages (append), attention of one new token
per row over the pages (attention), the bookkeeping of the pages (fork, compact), and the processing of logits before the next
token is chosen (logits).  `run` computes the plain forms in elementary torch operations; with `own` set it makes the calls a
user of the package makes.
"""
import functools
import math
import os
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
SIZE = {"fp16": 2, "bf16": 2, "fp32": 4}
DEV = "cuda"


@functools.lru_cache(maxsize=1)
def _w4a16():
    path = os.path.join(os.getcwd(), "w4a16-gemv-optimization-ladder_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import w4a16

    return w4a16


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one sequence of the 1B decoder (32 query heads, 8 key-value heads of 64), its cache of 512 nearly full: latency
        dict(name="attention_one", op="attention", rows=1, heads=32, kv_heads=8, head_dim=64, page_size=16, max_len=511,
             ragged=False, padded=False, dtype="fp16"),
        # an ordinary batch: 32 sequences of all lengths up to 4096, heads of 128 as in an 8B model
        dict(name="attention_batch", op="attention", rows=32, heads=32, kv_heads=8, head_dim=128, page_size=16, max_len=4096,
             ragged=True, padded=False, dtype="fp16"),
        # two long documents: few rows, so the length has to be split
        dict(name="attention_long", op="attention", rows=2, heads=32, kv_heads=8, head_dim=128, page_size=64, max_len=120001,
             ragged=True, padded=False, dtype="bf16"),
        # a large batch with padding rows, five query heads for each key-value head
        dict(name="attention_large", op="attention", rows=72, heads=40, kv_heads=8, head_dim=128, page_size=32, max_len=8191,
             ragged=True, padded=True, dtype="fp16"),
        # the new tokens of a decode step of the 1B decoder
        dict(name="append_step", op="append", tokens=64, seqs=64, heads=32, kv_heads=8, head_dim=64, page_size=16,
             first=700, padded=False, dtype="fp16"),
        # the prompts of eleven sequences at once, padded to a whole number of tiles
        dict(name="append_prompt", op="append", tokens=16384, seqs=11, heads=32, kv_heads=8, head_dim=128, page_size=16,
             first=0, padded=True, dtype="bf16"),
        # a beam step over the 1B decoder's layers: every child dropped, every parent forked again
        dict(name="fork_beams", op="fork", layers=16, forks=48, kv_heads=8, head_dim=64, page_size=16, max_len=900,
             dtype="fp16"),
        # a small cache compacted after sequences have left it
        dict(name="compact_small", op="compact", layers=16, pages=301, live=0.5, kv_heads=8, head_dim=64, page_size=16,
             dtype="fp16"),
        # a large one: 32 layers of an 8B model
        dict(name="compact_large", op="compact", layers=32, pages=4000, live=0.7, kv_heads=8, head_dim=128, page_size=16,
             dtype="bf16"),
        # the decoder's own vocabulary, one row with its history: latency
        dict(name="logits_one", op="logits", rows=1, vocab=128256, history=500, penalties=True, dense=False, pairs=0, mask=False,
             dtype="fp32"),
        # a batch under a grammar, with per-row bias pairs and long histories
        dict(name="logits_batch", op="logits", rows=64, vocab=128256, history=4096, penalties=True, dense=False, pairs=64,
             mask=True, dtype="fp32"),
        # an odd vocabulary in half precision with one bias for every token
        dict(name="logits_odd", op="logits", rows=17, vocab=50257, history=1023, penalties=True, dense=True, pairs=0, mask=False,
             dtype="fp16"),
    ]


def _spread(rng, low, high):
    """A whole number, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "fork", "compact", "logits", "logits"])
    dtype = rng.choice(["fp16", "bf16"])
    kv_heads, head_dim, page_size = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 128]), rng.choice([8, 16, 32, 64, 128])
    if op == "attention":
        rows = _spread(rng, 1, 80)
        most = min(120000, 300000 * 8 // (rows * kv_heads))
        return dict(op=op, rows=rows, heads=kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8, 12, 16]), kv_heads=kv_heads,
                    head_dim=head_dim, page_size=page_size, max_len=_spread(rng, 1, most), ragged=rng.random() < 0.7,
                    padded=rows > 4 and rng.random() < 0.3, dtype=dtype)
    if op == "append":
        seqs = _spread(rng, 1, 64)
        return dict(op=op, tokens=seqs * _spread(rng, 1, 16384 // seqs), seqs=seqs, heads=kv_heads * rng.choice([1, 2, 4, 7]),
                    kv_heads=kv_heads, head_dim=head_dim, page_size=page_size, first=rng.randrange(0, 1000),
                    padded=rng.random() < 0.3, dtype=dtype)
    if op == "fork":
        return dict(op=op, layers=rng.choice([2, 16, 24, 32]), forks=_spread(rng, 1, 128), kv_heads=kv_heads, head_dim=head_dim,
                    page_size=rng.choice([8, 16, 32]), max_len=_spread(rng, 17, 1500), dtype=dtype)
    if op == "compact":
        return dict(op=op, layers=rng.choice([2, 16, 24, 32]), pages=_spread(rng, 40, 3000), live=round(rng.uniform(0.2, 0.9), 2),
                    kv_heads=kv_heads, head_dim=head_dim, page_size=rng.choice([8, 16]), dtype=dtype)
    penalties = rng.random() < 0.8
    return dict(op=op, rows=_spread(rng, 1, 64), vocab=_spread(rng, 1000, 200000), history=_spread(rng, 1, 8000) if penalties else 0,
                penalties=penalties, dense=rng.random() < 0.4, pairs=rng.choice([0, 0, 5, 100]), mask=rng.random() < 0.6,
                dtype=rng.choice(["fp32", "fp32", "fp16", "bf16"]))


# ------------------------------------------------------------------------------------------------ inputs

def _lengths(n, top, ragged=True):
    """Lengths of n rows up to `top`: their sum does not depend on the seed, which only shuffles them."""
    return [-(-top * (i + 1) // n) if ragged else top for i in range(n)]


def _attention_lengths(c):
    dead = c["rows"] // 8 if c["padded"] else 0
    return _lengths(c["rows"] - dead, c["max_len"], c["ragged"]) + [0] * dead


def _fork_lengths(c):
    return _lengths(c["forks"], c["max_len"])


def _live(c):
    """(live pages, live pages that lie above the others' number and have to move)."""
    n = max(1, int(c["pages"] * c["live"]))
    return n, min(int(n * (1 - c["live"])), n, c["pages"] - n)


def _pool(gen, shape, dtype):
    return torch.randn(shape, dtype=dtype, device=DEV, generator=gen)


def _tables(gen, lens, page_size, pages):
    """A page table for sequences of these lengths: scattered pages, -1 past each sequence's last."""
    width = max(1, max(-(-n // page_size) for n in lens))
    used = torch.tensor([-(-n // page_size) for n in lens], device=DEV)
    at = torch.arange(width, device=DEV)[None, :]
    order = torch.randperm(pages, device=DEV, generator=gen)
    start = (torch.cumsum(used, 0) - used)[:, None]
    held = at < used[:, None]
    ids = order[(start + at).clamp(max=pages - 1)]
    return torch.where(held, ids, -1).to(torch.int32).contiguous()


def _angles(count, head_dim, theta=500000.0):
    inv = theta ** (-torch.arange(0, head_dim, 2, device=DEV, dtype=torch.float64) / head_dim)
    a = torch.arange(count, device=DEV, dtype=torch.float64)[:, None] * inv[None, :]
    a = torch.cat([a, a], dim=1)
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    c, dt = case, DTYPES[case["dtype"]]
    s = dict(case=case)
    if c["op"] == "attention":
        lens = _attention_lengths(c)
        lens = [lens[i] for i in torch.randperm(len(lens), generator=torch.Generator().manual_seed(seed)).tolist()]
        pages = sum(-(-n // c["page_size"]) for n in lens) + 3
        shape = (pages, c["kv_heads"], c["page_size"], c["head_dim"])
        s.update(q=_pool(gen, (c["rows"], c["heads"], c["head_dim"]), dt), k=_pool(gen, shape, dt), v=_pool(gen, shape, dt),
                 tables=_tables(gen, lens, c["page_size"], pages), lengths=torch.tensor(lens, dtype=torch.int32, device=DEV))
    elif c["op"] == "append":
        each = [len(range(i, c["tokens"], c["seqs"])) for i in range(c["seqs"])]
        lens = [c["first"] + n for n in each]
        pages = sum(-(-n // c["page_size"]) for n in lens) + 3
        shape = (pages, c["kv_heads"], c["page_size"], c["head_dim"])
        at = torch.cat([torch.arange(n) for n in each]) + c["first"]
        seqs = torch.cat([torch.full((n,), i) for i, n in enumerate(each)])
        dead = min(c["tokens"] // 9, 37) if c["padded"] else 0
        if dead:
            at[-dead:] = -1
        wide = _pool(gen, (c["tokens"], (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]), dt)  # one projection's output
        q, k, v = wide.split([n * c["head_dim"] for n in (c["heads"], c["kv_heads"], c["kv_heads"])], dim=1)
        cos, sin = _angles(max(lens), c["head_dim"])
        s.update(q=q.unflatten(1, (c["heads"], c["head_dim"])), kn=k.unflatten(1, (c["kv_heads"], c["head_dim"])),
                 vn=v.unflatten(1, (c["kv_heads"], c["head_dim"])), k=_pool(gen, shape, dt), v=_pool(gen, shape, dt), cos=cos, sin=sin,
                 tables=_tables(gen, lens, c["page_size"], pages), positions=at.to(DEV, torch.int32), seqs=seqs.to(DEV, torch.int32))
    elif c["op"] == "fork":
        n, lens = c["forks"], _fork_lengths(c)
        lens = [lens[i] for i in torch.randperm(n, generator=torch.Generator().manual_seed(seed)).tolist()]
        held = sum(-(-x // c["page_size"]) for x in lens)
        pages = held + 2 * n + 3
        shape = (c["layers"], pages, c["kv_heads"], c["page_size"], c["head_dim"])
        parents = _tables(gen, lens, c["page_size"], pages)
        tables = torch.cat([parents, torch.full_like(parents, -1)])
        refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
        refs[parents[parents >= 0].long()] = 1
        ids = torch.arange(2 * n, dtype=torch.int32, device=DEV)
        s.update(k=_pool(gen, shape, dt), v=_pool(gen, shape, dt), tables=tables, refs=refs, src=ids[:n].contiguous(), dst=ids[n:].contiguous(),
                 lengths=torch.tensor(lens + [0] * n, dtype=torch.int32, device=DEV))
    elif c["op"] == "compact":
        n, move = _live(c)
        shape = (c["layers"], c["pages"], c["kv_heads"], c["page_size"], c["head_dim"])
        low = torch.randperm(n, device=DEV, generator=gen)[: n - move]
        high = torch.randperm(c["pages"] - n, device=DEV, generator=gen)[:move] + n
        ids = torch.cat([low, high])[torch.randperm(n, device=DEV, generator=gen)]
        # each live page in one sequence's table, the first half of them shared with a second sequence
        width = 32
        both = torch.cat([ids, ids[: n // 2]])
        rows = -(-both.numel() // width)
        tables = torch.full((rows * width,), -1, dtype=torch.int32, device=DEV)
        tables[: both.numel()] = both.to(torch.int32)
        refs = torch.zeros(c["pages"], dtype=torch.int32, device=DEV)
        refs.index_add_(0, both, torch.ones_like(both, dtype=torch.int32))
        s.update(k=_pool(gen, shape, dt), v=_pool(gen, shape, dt), tables=tables.view(rows, width), refs=refs)
    else:
        b, vocab, h = c["rows"], c["vocab"], c["history"]
        s.update(logits=(torch.randn((b, vocab), device=DEV, generator=gen) * 4).to(dt), tokens=None, bias=None, ids=None, values=None, mask=None)
        if c["penalties"]:
            # few ids make most of a history, as in text
            tokens = (torch.rand((b, h), device=DEV, generator=gen).pow(3) * vocab).to(torch.int32).clamp(max=vocab - 1)
            total = torch.tensor(_lengths(b, h), dtype=torch.int32, device=DEV)
            s.update(tokens=tokens, total=total, prompt=total // 3, repetition=torch.rand(b, device=DEV, generator=gen) + 0.8,
                     frequency=torch.rand(b, device=DEV, generator=gen), presence=torch.rand(b, device=DEV, generator=gen) - 0.3)
        if c["dense"]:
            s["bias"] = torch.randn(vocab, device=DEV, generator=gen)
        if c["pairs"]:
            s["ids"] = torch.randint(-1, vocab, (b, c["pairs"]), device=DEV, generator=gen, dtype=torch.int32)
            s["values"] = torch.randn((b, c["pairs"]), device=DEV, generator=gen) * 10
        if c["mask"]:
            words = torch.randint(-(2 ** 31), 2 ** 31, (b, -(-vocab // 32)), device=DEV, generator=gen, dtype=torch.int64).to(torch.int32)
            words[b // 2] = 0  # a row whose grammar leaves nothing
            s["mask"] = words
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(s):
    if own:
        return _own(s)
    return {"attention": _attention, "append": _append, "fork": _fork, "compact": _compact, "logits": _logits}[s["case"]["op"]](s)


def _own(s):
    K, c = _w4a16(), s["case"]
    if c["op"] == "attention":
        return K.paged_attention(s["q"], s["k"], s["v"], s["tables"], s["lengths"])
    if c["op"] == "append":
        q = K.paged_append(s["q"], s["kn"], s["vn"], s["positions"], s["tables"], s["k"], s["v"], cos=s["cos"], sin=s["sin"], seqs=s["seqs"])
        return q, s["k"], s["v"]
    if c["op"] == "fork":
        K.free_sequences(s["tables"], s["lengths"], s["refs"], s["dst"])
        ok = K.fork_sequences(s["k"], s["v"], s["tables"], s["lengths"], s["refs"], s["src"], s["dst"])
        return ok, s["tables"], s["lengths"], s["refs"], s["k"], s["v"]
    if c["op"] == "compact":
        tables, refs, moved = K.compact_pages(s["k"], s["v"], s["tables"], s["refs"], inplace=False)
        return tables, refs, moved, s["k"], s["v"]
    if s["tokens"] is None:
        return K.process_logits(s["logits"], bias=s["bias"], bias_ids=s["ids"], bias_values=s["values"], mask=s["mask"])
    return K.process_logits(s["logits"], tokens=s["tokens"], prompt_lens=s["prompt"], total_lens=s["total"], repetition=s["repetition"],
                            frequency=s["frequency"], presence=s["presence"], bias=s["bias"], bias_ids=s["ids"], bias_values=s["values"],
                            mask=s["mask"])


def _attention(s):
    c = s["case"]
    rows, g, d = c["rows"], c["kv_heads"], c["head_dim"]
    pages = s["tables"].long().clamp(min=0)
    length = pages.shape[1] * c["page_size"]
    k, v = (x[pages].permute(0, 2, 1, 3, 4).reshape(rows, g, length, d).float() for x in (s["k"], s["v"]))
    score = s["q"].float().view(rows, g, -1, d) @ k.transpose(2, 3) * (1 / math.sqrt(d))
    past = torch.arange(length, device=DEV)[None, :] >= s["lengths"][:, None]
    score = score.masked_fill(past[:, None, None, :], -math.inf)
    top = score.amax(3, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = torch.exp(score - top)
    out = (p @ v) / p.sum(3, keepdim=True).clamp(min=1e-30)  # a row of no positions: zeros
    return out.view(rows, c["heads"], d).to(s["q"].dtype)


def _rotate(x, cos, sin):
    half = x.shape[-1] // 2
    x = x.float()
    return x * cos + torch.cat([-x[..., half:], x[..., :half]], dim=-1) * sin


def _append(s):
    c, dt = s["case"], s["q"].dtype
    at = s["positions"].long()
    cos, sin = (t[at.clamp(min=0)][:, None, :] for t in (s["cos"], s["sin"]))
    q = (_rotate(s["q"], cos, sin) * (at >= 0)[:, None, None]).to(dt)
    k, v, seqs = _rotate(s["kn"], cos, sin).to(dt), s["vn"], s["seqs"].long()
    if c["padded"]:
        kept = (at >= 0).nonzero()[:, 0]
        at, seqs, k, v = at[kept], seqs[kept], k[kept], v[kept]
    page, row = s["tables"][seqs, at // c["page_size"]].long(), at % c["page_size"]
    s["k"][page, :, row] = k
    s["v"][page, :, row] = v
    return q, s["k"], s["v"]


def _fork(s):
    c, tables, refs = s["case"], s["tables"], s["refs"]
    src, dst = s["src"].long(), s["dst"].long()
    # free the children
    old = tables[dst]
    refs.index_add_(0, old.clamp(min=0).view(-1).long(), -(old >= 0).view(-1).to(torch.int32))
    tables[dst] = -1
    s["lengths"][dst] = 0
    # fork the parents: whole pages are shared, a partial one is copied to the lowest free page
    length = s["lengths"][src]
    full, part = (length // c["page_size"])[:, None], length % c["page_size"] > 0
    free = torch.argsort((refs > 0).to(torch.int32), stable=True)
    rank = torch.cumsum(part, 0)
    ok = ~part | (rank <= (refs == 0).sum())
    new = free[(rank - 1).clamp(0, refs.numel() - 1)].to(torch.int32)
    rows, at = tables[src], torch.arange(tables.shape[1], device=DEV)[None, :]
    last = rows.gather(1, full.clamp(max=tables.shape[1] - 1).long())[:, 0]
    copied = part & ok
    shared = (at < full) & ok[:, None]
    tables[dst] = torch.where(shared, rows, torch.where((at == full) & copied[:, None], new[:, None], -1))
    s["lengths"][dst] = torch.where(ok, length, 0)
    refs.index_add_(0, torch.where(shared, rows, 0).view(-1).long(), shared.view(-1).to(torch.int32))
    refs.index_add_(0, torch.where(copied, new, 0).long(), copied.to(torch.int32))
    frm, to = last[copied].long(), new[copied].long()
    s["k"][:, to] = s["k"][:, frm]
    s["v"][:, to] = s["v"][:, frm]
    return ok.to(torch.int32), tables, s["lengths"], refs, s["k"], s["v"]


def _compact(s):
    refs, tables = s["refs"], s["tables"]
    live = refs > 0
    n = live.sum()
    ids = torch.arange(refs.numel(), device=DEV)
    frm, to = (live & (ids >= n)).nonzero()[:, 0], (~live & (ids < n)).nonzero()[:, 0]
    s["k"][:, to] = s["k"][:, frm]
    s["v"][:, to] = s["v"][:, frm]
    where = ids.to(torch.int32)
    where[frm] = to.to(torch.int32)
    moved = torch.where(tables >= 0, where[tables.clamp(min=0).long()], tables)
    counts = refs.clone()
    counts[to] = refs[frm]
    counts[frm] = 0
    return moved, counts, torch.full((1,), frm.numel(), dtype=torch.int32, device=DEV), s["k"], s["v"]


def _logits(s):
    c, x = s["case"], s["logits"].float()
    b, vocab = x.shape
    if s["tokens"] is not None:
        at = torch.arange(c["history"], device=DEV)[None, :]
        said, mine = at < s["total"][:, None], (at < s["total"][:, None]) & (at >= s["prompt"][:, None])
        ids = s["tokens"].long()
        seen = torch.zeros((b, vocab), device=DEV).scatter_add_(1, ids, said.float())
        count = torch.zeros((b, vocab), device=DEV).scatter_add_(1, ids, mine.float())
        r = s["repetition"][:, None]
        x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None] * count
        x = x - s["presence"][:, None] * (count > 0)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["ids"] is not None:
        x = x.scatter_add(1, s["ids"].long().clamp(min=0), s["values"] * (s["ids"] >= 0))
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device=DEV, dtype=torch.int32)) & 1
        x = x.masked_fill(bits.view(b, -1)[:, :vocab] == 0, -math.inf)
    return x.to(s["logits"].dtype)


# ------------------------------------------------------------------------------------------------ what a pass costs at least

def work(case):
    c, size = case, SIZE[case["dtype"]]
    if c["op"] == "attention":
        total = sum(_attention_lengths(c))
        return {"bytes": 2 * total * c["kv_heads"] * c["head_dim"] * size + 2 * c["rows"] * c["heads"] * c["head_dim"] * size,
                "flops": 4 * total * c["heads"] * c["head_dim"]}
    if c["op"] == "append":
        wide = (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"]
        angles = -(-c["tokens"] // c["seqs"]) * c["head_dim"] * 8
        return {"bytes": 2 * c["tokens"] * wide * size + angles, "flops": 3 * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["head_dim"]}
    if c["op"] in ("fork", "compact"):
        moves = sum(n % c["page_size"] > 0 for n in _fork_lengths(c)) if c["op"] == "fork" else _live(c)[1]
        page = 2 * c["layers"] * c["kv_heads"] * c["page_size"] * c["head_dim"] * size
        ints = 4 * c["pages"] * 4 if c["op"] == "compact" else 4 * c["forks"] * -(-c["max_len"] // c["page_size"])
        return {"bytes": 2 * moves * page + ints, "flops": 0}
    total = sum(_lengths(c["rows"], c["history"])) if c["penalties"] else 0
    each = c["rows"] * c["vocab"]
    return {"bytes": 2 * each * size + 4 * total + (each // 8 if c["mask"] else 0) + (4 * c["vocab"] if c["dense"] else 0) + 8 * c["rows"] * c["pairs"],
            "flops": 4 * each}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "attention":
        out = torch.zeros((c["rows"], c["heads"], c["head_dim"]), dtype=torch.float64, device=DEV)
        for t, n in enumerate(s["lengths"].tolist()):
            if n > 0:
                slot = torch.arange(n, device=DEV)
                page, row = s["tables"][t].long()[slot // c["page_size"]], slot % c["page_size"]
                k, v = (x[page, :, row].double().transpose(0, 1) for x in (s["k"], s["v"]))
                q = s["q"][t].double().unflatten(0, (c["kv_heads"], -1))
                p = torch.softmax(torch.einsum("ghd,gnd->ghn", q, k) / c["head_dim"] ** 0.5, dim=2)
                out[t] = torch.einsum("ghn,gnd->ghd", p, v).flatten(0, 1)
        return out
    if c["op"] == "append":
        q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
        at, h = s["positions"].long(), c["head_dim"] // 2
        real = (at >= 0).nonzero()[:, 0]

        def turned(x):
            a, b = x[real].double().split(h, dim=2)
            cos, sin = (t.double()[at[real]][:, None, :] for t in (s["cos"], s["sin"]))
            return torch.cat([a * cos[..., :h] - b * sin[..., :h], b * cos[..., h:] + a * sin[..., h:]], dim=2)

        q = torch.zeros_like(q).index_copy(0, real, turned(s["q"]))
        where = s["tables"].long()[s["seqs"].long()[real], at[real] // c["page_size"]] * c["page_size"] + at[real] % c["page_size"]
        flat = [x.transpose(1, 2).reshape(-1, c["kv_heads"], c["head_dim"]).index_copy(0, where, y)
                for x, y in ((k, turned(s["kn"])), (v, s["vn"][real].double()))]
        return (q, *(x.view(-1, c["page_size"], c["kv_heads"], c["head_dim"]).transpose(1, 2) for x in flat))
    if c["op"] == "fork":
        # one request after the other, on the host
        tables, lengths, refs = (s[n].tolist() for n in ("tables", "lengths", "refs"))
        free, k, v, ok = [p for p, n in enumerate(refs) if n == 0], s["k"], s["v"], []
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            whole = lengths[a] // c["page_size"]
            tables[b][:whole] = tables[a][:whole]
            for p in tables[a][:whole]:
                refs[p] += 1
            if lengths[a] % c["page_size"]:
                new = free.pop(0)
                tables[b][whole], refs[new] = new, 1
                k[:, new], v[:, new] = k[:, tables[a][whole]], v[:, tables[a][whole]]
            lengths[b] = lengths[a]
            ok.append(1)
        ints = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (ok, tables, lengths, refs)]
        return (*ints, k, v)
    if c["op"] == "compact":
        tables, refs = s["tables"].tolist(), s["refs"].tolist()
        n = sum(x > 0 for x in refs)
        moves = dict(zip([p for p in range(n, len(refs)) if refs[p] > 0], [p for p in range(n) if refs[p] == 0]))
        for a, b in moves.items():
            s["k"][:, b], s["v"][:, b] = s["k"][:, a], s["v"][:, a]
            refs[a], refs[b] = 0, refs[a]
        tables = [[moves.get(p, p) for p in row] for row in tables]
        ints = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (tables, refs, [len(moves)])]
        return (*ints, s["k"], s["v"])
    x = s["logits"].double()
    for b in range(c["rows"]):
        if s["tokens"] is not None:
            n, m = int(s["total"][b]), int(s["prompt"][b])
            r, f, p = (float(s[name][b]) for name in ("repetition", "frequency", "presence"))
            ids, _ = torch.unique(s["tokens"][b, :n].long(), return_counts=True)
            old = x[b, ids]
            x[b, ids] = torch.where(old > 0, old / r, old * r)
            ids, times = torch.unique(s["tokens"][b, m:n].long(), return_counts=True)
            x[b, ids] -= f * times.double() + p
        if s["ids"] is not None:
            real = s["ids"][b] >= 0
            x[b].index_add_(0, s["ids"][b][real].long(), s["values"][b][real].double())
    if s["bias"] is not None:
        x += s["bias"].double()
    if s["mask"] is not None:
        at = torch.arange(c["vocab"], device=DEV)
        x[(s["mask"][:, at // 32].long() >> (at % 32)) % 2 == 0] = -math.inf
    return x
