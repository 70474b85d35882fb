"""extend, fork, free, compact and copy of a paged cache's pages against a model on the host that
serves one request after the other, and the cache's contents through a random life of sequences."""
import random

import pytest
import torch

import w4a16 as K

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


class Model:
    """The bookkeeping one request at a time; contents[p] stands for what page p holds."""

    def __init__(self, sequences, width, pages, page_size):
        self.ps, self.width = page_size, width
        self.tables = [[-1] * width for _ in range(sequences)]
        self.lengths, self.refs = [0] * sequences, [0] * pages
        self.contents = list(range(pages))

    def _serve(self, requests):
        """requests: (key, valid, pages needed, what to do with the pages).  Returns ok."""
        free = [p for p, n in enumerate(self.refs) if n == 0]
        named, ok, used = set(), [], 0
        todo = []
        for key, valid, need, act in requests:
            good = valid and key not in named
            named.add(key)
            used += need if good else 0
            good = good and (need == 0 or used <= len(free))
            ok.append(int(good))
            if good:
                todo.append((act, free[used - need:used]))
        for act, pages in todo:
            act(pages)
        return ok

    def extend(self, seqs, counts):
        lengths = list(self.lengths)
        out = []
        for s, c in zip(seqs, counts):
            valid = 0 <= s < len(lengths) and c >= 0 and lengths[s] + c <= self.width * self.ps
            need = -(-(lengths[s] + c) // self.ps) - -(-lengths[s] // self.ps) if valid else 0

            def act(pages, s=s, c=c):
                at = -(-lengths[s] // self.ps)
                for i, p in enumerate(pages):
                    self.tables[s][at + i], self.refs[p] = p, 1
                self.lengths[s] += c

            out.append((s, valid, need, act))
        return self._serve(out)

    def fork(self, src, dst):
        lengths, tables = list(self.lengths), [list(r) for r in self.tables]
        out = []
        for a, b in zip(src, dst):
            valid = 0 <= a < len(lengths) and 0 <= b < len(lengths) and a != b and lengths[b] == 0
            n = lengths[a] if valid else 0

            def act(pages, a=a, b=b, n=n):
                for i in range(n // self.ps):
                    self.tables[b][i] = tables[a][i]
                    self.refs[tables[a][i]] += 1
                for p in pages:
                    self.tables[b][n // self.ps], self.refs[p] = p, 1
                    self.contents[p] = self.contents[tables[a][n // self.ps]]
                self.lengths[b] = n

            out.append((b, valid, int(n % self.ps > 0), act))
        return self._serve(out)

    def free(self, seqs):
        ok, named = [], set()
        for s in seqs:
            good = 0 <= s < len(self.lengths) and s not in named
            named.add(s)
            ok.append(int(good))
            if good:
                for i, p in enumerate(self.tables[s]):
                    if p >= 0:
                        self.refs[p] -= 1
                    self.tables[s][i] = -1
                self.lengths[s] = 0
        return ok

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        frm, to = [p for p in range(n, len(self.refs)) if self.refs[p] > 0], [p for p in range(n) if self.refs[p] == 0]
        where = dict(zip(frm, to))
        for a, b in where.items():
            self.refs[b], self.refs[a], self.contents[b] = self.refs[a], 0, self.contents[a]
        self.tables = [[where.get(p, p) for p in r] for r in self.tables]
        return len(where)

    def check(self, cache):
        assert cache.tables.tolist() == self.tables
        assert cache.lengths.tolist() == self.lengths
        assert cache.refs.tolist() == self.refs
        for x, sign in ((cache.k, 1), (cache.v, -1)):  # every value of a page in every layer
            want = torch.tensor(self.contents, device=DEV).to(x.dtype)[None, :, None, None, None] * sign
            want = want + torch.arange(x.shape[0], device=DEV).to(x.dtype)[:, None, None, None, None] * 0.25
            assert torch.equal(x, want.expand_as(x))


def _pair(sequences, width, pages, page_size, layers=3, kv_heads=2, dtype=torch.float16):
    cache = K.PagedKVCache(layers, pages, sequences, width * page_size, kv_heads=kv_heads, head_dim=64, page_size=page_size, dtype=dtype)
    ids = torch.arange(pages, device=DEV)[None, :, None, None, None] + torch.zeros_like(cache.k, dtype=torch.float32)
    layer = torch.arange(layers, device=DEV)[:, None, None, None, None] * 0.25
    cache.k.copy_(ids + layer)
    cache.v.copy_(-ids + layer)
    return cache, Model(sequences, width, pages, page_size)


@pytest.mark.parametrize("sequences,width,pages,page_size,seed", [(4, 3, 7, 1, 0), (12, 9, 40, 16, 1), (40, 30, 301, 8, 2), (100, 5, 1025, 4, 3)])
def test_random_life(sequences, width, pages, page_size, seed):
    rng = random.Random(seed)
    cache, model = _pair(sequences, width, pages, page_size)
    for step in range(60):
        n = rng.choice([0, 1, 2, 5, sequences])
        index = [rng.randrange(-1, sequences + 1) for _ in range(n)]  # out of range and repeated ones among them
        what = rng.choice(["extend", "extend", "extend", "fork", "fork", "free", "compact"])
        if what == "extend":
            counts = [rng.choice([-1, 0, 1, 2, page_size, rng.randrange(width * page_size + 2)]) for _ in range(n)]
            assert cache.extend(_i32(index), _i32(counts)).tolist() == model.extend(index, counts)
        elif what == "fork":
            dst = [rng.randrange(-1, sequences + 1) for _ in range(n)]
            assert cache.fork(_i32(index), _i32(dst)).tolist() == model.fork(index, dst)
        elif what == "free":
            index = index[: max(1, n // 2)] if n else []
            assert cache.free(_i32(index)).tolist() == model.free(index)
        else:
            assert cache.compact().tolist() == [model.compact()]
        model.check(cache)


@pytest.mark.parametrize("page_size", [2, 16])
def test_fork_of_a_sequence_whose_last_page_is_bad_is_refused(page_size):
    # there is nothing to copy: a child with a free page's old contents would answer in earnest
    cache, model = _pair(8, 4, 30, page_size)
    n = 3 * page_size - 1
    for x in (cache, model):
        x.extend(*((_i32([0, 1, 2]), _i32([n] * 3)) if x is cache else ([0, 1, 2], [n] * 3)))
    for entry in (-1, 30, 2 ** 31 - 1):
        cache.tables[1, 2] = entry
        before = [t.clone() for t in (cache.tables, cache.lengths, cache.refs, cache.k, cache.v)]
        assert cache.fork(_i32([1, 1]), _i32([4, 5])).tolist() == [0, 0]
        assert all(torch.equal(a, b) for a, b in zip(before, (cache.tables, cache.lengths, cache.refs, cache.k, cache.v)))
    assert cache.fork(_i32([1, 0, 1, 2]), _i32([4, 5, 6, 7])).tolist() == [0, 1, 0, 1]  # the others' pages are as if it were not there
    model.fork([0, 2], [5, 7])
    cache.tables[1, 2] = model.tables[1][2]
    model.check(cache)


def test_requests_past_the_free_pages_are_refused_in_order():
    cache, model = _pair(6, 4, 5, 16)
    seqs, counts = [0, 1, 2, 3, 4], [33, 16, 17, 0, 1]  # 3 + 1 pages, then 2 do not fit, 0 needed, 1 would
    assert cache.extend(_i32(seqs), _i32(counts)).tolist() == [1, 1, 0, 1, 0] == model.extend(seqs, counts)
    model.check(cache)
    assert cache.fork(_i32([0, 1, 0]), _i32([2, 3, 5])).tolist() == [1, 1, 0] == model.fork([0, 1, 0], [2, 3, 5])
    model.check(cache)


def test_largest_calls():
    n = 1024
    cache, model = _pair(2 * n, 3, 5000, 2, layers=1, kv_heads=1, dtype=torch.float32)
    counts = [i % 6 for i in range(n)]
    assert cache.extend(_i32(list(range(n))), _i32(counts)).tolist() == model.extend(range(n), counts)
    src, dst = [i // 2 for i in range(n)], list(range(2 * n - 1, n - 1, -1))
    assert cache.fork(_i32(src), _i32(dst)).tolist() == model.fork(src, dst)
    gone = list(range(0, 2 * n, 3)) * 3
    assert cache.free(_i32(gone)).tolist() == model.free(gone)
    assert cache.compact().tolist() == [model.compact()]
    model.check(cache)


def test_fork_of_a_sequence_that_another_request_fills():
    # request 0 fills sequence 1 from 0, request 1 reads 1 as it was before the call: empty
    cache, model = _pair(3, 4, 9, 16)
    cache.extend(_i32([0]), _i32([40]))
    model.extend([0], [40])
    assert cache.fork(_i32([0, 1]), _i32([1, 2])).tolist() == model.fork([0, 1], [1, 2]) == [1, 1]
    model.check(cache)
    assert cache.lengths.tolist() == [40, 40, 0]


def test_compact_beside_its_input_and_larger_pools():
    g = torch.Generator(device=DEV).manual_seed(0)
    pages = 70001
    refs = torch.randint(0, 3, (pages,), device=DEV, generator=g, dtype=torch.int32)
    k = torch.arange(pages, device=DEV).view(pages, 1, 1, 1).expand(pages, 1, 1, 16).contiguous().int()
    v = -k
    tables = torch.randperm(pages, device=DEV, generator=g).to(torch.int32)[None].contiguous()
    kept = tables.clone(), refs.clone()
    t, r, moved = K.compact_pages(k, v, tables, refs, inplace=False)
    assert torch.equal(tables, kept[0]) and torch.equal(refs, kept[1])
    n = int((refs > 0).sum())
    assert bool((r[:n] > 0).all()) and not r[n:].any() and int(moved) == int((refs[n:] > 0).sum())
    live = refs[tables.long()] > 0
    assert torch.equal(k[t[live].long(), 0, 0, 0], tables[live])
    assert torch.equal(v[t[live].long(), 0, 0, 0], -tables[live]) and torch.equal(r[t[live].long()], refs[tables[live].long()])
    t2, r2, moved = K.compact_pages(k, v, t, r)  # nothing left to do
    assert int(moved) == 0 and t2.data_ptr() == t.data_ptr() and torch.equal(r2[:n] > 0, torch.ones(n, dtype=torch.bool, device=DEV))
    empty = torch.zeros_like(refs)
    assert int(K.compact_pages(k, v, tables, empty)[2]) == 0


@pytest.mark.parametrize("shape,dtype", [((3, 9, 2, 16, 64), torch.float16), ((9, 1, 1, 8), torch.float16), ((2, 5, 3, 7, 80), torch.uint8),
                                         ((2, 40, 8, 64, 128), torch.bfloat16)])
def test_copy_pages(shape, dtype):
    k = torch.randint(0, 100, shape, device=DEV).to(dtype)
    v = torch.randint(0, 100, shape, device=DEV).to(dtype)
    pages = shape[-4]
    src, dst = [0, 3, 3, -1, pages, 2, 1], [pages - 1, 4, 2 if pages > 9 else -5, 0, 1, -1, 2 ** 31 - 1]
    want = [x.clone() for x in (k, v)]
    for a, b in zip(src, dst):
        if 0 <= a < pages and 0 <= b < pages:
            for x in want:
                x.movedim(-4, 0)[b] = x.movedim(-4, 0)[a]
    K.copy_pages(k, v, _i32(src), _i32(dst))
    # pages = 5 names page 4 twice as a destination, which the call does not promise anything about
    said = [p for p in range(pages) if dst.count(p) < 2]
    for x, y in zip((k, v), want):
        assert torch.equal(x.movedim(-4, 0)[said], y.movedim(-4, 0)[said])
    K.copy_pages(k, v, _i32([]), _i32([]))


def test_copy_pages_strided():
    big = torch.randn(4, 6, 16, 2, 64, device=DEV).half()
    k, v = big.transpose(2, 3)[::2, 1:], big.transpose(2, 3)[1::2, 1:]  # layers apart, token-major pages
    want = big.clone()
    want[0::2, 5], want[1::2, 5] = want[0::2, 2], want[1::2, 2]
    K.copy_pages(k, v, _i32([1]), _i32([4]))
    assert torch.equal(big, want)


def test_bookkeeping_in_a_graph():
    # extend by one, free and fork captured once and replayed with other indices
    cache, model = _pair(8, 6, 30, 4)
    seqs, ones, src, dst = _i32([0, 1, 2, 3]), _i32([1] * 4), _i32([0, 1]), _i32([4, 5])
    for _ in range(3):
        cache.extend(seqs, ones)
        model.extend([0, 1, 2, 3], [1] * 4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        cache.free(dst)
        cache.extend(seqs, ones)
        ok = cache.fork(src, dst)
    for a, b in (([0, 1], [4, 5]), ([2, 0], [5, 6]), ([3, 3], [4, 7])):
        src.copy_(_i32(a))
        dst.copy_(_i32(b))
        g.replay()
        model.free(b)
        model.extend([0, 1, 2, 3], [1] * 4)
        assert ok.tolist() == model.fork(a, b)
        model.check(cache)


def test_refusals_on_the_host():
    cache, _ = _pair(4, 3, 9, 16)
    s = _i32([0])
    bad = [lambda: cache.extend(s.long(), s), lambda: cache.extend(s, _i32([1, 2])), lambda: cache.extend(s.cpu(), s.cpu()),
           lambda: K.extend_sequences(cache.tables.long(), cache.lengths, cache.refs, s, s, page_size=16),
           lambda: K.extend_sequences(cache.tables, cache.lengths[:2], cache.refs, s, s, page_size=16),
           lambda: K.extend_sequences(cache.tables, cache.lengths, cache.refs, s, s, page_size=12),
           lambda: K.extend_sequences(cache.tables, cache.lengths, cache.refs, s, s, page_size=0),
           lambda: cache.extend(_i32([0] * 1025), _i32([0] * 1025)), lambda: cache.fork(s, _i32([1, 2])),
           lambda: K.fork_sequences(cache.k, cache.v[:2], cache.tables, cache.lengths, cache.refs, s, s),
           lambda: K.fork_sequences(cache.k, cache.v, cache.tables, cache.lengths, cache.refs[:5], s, s),
           lambda: K.copy_pages(cache.k[..., :32], cache.v[..., :32], s, s), lambda: K.copy_pages(cache.k[0, 0], cache.v[0, 0], s, s),
           lambda: K.compact_pages(cache.k, cache.v, cache.tables.t(), cache.refs), lambda: K.compact_pages(cache.k, cache.v, cache.tables, cache.refs[:4])]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        K.PagedKVCache(1, 4, 2, 64, kv_heads=1, head_dim=64, page_size=24)
