"""The serving operators together, on the decoder's own weights: prompts and single tokens of several
sequences through step_paged against the one-sequence step, with sequences forked, freed and the
cache compacted in between, and greedy generation under penalties, biases and a mask."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _decoder(seed=3, **kw):
    from w4a16.decode import LlamaDecodeConfig, W4A16LlamaDecoder

    return W4A16LlamaDecoder(LlamaDecodeConfig(layers=2, vocab=4096, max_len=160), seed=seed, **kw)


def _cache(dec, pages=60, sequences=8, page_size=16):
    import w4a16 as K

    c = dec.cfg
    return K.PagedKVCache(c.layers, pages, sequences, c.max_len, kv_heads=c.kv_heads, head_dim=c.head_dim, page_size=page_size)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _feed(dec, cache, prompts, pad=0):
    """Several sequences' tokens in one step: {sequence: tokens}, appended to what they hold."""
    seqs = list(prompts)
    before = cache.lengths[seqs].tolist()
    assert cache.extend(_i32(seqs), _i32([len(prompts[s]) for s in seqs])).tolist() == [1] * len(seqs)
    rows = [(t, s, n + i) for s, n in zip(seqs, before) for i, t in enumerate(prompts[s])] + [(0, 0, -1)] * pad
    tokens, ids, at = zip(*rows)
    logits = dec.step_paged(torch.tensor(tokens, device=DEV), _i32(ids), _i32(at), cache)
    last, out = -1, {}
    for s in seqs:
        last += len(prompts[s])
        out[s] = logits[last]
    return out


def _one_by_one(dec, tokens):
    """The same sequence through the one-sequence step over its own cache."""
    for i, t in enumerate(tokens):
        out = dec.step(token=t, pos=i)
    return out.clone()


def _near(a, b):
    assert (a - b).abs().max().item() <= 2e-2 * b.abs().max().item()


@pytest.mark.parametrize("kw", [dict(fused=True), dict(fused=False), dict(dense=True)], ids=["fused", "unfused", "dense"])
def test_several_sequences_match_one_at_a_time(kw):
    dec = _decoder(**kw)
    cache = _cache(dec)
    g = torch.Generator().manual_seed(0)
    texts = {s: torch.randint(0, 4096, (n,), generator=g).tolist() for s, n in ((0, 37), (3, 1), (5, 90))}
    out = _feed(dec, cache, texts, pad=3)           # 128 prompt tokens: the GEMM
    for s in texts:
        _near(out[s], _one_by_one(dec, texts[s]))
    new = {5: [17], 0: [4000]}                       # a decode step of two of them, and a new one
    for s, t in new.items():
        texts[s] += t
    texts[1] = [8, 9, 10]
    out = _feed(dec, cache, {**new, 1: texts[1]})
    for s in (5, 0, 1):
        _near(out[s], _one_by_one(dec, texts[s]))


@pytest.mark.parametrize("kw", [dict(), dict(dense=True)], ids=["int4", "dense"])
def test_any_number_of_tokens(kw):
    """None, one, the most that go through the GEMV, and one more, each with as many padding tokens as it
    takes after one real token: that token's logits are the same within the products' rounding."""
    dec = _decoder(**kw)
    want = _one_by_one(dec, [7])
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert dec.step_paged(none.long(), none, none, _cache(dec)).shape == (0, want.shape[-1])
    for n in (1, 2, 64, 65):
        cache = _cache(dec)
        cache.extend(_i32([2]), _i32([1]))
        got = dec.step_paged(torch.full((n,), 7, device=DEV), _i32([2] * n), _i32([0] + [-1] * (n - 1)), cache)
        assert got.shape[0] == n
        _near(got[0], want)


@pytest.mark.parametrize("kw,n", [(dict(), 6), (dict(dense=True), 6), (dict(), 70)], ids=["int4", "dense", "gemm"])
def test_tokens_outside_the_vocabulary(kw, n):
    """Of padding they are nobody's; of a real position they give NaN in their own sequence."""
    dec = _decoder(**kw)
    cache, clean = _cache(dec), _cache(dec)
    for c in (cache, clean):
        assert c.extend(_i32([0, 1]), _i32([2, 2])).tolist() == [1, 1]
    seqs, at = _i32([0, 0, 1] + [0] * (n - 3)), _i32([0, 1, 0] + [-1] * (n - 3))
    want = dec.step_paged(torch.tensor([5, 6, 7] + [0] * (n - 3), device=DEV), seqs, at, clean)
    pad = ([-1, 4096, 2 ** 62, -2 ** 63] * n)[:n - 3]
    out = dec.step_paged(torch.tensor([5, 6, 7] + pad, device=DEV), seqs, at, cache)
    assert torch.equal(out[:3], want[:3]) and torch.equal(cache.k, clean.k) and torch.equal(cache.v, clean.v)
    for bad in (-1, 4096):
        out = dec.step_paged(torch.tensor([5, bad, 7] + pad, device=DEV), seqs, at, cache)
        assert torch.equal(out[[0, 2]], want[[0, 2]]) and torch.isnan(out[1]).all()


def test_fork_free_and_compact_change_no_result():
    dec = _decoder()
    cache, plain = _cache(dec), _cache(dec)
    g = torch.Generator().manual_seed(1)
    texts = {s: torch.randint(0, 4096, (n,), generator=g).tolist() for s, n in ((0, 41), (1, 64), (2, 5))}
    _feed(dec, cache, texts)
    assert cache.fork(_i32([0, 0, 1]), _i32([4, 5, 6])).tolist() == [1, 1, 1]  # two share a partly filled page's sequence
    cache.free(_i32([1, 2]))
    assert int(cache.compact()) > 0
    live = int((cache.refs > 0).sum())
    assert not cache.refs[live:].any()
    # every child goes on in its own way; the same in a cache whose pages never moved (fed by the same
    # calls: the products' order of sums goes by the number of rows)
    new = {0: [11], 4: [12], 5: [13, 14], 6: [15]}
    out = _feed(dec, cache, new)
    whole = {0: texts[0] + [11], 4: texts[0] + [12], 5: texts[0] + [13, 14], 6: texts[1] + [15]}
    _feed(dec, plain, texts)
    plain.fork(_i32([0, 0, 1]), _i32([4, 5, 6]))
    want = _feed(dec, plain, new)
    for s in new:
        assert torch.equal(out[s], want[s])  # the pages' numbers are no part of the sums
        _near(out[s], _one_by_one(dec, whole[s]))
    cache.free(_i32([0, 4, 5, 6]))
    assert not cache.refs.any() and (cache.tables == -1).all() and not cache.lengths.any()


def test_decode_step_in_a_graph_with_the_cache_growing():
    dec = _decoder()
    cache, eager = _cache(dec), _cache(dec)
    texts = {0: [1, 2, 3], 1: list(range(30, 62))}
    _feed(dec, cache, texts)
    _feed(dec, eager, texts)
    seqs, ones, tokens = _i32([0, 1]), _i32([1, 1]), torch.tensor([5, 6], device=DEV)

    def step(c):
        positions = c.lengths.index_select(0, seqs.long())
        c.extend(seqs, ones)
        return dec.step_paged(tokens, seqs, positions, c)

    want = [step(eager).clone() for _ in range(20)]
    state = [t.clone() for t in (cache.tables, cache.lengths, cache.refs)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(cache)
    torch.cuda.current_stream().wait_stream(s)
    for t, v in zip((cache.tables, cache.lengths, cache.refs), state):
        t.copy_(v)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache)
    for w in want:  # one captured step, replayed across page ends
        graph.replay()
        assert torch.equal(out, w)
    assert torch.equal(cache.tables, eager.tables) and torch.equal(cache.refs, eager.refs)


def test_a_captured_step_keeps_its_workspaces_when_larger_steps_follow(monkeypatch):
    """The products' split-K workspaces grow with the number of tokens.  A graph captured before holds the addresses of
    the smaller ones, which must not go back to the allocator."""
    from w4a16 import kernels

    for name, empty in (("_WORKSPACE", {}), ("_GEMM_WS", {}), ("_OUTGROWN", [])):
        monkeypatch.setattr(kernels, name, empty)
    dec = _decoder()
    graphs = []
    for n in (2, 5, 65, 200):
        cache = _cache(dec)
        cache.extend(_i32([1]), _i32([150]))
        args = torch.arange(n, device=DEV), _i32([1] * n), _i32([i if i < 150 else -1 for i in range(n)]), cache
        want = dec.step_paged(*args)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = dec.step_paged(*args)
        used = list(kernels._WORKSPACE.values()) + list(kernels._GEMM_WS.values())
        graphs.append((graph, out, want, used, args))
    held = {b.data_ptr() for b in list(kernels._WORKSPACE.values()) + list(kernels._GEMM_WS.values()) + kernels._OUTGROWN}
    assert len(kernels._OUTGROWN) >= 1
    for _, _, _, used, _ in graphs:
        assert {b.data_ptr() for b in used} <= held
    sizes = sum(b.numel() for b in kernels._OUTGROWN)
    assert sizes <= sum(b.numel() for b in list(kernels._WORKSPACE.values()) + list(kernels._GEMM_WS.values()))
    del used
    junk = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=DEV) for _ in range(64)]
    for graph, out, want, _, _ in graphs:
        graph.replay()
        assert torch.equal(out, want)
    assert len(junk) == 64


def test_step_paged_refuses_another_models_cache():
    import w4a16 as K

    dec = _decoder()
    c = dec.cfg
    t = torch.zeros(1, dtype=torch.long, device=DEV)
    for kw in (dict(layers=1), dict(kv_heads=4), dict(head_dim=128), dict(dtype=torch.bfloat16)):
        a = dict(layers=c.layers, kv_heads=c.kv_heads, head_dim=c.head_dim, dtype=torch.float16) | kw
        cache = K.PagedKVCache(a.pop("layers"), 4, 2, 32, **a)
        with pytest.raises(ValueError):
            dec.step_paged(t, t.int(), t.int(), cache)


def _host_rules(x, ids, made, repetition, frequency, presence, bias, mask):
    x = x.double().clone()
    seen = torch.tensor(sorted(set(ids)), device=DEV)
    x[seen] = torch.where(x[seen] > 0, x[seen] / repetition, x[seen] * repetition)
    for t in set(made):
        x[t] -= frequency * made.count(t) + presence
    x = x + bias.double()
    at = torch.arange(x.numel(), device=DEV)
    return x.masked_fill((mask[at // 32].long() >> (at % 32)) % 2 == 0, float("-inf"))


def test_generation_under_rules_matches_an_eager_loop():
    dec = _decoder(seed=7)
    g = torch.Generator(device=DEV).manual_seed(2)
    bias = torch.randn(4096, device=DEV, generator=g) * 0.1
    mask = torch.randint(-2 ** 31, 2 ** 31, (128,), device=DEV, generator=g).int()
    rules = dict(repetition=1.5, frequency=0.25, presence=0.5, bias=bias, mask=mask)
    prompt = [5, 6, 7, 11]
    dec.fill_cache(20)
    k0, v0 = dec.k_cache.clone(), dec.v_cache.clone()
    plain = dec.generate(token=11, pos=20, n=12)
    for _ in range(2):  # captured, then replayed from the start
        dec.k_cache.copy_(k0)
        dec.v_cache.copy_(v0)
        toks = dec.generate(token=11, pos=20, n=12, prompt=prompt, **rules).tolist()
        dec.k_cache.copy_(k0)
        dec.v_cache.copy_(v0)
        t, made = 11, []
        for i in range(12):
            x = _host_rules(dec.step(token=t, pos=20 + i), prompt + made, made, **rules)
            # in fp32 the choice may fall on a token whose value is as good as the best one's
            assert x[toks[i]] >= x.max() - 1e-4 and torch.isfinite(x[toks[i]])
            t = toks[i]
            made.append(t)
    dec.k_cache.copy_(k0)
    dec.v_cache.copy_(v0)
    assert dec.generate(token=11, pos=20, n=12).tolist() == plain.tolist()  # without rules: as before
    dec.k_cache.copy_(k0)
    dec.v_cache.copy_(v0)
    assert dec.generate(token=11, pos=20, n=12, repetition=1.0).tolist() == plain.tolist()  # rules that change nothing
    with pytest.raises(ValueError):
        dec.generate(token=1, pos=0, n=2, prompt=[1] * 161)


def test_generation_refuses_rules_of_other_shapes():
    # a mask of truth values or of one word would be taken for other words, a bias of one value for all tokens'
    dec = _decoder(seed=7)
    for bad in (dict(mask=torch.ones(128, device=DEV, dtype=torch.bool)), dict(mask=torch.ones(1, device=DEV, dtype=torch.int32)),
                dict(mask=torch.ones(4096, device=DEV, dtype=torch.bool)), dict(bias=torch.ones(1, device=DEV)),
                dict(bias=torch.ones(1, 4096, device=DEV))):
        with pytest.raises(ValueError):
            dec.generate(token=1, pos=0, n=2, **bad)
