"""paged_append and paged_attention against float64 on the host-described cache: head layouts,
page sizes, lengths around page and tile edges, strided pools, sequences shared by rows, padding,
bad pages, garbage in unused places, offsets past 32 bits, streams and graphs."""
import pytest
import torch

import w4a16 as K

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def _cache(lens, kv_heads, page_size, head_dim, dtype, seed=0, spare=3, nhd=False):
    """k, v pages (scattered over the pool) and tables for sequences of these lengths."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    used = [-(-max(n, 0) // page_size) for n in lens]
    pages = sum(used) + spare
    shape = (pages, page_size, kv_heads, head_dim) if nhd else (pages, kv_heads, page_size, head_dim)
    k, v = (torch.randn(shape, device=DEV, generator=g).to(dtype) for _ in range(2))
    if nhd:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    tables = torch.full((len(lens), max(1, max(used))), -1, dtype=torch.int32)
    for s, n in enumerate(used):
        for i in range(n):
            tables[s, i] = order.pop()
    return k, v, tables.to(DEV), torch.tensor(order, device=DEV)


def _sequence(x, row, n):
    """Positions 0..n of a sequence, [kv_heads, n, head_dim] in float64."""
    at = torch.arange(n, device=DEV)
    return x[row.long()[at // x.shape[2]], :, at % x.shape[2]].double().transpose(0, 1)


def _check(out, q, k, v, tables, lens, seqs=None, scale=None):
    """With u half a step of the type: the probabilities are rounded to it before the product with V and
    the result once more.  fp32: a score is a sum of head_dim exact products whose error is at most
    (head_dim / 16 + 16) steps of 2^-22 of sum |q k| * scale, under 2^-13 here for head_dim <= 256 and
    inputs of unit variance (sum |q k| * scale < 0.8 * 16); it moves numerator and denominator, so
    2^-12.  Adding n terms in blocks of 16 costs n / 16 * 2^-23 = n * 2^-27 of sum p |v|."""
    u, d = HALF[q.dtype], q.shape[2]
    for t, n in enumerate(lens):
        row = tables[t if seqs is None else seqs[t]]
        if n <= 0:
            assert torch.equal(out[t], torch.zeros_like(out[t]))
            continue
        kk, vv = _sequence(k, row, n), _sequence(v, row, n)
        qq = q[t].double().unflatten(0, (k.shape[1], -1))
        p = torch.softmax(torch.einsum("ghd,gnd->ghn", qq, kk) * (d ** -0.5 if scale is None else scale), dim=2)
        ref = torch.einsum("ghn,gnd->ghd", p, vv).flatten(0, 1)
        size = torch.einsum("ghn,gnd->ghd", p, vv.abs()).flatten(0, 1)
        # an fp16 probability below 2^-14 is off by up to 2^-25
        tol = (u + 2.0 ** -12 + n * 2.0 ** -27) * size + u * ref.abs() + 2.0 ** -25 * n * (q.dtype == torch.float16) * vv.abs().mean() * 2
        err = (out[t].double() - ref).abs()
        assert (err <= tol).all(), (t, n, (err / tol).max().item())


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (32, 8), (40, 8), (16, 2), (9, 1), (16, 1), (24, 1), (34, 2)])
@pytest.mark.parametrize("head_dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_attention_head_layouts(heads, kv_heads, head_dim, dtype):
    lens = [1, 37, 300]
    k, v, tables, _ = _cache(lens, kv_heads, 16, head_dim, dtype, seed=heads)
    q = torch.randn(3, heads, head_dim, device=DEV).to(dtype)
    out = K.paged_attention(q, k, v, tables, torch.tensor(lens, dtype=torch.int32, device=DEV))
    _check(out, q, k, v, tables, lens)


@pytest.mark.parametrize("page_size", [1, 2, 8, 16, 64, 256])
@pytest.mark.parametrize("head_dim,dtype", [(64, torch.bfloat16), (128, torch.float16), (256, torch.float16), (256, torch.bfloat16)])
def test_attention_lengths_around_edges(page_size, head_dim, dtype):
    lens = [0, 1, 2, 7, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511, 513, 1000, -5]
    k, v, tables, _ = _cache(lens, 2, page_size, head_dim, dtype, seed=page_size)
    q = torch.randn(len(lens), 8, head_dim, device=DEV).to(dtype)
    out = K.paged_attention(q, k, v, tables, torch.tensor(lens, dtype=torch.int32, device=DEV))
    _check(out, q, k, v, tables, lens)


@pytest.mark.parametrize("rows,top", [(1, 20000), (3, 9001), (200, 400), (1500, 20), (700, 1)])
def test_attention_batches(rows, top):
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(0, top + 1, (rows,), generator=g).tolist()
    lens[0] = top
    k, v, tables, _ = _cache(lens, 4, 16, 64, torch.float16, seed=rows)
    q = torch.randn(rows, 16, 64, device=DEV).half()
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = K.paged_attention(q, k, v, tables, lengths)
    some = torch.randperm(rows, generator=g)[:40].tolist() + [0]
    _check(out[some], q[some], k, v, tables[some], [lens[i] for i in some])
    for _ in range(3):  # the same bits every time
        assert torch.equal(out, K.paged_attention(q, k, v, tables, lengths))


@pytest.mark.parametrize("rows,kv_heads,heads", [(1, 1, 1), (1, 8, 32), (3, 8, 32), (7, 8, 24), (18, 8, 8), (40, 8, 16), (2, 2, 32), (5, 1, 9)])
@pytest.mark.parametrize("head_dim,dtype", [(64, torch.float16), (128, torch.bfloat16), (256, torch.float16)])
def test_attention_of_few_rows_in_tables_of_any_width(rows, kv_heads, heads, head_dim, dtype):
    # the widths around which a row goes to 1, 2, 4 or 8 CTAs together, or is cut into parts
    lens = [0 if i % 5 == 3 else (i * 389) % 4097 for i in range(1, rows + 1)]
    lens[0] = 4096
    k, v, tables, _ = _cache(lens, kv_heads, 16, head_dim, dtype, seed=rows)
    q = torch.randn(rows, heads, head_dim, device=DEV).to(dtype)
    some = [0, rows - 1, rows // 2]
    for cap in (16, 128, 144, 256, 272, 512, 528, 1024, 1040, 2048, 2064, 4096, 4112):
        short = [min(n, cap) for n in lens]
        table = torch.full((rows, cap // 16), -1, dtype=torch.int32, device=DEV)
        n = min(cap // 16, tables.shape[1])
        table[:, :n] = tables[:, :n]
        lengths = torch.tensor(short, dtype=torch.int32, device=DEV)
        out = K.paged_attention(q, k, v, table, lengths)
        _check(out[some], q[some], k, v, table[some], [short[i] for i in some])
        assert not out[lengths == 0].any()
        assert torch.equal(out, K.paged_attention(q, k, v, table, lengths))


@pytest.mark.parametrize("head_dim,rows,top", [(64, 8, 200000), (128, 1500, 60000), (256, 3, 30000)])
def test_attention_one_long_row_among_short_ones(head_dim, rows, top):
    # nearly all work in one item, cut into hundreds of parts (by CTAs, by warps; 12 query heads of one
    # kv head: two blocks of heads with head_dim 256)
    lens = [top] + [1 + i % 3 for i in range(rows - 1)]
    k, v, tables, _ = _cache(lens, 1, 64, head_dim, torch.float16, seed=rows)
    q = torch.randn(rows, 12, head_dim, device=DEV).half()
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = K.paged_attention(q, k, v, tables, lengths)
    some = [0, 1, 2, rows - 1]
    _check(out[some], q[some], k, v, tables[some], [lens[i] for i in some])
    assert torch.equal(out, K.paged_attention(q, k, v, tables, lengths))


@pytest.mark.parametrize("rows", [1, 5, 127, 128, 129, 300, 2000])
def test_attention_padded_batches(rows):
    # rows of no positions before, between and behind the others, and nothing else
    g = torch.Generator().manual_seed(rows)
    lens = [0 if torch.rand((), generator=g) < 0.6 else int(torch.randint(1, 90, (), generator=g)) for _ in range(rows)]
    lens[-1] = 0
    k, v, tables, _ = _cache(lens, 2, 8, 64, torch.bfloat16, seed=rows)
    q = torch.randn(rows, 6, 64, device=DEV).bfloat16()
    out = K.paged_attention(q, k, v, tables, torch.tensor(lens, dtype=torch.int32, device=DEV))
    some = torch.randperm(rows, generator=g)[:60].tolist()
    _check(out[some], q[some], k, v, tables[some], [lens[i] for i in some])
    empty = torch.tensor([n == 0 for n in lens], device=DEV)
    assert not out[empty].any()
    assert not K.paged_attention(q, k, v, tables, torch.zeros(rows, dtype=torch.int32, device=DEV)).any()


def test_attention_workspace_of_a_call():
    # what a call takes is nothing or all; a smaller one than all is refused
    from w4a16 import _lib

    lens = [300, 7]
    for width, heads in ((20, 8), (20, 32), (5000, 8)):
        k, v, tables, _ = _cache(lens, 4, 16, 64, torch.float16)
        wide = torch.full((2, width), -1, dtype=torch.int32, device=DEV)
        wide[:, : tables.shape[1]] = tables
        q = torch.randn(2, heads, 64, device=DEV).half()
        n = torch.tensor(lens, dtype=torch.int32, device=DEV)
        want = K.paged_attention(q, k, v, wide, n)
        _check(want, q, k, v, wide, lens)
        need = _lib.lib().w4a16_paged_attention_call_bytes(_lib.DTYPE_F16, 2, heads, 4, 64, width, 16)
        full = _lib.lib().w4a16_paged_attention_workspace_bytes(heads, 4, 64)
        assert need == (full if width == 5000 else 0)
        assert torch.equal(K.paged_attention(q, k, v, wide, n, workspace=torch.empty(full, dtype=torch.uint8, device=DEV)), want)
        small = torch.empty(16, dtype=torch.uint8, device=DEV)
        with pytest.raises(RuntimeError):
            K.paged_attention(q, k, v, wide, n, workspace=small)


def test_attention_strides_and_scale():
    lens = [130, 77, 5]
    k, v, tables, _ = _cache(lens, 8, 16, 64, torch.float16, nhd=True)  # [pages, page_size, kv_heads, head_dim] storage
    wide = torch.randn(3, 48 * 64, device=DEV).half()
    q = wide[:, : 32 * 64].unflatten(1, (32, 64))
    big = torch.zeros(3, 40, 64, device=DEV).half()
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    out = K.paged_attention(q, k, v, tables, lengths, scale=0.3, out=big[:, 4:36])
    _check(out, q, k, v, tables, lens, scale=0.3)
    assert not big[:, :4].any() and not big[:, 36:].any()
    padded = torch.full((3, tables.shape[1] + 500), -1, dtype=torch.int32, device=DEV)  # a much wider table
    padded[:, : tables.shape[1]] = tables
    _check(K.paged_attention(q, k, v, padded, lengths, scale=0.3), q, k, v, tables, lens, scale=0.3)  # sums in another order
    assert torch.equal(K.paged_attention(q, k, v, padded[:, : tables.shape[1] + 1], lengths, scale=0.3), out)  # rows apart


def test_attention_rows_of_one_sequence():
    # a prompt's tokens as rows with growing lengths, mixed with another sequence's
    k, v, tables, _ = _cache([90, 40], 2, 8, 128, torch.bfloat16)
    lens, seqs = [1, 2, 33, 40, 90, 64, 0], [0, 0, 0, 1, 0, 0, 1]
    q = torch.randn(len(lens), 4, 128, device=DEV).bfloat16()
    out = K.paged_attention(q, k, v, tables, torch.tensor(lens, dtype=torch.int32, device=DEV),
                            seqs=torch.tensor(seqs, dtype=torch.int32, device=DEV))
    _check(out, q, k, v, tables, lens, seqs)


def test_attention_garbage_outside_the_lengths_and_infinities_inside():
    lens = [0, 5, 23, 64, 100]
    k, v, tables, free = _cache(lens, 2, 16, 64, torch.float16)
    q = torch.randn(5, 8, 64, device=DEV).half()
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = K.paged_attention(q, k, v, tables, lengths)
    for x in (k, v):  # NaN and infinities in every place that no row attends to
        x[free] = float("nan")
        for s, n in enumerate(lens):
            if n % 16:
                x[tables[s, n // 16].long(), :, n % 16:] = float("inf") if s % 2 else float("nan")
    assert torch.equal(K.paged_attention(q, k, v, tables, lengths), want)
    # a key of -inf in one kv head: probability 0 where q . k is -inf, by the formula NaN elsewhere
    q1 = q.abs()
    k[tables[4, 2].long(), 0, 3] = float("-inf")
    kk = _sequence(k, tables[4], 100)
    p = torch.softmax(torch.einsum("ghd,gnd->ghn", q1[4].double().unflatten(0, (2, 4)), kk) / 8, dim=2)
    out = K.paged_attention(q1, k, v, tables, lengths)[4].double()
    ref = torch.einsum("ghn,gnd->ghd", p, _sequence(v, tables[4], 100)).flatten(0, 1)
    assert torch.isfinite(ref).all() and (out - ref).abs().max() < 4e-3
    k[tables[4, 2].long(), 0, 3] = float("nan")
    out = K.paged_attention(q1, k, v, tables, lengths)[4]
    assert torch.isnan(out[:4]).all() and torch.isfinite(out[4:]).all()
    # large scores: the running maximum keeps the exponentials finite
    big = K.paged_attention(q * 100, k, v, tables, lengths)
    assert torch.isfinite(big[:4]).all()


@pytest.mark.parametrize("rows,kv_heads,n", [(1, 2, 500), (60, 4, 3000), (600, 4, 400), (2, 1, 60000)])
@pytest.mark.parametrize("above", [10, 16, 20])
@pytest.mark.parametrize("head_dim,dtype", [(64, torch.float16), (128, torch.float16), (64, torch.bfloat16)])
def test_attention_one_key_far_above_a_long_tail(rows, kv_heads, n, above, head_dim, dtype):
    """The first key scores about `above` over all others and its value is zero, so the result is what the
    others leave.  With u half a step of the type the result is rounded once.  A score is off by less than
    (head_dim / 16 + 16) steps of 2^-22 of sum |q k| * scale <= 32: 2^-12, in numerator and denominator:
    2^-11; adding up n terms costs n * 2^-27 of sum p |v|; the parts of a probability leave out at most
    2^-16 of it (bf16), or 2^-38 of the largest one (fp16), which is e^above of the others.  An fp16 result
    below 2^-14 (e^-20 times 500 values of about 1.3 is 1.3e-6) is a multiple of 2^-24: rounded by up to 2^-25."""
    g = torch.Generator(device=DEV).manual_seed(n)
    heads = 2 * kv_heads
    k, v, tables, _ = _cache([n] * rows, kv_heads, 16, head_dim, dtype, seed=n)
    q = (torch.randn(rows, heads, head_dim, device=DEV, generator=g) * 0.1 + 1).to(dtype)
    k.mul_(0.1)
    v.copy_(v.abs() + 0.5)
    first = tables[:, 0].long()
    k[first, :, 0] = above * head_dim ** -0.5
    v[first, :, 0] = 0
    out = K.paged_attention(q, k, v, tables, torch.full((rows,), n, dtype=torch.int32, device=DEV))
    for t in sorted({0, rows // 2, rows - 1}):
        kk, vv = _sequence(k, tables[t], n), _sequence(v, tables[t], n)
        s = torch.einsum("ghd,gnd->ghn", q[t].double().unflatten(0, (kv_heads, 2)), kk) * head_dim ** -0.5
        p = torch.softmax(s, dim=2)
        assert (s[:, :, 0] - s[:, :, 1:].amax(2) > above - 4).all()
        ref = torch.einsum("ghn,gnd->ghd", p, vv).flatten(0, 1)  # every value is positive
        lost = n * 2.0 ** -38 * vv.amax() + 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -16 * ref
        assert ((out[t].double() - ref).abs() <= (HALF[dtype] + 2.0 ** -11 + n * 2.0 ** -27) * ref + lost).all()


@pytest.mark.parametrize("heads,head_dim", [(1, 64), (16, 64), (1, 128), (9, 128), (1, 256)])
def test_attention_long_sums_have_no_bias(heads, head_dim):
    """Values of 1, so the result is 1 whatever the probabilities; many rows of one long sequence, so that a warp
    adds up thousands of tiles.  The result is rounded once (2^-12 below 1).  A sum of N tiles rounded to nearest
    is off by errors of no preferred sign, each below 2^-24 of it: 8 sqrt(N) 2^-24 is past any chance; the parts of
    the probabilities leave out 2^-22."""
    n, rows = 2 ** 24 // head_dim, 1200
    g = torch.Generator(device=DEV).manual_seed(heads)
    k = torch.randn(n // 256, 1, 256, head_dim, device=DEV, generator=g).half()
    v = torch.ones_like(k)
    q = torch.randn(rows, heads, head_dim, device=DEV, generator=g).half()
    tables = torch.arange(n // 256, dtype=torch.int32, device=DEV)[None]
    lengths = torch.full((rows,), n, dtype=torch.int32, device=DEV)
    out = K.paged_attention(q, k, v, tables, lengths, seqs=torch.zeros_like(lengths))
    assert ((out.double() - 1).abs() <= 2.0 ** -12 + 8 * (n / 16) ** 0.5 * 2.0 ** -24 + 2.0 ** -22).all()


@pytest.mark.parametrize("head_dim,dtype", [(64, torch.float16), (64, torch.bfloat16), (128, torch.bfloat16), (256, torch.bfloat16)])
@pytest.mark.parametrize("rows,group", [(60, 1), (60, 12), (900, 4)])
def test_attention_takes_both_parts_of_a_probability(rows, group, head_dim, dtype):
    """Three keys: two of score 0 with the values -h and -l, the type's nearest to x = e^s and to x - h, and
    one of score s < 0 with the value 1.  So the result is (x - h - l) / (2 + x), which two parts of the type
    leave of x: with b bits 2^-(2b + 1) of it (bf16 2^-17, fp16 2^-23), and one part 2^-b.  s is exact (one dimension of
    q is 1, the others 0); the exponential is off by 2^-22 and by the two roundings of its argument, below
    1.5 * 2^-24; adding up terms below 1 in fp32 costs less than 2^-23 each, of at most 9."""
    g = torch.Generator(device=DEV).manual_seed(rows)
    k = torch.zeros(rows, 1, 16, head_dim, dtype=dtype, device=DEV)
    v = torch.zeros_like(k)
    s = -(torch.rand(rows, device=DEV, generator=g) * 0.9 + 0.1).to(dtype)
    x = s.double().exp()
    h = x.to(dtype)
    low = (x - h.double()).to(dtype)
    k[:, 0, 2, 0] = s
    v[:, 0, 0], v[:, 0, 1], v[:, 0, 2] = -h[:, None], -low[:, None], 1
    q = torch.zeros(rows, group, head_dim, dtype=dtype, device=DEV)
    q[:, :, 0] = 1
    tables = torch.arange(rows, dtype=torch.int32, device=DEV)[:, None]
    out = K.paged_attention(q, k, v, tables, torch.full((rows,), 3, dtype=torch.int32, device=DEV), scale=1.0)
    ref = ((x - h.double() - low.double()) / (2 + x))[:, None, None]
    lost = 2.0 ** -23 if dtype == torch.float16 else 2.0 ** -17
    tol = HALF[dtype] * ref.abs() + (2.0 ** -22 + 1.5 * 2.0 ** -24 + 9 * 2.0 ** -23 + lost) / 2 + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((out.double() - ref).abs() <= tol).all()


def test_attention_bad_pages_give_nan_and_touch_nothing_else():
    lens = [40, 40, 40, 40, 40, 40]
    k, v, tables, _ = _cache(lens, 2, 16, 64, torch.float16)
    q = torch.randn(6, 4, 64, device=DEV).half()
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    want = K.paged_attention(q, k, v, tables, lengths)
    bad = tables.clone()
    bad[0, 1], bad[1, 0], bad[2, 2] = -1, k.shape[0], 2 ** 31 - 1
    out = K.paged_attention(q, k, v, bad, lengths)
    assert torch.isnan(out[:3]).all() and torch.equal(out[3:], want[3:])
    longer = lengths.clone()
    longer[3], longer[4] = 49, 2 ** 31 - 1  # past the tables' width
    out = K.paged_attention(q, k, v, tables, longer)
    assert torch.isnan(out[3:5]).all() and torch.equal(out[5], want[5]) and torch.equal(out[:3], want[:3])
    seqs = torch.tensor([0, 1, -1, 6, 4, 5], dtype=torch.int32, device=DEV)
    out = K.paged_attention(q, k, v, tables, lengths, seqs=seqs)
    assert torch.isnan(out[2:4]).all() and torch.equal(out[[0, 1, 4, 5]], want[[0, 1, 4, 5]])


# Rows with a bad page, sequence or length between good ones, in each form of the call: a cluster for an
# item; CTAs that take several items; warps; parts of few long items, joined by a CTA each and by heads.
FORMS = [("cluster", 6, 2, 8, 64, torch.float16, 40), ("cluster", 3, 8, 32, 128, torch.bfloat16, 500), ("items", 400, 4, 8, 64, torch.float16, 64),
         ("items", 32, 8, 32, 128, torch.bfloat16, 4096), ("items", 90, 4, 8, 256, torch.float16, 200), ("items", 100, 4, 64, 128, torch.float16, 300),
         ("warps", 1500, 4, 4, 64, torch.bfloat16, 60), ("warps", 700, 4, 48, 128, torch.float16, 40), ("parts", 40, 4, 16, 64, torch.float16, 5000),
         ("parts", 3, 4, 16, 128, torch.bfloat16, 30000), ("parts", 2, 1, 12, 64, torch.float16, 60000)]


@pytest.mark.parametrize("form,rows,kv_heads,heads,head_dim,dtype,top", FORMS)
def test_attention_bad_rows_leave_the_others_as_they_were(form, rows, kv_heads, heads, head_dim, dtype, top):
    g = torch.Generator().manual_seed(rows)
    lens = torch.randint(1, top + 1, (rows,), generator=g).tolist()
    lens[1::3] = [1 + n % 20 for n in lens[1::3]]  # short rows behind long ones
    lens[0] = top
    if rows > 3:
        lens[5::11] = [0] * len(lens[5::11])
    broken = set(range(0, rows, 6)) if rows > 6 else {0}
    k, v, tables, free = _cache(lens, kv_heads, 16, head_dim, dtype, seed=rows)
    q = torch.randn(rows, heads, head_dim, device=DEV).to(dtype)
    lengths, seqs = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (lens, list(range(rows))))
    want = K.paged_attention(q, k, v, tables, lengths, seqs=seqs)
    bad, other, hurt = tables.clone(), seqs.clone(), []
    for i, r in enumerate(sorted(broken)):
        pages = -(-lens[r] // 16)
        if pages == 0:
            continue
        hurt.append(r)
        if i % 4 == 0:
            bad[r, pages - 1] = -1
        elif i % 4 == 1:
            bad[r, :pages] = k.shape[0]
        elif i % 4 == 2:
            bad[r, 0] = 2 ** 31 - 1
        else:
            other[r] = rows if i % 8 == 3 else -1
    out = K.paged_attention(q, k, v, bad, lengths, seqs=other)
    kept = torch.tensor([r not in hurt for r in range(rows)], device=DEV)
    assert torch.isnan(out[~kept]).all() and torch.equal(out[kept], want[kept])
    # lengths past the tables: where another table is one page wider, the same lengths are good ones
    wide = torch.cat([tables, torch.full_like(tables[:, :1], int(free[0]))], 1)
    wide[hurt] = torch.where(wide[hurt] < 0, free[0].int(), wide[hurt])
    past = lengths.clone()
    past[hurt] = tables.shape[1] * 16 + 1
    want = K.paged_attention(q, k, v, wide, past)
    assert not torch.isnan(want).any()
    past[hurt[::2]] = 2 ** 31 - 1
    out = K.paged_attention(q, k, v, wide[:, :-1], past)
    assert torch.isnan(out[~kept]).all()
    if form == "cluster":  # chosen by the tables' width
        _check(out[kept], q[kept], k, v, tables[kept], [n for r, n in enumerate(lens) if r not in hurt])
    else:
        assert torch.equal(out[kept], want[kept])


def test_attention_offsets_past_32_bits():
    # the last pages of a pool of more than 2^32 elements
    pages = 2 ** 32 // (8 * 64 * 128) + 8
    k = torch.empty(pages, 8, 64, 128, dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    ids = torch.tensor([[pages - 1, 3, pages - 5, pages // 2 + 1]], dtype=torch.int32, device=DEV)
    for x in (k, v):
        x[ids[0].long()] = torch.randn(4, 8, 64, 128, device=DEV).bfloat16()
    q = torch.randn(1, 32, 128, device=DEV).bfloat16()
    out = K.paged_attention(q, k, v, ids, torch.tensor([250], dtype=torch.int32, device=DEV))
    _check(out, q, k, v, ids, [250])
    at = torch.tensor([0, 130], dtype=torch.int32, device=DEV)
    new = torch.randn(2, 8, 128, device=DEV).bfloat16()
    K.paged_append(None, new, new, at, ids, k, v, seqs=torch.zeros(2, dtype=torch.int32, device=DEV))
    assert torch.equal(k[pages - 1, :, 0], new[0]) and torch.equal(v[pages - 5, :, 2], new[1])


def test_attention_streams_and_graphs():
    lens = [3000, 10, 700]
    k, v, tables, _ = _cache(lens, 2, 16, 128, torch.float16)
    lengths = torch.tensor(lens, dtype=torch.int32, device=DEV)
    qs = [torch.randn(3, 8, 128, device=DEV).half() for _ in range(2)]
    want = [K.paged_attention(q, k, v, tables, lengths) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    got = [None, None]
    torch.cuda.synchronize()
    for _ in range(20):  # two calls at once
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = K.paged_attention(qs[i], k, v, tables, lengths)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for q in qs:  # two graphs, replayed on two streams at once, with lengths changed in between
        g, out = torch.cuda.CUDAGraph(), torch.empty_like(q)
        with torch.cuda.graph(g):
            K.paged_attention(q, k, v, tables, lengths, out=out)
        graphs.append(g)
        outs.append(out)
    for change in ([3000, 10, 700], [17, 1, 0]):
        lengths.copy_(torch.tensor(change, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for q, out in zip(qs, outs):
            _check(out, q, k, v, tables, change)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_calls_on_another_device_than_the_current_one():
    dev = torch.device("cuda", 1)
    k, v, tables, _ = _cache([70, 9], 2, 16, 64, torch.float16)
    q = torch.randn(2, 4, 64, device=DEV).half()
    n = torch.tensor([70, 9], dtype=torch.int32, device=DEV)
    want = K.paged_attention(q, k, v, tables, n)
    out = K.paged_attention(*(t.to(dev) for t in (q, k, v, tables, n)))
    assert out.device == dev and torch.equal(out.to(DEV), want)
    with pytest.raises(RuntimeError):
        K.paged_attention(q, k.to(dev), v.to(dev), tables, n)


# ------------------------------------------------------------------------------------- append

def _angles(n, d):
    a = torch.arange(n, device=DEV).double()[:, None] / 10000 ** (torch.arange(0, d, 2, device=DEV).double() / d)[None]
    a = torch.cat([a, a], 1)
    return a.cos().float(), a.sin().float()


def _turn(x, cos, sin):
    half = x.shape[-1] // 2
    x = x.double()
    return x * cos.double()[:, None] + torch.cat([-x[..., half:], x[..., :half]], -1) * sin.double()[:, None]


@pytest.mark.parametrize("tokens,heads,kv_heads,head_dim,page_size,dtype", [
    (1, 32, 8, 64, 16, torch.float16), (33, 8, 8, 128, 1, torch.bfloat16), (257, 7, 1, 256, 64, torch.float16),
    (5000, 4, 2, 64, 8, torch.bfloat16)])
@pytest.mark.parametrize("nhd", [False, True])
def test_append(tokens, heads, kv_heads, head_dim, page_size, dtype, nhd):
    g = torch.Generator().manual_seed(tokens)
    count = torch.bincount(torch.randint(0, 7, (tokens,), generator=g), minlength=7).tolist()
    lens = [n + 5 for n in count]
    k, v, tables, _ = _cache(lens, kv_heads, page_size, head_dim, dtype, nhd=nhd)
    at = torch.cat([torch.arange(n) for n in count]) + 5
    seqs = torch.cat([torch.full((n,), i) for i, n in enumerate(count)])
    mix = torch.randperm(tokens, generator=g)
    at, seqs = at[mix].to(DEV, torch.int32), seqs[mix].to(DEV, torch.int32)
    wide = torch.randn(tokens, heads + 2 * kv_heads, head_dim, device=DEV).to(dtype)
    q, kn, vn = wide.split([heads, kv_heads, kv_heads], dim=1)
    cos, sin = _angles(max(lens), head_dim)
    k0, v0 = k.clone(), v.clone()
    kept = wide.clone()
    out = K.paged_append(q, kn, vn, at, tables, k, v, cos=cos, sin=sin, seqs=seqs)
    assert torch.equal(wide, kept)
    c, s = cos[at.long()], sin[at.long()]
    u = HALF[dtype]
    # rounded once, from two fp32 products and a sum (3 half steps of 2^-24 of the products' sizes)
    for got, x in ((out, q), (k[tables[seqs.long(), at.long() // page_size].long(), :, at.long() % page_size], kn)):
        ref = _turn(x, c, s)
        size = _turn(x, c, s).abs() + 2 * x.abs().amax(-1, keepdim=True).double()
        assert ((got.double() - ref).abs() <= u * ref.abs() + 2.0 ** -22 * size + 2.0 ** -25 * (dtype == torch.float16)).all()
    page, row = tables[seqs.long(), at.long() // page_size].long(), at.long() % page_size
    v0[page, :, row] = vn
    assert torch.equal(v, v0)
    k0[page, :, row] = k[page, :, row]
    assert torch.equal(k, k0)  # nothing else was written
    # without angles: the values as they are; q in place
    k2, v2 = k.clone(), v.clone()
    assert torch.equal(K.paged_append(q, kn, vn, at, tables, k2, v2, seqs=seqs), q)
    assert torch.equal(k2[page, :, row], kn)
    same = K.paged_append(q, kn, vn, at, tables, k, v, cos=cos, sin=sin, seqs=seqs, out=q)
    assert same.data_ptr() == q.data_ptr() and torch.equal(q, out)


def test_append_padding_and_bad_indices():
    k, v, tables, _ = _cache([20, 20], 2, 16, 64, torch.float16)
    k0, v0 = k.clone(), v.clone()
    cos, sin = _angles(24, 64)
    q, kn, vn = (torch.randn(8, n, 64, device=DEV).half() for n in (4, 2, 2))
    bad = tables.clone()
    bad[1, 1] = k.shape[0]
    #                       padding, past the angles, past the table, bad page, bad sequences, good, padding
    at = torch.tensor([-1, 25, 2 ** 31 - 1, 17, 3, 3, 19, -2 ** 31], dtype=torch.int32, device=DEV)
    seqs = torch.tensor([0, 0, 0, 1, 2, -1, 0, 99], dtype=torch.int32, device=DEV)
    out = K.paged_append(q, kn, vn, at, bad, k, v, cos=cos, sin=sin, seqs=seqs)
    assert not out[0].any() and not out[7].any()
    assert torch.isnan(out[1:6]).all() and torch.isfinite(out[6]).all()
    page = tables[0, 1].long()
    assert torch.equal(v[page, :, 3], vn[6])
    k0[page, :, 3], v0[page, :, 3] = k[page, :, 3], vn[6]
    assert torch.equal(k, k0) and torch.equal(v, v0)


def test_refusals_on_the_host():
    k, v, tables, _ = _cache([20], 2, 16, 64, torch.float16)
    q = torch.randn(1, 4, 64, device=DEV).half()
    n = torch.tensor([20], dtype=torch.int32, device=DEV)
    bad = [
        dict(q=q.float()), dict(q=q[:, :3]), dict(q=q[0]), dict(q=q.cpu()), dict(q=torch.randn(1, 4, 128, device=DEV).half()[..., ::2]),
        dict(k=k.float(), v=v.float()), dict(v=v.bfloat16()), dict(v=v[:1]), dict(k=k[..., :32], v=v[..., :32]), dict(k=k[0], v=v[0]),
        dict(tables=tables.long()), dict(tables=tables[0]), dict(lengths=n.long()), dict(lengths=torch.cat([n, n])),
        dict(lengths=n.cpu()), dict(out=torch.empty(1, 4, 64, device=DEV)), dict(seqs=torch.zeros(2, dtype=torch.int32, device=DEV)),
        dict(k=k[:, :, :12], v=v[:, :, :12]),  # a page size that is no power of two
        dict(workspace=torch.empty(8, dtype=torch.uint8, device=DEV)), dict(workspace=torch.empty(1 << 26, dtype=torch.int8, device=DEV)),
    ]
    for change in bad:
        args = dict(q=q, k=k, v=v, tables=tables, lengths=n, out=None, seqs=None, workspace=None) | change
        with pytest.raises(RuntimeError):
            K.paged_attention(args["q"], args["k"], args["v"], args["tables"], args["lengths"], out=args["out"], seqs=args["seqs"],
                              workspace=args["workspace"])
    kn = torch.randn(1, 2, 64, device=DEV).half()
    cos, sin = _angles(24, 64)
    pos = n - 1
    for change in (dict(kn=kn.float()), dict(kn=kn[:, :1]), dict(pos=pos.long()), dict(cos=cos, sin=None), dict(cos=cos[:, :32], sin=sin[:, :32]),
                   dict(cos=cos.half(), sin=sin.half()), dict(cos=cos, sin=sin[:5]), dict(out=torch.empty(2, 4, 64, device=DEV).half())):
        args = dict(kn=kn, pos=pos, cos=None, sin=None, out=None) | change
        with pytest.raises(RuntimeError):
            K.paged_append(q, args["kn"], kn, args["pos"], tables, k, v, cos=args["cos"], sin=args["sin"], out=args["out"])
    # empty batches are fine
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    assert K.paged_attention(q[:0], k, v, tables, none).shape == (0, 4, 64)
    assert K.paged_append(q[:0], kn[:0], kn[:0], none, tables, k, v).shape == (0, 4, 64)
