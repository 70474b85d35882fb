"""Host-side refusals of the paged-cache and logits entry points of the C ABI: bad arguments return a
status before any CUDA call, so these run without a GPU.  No test here launches a kernel."""
import ctypes

import pytest

from w4a16 import _lib
from w4a16 import build as B

P = 1 << 12  # a plausible, aligned address that is never read


@pytest.fixture(scope="module")
def lib():
    B.build()
    return _lib.lib()


def pool(**kw):
    d = dict(k=P, v=P, dtype=_lib.DTYPE_F16, pages=8, kv_heads=2, page_size=16, head_dim=64, page_stride=2048, head_stride=1024,
             token_stride=64) | kw
    return ctypes.byref(_lib.PagePool(**d))


def tables(**kw):
    return ctypes.byref(_lib.PageTables(**(dict(ids=P, sequences=4, width=3, stride=3) | kw)))


def attention(lib, q=P, qs=256, lens=P, seqs=None, rows=4, heads=4, t=None, p=None, out=P, os=256, ws=P, wsb=1 << 30, scale=0.125):
    return lib.w4a16_paged_attention(q, qs, lens, seqs, rows, heads, t or tables(), p or pool(), scale, out, os, ws, wsb, None)


def append(lib, q=P, qs=256, k=P, ks=128, v=P, vs=128, pos=P, tokens=4, heads=4, t=None, cos=P, sin=P, rows=64, p=None, out=P, os=256):
    return lib.w4a16_paged_append(q, qs, k, ks, v, vs, pos, None, tokens, heads, t or tables(), cos, sin, rows, p or pool(), out, os, None)


BAD_POOLS = [(dict(k=0), -1), (dict(dtype=0), -4), (dict(dtype=7), -4), (dict(pages=0), -2), (dict(kv_heads=0), -2), (dict(page_size=12), -2),
             (dict(page_size=0), -2), (dict(page_size=8192), -2), (dict(head_dim=96), -2), (dict(page_stride=0), -3), (dict(token_stride=68), -3),
             (dict(head_stride=-1024), -3), (dict(v=P + 8), -3)]
BAD_TABLES = [(dict(ids=0), -1), (dict(sequences=0), -2), (dict(width=0), -2), (dict(stride=-1), -2), (dict(ids=P + 2), -3)]


def test_attention(lib):
    for change, status in BAD_POOLS:
        assert attention(lib, p=pool(**change)) == status, change
    for change, status in BAD_TABLES:
        assert attention(lib, t=tables(**change)) == status, change
    for kw, status in ((dict(q=None), -1), (dict(lens=None), -1), (dict(out=None), -1), (dict(rows=-1), -2), (dict(heads=3), -2),
                       (dict(heads=0), -2), (dict(q=P + 8), -3), (dict(out=P + 2), -3), (dict(qs=252), -3), (dict(os=128), -3),
                       (dict(lens=P + 1), -3), (dict(seqs=P + 2), -3), (dict(scale=0.0), -2), (dict(scale=-1.0), -2),
                       (dict(scale=float("nan")), -2), (dict(scale=float("inf")), -2)):
        assert attention(lib, **kw) == status, kw
    need = lib.w4a16_paged_attention_workspace_bytes(4, 2, 64)
    assert need > 0
    assert attention(lib, ws=None) == -1 and attention(lib, ws=P + 4) == -3 and attention(lib, wsb=need - 1) == -5
    assert lib.w4a16_paged_attention_call_bytes(_lib.DTYPE_F16, 4, 4, 2, 64, 100000, 16) == need
    for bad in ((0, 4, 4, 2, 64, 3, 16), (1, 0, 4, 2, 64, 3, 16), (1, 4, 3, 2, 64, 3, 16), (1, 4, 4, 2, 96, 3, 16), (1, 4, 4, 2, 64, 0, 16)):
        assert lib.w4a16_paged_attention_call_bytes(*bad) == 0
    assert attention(lib, rows=0) == 0
    assert lib.w4a16_paged_attention_workspace_bytes(3, 2, 64) == 0
    assert lib.w4a16_last_error_string()


def test_attention_scale_times_log2_e_is_a_number(lib):
    # the kernel's exponentials are powers of two: 2.5e38 * log2(e) is past fp32, and infinity times a score of 0 NaN
    for scale in (2.4e38, 3e38, 3.4e38):
        assert attention(lib, scale=scale) == -2, scale
    assert attention(lib, scale=2.0 ** 127, rows=0) == 0 and attention(lib, scale=2.0 ** -149, rows=0) == 0


def test_append(lib):
    for change, status in BAD_POOLS:
        assert append(lib, p=pool(**change)) == status, change
    for change, status in BAD_TABLES:
        assert append(lib, t=tables(**change)) == status, change
    for kw, status in ((dict(q=None), -1), (dict(k=None), -1), (dict(pos=None), -1), (dict(out=None), -1), (dict(tokens=-1), -2), (dict(heads=-1), -2),
                       (dict(cos=None), -2), (dict(rows=0), -2), (dict(ks=100), -3), (dict(v=P + 4), -3), (dict(cos=P + 4), -3), (dict(os=64), -3)):
        assert append(lib, **kw) == status, kw
    assert append(lib, tokens=0) == 0


def test_pages(lib):
    def state(**kw):
        return ctypes.byref(_lib.PageState(**(dict(tables=P, lengths=P, refs=P, sequences=4, width=3, pages=8, page_size=16, table_stride=3) | kw)))

    def blocks(**kw):
        return ctypes.byref(_lib.PageBlocks(**(dict(k=P, v=P, layers=2, pages=8, layer_stride=1 << 15, page_stride=4096, page_bytes=4096) | kw)))

    for change, status in ((dict(tables=0), -1), (dict(refs=0), -1), (dict(sequences=0), -2), (dict(page_size=10), -2), (dict(table_stride=2), -2),
                           (dict(lengths=P + 2), -3)):
        assert lib.w4a16_pages_extend(state(**change), P, P, 2, P, None) == status, change
        assert lib.w4a16_pages_free(state(**change), P, 2, P, None) == status, change
        assert lib.w4a16_pages_fork(state(**change), blocks(), P, P, 2, P, P, 64, None) == status, change
    for change, status in ((dict(k=0), -1), (dict(layers=0), -2), (dict(page_bytes=8192), -2), (dict(page_bytes=0), -2), (dict(page_bytes=4088), -3),
                           (dict(v=P + 8), -3), (dict(layer_stride=8), -3)):
        assert lib.w4a16_pages_copy(blocks(**change), P, P, 2, None) == status, change
        assert lib.w4a16_pages_compact(blocks(**change), P, P, 12, P, P, P, P, 1 << 20, None) == status, change
    assert lib.w4a16_pages_extend(state(), P, P, 1025, P, None) == -2 and lib.w4a16_pages_extend(state(), None, P, 1, P, None) == -1
    assert lib.w4a16_pages_extend(state(), None, None, 0, None, None) == 0
    wide = state(width=1 << 27, table_stride=1 << 27)  # 2^31 positions
    assert lib.w4a16_pages_extend(wide, P, P, 1, P, None) == -2 and lib.w4a16_pages_fork(wide, blocks(), P, P, 1, P, P, 64, None) == -2
    many = state(width=1 << 21, table_stride=1 << 21)  # 2^31 pages over 1024 rows
    assert lib.w4a16_pages_extend(many, P, P, 1024, P, None) == -2
    assert lib.w4a16_pages_free(state(), P, -1, P, None) == -2 and lib.w4a16_pages_free(state(), P + 1, 1, P, None) == -3
    assert lib.w4a16_pages_fork(state(pages=9), blocks(), P, P, 2, P, P, 64, None) == -2
    assert lib.w4a16_pages_fork(state(), blocks(), P, P, 9, P, P, 64, None) == -5
    assert lib.w4a16_pages_fork(state(), blocks(), P, P, 2, P, None, 64, None) == -1
    assert lib.w4a16_pages_copy(blocks(), None, None, 0, None) == 0 and lib.w4a16_pages_copy(blocks(), None, P, 1, None) == -1
    assert lib.w4a16_pages_compact(blocks(), P, P, 12, None, P, P, P, 1 << 20, None) == -1
    assert lib.w4a16_pages_compact(blocks(), P, P, -1, P, P, P, P, 1 << 20, None) == -2
    assert lib.w4a16_pages_compact(blocks(), P, P, 12, P, P, P, P, 8, None) == -5


def test_logits(lib):
    def call(**kw):
        d = _lib.LogitsDesc(**(dict(logits=P, out=P, dtype=0, rows=2, vocab=100, stride=100, out_stride=100) | kw))
        return lib.w4a16_process_logits(ctypes.byref(d), None)

    for kw, status in ((dict(logits=0), -1), (dict(out=0), -1), (dict(dtype=5), -4), (dict(tokens=P, token_bytes=2), -4), (dict(rows=-1), -2),
                       (dict(vocab=-1), -2), (dict(out_stride=99), -2), (dict(stride=-1), -2), (dict(pairs=3), -1), (dict(logits=P + 2), -3),
                       (dict(mask=P + 1), -3), (dict(out=P + 4), -2), (dict(out_stride=120), -2), (dict(bias=P + 2), -3)):
        assert call(**kw) == status, kw
    assert lib.w4a16_process_logits(None, None) == -1
    assert call(rows=0) == 0 and call(vocab=0) == 0


def test_workspace_bytes_from_python(lib):
    import w4a16 as K

    for heads, kv_heads, head_dim in ((32, 8, 64), (9, 1, 128), (24, 2, 256), (1, 1, 64)):
        need = K.paged_attention_workspace_bytes(heads, kv_heads, head_dim)
        assert need == lib.w4a16_paged_attention_workspace_bytes(heads, kv_heads, head_dim) > 0
    for bad in ((3, 2, 64), (0, 1, 64), (4, 0, 64), (4, 2, 96)):
        with pytest.raises(RuntimeError):
            K.paged_attention_workspace_bytes(*bad)


@pytest.mark.parametrize("cls,pack", [(_lib.PagePool, _lib.pack_pool), (_lib.PageTables, _lib.pack_tables), (_lib.PageState, _lib.pack_state),
                                      (_lib.PageBlocks, _lib.pack_blocks), (_lib.LogitsDesc, _lib.pack_logits)])
def test_packed_structures_are_the_declared_ones(cls, pack):
    values = range(1, len(cls._fields_) + 1)
    packed = cls.from_buffer_copy(pack(*values))
    assert len(pack(*values)) == ctypes.sizeof(cls) and [getattr(packed, name) for name, _ in cls._fields_] == list(values)


def test_python_calls_refuse_tensors_that_are_not_on_a_gpu():
    import torch

    import w4a16 as K

    k = torch.zeros(4, 2, 16, 64).half()
    i = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: K.paged_attention(k[:1, :, 0], k, k, i[None], i), lambda: K.paged_append(None, k[:1, :, 0], k[:1, :, 0], i, i[None], k, k),
                 lambda: K.copy_pages(k, k, i, i), lambda: K.extend_sequences(i[None], i, i, i, i, page_size=16),
                 lambda: K.free_sequences(i[None], i, i, i), lambda: K.fork_sequences(k, k, i[None], i, i, i, i),
                 lambda: K.compact_pages(k, k, i[None], i), lambda: K.process_logits(torch.zeros(1, 10))):
        with pytest.raises(RuntimeError):
            call()
