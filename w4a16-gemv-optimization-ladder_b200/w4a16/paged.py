"""Serving several sequences over a paged key-value cache.

The reference decodes one sequence through the Hugging Face cache (benchmarks/end_to_end.py:
24-42), and decode_attention here holds one sequence's cache as one block.  With several
sequences of different lengths the cache is cut into pages of `page_size` positions:

    k_pages, v_pages  fp16 or bf16 [pages, kv_heads, page_size, head_dim] (one layer's pool; any
                      strides with the last dimension contiguous, so [pages, page_size, kv_heads,
                      head_dim] storage is passed as its transpose(1, 2))
    tables            int32 [sequences, width]: the pages of each sequence in order, -1 past the last
    lengths           int32 [sequences]: positions held
    refs              int32 [pages]: table entries that hold the page, 0 for a free one

    paged_append      rotary embedding of new q and k, k and v written into their pages
    paged_attention   attention of one new token per row over its sequence's pages
    extend_sequences, fork_sequences, free_sequences, compact_pages, copy_pages
                      the pages' bookkeeping, on the device
    PagedKVCache      the tensors above for all layers of a model, with the calls as methods

Everything is read on the device, launched on the current stream and can be captured in a CUDA
graph; nothing is kept between calls.  Wrong dtypes, devices, shapes or layouts raise
RuntimeError before anything is launched; indices are checked in the kernels (a bad page, position
or sequence gives NaN, is skipped, or is refused, as each function says).
"""
import functools

import torch

from . import _lib

_POOL_DTYPES = {torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
# torch.cuda.current_stream(device).cuda_stream and torch.cuda.current_device(), without the objects
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _refuse(msg):
    raise RuntimeError(msg)


def _call(name, dev, *args):
    """Run a C entry on dev's current stream, its last argument.  The checks before it build their
    messages only when they fail: a decode step is short of host time."""
    fn, index = getattr(_lib.lib(), name), dev.index
    if _current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _raw_stream(index))
    if status:
        _lib.check(status, name)


def _pool(k_pages, v_pages):
    """One layer's pool, checked: its C description, kv_heads, page_size, head_dim."""
    dtype = _POOL_DTYPES.get(getattr(k_pages, "dtype", None))
    if dtype is None or k_pages.dim() != 4 or not k_pages.is_cuda:
        _refuse("k_pages must be an fp16 or bf16 CUDA tensor [pages, kv_heads, page_size, head_dim]")
    shape, stride = k_pages.shape, k_pages.stride()
    if not (isinstance(v_pages, torch.Tensor) and v_pages.device == k_pages.device and v_pages.dtype is k_pages.dtype
            and v_pages.shape == shape and v_pages.stride() == stride):
        _refuse("v_pages must have the device, dtype, shape and strides of k_pages")
    pages, kv_heads, page_size, head_dim = shape
    sp, sh, st, sd = stride
    if sd != 1:
        _refuse("the last dimension of the pages must be contiguous")
    # a dimension of one entry may carry any stride
    return _lib.pack_pool(k_pages.data_ptr(), v_pages.data_ptr(), dtype, pages, kv_heads, page_size, head_dim, sp if pages > 1 else 8,
                          sh if kv_heads > 1 else 8, st if page_size > 1 else 8), kv_heads, page_size, head_dim


@functools.lru_cache(maxsize=256)
def _bytes(name, *args):
    """The scratch that a C entry asks for: a function of the sizes alone."""
    return getattr(_lib.lib(), name)(*args)


@functools.lru_cache(maxsize=1024)
def _attention_bytes(index, *args):
    with torch.cuda.device(index):
        return _lib.lib().w4a16_paged_attention_call_bytes(*args)


def _tables(tables, dev):
    if not (isinstance(tables, torch.Tensor) and tables.device == dev and tables.dtype == torch.int32 and tables.dim() == 2):
        _refuse(f"tables must be an int32 [sequences, width] tensor on {dev}")
    sequences, width = tables.shape
    stride, one = tables.stride()
    if one != 1 and width > 1:
        _refuse("the rows of tables must be contiguous")
    return _lib.pack_tables(tables.data_ptr(), sequences, width, stride), width


def _index(t, n, name, dev):
    if not (isinstance(t, torch.Tensor) and t.device == dev and t.dtype == torch.int32 and t.dim() == 1
            and t.is_contiguous() and (n is None or t.shape[0] == n)):
        _refuse(f"{name} must be a contiguous int32 [{'n' if n is None else n}] tensor on {dev}")
    return t.data_ptr()


def _tokens(t, n, heads, head_dim, dtype, name, dev):
    """(address, elements between tokens) of a [tokens, heads, head_dim] tensor whose tokens are
    contiguous blocks (rows of a wider projection output will do)."""
    if not (isinstance(t, torch.Tensor) and t.device == dev and t.dtype == dtype and t.shape == (n, heads, head_dim)):
        _refuse(f"{name} must be a {dtype} [{n}, {heads}, {head_dim}] tensor on {dev}")
    sn, sh, sd = t.stride()
    if sd != 1 or (heads > 1 and sh != head_dim):
        _refuse(f"{name} must be contiguous within a token")
    return t.data_ptr(), sn if n > 1 else heads * head_dim


def paged_append(q, k, v, positions, tables, k_pages, v_pages, *, cos=None, sin=None, seqs=None, out=None):
    """Rotary embedding of new tokens' q and k, and the write of k and v into the cache's pages.

    q          [tokens, heads, head_dim] of the pool's dtype (rows of a wider tensor will do: the
               q, k, v slices of one projection's output), or None to write the cache only
    k, v       [tokens, kv_heads, head_dim]
    positions  int32 [tokens]: each token's position in its sequence; negative for a padding token,
               which writes nothing and whose q comes back zero
    seqs       int32 [tokens]: each token's row of `tables` (default: token t is sequence t)
    cos, sin   fp32 [>= positions, head_dim] rotate-half tables (both None: no rotation)
    out        where the rotated q goes (default a new tensor; q itself will do)

    Returns out.  A position past the tables' width or the angles, a sequence outside `tables` or a
    page outside the pool writes nothing to the cache and gives NaN.  A (sequence, position) may
    occur once per call."""
    pool, kvh, _, d = _pool(k_pages, v_pages)
    dev, dtype = k_pages.device, k_pages.dtype
    if not (isinstance(k, torch.Tensor) and k.dim() == 3):
        _refuse("k must be [tokens, kv_heads, head_dim]")
    n = k.shape[0]
    kp, ks = _tokens(k, n, kvh, d, dtype, "k", dev)
    vp, vs = _tokens(v, n, kvh, d, dtype, "v", dev)
    pos = _index(positions, n, "positions", dev)
    sq = _index(seqs, n, "seqs", dev) if seqs is not None else None
    tab, _ = _tables(tables, dev)
    cp = sp = None
    angles = 0
    if cos is not None or sin is not None:
        for name, t in (("cos", cos), ("sin", sin)):
            if not (isinstance(t, torch.Tensor) and t.device == dev and t.dtype == torch.float32 and t.dim() == 2
                    and t.shape[1] == d and t.is_contiguous()):
                _refuse(f"{name} must be a contiguous fp32 [positions, {d}] tensor on {dev} (cos and sin go together)")
        angles = cos.shape[0]
        if sin.shape[0] != angles:
            _refuse("cos and sin must have the same shape")
        cp, sp = cos.data_ptr(), sin.data_ptr()
    heads, qp, qs, op, os_ = 0, None, 0, None, 0
    if q is not None:
        if not (isinstance(q, torch.Tensor) and q.dim() == 3):
            _refuse("q must be [tokens, heads, head_dim]")
        heads = q.shape[1]
        qp, qs = _tokens(q, n, heads, d, dtype, "q", dev)
        if out is None:
            out = q.new_empty(n, heads, d)  # (numbers: a tuple costs half as much again)
            op, os_ = out.data_ptr(), heads * d
        else:
            op, os_ = _tokens(out, n, heads, d, dtype, "out", dev)
    if n:
        _call("w4a16_paged_append", dev, qp, qs, kp, ks, vp, vs, pos, sq, n, heads, tab, cp, sp, angles, pool, op, os_)
    return out


def paged_attention(q, k_pages, v_pages, tables, lengths, *, seqs=None, scale=None, out=None, workspace=None):
    """Attention of one query token per row over the pages of its sequence:
    out[t, h] = softmax_j(scale * q[t, h] . K[j, g]) V[j, g] over j < lengths[t], g = h // (heads // kv_heads).

    q        [rows, heads, head_dim] of the pool's dtype (rows of a wider tensor will do)
    lengths  int32 [rows]: positions each row attends to, its own token's included
    seqs     int32 [rows]: each row's row of `tables` (default: row t is sequence t); several rows may
             name one sequence, as the tokens of a prompt do with growing lengths
    scale    a positive number up to 2^127, default head_dim ** -0.5
    workspace  a uint8 CUDA tensor of at least paged_attention_workspace_bytes(heads, kv_heads, head_dim); default:
             one allocated for a call that takes it, so calls on several streams or in several graphs do not share it

    Returns out [rows, heads, head_dim], the same bits every time for tables of the same width (those of
    few rows in short tables go a faster way).  A row of length <= 0 is zero; a length past the tables'
    width, a sequence outside `tables` or a page outside the pool gives NaN."""
    pool, kvh, page_size, d = _pool(k_pages, v_pages)
    dev, dtype = k_pages.device, k_pages.dtype
    if not (isinstance(q, torch.Tensor) and q.dim() == 3):
        _refuse("q must be [rows, heads, head_dim]")
    n, heads = q.shape[0], q.shape[1]
    qp, qs = _tokens(q, n, heads, d, dtype, "q", dev)
    if heads == 0 or kvh == 0 or heads % kvh:
        _refuse(f"{heads} query heads are not a multiple of {kvh} kv heads")
    lens = _index(lengths, n, "lengths", dev)
    sq = _index(seqs, n, "seqs", dev) if seqs is not None else None
    tab, width = _tables(tables, dev)
    if out is None:
        out = q.new_empty(n, heads, d)
        op, os_ = out.data_ptr(), heads * d
    else:
        op, os_ = _tokens(out, n, heads, d, dtype, "out", dev)
    if n == 0:
        return out
    if workspace is None:
        size = _attention_bytes(dev.index, _POOL_DTYPES[dtype], n, heads, kvh, d, width, page_size)
        workspace = q.new_empty((size + 1) // 2) if size else None
        ws = workspace.data_ptr() if size else None
    else:
        if not (isinstance(workspace, torch.Tensor) and workspace.device == dev and workspace.dtype == torch.uint8
                and workspace.is_contiguous()):
            _refuse(f"workspace must be a contiguous uint8 tensor on {dev}")
        size, ws = workspace.numel(), workspace.data_ptr()
    _call("w4a16_paged_attention", dev, qp, qs, lens, sq, n, heads, tab, pool, float(d ** -0.5 if scale is None else scale),
          op, os_, ws, size)
    return out


def paged_attention_workspace_bytes(heads, kv_heads, head_dim):
    """Bytes of a workspace for any paged_attention call of these heads.  Its content does not matter; calls that may
    run at the same time (on two streams, in two graphs) need one each."""
    if head_dim not in (64, 128, 256) or heads <= 0 or kv_heads <= 0 or heads % kv_heads:
        _refuse(f"no paged attention of {heads} query heads over {kv_heads} kv heads of {head_dim} (64, 128 or 256)")
    return _bytes("w4a16_paged_attention_workspace_bytes", heads, kv_heads, head_dim)


# ------------------------------------------------------------------------------ page bookkeeping

def _state(tables, lengths, refs, page_size):
    if not (isinstance(tables, torch.Tensor) and tables.is_cuda and tables.dtype == torch.int32 and tables.dim() == 2
            and tables.is_contiguous()):
        _refuse("tables must be a contiguous int32 [sequences, width] CUDA tensor")
    dev = tables.device
    sequences, width = tables.shape
    return _lib.pack_state(tables.data_ptr(), _index(lengths, sequences, "lengths", dev), _index(refs, None, "refs", dev), sequences,
                           width, refs.shape[0], page_size, width)


def _blocks(k_pages, v_pages):
    """The pages' bytes in all layers, checked ([layers, pages, ...] or one layer's [pages, kv_heads,
    page_size, head_dim], every page one dense block): their C description, pages."""
    if not (isinstance(k_pages, torch.Tensor) and k_pages.is_cuda and k_pages.dim() in (4, 5)):
        _refuse("k_pages must be a CUDA tensor [layers, pages, kv_heads, page_size, head_dim] or [pages, kv_heads, page_size, head_dim]")
    shape, stride = k_pages.shape, k_pages.stride()
    if not (isinstance(v_pages, torch.Tensor) and v_pages.device == k_pages.device and v_pages.dtype == k_pages.dtype
            and v_pages.shape == shape and v_pages.stride() == stride):
        _refuse("v_pages must have the device, dtype, shape and strides of k_pages")
    size = k_pages.element_size()
    layers, ls = (shape[0], stride[0]) if len(shape) == 5 else (1, 0)
    pages, ps = shape[-4], stride[-4]
    elements = shape[-1] * shape[-2] * shape[-3]
    if stride[-3:] != (shape[-2] * shape[-1], shape[-1], 1):
        block = 1
        for st, n in sorted(zip(stride[-3:], shape[-3:])):  # dense in some order of its dimensions
            if n != 1 and st != block:
                _refuse("a page must be one dense block")
            block *= n
    return _lib.pack_blocks(k_pages.data_ptr(), v_pages.data_ptr(), layers, pages, ls * size if layers > 1 else 0,
                            (ps if pages > 1 else elements) * size, elements * size), pages


def extend_sequences(tables, lengths, refs, seqs, counts, *, page_size):
    """Sequence seqs[i] grows by counts[i] positions (int32 [n], n <= 1024) and receives the lowest free
    pages that it needs for them; tables, lengths and refs are updated in place.

    Returns ok, int32 [n]: 1, or 0 for a request that was refused and changed nothing (an index or
    count out of range, more positions than the table's row holds, a sequence named by an earlier
    request of the call, or no pages left: requests are served in order, and from the first that does
    not fit on all that need pages are refused)."""
    st = _state(tables, lengths, refs, page_size)
    dev = tables.device
    s = _index(seqs, None, "seqs", dev)
    n = seqs.shape[0]
    c = _index(counts, n, "counts", dev)
    ok = torch.empty_like(seqs)
    _call("w4a16_pages_extend", dev, st, s, c, n, ok.data_ptr())
    return ok


def fork_sequences(k_pages, v_pages, tables, lengths, refs, src, dst):
    """Sequence dst[i], which must be empty, becomes a copy of src[i] (int32 [n], n <= 1024): whole
    pages are shared, a partly filled last page is copied in every layer to the lowest free page.
    k_pages, v_pages: [layers, pages, kv_heads, page_size, head_dim] (or one layer's four dimensions).

    Returns ok, int32 [n], as extend_sequences does; a dst that is not empty, is its own src or was
    named by an earlier request is refused, and so is a src whose partly filled page is outside the
    pool.  All requests see the state from before the call."""
    b, pages = _blocks(k_pages, v_pages)
    st = _state(tables, lengths, refs, k_pages.shape[-2])
    dev = tables.device
    if k_pages.device != dev or refs.shape[0] != pages:
        _refuse(f"refs must have one entry for each of the {pages} pages, and k_pages be on {dev}")
    s = _index(src, None, "src", dev)
    n = src.shape[0]
    t = _index(dst, n, "dst", dev)
    ok = torch.empty_like(src)
    need = _bytes("w4a16_pages_fork_scratch_bytes", n)
    scratch = src.new_empty((need + 3) // 4)
    _call("w4a16_pages_fork", dev, st, b, s, t, n, ok.data_ptr(), scratch.data_ptr(), need)
    return ok


def free_sequences(tables, lengths, refs, seqs):
    """Sequence seqs[i] (int32 [n]) gives up every page in its row and becomes empty; a page that no
    row holds any more is free.  Returns ok, int32 [n]: 0 for an index out of range or named before."""
    st = _state(tables, lengths, refs, 1)
    dev = tables.device
    s = _index(seqs, None, "seqs", dev)
    ok = torch.empty_like(seqs)
    _call("w4a16_pages_free", dev, st, s, seqs.shape[0], ok.data_ptr())
    return ok


def copy_pages(k_pages, v_pages, src, dst):
    """Copies page src[i] to page dst[i] in every layer (int32 [n]).  A pair with an index outside
    the pool is skipped.  No page may be in both lists, or twice in dst."""
    b, _ = _blocks(k_pages, v_pages)
    dev = k_pages.device
    s = _index(src, None, "src", dev)
    n = src.shape[0]
    _call("w4a16_pages_copy", dev, b, s, _index(dst, n, "dst", dev), n)


def compact_pages(k_pages, v_pages, tables, refs, *, inplace=True):
    """Moves the live pages (refs > 0) to the front of the pool: with L of them, the k-th live page at
    or above L goes to the k-th free page below L, and no other page moves.

    Returns (tables, refs, moved): the tables and refs with the new page numbers (updated in place, or
    new tensors with inplace=False), and the number of pages moved, int32 [1] on the device."""
    b, pages = _blocks(k_pages, v_pages)
    dev = k_pages.device
    if not (isinstance(tables, torch.Tensor) and tables.device == dev and tables.dtype == torch.int32 and tables.is_contiguous()):
        _refuse(f"tables must be a contiguous int32 tensor on {dev}")
    r = _index(refs, pages, "refs", dev)
    new_tables, new_refs = (tables, refs) if inplace else (torch.empty_like(tables), torch.empty_like(refs))
    moved = refs.new_empty(1)
    need = _bytes("w4a16_pages_compact_scratch_bytes", pages)
    scratch = refs.new_empty((need + 3) // 4)
    _call("w4a16_pages_compact", dev, b, tables.data_ptr(), new_tables.data_ptr(), tables.numel(), r, new_refs.data_ptr(),
          moved.data_ptr(), scratch.data_ptr(), need)
    return new_tables, new_refs, moved


class PagedKVCache:
    """The paged cache of a model: k and v [layers, pages, kv_heads, page_size, head_dim], and the page
    tables of `sequences` sequences of at most `max_len` positions."""

    def __init__(self, layers, pages, sequences, max_len, *, kv_heads, head_dim, page_size=16, dtype=torch.float16,
                 device="cuda"):
        if page_size < 1 or page_size & (page_size - 1):
            raise ValueError(f"page_size {page_size} is not a power of two")
        dev = torch.device(device)
        self.page_size = page_size
        self.k = torch.zeros(layers, pages, kv_heads, page_size, head_dim, dtype=dtype, device=dev)
        self.v = torch.zeros_like(self.k)
        self.tables = torch.full((sequences, -(-max_len // page_size)), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)

    def extend(self, seqs, counts):
        return extend_sequences(self.tables, self.lengths, self.refs, seqs, counts, page_size=self.page_size)

    def fork(self, src, dst):
        return fork_sequences(self.k, self.v, self.tables, self.lengths, self.refs, src, dst)

    def free(self, seqs):
        return free_sequences(self.tables, self.lengths, self.refs, seqs)

    def compact(self):
        return compact_pages(self.k, self.v, self.tables, self.refs)[2]

    def append(self, layer, q, k, v, positions, *, cos=None, sin=None, seqs=None, out=None):
        return paged_append(q, k, v, positions, self.tables, self.k[layer], self.v[layer], cos=cos, sin=sin, seqs=seqs, out=out)

    def attention(self, layer, q, lengths, *, seqs=None, scale=None, out=None):
        return paged_attention(q, self.k[layer], self.v[layer], self.tables, lengths, seqs=seqs, scale=scale, out=out)
