"""Operators over a key-value cache in pages (include/mllmb200_lm.h): new rows into the pages, and attention of new tokens
over them.

A cache is two tensors, keys [pages, kv_heads, page, dim] and values [pages, kv_heads, page, vdim], bf16 or fp16, page a
multiple of 16, sizes multiples of 16 up to 256.  Rows are contiguous, the other strides are free (a cache laid out
[pages, page, kv_heads, dim] is passed as its transpose(1, 2)).  Position j of sequence s lies in page table[s, j // page],
row j % page; pages may lie in any order.  lengths[s] counts the tokens of a sequence with those of the call; its n rows stand
at positions lengths[s] - n and on.  table, lengths and q_start are int32 tensors on the device, and are read there: a
captured call replays with what they hold then.

Calls run on the current stream of the tensors' device, or on `stream` of that device (the tensors must be ready there); `out` is
allocated there too.  What the device finds wrong (page numbers, lengths) is reported by `check`."""
import ctypes as C
import struct

import torch

from . import lm
from .binding import _allocator

_PAGES = struct.Struct("@PP6q3P10i")
_LOOK = struct.Struct("@PP4qPP4ifi")
_DTYPES = {torch.bfloat16: lm.BF16, torch.float16: lm.F16}
_INT, _F32 = torch.int32, torch.float32
_sizes = {}  # bytes of workspace by sizes


def _fail(where, status):
    raise lm.EngineError(status, where, lm.STATUS.get(status))


def _refuse(where, *checks):
    """The first check that does not hold, as an error."""
    for ok, what in checks:
        if not ok():
            raise ValueError(f"{where}: {what}")
    raise ValueError(f"{where}: arguments")


try:  # the current device and its stream without the Python objects around them (4 us of a call that takes 10)
    _device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
except AttributeError:  # (names that torch does not promise)
    _device, _raw_stream = torch.cuda.current_device, lambda index: torch.cuda.current_stream(index).cuda_stream


def _on(index, stream, call, *tensors):
    """call(raw stream) with the tensors' device as the current one.  On a stream of the caller's the tensors' memory stays theirs until
    that stream is through, whatever becomes of the tensors meanwhile."""
    if stream is None:
        if index == _device():
            return call(_raw_stream(index))
        with torch.cuda.device(index):
            return call(_raw_stream(index))
    if stream.device.index != index:
        raise ValueError(f"a stream of {stream.device} for tensors of cuda:{index}")
    with torch.cuda.stream(stream):
        result = call(stream.cuda_stream)
    for t in tensors:
        if t is not None:
            t.record_stream(stream)
    return result


def _pages(where, k, v, table, lengths, q_start, rows):
    """(the call's mllmb200_lm_pages as bytes, sequences, kv heads, size of a key, of a value)"""
    dtype, device = _DTYPES.get(k.dtype), k.get_device()
    try:
        pages, heads, page, dim = k.shape
        v_pages, v_heads, v_rows, vdim = v.shape
        seqs, width = table.shape
        n_lengths, = lengths.shape
    except ValueError:
        _refuse(where, (lambda: k.dim() == v.dim() == 4, "keys and values are [pages, kv_heads, page, size]"), (lambda: False, "table is [sequences, pages], lengths [sequences]"))
    # (a third of the time of asking for strides)
    k_page, k_head, k_row, k_one = (heads * page * dim, page * dim, dim, 1) if k.is_contiguous() else k.stride()
    v_page, v_head, v_row, v_one = (v_heads * v_rows * vdim, v_rows * vdim, vdim, 1) if v.is_contiguous() else v.stride()
    ld_table, one = (width, 1) if table.is_contiguous() else table.stride()
    if not (dtype is not None and v.dtype == k.dtype and v_pages == pages and v_heads == heads and v_rows == page and k_one == 1 and v_one == 1 and
            table.dtype == _INT and lengths.dtype == _INT and n_lengths == seqs and lengths.is_contiguous() and (width < 2 or one == 1) and
            device >= 0 and v.get_device() == device and table.get_device() == device and lengths.get_device() == device and
            (q_start is None or (q_start.dtype == _INT and q_start.dim() == 1 and q_start.shape[0] == seqs + 1 and q_start.is_contiguous() and q_start.get_device() == device))):
        _refuse(where, (lambda: dtype is not None and v.dtype == k.dtype, "keys and values in bf16 or fp16"), (lambda: v.shape[:3] == k.shape[:3], "keys and values of the same pages"),
                (lambda: k_one == v_one == 1, "rows of keys and values are contiguous"), (lambda: table.dtype == lengths.dtype == _INT, "table and lengths in int32"),
                (lambda: n_lengths == seqs and lengths.is_contiguous() and (width < 2 or one == 1), "a length and a contiguous row of the table per sequence"),
                (lambda: q_start is None or (q_start.dtype == _INT and q_start.shape == (seqs + 1,) and q_start.is_contiguous()), "q_start [sequences + 1] in int32"),
                (lambda: False, "tensors on one GPU"))
    return _PAGES.pack(k.data_ptr(), v.data_ptr(), k_page, k_head, k_row, v_page, v_head, v_row, table.data_ptr(), lengths.data_ptr(), 0 if q_start is None else q_start.data_ptr(),
                       dtype, pages, page, heads, dim, vdim, ld_table, width, seqs, rows), seqs, heads, dim, vdim


def append(k_pages, v_pages, k, v, table, lengths, q_start=None, stream=None):
    """Rows of new keys [rows, kv_heads, dim] and values [rows, kv_heads, vdim] into their pages.  Sequence s brings the rows
    q_start[s] .. q_start[s + 1] - 1 (without q_start: as many as every other); rows behind the last sequence, and
    those whose position the table has no place for, are not stored."""
    if not (k.dim() == 3 and v.dim() == 3 and k_pages.dim() == 4 and v_pages.dim() == 4 and k.dtype == v.dtype == k_pages.dtype and k.get_device() == v.get_device() == k_pages.get_device() and
            k.shape[0] == v.shape[0] and k.shape[1] == v.shape[1] == k_pages.shape[1] and k.shape[2] == k_pages.shape[3] and v.shape[2] == v_pages.shape[3] and k.stride(2) == 1 and v.stride(2) == 1):
        _refuse("append", (lambda: k.dim() == v.dim() == 3 and k.dtype == v.dtype == k_pages.dtype and k.device == v.device == k_pages.device, "new keys and values [rows, kv_heads, size] of the cache's type"),
                (lambda: k.stride(2) == v.stride(2) == 1, "rows of keys and values are contiguous"), (lambda: False, "sizes of keys and values"))
    pages = _pages("append", k_pages, v_pages, table, lengths, q_start, k.shape[0])[0]
    st = _on(k.get_device(), stream, lambda s: lm.lib().mllmb200_lm_pages_append(pages, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), s),
             k_pages, v_pages, k, v, table, lengths, q_start)
    if st:
        _fail("append", st)


def _apart(out, q):
    """Whether every place of `out` is there once, and not where the queries lie (a block of rows may be done again from them)."""
    return out.numel() == 0 or (out.data_ptr() != q.data_ptr() and all(n < 2 or s for n, s in zip(out.shape, out.stride())))


def _attention(where, q, k_pages, v_pages, table, lengths, q_start, scale, window, keep, sink, bias, out, stream, exact):
    try:
        rows, heads, dim = q.shape
    except ValueError:
        _refuse(where, (lambda: False, "queries [rows, heads, dim]"))
    whole = q.is_contiguous()
    q_row, q_head, q_one = (heads * dim, dim, 1) if whole else q.stride()
    index = q.get_device()
    pages, seqs, kv_heads, k_dim, vdim = _pages(where, k_pages, v_pages, table, lengths, q_start, rows)
    if not (q.dtype == k_pages.dtype and index == k_pages.get_device() and q_one == 1 and dim == k_dim and
            (sink is None or (sink.dtype == _F32 and sink.shape == (heads,) and sink.is_contiguous() and sink.get_device() == index)) and
            (bias is None or (bias.dtype == _F32 and bias.dim() == 2 and bias.shape[0] == heads and bias.shape[1] > 0 and bias.is_contiguous() and bias.get_device() == index)) and
            (out is None or (out.shape == (rows, heads, vdim) and out.dtype == q.dtype and out.get_device() == index and out.stride(2) == 1 and _apart(out, q)))):
        _refuse(where, (lambda: q.dtype == k_pages.dtype and index == k_pages.get_device() and q_one == 1, "queries of the cache's type and device, rows contiguous"),
                (lambda: dim == k_dim, "size of queries and keys"), (lambda: sink is None or (sink.dtype == _F32 and sink.shape == (heads,) and sink.is_contiguous() and sink.get_device() == index), "sink [heads] in fp32"),
                (lambda: bias is None or (bias.dtype == _F32 and bias.dim() == 2 and bias.shape[0] == heads and bias.shape[1] > 0 and bias.is_contiguous() and bias.get_device() == index), "bias [heads, distances] in fp32"),
                (lambda: False, "out [rows, heads, vdim] of the queries' type, rows contiguous, every place once and not the queries' own"))
    L = lm.lib()
    decode = q_start is None
    key = (decode, rows, heads, kv_heads, dim, vdim, seqs) if decode else (rows, heads, kv_heads, dim, vdim, table.shape, k_pages.shape[2], window, keep)

    def call(s):
        o = out if out is not None else torch.empty_like(q) if vdim == dim and whole else q.new_empty((rows, heads, vdim))
        o_row, o_head = (heads * vdim, vdim) if out is None else (out.stride(0), out.stride(1))
        look = _LOOK.pack(q.data_ptr(), o.data_ptr(), q_row, q_head, o_row, o_head, 0 if sink is None else sink.data_ptr(), 0 if bias is None else bias.data_ptr(), heads,
                          0 if bias is None else bias.shape[1] - 1, window, keep, dim ** -0.5 if scale is None else scale, exact)
        need = _sizes.get(key)
        if need is None:  # (a function of the sizes)
            n = C.c_size_t()
            st = (L.mllmb200_lm_attn_decode_workspace if decode else L.mllmb200_lm_attn_prompt_workspace)(pages, look, C.byref(n))
            if st:
                return st, o
            if len(_sizes) > 4096:
                _sizes.clear()
            need = _sizes[key] = n.value
        run = L.mllmb200_lm_attn_decode if decode else L.mllmb200_lm_attn_prompt
        if not need:
            return run(pages, look, None, s), o
        take, give = _allocator()  # memory of the call, on its stream
        ws = take(need, s)
        try:
            return run(pages, look, ws, s), o
        finally:
            give(ws)
    st, o = _on(index, stream, call, q, k_pages, v_pages, table, lengths, q_start, sink, bias, out)
    if st:
        _fail(where, st)
    return o


def decode_attention(q, k_pages, v_pages, table, lengths, scale=None, window=0, keep=0, sink=None, bias=None, out=None, stream=None):
    """Attention of the newest tokens of every sequence, as many of each (at most 16; several: the tokens of a draft).  q:
    [sequences x tokens, heads, dim].  The lengths are split over the GPU.

    A token at position i sees key j if j <= i and (no window, or j > i - window, or j < keep).  Scores are scale q.k (default
    dim ** -0.5) + bias[head, min(i - j, distances - 1)]; sink: one more score per head, without a value.  A token that sees
    nothing gives zeros.  `out` must not overlap the queries."""
    return _attention("decode_attention", q, k_pages, v_pages, table, lengths, None, scale, window, keep, sink, bias, out, stream, False)


def prompt_attention(q, k_pages, v_pages, table, lengths, q_start, scale=None, window=0, keep=0, sink=None, bias=None, out=None, stream=None, exact=False):
    """The same for any number of tokens per sequence: sequence s has the rows q_start[s] .. q_start[s + 1] - 1 of q.  Rows behind
    the last sequence are left as they are in `out`.  exact: softmax weights meet the values as two numbers of 16 bits, as in
    decode_attention; without it heads of 64 and 128 round them to one, which errs about as much as the outputs' own rounding and
    is faster."""
    if q_start is None:
        raise ValueError("prompt_attention: q_start")
    return _attention("prompt_attention", q, k_pages, v_pages, table, lengths, q_start, scale, window, keep, sink, bias, out, stream, bool(exact))


def check(stream=None):
    """Waits for the stream; raises if a call on its device met a page number or a length outside of its cache."""
    stream = stream or torch.cuda.current_stream()
    with torch.cuda.device(stream.device):
        st = lm.lib().mllmb200_lm_operator_status(stream.cuda_stream)
    if st:
        _fail("paged operators", st)
