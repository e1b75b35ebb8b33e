"""Operators over a key-value cache in pages (include/mllmb200_lm.h): new rows into the pages, and attention of new tokens
over them.

A cache is two tensors, keys [pages, kv_heads, page, dim] and values [pages, kv_heads, page, vdim], bf16 or fp16, page a
multiple of 16, sizes multiples of 16 up to 256.  Rows are contiguous, the other strides are free (a cache laid out
[pages, page, kv_heads, dim] is passed as its transpose(1, 2)).  Position j of sequence s lies in page table[s, j // page],
row j % page; pages may lie in any order.  lengths[s] counts the tokens of a sequence with those of the call; its n rows stand
at positions lengths[s] - n and on.  table, lengths and q_start are int32 tensors on the device, and are read there: a
captured call replays with what they hold then.

Calls run on the current stream of the tensors' device, or on `stream` (the tensors must be ready there); `out` is allocated
there too.  What the device finds wrong (page numbers, lengths) is reported by `check`."""
import ctypes as C
import struct

import torch

from . import lm
from .binding import scratch

_PAGES = struct.Struct("@PP6q3P10i")
_LOOK = struct.Struct("@PP4qPP4if4x")
_DTYPES = {torch.bfloat16: lm.BF16, torch.float16: lm.F16}
_sizes = {}


def _fail(where, status):
    raise lm.EngineError(status, where, lm.STATUS.get(status))


def _on(device, stream, call):
    """call(raw stream) with the tensors' device as the current one."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return call(stream.cuda_stream)
    if device.index == torch.cuda.current_device():
        return call(torch.cuda.current_stream().cuda_stream)
    with torch.cuda.device(device):
        return call(torch.cuda.current_stream().cuda_stream)


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _pages(k, v, table, lengths, q_start, rows, where):
    kd, ks, vs = k.shape, k.stride(), v.stride()
    _need(len(kd) == 4 and v.dim() == 4 and kd[:3] == v.shape[:3], f"{where}: keys and values are [pages, kv_heads, page, size]")
    dtype = _DTYPES.get(k.dtype)
    _need(dtype is not None and v.dtype == k.dtype, f"{where}: keys and values in bf16 or fp16")
    _need(ks[3] == 1 and vs[3] == 1, f"{where}: rows of keys and values are contiguous")
    _need(table.dtype == lengths.dtype == torch.int32 and table.dim() == 2 and lengths.dim() == 1, f"{where}: table [sequences, pages] and lengths [sequences] in int32")
    seqs, width = table.shape
    _need(lengths.shape[0] == seqs and lengths.stride(0) == 1 and (width < 2 or table.stride(1) == 1), f"{where}: a length and a contiguous row of the table per sequence")
    start = 0
    if q_start is not None:
        _need(q_start.dtype == torch.int32 and q_start.dim() == 1 and q_start.shape[0] == seqs + 1 and q_start.is_contiguous(), f"{where}: q_start [sequences + 1] in int32")
        start = q_start.data_ptr()
    device = k.device
    _need(device.type == "cuda" and all(t is None or t.device == device for t in (v, table, lengths, q_start)), f"{where}: tensors on one GPU")
    return _PAGES.pack(k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], table.data_ptr(), lengths.data_ptr(), start, dtype, kd[0], kd[2],
                       kd[1], kd[3], v.shape[3], table.stride(0), width, seqs, rows)


def append(k_pages, v_pages, k, v, table, lengths, q_start=None, stream=None):
    """Rows of new keys [rows, kv_heads, dim] and values [rows, kv_heads, vdim] into their pages.  Sequence s brings the rows
    q_start[s] .. q_start[s + 1] - 1 (without q_start: as many as every other); rows behind the last sequence are not stored."""
    _need(k.dim() == 3 and v.dim() == 3 and k.dtype == v.dtype == k_pages.dtype and k.device == v.device == k_pages.device, "append: new keys and values [rows, kv_heads, size] of the cache's type")
    _need(k.shape[:2] == v.shape[:2] and (k.shape[1], k.shape[2]) == (k_pages.shape[1], k_pages.shape[3]) and v.shape[2] == v_pages.shape[3], "append: sizes of keys and values")
    _need(k.stride(2) == 1 and v.stride(2) == 1, "append: rows of keys and values are contiguous")
    pages = _pages(k_pages, v_pages, table, lengths, q_start, k.shape[0], "append")

    def call(s):
        return lm.lib().mllmb200_lm_pages_append(pages, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), s)
    st = _on(k.device, stream, call)
    if st:
        _fail("append", st)


def _attention(where, q, k_pages, v_pages, table, lengths, q_start, scale, window, keep, sink, bias, out, stream):
    _need(q.dim() == 3 and q.dtype == k_pages.dtype and q.device == k_pages.device and q.stride(2) == 1, f"{where}: queries [rows, heads, dim] of the cache's type, rows contiguous")
    rows, heads, dim = q.shape
    _need(dim == k_pages.shape[3], f"{where}: size of queries and keys")
    pages = _pages(k_pages, v_pages, table, lengths, q_start, rows, where)
    vdim, bias_max = v_pages.shape[3], 0
    if sink is not None:
        _need(sink.dtype == torch.float32 and sink.shape == (heads,) and sink.is_contiguous() and sink.device == q.device, f"{where}: sink [heads] in fp32")
    if bias is not None:
        _need(bias.dtype == torch.float32 and bias.dim() == 2 and bias.shape[0] == heads and bias.shape[1] > 0 and bias.is_contiguous() and bias.device == q.device, f"{where}: bias [heads, distances] in fp32")
        bias_max = bias.shape[1] - 1
    if out is not None:
        _need(out.shape == (rows, heads, vdim) and out.dtype == q.dtype and out.device == q.device and out.stride(2) == 1, f"{where}: out [rows, heads, vdim] of the queries' type")
    L = lm.lib()
    run, size = (L.mllmb200_lm_attn_decode, L.mllmb200_lm_attn_decode_workspace) if q_start is None else (L.mllmb200_lm_attn_prompt, L.mllmb200_lm_attn_prompt_workspace)

    def call(s):
        o = out if out is not None else torch.empty((rows, heads, vdim), dtype=q.dtype, device=q.device)
        look = _LOOK.pack(q.data_ptr(), o.data_ptr(), q.stride(0), q.stride(1), o.stride(0), o.stride(1), 0 if sink is None else sink.data_ptr(),
                          0 if bias is None else bias.data_ptr(), heads, bias_max, window, keep, dim ** -0.5 if scale is None else scale)
        key = (q_start is None, rows, heads, k_pages.shape[1], dim, vdim, table.shape)
        need = _sizes.get(key)
        if need is None:  # (a function of the sizes)
            n = C.c_size_t()
            st = size(pages, look, C.byref(n))
            if st:
                return st, o
            if len(_sizes) > 4096:
                _sizes.clear()
            need = _sizes[key] = n.value
        with scratch(need, s) as ws:
            return run(pages, look, ws, s), o
    st, o = _on(q.device, stream, call)
    if st:
        _fail(where, st)
    return o


def decode_attention(q, k_pages, v_pages, table, lengths, scale=None, window=0, keep=0, sink=None, bias=None, out=None, stream=None):
    """Attention of the newest tokens of every sequence, as many of each (at most 16; several: the tokens of a draft).  q:
    [sequences x tokens, heads, dim].  The lengths are split over the GPU.

    A token at position i sees key j if j <= i and (no window, or j > i - window, or j < keep).  Scores are scale q.k (default
    dim ** -0.5) + bias[head, min(i - j, distances - 1)]; sink: one more score per head, without a value.  A token that sees
    nothing gives zeros."""
    return _attention("decode_attention", q, k_pages, v_pages, table, lengths, None, scale, window, keep, sink, bias, out, stream)


def prompt_attention(q, k_pages, v_pages, table, lengths, q_start, scale=None, window=0, keep=0, sink=None, bias=None, out=None, stream=None):
    """The same for any number of tokens per sequence: sequence s has the rows q_start[s] .. q_start[s + 1] - 1 of q.  Rows behind
    the last sequence are left as they are in `out`."""
    _need(q_start is not None, "prompt_attention: q_start")
    return _attention("prompt_attention", q, k_pages, v_pages, table, lengths, q_start, scale, window, keep, sink, bias, out, stream)


def check(stream=None):
    """Waits for the stream; raises if a call met a page number or a length outside of its cache."""
    st = lm.lib().mllmb200_lm_operator_status((stream or torch.cuda.current_stream()).cuda_stream)
    if st:
        _fail("paged operators", st)
