"""Operators over a key-value cache in pages: storing rows, attention of a few tokens per sequence, attention of prompts,
against their definition in 64 bits."""
import ctypes as C

import numpy as np
import pytest
import torch

from mllm_b200 import lm, paged
from paged_case import Cache, attention64, check

BF16, FP16 = torch.bfloat16, torch.float16


# ------------------------------------------------------------------------------------------------ refusals, on the CPU
class Pages(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p)] + [(n, C.c_longlong) for n in ("k_page", "k_head", "k_row", "v_page", "v_head", "v_row")] + \
               [(n, C.c_void_p) for n in ("table", "lengths", "q_start")] + \
               [(n, C.c_int) for n in ("dtype", "pages", "page", "kv_heads", "dim", "vdim", "ld_table", "max_pages", "seqs", "rows")]


class Look(C.Structure):
    _fields_ = [("q", C.c_void_p), ("out", C.c_void_p)] + [(n, C.c_longlong) for n in ("q_row", "q_head", "out_row", "out_head")] + \
               [("sink", C.c_void_p), ("bias", C.c_void_p)] + [(n, C.c_int) for n in ("heads", "bias_max", "window", "keep")] + [("scale", C.c_float)]


def good():
    p = Pages(4096, 4096, 2048, 1024, 64, 2048, 1024, 64, 4096, 4096, None, lm.BF16, 8, 16, 2, 64, 64, 4, 4, 3, 3)
    return p, Look(4096, 4096, 256, 64, 256, 64, None, None, 4, 0, 0, 0, 0.125)


def test_layout_of_the_structures():
    assert C.sizeof(Pages) == paged._PAGES.size and C.sizeof(Look) == paged._LOOK.size


@pytest.mark.parametrize("change, status", [
    (dict(dtype=lm.F32), 2), (dict(page=8), 2), (dict(page=24), 2), (dict(dim=72), 2), (dict(dim=272), 2), (dict(vdim=0), 1), (dict(pages=0), 1), (dict(k=None), 1),
    (dict(k=4104), 1), (dict(k_row=66), 1), (dict(v_page=1), 1), (dict(lengths=None), 1), (dict(table=None), 1), (dict(rows=4), 1), (dict(seqs=-1), 1),
    (dict(max_pages=2 ** 27), 2), (dict(kv_heads=3), 1), (dict(rows=51), 2), (dict(heads=0), 1), (dict(heads=5), 1), (dict(heads=256), 2), (dict(window=-1), 1),
    (dict(keep=-1), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1), (dict(bias=4096, bias_max=-1), 1), (dict(q=None), 1), (dict(q=4098), 1), (dict(q_head=4), 1),
    (dict(out_row=2), 1)])
def test_refusals(change, status):
    p, look = good()
    for name, value in change.items():
        setattr(p if hasattr(p, name) else look, name, value)
    L, size = lm.lib(), C.c_size_t()
    as_bytes = lambda: (bytes(p), bytes(look))
    assert L.mllmb200_lm_attn_decode_workspace(*as_bytes(), C.byref(size)) == status
    assert L.mllmb200_lm_attn_decode(*as_bytes(), 4096, None) == status
    if "rows" not in change or status == 1:
        assert L.mllmb200_lm_attn_prompt(*as_bytes(), 4096, None) == status


def test_refusals_of_calls():
    p, look = good()
    L, size = lm.lib(), C.c_size_t()
    assert L.mllmb200_lm_attn_decode_workspace(bytes(p), bytes(look), C.byref(size)) == 0 and size.value > 0
    assert L.mllmb200_lm_attn_decode_workspace(None, bytes(look), C.byref(size)) == 1
    assert L.mllmb200_lm_attn_decode_workspace(bytes(p), None, C.byref(size)) == 1
    assert L.mllmb200_lm_attn_decode(bytes(p), bytes(look), None, None) == 1
    assert L.mllmb200_lm_attn_decode(bytes(p), bytes(look), 4100, None) == 1
    assert L.mllmb200_lm_pages_append(bytes(p), None, 128, 64, 4096, 128, 64, None) == 1
    assert L.mllmb200_lm_pages_append(bytes(p), 4096, 129, 64, 4096, 128, 64, None) == 1
    p.q_start = 4096
    assert L.mllmb200_lm_attn_decode(bytes(p), bytes(look), 4096, None) == 1
    p.q_start, p.rows = None, 0  # nothing to do
    assert L.mllmb200_lm_attn_decode(bytes(p), bytes(look), 4096, None) == 0
    assert L.mllmb200_lm_attn_prompt(bytes(p), bytes(look), 4096, None) == 0
    assert L.mllmb200_lm_pages_append(bytes(p), 4096, 128, 64, 4096, 128, 64, None) == 0
    p.seqs = 0
    assert L.mllmb200_lm_attn_decode(bytes(p), bytes(look), 4096, None) == 0


def test_python_refusals():
    k = torch.zeros(4, 2, 16, 64, dtype=BF16)
    q, table, lengths = torch.zeros(3, 4, 64, dtype=BF16), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    for args in ((q, k, k, table, lengths), (q.float(), k, k, table, lengths), (q, k, k.half(), table, lengths), (q, k, k, table.long(), lengths), (q, k, k, table, lengths[:2]),
                 (q[:, :, :48], k, k, table, lengths), (q, k, k[:3], table, lengths), (q, k.transpose(2, 3), k, table, lengths)):
        with pytest.raises(ValueError):
            paged.decode_attention(*args)
    with pytest.raises(ValueError):
        paged.prompt_attention(q, k, k, table, lengths, None)
    with pytest.raises(ValueError):
        paged.append(k, k, q, q, table, lengths)


# ------------------------------------------------------------------------------------------------ decode
def rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def run_decode(lengths, tokens, heads, kv, dim, vdim, page, dtype, window=0, keep=0, rel=False, layout="head", seed=0):
    c = Cache(lengths, kv, dim, vdim, page, dtype, seed, layout)
    q = rand((len(lengths) * tokens, heads, dim), dtype, seed + 1)
    sink, bias = (rand((heads,), torch.float32, seed + 2), rand((heads, 40), torch.float32, seed + 3)) if rel else (None, None)
    want = attention64(c, [tokens] * len(lengths), q, None, window, keep, sink, bias)
    c.on_gpu()
    cuda = lambda t: None if t is None else t.cuda()
    got = paged.decode_attention(q.cuda(), c.k, c.v, c.table, c.lengths, window=window, keep=keep, sink=cuda(sink), bias=cuda(bias))
    paged.check()
    check(got, *want, dim, dtype, False)
    return c, q, got


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[1], [2, 0, 16], [15, 16, 17, 31, 33], [127, 128, 129, 500], [3000]])
@pytest.mark.parametrize("heads, kv, dim, vdim, page", [(14, 2, 64, 64, 16), (12, 2, 128, 128, 48), (4, 4, 32, 96, 32), (3, 1, 256, 256, 16), (6, 1, 256, 64, 16)])
def test_decode_lengths(lengths, heads, kv, dim, vdim, page):
    run_decode(lengths, 1, heads, kv, dim, vdim, page, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens", [1, 2, 5, 16])
@pytest.mark.parametrize("window, keep", [(0, 0), (1, 0), (7, 3), (64, 17), (200, 400)])
@pytest.mark.parametrize("rel", [False, True])
def test_decode_masks(dtype, tokens, window, keep, rel):
    run_decode([700, 1, 0, tokens, 90, 65, 130], tokens, 8, 2, 64, 128, 32, dtype, window, keep, rel, seed=tokens)


@pytest.mark.gpu
def test_decode_many_heads_and_layouts():
    run_decode([40, 300], 1, 64, 1, 64, 64, 16, BF16)
    run_decode([40, 300], 3, 40, 2, 16, 16, 16, BF16)
    run_decode([5, 1000, 64], 4, 12, 4, 128, 128, 64, FP16, 33, 2, True, layout="token")
    run_decode([5, 1000, 64], 1, 12, 4, 48, 80, 16, BF16, layout="token")


@pytest.mark.gpu
def test_decode_many_sequences():
    """More than one launch takes (512), and lengths of nothing among them."""
    lengths = np.random.default_rng(1).integers(0, 60, 1100).tolist()
    run_decode(lengths, 1, 2, 1, 16, 16, 16, BF16)


@pytest.mark.gpu
def test_decode_many_sequences_in_blocks_of_rows():
    """Launches of 512 sequences, and more rows of a key head than a block holds (24 heads x 3 tokens)."""
    lengths = np.random.default_rng(2).integers(0, 40, 530).tolist()
    run_decode(lengths, 3, 24, 1, 64, 64, 16, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-35, 0.5])
@pytest.mark.parametrize("tokens", [1, 3])
def test_scales(scale, tokens):
    c = Cache([300, 5, 130], 2, 64, 64, 16, BF16, 4)
    q = rand((3 * tokens, 6, 64), BF16, 5)
    want = attention64(c, [tokens] * 3, q, scale)
    c.on_gpu()
    start = torch.arange(4, dtype=torch.int32, device="cuda") * tokens
    check(paged.decode_attention(q.cuda(), c.k, c.v, c.table, c.lengths, scale=scale), *want, 64, BF16, False)
    check(paged.prompt_attention(q.cuda(), c.k, c.v, c.table, c.lengths, start, scale=scale), *want, 64, BF16, True)


@pytest.mark.gpu
def test_strides_of_dimensions_of_one():
    """A single key head, a single row, a single head: their strides say nothing and may be anything."""
    c = Cache([40], 1, 64, 64, 16, BF16, 4)
    q = rand((1, 1, 64), BF16, 5)
    want = attention64(c, [1], q)
    c.on_gpu()
    odd = lambda t, *strides: torch.as_strided(t, t.shape, strides)
    k, v = odd(c.k, 16 * 64, 3, 64, 1), odd(c.v, 16 * 64, 5, 64, 1)
    qd = odd(q.cuda(), 7, 9, 1)
    start = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    check(paged.decode_attention(qd, k, v, c.table, c.lengths), *want, 64, BF16, False)
    check(paged.prompt_attention(qd, k, v, c.table, c.lengths, start), *want, 64, BF16, True)
    before = c.k.clone()
    paged.append(k, v, odd(q.cuda(), 3, 11, 1), odd(q.cuda(), 3, 11, 1), c.table, c.lengths)
    at = c.table_h[0, 39 // 16]
    assert torch.equal(c.k[at, 0, 39 % 16].cpu(), q[0, 0])
    before[at, 0, 39 % 16] = q[0, 0].cuda()
    assert torch.equal(torch.nan_to_num(c.k.float(), 9.0), torch.nan_to_num(before.float(), 9.0))
    # queries shared by all heads (a stride of 0)
    c = Cache([40, 70], 2, 64, 64, 16, BF16, 6)
    q = rand((2, 1, 64), BF16, 7)
    want = attention64(c, [1, 1], q.expand(2, 4, 64))
    c.on_gpu()
    check(paged.decode_attention(q.cuda().expand(2, 4, 64), c.k, c.v, c.table, c.lengths), *want, 64, BF16, False)


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls that run beside one another, each with scratch of its own."""
    c = Cache([900, 2000, 77], 2, 128, 128, 16, BF16, 8)
    q = rand((2, 3, 12, 128), BF16, 9).cuda()
    c.on_gpu()
    start = torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda")
    calls = [lambda x, s: paged.decode_attention(x, c.k, c.v, c.table, c.lengths, stream=s), lambda x, s: paged.prompt_attention(x, c.k, c.v, c.table, c.lengths, start, stream=s)]
    want = [call(x, None) for call, x in zip(calls, q)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[call(x, s) for call, x, s in zip(calls, q, streams)] for _ in range(20)]
    torch.cuda.synchronize()
    for pair in got:
        assert torch.equal(pair[0], want[0]) and torch.equal(pair[1], want[1])


@pytest.mark.gpu
def test_decode_same_bits_and_strides():
    """A sequence's result does not depend on how often it is computed; views of larger tensors give the same bits."""
    c, q, got = run_decode([900, 30, 411], 2, 8, 2, 128, 128, 16, BF16, 100, 5)
    again = paged.decode_attention(q.cuda(), c.k, c.v, c.table, c.lengths, window=100, keep=5)
    assert torch.equal(got, again)
    big_q, big_out = torch.randn(6, 10, 144, device="cuda").to(BF16), torch.full((8, 9, 256), 3.0, dtype=BF16, device="cuda")
    big_q[:, 1:9, 8:136] = q.cuda()
    table = torch.full((3, c.table.shape[1] + 3), 5, dtype=torch.int32, device="cuda")
    table[:, :c.table.shape[1]] = c.table
    out = paged.decode_attention(big_q[:, 1:9, 8:136], c.k, c.v, table[:, :c.table.shape[1]], c.lengths, window=100, keep=5, out=big_out[1:7, :8, 64:192])
    assert out.data_ptr() == big_out[1:7, :8, 64:192].data_ptr() and torch.equal(out, got)
    big_out[1:7, :8, 64:192] = 3.0
    assert (big_out == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("early, clean", [(146, []), (145, [1])])
def test_values_of_unseen_keys(prompt, early, clean):
    """Infinities and NaN in keys and values that only some tokens see reach those tokens alone."""
    lengths, tokens = [200, 70], 6
    c = Cache(lengths, 2, 64, 64, 16, BF16, 3)
    q = rand((12, 4, 64), BF16, 4)
    want, spread, big = attention64(c, [tokens] * 2, q, None, 50, 2)
    # of sequence 0 (positions 194 .. 199, window 50), key 196 is seen by tokens 2 .. 5, key 146 by tokens 0 and 1, key 145 by token 0
    for j, what in ((196, float("nan")), (early, float("inf"))):
        for t in (c.k, c.v):
            t[c.table_h[0, j // 16], :, j % 16] = what
    c.on_gpu()
    if prompt:
        start = torch.tensor([0, 6, 12], dtype=torch.int32, device="cuda")
        got = paged.prompt_attention(q.cuda(), c.k, c.v, c.table, c.lengths, start, window=50, keep=2)
    else:
        got = paged.decode_attention(q.cuda(), c.k, c.v, c.table, c.lengths, window=50, keep=2)
    hit = [t for t in range(6) if t not in clean]
    clean = clean + list(range(6, 12))
    check(got[clean], want[clean], spread[clean], big, 64, BF16, prompt)
    assert not torch.isfinite(got[hit].float()).any()


# ------------------------------------------------------------------------------------------------ prompts
def run_prompt(lengths, counts, heads, kv, dim, vdim, page, dtype, window=0, keep=0, rel=False, layout="head", seed=0, spare=2):
    c = Cache(lengths, kv, dim, vdim, page, dtype, seed, layout)
    q = rand((sum(counts) + spare, heads, dim), dtype, seed + 1)
    sink, bias = (rand((heads,), torch.float32, seed + 2), rand((heads, 40), torch.float32, seed + 3)) if rel else (None, None)
    n = sum(counts)
    want = attention64(c, counts, q[:n], None, window, keep, sink, bias)
    c.on_gpu()
    cuda = lambda t: None if t is None else t.cuda()
    start = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    out = torch.full((n + spare, heads, vdim), 7.0, dtype=dtype, device="cuda")
    got = paged.prompt_attention(q.cuda(), c.k, c.v, c.table, c.lengths, start, window=window, keep=keep, sink=cuda(sink), bias=cuda(bias), out=out)
    paged.check()
    assert (got[n:] == 7.0).all()  # rows behind the last sequence
    check(got[:n], *want, dim, dtype, True)
    return c, q, start, got


@pytest.mark.gpu
@pytest.mark.parametrize("lengths, counts", [([1], [1]), ([40], [40]), ([3, 0, 200], [3, 0, 1]), ([129, 64, 65], [129, 30, 65]), ([500, 77], [33, 77]), ([300], [300])])
@pytest.mark.parametrize("heads, kv, dim, vdim, page", [(14, 2, 64, 64, 16), (12, 2, 128, 128, 48), (4, 4, 32, 96, 32), (3, 1, 256, 256, 16), (8, 2, 128, 64, 64)])
def test_prompt_lengths(lengths, counts, heads, kv, dim, vdim, page):
    run_prompt(lengths, counts, heads, kv, dim, vdim, page, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("window, keep", [(0, 0), (1, 0), (7, 3), (64, 17), (150, 400), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("rel", [False, True])
def test_prompt_masks(dtype, dim, window, keep, rel):
    run_prompt([400, 1, 0, 90, 66], [150, 1, 0, 2, 66], 8, 2, dim, dim, 32, dtype, window, keep, rel, seed=dim)


@pytest.mark.gpu
def test_prompt_positions_before_the_start():
    """More rows than a sequence is long: those at negative positions see nothing."""
    c, q, start, got = run_prompt([3, 20], [9, 20], 4, 2, 64, 64, 16, BF16)
    assert (got[:6] == 0).all()
    run_prompt([3, 20], [9, 20], 4, 2, 64, 64, 16, BF16, 4, 1, True)
    run_prompt([3, 20], [9, 20], 4, 2, 64, 64, 16, BF16, 2 ** 31 - 1, 0, True)
    run_decode([2, 0, 5], 4, 4, 2, 64, 64, 16, BF16, rel=True)


@pytest.mark.gpu
def test_prompt_many_heads_layouts_sequences():
    run_prompt([40, 90], [40, 3], 64, 1, 64, 64, 16, BF16)
    run_prompt([5, 300, 64], [5, 100, 64], 12, 4, 128, 128, 64, FP16, 33, 2, True, layout="token")
    counts = np.random.default_rng(1).integers(0, 5, 700).tolist()
    run_prompt([n + i % 30 for i, n in enumerate(counts)], counts, 2, 1, 64, 64, 16, BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths, counts", [([3000], [9]), ([2100, 4, 0, 1300], [30, 4, 0, 1]), ([700, 3, 1500], [5, 7, 40])])
@pytest.mark.parametrize("heads, kv, dim, page", [(12, 2, 128, 48), (14, 2, 64, 16), (4, 4, 128, 64)])
@pytest.mark.parametrize("window, keep, rel", [(0, 0, False), (1100, 3, True)])
def test_prompt_few_rows_of_long_contexts(lengths, counts, heads, kv, dim, page, window, keep, rel):
    """The lengths are split and joined."""
    run_prompt(lengths, counts, heads, kv, dim, dim, page, BF16, window, keep, rel, seed=heads)


@pytest.mark.gpu
def test_prompt_values_of_unseen_keys_where_lengths_are_split():
    c = Cache([2000, 900], 2, 64, 64, 16, BF16, 3)
    q = rand((12, 4, 64), BF16, 4)
    want, spread, big = attention64(c, [6, 6], q)
    for t in (c.k, c.v):
        t[c.table_h[0, 1996 // 16], :, 1996 % 16] = float("nan")  # seen by the tokens at 1996 .. 1999 of sequence 0
    c.on_gpu()
    start = torch.tensor([0, 6, 12], dtype=torch.int32, device="cuda")
    got = paged.prompt_attention(q.cuda(), c.k, c.v, c.table, c.lengths, start)
    clean = [0, 1] + list(range(6, 12))
    check(got[clean], want[clean], spread[clean], big, 64, BF16, True)
    assert not torch.isfinite(got[2:6].float()).any()


# ------------------------------------------------------------------------------------------------ append, and a run of them together
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lengths, counts", [([1], [1]), ([40, 0, 17, 130], [40, 0, 2, 100]), ([3, 20], [9, 1])])
@pytest.mark.parametrize("layout", ["head", "token"])
def test_append(dtype, lengths, counts, layout):
    c = Cache(lengths, 3, 32, 48, 16, dtype, 5, layout)
    rows = sum(counts) + 2
    nk, nv = rand((rows, 3, 40), dtype, 6)[:, :, 8:], rand((rows, 3, 48), dtype, 7)
    want_k, want_v, row = c.k.clone(), c.v.clone(), 0
    for s, (n, count) in enumerate(zip(lengths, counts)):
        for t in range(count):
            j = n - count + t
            if j >= 0:
                want_k[c.table_h[s, j // 16], :, j % 16] = nk[row + t]
                want_v[c.table_h[s, j // 16], :, j % 16] = nv[row + t]
        row += count
    c.on_gpu()
    start = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")
    paged.append(c.k, c.v, nk.cuda(), nv.cuda(), c.table, c.lengths, start)
    paged.check()
    for got, want in ((c.k, want_k), (c.v, want_v)):
        assert torch.equal(torch.nan_to_num(got.cpu().float(), 11.0), torch.nan_to_num(want.float(), 11.0))


@pytest.mark.gpu
def test_bad_pages_and_lengths_are_reported():
    """Numbers of no page are not followed; the other sequences are right."""
    c = Cache([50, 50], 2, 64, 64, 16, BF16, 8)
    q = rand((2, 4, 64), BF16, 9)
    want, spread, big = attention64(c, [1, 1], q)
    c.table_h[0, 1] = c.pages
    c.on_gpu()
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for call in (lambda: paged.decode_attention(q.cuda(), c.k, c.v, c.table, c.lengths), lambda: paged.prompt_attention(q.cuda(), c.k, c.v, c.table, c.lengths, start)):
        got = call()
        with pytest.raises(lm.EngineError):
            paged.check()
        paged.check()  # reported once
        check(got[1:], want[1:], spread[1:], big, 64, BF16, True)
    c.table[0, 1], c.lengths[0] = c.table[0, 0], 10 ** 9
    before = c.k.clone()
    paged.append(c.k, c.v, rand((2, 2, 64), BF16, 1).cuda(), rand((2, 2, 64), BF16, 2).cuda(), c.table, torch.tensor([-5, 10 ** 9], dtype=torch.int32, device="cuda"))
    with pytest.raises(lm.EngineError):
        paged.check()
    assert torch.equal(torch.nan_to_num(before.float(), 11.0), torch.nan_to_num(c.k.float(), 11.0))


@pytest.mark.gpu
def test_graph_replays_read_tables_again():
    """A captured step (append, decode) follows the lengths and pages of its replays; so does another graph beside it."""
    c = Cache([70, 31], 2, 64, 64, 16, BF16, 10)
    q, nk, nv = rand((2, 4, 64), BF16, 11).cuda(), rand((2, 2, 64), BF16, 12).cuda(), rand((2, 2, 64), BF16, 13).cuda()
    keys, values = [t.clone() for t in c.keys], [t.clone() for t in c.values]
    c.on_gpu()
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")

    def step():
        paged.append(c.k, c.v, nk, nv, c.table, c.lengths)
        return paged.decode_attention(q, c.k, c.v, c.table, c.lengths), paged.prompt_attention(q, c.k, c.v, c.table, c.lengths, start)
    step()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for length in (70, 60, 33, 5):
        c.lengths_h = [length, max(1, length - 40)]
        c.lengths.copy_(torch.tensor(c.lengths_h, dtype=torch.int32))
        for s, n in enumerate(c.lengths_h):
            keys[s][n - 1], values[s][n - 1] = nk[s].cpu(), nv[s].cpu()
        c.keys, c.values = [t[:n] for t, n in zip(keys, c.lengths_h)], [t[:n] for t, n in zip(values, c.lengths_h)]
        want = attention64(c, [1, 1], q.cpu())
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in outs:
            check(a, *want, 64, BF16, False)
            check(b, *want, 64, BF16, True)


@pytest.mark.gpu
def test_streams():
    """On a stream of the caller's, behind what runs there."""
    c = Cache([300, 40], 2, 128, 128, 16, BF16, 14)
    q = rand((2, 4, 128), BF16, 15)
    want = attention64(c, [1, 1], q)
    c.on_gpu()
    qd, side = torch.zeros_like(q, device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        qd.copy_(q)
    got = paged.decode_attention(qd, c.k, c.v, c.table, c.lengths, stream=side)
    side.synchronize()
    check(got, *want, 128, BF16, False)
