"""How exactly the softmax weights of attention over pages enter the product with the values."""
import os
import re
import types

import numpy as np
import pytest
import torch

import lm_case
import lm_models as M
from mllm_b200 import paged, registry
from paged_case import HALF_STEP, Cache, attention64, check

BF16, FP16 = torch.bfloat16, torch.float16


def rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def starts(counts):
    return torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("heads, kv, dim, page", [(14, 2, 64, 16), (12, 2, 128, 48), (4, 4, 80, 32)])
@pytest.mark.parametrize("lengths, counts, window, keep, rel", [([300], [300], 0, 0, False), ([129, 64, 2100], [129, 30, 9], 0, 0, True), ([500, 77], [200, 77], 150, 4, False)])
def test_exact_weights_of_prompts(dtype, heads, kv, dim, page, lengths, counts, window, keep, rel):
    """Two halves of 16 bits carry a weight: nothing but the output's own rounding is of 16 bits (the bound without the term of
    weights in 16 bits)."""
    c = Cache(lengths, kv, dim, dim, page, dtype, dim + heads)
    q = rand((sum(counts), heads, dim), dtype, 1)
    sink, bias = (rand((heads,), torch.float32, 2), rand((heads, 40), torch.float32, 3)) if rel else (None, None)
    want = attention64(c, counts, q, None, window, keep, sink, bias)
    c.on_gpu()
    cuda = lambda t: None if t is None else t.cuda()
    got = paged.prompt_attention(q.cuda(), c.k, c.v, c.table, c.lengths, starts(counts), window=window, keep=keep, sink=cuda(sink), bias=cuda(bias), exact=True)
    paged.check()
    check(got, *want, dim, dtype, False)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_engine_prefill_on_pages_is_as_exact_as_on_slots(dim, tmp_path):
    """One layer of attention, 600 tokens, residual stream over pages and over slots.  Both carry a weight by two bf16 numbers: each off by
    2^-19 of it (rms), so is the sum over keys whose values have both signs, and a sum that lies 2^-19 elsewhere is rounded to the
    neighbouring bf16 number, 2^-7.5 away, once in 2^11.5 times: 2^-13.3 of the norm.  With weights of one number, off by
    2^-10.3, it would be 2^-8.9.  The bound lies between the two."""
    cfg = M.config(128, 200, [M.layer("attention", M.attention(6, 2, dim, dim, 37))], taps=0)
    folder, got = M.write(tmp_path, cfg, M.weights(cfg, 7)), []
    tokens = np.random.default_rng(1).integers(0, 200, 600).tolist()
    for page, pages in ((0, 0), (16, 64)):
        case = types.SimpleNamespace(model=registry.load(folder, "bfloat16", 2, 1024, 1024, page, pages)[0])
        got.append(lm_case.residual_after(case, tokens))
        case.model.close()
    assert np.linalg.norm(got[1] - got[0]) <= 2.0 ** -11 * np.linalg.norm(got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 80])
@pytest.mark.parametrize("top, late", [(18.0, False), (14.0, True)])
@pytest.mark.parametrize("value", [0.0, 1.0])
def test_many_small_weights_beside_a_large_one(dtype, dim, top, late, value):
    """A key whose score lies 14 or 18 above those of 65535 others: their weights, near 2^-20 and 2^-26 of its, sum up to what fp16 must not
    lose.  In fp16 a weight in two numbers is off by 2^-37 of the reference at most, whose own weight is at least 1 in the sum."""
    n = 65536
    c = Cache([64], 1, dim, dim, 64, dtype, 1)  # (its values are made anew below)
    c.lengths_h, pages = [n], n // 64
    c.keys, c.values = [torch.zeros(n, 1, dim, dtype=dtype)], [torch.ones(n, 1, dim, dtype=dtype)]
    at = n - 40 if late else 0
    c.keys[0][at, 0, 0], c.values[0][at] = top, value
    order = np.random.default_rng(2).permutation(pages)
    c.table_h, c.pages = np.ascontiguousarray(order[None].astype(np.int32)), pages
    c.k, c.v = (torch.empty(pages, 1, 64, dim, dtype=dtype) for _ in range(2))
    for pool, flat in ((c.k, c.keys[0]), (c.v, c.values[0])):
        pool[torch.from_numpy(order)] = flat.view(pages, 64, 1, dim).transpose(1, 2)
    q = torch.zeros(3, 2, dim, dtype=dtype)
    q[:, :, 0] = 1.0
    want, spread, big = attention64(c, [3], q, 1.0)
    c.on_gpu()
    start = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    for got, one in ((paged.decode_attention(q.cuda(), c.k, c.v, c.table, c.lengths, scale=1.0), False),
                     (paged.prompt_attention(q.cuda(), c.k, c.v, c.table, c.lengths, start, scale=1.0), True),
                     (paged.prompt_attention(q.cuda(), c.k, c.v, c.table, c.lengths, start, scale=1.0, exact=True), False)):
        half = HALF_STEP[dtype]
        bound = half * want.abs() * 1.01 + spread * ((half if one else 0.0) + 2.0 ** -16 + 2 * (dim / 16 + 4) * 2.0 ** -23 * big) + \
            (n * 2.0 ** -37 if dtype == FP16 else 0.0)
        off = (got.cpu().double() - want).abs()
        assert (off <= bound).all(), (float(off.max()), float(bound.min()), float(want.min()))
    paged.check()


LOWEST = torch.finfo(torch.float32).min


@pytest.mark.gpu
@pytest.mark.parametrize("dim, dtype", [(64, BF16), (128, FP16), (80, BF16)])
@pytest.mark.parametrize("distances", [40, 3001])
@pytest.mark.parametrize("sink", [None, 0.5, LOWEST])
def test_biases_of_the_lowest_value(dim, dtype, distances, sink):
    """Distance biases that say "as good as unseen" by the type's lowest number: all of them (a row shares its weight out evenly), the
    near ones (short rows have nothing else), the far ones.  Lowest plus a score is lowest again, in 32 bits and in 64."""
    lengths, counts, heads = [700, 9, 300, 4], [150, 9, 2, 4], 8
    c = Cache(lengths, 2, dim, dim, 32, dtype, 6)
    bias = rand((heads, distances), torch.float32, 7)
    bias[0::4] = LOWEST
    bias[1::4, :20] = LOWEST
    bias[2::4, 20:] = LOWEST
    sinks = None if sink is None else torch.full((heads,), sink)
    start, cuda = starts(counts), lambda t: None if t is None else t.cuda()
    q = rand((sum(counts), heads, dim), dtype, 8)
    want = attention64(c, counts, q, None, 0, 0, sinks, bias)
    few = rand((12, heads, dim), dtype, 9)
    want_few = attention64(c, [3] * 4, few, None, 0, 0, sinks, bias)
    c.on_gpu()
    look = dict(sink=cuda(sinks), bias=bias.cuda())
    check(paged.prompt_attention(q.cuda(), c.k, c.v, c.table, c.lengths, start, **look), *want, dim, dtype, True)
    check(paged.decode_attention(few.cuda(), c.k, c.v, c.table, c.lengths, **look), *want_few, dim, dtype, False)
    paged.check()


def test_polynomial_of_the_exponential():
    """The exponential that every fourth pair of weights takes (pair_exp2 of lm_paged_tc.cu, its constants read from there), in fp32 as the
    kernel computes it: off by 2^-18 of the result at most, 0 below 2^-126."""
    source = open(os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "mllm-advanced_b200", "csrc", "lm", "lm_paged_tc.cu")).read()
    body = source[source.index("float2 pair_exp2("):source.index("// weights 2^(score scale + base)")]
    c = [np.float32(x) for x in re.findall(r"pair_of\((0\.\d+)f, \1f\)", body)]
    big = np.float32(re.search(r"pair_of\((\d+\.0)f", body).group(1))
    assert len(c) == 5 and big == np.float32(1.5 * 2 ** 23 + 127)
    fma = lambda a, b, d: (a.astype(np.float64) * np.float64(b) + np.float64(d)).astype(np.float32)  # (a product of two is exact in 64 bits)
    mul = lambda a, b: a.astype(np.float64) * b.astype(np.float64)
    x = np.concatenate([np.linspace(-126, 16, 2_000_003), np.linspace(-2, 2, 500_001)]).astype(np.float32)
    t = x + big
    f = x - (t - big)
    p = fma(f, c[0], c[1])
    for k in c[2:]:
        p = (mul(p, f) + np.float64(k)).astype(np.float32)
    got = mul(p, (t.view(np.uint32) << 23).view(np.float32))
    want = np.exp2(x.astype(np.float64))
    assert np.abs(got / want - 1).max() <= 2.0 ** -18
    t = np.float32(-127) + big
    assert (np.array([t]).view(np.uint32) << 23).view(np.float32)[0] == 0
