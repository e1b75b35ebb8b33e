"""How exactly the softmax weights of attention over pages enter the product with the values."""
import types

import numpy as np
import pytest
import torch

import lm_case
import lm_models as M
from mllm_b200 import paged, registry
from paged_case import Cache, attention64, check

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
