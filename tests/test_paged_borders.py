"""Operators over pages at their borders: lengths beyond a table, tensors of other streams, odd arguments."""
import numpy as np
import pytest
import torch

from mllm_b200 import lm, paged
from paged_case import Cache

BF16 = torch.bfloat16


def rand(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("beyond, count", [(1, 1), (1, 3), (5, 3), (2 ** 31 - 1 - 64, 2)])
@pytest.mark.parametrize("ragged", [False, True])
def test_rows_beyond_a_full_table_are_not_stored(beyond, count, ragged):
    """Every place of the table names a page, and a length goes beyond them: rows with a place are stored there, the others nowhere."""
    c = Cache([64, 33], 2, 64, 64, 16, BF16, 3, wide=0)
    c.table_h[1, 3] = c.table_h[1, 2]  # (no number of no page anywhere)
    new = rand((2 * count, 2, 64), BF16, 4)
    want = c.k.clone(), c.v.clone()
    for s, n in enumerate((64 + beyond, 33)):
        for t in range(count):
            j = n - count + t
            if j < 64:
                for pool in want:
                    pool[c.table_h[s, j // 16], :, j % 16] = new[s * count + t]
    c.on_gpu()
    lengths = torch.tensor([64 + beyond, 33], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, count, 2 * count], dtype=torch.int32, device="cuda") if ragged else None
    paged.append(c.k, c.v, new.cuda(), new.cuda(), c.table, lengths, start)
    with pytest.raises(lm.EngineError) as e:
        paged.check()
    assert e.value.status == 7
    for got, w in zip((c.k, c.v), want):
        assert torch.equal(torch.nan_to_num(got.cpu().float(), 11.0), torch.nan_to_num(w.float(), 11.0))
