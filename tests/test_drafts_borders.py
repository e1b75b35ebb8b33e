"""Logits to probabilities and verification where a call can go wrong: barriers of clusters behind work of single lanes, rows in memory of
another form, sizes at the limits."""
import numpy as np
import pytest
import torch

from mllm_b200 import drafts
from test_drafts import rows, run_verify, softmax64


@pytest.mark.gpu
@pytest.mark.parametrize("seqs, k, vocab, odd", [(3, 33, 4099, False), (1, 64, 300001, True), (40, 1, 70000, True), (2, 0, 131073, False)])
def test_verification_after_work_of_single_lanes(seqs, k, vocab, odd):
    """The lanes of a warp look at different numbers of drafts and of sums before a cluster's CTAs meet; every call of many gives the
    same tokens as the definition in 64 bits."""
    rng = np.random.default_rng(vocab)
    target, draft = rows(rng, (seqs, k + 1, vocab)), rows(rng, (seqs, k, vocab))
    draft[:, :max(k - 1, 0)] = target[:, :max(k - 1, 0)]  # all but the last are accepted
    tokens = rng.integers(0, vocab, (seqs, k)).astype(np.int32)
    accept, pick = (rng.random((seqs, k)) * 0.99).astype(np.float32), rng.random(seqs).astype(np.float32)
    want_acc, want = run_verify(target, draft, tokens, accept, pick)
    pad = 1 if odd else 0  # rows of an odd distance are read number by number
    t, d = torch.zeros(seqs, k + 1, vocab + pad, device="cuda")[..., pad:], torch.zeros(seqs, k, vocab + pad, device="cuda")[..., pad:]
    t.copy_(torch.from_numpy(target)), d.copy_(torch.from_numpy(draft))
    x, u, r = (torch.from_numpy(a).cuda() for a in (tokens, accept, pick))
    for _ in range(50):
        acc, out = drafts.verify(t, d, x, u, r)
        assert np.array_equal(acc.cpu().numpy(), want_acc) and np.array_equal(out.cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows_, vocab", [(3, 200003), (37, 163841), (500, 2051)])
@pytest.mark.parametrize("t", [0.0, 0.7])
def test_probabilities_after_work_of_single_lanes(rows_, vocab, t):
    z = (torch.randn((rows_, vocab), generator=torch.Generator().manual_seed(vocab)) * 3).cuda()
    first = drafts.probabilities(z, t)
    if t == 0:
        assert torch.equal(first.cpu().double(), softmax64(z.cpu(), t))
    # (a sum is off by no more than its numbers: 2^-24 (6 arg + 8 + vocab / 2048 + 40) of each, arg < 40 here: 2.3e-5)
    assert torch.allclose(first.double().sum(dim=1).cpu(), torch.ones(rows_, dtype=torch.float64), atol=1e-4)
    for _ in range(20):
        assert torch.equal(drafts.probabilities(z, t), first)
