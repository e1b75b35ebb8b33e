"""Logits to probabilities and verification where a call can go wrong: barriers of clusters behind work of single lanes, rows in memory of
another form, sizes at the limits."""
import numpy as np
import pytest
import torch

import taralix_models as TM
from mllm_b200 import drafts, lm, registry
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


def test_rows_of_out_that_overlap_are_refused():
    """Shape and contiguous rows are not enough: rows nearer than vocab (an expanded row) would be written behind the tensor's end."""
    z = torch.zeros(4, 10)
    for out in (torch.zeros(1, 10).expand(4, 10), torch.zeros(40).as_strided((4, 10), (9, 1))):
        with pytest.raises(ValueError, match="overlap"):
            drafts.probabilities(z, out=out)
        with pytest.raises(ValueError, match="overlap"):
            lm.row_distance("step_probabilities", out, 4, 10)
    for out in (torch.zeros(4, 9), torch.zeros(4, 10).double(), torch.zeros(10, 4).T, torch.zeros(40)):
        with pytest.raises(ValueError, match="out \\["):
            lm.row_distance("step_probabilities", out, 4, 10)
    assert lm.row_distance("", torch.zeros(4, 12)[:, 1:11], 4, 10) == 12 and lm.row_distance("", torch.zeros(1, 10).as_strided((1, 10), (3, 1)), 1, 10) == 10
    assert lm.row_distance("", torch.zeros(0, 10), 0, 10) == 10


@pytest.mark.gpu
def test_overlapping_rows_of_out_are_refused_on_the_gpu(tmp_path):
    z = torch.randn(4, 10, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        drafts.probabilities(z, out=torch.zeros(1, 10, device="cuda").expand(4, 10))
    cfg = TM.config(64, 211, [TM.layer(TM.mixer(3, 20, 28, 36), TM.dense(72))])
    m, _ = registry.load(TM.write(tmp_path, cfg, TM.weights(cfg, 3)), "float32", 1, 64, 64)
    s = m.acquire()
    for out in (torch.zeros(1, 211, device="cuda").expand(3, 211), torch.zeros(3, 211)):
        with pytest.raises(ValueError):
            m.step_probabilities([(s, [1, 2, 3])], [0, 1, 2], out=out)
    assert m.length[s] == 0
    out = torch.zeros(2, 300, device="cuda")
    m.step_probabilities([(s, [1, 2, 3])], [0, 2], out=out[:, :211])
    assert (out[:, 211:] == 0).all() and torch.allclose(out.sum(dim=1), torch.ones(2, device="cuda"), atol=1e-5)
    m.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("at", [1, 2, 3])
def test_many_rows_from_an_odd_address(dtype, at):
    """Rows that are copied ahead from memory that begins inside a group of four numbers."""
    rows_, vocab, ld = 700, 1003, 1004
    logits = torch.randn(at + rows_ * ld, generator=torch.Generator().manual_seed(at)).to(dtype).cuda()[at:].view(rows_, ld)[:, :vocab]
    whole = torch.full((at + rows_ * ld,), -1.0, device="cuda")
    out = drafts.probabilities(logits, 0.8, out=whole[at:].view(rows_, ld)[:, :vocab])
    # (the groups fall otherwise, and with them the order of sums and the threads' maxima: 2^-24 (5 arg + 141) on either side, arg < 12)
    want = drafts.probabilities(logits.contiguous(), 0.8)
    assert ((out - want).abs() <= want * 2.0 ** -24 * 2 * (5 * 12 + 141)).all()
    assert (whole[:at] == -1).all() and (whole[at:].view(rows_, ld)[:, vocab:] == -1).all()


def test_rows_longer_than_32_bits_count_are_refused():
    L = lm.lib()
    for vocab in (2 ** 30 + 1, 2 ** 31 - 1):
        assert L.mllmb200_lm_probabilities(4096, lm.F32, 2 ** 31, 1, vocab, 1.0, 4096, 2 ** 31, None) == 2


@pytest.mark.gpu
def test_strides_of_a_vocabulary_of_one():
    """A dimension of one may have any stride."""
    odd = lambda t, *strides: torch.as_strided(t, t.shape, strides)
    z, out = torch.randn(3, 1, device="cuda"), torch.zeros(3, 1, device="cuda")
    assert (drafts.probabilities(odd(z, 1, 7), 0.5, out=odd(out, 1, 5)) == 1.0).all() and (out == 1.0).all()
    p = torch.ones(2, 2, 1, device="cuda")
    acc, new = drafts.verify(odd(p, 2, 1, 9), odd(p[:, :1].contiguous(), 1, 1, 4), torch.zeros(2, 1, dtype=torch.int32, device="cuda"), torch.zeros(2, 1, device="cuda") + 0.5,
                             torch.zeros(2, device="cuda") + 0.5)
    assert acc.tolist() == [1, 1] and new.tolist() == [[0, 0], [0, 0]]
