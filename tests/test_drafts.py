"""Logits to probabilities, and verification of drafted tokens, against their definitions in 64 bits."""
import numpy as np
import pytest
import torch

from mllm_b200 import drafts, lm


def test_refusals():
    L = lm.lib()
    probs = lambda logits=4096, dtype=lm.F32, ld=10, rows=2, vocab=10, t=1.0, out=4096, ld_out=10: L.mllmb200_lm_probabilities(logits, dtype, ld, rows, vocab, t, out, ld_out, None)
    assert [probs(logits=None), probs(dtype=7), probs(rows=-1), probs(vocab=0), probs(t=-1.0), probs(t=float("nan")), probs(t=float("inf")), probs(out=None),
            probs(ld_out=9), probs(rows=0)] == [1, 2, 1, 1, 1, 1, 1, 1, 1, 0]
    args = dict(target=4096, t_seq=30, t_row=10, draft=4096, d_seq=20, d_row=10, tokens=4096, ld_tokens=2, accept=4096, ld_accept=2, pick=4096, seqs=2, drafts=2, vocab=10,
                accepted=4096, out=4096, ld_out=3)
    verify = lambda **kw: L.mllmb200_lm_verify(*{**args, **kw}.values(), None)
    for kw in (dict(target=None), dict(draft=None), dict(tokens=None), dict(accept=None), dict(pick=None), dict(accepted=None), dict(out=None), dict(ld_out=2), dict(vocab=0),
               dict(seqs=-1), dict(drafts=-1), dict(t_row=-1)):
        assert verify(**kw) == 1, kw
    assert verify(seqs=0) == 0
    z = torch.zeros(2, 5)
    with pytest.raises(ValueError):
        drafts.probabilities(z)
    with pytest.raises(ValueError):
        drafts.verify(torch.zeros(1, 3, 5), torch.zeros(1, 3, 5), torch.zeros(1, 3, dtype=torch.int32), torch.zeros(1, 3), torch.zeros(1))


# ------------------------------------------------------------------------------------------------ probabilities
def softmax64(z, t):
    z = z.double()
    if t == 0:
        out = torch.zeros_like(z)
        for r in range(z.shape[0]):
            fine = torch.nan_to_num(z[r], -float("inf"), float("inf"), -float("inf"))
            if fine.max() > -float("inf"):
                out[r, int((fine == fine.max()).nonzero()[0])] = 1.0
        return out
    m = z.max(dim=1, keepdim=True).values
    w = torch.exp((z - m) / t)
    p = w / w.sum(dim=1, keepdim=True)
    p[(z == -float("inf")).all(dim=1)] = 0.0
    return p


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, vocab", [(1, 1), (3, 7), (2, 1023), (5, 4097), (1, 32000), (40, 5001), (2, 151936), (400, 300)])
@pytest.mark.parametrize("t", [0.0, 0.3, 1.0])
def test_probabilities(dtype, rows, vocab, t):
    z = (torch.randn((rows, vocab), generator=torch.Generator().manual_seed(vocab)) * 3).to(dtype)
    z[0, vocab // 2] = z[0].max()  # a tie
    want = softmax64(z, t)
    got = drafts.probabilities(z.cuda(), t).cpu().double()
    if t == 0:
        assert torch.equal(got, want)
        return
    # exp: its argument is off by three roundings, |z - m| / t of them times 2^-24, and CUDA's exp by 2 ulp; the sum by as many
    # roundings as a thread adds up, and one division
    arg = (z.double().max(dim=1, keepdim=True).values - z.double()) / t
    bound = want * 2.0 ** -24 * (3 * arg + 8 + 3 * arg.min(dim=1, keepdim=True).values + vocab / 256 + 40) + 1e-37
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows, vocab, z_at, z_pad, out_at, out_pad",
                         [(700, 1003, 0, 0, 0, 0), (400, 32001, 0, 0, 0, 0), (90, 50257, 0, 0, 0, 0), (90, 151935, 1, 2, 5, 2), (400, 32002, 3, 0, 2, 0), (60, 151937, 2, 0, 2, 3), (600, 1, 3, 5, 3, 1)])
@pytest.mark.parametrize("t", [0.0, 0.8])
def test_probabilities_of_many_rows(dtype, rows, vocab, z_at, z_pad, out_at, out_pad, t):
    """More rows than the GPU works on at a time; rows that begin anywhere in groups of four numbers."""
    g = torch.Generator().manual_seed(rows + vocab)
    inf = float("inf")
    z = (torch.randn((rows, vocab), generator=g) * 3).to(dtype)
    z[rows // 2, vocab // 3:] = -inf
    z[rows - 1] = torch.finfo(dtype).min
    z[rows - 2] = -inf
    z[rows - 3, vocab - 1] = inf
    z[rows - 4, vocab // 2] = float("nan")
    apart = torch.full((z_at + rows * (vocab + z_pad),), inf, dtype=dtype, device="cuda")
    logits = apart[z_at:].view(rows, vocab + z_pad)[:, :vocab]
    logits.copy_(z)
    whole = torch.full((out_at + rows * (vocab + out_pad) + 4,), -1.0, device="cuda")
    out = whole[out_at:out_at + rows * (vocab + out_pad)].view(rows, vocab + out_pad)[:, :vocab]
    drafts.probabilities(logits, t, out=out)
    got, want = out.cpu().double(), softmax64(z, t)
    assert (whole == -1).sum() == out_at + rows * out_pad + 4  # nothing beside the rows
    if t == 0:
        assert torch.equal(got, want)
        return
    assert got[rows - 3].isnan().all() and got[rows - 4].isnan().all()
    zd = z.double()
    arg = torch.nan_to_num((zd.max(dim=1, keepdim=True).values - zd) / t, 0.0, 0.0, 0.0)
    # In units of 2^-24: an exponent's argument is off by five roundings (difference, 1 / t, log2 e, their product, the whole), 5 |z - m| / t,
    # and exp2 by 4.  Above the line two exp2, a product and a quotient: 5 arg + 10.  Below it four exp2 (a thread's, warp's, CTA's
    # and cluster's maximum), the mean of 5 arg under the weights, at most 5 ln(vocab) < 60, and 40 + 15 sums: 131.  1e-37: below 2^-126
    bound = want * 2.0 ** -24 * (5 * arg + 141) + 1e-37
    fine = [r for r in range(rows) if r not in (rows - 3, rows - 4)]
    assert ((got - want).abs() <= bound)[fine].all()


@pytest.mark.gpu
@pytest.mark.parametrize("t", [0.0, 0.8])
def test_probabilities_of_long_rows(t):
    """Rows beyond what a cluster of CTAs holds."""
    vocab = 200003
    z = torch.randn((3, vocab), generator=torch.Generator().manual_seed(4)) * 3
    z[1, 7], z[1, 150000] = 40.0, 40.0
    z[2, :] = -float("inf")
    got, want = drafts.probabilities(z.cuda(), t).cpu().double(), softmax64(z, t)
    arg = 0.0 if t == 0 else torch.nan_to_num((z.double().max(dim=1, keepdim=True).values - z.double()) / t, 0.0)
    # (as above; a thread adds up vocab / 2048 weights)
    assert ((got - want).abs() <= want * 2.0 ** -24 * (6 * arg + 8 + vocab / 2048 + 40) + 1e-37).all()


@pytest.mark.gpu
def test_probabilities_of_masked_rows():
    inf, low = float("inf"), torch.finfo(torch.float32).min
    z = torch.randn(8, 3001)
    z[0, 5:] = -inf
    z[1, :] = -inf
    z[2, :] = low
    z[3, 100:] = low
    z[4, 17] = float("nan")
    z[5, 18] = inf
    z[6, :3000] = -inf
    for t in (0.0, 0.7):
        got, want = drafts.probabilities(z.cuda(), t).cpu().double(), softmax64(z, t)
        fine = [0, 1, 2, 3, 6, 7] if t else list(range(8))
        assert torch.allclose(got[fine], want[fine], rtol=1e-5, atol=1e-12)
        assert t == 0 or got[[4, 5]].isnan().all()
    assert drafts.probabilities(z.cuda(), 1e-42)[7].max() == 1.0  # as good as 0, without 0 / 0
    big = torch.zeros(9, 4000, device="cuda")
    out = drafts.probabilities(torch.randn(9, 4100, device="cuda")[:, 7:3007], 1.0, out=big[:, 9:3009])
    assert (big[:, :9] == 0).all() and (big[:, 3009:] == 0).all() and torch.allclose(out.sum(dim=1), torch.ones(9, device="cuda"), atol=1e-5)


# ------------------------------------------------------------------------------------------------ verification
def verify64(target, draft, tokens, accept, pick):
    """Sequence by sequence, exact products and running sums in 64 bits."""
    seqs, places, vocab = target.shape
    k, acc, out = places - 1, [], np.full((seqs, places), -1, np.int64)
    for s in range(seqs):
        n, refused = 0, False
        while n < k and 0 <= tokens[s, n] < vocab:
            x = tokens[s, n]
            if not float(accept[s, n]) * max(float(draft[s, n, x]), 0.0) < float(target[s, n, x]):
                refused = True
                break
            n += 1
        p = np.maximum(np.nan_to_num(target[s, n].astype(np.float64), nan=0.0), 0)
        mass = np.maximum(p - np.maximum(draft[s, n].astype(np.float64), 0), 0) if refused else p
        if not mass.sum() > 0:
            mass = p
        c = np.cumsum(mass)
        over = np.nonzero((c > float(pick[s]) * c[-1]) & (mass > 0))[0]
        some = np.nonzero(mass > 0)[0]
        out[s, :n] = tokens[s, :n]
        out[s, n] = over[0] if len(over) else some[-1] if len(some) else -1
        acc.append(n)
    return np.array(acc), out


def rows(rng, shape, sharp=2.0):
    z = rng.standard_normal(shape) * sharp
    w = np.exp(z - z.max(axis=-1, keepdims=True))
    return (w / w.sum(axis=-1, keepdims=True)).astype(np.float32)


def run_verify(target, draft, tokens, accept, pick):
    g = [torch.from_numpy(np.ascontiguousarray(x)).cuda() for x in (target, draft, tokens, accept, pick)]
    acc, out = drafts.verify(*g)
    want_acc, want = verify64(target, draft, tokens, accept, pick)
    assert np.array_equal(acc.cpu().numpy(), want_acc)
    assert np.array_equal(out.cpu().numpy(), want)
    return want_acc, want


@pytest.mark.gpu
@pytest.mark.parametrize("seqs, k, vocab", [(1, 1, 1), (1, 0, 50), (3, 4, 3), (5, 2, 1025), (2, 40, 300), (64, 5, 999), (7, 3, 32000), (2, 8, 151936), (700, 1, 64), (3, 2, 300001)])
def test_verify(seqs, k, vocab):
    rng = np.random.default_rng(seqs * 1000 + vocab)
    target, draft = rows(rng, (seqs, k + 1, vocab)), rows(rng, (seqs, k, vocab))
    near = rng.random((seqs, k)) < 0.5  # places where the models agree
    draft[near] = target[:, :k][near]
    tokens = rng.integers(0, vocab, (seqs, k)).astype(np.int32)
    for s in range(seqs):
        for i in range(k):
            if rng.random() < 0.8:
                tokens[s, i] = rng.choice(vocab, p=draft[s, i].astype(np.float64) / draft[s, i].astype(np.float64).sum())
    run_verify(target, draft, tokens, rng.random((seqs, k)).astype(np.float32), rng.random(seqs).astype(np.float32))


@pytest.mark.gpu
def test_verify_borders():
    """Numbers that 64 bits hold exactly: draws on the border between two tokens, no mass, ends of drafts, odd numbers."""
    V = 2048
    p = np.zeros((10, 3, V), np.float32)
    q = np.zeros((10, 2, V), np.float32)
    p[:, :, [3, 700, 2047]] = [0.25, 0.5, 0.25]
    q[:, :, [3, 700]] = [0.5, 0.5]
    tokens = np.full((10, 2), 700, np.int32)
    accept = np.full((10, 2), 0.5, np.float32)
    pick = np.array([0.0, 0.25, 0.2499999, 0.75, 0.9999999, 0.5, 0.5, 0.5, 0.0, 0.5], np.float32)
    tokens[5, 0] = -1              # no drafts
    tokens[6, 1] = V               # one draft
    tokens[7, 0] = 9               # not in either: 0.5 * 0 < 0 is false, and max(p - q, 0) has mass at 2047 alone
    p[8, 0], q[8, 0] = 0.0, 1.0    # refused, and the target has no mass
    p[9, 0, :], q[9, 0, 700] = np.nan, np.nan
    p[9, 0, 3], p[9, 0, 5] = 0.5, -1.0
    acc, out = run_verify(p, q, tokens, accept, pick)
    assert acc.tolist() == [2, 2, 2, 2, 2, 0, 1, 0, 0, 0]
    assert out[:, 0].tolist() == [700] * 5 + [700, 700, 2047, -1, 3]
    assert out[0].tolist() == [700, 700, 3] and out[1, 2] == 700 and out[2, 2] == 3 and out[3, 2] == 2047 and out[4, 2] == 2047
    same = p[:1, :2]               # refused where target and draft are the same: from the target
    acc, out = run_verify(p[:1], np.ascontiguousarray(same), np.full((1, 2), 9, np.int32), accept[:1], np.array([0.3], np.float32))
    assert acc[0] == 0 and out[0, 0] == 700


@pytest.mark.gpu
def test_verify_is_distributed_as_the_target():
    """20000 sequences of one draft over 6 tokens: what comes first is a draw of the target's distribution (chi-square of 5 degrees
    of freedom below 30: exceeded by a fair draw once in 10^5; the seed is fixed)."""
    n, V = 20000, 6
    p, q = np.array([0.3, 0.05, 0.25, 0.2, 0.1, 0.1], np.float32), np.array([0.1, 0.4, 0.1, 0.2, 0.15, 0.05], np.float32)
    rng = np.random.default_rng(3)
    tokens = rng.choice(V, size=(n, 1), p=q / q.sum(dtype=np.float64)).astype(np.int32)
    g = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()
    acc, out = drafts.verify(g(np.broadcast_to(p, (n, 2, V))), g(np.broadcast_to(q, (n, 1, V))), g(tokens), torch.rand(n, 1, generator=torch.Generator().manual_seed(1)).cuda(),
                             torch.rand(n, generator=torch.Generator().manual_seed(2)).cuda())
    seen = np.bincount(out[:, 0].cpu().numpy(), minlength=V)
    assert ((seen - n * p) ** 2 / (n * p)).sum() < 30
    assert abs(acc.float().mean().item() - np.minimum(p, q).sum()) < 0.02


@pytest.mark.gpu
def test_verify_strides_and_captured():
    rng = np.random.default_rng(9)
    S, k, V = 6, 3, 5000
    target, draft = rows(rng, (S, k + 1, V)), rows(rng, (S, k, V))
    tokens, accept, pick = rng.integers(0, V, (S, k)).astype(np.int32), rng.random((S, k)).astype(np.float32), rng.random(S).astype(np.float32)
    want_acc, want = verify64(target, draft, tokens, accept, pick)
    t, d = torch.zeros(S, k + 3, V + 9, device="cuda")[:, 1:k + 2, 5:V + 5], torch.zeros(S + 1, k, V + 1, device="cuda")[1:, :, 1:]
    t.copy_(torch.from_numpy(target)), d.copy_(torch.from_numpy(draft))
    x = torch.zeros(S, k + 2, dtype=torch.int32, device="cuda")[:, 2:]
    x.copy_(torch.from_numpy(tokens))
    u, r = torch.from_numpy(accept).cuda(), torch.from_numpy(pick).cuda()
    drafts.verify(t, d, x, u, r)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        acc, out = drafts.verify(t, d, x, u, r)
    for _ in range(2):
        g.replay()
        assert np.array_equal(acc.cpu().numpy(), want_acc) and np.array_equal(out.cpu().numpy(), want)
