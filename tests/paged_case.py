"""What the tests of the operators over pages share: caches in pages with everything that must not be read poisoned, and
attention in 64 bits written from its definition."""
import math

import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Cache:
    """Random keys and values of sequences, in pages of a pool in a random order.  Rows behind a sequence's length, pages that
    belong to nobody and table places behind a sequence's pages hold NaN, infinities and numbers of no page."""

    def __init__(self, lengths, kv_heads, dim, vdim, page, dtype, seed, layout="head", extra=3, wide=2):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.lengths_h, self.kv_heads, self.dim, self.vdim, self.page, self.dtype = list(lengths), kv_heads, dim, vdim, page, dtype
        need = [(max(n, 0) + page - 1) // page for n in lengths]
        self.pages = sum(need) + extra
        order = rng.permutation(self.pages)
        table = np.full((len(lengths), max(need, default=0) + wide), -7, np.int32)
        table[:, -1] = 2 ** 31 - 1
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
        self.table_h = table
        self.keys = [torch.randn((max(n, 0), kv_heads, dim), generator=g).to(dtype) for n in lengths]
        self.values = [torch.randn((max(n, 0), kv_heads, vdim), generator=g).to(dtype) for n in lengths]
        shape = (self.pages, kv_heads, page) if layout == "head" else (self.pages, page, kv_heads)
        self.k, self.v = (torch.full(shape + (d,), float("nan"), dtype=dtype) for d in (dim, vdim))
        self.k[::2], self.v[::2] = float("inf"), float("-inf")
        if layout != "head":
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        for s, n in enumerate(lengths):
            for j in range(max(n, 0)):
                self.k[table[s, j // page], :, j % page] = self.keys[s][j]
                self.v[table[s, j // page], :, j % page] = self.values[s][j]

    def on_gpu(self):
        self.table = torch.from_numpy(self.table_h).cuda()
        self.lengths = torch.tensor(self.lengths_h, dtype=torch.int32, device="cuda")
        strided = not self.k.is_contiguous()
        self.k, self.v = ((t.transpose(1, 2).contiguous().cuda().transpose(1, 2) if strided else t.cuda()) for t in (self.k, self.v))
        return self


def visible(i, n, window, keep):
    """Which of keys 0 .. n - 1 a token at position i sees."""
    j = torch.arange(n)
    seen = j <= i
    if window:
        seen &= (j > i - window) | (j < keep)
    return seen


def attention64(cache, counts, q, scale=None, window=0, keep=0, sink=None, bias=None):
    """(outputs, sums of weights times |values|, largest sum of |products| of a visible score) in 64 bits; rows in order."""
    heads = q.shape[1]
    group = heads // cache.kv_heads
    scale = cache.dim ** -0.5 if scale is None else scale
    out, spread, big, row = torch.zeros(q.shape[0], heads, cache.vdim, dtype=torch.float64), torch.zeros(q.shape[0], heads, cache.vdim, dtype=torch.float64), 0.0, 0
    for s, (count, n) in enumerate(zip(counts, cache.lengths_h)):
        k, v = cache.keys[s].double(), cache.values[s].double()
        for t in range(count):
            i = n - count + t
            seen = visible(i, max(n, 0), window, keep) if i >= 0 else torch.zeros(max(n, 0), dtype=torch.bool)
            if seen.any():
                j = seen.nonzero()[:, 0]
                for h in range(heads):
                    x = q[row + t, h].double()
                    z = (k[j, h // group] @ x) * scale
                    big = max(big, float((k[j, h // group].abs() @ x.abs()).max()) * abs(scale))
                    if bias is not None:
                        z = z + bias[h].double()[(i - j).clamp(max=bias.shape[1] - 1)]
                    m = z.max() if sink is None else max(z.max(), sink[h].double())
                    w = torch.exp(z - m)
                    w = w / (w.sum() + (0.0 if sink is None else math.exp(float(sink[h].double() - m))))
                    vs = v[j, h // group]
                    out[row + t, h] = w @ vs
                    spread[row + t, h] = w @ vs.abs()
        row += count
    return out, spread, big


def check(got, want, spread, big, dim, dtype, weights_in_16_bits):
    """Bound of the error: the output's own rounding; the weights' (half a step of 16 bits, or 2^-16 where two halves carry
    them, together with exp2's 2^-21); a score's sum over dim / 16 steps of the tensor core and its scaling, each off by at most 2^-23 of
    the sum of magnitudes, twice (weight and their sum).  Below 2^-14 fp16 numbers lie 2^-24 apart whatever their size, so that the output's
    rounding is 2^-25 there, not a share of the value (bf16: 2^-134)."""
    half, least = HALF_STEP[dtype], 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134
    bound = half * want.abs() * 1.01 + spread * ((half if weights_in_16_bits else 0.0) + 2.0 ** -16 + 2 * (dim / 16 + 4) * 2.0 ** -23 * max(big, 1.0)) + least
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got.cpu().double()).all()
    worst = float((off / bound).max())
    at = int((off / bound).argmax())
    assert worst <= 1.0, (worst, float(want.reshape(-1)[at]), float(off.reshape(-1)[at]), float(spread.reshape(-1)[at]))
