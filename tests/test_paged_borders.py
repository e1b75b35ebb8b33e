"""Operators over pages at their borders: lengths beyond a table, tensors of other streams, odd arguments."""
import contextlib
import ctypes as C
import pytest
import torch

from mllm_b200 import drafts, lm, paged
from paged_case import Cache
from test_paged import good

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


class FakeStream:
    """A stream as the calls see it, without a GPU."""

    def __init__(self, index, cuda_stream=77):
        self.device, self.cuda_stream, self.device_index = torch.device("cuda", index), cuda_stream, index


def test_a_stream_of_the_callers_keeps_the_tensors(monkeypatch):
    kept = []

    class Tensor:
        def record_stream(self, s):
            kept.append((self, s))
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    s, tensors = FakeStream(0), [Tensor(), None, Tensor()]
    assert paged._on(0, s, lambda raw: raw + 1, *tensors) == 78
    assert kept == [(tensors[0], s), (tensors[2], s)]
    ran = []
    with pytest.raises(ValueError, match="cuda:1 for tensors of cuda:0"):
        paged._on(0, FakeStream(1), ran.append, *tensors)
    assert not ran and len(kept) == 2


def test_check_asks_the_streams_device(monkeypatch):
    asked = []

    class Device(contextlib.nullcontext):
        def __init__(self, device):
            super().__init__()
            asked.append(device)

    class Library:
        def mllmb200_lm_operator_status(self, raw):
            asked.append(raw)
            return 7
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(lm, "lib", Library)
    with pytest.raises(lm.EngineError):
        paged.check(FakeStream(1))
    assert asked == [torch.device("cuda", 1), 77]


@pytest.mark.gpu
def test_tensors_dropped_behind_a_call_on_a_stream():
    """Temporaries of calls on a stream that is busy: their memory is not handed out while it is read."""
    c = Cache([300, 40], 2, 64, 64, 16, BF16, 14).on_gpu()
    q, z = rand((2, 4, 64), BF16, 15).cuda(), torch.randn(3, 5000, device="cuda")
    start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    want = [paged.decode_attention(q, c.k, c.v, c.table, c.lengths), paged.prompt_attention(q, c.k, c.v, c.table, c.lengths, start), drafts.probabilities(z)]
    side = torch.cuda.Stream()
    for i in range(3):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        args = (z.clone(),) if i == 2 else (q.clone(), c.k, c.v, c.table.clone(), c.lengths.clone())
        ready = torch.cuda.Event()
        ready.record()
        call = [paged.decode_attention, lambda *a, stream: paged.prompt_attention(*a, start, stream=stream), drafts.probabilities][i]
        side.wait_event(ready)
        got = call(*args, stream=side)
        shapes = [(a.shape, a.dtype) for a in args]
        del args
        junk = [torch.empty(shape, dtype=dtype, device="cuda").fill_(3) for shape, dtype in shapes for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(got, want[i])
        del junk


def test_outputs_that_overlap():
    q = torch.zeros(3, 4, 64)
    assert paged._apart(torch.zeros(3, 4, 64), q) and paged._apart(torch.zeros(6, 9, 64)[::2, 1:5], q) and paged._apart(torch.zeros(64).expand(1, 1, 64), q)
    assert not paged._apart(q, q) and not paged._apart(torch.zeros(1, 4, 64).expand(3, 4, 64), q) and not paged._apart(torch.zeros(3, 1, 64).expand(3, 4, 64), q)
    assert paged._apart(q[:0], q)


@pytest.mark.gpu
def test_outputs_that_overlap_are_refused():
    c = Cache([30, 40], 2, 64, 64, 16, BF16, 14).on_gpu()
    q, start = rand((2, 4, 64), BF16, 15).cuda(), torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for out in (q, torch.zeros(1, 4, 64, dtype=BF16, device="cuda").expand(2, 4, 64)):
        with pytest.raises(ValueError, match="every place once"):
            paged.decode_attention(q, c.k, c.v, c.table, c.lengths, out=out)
        with pytest.raises(ValueError, match="every place once"):
            paged.prompt_attention(q, c.k, c.v, c.table, c.lengths, start, out=out)


def test_rows_without_sequences_are_refused():
    """Rows that belong to no sequence have no answer; with row starts they lie behind the last sequence and are left as they are."""
    p, look = good()
    p.seqs, L, size = 0, lm.lib(), C.c_size_t()
    assert L.mllmb200_lm_attn_decode_workspace(bytes(p), bytes(look), C.byref(size)) == 1
    assert L.mllmb200_lm_attn_decode(bytes(p), bytes(look), 4096, None) == 1
    assert L.mllmb200_lm_pages_append(bytes(p), 4096, 128, 64, 4096, 128, 64, None) == 1
    p.q_start = 4096
    assert L.mllmb200_lm_attn_prompt(bytes(p), bytes(look), 4096, None) == 0
