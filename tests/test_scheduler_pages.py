"""Admission by pages, and slots given back when generation ends early, without a GPU but for the drafted case."""
import numpy as np
import pytest

from mllm_b200 import scheduler
from test_vupuzen import FakeModel, fake_reference


class FakePaged(FakeModel):
    """Slots that take pages as they grow."""

    def __init__(self, max_seqs, max_ctx, max_rows, page, pages):
        super().__init__(max_seqs, max_ctx, max_rows)
        self.page, self.pages, self.least = page, pages, pages

    def free_pages(self):
        n = self.pages - sum(-(-n // self.page) for n in self.length)
        assert n >= 0
        self.least = min(self.least, n)
        return n

    def step(self, entries, want=(), sample=False):
        out = super().step(entries, want, sample)
        self.free_pages()
        return out


def test_requests_wait_for_pages_that_others_hold():
    """Pages that a slot outside of the scheduler holds are not there for its requests; all the same every one is served."""
    m = FakePaged(4, 64, 64, 8, 14)
    mine = m.acquire()
    m.step([(mine, list(range(50)))])  # 7 pages
    prompts = [np.random.default_rng(i).integers(0, 50, n).tolist() for i, n in enumerate((20, 9, 30, 1, 17))]
    out = scheduler.generate(m, prompts, 14)
    assert out == [fake_reference(p, 14) for p in prompts]
    assert m.least < 3 and m.free_pages() == 7 and len(m.free) == 3
    with pytest.raises(RuntimeError, match="others hold"):
        scheduler.generate(m, [prompts[2] + prompts[0]], 14)  # 8 pages of the 14 are never free
    m.release(mine)
    assert scheduler.generate(m, [prompts[2] + prompts[0]], 14) == [fake_reference(prompts[2] + prompts[0], 14)]


def test_no_slot_at_all():
    m = FakeModel(1, 64, 32)
    m.acquire()
    with pytest.raises(RuntimeError, match="others hold"):
        scheduler.generate(m, [[1, 2]], 3)
