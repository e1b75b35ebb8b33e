"""Admission by pages, and slots given back when generation ends early, without a GPU but for the drafted case."""
import numpy as np
import pytest

import lm_models as M
import taralix_models as TM
from mllm_b200 import drafts, registry, scheduler
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


@pytest.mark.gpu
def test_slots_come_back_when_drafted_generation_ends_early(tmp_path, monkeypatch):
    cfg = TM.config(64, 211, [TM.layer(TM.mixer(3, 20, 28, 36), TM.dense(72))])
    folder = TM.write(tmp_path, cfg, TM.weights(cfg, 3))
    model, draft = (registry.load(folder, "float32", 2, 100, 64)[0] for _ in range(2))
    want = scheduler.generate_drafted(model, draft, [[5, 9], [4], [7, 8, 9]], 12, 3)
    real, calls = drafts.verify, []

    def failing(*args):
        calls.append(1)
        if len(calls) == 6:
            raise RuntimeError("a rank went away")
        return real(*args)
    monkeypatch.setattr(drafts, "verify", failing)
    with pytest.raises(RuntimeError, match="went away"):
        scheduler.generate_drafted(model, draft, [[5, 9], [4], [7, 8, 9]], 12, 3)
    assert len(model._free) == len(draft._free) == 2
    assert scheduler.generate_drafted(model, draft, [[5, 9], [4], [7, 8, 9]], 12, 3) == want
    model.close()
    draft.close()


@pytest.mark.gpu
def test_one_model_in_both_roles_and_a_slot_outside(tmp_path):
    """A model that drafts for itself takes two slots a request, on pages that a third slot holds some of."""
    mixer = {**M.attention(4, 2, 16, 16, 37), "window": 0, "keep": 0}
    cfg = M.config(64, 97, [M.layer("attention", mixer, 48)], taps=0)
    m, _ = registry.load(M.write(tmp_path, cfg, M.weights(cfg, 5)), "bfloat16", 5, 160, 160, 16, 20)
    mine = m.acquire()
    m.step([(mine, list(range(90)))])  # 6 pages
    prompts = [np.random.default_rng(n).integers(0, 97, n).tolist() for n in (40, 3, 17)]
    got = scheduler.generate_drafted(m, m, prompts, 40, 3)  # 5 + 3 + 4 pages in each of two roles: not all at once
    assert [len(x) for x in got] == [40] * 3 and m.free_pages() == 14
    with pytest.raises(RuntimeError, match="others hold"):
        scheduler.generate_drafted(m, m, [prompts[0] * 2], 40, 3)  # 8 and 8
    with pytest.raises(ValueError):
        scheduler.generate_drafted(m, m, [prompts[0] * 3], 41, 3)  # 11 and 11 of 20
    m.release(mine)
    assert m.free_pages() == 20 and len(m._free) == 5
    m.close()
