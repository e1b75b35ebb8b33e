"""The language-model engine on a cache in pages, with windows, and generation with drafted tokens: models of the Vupuzen design
against the float64 implementation in oracle/vupuzen_oracle.py, the Taralix design against its own greedy tokens."""
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "oracle"))

import lm_case  # noqa: E402
import lm_models as M  # noqa: E402
import taralix_models as TM  # noqa: E402
import vupuzen_oracle as V  # noqa: E402
from mllm_b200 import __main__ as cli  # noqa: E402
from mllm_b200 import lm, registry, scheduler, vupuzen  # noqa: E402

gpu = pytest.mark.gpu


def windowed(heads, kv, dim, vdim, bias_max, window, keep):
    return {**M.attention(heads, kv, dim, vdim, bias_max), "window": window, "keep": keep}


# windows alone, so that pages behind them are given up; a head size of the tensor-core kernel and others
WINDOWS = M.config(128, 200, [
    M.layer("attention", windowed(6, 2, 64, 64, 37, 40, 3), 96),
    M.layer("attention", windowed(4, 1, 24, 40, 90, 70, 0)),
    M.layer("retention", M.retention(3, 20, 28, 12, [0.9, 0.97, 1.0]), 72),
])
MODELS = {**M.MODELS, "windows": WINDOWS}


class Case(lm_case.Case):
    def __init__(self, folder, name, page, pages, max_seqs=6, max_ctx=1024, max_rows=1024):
        cfg = MODELS[name]
        self.cfg, self.w, self.dtype, self._oracle = cfg, M.weights(cfg, 7), "bfloat16", V
        self.model, runtime = registry.load(M.write(folder, cfg, self.w), "bfloat16", max_seqs, max_ctx, max_rows, page, pages)
        assert runtime == "engine"


# ------------------------------------------------------------------------------------------ host side
def test_window_of_the_config():
    d = vupuzen.layers_from_config(WINDOWS, lambda i: 10)
    assert [(x.get("window", 0), x.get("keep", 0)) for x in d] == [(40, 3), (70, 0), (0, 0)]
    assert [(x["window"], x["keep"]) for x in vupuzen.layers_from_config(M.MIXED, lambda i: 10) if x["mixer"] == lm.ATTENTION] == [(0, 0)] * 3


def test_page_sizes_that_are_refused():
    make = lambda dtype=lm.BF16, **kw: lm.LanguageModel({**vupuzen.model_config(M.MIXED, 1, 64, 64), **kw}, vupuzen.layers_from_config(M.MIXED, lambda i: 10), dtype)
    for kw, status in ((dict(page=16), 1), (dict(pages=4), 1), (dict(page=-16, pages=4), 1), (dict(page=24, pages=4), 2)):
        with pytest.raises(lm.EngineError) as e:
            make(**kw)
        assert e.value.status == status
    with pytest.raises(lm.EngineError) as e:
        make(lm.F32, page=16, pages=4)
    assert e.value.status == 2


# ------------------------------------------------------------------------------------------ the engine
@gpu
def test_window_without_pages_is_refused():
    with pytest.raises(lm.EngineError) as e:
        lm.LanguageModel(vupuzen.model_config(WINDOWS, 1, 64, 64), vupuzen.layers_from_config(WINDOWS, lambda i: 10))
    assert e.value.status == 2


@gpu
@pytest.mark.parametrize("name", sorted(MODELS))
@pytest.mark.parametrize("page", [16, 64])
def test_prompts_portions_and_single_tokens(name, page, tmp_path):
    case = Case(tmp_path, name, page, 6 * 1024 // page)
    tokens = case.tokens(330)
    want = case.oracle(tokens)
    for portions in ([330], [100, 1, 1, 30], [17]):
        case.check(case.run(tokens, portions), want)
    case.check(case.run(tokens[:40], [1]), want[:40])
    assert case.model.free_pages() == 6 * 1024 // page
    case.model.close()


@gpu
@pytest.mark.parametrize("name", ["mixed", "windows"])
def test_mixed_steps_and_decode(name, tmp_path):
    """Prompts, portions and single tokens of several sequences in one step, then graph-replayed decoding, all on pages that
    were other sequences' before."""
    case = Case(tmp_path, name, 16, 200)
    m = case.model
    seqs = [case.tokens(n, seed=n) for n in (150, 61, 9, 1)]
    slots = [m.acquire() for _ in seqs]
    m.step([(slots[1], seqs[1][:60]), (slots[2], seqs[2][:4])])
    entries = [(slots[0], seqs[0]), (slots[1], seqs[1][60:]), (slots[2], seqs[2][4:]), (slots[3], seqs[3])]
    ends, at = [], 0
    for _, t in entries:
        at += len(t)
        ends.append(at - 1)
    got = m.step(entries, ends, sample=True)
    for g, s in zip(got, seqs):
        case.check(g[None], case.oracle(s)[-1:])
    first = [int(m.read(s, m.length[s] - 1, 1)[0]) for s in slots]
    assert first == [int(g.argmax()) for g in got]
    m.decode(slots, 90)
    for s, prompt, f in zip(slots, seqs, first):
        new = [f] + m.read(s, len(prompt), 90).tolist()
        want = case.oracle(prompt + new[:-1])[len(prompt) - 1:]
        # every token is the oracle's largest logit, or within the bf16 error of it
        gap = want.max(axis=1) - want[np.arange(91), new]
        assert gap.max() < 0.5 * np.sqrt(np.mean(want ** 2)), float(gap.max())
        assert (gap == 0).mean() > 0.8
    m.check_device_status()
    m.close()


@gpu
def test_pages_are_counted_and_given_up(tmp_path):
    case = Case(tmp_path, "windows", 16, 30)
    m = case.model
    a = m.acquire()
    m.step([(a, case.tokens(100))])
    # 7 pages; position 100 sees from 31 on (window 70): place 0 holds the first tokens, place 1 (positions 16 .. 31) still shows one
    assert m.free_pages() == 23
    m.step([(a, case.tokens(29, 1))], [28], sample=True)  # 129 tokens, 9 pages
    assert m.free_pages() == 30 - 9
    m.decode([a], 63)                       # 192 tokens, 12 pages; at 129 nothing was behind a window of 70 and 64 tokens to go back
    assert m.free_pages() == 30 - 12
    m.decode([a], 0)                        # 16 .. 58 are behind now: places 1 and 2
    assert m.free_pages() == 30 - 12 + 2
    b = m.acquire()
    with pytest.raises(lm.EngineError) as e:
        m.step([(b, case.tokens(500, 2))])
    assert e.value.status == 6 and m.length[b] == 0 and m.free_pages() == 20
    with pytest.raises(lm.EngineError):
        m.decode([a], 400)
    m.step([(b, case.tokens(300, 2))])
    want = case.oracle(case.tokens(301, 2))
    case.check(m.step([(b, case.tokens(301, 2)[300:])], [0]), want[300:])
    m.release(a)
    m.release(b)
    assert m.free_pages() == 30
    m.close()


@gpu
def test_scheduler_waits_for_pages(tmp_path):
    """Fewer pages than the slots could hold: the same tokens as with as many as there can be."""
    prompts = [np.random.default_rng(i).integers(0, 200, n).tolist() for i, n in enumerate((90, 20, 60, 5, 33))]
    outs = []
    for pages in (200, 9):
        case = Case(tmp_path / str(pages), "windows", 16, pages)
        outs.append([registry.generate(case.model, "engine", [p], 30)[0] for p in prompts] if pages == 200 else registry.generate(case.model, "engine", prompts, 30))
        assert case.model.free_pages() == pages
        with pytest.raises(ValueError):
            scheduler.Scheduler(case.model).submit(list(range(100)), 1024 if pages == 200 else 60)
        case.model.close()
    same = sum(a == b for x, y in zip(*outs) for a, b in zip(x, y))
    assert same >= 0.8 * 150  # (a step of another shape rounds otherwise: near ties may fall differently)


# ------------------------------------------------------------------------------------------ drafted tokens
def taralix(folder, seed, max_seqs=3, width=100, dtype="float32", rows=256):
    cfg = TM.config(width, 211, [TM.layer(TM.mixer(3, 20, 28, 36), TM.dense(72)), TM.layer(TM.mixer(2, 36, 40, 36, kv_from=0))])
    path = TM.write(folder, cfg, TM.weights(cfg, seed))
    return registry.load(path, dtype, max_seqs, 300, rows)[0], path


@gpu
def test_truncate(tmp_path):
    m, _ = taralix(tmp_path / "a", 3)
    t = np.random.default_rng(1).integers(0, 211, 40).tolist()
    s = m.acquire()
    want = m.step([(s, t)], range(40))
    m.truncate(s, 25)
    got = m.step([(s, t[25:])], range(15))
    assert np.allclose(got, want[25:], rtol=0, atol=1e-4 * np.sqrt(np.mean(want ** 2)))
    for bad in (41, -1):
        with pytest.raises(lm.EngineError):
            m.truncate(s, bad)
    m.truncate(s, 0)
    assert np.allclose(m.step([(s, t)], range(40)), want, rtol=0, atol=1e-4 * np.sqrt(np.mean(want ** 2)))
    with pytest.raises(lm.EngineError):
        m.decode([s], 1)  # no current token
    m.close()
    case = Case(tmp_path / "b", "windows", 16, 60)
    s = case.model.acquire()
    case.model.step([(s, case.tokens(30))])
    with pytest.raises(lm.EngineError) as e:
        case.model.truncate(s, 3)
    assert e.value.status == 2
    case.model.truncate(s, 0)
    assert case.model.free_pages() == 60
    with pytest.raises(ValueError):
        scheduler.generate_drafted(case.model, case.model, [[1]], 3)
    case.model.close()


@gpu
def test_probabilities_of_a_step(tmp_path):
    m, _ = taralix(tmp_path, 3)
    t = np.random.default_rng(1).integers(0, 211, 20).tolist()
    s = m.acquire()
    z = m.step([(s, t)], [3, 19]).astype(np.float64)
    m.truncate(s, 0)
    p = m.step_probabilities([(s, t)], [3, 19], 0.7).cpu().numpy()
    w = np.exp((z - z.max(axis=1, keepdims=True)) / 0.7)
    assert np.allclose(p, w / w.sum(axis=1, keepdims=True), rtol=1e-4, atol=1e-9)
    m.close()


@gpu
@pytest.mark.parametrize("other", [False, True])
def test_greedy_tokens_with_drafts(other, tmp_path):
    """At temperature 0 the tokens are the model's own greedy ones, whether the drafts are good or not; more prompts than slots."""
    model, path = taralix(tmp_path / "a", 3)
    prompts = [np.random.default_rng(i).integers(0, 211, n).tolist() for i, n in enumerate((1, 40, 7, 22, 3))]
    want = scheduler.generate(model, prompts, 21)
    draft = taralix(tmp_path / "b", 5 if other else 3, width=64 if other else 100)[0]
    steps = model.stats()["launches"]
    for drafts in (1, 4):
        assert scheduler.generate_drafted(model, draft, prompts, 21, drafts) == want
    stop = {want[1][4]}
    cut = [w[:next((i + 1 for i, x in enumerate(w) if x in stop), len(w))] for w in want]
    assert scheduler.generate_drafted(model, draft, prompts, 21, 3, stop=stop) == cut
    assert model.stats()["launches"] > steps and len(model._free) == 3 and len(draft._free) == 3
    for m in (model, draft):
        m.check_device_status()
    with pytest.raises(ValueError):
        scheduler.generate_drafted(model, draft, [[]], 5)
    with pytest.raises(ValueError):
        scheduler.generate_drafted(model, draft, [[1]], 300)
    model.close()
    draft.close()


@gpu
def test_drafts_over_pages(tmp_path):
    """A model of attention layers without a convolution, on pages: taken back and forth over them, one request at a time where the
    pages hold no more; the tokens are its own greedy ones, but for near ties (a step of other shapes rounds otherwise)."""
    rng = np.random.default_rng(5)
    V_, W = 97, 64

    def model(pages, seed):
        layers = [dict(mixer=lm.ATTENTION, heads=4, kv_heads=2, dim=16, vdim=16, score_scale=0.25, sink=1, bias_rows=8, bias_max=20, window=24, keep=2, ff=48, ff_limit=2.0)] * 2
        m = lm.LanguageModel(dict(vocab=V_, width=W, conv_taps=0, max_seqs=3, max_ctx=160, max_rows=160, eps=1e-5, logit_scale=1.0, page=16, pages=pages), layers)
        r = np.random.default_rng(seed)
        bf = lambda n, k, s=1.0: M.f32_to_bf16((r.standard_normal((n, k)) * s / np.sqrt(k)).astype(np.float32))
        m.set_tensor(-1, "embed", bf(V_, W, 8.0))
        m.set_tensor(-1, "head", bf(V_, W, 3.0))
        m.set_tensor(-1, "final_norm", np.float32(1.0))
        for i in range(2):
            for name, n, k in (("q", 64, W), ("k", 32, W), ("v", 32, W), ("o", W, 64), ("gate", 48, W), ("up", 48, W), ("down", W, 48)):
                m.set_tensor(i, name, bf(n, k))
            m.set_tensor(i, "rel", r.standard_normal((8, 4)).astype(np.float32))
            for name in ("norm1", "norm1b", "norm2", "norm2b"):
                m.set_tensor(i, name, np.float32(1.0))
        return m

    prompts = [rng.integers(0, V_, n).tolist() for n in (40, 3, 17)]
    target, small = model(30, 1), model(30, 2)
    want = scheduler.generate(target, prompts, 40)
    for pages in (30, 5):  # 80 tokens are 5 pages
        m = model(pages, 1)
        got = scheduler.generate_drafted(m, small, prompts, 40, 3)
        assert m.free_pages() == pages and [len(x) for x in got] == [40] * 3
        agree = [next((i for i, (a, b) in enumerate(zip(x, y)) if a != b), 40) for x, y in zip(got, want)]
        assert sum(agree) >= 60, agree
        m.check_device_status()
        with pytest.raises(ValueError):
            scheduler.generate_drafted(m, small, [[1] * 110], 40 if pages == 5 else 60)
        m.close()
    target.close()
    small.close()


@gpu
def test_sampled_tokens_with_drafts(tmp_path):
    """The same seed gives the same tokens; the first token's distribution is the model's (200 runs over its likeliest tokens)."""
    model, _ = taralix(tmp_path / "a", 3, max_seqs=200, rows=1024)
    draft, _ = taralix(tmp_path / "b", 5, max_seqs=200, width=64, rows=1024)
    a = scheduler.generate_drafted(model, draft, [[5, 9, 2]] * 200, 3, 2, 1.0, seed=1)
    assert a == scheduler.generate_drafted(model, draft, [[5, 9, 2]] * 200, 3, 2, 1.0, seed=1)
    assert a != scheduler.generate_drafted(model, draft, [[5, 9, 2]] * 200, 3, 2, 1.0, seed=2)
    s = model.acquire()
    p = model.step_probabilities([(s, [5, 9, 2])], [2], 1.0)[0].cpu().numpy().astype(np.float64)
    seen = np.bincount([x[0] for x in a], minlength=211)
    # total variation of 200 draws over the tokens above 2 %: each is off by sqrt(p / 200) on average, four times that is allowed
    for t in np.nonzero(p > 0.02)[0]:
        assert abs(seen[t] / 200 - p[t]) < 4 * np.sqrt(p[t] / 200)
    model.close()
    draft.close()


@gpu
def test_command_line(tmp_path, capsys):
    model, path = taralix(tmp_path / "a", 3, dtype="bfloat16")
    want = scheduler.generate(model, [[4, 8, 15], [16]], 12)
    model.close()
    cli.main(["generate", "--model", path, "--tokens", "4,8,15", "--tokens", "16", "--max-new", "12", "--draft", path, "--drafts", "3"])
    lines = [[int(x) for x in line.split(",")] for line in capsys.readouterr().out.strip().splitlines()]
    assert [len(x) for x in lines] == [12, 12] and sum(a == b for x, y in zip(lines, want) for a, b in zip(x, y)) >= 12
    folder = M.write(tmp_path / "w", WINDOWS, M.weights(WINDOWS, 7))
    cli.main(["generate", "--model", folder, "--tokens", "4,8,15", "--max-new", "5", "--page", "16"])
    assert len(capsys.readouterr().out.strip().split(",")) == 5
