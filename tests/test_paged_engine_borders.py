"""The language-model engine on pages at its borders: windows of any size, slots taken back after their windows have left pages behind."""
import ctypes as C
import os
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "oracle"))

import lm_case  # noqa: E402
import lm_models as M  # noqa: E402
import vupuzen_oracle as V  # noqa: E402
from mllm_b200 import lm, registry, scheduler, vupuzen  # noqa: E402

gpu = pytest.mark.gpu
MOST = 2 ** 31 - 1


class Case(lm_case.Case):
    def __init__(self, folder, windows, pages, page=16, max_seqs=3, max_ctx=600, max_rows=600):
        """A model of attention layers alone, with these (window, first tokens)."""
        mixers = [{**M.attention(*size, 37), "window": w, "keep": k} for size, (w, k) in zip(((6, 2, 64, 64), (4, 1, 24, 40)), windows)]
        self.cfg = M.config(128, 200, [M.layer("attention", m, 96) for m in mixers], taps=0)
        self.w, self.dtype, self._oracle = M.weights(self.cfg, 7), "bfloat16", V
        self.model, _ = registry.load(M.write(folder, self.cfg, self.w), "bfloat16", max_seqs, max_ctx, max_rows, page, pages)


def test_pages_beyond_the_positions_that_are_counted():
    cfg = M.config(64, 50, [M.layer("attention", M.attention(2, 1, 16, 16, 37))])
    for ctx, page in ((MOST, 16), (64, MOST - 15), (2 ** 30, 16)):
        with pytest.raises(lm.EngineError) as e:
            lm.LanguageModel({**vupuzen.model_config(cfg, 1, 64, 64), "max_ctx": ctx, "page": page, "pages": 1}, vupuzen.layers_from_config(cfg, lambda i: 10))
        assert e.value.status == 2


@gpu
@pytest.mark.parametrize("windows", [((64, MOST), (64, MOST)), ((MOST, 0), (MOST, 0)), ((MOST, MOST), (40, 3)), ((600, 0), (599, 600))])
def test_windows_and_first_tokens_of_any_size(windows, tmp_path):
    """Everything stays visible to some layer: no page is given up, and the logits are those of the definition."""
    case = Case(tmp_path, windows, 110)
    m, tokens = case.model, case.tokens(500)
    want, slot, got = case.oracle(tokens), case.model.acquire(), []
    for i in range(0, 500, 100):
        got.append(m.step([(slot, tokens[i:i + 100])], range(100)))
        assert m.free_pages() == 110 - -(-(i + 100) // 16)
    case.check(np.concatenate(got), want)
    m.check_device_status()
    m.close()


@gpu
def test_taken_back_after_pages_were_given_up(tmp_path):
    """What the windows have left behind by 64 tokens is gone; the last 64 tokens, and those of the last step, can be taken back."""
    case = Case(tmp_path, ((24, 2), (20, 1)), 40)
    m, tokens = case.model, case.tokens(320)
    want, s = case.oracle(tokens), case.model.acquire()
    for a, b in ((0, 90), (90, 150), (150, 160), (160, 170)):
        got = m.step([(s, tokens[a:b])], range(b - a))
        case.check(got, want[a:b])
    # before the last step the slot held 160 tokens: of positions up to 160 - 64 - 24 = 72 places 1 .. 3 (16 .. 63) went
    assert m.free_pages() == 40 - 11 + 3
    m.truncate(s, 106)  # 64 tokens
    case.check(m.step([(s, tokens[106:170])], range(64)), want[106:170])
    m.truncate(s, 160)
    with pytest.raises(lm.EngineError) as e:  # a token at 70 sees from 47 on
        m.truncate(s, 70)
    assert e.value.status == 1 and m.free_pages() == 40 - 10 + 3 and m.length[s] == 160
    case.check(m.step([(s, tokens[160:300])], range(140)), want[160:300])
    m.truncate(s, 160)  # where the last step began
    case.check(m.step([(s, tokens[160:320])], range(160)), want[160:320])
    m.truncate(s, 0)
    assert m.free_pages() == 40
    case.check(m.step([(s, tokens[:30])], range(30)), want[:30])
    m.check_device_status()
    m.close()


@gpu
def test_taken_back_several_times(tmp_path):
    """How far a slot can be taken back goes by its furthest step, not by where it is when it is taken back."""
    case = Case(tmp_path, ((24, 2), (20, 1)), 40)
    m, tokens = case.model, case.tokens(230)
    want, s = case.oracle(tokens), case.model.acquire()
    for a, b in ((0, 150), (150, 190), (190, 200)):
        m.step([(s, tokens[a:b])])
    free = m.free_pages()
    m.truncate(s, 160)
    m.step([(s, tokens[160:161])])
    m.truncate(s, 126)  # the furthest step began at 190
    assert m.free_pages() == free + 13 - 8
    with pytest.raises(lm.EngineError) as e:  # (64 tokens of where it is now, but what they see went when it moved on from 190)
        m.truncate(s, 62)
    assert e.value.status == 1 and m.length[s] == 126 and m.free_pages() == free + 13 - 8
    case.check(m.step([(s, tokens[126:230])], range(104)), want[126:230])
    m.close()


@gpu
def test_drafts_behind_long_prompts_over_windows(tmp_path):
    """Prompts that the windows have left pages of, one request after the other: the model's own greedy tokens, but for near ties (a step
    of other shapes rounds otherwise)."""
    case = Case(tmp_path / "a", ((24, 2), (20, 1)), 60)
    other = Case(tmp_path / "b", ((24, 2), (20, 1)), 60)
    prompts = [case.tokens(n, seed=n) for n in (140, 230, 101)]
    want = scheduler.generate(case.model, prompts, 90)
    got = scheduler.generate_drafted(case.model, other.model, prompts, 90, 5)
    assert case.model.free_pages() == other.model.free_pages() == 60 and [len(x) for x in got] == [90] * 3
    for prompt, x, y in zip(prompts, got, want):
        logits = case.oracle(prompt + x[:-1])[len(prompt) - 1:]
        gap = logits.max(axis=1) - logits[np.arange(90), x]
        assert gap.max() < 0.5 * np.sqrt(np.mean(logits ** 2)) and (gap == 0).mean() > 0.8
        assert x[0] == y[0]
    for c in (case, other):
        c.model.check_device_status()
        c.model.close()


# the structures of callers that were built before there were pages
class OldConfig(C.Structure):
    _fields_ = [(n, C.c_int) for n in ("vocab", "width", "layers", "dtype", "conv_taps", "max_seqs", "max_ctx", "max_rows")] + \
               [("eps", C.c_float), ("logit_scale", C.c_float), ("norm_place", C.c_int), ("residual_scale", C.c_float)]


class OldLayer(C.Structure):
    _fields_ = lm.Layer._fields_[:-2]


def old_structures(layers):
    cfg = M.config(64, 50, [M.layer("attention", M.attention(2, 1, 16, 16, 37), 32)] * layers)
    now = [{"sink": 0, "bias_rows": 0, "bias_max": 0, "rot_dims": 0, "rot_base": 1.0, "ff": 0, "ff_limit": 0.0, "score_scale": 1.0, "weights_of": -1, "kv_rank": 0,
            "kv_from": -1, "act": lm.CLAMPED, "experts": 0, "top": 0, **d} for d in vupuzen.layers_from_config(cfg, lambda i: 10)]
    names = [n for n, *_ in OldLayer._fields_]
    descs = (OldLayer * layers)(*[OldLayer(**{n: d[n] for n in names}) for d in now])
    c = {**vupuzen.model_config(cfg, 1, 64, 64), "layers": layers, "dtype": lm.BF16, "norm_place": lm.NORM_SANDWICH, "residual_scale": 1.0}
    return OldConfig(**{n: c[n] for n, *_ in OldConfig._fields_}), descs


@pytest.mark.parametrize("layers", [1, 5])
def test_structures_of_older_callers(layers):
    """What lies behind a shorter structure is not read as pages: the model is as good as it was then (without a GPU: as far as its
    sizes are looked at)."""
    assert C.sizeof(OldLayer) < C.sizeof(lm.Layer)
    config, descs = old_structures(layers)
    noise = (C.c_char * 4096).from_buffer(bytearray(b"\xff" * 4096))
    C.memmove(noise, C.byref(config), C.sizeof(config))
    C.memmove(C.byref(noise, 2048), descs, C.sizeof(descs))
    h, L = C.c_void_p(), C.CDLL(lm.lib_path())
    st = L.mllmb200_lm_create(noise, C.byref(noise, 2048), C.byref(h))
    assert st == (0 if torch.cuda.is_available() else 3)
    if st == 0:
        n = C.c_int()
        assert L.mllmb200_lm_free_pages(h, C.byref(n)) == 0 and n.value == 0
        L.mllmb200_lm_destroy(h)
