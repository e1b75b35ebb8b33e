"""The language-model engine on pages at its borders: windows of any size, slots taken back after their windows have left pages behind."""
import os
import sys

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "oracle"))

import lm_case  # noqa: E402
import lm_models as M  # noqa: E402
import vupuzen_oracle as V  # noqa: E402
from mllm_b200 import lm, registry, vupuzen  # noqa: E402

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
