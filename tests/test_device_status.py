"""The device status word: operators on a caller's memory and engines are told apart, and nothing that was found is lost."""
import os
import subprocess

import numpy as np
import pytest
import torch

import lm_models as M
from mllm_b200 import lm, paged, registry

HERE = os.path.dirname(os.path.abspath(__file__))
OK, TIMEOUT, BAD_BLOB, BAD_PAGE = 0, 4, 5, 7


@pytest.mark.gpu
def test_readers_of_the_word(tmp_path):
    """Each reader takes the first of its own kinds and leaves the rest."""
    exe = str(tmp_path / "status_word")
    subprocess.run([os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-rdc=true", "-o", exe,
                    os.path.join(HERE, "status_word.cu"), os.path.join(HERE, "..", "mllm-advanced_b200", "csrc", "device_status.cu")], check=True)
    lines = [[int(x) for x in line.split()] for line in subprocess.run([exe], check=True, capture_output=True, text=True).stdout.splitlines()]
    assert lines == [[BAD_PAGE, OK, OK, OK, OK, OK], [OK, TIMEOUT, OK, OK, OK, OK], [OK, TIMEOUT, OK, BAD_BLOB, OK, OK], [TIMEOUT, TIMEOUT, BAD_PAGE, OK, OK, OK], [OK] * 6]


@pytest.mark.gpu
def test_an_engine_does_not_report_a_callers_pages(tmp_path):
    cfg = M.config(64, 50, [M.layer("attention", M.attention(2, 1, 64, 64, 37))])
    m, _ = registry.load(M.write(tmp_path, cfg, M.weights(cfg, 7)), "bfloat16", 1, 64, 64, 16, 4)
    k = torch.zeros(2, 1, 16, 64, dtype=torch.bfloat16, device="cuda")
    q, table = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.full((1, 1), 9, dtype=torch.int32, device="cuda")
    lengths, start = torch.ones(1, dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for call in (lambda: paged.decode_attention(q, k, k, table, lengths), lambda: paged.prompt_attention(q, k, k, table, lengths, start),
                 lambda: paged.append(k, k, q[:, :1], q[:, :1], table, lengths)):
        call()
        s = m.acquire()
        m.step([(s, np.arange(9).tolist())], [8])
        m.check_device_status()
        with pytest.raises(lm.EngineError) as e:
            paged.check()
        assert e.value.status == BAD_PAGE
        paged.check()
        m.release(s)
    m.close()
