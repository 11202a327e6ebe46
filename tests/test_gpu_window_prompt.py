"""decode_window over one very long prompt under a window, rows of it against the definition in 64 bits."""

import pytest
import torch

from _cache8 import problem, window64, window_bounds
from _util import log
from test_gpu_window import call, on_gpu

pytestmark = pytest.mark.gpu


def test_a_prompt_of_half_a_million_tokens():
    log("prompt: 524,288 tokens, window 4,096")
    n, window, sinks = 1 << 19, 4096, 5
    pr = problem(81, B=1, Hq=4, Hkv=1, D=64, Lq=n, T=n, lens=[n])
    out, lse = (t.cpu() for t in call(on_gpu(pr), window, sinks))
    for p in (0, 1, 63, 64, 255, 256, 4095, 4096, 4100, 65535, 65536, 100003, 262144, n - 2, n - 1):
        row = dict(pr, q=pr["q"][:, :, p:p + 1], seq_lens=torch.tensor([p + 1], dtype=torch.int32))
        ref = window64(row, window, sinks)
        ob, lb = window_bounds(row, *ref, out.dtype)
        assert ((out[:, :, p:p + 1].double() - ref[0]).abs() <= ob).all(), p
        assert ((lse[:, :, p:p + 1].double() - ref[1]).abs() <= lb).all(), p
