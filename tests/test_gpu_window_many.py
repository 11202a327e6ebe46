"""decode_window over very many short sequences, against the same few sequences by themselves."""

import pytest
import torch

from _cache8 import E4M3, problem
from _util import log
from test_gpu_window import call, check, on_gpu

pytestmark = pytest.mark.gpu


def many(B, **kw):
    """A problem of 8 sequences, checked, and the same on B rows that repeat them (queries are views; the last row last)."""
    pr = problem(71, B=8, T=64, lens=[64, 0, 1, 17, 33, 5, 64, 2], **kw)
    gp = on_gpu(pr)
    want = check(pr, gp=gp)
    big = dict(gp, block_table=gp["block_table"].repeat(B // 8, 1), seq_lens=gp["seq_lens"].repeat(B // 8))
    q = gp["q"]
    big["q"] = q[None].expand(B // 8, *q.shape).reshape(B, *q.shape[1:])
    return big, want


def same(got, want, B):
    for g, w in zip(got, want):
        assert torch.equal(g.view(B // 8, *w.shape), w[None].expand(B // 8, *w.shape))


def timed(big):
    call(big)
    best = float("inf")
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        call(big)
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("kw", [dict(Hq=4, Hkv=1, D=64), dict(Hq=8, Hkv=2, D=64, Lq=3)])
def test_time_grows_with_the_sequences_and_not_with_their_square(kw):
    log(f"many: {kw}")
    took = {}
    for B in (1 << 14, 1 << 17):
        big, want = many(B, **kw)
        same(call(big), want, B)
        took[B] = timed(big)
        log(f"  {B} sequences: {took[B]:.3f} ms")
    # 8 times the sequences: 8 times the time where it is linear, 64 times where it is not
    assert took[1 << 17] < 20 * took[1 << 14]
