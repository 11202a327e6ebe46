"""decode_window over very many short sequences, against the same few sequences by themselves."""

import pytest
import torch

from _cache8 import problem, window64, window_bounds
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


@pytest.mark.parametrize("B, kw", [(1 << 11, dict(Hq=32, Hkv=8, D=64, Lq=40)), (1 << 20, dict(Hq=16, Hkv=1, D=64, Lq=5))])
def test_very_many_rows(B, kw):
    """Items of 256 rows of thousands of sequences, and 84 million query rows, 2^32 threads and more where they are joined: every
    repetition of the 8 sequences has the same bits, and those are right."""
    log(f"many: {B} sequences, {kw}")
    big, _ = many(B, **kw)
    got = call(big)
    same(got, [t[:8] for t in got], B)
    pr = {k: v[:8].cpu() if k in ("q", "block_table", "seq_lens") else v.cpu() if torch.is_tensor(v) else v for k, v in big.items()}
    out, lse = (t[:8].cpu().double() for t in got)
    ref = window64(pr)
    ob, lb = window_bounds(pr, *ref, got[0].dtype)
    seen = ref[1] != -torch.inf
    assert (out[~seen] == 0).all() and (lse[~seen] == -torch.inf).all()
    assert ((out - ref[0]).abs() <= ob)[seen].all() and ((lse - ref[1]).abs() <= lb)[seen].all()
