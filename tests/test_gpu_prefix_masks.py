"""Masks that hide a sequence's first own tokens (a sliding window, left padding, a tree of draft tokens) under
logits far below zero, where the exponentials of the scores themselves underflow: decode_prefix against 64 bits."""

import math

import pytest
import torch

from _util import log
from sunshape_amd import hip_ops
from test_gpu_decode_prefix import _call, _check, _dev, _problem

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _low(p, low):
    """Every logit moved by `low`: one dim of the queries is 8 (times 1 / sqrt(64): 1), the keys' is `low`."""
    G = p["q"].shape[1] // p["cent"].shape[0]
    for h in range(p["cent"].shape[0]):
        p["q"][:, h * G:(h + 1) * G, :, int(p["perm"][h, 0])] = 8.0
        p["cent"][h, 0, :, 0] = low
    return p


def _hide(p, first, low=0.0):
    """The first own tokens at -inf (a number, or one per sequence), the others at `low`."""
    B, Hq, Lq, _ = p["q"].shape
    m = torch.full((B, 1, Lq, p["table"].shape[1] * p["codes"].shape[2]), low)
    for b in range(B):
        m[b, :, :, :first if isinstance(first, int) else first[b]] = -math.inf
    p["own_mask"] = m
    return p


def _both(p, what):
    for kernel in (0, 1):
        out, lse = _call(p, kernel=kernel)
        _check(p, out, lse, f"{what}, kernel {kernel}")


# 32 query rows of a KV head: every column of a tile is a row
BASE = dict(B=4, Hq=64, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, lens=[70, 200, 33, 130])


@pytest.mark.parametrize("T", [0, 45])
@pytest.mark.parametrize("low", [-80.0, -95.0, -300.0])
@pytest.mark.parametrize("first", [32, 64, 96])
def test_hidden_tiles_before_low_logits(first, low, T):
    """32 and 64: the first tiles of the first piece; 96: the first piece and the next one's first tile."""
    log(f"decode_prefix: {first} tokens hidden, logits near {low}, prefix {T}")
    _both(_hide(_low(_problem(T=T, **BASE), low), first), "low keys")


@pytest.mark.parametrize("low", [-95.0, -300.0, -1e30])
def test_low_masks_after_hidden_tiles(low):
    log(f"decode_prefix: a mask of -inf, then of {low}")
    p = _hide(_problem(T=0, **BASE), 32, low)
    if low < -1e20:  # the logits vanish beside the mask: every token alike, to the mask's last bit
        p["q"] = torch.zeros_like(p["q"])
    _both(p, f"mask {low}")


@pytest.mark.parametrize("qdt, vdt", [(BF, BF), (F16, F16), (F32, BF), (F16, BF)])
@pytest.mark.parametrize("D, bd", [(64, 2), (64, 8), (128, 4)])
def test_types_and_codebooks(qdt, vdt, D, bd):
    log(f"decode_prefix: hidden tiles, {qdt} queries, {vdt} values, head_dim {D}, dims of {bd}")
    for T in (0, 33):
        p = _problem(T=T, qdt=qdt, vdt=vdt, **{**BASE, "D": D, "Dv": D, "bd": bd})
        _both(_hide(_low(p, -95.0 * math.sqrt(D) / 8), [32, 150, 0, 64]), "types")


@pytest.mark.parametrize("heavy", [(), (3, 9)])
def test_more_rows_than_a_tile(heavy):
    """42 query rows a sequence, each with its own window: some rows see a tile that others do not."""
    log(f"decode_prefix: windows of rows, heavy {heavy}")
    p = _low(_problem(B=3, Hq=28, Hkv=2, Lq=3, D=64, Dv=64, bd=4, nc=256, T=20, lens=[70, 200, 131], heavy=heavy), -95.0)
    B, Hq, Lq, _ = p["q"].shape
    m = torch.full((B, Hq, Lq, p["table"].shape[1] * 16), -math.inf)
    for h in range(Hq):
        for i in range(Lq):
            m[:, h, i, 16 * (h % 8) + 5 * i:16 * (h % 8) + 5 * i + 30] = 0.0
    p["own_mask"] = m
    _both(p, "windows")
    p["plen"].zero_()
    _both(p, "windows, no prefix")


def test_every_row_hidden_but_the_last_token():
    log("decode_prefix: the last token alone")
    p = _low(_problem(T=0, **BASE), -95.0)
    _both(_hide(p, [n - 1 for n in BASE["lens"]]), "last token")


def test_graph_replays_with_hidden_tiles():
    log("decode_prefix: hidden tiles in a graph")
    p = _hide(_low(_problem(T=45, **BASE), -95.0), 64)
    d = {k: _dev(p[k]) for k in ("codes", "v", "perm", "cent", "ptable", "plen", "table", "lens", "own_mask")}
    q = _dev(p["q"]).contiguous()

    def call():
        return hip_ops.decode_prefix(q, d["codes"], d["v"], d["perm"], d["cent"], scale=p["scale"], prefix_table=d["ptable"],
                                     prefix_len=d["plen"], block_table=d["table"], seq_lens=d["lens"], mask=d["own_mask"],
                                     return_lse=True)

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call()
    for first in (32, 64, 96, 0):
        d["own_mask"].zero_()[..., :first] = -math.inf
        want = call()
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), first


@pytest.mark.parametrize("kw", [dict(nc=4096), dict(D=256, Dv=256), dict(nc=64, bd=2, vdt=F32), dict(D=128, Dv=64), dict(bd=1, nc=16),
                                dict(D=128, Dv=128, heavy=tuple(range(20))), dict(page=8)])
def test_hidden_tiles_under_other_codecs(kw):
    """The forms that take the decode kernels by chunks of rows."""
    log(f"decode_prefix: hidden tiles, {kw}")
    for T in (0, 45):
        p = _problem(T=T, **{**BASE, "Hq": 8, **kw})
        _low(p, -95.0 * math.sqrt(p["q"].shape[-1]) / 8)
        out, lse = _call(_hide(p, [32, 96, 0, 64]))
        _check(p, out, lse, "other codecs")
