"""decode_window over many query rows of a sequence (a prompt's chunk), large enough that its items of 256 rows serve it, against the
definition in 64 bits."""

import ctypes
import math

import pytest
import torch

from _cache8 import E4M3, problem, window64, window_bounds
from _step import DEV
from _util import log
from sunshape_amd import _native as N
from test_gpu_window import call, check, on_gpu

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def wide(pr, window=None, sinks=0):
    """The problem, seen to be one of the wide form: its workspace is that of partials of 256 rows."""
    B, Hq, Lq, D = pr["q"].shape
    P, Hkv, page, nb = pr["codes"].shape
    a = N.WindowArgs(window=window or 0, sinks=sinks, out_dtype=N.SSQ_BF16, num_pages=P)
    v8 = pr["v"].dtype == E4M3
    far = 1 << 32
    for k, v in dict(q=far, q_dtype=N.DTYPE_CODE[pr["q"].dtype], batch=B, num_q_heads=Hq, q_len=Lq, head_dim=D, num_kv_heads=Hkv, perm=far,
                     cent=far, block_dim=D // nb, n_blocks=nb, n_centroids=256, layout=N.SSQ_PAGED, seq_len=pr["block_table"].shape[1] * page,
                     codes=far, c_st=nb, block_table=far, seq_lens=far, page_size=page, v=far, v_dtype=N.SSQ_E4M3 if v8 else
                     N.DTYPE_CODE[pr["v"].dtype], value_dim=D, v_st=page, out=far).items():
        setattr(a.dec, k, v)
    a.v_scale = far if v8 else None
    items = B * ((Hq // Hkv * Lq + 255) // 256)
    cus = torch.cuda.get_device_properties(DEV).multi_processor_count
    want = Hkv * max(cus // Hkv, 1) * 2 * 256 * (D + 2) * 4 + items * 8
    assert N.lib().ssq_decode_window_workspace_size(ctypes.byref(a)) == want
    return pr


def chunk(seed, D=128, **kw):
    return problem(seed, B=1, Hq=256, Hkv=64, D=D, Lq=64, T=1900, **kw)


@pytest.mark.parametrize("D, bd, vt, qt", [(128, 4, E4M3, BF), (128, 2, BF, F16), (128, 8, F16, F32), (128, 4, BF, F32), (128, 2, E4M3, F16),
                                           (64, 4, BF, BF), (64, 2, F16, F32), (64, 8, E4M3, F16), (64, 4, E4M3, F32)])
def test_types_and_codecs(D, bd, vt, qt):
    log(f"wide: D {D} bd {bd} {vt} {qt}")
    check(wide(chunk(D + bd, D, bd=bd, vt=vt, qt=qt)))


@pytest.mark.parametrize("page, vt", [(16, E4M3), (64, BF), (256, E4M3)])
def test_ragged_windows(page, vt):
    """Groups of fewer rows than 256, sequences shorter than the chunk and empty ones, windows and sinks; 7 heads a KV head, so that
    groups begin inside a token's."""
    log(f"wide: ragged, pages of {page}, {vt}")
    for window, sinks in ((3000, 70), (3001, 0)):
        pr = problem(page, B=5, Hq=14, Hkv=2, D=64, Lq=300, T=9000, lens=[9000, 4501, 250, 0, 300], page=page, vt=vt)
        check(wide(pr, window, sinks), window, sinks)


def test_a_long_context_is_split():
    log("wide: 16,384 tokens")
    check(wide(problem(41, B=1, Hq=14, Hkv=2, D=64, Lq=300, T=16384, lens=[16381])))
    check(wide(problem(42, B=6, Hq=32, Hkv=8, D=128, Lq=64, T=4000)))


def test_what_no_row_sees_may_be_anything():
    window, sinks, Lq = 1700, 20, 64
    for vt in (E4M3, BF):
        log(f"wide: garbage {vt}")
        pr = chunk(43, vt=vt)
        wide(pr)
        n = int(pr["seq_lens"][0])
        seen = torch.zeros(pr["block_table"].shape[1] * 16, dtype=torch.bool)
        j = torch.arange(n)
        seen[:n] = (j > n - Lq - window) | (j < sinks)
        bad = {k: t.clone() if torch.is_tensor(t) else t for k, t in pr.items()}
        raw = bad["v"].view(torch.uint8) if vt == E4M3 else bad["v"]
        used = set()
        for c in range(bad["block_table"].shape[1]):
            s = seen[16 * c:16 * c + 16]
            if not s.any():
                bad["block_table"][0, c] = (-1, 2 ** 31 - 1, -2 ** 31)[c % 3]
                continue
            pg = int(bad["block_table"][0, c])
            used.add(pg)
            raw[pg][:, :, ~s] = 0x7F if vt == E4M3 else math.nan
            bad["codes"][pg][:, ~s] = 255
        for pg in set(range(len(raw))) - used:
            raw[pg] = 0xFF if vt == E4M3 else math.inf
            if vt == E4M3:
                bad["v_scale"][pg] = math.nan
        check(pr, window, sinks, gp=on_gpu(bad))


@pytest.mark.parametrize("vt", [E4M3, BF, F16])
def test_infinite_and_nan_values_reach_the_rows_that_see_them(vt):
    """One value a KV head, at a token that all, some or only the newest rows see; the other rows' bits are those without it."""
    log(f"wide: infinities and NaN, {vt}")
    window, sinks, Lq, n = 1750, 3, 64, 1900
    pr = wide(chunk(44, vt=vt, lens=[n]), window, sinks)
    bad = dict(pr)
    bad["v"] = pr["v"].clone()
    toks = [n - 1, n - 2, n - 33, n - Lq, n - Lq - 1, n - 700, n - Lq - window + 1, n - Lq - window + 40, n - window, 1, 100]
    kinds = (math.nan,) if vt == E4M3 else (math.nan, math.inf, -math.inf)
    at = {}
    for h in range(64):
        tok, dim, x = toks[h % len(toks)], (37 * h) % 128, kinds[h // len(toks) % len(kinds)]
        at[h] = tok, dim, x
        pg = int(pr["block_table"][0, tok // 16])
        if vt == E4M3:
            bad["v"].view(torch.uint8)[pg, h, dim, tok % 16] = (0x7F, 0xFF)[h % 2]
        else:
            bad["v"][pg, h, dim, tok % 16] = x
    zero = dict(pr)
    zero["v"] = pr["v"].clone()
    for h, (tok, dim, x) in at.items():
        zero["v"].view(torch.uint8 if vt == E4M3 else torch.int16)[int(pr["block_table"][0, tok // 16]), h, dim, tok % 16] = 0
    out, lse = (t.cpu() for t in call(on_gpu(bad), window, sinks))
    good, gl = (t.cpu() for t in call(on_gpu(zero), window, sinks))
    assert torch.equal(lse, gl) and torch.isfinite(good).all()
    p = n - Lq + torch.arange(Lq)
    for h, (tok, dim, x) in at.items():
        hit = (tok <= p) & ((tok > p - window) | (tok < sinks))
        for g in range(4 * h, 4 * h + 4):
            got, want = out[0, g], good[0, g].clone()
            want[hit, dim] = x
            assert torch.equal(got.nan_to_num(nan=1e30), want.nan_to_num(nan=1e30)), (h, tok, dim, x)
    # both infinities of a dim cancel to NaN where a row sees both
    if vt != E4M3:
        both = dict(pr)
        both["v"] = pr["v"].clone()
        for tok, x in ((n - 1, math.inf), (n - 5, -math.inf)):
            both["v"][int(pr["block_table"][0, tok // 16]), 0, 9, tok % 16] = x
        out = call(on_gpu(both), window, sinks)[0].cpu()[0, :4, :, 9]
        assert torch.isfinite(out[:, :-5]).all() and (out[:, -5:-1] == -math.inf).all() and torch.isnan(out[:, -1]).all()


def test_queries_that_are_not_finite():
    pr = wide(chunk(45))
    good = [t.cpu() for t in call(on_gpu(pr))]
    for x in (math.nan, -math.inf):
        log(f"wide: a query of {x}")
        bad = dict(pr)
        bad["q"] = pr["q"].clone()
        bad["q"][0, 6, 11, 7] = x
        out, lse = (t.cpu() for t in call(on_gpu(bad)))
        assert torch.isnan(out[0, 6, 11]).all()
        keep = torch.ones(256, 64, dtype=torch.bool)
        keep[6, 11] = False
        assert torch.equal(out[0][keep], good[0][0][keep]) and torch.equal(lse[0][keep], good[1][0][keep])


def test_scales_far_apart():
    """Page scales 2^-40 to 2^40, and pages that some rows of a group do not see 2^80 times the others."""
    log("wide: scales")
    check(wide(chunk(46, spread=40)))
    pr = chunk(47, spread=0, lens=[1900])
    for tok in (1899, 1900 - 64 - 1750 + 1):
        pr["v_scale"][int(pr["block_table"][0, tok // 16])] = 2.0 ** 80
    out, lse = (t.cpu().double() for t in call(on_gpu(wide(pr, 1750, 0)), 1750, 0))
    ref, rl, mag, pv = window64(pr, 1750, 0)
    ob, lb = window_bounds(pr, ref, rl, mag, pv, BF)
    # A weight with its page's scale is rounded to f16, in units in which the row's largest weight is at least 2^14 and the
    # largest scale that it sees is 1: a token's is off by half of f16's smallest step (2^-25) at the least, and its value by up to 448
    # times that.  So a row that sees 2^80 is exact to 1,750 * 2^-25 / 2^14 * 448 * 2^80 < 2^61 (rows that see one token of such
    # a page have dims in which that token is 0), the others to less than the bound has.
    p = 1900 - 64 + torch.arange(64)
    far = (p >= 1888) | (p - 1750 < 95)
    ob = ob + torch.where(far, 2.0 ** 61, 0.0)[None, None, :, None]
    assert ((out - ref).abs() <= ob).all() and ((lse - rl).abs() <= lb).all()
    assert (~far).any() and (ref[:, :, ~far].abs() < 1e6).all()


def test_logits_far_apart():
    log("wide: gains")
    check(wide(chunk(48, gain=1e-6, qt=F32)))
    pr = wide(chunk(48, gain=40.0, qt=F32))
    out, lse = (t.cpu().double() for t in call(on_gpu(pr)))
    ref, rl, mag, pv = window64(pr)
    ob, lb = window_bounds(pr, ref, rl, mag, pv, F32)
    # Weights down to e^-200 of the largest: in f16, with the largest at 2^14 or more, one is off by up to half of the smallest step
    # (2^-25) whatever its size, 2^-39 of the largest; a dim in which the tokens that count hold 0 shows it.  Values are at
    # most 448 * 2^3.
    ob = ob + 1900 * 2.0 ** -39 * 448 * 8
    assert ((out - ref).abs() <= ob).all() and ((lse - rl).abs() <= lb).all()


def test_strides_graph_and_streams():
    log("wide: strides, a graph, a stream")
    pr = wide(problem(49, B=1, Hq=256, Hkv=64, D=64, Lq=64, T=1900, per_head=False))
    g = on_gpu(pr)
    want = check(pr, gp=g)
    apart = torch.zeros(1, 256, 64, 64, 2, dtype=BF, device=DEV)
    apart[..., 0] = g["q"]
    odd = torch.zeros(1, 256, 64, 65, dtype=BF, device=DEV)
    odd[..., 1:] = g["q"]
    for q in (apart[..., 0], odd[..., 1:]):
        got = call({**g, "q": q})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = call(g)
    b = call(g)
    torch.cuda.synchronize()
    assert torch.equal(a[0], want[0]) and torch.equal(b[0], want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = call(g)
    for n in (1900, 700, 0, 1899):
        g["seq_lens"].fill_(n)
        graph.replay()
        got = out.clone(), lse.clone()
        eager = call(g)
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
