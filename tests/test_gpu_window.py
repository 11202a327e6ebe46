"""decode_window against the definition in 64 bits: types, layouts, lengths from none to many, windows, sinks, garbage in
what no row sees, infinities and NaN, splits along long contexts, graphs and streams."""

import math

import pytest
import torch

from _cache8 import E4M3, problem, window64, window_bounds
from _step import DEV
from _util import log
from sunshape_amd import hip_ops

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def on_gpu(pr):
    return {k: t.to(DEV) if torch.is_tensor(t) else t for k, t in pr.items()}


def call(gp, window=None, sinks=0, **kw):
    g = dict(gp)
    return hip_ops.decode_window(g.pop("q"), g.pop("codes"), g.pop("v"), g.pop("perm"), g.pop("cent"), window=window, sinks=sinks,
                                 return_lse=True, **{**g, **kw})


def check(pr, window=None, sinks=0, gp=None, **kw):
    out, lse = call(gp if gp is not None else on_gpu(pr), window, sinks, **kw)
    ref = window64(pr, window, sinks)
    ob, lb = window_bounds(pr, *ref, out.dtype)
    o, l = out.cpu().double(), lse.cpu().double()
    empty = ref[1] == -math.inf
    assert (o[empty] == 0).all() and (l[empty] == -math.inf).all()
    seen = ~empty
    eo = ((o - ref[0]).abs() / ob)[seen]
    el = ((l - ref[1]).abs() / lb)[seen]
    log(f"  worst of the bound: out {float(eo.max()) if eo.numel() else 0:.3f} lse {float(el.max()) if el.numel() else 0:.3f}")
    assert not torch.isnan(o).any()
    assert (eo <= 1).all() and (el <= 1).all()
    return out, lse


@pytest.mark.parametrize("vt", [E4M3, BF, F16])
@pytest.mark.parametrize("qt", [BF, F16, F32])
@pytest.mark.parametrize("D, bd", [(64, 2), (64, 4), (64, 8), (128, 2), (128, 4), (128, 8)])
def test_types_and_codecs(vt, qt, D, bd):
    log(f"window: {vt} {qt} D {D} bd {bd}")
    pr = problem(D + bd, B=3, Hq=8, Hkv=2, D=D, T=333, bd=bd, vt=vt, qt=qt)
    check(pr)


@pytest.mark.parametrize("Hq, Hkv, Lq", [(1, 1, 1), (2, 2, 1), (7, 1, 1), (16, 1, 1), (8, 2, 2), (14, 2, 3), (24, 2, 5), (8, 8, 40),
                                         (32, 1, 1), (33, 3, 3), (40, 2, 7), (64, 8, 6)])
@pytest.mark.parametrize("vt", [E4M3, BF])
def test_heads_and_rows(Hq, Hkv, Lq, vt):
    log(f"window: heads {Hq}/{Hkv} rows {Lq} {vt}")
    check(problem(Hq * Lq, B=2, Hq=Hq, Hkv=Hkv, D=64, Lq=Lq, T=170, vt=vt), window=50, sinks=3)
    check(problem(Hq * Lq + 1, B=2, Hq=Hq, Hkv=Hkv, D=128, Lq=Lq, T=170, vt=vt))


@pytest.mark.parametrize("page", [16, 32, 64, 256])
@pytest.mark.parametrize("vt", [E4M3, F16])
def test_pages_and_lengths(page, vt):
    lens = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]
    log(f"window: pages of {page} {vt}")
    pr = problem(page, B=len(lens), Hq=4, Hkv=2, D=64, T=300, lens=lens, page=page, vt=vt, per_head=False)
    for window, sinks in ((None, 0), (1, 0), (1, 1), (16, 0), (17, 2), (64, 64), (65, 100), (1000, 5)):
        check(pr, window, sinks)


@pytest.mark.parametrize("Lq", [2, 5, 17, 40])
def test_newest_tokens_with_windows(Lq):
    """Every row its own window: lengths below, at and past the new tokens', windows smaller and larger than they."""
    lens = [0, 1, Lq - 1, Lq, Lq + 1, 70, 130, 257, 400]
    for vt in (E4M3, BF):
        log(f"window: {Lq} new tokens {vt}")
        pr = problem(Lq, B=len(lens), Hq=4, Hkv=1, D=64, Lq=Lq, T=400, lens=lens, vt=vt)
        for window, sinks in ((None, 0), (1, 0), (3, 1), (33, 0), (64, 17), (100, 70), (399, 1)):
            check(pr, window, sinks)


@pytest.mark.parametrize("vt", [E4M3, BF])
@pytest.mark.parametrize("T, B, kw", [(5000, 3, {}), (20000, 1, {}), (9000, 5, dict(window=2500, sinks=200)),
                                      (3333, 9, dict(window=3000)), (70001, 1, dict(window=70000, sinks=1))])
def test_long_contexts_are_split(T, B, kw, vt):
    log(f"window: {B} of {T} {kw} {vt}")
    pr = problem(T, B=B, Hq=8, Hkv=2, D=128, T=T, vt=vt)
    check(pr, **kw)


def test_many_items_of_all_lengths():
    """More (sequence, row group) items than a wave has lanes, cut into equal shares: some empty, some long."""
    import numpy as np

    rng = np.random.default_rng(5)
    lens = [int(x) for x in rng.integers(0, 30, 150)] + [4000, 0, 2600, 1, 0]
    rng.shuffle(lens)
    log("window: 155 sequences")
    check(problem(1, B=len(lens), Hq=2, Hkv=1, D=64, T=4000, lens=lens))
    lens = [3000, 10, 2000]
    log("window: 100 new tokens, 3 sequences, 8 rows a token")
    check(problem(2, B=3, Hq=8, Hkv=1, D=64, Lq=100, T=3000, lens=lens), window=700, sinks=9)


def test_scales_of_pages_far_apart():
    log("window: page scales 2^-40 to 2^40")
    check(problem(3, B=4, Hq=8, Hkv=2, D=128, T=700, spread=40))


def test_logits_far_apart():
    """Rows whose largest logit moves by hundreds from tile to tile, and tiny and huge queries and codewords."""
    for gain in (1e-6, 40.0):
        for qt in (BF, F32):
            log(f"window: gain {gain} {qt}")
            check(problem(4, B=2, Hq=8, Hkv=2, D=64, T=900, gain=gain, qt=qt))
    pr = problem(5, B=2, Hq=8, Hkv=2, D=64, T=900, qt=F32)
    a = check(pr)
    for s in (2.0 ** 40, 2.0 ** -40):  # powers of two move nothing but exponents
        log(f"window: codewords times {s}")
        b = check({**pr, "cent": pr["cent"] * s, "q": pr["q"] / s})
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_what_no_row_sees_may_be_anything():
    """NaN values and scales, any codes and any table entries behind the end and between sinks and window."""
    for vt in (E4M3, BF, F16):
        for Lq in (1, 4):
            pr = problem(6, B=3, Hq=8, Hkv=2, D=64, Lq=Lq, T=600, lens=[600, 333, 250], vt=vt)
            for window, sinks in ((70, 5), (100, 0), (33, 40)):
                log(f"window: garbage {vt} {Lq} {window} {sinks}")
                bad = {k: t.clone() if torch.is_tensor(t) else t for k, t in pr.items()}
                raw = bad["v"].view(torch.uint8) if vt == E4M3 else bad["v"]
                used = set()
                for b in range(3):
                    n = int(pr["seq_lens"][b])
                    seen = torch.zeros(bad["block_table"].shape[1] * 16, dtype=torch.bool)
                    j = torch.arange(n)
                    seen[:n] = (j > n - Lq - window) | (j < sinks)
                    for c in range(bad["block_table"].shape[1]):
                        s = seen[16 * c:16 * c + 16]
                        if not s.any():
                            bad["block_table"][b, c] = (-1, 2 ** 31 - 1, -2 ** 31)[c % 3]
                            continue
                        pg = int(bad["block_table"][b, c])
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
    Lq, n, window = 6, 200, 40
    pr = problem(7, B=1, Hq=4, Hkv=1, D=64, Lq=Lq, T=n, lens=[n], vt=vt)
    for tok in (n - 1, n - 3, n - Lq - window + 2, n - Lq - window + 4, n - 30):
        for x in ((math.nan,) if vt == E4M3 else (math.nan, math.inf)):
            log(f"window: {x} at token {tok} of {n}, {vt}")
            bad = dict(pr)
            bad["v"] = pr["v"].clone()
            pg = int(pr["block_table"][0, tok // 16])
            if vt == E4M3:
                bad["v"].view(torch.uint8)[pg, 0, 5, tok % 16] = 0x7F
            else:
                bad["v"][pg, 0, 5, tok % 16] = x
            out, lse = (t.cpu() for t in call(on_gpu(bad), window, 0))
            good, gl = (t.cpu() for t in call(on_gpu(pr), window, 0))
            p = n - Lq + torch.arange(Lq)
            hit = (tok <= p) & (tok > p - window)
            assert torch.equal(lse, gl)
            for i in range(Lq):
                want = good[0, :, i].clone()
                if hit[i]:
                    assert (~torch.isfinite(out[0, :, i, 5])).all()
                    want[:, 5] = out[0, :, i, 5]
                assert torch.equal(out[0, :, i].nan_to_num(1.5), want.nan_to_num(1.5)), i


def test_queries_and_codewords_that_are_not_finite():
    log("window: NaN and infinite queries, infinite codewords")
    pr = problem(8, B=2, Hq=4, Hkv=1, D=64, T=500, lens=[500, 100])
    good = [t.cpu() for t in call(on_gpu(pr))]
    for x in (math.nan, math.inf, -math.inf):
        bad = dict(pr)
        bad["q"] = pr["q"].clone()
        bad["q"][0, 2, 0, 7] = x
        out, lse = (t.cpu() for t in call(on_gpu(bad)))
        assert torch.isnan(out[0, 2]).all()
        keep = torch.ones(2, 4, dtype=torch.bool)
        keep[0, 2] = False
        assert torch.equal(out[keep], good[0][keep]) and torch.equal(lse[keep], good[1][keep])
    # a codeword of -inf against positive queries: tokens that hold it weigh nothing
    bad = dict(pr)
    bad["cent"], bad["q"] = pr["cent"].clone(), pr["q"].clone()
    blk = 3
    bad["cent"][0, blk, 9, 1] = -math.inf
    bad["q"][..., pr["perm"][0, blk * 4 + 1]] = 0.5
    out, lse = (t.cpu().double() for t in call(on_gpu(bad)))
    ref = dict(bad)
    ref["cent"] = bad["cent"].clone()
    ref["cent"][0, blk, 9, 1] = -1e9
    want = window64(ref)
    ob, lb = window_bounds(ref, *want, BF)
    exact = {**ref, "cent": pr["cent"]}
    _, _, mag, pv = window64(exact)  # the bound's logits: those of the tokens that count
    ob, lb = window_bounds(ref, want[0], want[1], mag, want[3], BF)
    assert ((out - want[0]).abs() <= ob).all() and ((lse - want[1]).abs() <= lb).all()


def test_strides_views_and_shared_codecs():
    log("window: strides")
    pr = problem(9, B=3, Hq=8, Hkv=2, D=64, Lq=2, T=400, per_head=False)
    want = call(on_gpu(pr), 90, 4)
    g = on_gpu(pr)
    P = len(pr["codes"])
    codes = torch.zeros(P, 4, 16, 32, dtype=torch.uint8, device=DEV)
    codes[:, 1:3, :, 8:24] = g["codes"]
    v = torch.zeros(P, 3, 80, 16, dtype=torch.uint8, device=DEV).view(E4M3)
    v.view(torch.uint8)[:, :2, :64] = g["v"].view(torch.uint8)
    sc = torch.zeros(P, 5, device=DEV)
    sc[:, 1:5:2] = g["v_scale"]
    q = torch.zeros(3, 8, 2, 96, dtype=BF, device=DEV)
    q[..., 16:80] = g["q"]
    table = torch.zeros(3, 60, dtype=torch.int32, device=DEV)
    table[:, 5:5 + g["block_table"].shape[1]] = g["block_table"]
    view = {**g, "codes": codes[:, 1:3, :, 8:24], "v": v[:, :2, :64], "v_scale": sc[:, 1:5:2], "q": q[..., 16:80],
            "block_table": table[:, 5:5 + g["block_table"].shape[1]]}
    got = call(view, 90, 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # query dims apart, a codebook at an odd address
    apart = torch.zeros(3, 8, 2, 64, 2, dtype=BF, device=DEV)
    apart[..., 0] = g["q"]
    cent = torch.zeros(g["cent"].numel() + 1, device=DEV)
    cent[1:] = g["cent"].flatten()
    got = call({**g, "q": apart[..., 0], "cent": cent[1:].view(g["cent"].shape)}, 90, 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # a codec per head that is the same for all
    got = call({**g, "cent": g["cent"].expand(2, *g["cent"].shape).contiguous(), "perm": g["perm"].expand(2, -1).contiguous()}, 90, 4)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("out_dtype", [BF, F16, F32])
def test_out_dtype_and_scale_none(out_dtype):
    log(f"window: out {out_dtype}")
    pr = {**problem(10, B=2, Hq=8, Hkv=2, D=64, T=300, gain=0.2), "scale": None}
    out, _ = check(pr, out_dtype=out_dtype)
    assert out.dtype == out_dtype


def test_rotated_codec():
    log("window: rotation")
    from sunshape_amd.hip_ops import transform_rows

    pr = problem(11, B=2, Hq=8, Hkv=2, D=64, T=300, per_head=False)
    g = on_gpu(pr)
    rot = torch.linalg.qr(torch.randn(64, 64, generator=torch.Generator().manual_seed(1)))[0].to(DEV)
    out, lse = call(g, 77, 2, rotation=rot)
    turned = transform_rows(g["q"], rot, scale=pr["scale"])
    ident = torch.arange(64)
    check({**pr, "q": turned.cpu(), "perm": ident, "scale": None}, 77, 2, out_dtype=BF)
    want = call({**g, "q": turned, "perm": ident.to(DEV), "scale": None}, 77, 2, out_dtype=BF)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_empty_calls():
    log("window: empty")
    pr = problem(12, B=2, Hq=8, Hkv=2, D=64, T=40)
    g = on_gpu(pr)
    out, lse = call({**g, "block_table": g["block_table"][:, :0]})
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = call({**g, "seq_lens": torch.zeros(2, dtype=torch.int32, device=DEV)})
    assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = call({**g, "seq_lens": torch.tensor([-5, -2 ** 31], dtype=torch.int32, device=DEV)})
    assert (out == 0).all() and (lse == -math.inf).all()
    none = {**g, "q": g["q"][:0], "block_table": g["block_table"][:0], "seq_lens": g["seq_lens"][:0]}
    assert call(none)[0].shape == (0, 8, 1, 64)
    assert call({**g, "q": g["q"][:, :, :0]})[0].shape == (2, 8, 0, 64)
    # lengths past the table end at it
    cut = call({**g, "seq_lens": torch.tensor([40, 1000], dtype=torch.int32, device=DEV)})
    assert not torch.isnan(cut[0]).any()


def test_graph_streams_and_repeats():
    """Captured once, replayed over lengths, tables and queries that change between replays, with the program's own
    work around them; another stream; every call repeats itself bit for bit."""
    for T, B in ((400, 4), (6000, 4)):
        log(f"window: graph {T}")
        prs = [problem(20 + i, B=B, Hq=8, Hkv=2, D=128, T=T) for i in range(3)]
        P = max(len(p["codes"]) for p in prs)
        g = on_gpu(prs[0])
        buf = {**g, "codes": torch.zeros(P, 2, 16, 32, dtype=torch.uint8, device=DEV),
               "v": torch.zeros(P, 2, 128, 16, dtype=torch.uint8, device=DEV).view(E4M3), "v_scale": torch.ones(P, 2, device=DEV)}

        def fill(p):
            p = on_gpu(p)
            n = len(p["codes"])
            buf["codes"][:n] = p["codes"]
            buf["v"].view(torch.uint8)[:n] = p["v"].view(torch.uint8)
            buf["v_scale"][:n] = p["v_scale"]
            for k in ("q", "cent", "perm", "block_table", "seq_lens"):
                buf[k].copy_(p[k])

        fill(prs[0])
        call(buf, 3000, 4)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(buf, 3000, 4)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = call(buf, 3000, 4)
        for p in prs + prs[:1]:
            fill(p)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            want = call(on_gpu(p), 3000, 4)
            # the same call over a larger pool: the same bits
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
            assert torch.equal(call(buf, 3000, 4)[0], out)
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            again = call(buf, 3000, 4)
        side.synchronize()
        assert torch.equal(again[0], out)


def test_refusals():
    log("window: refusals")
    pr = problem(13, B=2, Hq=8, Hkv=2, D=64, T=40)
    g = on_gpu(pr)
    for bad, word in (
            (dict(v_scale=None), "v_scale"), (dict(v=g["v"].float().to(BF)), "v_scale"), (dict(v_scale=g["v_scale"].double()), "v_scale"),
            (dict(v_scale=g["v_scale"][:, :1]), "v_scale"), (dict(v_scale=g["v_scale"].cpu()), "v_scale"),
            (dict(block_table=g["block_table"].long()), "int32"), (dict(seq_lens=g["seq_lens"].long()), "int32"),
            (dict(block_table=g["block_table"][:1]), "block_table"), (dict(seq_lens=g["seq_lens"][:1]), "seq_lens"),
            (dict(q=g["q"][:, :7]), "divisible"), (dict(q=g["q"].double()), "dtype"), (dict(q=g["q"].cpu()), "device"),
            (dict(codes=g["codes"].to(torch.int16)), "codes"), (dict(v=g["v"][:, :, :32]), "value_dim"),
            (dict(heavy=[True] + [False] * 15), "passthrough"), (dict(v=g["v"].float(), v_scale=None), "8 or 16 bits"),
            (dict(window=0), "window"), (dict(window=-3), "window"), (dict(sinks=-1), "sinks"), (dict(out_dtype=torch.float64), "dtype"),
            (dict(cent=torch.zeros(2, 16, 300, 4, device=DEV), codes=g["codes"].to(torch.int16)), "byte codes"),
            (dict(cent=torch.zeros(2, 64, 256, 1, device=DEV), codes=torch.zeros(len(g["codes"]), 2, 16, 64, dtype=torch.uint8, device=DEV)),
             "block_dim")):
        with pytest.raises(RuntimeError, match=word):
            call({**g, **{k: v for k, v in bad.items() if k not in ("window", "sinks")}}, bad.get("window"), bad.get("sinks", 0))
    small = problem(14, B=1, Hq=2, Hkv=1, D=64, T=40)
    s = on_gpu(small)
    with pytest.raises(RuntimeError, match="page sizes"):  # pages of 8
        call({**s, "codes": s["codes"][:, :, :8].contiguous(), "v": s["v"].view(torch.uint8)[..., :8].contiguous().view(E4M3)})
    with pytest.raises(RuntimeError, match="aligned"):
        odd = torch.zeros(s["codes"].numel() + 1, dtype=torch.uint8, device=DEV)
        call({**s, "codes": odd[1:].view(s["codes"].shape)})
