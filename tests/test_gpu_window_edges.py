"""The 8-bit cache's operators where calls are large, far apart or odd: offsets past 32 bits, more heads than compute units, many
query rows, one page read often, pages that overlap."""

import pytest
import torch

from _cache8 import E4M3, problem, window64, window_bounds
from _util import log
from sunshape_amd import hip_ops

pytestmark = pytest.mark.gpu
DEV, BF = torch.device("cuda"), torch.bfloat16


def far(t, stride):
    """t's pages `stride` elements apart, the last ones more than 4 GiB from the first."""
    n = t.shape[0]
    assert (n - 1) * stride * t.element_size() > 1 << 32
    buf = torch.empty((n - 1) * stride + t[0].numel(), dtype=t.dtype, device=DEV)
    inner = torch.empty(t.shape[1:], dtype=t.dtype, device="meta").stride()
    return buf.as_strided(t.shape, (stride, *inner))


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def fill(dst, src):
    for i in range(src.shape[0]):
        dst[i].view(torch.uint8).copy_(src[i].view(torch.uint8))


def run(gp, **kw):
    pr = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in gp.items()}
    return hip_ops.decode_window(pr["q"], pr["codes"], pr["v"], pr["perm"], pr["cent"], block_table=pr["block_table"],
                                 seq_lens=pr["seq_lens"], scale=pr["scale"], v_scale=pr["v_scale"], return_lse=True, **kw)


@pytest.mark.parametrize("vt", [E4M3, BF])
def test_offsets_past_32_bits(vt):
    log(f"offsets past 32 bits, {vt}")
    pr = problem(31, B=1, Hq=8, Hkv=2, D=128, Lq=3, T=150, vt=vt)
    gp = {k: v.to(DEV) if torch.is_tensor(v) else v for k, v in pr.items()}
    near = run(gp, window=100, sinks=20)
    wide = dict(gp, codes=far(gp["codes"], (1 << 31) - (1 << 20)), v=far(gp["v"], (1 << 30) - (1 << 20)))
    fill(wide["codes"], gp["codes"])
    fill(wide["v"], gp["v"])
    for a, b in zip(near, run(wide, window=100, sinks=20)):
        assert torch.equal(a, b)
    # the same pools taken as a copy's, and an append's
    n = gp["codes"].shape[0]
    src, dst = torch.tensor([0, 1], device=DEV), torch.tensor([n - 1, n - 2], device=DEV)
    for pools in ([gp["codes"], gp["v"]], [wide["codes"], wide["v"]]):
        hip_ops.copy_pages(pools, src, dst)
    if vt == E4M3:
        v = torch.randn(1, 2, 40, 128, device=DEV).to(BF)
        slots = (torch.arange(40, device=DEV) + (n - 3) * 16)[None]
        scale = gp["v_scale"].clone()
        hip_ops.append_values(v, gp["v"], gp["v_scale"], slots)
        hip_ops.append_values(v, wide["v"], scale, slots)
        assert torch.equal(scale, gp["v_scale"])
        k = torch.randn(1, 2, 40, 128, device=DEV).to(BF)
        for pools, sc in ((gp, gp["v_scale"]), (wide, scale)):
            hip_ops.append_kv(k, v, gp["perm"], gp["cent"], codes_out=pools["codes"], v_out=pools["v"], slot_mapping=slots, v_scale=sc)
        assert torch.equal(scale, gp["v_scale"])
    for i in range(n):
        assert same_bits(gp["codes"][i], wide["codes"][i]) and same_bits(gp["v"][i], wide["v"][i])


@pytest.mark.parametrize("Hkv, lens", [(300, [40]), (300, [700, 3])])
def test_more_heads_than_compute_units(Hkv, lens):
    log(f"{Hkv} KV heads, lengths {lens}")
    pr = problem(32, B=len(lens), Hq=Hkv, Hkv=Hkv, D=64, T=max(lens), lens=lens, bd=8)
    out, lse = run(pr)
    ref, rl, mag, pv = window64(pr)
    ob, lb = window_bounds(pr, ref, rl, mag, pv, out.dtype)
    assert ((out.cpu().double() - ref).abs() <= ob).all()
    assert ((lse.cpu().double() - rl).abs() <= lb).all()


@pytest.mark.parametrize("vt", [E4M3, BF])
def test_a_long_chunk(vt):
    """2,500 newest tokens at once, of sequences that are longer, as long and shorter."""
    log(f"a long chunk, {vt}")
    pr = problem(33, B=3, Hq=4, Hkv=2, D=64, Lq=2500, T=2801, lens=[2801, 2500, 17], vt=vt)
    for kw in ({}, dict(window=130, sinks=5)):
        out, lse = run(pr, **kw)
        ref, rl, mag, pv = window64(pr, kw.get("window"), kw.get("sinks", 0))
        ob, lb = window_bounds(pr, ref, rl, mag, pv, out.dtype)
        assert ((out.cpu().double() - ref).abs() <= ob).all()
        got = lse.cpu().double()
        seen = torch.isfinite(rl)
        assert torch.equal(torch.isfinite(got), seen) and ((got - rl).abs() <= lb)[seen].all()


def test_one_page_read_often():
    """Sequences and places of a table may share pages, and one page may be copied to many."""
    pr = problem(34, B=6, Hq=8, Hkv=2, D=64, T=90)
    pr["block_table"][:] = 2
    pr["seq_lens"][:] = torch.tensor([90, 90, 1, 0, 33, 90])
    out, lse = run(pr)
    ref, rl, mag, pv = window64(pr)
    ob, _ = window_bounds(pr, ref, rl, mag, pv, out.dtype)
    assert ((out.cpu().double() - ref).abs() <= ob).all()
    pools = [t.to(DEV) for t in (pr["codes"], pr["v"], pr["v_scale"])]
    n = pools[0].shape[0]
    hip_ops.copy_pages(pools, torch.full((n - 1,), 2, device=DEV), torch.tensor([i for i in range(n) if i != 2], device=DEV))
    for t in pools:
        raw = t.view(torch.uint8)
        assert (raw == raw[2:3]).all()


def test_written_pages_that_overlap_are_refused():
    z = lambda *s, dt=torch.uint8: torch.zeros(*s, dtype=dt, device=DEV)  # noqa: E731
    one = z(1, dt=torch.int64)
    for bad in (z(1, 8).expand(4, 8), z(64).as_strided((4, 8), (4, 1))):
        with pytest.raises(RuntimeError, match="overlap"):
            hip_ops.copy_pages([z(4, 8)], one, one, into=[bad])
    hip_ops.copy_pages([z(1, 8).expand(4, 8)], one, one, into=[z(4, 8)])  # what is read may
    v, slots = z(1, 2, 1, 64, dt=BF), z(1, 1, dt=torch.int64)
    pages, scale = z(4, 2, 64, 16).view(E4M3), z(4, 2, dt=torch.float32)
    for p, s in ((pages, scale[:, :1].expand(4, 2)), (pages, scale[:1].expand(4, 2)), (pages[:1].expand(4, 2, 64, 16), scale),
                 (pages[:, :1].expand(4, 2, 64, 16), scale)):
        with pytest.raises(RuntimeError, match="memory of their own"):
            hip_ops.append_values(v, p, s, slots)


@pytest.mark.parametrize("window, sinks", [(None, 0), (40, 0), (40, 9)])
@pytest.mark.parametrize("T", [90, 5000])
def test_a_rows_scales_are_those_of_the_pages_it_sees(T, window, sinks):
    """Pages that some of the rows that share a tile do not see (yet, or any longer) have scales 2^80 times the others'."""
    log(f"scales that some rows see: {T} tokens, window {window}, sinks {sinks}")
    pr = problem(35, B=2, Hq=4, Hkv=2, D=64, Lq=24, T=T, lens=[T, T - 5], spread=0)
    for b in range(2):
        n = int(pr["seq_lens"][b])
        pr["v_scale"][pr["block_table"][b, (n - 1) // 16].long()] = 2.0 ** 80
        if window:  # the page that the first rows' windows begin in
            pr["v_scale"][pr["block_table"][b, (n - 24 - window + 1) // 16].long()] = 2.0 ** 80
    out, lse = run(pr, window=window, sinks=sinks)
    ref, rl, mag, pv = window64(pr, window, sinks)
    ob, lb = window_bounds(pr, ref, rl, mag, pv, out.dtype)
    assert ((out.cpu().double() - ref).abs() <= ob).all()
    assert ((lse.cpu().double() - rl).abs() <= lb).all()
    assert ref.abs().amax() > 1e20 and ref.abs().amin() < 1e6
