"""append_values, append_kv's 8-bit values and copy_pages against plain forms: every bit of the pages and scales."""

import math

import pytest
import torch

from _cache8 import E4M3, same_values, values_plain
from _step import DEV, codec_arrays
from _util import log
from sunshape_amd import hip_ops

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def pages_of(g, P, H, D, page, empty=False):
    v = (torch.randn(P, H, D, page, generator=g) * 64).clamp(-448, 448).to(E4M3)
    s = torch.exp2(torch.randint(-9, -4, (P, H), generator=g).float())
    if empty:
        v.view(torch.uint8).zero_()
        s.zero_()
    return v, s


def run(v, pages, scale, slots):
    gp, gs = pages.to(DEV), scale.to(DEV)
    hip_ops.append_values(v.to(DEV), gp, gs, slots.to(DEV))
    return gp.cpu(), gs.cpu()


def check(v, pages, scale, slots):
    want = values_plain(v, pages, scale, slots)
    got = run(v, pages, scale, slots)
    assert torch.equal(got[1], want[1])
    assert same_values(got[0], want[0])
    # nothing but the pages' earlier tokens and the new ones was touched, bits included
    P, page = len(pages), pages.shape[3]
    hit = torch.zeros(P, page, dtype=torch.bool)
    for x in slots.flatten().tolist():
        if 0 <= x < P * page:
            hit[x // page, x % page] = True
    rest = torch.ones(P, page, dtype=torch.bool)
    for pg in range(P):
        if hit[pg].any():
            rest[pg, :int(hit[pg].nonzero()[0])] = False  # may be rescaled
    rest &= ~hit
    a, b = got[0].view(torch.uint8).permute(0, 3, 1, 2), pages.view(torch.uint8).permute(0, 3, 1, 2)
    assert torch.equal(a[rest], b[rest])
    return got


def slots_of(g, B, S, P, page, pad=0.0, first=None):
    """Tokens of B sequences in distinct pages, padding between a sequence's tokens."""
    per = (S + page - 1) // page + 1
    assert B * per <= P
    table = torch.randperm(P, generator=g)[:B * per].view(B, per)
    start = torch.randint(0, page, (B, 1), generator=g) if first is None else torch.full((B, 1), first)
    live = torch.rand(B, S, generator=g) >= pad
    at = start + live.long().cumsum(1) - 1
    return torch.where(live, table.gather(1, at.clamp_min(0) // page) * page + at % page, -1 - torch.randint(0, 9, (B, S), generator=g))


@pytest.mark.parametrize("dt", [BF, F16, F32])
@pytest.mark.parametrize("H, D", [(1, 64), (2, 64), (3, 64), (8, 128), (2, 128), (1, 2), (3, 7), (2, 96), (1, 257), (2, 300)])
def test_steps_and_chunks(dt, H, D):
    g = torch.Generator().manual_seed(H * D)
    for B, S, page, pad in ((5, 1, 16, 0.0), (3, 5, 16, 0.4), (2, 50, 16, 0.0), (2, 131, 16, 0.3), (1, 100, 32, 0.0), (2, 90, 64, 0.5),
                            (1, 300, 256, 0.0)):
        log(f"values: {dt} H {H} D {D} B {B} S {S} page {page} pad {pad}")
        P = B * ((S + page - 1) // page + 1) + 2
        pages, scale = pages_of(g, P, H, D, page)
        v = (torch.randn(B, S, H, D, generator=g) * 10 ** float(torch.randn((), generator=g))).to(dt).transpose(1, 2)
        check(v, pages, scale, slots_of(g, B, S, P, page, pad))


@pytest.mark.parametrize("page", [16, 32, 48])
def test_every_offset_and_length(page):
    g = torch.Generator().manual_seed(page)
    H, D = 2, 64
    for first in range(page):
        for n in sorted({1, 2, 3, 4, 5, 15, 16, 17, page - first, page}):
            P = (first + n + page - 1) // page + 1
            pages, scale = pages_of(g, P, H, D, page)
            v = torch.randn(1, H, n, D, generator=g).to(BF)
            slots = (first + torch.arange(n))[None]
            if first % 5 == 0 and n == 5:
                log(f"values: page {page} offset {first}")
            check(v, pages, scale, slots)


def test_a_page_filled_token_by_token():
    """Scales only grow while a page fills, every token is within half a step of e4m3 (or of its subnormals) of what it was,
    twice where the scale grew; a page that starts over forgets its old scale."""
    g = torch.Generator().manual_seed(2)
    H, D, page = 2, 128, 16
    pages, scale = pages_of(g, 4, H, D, page)
    gp, gs = pages.to(DEV), scale.to(DEV)
    toks = [torch.randn(1, H, 1, D, generator=g).mul(4.0 ** (i - 8)).to(BF) for i in range(16)]
    last = torch.zeros(H)
    for i, t in enumerate(toks):
        hip_ops.append_values(t.to(DEV), gp, gs, torch.tensor([[2 * page + i]], device=DEV))
        now = gs[2].cpu()
        assert (now >= last).all()
        last = now
    got = gp[2].float().cpu() * gs[2].cpu()[:, None, None]
    for i, t in enumerate(toks):
        x = t[0, :, 0].float()
        err = (got[..., i] - x).abs()
        # one rounding: 2^-4 of the value or 2^-10 of the scale; rescaled ones lose at most as much again at the last scale
        assert (err <= x.abs() * 2.0 ** -4 + 2 * 2.0 ** -10 * last[:, None]).all(), i
    hip_ops.append_values((toks[0] * 1e-3).to(DEV), gp, gs, torch.tensor([[2 * page]], device=DEV))
    assert (gs[2].cpu() < last * 1e-3).all()


def test_edges_of_values():
    """Zeros, infinities, NaN, the largest and the smallest values, values at a border of the scale."""
    H, D, page = 1, 64, 16
    rows = []
    for fill in (0.0, math.nan, math.inf, -math.inf, 3.0e38, -3.0e38, 1e-38, 2.0 ** -100 * 448, 2.0 ** -100 * 449, 448.0, 448.5, 449.0, 896.0,
                 1.0, -1.75 * 256):
        r = torch.zeros(D)
        r[::2] = fill
        rows.append(r)
    for dt in (F32, BF):
        for i, r in enumerate(rows):
            for first in (0, 3):
                for other in (0.0, 1.0, math.nan):
                    log(f"values: edge {i} {dt} {first} {other}")
                    g = torch.Generator().manual_seed(i)
                    pages, scale = pages_of(g, 2, H, D, page)
                    v = torch.stack([r, torch.full((D,), other)])[None, None].to(dt)
                    check(v, pages, scale, torch.tensor([[first, first + 1]]))
    # memory as allocated: scales of 0 under a page that does not start at 0
    pages, scale = pages_of(torch.Generator(), 2, H, D, page, empty=True)
    check(torch.ones(1, H, 2, D).to(BF), pages, scale, torch.tensor([[5, 6]]))


def test_order_gaps_and_padding():
    """Offsets that skip, descend, or stand behind long padding; slots past the pages and far below 0."""
    g = torch.Generator().manual_seed(4)
    H, D, page, P = 2, 64, 16, 8
    v = torch.randn(1, H, 200, D, generator=g).to(BF)
    pages, scale = pages_of(g, P, H, D, page)
    for name, slots in (("gaps", torch.tensor([3, 5, 9, 10])), ("down", torch.tensor([9, 8, 7, 2])),
                        ("two pages down", torch.tensor([40, 39, 33, 17, 16, 31])),
                        ("behind padding", torch.cat((torch.tensor([18]), torch.full((150,), -1), torch.tensor([19, 20])))),
                        ("starts behind padding", torch.cat((torch.full((130,), -1), torch.tensor([64, 65, 66])))),
                        ("returns behind padding", torch.cat((torch.tensor([18]), torch.full((70,), -2 ** 60), torch.tensor([19, 33])))),
                        ("past the pages", torch.tensor([128, 2 ** 62, 5, 127])), ("none", torch.full((20,), -1))):
        log(f"values: {name}")
        check(v[:, :, :len(slots)], pages, scale, slots[None])


def test_strides_and_alignment():
    log("values: strides")
    g = torch.Generator().manual_seed(5)
    H, D, page, P = 2, 64, 16, 12
    v = torch.randn(2, H, 20, D, generator=g).to(BF)
    pages, scale = pages_of(g, P, H, D, page)
    slots = slots_of(g, 2, 20, P, page)
    want = run(v, pages, scale, slots)
    wide = torch.zeros(2, 20, H, D + 1, dtype=BF, device=DEV)  # odd strides: values load one by one
    wide[..., 1:] = v.transpose(1, 2).to(DEV)
    pool = torch.full((P, H + 1, D + 3, page), 9, dtype=torch.uint8, device=DEV).view(E4M3)
    pool.view(torch.uint8)[:, 1:, :D] = pages.view(torch.uint8).to(DEV)
    sc = torch.zeros(P, 5, device=DEV)
    sc[:, 1:5:2] = scale.to(DEV)
    sl = torch.full((2, 33), -1, device=DEV)
    sl[:, 7:27] = slots.to(DEV)
    hip_ops.append_values(wide[..., 1:].transpose(1, 2), pool[:, 1:, :D], sc[:, 1:5:2], sl[:, 7:27])
    assert torch.equal(pool.view(torch.uint8)[:, 1:, :D].cpu(), want[0].view(torch.uint8)) and torch.equal(sc[:, 1:5:2].cpu(), want[1])
    assert (pool.view(torch.uint8)[:, 0] == 9).all() and (pool.view(torch.uint8)[:, :, D:] == 9).all() and (sc[:, ::2] == 0).all()
    gp, gs = pages.to(DEV), scale.to(DEV)  # dims apart
    apart = torch.zeros(2, H, 20, D, 2, dtype=BF, device=DEV)
    apart[..., 0] = v.to(DEV)
    hip_ops.append_values(apart[..., 0], gp, gs, slots.to(DEV))
    assert torch.equal(gp.cpu().view(torch.uint8), want[0].view(torch.uint8))


@pytest.mark.parametrize("B, S, D, bd, nc", [(5, 1, 64, 4, 256), (3, 40, 128, 2, 256), (64, 1, 128, 4, 256), (1, 2100, 64, 8, 256), (2, 33, 64, 4, 300)])
def test_append_kv_writes_what_its_parts_write(B, S, D, bd, nc):
    """Codes are those of an append without values, values those of append_values; with rotation and norm on the way."""
    import numpy as np

    log(f"append 8: {B} {S} {D} {bd} {nc}")
    g = torch.Generator().manual_seed(S)
    H, page = 2, 16
    perm, cent, _, _ = codec_arrays(np.random.default_rng(S), H, D, bd, nc)
    P = B * ((S + page - 1) // page + 1) + 1
    pages, scale = pages_of(g, P, H, D, page)
    slots = slots_of(g, B, S, P, page, 0.2).to(DEV)
    k = torch.randn(B, S, H, D, generator=g).to(BF).to(DEV).transpose(1, 2)
    v = torch.randn(B, S, H, D, generator=g).to(BF).to(DEV).transpose(1, 2)
    cos, sin = hip_ops.rope_table(5000, D, device=DEV)
    pos = torch.randint(0, 5000, (B, S), generator=g).to(DEV)
    dt = hip_ops.index_dtype(nc)
    got = [torch.zeros(P, H, page, D // bd, dtype=dt, device=DEV) for _ in range(2)]
    turn = dict(cos=cos, sin=sin, positions=pos, k_weight=torch.ones(D, device=DEV, dtype=BF))
    perm, cent = perm.to(DEV), cent.to(DEV)
    gp, gs = pages.to(DEV), scale.to(DEV)
    hip_ops.append_kv(k, v, perm, cent, codes_out=got[0], v_out=gp, v_scale=gs, slot_mapping=slots, **turn)
    hip_ops.append_kv(k, None, perm, cent, codes_out=got[1], v_out=None, slot_mapping=slots, **turn)
    assert torch.equal(got[0], got[1])
    want = values_plain(v.cpu(), pages, scale, slots.cpu())
    assert torch.equal(gs.cpu(), want[1]) and same_values(gp.cpu(), want[0])


def test_graph_of_appends():
    """Captured once, replayed as the sequences grow."""
    import numpy as np

    log("append 8: graph")
    g = torch.Generator().manual_seed(9)
    B, H, D, page, P = 3, 2, 64, 16, 12
    perm, cent, _, _ = codec_arrays(np.random.default_rng(1), H, D, 4, 256)
    perm, cent = perm.to(DEV), cent.to(DEV)
    pages, scale = pages_of(g, P, H, D, page)
    gp, gs, codes = pages.to(DEV), scale.to(DEV), torch.zeros(P, H, page, D // 4, dtype=torch.uint8, device=DEV)
    k, v = (torch.zeros(B, H, 1, D, dtype=BF, device=DEV) for _ in range(2))
    slots = torch.full((B, 1), -1, device=DEV)

    def step():
        hip_ops.append_kv(k, v, perm, cent, codes_out=codes, v_out=gp, v_scale=gs, slot_mapping=slots)

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    want = (pages, scale)
    for i in range(20):
        new = torch.randn(B, H, 1, D, generator=g).mul(2.0 ** (i % 7)).to(BF)
        sl = torch.tensor([[(3 * b + i // 16) * page + i % 16] for b in range(B)])
        v.copy_(new)
        slots.copy_(sl)
        graph.replay()
        torch.cuda.synchronize()
        want = values_plain(new, *want, sl)
        assert torch.equal(gs.cpu(), want[1]) and same_values(gp.cpu(), want[0]), i


def test_values_refusals():
    log("values: refusals")
    g = torch.Generator().manual_seed(6)
    pages, scale = (t.to(DEV) for t in pages_of(g, 4, 2, 64, 16))
    v = torch.randn(1, 2, 3, 64).to(BF).to(DEV)
    slots = torch.tensor([[0, 1, 2]], device=DEV)
    before = pages.view(torch.uint8).clone(), scale.clone()
    for args, word in (((v.cpu(), pages, scale, slots), "device"), ((v, pages.float().to(BF), scale, slots), "float8"),
                       ((v, pages, scale.double(), slots), "v_scale"), ((v, pages, scale[:, :1], slots), "v_scale"),
                       ((v[:, :1], pages, scale, slots), "v_out"), ((v[..., :32], pages, scale, slots), "v_out"),
                       ((v.double(), pages, scale, slots), "dtype"), ((v, pages, scale, slots.int()), "int64"),
                       ((v, pages, scale, slots[:, :2]), "slot_mapping"), ((v, pages, scale, slots.cpu()), "slot_mapping"),
                       ((v[0], pages, scale, slots), "shape"), ((v, pages.view(torch.uint8)[..., :8].contiguous().view(E4M3), scale, slots), "multiple of 16"),
                       ((v, pages.view(torch.uint8).flatten()[16:16 + 3 * 2 * 64 * 16 + 1][1:].view(3, 2, 64, 16).view(E4M3), scale[:3], slots), "aligned")):
        with pytest.raises(RuntimeError, match=word):
            hip_ops.append_values(*args)
    import numpy as np

    perm, cent, _, _ = (t if not torch.is_tensor(t) else t.to(DEV) for t in codec_arrays(np.random.default_rng(1), 2, 64, 4, 256))
    codes = torch.zeros(4, 2, 16, 16, dtype=torch.uint8, device=DEV)
    kw = dict(codes_out=codes, slot_mapping=slots)
    for k in (dict(v_out=pages), dict(v_out=pages.float().to(BF), v_scale=scale), dict(v_out=None, v_scale=scale)):
        with pytest.raises(RuntimeError):
            hip_ops.append_kv(v, None if k["v_out"] is None else v, perm, cent, **kw, **k)
    assert torch.equal(pages.view(torch.uint8), before[0]) and torch.equal(scale, before[1]) and not codes.any()
    hip_ops.append_values(v[:, :, :0], pages, scale, slots[:, :0])
    assert torch.equal(pages.view(torch.uint8), before[0])


# ------------------------------------------------------------------------------------- copies
@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 500])
def test_copies(n):
    log(f"copy: {n} pages")
    g = torch.Generator().manual_seed(n)
    P = 2 * n + 3
    pools = [torch.randint(0, 256, s, generator=g, dtype=torch.int32).to(torch.uint8) for s in
             ((P, 2, 16, 16), (P, 2, 64, 16), (P, 8), (P, 4097), (P, 3), (P,), (P, 5, 0))]
    pools.append(torch.randn(P, 3, generator=g))
    order = torch.randperm(P, generator=g)
    src, dst = order[:n], order[n:2 * n]
    dev = [p.to(DEV) for p in pools]
    hip_ops.copy_pages(dev, src.to(DEV), dst.to(DEV))
    for p, d in zip(pools, dev):
        want = p.clone()
        want[dst] = p[src]
        assert torch.equal(d.cpu(), want)


def test_copies_between_pools_of_any_stride():
    log("copy: pools")
    g = torch.Generator().manual_seed(1)
    a = torch.randn(10, 2, 16, 5, generator=g).to(DEV)
    wide = torch.zeros(20, 2 * 16 * 5 + 7, device=DEV)
    b = wide[::2, 3:163].unflatten(1, (2, 16, 5))
    bits = torch.randint(0, 256, (10, 4, 16), generator=g, dtype=torch.int32).to(torch.uint8).to(DEV).view(E4M3)
    e = torch.zeros(10, 4, 16, dtype=torch.uint8, device=DEV).view(E4M3)
    src, dst = torch.tensor([0, 9, 4, 4, -1, 3, 10, 2], device=DEV), torch.tensor([3, 0, 1, 2, 4, -5, 5, 10], device=DEV)
    hip_ops.copy_pages([a, bits], src, dst, into=[b, e])
    for i, j in ((0, 3), (9, 0), (4, 1), (4, 2)):
        assert torch.equal(b[j], a[i]) and torch.equal(e.view(torch.uint8)[j], bits.view(torch.uint8)[i])
    assert not b[4:].any() and not e.view(torch.uint8)[4:].any() and not wide[1::2].any() and not wide[:, :3].any() and not wide[:, 163:].any()


def test_copy_refusals():
    log("copy: refusals")
    a = torch.zeros(4, 2, 16, device=DEV)
    i = torch.tensor([0], device=DEV)
    for args, kw, word in ((([], i, i), {}, "pools"), (([a] * 9, i, i), {}, "pools"), (([a.cpu()], i, i), {}, "device"),
                           (([a], i.int(), i.int()), {}, "int64"), (([a], i, torch.tensor([1, 2], device=DEV)), {}, "int64"),
                           (([a], i.cpu(), i), {}, "src and dst"), (([a.transpose(1, 2)], i, i), {}, "contiguous"),
                           (([a], i, i), dict(into=[a, a]), "pools"), (([a], i, i), dict(into=[a.double()]), "dtype"),
                           (([a], i, i), dict(into=[a[:, :1]]), "shape")):
        with pytest.raises(RuntimeError, match=word):
            hip_ops.copy_pages(*args, **kw)


def test_dims_that_share_memory_are_refused():
    """Written value dims have memory of their own, as written pages and heads do."""
    v, slots = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(1, 1, dtype=torch.int64, device=DEV)
    pages = torch.zeros(4, 2, 1, 16, dtype=torch.uint8, device=DEV).view(E4M3).expand(4, 2, 64, 16)
    with pytest.raises(RuntimeError, match="memory of their own"):
        hip_ops.append_values(v, pages, torch.zeros(4, 2, device=DEV), slots)
