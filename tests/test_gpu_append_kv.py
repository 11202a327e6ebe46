"""Append of raw keys and values to the paged cache (hip_ops.append_kv): the pages hold what the rotated,
rounded keys encode to (the oracle's encode, bit for bit), their passthrough values and the values, and nothing
else changes."""

import math

import numpy as np
import pytest
import torch

from _step import DEV, codec_arrays, unsigned
from _util import log
from oracle import vq_oracle as O
from sunshape_amd import hip_ops

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _slots(rng, B, S, page, pages, pad, scattered):
    """Distinct slots: runs through a sequence's pages from a random offset, or one by one anywhere."""
    if scattered:
        flat = rng.permutation(pages * page)[:B * S].reshape(B, S)
    else:
        per = (S + page - 1) // page + 1
        table = rng.permutation(pages)[:B * per].reshape(B, per)
        at = rng.integers(0, page, (B, 1)) + np.arange(S)[None]
        flat = np.take_along_axis(table, at // page, 1) * page + at % page
    gone = rng.random((B, S)) < pad
    return np.where(gone, rng.choice([-1, -7, pages * page, 1 << 40], (B, S)), flat)


def _run(case, kernel=0, grid=False, pages_fill=None):
    (B, Hkv, S, D, Dv, bd, nc, page, dt, vdt, vpdt, rot, inter, norm, heavy, per_head, pad, scattered, metric) = case
    rng = np.random.default_rng(B * 7 + S * 13 + D + nc)
    g = torch.Generator().manual_seed(B + S + D)
    nb = D // bd
    perm, cent, mask, sigma = codec_arrays(rng, Hkv, D, bd, nc, per_head, heavy)
    k = (torch.randn(B, S, Hkv, D, generator=g) * torch.from_numpy(sigma).float()).to(dt).transpose(1, 2)
    v = torch.randn(B, S, Hkv, Dv, generator=g).to(vdt).transpose(1, 2)
    pages = B * ((S + page - 1) // page + 1) + 3
    slots = _slots(rng, B, S, page, pages, pad, scattered)
    cos = sin = pos = w = E = None
    if rot:
        cos, sin = hip_ops.rope_table(S + 40, rot)
        pos = torch.from_numpy(rng.integers(0, 40, (B, 1)) + np.arange(S)[None])
    if norm:
        w = torch.from_numpy(sigma * (1 + 0.1 * rng.standard_normal(D))).to(dt)
    if metric:
        E = torch.eye(D) + 0.2 * torch.randn(D, D, generator=g)
    idt = hip_ops.index_dtype(nc)
    codes0 = torch.randint(0, 100, (pages, Hkv, page, nb), generator=g, dtype=torch.int32).to(idt)
    v0 = torch.randn(pages, Hkv, Dv, page, generator=g).to(vpdt)
    pt0 = torch.randn(pages, Hkv, page, len(heavy), bd, generator=g).to(dt) if heavy else None

    def dev(t):
        if t is None:
            return None
        return t.transpose(1, 2).contiguous().to(DEV).transpose(1, 2) if t.dim() == 4 and t.stride(1) < t.stride(2) else t.to(DEV)

    c, vp, pt = codes0.to(DEV), v0.to(DEV), None if pt0 is None else pt0.to(DEV)
    direct = hip_ops.cdist_direct(S, nc)
    hip_ops.append_kv(dev(k), dev(v), perm.to(DEV), cent.to(DEV), codes_out=c, v_out=vp,
                      slot_mapping=torch.from_numpy(slots).to(DEV), heavy=mask, pt_out=pt, cos=dev(cos), sin=dev(sin),
                      positions=dev(pos), k_weight=dev(w), interleaved=inter, metric=dev(E), direct=direct, kernel=kernel,
                      grid=hip_ops.encode_grid(cent.to(DEV), Hkv) if grid else None)
    torch.cuda.synchronize()
    # the rotated keys, from the operator that test_gpu_rope checks against the formulas
    kr = k
    if rot or norm:
        kr = hip_ops.qk_norm_rope(dev(k), None, dev(cos), dev(sin), dev(pos), q_weight=dev(w), interleaved=inter)[0].cpu()
    return dict(perm=perm, cent=cent, mask=mask, kr=kr, v=v, slots=slots, pages=pages, codes0=codes0, v0=v0, pt0=pt0,
                codes=c.cpu(), vp=vp.cpu(), pt=None if pt is None else pt.cpu(), E=E, direct=direct)


def _check(case, r):
    (B, Hkv, S, D, Dv, bd, nc, page, dt, vdt, vpdt, *_rest) = case
    want_c, want_v = unsigned(r["codes0"]).clone(), r["v0"].clone()
    want_p = None if r["pt0"] is None else r["pt0"].clone()
    live = (r["slots"] >= 0) & (r["slots"] < r["pages"] * page)
    bb, ss = np.nonzero(live)
    sl = torch.from_numpy(r["slots"][bb, ss])
    pg, off = sl // page, sl % page
    for h in range(Hkv):
        perm = (r["perm"][h] if r["perm"].ndim == 2 else r["perm"]).numpy()
        cent = (r["cent"][h] if r["cent"].ndim == 4 else r["cent"]).numpy()
        keys = r["kr"][:, h][bb, ss].float().numpy()
        hv = None if r["mask"] is None else np.array(r["mask"])
        if len(keys):
            kw = dict(metric=r["E"].numpy()) if r["E"] is not None else {}
            codes, kept = O.encode(keys, perm, cent, hv, direct=r["direct"], **kw)
            want_c[pg, h, off] = torch.from_numpy(codes.astype(np.int64) % 65536 if nc <= 65535 else codes.astype(np.int64))
            if want_p is not None:
                want_p[pg, h, off] = torch.from_numpy(kept[:, hv]).to(dt)
            want_v[pg, h, :, off] = r["v"][:, h][bb, ss].to(vpdt)
    assert torch.equal(unsigned(r["codes"]), want_c), "codes"
    assert torch.equal(r["vp"], want_v), "values"
    if want_p is not None:
        assert torch.equal(r["pt"], want_p), "passthrough"


#        B, Hkv, S,  D,  Dv, bd, nc, page, k dtype, v dtype, page dtype, rot, inter, norm, heavy, per head, pad, scattered, metric
CASES = [
    (1, 1, 1, 64, 64, 4, 256, 16, BF, BF, BF, 64, False, True, (), True, 0.0, False, False),
    (64, 8, 1, 128, 128, 4, 256, 16, BF, BF, BF, 128, False, True, (), True, 0.0, False, False),
    (7, 2, 5, 64, 64, 2, 256, 16, BF, BF, BF, 64, False, True, (1, 4, 9, 30), True, 0.4, False, False),
    (3, 2, 40, 64, 64, 2, 64, 16, F16, F16, F16, 32, True, False, (), False, 0.2, True, False),
    (2, 2, 33, 64, 96, 8, 256, 8, BF, F32, BF, 64, False, True, (), True, 0.0, False, False),   # values converted
    (2, 1, 21, 64, 40, 4, 256, 16, BF, BF, F32, 64, False, True, (), True, 0.1, False, False),  # to 32 bits
    (2, 1, 70, 64, 130, 4, 256, 16, F32, F32, F32, 64, True, True, (), True, 0.0, False, False),
    (2, 3, 9, 48, 24, 3, 100, 5, BF, BF, BF, 16, False, True, (), True, 0.0, False, False),     # odd pages and dims
    (2, 1, 9, 64, 64, 16, 32, 16, BF, BF, BF, 0, False, True, (), True, 0.0, False, False),     # norm only
    (4, 2, 6, 64, 64, 1, 16, 16, BF, BF, BF, 64, False, False, (3,), True, 0.0, False, False),
    (4, 2, 6, 64, 64, 4, 16, 16, BF, BF, BF, 64, False, True, (), True, 0.0, False, False),     # <= 25 rows: direct distances
    (3, 2, 4, 64, 64, 4, 300, 16, BF, BF, BF, 64, False, True, (2,), True, 0.3, False, False),  # 16-bit codes
    (2, 2, 3, 128, 128, 4, 4096, 16, BF, BF, BF, 128, False, True, (), True, 0.0, False, False),
    (3, 2, 8, 64, 64, 4, 256, 16, BF, BF, BF, 64, False, True, (), True, 0.0, False, True),     # a block metric
    (2, 2, 100, 64, 64, 4, 256, 32, BF, BF, BF, 0, False, False, (), True, 0.2, False, False),  # keys as they come
    (1, 2, 64, 256, 256, 4, 256, 16, BF, BF, BF, 256, False, True, (), False, 0.0, False, False),
]
IDS = [f"case{i}" for i in range(len(CASES))]


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_one_launch(case):
    log(f"append {case}")
    _check(case, _run(case))


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_many_rows_path(case):
    """kernel 1 takes the path of many rows (values, rotation, then the exact scan)."""
    if hip_ops.cdist_direct(case[2], case[6]):
        pass  # served by the exact scan too
    log(f"append, many rows' path {case}")
    _check(case, _run(case, kernel=1))


BIG = [
    (1, 8, 3001, 128, 128, 4, 256, 16, BF, BF, BF, 128, False, True, (), True, 0.1, False, False),     # the tile screen
    (3, 2, 2000, 64, 64, 2, 256, 16, BF, BF, BF, 64, False, True, (1, 7), True, 0.1, False, False),
    (2, 2, 700, 64, 64, 4, 4096, 16, F16, F16, F16, 64, True, True, (), True, 0.1, False, False),      # 16-bit codes
    (2, 2, 1500, 64, 64, 2, 1024, 16, BF, BF, BF, 64, False, True, (3,), False, 0.1, True, False),     # the wide scan
]


@pytest.mark.parametrize("case", BIG, ids=[f"big{i}" for i in range(len(BIG))])
def test_large(case):
    log(f"append, large {case}")
    _check(case, _run(case))


def test_large_with_a_search_grid():
    case = BIG[1]
    log(f"append, search grid {case}")
    _check(case, _run(case, grid=True))


def test_encode_leaves_padded_rows_out():
    """ssq_encode's own paged output takes negative slots as padding, on every kernel."""
    log("encode: padded rows")
    rng = np.random.default_rng(4)
    for bd, nc, S, grid, kernel in ((4, 256, 40, False, 0), (2, 256, 40, True, 0), (2, 256, 40, True, 3), (4, 64, 40, False, 0),
                                    (4, 256, 40, False, 1), (4, 300, 40, False, 0), (4, 4096, 300, False, 0)):
        perm, cent, mask, sigma = codec_arrays(rng, 2, 64, bd, nc, True, (1,))
        nb, pages = 64 // bd, 2 * (S // 16 + 2)
        k = (torch.randn(2, 2, S, 64) * torch.from_numpy(sigma).float()).to(BF).to(DEV)
        slots = torch.from_numpy(_slots(rng, 2, S, 16, pages, 0.3, False)).to(DEV)
        slots = torch.where(slots >= pages * 16, -1, slots)
        c = torch.full((pages, 2, 16, nb), 77, dtype=hip_ops.index_dtype(nc), device=DEV)
        pt = torch.full((pages, 2, 16, 1, bd), 5.0, dtype=BF, device=DEV)
        gr = hip_ops.encode_grid(cent.to(DEV), 2) if grid else None
        hip_ops.encode(k, perm.to(DEV), cent.to(DEV), heavy=mask, codes_out=c, pt_out=pt, slot_mapping=slots, grid=gr, kernel=kernel)
        want, wpt = hip_ops.encode(k, perm.to(DEV), cent.to(DEV), heavy=mask, grid=gr, kernel=kernel)
        live = slots >= 0
        b, s = live.nonzero(as_tuple=True)
        wc, wp = torch.full_like(c, 77), torch.full_like(pt, 5.0)
        wc[slots[b, s] // 16, :, slots[b, s] % 16] = want[b, :, s]
        wp[slots[b, s] // 16, :, slots[b, s] % 16] = wpt[b, :, s]
        assert torch.equal(c, wc) and torch.equal(pt, wp), (bd, nc, kernel)


def test_all_padding_nothing_written_and_empty():
    log("append: all padding, empty")
    rng = np.random.default_rng(1)
    perm, cent, _, _ = codec_arrays(rng, 1, 64, 4, 256)
    k = torch.randn(2, 1, 3, 64, device=DEV, dtype=BF)
    for kernel in (0, 1):
        c = torch.full((4, 1, 16, 16), 9, dtype=torch.uint8, device=DEV)
        v = torch.full((4, 1, 64, 16), 3.0, dtype=BF, device=DEV)
        hip_ops.append_kv(k, k, perm.to(DEV), cent.to(DEV), codes_out=c, v_out=v, kernel=kernel,
                          slot_mapping=torch.full((2, 3), -1, dtype=torch.int64, device=DEV))
        hip_ops.append_kv(k[:, :, :0], k[:, :, :0], perm.to(DEV), cent.to(DEV), codes_out=c, v_out=v, kernel=kernel,
                          slot_mapping=torch.zeros(2, 0, dtype=torch.int64, device=DEV))
        hip_ops.append_kv(k, k, perm.to(DEV), cent.to(DEV), codes_out=c[:0], v_out=v[:0], kernel=kernel,
                          slot_mapping=torch.zeros(2, 3, dtype=torch.int64, device=DEV))
        assert (c == 9).all() and (v == 3).all()


def test_keys_alone_and_bad_positions():
    """Values may be left out; a position outside the tables gives the codes of a NaN key, and harms no other row."""
    log("append: keys alone, positions outside the tables")
    rng = np.random.default_rng(2)
    perm, cent, _, _ = codec_arrays(rng, 1, 64, 4, 256)
    k = torch.randn(1, 1, 4, 64, device=DEV, dtype=BF)
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(8, 64))
    slots = torch.arange(4, device=DEV)[None]
    got = []
    for pos in ([[0, 1, 2, 3]], [[0, 8, 2, -5]]):
        c = torch.zeros(1, 1, 16, 16, dtype=torch.uint8, device=DEV)
        hip_ops.append_kv(k, None, perm.to(DEV), cent.to(DEV), codes_out=c, v_out=None, slot_mapping=slots, cos=cos, sin=sin,
                          positions=torch.tensor(pos, device=DEV))
        got.append(c)
    assert torch.equal(got[0][0, 0, [0, 2]], got[1][0, 0, [0, 2]])


def test_strided_pages():
    """Pages inside a larger allocation (every other page of it), keys and values in different stride orders."""
    log("append: strided pages")
    rng = np.random.default_rng(3)
    perm, cent, _, _ = codec_arrays(rng, 2, 64, 4, 256)
    k = torch.randn(3, 2, 20, 64, device=DEV, dtype=BF)
    v = torch.randn(3, 20, 2, 64, device=DEV, dtype=BF).transpose(1, 2)
    slots = torch.from_numpy(_slots(rng, 3, 20, 16, 12, 0.0, False)).to(DEV)
    for kernel in (0, 1):
        c0, v0 = torch.zeros(12, 2, 16, 16, dtype=torch.uint8, device=DEV), torch.zeros(12, 2, 64, 16, dtype=BF, device=DEV)
        cw, vw = torch.zeros(24, 2, 16, 19, dtype=torch.uint8, device=DEV), torch.zeros(24, 2, 64, 17, dtype=BF, device=DEV)
        for c, vp in ((c0, v0), (cw[::2, :, :, 2:18], vw[1::2, :, :, 1:])):
            hip_ops.append_kv(k, v, perm.to(DEV), cent.to(DEV), codes_out=c, v_out=vp, slot_mapping=slots, kernel=kernel)
        assert torch.equal(cw[::2, :, :, 2:18], c0) and torch.equal(vw[1::2, :, :, 1:], v0)
        assert (cw[1::2] == 0).all() and (vw[::2] == 0).all() and (cw[..., :2] == 0).all() and (vw[..., 0] == 0).all()


def test_rotated_codec():
    """A codec in rotated mode: the position rotation first, rounded to the keys' dtype, then the codec's R."""
    log("append: rotated codec")
    g = torch.Generator().manual_seed(8)
    R = torch.linalg.qr(torch.randn(64, 64, generator=g))[0].to(DEV)
    perm, cent, _, _ = codec_arrays(np.random.default_rng(5), 2, 64, 4, 256)
    perm, cent = perm.to(DEV), cent.to(DEV)
    k = torch.randn(2, 2, 9, 64, generator=g).to(BF).to(DEV)
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(16, 64))
    pos = torch.arange(9, device=DEV)[None].expand(2, 9)
    slots = torch.arange(18, device=DEV).view(2, 9)
    a, b = (torch.zeros(2, 2, 16, 16, dtype=torch.uint8, device=DEV) for _ in range(2))
    vp = torch.zeros(2, 2, 64, 16, dtype=BF, device=DEV)
    hip_ops.append_kv(k, k, perm, cent, codes_out=a, v_out=vp, slot_mapping=slots, cos=cos, sin=sin, positions=pos, rotation=R)
    kr, _ = hip_ops.qk_norm_rope(k, None, cos, sin, pos)
    hip_ops.encode(kr, perm, cent, codes_out=b, slot_mapping=slots, rotation=R)
    assert torch.equal(a, b)


def test_refusals():
    log("append: refusals")
    rng = np.random.default_rng(6)
    perm, cent, _, _ = codec_arrays(rng, 2, 64, 4, 256)
    k = torch.zeros(2, 2, 3, 64, device=DEV, dtype=BF)
    base = dict(keys=k, values=k, perm=perm.to(DEV), cent=cent.to(DEV), codes_out=torch.zeros(4, 2, 16, 16, dtype=torch.uint8, device=DEV),
                v_out=torch.zeros(4, 2, 64, 16, dtype=BF, device=DEV), slot_mapping=torch.zeros(2, 3, dtype=torch.int64, device=DEV))
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(4, 64))
    bad = [
        (dict(keys=k[0]), "shape"), (dict(values=k[:, :1]), "value_states"), (dict(values=None), "together"),
        (dict(v_out=base["v_out"][:3]), "v_out"), (dict(v_out=base["v_out"].transpose(2, 3)), "v_out"),
        (dict(codes_out=base["codes_out"].to(torch.int16)), "codes_out"), (dict(codes_out=base["codes_out"][:, :1]), "codes_out"),
        (dict(slot_mapping=base["slot_mapping"].int()), "slot_mapping"), (dict(slot_mapping=base["slot_mapping"][:, :2]), "slot_mapping"),
        (dict(slot_mapping=base["slot_mapping"].cpu()), "device"), (dict(heavy=[True] + [False] * 15), "passthrough"),
        (dict(cos=cos), "together"), (dict(cos=cos, sin=sin), "positions"), (dict(k_weight=torch.ones(63, device=DEV)), "k_weight"),
        (dict(kernel=2), "kernel"), (dict(perm=base["perm"][0][:32]), "permutation"),
        (dict(heavy=[True] + [False] * 15, pt_out=torch.zeros(4, 2, 16, 2, 4, device=DEV)), "pt_out"),
    ]
    for kw, word in bad:
        with pytest.raises(RuntimeError, match=word):
            hip_ops.append_kv(**{**base, **kw})


@pytest.mark.parametrize("B, S", [(16, 1), (2, 1100)])
def test_graph_replays(B, S):
    """Both paths captured and replayed on new inputs, beside eager calls; two captured graphs at once."""
    log(f"append: graphs {B} {S}")
    rng = np.random.default_rng(7)
    g = torch.Generator().manual_seed(11)
    perm, cent, _, _ = codec_arrays(rng, 4, 128, 4, 256)
    perm, cent = perm.to(DEV), cent.to(DEV)
    pages = B * (S // 16 + 2)
    k, v = (torch.randn(B, 4, S, 128, generator=g).to(BF).to(DEV) for _ in range(2))
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(S + 64, 128))
    pos = torch.arange(S, device=DEV)[None].expand(B, S).contiguous()
    slots = torch.from_numpy(_slots(rng, B, S, 16, pages, 0.1, False)).to(DEV)

    def make():
        return torch.zeros(pages, 4, 16, 32, dtype=torch.uint8, device=DEV), torch.zeros(pages, 4, 128, 16, dtype=BF, device=DEV)

    def call(c, vp):
        hip_ops.append_kv(k, v, perm, cent, codes_out=c, v_out=vp, slot_mapping=slots, cos=cos, sin=sin, positions=pos)

    bufs = [make(), make()]
    call(*bufs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*bufs[0])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for c, vp in bufs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(c, vp)
        graphs.append(graph)
    for step in range(3):
        k.mul_(0.9).add_(0.01)
        pos.add_(1)
        want = make()
        call(*want)
        for (c, vp), graph in zip(bufs, graphs):
            c.zero_()
            vp.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for c, vp in bufs:
            assert torch.equal(c, want[0]) and torch.equal(vp, want[1]), step


def _codes_of_append(k, perm, cent, direct, S=1):
    """Codes [n, nb] of rows k [n, D] appended as they are, by the form that appends take of themselves."""
    n, D = k.shape
    nb = cent.shape[1]
    pages = (n + 15) // 16
    c = torch.zeros(pages, 1, 16, nb, dtype=hip_ops.index_dtype(cent.shape[2]), device=DEV)
    hip_ops.append_kv(k.view(n // S, S, 1, D).transpose(1, 2), None, perm, cent, codes_out=c, v_out=None,
                      slot_mapping=torch.arange(n, device=DEV).view(n // S, S), direct=direct)
    return c.permute(0, 2, 1, 3).reshape(pages * 16, nb)[:n]


@pytest.mark.parametrize("direct", [False, True])
@pytest.mark.parametrize("bd, nc", [(1, 256), (2, 64), (2, 256), (4, 17), (4, 256), (8, 256), (3, 100), (4, 4096), (16, 1500)])
def test_ties_and_extremes(bd, nc, direct):
    """Codewords twice, codewords a step of fp32 apart, distances of zero, subnormal ones, infinities and NaN: the
    codes are those of the exact scan."""
    log(f"append_kv ties bd {bd} nc {nc} direct {direct}")
    rng = np.random.default_rng(bd * 1000 + nc)
    D = 48 if bd == 3 else 64
    nb = D // bd
    base = rng.standard_normal((1, nb, nc, bd)).astype(np.float32)
    half = nc // 2
    base[:, :, half:2 * half] = base[:, :, rng.permutation(half)]             # twice
    base[:, : nb // 2, half:2 * half] *= np.float32(1 + 2.0 ** -23)            # or a step apart
    cent = torch.from_numpy(base)
    pick = cent[0][torch.arange(nb), torch.from_numpy(rng.integers(0, nc, (24, nb)))].reshape(24, D)  # on codewords
    far = torch.from_numpy(rng.standard_normal((24, D)).astype(np.float32)) * 1e4
    odd = torch.from_numpy(rng.standard_normal((16, D)).astype(np.float32))
    odd[0], odd[1], odd[2, ::3], odd[3, ::5] = math.nan, math.inf, -math.inf, math.nan
    odd[4], odd[5] = 0.0, 3e38
    keys = torch.cat((pick, far, odd))
    perm = torch.from_numpy(rng.permutation(D))
    for scale in (1.0, 1e-19, 1e-22):
        dk, dc, dp = (keys * scale).to(DEV), (cent * scale).to(DEV), perm.to(DEV)
        want, _ = hip_ops.encode(dk.view(len(keys), 1, 1, D), dp, dc, kernel=1, direct=direct)
        want = want.view(len(keys), nb)
        for S in (1, 8):
            got = _codes_of_append(dk, dp, dc, direct, S)
            assert torch.equal(got, want), f"scale {scale}, {S} a sequence"
        half_keys = dk.to(BF)
        want, _ = hip_ops.encode(half_keys.view(len(keys), 1, 1, D), dp, dc, kernel=1, direct=direct)
        assert torch.equal(_codes_of_append(half_keys, dp, dc, direct), want.view(len(keys), nb)), f"bf16, scale {scale}"


@pytest.mark.parametrize("S, first", [(8, 0), (8, 7), (9, 15), (16, 1), (31, 8), (40, 3), (64, 0), (300, 13)])
@pytest.mark.parametrize("kernel", [0, 1])
def test_values_from_any_slot(S, first, kernel):
    """Runs of slots that begin anywhere in a page, with holes, over pages of 8, 16, 24 and 64 tokens."""
    log(f"append_kv values, {S} tokens from slot {first}")
    for page in (8, 16, 24, 64):
        rng = np.random.default_rng(S + page)
        B, Hkv, D, Dv = 3, 2, 64, 72
        per = (S + first) // page + 1
        table = rng.permutation(B * per + 2)[:B * per].reshape(B, per)
        at = first + np.arange(S)[None] + np.zeros((B, 1), np.int64)
        slots = np.take_along_axis(table, at // page, 1) * page + at % page
        slots[1, 0] = -1
        slots[2, S // 2] = -1
        g = torch.Generator().manual_seed(S)
        k, v = torch.randn(B, S, Hkv, D, generator=g).to(BF), torch.randn(B, S, Hkv, Dv, generator=g).to(BF)
        perm, cent, _, _ = codec_arrays(rng, Hkv, D, 4, 256)
        pages = B * per + 2
        v0 = torch.randn(pages, Hkv, Dv, page, generator=g).to(BF)
        vp = v0.to(DEV)
        c = torch.zeros(pages, Hkv, page, 16, dtype=torch.uint8, device=DEV)
        hip_ops.append_kv(k.to(DEV).transpose(1, 2), v.to(DEV).transpose(1, 2), perm.to(DEV), cent.to(DEV), codes_out=c,
                          v_out=vp, slot_mapping=torch.from_numpy(slots).to(DEV), kernel=kernel)
        want = v0.clone()
        for b in range(B):
            for s in range(S):
                if slots[b, s] >= 0:
                    want[slots[b, s] // page, :, :, slots[b, s] % page] = v[b, s]
        assert torch.equal(vp.cpu(), want), f"page {page}"


@pytest.mark.parametrize("bd, nc, D, Hkv, S", [(2, 64, 64, 2, 9000), (4, 16, 128, 4, 3000), (8, 128, 128, 4, 3000), (16, 200, 64, 1, 2000)])
def test_many_rows_of_small_codebooks(bd, nc, D, Hkv, S):
    """Codebooks that the encode serves by its exact scan keep to one launch: the same codes, with a search grid too
    where there is one."""
    log(f"append_kv small codebooks bd {bd} nc {nc} S {S}")
    rng = np.random.default_rng(nc)
    g = torch.Generator(device=DEV).manual_seed(nc)
    perm, cent, _, sigma = codec_arrays(rng, Hkv, D, bd, nc)
    perm, cent = perm.to(DEV), cent.to(DEV)
    k = (torch.randn(1, S, Hkv, D, generator=g, device=DEV) * torch.from_numpy(sigma).to(DEV).float()).to(BF).transpose(1, 2)
    v = torch.randn(1, S, Hkv, D, generator=g, device=DEV).to(BF).transpose(1, 2)
    pages = S // 16 + 2
    slots = 7 + torch.arange(S, device=DEV)[None]
    grids = [None] + ([hip_ops.encode_grid(cent, Hkv)] if bd == 2 else [])
    for grid in grids:
        got = []
        for kernel in (0, 1):
            c = torch.zeros(pages, Hkv, 16, D // bd, dtype=torch.uint8, device=DEV)
            vp = torch.zeros(pages, Hkv, D, 16, dtype=BF, device=DEV)
            hip_ops.append_kv(k, v, perm, cent, codes_out=c, v_out=vp, slot_mapping=slots, kernel=kernel, grid=grid)
            got.append((c, vp))
        assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
        flat = got[0][1].permute(0, 3, 1, 2).reshape(pages * 16, Hkv, D)[7:7 + S]
        assert torch.equal(flat, v[0].transpose(0, 1))
