"""Decode attention over a shared prefix (hip_ops.decode_prefix) against softmax attention in 64 bits."""

import math

import numpy as np
import pytest
import torch

from _step import DEV, codec_arrays, prefix_attention64
from _util import log
from sunshape_amd import hip_ops

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _problem(B, Hq, Hkv, Lq, D, Dv, bd, nc, T, lens, qdt=BF, vdt=BF, heavy=(), per_head=True, page=16, own_mask=None, seed=0,
             token_major=True, pt_dense=False):
    rng = np.random.default_rng(seed + 17 * B + T)
    g = torch.Generator().manual_seed(seed + B + T)
    nb = D // bd
    perm, cent, mask, _ = codec_arrays(rng, Hkv, D, bd, nc, per_head, heavy)
    lens = np.asarray(lens)
    width = int((lens.max() + page - 1) // page) if len(lens) else 0
    npre = (T + page - 1) // page
    total = npre + B * width + 2
    pool = rng.permutation(total)
    table = pool[npre:npre + B * width].reshape(B, width)
    own = (lens + page - 1) // page
    table = np.where(np.arange(width)[None] < own[:, None], table, 0).astype(np.int32)
    codes = torch.randint(0, nc, (total, Hkv, page, nb), generator=g, dtype=torch.int32).to(hip_ops.index_dtype(nc))
    v = torch.randn(total, Hkv, Dv, page, generator=g).to(vdt)
    pt = None
    if heavy:
        pt = torch.randn(total, Hkv, page, len(heavy), bd, generator=g).to(qdt)
    q = torch.randn(B, Lq, Hq, D, generator=g).mul(1.5).to(qdt)
    q = q.transpose(1, 2) if token_major else q.reshape(B, Hq, Lq, D)
    m = None
    if own_mask == "causal":
        last = torch.from_numpy(lens)[:, None] - Lq + torch.arange(Lq)[None]
        m = torch.zeros(B, 1, Lq, width * page).masked_fill_(torch.arange(width * page) > last[:, None, :, None], -math.inf)
    elif own_mask == "lowest":  # some rows: every own token at the type's lowest value
        m = torch.zeros(B, Hq, Lq, width * page)
        m[0] = torch.finfo(torch.float32).min
    elif own_mask == "empty":  # some rows lose all their own tokens
        m = torch.zeros(B, Hq, Lq, width * page)
        m[:, ::2] = -math.inf
    return dict(q=q, scale=1 / math.sqrt(D), perm=perm, cent=cent, mask=mask, codes=codes, v=v, pt=pt,
                ptable=torch.from_numpy(pool[:npre].astype(np.int32)), plen=torch.tensor([T], dtype=torch.int32),
                table=torch.from_numpy(table), lens=torch.from_numpy(lens.astype(np.int32)), own_mask=m, heavy=heavy)


def _dev(t):
    return None if t is None else t.to(DEV)


def _call(p, **kw):
    q = p["q"]
    dq = q.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    return hip_ops.decode_prefix(dq, _dev(p["codes"]), _dev(p["v"]), _dev(p["perm"]), _dev(p["cent"]), scale=p["scale"],
                                 prefix_table=_dev(p["ptable"]), prefix_len=_dev(p["plen"]), block_table=_dev(p["table"]),
                                 seq_lens=_dev(p["lens"]), mask=_dev(p["own_mask"]), heavy=p["mask"], pt=_dev(p["pt"]),
                                 return_lse=True, **kw)


def _check(p, out, lse, what):
    ref, rlse, mag, pv = prefix_attention64(p["q"], p["scale"], p["perm"], p["cent"], p["codes"], p["v"], p["ptable"],
                                            int(p["plen"]), p["table"], p["lens"], p["own_mask"], p["pt"], p["mask"])
    out, lse = out.cpu().double(), lse.cpu().double()
    empty = rlse == -math.inf
    assert (lse[empty] == -math.inf).all() and (out[empty] == 0).all(), f"{what}: rows with nothing to attend"
    # A logit: the codebook in two bf16 parts leaves 2^-17 of a codeword, and a 32-bit query as much of itself, and
    # the fp32 sum of D <= 256 terms rounds at most D 2^-24 of the sum of magnitudes: 2^-15 of it together.
    dx = 2.0 ** -15 * mag + 1e-5  # the exponential's and logarithm's own
    assert ((lse - rlse).abs()[~empty] <= dx[~empty] + 2.0 ** -22 * rlse.abs()[~empty]).all(), f"{what}: lse"
    # A probability is off by its logit's error, and rounded to the values' 16 bits (at most half a step); the
    # output is rounded once.
    half = torch.finfo(p["v"].dtype).eps / 2
    tiny = 2.0 ** -24 if p["v"].dtype == F16 else 0.0
    bound = half * ref.abs() + (2 * dx[..., None] + half + 1e-5) * pv + tiny * (1 + pv) + 1e-30
    err = (out - ref).abs()
    assert (err <= bound).all(), f"{what}: out {(err / bound).max().item():.2f} times the bound"


CASES = {
    "one": dict(B=1, Hq=1, Hkv=1, Lq=1, D=64, Dv=64, bd=4, nc=256, T=1, lens=[1]),
    "gqa": dict(B=5, Hq=14, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=517, lens=[37, 1, 16, 17, 0]),
    "rows33": dict(B=11, Hq=6, Hkv=2, Lq=1, D=64, Dv=64, bd=2, nc=256, T=333, lens=list(range(11))),
    "bd2_128": dict(B=9, Hq=32, Hkv=8, Lq=1, D=128, Dv=128, bd=2, nc=256, T=700, lens=[300, 5, 64, 65, 63, 1, 128, 0, 299]),
    "bd4_128": dict(B=40, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=1000, lens=[7 * i % 90 for i in range(40)]),
    "bd8_128": dict(B=20, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=8, nc=256, T=250, lens=[31] * 20),
    "nc64": dict(B=7, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=2, nc=64, T=129, lens=[40] * 7),
    "nc100": dict(B=7, Hq=8, Hkv=2, Lq=1, D=64, Dv=128, bd=4, nc=100, T=129, lens=[40] * 7),
    "f16": dict(B=6, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=260, lens=[40] * 6, qdt=F16, vdt=F16),
    "q_f32": dict(B=6, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=260, lens=[40] * 6, qdt=F32, vdt=BF),
    "v_f32": dict(B=6, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=260, lens=[40] * 6, vdt=F32),
    "shared_codec": dict(B=6, Hq=8, Hkv=4, Lq=1, D=64, Dv=64, bd=4, nc=256, T=100, lens=[20] * 6, per_head=False),
    "mixed": dict(B=6, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=150, lens=[20] * 6, heavy=(0, 3, 9)),
    "mixed_many": dict(B=3, Hq=4, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=80, lens=[9] * 3, heavy=tuple(range(0, 30, 3))),
    "mixed_64_8": dict(B=9, Hq=14, Hkv=2, Lq=1, D=64, Dv=64, bd=2, nc=256, T=517, lens=[20, 0, 1, 33] + [64] * 5, heavy=(0, 31, 7, 8)),
    "mixed_64_16": dict(B=5, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=8, nc=256, T=333, lens=[20, 0, 1, 33, 40], heavy=(1, 6)),
    "mixed_128_16": dict(B=21, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=1100, lens=[7 * i for i in range(21)], heavy=(0, 5, 6, 31)),
    "mixed_128_24": dict(B=5, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=8, nc=256, T=130, lens=[20, 0, 1, 33, 40], heavy=(15, 2, 3)),
    "mixed_128_32": dict(B=5, Hq=32, Hkv=2, Lq=2, D=128, Dv=128, bd=2, nc=64, T=200, lens=[20, 2, 3, 33, 40],
                         heavy=tuple(range(0, 64, 4)), own_mask="causal"),
    "mixed_128_40": dict(B=21, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=300, lens=[7 * i for i in range(21)], heavy=tuple(range(1, 31, 3))),
    "mixed_128_64": dict(B=3, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=8, nc=256, T=130, lens=[20, 0, 101], heavy=tuple(range(8))),
    "mixed_64_32": dict(B=3, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=130, lens=[20, 0, 101], heavy=tuple(range(1, 16, 2)), qdt=F16, vdt=F16),
    "mixed_64_4": dict(B=3, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=2, nc=256, T=130, lens=[20, 0, 101], heavy=(4, 30)),
    "mixed_64_6": dict(B=3, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=2, nc=256, T=130, lens=[20, 0, 101], heavy=(4, 30, 31)),
    "mixed_f16": dict(B=6, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=260, lens=[40] * 6, qdt=F16, vdt=F16, heavy=(3, 4, 30, 31)),
    "mixed_long": dict(B=2, Hq=4, Hkv=1, Lq=1, D=64, Dv=64, bd=4, nc=256, T=9000, lens=[2500, 3], heavy=(3, 4, 9, 11, 12, 15)),
    "wide": dict(B=4, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=4096, T=300, lens=[33, 2, 0, 70]),
    "wide_32bit": dict(B=2, Hq=2, Hkv=1, Lq=1, D=64, Dv=64, bd=16, nc=65536, T=40, lens=[9, 2]),
    "page8": dict(B=4, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=77, lens=[11, 8, 0, 9], page=8),
    "page64": dict(B=4, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=177, lens=[11, 80, 0, 64], page=64),
    "odd_dims": dict(B=3, Hq=4, Hkv=2, Lq=1, D=48, Dv=32, bd=3, nc=50, T=40, lens=[5, 6, 7]),
    "d256": dict(B=3, Hq=4, Hkv=2, Lq=1, D=256, Dv=256, bd=4, nc=256, T=140, lens=[5, 60, 7]),
    "verify": dict(B=5, Hq=8, Hkv=2, Lq=4, D=128, Dv=128, bd=4, nc=256, T=270, lens=[4, 30, 5, 64, 11], own_mask="causal"),
    "verify_f16": dict(B=3, Hq=14, Hkv=2, Lq=3, D=64, Dv=64, bd=2, nc=256, T=90, lens=[4, 30, 5], own_mask="causal", qdt=F16, vdt=F16),
    "head_major_q": dict(B=4, Hq=8, Hkv=2, Lq=3, D=64, Dv=64, bd=4, nc=256, T=90, lens=[4, 30, 5, 9], token_major=False),
    "mask_empty": dict(B=4, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=90, lens=[4, 30, 5, 9], own_mask="empty"),
    "mask_empty_no_prefix": dict(B=4, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=0, lens=[4, 30, 5, 9], own_mask="empty"),
    "mask_lowest": dict(B=4, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=90, lens=[4, 30, 5, 9], own_mask="lowest"),
    "no_prefix": dict(B=4, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=0, lens=[4, 300, 0, 9]),
    "no_own": dict(B=4, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=200, lens=[0, 0, 0, 0]),
    "nothing": dict(B=3, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=0, lens=[0, 2, 0]),
    "many_heads": dict(B=70, Hq=32, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=100, lens=[i % 33 for i in range(70)]),
    "long_own": dict(B=2, Hq=4, Hkv=1, Lq=1, D=128, Dv=128, bd=4, nc=256, T=65, lens=[2500, 3]),
    "g64": dict(B=2, Hq=96, Hkv=1, Lq=1, D=64, Dv=64, bd=4, nc=256, T=70, lens=[40, 3]),
}


@pytest.mark.parametrize("kernel", [0, 1])
@pytest.mark.parametrize("name", CASES)
def test_against_64_bits(name, kernel):
    log(f"decode_prefix {name} kernel {kernel}")
    p = _problem(**CASES[name])
    out, lse = _call(p, kernel=kernel)
    _check(p, out, lse, name)


@pytest.mark.parametrize("bits, nc, bd", [(8, 256, 4), (6, 64, 2), (4, 16, 2), (3, 8, 2)])
def test_packed_codes(bits, nc, bd):
    log(f"decode_prefix, packed codes of {bits} bits")
    p = _problem(B=5, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=bd, nc=nc, T=150, lens=[20, 0, 3, 64, 70])
    words = hip_ops.pack_codes(p["codes"].to(DEV), bits)
    packed = dict(p, codes=words)
    out, lse = _call(packed, code_bits=bits)
    _check(p, out, lse, f"{bits}-bit words")


def test_rotated_codec():
    log("decode_prefix, rotated codec")
    p = _problem(B=4, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=90, lens=[4, 30, 5, 9])
    g = torch.Generator().manual_seed(2)
    R = torch.linalg.qr(torch.randn(64, 64, generator=g, dtype=torch.float64))[0].float()
    out, lse = _call(p, rotation=R.to(DEV))
    qs = (p["q"] * p["scale"]).float()
    ref = dict(p, q=(qs.double() @ R.double().T).float(), scale=None, perm=torch.arange(64))
    _check(ref, out, lse, "rotated")


def test_lengths_on_the_device_shorter_than_the_tables():
    """Tables with room to spare: the lengths decide, and what the slots behind them hold is not seen (NaN and
    infinities there, and table entries behind the last page that name no page of the pool's first)."""
    log("decode_prefix: short lengths in long tables")
    p = _problem(B=6, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=400, lens=[100] * 6)
    used = torch.zeros(p["codes"].shape[0], 16, dtype=torch.bool)
    p["plen"] = torch.tensor([133], dtype=torch.int32)
    p["lens"] = torch.tensor([0, 1, 15, 16, 17, 99], dtype=torch.int32)
    for t in range(133):
        used[p["ptable"][t // 16], t % 16] = True
    for b in range(6):
        for t in range(int(p["lens"][b])):
            used[p["table"][b, t // 16], t % 16] = True
    v = p["v"].clone()
    v.permute(0, 3, 1, 2)[~used] = float("nan")
    v.permute(0, 3, 1, 2)[~used, :, ::2] = float("inf")
    for kernel in (0, 1):
        out, lse = _call(dict(p, v=v), kernel=kernel)
        _check(p, out, lse, f"short lengths, kernel {kernel}")


def test_large_logits():
    """Logits far apart (one token takes all), and all alike."""
    log("decode_prefix: large and equal logits")
    for f in (30.0, 0.0):
        p = _problem(B=5, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=300, lens=[40, 1, 0, 5, 33])
        p["q"] = p["q"] * f
        out, lse = _call(p)
        _check(p, out, lse, f"queries times {f}")


@pytest.mark.parametrize("qdt", [BF, F32])
def test_kept_blocks_codewords_and_unwritten_tokens(qdt):
    """A kept block's codewords are not read into the sum, nor what lies behind the lengths in the passthrough."""
    log(f"decode_prefix: kept blocks, {qdt}")
    p = _problem(B=6, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=400, lens=[100] * 6, heavy=(2, 9, 17, 18, 30, 31))
    p["plen"] = torch.tensor([133], dtype=torch.int32)
    p["lens"] = torch.tensor([0, 1, 15, 16, 17, 99], dtype=torch.int32)
    used = torch.zeros(p["codes"].shape[0], 16, dtype=torch.bool)
    for t in range(133):
        used[p["ptable"][t // 16], t % 16] = True
    for b in range(6):
        for t in range(int(p["lens"][b])):
            used[p["table"][b, t // 16], t % 16] = True
    p["q"] = p["q"].to(qdt)
    pt, cent = p["pt"].clone(), p["cent"].clone()
    pt.permute(0, 2, 1, 3, 4)[~used] = float("nan")
    cent[:, list(p["heavy"])] = float("nan")
    for kernel in (0, 1):
        out, lse = _call(dict(p, pt=pt, cent=cent), kernel=kernel)
        _check(p, out, lse, f"kept blocks, kernel {kernel}")


def test_keys_near_the_largest_f16():
    """log2(e) times a codeword or a kept value passes what f16 holds from 45,401 on."""
    log("decode_prefix: large f16 keys")
    p = _problem(B=5, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=300, lens=[40, 1, 0, 5, 33], qdt=F16, vdt=F16, heavy=(1, 5))
    rng = np.random.default_rng(5)
    p["cent"][:, 3] = torch.from_numpy(rng.choice([-65504.0, 65504.0, 50000.0, -46000.0], p["cent"][:, 3].shape)).float()
    p["pt"][:, :, :, 0] = torch.from_numpy(rng.choice([-65504.0, 65504.0, 50000.0], tuple(p["pt"][:, :, :, 0].shape))).to(F16)
    p["q"] = p["q"] * 2.0 ** -12
    out, lse = _call(p)
    # past f16's largest value the two parts leave 2^-12 of what the second one holds, less than half as much as the first
    ref, rlse, mag, pv = prefix_attention64(p["q"], p["scale"], p["perm"], p["cent"], p["codes"], p["v"], p["ptable"],
                                            int(p["plen"]), p["table"], p["lens"], None, p["pt"], p["mask"])
    dx = 2.0 ** -13 * mag + 1e-5
    assert ((lse.cpu().double() - rlse).abs() <= dx).all()
    half = torch.finfo(F16).eps / 2
    bound = half * ref.abs() + (2 * dx[..., None] + half + 1e-5) * pv + 2.0 ** -24 * (1 + pv)
    assert ((out.cpu().double() - ref).abs() <= bound).all()


def test_repeats_itself_and_streams():
    log("decode_prefix: repeats, side stream")
    p = _problem(B=33, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=900, lens=[i * 5 % 77 for i in range(33)])
    a = _call(p)
    b = _call(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = _call(p)
    side.synchronize()
    for x in (b, c):
        assert torch.equal(a[0], x[0]) and torch.equal(a[1], x[1])


def test_graph_replays_with_growing_lengths():
    """Two graphs of the step captured once, replayed as the sequences grow: the lengths live on the device."""
    log("decode_prefix: graphs")
    p = _problem(B=12, Hq=8, Hkv=2, Lq=1, D=128, Dv=128, bd=4, nc=256, T=500, lens=[90] * 12)
    d = {k: _dev(p[k]) for k in ("codes", "v", "perm", "cent", "ptable", "plen", "table", "lens")}
    q = p["q"].to(DEV).contiguous()

    def call():
        return hip_ops.decode_prefix(q, d["codes"], d["v"], d["perm"], d["cent"], scale=p["scale"], prefix_table=d["ptable"],
                                     prefix_len=d["plen"], block_table=d["table"], seq_lens=d["lens"], return_lse=True)

    call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    outs, graphs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for plen, n in ((500, 90), (1, 0), (317, 33), (0, 17), (0, 0)):
        d["plen"].fill_(plen)
        d["lens"].fill_(n)
        q.mul_(1.1)
        want = call()
        for o, graph in zip(outs, graphs):
            o[0].fill_(float("nan"))
            graph.replay()
            graph.replay()
        torch.cuda.synchronize()
        for o in outs:
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1]), (plen, n)


def test_refusals():
    log("decode_prefix: refusals")
    p = _problem(B=2, Hq=4, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=40, lens=[4, 9])
    base = dict(q=p["q"].to(DEV), codes=p["codes"].to(DEV), v=p["v"].to(DEV), perm=p["perm"].to(DEV), cent=p["cent"].to(DEV),
                prefix_table=p["ptable"].to(DEV), prefix_len=p["plen"].to(DEV), block_table=p["table"].to(DEV), seq_lens=p["lens"].to(DEV))
    bad = [
        (dict(q=base["q"][0]), "batch, heads"), (dict(q=base["q"][:, :3]), "divisible"), (dict(codes=base["codes"].int()), "codes"),
        (dict(v=base["v"][:-1]), "paged V"), (dict(prefix_table=base["prefix_table"].long()), "int32"),
        (dict(prefix_table=base["prefix_table"][None]), "prefix_table"), (dict(prefix_len=base["prefix_len"].repeat(2)), "prefix_len"),
        (dict(block_table=base["block_table"][:1]), "block_table"), (dict(seq_lens=base["seq_lens"][:1]), "seq_lens"),
        (dict(seq_lens=base["seq_lens"].cpu()), "device"), (dict(mask=torch.zeros(2, 16, device=DEV)), "4-D"),
        (dict(heavy=[True] + [False] * 15), "passthrough"), (dict(kernel=3), "kernel"),
        (dict(heavy=[True] + [False] * 15, pt=torch.zeros(2, 2, 16, 1, 4, device=DEV)), "passthrough values must"),
        (dict(codes=base["codes"][:, :, :4], v=base["v"][..., :4].contiguous()), "page_size"),
    ]
    for kw, word in bad:
        with pytest.raises(RuntimeError, match=word):
            hip_ops.decode_prefix(**{**base, **kw})
    empty = hip_ops.decode_prefix(**{**base, "q": base["q"][:0], "block_table": base["block_table"][:0], "seq_lens": base["seq_lens"][:0]})
    assert empty.shape == (0, 4, 1, 64)
