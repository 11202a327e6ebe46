"""The forms of the matrix-core kernel that only large calls of decode_prefix take: 64 rows an item, waves of more than
32 tiles (which read on in the page table), workgroups with several items, own pieces of several rounds.  Each case
says which form it means to reach, and the call's plan is asked whether it does."""

import ctypes
import math

import pytest
import torch

from _step import DEV
from _util import log
from sunshape_amd import _native as N
from sunshape_amd import hip_ops
from test_step_host import ALIGNED

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {F32: N.SSQ_F32, BF: N.SSQ_BF16, F16: N.SSQ_F16}


def _plan(c, width, kept):
    """rows of a prefix item / 32, row groups, slices, workgroups per KV head, own pieces at most, their fewest tiles"""
    a = N.PrefixArgs(prefix_table=ALIGNED, prefix_len=ALIGNED, prefix_cap=(c["T"] + 15) // 16 * 16)
    D, bd, hkv, hq, lq = c["D"], c["bd"], c["Hkv"], c["Hq"], c["Lq"]
    nb = D // bd
    d = dict(q=ALIGNED, q_dtype=CODE[c["qdt"]], q_sl=D, q_sh=lq * D, q_sb=hq * lq * D, batch=c["B"], num_q_heads=hq, q_len=lq,
             head_dim=D, num_kv_heads=hkv, perm=ALIGNED, cent=ALIGNED, cent_sh=nb * 256 * bd, block_dim=bd, n_blocks=nb,
             n_centroids=256, layout=N.SSQ_PAGED, seq_len=width * 16, codes=ALIGNED, c_st=nb, c_sh=16 * nb, c_sb=hkv * 16 * nb,
             block_table=ALIGNED if width else 0, bt_sb=width, seq_lens=ALIGNED, page_size=16, v=ALIGNED, v_dtype=CODE[c["vdt"]],
             value_dim=D, v_st=16, v_sh=D * 16, v_sb=hkv * D * 16, out=ALIGNED, o_sl=D, o_sh=lq * D, o_sb=hq * lq * D)
    for k, v in d.items():
        setattr(a.dec, k, v)
    for i in kept:
        a.dec.heavy_mask[i // 64] |= 1 << (i % 64)
    if kept:
        n = len(kept) * bd
        a.dec.pt, a.dec.pt_dtype, a.dec.pt_st, a.dec.pt_sh, a.dec.pt_sb = ALIGNED, CODE[c["vdt"]], n, 16 * n, hkv * 16 * n
    out = (ctypes.c_int32 * 6)()
    fn = getattr(N.lib(), "_Z22ssq_decode_prefix_planPK15ssq_prefix_argsPi")
    assert fn(ctypes.byref(a), out) == 0
    return dict(zip(("nr", "groups", "slices", "wgs", "pieces", "least"), out))


BASE = dict(Lq=1, D=64, bd=4, qdt=BF, vdt=BF, kept=(), window=None)
CASES = {
    # a batch on a long document, 64 rows an item
    "document": (dict(B=64, Hq=32, Hkv=8, D=128, T=16411, lens=[7 * i % 61 for i in range(64)]), "nr2"),
    "document_f16_verify": (dict(B=16, Hq=32, Hkv=8, D=128, Lq=4, T=16001, lens=[4 + 5 * i for i in range(16)], qdt=F16, vdt=F16), "nr2"),
    # one workgroup a KV head: more than 64 tiles a wave, 64 rows an item
    "deep": (dict(B=40, Hq=256, Hkv=256, T=9001, lens=[i % 5 for i in range(40)]), "nr2 deep"),
    "deep_f16": (dict(B=64, Hq=256, Hkv=256, bd=2, T=8210, lens=[0] * 64, qdt=F16, vdt=F16), "nr2 deep"),
    # several items a workgroup, of 64 and of 32 rows
    "rounds": (dict(B=150, Hq=128, Hkv=128, T=3001, lens=[i % 3 for i in range(150)]), "nr2 rounds"),
    "rounds_kept": (dict(B=40, Hq=256, Hkv=256, T=9001, lens=[i % 5 for i in range(40)], kept=(0, 5, 6)), "rounds deep"),
    "rounds_f32": (dict(B=70, Hq=256, Hkv=256, bd=8, T=4500, lens=[3] * 70, qdt=F32), "rounds deep32"),
    "rounds_kept_f16": (dict(B=33, Hq=256, Hkv=256, D=128, T=4200, lens=[0] * 33, kept=(3, 4, 9), qdt=F16, vdt=F16), "rounds deep32"),
    # own tokens: more pieces of the fewest tiles than waves, on few and on many sequences, and pieces of many tiles
    "own_few": (dict(B=12, Hq=64, Hkv=64, T=0, lens=[1400 - 100 * i for i in range(12)]), "own_rounds"),
    "own_many": (dict(B=70, Hq=64, Hkv=64, T=100, lens=[11 * i for i in range(70)]), "own_rounds"),
    "own_rows": (dict(B=9, Hq=128, Hkv=64, Lq=20, T=50, lens=[500 + 40 * i for i in range(9)]), "own_rounds"),
    "own_deep": (dict(B=2, Hq=64, Hkv=64, T=33, lens=[36011, 20000]), "own_rounds own_deep"),
    "own_deep_window": (dict(B=2, Hq=128, Hkv=64, Lq=16, T=0, lens=[36011, 20000], window=9000), "own_rounds own_deep"),
    "own_deep_kept_f16": (dict(B=3, Hq=64, Hkv=64, bd=2, T=0, lens=[30005, 9000, 17], kept=(1, 30), qdt=F16, vdt=F16), "own_rounds own_deep"),
}


def _problem(c):
    g = torch.Generator(device=DEV).manual_seed(5)
    B, Hq, Hkv, Lq, D, bd, T = (c[k] for k in ("B", "Hq", "Hkv", "Lq", "D", "bd", "T"))
    nb, lens = D // bd, torch.tensor(c["lens"], device=DEV, dtype=torch.int32)
    own, npre = (lens + 15) // 16, (T + 15) // 16
    width = int(own.max())
    total = npre + int(own.sum()) + 1
    pool = torch.randperm(total - 1, generator=g, device=DEV).to(torch.int32) + 1  # page 0 is none's
    table = torch.zeros(B, width, dtype=torch.int32, device=DEV)
    if width:
        table[torch.arange(width, device=DEV)[None] < own[:, None]] = pool[npre:]
    sigma = torch.exp(torch.rand(Hkv, D, generator=g, device=DEV) * math.log(15.0) + math.log(0.2))
    perm = torch.stack([torch.randperm(D, generator=g, device=DEV) for _ in range(Hkv)])
    p = dict(
        q=torch.randn(B, Hq, Lq, D, generator=g, device=DEV).mul(1.5).to(c["qdt"]), perm=perm,
        cent=torch.randn(Hkv, nb, 256, bd, generator=g, device=DEV) * torch.gather(sigma, 1, perm).view(Hkv, nb, 1, bd),
        codes=torch.randint(0, 256, (total, Hkv, 16, nb), generator=g, device=DEV, dtype=torch.uint8),
        v=torch.randn(total, Hkv, D, 16, generator=g, device=DEV).to(c["vdt"]), pt=None, heavy=None, mask=None,
        ptable=pool[:npre].contiguous(), plen=torch.tensor([T], dtype=torch.int32, device=DEV), table=table, lens=lens)
    p["v"][0] = float("nan")
    if c["kept"]:
        p["heavy"] = [i in c["kept"] for i in range(nb)]
        p["pt"] = torch.randn(total, Hkv, 16, len(c["kept"]), bd, generator=g, device=DEV).to(c["vdt"])
    if c["window"]:  # the last tokens, causal among the new ones
        at = torch.arange(width * 16, device=DEV)
        last = lens[:, None] - Lq + torch.arange(Lq, device=DEV)[None]
        seen = (at <= last[..., None]) & (at > last[..., None] - c["window"])
        p["mask"] = torch.zeros(B, 1, Lq, width * 16, device=DEV).masked_fill_(~seen[:, None], -math.inf)
    return p


def _call(p, scale, kernel=0):
    return hip_ops.decode_prefix(p["q"], p["codes"], p["v"], p["perm"], p["cent"], scale=scale, prefix_table=p["ptable"],
                                 prefix_len=p["plen"], block_table=p["table"], seq_lens=p["lens"], mask=p["mask"],
                                 heavy=p["heavy"], pt=p["pt"], return_lse=True, kernel=kernel)


def _head64(p, scale, h, c):
    """A KV head's rows in 64 bits: out [B, G, Lq, D], lse, the largest sum |q||k| of a row's logits, sum p |v|."""
    B, D, Lq, T, bd = c["B"], c["D"], c["Lq"], c["T"], c["bd"]
    G = c["Hq"] // c["Hkv"]

    def tokens(table, n):
        pages = table[:(n + 15) // 16].long()
        idx = p["codes"][pages, h].reshape(-1, D // bd)[:n].long()
        k = p["cent"][h].double().reshape(-1, bd)[idx + 256 * torch.arange(D // bd, device=DEV)]
        if p["heavy"]:
            k[:, torch.tensor(p["heavy"], device=DEV)] = p["pt"][pages, h].reshape(-1, len(c["kept"]), bd)[:n].double()
        return k.reshape(n, D), p["v"][pages, h].double().transpose(1, 2).reshape(-1, D)[:n]

    kp, vp = tokens(p["ptable"], T)
    q = (p["q"][:, h * G:(h + 1) * G] * scale).double()[..., p["perm"][h]].reshape(B, G * Lq, D)
    xp = (q.reshape(-1, D) @ kp.T.contiguous()).view(B, G * Lq, T)
    mp = (q.abs().reshape(-1, D) @ kp.abs().T.contiguous()).view(B, G * Lq, T)
    res = []
    for b in range(B):
        n = c["lens"][b]
        ko, vo = tokens(p["table"][b], n)
        x = torch.cat((xp[b], q[b] @ ko.T.contiguous()), 1)
        if p["mask"] is not None:
            x[:, T:] += p["mask"][b].expand(G, Lq, -1)[..., :n].reshape(G * Lq, n).double()
        mag = torch.cat((mp[b], q[b].abs() @ ko.abs().T.contiguous()), 1).amax(1) if T + n else x.new_zeros(G * Lq)
        v = torch.cat((vp, vo))
        if T + n == 0:
            res.append((x.new_zeros(G * Lq, D), x.new_full((G * Lq,), -math.inf), mag, x.new_zeros(G * Lq, D)))
            continue
        w = torch.softmax(x, 1)
        res.append((w @ v, torch.logsumexp(x, 1), mag, w @ v.abs()))
    return [torch.stack(t).view(B, G, Lq, *t[0].shape[1:]) for t in zip(*res)]


@pytest.mark.parametrize("name", CASES)
def test_forms_of_large_calls(name):
    c, want = CASES[name]
    c = {**BASE, **c}
    p = _problem(c)
    width = p["table"].shape[1]
    plan = _plan(c, width, c["kept"])
    log(f"decode_prefix {name}: {plan}")
    tiles = (c["T"] + 31) // 32
    slice_tiles = -(-tiles // plan["slices"]) if plan["slices"] else 0
    items = plan["groups"] * (-(-tiles // slice_tiles) if slice_tiles else 0)
    waves, groups = 4 * plan["wgs"], -(-(c["Hq"] // c["Hkv"] * c["Lq"]) // 32)
    own = [-(-n // 32) for n in c["lens"] for _ in range(groups)]
    reached = {
        "nr2": plan["nr"] == 2,
        "deep": slice_tiles > 4 * 64,
        "deep32": slice_tiles > 4 * 32,
        "rounds": items > plan["wgs"],
        "own_rounds": plan["pieces"] > 0 and sum(-(-t // plan["least"]) for t in own) > waves,
        "own_deep": sum(own) // waves > 64,
    }
    for w in want.split():
        assert reached[w], (w, plan)
    scale = 1 / math.sqrt(c["D"])
    out, lse = _call(p, scale)
    # the bounds of tests/test_gpu_decode_prefix.py, from the same arithmetic; f16's and bf16's half steps
    half = torch.finfo(c["vdt"]).eps / 2
    tiny = 2.0 ** -24 if c["vdt"] == F16 else 0.0
    G = c["Hq"] // c["Hkv"]
    for h in (0, c["Hkv"] // 2 - 1, c["Hkv"] - 1):
        ref, rlse, mag, pv = _head64(p, scale, h, c)
        o, s = out[:, h * G:(h + 1) * G].double(), lse[:, h * G:(h + 1) * G].double()
        empty = rlse == -math.inf
        assert (s[empty] == -math.inf).all() and (o[empty] == 0).all()
        dx = 2.0 ** -15 * mag + 1e-5
        assert ((s - rlse).abs()[~empty] <= (dx + 2.0 ** -22 * rlse.abs())[~empty]).all(), f"{name}, KV head {h}: lse"
        bound = half * ref.abs() + (2 * dx[..., None] + half + 1e-5) * pv + tiny * (1 + pv) + 1e-30
        err = (o - ref).abs()
        assert (err <= bound).all(), f"{name}, KV head {h}: out {(err / bound).max().item():.2f} times the bound"
    # every row against the decode kernels that serve every codec, which hold their own tests: both within their bounds,
    # a logit's magnitude at most that of the largest codeword of every block, sum p |v| at most the largest |v|
    out1, lse1 = _call(p, scale, kernel=1)
    top = p["cent"].abs().amax(2).reshape(c["Hkv"], c["D"])
    if p["heavy"]:
        kept = torch.tensor(p["heavy"], device=DEV).repeat_interleave(c["bd"])
        top[:, kept] = p["pt"].float().abs().amax()
    qa = torch.gather((p["q"].float().abs() * scale), 3, p["perm"].repeat_interleave(G, 0)[None, :, None].expand_as(p["q"]))
    dx = 2 * (2.0 ** -15 * (qa * top.repeat_interleave(G, 0)[None, :, None]).sum(-1) + 1e-5)
    live = lse1 != -math.inf
    assert torch.equal(live, lse != -math.inf)
    assert ((lse - lse1).abs()[live] <= (dx + 2.0 ** -21 * lse1.abs())[live]).all(), f"{name}: lse of every row"
    vmax = p["v"][1:].float().abs().amax()
    bound = half * (out.float().abs() + out1.float().abs()) + (2 * dx[..., None] + 2 * half) * vmax + 2 * tiny + 1e-30
    assert ((out.float() - out1.float()).abs() <= bound).all(), f"{name}: every row"
    again = _call(p, scale)
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])
