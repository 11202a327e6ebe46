"""Plain forms of the 8-bit cache's operators (CPU, 64 bits where they compute), and the inputs their GPU tests share."""

from __future__ import annotations

import math

import torch

from _step import codec_arrays, keys64

E4M3 = torch.float8_e4m3fn
LEAST = 2.0 ** -100
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}  # half a step, relative


def scale_of(top: float) -> float:
    """The smallest power of two s >= 2^-100 with top <= 448 s."""
    s = LEAST
    if top > 448.0 * LEAST:
        m, e = math.frexp(top)
        s = math.ldexp(1.0, e - 9 + (m > 0.875))
    assert top <= 448.0 * s and (s == LEAST or top > 224.0 * s)
    return s


def values_plain(v, pages, scale, slots):
    """append_values on CPU tensors: new (pages, scale)."""
    pages, scale = pages.clone(), scale.clone()
    P, H, D, page = pages.shape
    B, _, S, _ = v.shape
    runs = {}
    for b in range(B):
        for s in range(S):
            x = int(slots[b, s])
            if 0 <= x < P * page:
                runs.setdefault(x // page, []).append((x % page, b, s))
    raw = pages.view(torch.uint8)
    for pg, toks in runs.items():
        first = min(t[0] for t in toks)
        for h in range(H):
            rows = torch.stack([v[b, h, s].double() for _, b, s in toks])
            top = torch.where(torch.isfinite(rows), rows.abs(), 0.0).max().item()
            held = scale[pg, h].item()
            now = max(held, scale_of(top)) if first else scale_of(top)
            if first and now != held:
                old = pages[pg, h, :, :first].float() * (held / now)
                raw[pg, h, :, :first] = old.to(E4M3).view(torch.uint8)
            for (off, _, _), r in zip(toks, rows):
                x = torch.where(torch.isfinite(r), r / now, math.nan).float()  # exact, or below e4m3's smallest
                raw[pg, h, :, off] = x.to(E4M3).view(torch.uint8)
            scale[pg, h] = now
    return pages, scale


def same_values(a, b):
    """e4m3 tensors equal in value (any NaN equals any)."""
    x, y = a.float(), b.float()
    return bool(((x == y) | (torch.isnan(x) & torch.isnan(y))).all())


def problem(seed, *, B, Hq, Hkv, D, Lq=1, T, lens=None, bd=4, nc=256, page=16, vt=E4M3, qt=torch.bfloat16, per_head=True,
            spread=3, gain=2.0):
    """A random problem of decode_window (CPU tensors): pages in any order, lengths up to T."""
    import numpy as np

    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    perm, cent, _, _ = codec_arrays(rng, Hkv, D, bd, nc, per_head)
    lens = torch.tensor(lens if lens is not None else [T] + [int(rng.integers(0, T + 1)) for _ in range(B - 1)])
    width = (T + page - 1) // page
    need = (lens + page - 1) // page
    P = int(need.sum()) + 3
    order = torch.randperm(P, generator=g)
    table = torch.full((B, max(width, 1)), -7, dtype=torch.int32)  # what no row sees is not used
    at = 0
    for b in range(B):
        n = int(need[b])
        table[b, :n] = order[at:at + n].to(torch.int32)
        at += n
    nb = D // bd
    codes = torch.randint(0, nc, (P, Hkv, page, nb), generator=g, dtype=torch.int32).to(torch.uint8)
    v = torch.randn(P, Hkv, D, page, generator=g)
    scale = None
    if vt == E4M3:
        v = (v * 64).clamp(-448, 448).to(E4M3)
        scale = torch.exp2(torch.randint(-spread, spread + 1, (P, Hkv), generator=g).float())
    else:
        v = v.to(vt)
    norm = float(cent.square().mean().sqrt())
    q = (torch.randn(B, Lq, Hq, D, generator=g) * (gain / norm)).to(qt).transpose(1, 2)
    return dict(q=q, codes=codes, v=v, perm=perm, cent=cent, block_table=table, seq_lens=lens.to(torch.int32), v_scale=scale,
                scale=1.0 / math.sqrt(D))


def sees(n, Lq, i, window, sinks):
    p = n - Lq + i
    j = torch.arange(n)
    ok = j <= p
    return ok & ((j > p - window) | (j < sinks)) if window else ok


def window64(pr, window=None, sinks=0):
    """out, lse, the bound on a row's logits' errors, and sum p |v| (64 bits)."""
    q, perm, cent = pr["q"], pr["perm"], pr["cent"]
    B, Hq, Lq, D = q.shape
    P, Hkv, page, nb = pr["codes"].shape
    G = Hq // Hkv
    qs = (q * pr["scale"] if pr["scale"] is not None else q).double()
    out = torch.zeros(B, Hq, Lq, D, dtype=torch.float64)
    lse = torch.full((B, Hq, Lq), -math.inf, dtype=torch.float64)
    off, pv = torch.zeros(B, Hq, Lq, dtype=torch.float64), torch.zeros(B, Hq, Lq, D, dtype=torch.float64)
    for b in range(B):
        n = int(pr["seq_lens"][b])
        vis = [sees(n, Lq, i, window, sinks) for i in range(Lq)]
        need = torch.stack(vis).any(0)
        toks = need.nonzero()[:, 0]
        if not len(toks):
            continue
        pg, at = pr["block_table"][b].long()[toks // page], toks % page
        for h in range(Hkv):
            k = keys64(pr["codes"][pg, h, at], cent, None, None, h)
            v = pr["v"].view(torch.uint8)[pg, h, :, at].view(E4M3).double() if pr["v"].dtype == E4M3 else pr["v"][pg, h, :, at].double()
            if pr["v_scale"] is not None:
                v = v * pr["v_scale"].double()[pg, h][:, None]
            pm = perm[h] if perm.ndim == 2 else perm
            for i in range(Lq):
                m = vis[i][toks]
                if not m.any():
                    continue
                rows = qs[b, h * G:(h + 1) * G, i][:, pm]
                x = rows @ k[m].T
                p = torch.softmax(x, -1)
                out[b, h * G:(h + 1) * G, i] = p @ v[m]
                lse[b, h * G:(h + 1) * G, i] = torch.logsumexp(x, -1)
                off[b, h * G:(h + 1) * G, i] = (rows.abs() @ k[m].abs().T).amax(-1)
                pv[b, h * G:(h + 1) * G, i] = p @ v[m].abs()
    return out, lse, off, pv


def window_bounds(pr, out, lse, mag, pv, out_dtype):
    """What out and lse may be off by, from the roundings.

    A logit: codewords in two f16 parts (2^-22 of each product), fp32 queries too, and sums of 2 D (4 D) products
    in fp32, each partial sum rounded: (2^-21 + 4 * 128 * 2^-24) sum |q||k| at the very most, its factor of log2(e) and the
    subtraction of m (below 2^10 in size: 2^-14 absolute would need logits of 1,000; they stay below 2^7, 2^-17).
    A weight: twice that, its rounding to 16 bits (f16, or bf16 with bf16 values; halves of a step) and its page's
    factor; exp2 and the fp32 sums over at most 2^12 terms a lane and 2^11 joins: 2^-11 each at the very most."""
    p16 = HALF[torch.bfloat16] if pr["v"].dtype == torch.bfloat16 else HALF[torch.float16]
    logit = (2.0 ** -21 + 512 * 2.0 ** -24) * mag + 2.0 ** -17
    tiny = 2.0 ** -25 if out_dtype == torch.float16 else 0.0
    ob = HALF[out_dtype] * out.abs() * 1.001 + (p16 + 2.0 ** -12 + 2 * logit[..., None]) * pv * 1.001 + tiny + 1e-30
    lb = logit + 2.0 ** -12 + 2.0 ** -22 * torch.where(torch.isfinite(lse), lse.abs(), 0.0)
    return ob, lb
