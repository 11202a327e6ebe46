"""Plain 64-bit forms of the serving step's operators, on the CPU, and the inputs their GPU tests share."""

from __future__ import annotations

import math

import numpy as np
import torch

DEV = torch.device("cuda:0")


def turn64(x, w, cos, sin, positions, eps=1e-6, interleaved=False):
    """Norm and rotation of [B, H, S, D] from the formulas; also the sum of the magnitudes that a rotated
    dim is made of (the scale of its rounding errors)."""
    u = x.double()
    if w is not None:
        u = u / torch.sqrt(u.square().mean(-1, keepdim=True) + eps) * w.double()
    y, mag = u.clone(), u.abs()
    if cos is not None:
        r = cos.shape[1]
        c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
        i0 = torch.arange(r) * 2 if interleaved else torch.arange(r)
        i1 = i0 + 1 if interleaved else i0 + r
        a, b = u[..., i0], u[..., i1]
        y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
        mag[..., i0], mag[..., i1] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    return y, mag


def turn_bound(y, mag, dtype):
    """Rounding of the result (half a step of its dtype; f16 also of its subnormals) and of the fp32 work
    before it: the norm's r and two products, a rotation's product and sum, and the weight's none: 5 roundings
    of 2^-24 on each magnitude."""
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return torch.finfo(dtype).eps / 2 * y.abs() * (1 + 1e-6) + 6 * 2.0 ** -24 * mag + tiny + 1e-300


def codec_arrays(rng, Hkv, D, bd, nc, per_head=True, heavy=()):
    """perm, centroids, heavy mask, spread per channel (CPU tensors)."""
    nb = D // bd
    sigma = np.exp(rng.uniform(math.log(0.2), math.log(3.0), D))
    heads = Hkv if per_head else 1
    perm = np.stack([rng.permutation(D) for _ in range(heads)])
    cent = rng.standard_normal((heads, nb, nc, bd)) * sigma[perm].reshape(heads, nb, 1, bd)
    mask = None
    if heavy:
        mask = [i in heavy for i in range(nb)]
        cent[:, list(heavy)] = 0.0
    perm, cent = torch.from_numpy(perm), torch.from_numpy(cent.astype(np.float32))
    return (perm, cent, mask, sigma) if per_head else (perm[0], cent[0], mask, sigma)


def unsigned(codes):
    """Stored codes as int64."""
    c = codes.detach().cpu()
    return (c.to(torch.int64) & 0xFFFF) if c.dtype == torch.int16 else c.to(torch.int64)


def keys64(codes, cent, pt, mask, h):
    """Keys of KV head h in the codec's basis, [T, D], from codes [T, nb] (and kept values [T, n, bd])."""
    c = (cent[h] if cent.ndim == 4 else cent).double()
    nb, nc, bd = c.shape
    k = c.reshape(nb * nc, bd)[unsigned(codes) + torch.arange(nb) * nc]
    if mask is not None:
        k[:, torch.tensor(mask)] = pt.double()
    return k.reshape(len(k), nb * bd)


def prefix_attention64(q, scale, perm, cent, code_pages, v_pages, ptable, plen, table, lens, own_mask=None, pt=None, mask=None):
    """out, lse, and the scale of what may be off: the largest sum |q||k| of a row's logits, and sum p |v| (CPU)."""
    B, Hq, Lq, D = q.shape
    Hkv, page = code_pages.shape[1], code_pages.shape[2]
    G, Dv = Hq // Hkv, v_pages.shape[2]
    qs = (q * scale if scale is not None else q).double()
    out, lse = torch.zeros(B, Hq, Lq, Dv, dtype=torch.float64), torch.full((B, Hq, Lq), -math.inf, dtype=torch.float64)
    mag, pv = torch.zeros(B, Hq, Lq, dtype=torch.float64), torch.zeros(B, Hq, Lq, Dv, dtype=torch.float64)

    def tokens(tab, n, h):
        pages = tab[:(n + page - 1) // page].long()
        codes = code_pages[pages, h].reshape(-1, code_pages.shape[-1])[:n]
        p = None if pt is None else pt[pages, h].reshape(-1, pt.shape[3], pt.shape[4])[:n]
        k = keys64(codes, cent, p, mask, h) if n else torch.zeros(0, D, dtype=torch.float64)
        return k, v_pages[pages, h].double().transpose(1, 2).reshape(-1, Dv)[:n]

    for h in range(Hkv):
        kp, vp = tokens(ptable, plen, h)
        pm = perm[h] if perm.ndim == 2 else perm
        for b in range(B):
            ko, vo = tokens(table[b], int(lens[b]), h)
            k, v = torch.cat((kp, ko)), torch.cat((vp, vo))
            if not len(k):
                continue
            for g in range(G):
                for i in range(Lq):
                    row = qs[b, h * G + g, i][pm]
                    x = k @ row
                    if own_mask is not None:
                        m = own_mask.expand(B, Hq, Lq, own_mask.shape[-1])[b, h * G + g, i]
                        x[plen:] += m[:int(lens[b])].double()
                    if x.max() == -math.inf:
                        continue
                    p = torch.softmax(x, 0)
                    at = (b, h * G + g, i)
                    out[at], lse[at] = p @ v, torch.logsumexp(x, 0)
                    mag[at], pv[at] = (k.abs() @ row.abs()).max(), p @ v.abs()
    return out, lse, mag, pv
