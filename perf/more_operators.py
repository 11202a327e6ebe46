"""The paged cache with values in 8 bits, as cases that can be timed and checked.

Three operators: the append of values to pages in e4m3 with one scale per page and KV head, by itself
(``values``) or beside the keys' codes (``append``); causal attention of the newest tokens over such pages, or
16-bit ones, with a sliding window and first tokens that stay visible (``window``); and the copy of pages,
which forks and compacts a cache (``copy``).  ``prepare`` makes what the program holds before the call;
``run`` is the call, in elementary torch operations or, with ``own``, through the framework; ``exact`` is the
same from the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 16
E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LEAST = 2.0 ** -100  # the smallest scale of a page

# kind: the operator.  B sequences, Hq / Hkv query and KV heads, head_dim D (of keys and values), S new tokens
# a sequence, dtype of queries and values; bd: block dim, nc: codewords a block; T: the longest sequence's
# tokens, rag: lengths spread evenly between T / 4 and T; v8: values in 8 bits; window: 0 is all; N: pages.
DEFAULTS = {"B": 1, "Hq": 32, "Hkv": 8, "D": 128, "S": 1, "dtype": "bf16", "bd": 4, "nc": 256, "T": 0, "rag": False,
            "v8": True, "window": 0, "sinks": 0, "pad": 0.0, "N": 0}


def _case(kind, **kw):
    return {**DEFAULTS, "kind": kind, **kw}


def listed():
    return [
        # one chat's decode step in the small GQA layer: the smallest attention, fixed costs
        _case("window", name="window_chat_1", Hq=14, Hkv=2, D=64, T=517),
        # a full batch on 32k tokens each, everything visible: the largest, the cache's bytes
        _case("window", name="window_32k_full", B=64, T=32768),
        # chats of every length up to 8k at the default 4 bits/dim
        _case("window", name="window_8k_ragged", B=48, T=8192, rag=True, bd=2),
        # streaming chats: 4,096 tokens and 4 sinks stay visible of up to 32k
        _case("window", name="window_4k_sinks", B=64, T=32768, rag=True, window=4096, sinks=4),
        # verification of 5 tokens a sequence over 16-bit values, odd window, causal among the new tokens
        _case("window", name="window_verify_5", B=16, S=5, T=16001, rag=True, window=1001, sinks=17, dtype="f16", v8=False),
        # one long document: the work is split along it
        _case("window", name="window_long_1", T=131071),
        # a chunk of a long prompt, each token with its own window
        _case("window", name="window_chunk_512", S=512, T=16384, window=4096, sinks=4),
        # one decode step's keys and values of 64 sequences, values to 8 bits
        _case("append", name="append8_step_64", B=64),
        # a step of a mixed batch: 5 rows a sequence, a third of them padding
        _case("values", name="values8_mixed_padded", B=37, S=5, Hq=14, Hkv=2, D=64, pad=0.34, dtype="f16"),
        # a long prompt's values
        _case("values", name="values8_prompt_32k", S=32768),
        # 64 forks of one prompt: each its own copy of the last page
        _case("copy", name="copy_fork_64", N=64),
        # a cache compacted: 16,384 pages move
        _case("copy", name="copy_compact_16k", N=16384),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["window", "window", "window", "append", "values", "copy"])
    hq, hkv, d = rng.choice([(14, 2, 64), (32, 8, 128), (32, 8, 128), (64, 8, 128)])
    c = {"Hq": hq, "Hkv": hkv, "D": d, "dtype": rng.choice(["bf16", "bf16", "f16"])}
    if kind == "window":
        c["bd"], c["nc"] = rng.choice([(2, 256), (4, 256), (4, 256), (8, 256), (2, 64)])
        c["B"] = _log(rng, 1, 64)
        c["S"] = rng.choice([1, 1, 1, 1, 4, 13]) if c["B"] <= 32 else 1
        c["T"] = _log(rng, 16, min(131072, (1 << 20) // c["B"]))
        c["rag"] = rng.random() < 0.6
        c["v8"] = rng.random() < 0.75
        if rng.random() < 0.5:
            c["window"] = _log(rng, 1, c["T"])
            c["sinks"] = rng.choice([0, 0, 4, 37])
    elif kind == "copy":
        c["N"] = _log(rng, 1, 16384)
        c["bd"] = rng.choice([2, 4, 8])
    else:
        c["B"] = _log(rng, 1, 128)
        c["S"] = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, (1 << (11 if kind == "append" else 15)) // c["B"]))
        c["pad"] = rng.choice([0.0, 0.0, 0.3])
        if kind == "values":
            c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
    return _case(kind, **c)


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = {**DEFAULTS, **case}
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7193 + 41)
    dt = DTYPES[c["dtype"]]
    B, Hq, H, D, S, bd, nc = (c[k] for k in ("B", "Hq", "Hkv", "D", "S", "bd", "nc"))
    nb = D // bd
    s = {"case": c}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def pages8(n):  # e4m3 values and the scales of a cache that holds tokens: maxima of 3 to 6 times the spread
        v = randn(n, H, D, PAGE).mul_(64.0).clamp_(-448.0, 448.0).to(E4M3)
        return v, torch.exp2(torch.randint(-8, -5, (n, H), generator=g, device=dev).float())

    if c["kind"] == "copy":
        n = c["N"]
        v, vs = pages8(2 * n + 3)
        codes = torch.randint(0, 256, (2 * n + 3, H, PAGE, nb), generator=g, device=dev, dtype=torch.uint8)
        s["pools"] = [codes, v, vs]
        order = torch.randperm(2 * n + 3, generator=g, device=dev)
        s["src"], s["dst"] = order[:n].contiguous(), order[n:2 * n].contiguous()
        return s
    # one spread per channel, as K projections have
    sigma = torch.exp(torch.rand(D, generator=g, device=dev) * math.log(30.0) + math.log(0.1))
    s["perm"] = torch.randperm(D, generator=g, device=dev)
    s["cent"] = randn(H, nb, nc, bd) * sigma[s["perm"]].view(nb, 1, bd)
    if c["kind"] in ("append", "values"):
        s["k"] = (randn(B, S, H, D) * sigma).to(dt).transpose(1, 2)  # projections come token-major
        s["v"] = randn(B, S, H, D).to(dt).transpose(1, 2)
        per = (S + PAGE - 1) // PAGE + 1
        pages = B * per + 8
        first = torch.randint(0, PAGE, (B, 1), generator=g, device=dev)
        table = torch.randperm(pages, generator=g, device=dev)[:B * per].view(B, per)
        live = torch.rand(B, S, generator=g, device=dev) >= c["pad"]
        live[0, 0] = True
        at = first + torch.cumsum(live.long(), 1) - 1  # padding rows lie between a sequence's tokens
        s["slots"] = torch.where(live, torch.gather(table, 1, at.clamp_min(0) // PAGE) * PAGE + at % PAGE, -1)
        s["v_pages"], s["v_scale"] = pages8(pages)
        s["codes"] = torch.zeros(pages, H, PAGE, nb, dtype=torch.uint8, device=dev)
        return s
    # queries whose logits spread by a few nats, as trained heads have: the codewords' norm is taken out
    s["scale"] = 1.0 / math.sqrt(D)
    s["q"] = (randn(B, S, Hq, D) * (2.0 / sigma.square().mean().sqrt())).to(dt).transpose(1, 2)
    lens = torch.full((B,), c["T"], device=dev, dtype=torch.int64)
    if c["rag"]:
        u = torch.rand(B, generator=g, device=dev)
        lens = (c["T"] * (0.25 + 0.75 * u)).round().to(torch.int64).clamp_min(min(S, c["T"]))
        lens[0] = c["T"]
    width = (c["T"] + PAGE - 1) // PAGE
    used = (lens + PAGE - 1) // PAGE
    total = int(used.sum())
    pool = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    col = torch.arange(width, device=dev)
    at = (torch.cumsum(used, 0) - used)[:, None] + col[None]
    s["table"] = torch.where(col[None] < used[:, None], pool[at.clamp_max(total - 1)], 0).to(torch.int32).contiguous()
    s["lens"] = lens.to(torch.int32)
    s["codes"] = torch.randint(0, nc, (total, H, PAGE, nb), generator=g, device=dev, dtype=torch.uint8)
    s["v_scale"] = None
    if c["v8"]:
        s["v_pages"], s["v_scale"] = pages8(total)
    else:
        s["v_pages"] = randn(total, H, D, PAGE).to(dt)
    return s


# ------------------------------------------------------------------------------------- plain forms
def _nearest(x, cent):
    """The first codeword with the smallest distance sqrt(max(0, -2 x.c + |x|^2 + |c|^2)), its terms in the
    codec's order: each multiply-add rounded once to 32 bits (its product and sum held in 64), so that codes
    next to a border are the same ones.  x [H, N, nb, bd], cent [H, nb, nc, bd]."""
    bd = x.shape[-1]
    cn, xn = cent[..., 0] * cent[..., 0], x[..., 0] * x[..., 0]
    acc = (-2.0 * x[..., 0]).unsqueeze(-1) * cent[..., 0].unsqueeze(1)
    for d in range(1, bd):
        cn, xn = cn + cent[..., d] * cent[..., d], xn + x[..., d] * x[..., d]
        acc = torch.addcmul(acc.double(), (-2.0 * x[..., d]).double().unsqueeze(-1), cent[..., d].double().unsqueeze(1)).float()
    acc = acc + xn.unsqueeze(-1)
    acc = acc + cn.unsqueeze(1)
    return torch.sqrt(acc.clamp_min_(0.0).double()).float().argmin(-1)


def _values(s, c):
    """Values to e4m3 pages.  A page's scale is the smallest power of two that holds its tokens within 448, no
    less than what it holds already unless its first token is among the new ones."""
    B, H, S, D = s["v"].shape
    flat = s["slots"].flatten()
    row = torch.where(flat < 0, 0, torch.arange(B * S, device=flat.device))  # a padded row repeats the first, which is none
    slot = flat[row]
    page, off = slot // PAGE, slot % PAGE
    v = s["v"].float().transpose(1, 2).reshape(B * S, H, D)[row]
    P = s["v_pages"].shape[0]
    most = torch.where(torch.isfinite(v), v.abs(), 0.0).amax(-1)
    need = torch.zeros(P, H, device=v.device).scatter_reduce_(0, page[:, None].expand(-1, H), most, "amax")
    m, e = torch.frexp(need)  # 448 is 0.875 * 2^9
    need = torch.ldexp(torch.ones_like(need), e - 9 + (m > 0.875).to(e.dtype)).clamp_min(LEAST)
    first = torch.full((P,), PAGE, device=v.device).scatter_reduce_(0, page, off, "amin")
    held = s["v_scale"]
    scale = torch.where((first < PAGE)[:, None], torch.where((first > 0)[:, None], torch.maximum(need, held), need), held)
    old = torch.arange(PAGE, device=v.device)[None] < torch.where(first < PAGE, first, 0)[:, None]
    again = (s["v_pages"].float() * (held / scale)[..., None, None]).to(E4M3)
    bits = torch.where(old[:, None, None], again.view(torch.uint8), s["v_pages"].view(torch.uint8))
    bits[page, :, :, off] = (v / scale[page][..., None]).to(E4M3).view(torch.uint8)
    s["v_pages"].view(torch.uint8).copy_(bits)
    s["v_scale"].copy_(scale)


def _codes(s, c):
    B, H, S, D = s["k"].shape
    rows = s["k"].transpose(0, 1).reshape(H, B * S, D)[..., s["perm"]].reshape(H, B * S, D // c["bd"], c["bd"])
    codes = _nearest(rows.float(), s["cent"]).transpose(0, 1)
    flat = s["slots"].flatten()
    row = torch.where(flat < 0, 0, torch.arange(B * S, device=flat.device))
    slot = flat[row]
    s["codes"][slot // PAGE, :, slot % PAGE] = codes[row].to(torch.uint8)


def _window(s, c):
    B, Hq, S, D = s["q"].shape
    H, G = c["Hkv"], Hq // c["Hkv"]
    q = (s["q"] * s["scale"]).float()[..., s["perm"]].reshape(B, H, G * S, D)  # the query is scaled in its own type
    table = s["table"].long()
    idx = s["codes"][table].long()  # [B, n, H, PAGE, nb]
    k = s["cent"][torch.arange(H, device=q.device)[:, None, None], torch.arange(idx.shape[-1], device=q.device), idx]
    k = k.flatten(-2).transpose(1, 2).flatten(2, 3)  # [B, H, T.., D]
    del idx
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()).view(B, H, G, S, -1)
    del k
    v = s["v_pages"][table] if s["v_scale"] is None else s["v_pages"].view(torch.uint8)[table].view(E4M3)
    v = v.float()
    if s["v_scale"] is not None:
        v = v * s["v_scale"][table][..., None, None]
    v = v.permute(0, 2, 1, 4, 3).flatten(2, 3)
    j = torch.arange(x.shape[-1], device=x.device)
    p = (s["lens"].long()[:, None] - S + torch.arange(S, device=x.device))[..., None]
    seen = (j <= p) & ((j > p - c["window"]) | (j < c["sinks"])) if c["window"] else j <= p
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x = torch.exp(x - m)
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(B, H, G * S, -1), v).view(B, H, G, S, D) / total
    return {"out": out.reshape(B, Hq, S, D).to(s["q"].dtype), "lse": (m + total.log()).reshape(B, Hq, S)}


# ------------------------------------------------------------------------------------- the calls
def run(s):
    c = s["case"]
    if own:
        from sunshape_amd import hip_ops

        if c["kind"] == "copy":
            hip_ops.copy_pages(s["pools"], s["src"], s["dst"])
            return s["pools"]
        if c["kind"] == "values":
            hip_ops.append_values(s["v"], s["v_pages"], s["v_scale"], s["slots"])
            return {"values": s["v_pages"], "scales": s["v_scale"]}
        if c["kind"] == "append":
            hip_ops.append_kv(s["k"], s["v"], s["perm"], s["cent"], codes_out=s["codes"], v_out=s["v_pages"],
                              v_scale=s["v_scale"], slot_mapping=s["slots"])
            return {"codes": s["codes"], "values": s["v_pages"], "scales": s["v_scale"]}
        out, lse = hip_ops.decode_window(s["q"], s["codes"], s["v_pages"], s["perm"], s["cent"], block_table=s["table"],
                                         seq_lens=s["lens"], scale=s["scale"], window=c["window"] or None,
                                         sinks=c["sinks"], v_scale=s["v_scale"], return_lse=True)
        return {"out": out, "lse": lse}
    if c["kind"] == "copy":
        for pool in s["pools"]:
            bits = pool.view(torch.uint8) if pool.dtype == E4M3 else pool
            bits[s["dst"]] = bits[s["src"]]
        return s["pools"]
    if c["kind"] == "window":
        return _window(s, c)
    _values(s, c)
    if c["kind"] == "values":
        return {"values": s["v_pages"], "scales": s["v_scale"]}
    _codes(s, c)
    return {"codes": s["codes"], "values": s["v_pages"], "scales": s["v_scale"]}


# ------------------------------------------------------------------------------------- what it takes
def _seen(c, n, i):
    """Tokens that new token i of a sequence of n sees."""
    p = n - c["S"] + i + 1
    if p <= 0:
        return 0
    return min(p, c["window"] + min(c["sinks"], max(0, p - c["window"]))) if c["window"] else p


def work(case):
    c = {**DEFAULTS, **case}
    B, Hq, H, D, S, bd = (c[k] for k in ("B", "Hq", "Hkv", "D", "S", "bd"))
    size = 4 if c["dtype"] == "f32" else 2
    nb = D // bd
    if c["kind"] == "copy":
        return {"bytes": 2.0 * c["N"] * (H * PAGE * (nb + D) + 4 * H) + 16.0 * c["N"], "flops": 0.0}
    if c["kind"] != "window":
        rows = B * S * H * (1.0 - c["pad"])
        bytes_, flops = rows * D * (size + 1) + B * S * 8.0 + rows / min(S, PAGE) * 8.0, rows * 2.0 * D
        if c["kind"] == "append":
            bytes_ += rows * (D * size + nb) + H * nb * c["nc"] * bd * 4 + D * 8
            flops += rows * nb * c["nc"] * (2.0 * bd + 2.0)
        return {"bytes": bytes_, "flops": flops}
    lens = [c["T"]] * B
    if c["rag"]:  # evenly between T / 4 and T
        lens = [c["T"]] + [c["T"] * (0.25 + 0.75 * (i + 0.5) / (B - 1)) for i in range(B - 1)]
    tokens = pairs = 0.0
    for n in lens:
        tokens += min(n, _seen(c, n, S - 1) + S - 1)
        pairs += S * (_seen(c, n, 0) + _seen(c, n, S - 1)) / 2
    return {"bytes": tokens * H * (nb + D * (1 if c["v8"] else size)) + 2.0 * B * S * Hq * D * size + 4.0 * B * S * Hq
            + H * nb * c["nc"] * bd * 4 + D * 8, "flops": pairs * Hq * 4.0 * D}


# ------------------------------------------------------------------------------------- 64 bits
def _values64(s):
    """Stored values over their scale, unrounded, and the scales."""
    vals, scales = s["v_pages"].double(), s["v_scale"].double()
    b, i = (s["slots"] >= 0).nonzero(as_tuple=True)
    slot = s["slots"][b, i]
    new = s["v"].double()[b, :, i]  # [n, H, D]
    order = torch.argsort(slot)
    slot, new = slot[order], new[order]
    pages, counts = torch.unique_consecutive(slot // PAGE, return_counts=True)
    at = 0
    for page, n in zip(pages.tolist(), counts.tolist()):
        rows, off = new[at:at + n], slot[at:at + n] % PAGE
        at += n
        top = rows.abs().amax((0, 2)) / 448.0
        least = torch.exp2(torch.ceil(torch.log2(top.clamp_min(LEAST))))
        least = torch.where(least / 2 >= top, least / 2, least).clamp_min(LEAST)  # should the logarithm have been a hair high
        first = off[0]
        now = torch.where(first > 0, torch.maximum(least, scales[page]), least)
        keep = torch.arange(PAGE, device=off.device) < first
        vals[page] = torch.where(keep, vals[page] * (scales[page] / now)[:, None, None], vals[page])
        vals[page][:, :, off] = rows.permute(1, 2, 0) / now[:, None, None]
        scales[page] = now
    return vals, scales


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] == "copy":  # what it moves are stored values
        found = []
        for pool in s["pools"]:
            if pool.dtype == torch.uint8:
                found.append(None)
                continue
            moved = pool.double()
            moved.index_copy_(0, s["dst"], pool.double().index_select(0, s["src"]))
            found.append(moved)
        return found
    if c["kind"] in ("values", "append"):
        vals, scales = _values64(s)
        return {"values": vals, "scales": scales} if c["kind"] == "values" else {"codes": None, "values": vals, "scales": scales}
    B, Hq, S, D = s["q"].shape
    H, G = c["Hkv"], Hq // c["Hkv"]
    q = (s["q"] * s["scale"]).double()[..., s["perm"]]
    out = torch.empty(B, Hq, S, D, dtype=torch.float64, device=q.device)
    lse = torch.empty(B, Hq, S, dtype=torch.float64, device=q.device)
    for b, n in enumerate(s["lens"].tolist()):
        pages = s["table"][b, :(n + PAGE - 1) // PAGE].long()
        pos = n - S + torch.arange(S, device=q.device)
        tok = torch.arange(n, device=q.device)
        gone = tok[None] > pos[:, None]
        if c["window"]:
            gone = gone | ((tok[None] <= pos[:, None] - c["window"]) & (tok[None] >= c["sinks"]))
        for h in range(H):
            idx = s["codes"][pages, h].reshape(-1, D // c["bd"])[:n].long()
            k = torch.stack([s["cent"][h, j].double()[idx[:, j]] for j in range(idx.shape[1])], 1).reshape(n, D)
            v = s["v_pages"].view(torch.uint8)[pages, h].view(E4M3) if c["v8"] else s["v_pages"][pages, h]
            v = v.double()
            if c["v8"]:
                v = v * s["v_scale"][pages, h].double()[:, None, None]
            v = v.transpose(1, 2).reshape(-1, D)[:n]
            x = torch.matmul(q[b, h * G:(h + 1) * G], k.T)
            x = x.masked_fill(gone[None], -math.inf)
            lse[b, h * G:(h + 1) * G] = torch.logsumexp(x, -1)
            out[b, h * G:(h + 1) * G] = torch.softmax(x, -1) @ v
    return {"out": out, "lse": lse}
