"""A serving step's operators around the quantized-key cache, as cases that can be timed and checked.

Three operators: the per-head norm and position rotation of queries and keys (``rope``), the append of
raw keys and values to the paged cache with that rotation applied on the way (``append``), and decode
attention for a batch whose sequences share a long prefix (``prefix``).  ``prepare`` makes what the program
holds before the call; ``run`` is the call, in elementary torch operations or, with ``own``, through the
framework; ``exact`` is the same from the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

PAGE = 16
EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# kind: the operator.  B sequences, Hq / Hkv query and KV heads, head_dim D, S new tokens a sequence,
# dtype of queries, keys and values; rot: rotated dims (0: all), inter: pairs (2i, 2i + 1) instead of
# halves, norm: per-head RMS norm with weights; bd: block dim, nc: codewords a block, heavy: passthrough
# blocks, pad: the share of padded rows (slot -1); T: tokens of the shared prefix, own: the longest
# sequence's own tokens (ragged, log-spread), mask: causal over the S new tokens of each sequence.
DEFAULTS = {"B": 1, "Hq": 32, "Hkv": 8, "D": 128, "S": 1, "dtype": "bf16", "rot": 0, "inter": False, "norm": True,
            "bd": 4, "nc": 256, "heavy": 0, "pad": 0.0, "T": 0, "own": 0, "mask": False}


def _case(kind, **kw):
    return {**DEFAULTS, "kind": kind, **kw}


def listed():
    return [
        # one decode step of a full batch: the smallest call, where the launch is the cost
        _case("rope", name="rope_step_64", B=64),
        # a ragged prompt batch of the small GQA layer, half of each head rotated in adjacent pairs, no norm
        _case("rope", name="rope_partial_517", B=3, S=517, Hq=14, Hkv=2, D=64, dtype="f16", rot=32, inter=True, norm=False),
        # one long prompt: every query and key of 32k tokens once through
        _case("rope", name="rope_prompt_32k", S=32768),
        # one decode step's keys and values of 64 sequences into the pages
        _case("append", name="append_step_64", B=64),
        # a step of a mixed batch at 4 bits/dim with passthrough blocks: 5 rows a sequence, a third of them padding
        _case("append", name="append_mixed_padded", B=37, S=5, Hq=14, Hkv=2, D=64, bd=2, heavy=4, pad=0.34),
        # a chunk of a long prompt at 2 bits/dim
        _case("append", name="append_prompt_8k", S=8192),
        # a chunk at 3 bits/dim (4,096 codewords of dim 4, 16-bit codes), no norm
        _case("append", name="append_3bit_1k", S=1024, nc=4096, norm=False),
        # a few chats on a short system prompt: fixed costs
        _case("prefix", name="prefix_short", B=5, Hq=14, Hkv=2, D=64, T=517, own=37),
        # 48 chats of every length up to 2k on an 8k prompt at the default 4 bits/dim
        _case("prefix", name="prefix_8k_ragged", B=48, T=8192, own=2048, bd=2),
        # 64 sequences sampled from one 32k document
        _case("prefix", name="prefix_32k", B=64, T=32768, own=512),
        # speculative verification of 4 tokens a sequence, fp16, causal among the new tokens
        _case("prefix", name="prefix_verify_4", B=16, S=4, T=16001, own=300, dtype="f16", mask=True),
        # many samples from one long document, 8 query heads a KV head
        _case("prefix", name="prefix_64k_batch", B=128, Hq=64, T=65536, own=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "prefix", "prefix"])
    hq, hkv, d = rng.choice([(14, 2, 64), (32, 8, 128), (32, 8, 128), (64, 8, 128)])
    c = {"Hq": hq, "Hkv": hkv, "D": d, "dtype": rng.choice(["bf16", "bf16", "f16"])}
    c["norm"] = rng.random() < 0.5
    if kind == "rope":
        c["B"] = _log(rng, 1, 128)
        c["S"] = _log(rng, 1, (1 << 15) // c["B"])
        c["inter"] = rng.random() < 0.3
        c["rot"] = rng.choice([0, 0, d // 2])
        c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
        if c["dtype"] == "f32":
            c["S"] = max(1, c["S"] // 2)
    elif kind == "append":
        c["bd"], c["nc"] = rng.choice([(2, 256), (4, 256), (4, 256), (8, 256), (2, 64), (4, 4096)])
        c["B"] = _log(rng, 1, 128)
        most = 1 << (13 if c["nc"] == 256 else 12 if c["nc"] < 256 else 10)
        c["S"] = 1 if rng.random() < 0.4 else _log(rng, 1, max(1, most // c["B"]))
        c["heavy"] = 4 if c["bd"] <= 4 and c["nc"] == 256 and rng.random() < 0.3 else 0
        c["pad"] = rng.choice([0.0, 0.0, 0.3])
        c["inter"] = rng.random() < 0.3
        c["rot"] = rng.choice([0, 0, d // 2])
    else:
        c["bd"], c["nc"] = rng.choice([(2, 256), (4, 256), (4, 256), (8, 256), (2, 64)])
        c["B"] = _log(rng, 2, 128)
        c["S"] = rng.choice([1, 1, 1, 1, 3]) if c["B"] <= 32 else 1
        c["mask"] = c["S"] > 1
        c["T"] = _log(rng, 16, 65536 if c["B"] * hq <= 4096 else 32768)
        c["own"] = _log(rng, max(1, c["S"]), 2048 if c["B"] <= 64 else 700)
    return _case(kind, **c)


# ------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c = {**DEFAULTS, **case}
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 6113 + 29)
    dt = DTYPES[c["dtype"]]
    B, Hq, Hkv, D, S = (c[k] for k in ("B", "Hq", "Hkv", "D", "S"))
    s = {"case": c}

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    # one spread per channel, as K projections have
    sigma = torch.exp(torch.rand(D, generator=g, device=dev) * math.log(30.0) + math.log(0.1))
    if c["kind"] in ("rope", "append"):
        rot = c["rot"] or D
        start = torch.randint(0, 4096, (B, 1), generator=g, device=dev)
        s["positions"] = start + torch.arange(S, device=dev)[None]
        freq = 10000.0 ** (-torch.arange(0, rot, 2, device=dev, dtype=torch.float64) / rot)
        ang = torch.arange(4096 + S, device=dev, dtype=torch.float64)[:, None] * freq[None]
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
        s["wq"] = s["wk"] = None
        if c["norm"]:
            s["wq"] = (1.0 + 0.2 * randn(D)).to(dt)
            s["wk"] = (sigma * (1.0 + 0.1 * randn(D))).to(dt)
        # projections come token-major, [B, S, H, D] seen as [B, H, S, D]
        s["k"] = (randn(B, S, Hkv, D) * (1.0 if c["norm"] else sigma)).to(dt).transpose(1, 2)
        if c["kind"] == "rope":
            s["q"] = randn(B, S, Hq, D).to(dt).transpose(1, 2)
            return s
    bd, nc = c["bd"], c["nc"]
    nb = D // bd
    s["perm"] = torch.randperm(D, generator=g, device=dev)
    spread = sigma[s["perm"]].view(nb, 1, bd)
    s["cent"] = randn(Hkv, nb, nc, bd) * spread
    code_t = torch.uint8 if nc <= 256 else torch.int16
    s["heavy"] = None
    if c["heavy"]:
        kept = torch.sort(torch.topk(spread.square().sum((1, 2)), c["heavy"]).indices).values
        s["cent"][:, kept] = 0.0
        s["kept"] = kept
        s["heavy"] = [i in set(kept.tolist()) for i in range(nb)]
    if c["kind"] == "append":
        s["v"] = randn(B, S, Hkv, D).to(dt).transpose(1, 2)
        per = (S + PAGE - 1) // PAGE + 1
        pages = B * per + 8
        first = torch.randint(0, PAGE, (B, 1), generator=g, device=dev)
        table = torch.randperm(pages, generator=g, device=dev)[:B * per].view(B, per)
        at = first + torch.arange(S, device=dev)[None]
        s["slots"] = torch.gather(table, 1, at // PAGE) * PAGE + at % PAGE
        if c["pad"]:
            gone = torch.rand(B, S, generator=g, device=dev) < c["pad"]
            gone[0, 0] = False
            s["slots"] = torch.where(gone, -1, s["slots"])
        s["codes"] = torch.zeros(pages, Hkv, PAGE, nb, dtype=code_t, device=dev)
        s["v_pages"] = torch.zeros(pages, Hkv, D, PAGE, dtype=dt, device=dev)
        s["pt"] = torch.zeros(pages, Hkv, PAGE, c["heavy"], bd, dtype=dt, device=dev) if c["heavy"] else None
        return s
    # queries whose logits spread by a few nats, as trained heads have: the codewords' norm is taken out
    s["scale"] = 1.0 / math.sqrt(D)
    s["q"] = (randn(B, S, Hq, D) * (2.0 / sigma.square().mean().sqrt())).to(dt).transpose(1, 2)
    u = torch.rand(B, generator=g, device=dev)
    lo = max(1, S)
    lens = torch.exp(math.log(lo) + u * math.log(max(c["own"] / lo, 1.0))).round().to(torch.int64).clamp_(lo, c["own"])
    lens[0] = c["own"]
    per, pre = (lens + PAGE - 1) // PAGE, (c["T"] + PAGE - 1) // PAGE
    width = (c["own"] + PAGE - 1) // PAGE
    total = B * width + pre
    pool = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    s["prefix_table"] = pool[:pre].contiguous()
    col = torch.arange(width, device=dev)
    s["table"] = torch.where(col[None] < per[:, None], pool[pre:].view(B, width), 0).to(torch.int32).contiguous()
    s["lens"] = lens.to(torch.int32)
    s["prefix_len"] = torch.tensor([c["T"]], dtype=torch.int32, device=dev)
    s["codes"] = torch.randint(0, nc, (total, Hkv, PAGE, nb), generator=g, device=dev, dtype=torch.int32).to(code_t)
    s["v_pages"] = randn(total, Hkv, D, PAGE).to(dt)
    s["mask"] = None
    if c["mask"]:  # the S new tokens are the last of each sequence's own
        pos = torch.arange(width * PAGE, device=dev)
        last = lens[:, None] - S + torch.arange(S, device=dev)[None]
        s["mask"] = torch.zeros(B, 1, S, width * PAGE, device=dev)
        s["mask"].masked_fill_(pos[None, None, None] > last[:, None, :, None], -math.inf)
    return s


# ------------------------------------------------------------------------------------- plain forms
def _rotated(x, w, s, c):
    """Norm (its sum in 64 bits) and rotation of [B, H, S, D] in 32 bits, rounded once."""
    u = x.float()
    if w is not None:
        mean = u.double().square().mean(-1, keepdim=True)
        u = u * (1.0 / torch.sqrt(mean + EPS)).float() * w.float()
    rot = c["rot"] or c["D"]
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    a, b = (u[..., 0:rot:2], u[..., 1:rot:2]) if c["inter"] else (u[..., :rot // 2], u[..., rot // 2:rot])
    y0, y1 = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((y0, y1), -1).flatten(-2) if c["inter"] else torch.cat((y0, y1), -1)
    return torch.cat((y, u[..., rot:]), -1).to(x.dtype)


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


def _append(s, c):
    k = _rotated(s["k"], s["wk"], s, c)
    B, H, S, D = k.shape
    rows = k.transpose(0, 1).reshape(H, B * S, D)[..., s["perm"]].reshape(H, B * S, D // c["bd"], c["bd"])
    codes = _nearest(rows.float(), s["cent"]).transpose(0, 1)
    # a padded row repeats the first row, which is none
    slots = s["slots"].flatten()
    row = torch.where(slots < 0, 0, torch.arange(B * S, device=slots.device))
    slots = slots[row]
    page, off = slots // PAGE, slots % PAGE
    if c["heavy"]:
        codes[..., s["kept"]] = 0
        s["pt"][page, :, off] = rows[:, :, s["kept"]].transpose(0, 1)[row]
    s["codes"][page, :, off] = codes[row].to(s["codes"].dtype)
    s["v_pages"][page, :, :, off] = s["v"].permute(0, 2, 1, 3).reshape(B * S, H, D)[row]
    return {"codes": s["codes"], "values": s["v_pages"], "passthrough": s["pt"]}


def _pages(s, table, c):
    """Keys in the codec's basis and values of the pages in `table` [..., n]: [..., Hkv, n * PAGE, D] in 32 bits."""
    idx = s["codes"][table].long()  # [..., n, Hkv, PAGE, nb]
    h = torch.arange(c["Hkv"], device=idx.device)[:, None, None]
    k = s["cent"][h, torch.arange(idx.shape[-1], device=idx.device), idx]
    k = k.flatten(-2).transpose(-4, -3).flatten(-3, -2)
    v = s["v_pages"][table].float().transpose(-1, -2).transpose(-4, -3).flatten(-3, -2)
    return k, v


def _prefix(s, c):
    B, Hq, S, D = s["q"].shape
    H, G, T = c["Hkv"], c["Hq"] // c["Hkv"], c["T"]
    q = (s["q"] * s["scale"]).float()[..., s["perm"]].reshape(B, H, G, S, D)  # the query is scaled in its own type
    kp, vp = _pages(s, s["prefix_table"].long(), c)  # [H, T.., D]
    x = torch.matmul(q.transpose(0, 1).reshape(H, B * G * S, D), kp.transpose(-1, -2).contiguous())
    x = x.masked_fill(torch.arange(x.shape[-1], device=x.device) >= s["prefix_len"], -math.inf)
    ko, vo = _pages(s, s["table"].long(), c)  # [B, H, W, D]
    y = torch.matmul(q.reshape(B, H, G * S, D), ko.transpose(-1, -2).contiguous()).view(B, H, G, S, -1)
    if s["mask"] is not None:
        y = y + s["mask"][:, :, None]
    gone = torch.arange(y.shape[-1], device=y.device)[None] >= s["lens"][:, None]
    y = y.masked_fill(gone[:, None, None, None], -math.inf)
    vo = vo.masked_fill(gone[:, None, :, None], 0.0)
    x = x.view(H, B, G, S, -1).transpose(0, 1)
    m = torch.maximum(x.amax(-1), y.amax(-1))[..., None]
    x, y = torch.exp(x - m), torch.exp(y - m)
    total = x.sum(-1) + y.sum(-1)
    o = torch.matmul(x.transpose(0, 1).reshape(H, B * G * S, -1), vp[:, :x.shape[-1]]).view(H, B, G, S, D).transpose(0, 1)
    o = o + torch.matmul(y.reshape(B, H, G * S, -1), vo).view(B, H, G, S, D)
    out = (o / total[..., None]).reshape(B, Hq, S, D).to(s["v_pages"].dtype)
    return {"out": out, "lse": (m[..., 0] + total.log()).reshape(B, Hq, S)}


# ------------------------------------------------------------------------------------- the calls
def run(s):
    c = s["case"]
    if own:
        from sunshape_amd import hip_ops

        if c["kind"] == "rope":
            q, k = hip_ops.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["positions"], q_weight=s["wq"],
                                        k_weight=s["wk"], eps=EPS, interleaved=c["inter"])
            return {"q": q, "k": k}
        if c["kind"] == "append":
            hip_ops.append_kv(s["k"], s["v"], s["perm"], s["cent"], codes_out=s["codes"], v_out=s["v_pages"],
                              slot_mapping=s["slots"], heavy=s["heavy"], pt_out=s["pt"], cos=s["cos"], sin=s["sin"],
                              positions=s["positions"], k_weight=s["wk"], eps=EPS, interleaved=c["inter"])
            return {"codes": s["codes"], "values": s["v_pages"], "passthrough": s["pt"]}
        out, lse = hip_ops.decode_prefix(s["q"], s["codes"], s["v_pages"], s["perm"], s["cent"], scale=s["scale"],
                                         prefix_table=s["prefix_table"], prefix_len=s["prefix_len"],
                                         block_table=s["table"], seq_lens=s["lens"], mask=s["mask"], return_lse=True)
        return {"out": out, "lse": lse}
    if c["kind"] == "rope":
        return {"q": _rotated(s["q"], s["wq"], s, c), "k": _rotated(s["k"], s["wk"], s, c)}
    return _append(s, c) if c["kind"] == "append" else _prefix(s, c)


# ------------------------------------------------------------------------------------- what it takes
def work(case):
    c = {**DEFAULTS, **case}
    B, Hq, Hkv, D, S, bd = (c[k] for k in ("B", "Hq", "Hkv", "D", "S", "bd"))
    size = 4 if c["dtype"] == "f32" else 2
    nb, width = D // bd, 1 if c["nc"] <= 256 else 2
    book = Hkv * nb * c["nc"] * bd * 4 + D * 8
    turn = B * S * ((c["rot"] or D) * 4 + 8)  # a token's row of the tables and its position
    if c["kind"] == "rope":
        n = B * S * (Hq + Hkv) * D
        return {"bytes": 2.0 * n * size + turn, "flops": n * (7.0 if c["norm"] else 3.0)}
    if c["kind"] == "append":
        rows = B * S * Hkv * (1.0 - c["pad"])
        return {"bytes": rows * (3 * D * size + nb * width + c["heavy"] * bd * size) + turn + book,
                "flops": rows * ((nb - c["heavy"]) * c["nc"] * (2.0 * bd + 2.0) + 7.0 * D)}
    lo = max(1, S)
    spread = c["own"] / lo
    mean = (c["own"] - lo) / math.log(spread) if spread > 1 else c["own"]  # of a log-spread length
    tokens = Hkv * (c["T"] + c["own"] + (B - 1) * mean)
    pairs = B * S * Hq * (c["T"] + (c["own"] + (B - 1) * mean) / B)
    return {"bytes": tokens * (nb * width + D * size) + 2.0 * B * S * Hq * D * size + 4.0 * B * S * Hq + book,
            "flops": pairs * 4.0 * D}


# ------------------------------------------------------------------------------------- 64 bits
def _turned64(x, w, s, c):
    u = x.double()
    if w is not None:
        u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + EPS) * w.double()
    rot = c["rot"] or c["D"]
    z = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]][:, None]
    pair = u[..., :rot].unflatten(-1, (rot // 2, 2) if c["inter"] else (2, rot // 2))
    pair = pair if c["inter"] else pair.transpose(-1, -2)
    t = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
    t = t if c["inter"] else t.transpose(-1, -2)
    return torch.cat((t.flatten(-2), u[..., rot:]), -1)


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] == "rope":
        return {"q": _turned64(s["q"], s["wq"], s, c), "k": _turned64(s["k"], s["wk"], s, c)}
    if c["kind"] == "append":  # a code is an index; what the call moves has a value
        live = (s["slots"] >= 0).nonzero()
        b, i = live[:, 0], live[:, 1]
        page, off = s["slots"][b, i] // PAGE, s["slots"][b, i] % PAGE
        values = s["v_pages"].double()
        values[page, :, :, off] = s["v"][b, :, i].double()
        kept = None
        if c["heavy"]:
            k = _turned64(s["k"], s["wk"], s, c)[b, :, i]
            kept = s["pt"].double()
            kept[page, :, off] = k[..., s["perm"]].unflatten(-1, (-1, c["bd"]))[..., s["kept"], :]
        return {"codes": None, "values": values, "passthrough": kept}
    B, Hq, S, D = s["q"].shape
    H, G = c["Hkv"], Hq // c["Hkv"]
    q = (s["q"] * s["scale"]).double()[..., s["perm"]]
    out = torch.empty(B, Hq, S, D, dtype=torch.float64, device=q.device)
    lse = torch.empty(B, Hq, S, dtype=torch.float64, device=q.device)
    lens = s["lens"].tolist()

    def head(table, n, h):
        pages = table[:(n + PAGE - 1) // PAGE].long()
        idx = s["codes"][pages, h].reshape(-1, D // c["bd"])[:n].long()
        k = torch.stack([s["cent"][h, j].double()[idx[:, j]] for j in range(idx.shape[1])], 1).reshape(n, D)
        return k, s["v_pages"][pages, h].double().transpose(1, 2).reshape(-1, D)[:n]

    for h in range(H):
        rows = q[:, h * G:(h + 1) * G]
        kp, vp = head(s["prefix_table"], c["T"], h)
        x = (rows.reshape(-1, D) @ kp.T).view(B, G * S, -1)
        top = x.amax(-1)
        e = torch.exp(x - top[..., None])
        del x
        sums = e.sum(-1)
        acc = (e.view(B * G * S, -1) @ vp).view(B, G * S, D)
        del e
        for b in range(B):
            ko, vo = head(s["table"][b], lens[b], h)
            y = (rows[b].reshape(-1, D) @ ko.T).view(G, S, -1)
            if s["mask"] is not None:
                y = y + s["mask"][b, :, :, :lens[b]].double()
            y = y.view(G * S, -1)
            m = torch.maximum(top[b], y.amax(-1))
            w, f = torch.exp(top[b] - m), torch.exp(y - m[:, None])
            total = sums[b] * w + f.sum(-1)
            out[b, h * G:(h + 1) * G] = ((acc[b] * w[:, None] + f @ vo) / total[:, None]).view(G, S, D)
            lse[b, h * G:(h + 1) * G] = (m + total.log()).view(G, S)
    return {"out": out, "lse": lse}
