"""Norm and rotation of queries and keys (hip_ops.qk_norm_rope) against the formulas in 64 bits."""

import pytest
import torch

from _step import DEV, turn64, turn_bound
from _util import log
from sunshape_amd import hip_ops

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _make(B, H, S, D, dt, g, layout):
    if layout == "token":  # [B, S, H, D] projections seen as [B, H, S, D]
        return torch.randn(B, S, H, D, generator=g).to(dt).transpose(1, 2)
    if layout == "padded":  # rows inside a wider, unaligned buffer
        return torch.randn(B, H, S, D + 5, generator=g).to(dt)[..., 3:3 + D]
    return torch.randn(B, H, S, D, generator=g).to(dt)


def _check(got, x, w, cos, sin, pos, inter, what, eps=1e-6):
    ref, mag = turn64(x, w, cos, sin, pos, eps, inter)
    err = (got.cpu().double() - ref).abs()
    bound = turn_bound(ref, mag, x.dtype)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert (err <= bound).all(), f"{what}: {(err / bound).max().item():.3f} times the bound"


CASES = [
    # B, Hq, Hk, S, D, rot, interleaved, norm (0 none, 1 both, 2 queries only), dtype, layout
    (1, 1, 1, 1, 64, 64, False, 0, BF, "head"),
    (2, 14, 2, 5, 64, 64, False, 1, BF, "token"),
    (3, 14, 2, 17, 64, 32, True, 1, F16, "token"),
    (64, 32, 8, 1, 128, 128, False, 1, BF, "token"),
    (2, 32, 8, 300, 128, 64, False, 2, BF, "token"),
    (1, 3, 0, 9, 128, 128, True, 1, F32, "head"),
    (2, 5, 3, 7, 80, 80, False, 1, BF, "head"),       # head dim that is no power of two
    (2, 5, 3, 7, 96, 24, True, 1, F16, "token"),
    (1, 4, 2, 11, 128, 6, False, 1, BF, "token"),     # a rotated width that no 16-byte piece holds
    (2, 4, 1, 6, 64, 64, False, 1, BF, "padded"),     # unaligned rows
    (1, 2, 2, 3, 256, 256, False, 1, F32, "token"),
    (1, 2, 1, 3, 512, 512, False, 1, F32, "head"),
    (1, 2, 1, 3, 1024, 1024, True, 1, BF, "head"),
    (1, 1, 1, 2, 2, 2, False, 1, BF, "head"),
    (1, 2, 1, 2, 7, 4, False, 1, F32, "head"),        # an odd head dim
    (5, 40, 8, 700, 64, 64, False, 1, BF, "token"),   # rows enough for four heads a lane
    (2, 9, 2, 9000, 64, 32, True, 1, F32, "token"),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_against_formulas(case):
    B, Hq, Hk, S, D, rot, inter, norm, dt, layout = case
    log(f"rope {case}")
    g = torch.Generator().manual_seed(B * 1000 + S + D)
    q, k = _make(B, Hq, S, D, dt, g, layout), _make(B, Hk, S, D, dt, g, layout) if Hk else None
    cos, sin = hip_ops.rope_table(S + 50, rot)
    pos = torch.randint(0, S + 50, (B, S), generator=g)
    qw = (1 + 0.3 * torch.randn(D, generator=g)).to(BF) if norm else None
    kw = (1 + 0.3 * torch.randn(D, generator=g)).to(BF) if norm == 1 else None
    q0, k0 = q.to(DEV), None if k is None else k.to(DEV)
    if layout == "padded":  # .to() packs a view
        q0 = torch.zeros(B, Hq, S, D + 5, dtype=dt, device=DEV)[..., 3:3 + D].copy_(q0)
        k0 = torch.zeros(B, Hk, S, D + 5, dtype=dt, device=DEV)[..., 3:3 + D].copy_(k0)
    args = [cos.to(DEV), sin.to(DEV), pos.to(DEV)]
    gq, gk = hip_ops.qk_norm_rope(q0, k0, *args, q_weight=None if qw is None else qw.to(DEV),
                                  k_weight=None if kw is None else kw.to(DEV), interleaved=inter)
    _check(gq, q, qw, cos, sin, pos, inter, "q")
    if k is None:
        assert gk is None
    else:
        _check(gk, k, kw, cos, sin, pos, inter, "k")
    assert torch.equal(q0.cpu(), q)  # inputs are not written


@pytest.mark.parametrize("dt", [BF, F16, F32])
@pytest.mark.parametrize("inter", [False, True])
def test_paths_agree_bit_for_bit(dt, inter):
    """Aligned rows (whole pieces) and the same rows unaligned (element by element): the result does not
    depend on which kernel serves a call."""
    log(f"rope paths {dt} {inter}")
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, 4, 33, 128, generator=g).to(dt).to(DEV)
    w = torch.randn(128, generator=g).to(dt).to(DEV)
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(64, 128))
    pos = torch.randint(0, 64, (3, 33), generator=g).to(DEV)
    a, _ = hip_ops.qk_norm_rope(x, None, cos, sin, pos, q_weight=w, interleaved=inter)
    wide = torch.zeros(3, 4, 33, 131, dtype=dt, device=DEV)
    wide[..., 1:129] = x
    b, _ = hip_ops.qk_norm_rope(wide[..., 1:129], None, cos, sin, pos, q_weight=w, interleaved=inter)
    assert torch.equal(a, b)


def test_norm_alone_and_rotation_alone():
    log("rope: norm alone, rotation alone")
    g = torch.Generator().manual_seed(5)
    x = torch.randn(2, 3, 4, 64, generator=g).to(BF)
    w = torch.randn(64, generator=g)
    got, _ = hip_ops.qk_norm_rope(x.to(DEV), None, None, None, None, q_weight=w.to(DEV), eps=1e-3)
    _check(got, x, w, None, None, None, False, "norm", eps=1e-3)
    same, _ = hip_ops.qk_norm_rope(x.to(DEV), None, None, None, None)
    assert torch.equal(same.cpu(), x)


def test_far_positions_zeros_and_bad_positions():
    log("rope: far positions, zero rows, positions outside the tables")
    g = torch.Generator().manual_seed(7)
    cos, sin = hip_ops.rope_table(200000, 64)
    x = torch.randn(1, 2, 4, 64, generator=g)
    x[0, 0, 0] = 0.0  # r = 1 / sqrt(eps)
    pos = torch.tensor([[0, 199999, 200000, -1]])
    w = torch.ones(64)
    got, _ = hip_ops.qk_norm_rope(x.to(DEV), None, cos.to(DEV), sin.to(DEV), pos.to(DEV), q_weight=w.to(DEV))
    ok = pos[0] >= 0
    ok &= pos[0] < 200000
    _check(got[:, :, ok.to(DEV)], x[:, :, ok], w, cos, sin, pos[:, ok], False, "inside")
    assert torch.isnan(got[:, :, ~ok.to(DEV)]).all()
    assert (got[0, 0, 0] == 0).all()


def test_infinities_and_nan_stay_in_their_row():
    log("rope: infinities and NaN")
    x = torch.ones(1, 3, 1, 64)
    x[0, 0, 0, 5] = float("inf")
    x[0, 1, 0, 6] = float("nan")
    cos, sin = hip_ops.rope_table(8, 64)
    pos = torch.tensor([[3]])
    for w in (None, torch.ones(64)):
        got, _ = hip_ops.qk_norm_rope(x.to(BF).to(DEV), None, cos.to(DEV), sin.to(DEV), pos.to(DEV),
                                      q_weight=None if w is None else w.to(DEV))
        assert not torch.isfinite(got[0, 0]).all() and not torch.isfinite(got[0, 1]).all()
        assert torch.isfinite(got[0, 2]).all()


def test_empty_calls():
    log("rope: empty")
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(4, 64))
    for B, S in ((0, 1), (1, 0)):
        x = torch.zeros(B, 2, S, 64, device=DEV, dtype=BF)
        got, k = hip_ops.qk_norm_rope(x, x, cos, sin, torch.zeros(B, S, dtype=torch.int64, device=DEV))
        assert got.shape == x.shape and k.shape == x.shape


def test_refusals():
    log("rope: refusals")
    x = torch.zeros(2, 2, 3, 64, device=DEV, dtype=BF)
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(4, 64))
    pos = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    bad = [
        (dict(q=x[0]), "must be"), (dict(q=x.to(torch.int32)), "dtype"), (dict(k=x.float()), "key must be"),
        (dict(k=x[:, :, :2]), "key must be"), (dict(cos=None), "together"), (dict(positions=None), "positions"),
        (dict(positions=pos[:1]), "positions"), (dict(positions=pos.int()), "positions"), (dict(cos=cos.double()), "float32"),
        (dict(cos=cos[:, :16]), "alike"), (dict(cos=torch.cat((cos, cos), 1), sin=torch.cat((sin, sin), 1)), "rotate"),
        (dict(q_weight=torch.ones(32, device=DEV)), "q_weight"), (dict(k_weight=torch.ones(64)), "k_weight"),
        (dict(q_weight=torch.ones(64, device=DEV), k_weight=torch.ones(64, device=DEV, dtype=BF)), "share a dtype"),
        (dict(q_weight=torch.ones(64, device=DEV), eps=-1.0), "eps"),
        (dict(positions=pos.cpu()), "device"), (dict(cos=cos.cpu(), sin=sin.cpu()), "device"),
    ]
    for kw, word in bad:
        a = dict(q=x, k=x, cos=cos, sin=sin, positions=pos)
        a.update(kw)
        with pytest.raises(RuntimeError, match=word):
            hip_ops.qk_norm_rope(**a)


def test_graph_replays_and_side_stream():
    log("rope: graph, side stream")
    g = torch.Generator().manual_seed(9)
    x = torch.randn(8, 4, 1, 128, generator=g).to(BF).to(DEV)
    w = torch.randn(128, generator=g).to(DEV)
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(64, 128))
    pos = torch.zeros(8, 1, dtype=torch.int64, device=DEV)

    def call():
        return hip_ops.qk_norm_rope(x, x, cos, sin, pos, q_weight=w, k_weight=w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(a[0], call()[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(3):
        pos.fill_(step * 7)
        x.add_(0.25)
        want = call()
        out[0].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize("dt, D, rot, inter, norm", [(BF, 128, 128, False, True), (BF, 64, 32, True, False), (F16, 128, 64, True, True),
                                                     (F32, 128, 128, False, True), (BF, 256, 256, False, True)])
def test_many_rows_are_the_rows_by_themselves(dt, D, rot, inter, norm):
    """Many rows (four heads a lane, head counts that four does not divide) and the same tokens a few at a time."""
    log(f"rope, many rows {dt} {D} {rot} {inter} {norm}")
    Hq, Hkv = 11, 3
    lanes = D // (8 if dt == F32 else 16)
    S = -(-256 * 4096 // ((Hq + Hkv) * lanes)) + 5  # past 4,096 lanes a CU
    g = torch.Generator(device=DEV).manual_seed(D + rot)
    q = torch.randn(1, S, Hq, D, generator=g, device=DEV).to(dt).transpose(1, 2)
    k = torch.randn(1, S, Hkv, D, generator=g, device=DEV).to(dt).transpose(1, 2)
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g, device=DEV)).to(dt) if norm else None for _ in range(2))
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(S, rot))
    pos = torch.randperm(S, generator=g, device=DEV)[None]
    a, b = hip_ops.qk_norm_rope(q, k, cos, sin, pos, q_weight=qw, k_weight=kw, interleaved=inter)
    for s0 in list(range(0, S, S // 5)) + [S - 3]:
        s1 = min(s0 + 97, S)
        x, y = hip_ops.qk_norm_rope(q[:, :, s0:s1], k[:, :, s0:s1], cos, sin, pos[:, s0:s1], q_weight=qw, k_weight=kw, interleaved=inter)
        assert torch.equal(a[:, :, s0:s1], x) and torch.equal(b[:, :, s0:s1], y), s0
