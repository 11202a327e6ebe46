"""Infinities and NaN that decode_prefix meets.  What one pass over all
tokens gives (0 times infinity is NaN) does not depend on where the tokens are cut."""

import math

import pytest
import torch

from _util import log
from test_gpu_decode_prefix import _call, _problem

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _spike(p, at, logit):
    """Prefix token `at` beats all others by `logit`: a codeword of its own in block 0, along a query dim that is 1
    after the scale."""
    G = p["q"].shape[1] // p["cent"].shape[0]
    p["codes"][..., 0] = p["codes"][..., 0].clamp(min=1)
    for h in range(p["cent"].shape[0]):
        p["q"][:, h * G:(h + 1) * G, :, int(p["perm"][h, 0])] = math.sqrt(p["q"].shape[-1])
        p["cent"][h, 0, :, 0] = 0.0
        p["cent"][h, 0, 0, 0] = logit
    p["codes"][p["ptable"][at // 16].long(), :, at % 16, 0] = 0
    return p


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("T, at, where", [
    (64, 3, 40),      # another tile: another wave of the same workgroup
    (64, 3, 20),      # the same tile
    (2000, 3, 1500),  # another slice of the prefix
    (2000, 1900, 4),
    (2000, 700, 731),
    (300, 7, -1),     # an own token
])
def test_values_under_probabilities_that_underflow(T, at, where, bad):
    log(f"decode_prefix: a value of {bad} at {where}, the logit at {at} 400 above, prefix of {T}")
    p = _spike(_problem(B=3, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=T, lens=[70, 5, 0]), at, 400.0)
    clean = _call(p)
    v = p["v"].clone()
    if where >= 0:
        v[p["ptable"][where // 16].long(), :, 5, where % 16] = bad
        hit = torch.ones(3, dtype=torch.bool)
    else:
        v[p["table"][0, 3].long(), :, 5, 9] = bad
        hit = torch.tensor([True, False, False])
    for kernel in (0, 1):
        out, lse = _call(dict(p, v=v), kernel=kernel)
        assert torch.isnan(out[hit][..., 5]).all(), f"kernel {kernel}"
        assert torch.isfinite(out[~hit]).all() and torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 6:]).all()
        assert torch.isfinite(lse).all()
        if kernel == 0:
            assert torch.equal(out[..., 6:], clean[0][..., 6:]) and torch.equal(lse, clean[1])


@pytest.mark.parametrize("where", [20, 40, 100])
def test_values_of_hidden_tokens(where):
    """A token at a mask of -inf has probability 0, and 0 times an infinite value is NaN: in the piece with the visible
    tokens and in one that is hidden whole, wherever the sequence is cut."""
    log(f"decode_prefix: an infinite value at hidden token {where}")
    p = _problem(B=2, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=20, lens=[200, 150])
    v = p["v"].clone()
    v[p["table"][0, where // 16].long(), :, 5, where % 16] = math.inf
    m = torch.zeros(2, 1, 1, p["table"].shape[1] * 16)
    m[..., :128] = -math.inf
    p["own_mask"] = m
    for kernel in (0, 1):
        out, lse = _call(dict(p, v=v), kernel=kernel)
        assert torch.isnan(out[0, ..., 5]).all(), f"kernel {kernel}"
        assert torch.isfinite(out[1]).all() and torch.isfinite(out[..., :5]).all() and torch.isfinite(lse).all()


@pytest.mark.parametrize("T, lens", [(300, [70, 5, 0]), (0, [70, 5, 40]), (2000, [0, 0, 0])])
@pytest.mark.parametrize("qdt, vdt", [(BF, BF), (F16, F16), (F32, BF)])
def test_queries_of_nan(T, lens, qdt, vdt):
    """A row whose query holds a NaN is NaN, and no other row."""
    log(f"decode_prefix: a NaN query, {qdt}, prefix {T}")
    p = _problem(B=3, Hq=8, Hkv=2, Lq=1, D=64, Dv=64, bd=4, nc=256, T=T, lens=lens, qdt=qdt, vdt=vdt)
    p["q"][1, 6, 0, 11] = math.nan
    for kernel in (0, 1):
        out, lse = _call(p, kernel=kernel)
        bad = torch.zeros(3, 8, 1, dtype=torch.bool, device=out.device)
        bad[1, 6] = True
        assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all(), f"kernel {kernel}"
        assert torch.isfinite(out[~bad]).all() and torch.isfinite(lse[~bad]).all(), f"kernel {kernel}"


@pytest.mark.parametrize("kw", [dict(D=64, Dv=64, bd=4, nc=4096), dict(D=256, Dv=256, bd=4, nc=256), dict(D=64, Dv=64, bd=4, nc=256, vdt=F32),
                                dict(D=64, Dv=128, bd=4, nc=256), dict(D=128, Dv=128, bd=4, nc=256, heavy=tuple(range(20)))])
def test_queries_of_nan_under_other_codecs(kw):
    log(f"decode_prefix: a NaN query, {kw}")
    p = _problem(B=3, Hq=8, Hkv=2, Lq=2, T=300, lens=[70, 5, 0], **kw)
    p["q"][1, 6, 1, 11] = math.nan
    out, lse = _call(p)
    bad = torch.zeros(3, 8, 2, dtype=torch.bool, device=out.device)
    bad[1, 6, 1] = True
    assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
    assert torch.isfinite(out[~bad]).all() and torch.isfinite(lse[~bad]).all()


@pytest.mark.parametrize("heavy, bd, D", [((1,), 4, 64), ((0, 5, 6), 4, 128), ((2,), 8, 64), ((3, 8), 8, 128), ((4, 9), 2, 64)])
@pytest.mark.parametrize("dt", [BF, F16])
def test_infinite_kept_dims(heavy, bd, D, dt):
    """A kept key dim of infinity against a query dim of the other sign is a logit of -inf: a token that counts for
    nothing, as one of -30,000 does."""
    log(f"decode_prefix: infinite kept dims, heavy {heavy} of dims {bd}, head_dim {D}, {dt}")
    p = _problem(B=3, Hq=8, Hkv=2, Lq=1, D=D, Dv=D, bd=bd, nc=256, T=150, lens=[70, 5, 0], heavy=heavy, qdt=dt, vdt=dt)
    for h in range(2):  # the first kept dim's queries are 1
        p["q"][:, h * 4:(h + 1) * 4, :, int(p["perm"][h, min(heavy) * bd])] = 1.0

    def at(x):
        pt = p["pt"].clone()
        for t in (0, 33, 149):
            pt[p["ptable"][t // 16].long(), :, t % 16, 0, 0] = x
        pt[p["table"][0, 1].long(), :, 7, 0, 0] = x
        return dict(p, pt=pt)

    for kernel in (0, 1):
        want, out = _call(at(-30000.0), kernel=kernel), _call(at(-math.inf), kernel=kernel)
        assert torch.isfinite(want[0]).all() and torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]), f"kernel {kernel}"
