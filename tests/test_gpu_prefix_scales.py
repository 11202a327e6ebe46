"""decode_prefix with f16 queries over codebooks of any magnitude: a KV head's codewords are held as two f16 parts at
a scale of the head's own, so small and large ones keep the same relative precision."""

import math

import pytest
import torch

from _step import prefix_attention64
from _util import log
from test_gpu_decode_prefix import _call, _check, _problem

pytestmark = pytest.mark.gpu
F16 = torch.float16


def _scaled(size, qsize, bd=4, D=64, heavy=(), **kw):
    """Codewords (and kept values) of about `size`, queries of about `qsize`: logits of a few units."""
    p = _problem(B=5, Hq=8, Hkv=2, Lq=1, D=D, Dv=D, bd=bd, nc=256, T=300, lens=[40, 1, 0, 5, 33], qdt=F16, vdt=F16, heavy=heavy, **kw)
    g = torch.Generator().manual_seed(3)
    live = p["cent"] != 0  # kept blocks' codewords are zeros
    p["cent"] = torch.randn(p["cent"].shape, generator=g).mul(size) * live
    p["q"] = torch.randn(p["q"].shape, generator=g).clamp(-2.5, 2.5).mul(qsize).to(F16)
    if heavy:
        p["pt"] = torch.randn(p["pt"].shape, generator=g).mul(size).to(F16)
    return p


@pytest.mark.parametrize("size, qsize", [(1e-3, 2e3), (1e-5, 2.5e4), (1e-7, 2.5e4), (1.0, 2.0), (3e5, 1e-4), (1e9, 6e-5)])
@pytest.mark.parametrize("bd, D", [(2, 64), (4, 128), (8, 64)])
def test_codewords_of_every_size(size, qsize, bd, D):
    log(f"decode_prefix: f16, codewords of {size}, dims of {bd}, head_dim {D}")
    p = _scaled(size, qsize, bd, D)
    if size * qsize > 100:  # one token takes all, and the bound of the logits still holds
        p["scale"] = 2.0 ** -7
    for kernel in (0, 1):
        out, lse = _call(p, kernel=kernel)
        _check(p, out, lse, f"codewords of {size}, kernel {kernel}")


@pytest.mark.parametrize("size, qsize", [(1e-3, 2e3), (1e-5, 2.5e4), (1.0, 2.0)])
@pytest.mark.parametrize("heavy, bd, D", [((1, 5), 4, 64), (tuple(range(0, 30, 3)), 4, 128), ((2, 3), 8, 128), ((0, 31), 2, 64)])
def test_kept_dims_of_every_size(size, qsize, heavy, bd, D):
    log(f"decode_prefix: f16, kept values of {size}, {len(heavy)} blocks of dims {bd}, head_dim {D}")
    p = _scaled(size, qsize, bd, D, heavy)
    for kernel in (0, 1):
        out, lse = _call(p, kernel=kernel)
        _check(p, out, lse, f"kept values of {size}, kernel {kernel}")


def test_kept_dims_far_larger_than_the_codewords():
    """Codewords of 1e-4 beside kept values of 1e4 (what blocks are kept for), and the other way round."""
    log("decode_prefix: f16, kept dims and codewords of different sizes")
    for size, kept in ((1e-4, 1e4), (1e3, 1e-4)):
        p = _scaled(size, 1.0, heavy=(1, 5))
        p["pt"] = p["pt"].float().div(size).clamp(-4, 4).mul(kept).to(F16)
        q = p["q"].float()
        for h in range(2):  # each dim's share of a logit is about one
            dims = torch.ones(64, dtype=torch.bool)
            dims[p["perm"][h].view(16, 4)[[1, 5]].flatten()] = False
            q[:, 4 * h:4 * h + 4, :, dims] *= 1 / size
            q[:, 4 * h:4 * h + 4, :, ~dims] *= 1 / kept
        p["q"] = q.to(F16)
        for kernel in (0, 1):
            out, lse = _call(p, kernel=kernel)
            _check(p, out, lse, f"codewords {size}, kept {kept}, kernel {kernel}")


def test_heads_of_different_sizes():
    """Each KV head has a scale of its own; a codeword without a finite value does not set it."""
    log("decode_prefix: f16, heads of different sizes, unused codewords without a value")
    p = _scaled(1.0, 1.0)
    p["cent"][0] *= 1e-5
    p["cent"][1] *= 1e3
    q = p["q"].float()
    q[:, :4] *= 1.2e4
    q[:, 4:] *= 2e-3
    p["q"] = q.to(F16)
    p["codes"][..., 2] = p["codes"][..., 2].clamp(max=250)
    p["cent"][0, 2, 251] = math.inf
    p["cent"][0, 2, 252] = math.nan
    p["cent"][1, 2, 253] = -math.inf
    ref = prefix_attention64(p["q"], p["scale"], p["perm"], p["cent"], p["codes"], p["v"], p["ptable"], int(p["plen"]),
                             p["table"], p["lens"])
    assert torch.isfinite(ref[1]).all()
    for kernel in (0, 1):
        out, lse = _call(p, kernel=kernel)
        _check(p, out, lse, f"kernel {kernel}")
