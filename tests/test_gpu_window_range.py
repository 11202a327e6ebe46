"""decode_window at the ends of its values' ranges, against the definition in 64 bits, in each form that a call may take: a
workgroup's waves together (short contexts), shares of all tiles (long ones), and items of 256 rows (many new tokens)."""

import pytest
import torch

from _cache8 import E4M3, problem, window64, window_bounds
from _util import log
from test_gpu_window import call, on_gpu
from test_gpu_window_wide import wide

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def of_form(form, seed, **kw):
    if form == "together":
        return problem(seed, B=3, Hq=8, Hkv=2, D=128, Lq=2, T=400, per_head=False, **kw)
    if form == "shares":
        return problem(seed, B=2, Hq=8, Hkv=2, D=128, Lq=2, T=20000, per_head=False, **kw)
    return wide(problem(seed, B=1, Hq=256, Hkv=64, D=64, Lq=64, T=1900, per_head=False, **kw))


FORMS = ["together", "shares", "wide"]


def within(pr, out, lse, ref, bounds, floor=0.0):
    out, lse = out.cpu().double(), lse.cpu().double()
    empty = ref[1] == -torch.inf
    assert (out[empty] == 0).all() and (lse[empty] == -torch.inf).all()
    ob, lb = bounds
    assert torch.isfinite(out).all()
    eo, el = ((out - ref[0]).abs() / (ob + floor))[~empty], ((lse - ref[1]).abs() / lb)[~empty]
    log(f"  worst of the bound: out {float(eo.max()):.3f} lse {float(el.max()):.3f}")
    assert (eo <= 1).all() and (el <= 1).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("vt", [E4M3, BF])
@pytest.mark.parametrize("gain", [1e-6, 2.0])
def test_the_largest_values(form, vt, gain):
    """Values up to 3e38 average to what they are, alike ones too, with weights that are all alike (gain 1e-6) and that are not."""
    for alike in (False, True):
        log(f"range: values of 3e38, {form}, {vt}, gain {gain}, alike {alike}")
        pr = of_form(form, 61, vt=vt, gain=gain, spread=0)
        if vt == E4M3:
            pr["v_scale"].fill_(2.0 ** 119)
            if alike:
                pr["v"] = torch.full(pr["v"].shape, 448.0).to(E4M3)
        else:
            pr["v"] = torch.full(pr["v"].shape, 3e38).to(BF) if alike else (pr["v"].float().clamp(-3, 3) * 1e38).to(BF)
        ref = window64(pr)
        for out_dtype in (BF, F32):
            out, lse = call(on_gpu(pr), out_dtype=out_dtype)
            within(pr, out, lse, ref, window_bounds(pr, *ref, out_dtype))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("vt", [E4M3, BF])
def test_small_values(form, vt):
    """Values of about 2^-106 are held to as many bits as others: the sums' steps are 2^-149 at most, a token each."""
    log(f"range: values of 2^-106, {form}, {vt}")
    pr = of_form(form, 62, vt=vt, spread=0)
    if vt == E4M3:
        pr["v_scale"].fill_(2.0 ** -100)
        pr["v"] = (pr["v"].float() * 2.0 ** -9).to(E4M3)
    else:
        pr["v"] = (pr["v"].float() * 2.0 ** -106).to(BF)
    ref = window64(pr)
    # the bounds' own floor is far above these values: everything times 2^100, which is exact
    up = 2.0 ** 100
    big = [ref[0] * up, ref[1], ref[2], ref[3] * up]
    out, lse = call(on_gpu(pr), out_dtype=F32)
    # a product, or a sum of them, is rounded to a step of 2^-149 at the most, in units in which all weights sum to 2^-12 or more
    # (bf16 values: the largest weight is kept at 2^-8 until the sum is 2^-1, then taken 2^4 down)
    floor = pr["block_table"].shape[1] * 16 * 2.0 ** -149 * 2.0 ** 12 * up
    within(pr, out.double() * up, lse, big, window_bounds(pr, *big, F32), floor)
