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


def quiet(pr, seen_by_weight, nats=100.0):
    """Codeword 255 of block 0 gives a token `nats` less than others': the codes of tokens in `seen_by_weight` (page, place) pairs, and
    of no others.  Returns the problem with that codeword at 0 too, which the bounds' logits are of."""
    bd, D = pr["cent"].shape[-1], pr["q"].shape[-1]
    at = 0.5  # queries of block 0's dims
    pr["q"][..., pr["perm"][:bd]] = at
    pr["cent"][0, 255] = -nats / (pr["scale"] * bd * at)
    c0 = pr["codes"][..., 0]
    c0[c0 == 255] = 254
    for page, place in seen_by_weight:
        pr["codes"][page, :, place, 0] = 255
    calm = dict(pr, cent=pr["cent"].clone())
    calm["cent"][0, 255] = 0.0
    return calm


def last_page(pr, b, back=0):
    return int(pr["block_table"][b, (int(pr["seq_lens"][b]) - 1) // 16 - back])


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("r", [6, 10, 20, 28, 60, 118])
@pytest.mark.parametrize("how", ["weightless", "zero"])
def test_a_page_of_a_large_scale_that_counts_for_nothing(form, r, how):
    """A page 2^r above the others whose tokens have a weight of e^-100, or values of 0: the others are what comes out, to their own
    bits.  The rounding of weights to f16 counts from the row's largest weight: half of f16's smallest step, in units in which that weight is at
    least 2^14 times 2^-8, is 2^-31 of it, times 448 and the scale, a token."""
    log(f"range: a page 2^{r} up, {how}, {form}")
    pr = of_form(form, 63, spread=0)
    B = pr["q"].shape[0]
    far = sorted({last_page(pr, b, back) for b in range(B) if int(pr["seq_lens"][b]) > 200 for back in (0, 5)})
    pr["v_scale"][far] = 2.0 ** r
    if how == "zero":
        pr["v"].view(torch.uint8)[far] = 0
    calm = quiet(pr, [(pg, t) for pg in far for t in range(16)] if how == "weightless" else [])
    ref, mag = window64(pr), window64(calm)[2]
    floor = pr["block_table"].shape[1] * 16 * 2.0 ** -31 * 448
    for out_dtype in (BF, F32):
        out, lse = call(on_gpu(pr), out_dtype=out_dtype)
        within(pr, out, lse, ref, window_bounds(pr, ref[0], ref[1], mag, ref[3], out_dtype), floor)


@pytest.mark.parametrize("form", FORMS)
def test_scales_that_lie_anywhere(form):
    """Page scales of 2^-90 to 2^90, positive ones that are no powers of two: a row of them is held to the bits of its largest terms."""
    log(f"range: scales of 2^-90 to 2^90, {form}")
    pr = of_form(form, 64, spread=90)
    pr["v_scale"] = pr["v_scale"] * (1 + torch.rand(pr["v_scale"].shape, generator=torch.Generator().manual_seed(1)))
    ref = window64(pr)
    out, lse = call(on_gpu(pr), out_dtype=F32)
    within(pr, out, lse, ref, window_bounds(pr, *ref, F32))


@pytest.mark.parametrize("form", FORMS)
def test_scales_far_apart_beside_windows_and_nan(form):
    """The newest pages, which the older rows of a tile do not see, 2^40 above the others, and NaN values that some rows see."""
    log(f"range: scales, windows and NaN, {form}")
    pr = of_form(form, 65, spread=0, **({} if form == "wide" else {"lens": [385, 369, 193] if form == "together" else [19985, 7777]}))
    window = {"together": 100, "shares": 9000, "wide": 1750}[form]
    B, Lq = pr["q"].shape[0], pr["q"].shape[2]
    for b in range(B):
        pr["v_scale"][last_page(pr, b)] = 2.0 ** 40
    pr["v_scale"][last_page(pr, 0, 3)] = 2.0 ** 20
    bad = dict(pr, v=pr["v"].clone())
    n = int(pr["seq_lens"][0])
    toks = {0: n - 1, 1: n - 2, 5: n - Lq - window + 1, 7: n - 60}  # by dim; the third is seen by the first row alone
    for dim, tok in toks.items():
        bad["v"].view(torch.uint8)[int(pr["block_table"][0, tok // 16]), :, dim, tok % 16] = 0x7F
    ref = window64(pr, window, 3)
    ob, lb = window_bounds(pr, *ref, F32)
    out, lse = (t.cpu().double() for t in call(on_gpu(bad), window, 3, out_dtype=F32))
    for i in range(Lq):
        p = n - Lq + i
        for dim, tok in toks.items():
            if p - window < tok <= p:
                assert torch.isnan(out[0, :, i, dim]).all(), (i, dim)
                out[0, :, i, dim] = ref[0][0, :, i, dim]
    assert torch.isfinite(out).all()
    seen = ref[1] != -torch.inf
    assert (((out - ref[0]).abs() / ob)[seen] <= 1).all() and (((lse - ref[1]).abs() / lb)[seen] <= 1).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("vt", [BF, F16])
@pytest.mark.parametrize("nats", [30.0, 100.0])
def test_infinite_values_of_little_weight(form, vt, nats):
    """Infinite values of tokens whose weight is e^-30 or e^-100, the first tokens among them (what is summed before the weights
    that count): a row's dims are infinite where it sees one, NaN where it sees both or a NaN, and to the bit as without them elsewhere."""
    log(f"range: infinite values e^-{nats}, {form}, {vt}")
    inf, nan = torch.inf, torch.nan
    pr = of_form(form, 66, vt=vt, **({} if form == "wide" else {"lens": [400, 399, 250] if form == "together" else [20000, 19999]}))
    window = {"together": 300, "shares": 19000, "wide": 1800}[form]
    B, Hq, Lq, D = pr["q"].shape
    n0 = int(pr["seq_lens"][0])
    old = n0 - Lq - window + 1  # the oldest token that the first row sees, which the next does not
    # (token, dim, value) of sequence 0; the first quarter of what is seen and some of the newest tokens weigh little
    put = [(old, 0, inf), (old + 1, 1, -inf), (old + 40, 2, inf), (n0 - 1, 3, -inf), (n0 - 2, 4, inf), (old + 41, 5, inf),
           (n0 - 40, 5, -inf), (old + 70, 6, nan), (n0 - 33, 7, inf), (n0 - 33, 40, -inf), (old + 80, 41, inf), (old + 80, 42, nan),
           (n0 - 70, 42, inf)]
    few = sorted({t for t, _, _ in put} | set(range(old, old + window // 4)))
    quiet(pr, [(int(pr["block_table"][0, t // 16]), t % 16) for t in few], nats)
    bad = dict(pr, v=pr["v"].clone())
    zero = dict(pr, v=pr["v"].clone())
    for tok, dim, x in put:
        page = int(pr["block_table"][0, tok // 16])
        bad["v"][page, :, dim, tok % 16] = x
        zero["v"][page, :, dim, tok % 16] = 0
    out, lse = (t.cpu() for t in call(on_gpu(bad), window, 0, out_dtype=F32))
    want, wl = (t.cpu() for t in call(on_gpu(zero), window, 0, out_dtype=F32))
    assert torch.equal(lse, wl) and torch.isfinite(want).all()
    p = n0 - Lq + torch.arange(Lq)
    for dim in {d for _, d, _ in put}:
        total = torch.zeros(Lq)
        for tok, d, x in put:
            if d == dim:
                total = total + torch.where((p - window < tok) & (tok <= p), x, 0.0)
        hit = total != 0  # (NaN too)
        assert hit.any()
        want[0, :, hit, dim] = total[hit]
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out.nan_to_num(nan=7.0, posinf=inf, neginf=-inf), want.nan_to_num(nan=7.0, posinf=inf, neginf=-inf))


def test_infinite_values_in_pieces_that_weigh_nothing():
    """Parts of a long context whose weight in the join is 0 in 32 bits keep their infinities."""
    for vt in (BF, F16):
        log(f"range: infinite values, pieces without weight, {vt}")
        pr = problem(67, B=1, Hq=4, Hkv=1, D=64, T=60000, per_head=False, vt=vt)
        quiet(pr, [(int(pr["block_table"][0, t // 16]), t % 16) for t in range(30000)])
        pr["v"][int(pr["block_table"][0, 1000 // 16]), 0, 3, 5] = torch.inf
        pr["v"][int(pr["block_table"][0, 29000 // 16]), 0, 4, 5] = -torch.inf
        pr["v"][int(pr["block_table"][0, 50000 // 16]), 0, 5, 5] = torch.inf
        out = call(on_gpu(pr))[0].cpu()
        assert (out[..., 3] == torch.inf).all() and (out[..., 4] == -torch.inf).all() and (out[..., 5] == torch.inf).all()
        assert torch.isfinite(out[..., 6:]).all() and torch.isfinite(out[..., :3]).all()


@pytest.mark.parametrize("vt", [E4M3, BF])
def test_the_largest_values_over_many_tiles_a_wave(vt):
    """Alike values of 3e38 under alike weights, dozens of tiles a wave, so that its sum passes every threshold."""
    log(f"range: 3e38 over many tiles, {vt}")
    pr = problem(68, B=6, Hq=8, Hkv=8, D=64, T=30000, lens=[30000, 29999, 30000, 30000, 17000, 5], per_head=False, vt=vt, gain=1e-6, spread=0)
    if vt == E4M3:
        pr["v_scale"].fill_(2.0 ** 119)
        pr["v"] = torch.full(pr["v"].shape, 448.0).to(E4M3)
    else:
        pr["v"] = torch.full(pr["v"].shape, 3e38).to(BF)
    ref = window64(pr)
    out, lse = call(on_gpu(pr))
    within(pr, out, lse, ref, window_bounds(pr, *ref, BF))
