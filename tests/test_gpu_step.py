"""A serving loop's layer step over raw projections (PagedSunShapeCache.attend): norm, rotation, append and
attention together, with sequences that continue a shared prefix, against the same steps from their formulas."""

import math

import numpy as np
import pytest
import torch

from _step import DEV, codec_arrays, prefix_attention64, turn64
from _util import log
from sunshape_amd import hip_ops
from sunshape_amd.codec import SunShapeBlockCodec
from sunshape_amd.paged import PagedSunShapeCache

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def _cache(D, Hkv, heavy=(), seed=0, num_pages=128):
    perm, cent, mask, sigma = codec_arrays(np.random.default_rng(seed), Hkv, D, 4, 256, True, heavy)
    codec = SunShapeBlockCodec.from_buffers(perm, cent, mode="profileperm_mixed_precision" if heavy else "profileperm_baseline",
                                            mixed_high_precision_blocks=None if mask is None else torch.tensor(mask), device=DEV)
    return PagedSunShapeCache(codec, num_pages=num_pages, num_kv_heads=Hkv, value_dim=D, device=DEV), sigma


@pytest.mark.parametrize("D, Hq, Hkv, heavy", [(128, 8, 2, ()), (64, 14, 2, ()), (64, 4, 2, (0, 5))])
def test_steps_over_a_shared_prompt(D, Hq, Hkv, heavy):
    log(f"steps over a shared prompt: head_dim {D}, {Hq}/{Hkv} heads, heavy {heavy}")
    g = torch.Generator().manual_seed(D + Hq)
    cache, sigma = _cache(D, Hkv, heavy)
    codec = cache.codec
    cos, sin = hip_ops.rope_table(1024, D, device=DEV)
    qw, kw = torch.ones(D, dtype=BF, device=DEV), torch.from_numpy(sigma).to(BF).to(DEV)
    scale = 1 / math.sqrt(D)

    def project(n, S):
        return [torch.randn(n, S, h, D, generator=g).to(BF).to(DEV).transpose(1, 2) for h in (Hq, Hkv, Hkv)]

    def check(ids, q, out, first):
        """The step's output from the pages: the queries from their formula, attention in 64 bits."""
        B, _, S, _ = q.shape
        pos = torch.tensor([[f + i for i in range(S)] for f in first])
        qr = turn64(q.cpu(), qw.cpu(), cos.cpu(), sin.cpu(), pos)[0].to(BF)
        pre = cache.prefix_of.get(ids[0])
        table, lens = (t.cpu() for t in cache.tables(ids))
        plen = cache.seq_lens[pre] if pre is not None else 0
        ptab = torch.tensor(cache.block_tables[pre] if pre is not None else [], dtype=torch.int32)
        width = table.shape[1] * cache.page_size
        last = lens[:, None] - S + torch.arange(S)[None]
        m = torch.zeros(B, 1, S, width).masked_fill_(torch.arange(width) > last[:, None, :, None], -math.inf)
        ref, _, mag, pv = prefix_attention64(qr, scale, codec.effective_permutation().cpu(), codec.codebook().cpu(),
                                             cache.code_pages.cpu(), cache.v_pages.cpu(), ptab, plen, table, lens, m,
                                             None if cache.pt_pages is None else cache.pt_pages.cpu(), heavy and cache.heavy or None)
        # as in the attention's own test; a query dim next to a rounding border may round the other way: 2^-8 of
        # its share of a logit, for a few of D dims
        bound = 2.0 ** -8 * ref.abs() + (2 * (2.0 ** -15 * mag[..., None] + 1e-5) + 2.0 ** -8 + 2.0 ** -8 * mag[..., None] / 8) * pv
        assert ((out.cpu().double() - ref).abs() <= bound).all()

    # the prompt, in two chunks
    for S in (70, 13):
        q, k, v = project(1, S)
        first = [cache.seq_lens.get(0, 0)]
        check([0], q, cache.attend([0], q, k, v, cos=cos, sin=sin, q_weight=qw, k_weight=kw, scale=scale), first)
    ids = [5, 9, 11]
    cache.fork(0, ids)
    for S in (1, 1, 3, 1, 20):
        q, k, v = project(3, S)
        first = [cache.seq_lens[0] + cache.seq_lens.get(s, 0) for s in ids]
        before = cache.code_pages[cache.block_tables[0]].clone()
        out = cache.attend(ids, q, k, v, cos=cos, sin=sin, q_weight=qw, k_weight=kw, scale=scale)
        check(ids, q, out, first)
        # the appended codes are those of the rotated keys; the prompt's pages stay
        assert torch.equal(before, cache.code_pages[cache.block_tables[0]])
        kr, _ = hip_ops.qk_norm_rope(k, None, cos, sin, torch.tensor([[f + i for i in range(S)] for f in first], device=DEV), q_weight=kw)
        want, _ = hip_ops.encode(kr, codec.effective_permutation(), codec.codebook(), heavy=cache.heavy)
        for i, s in enumerate(ids):
            at = [cache.seq_lens[s] - S + j for j in range(S)]
            pages = torch.tensor([cache.block_tables[s][t // 16] for t in at], device=DEV)
            offs = torch.tensor([t % 16 for t in at], device=DEV)
            assert torch.equal(cache.code_pages[pages, :, offs], want[i].transpose(0, 1))
            assert torch.equal(cache.v_pages[pages, :, :, offs], v[i].transpose(0, 1))


def test_forked_equals_unforked():
    """A prompt held once and a prompt held by every sequence: outputs agree to rounding."""
    log("forked and unforked sequences")
    D, Hq, Hkv = 128, 8, 2
    g = torch.Generator().manual_seed(3)
    cos, sin = hip_ops.rope_table(512, D, device=DEV)
    shared, sigma = _cache(D, Hkv)
    apart, _ = _cache(D, Hkv)
    kw = torch.from_numpy(sigma).to(BF).to(DEV)
    q, k, v = (torch.randn(1, h, 100, D, generator=g).to(BF).to(DEV) for h in (Hq, Hkv, Hkv))
    kws = dict(cos=cos, sin=sin, k_weight=kw, scale=1 / math.sqrt(D))
    shared.attend([0], q, k, v, **kws)
    ids = [1, 2, 3, 4]
    shared.fork(0, ids)
    for s in ids:
        apart.attend([s], q, k, v, **kws)
    for _ in range(4):
        q, k, v = (torch.randn(4, h, 1, D, generator=g).to(BF).to(DEV) for h in (Hq, Hkv, Hkv))
        a, b = shared.attend(ids, q, k, v, **kws), apart.attend(ids, q, k, v, **kws)
        # both round probabilities and outputs to bf16: two half steps each
        assert ((a.double() - b.double()).abs() <= 4 * 2.0 ** -8 * v.abs().max() + 4 * 2.0 ** -8).all()
        rel = (a.double() - b.double()).norm() / b.double().norm()
        assert rel < 2 * 2.0 ** -8


def test_append_without_rotation_keeps_its_results():
    log("append with and without the operator")
    a, _ = _cache(64, 2)
    b, _ = _cache(64, 2)
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(3, 2, 21, 64, generator=g).to(BF).to(DEV) for _ in range(2))
    a.append([0, 1, 2], k, v)
    b.append([0, 1, 2], k, v, k_weight=None, cos=None, sin=None)
    c, _ = _cache(64, 2)
    slots = c.slot_mapping([0, 1, 2], 21)
    hip_ops.append_kv(k, v, c.codec.effective_permutation(), c.codec.codebook(), codes_out=c.code_pages, v_out=c.v_pages,
                      slot_mapping=slots)
    for x in (b, c):
        assert torch.equal(a.code_pages, x.code_pages) and torch.equal(a.v_pages, x.v_pages)


def test_fork_rules():
    log("fork: what is refused")
    cache, _ = _cache(64, 2)
    k = torch.randn(1, 2, 5, 64, device=DEV, dtype=BF)
    cache.append([0], k, k)
    cache.append([7], k, k)
    with pytest.raises(RuntimeError, match="prefix"):
        cache.fork(3, [1])  # holds nothing
    cache.fork(0, [1, 2])
    for args in ((0, [1]), (0, [0]), (0, [7]), (1, [8]), (0, [9, 9])):
        with pytest.raises(RuntimeError):
            cache.fork(*args)
    with pytest.raises(RuntimeError, match="no more tokens"):
        cache.append([0], k, k)
    with pytest.raises(RuntimeError, match="free them first"):
        cache.free(0)
    q = torch.randn(2, 4, 1, 64, device=DEV, dtype=BF)
    with pytest.raises(RuntimeError, match="same prefix"):
        cache.decode([1, 7], q)
    assert torch.isfinite(cache.decode([1, 2], q).float()).all()  # no own tokens yet
    cos, sin = hip_ops.rope_table(16, 64, device=DEV)
    with pytest.raises(RuntimeError, match="once"):
        cache.attend([1, 1], q, k.expand(2, -1, -1, -1)[:, :, :1], k.expand(2, -1, -1, -1)[:, :, :1], cos=cos, sin=sin)
    cache.free(1)
    cache.free(2)
    cache.append([0], k, k)
    cache.free(0)
    assert len(cache._free) == cache.num_pages - 1


def test_attend_refusals_leave_the_cache_as_it_was():
    log("attend: refusals")
    D, Hq, Hkv = 64, 4, 2
    cache, _ = _cache(D, Hkv)
    cos, sin = (t.to(DEV) for t in hip_ops.rope_table(64, D))
    q, k = torch.randn(2, Hq, 1, D, device=DEV).bfloat16(), torch.randn(2, Hkv, 1, D, device=DEV).bfloat16()
    before = (list(cache._free), dict(cache.seq_lens))
    for ids, args in (([1], (q, k, k)), ([1, 1], (q, k, k)), ([1, 2], (q[:1], k, k)), ([1, 2], (q, k[:1], k[:1])),
                      ([1, 2], (q, k[:, :1], k[:, :1])), ([1, 2], (q, k, k[:1]))):
        with pytest.raises(RuntimeError):
            cache.attend(ids, *args, cos=cos, sin=sin)
    with pytest.raises(RuntimeError):
        cache.append([1], k, k, cos=cos, sin=sin)
    assert (list(cache._free), dict(cache.seq_lens)) == before
    assert torch.isfinite(cache.attend([1, 2], q, k, k, cos=cos, sin=sin).float()).all()
