"""A serving loop over a cache with 8-bit values or a window (PagedSunShapeCache): steps, chunks, forks, releases, compaction
and new pools together, against the same steps from their formulas."""

import math

import numpy as np
import pytest
import torch

from _cache8 import E4M3, same_values, values_plain, window64, window_bounds
from _step import DEV, codec_arrays, turn64
from _util import log
from sunshape_amd import hip_ops
from sunshape_amd.codec import SunShapeBlockCodec
from sunshape_amd.paged import PagedSunShapeCache

pytestmark = pytest.mark.gpu
BF, F16 = torch.bfloat16, torch.float16


class Loop:
    """A cache, what its sequences' values ought to be (pages of their own on the CPU), and each sequence's codes as they
    were first written."""

    def __init__(self, D, Hq, Hkv, page, vt, window, sinks, seed):
        perm, cent, _, sigma = codec_arrays(np.random.default_rng(seed), Hkv, D, 4, 256, True)
        codec = SunShapeBlockCodec.from_buffers(perm, cent, mode="profileperm_baseline", device=DEV)
        self.cache = PagedSunShapeCache(codec, num_pages=96, num_kv_heads=Hkv, value_dim=D, page_size=page, value_dtype=vt,
                                        device=DEV, window=window, sinks=sinks)
        self.g = torch.Generator().manual_seed(seed)
        self.heads, self.D, self.scale = (Hq, Hkv, Hkv), D, 1 / math.sqrt(D)
        self.cos, self.sin = hip_ops.rope_table(1024, D, device=DEV)
        self.qw, self.kw = torch.ones(D, dtype=BF, device=DEV), torch.from_numpy(sigma).to(BF).to(DEV)
        self.values, self.codes, self.before = {}, {}, {}
        release = self.cache.release

        def noted(ids):  # the tables a step attended over, before it gives pages back
            self.before = {s: list(self.cache.block_tables[s]) for s in ids}
            return release(ids)

        self.cache.release = noted

    def pages(self, s, table=None):
        t = table or self.cache.block_tables[s]
        return [i for i, pg in enumerate(t) if pg >= 0], [pg for pg in t if pg >= 0]

    def stored(self, s, table=None):
        """Codes, values and scales of a sequence's pages on the CPU, zero where a page is released."""
        c = self.cache
        at, pg = self.pages(s, table)
        n = len(c.block_tables[s])
        codes = torch.zeros(n, *c.code_pages.shape[1:], dtype=torch.uint8)
        codes[at] = c.code_pages[pg].cpu()
        v = torch.zeros(n, *c.v_pages.shape[1:], dtype=c.v_pages.dtype)
        raw = torch.uint8 if v.dtype == E4M3 else torch.int16
        v.view(raw)[at] = c.v_pages.view(raw)[pg].cpu()
        scale = None
        if c.v_scale is not None:
            scale = torch.ones(n, self.heads[1])
            scale[at] = c.v_scale[pg].cpu()
        return codes, v, scale

    def expect_values(self, s, v, first):
        """The sequence's values after `first` tokens and the new ones [H, S, D]."""
        c, S = self.cache, v.shape[1]
        n = c._pages(first + S)
        old, sc = self.values.get(s, (torch.zeros(0, self.heads[1], self.D, c.page_size, dtype=c.v_pages.dtype),
                                      torch.zeros(0, self.heads[1])))
        raw = torch.uint8 if old.dtype == E4M3 else torch.int16
        new = torch.zeros(n, *old.shape[1:], dtype=old.dtype)
        new.view(raw)[:len(old)] = old.view(raw)
        sc = torch.cat([sc, torch.zeros(n - len(sc), self.heads[1])])
        slots = torch.arange(first, first + S)
        if old.dtype == E4M3:
            new, sc = values_plain(v[None], new, sc, slots[None])
        else:
            new[slots // c.page_size, :, :, slots % c.page_size] = v.to(old.dtype).transpose(0, 1)
        self.values[s] = new, sc

    def held_as_written(self):
        """Every live token's value is the formula's, its codes those it was given."""
        c = self.cache
        for s, n in c.seq_lens.items():
            codes, v, scale = self.stored(s)
            want, sc = self.values[s]
            at, _ = self.pages(s)
            for i in at:
                end = min(n - i * c.page_size, c.page_size)
                assert same_values(v[i, :, :, :end], want[i, :, :, :end]) and (scale is None or torch.equal(scale[i], sc[i]))
                have = self.codes.setdefault(s, {})
                for o in range(end):
                    row = codes[i, :, o]
                    assert torch.equal(row, have.setdefault(i * c.page_size + o, row))

    def expect(self, q, ids, out):
        """out [B, Hq, S, D] of the sequences' newest tokens: within the roundings of the 64-bit form over the stored pages."""
        c, S = self.cache, q.shape[2]
        pos = torch.tensor([[c.seq_lens[s] - S + i for i in range(S)] for s in ids])
        qr = turn64(q.cpu(), self.qw.cpu(), self.cos.cpu(), self.sin.cpu(), pos)[0].to(BF)
        for b, s in enumerate(ids):
            codes, v, scale = self.stored(s, self.before[s])  # what the step freed is still in its place
            pr = dict(q=qr[b:b + 1], codes=codes, v=v, perm=c.codec.effective_permutation().cpu(), cent=c.codec.codebook().cpu(),
                      block_table=torch.arange(len(codes))[None], seq_lens=torch.tensor([c.seq_lens[s]]), v_scale=scale,
                      scale=self.scale)
            ref, lse, mag, pv = window64(pr, c.window, c.sinks)
            # a query dim next to a rounding border may round the other way: a step of 2^-7, two after the
            # scale (2^-6), in dims with at most an eighth of a row's sum |q||k| (one in 2^13 dims is so near): a logit is off
            # by 2^-9 mag, a weight by twice that
            bound = window_bounds(pr, ref, lse, mag, pv, BF)[0] + 2.0 ** -8 * mag[..., None] * pv
            got = out[b:b + 1].cpu().double()
            assert ((got - ref).abs() <= bound).all(), (s, ((got - ref).abs() / bound).max())

    def step(self, ids, S):
        q, k, v = [torch.randn(len(ids), S, h, self.D, generator=self.g).to(BF).to(DEV).transpose(1, 2) for h in self.heads]
        first = [self.cache.seq_lens.get(s, 0) for s in ids]
        out = self.cache.attend(ids, q, k, v, cos=self.cos, sin=self.sin, q_weight=self.qw, k_weight=self.kw, scale=self.scale)
        for b, s in enumerate(ids):
            self.expect_values(s, v[b].cpu(), first[b])
        self.expect(q, ids, out)
        self.held_as_written()

    def fork(self, s, ids):
        self.cache.fork(s, ids)
        for i in ids:
            self.values[i], self.codes[i] = self.values[s], dict(self.codes[s])
        self.held_as_written()

    def free(self, s):
        self.cache.free(s)
        del self.values[s], self.codes[s]


@pytest.mark.parametrize("D, Hq, Hkv, page, vt, window, sinks", [
    (128, 8, 2, 16, E4M3, None, 0), (64, 14, 2, 16, E4M3, 40, 18), (128, 8, 2, 32, BF, 50, 4), (64, 4, 2, 64, F16, 70, 0)])
def test_a_serving_loop(D, Hq, Hkv, page, vt, window, sinks):
    log(f"serving loop: head_dim {D}, {Hq}/{Hkv} heads, pages of {page}, {vt} values, window {window}, sinks {sinks}")
    loop = Loop(D, Hq, Hkv, page, vt, window, sinks, seed=D + Hq + page)
    cache = loop.cache
    loop.step([0], 70)  # a prompt, and a chunk more
    loop.step([0], 37)
    loop.fork(0, [1, 2, 3])
    for _ in range(3):
        loop.step([0, 1, 2, 3], 1)
    loop.step([3, 1], 5)  # several new tokens, some of the sequences
    loop.free(0)
    loop.step([9], 33)
    cache.compact()
    loop.held_as_written()
    loop.step([1, 9, 2], 20)
    cache.resize(120)
    loop.held_as_written()
    loop.fork(9, [10])
    for _ in range(2):
        loop.step([10, 3, 2, 1, 9], 1)
    held = len({pg for t in cache.block_tables.values() for pg in t if pg >= 0})
    cache.resize(held + 6)
    loop.held_as_written()
    loop.step([10, 9, 1], 2)
    if window is not None:  # dead pages are back: no sequence holds more than its window, sinks and two partial pages
        per = cache._pages(window) + cache._pages(sinks) + 1
        assert all(sum(pg >= 0 for pg in t) <= per for s, t in cache.block_tables.items() if s in (10, 9, 1))
    for s in list(cache.seq_lens):
        cache.free(s)
    assert sorted(cache._free) == list(range(held + 6))


def test_appends_and_decodes_apart(D=128, Hq=8, Hkv=2):
    """append without rotation, decode with the softmax's logarithms, several rows of queries at once."""
    loop = Loop(D, Hq, Hkv, 16, E4M3, 64, 8, seed=5)
    cache = loop.cache
    for first, S in ((0, 50), (50, 9), (59, 1)):
        k, v = [torch.randn(2, S, h, D, generator=loop.g).to(BF).to(DEV).transpose(1, 2) for h in (Hkv, Hkv)]
        cache.append([4, 5], k, v)
        for b, s in enumerate((4, 5)):
            loop.expect_values(s, v[b].cpu(), first)
        loop.held_as_written()
    q = torch.randn(2, 3, Hq, D, generator=loop.g).to(BF).to(DEV).transpose(1, 2)
    out, lse = cache.decode([5, 4], q, scale=loop.scale, return_lse=True)
    for b, s in enumerate((5, 4)):
        codes, v, scale = loop.stored(s)
        pr = dict(q=q[b:b + 1].cpu(), codes=codes, v=v, perm=cache.codec.effective_permutation().cpu(), cent=cache.codec.codebook().cpu(),
                  block_table=torch.arange(len(codes))[None], seq_lens=torch.tensor([60]), v_scale=scale, scale=loop.scale)
        ref, ref_lse, mag, pv = window64(pr, 64, 8)
        ob, lb = window_bounds(pr, ref, ref_lse, mag, pv, out.dtype)
        assert ((out[b:b + 1].cpu().double() - ref).abs() <= ob).all()
        assert ((lse[b:b + 1].cpu().double() - ref_lse).abs() <= lb).all()


def test_a_captured_step():
    """Copies, an append and the attention in one graph, replayed over changing inputs and lengths in the same tensors."""
    log("a captured step")
    D, Hq, Hkv, B = 128, 8, 2, 3
    loop = Loop(D, Hq, Hkv, 16, E4M3, 40, 4, seed=8)
    cache = loop.cache
    codec, perm = cache.codec, cache.codec.effective_permutation()
    loop.step([0], 30)
    loop.fork(0, [1, 2])
    for s in range(B):  # pages for what follows
        while len(cache.block_tables[s]) < 4:
            cache.block_tables[s].append(cache._free.pop())
    table, lens = cache.tables(list(range(B)))
    spare = cache._free[:3]
    src, dst = [torch.tensor(x, device=DEV) for x in ([cache.block_tables[s][1] for s in range(B)], spare)]
    q, k, v = [torch.zeros(B, 1, h, D, dtype=BF, device=DEV).transpose(1, 2) for h in (Hq, Hkv, Hkv)]
    pos, slots = torch.zeros(B, 1, dtype=torch.int64, device=DEV), torch.zeros(B, 1, dtype=torch.int64, device=DEV)
    grid = codec.encode_search_grid(codec.centroids)

    def work():
        hip_ops.copy_pages(cache._pools(), src, dst)
        hip_ops.append_kv(k, v, perm, codec.centroids, codes_out=cache.code_pages, v_out=cache.v_pages, slot_mapping=slots,
                          positions=pos, cos=loop.cos, sin=loop.sin, k_weight=loop.kw, metric=codec.encode_metric(), grid=grid,
                          direct=hip_ops.cdist_direct(1, codec.n_centroids), v_scale=cache.v_scale)
        return hip_ops.decode_window(q, cache.code_pages, cache.v_pages, perm, codec.centroids, block_table=table, seq_lens=lens,
                                     scale=loop.scale, window=40, sinks=4, v_scale=cache.v_scale)

    def state():
        return [p.clone() for p in cache._pools()]

    def put(saved):
        for p, x in zip(cache._pools(), saved):
            p.view(torch.uint8).copy_(x.view(torch.uint8))

    slots.fill_(-1)  # a warm-up that appends nothing
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for n in range(30, 36):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=loop.g))
        pos.fill_(n)
        lens.fill_(n + 1)
        slots.copy_(torch.tensor([[cache.block_tables[s][n // 16] * 16 + n % 16] for s in range(B)]))
        before = state()
        graph.replay()
        got, after = out.clone(), state()
        put(before)
        eager = work()
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        for a, b in zip(after, cache._pools()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        put(after)
