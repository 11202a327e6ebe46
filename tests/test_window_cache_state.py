"""PagedSunShapeCache with 8-bit values or a window: its pages, forks, releases and moves on the CPU (stand-ins for the
operators that need the GPU; the copies are done by torch), and what it refuses."""

import math

import numpy as np
import pytest
import torch

from _step import codec_arrays
from sunshape_amd import hip_ops, paged
from sunshape_amd.codec import SunShapeBlockCodec
from sunshape_amd.paged import PagedSunShapeCache

BF, E4M3 = torch.bfloat16, torch.float8_e4m3fn


def _codec(D=64, bd=4, nc=256, heavy=()):
    perm, cent, mask, _ = codec_arrays(np.random.default_rng(0), 2, D, bd, nc, True, heavy)
    return SunShapeBlockCodec.from_buffers(perm, cent, mode="profileperm_mixed_precision" if heavy else "profileperm_baseline",
                                           mixed_high_precision_blocks=None if mask is None else torch.tensor(mask),
                                           device=torch.device("cpu"))


def _cache(codec=None, num_pages=12, page_size=16, value_dim=64, value_dtype=E4M3, **kw):
    return PagedSunShapeCache(codec or _codec(), num_pages=num_pages, num_kv_heads=2, value_dim=value_dim, page_size=page_size,
                              value_dtype=value_dtype, device=torch.device("cpu"), **kw)


def _state(cache):
    return (list(cache._free), {s: list(t) for s, t in cache.block_tables.items()}, dict(cache.seq_lens), dict(cache._refs),
            dict(cache._released), dict(cache.prefix_of))


@pytest.fixture
def ops(monkeypatch):
    """Stand-ins: `fail` names the ones that raise, `calls` are those made."""
    class Ops:
        fail, calls = set(), []

    Ops.fail, Ops.calls = set(), []

    def op(name, result):
        def call(*args, **kw):
            if name in Ops.fail:
                raise RuntimeError(f"{name} refuses")
            Ops.calls.append((name, args, kw))
            return result(*args, **kw)
        monkeypatch.setattr(paged.hip_ops, name, call)

    def copy(pools, src, dst, *, into=None):
        assert len(set(dst.tolist())) == len(dst) and (into is not None or not set(src.tolist()) & set(dst.tolist()))
        for p, o in zip(pools, into or pools):
            o[dst] = p[src]

    op("append_kv", lambda *a, **kw: None)
    op("append_values", lambda *a, **kw: None)
    op("encode", lambda *a, **kw: None)
    op("qk_norm_rope", lambda q, *a, **kw: (q, None))
    op("decode_window", lambda q, *a, **kw: q)
    op("copy_pages", copy)
    return Ops


def _rows(B, S, H=2, D=64):
    return torch.zeros(B, H, S, D, dtype=BF)


def _attend(cache, ids, S):
    cos, sin = hip_ops.rope_table(4096, 64)
    return cache.attend(ids, _rows(len(ids), S, 4), _rows(len(ids), S), _rows(len(ids), S), cos=cos, sin=sin)


def _mark(cache):
    """Every pool's pages numbered."""
    n = cache.num_pages
    cache.code_pages[:] = torch.arange(n, dtype=torch.uint8)[:, None, None, None]
    cache.v_pages.view(torch.uint8)[:] = torch.arange(n, dtype=torch.uint8)[:, None, None, None]
    if cache.v_scale is not None:
        cache.v_scale[:] = torch.arange(n).float()[:, None]


def _marks(cache, s):
    """The numbers on a sequence's pages, the same in every pool."""
    pg = [p for p in cache.block_tables[s] if p >= 0]
    got = [cache.code_pages[p, 0, 0, 0].item() for p in pg]
    assert got == [cache.v_pages.view(torch.uint8)[p, 1, 3, 2].item() for p in pg]
    assert cache.v_scale is None or got == [int(cache.v_scale[p, 1]) for p in pg]
    return got


def test_which_caches_are_refused():
    for kw, match in ((dict(codec=_codec(heavy=(1,))), "passthrough"), (dict(value_dim=32), "value_dim"),
                      (dict(codec=_codec(D=96), value_dim=96), "head_dim"), (dict(codec=_codec(bd=16)), "block_dim"),
                      (dict(codec=_codec(nc=300)), "byte codes"), (dict(page_size=48), "pages of"), (dict(window=0), "window"),
                      (dict(window=8, sinks=-1), "sinks"), (dict(sinks=4), "sinks"),
                      (dict(value_dtype=BF, sinks=4), "sinks"), (dict(value_dtype=torch.float32, window=8), "8 or 16 bits")):
        with pytest.raises(RuntimeError, match=match):
            _cache(**kw)
    assert not _cache(value_dtype=BF).causal  # and without either, all is as before
    assert _cache(value_dtype=BF, window=8, sinks=4).causal and _cache().causal


def test_scales_reach_the_operators(ops):
    cache = _cache(window=32, sinks=4)
    _attend(cache, [1], 5)
    cache.append([1], _rows(1, 3), _rows(1, 3))
    cache.decode([1], _rows(1, 2, 4), scale=0.5)
    by = {}
    for name, args, kw in ops.calls:
        by.setdefault(name, []).append((args, kw))
    assert by["append_kv"][0][1]["v_scale"] is cache.v_scale
    assert by["append_values"][0][0][1] is cache.v_pages and by["append_values"][0][0][2] is cache.v_scale
    for _, kw in by["decode_window"]:
        assert kw["v_scale"] is cache.v_scale and kw["window"] == 32 and kw["sinks"] == 4
    plain = _cache(value_dtype=BF, window=32)
    ops.calls.clear()
    _attend(plain, [1], 5)
    assert all("v_scale" not in kw for _, _, kw in ops.calls)


@pytest.mark.parametrize("length", [1, 15, 16, 17, 32, 40])
def test_forks_share_whole_pages_and_copy_the_last(ops, length):
    cache = _cache()
    _attend(cache, [0], length)
    whole, part = divmod(length, 16)
    _mark(cache)
    cache.fork(0, [1, 2])
    assert len(cache._free) == 12 - (whole + 3 * (part > 0))
    for s in (1, 2):
        assert cache.block_tables[s][:whole] == cache.block_tables[0][:whole] and cache.seq_lens[s] == length
        assert _marks(cache, s) == _marks(cache, 0)
    tails = [cache.block_tables[s][whole:] for s in (0, 1, 2)]
    assert len({t[0] for t in tails}) == 3 if part else tails == [[], [], []]
    _attend(cache, [0, 1, 2], 1)  # all of them go on, on pages of their own
    assert len({cache.block_tables[s][-1] for s in (0, 1, 2)}) == 3
    cache.free(0)  # the first as well as the last
    assert not set(cache._free) & set(cache.block_tables[1] + cache.block_tables[2])
    cache.fork(1, [3])
    for s in (2, 1, 3):
        cache.free(s)
    assert sorted(cache._free) == list(range(12)) and cache._refs == {} and cache.seq_lens == {} and cache._released == {}


def test_forks_that_are_refused(ops):
    cache = _cache(num_pages=4)
    _attend(cache, [0], 20)
    before = _state(cache)
    for ids, match in (([1, 2, 3], "out of pages"), ([1, 1], "distinct"), ([0], "distinct")):
        with pytest.raises(RuntimeError, match=match):
            cache.fork(0, ids)
        assert _state(cache) == before
    with pytest.raises(RuntimeError, match="no tokens"):
        cache.fork(9, [1])
    ops.fail.add("copy_pages")
    with pytest.raises(RuntimeError, match="copy_pages refuses"):
        cache.fork(0, [1])
    assert _state(cache) == before
    cache.fork(0, [])
    assert _state(cache) == before


@pytest.mark.parametrize("op", ["append_kv", "qk_norm_rope", "decode_window"])
def test_a_step_that_is_refused(ops, op):
    cache = _cache(window=8)
    _attend(cache, [0], 40)
    cache.fork(0, [1])
    before = _state(cache)
    ops.fail.add(op)
    with pytest.raises(RuntimeError, match=f"{op} refuses"):
        _attend(cache, [0, 1, 2], 30)
    assert _state(cache) == before


@pytest.mark.parametrize("page_size", [16, 64])
@pytest.mark.parametrize("window, sinks", [(1, 0), (16, 1), (30, 17), (64, 16), (100, 0), (5, 1000)])
def test_released_pages_are_those_no_later_token_sees(ops, window, sinks, page_size):
    cache = _cache(num_pages=40, page_size=page_size, window=window, sinks=sinks)
    for S in (3, 40, 1, 1, 64, 1, 90, 17):
        _attend(cache, [0], S)
        n = cache.seq_lens[0]
        live = [any(t > n - 1 - window or t < sinks for t in range(i * page_size, min((i + 1) * page_size, n)))
                for i in range(cache._pages(n))]
        assert [pg >= 0 for pg in cache.block_tables[0]] == live
        assert sorted(cache._free + [pg for pg in cache.block_tables[0] if pg >= 0]) == list(range(40))
        # the newest tokens' queries are served as far back as their pages are there
        for rows in range(1, 40):
            seen = [t for i in range(rows) for t in range(max(0, n - rows + i + 1)) if t > n - rows + i - window or t < sinks]
            gone = any(not live[t // page_size] for t in seen)
            if gone:
                with pytest.raises(RuntimeError, match="released"):
                    cache.decode([0], _rows(1, rows, 4))
            elif n - rows >= 0:
                cache.decode([0], _rows(1, rows, 4))
    bt, _ = cache.tables([0])
    assert bt.tolist()[0] == cache.block_tables[0]


def test_releases_of_shared_pages(ops):
    cache = _cache(window=16)
    _attend(cache, [0], 48)  # pages 0 and 1 are dead behind the last token
    assert [pg >= 0 for pg in cache.block_tables[0]] == [False, False, True]
    cache.fork(0, [1])
    assert cache._refs == {cache.block_tables[0][2]: 2} and len(cache._free) == 11
    _attend(cache, [0], 16)
    assert cache._refs == {} and len(cache._free) == 10  # the other still holds its page
    _attend(cache, [1], 16)
    assert len(cache._free) == 10
    with pytest.raises(RuntimeError, match="released"):  # a fork is as far on as what it continues
        cache.decode([1], _rows(1, 2, 4))
    assert cache.release([0, 1, 5]) == 0
    assert _cache().release([0]) == 0  # no window, nothing to give back


def test_compact_and_resize(ops):
    cache = _cache(num_pages=12, window=32)
    for s in (0, 1, 2):
        _attend(cache, [s], 40)
    cache.fork(1, [3])
    cache.free(0)
    _attend(cache, [1], 30)
    _mark(cache)
    marks = {s: _marks(cache, s) for s in (1, 2, 3)}
    holes = {s: [pg < 0 for pg in t] for s, t in cache.block_tables.items()}
    held = len({pg for t in cache.block_tables.values() for pg in t if pg >= 0})

    def same():
        assert {s: _marks(cache, s) for s in (1, 2, 3)} == marks
        assert {s: [pg < 0 for pg in t] for s, t in cache.block_tables.items()} == holes
        pages = {pg for t in cache.block_tables.values() for pg in t if pg >= 0}
        assert pages == set(range(held)) and sorted(cache._free) == list(range(held, cache.num_pages))
        assert all(sum(pg in t for t in cache.block_tables.values()) == n for pg, n in cache._refs.items())

    assert cache.compact() == held
    same()
    copies = len([c for c in ops.calls if c[0] == "copy_pages"])
    assert cache.compact() == held
    same()
    assert len([c for c in ops.calls if c[0] == "copy_pages"]) == copies  # nothing to move
    before = _state(cache)
    with pytest.raises(RuntimeError, match="are held"):
        cache.resize(held - 1)
    ops.fail.add("copy_pages")
    with pytest.raises(RuntimeError, match="refuses"):
        cache.resize(30)
    assert _state(cache) == before and cache.code_pages.shape[0] == 12
    ops.fail.clear()
    for n in (30, held):
        cache.resize(n)
        assert cache.num_pages == n and all(p.shape[0] == n for p in cache._pools())
        same()
    assert cache._free == []
    for s in (1, 2, 3):
        cache.free(s)
    assert cache.compact() == 0
    cache.resize(0)
    assert cache._free == []


def test_moves_of_an_ordinary_cache(ops):
    """compact and resize take the caches that were there before too: kept blocks, and sequences that continue others."""
    cache = _cache(_codec(heavy=(1, 3)), value_dtype=BF)
    for s in (4, 0):
        cache.slot_mapping([s], 20)
    cache.fork(0, [1])
    cache.slot_mapping([1], 5)
    cache.free(4)
    _mark(cache)
    marks = {s: _marks(cache, s) for s in (0, 1)}
    assert cache.compact() == 3 and {s: _marks(cache, s) for s in (0, 1)} == marks
    cache.resize(7)
    assert {s: _marks(cache, s) for s in (0, 1)} == marks and cache.pt_pages.shape[0] == 7 and cache.prefix_of == {1: 0}


def test_masks_and_repeated_sequences_are_refused(ops):
    cache = _cache()
    _attend(cache, [0], 4)
    before = _state(cache)
    with pytest.raises(RuntimeError, match="no mask"):
        cache.decode([0], _rows(1, 1, 4), mask=torch.zeros(1, 1, 1, 16))
    cos, sin = hip_ops.rope_table(64, 64)
    for turn in ({}, dict(cos=cos, sin=sin)):
        with pytest.raises(RuntimeError, match="once"):
            cache.append([0, 0], _rows(2, 1), _rows(2, 1), **turn)
    assert _state(cache) == before
    assert math.isfinite(cache.v_scale.sum())


def test_heads_that_do_not_divide_are_refused_before_anything_is_appended(ops):
    """8-bit values of a page are rounded to a scale that grows with the new ones: a step that decode would refuse must not get there."""
    for cache in (_cache(), _cache(value_dtype=BF, window=20)):
        _attend(cache, [0], 4)
        before = _state(cache)
        ops.calls.clear()
        cos, sin = hip_ops.rope_table(64, 64)
        with pytest.raises(RuntimeError, match="divisible"):
            cache.attend([0], _rows(1, 1, 3), _rows(1, 1), _rows(1, 1), cos=cos, sin=sin)
        assert _state(cache) == before and not [c for c in ops.calls if c[0] == "append_kv"]
