"""A step that PagedSunShapeCache refuses leaves its lengths, tables and free pages as they were (CPU: the pages are
host tensors, which the operators refuse, and stand-ins where a step is to succeed)."""

import numpy as np
import pytest
import torch

from _step import codec_arrays
from sunshape_amd import hip_ops, paged
from sunshape_amd.codec import SunShapeBlockCodec
from sunshape_amd.paged import PagedSunShapeCache

BF = torch.bfloat16


def _cache(num_pages=6, page_size=16):
    perm, cent, _, _ = codec_arrays(np.random.default_rng(0), 2, 64, 4, 256, True)
    codec = SunShapeBlockCodec.from_buffers(perm, cent, mode="profileperm_baseline", device=torch.device("cpu"))
    return PagedSunShapeCache(codec, num_pages=num_pages, num_kv_heads=2, value_dim=64, page_size=page_size, device=torch.device("cpu"))


def _state(cache):
    return (list(cache._free), {s: list(t) for s, t in cache.block_tables.items()}, dict(cache.seq_lens), dict(cache.prefix_of))


@pytest.fixture
def stand_ins(monkeypatch):
    """Operators that take their arguments and compute nothing; `fail` names one that raises."""
    fail = set()

    def op(name, result):
        def call(*args, **kw):
            if name in fail:
                raise RuntimeError(f"{name} refuses")
            return result(*args)
        monkeypatch.setattr(paged.hip_ops, name, call)

    op("append_kv", lambda *a: None)
    op("qk_norm_rope", lambda q, *a: (q, None))
    op("decode", lambda q, *a: q)
    op("decode_prefix", lambda q, *a: q)
    op("encode", lambda *a: None)
    return fail


def _rows(B, S, H=2, D=64):
    return torch.zeros(B, H, S, D, dtype=BF)


def test_a_pool_that_runs_out_is_left_as_it_was(stand_ins):
    cache = _cache(num_pages=6)
    cos, sin = hip_ops.rope_table(256, 64)
    cache.attend([7], _rows(1, 20, 4), _rows(1, 20), _rows(1, 20), cos=cos, sin=sin)
    before = _state(cache)
    assert len(before[0]) == 4
    # 7 has room for 12 more; 1 and 2 take three pages, 3 a fourth and fifth
    for step in (lambda: cache.slot_mapping([7, 1, 2, 3], 33), lambda: cache.slot_mapping([1, 1, 1], 32),
                 lambda: cache.append([7, 1, 2, 3], _rows(4, 33), _rows(4, 33)),
                 lambda: cache.append([7, 1, 2, 3], _rows(4, 33), _rows(4, 33), cos=cos, sin=sin),
                 lambda: cache.attend([1, 2, 3], _rows(3, 20, 4), _rows(3, 20), _rows(3, 20), cos=cos, sin=sin)):
        with pytest.raises(RuntimeError, match="out of pages"):
            step()
        assert _state(cache) == before
    assert cache.slot_mapping([7, 1, 1], 12).shape == (3, 12)  # what fits is given
    assert cache.seq_lens == {7: 32, 1: 24} and len(cache._free) == 2


@pytest.mark.parametrize("op", ["append_kv", "qk_norm_rope", "decode"])
def test_an_operator_that_refuses(stand_ins, op):
    cache = _cache(num_pages=8)
    cos, sin = hip_ops.rope_table(256, 64)
    cache.attend([7], _rows(1, 20, 4), _rows(1, 20), _rows(1, 20), cos=cos, sin=sin)
    before = _state(cache)
    stand_ins.add(op)
    for S in (1, 20):
        with pytest.raises(RuntimeError, match=f"{op} refuses"):
            cache.attend([7, 1, 2], _rows(3, S, 4), _rows(3, S), _rows(3, S), cos=cos, sin=sin)
        assert _state(cache) == before
    if op == "append_kv":
        with pytest.raises(RuntimeError, match="append_kv refuses"):
            cache.append([1, 7], _rows(2, 3), _rows(2, 3), k_weight=torch.ones(64))
        assert _state(cache) == before
    stand_ins.clear()
    cache.attend([7, 1, 2], _rows(3, 1, 4), _rows(3, 1), _rows(3, 1), cos=cos, sin=sin)
    assert cache.seq_lens == {7: 21, 1: 1, 2: 1}


def test_a_forked_sequence_whose_step_is_refused(stand_ins):
    cache = _cache()
    cos, sin = hip_ops.rope_table(256, 64)
    cache.attend([7], _rows(1, 20, 4), _rows(1, 20), _rows(1, 20), cos=cos, sin=sin)
    cache.fork(7, [1, 2])
    before = _state(cache)
    stand_ins.add("decode_prefix")
    with pytest.raises(RuntimeError, match="decode_prefix refuses"):
        cache.attend([1, 2], _rows(2, 1, 4), _rows(2, 1), _rows(2, 1), cos=cos, sin=sin)
    assert _state(cache) == before


def test_an_append_without_rotation_that_is_refused():
    """Encoding on the host is refused: after the slots were taken."""
    cache = _cache()
    before = _state(cache)
    for kw in ({}, dict(k_weight=torch.ones(64))):
        with pytest.raises(RuntimeError):
            cache.append([1, 2], _rows(2, 3), _rows(2, 3), **kw)
        assert _state(cache) == before


def test_positions_past_the_tables(stand_ins):
    cache = _cache(num_pages=8)
    cos, sin = hip_ops.rope_table(24, 64)
    cache.attend([7], _rows(1, 20, 4), _rows(1, 20), _rows(1, 20), cos=cos, sin=sin)
    cache.fork(7, [1])
    before = _state(cache)
    for ids, S in (([1], 5), ([2], 25)):
        with pytest.raises(RuntimeError, match=r"outside the rotation's tables \(24 rows\)"):
            cache.attend(ids, _rows(1, S, 4), _rows(1, S), _rows(1, S), cos=cos, sin=sin)
        with pytest.raises(RuntimeError, match="outside the rotation's tables"):
            cache.append(ids, _rows(1, S), _rows(1, S), cos=cos, sin=sin)
        assert _state(cache) == before
    cache.attend([1], _rows(1, 4, 4), _rows(1, 4), _rows(1, 4), cos=cos, sin=sin)  # up to the last row
    cache.append([2], _rows(1, 24), _rows(1, 24), cos=cos, sin=sin)
    cache.append([3], _rows(1, 30), _rows(1, 30), k_weight=torch.ones(64))  # no rotation, no end
    cache.append([2], _rows(1, 0), _rows(1, 0), cos=cos, sin=sin)  # nothing new


def test_a_sine_without_its_cosine():
    """append takes both tables or neither: one alone is refused, not left aside."""
    cache = _cache()
    _, sin = hip_ops.rope_table(24, 64)
    before = _state(cache)
    with pytest.raises(RuntimeError, match="cos and sin"):
        cache.append([1], _rows(1, 3), _rows(1, 3), sin=sin)
    assert _state(cache) == before


def test_fork_of_a_sequence_without_tokens(stand_ins):
    cache = _cache()
    cache.append([1], _rows(1, 0), _rows(1, 0))
    for prefix in (1, 9):
        with pytest.raises(RuntimeError, match="holds no tokens"):
            cache.fork(prefix, [2])
    assert cache.prefix_of == {}
    cache.append([1], _rows(1, 1), _rows(1, 1), k_weight=torch.ones(64))
    cache.fork(1, [2])
