"""Steps of PagedSunShapeCache that the operators refuse: nothing of them stays, and what follows is what it would have
been without them."""

import math

import pytest
import torch

from _step import DEV
from _util import log
from sunshape_amd import hip_ops
from test_gpu_step import _cache

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("forked", [False, True])
def test_refused_steps_leave_nothing(forked):
    log(f"attend: refusals, forked {forked}")
    D, Hq, Hkv = 64, 8, 2
    g = torch.Generator().manual_seed(1)
    cos, sin = hip_ops.rope_table(100, D, device=DEV)
    kw = dict(cos=cos, sin=sin, scale=1 / math.sqrt(D))

    def rows(B, S, d=D, dt=BF):
        return [torch.randn(B, h, S, d, generator=g).to(dt).to(DEV) for h in (Hq, Hkv, Hkv)]

    caches = [_cache(D, Hkv, num_pages=12)[0] for _ in range(2)]
    q, k, v = rows(1, 37)
    for c in caches:
        c.attend([0], q, k, v, **kw)
        if forked:
            c.fork(0, [1, 2])
    tried = caches[0]
    ids = [1, 2]

    def state(c):
        return list(c._free), {s: list(t) for s, t in c.block_tables.items()}, dict(c.seq_lens), dict(c.prefix_of)

    for S in (1, 20):
        q, k, v = rows(2, S)
        before = state(tried)
        end = (37 if forked else 0) + tried.seq_lens.get(1, 0) + S
        bad = [
            dict(k_weight=torch.ones(D // 2, device=DEV)), dict(q_weight=torch.ones(D + 1, device=DEV)),
            dict(k_weight=torch.ones(D)), dict(eps=-1.0, k_weight=torch.ones(D, device=DEV)),
            dict(value_states=v[..., :D // 2].contiguous()), dict(value_states=v.double()), dict(key_states=k.double()),
            dict(key_states=rows(2, S, 2 * D)[1]), dict(query=rows(2, S, 2 * D)[0]), dict(query=q[:, :Hq - 1]),
            dict(cos=cos[:, :8]), dict(cos=cos.double(), sin=sin.double()), dict(cos=cos[:end - 1], sin=sin[:end - 1]),
        ]
        for b in bad:
            with pytest.raises(RuntimeError):
                tried.attend(ids, **{**dict(query=q, key_states=k, value_states=v), **kw, **b})
            assert state(tried) == before, list(b)
        for b in (dict(value_states=v[..., :D // 2].contiguous()), dict(key_states=rows(2, S, 2 * D)[1])):
            with pytest.raises(RuntimeError):  # without the rotation
                tried.append(ids, **{**dict(key_states=k, value_states=v), **b})
            assert state(tried) == before, list(b)
        with pytest.raises(RuntimeError, match="out of pages"):
            tried.attend(ids, *rows(2, 90), **{**kw, "cos": cos.repeat(2, 1), "sin": sin.repeat(2, 1)})
        assert state(tried) == before
        a, b = (c.attend(ids, q, k, v, **kw) for c in caches)
        assert torch.equal(a, b) and state(caches[0]) == state(caches[1])
