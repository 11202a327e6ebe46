"""append_kv with positions outside the tables: what is stored is what encode gives for the NaN rows that
qk_norm_rope returns, and no other row changes."""

import numpy as np
import pytest
import torch

from _step import DEV, codec_arrays
from _util import log
from sunshape_amd import hip_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S", [4, 4096])
@pytest.mark.parametrize("rot", [64, 32])
def test_codes_of_rows_without_a_position(S, rot):
    log(f"append: positions outside the tables, {S} tokens, {rot} rotated dims")
    rng = np.random.default_rng(2)
    perm, cent, _, _ = (t.to(DEV) if torch.is_tensor(t) else t for t in codec_arrays(rng, 8, 64, 4, 256))
    g = torch.Generator().manual_seed(S + rot)
    k = torch.randn(1, 8, S, 64, generator=g).to(torch.bfloat16).to(DEV)
    cos, sin = hip_ops.rope_table(S, rot, device=DEV)
    pos = torch.arange(S, device=DEV)[None].clone()
    pos[0, 1::2] = torch.where(torch.arange(S // 2, device=DEV) % 2 == 0, S, -5)
    pages = S // 16 + 1
    codes = torch.full((pages, 8, 16, 16), 99, dtype=torch.uint8, device=DEV)
    slots = torch.arange(S, device=DEV)[None]
    hip_ops.append_kv(k, None, perm, cent, codes_out=codes, v_out=None, slot_mapping=slots, cos=cos, sin=sin, positions=pos)
    kr, _ = hip_ops.qk_norm_rope(k, None, cos, sin, pos)
    assert torch.isnan(kr[0, :, 1::2, :rot]).all() and torch.isfinite(kr[0, :, ::2]).all()
    want, _ = hip_ops.encode(kr, perm, cent)
    got = codes.transpose(1, 2).reshape(-1, 8, 16)
    assert torch.equal(got[:S], want[0].transpose(0, 1))
    assert (got[S:] == 99).all()
