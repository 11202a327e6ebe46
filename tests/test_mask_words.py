"""The heavy-block mask as the operators' two words: any iterable of truth values, once through."""

import numpy as np
import torch

from sunshape_amd import _native as N


def test_every_kind_of_mask():
    want = (0b100101, 1 << 5)
    blocks = [i in (0, 2, 5, 69) for i in range(72)]
    for mask in (blocks, tuple(blocks), torch.tensor(blocks), np.array(blocks), [int(x) for x in blocks],
                 [np.bool_(x) for x in blocks], (x for x in blocks), iter(blocks), map(int, blocks)):
        assert N.mask_words_signed(mask) == want, type(mask)
    assert N.mask_words_signed(None) == N.mask_words_signed([]) == (0, 0)
    assert N.mask_words_signed(x for x in [True] * 64) == (-1, 0)
