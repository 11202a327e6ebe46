"""Host-side checks of ssq_qk_norm_rope, ssq_append and ssq_decode_prefix: refusals come back as a status and a
message before anything is launched (no GPU call is made here), and sizes follow from the arguments alone."""

import ctypes

import pytest
import torch

from sunshape_amd import _native as N
from sunshape_amd import hip_ops

ALIGNED = 1 << 32  # addresses the host code only inspects


def _rope_args(**kw):
    a = N.RopeArgs(dtype=N.SSQ_BF16, q=ALIGNED, q_out=ALIGNED, k=ALIGNED, k_out=ALIGNED, batch=1, seq_len=1, head_dim=64,
                   num_q_heads=2, num_k_heads=1)
    a.rope.cos = a.rope.sin = a.rope.positions = ALIGNED
    a.rope.ld, a.rope.max_pos, a.rope.rot_dim = 32, 16, 64
    for k, v in kw.items():
        setattr(a.rope if k in dict(N.Rope._fields_) else a, k, v)
    return a


@pytest.mark.parametrize("bad, word", [
    (dict(dtype=3), "dtype"), (dict(head_dim=0), "head_dim"), (dict(head_dim=2048), "head_dim"), (dict(q=0), "q and q_out"),
    (dict(k_out=0), "k and k_out"), (dict(rot_dim=63), "rot_dim"), (dict(rot_dim=66), "rot_dim"), (dict(rot_dim=0), "rot_dim"),
    (dict(max_pos=0), "table"), (dict(ld=31), "table"), (dict(interleaved=2), "interleaved"), (dict(sin=0), "cos, sin"),
    (dict(positions=0), "positions"), (dict(q_weight=ALIGNED, w_dtype=7), "weight"), (dict(k_weight=ALIGNED, eps=-1.0), "eps"),
    (dict(num_q_heads=0), "head counts"), (dict(batch=-1), "batch"),
])
def test_rope_refusals(bad, word):
    a = _rope_args(**bad)
    assert N.lib().ssq_qk_norm_rope(ctypes.byref(a), None) == N.SSQ_ERR_INVALID
    assert word.encode() in N.lib().ssq_last_error()


def test_rope_struct_size_and_empty():
    a = _rope_args(struct_size=8)
    assert N.lib().ssq_qk_norm_rope(ctypes.byref(a), None) == N.SSQ_ERR_ABI
    assert N.lib().ssq_qk_norm_rope(None, None) == N.SSQ_ERR_INVALID
    assert N.lib().ssq_qk_norm_rope(ctypes.byref(_rope_args(batch=0)), None) == N.SSQ_OK
    assert N.lib().ssq_qk_norm_rope(ctypes.byref(_rope_args(seq_len=0)), None) == N.SSQ_OK


def _append_args(**kw):
    a = N.AppendArgs(num_pages=8, v=ALIGNED, v_dtype=N.SSQ_BF16, value_dim=64, vp_dtype=N.SSQ_BF16, v_pages=ALIGNED)
    e = dict(keys=ALIGNED, k_dtype=N.SSQ_BF16, k_sb=64, k_sh=64, k_ss=64, batch=2, num_kv_heads=1, seq_len=1, head_dim=64,
             perm=ALIGNED, cent=ALIGNED, block_dim=4, n_blocks=16, n_centroids=256, codes=ALIGNED, slot_mapping=ALIGNED,
             page_size=16)
    for k, v in e.items():
        setattr(a.enc, k, v)
    for k, v in kw.items():
        if k == "heavy":
            a.enc.heavy_mask[0] = v
        else:
            setattr(a.enc if k in e or k in ("kernel", "direct_dist", "pt_dtype") else a.rope if k in dict(N.Rope._fields_)
                    else a, k, v)
    return a


@pytest.mark.parametrize("bad, word, status", [
    (dict(keys=0), "non-NULL", 1), (dict(slot_mapping=0), "slot_mapping", 1), (dict(page_size=0), "page_size", 1),
    (dict(num_pages=-1), "num_pages", 1), (dict(seq_len=1 << 30, batch=4), "too many rows", 1), (dict(k_dtype=5), "k_dtype", 1),
    (dict(block_dim=17), "block_dim", 1), (dict(n_blocks=15), "n_blocks", 1), (dict(n_centroids=0), "n_centroids", 1),
    (dict(heavy=1), "passthrough", 1), (dict(v_pages=0), "v_pages", 1), (dict(v_dtype=9), "value dtype", 1),
    (dict(value_dim=0), "value_dim", 1), (dict(kernel=2), "kernel", 4), (dict(kernel=3), "kernel", 4),
    (dict(direct_dist=2), "direct_dist", 1), (dict(cos=ALIGNED), "positions", 1),
    (dict(n_centroids=4096, codes=ALIGNED + 1), "aligned", 1), (dict(num_kv_heads=70000), "heads", 1),
])
def test_append_refusals(bad, word, status):
    a = _append_args(**bad)
    assert N.lib().ssq_append(ctypes.byref(a), None, 0, None) == status
    assert word.encode() in N.lib().ssq_last_error()
    assert N.lib().ssq_append_workspace_size(ctypes.byref(a)) == 0


def test_append_sizes():
    lib = N.lib()
    a = _append_args()
    a.enc.struct_size = 8
    assert lib.ssq_append(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_ABI
    assert lib.ssq_append(ctypes.byref(N.AppendArgs(struct_size=4)), None, 0, None) == N.SSQ_ERR_ABI
    assert lib.ssq_append(ctypes.byref(_append_args(batch=0)), None, 0, None) == N.SSQ_OK
    assert lib.ssq_append_workspace_size(ctypes.byref(_append_args())) == 0  # a decode step: one launch
    # many rows: the rotated keys and the checked slots; without norm and rotation the slots alone
    big = dict(batch=4, seq_len=8192)
    rope = dict(cos=ALIGNED, sin=ALIGNED, positions=ALIGNED, ld=32, max_pos=16, rot_dim=64)
    n = 4 * 8192
    assert lib.ssq_append_workspace_size(ctypes.byref(_append_args(**big))) == n * 8
    assert lib.ssq_append_workspace_size(ctypes.byref(_append_args(**big, **rope))) == n * 8 + n * 64 * 2
    a = _append_args(**big, **rope)
    assert lib.ssq_append(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_INVALID
    assert b"workspace" in lib.ssq_last_error()


def _prefix_args(**kw):
    a = N.PrefixArgs(prefix_table=ALIGNED, prefix_len=ALIGNED, prefix_cap=1024)
    d = dict(q=ALIGNED, q_dtype=N.SSQ_BF16, q_sb=1024, q_sh=64, q_sl=1024, batch=4, num_q_heads=8, q_len=1, head_dim=64,
             num_kv_heads=2, perm=ALIGNED, cent=ALIGNED, block_dim=4, n_blocks=16, n_centroids=256, layout=N.SSQ_PAGED,
             seq_len=256, codes=ALIGNED, c_sb=512, c_sh=256, c_st=16, block_table=ALIGNED, bt_sb=16, seq_lens=ALIGNED,
             page_size=16, v=ALIGNED, v_dtype=N.SSQ_BF16, value_dim=64, v_sb=2048, v_sh=1024, v_st=16, out=ALIGNED, o_sb=512,
             o_sh=64, o_sl=64)
    for k, v in d.items():
        setattr(a.dec, k, v)
    for k, v in kw.items():
        setattr(a.dec if k in dict(N.DecodeArgs._fields_) and k != "struct_size" else a, k, v)
    return a


@pytest.mark.parametrize("bad, word", [
    (dict(layout=0), "paged"), (dict(scores=ALIGNED), "scores"), (dict(kernel=2), "kernel"), (dict(num_splits=2), "num_splits"),
    (dict(prefix_cap=-1), "prefix_cap"), (dict(prefix_table=0), "prefix_table"), (dict(prefix_len=0), "prefix_len"),
    (dict(num_q_heads=7), "divisible"), (dict(v=0), "v and out"), (dict(out=0), "v and out"), (dict(page_size=4), "page_size"),
    (dict(page_size=24), "page_size"), (dict(block_table=0), "block_table"), (dict(batch=0), "empty"), (dict(q_len=0), "empty"),
    (dict(value_dim=20), "value_dim"), (dict(batch=1 << 20), "too many|batch"), (dict(q_len=1 << 20), "too many"),
    (dict(batch=40000), "65535"),
])
def test_prefix_refusals(bad, word):
    import re

    a = _prefix_args(**bad)
    assert N.lib().ssq_decode_prefix(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_INVALID
    assert re.search(word, N.lib().ssq_last_error().decode())
    assert N.lib().ssq_decode_prefix_workspace_size(ctypes.byref(a)) == 0


def test_prefix_sizes():
    lib = N.lib()
    a = _prefix_args()
    assert lib.ssq_decode_prefix_workspace_size(ctypes.byref(a)) > 0
    assert lib.ssq_decode_prefix(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_INVALID
    assert b"workspace" in lib.ssq_last_error()
    a.dec.struct_size = 8
    assert lib.ssq_decode_prefix(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_ABI
    assert lib.ssq_decode_prefix(ctypes.byref(_prefix_args(struct_size=8)), None, 0, None) == N.SSQ_ERR_ABI
    both = lib.ssq_decode_prefix_workspace_size(ctypes.byref(_prefix_args()))
    own = lib.ssq_decode_prefix_workspace_size(ctypes.byref(_prefix_args(prefix_cap=0, prefix_table=0, prefix_len=0)))
    pre = lib.ssq_decode_prefix_workspace_size(ctypes.byref(_prefix_args(seq_len=0, block_table=0, seq_lens=0)))
    assert own > 0 and pre > 0 and own + pre == both


def test_python_surface_needs_a_device():
    t = torch.zeros(1, 2, 1, 64)
    i = torch.zeros(1, 1, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hip_ops.qk_norm_rope(t, None, None, None, None)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hip_ops.append_kv(t, t, i, t, codes_out=t, v_out=t, slot_mapping=i)
    with pytest.raises(RuntimeError, match="no CPU path"):
        hip_ops.decode_prefix(t, t, t, i, t, prefix_table=i, prefix_len=i, block_table=i, seq_lens=i)
    for bad in (dict(max_position=0, rot_dim=64), dict(max_position=8, rot_dim=63), dict(max_position=8, rot_dim=0)):
        with pytest.raises(RuntimeError):
            hip_ops.rope_table(**bad)


def test_rope_table_values():
    """Angles in 64 bits: fp32 ones would be off by up to position * 2^-24."""
    cos, sin = hip_ops.rope_table(100001, 8, base=500000.0)
    assert cos.shape == sin.shape == (100001, 4) and cos.dtype == torch.float32
    import math

    for pos in (0, 1, 77777, 100000):
        for i in range(4):
            ang = pos * 500000.0 ** (-2 * i / 8)
            assert abs(cos[pos, i].item() - math.cos(ang)) < 1e-7 and abs(sin[pos, i].item() - math.sin(ang)) < 1e-7
