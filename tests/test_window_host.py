"""Host-side checks of ssq_append_values, ssq_append8, ssq_decode_window and ssq_copy_pages: refusals come back as a status and
a message before anything is launched (no GPU call is made here), and sizes follow from the arguments alone."""

import ctypes

import pytest
import torch

from sunshape_amd import _native as N
from sunshape_amd import hip_ops
from sunshape_amd._abi import CopyPool

ALIGNED = 1 << 32  # addresses the host code only inspects
E4M3 = torch.float8_e4m3fn


def _values_args(**kw):
    a = N.ValuesArgs(v=ALIGNED, v_dtype=N.SSQ_BF16, v_sb=128, v_sh=64, v_ss=64, batch=2, num_kv_heads=2, seq_len=1, value_dim=64,
                     v_pages=ALIGNED, vp_sb=2048, vp_sh=1024, vp_sd=16, v_scale=ALIGNED, vs_sb=2, vs_sh=1, slot_mapping=ALIGNED,
                     sm_sb=1, page_size=16, num_pages=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad, word", [
    (dict(v=0), "non-NULL"), (dict(v_pages=0), "non-NULL"), (dict(v_scale=0), "non-NULL"), (dict(slot_mapping=0), "non-NULL"),
    (dict(v_dtype=3), "v_dtype"), (dict(v_dtype=-1), "v_dtype"), (dict(batch=-1), "batch"), (dict(seq_len=-1), "seq_len"),
    (dict(num_kv_heads=0), "heads"), (dict(num_kv_heads=65536), "heads"), (dict(value_dim=0), "value_dim"),
    (dict(value_dim=8193), "value_dim"), (dict(page_size=8), "page_size"), (dict(page_size=24), "page_size"),
    (dict(page_size=0), "page_size"), (dict(num_pages=-1), "num_pages"), (dict(num_pages=1 << 40), "num_pages"),
    (dict(v_pages=ALIGNED + 8), "aligned"), (dict(vp_sd=24), "aligned"), (dict(vp_sb=8), "aligned"), (dict(vp_sh=1), "aligned"),
    (dict(batch=1 << 16, seq_len=1 << 16), "too many rows")])
def test_values_refusals(bad, word):
    assert N.lib().ssq_append_values(ctypes.byref(_values_args(**bad)), None) == N.SSQ_ERR_INVALID
    assert word.encode() in N.lib().ssq_last_error()


def test_values_sizes():
    lib = N.lib()
    assert lib.ssq_append_values(None, None) == N.SSQ_ERR_INVALID
    assert lib.ssq_append_values(ctypes.byref(_values_args(struct_size=8)), None) == N.SSQ_ERR_ABI
    for empty in (dict(batch=0), dict(seq_len=0), dict(num_pages=0)):
        assert lib.ssq_append_values(ctypes.byref(_values_args(**empty)), None) == N.SSQ_OK


def _append8_args(**kw):
    a = N.Append8Args(v_scale=ALIGNED, vs_sb=1, vs_sh=1)
    own = dict(num_pages=8, v=ALIGNED, v_dtype=N.SSQ_BF16, v_sb=64, v_sh=64, v_ss=64, value_dim=64, vp_dtype=N.SSQ_E4M3, v_pages=ALIGNED,
               vp_sb=1024, vp_sh=1024, vp_sd=16)
    e = dict(keys=ALIGNED, k_dtype=N.SSQ_BF16, k_sb=64, k_sh=64, k_ss=64, batch=2, num_kv_heads=1, seq_len=1, head_dim=64,
             perm=ALIGNED, cent=ALIGNED, block_dim=4, n_blocks=16, n_centroids=256, codes=ALIGNED, slot_mapping=ALIGNED,
             page_size=16)
    for k, v in {**own, **e, **kw}.items():
        setattr(a.app if k in own else a.app.enc if k in e else a, k, v)
    return a


@pytest.mark.parametrize("bad, word", [
    (dict(keys=0), "non-NULL"), (dict(v=0), "non-NULL"), (dict(v_pages=0), "non-NULL"), (dict(v_scale=0), "non-NULL"),
    (dict(vp_dtype=N.SSQ_BF16), "8-bit"), (dict(vp_dtype=9), "8-bit"), (dict(v_dtype=N.SSQ_E4M3), "v_dtype"),
    (dict(page_size=8), "page_size"), (dict(v_pages=ALIGNED + 4), "aligned"), (dict(n_blocks=15), "n_blocks"),
    (dict(num_pages=-1), "num_pages"), (dict(value_dim=9000), "value_dim")])
def test_append8_refusals(bad, word):
    a = _append8_args(**bad)
    assert N.lib().ssq_append8(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_INVALID
    assert word.encode() in N.lib().ssq_last_error()
    assert N.lib().ssq_append8_workspace_size(ctypes.byref(a)) == 0


def test_append8_sizes():
    lib = N.lib()
    a = _append8_args()
    a.struct_size = 8
    assert lib.ssq_append8(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_ABI
    a = _append8_args()
    a.app.struct_size = 8
    assert lib.ssq_append8(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_ABI
    assert lib.ssq_append8(None, None, 0, None) == N.SSQ_ERR_INVALID
    assert lib.ssq_append8(ctypes.byref(_append8_args(batch=0)), None, 0, None) == N.SSQ_OK
    assert lib.ssq_append8_workspace_size(ctypes.byref(_append8_args())) == 0
    n = 4 * 8192  # many rows: the keys' part needs what it needs with 16-bit values
    big = _append8_args(batch=4, seq_len=8192)
    assert lib.ssq_append8_workspace_size(ctypes.byref(big)) == lib.ssq_append_workspace_size(
        ctypes.byref(_with_16_bits(big))) == 8 * n
    assert lib.ssq_append8(ctypes.byref(big), None, 0, None) == N.SSQ_ERR_INVALID


def _with_16_bits(a):
    b = N.AppendArgs()
    ctypes.memmove(ctypes.byref(b), ctypes.byref(a.app), ctypes.sizeof(b))
    b.vp_dtype = N.SSQ_BF16
    return b


def _window_args(**kw):
    a = N.WindowArgs(window=0, sinks=0, out_dtype=N.SSQ_BF16, num_pages=8, v_scale=ALIGNED, vs_sb=2, vs_sh=1)
    d = dict(q=ALIGNED, q_dtype=N.SSQ_BF16, q_sb=256, q_sh=64, q_sl=256, batch=2, num_q_heads=4, q_len=1, head_dim=64, num_kv_heads=2,
             has_scale=1, scale=0.125, perm=ALIGNED, cent=ALIGNED, cent_sh=0, block_dim=4, n_blocks=16, n_centroids=256,
             layout=N.SSQ_PAGED, seq_len=64, codes=ALIGNED, c_st=16, c_sh=256, c_sb=512, block_table=ALIGNED, bt_sb=4, seq_lens=ALIGNED,
             page_size=16, v=ALIGNED, v_dtype=N.SSQ_E4M3, value_dim=64, v_st=16, v_sh=1024, v_sb=2048, out=ALIGNED, o_sb=256, o_sh=64,
             o_sl=64)
    for k, v in {**d, **kw}.items():
        if k == "heavy":
            a.dec.heavy_mask[0] = v
        else:
            setattr(a.dec if k in dict(N.DecodeArgs._fields_) and k != "num_pages" else a, k, v)
    return a


@pytest.mark.parametrize("bad, word, status", [
    (dict(layout=N.SSQ_CONTIGUOUS), "pages", 1), (dict(v=0), "values", 1), (dict(mask=ALIGNED), "mask", 1),
    (dict(scores=ALIGNED), "scores", 1), (dict(seq_len=8), "block table", 1), (dict(seq_len=0), "block table", 1),
    (dict(window=-1), "window", 1), (dict(sinks=-1), "sinks", 1), (dict(out_dtype=3), "out_dtype", 1), (dict(num_pages=0), "num_pages", 1),
    (dict(num_pages=1 << 31), "num_pages", 1), (dict(v_scale=0), "v_scale", 1), (dict(v_dtype=N.SSQ_BF16), "v_scale", 1),
    (dict(v_dtype=N.SSQ_F32, v_scale=0), "8 or 16 bits", 4), (dict(batch=-1), "batch", 1), (dict(q_len=-3), "q_len", 1),
    (dict(num_kv_heads=0), "heads", 1), (dict(num_q_heads=3), "divisible", 1), (dict(q_len=(1 << 20) + 1), "too many query rows", 1),
    (dict(batch=1 << 20, num_q_heads=64, num_kv_heads=64), "too many query rows", 1),
    (dict(seq_len=1 << 30, batch=1 << 16), "too many query rows", 4), (dict(seq_len=(1 << 30) + 16), "too long", 4),
    (dict(q=0), "non-NULL", 1), (dict(cent=0), "non-NULL", 1), (dict(out=0), "out", 1), (dict(block_table=0), "block_table", 1),
    (dict(seq_lens=0), "seq_lens", 1), (dict(q_dtype=3), "q_dtype", 1), (dict(page_size=8), "page size", 4),
    (dict(page_size=48), "page_size", 1), (dict(page_size=512, seq_len=512), "page_size", 1), (dict(heavy=1, pt=ALIGNED), "passthrough", 4),
    (dict(head_dim=32, n_blocks=8, value_dim=32), "head_dim", 4), (dict(value_dim=128), "value_dim", 4),
    (dict(block_dim=16, n_blocks=4), "block_dim", 4), (dict(block_dim=1, n_blocks=64), "block_dim", 4),
    (dict(n_centroids=300), "byte codes", 4), (dict(code_bits=8), "byte codes", 4), (dict(cent=ALIGNED + 4), "centroids", 1),
    (dict(codes=ALIGNED + 2), "code rows", 1), (dict(c_st=18), "code rows", 1), (dict(v=ALIGNED + 8), "value rows", 1),
    (dict(v_st=24), "value rows", 1), (dict(v_st=-16), "dim stride", 1), (dict(c_sb=1 << 31), "page strides", 1),
    (dict(v_sb=1 << 30), "page strides", 1), (dict(vs_sb=-1), "page strides", 1), (dict(c_st=-16), "page strides", 1)])
def test_window_refusals(bad, word, status):
    a = _window_args(**bad)
    assert N.lib().ssq_decode_window(ctypes.byref(a), ALIGNED, 1 << 40, None) == status
    assert word.encode() in N.lib().ssq_last_error(), N.lib().ssq_last_error()
    assert N.lib().ssq_decode_window_workspace_size(ctypes.byref(a)) == 0


def test_window_sizes():
    lib = N.lib()
    assert lib.ssq_decode_window(None, None, 0, None) == N.SSQ_ERR_INVALID
    a = _window_args()
    a.struct_size = 8
    assert lib.ssq_decode_window(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_ABI
    a = _window_args()
    a.dec.struct_size = 8
    assert lib.ssq_decode_window(ctypes.byref(a), None, 0, None) == N.SSQ_ERR_ABI
    for empty in (dict(batch=0), dict(num_q_heads=0), dict(q_len=0)):
        assert lib.ssq_decode_window(ctypes.byref(_window_args(**empty)), None, 0, None) == N.SSQ_OK
        assert lib.ssq_decode_window_workspace_size(ctypes.byref(_window_args(**empty))) == 0
    # a few tiles a sequence: workgroups join in their own memory; a long context leaves partials
    size = lambda **kw: lib.ssq_decode_window_workspace_size(ctypes.byref(_window_args(**kw)))  # noqa: E731
    assert size(seq_len=256) == 0 and size(seq_len=1 << 17, window=256) == 0
    long = size(seq_len=1 << 17)
    assert long > 0 and size(seq_len=1 << 29, num_pages=(1 << 31) - 1) == long  # and do not grow with it
    assert size(seq_len=1 << 17, window=(1 << 31) - 1, sinks=(1 << 31) - 1) == long
    a = _window_args(seq_len=1 << 17)
    for ws, n in ((ALIGNED, long - 1), (None, long), (ALIGNED + 4, long)):
        assert lib.ssq_decode_window(ctypes.byref(a), ws, n, None) == N.SSQ_ERR_INVALID
        assert b"workspace" in lib.ssq_last_error()


def _copy_args(*pools, **kw):
    a = N.CopyArgs(n_pools=len(pools) or 1, src_pages=ALIGNED, dst_pages=ALIGNED, n_pairs=4)
    for i, p in enumerate(pools or (dict(),)):
        a.pool[i] = CopyPool(**{**dict(src=ALIGNED, dst=ALIGNED, src_stride=64, dst_stride=64, src_pages=8, dst_pages=8, bytes=64), **p})
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("a, word, status", [
    (_copy_args(n_pools=0), "n_pools", 1), (_copy_args(n_pools=9), "n_pools", 1), (_copy_args(n_pairs=-1), "n_pairs", 1),
    (_copy_args(n_pairs=1 << 31), "n_pairs", 1), (_copy_args(src_pages=0), "non-NULL", 1), (_copy_args(dst_pages=0), "non-NULL", 1),
    (_copy_args(dict(), dict(src=0)), "pool 1 is NULL", 1), (_copy_args(dict(dst=0)), "pool 0 is NULL", 1),
    (_copy_args(dict(bytes=-1)), "bad pool", 1), (_copy_args(dict(src_pages=-1)), "bad pool", 1),
    (_copy_args(dict(bytes=(1 << 63) - 1)), "too large", 4)])
def test_copy_refusals(a, word, status):
    assert N.lib().ssq_copy_pages(ctypes.byref(a), None) == status
    assert word.encode() in N.lib().ssq_last_error()


def test_copy_sizes():
    lib = N.lib()
    assert lib.ssq_copy_pages(None, None) == N.SSQ_ERR_INVALID
    assert lib.ssq_copy_pages(ctypes.byref(_copy_args(struct_size=8)), None) == N.SSQ_ERR_ABI
    assert lib.ssq_copy_pages(ctypes.byref(_copy_args(n_pairs=0, src_pages=0, dst_pages=0)), None) == N.SSQ_OK
    assert lib.ssq_copy_pages(ctypes.byref(_copy_args(dict(bytes=0, src=0, dst=0))), None) == N.SSQ_OK


def test_operators_without_a_gpu_say_so():
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    with pytest.raises(RuntimeError, match="value_states"):
        hip_ops.append_values(z(1, 2, 1, 64), z(4, 2, 64, 16, dt=E4M3), z(4, 2, dt=torch.float32), z(1, 1, dt=torch.int64))
    with pytest.raises(RuntimeError, match="query"):
        hip_ops.decode_window(z(1, 2, 1, 64), z(4, 2, 16, 16, dt=torch.uint8), z(4, 2, 64, 16), torch.arange(64), z(16, 256, 4),
                              block_table=z(1, 4, dt=torch.int32), seq_lens=z(1, dt=torch.int32))
    with pytest.raises(RuntimeError, match="pool"):
        hip_ops.copy_pages([z(4, 2)], z(1, dt=torch.int64), z(1, dt=torch.int64))


def test_window_takes_every_prompt_whose_shares_can_be_counted():
    """What is refused is a cost axis past 32 bits: items of the form that the call takes, with the tiles that they can see."""
    lib = N.lib()
    size = lambda **kw: lib.ssq_decode_window_workspace_size(ctypes.byref(_window_args(**kw)))  # noqa: E731
    prompt = dict(num_q_heads=32, num_kv_heads=8, head_dim=128, n_blocks=32, c_st=32, c_sh=512, value_dim=128)
    for kw in (dict(batch=1, q_len=1 << 19, seq_len=1 << 19, window=4096, sinks=4), dict(batch=1, q_len=1 << 19, seq_len=1 << 19),
               dict(batch=16, q_len=1 << 17, seq_len=1 << 17), dict(batch=1, q_len=1 << 20, seq_len=1 << 20, window=4096)):
        assert size(**prompt, **kw) > 0, lib.ssq_last_error()
    # 2^22 items of 256 rows, which cost 5 tiles each beside those of 64 tokens: 506 of them fit, 507 do not
    most = dict(batch=1, num_q_heads=1024, num_kv_heads=1, q_len=1 << 20)
    assert size(**most, seq_len=506 * 64) > 0
    assert size(**most, seq_len=507 * 64) == 0 and b"too many query rows" in lib.ssq_last_error()
    a = _window_args(**most, seq_len=507 * 64)
    assert lib.ssq_decode_window(ctypes.byref(a), ALIGNED, 1 << 40, None) == N.SSQ_ERR_UNSUPPORTED
    # under a window they are those that it holds: 256 + 17 tokens' and one sink's
    assert size(**most, seq_len=1 << 22, window=17, sinks=1) > 0
    # 2^24 sequences of one row: shares of single waves, 2 tiles beside those of 64 tokens
    many = dict(batch=1 << 24, num_q_heads=1, num_kv_heads=1, q_len=1)
    assert size(**many, seq_len=125 * 64) > 0
    assert size(**many, seq_len=126 * 64) == 0 and b"too many query rows" in lib.ssq_last_error()
