"""Drives the host code of ssq_append_values, ssq_append8, ssq_decode_window and ssq_copy_pages (argument checks, choice of
form, launch plans, workspace sizes) with arbitrary arguments, for tests/test_window_sanitizers.py, as tests/host_step_fuzz.py does
for the other steps' entry points: a process that sees no GPU, the host-sanitized library, addresses that the
host code only inspects.

usage: python host_window_fuzz.py <libsunshape_amd_hostsan.so> <examples>
"""

import ctypes
import importlib.util
import os
import random
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
_spec = importlib.util.spec_from_file_location("ssq_abi", os.path.join(HERE, "..", "sunshape_amd", "_abi.py"))
abi = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(abi)

lib = ctypes.CDLL(sys.argv[1])
N_EXAMPLES = int(sys.argv[2]) if len(sys.argv) > 2 else 3000
P, vp, sz = ctypes.POINTER, ctypes.c_void_p, ctypes.c_size_t
lib.ssq_append_values.argtypes = [P(abi.ValuesArgs), vp]
lib.ssq_append8_workspace_size.argtypes, lib.ssq_append8_workspace_size.restype = [P(abi.Append8Args)], sz
lib.ssq_append8.argtypes = [P(abi.Append8Args), vp, sz, vp]
lib.ssq_decode_window_workspace_size.argtypes, lib.ssq_decode_window_workspace_size.restype = [P(abi.WindowArgs)], sz
lib.ssq_decode_window.argtypes = [P(abi.WindowArgs), vp, sz, vp]
lib.ssq_copy_pages.argtypes = [P(abi.CopyArgs), vp]
lib.ssq_last_error.restype = ctypes.c_char_p

ALIGNED, BIG = 1 << 32, (1 << 63) - 1
EDGE = {ctypes.c_int32: [-(1 << 31), -1, 0, 1, 2, 7, 16, 255, 256, 257, 65536, 1 << 20, (1 << 30) + 1, (1 << 31) - 1],
        ctypes.c_int64: [-BIG - 1, -(1 << 40), -1, 0, 1, 3, 8, 16, 1 << 22, 1 << 30, 1 << 31, 1 << 40, BIG],
        ctypes.c_uint32: [0, 8, 1 << 31],
        ctypes.c_float: [0.0, float("nan"), float("inf"), -1.0],
        ctypes.c_void_p: [0, ALIGNED + 1, ALIGNED + 4, ALIGNED + 8]}
rng = random.Random(11)


def addr():
    return ALIGNED + 256 * rng.randint(1, 1 << 24)


def edges(*structs):
    """None to three fields overwritten with edge values."""
    for _ in range(rng.choice([0, 0, 1, 1, 1, 2, 3])):
        s = rng.choice(structs)
        name, kind = rng.choice([f for f in s._fields_ if f[1] in EDGE])
        setattr(s, name, rng.choice(EDGE[kind]))


def status(rc):
    assert rc in (0, 1, 2, 3, 4), rc
    if rc:
        assert lib.ssq_last_error()


def values_fields():
    B, S, h, dv = rng.choice([0, 1, 3, 64]), rng.choice([0, 1, 7, 1000, 1 << 20]), rng.choice([1, 2, 8, 65535]), rng.choice([1, 64, 128, 8192])
    page = rng.choice([16, 16, 32, 48, 256, 1 << 20])
    return B, S, h, dv, page, dict(v=addr(), v_dtype=rng.randint(0, 2), v_ss=dv, v_sh=S * dv, v_sb=h * S * dv, v_pages=addr(), vp_sd=page,
                                   vp_sh=dv * page, vp_sb=h * dv * page, value_dim=dv)


def values():
    B, S, h, dv, page, kw = values_fields()
    a = abi.ValuesArgs(batch=B, num_kv_heads=h, seq_len=S, v_scale=addr(), vs_sb=h, vs_sh=1, slot_mapping=addr(), sm_sb=S,
                       page_size=page, num_pages=rng.choice([0, 1, 100, 1 << 30, (1 << 31) - 1]), **kw)
    edges(a)
    status(lib.ssq_append_values(ctypes.byref(a), None))


def append8():
    B, S, h, dv, page, kw = values_fields()
    hd, bd = rng.choice([64, 128]), rng.choice([2, 4, 8])
    nb, nc = hd // bd, rng.choice([16, 256, 300, 65536])
    a = abi.Append8Args(v_scale=addr(), vs_sb=h, vs_sh=1)
    for k, v in dict(kw, vp_dtype=3, num_pages=rng.choice([0, 100, 1 << 30, (1 << 31) - 1])).items():
        setattr(a.app, k, v)
    for k, v in dict(keys=addr(), k_dtype=rng.randint(0, 2), k_ss=hd, k_sh=S * hd, k_sb=h * S * hd, batch=B, num_kv_heads=h, seq_len=S,
                     head_dim=hd, perm=addr(), perm_sh=rng.choice([0, hd]), cent=addr(), cent_sh=rng.choice([0, nb * nc * bd]), block_dim=bd,
                     n_blocks=nb, n_centroids=nc, codes=addr(), c_st=nb, c_sh=page * nb, c_sb=h * page * nb, slot_mapping=addr(), sm_sb=S,
                     page_size=page, kernel=rng.choice([0, 0, 1]), direct_dist=rng.choice([0, 0, 1])).items():
        setattr(a.app.enc, k, v)
    if rng.random() < 0.5:
        for k, v in dict(cos=addr(), sin=addr(), positions=addr(), ld=hd // 2, max_pos=4096, rot_dim=hd, p_sb=1, p_ss=1).items():
            setattr(a.app.rope, k, v)
    edges(a, a.app, a.app.enc, a.app.rope)
    n = lib.ssq_append8_workspace_size(ctypes.byref(a))
    status(lib.ssq_append8(ctypes.byref(a), ALIGNED if n else None, n, None))
    if n:
        status(lib.ssq_append8(ctypes.byref(a), ALIGNED, n - 1, None))


def window():
    hd = rng.choice([64, 128, 128, 96])
    bd = rng.choice([2, 4, 4, 8, 16])
    nb, nc, hkv = hd // bd, rng.choice([16, 64, 256, 256, 300]), rng.choice([1, 2, 8, 16, 65536])
    hq, B, Lq = hkv * rng.choice([0, 1, 4, 7, 8]), rng.choice([0, 1, 5, 64, 700]), rng.choice([0, 1, 1, 5, 512, 1 << 20])
    page, width, vt = rng.choice([16, 16, 32, 64, 256]), rng.choice([0, 1, 33, 5000, 1 << 22]), rng.choice([1, 2, 3, 3])
    a = abi.WindowArgs(window=rng.choice([0, 0, 1, 4096, (1 << 31) - 1]), sinks=rng.choice([0, 4, (1 << 31) - 1]), out_dtype=rng.randint(0, 2),
                       num_pages=rng.choice([1, 1000, (1 << 31) - 1]), v_scale=addr() if vt == 3 else 0, vs_sb=hkv, vs_sh=1)
    for k, v in dict(q=addr(), q_dtype=rng.randint(0, 2), q_sl=hd, q_sh=Lq * hd, q_sb=hq * Lq * hd, batch=B, num_q_heads=hq, q_len=Lq,
                     head_dim=hd, num_kv_heads=hkv, has_scale=1, scale=0.125, perm=addr(), cent=addr(), cent_sh=rng.choice([0, nb * nc * bd]),
                     block_dim=bd, n_blocks=nb, n_centroids=nc, layout=1, seq_len=min(width * page, (1 << 31) - 1), codes=addr(), c_st=nb,
                     c_sh=page * nb, c_sb=hkv * page * nb, block_table=addr(), bt_sb=width, seq_lens=addr(), page_size=page, v=addr(),
                     v_dtype=vt, value_dim=hd, v_st=page, v_sh=hd * page, v_sb=hkv * hd * page, out=addr(), o_sl=hd, o_sh=Lq * hd,
                     o_sb=hq * Lq * hd, lse=rng.choice([0, addr()])).items():
        setattr(a.dec, k, v)
    edges(a, a.dec, a.dec)
    n = lib.ssq_decode_window_workspace_size(ctypes.byref(a))
    status(lib.ssq_decode_window(ctypes.byref(a), ALIGNED if n else None, n, None))
    if n:
        status(lib.ssq_decode_window(ctypes.byref(a), ALIGNED, n - 1, None))


def copies():
    a = abi.CopyArgs(n_pools=rng.randint(1, 8), src_pages=addr(), dst_pages=addr(), n_pairs=rng.choice([0, 1, 64, 1 << 20, (1 << 31) - 1]))
    for k in range(8):
        n = rng.choice([0, 1, 8, 2048, 1 << 20, 1 << 32])
        p = abi.CopyPool(src=addr(), dst=addr(), src_stride=n, dst_stride=n, src_pages=rng.choice([0, 5, BIG]), dst_pages=rng.choice([0, 5, BIG]),
                         bytes=n)
        edges(p)
        a.pool[k] = p
    edges(a)
    status(lib.ssq_copy_pages(ctypes.byref(a), None))


if __name__ == "__main__":
    for f in (values, append8, window, copies):
        for i in range(N_EXAMPLES):
            f()
        print(f.__name__, N_EXAMPLES, flush=True)
    print(f"host window fuzz: {4 * N_EXAMPLES} examples, no sanitizer report")
