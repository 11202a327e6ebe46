"""Drives the host code of ssq_qk_norm_rope, ssq_append and ssq_decode_prefix (argument checks, choice of form, launch
plans, workspace sizes) with arbitrary arguments, for tests/test_step_sanitizers.py, as tests/host_abi_fuzz.py does
for the other entry points: a process that sees no GPU, the host-sanitized library, addresses that the host code
only inspects.

usage: python host_step_fuzz.py <libsunshape_amd_hostsan.so> <examples>
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
lib.ssq_qk_norm_rope.argtypes = [P(abi.RopeArgs), vp]
lib.ssq_append_workspace_size.argtypes, lib.ssq_append_workspace_size.restype = [P(abi.AppendArgs)], sz
lib.ssq_append.argtypes = [P(abi.AppendArgs), vp, sz, vp]
lib.ssq_decode_prefix_workspace_size.argtypes, lib.ssq_decode_prefix_workspace_size.restype = [P(abi.PrefixArgs)], sz
lib.ssq_decode_prefix.argtypes = [P(abi.PrefixArgs), vp, sz, vp]
lib.ssq_last_error.restype = ctypes.c_char_p

ALIGNED = 1 << 32
EDGE = {ctypes.c_int32: [-(1 << 31), -1, 0, 1, 2, 7, 16, 255, 256, 257, 65536, 1 << 20, (1 << 30) + 1, (1 << 31) - 1],
        ctypes.c_int64: [-(1 << 40), -1, 0, 1, 2, 3, 7, 8, 12, 1 << 31, 1 << 40],
        ctypes.c_uint32: [0, 8, 1 << 31],
        ctypes.c_float: [0.0, float("nan"), float("inf"), -1.0],
        ctypes.c_double: [0.0, float("nan"), float("inf"), -1.0],
        ctypes.c_void_p: [0, ALIGNED + 1, ALIGNED + 2, ALIGNED + 8]}
rng = random.Random(7)


def addr():
    return ALIGNED + 256 * rng.randint(1, 1 << 24)


def put(struct, **kw):
    for k, v in kw.items():
        setattr(struct, k, v)


def edges(*structs):
    """None to three fields overwritten with edge values."""
    for _ in range(rng.choice([0, 0, 1, 1, 1, 2, 3])):
        s = rng.choice(structs)
        name, kind = rng.choice([f for f in s._fields_ if f[1] in EDGE])
        setattr(s, name, rng.choice(EDGE[kind]))


def turn(t, head_dim):
    if rng.random() < 0.8:
        rot = 2 * rng.randint(1, head_dim // 2)
        put(t, cos=addr(), sin=addr(), positions=addr(), ld=rot // 2, max_pos=rng.choice([1, 4096]), rot_dim=rot,
            interleaved=rng.randint(0, 1), p_sb=1, p_ss=1)
    put(t, w_dtype=rng.randint(0, 2), eps=1e-6)


def status(rc):
    assert rc in (0, 1, 2, 3, 4), rc
    if rc:
        assert lib.ssq_last_error()


def rope():
    hd, hq, hk = rng.choice([2, 48, 64, 128, 256, 1024]), rng.choice([1, 14, 32]), rng.choice([0, 2, 8])
    B, S = rng.choice([0, 1, 3, 64]), rng.choice([0, 1, 517, 1 << 20])
    a = abi.RopeArgs(dtype=rng.randint(0, 2), q=addr(), q_sb=S * hq * hd, q_sh=hd, q_ss=hq * hd, q_out=addr(), qo_sb=S * hq * hd,
                     qo_sh=hd, qo_ss=hq * hd, k=addr(), k_sb=S * hk * hd, k_sh=hd, k_ss=hk * hd, k_out=addr(), ko_sb=S * hk * hd,
                     ko_sh=hd, ko_ss=hk * hd, batch=B, seq_len=S, head_dim=hd, num_q_heads=hq, num_k_heads=hk,
                     q_weight=rng.choice([0, addr()]), k_weight=rng.choice([0, addr()]))
    turn(a.rope, hd)
    edges(a, a.rope)
    status(lib.ssq_qk_norm_rope(ctypes.byref(a), None))


def append():
    hd = rng.choice([32, 64, 128, 256, 1024])
    bd = rng.choice([b for b in (1, 2, 3, 4, 8, 16) if hd % b == 0 and hd // b <= 128] or [8])
    nb, nc, hkv = hd // bd, rng.choice([1, 16, 64, 256, 257, 4096, 65536, 1 << 20]), rng.choice([1, 2, 8])
    B, S, page = rng.choice([0, 1, 3, 64]), rng.choice([0, 1, 7, 8, 1000, 1 << 20]), rng.choice([1, 5, 8, 16, 64])
    a = abi.AppendArgs(num_pages=rng.choice([0, 100, 100, 1 << 30, (1 << 63) - 1, -(1 << 63)]), k_weight=rng.choice([0, addr()]))
    e = a.enc
    put(e, keys=addr(), k_dtype=rng.randint(0, 2), k_ss=hd, k_sh=S * hd, k_sb=hkv * S * hd, batch=B, num_kv_heads=hkv, seq_len=S,
        head_dim=hd, perm=addr(), perm_sh=rng.choice([0, hd]), cent=addr(), cent_sh=rng.choice([0, nb * nc * bd]), block_dim=bd,
        n_blocks=nb, n_centroids=nc, codes=addr(), c_st=nb, c_sh=page * nb, c_sb=hkv * page * nb, slot_mapping=addr(), sm_sb=S,
        page_size=page, kernel=rng.choice([0, 0, 1]), direct_dist=rng.choice([0, 0, 1]))
    heavy = [i for i in range(nb) if rng.random() < 0.1] if rng.random() < 0.4 else []
    for i in heavy:
        e.heavy_mask[i // 64] |= 1 << (i % 64)
    if heavy:
        n = len(heavy) * bd
        put(e, pt=addr(), pt_dtype=rng.randint(0, 2), pt_st=n, pt_sh=page * n, pt_sb=hkv * page * n)
    if rng.random() < 0.2:
        put(e, metric=addr(), metric_sh=hd * hd)
    if rng.random() < 0.8:
        dv = rng.choice([1, 24, 64, 128, 200, 8192])
        put(a, v=addr(), v_dtype=rng.randint(0, 2), v_ss=dv, v_sh=S * dv, v_sb=hkv * S * dv, value_dim=dv, vp_dtype=rng.randint(0, 2),
            v_pages=addr(), vp_sd=page, vp_sh=dv * page, vp_sb=hkv * dv * page)
    turn(a.rope, hd)
    edges(a, e, e, a.rope)
    n = lib.ssq_append_workspace_size(ctypes.byref(a))
    status(lib.ssq_append(ctypes.byref(a), ALIGNED if n else None, n, None))
    if n:
        status(lib.ssq_append(ctypes.byref(a), ALIGNED, n - 1, None))


def prefix():
    hd = rng.choice([32, 64, 64, 128, 128, 256])
    bd = rng.choice([b for b in (1, 2, 4, 8, 16) if hd // b <= 128])
    nb, nc, hkv = hd // bd, rng.choice([16, 64, 256, 256, 4096, 65536]), rng.choice([1, 2, 8, 16])
    hq, B, Lq = hkv * rng.choice([1, 4, 7, 8]), rng.choice([1, 5, 64, 700]), rng.choice([1, 1, 3, 64])
    page, width = rng.choice([8, 16, 16, 64, 256]), rng.choice([0, 1, 33, 5000])
    dv = rng.choice([hd, hd, 64])
    a = abi.PrefixArgs(prefix_table=addr(), prefix_len=addr(), prefix_cap=page * rng.choice([0, 1, 33, 4096, 1 << 20]))
    d = a.dec
    put(d, q=addr(), q_dtype=rng.randint(0, 2), q_sl=hd, q_sh=Lq * hd, q_sb=hq * Lq * hd, batch=B, num_q_heads=hq, q_len=Lq, head_dim=hd,
        num_kv_heads=hkv, has_scale=1, scale=0.125, perm=addr(), cent=addr(), cent_sh=rng.choice([0, nb * nc * bd]), block_dim=bd,
        n_blocks=nb, n_centroids=nc, layout=1, seq_len=width * page, codes=addr(), c_st=nb, c_sh=page * nb, c_sb=hkv * page * nb,
        block_table=addr() if width else 0, bt_sb=width, seq_lens=addr(), page_size=page, v=addr(), v_dtype=rng.randint(0, 2),
        value_dim=dv, v_st=page, v_sh=dv * page, v_sb=hkv * dv * page, out=addr(), o_sl=dv, o_sh=Lq * dv, o_sb=hq * Lq * dv,
        lse=rng.choice([0, addr()]), kernel=rng.choice([0, 0, 0, 1]), code_bits=rng.choice([0, 0, 0, 4, 6, 8]) if nc <= 256 else 0)
    heavy = [i for i in range(nb) if rng.random() < 0.1] if rng.random() < 0.4 else []
    for i in heavy:
        d.heavy_mask[i // 64] |= 1 << (i % 64)
    if heavy:
        n = len(heavy) * bd
        put(d, pt=addr(), pt_dtype=rng.randint(0, 2), pt_st=n, pt_sh=page * n, pt_sb=hkv * page * n)
    if rng.random() < 0.3:
        put(d, mask=addr(), m_st=1)
    edges(a, d, d, d)
    n = lib.ssq_decode_prefix_workspace_size(ctypes.byref(a))
    status(lib.ssq_decode_prefix(ctypes.byref(a), ALIGNED if n else None, n, None))
    if n:
        status(lib.ssq_decode_prefix(ctypes.byref(a), ALIGNED, n - 1, None))


if __name__ == "__main__":
    for f in (rope, append, prefix):
        for i in range(N_EXAMPLES):
            f()
        print(f.__name__, N_EXAMPLES, flush=True)
    print(f"host step fuzz: {3 * N_EXAMPLES} examples, no sanitizer report")
