"""What attn_var and the K / V cache refuse, and the host side of AttnSeqs: no GPU needed."""
import ctypes as C
import glob
import os
import subprocess

import numpy as np
import pytest
import torch

from cikm2020_dmt_amd import _lib as L
from cikm2020_dmt_amd import kv_cache, ops


def test_struct_layouts():
    lib = L.load()
    assert C.sizeof(L.AttnVarDesc) == lib.dmt_struct_size(15) and C.sizeof(L.KvAttnDesc) == lib.dmt_struct_size(16)


def test_seqs_offsets_and_bounds():
    s = ops.AttnSeqs([3, 0, 5], device="cpu")
    assert s.q_off.tolist() == [0, 3, 3] and (s.max_q, s.end_q, s.total_q, s.k_shared) == (5, 8, 8, False) and s.k_lens is s.q_lens
    s = ops.AttnSeqs(np.array([3, 5]), [4, 6], q_off=[10, 0], k_off=torch.tensor([0, 2]), device="cpu", max_k=9)
    assert (s.end_q, s.total_q, s.end_k, s.k_shared, s.max_q, s.max_k) == (13, 8, 8, True, 5, 9)
    s = ops.AttnSeqs([], device="cpu")
    assert (s.B, s.max_q, s.end_q) == (0, 0, 0)


@pytest.mark.parametrize("kw,msg", [(dict(q_lens=[3, -1]), "must lie in"), (dict(q_lens=[3, 5], q_off=[0, 2]), "share query rows"),
                                    (dict(q_lens=[3, 5], q_off=[0]), "one length and offset"), (dict(q_lens=[3], k_off=[0]), "without k_lens"),
                                    (dict(q_lens=[3, 5], max_q=4), "passes max_q"), (dict(q_lens=[2 ** 31]), "must lie in"),
                                    (dict(q_lens=[1.5]), "integers"), (dict(q_lens=[[1]]), "integers"), (dict(q_lens=[3], q_off=[-1]), "must lie in")])
def test_seqs_refusals(kw, msg):
    with pytest.raises(ValueError, match=msg):
        ops.AttnSeqs(device="cpu", **kw)


def _desc(**kw):
    d = L.AttnVarDesc()
    base = dict(dtype=L.DMT_BF16, B=1, Hq=2, Hkv=1, dh=32, max_q=4, max_k=4, rows_q=4, rows_k=4, Q=1024, q_rs=64, K=1024, k_rs=32, V=1024, v_rs=32,
                q_off=64, q_lens=64, k_off=64, k_lens=64, scale=1.0, cap=0.0, out=1024, o_rs=64, lse=64, dout=1024, do_rs=64, dQ=1024, dq_rs=64,
                dK=1024, dk_rs=32, dV=1024, dv_rs=32, ws=1024, ws_bytes=1 << 20)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    return d


BAD = [(dict(dtype=2), "needs bf16"), (dict(dh=33), "needs bf16"), (dict(dh=136), "needs bf16"), (dict(Hkv=0), "needs bf16"), (dict(Hq=3, Hkv=2), "needs bf16"),
       (dict(B=-1), "negative"), (dict(B=70000), "65535"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(cap=-1.0), "cap"),
       (dict(cap=float("inf")), "cap"), (dict(q_doc=64), "go together"), (dict(q_rs=63), "shorter"), (dict(k_rs=33), "aligned"), (dict(V=1032), "aligned"),
       (dict(Q=None), "NULL"), (dict(k_lens=None), "NULL"), (dict(out=None), "NULL"), (dict(rows_k=2 ** 31), "int32"), (dict(k_rs=1 << 24), "16 MB"),
       (dict(q_doc=64, k_doc=64), "doc_ranges"), (dict(q_doc=64, k_doc=64, doc_ranges=1032), "doc_ranges")]


@pytest.mark.parametrize("kw,msg", BAD)
def test_c_entry_refuses(kw, msg):
    lib, d = L.load(), _desc(**kw)
    assert lib.dmt_attn_var_fwd(C.byref(d), None) == -1 and msg in lib.dmt_last_error().decode()
    assert lib.dmt_attn_var_bwd(C.byref(d), None) == -1


@pytest.mark.parametrize("kw,msg", [(dict(lse=None), "NULL"), (dict(dK=None), "NULL"), (dict(do_rs=60), "stride"), (dict(dV=8), "aligned"),
                                    (dict(dslopes=64), "dslopes"), (dict(ws_bytes=0), "workspace"), (dict(ws=1032), "workspace")])
def test_c_backward_refuses(kw, msg):
    lib, d = L.load(), _desc(**kw)
    assert lib.dmt_attn_var_bwd(C.byref(d), None) == -1 and msg in lib.dmt_last_error().decode()


def test_nothing_to_do_launches_nothing():
    lib = L.load()
    for kw in (dict(B=0), dict(max_q=0), dict(rows_q=0)):
        assert lib.dmt_attn_var_fwd(C.byref(_desc(**kw)), None) == 0
    assert lib.dmt_attn_var_bwd(C.byref(_desc(B=0)), None) == 0
    assert lib.dmt_attn_var_fwd(None, None) == -1


def test_cpu_tensors_are_refused():
    x = torch.zeros((4, 32))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.attn_var(x, x, x, ops.AttnSeqs([4], device="cpu"), 1)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv_cache.kv_plan(i, i, i[:, None].contiguous(), i, i[:1], 4)


CACHE = (2, 32, 8, 1024, 1024, 64, 64)


@pytest.mark.parametrize("c", [(0, 32, 8, 1024, 1024, 64, 64), (2, 24, 8, 1024, 1024, 64, 64), (2, 144, 8, 1024, 1024, 64, 64), (2, 32, 0, 1024, 1024, 64, 64),
                               (2, 32, 1 << 26, 1024, 1024, 64, 64), (2, 32, 8, 1032, 1024, 64, 64), (2, 32, 8, 1024, None, 64, 64), (2, 32, 8, 1024, 1024, None, 64)])
def test_bad_caches_are_refused(c):
    lib = L.load()
    assert lib.dmt_kv_append(*c, 1, 1024, 64, 1024, 64, 64, 64, 64, 1, None) == -1 and b"bad cache" in lib.dmt_last_error()
    assert lib.dmt_kv_read(*c, 1, 64, 1024, 64, 1024, 64, None) == -1
    d = L.KvAttnDesc()
    d.Hkv, d.dh, d.n_blocks, d.k, d.v, d.k_scale, d.v_scale = c
    assert lib.dmt_kv_attn(C.byref(d), None) == -1 and b"bad cache" in lib.dmt_last_error()


def test_kv_entries_refuse():
    lib = L.load()
    assert lib.dmt_kv_append(*CACHE, 1, 1024, 60, 1024, 64, 64, 64, 64, 1, None) == -1 and b"rows of at least" in lib.dmt_last_error()
    assert lib.dmt_kv_append(*CACHE, 1, 1024, 64, 1024, 64, None, 64, 64, 1, None) == -1 and b"NULL" in lib.dmt_last_error()
    assert lib.dmt_kv_append(*CACHE, -1, 1024, 64, 1024, 64, 64, 64, 64, 1, None) == -1
    assert lib.dmt_kv_append(*CACHE, 0, None, 64, None, 64, None, None, None, 0, None) == 0
    assert lib.dmt_kv_read(*CACHE, 0, None, None, 64, None, 64, None) == 0
    assert lib.dmt_kv_read(*CACHE, 1, 64, 1032, 64, 1024, 64, None) == -1
    assert lib.dmt_kv_plan(1, 4, 64, 64, 64, 4, 64, 4, 64, 64, 64, 64, 64, 64, 64, None, 0, None) == -1 and b"workspace" in lib.dmt_last_error()
    assert lib.dmt_kv_plan(-1, 4, 64, 64, 64, 4, 64, 4, 64, 64, 64, 64, 64, 64, 64, 64, 99, None) == -1
    assert lib.dmt_kv_plan(1, 4, 64, 64, 64, 4, 64, 4, 64, 64, 64, None, 64, 64, 64, 64, 99, None) == -1
    assert lib.dmt_kv_release(1, None, 64, 64, 4, 64, 64, 4, None) == -1
    assert lib.dmt_kv_release(0, None, None, None, 4, None, None, 4, None) == 0


@pytest.mark.parametrize("kw,msg", [(dict(Hq=3), "multiple"), (dict(scale=-1.0), "scale"), (dict(cap=-1.0), "scale"), (dict(q_rs=68), "aligned"),
                                    (dict(out=None), "NULL"), (dict(table=None), "NULL"), (dict(n=70000), "65535"), (dict(max_q=-1), "max_q")])
def test_kv_attn_refuses(kw, msg):
    lib, d = L.load(), L.KvAttnDesc()
    base = dict(n=1, Hq=2, Hkv=2, dh=32, n_blocks=8, max_q=1, max_len=64, width=1, rows=1, k=1024, v=1024, k_scale=64, v_scale=64, Q=1024, q_rs=64,
                table=64, lens=64, row_off=64, scale=1.0, cap=0.0, causal=1, out=1024, o_rs=64, ws=1024, ws_bytes=1 << 30)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    assert lib.dmt_kv_attn(C.byref(d), None) == -1 and msg in lib.dmt_last_error().decode()
    for zero in ("n", "max_q", "rows"):
        for k, v in {**base, zero: 0}.items():
            setattr(d, k, v)
        assert lib.dmt_kv_attn(C.byref(d), None) == 0


def test_outputs_in_place_of_inputs_are_refused():
    lib = L.load()
    for same in ("Q", "K", "V"):
        d = _desc(Q=2048, K=4096, V=8192, out={"Q": 2048, "K": 4096, "V": 8192}[same])
        assert lib.dmt_attn_var_fwd(C.byref(d), None) == -1 and b"operand" in lib.dmt_last_error()
    assert lib.dmt_kv_plan(1, 4, 64, 68, 72, 4, 76, 4, 80, 84, 64, 88, 92, 96, 100, 128, 99, None) == -1 and b"lens_out" in lib.dmt_last_error()
    assert lib.dmt_kv_plan(1, 4, 64, 68, 72, 4, 76, 4, 80, 84, 104, 88, 92, 96, 80, 128, 99, None) == -1 and b"state" in lib.dmt_last_error()


@pytest.mark.parametrize("kw", [dict(max_q=2 ** 31 - 1, Hq=4), dict(n=65535, max_q=2 ** 24), dict(n=65535, Hq=65535, Hkv=65535)])
def test_kv_attn_refuses_launches_that_do_not_fit(kw):
    lib, d = L.load(), L.KvAttnDesc()
    base = dict(n=1, Hq=2, Hkv=2, dh=32, n_blocks=8, max_q=1, max_len=2 ** 31 - 64, width=2 ** 24, rows=1, k=1024, v=1024, k_scale=64, v_scale=64, Q=1024,
                q_rs=1 << 21, table=64, lens=64, row_off=64, scale=1.0, cap=0.0, causal=1, out=2048, o_rs=1 << 21, ws=1024, ws_bytes=1 << 62)
    for k, v in {**base, **kw}.items():
        setattr(d, k, v)
    assert lib.dmt_kv_attn(C.byref(d), None) == -1 and b"2^31 workgroups" in lib.dmt_last_error()
    assert lib.dmt_kv_attn_ws_bytes(C.byref(d)) == 0


def test_release_needs_device_tensors():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        kv_cache.kv_release(i, i, i[:, None].contiguous(), i, i[:1])


@pytest.mark.parametrize("rs", ["q_rs", "k_rs", "v_rs", "o_rs", "do_rs"])
def test_row_strides_that_32_rows_cannot_hold_are_refused(rs):
    """rows are addressed by 32-bit offsets from the first row of a wavefront (or of a 64-row tile): 2^24 bytes a row at most, o_rs included"""
    lib, d = L.load(), _desc(**{rs: 1 << 23})
    assert lib.dmt_attn_var_bwd(C.byref(d), None) == -1 and b"stride" in lib.dmt_last_error()


@pytest.mark.parametrize("kw", [dict(cap=1.1e38), dict(scale=1.1e38), dict(cap=3e38)])
def test_caps_and_scales_whose_log2_form_overflows_are_refused(kw):
    """(2 cap log2 e has to be finite: past 1e38 it was not, and the scores came out NaN)"""
    lib, d = L.load(), _desc(**kw)
    assert lib.dmt_attn_var_fwd(C.byref(d), None) == -1 and b"1e38" in lib.dmt_last_error()
    k = L.KvAttnDesc()
    base = dict(n=1, Hq=2, Hkv=2, dh=32, n_blocks=8, max_q=1, max_len=64, width=1, rows=1, k=1024, v=1024, k_scale=64, v_scale=64, Q=1024, q_rs=64,
                table=64, lens=64, row_off=64, scale=1.0, cap=0.0, causal=1, out=1024, o_rs=64, ws=1024, ws_bytes=1 << 30)
    for n, v in {**base, **kw}.items():
        setattr(k, n, v)
    assert lib.dmt_kv_attn(C.byref(k), None) == -1 and b"1e38" in lib.dmt_last_error()


def test_other_flags_build_every_object_again():
    """the flags stand in the Makefile, and some of them are needed for right results: objects of an earlier Makefile are not linked"""
    csrc = os.path.join(os.path.dirname(L.__file__), "csrc")
    plan = subprocess.run(["make", "-n", "-W", "Makefile", "-C", csrc], check=True, capture_output=True, text=True).stdout
    for f in glob.glob(os.path.join(csrc, "*.hip")):
        assert "-c " + os.path.basename(f) in plan, f
