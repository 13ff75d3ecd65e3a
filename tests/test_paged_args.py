"""Refusals of the paged-cache entry points that need no GPU: the C ABI's argument checks run before
any device access, and the Python side checks shapes before it asks for the device."""
import ctypes

import pytest
import torch

import usagi_b200 as ub
from usagi_b200 import _lib

class Call(ctypes.Structure):
    """bsattn_paged_call of include/bsattn.h."""
    _fields_ = [("k_pages", ctypes.c_void_p), ("v_pages", ctypes.c_void_p),
                ("page_strides", ctypes.c_int64 * 6), ("block_table", ctypes.c_void_p),
                ("table_stride", ctypes.c_int64), ("seq_lens", ctypes.c_void_p),
                ("q_lens", ctypes.c_void_p)] + [(n, ctypes.c_int32) for n in (
                    "max_pages", "n_pages", "page_size", "B", "Hq", "Hkv", "Tq", "dtype_flags")] + \
               [("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
                ("stream", ctypes.c_void_p)]


def _record(a):
    return ctypes.byref(Call(a["kp"], a["vp"], (ctypes.c_int64 * 6)(*a["st"]), a["table"], a["ts"],
                             a["sl"], a["ql"], a["mp"], a["np"], a["ps"], a["B"], a["Hq"], a["Hkv"],
                             a["Tq"], a["flags"], a["ws"], a["wsb"], None))


CACHE = dict(kp=16, vp=16, st=[128] * 6, table=16, ts=4, mp=4, np=8, ps=16, sl=16, ql=0, B=1, Hq=2,
             Hkv=1, Tq=1, flags=0, ws=16, wsb=256)


def _fwd(**kw):
    a = dict(CACHE, q=16, o=16, lse=None, window=0, glob=0, prefix=0, cnt=16)
    a.update(kw)
    return _lib.load().bsattn_paged_fwd(_record(a), a["q"], a["o"], a["lse"], a["window"],
                                        a["glob"], a["prefix"], 0.0, 16, 1 << 20, a["cnt"])


def _append(**kw):
    a = dict(CACHE, q=16, k=16, v=16, ins=[128] * 9, qo=16, inv=16, rot=128)
    a.update(kw)
    ins = None if a["ins"] is None else (ctypes.c_int64 * 9)(*a["ins"])
    return _lib.load().bsattn_paged_append(_record(a), a["q"], a["k"], a["v"], ins, a["qo"],
                                           a["inv"], a["rot"], 0)


@pytest.mark.parametrize("call", [_fwd, _append])
def test_cache_arguments(call):
    for name in ("kp", "vp", "table", "sl"):
        assert call(**{name: 0}) == _lib.E_NULL, name
    assert call(q=None) == _lib.E_NULL
    for kw in (dict(B=0), dict(Hkv=0), dict(Tq=0), dict(mp=0), dict(np=0), dict(ts=-1),
               dict(ps=8), dict(ps=48), dict(ps=2048), dict(mp=1 << 27)):
        assert call(**kw) == _lib.E_SHAPE, kw
    assert call(kp=24) == _lib.E_ALIGN
    for bad in (132, 0, -128):
        assert call(st=[128, 128, bad, 128, 128, 128]) == _lib.E_ALIGN
    assert call(ws=0) == _lib.E_WORKSPACE
    assert call(wsb=4) == _lib.E_WORKSPACE


def test_attention_arguments():
    for kw in (dict(window=-1), dict(glob=-1, window=1), dict(glob=1), dict(window=1 << 25),
               dict(prefix=-16), dict(prefix=24), dict(prefix=80), dict(prefix=16, window=1)):
        assert _fwd(**kw) == _lib.E_SHAPE, kw
    assert _fwd(o=None) == _lib.E_NULL
    assert _fwd(cnt=None) == _lib.E_NULL
    assert _fwd(flags=4) == _lib.E_DTYPE
    assert _fwd(q=24) == _lib.E_ALIGN
    assert _fwd(o=24) == _lib.E_ALIGN


def test_append_arguments():
    assert _append(k=None) == _lib.E_NULL
    assert _append(ins=None) == _lib.E_NULL
    assert _append(qo=None) == _lib.E_NULL
    assert _append(flags=1) == _lib.E_DTYPE
    for rot in (0, 8, 24, 144, -16):
        assert _append(rot=rot) == _lib.E_SHAPE, rot
    assert _append(k=24) == _lib.E_ALIGN
    assert _append(ins=[128] * 8 + [100]) == _lib.E_ALIGN


def test_null_call_record():
    lib = _lib.load()
    assert lib.bsattn_paged_fwd(None, 16, 16, None, 0, 0, 0, 0.0, 16, 1 << 20, 16) == _lib.E_NULL
    assert lib.bsattn_paged_append(None, 16, 16, 16, (ctypes.c_int64 * 9)(), 16, None, 0, 0) == _lib.E_NULL


def test_error_code_has_a_text():
    assert "page" in _lib.strerror(_lib.E_PAGE)


def test_python_side():
    kp = torch.zeros(4, 2, 16, 128, dtype=torch.float16)
    table = torch.zeros(1, 4, dtype=torch.int32)
    lens = torch.ones(1, dtype=torch.int32)
    q = torch.zeros(1, 4, 1, 128, dtype=torch.float16)
    k = torch.zeros(1, 2, 1, 128, dtype=torch.float16)
    for call in (lambda: ub.paged_attn_fwd(q, kp, kp, table, lens),
                 lambda: ub.shared_prefix_attn_fwd(q, kp, kp, table, lens, prefix_len=16),
                 lambda: ub.paged_kv_append(kp, kp, table, lens, k, k)):
        with pytest.raises(ValueError, match="no CPU path"):
            call()
    with pytest.raises(TypeError):
        ub.paged_attn_fwd(q.float(), kp.float(), kp.float(), table, lens)
    with pytest.raises(ValueError):
        ub.paged_attn_fwd(q, kp[..., :64], kp[..., :64], table, lens)
    with pytest.raises(ValueError):
        ub.paged_attn_fwd(q[0], kp, kp, table, lens)
    with pytest.raises(ValueError, match="window"):
        ub.paged_attn_fwd(q, kp, kp, table, lens, window=0)
    with pytest.raises(ValueError, match="window"):
        ub.paged_attn_fwd(q, kp, kp, table, lens, global_blocks=1)
    for bad in (None, 3, kp.numpy()):
        with pytest.raises(TypeError, match="tensor"):
            ub.paged_attn_fwd(bad, kp, kp, table, lens)
        with pytest.raises(TypeError, match="tensor"):
            ub.paged_attn_fwd(q, kp, bad, table, lens)


def test_inv_freq():
    f = ub.rope_inv_freq(64, 10000.0, "cpu")
    assert f.dtype == torch.float64 and f.shape == (32,)
    assert f[0] == 1.0 and abs(f[16].item() - 0.01) < 1e-15
