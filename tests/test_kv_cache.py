"""Argument checks of the operators over a key / value cache (CPU only: nothing
here launches a kernel)."""

import ctypes

import pytest
import torch

import fastalgebraictransformer_amd as F
from fastalgebraictransformer_amd import _lib

P = ctypes.c_void_p(16)


def _msg():
    return _lib.load().kat_last_error().decode()


def test_cpu_tensors_are_refused():
    q, kv = torch.zeros(1, 2, 8), torch.zeros(1, 2, 5, 8)
    s = torch.ones(2)
    with pytest.raises(AssertionError):
        F.rational_attention_tree(kv, kv, kv, s, 1.0, torch.zeros(5, dtype=torch.int32))
    with pytest.raises(AssertionError):
        F.rational_attention_decode_accumulate(q, kv, kv, s, 1.0, torch.zeros(1, 2, 5))
    with pytest.raises(AssertionError):
        F.rational_attention_key_weights(kv, kv, s, 1.0, torch.zeros(1, 2, 5))
    with pytest.raises(AssertionError):
        F.kv_cache_evict(kv, kv, torch.zeros(1, 2, 5), torch.zeros(1, 2, 5, dtype=torch.int32),
                         torch.zeros(1, dtype=torch.int32), 3)


def _tree(N=4, T=9, D=64, dtype=1, strides=None, ws=0, parents=P, esz=2):
    lib = _lib.load()
    st = _lib.i64_array(strides or [64] * 12)
    return lib.kat_attn_tree(P, P, P, P, None, P, parents, N, None, None, None, None, ws, 1, 2, N, T, D, st,
                             1.0, 1e-6, dtype, None)


def test_tree_refusals():
    assert _tree(N=65) == 2 and "65 tokens" in _msg()
    assert _tree(N=-1) == 1 and "negative" in _msg()
    assert _tree(D=264) == 2 and "head dim 264" in _msg()
    assert _tree(D=100) == 2 and _tree(D=64, dtype=3) == 2
    assert _tree(strides=[64] * 11 + [60]) == 2 and "aligned" in _msg()
    assert _tree(strides=[64] * 5 + [8] + [64] * 6) == 1 and "row stride" in _msg()
    assert _tree(parents=None) == 1 and "null" in _msg()
    assert _tree(N=0) == 0  # nothing to do
    # a long cache of few heads is split and needs its workspace
    assert _lib.load().kat_attn_tree_workspace_size(1, 2, 4, 5000, 64, 1) > 0
    assert _tree(T=5000) == 1 and "workspace" in _msg()
    assert _lib.load().kat_attn_tree_workspace_size(1, 2, 65, 5000, 64, 1) == 0


def test_accumulate_refusals():
    lib = _lib.load()

    def call(D=64, T=9, wp=True, weights=P, strides=None, ws=0):
        return lib.kat_attn_decode_accum(P, P, P, P, None, P, weights, None, None,
                                         _lib.i64_array([9, 9, 0, 0]) if wp else None, None, ws, 1, 2, T, D,
                                         _lib.i64_array(strides or [64] * 10), 1.0, 1e-6, 1, None)
    assert call(D=12) == 2 and "head dim 12" in _msg()
    assert call(weights=None) == 1 and call(wp=False) == 1 and "null" in _msg()
    assert call(T=-1) == 1 and call(T=1 << 30) == 2
    assert call(strides=[64] * 4 + [8] + [64] * 5) == 1 and "row stride" in _msg()
    # few rows take one launch and no workspace, a long cache of few heads does
    assert lib.kat_attn_decode_accum_workspace_size(1, 2, 9, 64, 1) == 0
    assert lib.kat_attn_decode_accum_workspace_size(1, 2, 5000, 64, 1) > 2 * 5000 * 4
    assert call(T=5000) == 1 and "workspace 0 bytes" in _msg()


def test_key_weights_refusals():
    lib = _lib.load()

    def call(D=64, T=9, L=P, last=0, strides=None, dtype=1):
        return lib.kat_attn_key_weights(P, P, L, P, P, None, 0, None, 0, 1, 2, T, D, last,
                                        _lib.i64_array(strides or [64] * 11), 1.0, 1e-6, dtype, None)
    assert call(D=20) == 2 and call(D=64, dtype=3) == 2
    assert call(D=260, dtype=0) == 2 and "head dim 260" in _msg()
    assert call(L=None) == 1 and call(last=-1) == 1
    assert call(T=0) == 0
    assert call(strides=[64, 64, 1 << 25] + [64] * 8) == 2 and "stride too large" in _msg()
    assert lib.kat_attn_key_weights_workspace_size(1, 1, 4096, 64, 0, 1) > 0
    assert call(T=4096) == 1 and "workspace" in _msg()


def test_evict_refusals():
    lib = _lib.load()

    def call(D=64, keep=4, recent=0, in_place=0, out=ctypes.c_void_p(32), dtype=1, ws=0, T=9):
        return lib.kat_kv_evict(P, P, P, P, None, out, out, out, out, None, P if ws else None, ws, 1, 2, T, D, keep,
                                recent, in_place, _lib.i64_array([64] * 20), dtype, None)
    assert call(recent=5) == 1 and "recent 5" in _msg()
    assert call(D=12) == 2 and "16-byte pieces" in _msg()
    assert call(dtype=9) == 2 and call(keep=-1) == 1
    assert call(in_place=1) == 1 and "in place" in _msg()
    assert call(out=None) == 1 and "null" in _msg()
    assert call(T=0) == 0
    assert call(in_place=1, out=P) == 1 and "workspace" in _msg()
    assert lib.kat_kv_evict(P, P, P, P, P, P, P, P, P, P, None, 0, 1, 2, 9, 64, 4, 0, 0, _lib.i64_array([64] * 20), 1,
                            None) == 1 and "lengths_out" in _msg()
    assert lib.kat_kv_evict_workspace_size(2, 3, 10) == 6 * 21 * 4
