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


# ------------------------------------------------- the oracle's own pins ----

def test_oracle_rows_and_weights_are_those_of_the_attention():
    import oracle as O
    from oracle import cache as C
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 2, 23, 8, generator=g, dtype=torch.float64) for _ in range(3))
    slopes = F.compute_alibi_slopes(2)
    o, L = O.attention_fwd(q, k, v, slopes, 0.3)
    for h in range(2):
        cols = torch.zeros(23, dtype=torch.float64)
        for i in (0, 7, 22):
            dist = i - torch.arange(i + 1)
            ro, rL, p, A, E = C.attention_rows(q[0, h, i], k[0, h, :i + 1], v[0, h, :i + 1], slopes[h], 0.3, dist)
            assert float((ro - o[0, h, i]).abs().max()) <= 1e-12 and abs(float(rL - L[0, h, i])) <= 1e-12
            assert 0 < E < 1e-3 and bool((A >= ro.abs() - 1e-12).all())
            cols[:i + 1] += p
        w = sum(C.key_weights(q[0, h, :i + 1], k[0, h, :i + 1], slopes[h], 0.3, L[0, h, :i + 1], None, 1)[0].new_zeros(23)
                .index_add(0, torch.arange(i + 1), C.key_weights(q[0, h, :i + 1], k[0, h, :i + 1], slopes[h], 0.3,
                                                                 L[0, h, :i + 1], None, 1)[0]) for i in (0, 7, 22))
        assert float((w - cols).abs().max()) <= 1e-12
        total, _ = C.key_weights(q[0, h], k[0, h], slopes[h], 0.3, L[0, h], None, None)
        assert abs(float(total.sum()) - 23) <= 23 * 1e-4  # every query hands out L / (L + eps)


def test_oracle_trees_and_evictions():
    from oracle import cache as C
    assert C.tree_lines([-1, 0, 0, 2, -1, 7, 4, -2, 7, 9]) == [[0], [0, 1], [0, 2], [0, 2, 3], [4], None, [4, 6],
                                                               None, None, None]
    pos = [0, 1, 2, 3, 4, 5]
    assert C.evict_rows([3.0, 1.0, 3.0, 0.0, 2.0, 0.0], pos, 6, 3, 0) == [0, 2, 4]
    assert C.evict_rows([3.0, 1.0, 3.0, 0.0, 2.0, 0.0], pos, 6, 3, 2) == [0, 4, 5]
    assert C.evict_rows([3.0, 3.0, 3.0, 0.0], pos, 4, 2, 0) == [0, 1]           # ties: the lower row
    assert C.evict_rows([3.0, float("nan"), 4.0, 0.0], pos, 4, 2, 0) == [1, 2]  # a NaN above every number
    assert C.evict_rows([3.0, 1.0], pos, 2, 5, 1) == [0, 1]


@pytest.mark.parametrize("B,H,T", [(1, 1, 1), (16, 16, 4096), (1, 8, 100000)])
def test_workspaces_are_bounded(B, H, T):
    # the partial sums of a call stay a small part of the cache it reads
    lib = _lib.load()
    cache = 2 * B * H * T * 128 * 2
    assert lib.kat_attn_tree_workspace_size(B, H, 64, T, 128, 1) <= max(cache, 64 << 20)
    assert lib.kat_attn_decode_accum_workspace_size(B, H, T, 128, 1) <= max(cache // 8, 8 << 20)
    assert lib.kat_attn_key_weights_workspace_size(B, H, T, 128, 64, 1) <= max(cache // 8, 8 << 20)


@pytest.mark.parametrize("dtype", [None, torch.bfloat16, torch.float16])
def test_depths_of_drafted_tokens_under_autocast(dtype):
    from fastalgebraictransformer_amd.algebraic_model import AlgebraicTransformerLM
    g = torch.Generator().manual_seed(0)
    chain = torch.arange(64) - 1
    tree = torch.tensor([-1] + [int(torch.randint(-1, i, (1,), generator=g)) for i in range(1, 64)])
    parents = torch.stack((chain, tree, torch.full((64,), -1))).to(torch.int32)
    want = torch.zeros_like(parents)
    for b in range(3):
        for i in range(64):
            want[b, i] = 0 if parents[b, i] < 0 else want[b, int(parents[b, i])] + 1
    with torch.autocast("cpu", dtype=dtype or torch.bfloat16, enabled=dtype is not None):
        got = AlgebraicTransformerLM._depths(parents)
    assert torch.equal(got, want.long())
