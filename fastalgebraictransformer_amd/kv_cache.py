"""Operators over a key / value cache beside the plain decode.

Extensions beyond the reference API, for serving: the attention of a tree of
drafted tokens (speculative decoding), and a cache bounded by the attention
weight its keys have received -- collected over a prompt
(``rational_attention_key_weights``) and over each decoded token
(``rational_attention_decode_accumulate``), and used to evict
(``kv_cache_evict``). ``generate(cache_keep=...)`` and ``forward_tree`` of the
model use them. CUDA tensors only; no gradients. The launches go to the
``kat_attn_tree``, ``kat_attn_decode_accum``, ``kat_attn_key_weights`` and
``kat_kv_evict`` entry points of libkat.so on the current stream of the
tensors' device, and can be captured in a HIP graph.

Caches are [B, H, T, D] with any (b, h, t) strides and a unit last-dim stride
(e.g. permuted views of token-major [B, T, H, D] buffers), rows 16-byte
aligned; ``positions`` are int32 and ``weights`` fp32, [B, H, T].
"""

import torch

from . import _lib
from .forward import _bht_strides, _key_mask_arg, _unit_d
from .fused_ops import EPS

MAX_TREE = 64  # drafted tokens per call


def _slopes_arg(alibi_slopes, q):
    s = alibi_slopes.to(device=q.device, dtype=torch.float32).contiguous()
    assert s.numel() == q.shape[1], "alibi_slopes must have n_heads entries"
    return s


def _lengths_arg(lengths, q):
    if lengths is None:
        return None
    n = lengths.to(device=q.device, dtype=torch.int32).contiguous()
    assert n.numel() == q.shape[0], "lengths must have B entries"
    return n


def _unit_t(t):
    return t if t.shape[-1] <= 1 or t.stride(-1) == 1 else t.contiguous()


def _positions_arg(positions, B, H, T, q):
    if positions is None:
        return None
    assert tuple(positions.shape) == (B, H, T), f"positions must be [B, H, T] = [{B}, {H}, {T}]"
    return _unit_t(positions.to(device=q.device, dtype=torch.int32))


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(nbytes, q):
    return torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None


def _check_rows(name, t, shape, dtype, device):
    """A tensor that a kernel writes in place: it cannot be converted."""
    assert tuple(t.shape) == shape, f"{name} must be {list(shape)}"
    assert t.dtype == dtype and t.device == device, f"{name} must be {dtype} on {device}"
    assert t.shape[-1] <= 1 or t.stride(-1) == 1, f"{name} must have a unit last-dim stride"
    for size, stride in zip(t.shape[:-1], t.stride()[:-1]):
        assert size <= 1 or stride >= t.shape[-1], f"{name} must not overlap itself"


def rational_attention_tree(q, k_cache, v_cache, alibi_slopes, scale, parents, lengths=None,
                            positions=None, eps=EPS):
    """Attention of N drafted tokens per batch row over a KV cache and, among
    themselves, each over its own ancestors: the pass that scores every branch
    of a speculative draft at once.

    q: [B, H, N, D], N <= 64; k_cache, v_cache: [B, H, T, D], of whose first
    ``lengths[b]`` rows (int32 [B] on the device, default T) the last N hold the
    drafted tokens' keys and values. ``parents`` (int32 [B, N], or [N] for all
    rows): the token that token i hangs on (less than i), -1 for the context;
    any other value marks an absent token, and tokens below one are absent too.
    A token sees the context, itself and its ancestors. ALiBi distances count
    along the branch: a token sits ``depth`` positions past the context; with
    ``positions`` (int32 [B, H, T], caches with evicted rows) they are
    differences of the rows' positions. Absent tokens, and rows with fewer than
    N keys cached, give zeros. Rows a token does not see may hold anything.

    Returns (out [B, H, N, D] in q's dtype and row order, L [B, H, N] fp32
    without eps). With N = 1 and parents -1 it is rational_attention_decode."""
    r = _lib.ops().tree(q, k_cache, v_cache, alibi_slopes, scale, parents, lengths, positions, eps)
    if r is not None:
        return r
    assert q.is_cuda and k_cache.is_cuda and v_cache.is_cuda
    B, H, N, D = q.shape
    T = k_cache.shape[2]
    assert tuple(k_cache.shape) == (B, H, T, D) and tuple(v_cache.shape) == (B, H, T, D)
    assert N <= MAX_TREE, f"at most {MAX_TREE} drafted tokens"
    assert tuple(parents.shape) in ((N,), (B, N)), f"parents must be [N] or [B, N] = [{B}, {N}]"
    lib = _lib.load()
    q, k, v = _unit_d(q), _unit_d(k_cache.to(q.dtype)), _unit_d(v_cache.to(q.dtype))
    slopes = _slopes_arg(alibi_slopes, q)
    parents = _unit_t(parents.to(device=q.device, dtype=torch.int32))
    lengths = _lengths_arg(lengths, q)
    positions = _positions_arg(positions, B, H, T, q)
    out = torch.empty((B, H, N, D), dtype=q.dtype, device=q.device)
    L = torch.empty((B, H, N), dtype=torch.float32, device=q.device)
    code = _lib.dtype_code(q)
    strides = _lib.i64_array(_bht_strides(q) + _bht_strides(k) + _bht_strides(v) + _bht_strides(out))
    ps = _lib.i64_array(positions.stride()[:2] if positions is not None else (0, 0))
    with torch.cuda.device(q.device):
        nbytes = lib.kat_attn_tree_workspace_size(B, H, N, T, D, code)
        ws = _workspace(nbytes, q)
        _lib.check(lib.kat_attn_tree(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                     L.data_ptr(), slopes.data_ptr(), parents.data_ptr(),
                                     parents.stride(0) if parents.dim() == 2 else 0, _ptr(lengths),
                                     _ptr(positions), ps, _ptr(ws), nbytes, B, H, N, T, D, strides,
                                     float(scale), float(eps), code, _lib.stream(q)),
                   "kat_attn_tree")
    return out, L


def rational_attention_decode_accumulate(q, k_cache, v_cache, alibi_slopes, scale, weights,
                                         lengths=None, positions=None, eps=EPS):
    """rational_attention_decode that also adds the attention weights to the
    keys' running totals: ``weights`` (fp32 [B, H, T]) gains f_j / (L + eps) at
    the filled rows j < lengths[b], in place.

    With ``positions`` (int32 [B, H, T]) the query's distance to row j is
    positions[lengths[b] - 1] - positions[j], for caches whose rows have been
    evicted; without, rows are positions. Other arguments, types and head dims
    as rational_attention_decode. Returns (out [B, H, D], L [B, H])."""
    r = _lib.ops().decode_accumulate(q, k_cache, v_cache, alibi_slopes, scale, weights, lengths,
                                     positions, eps)
    if r is not None:
        return r
    assert q.is_cuda and k_cache.is_cuda and v_cache.is_cuda
    B, H, D = q.shape
    T = k_cache.shape[2]
    assert tuple(k_cache.shape) == (B, H, T, D) and tuple(v_cache.shape) == (B, H, T, D)
    _check_rows("weights", weights, (B, H, T), torch.float32, q.device)
    lib = _lib.load()
    q, k, v = _unit_d(q), _unit_d(k_cache.to(q.dtype)), _unit_d(v_cache.to(q.dtype))
    slopes = _slopes_arg(alibi_slopes, q)
    lengths = _lengths_arg(lengths, q)
    positions = _positions_arg(positions, B, H, T, q)
    out = torch.empty((B, H, D), dtype=q.dtype, device=q.device)
    L = torch.empty((B, H), dtype=torch.float32, device=q.device)
    code = _lib.dtype_code(q)
    strides = _lib.i64_array((q.stride(0), q.stride(1)) + _bht_strides(k) + _bht_strides(v) +
                             (out.stride(0), out.stride(1)))
    wp = _lib.i64_array(weights.stride()[:2] + (positions.stride()[:2] if positions is not None
                                                else (0, 0)))
    with torch.cuda.device(q.device):
        nbytes = lib.kat_attn_decode_accum_workspace_size(B, H, max(T, 1), D, code)
        ws = _workspace(nbytes, q)
        _lib.check(lib.kat_attn_decode_accum(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                             out.data_ptr(), L.data_ptr(), slopes.data_ptr(),
                                             weights.data_ptr(), _ptr(lengths), _ptr(positions), wp,
                                             _ptr(ws), nbytes, B, H, T, D, strides, float(scale),
                                             float(eps), code, _lib.stream(q)),
                   "kat_attn_decode_accum")
    return out, L


def rational_attention_key_weights(q, k, alibi_slopes, scale, L, key_mask=None, last=None, eps=EPS):
    """The attention weight that each key of a prompt receives, summed over its
    queries: w[b, h, j] = sum over i >= j of f_ij / (L_i + eps), fp32 [B, H, T].

    q, k: [B, H, T, D] as the causal forward took them, L [B, H, T] the row sums
    it returned (rational_attention_forward). ``last``: only the last ``last``
    queries count (default all). ``key_mask`` ([B, T], 0 drops a token): a
    dropped token neither gives nor receives weight; L is then the masked
    attention's."""
    assert last is None or last >= 1, "last must be at least 1"
    n = 0 if last is None else min(int(last), 1 << 40)
    r = _lib.ops().key_weights(q, k, alibi_slopes, scale, L, key_mask, n, eps)
    if r is not None:
        return r
    assert q.is_cuda and k.is_cuda and L.is_cuda
    assert q.shape == k.shape and tuple(L.shape) == tuple(q.shape[:3])
    B, H, T, D = q.shape
    assert key_mask is None or tuple(key_mask.shape) == (B, T), f"key_mask must be [B, T] = [{B}, {T}]"
    lib = _lib.load()
    q, k = _unit_d(q), _unit_d(k.to(q.dtype))
    L = L.to(device=q.device, dtype=torch.float32)
    slopes = _slopes_arg(alibi_slopes, q)
    mask = _key_mask_arg(key_mask, B, T, q.device)
    w = torch.empty((B, H, T), dtype=torch.float32, device=q.device)
    code = _lib.dtype_code(q)
    strides = _lib.i64_array(_bht_strides(q) + _bht_strides(k) + _bht_strides(L) + w.stride()[:2])
    with torch.cuda.device(q.device):
        nbytes = lib.kat_attn_key_weights_workspace_size(B, H, T, D, n, code)
        ws = _workspace(nbytes, q)
        _lib.check(lib.kat_attn_key_weights(q.data_ptr(), k.data_ptr(), L.data_ptr(), w.data_ptr(),
                                            slopes.data_ptr(), _ptr(mask), T, _ptr(ws), nbytes, B,
                                            H, T, D, n, strides, float(scale), float(eps), code,
                                            _lib.stream(q)), "kat_attn_key_weights")
    return w


def kv_cache_evict(k_cache, v_cache, weights, positions, lengths, keep, recent=0, out=None):
    """Keep at most ``keep`` rows of every (batch, head) of a cache: the rows
    whose positions are among the newest ``recent`` (above positions[n - 1] -
    recent, n = lengths[b]), then those with the largest ``weights``, ties to the
    lower row; a NaN weight ranks above every number. ``lengths`` (int32 [B])
    may be None for full caches, except in place.

    In place (``out`` None): the kept rows of all four tensors end in rows 0 ..
    min(n, keep) - 1, those already there staying where they are (so rows are
    not in the order of their positions afterwards), and ``lengths`` becomes
    min(n, keep). With ``out`` = (k, v, weights, positions, lengths) of another
    cache with at least ``keep`` rows, the kept rows go there in their order and
    the inputs stay as they are (out's ``lengths`` too is another tensor than the
    one given); rows behind them are left alone.
    Returns the five tensors that hold the result."""
    if out is not None:
        out = tuple(out)
        assert len(out) == 5, "out must be (k, v, weights, positions, lengths)"
    res = (k_cache, v_cache, weights, positions, lengths) if out is None else out
    if _lib.ops().evict(k_cache, v_cache, weights, positions, lengths, out, keep, recent):
        return res
    assert k_cache.is_cuda and v_cache.is_cuda
    B, H, T, D = k_cache.shape
    assert tuple(v_cache.shape) == (B, H, T, D) and v_cache.dtype == k_cache.dtype
    assert 0 <= recent <= keep, "recent must lie in [0, keep]"
    assert out is not None or lengths is not None, "an eviction in place updates lengths"
    dev, dt, S = k_cache.device, k_cache.dtype, res[0].shape[2]
    _lib.dtype_code(k_cache)
    # what is written cannot be converted
    for name, t, shape, dtype in (("k", res[0], (B, H, S, D), dt), ("v", res[1], (B, H, S, D), dt),
                                  ("weights", res[2], (B, H, S), torch.float32),
                                  ("positions", res[3], (B, H, S), torch.int32),
                                  ("lengths", res[4], (B,), torch.int32)):
        _check_rows(name if out is None else f"out's {name}", t, shape, dtype, dev)
    assert S >= min(keep, T), "out must have room for the kept rows"
    if B * H * T * D == 0:  # nothing to move
        res[4].zero_()
        return res
    if out is not None:
        assert tuple(weights.shape) == (B, H, T), f"weights must be [B, H, T] = [{B}, {H}, {T}]"
        k_cache, v_cache = _unit_d(k_cache), _unit_d(v_cache.to(dev))
        weights = _unit_t(weights.to(device=dev, dtype=torch.float32))
        positions = _positions_arg(positions, B, H, T, k_cache)
        lengths = _lengths_arg(lengths, k_cache)
    if not _lib.ops().evict(k_cache, v_cache, weights, positions, lengths, out, keep, recent):
        raise RuntimeError("kv_cache_evict takes plain CUDA tensors only")
    return res
