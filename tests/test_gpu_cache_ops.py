"""The operators over a key / value cache (kv_cache.py) against their
definitions in 64 bits (oracle/cache.py).

Tolerances, derived before any run. u = finfo.eps / 2 of the tensors' type. An
attention output o = sum p v is off by at most
    (2 E + r) A + u |o| + floor,   A = sum p |v|,
E the relative error of an fp32 weight (the oracle's bound; once in the
products and once in L), r = u^2 for 16-bit types, whose weights enter the
product of a tree as a rounded value and the rounded rest, and 0 for fp32; fp16
weights below its normal range (16 f < 2^-14) are off by 2^-25 absolutely, so
floor = 2^-25 sum |v| / (16 (L + eps)). L is off by E L, a weight p by 2 E p + u32 p."""

import math

import pytest
import torch

import fastalgebraictransformer_amd as F
from oracle import cache as C

pytestmark = pytest.mark.gpu
dev = "cuda"
U32 = C.U32


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def rand(shape, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(dev)


def caches(B, H, T, D, dtype, seed):
    """Token-major caches [B, T, H, D] as [B, H, T, D] views."""
    return (rand((B, T, H, D), dtype, seed).permute(0, 2, 1, 3),
            rand((B, T, H, D), dtype, seed + 1).permute(0, 2, 1, 3))


def positions_like(B, H, T, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(1, 4, (B, H, T), generator=g).cumsum(-1).to(torch.int32).to(dev)


def check_out(got, ref, A, E, v, L, dtype, what, product_rounds):
    u = unit(dtype)
    tol = (2 * E + (u * u if product_rounds and dtype != torch.float32 else 0.0)) * A + u * ref.abs() + 1e-30
    if dtype == torch.float16 and product_rounds:
        tol = tol + 2.0 ** -25 * v.double().cpu().abs().sum(0) / (16 * (float(L) + 1e-6))
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25  # the output's own subnormal spacing
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: {float((err - tol).max()):.3e} past the bound, err {float(err.max()):.3e}"


DIMS = [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.bfloat16, 256), (torch.float16, 128),
        (torch.float16, 200), (torch.bfloat16, 8), (torch.bfloat16, 96), (torch.float32, 32),
        (torch.float32, 64), (torch.float32, 128), (torch.float32, 20), (torch.float32, 100)]


# ------------------------------------------------------------------- tree ----

def random_parents(B, N, seed, absent=False):
    g = torch.Generator().manual_seed(seed)
    p = ((torch.rand(B, N, generator=g) * (torch.arange(N) + 1)).floor() - 1).to(torch.int32)
    if absent:  # padding, a parent that is not before its token, one out of range
        bad = torch.rand(B, N, generator=g) < 0.15
        p = torch.where(bad, torch.randint(-5, N + 70, (B, N), generator=g).to(torch.int32), p)
    return p


def check_tree(o, L, q, k, v, slopes, scale, parents, lengths, positions, what=""):
    B, H, N, D = q.shape
    T = k.shape[2]
    qc, kc, vc = q.cpu(), k.cpu(), v.cpu()
    for b in range(B):
        n = T if lengths is None else min(int(lengths[b]), T)
        lines = C.tree_lines((parents[b] if parents.dim() == 2 else parents).tolist())
        c = n - N
        for h in range(H):
            for i in range(N):
                where = f"{what} b={b} h={h} i={i}"
                if c < 0 or lines[i] is None:
                    assert bool((o[b, h, i] == 0).all()) and float(L[b, h, i]) == 0, where
                    continue
                rows = torch.tensor(list(range(c)) + [c + j for j in lines[i]])
                at = torch.arange(c + len(lines[i])) if positions is None else positions[b, h].cpu()[rows]
                ro, rL, _, A, E = C.attention_rows(qc[b, h, i], kc[b, h][rows], vc[b, h][rows], slopes[h],
                                                   scale, at[-1] - at, fused=q.dtype != torch.float32)
                assert abs(float(L[b, h, i]) - float(rL)) <= E * float(rL), where
                check_out(o[b, h, i], ro, A, E, vc[b, h][rows], rL, q.dtype, where, True)


@pytest.mark.parametrize("N", [1, 7, 16, 33, 64])
@pytest.mark.parametrize("dtype,D", DIMS)
def test_tree_matches_definition(gpu, dtype, D, N):
    B, H, T = 2, 2, 150
    k, v = caches(B, H, T, D, dtype, D + N)
    q = rand((B, N, H, D), dtype, D + N + 2).permute(0, 2, 1, 3)
    parents = random_parents(B, N, N)
    lengths = torch.tensor([T, N + 5], dtype=torch.int32)
    slopes = F.compute_alibi_slopes(H)
    scale = 1.0 / math.sqrt(D)
    o, L = F.rational_attention_tree(q, k, v, slopes.to(dev), scale, parents.to(dev), lengths=lengths.to(dev))
    torch.cuda.synchronize()
    assert o.shape == q.shape and o.dtype == dtype and L.shape == (B, H, N)
    check_tree(o, L, q, k, v, slopes, scale, parents, lengths, None)


@pytest.mark.parametrize("n", [5, 37, 64, 65, 700])
@pytest.mark.parametrize("dtype,D,N", [(torch.bfloat16, 64, 5), (torch.float32, 64, 20), (torch.float16, 128, 37)])
def test_tree_lengths_positions_and_absent_tokens(gpu, dtype, D, N, n):
    B, H, T = 3, 2, 701
    k, v = caches(B, H, T, D, dtype, n)
    q = rand((B, H, N, D), dtype, n + 2)
    parents = random_parents(B, N, n, absent=True)
    lengths = torch.tensor([n, 0, N - 1 if n % 2 else 10 ** 6], dtype=torch.int32)
    slopes = F.compute_alibi_slopes(H)
    pos = positions_like(B, H, T, n)
    for positions in (None, pos):
        o, L = F.rational_attention_tree(q, k, v, slopes.to(dev), 0.11, parents.to(dev),
                                         lengths=lengths.to(dev), positions=positions)
        torch.cuda.synchronize()
        check_tree(o, L, q, k, v, slopes, 0.11, parents, lengths, positions, f"positions={positions is not None}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_tree_ignores_what_a_token_does_not_see(gpu, dtype):
    # rows of absent tokens, of other branches and past the filled ones hold
    # inf and NaN; the tokens that do not see them get the same results
    B, H, T, D, N = 1, 2, 200, 64, 12
    parents = torch.tensor([-1, 0, 0, 1, 2, -1, 5, -3, 7, 4, 3, 6], dtype=torch.int32)
    lengths = torch.tensor([170], dtype=torch.int32)
    c = 170 - N
    k, v = caches(B, H, T, D, dtype, 1)
    q = rand((B, H, N, D), dtype, 3)
    slopes = F.compute_alibi_slopes(H)
    args = (slopes.to(dev), 0.125, parents.to(dev))
    o, L = F.rational_attention_tree(q, k, v, *args, lengths=lengths.to(dev))
    k2, v2, q2 = k.clone(), v.clone(), q.clone()
    for j, x in ((7, float("nan")), (8, float("inf")), (6, float("-inf"))):
        k2[:, :, c + j] = x
        v2[:, :, c + j] = x
    q2[:, :, 7:9] = float("nan")
    k2[:, :, 170:] = float("nan")
    v2[:, :, 170:] = float("nan")
    o2, L2 = F.rational_attention_tree(q2, k2, v2, *args, lengths=lengths.to(dev))
    torch.cuda.synchronize()
    clean = [i for i in range(N) if i not in (6, 11)]  # 11 hangs on 6
    assert bool(torch.isfinite(o2[:, :, clean]).all())
    assert torch.equal(L2[:, :, clean], L[:, :, clean])
    check_tree(o2[:, :, :6], L2[:, :, :6], q[:, :, :6], torch.cat((k[:, :, :c], k[:, :, c:c + 6]), 2),
               torch.cat((v[:, :, :c], v[:, :, c:c + 6]), 2), slopes, 0.125, parents[:6], None, None)
    assert float(o2[:, :, 7:9].abs().max()) == 0
    assert not bool(torch.isfinite(o2[:, :, 6]).any())  # it sees its own row


def test_tree_of_one_token_is_the_decode(gpu):
    B, H, T, D = 3, 4, 513, 128
    k, v = caches(B, H, T, D, torch.bfloat16, 5)
    q = rand((B, H, D), torch.bfloat16, 6)
    slopes = F.compute_alibi_slopes(H).to(dev)
    lengths = torch.tensor([513, 1, 77], dtype=torch.int32, device=dev)
    a, la = F.rational_attention_decode(q, k, v, slopes, 0.09, lengths=lengths)
    root = torch.full((1,), -1, dtype=torch.int32, device=dev)
    b, lb = F.rational_attention_tree(q[:, :, None], k, v, slopes, 0.09, root, lengths=lengths)
    torch.cuda.synchronize()
    assert torch.allclose(la, lb[:, :, 0], rtol=1e-5)
    # each is off by (u + E) A + u |o|; A <= 4 here (|v| <= 4.5 or so)
    assert float((a - b[:, :, 0]).abs().max()) <= 4 * 2.0 ** -8 * 4


def test_tree_chain_is_the_causal_attention(gpu):
    # a chain of drafted tokens is a piece of the causal prompt
    B, H, T, D, N = 2, 3, 300, 64, 31
    q, k, v = (rand((B, H, T, D), torch.float32, s) for s in (1, 2, 3))
    slopes = F.compute_alibi_slopes(H).to(dev)
    o, L = F.rational_attention_forward(q, k, v, slopes, 0.125)
    chain = torch.arange(-1, N - 1, dtype=torch.int32, device=dev)
    ot, Lt = F.rational_attention_tree(q[:, :, T - N:], k, v, slopes, 0.125, chain)
    torch.cuda.synchronize()
    assert float((ot - o[:, :, T - N:]).abs().max()) <= 2e-5 * float(o.abs().max())
    assert torch.allclose(Lt, L[:, :, T - N:], rtol=2e-5)


def test_tree_long_cache_splits_and_is_deterministic(gpu):
    B, H, T, D, N = 1, 2, 9001, 128, 48
    k, v = caches(B, H, T, D, torch.bfloat16, 11)
    q = rand((B, H, N, D), torch.bfloat16, 12)
    parents = random_parents(B, N, 13)
    slopes = F.compute_alibi_slopes(H)
    run = lambda: F.rational_attention_tree(q, k, v, slopes.to(dev), 0.088, parents.to(dev))
    o, L = run()
    o2, L2 = run()
    torch.cuda.synchronize()
    assert torch.equal(o, o2) and torch.equal(L, L2)
    check_tree(o, L, q, k, v, slopes, 0.088, parents, None, None)


@pytest.mark.parametrize("N", [9, 30, 61])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 256),
                                     (torch.float32, 32), (torch.float32, 64), (torch.float32, 128)])
def test_tree_of_full_grids(gpu, dtype, D, N):
    # more heads than blocks fit: one block takes all its tiles, many times round
    # its ring; three (b, h) checked
    B, H, T = 33, 16, 700
    k, v = caches(B, H, T, D, dtype, N)
    q = rand((B, N, H, D), dtype, N + 2).permute(0, 2, 1, 3)
    parents = random_parents(B, N, N)
    lengths = torch.randint(T - 300, T + 1, (B,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    slopes = F.compute_alibi_slopes(H)
    for positions in (None, positions_like(B, H, T, N)):
        o, L = F.rational_attention_tree(q, k, v, slopes.to(dev), 0.09, parents.to(dev), lengths=lengths.to(dev),
                                         positions=positions)
        torch.cuda.synchronize()
        for b, h in ((0, 0), (17, 5), (B - 1, H - 1)):
            one = lambda t: t[b:b + 1, h:h + 1]
            check_tree(one(o), one(L), one(q), one(k), one(v), slopes[h:h + 1], 0.09, parents[b:b + 1],
                       lengths[b:b + 1], None if positions is None else one(positions))


# ------------------------------------------------------------- accumulate ----

def check_accumulate(o, L, total, old, q, k, v, slopes, scale, lengths, positions):
    B, H, D = q.shape
    T = k.shape[2]
    qc, kc, vc = q.cpu(), k.cpu(), v.cpu()
    for b in range(B):
        n = T if lengths is None else max(0, min(int(lengths[b]), T))
        for h in range(H):
            at = torch.arange(n) if positions is None else positions[b, h, :n].cpu()
            dist = at[-1] - at if n else at
            ro, rL, p, A, E = C.attention_rows(qc[b, h], kc[b, h, :n], vc[b, h, :n], slopes[h], scale, dist)
            assert abs(float(L[b, h]) - float(rL)) <= E * float(rL)
            check_out(o[b, h], ro, A, E, vc[b, h, :n], rL, q.dtype, f"b={b} h={h}", False)
            was = old[b, h].double().cpu()
            err = (total[b, h, :n].double().cpu() - was[:n] - p).abs()
            assert bool((err <= (2 * E + 4 * U32) * p + U32 * (was[:n].abs() + p)).all()), (b, h)
            assert torch.equal(total[b, h, n:].cpu(), old[b, h, n:].cpu())


@pytest.mark.parametrize("n", [1, 2, 63, 257, 1500])
@pytest.mark.parametrize("dtype,D", DIMS)
def test_accumulate_matches_definition(gpu, dtype, D, n):
    B, H, T = 3, 2, 1501
    k, v = caches(B, H, T, D, dtype, n + D)
    q = rand((B, H, D), dtype, n + D + 2)
    lengths = torch.tensor([n, 0, T + 5], dtype=torch.int32)
    slopes = F.compute_alibi_slopes(H)
    scale = 1.0 / math.sqrt(D)
    for positions in (None, positions_like(B, H, T, n)):
        # the totals are a view into a larger buffer
        buf = torch.rand(B, H + 1, T + 3, generator=torch.Generator().manual_seed(n)).to(dev)
        old = buf.clone()
        total = buf[:, :H, 1:T + 1]
        o, L = F.rational_attention_decode_accumulate(q, k, v, slopes.to(dev), scale, total,
                                                      lengths=lengths.to(dev), positions=positions)
        torch.cuda.synchronize()
        check_accumulate(o, L, total, old[:, :H, 1:T + 1], q, k, v, slopes, scale, lengths, positions)
        total.copy_(old[:, :H, 1:T + 1])
        assert torch.equal(buf, old)  # nothing outside the view


@pytest.mark.parametrize("n", [1, 31, 129])
@pytest.mark.parametrize("dtype,D", DIMS)
def test_accumulate_of_few_rows(gpu, dtype, D, n):
    # a block per (b, h), which finishes its totals itself
    B, H, T = 3, 2, 130
    k, v = caches(B, H, T, D, dtype, n + D)
    q = rand((B, H, D), dtype, n + D + 2)
    lengths = torch.tensor([n, 0, T + 5], dtype=torch.int32)
    slopes = F.compute_alibi_slopes(H)
    for positions in (None, positions_like(B, H, T, n)):
        total = torch.rand(B, H, T, generator=torch.Generator().manual_seed(n)).to(dev)
        old = total.clone()
        o, L = F.rational_attention_decode_accumulate(q, k, v, slopes.to(dev), 0.1, total,
                                                      lengths=lengths.to(dev), positions=positions)
        torch.cuda.synchronize()
        check_accumulate(o, L, total, old, q, k, v, slopes, 0.1, lengths, positions)


@pytest.mark.parametrize("dtype,D,T", [(torch.bfloat16, 64, 700), (torch.float16, 256, 300), (torch.float32, 128, 300),
                                       (torch.float16, 8, 8192), (torch.float16, 8, 8193)])
def test_accumulate_of_full_grids(gpu, dtype, D, T):
    # more heads than CUs: a block per (b, h) up to 8192 rows, chunks beyond; three
    # (b, h) checked
    B, H = 33, 16
    k, v = caches(B, H, T, D, dtype, T)
    q = rand((B, H, D), dtype, T + 2)
    lengths = torch.randint(T // 2, T + 1, (B,), generator=torch.Generator().manual_seed(1)).to(torch.int32)
    lengths[0] = T
    slopes = F.compute_alibi_slopes(H)
    total = torch.rand(B, H, T, generator=torch.Generator().manual_seed(T)).to(dev)
    old, positions = total.clone(), positions_like(B, H, T, T)
    o, L = F.rational_attention_decode_accumulate(q, k, v, slopes.to(dev), 0.1, total, lengths=lengths.to(dev),
                                                  positions=positions)
    torch.cuda.synchronize()
    for b, h in ((0, 0), (17, 5), (B - 1, H - 1)):
        one = lambda t: t[b:b + 1, h:h + 1]
        check_accumulate(one(o), one(L), one(total), one(old), one(q), one(k), one(v), slopes[h:h + 1], 0.1,
                         lengths[b:b + 1], one(positions))


def test_accumulate_agrees_with_decode_and_adds_up(gpu):
    B, H, T, D = 2, 4, 2000, 64
    k, v = caches(B, H, T, D, torch.bfloat16, 21)
    slopes = F.compute_alibi_slopes(H).to(dev)
    total = torch.zeros(B, H, T, device=dev)
    for step in range(3):
        q = rand((B, H, D), torch.bfloat16, 30 + step)
        o, L = F.rational_attention_decode_accumulate(q, k, v, slopes, 0.125, total)
        a, la = F.rational_attention_decode(q, k, v, slopes, 0.125)
        torch.cuda.synchronize()
        assert torch.allclose(L, la, rtol=1e-5)
        assert float((o - a).abs().max()) <= 2 * 2.0 ** -8 * float(a.abs().max())
    # every query hands out L / (L + eps)
    assert torch.allclose(total.sum(-1), torch.full((B, H), 3.0, device=dev), rtol=1e-4)


# ------------------------------------------------------------ key weights ----

@pytest.mark.parametrize("T", [1, 15, 64, 65, 333])
@pytest.mark.parametrize("dtype,D", DIMS + [(torch.float32, 256)])
def test_key_weights_match_definition(gpu, dtype, D, T):
    B, H = 2, 2
    qkv = rand((B, T, 3, H, D), dtype, T + D).permute(2, 0, 3, 1, 4)
    q, k, v = qkv[0], qkv[1], qkv[2]
    slopes = F.compute_alibi_slopes(H)
    scale = 1.0 / math.sqrt(D)
    _, L = F.rational_attention_forward(q, k, v, slopes.to(dev), scale)
    for last in (None, 1, 17):
        w = F.rational_attention_key_weights(q, k, slopes.to(dev), scale, L, last=last)
        torch.cuda.synchronize()
        assert w.shape == (B, H, T) and w.dtype == torch.float32
        for b in range(B):
            for h in range(H):
                ref, tol = C.key_weights(q[b, h].cpu(), k[b, h].cpu(), slopes[h], scale, L[b, h].cpu(), None, last)
                err = (w[b, h].double().cpu() - ref).abs()
                assert bool((err <= tol + 1e-30).all()), (b, h, last, float((err - tol).max()))


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)])
def test_key_weights_with_dropped_tokens(gpu, dtype, D):
    B, H, T = 3, 2, 201
    q, k = rand((B, H, T, D), dtype, 1), rand((B, H, T, D), dtype, 2)
    mask = torch.ones(B, T, dtype=torch.bool)
    mask[0, :130] = False                                    # left padding
    mask[1] = torch.rand(T, generator=torch.Generator().manual_seed(3)) < 0.5
    mask[2] = False                                          # no token at all
    slopes = F.compute_alibi_slopes(H)
    L = torch.rand(B, H, T, generator=torch.Generator().manual_seed(4)) + 0.5
    # whatever a dropped token holds is ignored
    q2, k2, L2 = q.clone(), k.clone(), L.clone()
    for b in range(B):
        q2[b, :, ~mask[b].to(dev)] = float("nan")
        k2[b, :, ~mask[b].to(dev)] = float("inf")
        L2[b, :, ~mask[b]] = float("nan")
    for last in (None, 70):
        w = F.rational_attention_key_weights(q2, k2, slopes.to(dev), 0.1, L2.to(dev), key_mask=mask.to(dev), last=last)
        torch.cuda.synchronize()
        for b in range(B):
            for h in range(H):
                ref, tol = C.key_weights(q[b, h].cpu(), k[b, h].cpu(), slopes[h], 0.1, L[b, h], mask[b], last)
                err = (w[b, h].double().cpu() - ref).abs()
                assert bool((err <= tol + 1e-30).all()), (b, h, last, float((err - tol).max()))
                assert float(w[b, h][~mask[b].to(dev)].abs().sum()) == 0


# one call per way a grid is laid out, at head dims that end in the third quarter of
# their layout's columns and at full ones
@pytest.mark.parametrize("dtype,B,H,T,D", [
    (torch.bfloat16, 6, 2, 200, 96), (torch.float16, 12, 4, 333, 40), (torch.float32, 6, 12, 256, 48),
    (torch.bfloat16, 6, 1, 1301, 80), (torch.float32, 6, 1, 1301, 96), (torch.float32, 18, 16, 130, 80),
    (torch.float16, 60, 12, 257, 128), (torch.bfloat16, 60, 12, 257, 192), (torch.float32, 6, 2, 300, 160),
    (torch.float32, 6, 2, 300, 256)])
def test_key_weights_with_runs_of_dropped_tokens(gpu, dtype, B, H, T, D):
    q, k = rand((B, H, T, D), dtype, 11), rand((B, H, T, D), dtype, 12)
    mask = torch.ones(B, T, dtype=torch.bool)
    for b in range(B):
        if b % 6 == 0: mask[b, :2 * T // 3] = False              # left padding
        elif b % 6 == 1: mask[b, T // 4:] = False                # right padding
        elif b % 6 == 2: mask[b, 5:T - 7] = False                # only the ends
        elif b % 6 == 3: mask[b, T // 5:T // 5 + 1 + 3 * T // 8] = False  # a hole
        elif b % 6 == 4: mask[b] = False
    slopes = F.compute_alibi_slopes(H)
    L = torch.rand(B, H, T, generator=torch.Generator().manual_seed(13)) + 0.5
    q2, k2, L2 = q.clone(), k.clone(), L.clone()
    for b in range(B):
        q2[b, :, ~mask[b].to(dev)] = float("inf")
        k2[b, :, ~mask[b].to(dev)] = float("nan")
        L2[b, :, ~mask[b]] = float("nan")
    for last in (None, T // 3):
        w = F.rational_attention_key_weights(q2, k2, slopes.to(dev), 0.1, L2.to(dev), key_mask=mask.to(dev), last=last)
        torch.cuda.synchronize()
        for b in range(6):
            for h in {0, H - 1}:
                ref, tol = C.key_weights(q[b, h].cpu(), k[b, h].cpu(), slopes[h], 0.1, L[b, h], mask[b], last)
                err = (w[b, h].double().cpu() - ref).abs()
                assert bool((err <= tol + 1e-30).all()), (b, h, last, float((err - tol).max()))
        assert float(w.masked_select(~mask.to(dev)[:, None].expand(B, H, T)).abs().sum()) == 0
        for b in range(6, B):  # the other rows: finite, and not zero where a query counts
            assert bool(torch.isfinite(w[b]).all())
            assert bool((w[b].sum(-1) > 0).all()) == bool(mask[b, T - (last or T):].any())


@pytest.mark.parametrize("B,H,T", [(1, 2, 2500), (8, 16, 700)])
def test_key_weights_of_split_and_full_grids(gpu, B, H, T):
    # grids that split the queries and grids that do not: rows add up to the
    # weight every query hands out
    D = 64
    q, k, v = (rand((B, H, T, D), torch.bfloat16, s) for s in (1, 2, 3))
    slopes = F.compute_alibi_slopes(H).to(dev)
    _, L = F.rational_attention_forward(q, k, v, slopes, 0.125)
    w = F.rational_attention_key_weights(q, k, slopes, 0.125, L)
    again = F.rational_attention_key_weights(q, k, slopes, 0.125, L)
    torch.cuda.synchronize()
    assert torch.equal(w, again)
    # the forward's own L may be off by 1e-4 of itself (fp32 sums, its sigma form)
    assert torch.allclose(w.sum(-1), torch.full((B, H), float(T), device=dev), rtol=2e-4)
    i = T // 2
    one = F.rational_attention_key_weights(q[:, :, :i + 1], k[:, :, :i + 1], slopes, 0.125, L[:, :, :i + 1], last=1)
    o, Ld = F.rational_attention_decode(q[:, :, i].contiguous(), k[:, :, :i + 1], v[:, :, :i + 1], slopes, 0.125)
    total = torch.zeros(B, H, i + 1, device=dev)
    F.rational_attention_decode_accumulate(q[:, :, i].contiguous(), k[:, :, :i + 1], v[:, :, :i + 1], slopes, 0.125, total)
    torch.cuda.synchronize()
    assert float((one - total).abs().max()) <= 2e-4 * float(total.max())


# ------------------------------------------------------------------ evict ----

def check_evict(old, new, n0, keep, recent, in_place, behind=None):
    """old, new: (k, v, weights, positions, lengths) before and after."""
    B, H = old[2].shape[:2]
    for b in range(B):
        n = max(0, min(n0[b], old[2].shape[2]))
        m = min(n, keep)
        assert int(new[4][b]) == m
        for h in range(H):
            rows = C.evict_rows(old[2][b, h].tolist(), old[3][b, h].tolist(), n, keep, recent)
            if in_place:  # the kept rows past m go, in order, where rows are given up
                movers, holes = [j for j in rows if j >= m], [j for j in range(m) if j not in rows]
                at = list(range(m))
                for d, s in zip(holes, movers):
                    at[d] = s
                rows = at
            rows = torch.tensor(rows, dtype=torch.long)
            for i, (x, y) in enumerate(zip(old[:4], new[:4])):
                assert torch.equal(y[b, h, :m].cpu().view(torch.uint8 if y.dtype == torch.bool else y.dtype),
                                   x[b, h].cpu()[rows]) or \
                    bool(torch.isnan(x[b, h].float()).any()) and torch.equal(
                        torch.nan_to_num(y[b, h, :m].cpu()), torch.nan_to_num(x[b, h].cpu()[rows])), (b, h, i)
                rest = (x if in_place else behind[i])[b, h].cpu()[m:]
                assert torch.equal(torch.nan_to_num(y[b, h].cpu()[m:]), torch.nan_to_num(rest)), (b, h, i)


def evict_case(B, H, T, D, dtype, seed, ties=False):
    g = torch.Generator().manual_seed(seed)
    k, v = caches(B, H, T, D, dtype, seed)
    w = torch.randn(B, H, T, generator=g).exp()
    if ties:  # few distinct totals, and zeros of both signs
        w = (w * 2).floor() * torch.where(torch.rand(B, H, T, generator=g) < 0.5, 1.0, -0.0)
    return k, v, w.to(dev), positions_like(B, H, T, seed), g


@pytest.mark.parametrize("T,keep,recent", [(1, 1, 0), (1, 0, 0), (70, 69, 0), (70, 8, 8), (333, 100, 20),
                                           (1024, 1, 1), (1025, 700, 64), (5000, 512, 100)])
@pytest.mark.parametrize("ties", [False, True])
def test_evict_matches_definition(gpu, T, keep, recent, ties):
    B, H, D = 3, 2, 64
    k, v, w, p, g = evict_case(B, H, T, D, torch.bfloat16, T + keep, ties)
    n0 = [T, max(0, keep - 1), T // 2]
    lengths = torch.tensor(n0, dtype=torch.int32, device=dev)
    old = [t.clone() for t in (k, v, w, p, lengths)]
    out = (torch.full((B, keep + 2, H, D), 7.0, dtype=k.dtype, device=dev).permute(0, 2, 1, 3),
           torch.full((B, keep + 2, H, D), 8.0, dtype=k.dtype, device=dev).permute(0, 2, 1, 3),
           torch.full((B, H, keep + 2), 9.0, device=dev),
           torch.full((B, H, keep + 2), 10, dtype=torch.int32, device=dev),
           torch.full((B,), -1, dtype=torch.int32, device=dev))
    behind = [t.clone() for t in out]
    res = F.kv_cache_evict(k, v, w, p, lengths, keep, recent=recent, out=out)
    torch.cuda.synchronize()
    assert all(a is b for a, b in zip(res, out))
    check_evict(old, res, n0, keep, recent, False, behind)
    assert all(torch.equal(a, b) for a, b in zip(old, (k, v, w, p, lengths)))
    res = F.kv_cache_evict(k, v, w, p, lengths, keep, recent=recent)
    torch.cuda.synchronize()
    check_evict(old, res, n0, keep, recent, True)


@pytest.mark.parametrize("T", [20000, 33000, 70000])
def test_evict_long_caches(gpu, T):
    # every form of the selection's key storage (held in registers, or not)
    B, H, D, keep = 1, 2, 16, 1000
    k, v, w, p, _ = evict_case(B, H, T, D, torch.float16, T, ties=T > 60000)
    lengths = torch.tensor([T - 3], dtype=torch.int32, device=dev)
    old = [t.clone() for t in (k, v, w, p, lengths)]
    res = F.kv_cache_evict(k, v, w, p, lengths, keep, recent=37)
    torch.cuda.synchronize()
    check_evict(old, res, [T - 3], keep, 37, True)


@pytest.mark.parametrize("dtype,D", [(torch.float32, 4), (torch.bfloat16, 8), (torch.float16, 328),
                                     (torch.float64, 6)])
def test_evict_types_and_odd_totals(gpu, dtype, D):
    # infinities rank as numbers, a NaN above them; positions out of order
    B, H, T, keep = 1, 3, 50, 13
    k, v, w, p, g = evict_case(B, H, T, D, dtype, D)
    w[0, 0, [3, 40]] = float("inf")
    w[0, 0, [5, 6, 7]] = float("-inf")
    w[0, 1, [9, 30]] = float("nan")
    w[0, 2] = 0.0
    p = p[:, :, torch.randperm(T, generator=g).to(dev)].contiguous()
    old = [t.clone() for t in (k, v, w, p)] + [torch.tensor([T])]
    lengths = torch.tensor([T], dtype=torch.int32, device=dev)
    res = F.kv_cache_evict(k, v, w, p, lengths, keep, recent=4)
    torch.cuda.synchronize()
    check_evict(old, res, [T], keep, 4, True)


# --------------------------------------------------------------- together ----

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_eviction_decode_and_tree_together(gpu, dtype):
    # a prompt's weights, its eviction into a small cache, decoded tokens that add
    # theirs and evict in place, then a drafted tree over what is left: the same
    # run in plain 64-bit arithmetic over the rows the operators kept
    B, H, T, D, keep, room, N = 2, 2, 90, 64, 40, 60, 9
    slopes = F.compute_alibi_slopes(H)
    sl, scale = slopes.to(dev), 0.125
    qkv = rand((B, T, 3, H, D), dtype, 1).permute(2, 0, 3, 1, 4)
    q, k, v = qkv[0], qkv[1], qkv[2]
    _, L = F.rational_attention_forward(q, k, v, sl, scale)
    w = F.rational_attention_key_weights(q, k, sl, scale, L)
    pos = torch.arange(T, dtype=torch.int32, device=dev).expand(B, H, T)
    cache = (torch.zeros(B, room, H, D, dtype=dtype, device=dev).permute(0, 2, 1, 3),
             torch.zeros(B, room, H, D, dtype=dtype, device=dev).permute(0, 2, 1, 3),
             torch.zeros(B, H, room, device=dev), torch.zeros(B, H, room, dtype=torch.int32, device=dev),
             torch.zeros(B, dtype=torch.int32, device=dev))
    F.kv_cache_evict(k, v, w, pos, None, keep, recent=8, out=cache)
    kc, vc, wc, pc, n = cache
    torch.cuda.synchronize()
    old = (k, v, w, pos, None)
    check_evict(old, cache, [T, T], keep, 8, False, [torch.zeros_like(t) for t in cache[:4]])
    for step in range(25):
        if int(n[0]) == room:
            before = [t.clone() for t in cache]
            F.kv_cache_evict(kc, vc, wc, pc, n, keep, recent=8)
            torch.cuda.synchronize()
            check_evict(before, cache, [room, room], keep, 8, True)
        r = int(n[0])
        kc[:, :, r], vc[:, :, r] = rand((B, H, D), dtype, 100 + step), rand((B, H, D), dtype, 200 + step)
        wc[:, :, r], pc[:, :, r] = 0.0, T + step
        n += 1
        was = wc.clone()
        qt = rand((B, H, D), dtype, 300 + step)
        o, Ld = F.rational_attention_decode_accumulate(qt, kc, vc, sl, scale, wc, lengths=n, positions=pc)
        torch.cuda.synchronize()
        check_accumulate(o, Ld, wc, was, qt, kc, vc, slopes, scale, n, pc)
    r = int(n[0])
    F.kv_cache_evict(kc, vc, wc, pc, n, keep, recent=8)
    torch.cuda.synchronize()
    r = int(n[0])
    parents = random_parents(1, N, 5)[0]
    depth = torch.tensor([len(x) for x in C.tree_lines(parents.tolist())], dtype=torch.int32, device=dev)
    kc[:, :, r:r + N], vc[:, :, r:r + N] = rand((B, H, N, D), dtype, 7), rand((B, H, N, D), dtype, 8)
    pc[:, :, r:r + N] = T + 24 + depth
    n += N
    qn = rand((B, H, N, D), dtype, 9)
    o, Lt = F.rational_attention_tree(qn, kc, vc, sl, scale, parents.to(dev), lengths=n, positions=pc)
    torch.cuda.synchronize()
    check_tree(o, Lt, qn, kc, vc, slopes, scale, parents, n, pc)
