"""How the operators over a key / value cache are called: captured and replayed,
on other streams, with arguments that need converting, with caches past 2^31
bytes, and with arguments that are refused."""

import pytest
import torch

import fastalgebraictransformer_amd as F
from oracle import cache as C
from test_gpu_cache_ops import (caches, check_accumulate, check_evict, check_tree, positions_like, rand,
                                random_parents)

pytestmark = pytest.mark.gpu
dev = "cuda"


class Case:
    """One call of every operator on fixed inputs, split over blocks and not."""

    def __init__(self, seed, T):
        self.B, self.H, self.T, self.D, self.N = 2, 2, T, 64, 20
        B, H, D, N = self.B, self.H, self.D, self.N
        self.k, self.v = caches(B, H, T, D, torch.bfloat16, seed)
        self.q = rand((B, N, H, D), torch.bfloat16, seed + 2).permute(0, 2, 1, 3)
        self.q1 = rand((B, H, D), torch.bfloat16, seed + 3)
        self.qt = rand((B, H, T, D), torch.bfloat16, seed + 4)
        self.slopes = F.compute_alibi_slopes(H).to(dev)
        self.parents = random_parents(B, N, seed).to(dev)
        self.n = torch.tensor([T, T - 7], dtype=torch.int32, device=dev)
        self.pos = positions_like(B, H, T, seed)
        self.L = torch.rand(B, H, T, device=dev) + 1
        self.total = torch.rand(B, H, T, device=dev)
        self.first = self.total.clone()
        self.out = (torch.zeros(B, H, T // 2, D, dtype=torch.bfloat16, device=dev),
                    torch.zeros(B, H, T // 2, D, dtype=torch.bfloat16, device=dev),
                    torch.zeros(B, H, T // 2, device=dev), torch.zeros(B, H, T // 2, dtype=torch.int32, device=dev),
                    torch.zeros(B, dtype=torch.int32, device=dev))

    def run(self):
        self.total.copy_(self.first)
        a = F.rational_attention_tree(self.q, self.k, self.v, self.slopes, 0.1, self.parents, lengths=self.n,
                                      positions=self.pos)
        b = F.rational_attention_decode_accumulate(self.q1, self.k, self.v, self.slopes, 0.1, self.total,
                                                   lengths=self.n)
        c = F.rational_attention_key_weights(self.qt, self.k, self.slopes, 0.1, self.L)
        d = F.kv_cache_evict(self.k, self.v, self.total, self.pos, self.n, self.T // 2, recent=9, out=self.out)
        # and in place, on copies
        e = F.kv_cache_evict(self.k.clone(), self.v.clone(), self.total.clone(), self.pos.clone(), self.n.clone(),
                             self.T // 2, recent=9)
        return a + b + (c, self.total) + tuple(d) + tuple(e)


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("T", [120, 3001])
def test_captured_and_replayed(gpu, T):
    # two graphs, replayed in turn with eager work and synchronisations between
    # (each has workspaces of its own); every replay against the eager result
    cases = [Case(1, T), Case(50, T)]
    want = [[t.clone() for t in c.run()] for c in cases]
    graphs, got = [], []
    for c in cases:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            c.run()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = c.run()
        graphs.append(g)
        got.append(r)
    for i in range(4):
        for j in (0, 1):
            graphs[j].replay()
            if i % 2:
                torch.cuda.synchronize()
            assert same(got[j], want[j]), (i, j)
            assert same(cases[1 - j].run(), want[1 - j])
            junk = torch.randn(300, 300, device=dev) @ torch.randn(300, 300, device=dev)
            del junk
    for j in (1, 0):  # back to back
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert same(got[0], want[0]) and same(got[1], want[1])
    # another length in the same buffers
    cases[0].n.copy_(torch.tensor([T // 3, 25], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    other = [t.clone() for t in got[0]]
    for t in cases[0].out:
        t.zero_()
    assert same([t for i, t in enumerate(cases[0].run()) if i not in (6, 7, 8, 9)],
                [t for i, t in enumerate(other) if i not in (6, 7, 8, 9)])


@pytest.mark.parametrize("T", [120, 3001])
def test_two_calls_at_once_on_two_streams(gpu, T):
    cases = [Case(2, T), Case(60, T)]
    want = [[t.clone() for t in c.run()] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for rep in range(5):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(c.run())
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert same(g, w), rep


def test_arguments_are_converted(gpu):
    # other integer types, float slopes on the host, masks as numbers, caches of
    # another dtype, strided inputs: the same results as the plain call
    c = Case(3, 200)
    B, H, T, D = c.B, c.H, c.T, c.D
    a = F.rational_attention_tree(c.q, c.k, c.v, c.slopes, 0.1, c.parents, lengths=c.n, positions=c.pos)
    wide = torch.stack((c.k, c.k), -1)[..., 0]  # last-dim stride 2
    b = F.rational_attention_tree(c.q, wide, c.v.float(), c.slopes.cpu().double(), 0.1, c.parents.long().cpu(),
                                  lengths=c.n.tolist() and c.n.long(), positions=c.pos.long())
    assert same(a, b)
    one = random_parents(1, c.N, 5)[0].to(dev)
    assert same(F.rational_attention_tree(c.q, c.k, c.v, c.slopes, 0.1, one),
                F.rational_attention_tree(c.q, c.k, c.v, c.slopes, 0.1, one.expand(B, c.N)))
    t1, t2 = c.total.clone(), c.total.clone()
    a = F.rational_attention_decode_accumulate(c.q1, c.k, c.v, c.slopes, 0.1, t1, lengths=c.n)
    b = F.rational_attention_decode_accumulate(c.q1, wide, c.v.float(), c.slopes.double(), 0.1, t2, lengths=c.n.long())
    assert same(a, b) and torch.equal(t1, t2)
    mask = torch.rand(B, T, device=dev) < 0.7
    a = F.rational_attention_key_weights(c.qt, c.k, c.slopes, 0.1, c.L, key_mask=mask, last=50)
    for m in (mask.float() * 3, mask.to(torch.uint8) * 5, mask.t().contiguous().t(), mask.long()):
        assert torch.equal(a, F.rational_attention_key_weights(c.qt, c.k, c.slopes, 0.1, c.L, key_mask=m, last=50))
    b = F.rational_attention_key_weights(c.qt, wide, c.slopes.double(), 0.1, c.L.double(), key_mask=mask, last=50)
    assert torch.equal(a, b)
    assert torch.equal(F.rational_attention_key_weights(c.qt, c.k, c.slopes, 0.1, c.L, last=10 ** 30),
                       F.rational_attention_key_weights(c.qt, c.k, c.slopes, 0.1, c.L))
    res = [t.clone() for t in F.kv_cache_evict(c.k, c.v, c.total, c.pos, c.n, 90, recent=4, out=c.out)]
    again = F.kv_cache_evict(wide, c.v, c.total.double(), c.pos.long(), c.n.long(), 90, recent=4, out=c.out)
    assert same(res, again)


def test_dims_of_one_element_have_no_stride(gpu):
    # views whose strides of single-element dims are odd numbers
    k, v = rand((1, 1, 40, 64), torch.bfloat16, 1), rand((1, 1, 40, 64), torch.bfloat16, 2)
    q = rand((1, 1, 1, 64), torch.bfloat16, 3)
    odd = lambda t, *s: t.as_strided(t.shape, s)
    s = torch.tensor([0.1], device=dev)
    root = torch.full((1,), -1, dtype=torch.int32, device=dev)
    ko, vo, qo = odd(k, 3, 5, 64, 1), odd(v, 1, 7, 64, 1), odd(q, 3, 1, 5, 1)
    want = F.rational_attention_tree(q, k, v, s, 0.2, root)
    assert same(want, F.rational_attention_tree(qo, ko, vo, s, 0.2, root))
    t1, t2 = torch.zeros(1, 1, 40, device=dev), torch.zeros(1, 1, 40, device=dev)
    want = F.rational_attention_decode_accumulate(q[:, :, 0], k, v, s, 0.2, t1)
    got = F.rational_attention_decode_accumulate(odd(q[:, :, 0], 3, 9, 1), ko, vo, s, 0.2, odd(t2, 1, 1, 1))
    assert same(want, got) and torch.equal(t1, t2)
    L = torch.rand(1, 1, 40, device=dev) + 1
    assert torch.equal(F.rational_attention_key_weights(k, v, s, 0.2, L),
                       F.rational_attention_key_weights(ko, vo, s, 0.2, odd(L, 3, 1, 1)))
    one = (odd(q, 3, 1, 5, 1), odd(q.clone(), 7, 3, 1, 1), odd(torch.ones(1, 1, 1, device=dev), 0, 0, 0),
           torch.zeros(1, 1, 1, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev))
    F.kv_cache_evict(ko, vo, t1, torch.arange(40, dtype=torch.int32, device=dev).view(1, 1, 40), None, 1, out=one)
    j = int(t1[0, 0].argmax())
    torch.cuda.synchronize()
    assert torch.equal(one[0][0, 0, 0], k[0, 0, j]) and torch.equal(one[1][0, 0, 0], v[0, 0, j])
    assert int(one[3]) == j and int(one[4]) == 1


def test_empty_calls(gpu):
    s = F.compute_alibi_slopes(2).to(dev)
    kv = torch.zeros(3, 2, 0, 64, dtype=torch.bfloat16, device=dev)
    q = rand((3, 2, 64), torch.bfloat16, 1)
    i32 = dict(dtype=torch.int32, device=dev)
    o, L = F.rational_attention_tree(q[:, :, None], kv, kv, s, 0.1, torch.full((1,), -1, **i32))
    assert float(o.abs().max()) == 0 and float(L.abs().max()) == 0
    w = torch.zeros(3, 2, 0, device=dev)
    o, L = F.rational_attention_decode_accumulate(q, kv, kv, s, 0.1, w)
    assert float(o.abs().max()) == 0 and float(L.abs().max()) == 0
    assert F.rational_attention_key_weights(kv, kv, s, 0.1, w).shape == (3, 2, 0)
    n = torch.full((3,), 5, **i32)
    F.kv_cache_evict(kv, kv, w, torch.zeros(3, 2, 0, **i32), n, 4)
    assert n.tolist() == [0, 0, 0]
    k = rand((0, 2, 7, 64), torch.bfloat16, 1)
    assert F.rational_attention_tree(k, k, k, s, 0.1, torch.zeros(7, **i32))[0].shape == (0, 2, 7, 64)
    o, L = F.rational_attention_tree(rand((1, 2, 0, 64), torch.bfloat16, 1), rand((1, 2, 7, 64), torch.bfloat16, 1),
                                     rand((1, 2, 7, 64), torch.bfloat16, 2), s, 0.1, torch.zeros(0, **i32))
    assert o.shape == (1, 2, 0, 64) and L.shape == (1, 2, 0)


def test_refused_arguments(gpu):
    c = Case(4, 100)
    B, H, T, D = c.B, c.H, c.T, c.D
    tree = lambda **kw: F.rational_attention_tree(*[kw.get(n, getattr(c, n)) for n in ("q", "k", "v", "slopes")], 0.1,
                                                  kw.get("parents", c.parents), lengths=kw.get("n", c.n),
                                                  positions=kw.get("pos", c.pos))
    for bad in (dict(k=c.k[:, :, :50]), dict(k=c.k[:, :1]), dict(parents=c.parents[:, :-1]), dict(n=c.n[:1]),
                dict(pos=c.pos[:, :, :-1]), dict(slopes=c.slopes[:1]), dict(q=c.q.repeat(1, 1, 4, 1))):
        with pytest.raises(AssertionError):
            tree(**bad)
    with pytest.raises(RuntimeError, match="aligned"):  # rows of odd offset
        tree(k=torch.zeros(B, H, T, D + 4, dtype=torch.bfloat16, device=dev)[..., 4:])
    with pytest.raises(RuntimeError, match="head dim"):
        kv = torch.zeros(B, H, T, 12, dtype=torch.bfloat16, device=dev)
        tree(q=kv[:, :, :c.N], k=kv, v=kv)
    for w in (c.total.half(), c.total[:, :, :-1], c.total[:, :1].expand(B, H, T), c.total.cpu(),
              c.total.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(AssertionError):
            F.rational_attention_decode_accumulate(c.q1, c.k, c.v, c.slopes, 0.1, w)
    with pytest.raises(AssertionError):
        F.rational_attention_key_weights(c.qt, c.k, c.slopes, 0.1, c.L, last=0)
    with pytest.raises(AssertionError):
        F.rational_attention_key_weights(c.qt, c.k, c.slopes, 0.1, c.L, key_mask=torch.ones(B, T + 1, device=dev))
    with pytest.raises(AssertionError):
        F.rational_attention_key_weights(c.qt, c.k, c.slopes, 0.1, c.L[:, :, 1:])
    ev = lambda keep=20, recent=4, out=None, **kw: F.kv_cache_evict(
        *[kw.get(n, getattr(c, n)) for n in ("k", "v", "total", "pos", "n")], keep, recent=recent, out=out)
    for bad in (dict(recent=21), dict(recent=-1), dict(keep=-1, recent=0), dict(n=None), dict(n=c.n.long()),
                dict(total=c.total.double()), dict(pos=c.pos[:, :1].expand(B, H, T)), dict(v=c.v.float()),
                dict(v=c.v[:, :, :-1]), dict(k=c.k[:, :1].expand(B, H, T, D)), dict(out=c.out[:4]),
                dict(keep=51, out=c.out), dict(out=c.out[:4] + (c.n.long(),)),
                dict(out=(c.out[0][:, :, ::2],) + c.out[1:])):
        with pytest.raises(AssertionError):
            ev(**bad)
    with pytest.raises(RuntimeError, match="lengths_out"):
        ev(out=c.out[:4] + (c.n,))
    assert torch.equal(c.total, c.first) and c.n.tolist() == [T, T - 7]  # nothing was written


@pytest.mark.parametrize("T", [70, 5000])
def test_rows_without_keys_are_zero_with_eps_0(gpu, T):
    B, H, D, N = 2, 2, 64, 5
    q, k, v = (rand((B, H, n, D), torch.bfloat16, s) for n, s in ((N, 1), (T, 2), (T, 3)))
    slopes = torch.tensor([0.5, 0.1], device=dev)
    parents = torch.tensor([-1, 0, -7, 2, 1], dtype=torch.int32, device=dev)  # 2 and, below it, 3 are absent
    n = torch.tensor([T, N - 1], dtype=torch.int32, device=dev)               # row 1: no room for the tokens
    o, L = F.rational_attention_tree(q, k, v, slopes, 0.125, parents, lengths=n, eps=0.0)
    assert float(o[0, :, 2:4].abs().max()) == 0 and float(o[1].abs().max()) == 0 and float(L[1].abs().max()) == 0
    assert bool(torch.isfinite(o).all()) and float(o[0, :, 4].abs().max()) > 0
    n[1] = 0
    total = rand((B, H, T), torch.float32, 4)
    before = total.clone()
    o, L = F.rational_attention_decode_accumulate(q[:, :, 0], k, v, slopes, 0.125, total, lengths=n, eps=0.0)
    assert float(o[1].abs().max()) == 0 and float(L[1].abs().max()) == 0 and torch.equal(total[1], before[1])
    assert bool(torch.isfinite(o).all()) and bool((total[0] >= before[0]).all())


def test_caches_past_2_31_bytes(gpu):
    # one head of a wide token-major cache: rows 64 KB apart, the last past 2^31
    T, heads, D, N = 33000, 512, 64, 6
    big = torch.empty(2, 1, T, heads, D, dtype=torch.bfloat16, device=dev)
    k, v = (big[i][:, :, 511:].permute(0, 2, 1, 3) for i in (0, 1))
    k.copy_(rand((1, 1, T, D), torch.bfloat16, 1))
    v.copy_(rand((1, 1, T, D), torch.bfloat16, 2))
    assert (T - 1) * k.stride(2) * 2 > 2 ** 31
    slopes = torch.tensor([2.0 ** -12], device=dev)  # gentle: far rows count
    q = rand((1, 1, N, D), torch.bfloat16, 3)
    parents = random_parents(1, N, 4)
    o, L = F.rational_attention_tree(q, k, v, slopes, 0.125, parents.to(dev))
    check_tree(o, L, q, k, v, slopes.cpu(), 0.125, parents, None, None)
    total = torch.zeros(1, 1, T, device=dev)
    o, L = F.rational_attention_decode_accumulate(q[:, :, 0], k, v, slopes, 0.125, total)
    torch.cuda.synchronize()
    check_accumulate(o, L, total, torch.zeros_like(total), q[:, :, 0], k, v, slopes.cpu(), 0.125, None, None)
    Lq = torch.rand(1, 1, T, device=dev) + 1
    w = F.rational_attention_key_weights(v, k, slopes, 0.125, Lq, last=3)  # v as the queries: both wide
    ref, tol = C.key_weights(v[0, 0].cpu(), k[0, 0].cpu(), slopes[0].cpu(), 0.125, Lq[0, 0].cpu(), None, 3)
    assert bool(((w[0, 0].double().cpu() - ref).abs() <= tol + 1e-30).all())
    pos = torch.arange(T, dtype=torch.int32, device=dev).view(1, 1, T)
    n = torch.tensor([T], dtype=torch.int32, device=dev)
    old = [t.clone(memory_format=torch.contiguous_format) for t in (k, v, total, pos, n)]
    total[0, 0, -500:] += 1.0
    old[2].copy_(total)
    F.kv_cache_evict(k, v, total, pos, n, 700, recent=10)
    torch.cuda.synchronize()
    check_evict(old, (k, v, total, pos, n), [T], 700, 10, True)
