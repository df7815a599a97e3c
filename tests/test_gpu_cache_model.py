"""The model on the operators over a key / value cache: bounded generation and
drafted tokens, against the plain generate() and forward()."""

import pytest
import torch

import fastalgebraictransformer_amd as F

pytestmark = pytest.mark.gpu
dev = "cuda"


def small_model(seed, **kw):
    torch.manual_seed(seed)
    return F.AlgebraicTransformerLM(vocab_size=300, d_model=128, n_head=2, n_layers=2, dropout=0.0,
                                    **kw).cuda().eval()


def test_bounded_generation_with_room_is_the_plain_one(gpu):
    # a budget that nothing exceeds: token for token the uncached greedy result
    m = small_model(0, block_size=128)
    prompt = torch.randint(0, 300, (2, 20), device=dev)
    a = m.generate(prompt, 30, top_k=1, cache_keep=64)
    b = m.generate(prompt, 30, top_k=1, use_cache=False)
    assert torch.equal(a, b)


@pytest.mark.parametrize("autocast", [False, True])
def test_bounded_generation_graph_matches_eager(gpu, autocast):
    # evictions of the prompt and, several times, between the replays; past block_size
    m = small_model(1, block_size=64)
    prompt = torch.randint(0, 300, (3, 50), device=dev)
    outs = []
    for use_graph in (True, False):
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            outs.append(m.generate(prompt, 60, top_k=1, cache_keep=24, use_graph=use_graph))
    assert outs[0].shape == (3, 110) and torch.equal(outs[0], outs[1])


def test_bounded_cache_holds_the_attention_weights(gpu):
    # without evictions the totals are the column sums of the attention: every
    # query hands out one unit (less eps / L)
    m = small_model(2)
    ids = torch.randint(0, 300, (2, 33), device=dev)
    with torch.no_grad():
        caches = m.new_kv_caches(64, keep=63)
        m.forward_cached(ids[:, :30], caches, 0)
        from fastalgebraictransformer_amd.algebraic_model import _DecodeStep
        step = _DecodeStep(m, caches, 2, ids.device, use_graph=True)
        for i in range(30, 33):
            logits = step(ids[:, i:i + 1], i, i)
        full, _ = m(ids)
    assert float((logits - full[:, -1]).abs().max()) <= 1e-4 * max(1.0, float(full.abs().max()))
    for c in caches:
        assert torch.allclose(c.weights.sum(-1), torch.full((2, 2), 33.0, device=dev), rtol=1e-4)
        assert torch.equal(c.positions[:, :, :33].cpu(),
                           torch.arange(33, dtype=torch.int32).expand(2, 2, 33))


@pytest.mark.parametrize("bounded", [False, True])
def test_tree_logits_are_those_of_each_branch(gpu, bounded):
    m = small_model(3)
    ids = torch.randint(0, 300, (2, 25), device=dev)
    tokens = torch.randint(0, 300, (2, 6), device=dev)
    parents = torch.tensor([[-1, 0, 0, 1, 2, 4], [-1, -1, 1, 2, 2, 0]], dtype=torch.int32, device=dev)
    lines = [[[0], [0, 1], [0, 2], [0, 1, 3], [0, 2, 4], [0, 2, 4, 5]],
             [[0], [1], [1, 2], [1, 2, 3], [1, 2, 4], [0, 5]]]
    path = torch.tensor([[0, 2, 4], [1, 2, 3]], device=dev)
    with torch.no_grad():
        caches = m.new_kv_caches(64, keep=40 if bounded else None)
        m.forward_cached(ids, caches, 0)
        logits = m.forward_tree(tokens, parents, caches, 25)
        for b in range(2):
            for i in range(6):
                ctx = torch.cat((ids[b], tokens[b, lines[b][i]]))[None]
                ref = m(ctx)[0][0, -1]
                assert float((logits[b, i] - ref).abs().max()) <= 1e-4 * max(1.0, float(ref.abs().max())), (b, i)
        # the accepted branch is then part of the context
        m.accept_drafted(caches, 25, path)
        nxt = torch.randint(0, 300, (2, 1), device=dev)
        got = m.forward_tree(nxt, torch.tensor([-1]), caches, 28)[:, 0]
        for b in range(2):
            ref = m(torch.cat((ids[b], tokens[b, path[b]], nxt[b]))[None])[0][0, -1]
            assert float((got[b] - ref).abs().max()) <= 1e-4 * max(1.0, float(ref.abs().max())), b


def test_drafted_generation_is_the_greedy_one(gpu):
    m = small_model(4, block_size=160)
    prompt = torch.randint(0, 300, (1, 17), device=dev)
    want = m.generate(prompt, 40, top_k=1)
    passes = []

    def good(idx):  # the right continuation as a chain, beside wrong branches
        passes.append(1)
        right = want[0, idx.size(1):idx.size(1) + 4]
        k = len(right)
        wrong = torch.zeros(3, dtype=torch.long, device=dev)
        return torch.cat((wrong, right)), [-1, 0, -1] + [-1] + list(range(3, 2 + k)) if k else [-1, 0, -1]

    assert torch.equal(m.generate_drafted(prompt, 40, good), want)
    assert len(passes) <= 9
    g = torch.Generator().manual_seed(0)
    bad = lambda idx: (torch.randint(0, 300, (5,), generator=g), torch.tensor([-1, 0, 1, -1, 3]))
    assert torch.equal(m.generate_drafted(prompt, 40, bad), want)
    none = lambda idx: ([], [])
    assert torch.equal(m.generate_drafted(prompt, 3, none), want[:, :20])
