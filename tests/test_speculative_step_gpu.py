"""The three operators as a serving loop uses them: attention of the drafted tree, verification of what the model made of it,
move of the accepted rows, and the next step's attention on the shortened cache."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests import speculative_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from vkop_b200 import capi as c
    return c


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 128, 16), (torch.float16, 64, 24), (torch.float32, 40, 5)])
def test_steps_of_a_serving_loop(capi, tree, dtype, dim, page):
    batch, nodes, heads, group, vocab, layers = 4, 10, 2, 4, 501, 2
    g = torch.Generator().manual_seed(1)
    room = 200
    k, v, table = ref.paged([room] * batch, page, heads, dim, dtype, g)
    k, v = (torch.stack([x, torch.randn(x.shape, generator=g).to(dtype)]).cuda() for x in (k, v))
    table, context = table.cuda(), torch.tensor([0, 7, 63, 130], dtype=torch.int32).cuda()
    embed = torch.randn(vocab, heads * group * dim, generator=g).cuda()
    kept = [[] for _ in range(batch)]  # per sequence: (key, value) of every accepted row, as the cache should hold them
    start = context.clone()
    for b in range(batch):
        for pos in range(int(context[b])):
            at = int(table[b, pos // page]), pos % page
            kept[b].append((k[:, at[0], at[1]].clone(), v[:, at[0], at[1]].clone()))
    for step in range(3):
        parents = ref.random_tree(batch, nodes, g).cuda() if tree else None
        fresh = [torch.randn(layers, batch, nodes, heads, dim, generator=g).to(dtype).cuda() for _ in range(2)]
        pos = context[:, None].long() + torch.arange(nodes, device="cuda")[None]
        pages = table.long().gather(1, pos // page)
        for cache, new in zip((k, v), fresh):
            cache[:, pages, pos % page] = new
        q = torch.randn(batch, nodes, heads * group, dim, generator=g).to(dtype).cuda()
        outs = [capi.tree_attention(q, k[i], v[i], table, context, parents=parents, return_lse=True) for i in range(layers)]
        for i in range(layers):
            ref.check_attend(outs[i], q.cpu(), k[i].cpu(), v[i].cpu(), table.cpu(), context.cpu(), None if parents is None else parents.cpu())
        logits = outs[-1][0].float().view(batch, nodes, -1) @ embed.T
        probs = capi.softmax(logits, inv_temperature=0.2)
        draft = capi.softmax(logits + torch.randn(logits.shape, generator=g).cuda(), inv_temperature=0.2)
        up = parents.long() if tree else (torch.arange(nodes, device="cuda") - 1).clamp(min=0).expand(batch, nodes)
        rows = draft.gather(1, up[:, :, None].expand(-1, -1, vocab))
        tokens = torch.multinomial(rows.cpu().view(-1, vocab), 1, generator=g).view(batch, nodes).to(torch.int32).cuda()
        u = torch.rand(batch, nodes, generator=g).cuda()
        path, count, token = capi.draft_verify(probs, tokens, u, draft=draft, parents=parents)
        want = ref.verify(probs, tokens, u, draft, None if parents is None else parents.cpu())
        assert np.array_equal(path.cpu().numpy(), want[0]) and np.array_equal(token.cpu().numpy(), want[2])
        assert (token >= 0).all() and (count >= 1).all()
        longer = capi.cache_compact(k, v, table, context, path, count)
        assert torch.equal(longer, context + count)
        for b in range(batch):
            kept[b] += [(fresh[0][:, b, int(n)], fresh[1][:, b, int(n)]) for n in path[b, : int(count[b])]]
            assert len(kept[b]) == int(longer[b])
            for p, (kk, vv) in enumerate(kept[b]):
                at = int(table[b, p // page]), p % page
                assert torch.equal(k[:, at[0], at[1]], kk) and torch.equal(v[:, at[0], at[1]], vv), (b, p)
        context = longer
    assert (context > start + 2).all()


def test_a_step_in_one_graph(capi):
    """Attention, softmax, verification and the move captured together and replayed."""
    batch, nodes, heads, dim, page, vocab = 3, 6, 2, 64, 16, 300
    g = torch.Generator().manual_seed(2)
    lengths = torch.tensor([40, 0, 90], dtype=torch.int32)
    k, v, table = ref.paged(lengths + nodes, page, heads, dim, torch.float16, g)
    parents = ref.random_tree(batch, nodes, g)
    q = torch.randn(batch, nodes, heads, dim, generator=g).half()
    embed = torch.randn(vocab, heads * dim, generator=g)
    tokens = torch.randint(0, vocab, (batch, nodes), generator=g, dtype=torch.int32)
    u = torch.rand(batch, nodes, generator=g)
    d = [x.cuda() for x in (q, k, v, table, lengths, parents, tokens, u, embed)]

    def step(k, v):
        out = capi.tree_attention(d[0], k, v, d[3], d[4], parents=d[5])
        probs = capi.softmax(out.float().view(batch, nodes, -1) @ d[8].T)
        path, count, token = capi.draft_verify(probs, d[6], d[7], parents=d[5])
        return out, path, count, token, capi.cache_compact(k, v, d[3], d[4], path, count), k, v

    want = step(d[1].clone(), d[2].clone())
    torch.cuda.synchronize()
    gk, gv = d[1].clone(), d[2].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(gk, gv)
    for _ in range(2):
        gk.copy_(d[1])
        gv.copy_(d[2])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want))
