"""Move of the accepted path's cache rows: bytes are copied, so everything is compared bit for bit."""
from __future__ import annotations

import pytest
import torch

from tests import speculative_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def capi():
    from vkop_b200 import capi as c
    return c


def make(batch, nodes, layers, heads, dim, page, top, dtype, seed, columns=None):
    g = torch.Generator().manual_seed(seed)
    context = torch.randint(0, top + 1, (batch,), generator=g, dtype=torch.int32)
    k, v, table = ref.paged(context + nodes, page, heads, dim, dtype, g, columns=columns)
    k, v = (torch.randn(layers, *x.shape, generator=g).to(dtype) for x in (k, v))
    count = torch.randint(0, nodes + 1, (batch,), generator=g, dtype=torch.int32)
    path = torch.full((batch, nodes), -1, dtype=torch.int32)
    for b in range(batch):
        n = int(count[b])
        if n:
            path[b, :n] = torch.cat([torch.zeros(1), 1 + torch.randperm(nodes - 1, generator=g)[: n - 1].sort()[0]]).to(torch.int32)
    return k, v, table, context, path, count


def check(capi, k, v, table, context, path, count, place=lambda t: t.cuda()):
    gk, gv = place(k), place(v) if v is not None else None
    lengths = capi.cache_compact(gk, gv, table.cuda(), context.cuda(), path.cuda(), count.cuda())
    torch.cuda.synchronize()
    for got, c in ((gk, k), (gv, v)):
        if c is not None:
            want, n = ref.compact(c, table, context, path, count)
            assert torch.equal(got.cpu().view(torch.uint8 if c.dtype != torch.float32 else torch.int32) if got.is_contiguous() else got.cpu(),
                               want.view(torch.uint8 if c.dtype != torch.float32 else torch.int32) if got.is_contiguous() else want)
    assert lengths.dtype == torch.int32 and lengths.tolist() == n


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,nodes,layers,heads,dim,page", [(1, 1, 1, 1, 8, 16), (3, 2, 2, 1, 64, 1), (5, 17, 3, 8, 128, 16), (2, 64, 1, 5, 40, 24), (4, 200, 2, 2, 64, 7), (3, 30, 2, 3, 5, 16), (2, 9, 1, 1, 1, 4)])
def test_rows_move_and_nothing_else(capi, dtype, batch, nodes, layers, heads, dim, page):
    for seed in range(3):
        check(capi, *make(batch, nodes, layers, heads, dim, page, 60, dtype, seed))


def test_every_node_accepted_and_none(capi):
    k, v, table, context, path, count = make(3, 12, 2, 2, 64, 16, 40, torch.float16, 4)
    path[:] = torch.arange(12)
    count[:] = torch.tensor([12, 0, 1])
    check(capi, k, v, table, context, path, count)


def test_the_last_nodes_move_to_the_front(capi):
    """Sources lie far behind targets, and targets are sources of later rows."""
    k, v, table, context, path, count = make(2, 40, 2, 2, 64, 16, 33, torch.bfloat16, 5)
    path[:] = -1
    path[0, :21] = torch.cat([torch.zeros(1), torch.arange(20, 40)]).int()
    path[1, :20] = torch.cat([torch.zeros(1), torch.arange(1, 39, 2)]).int()
    count[:] = torch.tensor([21, 20])
    check(capi, k, v, table, context, path, count)


def test_one_cache_and_one_layer(capi):
    k, v, table, context, path, count = make(3, 12, 1, 2, 64, 16, 40, torch.float16, 6)
    check(capi, k, None, table, context, path, count)
    gk, gv = k[0].cuda(), v[0].cuda()
    capi.cache_compact(gk, gv, table.cuda(), context.cuda(), path.cuda(), count.cuda())
    assert torch.equal(gk.cpu(), ref.compact(k, table, context, path, count)[0][0])
    assert torch.equal(gv.cpu(), ref.compact(v, table, context, path, count)[0][0])


def test_layouts(capi):
    c = make(3, 12, 2, 4, 64, 16, 40, torch.float16, 7)
    check(capi, *c, place=lambda t: t.cuda().permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4))  # heads before slots

    def odd(t):
        big = torch.zeros(*t.shape[:4], t.shape[4] + 1, dtype=t.dtype, device="cuda")[..., 1:]
        return big.copy_(t)

    check(capi, *c, place=odd)

    def inside(t):
        big = torch.zeros(t.shape[0] + 1, t.shape[1], t.shape[2], t.shape[3] + 2, t.shape[4], dtype=t.dtype, device="cuda")[1:, :, :, 1:-1]
        return big.copy_(t)

    check(capi, *c, place=inside)


def test_bad_paths_pages_and_counts(capi):
    k, v, table, context, path, count = make(6, 12, 2, 2, 64, 16, 60, torch.float16, 8)
    path[:] = torch.tensor([0, 2, 3, 5, 8, 9, 11, -1, -1, -1, -1, -1], dtype=torch.int32)
    count[:] = torch.tensor([7, 7, 7, 9, 99, -4])
    path[0, 3], path[1, 4], path[2, 2] = 3, 12, -1          # repeated, past the nodes, not there
    check(capi, k, v, table, context, path, count)
    count[:] = 7
    table[3, int(context[3]) // 16], table[4, int(context[4] + 8) // 16] = -1, k.shape[1]
    check(capi, k, v, table, context, path, count)
    check(capi, k, v, table[:, :3].contiguous(), context, path, count)
    check(capi, k, v, table[:, :0].contiguous(), context, path, count)


def test_offsets_past_32_bits(capi):
    pages, page = 70000, 16
    k = torch.empty(1, pages, page, 16, 128, dtype=torch.float16, device="cuda")
    assert k.numel() > 2**31
    k[0, 69999], k[0, 3] = 1.0, 2.0
    k[0, 69999, :, 0, 0] = torch.arange(16, device="cuda").half()
    lengths = capi.cache_compact(k, None, torch.tensor([[3, 69999]], dtype=torch.int32).cuda(), torch.tensor([15], dtype=torch.int32).cuda(),
                                 torch.tensor([[0, 4, 6, -1, -1, -1, -1]], dtype=torch.int32).cuda(), torch.tensor([3], dtype=torch.int32).cuda())
    assert lengths.tolist() == [18]
    assert k[0, 69999, :, 0, 0].tolist() == [3.0, 5.0, 2.0, 3.0] + list(range(4, 16))  # positions 16, 17 hold nodes 4, 6


def test_streams_and_graphs(capi):
    k, v, table, context, path, count = make(3, 12, 2, 2, 64, 16, 40, torch.float16, 9)
    gk, gv = k.cuda(), v.cuda()
    args = [t.cuda() for t in (table, context, path, count)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lengths = capi.cache_compact(gk, gv, *args)
    for seed in (10, 11):
        _, _, _, _, path, count = make(3, 12, 2, 2, 64, 16, 40, torch.float16, seed)
        gk.copy_(k)
        gv.copy_(v)
        args[2].copy_(path)
        args[3].copy_(count)
        graph.replay()
        torch.cuda.synchronize()
        want, n = ref.compact(k, table, context, path, count)
        assert torch.equal(gk.cpu(), want) and lengths.tolist() == n
