"""Attention of a token tree over a paged cache against a 64-bit statement, within bounds that count roundings."""
from __future__ import annotations

import pytest
import torch

from tests import speculative_reference as ref

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module")
def capi():
    from vkop_b200 import capi as c
    return c


def run(capi, q, k, v, table, context, parents=None, num_nodes=None, scale=None, **kw):
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    got = capi.tree_attention(dev(q), dev(k), dev(v), dev(table), dev(context), parents=dev(parents), num_nodes=dev(num_nodes),
                              scale=scale, return_lse=True, **kw)
    torch.cuda.synchronize()
    return got


def case(batch, nodes, kv_heads, group, dim, page, context, dtype, tree, seed=0, used=None, fill=NAN, columns=None):
    g = torch.Generator().manual_seed(seed)
    context = torch.tensor(context, dtype=torch.int32)
    n = torch.full((batch,), nodes) if used is None else torch.tensor(used)
    k, v, table = ref.paged(context.clamp(min=0) + n, page, kv_heads, dim, dtype, g, fill=fill, columns=columns)
    q = (2 * torch.randn(batch, nodes, kv_heads * group, dim, generator=g)).to(dtype)
    return q, k, v, table, context, ref.random_tree(batch, nodes, g) if tree else None, None if used is None else n.to(torch.int32)


def check(capi, *c, **kw):
    got = run(capi, *c, **kw)
    ref.check_attend(got, *c, scale=kw.get("scale"), what=str(tuple(c[0].shape)))
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("nodes,kv_heads,group,tree", [(1, 2, 1, False), (1, 1, 4, False), (3, 2, 5, False), (7, 1, 8, True), (33, 2, 1, True), (64, 1, 3, True)])
@pytest.mark.parametrize("page", [16, 24, 128])
def test_matches_the_formula(capi, dtype, dim, nodes, kv_heads, group, tree, page):
    check(capi, *case(4, nodes, kv_heads, group, dim, page, [0, 1, 127, 300], dtype, tree, seed=nodes))


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 8), (torch.bfloat16, 40), (torch.float16, 80), (torch.bfloat16, 96), (torch.float32, 256), (torch.bfloat16, 256)])
def test_head_sizes(capi, dtype, dim):
    check(capi, *case(2, 6, 2, 3, dim, 7, [50, 201], dtype, True, seed=dim))


@pytest.mark.parametrize("length", [126, 127, 128, 129, 255, 256, 257, 511, 513, 1023, 2049, 4500])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_lengths_around_tiles_and_parts(capi, dtype, length):
    check(capi, *case(1, 5, 1, 2, 128, 16, [length], dtype, True, seed=length))
    check(capi, *case(2, 20, 1, 8, 64, 48, [length, length // 3], dtype, True, seed=length))


@pytest.mark.parametrize("nodes,group", [(128, 1), (128, 3), (16, 16), (128, 8), (65, 4)])
def test_many_rows(capi, nodes, group):
    check(capi, *case(2, nodes, 2, group, 64, 32, [200, 77], torch.bfloat16, True, seed=nodes))
    check(capi, *case(1, nodes, 1, group, 128, 32, [400], torch.float16, False, seed=nodes))


@pytest.mark.parametrize("page", [1, 3, 5, 8, 16, 40, 48, 96, 256, 1000])
def test_page_sizes(capi, page):
    check(capi, *case(3, 4, 2, 2, 64, page, [0, 19, 140], torch.float16, True, seed=page))
    check(capi, *case(2, 6, 2, 3, 128, page, [1301, 777], torch.bfloat16, True, seed=page))
    check(capi, *case(1, 40, 1, 5, 64, page, [900], torch.bfloat16, True, seed=page))


@pytest.mark.parametrize("dim", [64, 80])
def test_padding_nodes_and_empty_sequences_are_zero(capi, dim):
    c = case(5, 9, 2, 4, dim, 16, [0, 33, 0, 500, 40], torch.bfloat16, True, seed=3, used=[0, 0, 1, 9, 4])
    out, lse = check(capi, *c)
    assert (out[0] == 0).all() and (lse[0] == -INF).all() and (out[4, 4:] == 0).all() and (lse[4, 4:] == -INF).all()
    # counts outside the range are taken as its ends, a negative context as 0
    q, k, v, table, context, parents, _ = c
    wild = run(capi, q, k, v, table, torch.tensor([-5, 33, -1, 500, 40], dtype=torch.int32), parents, torch.tensor([-2, 0, 1, 99, 4], dtype=torch.int32))
    assert torch.equal(wild[0], out) and torch.equal(wild[1], lse)


@pytest.mark.parametrize("batch,kv_heads,length", [(3, 2, 1500), (40, 8, 700)])
def test_padding_nodes_of_long_sequences(capi, batch, kv_heads, length):
    """Few sequences, whose rows several CTAs share, and many, of which a CTA takes several in turn."""
    g = torch.Generator().manual_seed(4)
    used = torch.randint(0, 6, (batch,), generator=g).tolist()
    context = torch.randint(length // 2, length, (batch,), generator=g).tolist()
    c = case(batch, 5, kv_heads, 2, 64, 16, context, torch.float16, True, seed=8, used=used)
    out, lse = check(capi, *c)
    pad = torch.arange(5)[None] >= torch.tensor(used)[:, None]
    assert (out.cpu()[pad] == 0).all() and (lse.cpu()[pad] == -INF).all()


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 64), (torch.bfloat16, 128), (torch.float32, 64)])
def test_what_masked_places_hold_does_not_matter(capi, dtype, dim):
    """NaN and infinities behind the sequences (in every case here) and in drafted rows of other branches."""
    q, k, v, table, context, parents, _ = case(2, 12, 2, 4, dim, 16, [100, 140], dtype, True, seed=5)
    parents[:] = torch.tensor([0, 0, 0, 1, 1, 2, 2, 3, 4, 5, 6, 9], dtype=torch.int32)
    for b, node, bad in ((0, 5, NAN), (0, 7, INF), (1, 2, -INF), (1, 11, NAN)):
        pos = int(context[b]) + node
        page, slot = int(table[b, pos // 16]), pos % 16
        k[page, slot], v[page, slot] = bad, bad
    out, lse = run(capi, q, k, v, table, context, parents)
    clean_k, clean_v = torch.nan_to_num(k, 0, 0, 0), torch.nan_to_num(v, 0, 0, 0)
    want, want_lse = run(capi, q, clean_k, clean_v, table, context, parents)
    hit = torch.zeros(2, 12, dtype=torch.bool)
    for b, node in ((0, 5), (0, 7), (1, 2), (1, 11)):
        hit[b] |= torch.from_numpy(ref.ancestors(parents[b], 12)[:, node].copy())
    assert torch.equal(out.cpu()[~hit], want.cpu()[~hit]) and torch.equal(lse.cpu()[~hit], want_lse.cpu()[~hit])
    assert hit.sum() == 10
    # a value alone that is not finite reaches the rows that attend it, and only those
    v2 = clean_v.clone()
    pos = int(context[0]) + 5
    v2[int(table[0, pos // 16]), pos % 16] = INF
    out2, lse2 = run(capi, q, clean_k, v2, table, context, parents)
    sees = torch.from_numpy(ref.ancestors(parents[0], 12)[:, 5].copy())
    assert torch.equal(out2[0].cpu()[~sees], want[0].cpu()[~sees]) and not torch.isfinite(out2[0].cpu()[sees]).any()
    assert torch.equal(out2[1], want[1]) and torch.equal(lse2, want_lse)


@pytest.mark.parametrize("dtype,dim", [(torch.float16, 128), (torch.float32, 64)])
def test_pages_that_are_not_there_are_left_out(capi, dtype, dim):
    q, k, v, table, context, parents, _ = case(3, 6, 1, 2, dim, 16, [200, 90, 64], dtype, True, seed=7)
    table[0, 3], table[0, 7], table[1, 0], table[1, 6] = -1, k.shape[0], 1 << 30, -7
    check(capi, q, k, v, table, context, parents)
    table[2, :] = -1  # nothing at all: rows of zeros
    out, lse = check(capi, q, k, v, table, context, parents)
    assert (out[2] == 0).all() and (lse[2] == -INF).all()
    # a table that ends before the sequence does
    check(capi, q, k, v, table[:, :4].contiguous(), context, parents)
    check(capi, q, k, v, table[:, :0].contiguous(), context, parents)


def test_parents_out_of_range_have_no_ancestors(capi):
    q, k, v, table, context, parents, _ = case(2, 10, 1, 2, 64, 16, [40, 0], torch.float16, True, seed=9)
    parents[0, 3], parents[0, 5], parents[1, 1], parents[1, 9], parents[1, 0] = -1, 5, 9, 70, 5
    check(capi, q, k, v, table, context, parents)


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16), (64, torch.float32)])
def test_layouts(capi, dim, dtype):
    """Heads before slots in the cache, queries and outputs inside larger tensors, rows off the 16-byte boundary."""
    q, k, v, table, context, parents, _ = case(3, 5, 4, 2, dim, 16, [60, 17, 300], dtype, True, seed=12)
    want = check(capi, q, k, v, table, context, parents)
    t = [x.cuda() for x in (table, context, parents)]

    def go(q, k, v, table=t[0], **kw):
        return capi.tree_attention(q, k, v, table, t[1], parents=t[2], return_lse=True, **kw)

    hk, hv = (x.cuda().permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    fused = torch.randn(3, 5, 24, dim, device="cuda").to(dtype)
    fused[:, :, 3:11] = q.cuda()
    held = torch.zeros(3, 7, 10, dim, dtype=dtype, device="cuda")
    for got in (go(q.cuda(), hk, hv), go(fused[:, :, 3:11], k.cuda(), v.cuda()), go(q.cuda(), k.cuda(), hv, out=held[:, 1:6, 1:9])):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert (held[:, 0] == 0).all() and (held[:, 6] == 0).all() and (held[:, :, 0] == 0).all() and (held[:, :, 9] == 0).all()
    wide = torch.full((3, t[0].shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    wide[:, : t[0].shape[1]] = t[0]
    got = go(q.cuda(), k.cuda(), v.cuda(), table=wide[:, : t[0].shape[1]])
    assert torch.equal(got[0], want[0])
    off = torch.zeros(k.numel() + 1, dtype=dtype, device="cuda")[1:].view(k.shape)
    off.copy_(k)
    got = go(q.cuda(), off, v.cuda())
    ref.check_attend(got, q, k, v, table, context, parents, what="off the boundary")
    odd = torch.zeros(*k.shape[:3], dim + 1, dtype=dtype, device="cuda")[..., :dim]
    odd.copy_(v)
    got = go(q.cuda(), k.cuda(), odd)
    ref.check_attend(got, q, k, v, table, context, parents, what="odd strides")
    qo = torch.zeros(*q.shape[:3], dim + 1, dtype=dtype, device="cuda")[..., 1:]
    qo.copy_(q)
    got = go(qo, k.cuda(), v.cuda())
    ref.check_attend(got, q, k, v, table, context, parents, what="queries off the boundary")
    oo = torch.zeros(*q.shape[:3], dim + 1, dtype=dtype, device="cuda")[..., 1:]
    got = go(q.cuda(), k.cuda(), v.cuda(), out=oo)
    ref.check_attend(got, q, k, v, table, context, parents, what="outputs off the boundary")


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 3.0])
def test_scales(capi, scale):
    check(capi, *case(2, 6, 1, 4, 64, 16, [300, 5], torch.float16, True, seed=14), scale=scale)


def test_scores_of_every_size(capi):
    """Maxima that rise from tile to tile and jump up and down by far more than the exponential's range."""
    q, k, v, table, context, parents, _ = case(2, 4, 1, 2, 64, 16, [1500, 700], torch.bfloat16, True, seed=15)
    for b in range(2):
        for pos in range(int(context[b]) + 4):
            k[int(table[b, pos // 16]), pos % 16] *= [0.01, 30.0, 0.5, -20.0, 1.0][pos // 130 % 5] * (1 + pos / 1000)
    check(capi, q, k, v, table, context, parents)


def test_long_context_and_a_bound_that_is_too_small(capi):
    c = case(1, 3, 1, 2, 64, 64, [70001], torch.float16, True, seed=16)
    a = check(capi, *c, max_context=70001)
    for bound in (1, 5000, 200000):
        check(capi, *c, max_context=bound)
    assert a[0].shape == (1, 3, 2, 64)


@pytest.mark.parametrize("batch,nodes,kv_heads,group,dim,top", [(1500, 3, 1, 2, 64, 2500), (700, 1, 3, 1, 128, 300), (40, 70, 2, 4, 64, 4000), (3, 128, 2, 8, 128, 9000)])
def test_many_sequences_of_every_length(capi, batch, nodes, kv_heads, group, dim, top):
    """Long lists of tiles, several sequences a thread of the scan, several groups of rows a head: against the general kernel,
    which takes outputs off the 16-byte boundary.  Both are off the formula by at most (2 rel + t) sum p|v| + t |o| with t half a
    step of 16 bits and rel of 32-bit roundings (far below t here): by less than 3 t max|v| each."""
    g = torch.Generator(device="cuda").manual_seed(batch)
    context = (torch.rand(batch, generator=g, device="cuda") ** 2 * (top + 1)).int()
    used = torch.randint(0, nodes + 1, (batch,), generator=g, device="cuda", dtype=torch.int32)
    page, wide = 16, -(-(top + nodes) // 16)
    need = (context + used + page - 1) // page
    pool = int(need.sum()) + 3
    order = torch.randperm(pool, generator=g, device="cuda")
    at = torch.arange(wide, device="cuda")[None]
    table = torch.where(at < need[:, None], order[(need.cumsum(0)[:, None] - need[:, None] + at).clamp(max=pool - 1).long()], -1).to(torch.int32)
    k, v = (torch.empty(pool, page, kv_heads, dim, dtype=torch.float16, device="cuda").normal_(generator=g) for _ in range(2))
    q = torch.randn(batch, nodes, kv_heads * group, dim, generator=g, device="cuda").half()
    parents = ref.random_tree(batch, nodes, torch.Generator().manual_seed(1)).cuda()
    args = dict(parents=parents, num_nodes=used, return_lse=True, max_context=top)
    fast = capi.tree_attention(q, k, v, table, context, **args)
    odd = torch.zeros(batch, nodes, kv_heads * group, dim + 1, dtype=torch.float16, device="cuda")[..., 1:]
    slow = capi.tree_attention(q, k, v, table, context, out=odd, **args)
    assert ((fast[0].float() - slow[0].float()).abs() <= 6 * 2.0**-11 * float(v.abs().max())).all()
    live = torch.isfinite(slow[1])
    assert torch.equal(live, torch.isfinite(fast[1])) and ((fast[1] - slow[1])[live].abs() <= 1e-4).all()


def test_calls_at_the_same_time(capi):
    """Two streams, each with scratch memory of its own."""
    cs = [[None if t is None else t.cuda() for t in case(2, 8, 2, 4, 128, 16, lengths, torch.float16, True, seed=30 + i)] for i, lengths in enumerate(([9000, 5000], [7000, 8000]))]
    want = [capi.tree_attention(*c[:5], parents=c[5]) for c in cs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cs]
    got = [[], []]
    for _ in range(10):
        for i, (st, c) in enumerate(zip(streams, cs)):
            with torch.cuda.stream(st):
                got[i].append(capi.tree_attention(*c[:5], parents=c[5]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in got[i])


def test_wrapper_refusals(capi):
    q, k, v, table, context, parents, _ = [None if t is None else t.cuda() for t in case(2, 4, 1, 2, 64, 16, [40, 9], torch.float16, True, seed=33)]
    for bad in (dict(context=context.long()), dict(context=context[:1]), dict(parents=parents.long()), dict(parents=parents[:, :3].contiguous()),
                dict(num_nodes=context.float()), dict(out=torch.empty_like(q)[:, :2]), dict(out=q.float())):
        with pytest.raises(ValueError):
            capi.tree_attention(**(dict(q=q, k_cache=k, v_cache=v, page_table=table, context=context) | bad))
    with pytest.raises(RuntimeError):
        capi.tree_attention(q, k, v, table.cpu(), context)
    with pytest.raises(capi.VkopError) as e:
        capi.tree_attention(q, k, v, table, context, scale=float("inf"))
    assert e.value.status == capi.INVALID_ARG
    with pytest.raises(capi.VkopError):
        capi.tree_attention(q.expand(2, 4, 2, 64).repeat(1, 40, 1, 1), k, v, table, context)


def test_a_context_past_the_table(capi):
    """Lengths that the table cannot hold: the positions it has are attended, the drafted ones are out of reach."""
    for dim in (64, 80):
        q, k, v, table, context, parents, _ = case(2, 4, 1, 2, dim, 16, [400, 90], torch.float16, True, seed=23)
        far = torch.tensor([2**31 - 1, 100000], dtype=torch.int32)
        table[table < 0] = 1 << 20
        got = run(capi, q, k, v, table, far, parents)
        pages = table.shape[1] * 16
        # the same as a context that ends with the table, without drafted positions (their pages are not there)
        wide = torch.cat([table, torch.full((2, 1), -1, dtype=torch.int32)], 1)
        ref.check_attend(got, q, k, v, wide, torch.full((2,), pages, dtype=torch.int32), parents, what="past the table")


def test_offsets_past_32_bits(capi):
    """Pages more than 2^31 elements into the cache."""
    pages, page, dim = 70000, 16, 128
    k = torch.empty(pages, page, 16, dim, dtype=torch.float16, device="cuda")
    v = torch.empty(pages, page, 16, dim, dtype=torch.float16, device="cuda")
    assert k.numel() > 2**31
    g = torch.Generator().manual_seed(18)
    use = [69999, 5, 66000]
    small_k, small_v = (torch.randn(3, page, 16, dim, generator=g).half() for _ in range(2))
    for i, p in enumerate(use):
        k[p], v[p] = small_k[i].cuda(), small_v[i].cuda()
    q = torch.randn(1, 4, 16, dim, generator=g).half()
    context = torch.tensor([40], dtype=torch.int32)
    got = capi.tree_attention(q.cuda(), k, v, torch.tensor([use], dtype=torch.int32).cuda(), context.cuda(), return_lse=True)
    ref.check_attend(got, q, small_k, small_v, torch.tensor([[0, 1, 2]], dtype=torch.int32), context, what="far pages")


def test_repeats_give_the_same_bits(capi):
    c = [None if t is None else t.cuda() for t in case(3, 20, 2, 4, 128, 16, [2000, 900, 33], torch.bfloat16, True, seed=21)]
    first = capi.tree_attention(*c[:5], parents=c[5])
    for _ in range(5):
        assert torch.equal(capi.tree_attention(*c[:5], parents=c[5]), first)


def test_workspaces_streams_and_graphs(capi):
    c = [None if t is None else t.cuda() for t in case(2, 8, 2, 4, 128, 16, [3000, 1800], torch.float16, True, seed=22)]
    want = capi.tree_attention(*c[:5], parents=c[5])
    need = capi.tree_attention_workspace_bytes(*c[:4])
    assert need > 0
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # scratch may hold anything (these are NaNs)
    assert torch.equal(capi.tree_attention(*c[:5], parents=c[5], workspace=ws), want)
    with pytest.raises(capi.VkopError) as e:
        capi.tree_attention(*c[:5], parents=c[5], workspace=ws[: need - 16])
    assert e.value.status == capi.WORKSPACE_TOO_SMALL
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = capi.tree_attention(*c[:5], parents=c[5])
    side.synchronize()
    assert torch.equal(got, want)
    # two captured calls on one workspace, replayed in turn with other contexts
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(capi.tree_attention(*c[:5], parents=c[5], workspace=ws))
        graphs.append(graph)
    for lengths in ([3000, 1800], [17, 2000]):
        c[4].copy_(torch.tensor(lengths, dtype=torch.int32))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = capi.tree_attention(*c[:5], parents=c[5])
        assert all(torch.equal(o, want) for o in outs)


def test_empty_batch(capi):
    k = torch.zeros(2, 16, 1, 64, dtype=torch.float16, device="cuda")
    out = capi.tree_attention(torch.zeros(0, 3, 2, 64, dtype=torch.float16, device="cuda"), k, k, torch.zeros(0, 4, dtype=torch.int32, device="cuda"),
                              torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert out.shape == (0, 3, 2, 64)
