"""Verification of drafted tokens: decisions are whole numbers and have to equal those of a sequential 64-bit walk."""
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


def make(batch, nodes, vocab, dtype, tree, draft_rows, seed, index=torch.int32, near=0.7):
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(batch, nodes, vocab, generator=g)
    p = torch.softmax(x, -1)
    q = torch.softmax(x + near * torch.randn(batch, nodes, vocab, generator=g), -1)
    parents = ref.random_tree(batch, nodes, g) if tree else None
    up = (parents.long() if tree else (torch.arange(nodes) - 1).clamp(min=0).expand(batch, nodes)).clamp(min=0)
    tokens = torch.zeros(batch, nodes, dtype=index)
    for b in range(batch):
        for i in range(1, nodes):
            tokens[b, i] = torch.multinomial(q[b, up[b, i]], 1, generator=g)[0]
    u = torch.rand(batch, nodes, generator=g)
    return p.to(dtype), q[:, :draft_rows].to(dtype).contiguous() if draft_rows else None, tokens, u, parents


def check(capi, p, q, tokens, u, parents=None, num_nodes=None):
    dev = [None if t is None else t.cuda() for t in (p, tokens, u, q, parents, num_nodes)]
    path, count, token, chance = capi.draft_verify(*dev[:3], draft=dev[3], parents=dev[4], num_nodes=dev[5], chances=True)
    torch.cuda.synchronize()
    want = ref.verify(p, tokens, u, q, parents, num_nodes)
    assert np.array_equal(path.cpu().numpy(), want[0])
    assert np.array_equal(count.cpu().numpy(), want[1])
    assert token.dtype == tokens.dtype and np.array_equal(token.cpu().numpy(), want[2])
    # one rounding to 32 bits (half a step, 2^-24), 64-bit sums of up to 2^18 terms (2^-35) and their quotient
    assert np.all(np.abs(chance.cpu().numpy() - want[3]) <= 2.0**-23 * want[3])
    return path, count, token, chance


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,nodes,vocab", [(1, 1, 1), (2, 3, 7), (3, 5, 1000), (5, 33, 4099), (2, 4, 128257), (150, 3, 517), (300, 2, 64)])
@pytest.mark.parametrize("tree,rows", [(False, "all"), (True, "all"), (True, 0), (False, 0), (True, "some")])
def test_matches_the_sequential_walk(capi, dtype, batch, nodes, vocab, tree, rows):
    rows = {"all": nodes, "some": (nodes + 1) // 2}.get(rows, rows)
    p, q, tokens, u, parents = make(batch, nodes, vocab, dtype, tree, rows, seed=batch * 1000 + nodes)
    g = torch.Generator().manual_seed(5)
    used = torch.randint(0, nodes + 1, (batch,), generator=g, dtype=torch.int32)
    check(capi, p, q, tokens, u, parents)
    check(capi, p, q, tokens, u, parents, used)


def test_many_siblings_exhaust_a_node(capi):
    """All children of node 0: repeated residuals of one distribution, and certain drafts with tokens drawn twice."""
    p, q, tokens, u, _ = make(6, 40, 300, torch.float32, False, 40, seed=2, near=2.0)
    parents = torch.zeros(6, 40, dtype=torch.int32)
    g = torch.Generator().manual_seed(6)
    for b in range(6):
        tokens[b, 1:] = torch.multinomial(q[b, 0], 39, replacement=True, generator=g)
    u[:, 1:] = 0.97 + 0.03 * u[:, 1:]  # rejections mostly
    _, _, _, chance = check(capi, p, q, tokens, u, parents)
    assert (chance[:, 2:] > 0).any()  # a residual of a residual was tested
    check(capi, p, None, tokens, u, parents)
    tokens[:, 1:] = torch.randint(0, 5, (6, 39), generator=g)
    check(capi, p, None, tokens, u, parents)


def test_more_nodes_than_threads(capi):
    p, _, _, u, _ = make(1, 1, 50, torch.float32, False, 0, seed=3)
    n = 1024
    p = p.expand(1, n, 50).contiguous()
    tokens = torch.arange(n, dtype=torch.int32)[None] % 49  # token 49 is drafted by nobody
    u = torch.rand(1, n, generator=torch.Generator().manual_seed(4)) * 1e-6 + 0.999
    for parents in (torch.zeros(1, n, dtype=torch.int32), torch.where(torch.arange(n) > 600, 600, -1)[None].to(torch.int32)):
        _, _, token, _ = check(capi, p, None, tokens, u, parents)
    # children of node 0 numbered above the thread count only
    check(capi, p, None, tokens, u, torch.where(torch.arange(n) > 600, 0, -1)[None].to(torch.int32))


def test_equal_distributions_are_accepted_and_leave_nothing(capi):
    p, _, tokens, u, _ = make(4, 6, 1000, torch.float32, False, 0, seed=7)
    tokens = torch.stack([torch.multinomial(p[b, 0], 6, replacement=True, generator=torch.Generator().manual_seed(b)) for b in range(4)]).to(torch.int32)
    q = p.clone()
    path, count, _, chance = check(capi, p, q, tokens, u)
    assert (count == 6).all() and (chance[:, 1:] == 1).all()
    # a token that neither distribution holds is rejected, and the residual is empty: the last token comes from p itself
    p[:, 0, 3] = 0
    q = p.clone()
    tokens[:, 1] = 3
    _, count, token, _ = check(capi, p, q, tokens, u)
    assert (count == 1).all() and (token >= 0).all() and (token != 3).all()


def test_ends_of_the_uniform_range_and_degenerate_rows(capi):
    p = torch.zeros(5, 2, 4000)
    p[0, 0, 1234] = 1.0                      # one token holds everything
    p[1, 0, 5] = p[1, 0, 3999] = 0.5
    p[2, 0] = 0.0                            # nothing to draw
    p[3, 0] = torch.tensor(float("nan"))     # not numbers: nothing either
    p[4, 0, :6] = torch.tensor([1e-40, -1.0, float("nan"), 0.25, 1e-40, -0.0])
    tokens = torch.tensor([[0, 1234], [0, 17], [0, 0], [0, 0], [0, 0]], dtype=torch.int64)
    for first in (0.0, 0.49999, 0.5, 1 - 2.0**-24):
        u = torch.tensor([[first, 0.0]] * 5)
        _, _, token, _ = check(capi, p, None, tokens, u)
        assert token[2] == -1 and token[3] == -1 and token[4] == 3
    # a number outside [0, 1) still gives a token that the distribution holds
    u = torch.tensor([[1.0, 1.0], [7.0, 1.0], [1.0, 1.0], [1.0, 1.0], [float("nan"), 1.0]])
    _, _, token, _ = capi.draft_verify(p.cuda(), tokens.cuda(), u.cuda(), chances=True)
    assert token.tolist() == [1234, 3999, -1, -1, 3]


def test_residuals_of_entries_that_are_no_probabilities(capi):
    p, q, tokens, u, _ = make(4, 3, 900, torch.float32, False, 3, seed=12, near=2.0)
    nan, inf = float("nan"), float("inf")
    odd = torch.tensor([nan, -1.0, 1e-40, 0.0, -0.0, -inf, 2.0**-126])
    for b in range(4):
        p[b, 0, 10 * b:10 * b + 7], q[b, 0, 50 + b:57 + b] = odd, odd.flip(0)
        p[b, 0, 200 + b:207 + b], q[b, 0, 200 + b:207 + b] = odd, odd.roll(2)
    p[3, 0, 400] = inf
    u[:, 1:] = 0.9999
    check(capi, p, q, tokens, u)
    check(capi, p, None, tokens, u)


def test_bad_tokens_and_parents_are_passed_over(capi):
    p, q, tokens, u, parents = make(3, 12, 100, torch.float32, True, 12, seed=11)
    tokens[0, 3], tokens[1, 5], tokens[2, 1] = -1, 100, 1 << 30
    parents[0, 4], parents[1, 6], parents[2, 2], parents[2, 7] = -1, 6, 11, 50
    u[:] = u * 0.2  # acceptances mostly
    check(capi, p, q, tokens, u, parents)
    check(capi, p, None, tokens.to(torch.int64), u, parents, torch.tensor([12, 40, -3], dtype=torch.int32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_strides_and_rows_off_the_vector_boundary(capi, dtype):
    p, q, tokens, u, parents = make(3, 6, 3001, dtype, True, 6, seed=13, near=2.0)
    for shift_p, shift_q in ((1, 1), (3, 2), (0, 1)):
        big_p, big_q = torch.zeros(3, 8, 3010, dtype=dtype, device="cuda"), torch.zeros(4, 6, 3013, dtype=dtype, device="cuda")
        vp, vq = big_p[:, 1:7, shift_p:shift_p + 3001], big_q[1:, :, shift_q:shift_q + 3001]
        vp.copy_(p)
        vq.copy_(q)
        path, count, token = capi.draft_verify(vp, tokens.cuda(), u.cuda(), draft=vq, parents=parents.cuda())
        want = ref.verify(p, tokens, u, q, parents)
        assert np.array_equal(path.cpu().numpy(), want[0]) and np.array_equal(count.cpu().numpy(), want[1])
        assert np.array_equal(token.cpu().numpy(), want[2])


def test_the_tokens_have_the_targets_distribution(capi):
    """First token after node 0, whether drafted or drawn: frequencies of 40000 walks against p (5 sigma)."""
    n = 40000
    p = torch.tensor([0.35, 0.05, 0.25, 0.05, 0.2, 0.1])
    q = torch.tensor([0.1, 0.3, 0.1, 0.3, 0.1, 0.1])
    g = torch.Generator().manual_seed(17)
    parents = torch.zeros(n, 4, dtype=torch.int32)
    for draft in (True, False):
        tokens = torch.multinomial(q.expand(n, 6), 4, replacement=True, generator=g).to(torch.int32)
        u = torch.rand(n, 4, generator=g)
        rows = p.expand(n, 4, 6).contiguous().cuda()
        path, count, token = capi.draft_verify(rows, tokens.cuda(), u.cuda(), draft=q.expand(n, 4, 6).contiguous().cuda() if draft else None, parents=parents.cuda())
        path, count, token = path.cpu().long(), count.cpu(), token.cpu()
        first = torch.where(count > 1, tokens.gather(1, path[:, 1:2].clamp(min=0))[:, 0], token)
        freq = torch.bincount(first.long(), minlength=6) / n
        assert torch.all((freq - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)), (draft, freq)


def test_streams_and_graphs(capi):
    p, q, tokens, u, parents = make(8, 9, 5000, torch.bfloat16, True, 9, seed=19)
    dev = [t.cuda() for t in (p, tokens, u, q, parents)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = capi.draft_verify(*dev[:3], draft=dev[3], parents=dev[4])
    side.synchronize()
    want = ref.verify(p, tokens, u, q, parents)
    assert all(np.array_equal(a.cpu().numpy(), w) for a, w in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = capi.draft_verify(*dev[:3], draft=dev[3], parents=dev[4])
    for seed in (20, 21):
        p, q, tokens, u, parents = make(8, 9, 5000, torch.bfloat16, True, 9, seed=seed)
        for d, t in zip(dev, (p, tokens, u, q, parents)):
            d.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = ref.verify(p, tokens, u, q, parents)
        assert all(np.array_equal(a.cpu().numpy(), w) for a, w in zip(held, want))


def test_calls_at_the_same_time(capi):
    cases = [make(6, 9, 30000, torch.float32, True, 9, seed=40 + i, near=2.0) for i in range(2)]
    want = [ref.verify(p, tokens, u, q, parents) for p, q, tokens, u, parents in cases]
    dev = [[t.cuda() for t in c] for c in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(10):
        for i, (st, (p, q, tokens, u, parents)) in enumerate(zip(streams, dev)):
            with torch.cuda.stream(st):
                got[i].append(capi.draft_verify(p, tokens, u, draft=q, parents=parents))
    torch.cuda.synchronize()
    assert all(np.array_equal(a.cpu().numpy(), w) for i in range(2) for g in got[i] for a, w in zip(g, want[i]))


def test_wrapper_refusals(capi):
    p, q, tokens, u, parents = [t.cuda() for t in make(2, 4, 50, torch.float32, True, 4, seed=44)]
    for bad in (dict(u=u.double()), dict(u=u[:, :3]), dict(tokens=tokens.short()), dict(tokens=tokens.T.contiguous().T), dict(parents=parents.long()),
                dict(draft=q.half()), dict(draft=q[:1]), dict(draft=q[..., :49]), dict(target=p[..., ::2]), dict(target=p[:, :1].expand(2, 4, 50)),
                dict(num_nodes=parents[:, 0])):
        with pytest.raises(ValueError):
            capi.draft_verify(**(dict(target=p, tokens=tokens, u=u, draft=q, parents=parents) | bad))
    with pytest.raises(RuntimeError):
        capi.draft_verify(p, tokens.cpu(), u)
    with pytest.raises(capi.VkopError) as e:  # more distributions than nodes
        capi.draft_verify(p, tokens, u, draft=torch.cat([q, q], 1))
    assert e.value.status == capi.INVALID_ARG


def test_empty_batch(capi):
    path, count, token = capi.draft_verify(torch.zeros(0, 3, 10).cuda(), torch.zeros(0, 3, dtype=torch.int32).cuda(), torch.zeros(0, 3).cuda())
    assert path.shape == (0, 3) and count.shape == (0,) and token.shape == (0,)
