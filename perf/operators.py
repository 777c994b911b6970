"""What the operators of a speculative decoding step cost: verification of drafted tokens (vkop_b200.capi.draft_verify),
attention of a tree of drafted tokens over a paged cache (tree_attention) and the move of the accepted path's cache rows
(cache_compact).

Conventions shared by the three: node 0 of a sequence is the last token already decided, nodes 1.. are drafted, a node's
parent has a smaller number, node i's key and value lie in the cache at position context + i.

`own` False: the operators written out in elementary torch operations; True: the framework's calls.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # -- verification: rows of the vocabulary-selection workloads (128256 columns f32, 256000 columns bf16)
        # one user, four drafted tokens in a chain with the draft's distributions: latency
        dict(name="verify_chain_one", op="verify", batch=1, nodes=5, vocab=128256, dtype="f32", tree=False, draft=True, ragged=False),
        # a full serving batch of the 64-row workload, five drafted tokens each
        dict(name="verify_chain_batch", op="verify", batch=64, nodes=6, vocab=128256, dtype="f32", tree=False, draft=True, ragged=False),
        # trees of tokens drafted with certainty (the best few of a small head), padded batch
        dict(name="verify_tree_certain", op="verify", batch=32, nodes=32, vocab=32000, dtype="f16", tree=True, draft=False, ragged=True),
        # trees drawn from the draft's distributions over the largest vocabulary
        dict(name="verify_tree_drawn", op="verify", batch=16, nodes=26, vocab=256000, dtype="bf16", tree=True, draft=True, ragged=False),
        # -- attention
        # a single new token of one user: latency
        dict(name="attend_one_token", op="attend", batch=1, nodes=1, kv_heads=8, group=4, dim=128, page=16, context=1023, dtype="bf16", tree=False, ragged=False, lse=False),
        # a serving batch with chains of five, contexts of every length up to 8192
        dict(name="attend_chain_batch", op="attend", batch=32, nodes=5, kv_heads=8, group=4, dim=128, page=16, context=8192, dtype="bf16", tree=False, ragged=True, lse=False),
        # many heads without sharing, short rows of 64, middle-sized trees
        dict(name="attend_tree_heads", op="attend", batch=16, nodes=26, kv_heads=16, group=1, dim=64, page=32, context=3001, dtype="f16", tree=True, ragged=True, lse=True),
        # large trees: 256 rows share a head's keys
        dict(name="attend_tree_wide", op="attend", batch=8, nodes=64, kv_heads=8, group=4, dim=128, page=64, context=16384, dtype="bf16", tree=True, ragged=False, lse=False),
        # one long document
        dict(name="attend_tree_long", op="attend", batch=1, nodes=32, kv_heads=8, group=8, dim=128, page=64, context=131071, dtype="f16", tree=True, ragged=False, lse=True),
        # -- moving the accepted rows: one layer at a time, and all layers of a cache in one call
        dict(name="compact_layer", op="compact", batch=4, nodes=16, layers=1, kv_heads=8, dim=128, page=16, context=255, dtype="bf16"),
        dict(name="compact_cache", op="compact", batch=64, nodes=64, layers=16, kv_heads=8, dim=128, page=16, context=200, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["verify", "attend", "attend", "compact"])
    if op == "verify":
        tree, vocab, dtype = rng.random() < 0.5, _log(rng, 1000, 256000), rng.choice(["f32", "f16", "bf16"])
        nodes = _log(rng, 1, 64) if tree else _log(rng, 1, 16)
        most = max(1, min(64, 190_000_000 // (nodes * vocab * (4 if dtype == "f32" else 2))))
        return dict(op=op, batch=_log(rng, 1, most), nodes=nodes, vocab=vocab, dtype=dtype, tree=tree, draft=rng.random() < 0.6, ragged=rng.random() < 0.5)
    if op == "attend":
        kv_heads, group, dim = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 4, 5, 8]), rng.choice([64, 128])
        tree, context = rng.random() < 0.6, _log(rng, 1, 131072)
        nodes = _log(rng, 1, 64) if tree else _log(rng, 1, 16)
        most = 260_000_000 // (context * kv_heads * dim)
        most = min(most, int(1.3e11 // (4 * nodes * group * kv_heads * context * dim)))
        return dict(op=op, batch=_log(rng, 1, max(1, min(64, most))), nodes=nodes, kv_heads=kv_heads, group=group, dim=dim, page=rng.choice([8, 16, 24, 32, 64, 128]),
                    context=context, dtype=rng.choice(["f16", "bf16"]), tree=tree, ragged=rng.random() < 0.5, lse=rng.random() < 0.5)
    return dict(op=op, batch=_log(rng, 1, 64), nodes=_log(rng, 2, 64), layers=_log(rng, 1, 16), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]),
                page=rng.choice([8, 16, 24, 32, 64]), context=_log(rng, 1, 200), dtype=rng.choice(["f16", "bf16"]))


# ---------------------------------------------------------------------------------------------------------------------
# inputs


def _parents(case, g):
    b, n = case["batch"], case["nodes"]
    at = torch.arange(n, device="cuda")
    if case.get("tree"):  # every earlier node is as likely a parent: depth about log(n)
        up = (torch.rand(b, n, generator=g, device="cuda") * at).long().clamp(max=(at - 1).clamp(min=0))
    else:
        up = (at - 1).expand(b, n)
    return up.clamp(min=0).to(torch.int32).contiguous()


def _nodes(case, g):
    """Nodes in use a sequence, or None where all are."""
    if not case.get("ragged"):
        return None
    return torch.randint(1, case["nodes"] + 1, (case["batch"],), generator=g, device="cuda", dtype=torch.int32)


def _prepare_verify(case, g):
    b, n, v, dt = case["batch"], case["nodes"], case["vocab"], DTYPES[case["dtype"]]
    target = torch.empty(b, n, v, dtype=dt, device="cuda")
    draft = torch.empty(b, n, v, dtype=dt, device="cuda") if case["draft"] else None
    parents, tokens = _parents(case, g), torch.zeros(b, n, dtype=torch.int32, device="cuda")
    guess = torch.empty(b, n, n, dtype=torch.int64, device="cuda")
    for i in range(b):  # a sequence at a time: no second copy of all rows in 32 bits
        x = torch.randn(n, v, generator=g, device="cuda")
        x.scatter_add_(1, torch.randint(0, v, (n, 20), generator=g, device="cuda"), 8 + torch.randn(n, 20, generator=g, device="cuda"))
        y = x + 0.5 * torch.randn(n, v, generator=g, device="cuda")
        q = torch.softmax(y / 0.8, -1)
        target[i] = torch.softmax(x / 0.8, -1).to(dt)
        if draft is not None:
            draft[i] = q.to(dt)
        guess[i] = torch.multinomial(q, n, replacement=True, generator=g)  # row r: what r's children may be
    at = torch.arange(n, device="cuda").expand(b, n)
    tokens[:] = guess.gather(1, parents.long()[:, :, None].expand(b, n, n)).gather(2, at[:, :, None])[:, :, 0].to(torch.int32)
    return dict(target=target, draft=draft, tokens=tokens, parents=parents if case["tree"] else None, num_nodes=_nodes(case, g),
                u=torch.rand(b, n, generator=g, device="cuda"))


def _table(lengths, pages_a_sequence, pool, g):
    """Pages in random order, as a cache in use has them; entries behind a sequence's last page are -1."""
    b = lengths.numel()
    order = torch.randperm(pool, generator=g, device="cuda")[: b * pages_a_sequence].view(b, pages_a_sequence)
    used = torch.arange(pages_a_sequence, device="cuda")[None] < lengths[:, None]
    return torch.where(used, order, -1).to(torch.int32).contiguous()


def _prepare_attend(case, g):
    b, n, h, d, page, dt = case["batch"], case["nodes"], case["kv_heads"], case["dim"], case["page"], DTYPES[case["dtype"]]
    top = case["context"]
    context = torch.randint(0 if top < 4 else top // 4, top + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else torch.full((b,), top, dtype=torch.int32, device="cuda")
    wide = -(-(top + n) // page)
    pool = b * wide + 3
    cache = [torch.empty(pool, page, h, d, dtype=dt, device="cuda").normal_(generator=g) for _ in range(2)]
    q = 2 * torch.randn(b, n, h * case["group"], d, generator=g, device="cuda")
    return dict(q=q.to(dt), k=cache[0], v=cache[1], table=_table((context + n + page - 1) // page, wide, pool, g), context=context,
                parents=_parents(case, g) if case["tree"] else None, num_nodes=_nodes(case, g), scale=1 / math.sqrt(d), max_context=top, lse=case["lse"])


def _prepare_compact(case, g):
    b, n, h, d, page, layers, dt = case["batch"], case["nodes"], case["kv_heads"], case["dim"], case["page"], case["layers"], DTYPES[case["dtype"]]
    top = case["context"]
    context = torch.randint(top // 2, top + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    wide = -(-(top + n) // page)
    pool = b * wide + 3
    cache = [torch.empty(layers, pool, page, h, d, dtype=dt, device="cuda").normal_(generator=g) for _ in range(2)]
    # the accepted path: node 0 and an ascending choice of the others, as a walk down a tree leaves it
    some = min(n, 12)
    count = torch.randint(1, some + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
    pick = 1 + torch.rand(b, n - 1, generator=g, device="cuda").argsort(1)[:, : some - 1]
    at = torch.arange(some, device="cuda")[None]
    pick = torch.where(at[:, 1:] < count[:, None], pick, n).sort(1)[0]
    path = torch.full((b, n), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    path[:, 1:some] = torch.where(at[:, 1:] < count[:, None], pick, -1).to(torch.int32)
    return dict(k=cache[0], v=cache[1], table=_table((context + n + page - 1) // page, wide, pool, g), context=context, path=path, count=count)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"verify": _prepare_verify, "attend": _prepare_attend, "compact": _prepare_compact}[case["op"]](case, g) | {"op": case["op"]}


# ---------------------------------------------------------------------------------------------------------------------
# plain forms


def _verify(s):
    """64 bits: every decision is a comparison with a border."""
    p, q, tokens, u = s["target"], s["draft"], s["tokens"].long(), s["u"].double()
    b, n, v = p.shape
    row = torch.arange(b, device=p.device)
    parents = s["parents"].long() if s["parents"] is not None else (torch.arange(n, device=p.device) - 1).expand(b, n)
    used = s["num_nodes"].long() if s["num_nodes"] is not None else torch.full((b,), n, device=p.device)
    cur = torch.zeros(b, dtype=torch.long, device=p.device)
    c, mass = torch.zeros(b, dtype=torch.double, device=p.device), torch.ones(b, dtype=torch.double, device=p.device)
    gone = torch.zeros(b, n, dtype=torch.bool, device=p.device)  # rejected children of the present node
    path, chance = torch.full((b, n), -1, dtype=torch.int32, device=p.device), torch.zeros(b, n, device=p.device)
    path[:, 0] = torch.where(used > 0, 0, -1)
    count = (used > 0).to(torch.int32)
    for i in range(1, n):  # each test depends on the one before
        tested = (parents[:, i] == cur) & (i < used)
        t = tokens[:, i]
        pt = p[row, cur, t].double()
        if q is not None:
            qt = q[row, cur, t].double()
            left, scaled = (pt - c * qt).clamp(min=0), mass * qt
        else:
            left, scaled = torch.where((gone & (tokens == t[:, None])).any(1), 0, pt), mass
        took = tested & (u[:, i] * scaled < left)
        chance[:, i] = torch.where(tested, torch.where(left >= scaled, (left > 0).double(), left / scaled), 0).float()
        path[row, count.long().clamp(max=n - 1)] = torch.where(took, i, path[row, count.long().clamp(max=n - 1)]).to(torch.int32)
        lost = tested & ~took
        if q is not None:
            c = torch.where(lost, c + mass, c)
            mass = torch.where(lost, (p[row, cur].double() - c[:, None] * q[row, cur].double()).clamp(min=0).sum(1), mass)
        else:
            mass = torch.where(lost, (mass - left).clamp(min=0), mass)
            gone[:, i] = lost
        count += took.to(torch.int32)
        cur = torch.where(took, i, cur)
        c, mass = torch.where(took, 0, c), torch.where(took, 1, mass)
        gone &= ~took[:, None]
    full = p[row, cur].double()
    if q is not None:
        w = (full - c[:, None] * q[row, cur].double()).clamp(min=0)
    else:
        w = full.scatter_reduce(1, tokens, torch.where(gone, 0.0, 1.0).double(), "prod")
    w = torch.where((w.sum(1) > 0)[:, None], w, full)
    run = w.cumsum(1)
    token = (run <= u[:, :1] * run[:, -1:]).sum(1)
    return path, count, torch.where((count > 0) & (run[:, -1] > 0), token, -1).to(torch.int32), chance


def _sees(s, n):
    """[b, n, n]: whether node i has node j above it or is j."""
    b = s["q"].shape[0]
    if s["parents"] is None:
        return torch.ones(n, n, dtype=torch.bool, device="cuda").tril().expand(b, n, n)
    up = torch.zeros(b, n, n, device="cuda")
    up.scatter_(2, s["parents"].long()[:, :, None], 1)
    up[:, 0] = 0
    see = torch.eye(n, device="cuda").expand(b, n, n)
    for _ in range(max(1, n - 1).bit_length()):  # ancestors within 1, 2, 4, ... steps
        see = ((see + up @ see) > 0).float()
        up = ((up @ up) > 0).float()
    return see > 0


def _attend(s):
    q, k, v, table, context = s["q"].float(), s["k"], s["v"], s["table"].long(), s["context"].long()
    b, n, heads, d = q.shape
    page, h = k.shape[1], k.shape[2]
    length = table.shape[1] * page
    used = s["num_nodes"].long() if s["num_nodes"] is not None else torch.full((b,), n, device="cuda")
    keys = k[table.clamp(min=0)].view(b, length, h, d).permute(0, 2, 3, 1).float()
    values = v[table.clamp(min=0)].view(b, length, h, d).permute(0, 2, 1, 3).float()
    at = torch.arange(length, device="cuda")
    draft = at[None] - context[:, None]  # the node at a position, where it is one
    see = _sees(s, n).gather(2, draft.clamp(0, n - 1)[:, None].expand(b, n, length)) & ((draft >= 0) & (draft < used[:, None]))[:, None]
    see = (see | (draft < 0)[:, None]) & (torch.arange(n, device="cuda") < used[:, None])[:, :, None]
    rows = q.view(b, n, h, heads // h, d).permute(0, 2, 3, 1, 4).reshape(b, h, -1, d) * s["scale"]
    x = (rows @ keys).view(b, h, heads // h, n, length).masked_fill_(~see[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top > -math.inf, top, 0)).exp_()
    total = x.sum(-1, keepdim=True)
    # entries past a sequence are not numbers that count: their weight is 0, and so is their value here
    values = values.masked_fill(~(draft < used[:, None])[:, None, :, None], 0)
    out = (x.view(b, h, -1, length) @ values).view(b, h, heads // h, n, d) / torch.where(total > 0, total, 1)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, n, heads, d).to(s["q"].dtype)
    return (out, (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(b, n, heads)) if s["lse"] else out


def _compact(s):
    k, v, table, context, path, count = s["k"], s["v"], s["table"].long(), s["context"].long(), s["path"].long(), s["count"].long()
    page, n = k.shape[2], path.shape[1]
    at = torch.arange(n, device="cuda").expand_as(path)
    seq, rank = torch.nonzero((at > 0) & (at < count[:, None]), as_tuple=True)
    old, new = context[seq] + path[seq, rank], context[seq] + rank
    old, new = (table[seq, old // page], old % page), (table[seq, new // page], new % page)
    k[:, new[0], new[1]] = k[:, old[0], old[1]]
    v[:, new[0], new[1]] = v[:, old[0], old[1]]
    return k, v, (context + count).to(torch.int32)


def run(s):
    if own:
        from vkop_b200 import capi

        if s["op"] == "verify":
            return capi.draft_verify(s["target"], s["tokens"], s["u"], draft=s["draft"], parents=s["parents"], num_nodes=s["num_nodes"], chances=True)
        if s["op"] == "attend":
            return capi.tree_attention(s["q"], s["k"], s["v"], s["table"], s["context"], parents=s["parents"], num_nodes=s["num_nodes"], scale=s["scale"],
                                       max_context=s["max_context"], return_lse=s["lse"])
        return s["k"], s["v"], capi.cache_compact(s["k"], s["v"], s["table"], s["context"], s["path"], s["count"])
    return {"verify": _verify, "attend": _attend, "compact": _compact}[s["op"]](s)


# ---------------------------------------------------------------------------------------------------------------------


def work(case):
    b, n = case["batch"], case["nodes"]
    size = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "verify":  # the row that the last token is drawn from (and the draft's, where there is one), a value of each for a test, the answers
        rows = 2 if case["draft"] else 1
        return {"bytes": b * (rows * case["vocab"] * size + n * (rows * size + 24)), "flops": b * case["vocab"] * (4.0 if case["draft"] else 2.0)}
    h, d = case["kv_heads"], case["dim"]
    if case["op"] == "attend":
        # mean lengths: contexts of a ragged batch lie between a quarter of the longest and the longest, its node counts between 1 and all
        mean = case["context"] * (0.625 if case["ragged"] and case["context"] >= 4 else 1.0)
        live = (n + 1) / 2 if case["ragged"] else n
        heads = h * case["group"]
        return {"bytes": b * (2 * (mean + live) * h * d * size + 2 * n * heads * d * size + (4 * n * heads if case["lse"] else 0)),
                "flops": 4.0 * b * live * heads * d * (mean + (live + 1) / 2)}
    moved = (min(n, 12) + 1) / 2 - 1  # accepted drafted tokens a sequence, on average
    return {"bytes": max(1.0, b * (case["layers"] * 2 * 2 * moved * h * d * size + 8 * n)), "flops": 0.0}


# ---------------------------------------------------------------------------------------------------------------------
# the same in 64 bits, sequence by sequence, straight from the definitions


def _exact_verify(s):
    p, q = s["target"], s["draft"]
    b, n, v = p.shape
    paths, counts, last, chances = [], [], [], []
    for i in range(b):
        tokens, u = s["tokens"][i].tolist(), s["u"][i].double().tolist()
        up = s["parents"][i].tolist() if s["parents"] is not None else [j - 1 for j in range(n)]
        used = int(s["num_nodes"][i]) if s["num_nodes"] is not None else n
        node, path, chance = 0, [0], [0.0] * n
        rest = p[i, 0].double()  # the distribution that the present node's token has, given the rejections so far
        while True:
            took = None
            for j in [j for j in range(1, used) if up[j] == node]:
                have = float(rest[tokens[j]])
                asked = float(q[i, node, tokens[j]].double()) if q is not None else 1.0
                chance[j] = (1.0 if have > 0 else 0.0) if have >= asked else have / asked
                if u[j] * asked < have:
                    took = j
                    break
                if q is not None:
                    rest = (rest - q[i, node].double()).clamp(min=0)
                    rest = rest / rest.sum() if float(rest.sum()) > 0 else rest
                else:
                    total = max(1.0 - have, 0.0)
                    rest = rest.clone()
                    rest[tokens[j]] = 0
                    rest = rest / total if total > 0 else rest
            if took is None:
                break
            node, rest = took, p[i, took].double()
            path.append(took)
        if not float(rest.sum()) > 0:
            rest = p[i, node].double()
        run = rest.cumsum(0)
        last.append(int((run <= u[0] * run[-1]).sum()))
        paths.append(path + [-1] * (n - len(path)))
        counts.append(len(path))
        chances.append(chance)
    whole = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return whole(paths), whole(counts), whole(last), torch.tensor(chances, dtype=torch.float64)


def _exact_attend(s):
    b, n, heads, d = s["q"].shape
    h, page = s["k"].shape[2], s["k"].shape[1]
    out, lse = torch.zeros(b, n, heads, d, dtype=torch.float64, device="cuda"), torch.full((b, n, heads), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(b):
        c, used = int(s["context"][i]), int(s["num_nodes"][i]) if s["num_nodes"] is not None else n
        see = torch.zeros(used, used, dtype=torch.bool)
        up = s["parents"][i].tolist() if s["parents"] is not None else [j - 1 for j in range(n)]
        for j in range(used):
            if j:
                see[j] = see[up[j]]
            see[j, j] = True
        at = torch.arange(c + used, device="cuda")
        pages, slots = s["table"][i].long()[at // page], at % page
        for g in range(h):
            k, v = s["k"][pages, slots, g].double(), s["v"][pages, slots, g].double()
            for r in range(heads // h):
                x = s["q"][i, :used, g * (heads // h) + r].double() @ k.T * s["scale"]
                x[:, c:] = x[:, c:].masked_fill(~see.cuda(), -math.inf)
                lse[i, :used, g * (heads // h) + r] = torch.logsumexp(x, -1)
                out[i, :used, g * (heads // h) + r] = torch.softmax(x, -1) @ v
    return (out, lse) if s["lse"] else out


def _exact_compact(s):
    k, v = s["k"].double(), s["v"].double()
    page = k.shape[2]
    for i in range(s["count"].numel()):
        c, table = int(s["context"][i]), s["table"][i].tolist()
        for rank, node in enumerate(s["path"][i, : int(s["count"][i])].tolist()):
            old, new = c + node, c + rank  # ascending, so that a row is read before another is written over it
            for x in (k, v):
                x[:, table[new // page], new % page] = x[:, table[old // page], old % page]
    return k, v, s["context"] + s["count"]


def exact(case, seed):
    s = prepare(case, seed)
    return {"verify": _exact_verify, "attend": _exact_attend, "compact": _exact_compact}[case["op"]](s)
