"""Plain 64-bit statements of the speculative decoding operators, sequence by sequence (numpy, CPU), and the bounds that the
tests hold the kernels to."""
from __future__ import annotations

import numpy as np
import torch


def clean(x):
    x = np.asarray(x, np.float64)
    return np.where(x >= 2.0**-126, np.minimum(x, 2.0**128), 0.0)  # NaN compares false


def verify(target, tokens, u, draft=None, parents=None, num_nodes=None):
    """(path, count, token, chance) as the header defines them."""
    target = target.double().cpu().numpy()
    tokens, u = tokens.cpu().numpy(), u.cpu().numpy().astype(np.float64)
    draft = None if draft is None else draft.double().cpu().numpy()
    B, N, V = target.shape
    path, count = np.full((B, N), -1, np.int64), np.zeros(B, np.int64)
    token, chance = np.full(B, -1, np.int64), np.zeros((B, N))
    for b in range(B):
        used = N if num_nodes is None else min(max(int(num_nodes[b]), 0), N)
        if used == 0:
            continue
        up = [i - 1 if parents is None else int(parents[b, i]) for i in range(N)]
        kept, cur = [0], 0
        while True:
            p = clean(target[b, cur])
            q = clean(draft[b, cur]) if draft is not None and cur < draft.shape[1] else None
            c, mass, gone, took = 0.0, 1.0, set(), None
            for i in [i for i in range(1, used) if up[i] == cur and 0 <= tokens[b, i] < V]:
                t = int(tokens[b, i])
                if q is not None:
                    if c > 0:
                        mass = np.maximum(p - c * q, 0).sum()
                    left, scaled = max(p[t] - c * q[t], 0.0), mass * q[t]
                else:
                    left, scaled = 0.0 if t in gone else p[t], mass
                chance[b, i] = float(left > 0) if left >= scaled else left / scaled
                if u[b, i] * scaled < left:
                    took = i
                    break
                if q is not None:
                    c += mass
                else:
                    mass = max(mass - left, 0.0)
                    gone.add(t)
            if took is None:
                break
            cur = took
            kept.append(took)
        w = np.maximum(p - c * q, 0) if q is not None else p.copy()
        w[list(gone)] = 0
        w = w if w.sum() > 0 else p
        run = np.cumsum(w)
        if run[-1] > 0:
            token[b] = min(int((run <= u[b, 0] * run[-1]).sum()), int(np.nonzero(w)[0][-1]))
        path[b, : len(kept)] = kept
        count[b] = len(kept)
    return path, count, token, chance


def ancestors(parents, n):
    """sees[i, j]: node j is node i or above it."""
    sees = np.eye(n, dtype=bool)
    for i in range(1, n):
        up = i - 1 if parents is None else int(parents[i])
        if 0 <= up < i:
            sees[i] |= sees[up]
    return sees


def attend(q, k, v, table, context, parents=None, num_nodes=None, scale=None):
    """(out, lse, tol_out, tol_lse), all in 64 bits.

    The bounds count roundings of at most half a step each: eps = step of the inputs' type, e = step of 32 bits.
      scores   a product of two 16-bit numbers is exact in 32 bits; D additions and the scale: off by at most
               (D + 4) e max sum|q k||scale| =: ds (absolute, natural units; as much for 32-bit inputs, whose products round);
      weights  exp off by ds, the exponential function and its argument by 4 steps, and the running maximum's rescalings and
               the join by 4 steps in each of at most `tiles` tiles; once to the inputs' type for the product with the values;
      sums     `len` additions of at most e each relative to sum p|v| (tree or tile order does not make it worse)."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    t_eps, e = {torch.float32: 2.0**-23, torch.float16: 2.0**-10, torch.bfloat16: 2.0**-7}[attend.dtype] / 2, 2.0**-24
    B, N, H, D = q.shape
    P, S, KH, _ = k.shape
    scale = D**-0.5 if scale is None else scale
    out, lse = torch.zeros(B, N, H, D, dtype=torch.float64), torch.full((B, N, H), -np.inf, dtype=torch.float64)
    tol_out, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(B):
        c, used = max(int(context[b]), 0), N if num_nodes is None else min(max(int(num_nodes[b]), 0), N)
        sees = ancestors(None if parents is None else parents[b], used) if used else np.zeros((0, 0), bool)
        pos = torch.arange(c + used)
        inside = pos // S < table.shape[1]
        page = torch.where(inside, table[b].long().cpu()[(pos // S).clamp(max=max(table.shape[1] - 1, 0))], -1) if table.shape[1] else -torch.ones_like(pos)
        good = (page >= 0) & (page < P)
        for i in range(used):
            see = good & ((pos < c) | torch.from_numpy(np.concatenate([np.zeros(c, bool), sees[i]])))
            at = torch.nonzero(see)[:, 0]
            if at.numel() == 0:
                continue
            kk, vv = k[page[at], at % S], v[page[at], at % S]  # [L, KH, D]
            kk, vv = (x.repeat_interleave(H // KH, 1) for x in (kk, vv))
            s = torch.einsum("hd,lhd->hl", q[b, i], kk) * scale
            w = torch.softmax(s, -1)
            out[b, i] = torch.einsum("hl,lhd->hd", w, vv)
            lse[b, i] = torch.logsumexp(s, -1)
            ds = (D + 4) * 2 * e * (torch.einsum("hd,lhd->hl", q[b, i].abs(), kk.abs()) * abs(scale)).amax(-1)
            L = at.numel()
            rel = 2 * ds + (4 * (L // 32 + 2) + L) * e
            mass = torch.einsum("hl,lhd->hd", w, vv.abs())
            tol_out[b, i] = (2 * rel[:, None] + t_eps) * mass + t_eps * out[b, i].abs() + 2.0**-24 * (attend.dtype == torch.float16)
            tol_lse[b, i] = rel + 4 * e * lse[b, i].abs() + 8 * e
    return out, lse, tol_out, tol_lse


def check_attend(got, q, k, v, table, context, parents=None, num_nodes=None, scale=None, what=""):
    attend.dtype = q.dtype
    out, lse, tol_out, tol_lse = attend(q, k, v, table, context, parents, num_nodes, scale)
    for name, g, w, tol in (("out", got[0], out, tol_out), ("lse", got[1], lse, tol_lse)):
        g = g.double().cpu()
        same = (g == w) | (torch.isnan(g) & torch.isnan(w))
        bad = ~(same | ((g - w).abs() <= tol))
        if bad.any():
            at = tuple(torch.nonzero(bad)[0].tolist())
            raise AssertionError(f"{what} {name} at {at}: got {g[at]}, want {w[at]} +- {tol[at]}; {int(bad.sum())} of {bad.numel()}")


def compact(cache, table, context, path, count):
    """The cache after the move of the accepted rows (a copy), [layers, pages, page_size, heads, dim]."""
    cache, out = cache.clone(), cache.clone()
    L, P, S = cache.shape[:3]
    lengths = []
    for b in range(len(context)):
        n = 0
        for i in range(min(max(int(count[b]), 0), path.shape[1])):
            if int(path[b, i]) >= path.shape[1] or int(path[b, i]) <= (int(path[b, i - 1]) if i else -1):
                break
            n += 1
        lengths.append(max(int(context[b]), 0) + n)
        for i in range(1, n):
            old, new = max(int(context[b]), 0) + int(path[b, i]), max(int(context[b]), 0) + i
            if max(old, new) // S >= table.shape[1]:
                continue
            a, z = int(table[b, old // S]), int(table[b, new // S])
            if 0 <= a < P and 0 <= z < P and old != new:
                out[:, z, new % S] = cache[:, a, old % S]
    return out, lengths


def random_tree(batch, nodes, g):
    at = torch.arange(nodes)
    return (torch.rand(batch, nodes, generator=g) * at).long().clamp(max=(at - 1).clamp(min=0)).to(torch.int32)


def paged(lengths, page, heads, dim, dtype, g, spare=3, columns=None, fill=None):
    """A cache whose sequences lie in pages in random order; entries of the table behind a sequence are -1 and everything
    behind a sequence's last row, spare pages included, holds `fill` where it is given."""
    need = [-(-int(n) // page) for n in lengths]
    columns = max(max(need), 1) if columns is None else columns
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g).tolist()
    table = torch.full((len(lengths), columns), -1, dtype=torch.int32)
    k, v = (torch.randn(pool, page, heads, dim, generator=g).to(dtype) for _ in range(2))
    live = torch.zeros(pool, page, dtype=torch.bool)
    for b, n in enumerate(need):
        for j in range(n):
            table[b, j] = order.pop()
            live[int(table[b, j]), : min(page, int(lengths[b]) - j * page)] = True
    if fill is not None:
        k[~live], v[~live] = fill, fill
    return k, v, table
