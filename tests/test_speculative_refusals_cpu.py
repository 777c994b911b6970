"""What the speculative decoding entry points refuse, and what they plan: no device is needed, nothing is launched."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from tests import speculative_reference as ref
from vkop_b200 import capi

P = 4096  # a pointer that is never followed: every call here is refused, or has an empty batch


def verify_desc(**kw):
    d = dict(batch=2, vocab=100, target_batch_stride=0, target_node_stride=0, draft_batch_stride=0, draft_node_stride=0, nodes=4, draft_rows=4, dtype=capi.F32,
             index_dtype=capi.I32)
    return capi.DraftVerifyDesc(**(d | kw))


def verify(d, target=P, draft=P, tokens=P, parents=None, used=None, u=P, path=P, count=P, token=P, chance=None):
    return capi.lib().vkop_cuda_draft_verify(C.byref(d) if d is not None else None, target, draft, tokens, parents, used, u, path, count, token, chance, None)


def test_draft_verify_refusals():
    n0 = capi.launch_count()
    for kw in (dict(batch=-1), dict(vocab=0), dict(vocab=2**31), dict(nodes=0), dict(nodes=1025), dict(draft_rows=-1), dict(draft_rows=5), dict(dtype=3), dict(dtype=-1),
               dict(index_dtype=2), dict(target_node_stride=99), dict(draft_node_stride=99), dict(target_batch_stride=-4), dict(draft_batch_stride=-1)):
        assert verify(verify_desc(**kw)) == capi.INVALID_ARG, kw
    assert verify(None) == capi.INVALID_ARG
    for name in ("target", "draft", "tokens", "u", "path", "count", "token"):
        assert verify(verify_desc(), **{name: None}) == capi.INVALID_ARG, name
    for name, d in (("target", {}), ("draft", {}), ("tokens", {}), ("parents", {}), ("used", {}), ("u", {}), ("path", {}), ("count", {}), ("token", {}), ("chance", {})):
        assert verify(verify_desc(**d), **{name: P + 2}) == capi.INVALID_ARG, name
    assert verify(verify_desc(dtype=capi.F16), target=P + 1) == capi.INVALID_ARG
    assert verify(verify_desc(index_dtype=capi.I64), tokens=P + 4) == capi.INVALID_ARG
    assert verify(verify_desc(batch=0), None, None, None) == capi.OK
    assert capi.launch_count() == n0


def attention_desc(**kw):
    d = dict(batch=2, num_pages=10, max_context=100, nodes=4, q_heads=8, kv_heads=2, head_dim=64, page_size=16, max_pages=8, dtype=capi.F16, scale=0.125)
    return capi.TreeAttentionDesc(**(d | kw))


def attention(d, q=P, k=P, v=P, table=P, context=P, parents=None, used=None, out=P, lse=None, ws=P, nbytes=1 << 40):
    return capi.lib().vkop_cuda_tree_attention(C.byref(d) if d is not None else None, q, k, v, table, context, parents, used, out, lse, ws, nbytes, None)


def test_tree_attention_refusals():
    n0 = capi.launch_count()
    need = C.c_size_t(0)
    for kw, status in ((dict(batch=-1), -1), (dict(batch=65536), -1), (dict(num_pages=-1), -1), (dict(max_context=-1), -1), (dict(nodes=0), -1), (dict(nodes=129), -1),
                       (dict(kv_heads=0), -1), (dict(q_heads=1), -1), (dict(q_heads=7), -1), (dict(q_heads=1024), -1), (dict(head_dim=0), -1), (dict(head_dim=12), -1),
                       (dict(head_dim=264), -1), (dict(page_size=0), -1), (dict(page_size=65537), -1), (dict(max_pages=-1), -1), (dict(dtype=3), -1),
                       (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1), (dict(q_node_stride=-8), -1), (dict(v_page_stride=-1), -1), (dict(table_stride=7), -1),
                       (dict(page_size=65536, max_pages=40000), -2), (dict(kv_heads=1024, q_heads=1024 * 8, nodes=128), -2)):
        assert attention(attention_desc(**kw)) == status, kw
        assert capi.lib().vkop_cuda_tree_attention_workspace(C.byref(attention_desc(**kw)), C.byref(need)) == status, kw
    assert attention(None) == capi.INVALID_ARG
    for name in ("q", "k", "v", "table", "context", "out"):
        assert attention(attention_desc(), **{name: None}) == capi.INVALID_ARG, name
    for name in ("q", "k", "v", "out"):
        assert attention(attention_desc(), **{name: P + 1}) == capi.INVALID_ARG, name
    for name in ("table", "context", "parents", "used", "lse"):
        assert attention(attention_desc(), **{name: P + 2}) == capi.INVALID_ARG, name
    long = attention_desc(batch=1, max_context=100000, max_pages=7000)
    assert capi.lib().vkop_cuda_tree_attention_workspace(C.byref(long), C.byref(need)) == capi.OK and need.value > 0
    assert attention(long, ws=None, nbytes=0) == capi.WORKSPACE_TOO_SMALL
    assert attention(long, nbytes=need.value - 1) == capi.WORKSPACE_TOO_SMALL
    assert attention(long, ws=P + 8) == capi.INVALID_ARG
    assert capi.lib().vkop_cuda_tree_attention_workspace(C.byref(long), None) == capi.INVALID_ARG
    assert attention(attention_desc(batch=0), None, None, None, None, None, out=None) == capi.OK
    assert capi.launch_count() == n0


def compact_desc(**kw):
    d = dict(batch=2, num_pages=10, layers=2, nodes=8, kv_heads=2, head_dim=64, page_size=16, max_pages=8, dtype=capi.F16)
    return capi.CacheCompactDesc(**(d | kw))


def compact(d, k=P, v=2 * P, table=P, context=P, path=P, count=P, out=16 * P):
    return capi.lib().vkop_cuda_cache_compact(C.byref(d) if d is not None else None, k, v, table, context, path, count, out, None)


def test_cache_compact_refusals():
    n0 = capi.launch_count()
    for kw in (dict(batch=-1), dict(num_pages=-1), dict(layers=-1), dict(layers=32768), dict(nodes=0), dict(nodes=1025), dict(kv_heads=0), dict(head_dim=0), dict(page_size=0),
               dict(max_pages=-1), dict(dtype=7), dict(k_layer_stride=-1), dict(v_head_stride=-2), dict(table_stride=3), dict(reserved=1)):
        assert compact(compact_desc(**kw)) == capi.INVALID_ARG, kw
    assert compact(None) == capi.INVALID_ARG
    for name in ("k", "table", "context", "path", "count", "out"):
        assert compact(compact_desc(), **{name: None}) == capi.INVALID_ARG, name
    assert compact(compact_desc(), v=P) == capi.INVALID_ARG          # one cache twice
    assert compact(compact_desc(), out=P + 4) == capi.INVALID_ARG    # overlaps context
    assert compact(compact_desc(), out=P) == capi.INVALID_ARG
    for name in ("k", "v"):
        assert compact(compact_desc(), **{name: 3 * P + 1}) == capi.INVALID_ARG, name
    for name in ("table", "context", "path", "count", "out"):
        assert compact(compact_desc(), **{name: 3 * P + 2}) == capi.INVALID_ARG, name
    assert compact(compact_desc(batch=0), None, None, None, None, None, None, None) == capi.OK
    assert capi.launch_count() == n0


def test_python_wrappers_refuse_host_memory():
    t, i = torch.zeros(1, 2, 10), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA device memory only"):
        capi.draft_verify(t, i, torch.zeros(1, 2))
    k = torch.zeros(2, 16, 1, 64)
    with pytest.raises(RuntimeError, match="CUDA device memory only"):
        capi.tree_attention(torch.zeros(1, 2, 1, 64), k, k, i, i[:, 0])
    with pytest.raises(RuntimeError, match="CUDA device memory only"):
        capi.cache_compact(k, k, i, i[:, 0], i, i[:, 0])


def test_shapes_and_types_that_the_wrappers_refuse():
    """The descriptor of the attention is built without touching the tensors' memory: the checks run on the CPU."""
    q, k, table = torch.zeros(2, 3, 4, 64, dtype=torch.float16), torch.zeros(5, 16, 2, 64, dtype=torch.float16), torch.zeros(2, 4, dtype=torch.int32)
    assert capi.tree_attention_workspace_bytes(q, k, k, table) >= 0
    for bad in ((q.double(), k, k, table), (q[0], k, k, table), (q, k, k[:, :8], table), (q, k.float(), k.float(), table), (q[..., ::2], k, k, table),
                (q[:, :1].expand(2, 3, 4, 64), k, k, table), (q, k, k, table.long()), (q, k, k, table[:1]), (q, k, k, table.T.contiguous().T),
                (q, k[:1].expand(5, 16, 2, 64), k, table)):
        with pytest.raises(ValueError):
            capi.tree_attention_workspace_bytes(*bad)
    # one sequence, one page, one head: strides of dimensions of one do not matter
    assert capi.tree_attention_workspace_bytes(q[:1, :1, :1].expand(1, 1, 1, 64), k[:1, :, :1], k[:1, :, :1], table[:1, :1]) >= 0


def test_a_scale_that_overflows_in_units_of_log2_is_refused():
    """Scores are kept as scale * log2(e) * q k: 2.4e38 is finite, 2.4e38 * 1.4427 is not."""
    need = C.c_size_t(0)
    for scale in (2.4e38, -2.4e38):
        assert attention(attention_desc(scale=scale)) == capi.INVALID_ARG
        assert capi.lib().vkop_cuda_tree_attention_workspace(C.byref(attention_desc(scale=scale)), C.byref(need)) == capi.INVALID_ARG
    assert attention(attention_desc(scale=2.3e38, batch=0)) == capi.OK


def test_rows_too_long_to_count_are_refused():
    """A row of all heads has at most 2^30 elements: its columns are counted in 32 bits."""
    assert compact(compact_desc(kv_heads=65536, head_dim=65536)) == capi.UNSUPPORTED
    assert compact(compact_desc(kv_heads=32768, head_dim=65536, batch=0), None, None, None, None, None, None, None) == capi.UNSUPPORTED
    assert compact(compact_desc(kv_heads=16384, head_dim=65536, batch=0), None, None, None, None, None, None, None) == capi.OK


def test_a_broadcast_workspace_is_refused(monkeypatch):
    """Its elements are more than its memory: the length that the entry point checks would be wrong."""
    monkeypatch.setattr(capi, "_one_device", lambda what, *tensors: 0)
    monkeypatch.setattr(capi, "_call", lambda *a: None)
    q, k = torch.zeros(1, 3, 4, 64, dtype=torch.float16), torch.zeros(5, 16, 2, 64, dtype=torch.float16)
    table, context = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for bad in (torch.zeros(1, dtype=torch.uint8).expand(1 << 20), torch.zeros(1 << 20, dtype=torch.uint8)[::2], torch.zeros(1 << 20)):
        with pytest.raises(ValueError, match="workspace"):
            capi.tree_attention(q, k, k, table, context, workspace=bad)
    capi.tree_attention(q, k, k, table, context, workspace=torch.zeros(1 << 20, dtype=torch.uint8))


# ---- the 64-bit statements that the GPU tests compare with, checked against each other and by hand ----


def test_reference_walk_by_hand():
    p = torch.tensor([[[0.5, 0.3, 0.2], [0.1, 0.8, 0.1], [1.0, 0, 0]]])
    q = torch.tensor([[[0.25, 0.5, 0.25], [0.1, 0.1, 0.8], [0, 0, 1.0]]])
    tokens = torch.tensor([[0, 1, 2]], dtype=torch.int32)
    # node 1: 0.3 / 0.5 = 0.6 > 0.55 accepted; node 2: 0.1 / 0.8 < 0.2 rejected; left: (0, 0.7, 0)
    path, count, token, chance = ref.verify(p, tokens, torch.tensor([[0.5, 0.55, 0.2]]), q)
    assert path.tolist() == [[0, 1, -1]] and count.tolist() == [2] and token.tolist() == [1]
    assert np.allclose(chance, [[0, 0.6, 0.125]])
    # node 1 rejected: left (0.25, 0, 0)
    path, count, token, _ = ref.verify(p, tokens, torch.tensor([[0.9, 0.65, 0.2]]), q)
    assert path.tolist() == [[0, -1, -1]] and token.tolist() == [0]
    # certain drafts, both children of node 0: 0.3 rejected, then 0.2 / 0.7
    up = torch.zeros(1, 3, dtype=torch.int32)
    path, count, token, chance = ref.verify(p, tokens, torch.tensor([[0.0, 0.5, 0.5]]), None, up)
    assert path.tolist() == [[0, -1, -1]] and token.tolist() == [0] and np.allclose(chance, [[0, 0.3, 0.2 / 0.7]])


def test_reference_residuals_equal_the_recursive_form():
    """max(max(p - c q, 0) / D - q, 0) in turn, normalised each time, against the closed form that the operator uses."""
    rng = np.random.default_rng(3)
    p, q = rng.dirichlet(np.ones(50)), rng.dirichlet(np.ones(50))
    rest, c, mass = p, 0.0, 1.0
    for _ in range(4):
        rest = np.maximum(rest - q, 0)
        rest = rest / rest.sum()
        c += mass
        mass = np.maximum(p - c * q, 0).sum()
        assert np.allclose(np.maximum(p - c * q, 0) / mass, rest, rtol=1e-9, atol=1e-15)


def test_reference_masks_and_bad_pages():
    g = torch.Generator().manual_seed(0)
    k, v, table = ref.paged([9], 4, 1, 8, torch.float32, g)
    q = torch.randn(1, 4, 1, 8, generator=g)
    parents = torch.tensor([[0, 0, 0, 1]], dtype=torch.int32)
    context = torch.tensor([5], dtype=torch.int32)
    ref.attend.dtype = torch.float32
    out = ref.attend(q, k, v, table, context, parents)[0]
    rows = [[0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 4, 5, 6], [0, 1, 2, 3, 4, 5, 7], [0, 1, 2, 3, 4, 5, 6, 8]]
    for i, at in enumerate(rows):
        at = torch.tensor(at)
        kk, vv = k[table[0].long()[at // 4], at % 4, 0].double(), v[table[0].long()[at // 4], at % 4, 0].double()
        w = torch.softmax(kk @ q[0, i, 0].double() * 8**-0.5, 0)
        assert torch.allclose(out[0, i, 0], w @ vv)
    table[0, 1] = 77  # not there: positions 4 .. 7 are left out
    out = ref.attend(q, k, v, table, context, parents)[0]
    at = torch.arange(4)
    w = torch.softmax(k[table[0, 0].long(), at, 0].double() @ q[0, 0, 0].double() * 8**-0.5, 0)
    assert torch.allclose(out[0, 0, 0], w @ v[table[0, 0].long(), at, 0].double())
