"""ctypes binding of the C ABI declared in ``include/vkop_cuda.h``.

The wrappers take torch CUDA tensors (device memory only; nothing is computed
by torch) and enqueue on torch's current stream.  A missing or unloadable
``libvkop_cuda.so`` raises; there is no fallback.
"""
from __future__ import annotations

import ctypes as C
import os

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libvkop_cuda.so")

F32, F16, BF16 = 0, 1, 2
I32, I64 = 0, 1
VALUE_PROBABILITY, VALUE_RAW = 0, 1
PATH_AUTO, PATH_CHUNK, PATH_RADIX, PATH_STREAM, PATH_BULK = 0, 1, 2, 3, 4
FLAG_INPUT_READY = 1
OK, INVALID_ARG, UNSUPPORTED, WORKSPACE_TOO_SMALL, CUDA_ERROR, TIMEOUT = 0, -1, -2, -3, -4, -5

EXPORTS = [
    "vkop_cuda_version", "vkop_cuda_status_string", "vkop_cuda_launch_count", "vkop_cuda_workspace_init",
    "vkop_cuda_softmax_topk_workspace", "vkop_cuda_softmax_topk", "vkop_cuda_topk", "vkop_cuda_softmax",
    "vkop_cuda_packet_bytes", "vkop_cuda_softmax_topk_partial", "vkop_cuda_softmax_topk_merge",
    "vkop_cuda_nms_workspace", "vkop_cuda_nms",
    "vkop_cuda_static_scratch_bytes", "vkop_cuda_softmax_topk_static",
    "vkop_cuda_packets_push", "vkop_cuda_packets_wait", "vkop_cuda_packets_exchange_all_ranks", "vkop_cuda_yolo_nms",
    "vkop_cuda_sample_topk", "vkop_cuda_topk_axis_workspace", "vkop_cuda_topk_axis",
    "vkop_cuda_draft_verify", "vkop_cuda_tree_attention_workspace", "vkop_cuda_tree_attention", "vkop_cuda_cache_compact",
]


class SoftmaxTopkDesc(C.Structure):
    _fields_ = [("rows", C.c_int64), ("cols", C.c_int64), ("row_stride", C.c_int64), ("dtype", C.c_int32),
                ("k", C.c_int32), ("index_dtype", C.c_int32), ("value_kind", C.c_int32),
                ("inv_temperature", C.c_float), ("largest", C.c_int32), ("path", C.c_int32), ("splits", C.c_int32),
                ("index_offset", C.c_int64), ("flags", C.c_int32), ("reserved", C.c_int32)]


class SoftmaxDesc(C.Structure):
    _fields_ = [("outer", C.c_int64), ("axis_len", C.c_int64), ("inner", C.c_int64), ("dtype", C.c_int32),
                ("inv_temperature", C.c_float)]


class TopkAxisDesc(C.Structure):
    _fields_ = [("outer", C.c_int64), ("axis_len", C.c_int64), ("inner", C.c_int64), ("dtype", C.c_int32),
                ("k", C.c_int32), ("index_dtype", C.c_int32), ("largest", C.c_int32), ("sorted", C.c_int32),
                ("path", C.c_int32)]


class NmsDesc(C.Structure):
    _fields_ = [("num_batch", C.c_int32), ("num_class", C.c_int32), ("num_boxes", C.c_int32),
                ("center_point_box", C.c_int32), ("max_output_boxes_per_class", C.c_int32), ("pre_topk", C.c_int32),
                ("iou_threshold", C.c_float), ("score_threshold", C.c_float), ("capacity_rows", C.c_int64)]


class DraftVerifyDesc(C.Structure):
    _fields_ = [("batch", C.c_int64), ("vocab", C.c_int64), ("target_batch_stride", C.c_int64),
                ("target_node_stride", C.c_int64), ("draft_batch_stride", C.c_int64), ("draft_node_stride", C.c_int64),
                ("nodes", C.c_int32), ("draft_rows", C.c_int32), ("dtype", C.c_int32), ("index_dtype", C.c_int32)]


class TreeAttentionDesc(C.Structure):
    _fields_ = [("batch", C.c_int64), ("num_pages", C.c_int64), ("max_context", C.c_int64),
                ("q_batch_stride", C.c_int64), ("q_node_stride", C.c_int64), ("q_head_stride", C.c_int64),
                ("out_batch_stride", C.c_int64), ("out_node_stride", C.c_int64), ("out_head_stride", C.c_int64),
                ("k_page_stride", C.c_int64), ("k_token_stride", C.c_int64), ("k_head_stride", C.c_int64),
                ("v_page_stride", C.c_int64), ("v_token_stride", C.c_int64), ("v_head_stride", C.c_int64),
                ("table_stride", C.c_int64), ("nodes", C.c_int32), ("q_heads", C.c_int32), ("kv_heads", C.c_int32),
                ("head_dim", C.c_int32), ("page_size", C.c_int32), ("max_pages", C.c_int32), ("dtype", C.c_int32),
                ("scale", C.c_float)]


class CacheCompactDesc(C.Structure):
    _fields_ = [("batch", C.c_int64), ("num_pages", C.c_int64), ("k_layer_stride", C.c_int64),
                ("k_page_stride", C.c_int64), ("k_token_stride", C.c_int64), ("k_head_stride", C.c_int64),
                ("v_layer_stride", C.c_int64), ("v_page_stride", C.c_int64), ("v_token_stride", C.c_int64),
                ("v_head_stride", C.c_int64), ("table_stride", C.c_int64), ("layers", C.c_int32), ("nodes", C.c_int32),
                ("kv_heads", C.c_int32), ("head_dim", C.c_int32), ("page_size", C.c_int32), ("max_pages", C.c_int32),
                ("dtype", C.c_int32), ("reserved", C.c_int32)]


class VkopError(RuntimeError):
    def __init__(self, status: int, where: str):
        self.status = status
        super().__init__(f"{where}: {status_string(status)} ({status})")


_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} is missing: build it with `python -m vkop_b200.build` "
                               "(there is no CPU fallback)")
        L = C.CDLL(LIB_PATH)
        L.vkop_cuda_status_string.restype = C.c_char_p
        L.vkop_cuda_launch_count.restype = C.c_uint64
        L.vkop_cuda_packet_bytes.restype = C.c_size_t
        L.vkop_cuda_packet_bytes.argtypes = [C.c_int32]
        vp, sz = C.c_void_p, C.c_size_t
        L.vkop_cuda_workspace_init.argtypes = [vp, sz, vp]
        L.vkop_cuda_softmax_topk_workspace.argtypes = [C.POINTER(SoftmaxTopkDesc), C.POINTER(sz)]
        L.vkop_cuda_softmax_topk.argtypes = [C.POINTER(SoftmaxTopkDesc), vp, vp, vp, vp, sz, vp]
        L.vkop_cuda_topk.argtypes = [C.POINTER(SoftmaxTopkDesc), vp, vp, vp, vp, sz, vp]
        L.vkop_cuda_softmax.argtypes = [C.POINTER(SoftmaxDesc), vp, vp, vp]
        L.vkop_cuda_topk_axis_workspace.argtypes = [C.POINTER(TopkAxisDesc), C.POINTER(sz)]
        L.vkop_cuda_topk_axis.argtypes = [C.POINTER(TopkAxisDesc), vp, vp, vp, vp, sz, vp]
        L.vkop_cuda_softmax_topk_partial.argtypes = [C.POINTER(SoftmaxTopkDesc), vp, vp, vp, sz, vp]
        L.vkop_cuda_softmax_topk_merge.argtypes = [C.POINTER(SoftmaxTopkDesc), vp, C.c_int32, vp, vp, vp]
        L.vkop_cuda_nms_workspace.argtypes = [C.POINTER(NmsDesc), C.POINTER(sz)]
        L.vkop_cuda_nms.argtypes = [C.POINTER(NmsDesc), vp, vp, vp, vp, vp, sz, vp]
        L.vkop_cuda_packets_push.argtypes = [vp, sz, vp, vp, C.c_int32, C.c_int32, C.c_uint32, vp, vp]
        L.vkop_cuda_packets_wait.argtypes = [vp, C.c_int32, C.c_uint32, C.c_uint32, vp, vp]
        L.vkop_cuda_packets_exchange_all_ranks.argtypes = [vp, sz, vp, vp, C.c_int32, C.c_uint32, vp, C.c_uint32, vp, vp]
        L.vkop_cuda_yolo_nms.argtypes = [C.POINTER(NmsDesc), vp, vp, vp, vp, sz, vp]
        L.vkop_cuda_sample_topk.argtypes = [vp, C.c_int32, vp, C.c_int32, C.c_int64, C.c_int32, C.c_float, vp, vp, vp, vp]
        L.vkop_cuda_draft_verify.argtypes = [C.POINTER(DraftVerifyDesc)] + [vp] * 11
        L.vkop_cuda_tree_attention_workspace.argtypes = [C.POINTER(TreeAttentionDesc), C.POINTER(sz)]
        L.vkop_cuda_tree_attention.argtypes = [C.POINTER(TreeAttentionDesc)] + [vp] * 10 + [sz, vp]
        L.vkop_cuda_cache_compact.argtypes = [C.POINTER(CacheCompactDesc)] + [vp] * 8
        L.vkop_cuda_static_scratch_bytes.restype = sz
        L.vkop_cuda_softmax_topk_static.argtypes = [C.POINTER(SoftmaxTopkDesc), vp, vp, vp, vp]
        _lib = L
    return _lib


def status_string(status: int) -> str:
    return lib().vkop_cuda_status_string(C.c_int(status)).decode()


def launch_count() -> int:
    return int(lib().vkop_cuda_launch_count())


def check(status: int, where: str) -> None:
    if status != OK:
        raise VkopError(status, where)


_TORCH_DTYPE = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


def dtype_tag(t: torch.Tensor) -> int:
    return _TORCH_DTYPE[t.dtype]


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t) -> int | None:
    return None if t is None else t.data_ptr()


class Workspace:
    """Caller-owned scratch memory (a torch byte tensor), cleared once on creation."""

    def __init__(self, nbytes: int, device="cuda"):
        self.nbytes = int(nbytes)
        self.buf = torch.empty(max(self.nbytes, 16), dtype=torch.uint8, device=device)
        check(lib().vkop_cuda_workspace_init(self.buf.data_ptr(), self.buf.numel(), _stream()), "workspace_init")

    @property
    def ptr(self) -> int:
        return self.buf.data_ptr()


def make_desc(logits: torch.Tensor, k: int, inv_temperature: float = 1.0, index_dtype: int = I32,
              value_kind: int = VALUE_PROBABILITY, largest: bool = True, path: int = PATH_AUTO, splits: int = 0,
              index_offset: int = 0, flags: int = 0) -> SoftmaxTopkDesc:
    assert logits.dim() == 2 and logits.stride(1) == 1
    return SoftmaxTopkDesc(rows=logits.shape[0], cols=logits.shape[1], row_stride=logits.stride(0),
                           dtype=dtype_tag(logits), k=k, index_dtype=index_dtype, value_kind=value_kind,
                           inv_temperature=inv_temperature, largest=int(largest), path=path, splits=splits,
                           index_offset=index_offset, flags=flags, reserved=0)


def softmax_topk_workspace_bytes(desc: SoftmaxTopkDesc) -> int:
    n = C.c_size_t(0)
    check(lib().vkop_cuda_softmax_topk_workspace(C.byref(desc), C.byref(n)), "softmax_topk_workspace")
    return int(n.value)


def softmax_topk(logits: torch.Tensor, k: int, inv_temperature: float = 1.0, index_dtype: int = I32,
                 value_kind: int = VALUE_PROBABILITY, path: int = PATH_AUTO, splits: int = 0, index_offset: int = 0,
                 workspace: Workspace | None = None, out=None, standalone_topk: bool = False, largest: bool = True,
                 flags: int = 0):
    """Fused softmax + top-k of a 2-D CUDA tensor.  Returns (values [rows,k] in the logits dtype, indices)."""
    if not logits.is_cuda:
        raise RuntimeError("vkop_b200 runs on CUDA device memory only")
    desc = make_desc(logits, k, inv_temperature, index_dtype, value_kind, largest, path, splits, index_offset, flags)
    need = softmax_topk_workspace_bytes(desc)
    if workspace is None or workspace.nbytes < need:
        workspace = Workspace(need, logits.device)
    if out is None:
        values = torch.empty((logits.shape[0], k), dtype=logits.dtype, device=logits.device)
        indices = torch.empty((logits.shape[0], k), dtype=torch.int64 if index_dtype == I64 else torch.int32,
                              device=logits.device)
    else:
        values, indices = out
    fn = lib().vkop_cuda_topk if standalone_topk else lib().vkop_cuda_softmax_topk
    check(fn(C.byref(desc), logits.data_ptr(), values.data_ptr(), indices.data_ptr(), workspace.ptr,
             workspace.buf.numel(), _stream()), "topk" if standalone_topk else "softmax_topk")
    return values, indices


def topk_axis(x: torch.Tensor, k: int, axis: int = -1, largest: bool = True, sorted: bool = True, index_dtype: int = I32,
              path: int = PATH_AUTO, workspace: Workspace | None = None):
    """TopK of a contiguous CUDA tensor along any axis.  Returns (values, indices) shaped like x with shape[axis] = k;
    sorted=False gives the k entries in ascending index order."""
    if not x.is_cuda or not x.is_contiguous():
        raise RuntimeError("vkop_b200 runs on contiguous CUDA device memory only")
    axis = axis % x.dim()
    outer = int(torch.Size(x.shape[:axis]).numel())
    inner = int(torch.Size(x.shape[axis + 1:]).numel())
    desc = TopkAxisDesc(outer=outer, axis_len=x.shape[axis], inner=inner, dtype=dtype_tag(x), k=k, index_dtype=index_dtype,
                        largest=int(largest), sorted=int(sorted), path=path)
    n = C.c_size_t(0)
    check(lib().vkop_cuda_topk_axis_workspace(C.byref(desc), C.byref(n)), "topk_axis_workspace")
    if workspace is None or workspace.nbytes < n.value:
        workspace = Workspace(int(n.value), x.device)
    shape = list(x.shape)
    shape[axis] = k
    values = torch.empty(shape, dtype=x.dtype, device=x.device)
    indices = torch.empty(shape, dtype=torch.int64 if index_dtype == I64 else torch.int32, device=x.device)
    check(lib().vkop_cuda_topk_axis(C.byref(desc), x.data_ptr(), values.data_ptr(), indices.data_ptr(), workspace.ptr,
                                    workspace.buf.numel(), _stream()), "topk_axis")
    return values, indices


def yolo_nms(head: torch.Tensor, center_point_box: int = 1, max_output_boxes_per_class: int = 0,
             iou_threshold: float = 0.0, score_threshold: float = 0.0, pre_topk: int = 0, capacity_rows: int | None = None,
             workspace: Workspace | None = None, out=None):
    """NMS on a detection head [B, 4 + C, N] (coordinate planes, then score planes), read in place.
    Returns (rows int32 [capacity, 3], count int32 [1]) like nms()."""
    if not head.is_cuda:
        raise RuntimeError("vkop_b200 runs on CUDA device memory only")
    assert head.dtype == torch.float32 and head.dim() == 3 and head.shape[1] > 4 and head.is_contiguous()
    B, planes, N = head.shape
    Cn = planes - 4
    if capacity_rows is None:
        per = max_output_boxes_per_class if max_output_boxes_per_class > 0 else (pre_topk if pre_topk > 0 else N)
        capacity_rows = B * Cn * min(per, N)
    desc = NmsDesc(num_batch=B, num_class=Cn, num_boxes=N, center_point_box=center_point_box,
                   max_output_boxes_per_class=max_output_boxes_per_class, pre_topk=pre_topk,
                   iou_threshold=iou_threshold, score_threshold=score_threshold, capacity_rows=capacity_rows)
    need = nms_workspace_bytes(desc)
    if workspace is None or workspace.nbytes < need:
        workspace = Workspace(need, head.device)
    if out is None:
        rows = torch.empty((max(capacity_rows, 1), 3), dtype=torch.int32, device=head.device)
        count = torch.empty(1, dtype=torch.int32, device=head.device)
    else:
        rows, count = out
    check(lib().vkop_cuda_yolo_nms(C.byref(desc), head.data_ptr(), rows.data_ptr(), count.data_ptr(), workspace.ptr,
                                   workspace.buf.numel(), _stream()), "yolo_nms")
    return rows, count


def sample_topk(values: torch.Tensor, indices: torch.Tensor, top_p: float, u: torch.Tensor):
    """Sampling tail over the survivors of softmax_topk.  Returns (choice int32 [rows], token [rows])."""
    if not (values.is_cuda and indices.is_cuda and u.is_cuda):
        raise RuntimeError("vkop_b200 runs on CUDA device memory only")
    rows, k = values.shape
    assert indices.shape == values.shape and u.shape == (rows,) and u.dtype == torch.float32
    values, indices, u = values.contiguous(), indices.contiguous(), u.contiguous()
    choice = torch.empty(rows, dtype=torch.int32, device=values.device)
    token = torch.empty(rows, dtype=indices.dtype, device=values.device)
    check(lib().vkop_cuda_sample_topk(values.data_ptr(), dtype_tag(values), indices.data_ptr(),
                                      I64 if indices.dtype == torch.int64 else I32, rows, k, float(top_p), u.data_ptr(),
                                      choice.data_ptr(), token.data_ptr(), _stream()), "sample_topk")
    return choice, token


# The bindings below are on the path of every decoding step: checks and bookkeeping are kept to a few microseconds.
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else \
    (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _one_device(what: str, *tensors) -> int:
    """The index of the device that all the tensors lie on (None among them is passed over)."""
    index = tensors[0].get_device()  # -1 on the host
    for t in tensors:
        if t is not None and t.get_device() != index:
            index = -1
    if index < 0:
        raise RuntimeError(f"{what}: vkop_b200 runs on CUDA device memory only, all tensors on one device")
    return index


def _call(index: int, what: str, fn, *args) -> None:
    """Calls a C entry point with the device current and its current stream as the last argument."""
    if torch.cuda.current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status != OK:
        raise VkopError(status, what)


def _whole(what: str, name: str, t, shape, dtype=torch.int32):
    """Checks a small dense argument: its type, its shape and that it is contiguous."""
    if t is not None and (t.dtype != dtype or t.shape != shape or not t.is_contiguous()):
        raise ValueError(f"{what}: {name} is a contiguous {dtype} tensor of shape {tuple(shape)}, "
                         f"got {t.dtype} {tuple(t.shape)}")


def _strides(what: str, name: str, t: torch.Tensor, ndim: int):
    """Strides of the leading dimensions, in elements (0: dense); the last dimension is contiguous and nothing is broadcast."""
    if t.dim() != ndim or t.dtype not in _TORCH_DTYPE:
        raise ValueError(f"{what}: {name} is a float32, float16 or bfloat16 tensor of {ndim} dimensions")
    if t.is_contiguous():
        return (0,) * (ndim - 1)
    strides, shape = t.stride(), t.shape
    if (strides[-1] != 1 and shape[-1] > 1) or any(s == 0 and n > 1 for s, n in zip(strides, shape)):
        raise ValueError(f"{what}: {name} has a contiguous last dimension and no broadcast one")
    return [s if n > 1 else 0 for s, n in zip(strides[:-1], shape[:-1])]


def _table(what: str, t: torch.Tensor, batch: int) -> int:
    """Checks a page table; returns the stride of its rows (0: dense)."""
    if t.dtype != torch.int32 or t.dim() != 2 or t.shape[0] != batch or \
            not (t.is_contiguous() or (t.stride(1) == 1 and t.stride(0) >= t.shape[1])):
        raise ValueError(f"{what}: page_table is int32 [batch, max_pages]")
    return t.stride(0) if batch > 1 else 0


def draft_verify(target: torch.Tensor, tokens: torch.Tensor, u: torch.Tensor, draft: torch.Tensor | None = None,
                 parents: torch.Tensor | None = None, num_nodes: torch.Tensor | None = None, chances: bool = False):
    """Verifies a tree (parents given) or chain of drafted tokens against the target's probabilities.

    target [batch, nodes, vocab]; tokens int32 or int64 [batch, nodes] (column 0, the last token already decided, is not
    read); u float32 [batch, nodes] uniform numbers, column 0 for the last token; draft [batch, draft_rows, vocab], the
    distributions that the children of nodes 0 .. draft_rows - 1 were drawn from, or None for tokens drafted with certainty;
    parents int32 [batch, nodes]; num_nodes int32 [batch].
    Returns (path int32 [batch, nodes], count int32 [batch], token [batch]), and chance float32 [batch, nodes] if asked."""
    what = "draft_verify"
    index = _one_device(what, target, tokens, u, draft, parents, num_nodes)
    ts = _strides(what, "target", target, 3)
    batch, nodes, vocab = target.shape
    ds, rows = (0, 0), 0
    if draft is not None:
        ds, rows = _strides(what, "draft", draft, 3), draft.shape[1]
        if draft.dtype != target.dtype or draft.shape[0] != batch or draft.shape[2] != vocab:
            raise ValueError("draft_verify: draft has the type, batch and vocabulary of target")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError("draft_verify: tokens are int32 or int64")
    _whole(what, "tokens", tokens, (batch, nodes), tokens.dtype)
    _whole(what, "u", u, (batch, nodes), torch.float32)
    _whole(what, "parents", parents, (batch, nodes))
    _whole(what, "num_nodes", num_nodes, (batch,))
    desc = DraftVerifyDesc(batch, vocab, ts[0], ts[1], ds[0], ds[1], nodes, rows, dtype_tag(target),
                           I64 if tokens.dtype == torch.int64 else I32)
    path, token = torch.empty_like(tokens, dtype=torch.int32), tokens.new_empty(batch)
    count = path.new_empty(batch)
    chance = torch.empty_like(u) if chances else None
    _call(index, what, lib().vkop_cuda_draft_verify, C.byref(desc), target.data_ptr(), _ptr(draft), tokens.data_ptr(), _ptr(parents),
          _ptr(num_nodes), u.data_ptr(), path.data_ptr(), count.data_ptr(), token.data_ptr(), _ptr(chance))
    return (path, count, token, chance) if chances else (path, count, token)


def _tree_attention_desc(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                         scale: float | None, max_context: int, out: torch.Tensor | None) -> TreeAttentionDesc:
    what = "tree_attention"
    qs, ks, vs = _strides(what, "q", q, 4), _strides(what, "k_cache", k_cache, 4), _strides(what, "v_cache", v_cache, 4)
    os_ = _strides(what, "out", out, 4) if out is not None else (0, 0, 0)
    batch, nodes, heads, dim = q.shape
    pages, page_size, kv_heads, kv_dim = k_cache.shape
    if k_cache.shape != v_cache.shape or kv_dim != dim or k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError("tree_attention: k_cache and v_cache are [pages, page_size, kv_heads, head_dim] of q's type and head_dim")
    if out is not None and (out.shape != q.shape or out.dtype != q.dtype):
        raise ValueError("tree_attention: out has the shape and type of q")
    return TreeAttentionDesc(batch, pages, max_context, *qs, *os_, *ks, *vs, _table(what, page_table, batch), nodes,
                             heads, kv_heads, dim, page_size, page_table.shape[1], dtype_tag(q),
                             dim ** -0.5 if scale is None else scale)


def tree_attention_workspace_bytes(q, k_cache, v_cache, page_table, max_context: int = 0) -> int:
    """Scratch that tree_attention needs for tensors of these shapes."""
    n = C.c_size_t(0)
    desc = _tree_attention_desc(q, k_cache, v_cache, page_table, None, max_context, None)
    check(lib().vkop_cuda_tree_attention_workspace(C.byref(desc), C.byref(n)), "tree_attention_workspace")
    return int(n.value)


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                   context: torch.Tensor, parents: torch.Tensor | None = None, num_nodes: torch.Tensor | None = None,
                   scale: float | None = None, max_context: int = 0, return_lse: bool = False,
                   workspace: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """Attention of the nodes of a token tree (parents None: a chain) over a paged cache that holds the context and, from
    position context[b] on, the nodes themselves.

    q [batch, nodes, q_heads, head_dim]; k_cache, v_cache [pages, page_size, kv_heads, head_dim], any strides with a
    contiguous last dimension; page_table int32 [batch, max_pages]; context, num_nodes int32 [batch]; parents int32
    [batch, nodes]; max_context: an upper bound of context that the caller knows (0: the table's width).  workspace: a
    uint8 tensor of tree_attention_workspace_bytes() to use instead of torch's allocator.
    Returns out like q, and lse float32 [batch, nodes, q_heads] if asked."""
    what = "tree_attention"
    index = _one_device(what, q, k_cache, v_cache, page_table, context, parents, num_nodes, workspace, out)
    desc = _tree_attention_desc(q, k_cache, v_cache, page_table, scale, max_context, out)
    batch, nodes, heads = desc.batch, desc.nodes, desc.q_heads
    _whole(what, "context", context, (batch,))
    _whole(what, "parents", parents, (batch, nodes))
    _whole(what, "num_nodes", num_nodes, (batch,))
    if workspace is not None and (workspace.dtype != torch.uint8 or not workspace.is_contiguous()):
        raise ValueError("tree_attention: workspace is a contiguous uint8 tensor")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)  # half the cost of new_empty(shape)
    lse = torch.empty(batch, nodes, heads, dtype=torch.float32, device=q.device) if return_lse else None
    L, ref = lib(), C.byref(desc)
    if workspace is None:
        need = C.c_size_t(0)
        check(L.vkop_cuda_tree_attention_workspace(ref, C.byref(need)), what)
        if need.value:
            workspace = q.new_empty(need.value, dtype=torch.uint8)
    nbytes = 0 if workspace is None else workspace.numel()
    _call(index, what, L.vkop_cuda_tree_attention, ref, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(),
          context.data_ptr(), _ptr(parents), _ptr(num_nodes), out.data_ptr(), _ptr(lse), _ptr(workspace), nbytes)
    return (out, lse) if return_lse else out


def cache_compact(k_cache: torch.Tensor, v_cache: torch.Tensor | None, page_table: torch.Tensor, context: torch.Tensor,
                  path: torch.Tensor, count: torch.Tensor) -> torch.Tensor:
    """Moves the cache rows of an accepted path (as draft_verify returns it) to the front of the drafted positions, in
    place.  k_cache, v_cache [layers, pages, page_size, kv_heads, head_dim], or without the first dimension for one layer.
    Returns the new context lengths, int32 [batch]."""
    what = "cache_compact"
    index = _one_device(what, k_cache, v_cache, page_table, context, path, count)
    if k_cache.dim() == 4:
        k_cache, v_cache = k_cache[None], v_cache[None] if v_cache is not None else None
    ks = _strides(what, "k_cache", k_cache, 5)
    vs = _strides(what, "v_cache", v_cache, 5) if v_cache is not None else (0, 0, 0, 0)
    if v_cache is not None and (v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype):
        raise ValueError("cache_compact: k_cache and v_cache have one shape and type")
    layers, pages, page_size, heads, dim = k_cache.shape
    batch = context.shape[0]
    if path.dim() != 2:
        raise ValueError("cache_compact: path is int32 [batch, nodes]")
    nodes = path.shape[1]
    _whole(what, "context", context, (batch,))
    _whole(what, "path", path, (batch, nodes))
    _whole(what, "count", count, (batch,))
    desc = CacheCompactDesc(batch, pages, *ks, *vs, _table(what, page_table, batch), layers, nodes, heads, dim,
                            page_size, page_table.shape[1], dtype_tag(k_cache), 0)
    lengths = torch.empty_like(context)
    _call(index, what, lib().vkop_cuda_cache_compact, C.byref(desc), k_cache.data_ptr(), _ptr(v_cache), page_table.data_ptr(),
          context.data_ptr(), path.data_ptr(), count.data_ptr(), lengths.data_ptr())
    return lengths


def packets_push(packets: torch.Tensor, peer_slots: torch.Tensor, peer_flags: torch.Tensor, rank: int, world: int,
                 seq: int, tickets: torch.Tensor) -> None:
    """peer_slots / peer_flags: int64 CUDA tensors holding one device pointer per rank."""
    check(lib().vkop_cuda_packets_push(packets.data_ptr(), packets.numel() * packets.element_size(), peer_slots.data_ptr(),
                                       peer_flags.data_ptr(), rank, world, seq, tickets.data_ptr(), _stream()), "packets_push")


def packets_wait(flags: torch.Tensor, world: int, seq: int, status: torch.Tensor, max_polls: int = 1 << 20) -> None:
    check(lib().vkop_cuda_packets_wait(flags.data_ptr(), world, seq, max_polls, status.data_ptr(), _stream()), "packets_wait")


def packets_exchange_all_ranks(packet_ptrs: torch.Tensor, packets_bytes: int, peer_slots: torch.Tensor, peer_flags: torch.Tensor,
                               world: int, seq: int, ticket_ptrs: torch.Tensor, status: torch.Tensor, max_polls: int = 1 << 20) -> None:
    """Every rank's push and bounded wait of one step in one cooperative launch (ranks emulated on one GPU).
    packet_ptrs / ticket_ptrs / peer_slots / peer_flags: int64 CUDA tensors of one device pointer per rank."""
    check(lib().vkop_cuda_packets_exchange_all_ranks(packet_ptrs.data_ptr(), packets_bytes, peer_slots.data_ptr(), peer_flags.data_ptr(),
                                                     world, seq, ticket_ptrs.data_ptr(), max_polls, status.data_ptr(), _stream()),
          "packets_exchange_all_ranks")


def static_scratch_bytes() -> int:
    return int(lib().vkop_cuda_static_scratch_bytes())


def softmax_topk_static(logits: torch.Tensor, k: int, inv_temperature: float = 1.0, index_dtype: int = I32,
                        value_kind: int = VALUE_PROBABILITY, out=None):
    """Fused softmax + top-k through the entry point that takes no workspace and allocates nothing
    (the outputs are still the caller's: pass `out`, or they are created here with torch)."""
    if not logits.is_cuda:
        raise RuntimeError("vkop_b200 runs on CUDA device memory only")
    desc = make_desc(logits, k, inv_temperature, index_dtype, value_kind, True, PATH_AUTO, 0, 0, 0)
    if out is None:
        values = torch.empty((logits.shape[0], k), dtype=logits.dtype, device=logits.device)
        indices = torch.empty((logits.shape[0], k), dtype=torch.int64 if index_dtype == I64 else torch.int32,
                              device=logits.device)
    else:
        values, indices = out
    check(lib().vkop_cuda_softmax_topk_static(C.byref(desc), logits.data_ptr(), values.data_ptr(), indices.data_ptr(),
                                              _stream()), "softmax_topk_static")
    return values, indices


def softmax(x: torch.Tensor, axis: int = -1, inv_temperature: float = 1.0) -> torch.Tensor:
    if not x.is_cuda:
        raise RuntimeError("vkop_b200 runs on CUDA device memory only")
    x = x.contiguous()
    axis = axis % x.dim()
    outer = 1
    for s in x.shape[:axis]:
        outer *= s
    inner = 1
    for s in x.shape[axis + 1:]:
        inner *= s
    desc = SoftmaxDesc(outer=outer, axis_len=x.shape[axis], inner=inner, dtype=dtype_tag(x),
                       inv_temperature=inv_temperature)
    out = torch.empty_like(x)
    check(lib().vkop_cuda_softmax(C.byref(desc), x.data_ptr(), out.data_ptr(), _stream()), "softmax")
    return out


def packet_bytes(k: int) -> int:
    return int(lib().vkop_cuda_packet_bytes(k))


def softmax_topk_partial(shard: torch.Tensor, k: int, index_offset: int, inv_temperature: float = 1.0,
                         workspace: Workspace | None = None, packets: torch.Tensor | None = None,
                         path: int = PATH_AUTO, splits: int = 0):
    """Per-shard packets [rows, packet_bytes/4] (uint32 words held in an int32 tensor)."""
    desc = make_desc(shard, k, inv_temperature, index_offset=index_offset, path=path, splits=splits)
    need = softmax_topk_workspace_bytes(desc)
    if workspace is None or workspace.nbytes < need:
        workspace = Workspace(need, shard.device)
    if packets is None:
        packets = torch.empty((shard.shape[0], packet_bytes(k) // 4), dtype=torch.int32, device=shard.device)
    check(lib().vkop_cuda_softmax_topk_partial(C.byref(desc), shard.data_ptr(), packets.data_ptr(), workspace.ptr,
                                               workspace.buf.numel(), _stream()), "softmax_topk_partial")
    return packets


def softmax_topk_merge(packets: torch.Tensor, rows: int, k: int, dtype: torch.dtype, inv_temperature: float = 1.0,
                       index_dtype: int = I32, out=None):
    """packets: [shards, rows, words] as gathered.  Returns (values, indices)."""
    shards = packets.shape[0]
    desc = SoftmaxTopkDesc(rows=rows, cols=1, row_stride=0, dtype=_TORCH_DTYPE[dtype], k=k, index_dtype=index_dtype,
                           value_kind=VALUE_PROBABILITY, inv_temperature=inv_temperature, largest=1, path=0, splits=0,
                           index_offset=0)
    if out is None:
        values = torch.empty((rows, k), dtype=dtype, device=packets.device)
        indices = torch.empty((rows, k), dtype=torch.int64 if index_dtype == I64 else torch.int32,
                              device=packets.device)
    else:
        values, indices = out
    check(lib().vkop_cuda_softmax_topk_merge(C.byref(desc), packets.data_ptr(), shards, values.data_ptr(),
                                             indices.data_ptr(), _stream()), "softmax_topk_merge")
    return values, indices


def nms_workspace_bytes(desc: NmsDesc) -> int:
    n = C.c_size_t(0)
    check(lib().vkop_cuda_nms_workspace(C.byref(desc), C.byref(n)), "nms_workspace")
    return int(n.value)


def nms(boxes: torch.Tensor, scores: torch.Tensor, center_point_box: int = 0, max_output_boxes_per_class: int = 0,
        iou_threshold: float = 0.0, score_threshold: float = 0.0, pre_topk: int = 0, capacity_rows: int | None = None,
        workspace: Workspace | None = None, out=None):
    """Returns (rows int32 [capacity,3] device tensor, count int32 [1] device tensor)."""
    if not (boxes.is_cuda and scores.is_cuda):
        raise RuntimeError("vkop_b200 runs on CUDA device memory only")
    B, N, four = boxes.shape
    assert four == 4 and boxes.dtype == torch.float32 and scores.dtype == torch.float32
    Cn = scores.shape[1]
    assert scores.shape[0] == B and scores.shape[2] == N
    boxes, scores = boxes.contiguous(), scores.contiguous()
    if capacity_rows is None:
        per = max_output_boxes_per_class if max_output_boxes_per_class > 0 else (pre_topk if pre_topk > 0 else N)
        capacity_rows = B * Cn * min(per, N)
    desc = NmsDesc(num_batch=B, num_class=Cn, num_boxes=N, center_point_box=center_point_box,
                   max_output_boxes_per_class=max_output_boxes_per_class, pre_topk=pre_topk,
                   iou_threshold=iou_threshold, score_threshold=score_threshold, capacity_rows=capacity_rows)
    need = nms_workspace_bytes(desc)
    if workspace is None or workspace.nbytes < need:
        workspace = Workspace(need, boxes.device)
    if out is None:
        rows = torch.empty((max(capacity_rows, 1), 3), dtype=torch.int32, device=boxes.device)
        count = torch.empty(1, dtype=torch.int32, device=boxes.device)
    else:
        rows, count = out
    check(lib().vkop_cuda_nms(C.byref(desc), boxes.data_ptr(), scores.data_ptr(), rows.data_ptr(), count.data_ptr(),
                              workspace.ptr, workspace.buf.numel(), _stream()), "nms")
    return rows, count
