"""GQA decode attention with sinks over compacted indices (HIP, MFMA).

The consumer of the Drop + Reposition metadata: one decode step per layer
reading each request's keys through ``kv_indptr`` / ``kv_indices`` (a full
layer's compacted rows from ``compact_rows`` / ``ContextDecodeRegistry.fill``,
or a sliding-window layer's from ``fill_window``), normalised with per-head
sink logits exactly as the reference's ``o * sigmoid(lse - sink)``
(``akv/system/sglang/srt/layers/attention/context_backend.py:254-272``).
``tree_attention`` is its form for several drafted tokens per request, the
step that verifies a tree of them (speculative decoding, which the reference
rejects: ``akv/system/sglang/srt/context_system/capabilities.py:72-73``).
"""

import torch

from . import _lib
from .ops import _on_device, current_stream_handle

_INDEX = {torch.int32: _lib.AKV_I32, torch.int64: _lib.AKV_I64}
_TREE_DTYPES = {torch.bfloat16: _lib.AKV_BF16, torch.float16: _lib.AKV_F16, torch.float32: _lib.AKV_F32}


def workspace_bytes(n_requests, kv_heads, head_dim, max_len):
    return _lib.calls().akv_decode_attention_workspace_bytes(n_requests, kv_heads, head_dim, max_len)


def decode_attention(q, k_buffer, v_buffer, kv_indptr, kv_indices, out, *, scale, max_len, sinks=None,
                     workspace=None, status=None):
    """``out[b, h] = softmax-with-sink(scale * q[b, h] . K_j) . V_j`` over request b's indices.

    ``q``/``out``: ``[B, q_heads, D]`` (bf16 q; bf16 or f32 out); ``k_buffer``/
    ``v_buffer``: one layer's ``[slots, kv_heads, D]`` bf16 pool; ``kv_indptr``
    int32 ``[B+1]``; ``kv_indices`` int32; ``sinks`` f32 ``[q_heads]``;
    ``max_len``: host bound on every request's key count.  ``status``: the
    compaction's device status word when the indices come from it (the
    kernels then skip their work on the device when it reports them
    unusable).
    """
    if q.dtype != torch.bfloat16 or q.ndim != 3 or q.stride(-1) != 1:
        raise ValueError("q must be bf16 [B, q_heads, head_dim] with unit dim stride")
    if (k_buffer.dtype != torch.bfloat16 or v_buffer.dtype != torch.bfloat16 or k_buffer.ndim != 3
            or v_buffer.shape != k_buffer.shape or k_buffer.stride(-1) != 1 or v_buffer.stride(-1) != 1):
        raise ValueError("K/V must be matching bf16 [slots, kv_heads, head_dim] buffers")
    if out.dtype not in (torch.bfloat16, torch.float32) or out.shape != q.shape or out.stride(-1) != 1:
        raise ValueError("out must be bf16 or f32 shaped like q")
    if kv_indptr.dtype != torch.int32 or kv_indices.dtype != torch.int32 or len(kv_indptr) != q.shape[0] + 1:
        raise ValueError("kv_indptr / kv_indices must be int32, indptr of length B + 1")
    if sinks is not None and (sinks.dtype != torch.float32 or sinks.shape != (q.shape[1],)):
        raise ValueError("sinks must be f32 [q_heads]")
    if q.shape[2] != k_buffer.shape[2]:
        raise ValueError("q and K head dims differ")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1 or status.device != q.device):
        raise ValueError("status must be an int32 device word on q's device")
    n, hq, d = q.shape
    hkv = k_buffer.shape[1]
    need = workspace_bytes(n, hkv, d, max_len)
    if workspace is None:
        workspace = torch.empty(max(4, (need + 3) // 4), dtype=torch.float32, device=q.device)
    lib = _lib.calls()
    with _on_device(q.device):
        rc = lib.akv_decode_attention(
            q.data_ptr(), q.stride(0), q.stride(1), k_buffer.data_ptr(), v_buffer.data_ptr(),
            k_buffer.stride(0), k_buffer.stride(1), v_buffer.stride(0), v_buffer.stride(1), n, hq, hkv, d,
            kv_indptr.data_ptr(), kv_indices.data_ptr(), _lib.ptr(sinks), float(scale), out.data_ptr(),
            _lib.AKV_F32 if out.dtype == torch.float32 else _lib.AKV_BF16, out.stride(0), out.stride(1),
            int(max_len), workspace.data_ptr(), workspace.numel() * workspace.element_size(), _lib.ptr(status),
            current_stream_handle(q.device),
        )
    _lib.check(rc, "akv_decode_attention")
    return out


def tree_workspace_bytes(n_tokens, n_requests, q_heads, kv_heads, head_dim, max_len, max_new):
    """Device bytes ``tree_attention`` needs for every batch of up to these
    tokens and requests, under bounds of up to these."""
    need = _lib.calls().akv_tree_attention_workspace_bytes(n_tokens, n_requests, q_heads, kv_heads, head_dim, max_len,
                                                           max_new)
    if need < 0:
        raise ValueError("tree attention takes head dims that are multiples of 8 up to 128 and whole q groups")
    return need


def tree_attention(q, k_buffer, v_buffer, qo_indptr, kv_indptr, kv_indices, out, *, scale, max_len, max_new,
                   page_size=1, tree_mask=None, key_starts=None, sinks=None, workspace=None, status=None):
    """Attention of each request's drafted tokens over the cache and each other.

    ``q`` / ``out``: ``[N, q_heads, D]`` (bf16 or fp16 q; q's dtype or f32
    out), request b's tokens ``qo_indptr[b]:qo_indptr[b + 1]``, n of them;
    ``k_buffer`` / ``v_buffer``: one layer's ``[slots, kv_heads, D]`` pool,
    which holds the drafted tokens' own rows already.  Request b's
    ``kv_indptr[b + 1] - kv_indptr[b]`` keys end in those n; they lie at the
    slots ``kv_indices[kv_indptr[b]:]`` (1-D, ``context_decode_indices``), or on
    the pages of row b of a 2-D block table (``context_step_maps``), with
    ``page_size`` slots each.  Token i sees the request's earlier keys from
    rank ``key_starts[i]`` on (None: all), and of the drafted tokens those whose
    bit is set in its ``tree_mask`` row (int64 words ``[N, words]``, 0 past the
    last; None: a chain, each token itself and those before it).  A token that sees no key
    gets 0; a key at a slot outside the pool is seen by none.  ``sinks``: f32
    ``[q_heads]``.  ``max_len`` (keys a request's tokens reach: its keys, or
    window + n + 1) and ``max_new`` (its tokens) are host bounds that size the
    launch and the workspace; the results depend on them only in the order of
    their fp32 sums (and in whether an infinite value that a token sees makes
    that dim of its row infinite or NaN).  Rows of ``out``, which must not
    overlap ``q``, behind the last token stay as they are.  Head dims: multiples
    of 8 up to 128.  Weights are relative to a row's first scores and may grow to
    2^32 before they are rescaled, so bf16 values that a token sees are taken
    up to 2^94 in magnitude.  ``status``: as for ``decode_attention``.
    """
    # one read of every property: the checks are most of a small call's time
    dtype, at, q_shape, q_stride = q.dtype, q.get_device(), q.shape, q.stride()
    if dtype not in (torch.bfloat16, torch.float16) or len(q_shape) != 3 or q_stride[2] != 1:
        raise ValueError("q must be bf16 or fp16 [tokens, q_heads, head_dim] with unit dim stride")
    n, hq, d = q_shape
    pool, k_stride, v_stride = k_buffer.shape, k_buffer.stride(), v_buffer.stride()
    if len(pool) != 3 or v_buffer.shape != pool or pool[2] != d or k_buffer.dtype != dtype \
            or v_buffer.dtype != dtype or k_stride[2] != 1 or v_stride[2] != 1:
        raise ValueError("K/V must be matching [slots, kv_heads, head_dim] buffers of q's dtype and head_dim")
    out_dtype, out_stride = out.dtype, out.stride()
    if out.shape != q_shape or (out_dtype != dtype and out_dtype != torch.float32) or out_stride[2] != 1:
        raise ValueError("out must be shaped like q, of its dtype or f32")
    q_ptr, out_ptr = q.data_ptr(), out.data_ptr()
    if out_ptr == q_ptr and n:
        raise ValueError("out must not be q")
    indptr_t = _INDEX.get(qo_indptr.dtype)
    n_requests = qo_indptr.numel() - 1
    if indptr_t is None or kv_indptr.dtype != qo_indptr.dtype or qo_indptr.ndim != 1 or kv_indptr.ndim != 1 \
            or kv_indptr.numel() != n_requests + 1 or not qo_indptr.is_contiguous() or not kv_indptr.is_contiguous():
        raise ValueError("qo_indptr and kv_indptr must be contiguous [requests + 1] of one int32/int64 dtype")
    list_shape, list_stride = kv_indices.shape, kv_indices.stride()
    if kv_indices.dtype != torch.int32 or len(list_shape) not in (1, 2) or (list_stride[-1] != 1 and kv_indices.numel()):
        raise ValueError("kv_indices must be int32: a list of slots or a block table [requests, pages]")
    width, stride = list_shape[-1], 0
    if len(list_shape) == 2:
        stride = list_stride[0] if n_requests > 1 else max(1, width)
        if list_shape[0] != n_requests or stride < max(1, width):
            raise ValueError("the block table needs a row per request, without overlap")
    elif page_size != 1:
        raise ValueError("pages need a block table")
    mask_args = (None, 0, 0)
    if tree_mask is not None:
        mask_shape, mask_stride = tree_mask.shape, tree_mask.stride()
        if tree_mask.dtype != torch.int64 or len(mask_shape) != 2 or mask_shape[0] != n \
                or (mask_stride[1] != 1 and tree_mask.numel()) or tree_mask.get_device() != at:
            raise ValueError("tree_mask must be int64 words [tokens, words] on q's device")
        # (an empty tensor has no address, and no address is a chain: words of none are never read)
        mask_args = (tree_mask.data_ptr() or q_ptr, mask_stride[0], mask_shape[1])
    if key_starts is not None and (key_starts.dtype != torch.int32 or key_starts.ndim != 1 or key_starts.numel() != n
                                   or not key_starts.is_contiguous() or key_starts.get_device() != at):
        raise ValueError("key_starts must be contiguous int32 [tokens] on q's device")
    if sinks is not None and (sinks.dtype != torch.float32 or sinks.ndim != 1 or sinks.numel() != hq
                              or not sinks.is_contiguous() or sinks.get_device() != at):
        raise ValueError("sinks must be f32 [q_heads] on q's device")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1 or status.get_device() != at):
        raise ValueError("status must be an int32 device word on q's device")
    if at < 0 or not (k_buffer.get_device() == v_buffer.get_device() == out.get_device() == qo_indptr.get_device()
                      == kv_indptr.get_device() == kv_indices.get_device() == at):
        raise ValueError("tree attention's tensors must be on one GPU")
    if n == 0 or n_requests <= 0:
        return out
    device, hk = q.device, pool[1]
    lib = _lib.calls()
    if workspace is None:
        need = lib.akv_tree_attention_workspace_bytes(n, n_requests, hq, hk, d, int(max_len), int(max_new))
        workspace = torch.empty(max(16, need), dtype=torch.uint8, device=device)
    elif workspace.get_device() != at or not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous, on q's device")
    with _on_device(device):
        rc = lib.akv_tree_attention(
            q_ptr, q_stride[0], q_stride[1], k_buffer.data_ptr(), v_buffer.data_ptr(), k_stride[0], k_stride[1],
            v_stride[0], v_stride[1], pool[0], _TREE_DTYPES[dtype], n, n_requests, hq, hk, d, qo_indptr.data_ptr(),
            kv_indptr.data_ptr(), indptr_t, kv_indices.data_ptr(), stride, width, int(page_size), *mask_args,
            None if key_starts is None else key_starts.data_ptr(), None if sinks is None else sinks.data_ptr(),
            float(scale), out_ptr, _TREE_DTYPES[out_dtype], out_stride[0], out_stride[1], int(max_len), int(max_new),
            workspace.data_ptr(), workspace.nbytes, None if status is None else status.data_ptr(),
            current_stream_handle(device),
        )
    if rc:
        _lib.check(rc, "akv_tree_attention")
    return out
