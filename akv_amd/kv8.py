"""A KV cache held in 8 bits, with a scale for each block of slots and head.

A layer's cache: ``k_buffer`` / ``v_buffer`` ``[slots, kv_heads, D]`` of
``torch.float8_e4m3fn`` or ``torch.float8_e5m2`` codes, and ``k_scales`` /
``v_scales`` f32 ``[blocks, kv_heads]``, block ``slot // scale_block``; a value
is its code times its scale.  ``scale_block`` is a power of two up to 64: 1 for
pools whose slots are handed out one by one, up to the page size for pages,
which are filled in order.  Half the bytes of the bf16 pool, on the same path:

* ``append_kv8``              new K/V rows, rotated on the way (beside
                              ``qk_norm.qk_norm_rope``, which may norm and
                              rotate before it);
* ``reposition_kv8_layers``   the Reposition of kept rows (beside
                              ``ops.reposition_kv_layers_gated``, and like it
                              fed by ``tables.compact_rows`` / ``compact_pages``);
* ``attention_kv8``           attention of new tokens over the cache (beside
                              ``attention.tree_attention``, over the metadata
                              of ``page_table``).

``transfer.copy_kv_rows`` moves its rows between pools as they are (rows of codes,
and with ``scale_block`` 1 rows of scales).  The reference keeps unquantized KV
only (``akv/system/sglang/kernels/ops/attention/context_reposition.py:149-152``).
"""

import torch

from . import _lib
from .ops import _KV_DTYPES, _on_device, _raw_device, current_stream_handle

_INDEX = {torch.int32: _lib.AKV_I32, torch.int64: _lib.AKV_I64}
_POINTERS = (torch.int64, torch.uint64)
_FORMATS = {torch.float8_e4m3fn: _lib.AKV_E4M3, torch.float8_e5m2: _lib.AKV_E5M2}


def _cache(k_buffer, v_buffer, k_scales, v_scales, scale_block, at):
    """Checks one layer's cache on device index ``at``; returns its format, shape
    and the four tensors' strides."""
    form, shape = _FORMATS.get(k_buffer.dtype), k_buffer.shape
    k_stride, v_stride = k_buffer.stride(), v_buffer.stride()
    if form is None or len(shape) != 3 or v_buffer.shape != shape or v_buffer.dtype != k_buffer.dtype \
            or k_stride[2] != 1 or v_stride[2] != 1:
        raise ValueError("K/V must be matching float8_e4m3fn or float8_e5m2 [slots, kv_heads, head_dim] buffers")
    if type(scale_block) is not int or not 0 < scale_block <= 64 or scale_block & (scale_block - 1):
        raise ValueError("scale_block must be a power of two up to 64")
    k_blocks, v_blocks = k_scales.shape, v_scales.shape
    if k_scales.dtype != torch.float32 or v_scales.dtype != torch.float32 or len(k_blocks) != 2 or len(v_blocks) != 2 \
            or min(k_blocks[0], v_blocks[0]) * scale_block < shape[0] or not k_blocks[1] == v_blocks[1] == shape[1]:
        raise ValueError("k_scales / v_scales must be f32 [slots / scale_block, kv_heads]")
    if at < 0 or not (k_buffer.get_device() == v_buffer.get_device() == k_scales.get_device()
                      == v_scales.get_device() == at):
        raise ValueError("the 8-bit cache's tensors must be on one GPU")
    return form, shape, k_stride, v_stride, k_scales.stride(), v_scales.stride()


def _launch(call, device, args):
    """``call(*args)`` with ``device`` current."""
    if _raw_device() == device.index:
        return call(*args)
    with _on_device(device):
        return call(*args)


def append_kv8(k, v, slot_map, k_buffer, v_buffer, k_scales, v_scales, *, scale_block=1, positions=None,
               cos_sin_cache=None, rotary_dim=None, is_neox_style=True, q=None, q_out=None):
    """New K/V rows into the cache, K (and ``q``) rotated on the way.

    ``k`` / ``v`` ``[N, kv_heads, D]`` in bf16, fp16 or fp32 (views of a fused
    projection will do), D a multiple of 16 up to 128; ``slot_map`` int32 or
    int64 ``[N]``, entries outside the pool (-1: padding) take nothing.  With
    ``cos_sin_cache`` ``[positions, rotary_dim]``, K's first ``rotary_dim`` dims
    are rotated by its rows ``positions`` ``[N]`` in fp32, and ``q`` ``[N,
    q_heads, D]`` goes, rotated and rounded once, to ``q_out`` (which may be
    ``q``); a position outside the table gives NaN.  Without a table K is stored
    as it is (rows that ``qk_norm_rope`` left in ``k_out``).

    A block's tokens follow one another in a call, their slots distinct and
    ascending by 1, and blocks are filled in order (the list is not checked: a block that is
    come to twice has no defined content).  Scales that blocks or heads share
    (stride 0) are refused, here and by the Reposition.  A block begun by a call gets, per head, the
    smallest power of two s >= 2^-100 that holds its rows (magnitude <= 448 s, or
    57344 s in e5m2) as its scale; behind earlier rows its scale is
    doubled as often as the new rows need, and the earlier codes are rounded
    again in its units.  Values are rounded to nearest even; infinities and NaN do
    not enter the scales, and stay what the format has of them (e4m3: NaN).
    """
    dtype, at = k.dtype, k.get_device()
    k_shape, k_stride, v_stride = k.shape, k.stride(), v.stride()
    if dtype not in _KV_DTYPES or len(k_shape) != 3 or k_stride[2] != 1 or v.shape != k_shape or v.dtype != dtype \
            or v.get_device() != at or v_stride[2] != 1:
        raise ValueError("k and v must be matching float32, float16 or bfloat16 [tokens, kv_heads, head_dim] rows")
    n, hk, d = k_shape
    form, pool, kb, vb, ks, vs = _cache(k_buffer, v_buffer, k_scales, v_scales, scale_block, at)
    if pool[1] != hk or pool[2] != d:
        raise ValueError("the cache must have k's heads and head_dim")
    slots_t = _INDEX.get(slot_map.dtype)
    if slots_t is None or slot_map.shape != (n,) or slot_map.get_device() != at or not slot_map.is_contiguous():
        raise ValueError("slot_map must be a contiguous int32/int64 [tokens] tensor on k's device")
    q_args, out_args, hq = (None, 0, 0), (None, 0, 0), 0
    if cos_sin_cache is None:
        if positions is not None or q is not None or q_out is not None or rotary_dim is not None:
            raise ValueError("the rotation needs positions and a cos/sin cache")
        rope = (None, _lib.AKV_I32, None, _lib.AKV_F32, 0, 0)
        rotary_dim = 0
    else:
        table, table_t, rope_shape = cos_sin_cache.stride(), _KV_DTYPES.get(cos_sin_cache.dtype), cos_sin_cache.shape
        if rotary_dim is None:
            rotary_dim = d
        if type(rotary_dim) is not int or not 0 < rotary_dim <= d or rotary_dim % 2 or len(rope_shape) != 2 \
                or rope_shape[1] != rotary_dim or table[1] != 1 or table_t is None \
                or cos_sin_cache.get_device() != at:
            raise ValueError("the rotation needs a native cos/sin cache matching rotary_dim")
        positions_t = None if positions is None else _INDEX.get(positions.dtype)
        if positions_t is None or positions.shape != (n,) or positions.get_device() != at \
                or not positions.is_contiguous():
            raise ValueError("positions must be a contiguous int32/int64 [tokens] tensor on k's device")
        rope = (positions.data_ptr(), positions_t, cos_sin_cache.data_ptr(), table_t, table[0], rope_shape[0])
        if (q is None) != (q_out is None):
            raise ValueError("q and q_out go together")
        if q is not None:
            q_shape, q_stride, out_stride = q.shape, q.stride(), q_out.stride()
            if len(q_shape) != 3 or q_shape[0] != n or q_shape[2] != d or q.dtype != dtype or q.get_device() != at \
                    or q_stride[2] != 1 or q_out.shape != q_shape or q_out.dtype != dtype \
                    or q_out.get_device() != at or out_stride[2] != 1:
                raise ValueError("q and q_out must be [tokens, q_heads, head_dim] rows of k's dtype and device")
            hq = q_shape[1]
            q_args, out_args = (q.data_ptr(), q_stride[0], q_stride[1]), (q_out.data_ptr(), out_stride[0], out_stride[1])
    if n == 0:
        return
    device = k.device
    rc = _launch(_lib.calls().akv_kv8_append, device, (
        *q_args, k.data_ptr(), k_stride[0], k_stride[1], v.data_ptr(), v_stride[0], v_stride[1],
        _KV_DTYPES[dtype], n, hq, hk, d, rotary_dim, 1 if is_neox_style else 0, *rope, *out_args,
        slot_map.data_ptr(), slots_t, k_buffer.data_ptr(), v_buffer.data_ptr(), form, pool[0], kb[0], kb[1], vb[0],
        vb[1], k_scales.data_ptr(), v_scales.data_ptr(), scale_block, ks[0], ks[1], vs[0], vs[1],
        current_stream_handle(device),
    ))
    if rc:
        _lib.check(rc, "akv_kv8_append")


def reposition_kv8_layers(k_data_ptrs, v_data_ptrs, k_scale_ptrs, v_scale_ptrs, k_layout, v_layout, k_scale_layout,
                          v_scale_layout, source_slots, destination_slots, position_pairs, cos_sin_cache, *,
                          scale_block=1, is_neox_style=True, skip_unmapped=False, rotary_dim=None, status=None):
    """``ops.reposition_kv_layers`` over per-layer 8-bit caches, in one launch.

    The four ``*_ptrs`` are device tables of per-layer base addresses of code
    buffers and scales; every layer shares the exemplars' shapes, dtypes and
    strides.  A moved token's values are taken at its source's scale, K's rotary
    part turned in fp32 from ``position_pairs[t, 0]`` to ``[t, 1]`` (nothing is
    done where they are equal), and stored at its destination as ``append_kv8``
    stores rows: a block's destinations follow one another in the lists, ascending by
    1, and sources lie outside the blocks that the call writes.  With ``scale_block`` 1 a
    row that only moves keeps its values exactly, its scale a power of two as
    ``append_kv8`` leaves it: the least that holds the row (half as large where rounding
    took the row there; for zeros the least of all); rows under other scales are rounded
    again.  Slots outside the pool are passed over (with ``skip_unmapped`` 0, too): without
    a source a destination and its scale stay as they are, but in a block that other
    rows of the call come to its slot holds nothing any more.  A position outside the
    table gives a NaN K row.  ``status``: as for ``reposition_kv_layers_gated``.
    """
    at = k_layout.get_device()
    form, pool, kb, vb, ks, vs = _cache(k_layout, v_layout, k_scale_layout, v_scale_layout, scale_block, at)
    tables = (k_data_ptrs, v_data_ptrs, k_scale_ptrs, v_scale_ptrs)
    layers = k_data_ptrs.numel()
    for t in tables:
        if t.shape != (layers,) or t.dtype not in _POINTERS or not t.is_contiguous() or t.get_device() != at:
            raise ValueError("Reposition requires contiguous 64-bit layer pointer tables on the KV device")
    count = source_slots.numel()
    for t in (source_slots, destination_slots):
        if t.shape != (count,) or t.dtype != torch.int32 or not t.is_contiguous() or t.get_device() != at:
            raise ValueError("Reposition requires contiguous int32 slot vectors on the KV device")
    pair_stride, rope_shape = position_pairs.stride(), cos_sin_cache.shape
    if position_pairs.shape != (count, 2) or position_pairs.dtype != torch.int32 or pair_stride[1] != 1 \
            or position_pairs.get_device() != at:
        raise ValueError("Reposition requires int32 [N, 2] positions on the KV device")
    if rotary_dim is None:
        rotary_dim = pool[2]
    table, table_t = cos_sin_cache.stride(), _KV_DTYPES.get(cos_sin_cache.dtype)
    if type(rotary_dim) is not int or not 0 < rotary_dim <= pool[2] or rotary_dim % 2 or len(rope_shape) != 2 \
            or rope_shape[1] != rotary_dim or table[1] != 1 or table_t is None \
            or cos_sin_cache.get_device() != at:
        raise ValueError("Reposition requires a native cos/sin cache matching rotary_dim")
    if status is not None and (status.dtype != torch.int32 or status.numel() < 1 or status.get_device() != at):
        raise ValueError("status must be an int32 device word on the KV device")
    if count == 0 or layers == 0:
        return
    device = k_layout.device
    rc = _launch(_lib.calls().akv_kv8_reposition, device, (
        k_data_ptrs.data_ptr(), v_data_ptrs.data_ptr(), k_scale_ptrs.data_ptr(), v_scale_ptrs.data_ptr(), layers, form,
        pool[1], pool[2], rotary_dim, pool[0], kb[0], kb[1], vb[0], vb[1], scale_block, ks[0], ks[1], vs[0], vs[1],
        source_slots.data_ptr(), destination_slots.data_ptr(), position_pairs.data_ptr(), pair_stride[0], count,
        cos_sin_cache.data_ptr(), table_t, table[0], rope_shape[0], 1 if is_neox_style else 0, 1 if skip_unmapped else 0,
        None if status is None else status.data_ptr(), current_stream_handle(device),
    ))
    if rc:
        _lib.check(rc, "akv_kv8_reposition")


def attention_kv8_workspace_bytes(n_tokens, n_requests, q_heads, kv_heads, head_dim, max_len, max_new):
    """Device bytes ``attention_kv8`` needs for every batch of up to these tokens
    and requests, under bounds of up to these."""
    need = _lib.calls().akv_kv8_attention_workspace_bytes(n_tokens, n_requests, q_heads, kv_heads, head_dim, max_len,
                                                          max_new)
    if need < 0:
        raise ValueError("attention over an 8-bit cache takes head dims that are multiples of 16 up to 128 and whole "
                         "q groups")
    return need


def attention_kv8(q, k_buffer, v_buffer, k_scales, v_scales, qo_indptr, kv_indptr, kv_indices, out, *, scale, max_len,
                  max_new, page_size=1, scale_block=1, tree_mask=None, key_starts=None, first_keys=0, sinks=None,
                  workspace=None, status=None):
    """Attention of each request's new tokens over an 8-bit cache.

    ``attention.tree_attention`` for a cache with scales, of any number of new
    tokens: one decodes, a tree verifies drafted tokens, a long chain extends by
    a chunk.  ``q`` / ``out`` ``[N, q_heads, D]`` (bf16 or fp16 q; q's dtype or
    f32 out), D a multiple of 16 up to 128; the cache holds the new tokens' own
    rows already.  Requests, slots or block tables, ``tree_mask``, ``sinks``,
    ``workspace`` and ``status`` are as there.  An earlier key of rank j is seen
    by token i if ``j < first_keys`` or ``j >= key_starts[i]`` (None: all), a
    sliding window with a few first keys that stay visible; ``max_len`` is then
    first_keys + window + n + 1.  Codes enter the products exactly; a weight times
    its key's V scale is rounded once to bf16 (fp16 q: to the sum of two bf16 values), and sums are
    fp32.  A code that is infinite or NaN makes that dim of the rows that see its
    key infinite or NaN, and reaches no other row.
    """
    # one read of every property: the checks are most of a small call's time
    dtype, at, q_shape, q_stride = q.dtype, q.get_device(), q.shape, q.stride()
    if dtype not in (torch.bfloat16, torch.float16) or len(q_shape) != 3 or q_stride[2] != 1:
        raise ValueError("q must be bf16 or fp16 [tokens, q_heads, head_dim] with unit dim stride")
    n, hq, d = q_shape
    form, pool, kb, vb, ks, vs = _cache(k_buffer, v_buffer, k_scales, v_scales, scale_block, at)
    if pool[2] != d:
        raise ValueError("q and the cache must have one head_dim")
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
    if type(first_keys) is not int or not 0 <= first_keys < 2 ** 31:
        raise ValueError("first_keys must be a count of keys")
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
    if not (out.get_device() == qo_indptr.get_device() == kv_indptr.get_device() == kv_indices.get_device() == at):
        raise ValueError("the attention's tensors must be on one GPU")
    if n == 0 or n_requests <= 0:
        return out
    device, hk = q.device, pool[1]
    lib = _lib.calls()
    if workspace is None:
        need = lib.akv_kv8_attention_workspace_bytes(n, n_requests, hq, hk, d, int(max_len), int(max_new))
        workspace = torch.empty(max(16, need), dtype=torch.uint8, device=device)
    elif workspace.get_device() != at or not workspace.is_contiguous():
        raise ValueError("the workspace must be contiguous, on q's device")
    rc = _launch(lib.akv_kv8_attention, device, (
        q_ptr, q_stride[0], q_stride[1], _KV_DTYPES[dtype], k_buffer.data_ptr(), v_buffer.data_ptr(), form, kb[0],
        kb[1], vb[0], vb[1], pool[0], k_scales.data_ptr(), v_scales.data_ptr(), scale_block, ks[0], ks[1], vs[0],
        vs[1], n, n_requests, hq, hk, d, qo_indptr.data_ptr(), kv_indptr.data_ptr(), indptr_t,
        kv_indices.data_ptr(), stride, width, int(page_size), *mask_args,
        None if key_starts is None else key_starts.data_ptr(), first_keys,
        None if sinks is None else sinks.data_ptr(), float(scale), out_ptr, _KV_DTYPES[out_dtype], out_stride[0],
        out_stride[1], int(max_len), int(max_new), workspace.data_ptr(), workspace.nbytes,
        None if status is None else status.data_ptr(), current_stream_handle(device),
    ))
    if rc:
        _lib.check(rc, "akv_kv8_attention")
    return out
