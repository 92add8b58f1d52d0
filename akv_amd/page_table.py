"""Decode metadata over compacted request rows (host side of the HIP kernels).

Mirrors the reference's decode-index path:

* ``context_decode_indices`` / ``context_window_lengths``
  (``akv/system/sglang/kernels/ops/attention/context_page_table.py:7-76``)
  -> ``akv_decode_indices`` / ``akv_window_lengths``;
* ``kv_indptr[1:] = cumsum(seq_lens)`` (``akv/system/sglang.patch:2266-2268``)
  -> ``akv_build_indptr``;
* ``ReqToTokenPool.write`` through side rows (``sglang.patch:4230-4235``)
  -> ``akv_write_row_slots``;
* the new tokens' side of a step (slots, positions, block tables, tree masks),
  which the reference builds on the host -> ``akv_step_maps``.

The reference's decode registry (``context_backend.py:666-809``) calls these
with its own int64 rows ``(raw_ids_ptr, positions_ptr, prompt_len, active,
next_pos, row_ptr)``, one per request-table row; a row of zeros is an
ordinary request read straight from its table row.
"""

import torch

from . import _lib
from .ops import _on_device, current_stream_handle

_INDEX_DTYPES = {torch.int32: _lib.AKV_I32, torch.int64: _lib.AKV_I64}


def _idx(t, name):
    if t is None:
        return None, _lib.AKV_I32
    code = _INDEX_DTYPES.get(t.dtype)
    if code is None or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32/int64 tensor")
    return t.data_ptr(), code


def _status_ptr(status, device):
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() < 1 or status.device != device:
        raise ValueError("status must be an int32 device word on the output's device")
    return status.data_ptr()


def context_decode_indices(registry, table, rows, lengths, indptr, output, *, starts=None,
                           mapping=None, multiplier=1, status=None):
    """``out[indptr[b] + i] = T(row[raw])`` over ``len(lengths)`` requests.

    ``status``: the compaction's device status word when the registry rows
    point at its decode layout; the kernel then skips its reads and writes
    on the device when that compaction's outputs are unusable."""
    if registry.dtype != torch.int64 or registry.ndim != 2 or registry.shape[1] != 6:
        raise ValueError("registry must be int64 [rows, 6]")
    if table.dtype != torch.int32 or table.stride(-1) != 1:
        raise ValueError("the request table must be int32 with unit column stride")
    rows_p, rows_t = _idx(rows, "rows")
    len_p, len_t = _idx(lengths, "lengths")
    ind_p, ind_t = _idx(indptr, "indptr")
    out_p, out_t = _idx(output, "output")
    st_p, st_t = _idx(starts, "starts")
    map_p, map_t = _idx(mapping, "mapping")
    device = output.device
    with _on_device(device):
        rc = _lib.calls().akv_decode_indices(
            registry.data_ptr(), table.data_ptr(), table.stride(0), rows_p, rows_t, len_p, len_t,
            ind_p, ind_t, out_p, out_t, st_p, st_t, map_p, map_t, int(multiplier), len(lengths),
            _status_ptr(status, device), current_stream_handle(device),
        )
    _lib.check(rc, "akv_decode_indices")


def context_window_lengths(registry, rows, lengths, output, window, *, starts=None):
    """Visible key counts for an inclusive ``window``; optionally ``starts = lengths - output``."""
    rows_p, rows_t = _idx(rows, "rows")
    len_p, len_t = _idx(lengths, "lengths")
    out_p, out_t = _idx(output, "output")
    if starts is not None and starts.dtype != lengths.dtype:
        raise ValueError("starts must have the dtype of lengths")
    device = output.device
    with _on_device(device):
        rc = _lib.calls().akv_window_lengths(
            registry.data_ptr(), rows_p, rows_t, len_p, len_t, out_p, out_t, _lib.ptr(starts),
            int(window), len(lengths), current_stream_handle(device),
        )
    _lib.check(rc, "akv_window_lengths")


def build_indptr(lengths, indptr, *, last_page_len=None, page_size=1):
    """``indptr[0] = 0; indptr[1:] = cumsum(lengths)`` (+ last-page lengths)."""
    len_p, len_t = _idx(lengths, "lengths")
    ind_p, ind_t = _idx(indptr, "indptr")
    if last_page_len is not None and last_page_len.dtype != torch.int32:
        raise ValueError("last_page_len must be int32")
    device = indptr.device
    with _on_device(device):
        rc = _lib.calls().akv_build_indptr(
            len_p, len_t, len(lengths), ind_p, ind_t, _lib.ptr(last_page_len), int(page_size), 1,
            current_stream_handle(device),
        )
    _lib.check(rc, "akv_build_indptr")


def table_indptr(batch, stride, indptr):
    """Page-table form ``indptr[b] = b * stride`` for ``b`` in ``[0, batch]``."""
    ind_p, ind_t = _idx(indptr, "indptr")
    if stride == 1:
        # a scale of 1 would select the cumulative-sum form
        raise ValueError("table_indptr needs a row stride other than 1")
    device = indptr.device
    with _on_device(device):
        rc = _lib.calls().akv_build_indptr(
            None, _lib.AKV_I32, batch, ind_p, ind_t, None, 1, int(stride), current_stream_handle(device)
        )
    _lib.check(rc, "akv_build_indptr")


def write_row_slots(pointers, rows, columns, values):
    """``((int32*)pointers[rows[i]])[columns[i]] = values[i]`` (side-row scatter)."""
    if pointers.dtype != torch.int64:
        raise ValueError("row pointers must be int64 addresses")
    rows_p, rows_t = _idx(rows, "rows")
    col_p, col_t = _idx(columns, "columns")
    val_p, val_t = _idx(values, "values")
    device = pointers.device
    with _on_device(device):
        rc = _lib.calls().akv_write_row_slots(
            pointers.data_ptr(), rows_p, rows_t, col_p, col_t, val_p, val_t, rows.numel(),
            current_stream_handle(device),
        )
    _lib.check(rc, "akv_write_row_slots")


def write_req_to_token_pool(req_to_token, req_pool_indices, prefix_tensors, pre_lens, seq_lens, extend_lens,
                            out_cache_loc, row_pointers=None, *, prefix_dtype=torch.int64):
    """Extend write of request rows: ``write_req_to_token_pool_triton`` with
    ``RowPointers`` (``akv/system/sglang.patch:238-278``).

    For request ``b`` (table row ``r = req_pool_indices[b]``, or the side row
    ``row_pointers[r]`` when given): the first ``pre_lens[b]`` entries come
    from the array at address ``prefix_tensors[b]`` (``prefix_dtype``), the
    next ``seq_lens[b] - pre_lens[b]`` from ``out_cache_loc`` after the
    earlier requests' ``extend_lens``.
    """
    if req_to_token.dtype != torch.int32 or req_to_token.stride(-1) != 1:
        raise ValueError("the request table must be int32 with unit column stride")
    if prefix_tensors.dtype != torch.int64 or (row_pointers is not None and row_pointers.dtype != torch.int64):
        raise ValueError("prefix tensors and row pointers must be int64 addresses")
    if pre_lens.dtype != seq_lens.dtype or extend_lens.dtype != seq_lens.dtype:
        raise ValueError("pre_lens, seq_lens and extend_lens must share one dtype")
    rows_p, rows_t = _idx(req_pool_indices, "req_pool_indices")
    len_t = _idx(seq_lens, "seq_lens")[1]
    loc_p, loc_t = _idx(out_cache_loc, "out_cache_loc")
    prefix_t = _INDEX_DTYPES.get(prefix_dtype)
    if prefix_t is None:
        raise ValueError("prefix_dtype must be int32 or int64")
    device = req_to_token.device
    with _on_device(device):
        rc = _lib.calls().akv_write_extend_rows(
            req_to_token.data_ptr(), req_to_token.stride(0), _lib.ptr(row_pointers), rows_p, rows_t,
            prefix_tensors.data_ptr(), prefix_t, pre_lens.data_ptr(), seq_lens.data_ptr(), extend_lens.data_ptr(),
            len_t, loc_p, loc_t, len(req_pool_indices), current_stream_handle(device),
        )
    _lib.check(rc, "akv_write_extend_rows")


def context_step_maps(registry, table, rows, seq_lens, new_lens, qo_indptr, kv_indptr, slot_map, positions, *,
                      block_tables=None, page_size=1, parents=None, tree_mask=None, window=None, window_mask=None,
                      window_starts=None, status=None):
    """The metadata of a step's new tokens from request lengths, in one launch.

    Request b has ``seq_lens[b]`` ranks, the last ``new_lens[b]`` of them new
    (decoded or drafted tokens, or a prefill chunk), whose slots and positions
    follow from its registry row as in ``context_decode_indices``.  Writes

    * ``qo_indptr`` / ``kv_indptr`` ``[B + 1]``: cumulative sums of both;
    * ``slot_map`` / ``positions`` ``[N]``: each new token's slot and position;
      -1 and 0 behind the last one, so a padded batch stores nothing there;
    * ``block_tables`` int32 ``[B, pages]``: the page of every ``page_size``-th
      rank, -1 behind the request's last;
    * ``tree_mask`` int64 ``[N, words]``: bit a of token i's row when new token
      a is i or one of its ancestors.  ``parents`` int32 ``[N]`` names each
      token's parent by its number among the request's new tokens (an earlier
      one; anything else: none); without it a request's tokens are a chain.  A
      tree's node i has the position of the first new rank plus its depth, a
      chain's that of its own rank;
    * for layers with a sliding ``window`` (a key is visible when
      ``q_pos - k_pos <= window``): ``window_mask``, the ancestors inside it
      (itself too),
      and ``window_starts`` int32 ``[N]``, the first earlier key inside it.

    ``rows`` may be int32 or int64; ``seq_lens`` and ``new_lens`` share either,
    as do the indptrs; a mask has a word per 64 new tokens of a request.  A
    request of length 0 (a padded batch's last ones) may name any row.
    ``status``: as for ``context_decode_indices``.
    """
    # one read of every property: the checks are most of the call's time
    at = slot_map.get_device()
    if registry.dtype != torch.int64 or registry.ndim != 2 or registry.shape[1] != 6 or not registry.is_contiguous():
        raise ValueError("registry must be contiguous int64 [rows, 6]")
    table_shape, table_stride = table.shape, table.stride()
    if table.dtype != torch.int32 or len(table_shape) != 2 or table_stride[1] != 1:
        raise ValueError("the request table must be int32 [rows, width] with unit column stride")
    batch = seq_lens.numel()
    if new_lens.dtype != seq_lens.dtype or new_lens.numel() != batch or rows.numel() != batch:
        raise ValueError("rows, seq_lens and new_lens must have one entry per request, the lengths one dtype")
    if qo_indptr.dtype != kv_indptr.dtype or qo_indptr.numel() != batch + 1 or kv_indptr.numel() != batch + 1:
        raise ValueError("qo_indptr and kv_indptr must be [requests + 1] of one dtype")
    rows_p, rows_t = _idx(rows, "rows")
    seq_p, len_t = _idx(seq_lens, "seq_lens")
    new_p, _ = _idx(new_lens, "new_lens")
    qo_p, ind_t = _idx(qo_indptr, "qo_indptr")
    kv_p, _ = _idx(kv_indptr, "kv_indptr")
    slot_p, slot_t = _idx(slot_map, "slot_map")
    pos_p, pos_t = _idx(positions, "positions")
    n = slot_map.numel()
    if positions.numel() != n:
        raise ValueError("slot_map and positions must have one entry per token")
    one_device = at >= 0 and (at == registry.get_device() == table.get_device() == rows.get_device()
                              == seq_lens.get_device() == new_lens.get_device() == qo_indptr.get_device()
                              == kv_indptr.get_device() == positions.get_device())
    block_args = (None, 0, 0)
    if block_tables is not None:
        shape, stride = block_tables.shape, block_tables.stride()
        if block_tables.dtype != torch.int32 or len(shape) != 2 or shape[0] != batch \
                or (stride[1] != 1 and block_tables.numel()) or (batch > 1 and stride[0] < shape[1]):
            raise ValueError("block_tables must be int32 [requests, pages] with unit column stride, without overlap")
        block_args = (block_tables.data_ptr(), stride[0], shape[1])
        one_device &= block_tables.get_device() == at
    if parents is not None:
        if parents.dtype != torch.int32 or parents.numel() != n or not parents.is_contiguous():
            raise ValueError("parents must be contiguous int32 with one entry per token")
        one_device &= parents.get_device() == at
    if window is None and (window_mask is not None or window_starts is not None):
        raise ValueError("window_mask and window_starts need a window")
    mask_args = [(None, 0, 0), (None, 0, 0)]
    for i, mask in enumerate((tree_mask, window_mask)):
        if mask is None:
            continue
        shape, stride = mask.shape, mask.stride()
        if mask.dtype != torch.int64 or len(shape) != 2 or shape[0] != n or (stride[1] != 1 and mask.numel()) \
                or (n > 1 and stride[0] < shape[1]):
            raise ValueError("masks must be int64 words [tokens, words] with unit word stride, without overlap")
        mask_args[i] = (mask.data_ptr(), stride[0], shape[1])
        one_device &= mask.get_device() == at
    if window_starts is not None:
        if window_starts.dtype != torch.int32 or window_starts.numel() != n or not window_starts.is_contiguous():
            raise ValueError("window_starts must be contiguous int32 with one entry per token")
        one_device &= window_starts.get_device() == at
    if not one_device:
        raise ValueError("step maps' tensors must be on one GPU")
    device = slot_map.device
    with _on_device(device):
        rc = _lib.calls().akv_step_maps(
            registry.data_ptr(), table.data_ptr(), table_stride[0], table_shape[1], rows_p, rows_t, seq_p, new_p,
            len_t, batch, qo_p, kv_p, ind_t, n, slot_p, slot_t, pos_p, pos_t, *block_args, int(page_size),
            None if parents is None else parents.data_ptr(), *mask_args[0], 0 if window is None else int(window),
            *mask_args[1], None if window_starts is None else window_starts.data_ptr(), _status_ptr(status, device),
            current_stream_handle(device),
        )
    if rc:
        _lib.check(rc, "akv_step_maps")
