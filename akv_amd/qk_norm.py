"""Per-head norms of queries and keys with the rotation and the pool write.

What a layer whose attention norms its heads does between the QKV product and
the attention over the pool: RMS norms of every q and k head, the position
rotation from the model's cos / sin table (the layout and pair styles the
Reposition reads, ``akv/system/sglang/kernels/ops/attention/
context_reposition.py:82-102``), and the new K and V rows stored at their
slots, in one launch of ``akv_qk_norm_rope``.  The keys it stores are the ones
``reposition_kv_layers`` moves later.
"""

import torch

from . import _lib
from .ops import _KV_DTYPES, _on_device, current_stream_handle

_INDEX = {torch.int32: _lib.AKV_I32, torch.int64: _lib.AKV_I64}


def qk_norm_rope(q, k, v, q_weight, k_weight, positions, cos_sin_cache, q_out, *, eps=1e-6, k_out=None,
                 slot_map=None, k_buffer=None, v_buffer=None, rotary_dim=None, is_neox_style=True):
    """``y = rotate(x / sqrt(mean(x^2) + eps) * weight)`` of every q and k head row.

    ``q`` ``[N, q_heads, D]``, ``k`` / ``v`` ``[N, kv_heads, D]`` (views of a
    fused projection will do: any token and head strides); ``q_weight`` /
    ``k_weight`` ``[D]`` or None (1); ``positions`` int32 or int64 ``[N]``, rows
    of ``cos_sin_cache`` ``[positions, rotary_dim]``.  Norm and rotation are in
    fp32 (a row's squares too: past its range the row comes out as 0), rounded
    once.  q goes to ``q_out`` (which may be ``q``), k to
    ``k_out`` (which may be ``k``) and, with ``k_buffer`` / ``v_buffer``
    ``[slots, kv_heads, D]``, k and v to rows ``slot_map`` int32 or int64
    ``[N]``, whose valid entries are distinct.  A token whose slot is outside
    the pool (-1: padding) writes no pool row; one whose position is outside
    the table gets NaN in q_out / k_out and no K pool row.  ``v`` is read only
    for the pool and may be None without it.  Head dims up to 512; rows that
    are 16-byte aligned, with D and rotary_dim multiples of 16, take the
    vector kernel.
    """
    # one read of every property: the checks are most of a small call's time
    dtype, at = q.dtype, q.get_device()
    if dtype not in _KV_DTYPES:
        raise ValueError("q, k and v must be float32, float16 or bfloat16")
    q_shape, k_shape, q_stride, k_stride = q.shape, k.shape, q.stride(), k.stride()
    if len(q_shape) != 3 or len(k_shape) != 3 or q_stride[2] != 1 or k_stride[2] != 1:
        raise ValueError("q and k must be [tokens, heads, head_dim] with unit dim stride")
    n, hq, d = q_shape
    hk = k_shape[1]
    if k.dtype != dtype or k.get_device() != at or k_shape[0] != n or k_shape[2] != d:
        raise ValueError("q and k must share tokens, head_dim, dtype and device")
    out_stride = q_out.stride()
    if q_out.shape != q_shape or q_out.dtype != dtype or q_out.get_device() != at or out_stride[2] != 1:
        raise ValueError("q_out must be shaped like q, of its dtype and device")
    k_out_args = (None, 0, 0)
    if k_out is not None:
        stride = k_out.stride()
        if k_out.shape != k_shape or k_out.dtype != dtype or k_out.get_device() != at or stride[2] != 1:
            raise ValueError("k_out must be shaped like k, of its dtype and device")
        k_out_args = (k_out.data_ptr(), stride[0], stride[1])
    weight = q_weight if q_weight is not None else k_weight
    weight_dtype = torch.float32 if weight is None else weight.dtype
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype != weight_dtype or w.dtype not in _KV_DTYPES or w.get_device() != at
                              or w.ndim != 1 or w.numel() != d or not w.is_contiguous()):
            raise ValueError("norm weights must be contiguous [head_dim] vectors of one floating-point dtype")
    positions_t = _INDEX.get(positions.dtype)
    if positions_t is None or positions.ndim != 1 or positions.numel() != n or positions.get_device() != at \
            or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int32/int64 [tokens] tensor")
    if rotary_dim is None:
        rotary_dim = d
    table_shape, table_stride = cos_sin_cache.shape, cos_sin_cache.stride()
    table_t = _KV_DTYPES.get(cos_sin_cache.dtype)
    if type(rotary_dim) is not int or not 0 < rotary_dim <= d or rotary_dim % 2 or len(table_shape) != 2 \
            or table_shape[1] != rotary_dim or table_stride[1] != 1 or table_t is None \
            or cos_sin_cache.get_device() != at:
        raise ValueError("the rotation needs a native cos/sin cache matching rotary_dim")
    if k_buffer is None:
        if v_buffer is not None or slot_map is not None:
            raise ValueError("the pool write needs k_buffer, v_buffer and slot_map")
        if k_out is None:
            raise ValueError("k needs k_out, the pool, or both")
        pool = (None, _lib.AKV_I32, None, None, 0, 0, 0, 0, 0)
        v_args = (None, 0, 0)
    else:
        if v_buffer is None or slot_map is None:
            raise ValueError("the pool write needs k_buffer, v_buffer and slot_map")
        v_stride = None if v is None else v.stride()
        if v is None or v.shape != k_shape or v.dtype != dtype or v.get_device() != at or v_stride[2] != 1:
            raise ValueError("v must be shaped like k, of its dtype and device, with unit dim stride")
        pool_shape, kp_stride, vp_stride = k_buffer.shape, k_buffer.stride(), v_buffer.stride()
        if len(pool_shape) != 3 or pool_shape[1] != hk or pool_shape[2] != d or v_buffer.shape != pool_shape \
                or k_buffer.dtype != dtype or v_buffer.dtype != dtype or k_buffer.get_device() != at \
                or v_buffer.get_device() != at or kp_stride[2] != 1 or vp_stride[2] != 1:
            raise ValueError("the pool must be [slots, kv_heads, head_dim] buffers of k's dtype and device")
        slots_t = _INDEX.get(slot_map.dtype)
        if slots_t is None or slot_map.ndim != 1 or slot_map.numel() != n or slot_map.get_device() != at \
                or not slot_map.is_contiguous():
            raise ValueError("slot_map must be a contiguous int32/int64 [tokens] tensor")
        pool = (slot_map.data_ptr(), slots_t, k_buffer.data_ptr(), v_buffer.data_ptr(), pool_shape[0], kp_stride[0],
                kp_stride[1], vp_stride[0], vp_stride[1])
        v_args = (v.data_ptr(), v_stride[0], v_stride[1])
    if at < 0:
        raise ValueError("q must be on a GPU")
    if n == 0:
        return q_out
    device = q.device
    with _on_device(device):
        rc = _lib.calls().akv_qk_norm_rope(
            q.data_ptr(), q_stride[0], q_stride[1], k.data_ptr(), k_stride[0], k_stride[1], *v_args,
            _KV_DTYPES[dtype], n, hq, hk, d, rotary_dim, 1 if is_neox_style else 0,
            None if q_weight is None else q_weight.data_ptr(), None if k_weight is None else k_weight.data_ptr(),
            _KV_DTYPES[weight_dtype], float(eps), positions.data_ptr(), positions_t, cos_sin_cache.data_ptr(), table_t,
            table_stride[0], table_shape[0], q_out.data_ptr(), out_stride[0], out_stride[1], *k_out_args, *pool,
            current_stream_handle(device),
        )
    if rc:
        _lib.check(rc, "akv_qk_norm_rope")
    return q_out
