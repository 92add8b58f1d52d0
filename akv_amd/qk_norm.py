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
    fp32, rounded once.  q goes to ``q_out`` (which may be ``q``), k to
    ``k_out`` (which may be ``k``) and, with ``k_buffer`` / ``v_buffer``
    ``[slots, kv_heads, D]``, k and v to rows ``slot_map`` int32 or int64
    ``[N]``, whose valid entries are distinct.  A token whose slot is outside
    the pool (-1: padding) writes no pool row; one whose position is outside
    the table gets NaN in q_out / k_out and no K pool row.  ``v`` is read only
    for the pool and may be None without it.  Head dims up to 512; rows that
    are 16-byte aligned, with D and rotary_dim multiples of 16, take the
    vector kernel.
    """
    device, dtype = q.device, q.dtype
    if dtype not in _KV_DTYPES:
        raise ValueError("q, k and v must be float32, float16 or bfloat16")
    if q.ndim != 3 or k.ndim != 3 or q.stride(2) != 1 or k.stride(2) != 1:
        raise ValueError("q and k must be [tokens, heads, head_dim] with unit dim stride")
    n, hq, d = q.shape
    hk = k.shape[1]
    if k.dtype != dtype or k.device != device or k.shape[0] != n or k.shape[2] != d:
        raise ValueError("q and k must share tokens, head_dim, dtype and device")
    if q_out.shape != q.shape or q_out.dtype != dtype or q_out.device != device or q_out.stride(2) != 1:
        raise ValueError("q_out must be shaped like q, of its dtype and device")
    if k_out is not None and (k_out.shape != k.shape or k_out.dtype != dtype or k_out.device != device
                              or k_out.stride(2) != 1):
        raise ValueError("k_out must be shaped like k, of its dtype and device")
    weight = q_weight if q_weight is not None else k_weight
    for w in (q_weight, k_weight):
        if w is not None and (w.shape != (d,) or w.dtype != weight.dtype or w.dtype not in _KV_DTYPES
                              or w.device != device or not w.is_contiguous()):
            raise ValueError("norm weights must be contiguous [head_dim] vectors of one floating-point dtype")
    if positions.dtype not in _INDEX or positions.shape != (n,) or positions.device != device \
            or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int32/int64 [tokens] tensor")
    rotary_dim = d if rotary_dim is None else rotary_dim
    if type(rotary_dim) is not int or not 0 < rotary_dim <= d or rotary_dim % 2 or cos_sin_cache.ndim != 2 \
            or cos_sin_cache.shape[1] != rotary_dim or cos_sin_cache.stride(1) != 1 \
            or cos_sin_cache.dtype not in _KV_DTYPES or cos_sin_cache.device != device:
        raise ValueError("the rotation needs a native cos/sin cache matching rotary_dim")
    if (k_buffer is None) != (v_buffer is None) or (k_buffer is None) != (slot_map is None):
        raise ValueError("the pool write needs k_buffer, v_buffer and slot_map")
    if k_buffer is None:
        if k_out is None:
            raise ValueError("k needs k_out, the pool, or both")
        pool = (None, _lib.AKV_I32, None, None, 0, 0, 0, 0, 0)
        v_args = (None, 0, 0)
    else:
        if v is None or v.shape != k.shape or v.dtype != dtype or v.device != device or v.stride(2) != 1:
            raise ValueError("v must be shaped like k, of its dtype and device, with unit dim stride")
        for t in (k_buffer, v_buffer):
            if t.ndim != 3 or t.shape[1:] != k.shape[1:] or t.shape[0] != k_buffer.shape[0] or t.dtype != dtype \
                    or t.device != device or t.stride(2) != 1:
                raise ValueError("the pool must be [slots, kv_heads, head_dim] buffers of k's dtype and device")
        if slot_map.dtype not in _INDEX or slot_map.shape != (n,) or slot_map.device != device \
                or not slot_map.is_contiguous():
            raise ValueError("slot_map must be a contiguous int32/int64 [tokens] tensor")
        pool = (slot_map.data_ptr(), _INDEX[slot_map.dtype], k_buffer.data_ptr(), v_buffer.data_ptr(),
                k_buffer.shape[0], k_buffer.stride(0), k_buffer.stride(1), v_buffer.stride(0), v_buffer.stride(1))
        v_args = (v.data_ptr(), v.stride(0), v.stride(1))
    if device.type != "cuda":
        raise ValueError("q must be on a GPU")
    k_out_args = (None, 0, 0) if k_out is None else (k_out.data_ptr(), k_out.stride(0), k_out.stride(1))
    if n == 0:
        return q_out
    lib = _lib.calls()
    with _on_device(device):
        rc = lib.akv_qk_norm_rope(
            q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1), *v_args,
            _KV_DTYPES[dtype], n, hq, hk, d, rotary_dim, 1 if is_neox_style else 0, _lib.ptr(q_weight),
            _lib.ptr(k_weight), _lib.AKV_F32 if weight is None else _KV_DTYPES[weight.dtype], float(eps),
            positions.data_ptr(), _INDEX[positions.dtype], cos_sin_cache.data_ptr(), _KV_DTYPES[cos_sin_cache.dtype],
            cos_sin_cache.stride(0), cos_sin_cache.shape[0], q_out.data_ptr(), q_out.stride(0), q_out.stride(1),
            *k_out_args, *pool, current_stream_handle(device),
        )
    _lib.check(rc, "akv_qk_norm_rope")
    return q_out
