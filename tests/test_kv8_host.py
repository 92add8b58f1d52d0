"""What the operators of the 8-bit cache refuse, without a GPU: the wrappers'
checks and the C ABI's, none of which reaches a launch."""

import pytest
import torch

from akv_amd import _lib, kv8

BF16, F16, F32, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def _zeros8(*shape, dtype=E4):
    return torch.zeros(shape, dtype=torch.uint8).view(dtype)


def _append(**change):
    a = dict(k=torch.zeros(5, 2, 64, dtype=BF16), v=torch.zeros(5, 2, 64, dtype=BF16), slots=torch.zeros(5, dtype=I64),
             kb=_zeros8(9, 2, 64), vb=_zeros8(9, 2, 64), ks=torch.zeros(9, 2), vs=torch.zeros(9, 2),
             positions=torch.zeros(5, dtype=I64), cos_sin_cache=torch.zeros(8, 64), q=torch.zeros(5, 4, 64, dtype=BF16),
             q_out=torch.zeros(5, 4, 64, dtype=BF16))
    a.update(change)
    args = [a.pop(n) for n in ("k", "v", "slots", "kb", "vb", "ks", "vs")]
    return kv8.append_kv8(*args, **a)


NO_ROPE = dict(positions=None, cos_sin_cache=None, q=None, q_out=None)


@pytest.mark.parametrize("change,message", [
    (dict(k=torch.zeros(5, 2, 64, dtype=torch.float64)), "k and v must be matching"),
    (dict(k=torch.zeros(5, 64, 2, dtype=BF16).transpose(1, 2)), "k and v must be matching"),
    (dict(v=torch.zeros(5, 2, 64, dtype=F16)), "k and v must be matching"),
    (dict(v=torch.zeros(4, 2, 64, dtype=BF16)), "k and v must be matching"),
    (dict(kb=torch.zeros(9, 2, 64, dtype=BF16)), "K/V must be matching float8"),
    (dict(kb=_zeros8(9, 2, 64, dtype=E5)), "K/V must be matching float8"),
    (dict(vb=_zeros8(8, 2, 64)), "K/V must be matching float8"),
    (dict(kb=_zeros8(9, 64, 2).transpose(1, 2), vb=_zeros8(9, 64, 2).transpose(1, 2)), "K/V must be matching float8"),
    (dict(ks=torch.zeros(9, 2, dtype=BF16)), "k_scales / v_scales must be f32"),
    (dict(vs=torch.zeros(8, 2)), "k_scales / v_scales must be f32"),
    (dict(vs=torch.zeros(9, 3)), "k_scales / v_scales must be f32"),
    (dict(scale_block=4, ks=torch.zeros(2, 2)), "k_scales / v_scales must be f32"),
    (dict(scale_block=3), "scale_block must be"),
    (dict(scale_block=0), "scale_block must be"),
    (dict(scale_block=128), "scale_block must be"),
    (dict(scale_block=2.0), "scale_block must be"),
    (dict(), "must be on one GPU"),
])
def test_append_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        _append(**change)


def _attend(**change):
    a = dict(q=torch.zeros(6, 4, 64, dtype=BF16), k=_zeros8(9, 2, 64), v=_zeros8(9, 2, 64), ks=torch.zeros(9, 2),
             vs=torch.zeros(9, 2), qo=torch.zeros(3, dtype=I32), kv=torch.zeros(3, dtype=I32),
             indices=torch.zeros(9, dtype=I32), out=torch.zeros(6, 4, 64, dtype=BF16), scale=1.0, max_len=9, max_new=3)
    a.update(change)
    args = [a.pop(n) for n in ("q", "k", "v", "ks", "vs", "qo", "kv", "indices", "out")]
    return kv8.attention_kv8(*args, **a)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(6, 4, 64)), "q must be bf16 or fp16"),
    (dict(q=torch.zeros(6, 64, 4, dtype=BF16).transpose(1, 2)), "q must be bf16 or fp16"),
    (dict(k=torch.zeros(9, 2, 64, dtype=BF16)), "K/V must be matching float8"),
    (dict(vs=torch.zeros(9, 2, dtype=F16)), "k_scales / v_scales must be f32"),
    (dict(scale_block=6), "scale_block must be"),
    (dict(), "must be on one GPU"),
])
def test_attention_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        _attend(**change)


def _move(**change):
    a = dict(kp=torch.zeros(3, dtype=I64), vp=torch.zeros(3, dtype=I64), ksp=torch.zeros(3, dtype=I64),
             vsp=torch.zeros(3, dtype=I64), k=_zeros8(9, 2, 64), v=_zeros8(9, 2, 64), ks=torch.zeros(9, 2),
             vs=torch.zeros(9, 2), src=torch.zeros(5, dtype=I32), dst=torch.zeros(5, dtype=I32),
             pairs=torch.zeros(5, 2, dtype=I32), table=torch.zeros(8, 64))
    a.update(change)
    args = [a.pop(n) for n in ("kp", "vp", "ksp", "vsp", "k", "v", "ks", "vs", "src", "dst", "pairs", "table")]
    return kv8.reposition_kv8_layers(*args, **a)


@pytest.mark.parametrize("change,message", [
    (dict(v=_zeros8(9, 2, 32)), "K/V must be matching float8"),
    (dict(ks=torch.zeros(9)), "k_scales / v_scales must be f32"),
    (dict(scale_block=-2), "scale_block must be"),
    (dict(), "must be on one GPU"),
])
def test_reposition_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        _move(**change)


def test_workspace_sizes():
    assert kv8.attention_kv8_workspace_bytes(0, 0, 8, 2, 64, 0, 0) >= 0
    # requests of one workgroup need no partial results
    assert kv8.attention_kv8_workspace_bytes(8, 1, 8, 2, 64, 100, 8) == 16
    assert kv8.attention_kv8_workspace_bytes(8, 1, 8, 2, 64, 20000, 8) > 8 * 8 * 66 * 4
    for sizes in ((8, 1, 8, 2, 72, 100, 8), (8, 1, 8, 2, 144, 100, 8), (8, 1, 8, 3, 64, 100, 8), (-1, 1, 8, 2, 64, 9, 8),
                  (8, 1, 8, 2, 64, -1, 8), (8, 1, 8, 2, 64, 9, -1), (8, 1, 8, 0, 64, 9, 8)):
        with pytest.raises(ValueError):
            kv8.attention_kv8_workspace_bytes(*sizes)


_FAKE = 1 << 20  # an aligned address that is never dereferenced


def _call(name, **change):
    """The entry point with plausible arguments by name, some changed."""
    lib = _lib.load()
    pool = dict(k_stride_slot=128, k_stride_head=64, v_stride_slot=128, v_stride_head=64)
    scales = dict(scale_block=1, ks_stride_block=2, ks_stride_head=1, vs_stride_block=2, vs_stride_head=1)
    values = {
        "akv_kv8_append": dict(
            q=_FAKE, q_stride_t=256, q_stride_h=64, k=_FAKE, k_stride_t=128, k_stride_h=64, v=_FAKE, v_stride_t=128,
            v_stride_h=64, dtype=_lib.AKV_BF16, n_tokens=6, q_heads=4, kv_heads=2, head_dim=64, rotary_dim=64,
            is_neox=1, positions=_FAKE, positions_dtype=_lib.AKV_I64, cos_sin=_FAKE, cos_sin_dtype=_lib.AKV_F32,
            rope_stride=64, rope_rows=10, q_out=_FAKE, qo_stride_t=256, qo_stride_h=64, slots=_FAKE,
            slots_dtype=_lib.AKV_I64, k_pool=_FAKE, v_pool=_FAKE, format=_lib.AKV_E4M3, pool_slots=9, **pool,
            k_scales=_FAKE, v_scales=_FAKE, **scales, stream=None),
        "akv_kv8_reposition": dict(
            k_ptrs=_FAKE, v_ptrs=_FAKE, k_scale_ptrs=_FAKE, v_scale_ptrs=_FAKE, n_layers=3, format=_lib.AKV_E5M2,
            n_heads=2, head_dim=64, rotary_dim=64, pool_slots=9, **pool, **scales, src=_FAKE, dst=_FAKE, pairs=_FAKE,
            pair_stride=2, n_tokens=5, cos_sin=_FAKE, cos_sin_dtype=_lib.AKV_F32, rope_stride=64, rope_rows=10,
            is_neox=1, skip_unmapped=0, status=None, stream=None),
        "akv_kv8_attention": dict(
            q=_FAKE, q_stride_t=256, q_stride_h=64, dtype=_lib.AKV_BF16, k_buffer=_FAKE, v_buffer=_FAKE,
            format=_lib.AKV_E4M3, **pool, pool_slots=9, k_scales=_FAKE, v_scales=_FAKE, **scales, n_tokens=6,
            n_requests=2, q_heads=4, kv_heads=2, head_dim=64, qo_indptr=_FAKE, kv_indptr=_FAKE,
            indptr_dtype=_lib.AKV_I32, kv_indices=_FAKE, table_stride=0, table_width=9, page_size=1, tree_mask=None,
            mask_stride=0, mask_words=0, key_starts=None, first_keys=0, sinks=None, scale=1.0, out=_FAKE,
            out_dtype=_lib.AKV_BF16, out_stride_t=256, out_stride_h=64, max_len=9, max_new=3, workspace=_FAKE,
            workspace_bytes=1 << 20, status=None, stream=None),
    }[name]
    assert not set(change) - set(values)
    values.update(change)
    fn = getattr(lib, name)
    assert len(values) == len(fn.argtypes)
    return fn(*values.values())


APPEND, MOVE, READ = "akv_kv8_append", "akv_kv8_reposition", "akv_kv8_attention"


@pytest.mark.parametrize("name,change,message", [
    (APPEND, dict(format=_lib.AKV_BF16), "must be e4m3 or e5m2"),
    (APPEND, dict(kv_heads=0), "0 KV heads"),
    (APPEND, dict(head_dim=72), "head_dim 72"),
    (APPEND, dict(head_dim=144), "head_dim 144"),
    (APPEND, dict(rotary_dim=33), "rotary_dim 33"),
    (APPEND, dict(rotary_dim=66), "rotary_dim 66"),
    (APPEND, dict(scale_block=24), "scale_block 24"),
    (APPEND, dict(scale_block=128), "scale_block 128"),
    (APPEND, dict(pool_slots=-1), "negative size"),
    (APPEND, dict(dtype=9), "dtypes must be"),
    (APPEND, dict(cos_sin_dtype=9), "dtypes must be"),
    (APPEND, dict(slots_dtype=9), "int32 or int64"),
    (APPEND, dict(n_tokens=-1), "invalid size"),
    (APPEND, dict(q_heads=-1), "invalid size"),
    (APPEND, dict(rotary_dim=0), "q without a rotation"),
    (APPEND, dict(n_tokens=1 << 40), "tokens"),
    (APPEND, dict(n_tokens=(1 << 31) - 1), "batch too large"),
    (APPEND, dict(q_out=None), "null device pointer"),
    (APPEND, dict(positions=None), "null device pointer"),
    (APPEND, dict(v=None), "null device pointer"),
    (APPEND, dict(k_pool=None), "null device pointer"),
    (APPEND, dict(v_scales=None), "null device pointer"),
    (MOVE, dict(format=0), "must be e4m3 or e5m2"),
    (MOVE, dict(n_heads=-1), "-1 KV heads"),
    (MOVE, dict(head_dim=8), "head_dim 8"),
    (MOVE, dict(rotary_dim=0), "rotary_dim 0"),
    (MOVE, dict(scale_block=0), "scale_block 0"),
    (MOVE, dict(cos_sin_dtype=5), "cos_sin dtype 5"),
    (MOVE, dict(n_layers=-1), "negative size"),
    (MOVE, dict(pair_stride=-1), "negative size"),
    (MOVE, dict(n_tokens=1 << 31), "tokens"),
    (MOVE, dict(n_tokens=(1 << 31) - 1), "batch too large"),
    (MOVE, dict(v_scale_ptrs=None), "null device pointer"),
    (MOVE, dict(pairs=None), "null device pointer"),
    (READ, dict(n_tokens=-1), "negative size"),
    (READ, dict(first_keys=-1), "negative size"),
    (READ, dict(head_dim=72), "head_dim 72"),
    (READ, dict(head_dim=144), "head_dim 144"),
    (READ, dict(q_heads=5), "5 q heads over 2"),
    (READ, dict(dtype=_lib.AKV_F32), "q must be bf16 or fp16"),
    (READ, dict(format=_lib.AKV_F16), "must be e4m3 or e5m2"),
    (READ, dict(out_dtype=_lib.AKV_F16), "q's type or be f32"),
    (READ, dict(scale_block=48), "scale_block 48"),
    (READ, dict(indptr_dtype=7), "int32 or int64"),
    (READ, dict(page_size=0), "page_size must be positive"),
    (READ, dict(page_size=16), "pages need a block table"),
    (READ, dict(scale=0.0), "scale must be positive"),
    (READ, dict(scale=float("nan")), "scale must be positive"),
    (READ, dict(kv_indices=None), "null device pointer"),
    (READ, dict(k_scales=None), "null device pointer"),
    (READ, dict(q_stride_h=60), "16-byte aligned"),
    (READ, dict(k_stride_head=72), "16-byte aligned"),
    (READ, dict(v_buffer=_FAKE + 8), "16-byte aligned"),
    (READ, dict(workspace_bytes=15), "workspace holds 15 bytes"),
    (READ, dict(max_len=5000), "workspace holds 1048576 bytes"),
    (READ, dict(k_stride_slot=1 << 31), "batch too large"),
    (READ, dict(n_tokens=1 << 40), "batch too large"),
])
def test_entry_points_refuse(name, change, message):
    assert _call(name, **change) == _lib.AKV_EINVAL
    assert message in _lib.last_error()


def test_nothing_to_do_is_no_error():
    assert _call(APPEND, n_tokens=0) == 0
    assert _call(APPEND, pool_slots=0, k_pool=None, v_pool=None, k_scales=None, v_scales=None, q_heads=0) == 0
    assert _call(MOVE, n_tokens=0) == 0
    assert _call(MOVE, n_layers=0) == 0
    assert _call(READ, n_tokens=0) == 0
    assert _call(READ, n_requests=0) == 0


@pytest.mark.parametrize("q_heads,kv_heads,head_dim", [(64, 8, 64), (32, 8, 128), (8, 1, 64), (4, 4, 96)])
def test_a_workspace_serves_every_smaller_batch(q_heads, kv_heads, head_dim):
    def need(requests, tokens, max_len, max_new):
        assert _call(READ, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, n_requests=requests, n_tokens=tokens,
                     max_len=max_len, max_new=max_new, workspace_bytes=0) == _lib.AKV_EINVAL
        words = _lib.last_error().split()
        assert words[-2] == "needs"
        return int(words[-1])

    lens = (1, 256, 257, 512, 513, 1000, 1024, 1025, 2048, 2049, 30000)
    for max_new in (1, 8, 9, 40, 300):
        before = 0
        for max_len in lens:
            sizes = [kv8.attention_kv8_workspace_bytes(r * max_new, r, q_heads, kv_heads, head_dim, max_len, max_new)
                     for r in (1, 2, 15, 16, 17, 127, 128, 129, 600)]
            assert sizes == sorted(sizes) and sizes[0] >= 16 and sizes[0] >= before
            before = sizes[0]
            for requests in (1, 15, 16, 32, 128, 600):
                for tokens in (requests, requests * max_new):
                    for bound in (b for b in lens if b <= max_len):
                        for new in (1, max_new):
                            assert need(requests, tokens, bound, new) <= sizes[-1]
    for max_len in lens:
        sizes = [kv8.attention_kv8_workspace_bytes(4000, 16, q_heads, kv_heads, head_dim, max_len, n)
                 for n in (1, 2, 5, 8, 9, 17, 64, 65, 300)]
        assert sizes == sorted(sizes)
