"""What the drafted-token operators refuse, without a GPU: the wrappers'
checks and the C ABI's, none of which reaches a launch."""

import re
from pathlib import Path

import pytest
import torch

from akv_amd import _lib, attention, page_table, qk_norm

BF16, F16, F32, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.int32, torch.int64


def _tree(**change):
    a = dict(q=torch.zeros(6, 4, 64, dtype=BF16), k=torch.zeros(9, 2, 64, dtype=BF16),
             v=torch.zeros(9, 2, 64, dtype=BF16), qo=torch.zeros(3, dtype=I32), kv=torch.zeros(3, dtype=I32),
             indices=torch.zeros(9, dtype=I32), out=torch.zeros(6, 4, 64, dtype=BF16), scale=1.0, max_len=9, max_new=3)
    a.update(change)
    args = [a.pop(n) for n in ("q", "k", "v", "qo", "kv", "indices", "out")]
    return attention.tree_attention(*args, **a)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(6, 4, 64)), "q must be bf16 or fp16"),
    (dict(q=torch.zeros(6, 64, 4, dtype=BF16).transpose(1, 2)), "q must be bf16 or fp16"),
    (dict(k=torch.zeros(9, 2, 64, dtype=F16)), "K/V must be matching"),
    (dict(v=torch.zeros(8, 2, 64, dtype=BF16)), "K/V must be matching"),
    (dict(k=torch.zeros(9, 2, 32, dtype=BF16), v=torch.zeros(9, 2, 32, dtype=BF16)), "K/V must be matching"),
    (dict(out=torch.zeros(6, 4, 64, dtype=F16)), "out must be shaped like q"),
    (dict(out=torch.zeros(5, 4, 64, dtype=BF16)), "out must be shaped like q"),
    (dict(qo=torch.zeros(3, dtype=I64)), "of one int32/int64 dtype"),
    (dict(kv=torch.zeros(4, dtype=I32)), "of one int32/int64 dtype"),
    (dict(qo=torch.zeros(6, dtype=I32)[::2]), "of one int32/int64 dtype"),
    (dict(indices=torch.zeros(9, dtype=I64)), "kv_indices must be int32"),
    (dict(indices=torch.zeros(18, dtype=I32)[::2]), "kv_indices must be int32"),
    (dict(indices=torch.zeros(3, 4, dtype=I32)), "a row per request"),
    (dict(indices=torch.zeros(1, 4, dtype=I32).expand(2, 4)), "without overlap"),
    (dict(page_size=16), "pages need a block table"),
    (dict(tree_mask=torch.zeros(6, dtype=I64)), "tree_mask must be"),
    (dict(tree_mask=torch.zeros(6, 1, dtype=I32)), "tree_mask must be"),
    (dict(tree_mask=torch.zeros(5, 1, dtype=I64)), "tree_mask must be"),
    (dict(key_starts=torch.zeros(6, dtype=I64)), "key_starts must be"),
    (dict(key_starts=torch.zeros(5, dtype=I32)), "key_starts must be"),
    (dict(sinks=torch.zeros(4, dtype=BF16)), "sinks must be"),
    (dict(sinks=torch.zeros(8)[::2]), "sinks must be"),
    (dict(status=torch.zeros(1)), "status must be"),
    (dict(), "must be on one GPU"),
])
def test_tree_attention_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        _tree(**change)


def test_tree_attention_refuses_its_own_input_as_output():
    q = torch.zeros(6, 4, 64, dtype=BF16)
    with pytest.raises(ValueError, match="out must not be q"):
        _tree(q=q, out=q)


def test_tree_workspace_sizes():
    assert attention.tree_workspace_bytes(0, 0, 8, 2, 64, 0, 0) >= 0
    # requests of one workgroup need no partial results
    assert attention.tree_workspace_bytes(8, 1, 8, 2, 64, 100, 8) == 16
    assert attention.tree_workspace_bytes(8, 1, 8, 2, 64, 20000, 8) > 8 * 8 * 66 * 4
    for sizes in ((8, 1, 8, 2, 60, 100, 8), (8, 1, 8, 2, 136, 100, 8), (8, 1, 8, 3, 64, 100, 8), (-1, 1, 8, 2, 64, 9, 8),
                  (8, 1, 8, 2, 64, -1, 8), (8, 1, 8, 2, 64, 9, -1), (8, 1, 8, 0, 64, 9, 8)):
        with pytest.raises(ValueError):
            attention.tree_workspace_bytes(*sizes)


_FAKE = 1 << 20  # an aligned address that is never dereferenced


def _call(name, **change):
    """The entry point with plausible arguments by name, some changed."""
    lib = _lib.load()
    values = {
        "akv_tree_attention": dict(
            q=_FAKE, q_stride_t=256, q_stride_h=64, k_buffer=_FAKE, v_buffer=_FAKE, k_stride_slot=128,
            k_stride_head=64, v_stride_slot=128, v_stride_head=64, pool_slots=9, dtype=_lib.AKV_BF16, n_tokens=6,
            n_requests=2, q_heads=4, kv_heads=2, head_dim=64, qo_indptr=_FAKE, kv_indptr=_FAKE,
            indptr_dtype=_lib.AKV_I32, kv_indices=_FAKE, table_stride=0, table_width=9, page_size=1, tree_mask=None,
            mask_stride=0, mask_words=0, key_starts=None, sinks=None, scale=1.0, out=_FAKE, out_dtype=_lib.AKV_BF16,
            out_stride_t=256, out_stride_h=64, max_len=9, max_new=3, workspace=_FAKE, workspace_bytes=1 << 20,
            status=None, stream=None),
        "akv_qk_norm_rope": dict(
            q=_FAKE, q_stride_t=256, q_stride_h=64, k=_FAKE, k_stride_t=128, k_stride_h=64, v=_FAKE, v_stride_t=128,
            v_stride_h=64, dtype=_lib.AKV_BF16, n_tokens=6, q_heads=4, kv_heads=2, head_dim=64, rotary_dim=64,
            is_neox=1, q_weight=None, k_weight=None, weight_dtype=_lib.AKV_F32, eps=1e-6, positions=_FAKE,
            positions_dtype=_lib.AKV_I64, cos_sin=_FAKE, cos_sin_dtype=_lib.AKV_F32, rope_stride=64, rope_rows=10,
            q_out=_FAKE, qo_stride_t=256, qo_stride_h=64, k_out=None, ko_stride_t=0, ko_stride_h=0, slots=_FAKE,
            slots_dtype=_lib.AKV_I64, k_pool=_FAKE, v_pool=_FAKE, pool_slots=9, kp_stride_slot=128,
            kp_stride_head=64, vp_stride_slot=128, vp_stride_head=64, stream=None),
        "akv_step_maps": dict(
            registry=_FAKE, table=_FAKE, row_stride=8, table_width=8, rows=_FAKE, rows_dtype=_lib.AKV_I64,
            seq_lens=_FAKE, new_lens=_FAKE, lens_dtype=_lib.AKV_I64, n_requests=2, qo_indptr=_FAKE, kv_indptr=_FAKE,
            indptr_dtype=_lib.AKV_I32, n_tokens=3, slot_map=_FAKE, slots_dtype=_lib.AKV_I64, positions=_FAKE,
            positions_dtype=_lib.AKV_I64, block_tables=None, block_stride=0, block_width=0, page_size=1, parents=None,
            tree_mask=None, tree_stride=0, tree_words=0, window=0, window_mask=None, window_stride=0, window_words=0,
            window_starts=None, status=None, stream=None),
    }[name]
    assert not set(change) - set(values)
    values.update(change)
    fn = getattr(lib, name)
    assert len(values) == len(fn.argtypes)
    return fn(*values.values())


@pytest.mark.parametrize("name,change,message", [
    ("akv_tree_attention", dict(n_tokens=-1), "negative size"),
    ("akv_tree_attention", dict(table_stride=-4), "negative size"),
    ("akv_tree_attention", dict(head_dim=60), "head_dim 60"),
    ("akv_tree_attention", dict(head_dim=136), "head_dim 136"),
    ("akv_tree_attention", dict(q_heads=5), "5 q heads over 2"),
    ("akv_tree_attention", dict(kv_heads=0), "over 0 KV heads"),
    ("akv_tree_attention", dict(dtype=_lib.AKV_F32), "must be bf16 or fp16"),
    ("akv_tree_attention", dict(out_dtype=_lib.AKV_F16), "q's type or be f32"),
    ("akv_tree_attention", dict(indptr_dtype=7), "int32 or int64"),
    ("akv_tree_attention", dict(page_size=0), "page_size must be positive"),
    ("akv_tree_attention", dict(page_size=16), "pages need a block table"),
    ("akv_tree_attention", dict(scale=0.0), "scale must be positive"),
    ("akv_tree_attention", dict(scale=float("nan")), "scale must be positive"),
    ("akv_tree_attention", dict(scale=float("inf")), "scale must be positive"),
    ("akv_tree_attention", dict(kv_indices=None), "null device pointer"),
    ("akv_tree_attention", dict(workspace=None), "null device pointer"),
    ("akv_tree_attention", dict(q_stride_h=60), "16-byte aligned"),
    ("akv_tree_attention", dict(v_buffer=_FAKE + 8), "16-byte aligned"),
    ("akv_tree_attention", dict(workspace=_FAKE + 4), "16-byte aligned"),
    ("akv_tree_attention", dict(workspace_bytes=15), "workspace holds 15 bytes"),
    ("akv_tree_attention", dict(workspace_bytes=1 << 20, max_len=5000), "workspace holds 1048576 bytes"),
    ("akv_tree_attention", dict(k_stride_slot=1 << 31), "batch too large"),
    ("akv_tree_attention", dict(n_tokens=1 << 40), "batch too large"),
    ("akv_qk_norm_rope", dict(dtype=9), "dtypes must be"),
    ("akv_qk_norm_rope", dict(weight_dtype=9), "dtypes must be"),
    ("akv_qk_norm_rope", dict(slots_dtype=9), "int32 or int64"),
    ("akv_qk_norm_rope", dict(n_tokens=-1), "negative size"),
    ("akv_qk_norm_rope", dict(head_dim=513, rotary_dim=64), "head_dim 513"),
    ("akv_qk_norm_rope", dict(rotary_dim=0), "rotary_dim 0"),
    ("akv_qk_norm_rope", dict(rotary_dim=33), "rotary_dim 33"),
    ("akv_qk_norm_rope", dict(rotary_dim=66), "rotary_dim 66"),
    ("akv_qk_norm_rope", dict(eps=-1.0), "eps must be"),
    ("akv_qk_norm_rope", dict(eps=float("nan")), "eps must be"),
    ("akv_qk_norm_rope", dict(q_heads=1 << 20), "q and 2 KV heads"),
    ("akv_qk_norm_rope", dict(q_out=None), "null device pointer"),
    ("akv_qk_norm_rope", dict(positions=None), "null device pointer"),
    ("akv_qk_norm_rope", dict(v=None), "the pool needs"),
    ("akv_qk_norm_rope", dict(slots=None), "the pool needs"),
    ("akv_qk_norm_rope", dict(k_pool=None, v_pool=None), "nowhere to go"),
    ("akv_step_maps", dict(n_requests=-1), "negative size"),
    ("akv_step_maps", dict(n_tokens=-1), "negative size"),
    ("akv_step_maps", dict(n_requests=70000), "exceeds one launch"),
    ("akv_step_maps", dict(page_size=0), "page_size must be positive"),
    ("akv_step_maps", dict(lens_dtype=5), "int32 or int64"),
    ("akv_step_maps", dict(window_starts=_FAKE, window=-1), "need a window"),
    ("akv_step_maps", dict(window_mask=_FAKE, window_words=1, window=1 << 31), "need a window"),
    ("akv_step_maps", dict(registry=None), "null device pointer"),
    ("akv_step_maps", dict(slot_map=None), "null device pointer"),
])
def test_entry_points_refuse(name, change, message):
    assert _call(name, **change) == _lib.AKV_EINVAL
    assert message in _lib.last_error()


def test_nothing_to_do_is_no_error():
    assert _call("akv_tree_attention", n_tokens=0) == 0
    assert _call("akv_tree_attention", n_requests=0) == 0
    assert _call("akv_qk_norm_rope", n_tokens=0) == 0
    assert _call("akv_qk_norm_rope", q_heads=0, kv_heads=0) == 0


def _norm(**change):
    a = dict(q=torch.zeros(5, 4, 64, dtype=BF16), k=torch.zeros(5, 2, 64, dtype=BF16),
             v=torch.zeros(5, 2, 64, dtype=BF16), wq=torch.ones(64, dtype=BF16), wk=torch.ones(64, dtype=BF16),
             positions=torch.zeros(5, dtype=I64), table=torch.zeros(8, 64), out=torch.zeros(5, 4, 64, dtype=BF16),
             slot_map=torch.zeros(5, dtype=I64), k_buffer=torch.zeros(9, 2, 64, dtype=BF16),
             v_buffer=torch.zeros(9, 2, 64, dtype=BF16))
    a.update(change)
    args = [a.pop(n) for n in ("q", "k", "v", "wq", "wk", "positions", "table", "out")]
    return qk_norm.qk_norm_rope(*args, **a)


@pytest.mark.parametrize("change,message", [
    (dict(q=torch.zeros(5, 4, 64, dtype=torch.float64)), "q, k and v must be float32"),
    (dict(q=torch.zeros(5, 64, 4, dtype=BF16).transpose(1, 2)), "unit dim stride"),
    (dict(k=torch.zeros(4, 2, 64, dtype=BF16)), "q and k must share"),
    (dict(k=torch.zeros(5, 2, 64, dtype=F16)), "q and k must share"),
    (dict(out=torch.zeros(5, 4, 64, dtype=F32)), "q_out must be"),
    (dict(k_out=torch.zeros(5, 4, 64, dtype=BF16)), "k_out must be"),
    (dict(wq=torch.ones(32, dtype=BF16)), "norm weights must be"),
    (dict(wq=torch.ones(64)), "norm weights must be"),
    (dict(wk=torch.ones(128, dtype=BF16)[::2]), "norm weights must be"),
    (dict(positions=torch.zeros(5)), "positions must be"),
    (dict(positions=torch.zeros(6, dtype=I64)), "positions must be"),
    (dict(rotary_dim=32), "cos/sin cache"),
    (dict(rotary_dim=63), "cos/sin cache"),
    (dict(table=torch.zeros(64, 8).T), "cos/sin cache"),
    (dict(slot_map=None), "the pool write needs"),
    (dict(v_buffer=None), "the pool write needs"),
    (dict(slot_map=None, k_buffer=None, v_buffer=None), "k needs k_out"),
    (dict(v=None), "v must be shaped like k"),
    (dict(k_buffer=torch.zeros(9, 3, 64, dtype=BF16)), "the pool must be"),
    (dict(v_buffer=torch.zeros(8, 2, 64, dtype=BF16)), "the pool must be"),
    (dict(slot_map=torch.zeros(5)), "slot_map must be"),
    (dict(), "q must be on a GPU"),
])
def test_qk_norm_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        _norm(**change)


def _maps(**change):
    a = dict(registry=torch.zeros(3, 6, dtype=I64), table=torch.zeros(3, 8, dtype=I32), rows=torch.zeros(2, dtype=I64),
             seq=torch.zeros(2, dtype=I64), new=torch.zeros(2, dtype=I64), qo=torch.zeros(3, dtype=I32),
             kv=torch.zeros(3, dtype=I32), slots=torch.zeros(4, dtype=I64), positions=torch.zeros(4, dtype=I64))
    a.update(change)
    args = [a.pop(n) for n in ("registry", "table", "rows", "seq", "new", "qo", "kv", "slots", "positions")]
    return page_table.context_step_maps(*args, **a)


@pytest.mark.parametrize("change,message", [
    (dict(registry=torch.zeros(3, 5, dtype=I64)), "registry must be"),
    (dict(table=torch.zeros(8, 3, dtype=I32).T), "the request table must be"),
    (dict(new=torch.zeros(2, dtype=I32)), "one entry per request"),
    (dict(rows=torch.zeros(3, dtype=I64)), "one entry per request"),
    (dict(kv=torch.zeros(2, dtype=I32)), r"\[requests \+ 1\]"),
    (dict(kv=torch.zeros(3, dtype=I64)), r"\[requests \+ 1\]"),
    (dict(slots=torch.zeros(4)), "slot_map must be"),
    (dict(positions=torch.zeros(5, dtype=I64)), "one entry per token"),
    (dict(block_tables=torch.zeros(3, 4, dtype=I32)), "block_tables must be"),
    (dict(block_tables=torch.zeros(1, 4, dtype=I32).expand(2, 4)), "block_tables must be"),
    (dict(parents=torch.zeros(4, dtype=I64)), "parents must be"),
    (dict(parents=torch.zeros(3, dtype=I32)), "parents must be"),
    (dict(window_starts=torch.zeros(4, dtype=I32)), "need a window"),
    (dict(tree_mask=torch.zeros(4, dtype=I64)), "masks must be"),
    (dict(tree_mask=torch.zeros(3, 1, dtype=I64)), "masks must be"),
    (dict(window=4, window_mask=torch.zeros(1, 2, dtype=I64).expand(4, 2)), "masks must be"),
    (dict(window=4, window_starts=torch.zeros(4, dtype=I64)), "window_starts must be"),
    (dict(), "must be on one GPU"),
])
def test_step_maps_refuse(change, message):
    with pytest.raises(ValueError, match=message):
        _maps(**change)


def _need(q_heads, kv_heads, head_dim, requests, tokens, max_len, max_new):
    """What the call itself asks for: it is refused without."""
    assert _call("akv_tree_attention", q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim, n_requests=requests,
                 n_tokens=tokens, max_len=max_len, max_new=max_new, workspace_bytes=0) == _lib.AKV_EINVAL
    words = _lib.last_error().split()
    assert words[-2] == "needs"
    return int(words[-1])


@pytest.mark.parametrize("q_heads,kv_heads,head_dim", [(64, 8, 64), (32, 8, 128), (8, 1, 64), (4, 4, 96)])
def test_a_workspace_serves_every_smaller_batch(q_heads, kv_heads, head_dim):
    """On both sides of the launch rules: 128 workgroups, 4 tiles, 1024 keys,
    rows of one to four subtiles."""
    lens = (1, 256, 257, 512, 513, 1000, 1024, 1025, 30000)
    for max_new in (1, 8, 9, 40, 300):
        before = 0
        for max_len in lens:
            sizes = [attention.tree_workspace_bytes(r * t, r, q_heads, kv_heads, head_dim, max_len, max_new)
                     for r in (1, 2, 15, 16, 17, 127, 128, 129, 600) for t in (max_new,)]
            assert sizes == sorted(sizes) and sizes[0] >= 16
            assert sizes[0] >= before
            before = sizes[0]
            whole = sizes[-1]
            for requests in (1, 15, 16, 32, 128, 600):
                for tokens in (requests, requests * max_new):
                    for bound in (b for b in lens if b <= max_len):
                        for new in (1, max_new):
                            assert _need(q_heads, kv_heads, head_dim, requests, tokens, bound, new) <= whole
    for max_len in lens:
        sizes = [attention.tree_workspace_bytes(4000, 16, q_heads, kv_heads, head_dim, max_len, n)
                 for n in (1, 2, 5, 8, 9, 17, 64, 65, 300)]
        assert sizes == sorted(sizes)


@pytest.mark.parametrize("name,change,message", [
    ("akv_tree_attention", dict(k_buffer=None), "null device pointer"),
    ("akv_tree_attention", dict(kv_indices=None, table_width=1), "null device pointer"),
    ("akv_qk_norm_rope", dict(v_pool=None), "the pool needs"),
    ("akv_qk_norm_rope", dict(k_pool=None, v_pool=None, pool_slots=1), "nowhere to go"),
    ("akv_qk_norm_rope", dict(k_pool=None, v_pool=None, pool_slots=0, slots=None), "nowhere to go"),
    ("akv_step_maps", dict(table=None), "null device pointer"),
])
def test_no_address_is_for_nothing_alone(name, change, message):
    assert _call(name, **change) == _lib.AKV_EINVAL
    assert message in _lib.last_error()


def test_asm_names_the_registers_it_writes():
    """Scalar registers that an asm statement writes by name are among its
    clobbers, so that the compiler keeps nothing in them across it."""
    found = 0
    for path in (Path(_lib.__file__).parent / "csrc").iterdir():
        text = path.read_text() if path.suffix in (".hip", ".h") else ""
        for asm in re.findall(r"\basm(?:\s+volatile)?\s*\((.*?)\);", text, re.S):
            for register in re.findall(r"\bs_mov_b(?:32|64)\s+(m0|vcc|exec|s\d+)\b", asm):
                found += 1
                assert f'"{register}"' in asm, (path.name, asm)
    assert found >= 2
