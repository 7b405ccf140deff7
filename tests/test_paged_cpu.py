"""Refusals of the paged-cache entry points: every case is turned away on the host, before any launch."""
import ctypes

import pytest
import torch

import turboquant_b200 as tq
from turboquant_b200._lib import TqbPagedAttentionParams, TqbPagedLayer, TqbRopeParams, lib

A = 1 << 20   # an aligned address that nothing reads


def layer(**kw):
    d = dict(k_indices=A, k_scales=A, v_indices=A, v_scales=A, num_pages=4, num_kv_heads=2, page_size=16, head_dim=128, bits=4, reserved=0)
    return TqbPagedLayer(**{**d, **kw})


def attend(p=None, lay=None):
    d = dict(q=A, out=A, block_table=A, kv_lens=A, scratch=A, scratch_bytes=1 << 30, q_row_stride=0, table_stride=4, max_blocks=4,
             num_requests=3, num_q_heads=8, q_dtype=2, out_dtype=2, softmax_scale=0.1)
    return lib.tqb_paged_attention(ctypes.byref(lay or layer()), ctypes.byref(TqbPagedAttentionParams(**{**d, **(p or {})})), None)


BAD_LAYERS = [(dict(bits=2), 2), (dict(bits=5), 2), (dict(head_dim=100), 1), (dict(head_dim=0), 1), (dict(head_dim=96), 9), (dict(head_dim=512), 9),
              (dict(page_size=8), 7), (dict(page_size=48), 7), (dict(page_size=2048), 7), (dict(num_kv_heads=0), 7), (dict(num_pages=-1), 7),
              (dict(k_indices=None), 6), (dict(v_scales=None), 6), (dict(k_scales=A + 2), 8), (dict(v_indices=A + 8), 8)]


@pytest.mark.parametrize("change,status", BAD_LAYERS)
def test_layers(change, status):
    bad = layer(**change)
    assert attend(lay=bad) == status
    ref = ctypes.byref(bad)
    assert lib.tqb_paged_append(ref, A, 256, 128, A, 256, 128, 2, A, 3, None) == status
    assert lib.tqb_paged_dequantize(ref, A, 3, A, A, 2, None) == status
    assert lib.tqb_paged_append_rope(ref, ctypes.byref(rope_params()), A, 256, 128, A, None) == status


@pytest.mark.parametrize("change,status", [
    (dict(num_requests=-1), 7), (dict(num_requests=0), 0), (dict(num_requests=4097), 12), (dict(num_q_heads=0), 7), (dict(num_q_heads=7), 3),
    (dict(max_blocks=-1), 7), (dict(table_stride=3), 7), (dict(q_dtype=3), 7), (dict(out_dtype=-1), 7), (dict(q_row_stride=-8), 7),
    (dict(q_row_stride=512), 7), (dict(q_row_stride=1028), 8), (dict(q=None), 6), (dict(out=None), 6), (dict(kv_lens=None), 6), (dict(block_table=None), 6),
    (dict(scratch=None), 6), (dict(scratch_bytes=100), 7), (dict(q=A + 2), 8), (dict(out=A + 8), 8), (dict(kv_lens=A + 1), 8)])
def test_attention(change, status):
    assert attend(change) == status


def test_attention_without_arguments():
    assert lib.tqb_paged_attention(None, None, None) == 6
    assert lib.tqb_paged_attention(ctypes.byref(layer()), None, None) == 6
    assert lib.tqb_paged_scratch_bytes(0, 8, 128) == 0 and lib.tqb_paged_scratch_bytes(32, 8, 128) > 8192


def rope_params(**kw):
    d = dict(q=A, q_out=A, k=A, k_out=A, q_token_stride=1024, q_head_stride=128, q_out_token_stride=1024, q_out_head_stride=128, k_token_stride=256,
             k_head_stride=128, k_out_token_stride=256, k_out_head_stride=128, q_weight=None, k_weight=None, positions=A, inv_freq=A, num_tokens=3,
             num_q_heads=8, num_kv_heads=2, head_dim=128, rot_dim=128, dtype=2, flags=0, eps=1e-6)
    return TqbRopeParams(**{**d, **kw})


ROPE = [(dict(dtype=3), 7), (dict(head_dim=100), 1), (dict(head_dim=32), 9), (dict(rot_dim=144), 7), (dict(rot_dim=24), 7), (dict(rot_dim=-16), 7),
        (dict(num_tokens=-1), 7), (dict(num_q_heads=-1), 7), (dict(eps=-1.0), 7), (dict(eps=float("nan")), 7), (dict(flags=8), 7), (dict(positions=None), 6),
        (dict(inv_freq=None), 6), (dict(positions=A + 4, flags=4), 8), (dict(q_out=None), 6), (dict(q=A + 8), 8), (dict(q_head_stride=4), 8),
        (dict(q_token_stride=-1024), 7), (dict(q_weight=A + 2), 8), (dict(k_token_stride=129), 8), (dict(k_weight=A + 4), 8)]


@pytest.mark.parametrize("change,status", ROPE + [(dict(k_out=None), 6), (dict(num_tokens=0), 0)])
def test_norm_rope(change, status):
    assert lib.tqb_qk_norm_rope(ctypes.byref(rope_params(**change)), None) == status


@pytest.mark.parametrize("change,status", ROPE + [(dict(num_kv_heads=3), 3), (dict(head_dim=64, rot_dim=64), 3), (dict(k=None), 6), (dict(num_tokens=0), 0)])
def test_append_rope(change, status):
    assert lib.tqb_paged_append_rope(ctypes.byref(layer()), ctypes.byref(rope_params(**change)), A, 256, 128, A, None) == status


def test_append_and_dequantize():
    ref = ctypes.byref(layer())
    assert lib.tqb_qk_norm_rope(None, None) == 6
    assert lib.tqb_paged_append_rope(ref, None, A, 256, 128, A, None) == 6
    assert lib.tqb_paged_append_rope(ref, ctypes.byref(rope_params()), None, 256, 128, A, None) == 6
    assert lib.tqb_paged_append_rope(ref, ctypes.byref(rope_params()), A, 256, 128, None, None) == 6
    assert lib.tqb_paged_append(ref, A, 256, 128, A, 256, 128, 2, A, 0, None) == 0
    assert lib.tqb_paged_append(ref, A, 256, 128, A, 256, 128, 2, A, -1, None) == 7
    assert lib.tqb_paged_append(ref, A, 256, 128, A, 256, 128, 4, A, 1, None) == 7
    assert lib.tqb_paged_append(ref, None, 256, 128, A, 256, 128, 2, A, 1, None) == 6
    assert lib.tqb_paged_append(ref, A, 256, 128, A, 256, 128, 2, None, 1, None) == 6
    assert lib.tqb_paged_append(ref, A, 256, 128, A, 256, 128, 2, A + 4, 1, None) == 8
    assert lib.tqb_paged_append(ref, A, 257, 128, A, 256, 128, 2, A, 1, None) == 8
    assert lib.tqb_paged_append(ref, A, 256, -128, A, 256, 128, 2, A, 1, None) == 7
    assert lib.tqb_paged_dequantize(ref, A, 0, A, A, 2, None) == 0
    assert lib.tqb_paged_dequantize(ref, A, -1, A, A, 2, None) == 7
    assert lib.tqb_paged_dequantize(ref, A, 1, A, A, 7, None) == 7
    assert lib.tqb_paged_dequantize(ref, A, 1, A, None, 2, None) == 6
    assert lib.tqb_paged_dequantize(ref, A, 1, A, A + 8, 2, None) == 8


@pytest.mark.parametrize("at,value,status", [(2, -1, 7), (2, 4097, 12), (4, 3, 7), (5, -1, 7), (8, 24, 7), (8, 8, 7), (8, 2048, 7), (11, -1, 7), (0, None, 6), (1, None, 6),
                                             (3, None, 6), (6, None, 6), (7, None, 6), (9, None, 6), (10, None, 6), (12, None, 6), (13, None, 6), (14, None, 6)])
def test_plan(at, value, status):
    args = [A, A, 3, A, 4, 4, A, A, 16, A, A, 5, A, A, A, None]
    args[at] = value
    assert lib.tqb_paged_plan(*args) == status


@pytest.mark.parametrize("at,value,status", [(2, -1, 7), (2, 5000, 12), (4, 3, 7), (7, -1, 7), (9, 17, 7), (0, None, 6), (1, None, 6), (3, None, 6), (6, None, 6), (8, None, 6)])
def test_release(at, value, status):
    args = [A, A, 3, A, 4, 4, A, 9, A, 16, None]
    args[at] = value
    assert lib.tqb_paged_release(*args) == status


def test_tensors_of_the_host_are_refused():
    i, s = torch.zeros((2, 1, 16, 64), dtype=torch.uint8), torch.zeros((2, 1, 16, 4), dtype=torch.int16)
    with pytest.raises(ValueError):
        tq.PagedLayer(i, s, i, s, 4)
    with pytest.raises(ValueError):
        tq.QkNormRope(torch.ones(64))
    z = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError):
        tq.paged_plan(z, z, torch.zeros((4, 2), dtype=torch.int32), z, z, 16, 4)
    with pytest.raises(ValueError):
        tq.paged_release(torch.zeros(4, dtype=torch.uint8), z, torch.zeros((4, 2), dtype=torch.int32), z, z, 16)


def test_caches_of_other_formats_are_refused():
    for kw in (dict(norm_mode=tq.QuantNormMode.L2Norm), dict(outlier_blocks=0), dict(outlier_blocks=2)):
        with pytest.raises(tq.TqbRuntimeError):
            tq.PagedPqoCache(tq.CacheConfig(4, 128, 8, 1, **kw), 4)
    with pytest.raises(tq.DimensionMismatch):
        tq.PagedPqoCache(tq.CacheConfig(4, 128, 8, 1, batch=2), 4)


MANY = (1 << 30) + 1


def test_counts_beyond_32_bits_are_refused():
    ref = ctypes.byref(layer())
    args = [A, A, 3, A, 4, 4, A, A, 16, A, A, MANY, A, A, A, None]
    assert lib.tqb_paged_plan(*args) == 12
    for change in (dict(), dict(rot_dim=64), dict(q=None)):
        assert lib.tqb_qk_norm_rope(ctypes.byref(rope_params(num_tokens=MANY, **change)), None) == 12
        assert lib.tqb_paged_append_rope(ref, ctypes.byref(rope_params(num_tokens=MANY, **change)), A, 256, 128, A, None) == 12
    big = layer(num_pages=1 << 20, num_kv_heads=256)   # 2^32 rows
    assert attend(lay=big) == 12
    assert lib.tqb_paged_append(ctypes.byref(big), A, 1 << 15, 128, A, 1 << 15, 128, 2, A, 3, None) == 12
    assert lib.tqb_paged_dequantize(ctypes.byref(big), A, 3, A, A, 2, None) == 12
    assert attend(dict(num_q_heads=1 << 30)) == 12


def test_append_rope_of_keys_beyond_shared_memory_is_refused():
    wide = layer(num_kv_heads=410)   # 410 * 4 blocks of 80 bytes
    p = rope_params(num_kv_heads=410, k_token_stride=410 * 128)
    assert lib.tqb_paged_append_rope(ctypes.byref(wide), ctypes.byref(p), A, 410 * 128, 128, A, None) == 9


def test_packed_arguments_are_the_c_structures():
    from turboquant_b200 import paged
    for packed, c in ((paged._LAYER, TqbPagedLayer), (paged._ROPE, TqbRopeParams), (paged._ATTEND, TqbPagedAttentionParams)):
        assert packed.size == ctypes.sizeof(c)
        names = [n for n, _ in c._fields_]
        values = [0.25 * (i + 1) if t is ctypes.c_float else i + 1 for i, (_, t) in enumerate(c._fields_)]
        made = c.from_buffer_copy(packed.pack(*values))
        assert [getattr(made, n) for n in names] == values
