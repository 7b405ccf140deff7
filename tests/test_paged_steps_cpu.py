"""Refusals of the paged cache's entry points that are decided on the host, before any launch."""
import ctypes

import pytest
import torch

import turboquant_b200 as tq
from test_paged_cpu import A, layer, rope_params
from turboquant_b200 import paged
from turboquant_b200._lib import TqbPagedAttentionParams, lib


def attention(**kw):
    d = dict(q=A, out=A, block_table=A, kv_lens=A, scratch=A, scratch_bytes=1 << 30, q_row_stride=0, table_stride=4, max_blocks=4,
             num_requests=3, num_q_heads=8, q_dtype=2, out_dtype=2, softmax_scale=0.1)
    return TqbPagedAttentionParams(**{**d, **kw})


@pytest.mark.parametrize("cu,rows,change,status", [(None, 3, {}, 6), (A + 2, 3, {}, 8), (A, -1, {}, 7), (A, 0, {}, 0), (A, 3, dict(num_requests=0), 0),
                                                   (A, 3, dict(num_requests=4097), 12), (A, 3, dict(q=None), 6), (A, 3, dict(num_q_heads=7), 3)])
def test_rows_of_a_step(cu, rows, change, status):
    assert lib.tqb_paged_attention_rows(ctypes.byref(layer()), ctypes.byref(attention(**change)), cu, rows, None) == status


@pytest.mark.parametrize("at,value,status", [(2, -1, 7), (2, 4097, 12), (4, 3, 7), (7, -1, 7), (9, 24, 7), (12, -1, 7), (12, (1 << 30) + 1, 12), (6, None, 6),
                                             (8, None, 6), (10, None, 6), (13, None, 6), (14, None, 6), (15, None, 6)])
def test_plan_of_a_list_of_known_length(at, value, status):
    args = [A, A, 3, A, 4, 4, A, 9, A, 16, A, A, 5, A, A, A, None, None]
    args[at] = value
    assert lib.tqb_paged_plan_bounded(*args) == status


def test_rotations_whose_units_and_stride_pass_31_bits_are_refused():
    """Two units a token: 2,147,476,000 of them, and the grid's stride on top."""
    p = rope_params(num_tokens=1073738000, num_q_heads=1, num_kv_heads=1)
    assert lib.tqb_qk_norm_rope(ctypes.byref(p), None) == 12


@pytest.mark.parametrize("hkv,hq", [(1 << 21, 1 << 21), (2, 1 << 25)])
def test_heads_beyond_the_quotients_of_the_work_line_are_refused(hkv, hq):
    """2^21 KV heads, or as many groups of eight query heads, of one request: few units, but too many heads."""
    few = layer(num_kv_heads=hkv, num_pages=1, page_size=16)
    p = attention(num_q_heads=hq, num_requests=1, max_blocks=1, table_stride=1)
    assert lib.tqb_paged_attention(ctypes.byref(few), ctypes.byref(p), None) == 12


def test_capture_is_asked_of_the_cache_s_own_device(monkeypatch):
    """A cache on another device than the current one: whether its stream is being captured, and which one that is, are asked
    with its device current."""
    now, used = [0], []

    class On:
        def __init__(self, device):
            self.index = torch.device(device).index if not isinstance(device, int) else device

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *a):
            now[0] = self.before

    class Layer:
        def __init__(self, index):
            self.index = index

        def attend_scratch(self, heads):
            return "kept"

        def attend(self, q, table, lens, scale, out=None, scratch=None, cu=None):
            used.append(scratch)
            return q

    monkeypatch.setattr(torch.cuda, "device", On)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == 1)   # device 1 captures, device 0 does not
    monkeypatch.setattr(paged, "_current_device", lambda: now[0])
    monkeypatch.setattr(paged, "_raw_stream", lambda index: 5)
    step = tq.PagedStep(None, None, None, None, None)
    for index, scratch in ((1, None), (0, "kept")):
        cache = object.__new__(tq.PagedPqoCache)
        cache.device, cache.layers, cache.block_table, cache._scratch = torch.device("cuda", index), [Layer(index)], None, {}
        cache.decode(0, torch.zeros(2, 4, 64), step, tq.AttendConfig(0.1))
        assert used.pop() == scratch
