"""Steps of a paged batch in which requests are idle, bring one token or a piece of a prompt: queries and outputs lie in the
order of the step's tokens.  Plans and attention where they are at their limits."""
import numpy as np
import pytest
import torch

import paged_ref as ref
import turboquant_b200 as tq
from test_gpu_paged import DT, check_attention, filled, gen, table_of

pytestmark = pytest.mark.gpu


def rope_of(dim):
    return tq.QkNormRope((1e4 ** -(torch.arange(0, dim, 2, device="cuda").double() / dim)).float())


def check_rows(out, q, layer, table, kv, cu, scale, before=None):
    """Rows of requests that bring one token are those of the 64-bit form; the others are `before`, or zeros."""
    live = [r for r in range(len(cu) - 1) if cu[r + 1] - cu[r] == 1 and 0 <= cu[r] < q.shape[0]]
    at = torch.tensor([cu[r] for r in live], device="cuda", dtype=torch.long)
    if live:
        check_attention(out[at], q[at], layer, table[live], torch.tensor([kv[r] for r in live], device="cuda"), scale, out.dtype)
    rest = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    rest[at] = False
    assert bool((out[rest] == (0 if before is None else before)).all())


@pytest.mark.parametrize("bits,dtype", [(4, "bf16"), (3, "f16"), (4, "f32")])
def test_documented_sequence_with_idle_requests(bits, dtype):
    """plan, append_rope, decode_tokens: with requests idle, and with pieces of prompts in the same step."""
    g, dt, dim, hq, hkv, page, requests = gen(1), DT[dtype], 128, 8, 2, 16, 6
    cache, rope, att = tq.PagedPqoCache(tq.CacheConfig(bits, dim, hkv, 1), 80, page, requests), rope_of(dim), tq.AttendConfig(dim ** -0.5, hq // hkv)
    lens = [0] * requests
    for new, pad in (([30, 20, 0, 50, 1, 0], 2), ([1, 0, 0, 1, 0, 0], 0), ([1, 0, 0, 1, 0, 0], 4), ([0, 1, 1, 0, 1, 1], 2), ([0, 1, 9, 1, 0, 1], 0),
                     ([0] * 6, 3), ([0, 0, 0, 0, 0, 1], 0), ([1] * 6, 0)):
        rows = sum(new) + pad
        step = cache.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), rows)
        step.check()
        q, k, v = torch.randn((rows, hq + 2 * hkv, dim), generator=g, device="cuda").to(dt).split([hq, hkv, hkv], 1)
        q = cache.append_rope(0, rope, q, k, v, step)
        lens = [s + n for s, n in zip(lens, new)]
        cu = [0] + np.cumsum(new).tolist()
        check_rows(cache.decode_tokens(0, q, step, att).fused, q, cache.layers[0], cache.block_table, lens, cu, dim ** -0.5)
        given = torch.full_like(q, 7)
        assert cache.decode_tokens(0, q, step, att, out=given).fused is given
        check_rows(given, q, cache.layers[0], cache.block_table, lens, cu, dim ** -0.5, before=7)
        if all(n == 1 for n in new):
            assert torch.equal(cache.decode(0, q, step, att).fused, given)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hkv,group", [(8, 4), (1, 12), (2, 8)])
def test_rows_of_long_requests(hkv, group, dtype):
    """Requests that many CTAs share, idle ones between them, over queries that are the outputs too."""
    g, dt, dim, page = gen(2), DT[dtype], 128, 64
    kv, new = [9000, 700, 0, 64, 5000, 1], [1, 0, 0, 1, 1, 3]
    pages = sum(-(-n // page) for n in kv)
    layer, table = filled(pages, hkv, page, dim, 4, g), table_of(kv, page, pages, g)
    cu = [0] + np.cumsum(new).tolist()
    lens, starts = torch.tensor(kv, dtype=torch.int32, device="cuda"), torch.tensor(cu, dtype=torch.int32, device="cuda")
    wide = torch.randn((8, (group + 2) * hkv, dim), generator=g, device="cuda").to(dt)
    q, scratch = wide[:, : group * hkv], layer.attend_scratch(group * hkv)
    out = layer.attend(q, table, lens, dim ** -0.5, scratch=scratch, cu=starts)
    check_rows(out, q, layer, table, kv, cu, dim ** -0.5)
    alone = layer.attend(q[:3].contiguous(), table[[0, 3, 4]].contiguous(), lens[[0, 3, 4]], dim ** -0.5)
    assert torch.equal(out[:3], alone)   # the work is shared out as without the others
    for _ in range(3):
        x = q.clone(memory_format=torch.contiguous_format)
        assert layer.attend(x, table, lens, dim ** -0.5, out=x, scratch=scratch, cu=starts) is x
        assert torch.equal(x[:3], out[:3]) and torch.equal(x[3:], q[3:])
    assert bool((scratch[:16384] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_that_do_not_exist_are_left_out(dtype):
    """First tokens outside the rows, a request without stored tokens, none with a row at all."""
    g, dt, dim, page, hkv, group = gen(3), DT[dtype], 64, 16, 2, 3
    layer, table = filled(40, hkv, page, dim, 4, g), table_of([100, 50, 0, 20], page, 40, g)
    lens = torch.tensor([100, 50, 0, 20], dtype=torch.int32, device="cuda")
    q = torch.randn((3, hkv * group, dim), generator=g, device="cuda").to(dt)
    for cu in ([0, 1, 2, 3, 4], [2, 3, 4, 5, 6], [-1, 0, 1, 2, 3], [0, 0, 0, 0, 0], [-(2 ** 31), 2 ** 31 - 1, 0, 1, 2], [3, 4, 5, 6, 7]):
        out = layer.attend(q, table, lens, 0.1, out=torch.full_like(q, 7), cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
        want = torch.full_like(q, 7)
        for r in range(4):
            if cu[r + 1] - cu[r] == 1 and 0 <= cu[r] < 3:
                want[cu[r]] = 9
                if lens[r] == 0:
                    assert bool((out[cu[r]] == 0).all())
                else:
                    one = torch.tensor([int(lens[r])], dtype=torch.int32, device="cuda")
                    check_attention(out[cu[r]][None], q[cu[r]][None], layer, table[r][None], one, 0.1, dt)
        assert bool((out[want == 7] == 7).all())
    assert layer.attend(q[:0], table, lens, 0.1, cu=torch.zeros(5, dtype=torch.int32, device="cuda")).shape == (0, hkv * group, dim)


def test_captured_steps_with_requests_that_come_and_go():
    """One graph of plan, rows and attention for every batch: each request's own query meets its own pages."""
    g, hq, hkv, dim, page, requests, dt = gen(4), 8, 2, 128, 16, 4, torch.bfloat16
    cache, rope, att = tq.PagedPqoCache(tq.CacheConfig(4, dim, hkv, 1), 60, page, requests), rope_of(dim), tq.AttendConfig(dim ** -0.5, hq // hkv)
    qkv, new = torch.zeros((requests, hq + 2 * hkv, dim), device="cuda", dtype=dt), torch.zeros(requests, dtype=torch.int32, device="cuda")

    def one():
        step = cache.plan(new, requests)
        q, k, v = qkv.split([hq, hkv, hkv], 1)
        turned = cache.append_rope(0, rope, q, k, v, step)
        return step, turned, cache.decode_tokens(0, turned, step, att).fused

    one()   # before the capture; nothing is new
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step, turned, out = one()
    lens = [0] * requests
    for i in range(30):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        some = [int((i + r) % (r + 2) != 0) for r in range(requests)]
        new.copy_(torch.tensor(some, dtype=torch.int32))
        graph.replay()
        lens = [a + b for a, b in zip(lens, some)]
        step.check()
        check_rows(out, turned, cache.layers[0], cache.block_table, lens, [0] + np.cumsum(some).tolist(), dim ** -0.5)


def test_rows_that_do_not_fit_are_refused():
    i32 = dict(dtype=torch.int32, device="cuda")
    g = gen(5)
    layer, table, lens = filled(4, 2, 16, 64, 4, g), torch.zeros((3, 2), **i32), torch.ones(3, **i32)
    q, cu = torch.zeros((5, 4, 64), dtype=torch.bfloat16, device="cuda"), torch.zeros(4, **i32)
    wrong = (tq.DimensionMismatch, TypeError, ValueError, tq.TqbRuntimeError)
    for call in (lambda: layer.attend(q, table, lens, 0.1, cu=cu[:3]), lambda: layer.attend(q, table, lens, 0.1, cu=cu.long()),
                 lambda: layer.attend(q, table, lens, 0.1, cu=cu.cpu()), lambda: layer.attend(q, table, lens[:2], 0.1, cu=cu),
                 lambda: layer.attend(q, table[0], lens, 0.1, cu=cu), lambda: layer.attend(q, table, lens, 0.1),
                 lambda: layer.attend(q, table, lens, 0.1, out=q[:3], cu=cu)):
        with pytest.raises(wrong):
            call()


@pytest.mark.parametrize("count,status", [(3, 0), (4, 1), (2 ** 31 - 1, 1)])
@pytest.mark.parametrize("capacity", [40, 5000])
def test_plan_of_a_count_beyond_its_list(count, status, capacity):
    """A wrong number of free pages: no page is taken from behind the list, and a step that needs none goes on."""
    i32 = dict(dtype=torch.int32, device="cuda")
    seq, table, free = torch.tensor([16, 5], **i32), torch.tensor([[7, -1, -1], [9, -1, -1]], **i32), torch.tensor([0, 1, 2], **i32)
    state = torch.tensor([count, 0, 0, 0], **i32)
    step = tq.paged_plan(seq, torch.tensor([20, 3], **i32), table, free, state, 16, capacity)
    if status:
        assert step.state.tolist() == [count, 0, 1, 0] and table.tolist() == [[7, -1, -1], [9, -1, -1]] and step.kv_lens.tolist() == [16, 5]
        assert step.slots.tolist() == [-1] * capacity and step.cu.tolist() == [0, 0, 0]
    else:
        assert step.state.tolist() == [1, 0, 0, 0] and table.tolist() == [[7, 2, 1], [9, -1, -1]]
    table = torch.tensor([[7, -1, -1], [9, -1, -1]], **i32)
    step = tq.paged_plan(seq, torch.tensor([0, 3], **i32), table, free, state, 16, capacity)
    assert step.state.tolist() == [count, 0, 0, 0] and step.slots[:3].tolist() == [149, 150, 151]


def test_a_step_that_did_not_fit_is_told_after_later_ones():
    """Also where a captured plan is replayed on and on, and where a release in between was refused."""
    cache = tq.PagedPqoCache(tq.CacheConfig(4, 64, 1, 1), 4, 16, 2)
    new = torch.zeros(2, dtype=torch.int32, device="cuda")
    cache.plan(new, 70)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.plan(new, 70)
    for some, status in (([20, 20], 0), ([40, 1], 1), ([1, 0], 0), ([60, 11], 2), ([3, 3], 0)):   # (81 tokens are more than the table's 64)
        new.copy_(torch.tensor(some, dtype=torch.int32))
        graph.replay()
        assert int(cache.state[2]) == status
    assert cache.seq_lens.tolist() == [24, 23]
    with pytest.raises(tq.TqbRuntimeError) as e:
        cache.check()
    assert e.value.status == 2
    cache.check()
    graph.replay()
    cache.check()
    cache.seq_lens[1] = -1
    cache.release(torch.tensor([False, True], device="cuda"))   # refused: the length is negative
    cache.seq_lens[1] = 26
    graph.replay()
    assert int(cache.state[2]) == 0
    with pytest.raises(tq.TqbRuntimeError) as e:
        cache.check()
    assert e.value.status == 2
    cache.seq_lens[1] = -1
    cache.release(torch.tensor([False, True], device="cuda"))
    with pytest.raises(tq.TqbRuntimeError):
        cache.check()
    cache.check()
    with pytest.raises(tq.DimensionMismatch):
        tq.paged_plan(cache.seq_lens, new, cache.block_table, cache.free_pages, cache.state, 16, 4, failed=new)


@pytest.mark.parametrize("dim,group", [(64, 4), (128, 4), (128, 8), (256, 2)])
@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("vscale", [1.0, 1e-4, 1e-6, 3e-7])
def test_values_of_small_scales_keep_their_precision(vscale, bits, dim, group):
    """The error's norm, over that of a head's output.  A weight is rounded to f16 twice, each time by up to 2^-11 of itself:
    2.9e-4 rms and less.  Below 2^-14 a product is off by up to 2^-25 (2^-25 / sqrt(3) rms); the largest weight is held as 2^11 at least, so that
    700 of them make 2^-25 / sqrt(3) * sqrt(700) / (2^11 * 3e-7) = 7.4e-4 of the output at the smallest scale here."""
    g, page, hkv, lens = gen(9), 32, 2, [65, 700]
    layer = filled(30, hkv, page, dim, bits, g, 0.0)
    layer.tensors[3].copy_((layer.tensors[3].view(torch.float16).float() * vscale).half().view(torch.int16))
    table, ln = table_of(lens, page, 30, g), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((2, hkv * group, dim), generator=g, device="cuda").to(torch.bfloat16)
    out = layer.attend(q, table, ln, dim ** -0.5, out=torch.empty((2, hkv * group, dim), device="cuda"))
    want, _, _ = ref.attend(q, layer.tensors, bits, table, ln, dim ** -0.5)
    off = (out.double() - want).norm(dim=-1) / want.norm(dim=-1)
    assert float(off.mean()) <= 2.0 ** -10, float(off.mean())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens,hq,hkv", [(3, 8, 2), (1, 4, 4), (70, 1, 1), (129, 5, 2)])
def test_rows_that_lie_head_after_head(tokens, hq, hkv, dtype):
    """Outputs [heads, tokens, dim], new ones and the inputs themselves; rows that overlap are refused."""
    g, dt, dim = gen(6), DT[dtype], 128
    rope, pos = rope_of(dim), torch.arange(tokens, device="cuda")
    q, k = (torch.randn((h, tokens, dim), generator=g, device="cuda").to(dt).transpose(0, 1) for h in (hq, hkv))
    want = rope(q.contiguous(), k.contiguous(), pos)
    outs = [torch.zeros((h, tokens, dim), device="cuda", dtype=dt).transpose(0, 1) for h in (hq, hkv)]
    got = rope(q, k, pos, q_out=outs[0], k_out=outs[1])
    assert got[0] is outs[0] and torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    rope(q, k, pos, q_out=q, k_out=k)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    flat = torch.zeros(1 << 18, device="cuda", dtype=dt)
    if tokens > 1 and hq > 1:
        for strides in ((dim, dim, 1), (0, dim, 1), (dim, 0, 1), (2 * dim, dim, 1), (dim // 2, tokens * dim, 1)):
            if strides[0] < (hq - 1) * strides[1] + dim and strides[1] < (tokens - 1) * strides[0] + dim or min(strides[:2]) < dim:
                with pytest.raises(ValueError):
                    rope(q, k, pos, q_out=flat.as_strided((tokens, hq, dim), strides))
