"""Paged cache on the GPU, where single sizes do not lead: prompts of thousands of tokens, tables wider than 32-bit counts of
their groups, keys that fill a CTA's shared memory, outputs over their inputs, and work areas that streams and graphs share."""
import pytest
import torch

import paged_ref as ref
import turboquant_b200 as tq
from test_gpu_paged import DT, check_attention, close, filled, gen, layer_of, stored, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,hq,hkv,rot,norm,interleaved", [(64, 6, 2, 64, True, False), (128, 8, 3, 128, True, True), (128, 4, 4, 64, True, False),
                                                             (128, 5, 1, 32, False, True), (256, 3, 1, 256, True, False), (64, 3, 3, 0, True, False)])
def test_norm_rope_of_many_tokens(dim, hq, hkv, rot, norm, interleaved, dtype):
    g, dt = gen(dim + hq), DT[dtype]
    inv = (1e4 ** -(torch.arange(0, rot, 2, device="cuda").double() / max(rot, 1))).float()
    wq, wk = (torch.randn(dim, generator=g, device="cuda").to(dt) for _ in range(2))
    rope = tq.QkNormRope(inv, wq, wk, eps=1e-6, norm=norm, interleaved=interleaved)
    for tokens in (1183, 1184, 5003):   # on both sides of a CTA a token, and several rounds of the grid
        qkv = torch.randn((tokens, hq + 2 * hkv, dim), generator=g, device="cuda").to(dt)
        q, k = qkv[:, :hq], qkv[:, hq:hq + hkv]
        pos = torch.arange(tokens, device="cuda", dtype=torch.int32).flip(0)
        qo, ko = rope(q, k, pos)
        for got, x, w in ((qo, q, wq), (ko, k, wk)):
            want = ref.norm_rope(x, w, pos, inv, 1e-6, norm, interleaved)
            close(got, want, dt, want.abs().amax(-1, keepdim=True))
        q2, k2 = q.clone(), k.clone()
        rope(q2, k2, pos, q_out=q2, k_out=k2)
        assert torch.equal(q2, qo) and torch.equal(k2, ko)


@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,hq,hkv,rot,norm", [(128, 8, 3, 128, True), (64, 4, 1, 64, False), (128, 2, 2, 64, True), (256, 2, 1, 256, True), (64, 2, 4, 0, True)])
def test_append_rope_of_many_tokens(dim, hq, hkv, rot, norm, dtype, bits):
    g, dt, page, tokens = gen(dim), DT[dtype], 64, 2501
    a, b = (layer_of(45, hkv, page, dim, bits) for _ in range(2))
    q, k, v = (torch.randn((tokens, h, dim), generator=g, device="cuda").to(dt) for h in (hq, hkv, hkv))
    inv = (1e4 ** -(torch.arange(0, rot, 2, device="cuda").double() / max(rot, 1))).float()
    rope = tq.QkNormRope(inv, None, torch.randn(dim, generator=g, device="cuda").to(dt), norm=norm)
    pos = torch.randint(0, 1 << 17, (tokens,), generator=g, device="cuda")
    slots = torch.randperm(45 * page, generator=g, device="cuda")[:tokens]
    slots[::7] = -1
    qo, ko = rope(q, k, pos)
    a.append(ko, v, slots)
    assert torch.equal(b.append_rope(rope, q, k, v, pos, slots), qo)
    for x, y in zip(a.tensors, b.tensors):
        assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_of_many_tokens_in_and_out(dtype, bits):
    """More 32-blocks than a round of the grids takes."""
    g, dt, dim, heads, page, tokens = gen(1), DT[dtype], 128, 8, 128, 3001
    layer = layer_of(24, heads, page, dim, bits)
    kv = torch.randn((2, tokens, heads, dim), generator=g, device="cuda").to(dt)
    slots = torch.randperm(24 * page, generator=g, device="cuda")[:tokens]
    slots[5::11] = -1
    layer.append(kv[0], kv[1], slots)
    ok = slots >= 0
    got, back = stored(layer, slots[ok]), layer.dequantize(slots, dt)
    for i in range(2):
        wi, ws = tq.block_quantize(kv[i][ok].reshape(-1, dim).contiguous(), bits)
        assert torch.equal(got[2 * i].reshape(wi.shape), wi) and torch.equal(got[2 * i + 1].reshape(ws.shape), ws)
        assert torch.equal(back[i][ok].reshape(-1, dim), tq.block_dequantize(wi, ws, bits, dim, dtype=dt))
        assert bool((back[i][~ok] == 0).all())


def test_append_rope_of_more_heads_than_eight_tokens_have_room_for():
    g, dim, hkv, page, tokens = gen(2), 256, 64, 16, 1300   # keys of a token: 64 * 8 * 144 bytes
    a, b = (layer_of(82, hkv, page, dim, 4) for _ in range(2))
    k, v = (torch.randn((tokens, hkv, dim), generator=g, device="cuda") for _ in range(2))
    q = torch.randn((tokens, 1, dim), generator=g, device="cuda")
    rope = tq.QkNormRope(1.0 / torch.arange(1, 129, device="cuda"))
    pos, slots = torch.arange(tokens, device="cuda"), torch.randperm(82 * page, generator=g, device="cuda")[:tokens]
    qo, ko = rope(q, k, pos)
    a.append(ko, v, slots)
    assert torch.equal(b.append_rope(rope, q, k, v, pos, slots), qo)
    for x, y in zip(a.tensors, b.tensors):
        assert torch.equal(x, y)


def test_rows_broadcast_over_heads():
    """A head stride of zero: every head reads the same row."""
    g, dim, page = gen(3), 128, 16
    layer = layer_of(4, 4, page, dim, 4)
    k = torch.randn((20, 1, dim), generator=g, device="cuda").to(torch.bfloat16)
    slots = torch.arange(20, device="cuda")
    layer.append(k.expand(20, 4, dim), k.expand(20, 4, dim), slots)
    got = stored(layer, slots)
    wi, ws = tq.block_quantize(k.reshape(-1, dim).contiguous(), 4)
    for h in range(4):
        assert torch.equal(got[0][:, h], wi) and torch.equal(got[3][:, h], ws)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens", [[5000, 33], [1, 20011]])
def test_attention_of_a_table_wider_than_its_groups_can_be_counted(lens, dtype):
    g, dt, page, dim, hkv, group = gen(4), DT[dtype], 1024, 64, 8, 2
    pages = sum(-(-n // page) for n in lens) + 1
    layer = filled(pages, hkv, page, dim, 4, g)
    table = table_of(lens, page, pages, g, blocks=1 << 21)   # 2^31 tokens a request
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((2, hkv * group, dim), generator=g, device="cuda").to(dt)
    out = layer.attend(q, table, ln, dim ** -0.5)
    check_attention(out, q, layer, table[:, :32].contiguous(), ln, dim ** -0.5, dt)
    assert torch.equal(out, layer.attend(q, table, ln, dim ** -0.5))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("lens,group", [([9000, 3], 4), ([64] * 150, 12)])
def test_attention_over_its_own_queries(lens, group, dtype):
    g, dt, page, dim, hkv = gen(5), DT[dtype], 64, 128, 2
    pages = sum(-(-n // page) for n in lens)
    layer, table = filled(pages, hkv, page, dim, 3, g), table_of(lens, page, pages, g)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((len(lens), hkv * group, dim), generator=g, device="cuda").to(dt)
    want = layer.attend(q, table, ln, 0.1)
    for _ in range(3):
        x = q.clone()
        assert layer.attend(x, table, ln, 0.1, out=x) is x and torch.equal(x, want)


def test_attention_of_pages_that_requests_share():
    """A common beginning is stored once; and a page may stand in a table twice."""
    g, page, dim, hkv, group = gen(6), 32, 128, 4, 4
    layer = filled(40, hkv, page, dim, 4, g)
    table = torch.tensor([[3, 4, 5, 6], [3, 4, 9, 10], [3, 3, 3, 3]], dtype=torch.int32, device="cuda")
    ln = torch.tensor([128, 97, 100], dtype=torch.int32, device="cuda")
    q = torch.randn((3, hkv * group, dim), generator=g, device="cuda").to(torch.bfloat16)
    check_attention(layer.attend(q, table, ln, dim ** -0.5), q, layer, table, ln, dim ** -0.5, torch.bfloat16)


def test_two_graphs_and_an_eager_call_with_one_work_area():
    """One after the other, two captured calls and an eager one may share a work area."""
    g, page, dim, hkv, group = gen(7), 64, 128, 8, 4
    layer = filled(200, hkv, page, dim, 4, g)
    scratch = layer.attend_scratch(hkv * group)
    lens = [[6000], [40, 3000, 1000]]
    tables = [table_of(x, page, 200, g) for x in lens]
    ln = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in lens]
    q = [torch.randn((len(x), hkv * group, dim), generator=g, device="cuda").to(torch.bfloat16) for x in lens]
    want = [layer.attend(*x, 0.1) for x in zip(q, tables, ln)]
    outs, graphs = [torch.empty_like(x) for x in q], []
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            layer.attend(q[i], tables[i], ln[i], 0.1, out=outs[i], scratch=scratch)
        graphs.append(graph)
    for _ in range(4):
        for i in range(2):
            outs[i].fill_(3)
            graphs[i].replay()
            assert torch.equal(outs[i], want[i])
        assert torch.equal(layer.attend(q[1], tables[1], ln[1], 0.1, scratch=scratch), want[1])
    assert bool((scratch[:16384] == 0).all())


def test_cache_decodes_under_capture_and_on_streams():
    cfg = tq.CacheConfig(4, 128, 2, 1)
    cache = tq.PagedPqoCache(cfg, 64, page_size=16, max_requests=3)
    g = gen(8)
    step = cache.plan(torch.tensor([200, 0, 60], dtype=torch.int32, device="cuda"), 260)
    step.check()
    k, v = (torch.randn((260, 2, 128), generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    cache.append(0, k, v, step)
    q = torch.randn((3, 8, 128), generator=g, device="cuda").to(torch.bfloat16)
    att = tq.AttendConfig(128 ** -0.5, 4)
    want = cache.decode(0, q, step, att).fused
    assert bool((want[1] == 0).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = cache.decode(0, q, step, att).fused
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = cache.decode(0, q, step, att).fused
    captured.zero_()
    graph.replay()
    assert torch.equal(other, want) and torch.equal(captured, want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_of_lengths_beyond_the_table_and_below_zero(dtype):
    g, dt, page, dim, hkv, group = gen(9), DT[dtype], 32, 64, 3, 5
    layer = filled(20, hkv, page, dim, 4, g)
    table = table_of([96, 96, 96], page, 20, g)
    q = torch.randn((3, hkv * group, dim), generator=g, device="cuda").to(dt)
    out = layer.attend(q, table, torch.tensor([97, -5, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), 0.1)
    cut = torch.tensor([96, 0, 96], dtype=torch.int32, device="cuda")
    assert torch.equal(out, layer.attend(q, table, cut, 0.1)) and bool((out[1] == 0).all())
    check_attention(out, q, layer, table, cut, 0.1, dt)


@pytest.mark.parametrize("bits,group,page", [(3, 3, 1024), (4, 17, 16), (3, 20, 256), (4, 1, 512)])
@pytest.mark.parametrize("scale", [0.0, -0.1, 0.5])
def test_attention_of_odd_groups_pages_and_scales(bits, group, page, scale):
    lens = [1500, 1, 0, 777, 16]
    for dim, dtype in ((64, "f16"), (128, "bf16"), (256, "f32")):
        g, dt, hkv = gen(dim + group), DT[dtype], 3
        pages = sum(-(-n // page) for n in lens)
        layer, table = filled(pages, hkv, page, dim, bits, g), table_of(lens, page, pages, g)
        ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
        q = torch.randn((5, hkv * group, dim), generator=g, device="cuda").to(dt)
        check_attention(layer.attend(q, table, ln, scale), q, layer, table, ln, scale, dt)


@pytest.mark.parametrize("dtype,bits", [("bf16", 4), ("f32", 3)])
@pytest.mark.parametrize("every", [0, 1, 97])
def test_attention_of_as_many_requests_as_may_be(every, dtype, bits):
    """4,096 requests: none with tokens, all, and a few of a padded batch."""
    g, dt, page, dim, hkv, group, n = gen(10), DT[dtype], 16, 64, 1, 2, 4096
    lens = [(1 + i * 31 % 70) if every and i % every == every - 1 else 0 for i in range(n)]
    pages = sum(-(-x // page) for x in lens) + 1
    layer = filled(pages, hkv, page, dim, bits, g)
    table, ln = table_of(lens, page, pages, g), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((n, hkv * group, dim), generator=g, device="cuda").to(dt)
    out = layer.attend(q, table, ln, 0.1, out=torch.full_like(q, 7))
    check_attention(out, q, layer, table, ln, 0.1, dt)
    assert bool((out[ln == 0] == 0).all())


@pytest.mark.parametrize("rot", [128, 64])
@pytest.mark.parametrize("tokens", [5, 1500])
def test_queries_or_keys_may_be_missing(tokens, rot):
    """At the C entry points: a null q or k is left out, and the rotated keys of an append are written too where wanted."""
    from turboquant_b200.paged import _call, lib
    g, dt, hq, hkv, d = gen(rot), torch.bfloat16, 6, 2, 128
    q, k, v = (torch.randn((tokens, h, d), generator=g, device="cuda").to(dt) for h in (hq, hkv, hkv))
    w = torch.randn(d, generator=g, device="cuda").to(dt)
    rope = tq.QkNormRope(1.0 / torch.arange(1, rot // 2 + 1, device="cuda"), w, w)
    pos = torch.arange(tokens, device="cuda")
    qo, ko = rope(q, k, pos)
    none, rows = (0, 0, 0), lambda t: (t.data_ptr(), t.stride(0), t.stride(1))
    a, b = torch.zeros_like(q), torch.zeros_like(k)
    _call(0, lib.tqb_qk_norm_rope, rope._params(rows(q), rows(a), none, none, tokens, hq, hkv, d, dt, pos))
    _call(0, lib.tqb_qk_norm_rope, rope._params(none, none, rows(k), rows(b), tokens, hq, hkv, d, dt, pos))
    assert torch.equal(a, qo) and torch.equal(b, ko)
    one, two = (layer_of(100, hkv, 16, d, 4) for _ in range(2))
    slots = torch.randperm(1600, generator=g, device="cuda")[:tokens]
    one.append(ko, v, slots)
    c = torch.zeros_like(k)
    _call(0, lib.tqb_paged_append_rope, two._c, rope._params(none, none, rows(k), rows(c), tokens, hq, hkv, d, dt, pos), *rows(v), slots.data_ptr())
    assert torch.equal(c, ko)
    for x, y in zip(one.tensors, two.tensors):
        assert torch.equal(x, y)


def test_arguments_that_do_not_fit_are_refused():
    dt, i32 = torch.bfloat16, dict(dtype=torch.int32, device="cuda")
    layer = layer_of(4, 2, 16, 64, 4)
    k = torch.zeros((3, 2, 64), dtype=dt, device="cuda")
    q, slots, pos = torch.zeros((3, 4, 64), dtype=dt, device="cuda"), torch.arange(3, device="cuda"), torch.arange(3, device="cuda")
    rope = tq.QkNormRope(torch.ones(32, device="cuda"), torch.ones(64, dtype=dt, device="cuda"))
    table, lens = torch.zeros((3, 2), **i32), torch.ones(3, **i32)
    wrong = (tq.DimensionMismatch, TypeError, ValueError, tq.TqbRuntimeError)
    before = [t.clone() for t in layer.tensors]
    for call in (lambda: layer.append(k, k[:2], slots), lambda: layer.append(k, k.float(), slots), lambda: layer.append(k, k, slots[:2]),
                 lambda: layer.append(k, k, slots.int()), lambda: layer.append(k[:, :1], k[:, :1], slots), lambda: layer.append(k.double(), k.double(), slots),
                 lambda: layer.append(k.cpu(), k, slots), lambda: layer.append_rope(rope, q.float(), k, k, pos, slots),
                 lambda: layer.append_rope(rope, q, k, k, pos[:2], slots), lambda: layer.append_rope(rope, q, k, k, pos.float(), slots),
                 lambda: layer.append_rope(rope, q, k, k, pos, slots, q_out=q[:2]), lambda: layer.append_rope(rope, q, k, k, pos, slots, q_out=q.transpose(0, 1)),
                 lambda: rope(q, k, pos, q_out=q[:1].expand(3, 4, 64)), lambda: rope(q, k.half(), pos), lambda: rope(q.half(), k.half(), pos),
                 lambda: rope(q[..., :32], k[..., :32], pos), lambda: rope(q[0], k, pos),
                 lambda: layer.attend(q, table, lens.long(), 0.1), lambda: layer.attend(q, table[:2], lens, 0.1), lambda: layer.attend(q[..., :32], table, lens, 0.1),
                 lambda: layer.attend(q[:, :3], table, lens, 0.1), lambda: layer.attend(q, table.t().contiguous().t(), lens, 0.1),
                 lambda: layer.attend(q, table, lens, 0.1, scratch=torch.zeros(64, dtype=torch.uint8, device="cuda")),
                 lambda: layer.attend(q, table, lens, 0.1, out=q[:2]), lambda: layer.attend(q, table, lens, 0.1, out=q.double()),
                 lambda: layer.attend(q.double(), table, lens, 0.1), lambda: layer.dequantize(slots.int()), lambda: layer.dequantize(slots, torch.float64),
                 lambda: tq.paged_plan(lens, lens[:2], table, lens, torch.zeros(4, **i32), 16, 3),
                 lambda: tq.paged_plan(lens, lens, table, lens, torch.zeros(3, **i32), 16, 3), lambda: tq.paged_plan(lens, lens, table, lens, torch.zeros(4, **i32), 15, 3),
                 lambda: tq.paged_plan(lens, lens, table, lens, torch.zeros(4, **i32), 16, -1),
                 lambda: tq.PagedLayer(*layer.tensors, 5), lambda: tq.PagedLayer(*layer.tensors, 3), lambda: tq.PagedLayer(*layer.tensors[:3], layer.tensors[3].half(), 4),
                 lambda: tq.QkNormRope(torch.ones(31, device="cuda"))(q, k, pos), lambda: tq.QkNormRope(torch.ones(64, device="cuda"))(q, k, pos)):
        with pytest.raises(wrong):
            call()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(before, layer.tensors))
