"""Paged cache on the GPU against plain 64-bit forms: plan and release, norm and rotation, rows into pages and back,
attention of one new token of each request, and all of them together as a batch of requests uses them."""
import math

import numpy as np
import pytest
import torch

import paged_ref as ref
import turboquant_b200 as tq

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def gen(seed=0):
    return torch.Generator(device="cuda").manual_seed(seed)


# ---- plan and release -------------------------------------------------------------------------------------------------
def make_state(seq, page, blocks, spare, seed):
    g = np.random.default_rng(seed)
    used = [-(-s // page) for s in seq]
    perm = g.permutation(sum(used) + spare).astype(np.int32)
    table = np.full((len(seq), blocks), -1, np.int32)
    at = 0
    for r, u in enumerate(used):
        table[r, :u] = perm[at:at + u]
        at += u
    return table, perm[at:].copy()


def plan_on_gpu(seq, new, table, free, count, page, capacity, in_place=False):
    dev = dict(dtype=torch.int32, device="cuda")
    s, n = torch.tensor(seq, **dev), torch.tensor(new, **dev)
    t, f = torch.tensor(table, **dev), torch.tensor(free, **dev)
    st = torch.tensor([count, 0, 0, 0], **dev)
    more = dict(kv_lens=s, state_out=st) if in_place else {}
    step = tq.paged_plan(s, n, t, f, st, page, capacity, **more)
    if not in_place:
        assert s.tolist() == list(seq) and st.tolist() == [count, 0, 0, 0]
    return step, t


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests,page,chunk,extra", [(1, 16, 1, 0), (1, 64, 200, 3), (7, 16, 40, 1), (64, 64, 1, 0), (300, 32, 90, 17),
                                                      (1500, 16, 3, 0), (4096, 128, 1, 5)])
def test_plan(requests, page, chunk, extra, in_place):
    g = np.random.default_rng(requests + page)
    seq = [int(x) for x in g.integers(0, 5 * page, requests)]
    seq[0] = 0
    new = [int(x) for x in g.integers(0, chunk + 1, requests)]
    new[-1] = max(new[-1], 1)
    blocks = max(-(-(s + n) // page) for s, n in zip(seq, new))
    spare = sum(-(-(s + n) // page) - -(-s // page) for s, n in zip(seq, new)) + extra
    table, free = make_state(seq, page, blocks, spare, 1)
    capacity = sum(new) + extra
    step, t = plan_on_gpu(seq, new, table, free, len(free), page, capacity, in_place)
    slots, pos, cu, kv, tab, left = ref.plan(seq, new, table.tolist(), free.tolist(), len(free), page, capacity)
    assert step.state.tolist() == [left, 0, 0, 0]
    assert step.slots.tolist() == slots and step.positions.tolist() == pos
    assert step.cu.tolist() == cu and step.kv_lens.tolist() == kv and t.tolist() == tab
    step.check()


def test_plan_without_requests_or_tokens():
    step, _ = plan_on_gpu([], [], np.zeros((0, 4), np.int32), np.arange(3), 3, 16, 5)
    assert step.slots.tolist() == [-1] * 5 and step.cu.tolist() == [0] and step.state.tolist() == [3, 0, 0, 0]
    step, t = plan_on_gpu([5, 0], [0, 0], [[2], [-1]], [0, 1], 2, 16, 0)
    assert step.slots.numel() == 0 and step.kv_lens.tolist() == [5, 0] and t.tolist() == [[2], [-1]]


@pytest.mark.parametrize("capacity", [40, 5000])
@pytest.mark.parametrize("seq,new,count,status", [([16, 5], [20, 3], 1, 1), ([16, -1], [1, 1], 9, 2), ([16, 5], [1, -3], 9, 2), ([16, 60], [1, 10], 9, 2),
                                                  ([2 ** 31 - 1, 0], [1, 0], 9, 2), ([0, 0], [30, 4981], 9, 2), ([16, 5], [1, 1], -4, 1)])
def test_plan_that_does_not_fit(seq, new, count, status, capacity):
    table = [[7, 8, -1, -1], [9, 3, -1, -1]]
    step, t = plan_on_gpu(seq, new, table, [0, 1, 2, 4, 5, 6, 10, 11, 12], count, 16, capacity)
    assert step.state.tolist() == [max(count, 0), 0, status, 0]
    assert t.tolist() == table and step.kv_lens.tolist() == seq
    assert step.cu.tolist() == [0, 0, 0] and step.slots.tolist() == [-1] * capacity and step.positions.tolist() == [0] * capacity
    with pytest.raises(tq.TqbRuntimeError):
        step.check()


def test_plan_over_capacity():
    step, t = plan_on_gpu([0, 0], [20, 21], [[-1, -1], [-1, -1]], [0, 1, 2, 3], 4, 16, 40)
    assert step.state.tolist() == [4, 0, 3, 0] and t.tolist() == [[-1, -1], [-1, -1]]


def test_plans_and_releases_in_a_row():
    page, requests, blocks, pages = 16, 9, 6, 40
    g = np.random.default_rng(3)
    cache = tq.PagedPqoCache(tq.CacheConfig(4, 64, 1, 1), pages, page, requests, blocks)
    seq, table = [0] * requests, [[-1] * blocks for _ in range(requests)]
    free, left = list(range(pages - 1, -1, -1)), pages
    for i in range(30):
        if i % 3 == 2:
            mask = [bool(x) for x in g.integers(0, 2, requests)]
            cache.release(torch.tensor(mask, device="cuda"))
            for r in range(requests):
                if mask[r]:
                    for b in range(-(-seq[r] // page)):
                        free[left] = table[r][b]
                        table[r][b] = -1
                        left += 1
                    seq[r] = 0
        new = [int(x) for x in g.integers(0, 12, requests)]
        cap = 120
        step = cache.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), cap)
        need = sum(-(-(s + n) // page) - -(-s // page) for s, n in zip(seq, new))
        if need > left or any(s + n > blocks * page for s, n in zip(seq, new)):
            assert int(step.state[2]) in (1, 2)
        else:
            slots, pos, cu, seq, table, left = ref.plan(seq, new, table, free, left, page, cap)
            assert step.slots.tolist() == slots and step.positions.tolist() == pos
        assert cache.seq_lens.tolist() == seq and cache.block_table.tolist() == table and int(cache.state[0]) == left
        assert cache.free_pages.tolist()[:left] == free[:left]


def test_release_that_cannot_be_done_changes_nothing():
    dev = dict(dtype=torch.int32, device="cuda")
    seq, table, free = torch.tensor([40, 16], **dev), torch.tensor([[1, 2, 3], [0, -1, -1]], **dev), torch.tensor([4, 0, 0], **dev)
    state = torch.tensor([1, 0, 0, 0], **dev)
    tq.paged_release(torch.tensor([1, 0], dtype=torch.uint8, device="cuda"), seq, table, free, state, 16)
    assert state.tolist() == [1, 0, 1, 0] and seq.tolist() == [40, 16] and table.tolist() == [[1, 2, 3], [0, -1, -1]]
    seq[0] = 49
    tq.paged_release(torch.tensor([1, 1], dtype=torch.uint8, device="cuda"), seq, table, free, state, 16)
    assert state.tolist() == [1, 0, 2, 0] and seq.tolist() == [49, 16]


# ---- norm and rotation ------------------------------------------------------------------------------------------------
def close(got, want, dtype, row):
    """One rounding to the type (half a step), and f32 arithmetic: the norm's sum of up to 256 squares in a tree of 13
    roundings that the root halves, root and quotient, two products, the angle rounded at up to pi (2 steps), sine and
    cosine (2), two products and a sum: below 32 steps of 2^-24 of the row's largest value."""
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -19 * row
    err = (got.double() - want).abs()
    # a subnormal f16 result is rounded to the fixed step 2^-24
    tol = tol + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.3f} of the tolerance"


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,hq,hkv,rot", [(64, 4, 4, 64), (64, 7, 1, 32), (128, 32, 8, 128), (128, 5, 1, 96), (128, 3, 3, 0), (256, 8, 2, 256), (256, 1, 1, 16)])
def test_norm_rope(dim, hq, hkv, rot, dtype, norm, interleaved):
    g, dt = gen(dim + hq), DT[dtype]
    for tokens in (1, 3, 130):
        qkv = (torch.randn((tokens, (hq + 2 * hkv) * dim), generator=g, device="cuda") * 2).to(dt)
        q, k = qkv[:, : hq * dim].view(tokens, hq, dim), qkv[:, hq * dim: (hq + hkv) * dim].view(tokens, hkv, dim)
        wq, wk = (torch.randn(dim, generator=g, device="cuda").to(dt) for _ in range(2))
        inv = (1e4 ** -(torch.arange(0, rot, 2, device="cuda").double() / max(rot, 1))).float()
        pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda")
        pos[0] = 0 if tokens > 1 else 2 ** 31 - 1
        if tokens == 3:
            pos = pos.int()
        rope = tq.QkNormRope(inv, wq, None if tokens == 3 else wk, eps=1e-5, norm=norm, interleaved=interleaved)
        qo, ko = rope(q, k, pos)
        for got, x, w in ((qo, q, wq), (ko, k, None if tokens == 3 else wk)):
            want = ref.norm_rope(x, w, pos, inv, 1e-5, norm, interleaved)
            close(got, want, dt, want.abs().amax(-1, keepdim=True))
        # in place, in the strided rows
        before = qkv.clone()
        rope(q, k, pos, q_out=q, k_out=k)
        assert torch.equal(q, qo) and torch.equal(k, ko)
        assert torch.equal(qkv[:, (hq + hkv) * dim:], before[:, (hq + hkv) * dim:])


def test_norm_rope_of_nothing_and_of_rows_that_are_not_dense():
    rope = tq.QkNormRope(torch.ones(32, device="cuda"))
    q = torch.empty((0, 4, 64), device="cuda", dtype=torch.bfloat16)
    qo, ko = rope(q, q, torch.empty(0, dtype=torch.int32, device="cuda"))
    assert qo.shape == (0, 4, 64)
    x = torch.randn((6, 64, 4), device="cuda", generator=gen()).to(torch.bfloat16).transpose(1, 2)
    pos = torch.arange(6, device="cuda")
    a, b = rope(x, x, pos), rope(x.contiguous(), x.contiguous(), pos)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---- rows into pages and back -------------------------------------------------------------------------------------------
def layer_of(pages, heads, page, dim, bits, fill=None):
    a = []
    for _ in range(2):
        a.append(torch.zeros((pages, heads, page, dim * bits // 8), dtype=torch.uint8, device="cuda"))
        a.append(torch.zeros((pages, heads, page, dim // 32), dtype=torch.int16, device="cuda"))
    if fill is not None:
        for t in a:
            t.fill_(fill)
    return tq.PagedLayer(*a, bits)


def stored(layer, slots):
    p = layer.page_size
    return [t[slots // p, :, slots % p] for t in layer.tensors]


@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,heads,page", [(64, 1, 16), (64, 5, 64), (128, 8, 64), (128, 3, 16), (256, 2, 32)])
def test_append_stores_the_bytes_of_block_quantize(dim, heads, page, dtype, bits):
    g, dt = gen(dim + heads), DT[dtype]
    for tokens in (1, 77, 700):
        pages = -(-tokens // page) + 3
        layer = layer_of(pages, heads, page, dim, bits, 0x55)
        kv = torch.randn((tokens, 2 * heads, dim), generator=g, device="cuda") * torch.exp(torch.randn(dim, generator=g, device="cuda"))
        kv[0, 0] = 0
        kv[tokens // 2, :, : dim // 2] *= 1e-12
        kv = kv.to(dt)
        k, v = kv[:, :heads], kv[:, heads:]
        slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
        if tokens > 5:
            slots[3], slots[4], slots[5] = -1, pages * page, -(1 << 40)
        layer.append(k, v, slots)
        ok = (slots >= 0) & (slots < pages * page)
        got = stored(layer, slots[ok])
        for x, idx, sc in ((k, got[0], got[1]), (v, got[2], got[3])):
            wi, ws = tq.block_quantize(x[ok].reshape(-1, dim).contiguous(), bits)
            assert torch.equal(idx.reshape(wi.shape), wi) and torch.equal(sc.reshape(ws.shape), ws)
        rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
        rest[slots[ok]] = False
        for t, b in zip(stored(layer, rest.nonzero()[:, 0]), (0x55, 0x55, 0x55, 0x55)):
            assert bool((t == b).all())


@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,hq,hkv,rot,norm,interleaved", [(64, 6, 2, 64, True, False), (128, 32, 8, 128, True, False), (128, 8, 8, 64, False, True), (256, 3, 1, 256, True, True)])
def test_append_rope_is_the_two_calls_in_one(dim, hq, hkv, rot, norm, interleaved, dtype, bits):
    g, dt, page = gen(dim + hq), DT[dtype], 16
    for tokens in (1, 45):
        a, b = layer_of(6, hkv, page, dim, bits), layer_of(6, hkv, page, dim, bits)
        qkv = (torch.randn((tokens, hq + 2 * hkv, dim), generator=g, device="cuda") * 3).to(dt)
        q, k, v = qkv.split([hq, hkv, hkv], 1)
        w = torch.randn(dim, generator=g, device="cuda").to(dt)
        inv = (1e4 ** -(torch.arange(0, rot, 2, device="cuda").double() / rot)).float()
        pos = torch.randint(0, 100000, (tokens,), generator=g, device="cuda").int()
        slots = torch.randperm(6 * page, generator=g, device="cuda")[:tokens]
        if tokens > 2:
            slots[2] = -1
        rope = tq.QkNormRope(inv, w, w, norm=norm, interleaved=interleaved)
        qo, ko = rope(q, k, pos)
        a.append(ko, v, slots)
        got = b.append_rope(rope, q, k, v, pos, slots)
        assert torch.equal(got, qo)
        for x, y in zip(a.tensors, b.tensors):
            assert torch.equal(x, y)


@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,heads,page", [(64, 3, 16), (128, 8, 64), (256, 1, 128)])
def test_dequantize_gives_the_values_of_block_dequantize(dim, heads, page, dtype, bits):
    g = gen(dim)
    layer = layer_of(5, heads, page, dim, bits)
    n = 5 * page
    kv = torch.randn((2, n, heads, dim), generator=g, device="cuda")
    layer.append(kv[0], kv[1], torch.randperm(n, generator=g, device="cuda"))
    for count in (0, 1, 53):
        slots = torch.randint(0, n, (count,), generator=g, device="cuda")
        if count > 3:
            slots[1], slots[2] = -1, n
        ok = (slots >= 0) & (slots < n)
        for got, (idx, sc) in zip(layer.dequantize(slots, DT[dtype]), (stored(layer, slots.clamp(0, n - 1))[:2], stored(layer, slots.clamp(0, n - 1))[2:])):
            if count == 0:
                assert got.shape == (0, heads, dim)
                continue
            want = tq.block_dequantize(idx.reshape(-1, dim * bits // 8).contiguous(), sc.reshape(-1, dim // 32).contiguous(), bits, dim, dtype=DT[dtype])
            want = want.view(count, heads, dim) * ok[:, None, None].to(DT[dtype])
            assert torch.equal(got, want)


# ---- attention ----------------------------------------------------------------------------------------------------------
def filled(pages, heads, page, dim, bits, g, spread=0.5):
    layer = layer_of(pages, heads, page, dim, bits)
    for i in (0, 2):
        layer.tensors[i].copy_(torch.randint(0, 256, layer.tensors[i].shape, generator=g, device="cuda", dtype=torch.uint8))
        s = torch.exp(spread * torch.randn(layer.tensors[i + 1].shape, generator=g, device="cuda")).half()
        layer.tensors[i + 1].copy_((-s).view(torch.int16))
    return layer


def table_of(lens, page, pages, g, blocks=None):
    need = [-(-n // page) for n in lens]
    t = torch.full((len(lens), blocks or max(1, max(need))), -1, dtype=torch.int32, device="cuda")
    perm, at = torch.randperm(pages, generator=g, device="cuda").int(), 0
    for r, n in enumerate(need):
        t[r, :n] = perm[at:at + n]
        at += n
    return t


def check_attention(out, q, layer, table, lens, scale, dtype):
    """Off by half a step of the type; and, relative to the size that the weights act on: a score off by `serr` changes a
    weight and the weights' sum by as much each; 16-bit queries take weights and weights times scales rounded to f16
    (2^-11 each), f32 ones do not; 2^-13 (f32: 2^-17) is left for the f32 sums."""
    want, slack, serr = ref.attend(q, layer.tensors, layer.bits, table, lens, scale)
    narrow = q.dtype != torch.float32
    rel = (2 * serr + 2.0 ** -10 + 2.0 ** -13) if narrow else (2 * serr * 2.0 ** -4 + 2.0 ** -17)
    tol = torch.finfo(dtype).eps / 2 * want.abs() + 1.01 * rel * slack + (2.0 ** -25 if dtype == torch.float16 else 0)
    err = (out.double() - want).abs()
    assert out.dtype == dtype and bool(torch.isfinite(out).all())
    assert bool((err <= tol).all()), f"off by {float((err / tol.clamp(min=1e-300)).max()):.3f} of the tolerance"
    return want


LENS = [1, 15, 16, 17, 63, 64, 65, 0, 127, 130, 400, 2, 33]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("dim,hkv,group,page", [(64, 2, 1, 16), (64, 1, 7, 64), (128, 8, 4, 64), (128, 2, 8, 16), (128, 1, 1, 32), (128, 1, 12, 16), (256, 2, 2, 16), (256, 1, 5, 128)])
def test_attention_of_short_requests(dim, hkv, group, page, bits, dtype):
    g, dt = gen(dim + group), DT[dtype]
    pages = sum(-(-n // page) for n in LENS) + 2
    layer = filled(pages, hkv, page, dim, bits, g)
    table = table_of(LENS, page, pages, g)
    # whatever lies behind a request's last token must not matter: NaN and infinite scales
    for r, n in enumerate(LENS):
        if n % page:
            for i in (1, 3):
                layer.tensors[i][int(table[r, n // page]), :, n % page:] = 0x7E00 if i == 1 else 0x7C00
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    qkv = (torch.randn((len(LENS), (group + 2) * hkv * dim), generator=g, device="cuda") * 2).to(dt)
    q = qkv[:, : group * hkv * dim].view(len(LENS), group * hkv, dim)
    out = layer.attend(q, table, lens, dim ** -0.5)
    check_attention(out, q, layer, table, lens, dim ** -0.5, dt)
    assert bool((out[LENS.index(0)] == 0).all())
    again = layer.attend(q.contiguous(), table, lens, dim ** -0.5, out=torch.full_like(out, 7))
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("lens,hkv,group", [([9000], 8, 4), ([70001], 1, 8), ([20000, 0, 0, 3], 2, 1), ([3000, 1, 999, 4097, 64], 8, 8)])
def test_attention_split_over_the_length(lens, hkv, group, bits, dtype):
    g, dt, page, dim = gen(len(lens)), DT[dtype], 64, 128
    pages = sum(-(-n // page) for n in lens) + 1
    layer = filled(pages, hkv, page, dim, bits, g)
    table = table_of(lens, page, pages, g)
    ln = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((len(lens), group * hkv, dim), generator=g, device="cuda").to(dt)
    scratch = layer.attend_scratch(group * hkv)
    out = layer.attend(q, table, ln, dim ** -0.5, scratch=scratch)
    check_attention(out, q, layer, table, ln, dim ** -0.5, dt)
    for _ in range(3):
        assert torch.equal(out, layer.attend(q, table, ln, dim ** -0.5, scratch=scratch))
    assert bool((scratch[:8192] == 0).all())


@pytest.mark.parametrize("bits", [3, 4])
def test_attention_of_many_requests(bits):
    g, page, dim, hkv, group = gen(5), 16, 64, 2, 2
    lens = [int(x) for x in np.random.default_rng(0).integers(0, 90, 1300)]
    pages = sum(-(-n // page) for n in lens) + 1
    layer = filled(pages, hkv, page, dim, bits, g)
    table, ln = table_of(lens, page, pages, g), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((len(lens), hkv * group, dim), generator=g, device="cuda").to(torch.bfloat16)
    check_attention(layer.attend(q, table, ln, 0.2), q, layer, table, ln, 0.2, torch.bfloat16)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_leaves_pages_out_that_do_not_exist(dtype):
    g, page, dim, hkv, group, lens = gen(8), 16, 128, 2, 4, [100, 40, 500]
    pages = sum(-(-n // page) for n in lens)
    layer = filled(pages, hkv, page, dim, 4, g)
    table, ln = table_of(lens, page, pages, g), torch.tensor(lens, dtype=torch.int32, device="cuda")
    table[0, 2], table[0, 5], table[2, 0], table[2, 17] = -1, pages, 2 ** 31 - 1, -(2 ** 31)
    table[1] = -7
    q = torch.randn((3, hkv * group, dim), generator=g, device="cuda").to(DT[dtype])
    out = layer.attend(q, table, ln, dim ** -0.5)
    check_attention(out, q, layer, table, ln, dim ** -0.5, DT[dtype])
    assert bool((out[1] == 0).all())
    # lengths beyond the table are cut, negative ones are none
    long = torch.tensor([2 ** 31 - 1, -5, 4000], dtype=torch.int32, device="cuda")
    out = layer.attend(q, table, long, dim ** -0.5)
    check_attention(out, q, layer, table, long, dim ** -0.5, DT[dtype])


@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("qscale,vscale", [(1e-3, 1.0), (60.0, 1.0), (1.0, 900.0), (1.0, 3e4), (1.0, 1e-4), (200.0, 2e4)])
def test_attention_of_far_scales(qscale, vscale, bits):
    """Peaked and flat softmaxes, values near the ends of f16."""
    g, page, dim, hkv, group, lens = gen(9), 32, 128, 2, 4, [700, 65, 3]
    pages = sum(-(-n // page) for n in lens)
    layer = filled(pages, hkv, page, dim, bits, g, 0.0)
    layer.tensors[3].copy_((layer.tensors[3].view(torch.float16).float() * vscale).half().view(torch.int16))
    table, ln = table_of(lens, page, pages, g), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = (torch.randn((3, hkv * group, dim), generator=g, device="cuda") * qscale).to(torch.bfloat16)
    out = layer.attend(q, table, ln, dim ** -0.5, out=torch.empty((3, hkv * group, dim), dtype=torch.float32, device="cuda"))
    check_attention(out, q, layer, table, ln, dim ** -0.5, torch.float32)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_passes_on_what_is_not_a_number(dtype):
    g, page, dim, lens = gen(10), 16, 128, [50, 50, 50]
    layer = filled(12, 1, page, dim, 4, g)
    table, ln = table_of(lens, page, 12, g), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((3, 4, dim), generator=g, device="cuda").to(DT[dtype])
    q[1, 2, 5] = math.nan
    out = layer.attend(q, table, ln, dim ** -0.5)
    assert bool(out[1, 2].isnan().all())
    keep = torch.ones((3, 4), dtype=torch.bool, device="cuda")
    keep[1, 2] = False
    assert bool(out[keep].isfinite().all())


def test_attention_in_a_graph_serves_other_lengths():
    g, page, dim, hkv, group = gen(11), 64, 128, 8, 4
    layer = filled(200, hkv, page, dim, 4, g)
    lens = [3000, 17, 0, 900]
    table, ln = table_of([3000] * 4, page, 200, g), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((4, hkv * group, dim), generator=g, device="cuda").to(torch.bfloat16)
    out, scratch = torch.empty_like(q), layer.attend_scratch(hkv * group)
    layer.attend(q, table, ln, dim ** -0.5, out=out, scratch=scratch)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.attend(q, table, ln, dim ** -0.5, out=out, scratch=scratch)
        layer.attend(q, table, ln, dim ** -0.5, out=out, scratch=scratch)
    for lens in ([3000, 17, 0, 900], [1, 2, 3, 4], [0, 0, 0, 0], [3000, 3000, 3000, 2999]):
        ln.copy_(torch.tensor(lens, dtype=torch.int32))
        out.fill_(3)
        graph.replay()
        check_attention(out, q, layer, table, ln, dim ** -0.5, torch.bfloat16)


def test_attention_on_two_streams():
    g, page, dim, hkv, group, lens = gen(12), 64, 128, 4, 4, [5000, 3, 1000]
    pages = sum(-(-n // page) for n in lens)
    layer = filled(pages, hkv, page, dim, 4, g)
    table, ln = table_of(lens, page, pages, g), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((3, hkv * group, dim), generator=g, device="cuda").to(torch.bfloat16)
    want = layer.attend(q, table, ln, 0.1)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for s, o in zip(streams, got):
            with torch.cuda.stream(s):
                o.append(layer.attend(q, table, ln, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for o in got for x in o)


def test_offsets_past_32_bits():
    g, page, dim, hkv, group = gen(13), 64, 256, 8, 2
    pages = 70000   # 4.6 GB of keys' indices
    layer = layer_of(pages, hkv, page, dim, 4)
    use = torch.tensor([pages - 1, 3, pages - 2, 65537], dtype=torch.int32, device="cuda")
    slots = (use.long()[:, None] * page + torch.arange(page, device="cuda")).view(-1)[:250]
    kv = torch.randn((2, 250, hkv, dim), generator=g, device="cuda").to(torch.bfloat16)
    layer.append(kv[0], kv[1], slots)
    k, _ = layer.dequantize(slots, torch.bfloat16)
    wi, ws = tq.block_quantize(kv[0].reshape(-1, dim).contiguous(), 4)
    assert torch.equal(k.reshape(-1, dim), tq.block_dequantize(wi, ws, 4, dim, dtype=torch.bfloat16))
    q = torch.randn((1, hkv * group, dim), generator=g, device="cuda").to(torch.bfloat16)
    ln = torch.tensor([250], dtype=torch.int32, device="cuda")
    check_attention(layer.attend(q, use[None], ln, dim ** -0.5), q, layer, use[None], ln, dim ** -0.5, torch.bfloat16)


# ---- together -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits,dim", [(4, 128), (3, 128), (4, 64)])
def test_requests_of_different_lengths_together(bits, dim):
    """Prompts and decode steps of a batch whose requests come and go, against one PqoCache for each request."""
    g, hq, hkv, page, requests, layers, dt = gen(14), 8, 2, 16, 5, 2, torch.bfloat16
    cache = tq.PagedPqoCache(tq.CacheConfig(bits, dim, hkv, layers), 60, page, requests)
    alone = {}
    inv = (1e4 ** -(torch.arange(0, dim, 2, device="cuda").double() / dim)).float()
    rope = [tq.QkNormRope(inv, torch.randn(dim, generator=g, device="cuda").to(dt), torch.randn(dim, generator=g, device="cuda").to(dt)) for _ in range(layers)]
    att = tq.AttendConfig(dim ** -0.5, hq // hkv)
    lens = [0] * requests
    script = [[37, 0, 5, 0, 0], [1, 18, 1, 0, 0], [1, 1, 1, 70, 0], [1] * 5, "release", [1, 9, 1, 1, 1], [1] * 5, [1] * 5]
    for new in script:
        if new == "release":
            cache.release(torch.tensor([False, True, False, False, True], device="cuda"))
            for r in (1, 4):
                lens[r] = 0
                alone.pop(r)
            continue
        total = sum(new)
        step = cache.plan(torch.tensor(new, dtype=torch.int32, device="cuda"), total + 3)
        step.check()
        for layer in range(layers):
            qkv = torch.randn((total, hq + 2 * hkv, dim), generator=g, device="cuda").to(dt)
            q, k, v = qkv.split([hq, hkv, hkv], 1)
            turned, ko = rope[layer](q, k, step.positions[:total])
            assert torch.equal(cache.append_rope(layer, rope[layer], q, k, v, step), turned)
            at = 0
            out = None
            if all(n == 1 for n in new):
                out = cache.decode(layer, turned, step, att).fused
            for r, n in enumerate(new):
                if n == 0:
                    continue
                one = alone.setdefault(r, tq.PqoCache(tq.CacheConfig(bits, dim, hkv, layers)))
                rows = lambda x: x[at:at + n].transpose(0, 1)[None].contiguous()  # noqa: E731
                if out is not None:
                    want = one.decode(layer, rows(ko), rows(v), rows(turned), att).fused[0, :, 0]
                    # both are within a few 2^-9 of the exact result (each rounds to bf16 and errs a little before)
                    assert torch.allclose(out[r].float(), want.float(), rtol=2.0 ** -7, atol=2.0 ** -8)
                else:
                    one.prefill(layer, rows(ko), rows(v))
                at += n
        lens = [s + n for s, n in zip(lens, new)]
    for r in range(requests):
        slots = torch.arange(lens[r], device="cuda")
        slots = cache.block_table[r].long()[slots // page] * page + slots % page
        for layer in range(layers):
            got = cache.dequantize(layer, slots)
            want = alone[r].dequantize_full(layer)
            for x, y in zip(got, want):
                assert torch.equal(x.transpose(0, 1), y[0])


def test_step_in_a_graph():
    """Plan, rows and attention captured once and replayed token after token."""
    g, hq, hkv, dim, page, requests, dt = gen(15), 8, 2, 128, 16, 3, torch.bfloat16
    cache = tq.PagedPqoCache(tq.CacheConfig(4, dim, hkv, 1), 30, page, requests)
    other = tq.PagedPqoCache(tq.CacheConfig(4, dim, hkv, 1), 30, page, requests)
    rope = tq.QkNormRope((1e4 ** -(torch.arange(0, dim, 2, device="cuda").double() / dim)).float())
    att = tq.AttendConfig(dim ** -0.5, hq // hkv)
    qkv = torch.zeros((requests, hq + 2 * hkv, dim), device="cuda", dtype=dt)
    new = torch.ones(requests, dtype=torch.int32, device="cuda")

    def one(c):
        step = c.plan(new, requests)
        q, k, v = qkv.split([hq, hkv, hkv], 1)
        return c.decode(0, c.append_rope(0, rope, q, k, v, step), step, att).fused

    one(other)   # before the capture
    other.release(torch.ones(requests, dtype=torch.bool, device="cuda"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one(cache)
    for i in range(40):
        qkv.copy_(torch.randn(qkv.shape, generator=g, device="cuda"))
        new[1] = i % 2
        graph.replay()
        assert torch.equal(out, one(other))
        assert cache.seq_lens.tolist() == other.seq_lens.tolist() and int(cache.state[2]) == 0
