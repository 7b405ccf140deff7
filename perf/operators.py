"""Measured cases of the paged-cache operators: the same work in plain torch operations and through `turboquant_b200`.

  plan      block tables, slot map and positions of a step, built on the GPU from the requests' lengths
  rope      norms of queries and keys for each head with the position rotation in the same pass
  step_in   the same for a step's queries and keys, with the keys and the values packed into their pages
  store     keys and values packed into their pages, and read back as the values they stand for
  readback  rows of the pages handed back dequantized, as an engine's own attention takes them for a shared prefix
  attend    attention of one new token of each request over the paged packed cache

A page holds `page` tokens of every KV head of a layer: indices [pages, kv_heads, page, head_dim * bits / 8] u8 and scales
[pages, kv_heads, page, head_dim / 32] (f16 bits, the sign marks the outlier codebook).  A block of 32 values x is stored
as the codes of s .* H x / sqrt(32) over a scale (H: the 32-point Walsh-Hadamard matrix, s: a fixed sign pattern).
Shapes are those of the benchmark and the tests (8 KV heads, groups of 1 to 8 query heads, batch 64 at 8,192 tokens, one
sequence of 131,072) and odd sizes between them.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
R = 2.1573                   # the outermost centroid of both codebooks
C3 = [-2.1573, -1.3336, -0.7434, -0.2428, 0.2428, 0.7434, 1.3336, 2.1573]
B3 = [-1.7455, -1.0385, -0.4931, 0.0, 0.4931, 1.0385, 1.7455]
SIGNS = [1, -1, 1, 1, -1, -1, 1, -1, 1, 1, -1, 1, -1, 1, -1, -1, 1, -1, -1, 1, 1, -1, 1, -1, -1, 1, 1, 1, -1, -1, 1, -1]


def listed():
    return [
        # the bookkeeping of one decode step of a running batch: every request gets one token
        dict(name="plan_decode_64", op="plan", requests=64, longest=8192, chunk=1, page=64),
        # a step that mixes chunks of prompts with decoding requests
        dict(name="plan_mixed_211", op="plan", requests=211, longest=5003, chunk=511, page=16),
        # one token of one request: latency
        dict(name="rope_token", op="rope", tokens=1, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16", norm=True, interleaved=False, far=131072),
        # a prompt of odd length, neighbouring elements rotated together
        dict(name="rope_prompt_8191", op="rope", tokens=8191, q_heads=32, kv_heads=8, head_dim=128, dtype="f16", norm=True, interleaved=True, far=8192),
        # what a decode step of a batch of 64 does before its attention
        dict(name="step_in_64_4bit", op="step_in", tokens=64, q_heads=32, kv_heads=8, head_dim=128, bits=4, dtype="bf16", norm=True, interleaved=False, far=8192, page=64),
        # prompts of a model without norms of queries and keys
        dict(name="step_in_6007_3bit", op="step_in", tokens=6007, q_heads=16, kv_heads=8, head_dim=128, bits=3, dtype="bf16", norm=False, interleaved=False, far=32768, page=32),
        # a prompt whose keys are rotated elsewhere
        dict(name="store_16384_d64", op="store", tokens=16384, kv_heads=8, head_dim=64, bits=4, dtype="f16", page=64),
        # a shared prefix handed to an engine's own attention
        dict(name="readback_32k_4bit", op="readback", tokens=32768, kv_heads=8, head_dim=128, bits=4, dtype="bf16", page=64),
        # one short request
        dict(name="attend_one_1000", op="attend", requests=1, longest=1000, ragged=False, q_heads=16, kv_heads=8, head_dim=128, bits=4, dtype="bf16", page=64),
        # a full batch of requests of different lengths
        dict(name="attend_64_ragged_8k", op="attend", requests=64, longest=8192, ragged=True, q_heads=32, kv_heads=8, head_dim=128, bits=4, dtype="bf16", page=64),
        # one long document, 8 query heads for each KV head
        dict(name="attend_one_128k", op="attend", requests=1, longest=131072, ragged=False, q_heads=64, kv_heads=8, head_dim=128, bits=4, dtype="f16", page=128),
        # many short chats, 3-bit
        dict(name="attend_97_ragged_2k_3bit", op="attend", requests=97, longest=2003, ragged=True, q_heads=16, kv_heads=8, head_dim=128, bits=3, dtype="bf16", page=16),
    ]


def _log(rng, lo, hi):
    """An odd or even size between lo and hi, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "rope", "step_in", "store", "readback", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        return dict(op=op, requests=_log(rng, 1, 256), longest=_log(rng, 10, 8192), chunk=rng.choice([1, _log(rng, 2, 512)]), page=page)
    hkv, dim, dtype = rng.choice([1, 2, 8]), rng.choice([64, 128, 256]), rng.choice(["bf16", "bf16", "f16"])
    hq, bits = hkv * rng.choice([1, 2, 4, 8]), rng.choice([3, 4])
    if op == "rope":
        return dict(op=op, tokens=_log(rng, 1, 8192), q_heads=hq, kv_heads=hkv, head_dim=dim, dtype=rng.choice([dtype, dtype, "f32"]), norm=rng.random() < 0.7,
                    interleaved=rng.random() < 0.4, far=_log(rng, 1000, 1000000))
    if op == "step_in":
        return dict(op=op, tokens=_log(rng, 1, 4096), q_heads=hq, kv_heads=hkv, head_dim=dim, bits=bits, dtype=dtype, norm=rng.random() < 0.5,
                    interleaved=rng.random() < 0.3, far=_log(rng, 1000, 100000), page=page)
    if op in ("store", "readback"):
        return dict(op=op, tokens=_log(rng, 1, 16384), kv_heads=hkv, head_dim=dim, bits=bits, dtype=dtype, page=page)
    longest = _log(rng, 1, 65536)
    n = _log(rng, 1, max(1, min(200, 200000 // longest)))
    return dict(op=op, requests=n, longest=longest, ragged=rng.random() < 0.7, q_heads=hq, kv_heads=hkv, head_dim=dim, bits=bits, dtype=dtype, page=page)


# ---- sizes that follow from a case ----------------------------------------------------------------------------------
def _lens(c):
    """The requests' stored lengths: the longest, and lengths down to a sixteenth of it, spread over their logarithm."""
    rng = random.Random(c["requests"] * 1000003 + c["longest"])
    if not c.get("ragged", True):
        return [c["longest"]] * c["requests"]
    return [c["longest"]] + [_log(rng, max(1.0, c["longest"] / 16), c["longest"]) for _ in range(c["requests"] - 1)]


def _new(c):
    """Tokens that each request of a `plan` case brings: one, or for every third request a chunk of a prompt."""
    rng = random.Random(c["requests"] * 7919 + c["chunk"])
    return [rng.randint(1, c["chunk"]) if i % 3 == 0 else 1 for i in range(c["requests"])]


def _row(c):
    """Bytes of one packed row with its scales."""
    return c["head_dim"] * c["bits"] // 8 + c["head_dim"] // 16


def work(c):
    op, b = c["op"], SIZE.get(c.get("dtype"), 0)
    if op == "plan":
        s, n, p = _lens(c), _new(c), c["page"]
        taken = sum(-(-(x + y) // p) - -(-x // p) for x, y in zip(s, n))
        return {"bytes": 16 * c["requests"] + 8 * taken + 12 * sum(n), "flops": 0}
    if op == "attend":
        toks = sum(_lens(c))
        return {"bytes": 2 * toks * c["kv_heads"] * _row(c) + 2 * c["requests"] * c["q_heads"] * c["head_dim"] * b,
                "flops": 4 * toks * c["q_heads"] * c["head_dim"]}
    t, kv, d = c["tokens"], c["kv_heads"], c["head_dim"]
    if op == "rope":
        n = t * (c["q_heads"] + kv) * d
        return {"bytes": 2 * n * b + 4 * t, "flops": 8 * n}
    if op == "step_in":
        q, n = t * c["q_heads"] * d, t * kv * d
        return {"bytes": 2 * q * b + 2 * n * b + 2 * t * kv * _row(c) * 2 + 2 * n * b + 12 * t, "flops": 8 * (q + n) + 32 * n}
    if op == "store":
        n = t * kv * d
        return {"bytes": 2 * n * b + 2 * t * kv * _row(c) * 2 + 2 * n * b + 8 * t, "flops": 32 * n}
    n = t * kv * d
    return {"bytes": 2 * t * kv * _row(c) + 2 * n * b + 8 * t, "flops": 14 * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _codes(rows, dim, bits, g):
    """Packed codes of rows as they come of normal values: [*rows, dim * bits / 8]."""
    x = torch.randn((*rows, dim), generator=g, device="cuda", dtype=torch.bfloat16)
    if bits == 4:
        c = (x * (7.5 / R) + 7.5).round_().clamp_(0, 15).to(torch.uint8)
        return c[..., 0::2] | (c[..., 1::2] << 4)
    c = torch.bucketize(x, torch.tensor(B3, device="cuda", dtype=torch.bfloat16)).int().view(*rows, dim // 8, 8)
    w = (c << torch.arange(0, 24, 3, device="cuda", dtype=torch.int32)).sum(-1, dtype=torch.int32)
    return torch.stack([w & 255, (w >> 8) & 255, w >> 16], -1).to(torch.uint8).view(*rows, dim * 3 // 8)


def _scales(rows, dim, g):
    s = torch.randn((*rows, dim // 32), generator=g, device="cuda") * 0.3
    return -torch.exp(s).half().view(torch.int16).view(torch.float16)


def _pages(c, pages, g):
    rows = (pages, c["kv_heads"], c["page"])
    a = []
    for _ in range(2):
        a += [_codes(rows, c["head_dim"], c["bits"], g), _scales(rows, c["head_dim"], g).view(torch.int16)]
    return dict(k_idx=a[0], k_sc=a[1], v_idx=a[2], v_sc=a[3])


def _empty_pages(c, pages):
    rows = (pages, c["kv_heads"], c["page"])
    idx = lambda: torch.zeros((*rows, c["head_dim"] * c["bits"] // 8), dtype=torch.uint8, device="cuda")  # noqa: E731
    sc = lambda: torch.zeros((*rows, c["head_dim"] // 32), dtype=torch.int16, device="cuda")  # noqa: E731
    return dict(k_idx=idx(), k_sc=sc(), v_idx=idx(), v_sc=sc())


def _inv_freq(dim):
    return (1.0 / (500000.0 ** (torch.arange(0, dim, 2, dtype=torch.float64) / dim))).float().cuda()


def _rope_state(c, g):
    t, hq, kv, d, dt = c["tokens"], c["q_heads"], c["kv_heads"], c["head_dim"], DTYPES[c["dtype"]]
    # queries, keys and values lie side by side in a token's row, as one projection leaves them
    qkv = (torch.randn((t, (hq + 2 * kv) * d), generator=g, device="cuda") * 1.5).to(dt)
    s = dict(q=qkv[:, : hq * d].view(t, hq, d), k=qkv[:, hq * d: (hq + kv) * d].view(t, kv, d), v=qkv[:, (hq + kv) * d:].view(t, kv, d))
    first = torch.randint(0, max(1, c["far"] - t), (1,), generator=g, device="cuda")
    s["positions"] = (first + torch.arange(t, device="cuda")).int()
    s["inv_freq"] = _inv_freq(d)
    s["q_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) if c["norm"] else None
    s["k_weight"] = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dt) if c["norm"] else None
    return s


def _slots(c, g, pages):
    """A slot for each token: whole pages in any order, the tokens of a page in a row."""
    p = c["page"]
    perm = torch.randperm(pages, generator=g, device="cuda")
    return (perm[:, None] * p + torch.arange(p, device="cuda")).view(-1)[: c["tokens"]].contiguous()


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(case=c)
    if c["op"] == "plan":
        lens, new, p = _lens(c), _new(c), c["page"]
        used = [-(-x // p) for x in lens]
        wide = max(-(-(x + y) // p) for x, y in zip(lens, new)) + 1
        total = sum(used) + sum(-(-(x + y) // p) - -(-x // p) for x, y in zip(lens, new)) + 37
        perm = torch.randperm(total, generator=g, device="cuda").int()
        col, cnt = torch.arange(wide, device="cuda"), torch.tensor(used, device="cuda")
        at = (cnt.cumsum(0) - cnt)[:, None] + col
        s["block_table"] = torch.where(col < cnt[:, None], perm[at.clamp(max=total - 1)], -1)
        s["free_pages"] = perm[sum(used):].contiguous()
        s["state"] = torch.tensor([total - sum(used), 0, 0, 0], dtype=torch.int32, device="cuda")
        s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["new_tokens"] = torch.tensor(new, dtype=torch.int32, device="cuda")
        s["capacity"] = sum(new) + 5
        return s
    if c["op"] == "rope":
        return {**s, **_rope_state(c, g)}
    if c["op"] == "attend":
        lens, p, hq, d, dt = _lens(c), c["page"], c["q_heads"], c["head_dim"], DTYPES[c["dtype"]]
        cnt = torch.tensor([-(-x // p) for x in lens], device="cuda")
        pages = int(cnt.sum()) + 3
        perm, col = torch.randperm(pages, generator=g, device="cuda").int(), torch.arange(int(cnt.max()), device="cuda")
        s["block_table"] = torch.where(col < cnt[:, None], perm[((cnt.cumsum(0) - cnt)[:, None] + col).clamp(max=pages - 1)], -1)
        s["kv_lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["q"] = (torch.randn((c["requests"], hq, d), generator=g, device="cuda") * 1.5).to(dt)
        return {**s, **_pages(c, pages, g)}
    pages = -(-c["tokens"] // c["page"]) + 3
    if c["op"] == "readback":
        return {**s, **_pages(c, pages, g), "slots": _slots(c, g, pages)}
    if c["op"] == "step_in":
        s |= _rope_state(c, g)
    else:
        shape = (c["tokens"], c["kv_heads"], c["head_dim"])
        spread = torch.exp(torch.randn(c["head_dim"], generator=g, device="cuda") * 0.5)
        s["k"], s["v"] = ((torch.randn(shape, generator=g, device="cuda") * spread).to(DTYPES[c["dtype"]]) for _ in range(2))
    return {**s, **_empty_pages(c, pages), "slots": _slots(c, g, pages)}


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _rotation(dtype):
    """The matrix x -> s .* H x / sqrt(32)."""
    i = torch.arange(32, device="cuda")
    bits = (i[:, None] & i).unsqueeze(-1).bitwise_right_shift(torch.arange(5, device="cuda")).bitwise_and(1).sum(-1)
    return (1 - 2 * (bits & 1)).to(dtype) * torch.tensor(SIGNS, device="cuda", dtype=dtype)[:, None] / math.sqrt(32.0)


def _centroids(bits, dtype):
    if bits == 4:
        return -R + torch.arange(16, device="cuda", dtype=dtype) * (2 * R / 15)
    return torch.tensor(C3, device="cuda", dtype=dtype)


def _borders(bits, dtype):
    if bits == 4:
        return -R + (torch.arange(15, device="cuda", dtype=dtype) + 0.5) * (2 * R / 15)
    return torch.tensor(B3, device="cuda", dtype=dtype)


def _unpack(packed, bits):
    if bits == 4:
        return torch.stack([packed & 15, packed >> 4], -1).flatten(-2).int()
    b = packed.view(*packed.shape[:-1], -1, 3).int()
    w = b[..., 0] | (b[..., 1] << 8) | (b[..., 2] << 16)
    return ((w[..., None] >> torch.arange(0, 24, 3, device="cuda", dtype=torch.int32)) & 7).flatten(-2)


def _values(packed, scales, bits):
    """Rows in the rotated domain, [..., dim / 32, 32]."""
    x = _centroids(bits, torch.float32)[_unpack(packed, bits)].unflatten(-1, (-1, 32))
    return x * scales.view(torch.float16).float().abs()[..., None]


def _plain_plan(s):
    p, bt = s["case"]["page"], s["block_table"]
    seq, new, total = s["seq_lens"].long(), s["new_tokens"].long(), s["new_tokens"].long().sum()
    have, want = (seq + p - 1) // p, (seq + new + p - 1) // p
    need = want - have
    col = torch.arange(bt.shape[1], device="cuda")
    nth = (need.cumsum(0) - need)[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < want[:, None])
    free = s["state"][0].long()
    table = torch.where(fresh, s["free_pages"][(free - 1 - nth).clamp(0, len(s["free_pages"]) - 1)], bt)
    cu = torch.cat([torch.zeros_like(total)[None], new.cumsum(0)])
    t = torch.arange(s["capacity"], device="cuda")
    r = (torch.searchsorted(cu, t, right=True) - 1).clamp(max=len(seq) - 1)
    pos = seq[r] + t - cu[r]
    live = t < total
    slots = table[r, (pos // p).clamp(max=bt.shape[1] - 1)].long() * p + pos % p
    state = torch.stack([free - need.sum(), torch.zeros_like(free), torch.zeros_like(free), torch.zeros_like(free)]).int()
    return (torch.where(live, slots, -1), torch.where(live, pos, 0).int(), cu.int(), (seq + new).int(), table, state)


def _plain_turn(x, weight, s, norm):
    c = s["case"]
    y = x.float()
    if norm:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight.float()
    a = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    co, si = a.cos().float(), a.sin().float()
    if c["interleaved"]:
        y1, y2 = y[..., 0::2], y[..., 1::2]
        return torch.stack([y1 * co - y2 * si, y2 * co + y1 * si], -1).flatten(-2).to(x.dtype)
    y1, y2 = y.chunk(2, -1)
    return torch.cat([y1 * co - y2 * si, y2 * co + y1 * si], -1).to(x.dtype)


def _plain_store(x, idx, sc, slots, bits):
    """In 64 bits where a value next to a border is told from its neighbour."""
    t, kv, d = x.shape
    y = x.double().view(t, kv, d // 32, 32) @ _rotation(torch.float64).T
    scale = (y.abs().amax(-1) / R).clamp(min=1e-10)
    code = torch.bucketize(y / scale[..., None], _borders(bits, torch.float64)).int().view(t, kv, d // 8, 8)
    w = (code.long() << torch.arange(0, 8 * bits, bits, device="cuda")).sum(-1)
    packed = ((w[..., None] >> torch.arange(0, 8 * bits, 8, device="cuda")) & 255).to(torch.uint8).flatten(-2)
    p = idx.shape[2]
    idx[slots // p, :, slots % p] = packed
    sc[slots // p, :, slots % p] = (-scale.half()).view(torch.int16)


def _plain_rows(s, slots, dtype):
    p, bits, m = s["k_idx"].shape[2], s["case"]["bits"], _rotation(torch.float32)
    a, b = slots // p, slots % p
    k = _values(s["k_idx"][a, :, b], s["k_sc"][a, :, b], bits) @ m
    v = _values(s["v_idx"][a, :, b], s["v_sc"][a, :, b], bits) @ m
    return k.flatten(-2).to(dtype), v.flatten(-2).to(dtype)


def _plain_attend(s):
    c, q = s["case"], s["q"]
    n, hq, d = q.shape
    kv, m = c["kv_heads"], _rotation(torch.float32)
    pages = s["block_table"].clamp(min=0).long()

    def rows(idx, sc):   # [requests, kv heads, tokens, dim]
        return _values(idx[pages], sc[pages], c["bits"]).flatten(-2).transpose(1, 2).flatten(2, 3)

    qr = (q.float().view(n, hq, d // 32, 32) @ m.T).view(n, kv, hq // kv, d)
    logit = (qr @ rows(s["k_idx"], s["k_sc"]).transpose(-1, -2)) / math.sqrt(d)
    alive = torch.arange(logit.shape[-1], device="cuda") < s["kv_lens"][:, None, None, None]
    logit = logit.masked_fill(~alive, -math.inf)
    p = torch.exp(logit - logit.amax(-1, keepdim=True).clamp(min=-1e30))
    out = (p @ rows(s["v_idx"], s["v_sc"])) / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return (out.view(n, hq, d // 32, 32) @ m).view(n, hq, d).to(q.dtype)


def _plain(s):
    c = s["case"]
    if c["op"] == "plan":
        return _plain_plan(s)
    if c["op"] == "rope":
        return _plain_turn(s["q"], s["q_weight"], s, c["norm"]), _plain_turn(s["k"], s["k_weight"], s, c["norm"])
    if c["op"] == "attend":
        return _plain_attend(s)
    dt = DTYPES[c["dtype"]]
    if c["op"] == "readback":
        return _plain_rows(s, s["slots"], dt)
    q, k = (), s["k"]
    if c["op"] == "step_in":
        q, k = (_plain_turn(s["q"], s["q_weight"], s, c["norm"]),), _plain_turn(k, s["k_weight"], s, c["norm"])
    _plain_store(k, s["k_idx"], s["k_sc"], s["slots"], c["bits"])
    _plain_store(s["v"], s["v_idx"], s["v_sc"], s["slots"], c["bits"])
    return (*q, *_plain_rows(s, s["slots"], dt))


# ---- the framework's operators --------------------------------------------------------------------------------------
def _own(s):
    import turboquant_b200 as tq
    c = s["case"]
    if c["op"] == "plan":
        step = tq.paged_plan(s["seq_lens"], s["new_tokens"], s["block_table"], s["free_pages"], s["state"], c["page"], s["capacity"])
        return step.slots, step.positions, step.cu, step.kv_lens, s["block_table"], step.state
    if "inv_freq" in s and "turn" not in s:   # what a program builds once for a layer
        s["turn"] = tq.QkNormRope(s["inv_freq"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS, norm=c["norm"], interleaved=c["interleaved"])
    if c["op"] == "rope":
        return s["turn"](s["q"], s["k"], s["positions"])
    if "layer" not in s:
        s["layer"] = tq.PagedLayer(s["k_idx"], s["k_sc"], s["v_idx"], s["v_sc"], c["bits"])
    layer = s["layer"]
    if c["op"] == "attend":
        if "scratch" not in s:
            s["scratch"] = layer.attend_scratch(c["q_heads"])
        return layer.attend(s["q"], s["block_table"], s["kv_lens"], 1.0 / math.sqrt(c["head_dim"]), scratch=s["scratch"])
    q, dt = (), DTYPES[c["dtype"]]
    if c["op"] == "step_in":
        q = (layer.append_rope(s["turn"], s["q"], s["k"], s["v"], s["positions"], s["slots"]),)
    elif c["op"] == "store":
        layer.append(s["k"], s["v"], s["slots"])
    return (*q, *layer.dequantize(s["slots"], dt))


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _h32():
    h = torch.ones((1, 1), dtype=torch.float64, device="cuda")
    for _ in range(5):
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(32.0)


def _exact_turn(x, w, s):
    c, y = s["case"], x.double()
    if c["norm"]:
        y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + EPS) * w.double()
    half = y.shape[-1] // 2
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * s["inv_freq"].double())
    u = torch.complex(y[..., first], y[..., second]) * z[:, None]
    out = torch.empty_like(y)
    out[..., first], out[..., second] = u.real, u.imag
    return out


def _exact_coded(x, bits):
    """What the codes of rows x [..., dim] stand for."""
    h, sign = _h32(), torch.tensor(SIGNS, device="cuda", dtype=torch.float64)
    y = (x.double().unflatten(-1, (-1, 32)) @ h) * sign
    scale = torch.clamp(y.abs().amax(-1, keepdim=True) / R, min=1e-10)
    grid = torch.tensor([-R + i * 2 * R / 15 for i in range(16)] if bits == 4 else C3, device="cuda", dtype=torch.float64)
    edge = torch.tensor([-R + (i + 0.5) * 2 * R / 15 for i in range(15)] if bits == 4 else B3, device="cuda", dtype=torch.float64)
    code = torch.searchsorted(edge, (y / scale).contiguous())
    return ((grid[code] * scale.half().double() * sign) @ h).flatten(-2)


def _exact_rows(idx, sc, bits):
    """What packed rows idx [..., bytes] with scales sc [..., blocks] stand for."""
    grid = torch.tensor([-R + i * 2 * R / 15 for i in range(16)] if bits == 4 else C3, device="cuda", dtype=torch.float64)
    bit = (idx[..., None] >> torch.arange(8, device="cuda", dtype=torch.uint8)) & 1
    bit = bit.flatten(-2).unflatten(-1, (-1, bits)).long()
    code = (bit << torch.arange(bits, device="cuda")).sum(-1)
    y = grid[code].unflatten(-1, (-1, 32)) * sc.view(torch.float16).double().abs()[..., None]
    return ((y * torch.tensor(SIGNS, device="cuda", dtype=torch.float64)) @ _h32()).flatten(-2)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "plan":
        return None   # whole numbers
    if c["op"] == "rope":
        return _exact_turn(s["q"], s["q_weight"], s), _exact_turn(s["k"], s["k_weight"], s)
    if c["op"] == "store":
        return _exact_coded(s["k"], c["bits"]), _exact_coded(s["v"], c["bits"])
    if c["op"] == "step_in":   # keys are rounded to their type before they are packed
        k = _exact_turn(s["k"], s["k_weight"], s).to(DTYPES[c["dtype"]])
        return _exact_turn(s["q"], s["q_weight"], s), _exact_coded(k, c["bits"]), _exact_coded(s["v"], c["bits"])
    p = c["page"]
    if c["op"] == "readback":
        a, b = s["slots"] // p, s["slots"] % p
        return (_exact_rows(s["k_idx"][a, :, b], s["k_sc"][a, :, b], c["bits"]), _exact_rows(s["v_idx"][a, :, b], s["v_sc"][a, :, b], c["bits"]))
    kv, d, out = c["kv_heads"], c["head_dim"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, n in enumerate(_lens(c)):
        pages = s["block_table"][r, : -(-n // p)].long()
        for h in range(kv):
            k = _exact_rows(s["k_idx"][pages, h].flatten(0, 1)[:n], s["k_sc"][pages, h].flatten(0, 1)[:n], c["bits"])
            v = _exact_rows(s["v_idx"][pages, h].flatten(0, 1)[:n], s["v_sc"][pages, h].flatten(0, 1)[:n], c["bits"])
            q = s["q"][r].view(kv, -1, d)[h].double()
            out[r].view(kv, -1, d)[h] = torch.softmax(q @ k.T / math.sqrt(d), -1) @ v
    return out
