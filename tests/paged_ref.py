"""Plain 64-bit forms of the paged-cache operators, for the tests."""
import math

import torch

R = 2.1573
CENT = {4: [-R + i * 2 * R / 15 for i in range(16)], 3: [-2.1573, -1.3336, -0.7434, -0.2428, 0.2428, 0.7434, 1.3336, 2.1573]}
SIGNS = [1, -1, 1, 1, -1, -1, 1, -1, 1, 1, -1, 1, -1, 1, -1, -1, 1, -1, -1, 1, 1, -1, 1, -1, -1, 1, 1, 1, -1, -1, 1, -1]


def hadamard(device):
    h = torch.ones((1, 1), dtype=torch.float64, device=device)
    for _ in range(5):
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(32.0)


def signs(device):
    return torch.tensor(SIGNS, dtype=torch.float64, device=device)


def rotated_rows(idx, sc, bits):
    """Packed rows [..., bytes], scales [..., blocks] (int16) -> values in the rotated domain [..., blocks, 32]."""
    bit = (idx[..., None] >> torch.arange(8, device=idx.device, dtype=torch.uint8)) & 1
    code = (bit.flatten(-2).unflatten(-1, (-1, bits)).long() << torch.arange(bits, device=idx.device)).sum(-1)
    y = torch.tensor(CENT[bits], dtype=torch.float64, device=idx.device)[code].unflatten(-1, (-1, 32))
    return y * sc.view(torch.float16).double().abs()[..., None]


def rows(idx, sc, bits):
    y = rotated_rows(idx, sc, bits)
    return ((y * signs(idx.device)) @ hadamard(idx.device)).flatten(-2)


def plan(seq, new, table, free, count, page, capacity):
    """The plan with plain loops: (slots, positions, cu, kv_lens, table, pages left)."""
    table = [list(r) for r in table]
    cu, slots, pos, left = [0], [], [], count
    for r, (s, n) in enumerate(zip(seq, new)):
        for b in range(-(-s // page), -(-(s + n) // page)):
            left -= 1
            table[r][b] = free[left]
        for p in range(s, s + n):
            pos.append(p)
            slots.append(table[r][p // page] * page + p % page)
        cu.append(len(slots))
    pad = capacity - len(slots)
    return slots + [-1] * pad, pos + [0] * pad, cu, [s + n for s, n in zip(seq, new)], table, left


def norm_rope(x, weight, positions, inv_freq, eps, norm, interleaved):
    y = x.double()
    if norm:
        y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + eps)
        y = y * weight.double() if weight is not None else y
    half = inv_freq.shape[0]
    i = torch.arange(half, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    ang = (positions.double()[:, None] * inv_freq.double())[:, None]
    out = y.clone()
    out[..., a] = y[..., a] * ang.cos() - y[..., b] * ang.sin()
    out[..., b] = y[..., b] * ang.cos() + y[..., a] * ang.sin()
    return out


def attend(q, arrays, bits, table, lens, scale, cut=None):
    """Returns (out, slack): slack[r, h, d] is the sum over the tokens of p |v block|, the size that a relative error of the
    weights acts on (the rotation keeps the 2-norm of a block, so no element is off by more), and the largest
    |score error| that a query known to 2^-16 of its largest rotated component allows."""
    k_idx, k_sc, v_idx, v_sc = arrays
    n, hq, d = q.shape
    pages, kv, page, _ = k_idx.shape
    out = torch.zeros((n, hq, d), dtype=torch.float64, device=q.device)
    slack, serr = torch.zeros_like(out), torch.zeros((n, hq, 1), dtype=torch.float64, device=q.device)
    h32, sg = hadamard(q.device), signs(q.device)
    for r in range(n):
        length = min(int(lens[r]), table.shape[1] * page)
        if length <= 0:
            continue
        t = torch.arange(length, device=q.device)
        pg = table[r].long()[t // page]
        ok = (pg >= 0) & (pg < pages)
        pg, off = pg[ok], (t % page)[ok]
        if pg.numel() == 0:
            continue
        k = rotated_rows(k_idx[pg, :, off], k_sc[pg, :, off], bits)     # [tokens, kv, blocks, 32]
        v = rotated_rows(v_idx[pg, :, off], v_sc[pg, :, off], bits)
        qr = ((q[r].double().view(kv, -1, d // 32, 32) @ h32) * sg)     # [kv, g, blocks, 32]
        s = torch.einsum("hgbe,thbe->hgt", qr, k) * scale
        p = torch.softmax(s, -1)
        o = torch.einsum("hgt,thbe->hgbe", p, v)
        out[r] = ((o * sg) @ h32).reshape(hq, d)
        size = torch.einsum("hgt,thb->hgb", p, v.norm(dim=-1))
        slack[r] = size.repeat_interleave(32, -1).reshape(hq, d)
        serr[r] = (qr.abs().amax((-1, -2)) * 2.0 ** -16 * k.abs().sum((-1, -2)).amax(0)[:, None] * abs(scale)).reshape(hq, 1)
    return out, slack, serr
