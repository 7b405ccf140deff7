"""Paged attention split over long requests, against bounds that a lost or doubled page cannot pass."""
import pytest
import torch

import paged_ref as ref
from test_gpu_paged import DT, filled, gen, table_of

pytestmark = pytest.mark.gpu
PAGE, DIM = 16, 128


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("lens,hkv,group", [([9000], 8, 4), ([20000, 0, 0, 3], 2, 1), ([131072], 1, 4), ([131000], 1, 8), ([70001], 1, 12),
                                            ([3000, 1, 999, 4097, 64], 8, 8), ([1 + 37 * i for i in range(120)], 2, 3)])
def test_no_part_of_a_request_is_lost(lens, hkv, group, bits, dtype):
    """Flat softmaxes, outputs in f32.  A head's error by norm: 16-bit queries take weights and products rounded to f16, 2^-11 each
    and independent of one another (2.9e-4 rms), f32 ones f32 sums (below 2^-16).  Sixteen of n tokens left out or taken twice change a head by
    sqrt(16 / n) of its norm, 1.1 % at 131,072: the oracle without a page shows by how much at least."""
    g, dt = gen(len(lens) + hkv), DT[dtype]
    pages = sum(-(-n // PAGE) for n in lens) + 1
    layer = filled(pages, hkv, PAGE, DIM, bits, g)
    table, ln = table_of(lens, PAGE, pages, g), torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = (torch.randn((len(lens), group * hkv, DIM), generator=g, device="cuda") * 2.0 ** -5).to(dt)
    scratch, out = layer.attend_scratch(group * hkv), torch.empty((len(lens), group * hkv, DIM), device="cuda")
    layer.attend(q, table, ln, DIM ** -0.5, out=out, scratch=scratch)
    want, _, _ = ref.attend(q, layer.tensors, bits, table, ln, DIM ** -0.5)
    size, bound = want.norm(dim=-1), 2.0 ** -16 if dtype == "f32" else 2.0 ** -9
    off = (out.double() - want).norm(dim=-1) / size.clamp(min=1e-300)
    assert float(off.max()) <= bound, float(off.max())
    r = lens.index(max(lens))
    last = (lens[r] - 1) // PAGE
    for lost in (0, last // 3, last - 1):
        other = table[r: r + 1].clone()
        other[0, lost] = -1
        less, _, _ = ref.attend(q[r: r + 1], layer.tensors, bits, other, ln[r: r + 1], DIM ** -0.5)
        assert float(((less[0] - want[r]).norm(dim=-1) / size[r]).min()) > 2 * bound
    for _ in range(2):
        assert torch.equal(out, layer.attend(q, table, ln, DIM ** -0.5, out=torch.empty_like(out), scratch=scratch))
    assert bool((scratch[:16384] == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("bits", [3, 4])
@pytest.mark.parametrize("power", [10, 20, 23, 24, 25, 26, 30, 60, 90, 112])
def test_scores_far_from_zero_still_have_a_softmax(power, bits, dtype):
    """One token has weight 1 whatever its score is, from -1e36 to 1e36: the value itself, but for the rounding of weight and product."""
    g, dt, n = gen(power), DT[dtype], 24
    layer = filled(n, 2, PAGE, DIM, bits, g, 0.0)
    table, ln = torch.arange(n, dtype=torch.int32, device="cuda")[:, None].contiguous(), torch.ones(n, dtype=torch.int32, device="cuda")
    q = (torch.randn((n, 8, DIM), generator=g, device="cuda") * 2.0 ** power).to(dt)
    out = layer.attend(q, table, ln, DIM ** -0.5, out=torch.empty((n, 8, DIM), device="cuda"))
    want = ref.rows(layer.tensors[2][:, :, 0], layer.tensors[3][:, :, 0], bits).repeat_interleave(4, 1)
    assert float(((out.double() - want).norm(dim=-1) / want.norm(dim=-1)).max()) <= 2.0 ** -10
