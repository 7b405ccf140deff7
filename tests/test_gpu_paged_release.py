"""Release of requests that share pages: each page goes back once, when nobody holds it any more."""
import numpy as np
import pytest
import torch

import turboquant_b200 as tq

pytestmark = pytest.mark.gpu
I32 = dict(dtype=torch.int32, device="cuda")


def model(mask, seq, table, free, left, room, page):
    """(seq, table, free list, status) by plain loops."""
    used = [-(-s // page) for s in seq]
    kept = {p for r, m in enumerate(mask) if not m for p in table[r][: used[r]] if p >= 0}
    back = []
    for r, m in enumerate(mask):
        for p in table[r][: used[r]] if m else []:
            if p >= 0 and p not in kept:
                kept.add(p)
                back.append(p)
    if left + len(back) > room:
        return seq, table, free[:left], 1
    table = [[-1] * used[r] + row[used[r]:] if mask[r] else row for r, row in enumerate(table)]
    return [0 if m else s for m, s in zip(mask, seq)], table, free[:left] + back, 0


def check(mask, seq, table, free, left, page, room=None):
    t, s = torch.tensor(table, **I32), torch.tensor(seq, **I32)
    f = torch.full((room if room is not None else left + t.numel() + 1,), -9, **I32)
    f[:left] = torch.tensor(free[:left], **I32)
    state = torch.tensor([left, 0, 0, 0], **I32)
    tq.paged_release(torch.tensor(mask, device="cuda"), s, t, f, state, page)
    seq, table, free, status = model(mask, seq, table, free, left, f.numel(), page)
    assert state.tolist() == [len(free), 0, status, 0]
    assert s.tolist() == seq and t.tolist() == table and f[: len(free)].tolist() == free
    assert bool((f[len(free):] == -9).all())
    return s, t, f, state


def test_pages_of_two_ended_requests_are_handed_out_once():
    s, t, f, state = check([True, True, False], [32, 32, 0], [[3, 4, -1, -1], [3, 5, -1, -1], [-1] * 4], [0, 1, 2], 3, 16)
    assert f[:6].tolist() == [0, 1, 2, 3, 4, 5]
    step = tq.paged_plan(s, torch.tensor([32, 60, 0], **I32), t, f, state, 16, 92)
    step.check()
    assert len(set(step.slots.tolist())) == 92 and int(step.state[0]) == 0


def test_a_page_stays_with_the_request_that_goes_on():
    s, t, f, state = check([True, False, False], [40, 33, 16], [[3, 4, 5], [3, 4, 6], [5, -1, -1]], [0], 1, 16)
    assert int(state[0]) == 1
    s, t, f, state = check([False, True, False], s.tolist(), t.tolist(), f.tolist(), 1, 16)
    assert f[:4].tolist() == [0, 3, 4, 6]   # page 5 is the third request's
    check([True] * 3, s.tolist(), t.tolist(), f.tolist(), 4, 16)


def test_entries_behind_a_length_hold_nothing_and_holes_are_no_pages():
    check([True, False], [20, 16], [[7, 8, 9], [1, 7, 8]], [], 0, 16)
    check([True, False], [48, 48], [[-1, 8, -7], [-1, -1, 2]], [4], 1, 16)
    check([True, True], [48, 48], [[2, 2, 2], [-3, 2, 6]], [4], 1, 16)
    check([True, False], [0, 0], [[-1], [-1]], [4], 1, 16)
    check([False, False], [9, 9], [[1], [2]], [4], 1, 16)


@pytest.mark.parametrize("room,fits", [(7, True), (6, False)])
def test_room_is_needed_for_what_goes_back_only(room, fits):
    table = [[3, 4, 5, 6], [3, 4, 5, 7], [6, 8, -1, -1]]
    s, t, f, state = check([True, True, False], [64, 64, 32], table, [0, 1, 2], 3, 16, room)
    assert (t.tolist() != table) == fits and int(state[2]) == (0 if fits else 1)


@pytest.mark.parametrize("requests,blocks,ids,page,seed", [(3, 2000, 2500, 16, 0), (64, 40, 900, 64, 1), (1500, 9, 6000, 32, 2), (4096, 3, 5000, 128, 3),
                                                           (9, 700, 2 ** 31, 16, 4), (40, 90, 1 << 22, 1024, 5)])
def test_random_sharing(requests, blocks, ids, page, seed):
    """Common beginnings, pages that stand twice in a row, holes, page numbers far apart."""
    g = np.random.default_rng(seed)
    pool = g.integers(0, ids, size=requests * blocks // 2 + 1, dtype=np.int64)
    pool[0], pool[-1] = ids - 1, 0
    table = pool[g.integers(0, len(pool), (requests, blocks))]
    table[: requests // 2, : blocks // 2] = table[0, : blocks // 2]
    table[g.random((requests, blocks)) < 0.02] = -1
    seq = [int(x) for x in g.integers(0, blocks * page + 1, requests)]
    for share in (0.1, 0.5, 1.0):
        mask = [bool(x) for x in g.random(requests) < share]
        s, t, f, state = check(mask, seq, table.tolist(), [5, 6], 2, page)
        rest, left = [not m for m in mask], int(state[0])
        check(rest, s.tolist(), t.tolist(), f.tolist(), left, page, room=left + table.size + 1)


def test_cache_whose_requests_share_a_beginning():
    """A prompt stored once and read by three requests: rows of those that go on stay as they are through releases and plans."""
    g = torch.Generator(device="cuda").manual_seed(6)
    cache = tq.PagedPqoCache(tq.CacheConfig(4, 64, 2, 1), 12, 16, 3)
    k = torch.randn((48, 2, 64), generator=g, device="cuda")
    cache.append(0, k, k, cache.plan(torch.tensor([48, 0, 0], **I32), 48))
    cache.block_table[1, :2], cache.block_table[2, :3] = cache.block_table[0, :2], cache.block_table[0, :3]
    cache.seq_lens.copy_(torch.tensor([48, 32, 48], **I32))
    rows = lambda r, n: cache.dequantize(0, cache.block_table[r].long()[torch.arange(n, device="cuda") // 16] * 16 + torch.arange(n, device="cuda") % 16)  # noqa: E731
    want = [t.clone() for t in rows(0, 48)]
    for ended in ([True, False, False], [False, False, True]):
        cache.release(torch.tensor(ended, device="cuda"))
        new = torch.tensor([20 if e else 0 for e in ended], **I32)
        step = cache.plan(new, 20)
        step.check()
        other = torch.randn((20, 2, 64), generator=g, device="cuda")
        cache.append(0, other, other, step)
        for a, b in zip(rows(1, 32), want):
            assert torch.equal(a, b[:32])
    cache.release(torch.ones(3, dtype=torch.bool, device="cuda"))
    assert int(cache.state[0]) == 12 and sorted(cache.free_pages.tolist()) == list(range(12))
