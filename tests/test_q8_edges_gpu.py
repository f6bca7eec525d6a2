"""The 8-bit cache's operators where a block, a warp or a call has nothing of its own to do, and what else the widest use of them meets."""

import math

import pytest
import torch

from tests.test_q8_cache_gpu import BF16, Attend, Write, forced, ops  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("splits", [0, 2, 4, 8])
@pytest.mark.parametrize("H,KVH,D", [(12, 2, 128), (14, 2, 64), (5, 5, 128)])
def test_queries_of_nan_beside_shares_without_keys(ops, forced, H, KVH, D, splits):  # noqa: F811
    """Short prompts beside a long context, keys cut over 2, 4 and 8 blocks (0: by the rule, which goes by the longest): most blocks of a short
    prompt's row tiles have no keys.  Queries with NaN in every odd column, in the last rows of a tile and in its first: their own rows are NaN,
    every other row has the bits that it has beside clean queries."""
    a = Attend([40, 130, 17, 1, 64, 33], [40, 130, 17, 1, 4000, 33], H, KVH, D, 16)
    a.step.num_decode = 0
    G, odd = H // KVH, torch.zeros(a.q.shape[0], H, dtype=torch.bool, device=a.q.device)
    start = 0
    for n in a.q_lens:
        for row in range(n * G):                                   # (a row tile is 128 (token, head-in-group) pairs)
            if row % 128 >= 120 or row % 128 < 3:
                odd[start + row // G, row % G] = True
        start += n
    forced(row_tiles=1 if splits else 0, portion_splits=splits)
    clean = a.run(ops).clone().view(a.q.shape)
    a.check()
    q = a.q.clone()
    a.q[..., 1::2][odd] = math.nan
    for _ in range(20):
        a.out.fill_(7.0)
        got = a.run(ops).view(a.q.shape)
        assert got[odd].isnan().all()
        assert torch.equal(got[~odd], clean[~odd])
    a.q = q
    assert torch.equal(a.run(ops).view(a.q.shape), clean)


@pytest.mark.parametrize("slot", [-2, -3, -(1 << 31)])
@pytest.mark.parametrize("case", [([200], [5], 4, 2, 64, 64, 256, BF16), ([1300], [7], 4, 2, 128, 128, 256, BF16), ([1, 5], [9, 3], 4, 2, 64, 64, 16, BF16),
                                  ([40, 9], [5, 0], 3, 1, 80, 80, 64, BF16)], ids=lambda c: f"{len(c[0])}x{max(c[0])}-{c[4]}")
def test_any_negative_slot_is_a_token_that_is_not_written(ops, case, slot):  # noqa: F811
    """Tokens without a place in the middle of pages, at the edges of spans of 1, 16 and 64 tokens among them: the page's other rows are one
    run all the same, with one scale."""
    w = Write(*case)
    for t in (1, 2, 14, 15, 16, 31, 47, 48, 63, 64, 100, 127, 128, 191, 640, 895):
        if t < w.slots.shape[0] - 1:
            w.slots[t] = slot
    w.run(ops)
    w.check()


@pytest.mark.parametrize("n", [0, 3, 600])
def test_maps_of_a_step_without_requests(ops, n):  # noqa: F811
    """The page tables take what is to go into them, the query starts begin at 0, tokens that no request brings have no place."""
    i32 = torch.int32
    tables = torch.randint(1, 999, (2, 5, 9), dtype=i32, device="cuda")
    g = torch.Generator().manual_seed(n)
    updates = torch.stack([torch.randint(0, m, (n,), generator=g) for m in (2, 5, 9, 5000)], 1).int()
    want = tables.clone().cpu()
    for a, b, c, p in updates.tolist():
        want[a, b, c] = p
    new = lambda *s: torch.full(s, -77, dtype=i32, device="cuda")  # noqa: E731
    out = [new(1), new(0), new(4), new(4), new(2, 4), new(2, 0, 9)]
    ops.step_maps(new(3, 0), updates.cuda(), tables, 16, *out)
    assert torch.equal(tables.cpu(), want)
    assert out[0].tolist() == [0] and not out[2].any() and not out[3].any() and out[4].eq(-1).all()


def test_clusters_switched_off_after_the_first_call(ops):  # noqa: F811
    a = Attend([1] * 8, [2048 - 37 * i for i in range(8)], 12, 2, 128, 64)
    launches = []
    try:
        for on in (1, 0, 1):
            ops.lib.ts_set_clusters(on)
            before = ops.launches
            a.out.fill_(7.0)
            a.run(ops)
            a.check()
            launches.append(ops.launches - before)
    finally:
        ops.lib.ts_set_clusters(1)
    assert launches == [1, 2, 1]
