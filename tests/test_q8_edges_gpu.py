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


# Long contexts.  Values of + and - the same size in the two halves of a context cancel, so that a block's or a warp's share of the keys that got
# lost, or counted twice, shows as 1 / 128 of them and more.  The bound charges a weight's rounding to a half float as it is: 2^-11 of it, or, where
# weight * scale lies below 2^-14 of the row's largest, 2^-25 of that largest (a reference below the largest rounds finer); the sums' by the
# longest chain of additions, a quarter of the keys (four warps a block) and the merges' 140 for single tokens, all of them for portions; scores and
# exponentials as in test_q8_cache_gpu.py.

def halves_that_cancel(a):
    """The requests' values: the same size, with the other sign in the second half of what is seen of each context, and some noise."""
    noise = torch.randn(a.v.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") * 20
    v = noise + 150
    for b, n in enumerate(a.lens):
        held = -(-n // a.page)
        first = max(0, n - a.window) // a.page if a.window else 0
        v[a.tables[b, (first + held) // 2:held].long()] -= 300
    a.v, a.vs = v.to(a.v.dtype), torch.full_like(a.vs, 2.0 ** -7)


def sharp(a, b, chain, leave_out=None):
    """(outputs of request ``b`` in 64 bits, what each may be off by); ``leave_out``: keys whose weights are dropped."""
    H, D = a.q.shape[1:]
    G, n, t = H // a.KVH, a.lens[b], sum(a.q_lens[:b])
    ids = a.tables[b, :-(-n // a.page)].long()
    outs, bounds = [], []
    j, pos = torch.arange(n, device="cuda"), torch.arange(n - a.q_lens[b], n, device="cuda")[:, None]
    seen = (j <= pos) & ((j > pos - a.window) if a.window else True)
    for h in range(H):
        k, v8 = ((x[ids, h // G].double()).flatten(0, 1)[:n] for x in (a.k, a.v))
        ks, vs = (s[ids, h // G].double().repeat_interleave(a.page)[:n] for s in (a.ks, a.vs))
        q = a.q[t:t + a.q_lens[b], h].double()
        s = (q @ (k * ks[:, None]).T * a.scale).masked_fill(~seen, -math.inf)
        w = torch.softmax(s, -1)
        if leave_out is not None:
            w[:, leave_out] = 0
            w = w / w.sum(-1, keepdim=True)
        x = w * vs
        top = x.amax(-1, keepdim=True)
        off = torch.where(x >= 2.0 ** -14 * top, 2.0 ** -11 * x, torch.where(seen, 2.0 ** -25 * top, torch.zeros_like(top)))
        size, want = x @ v8.abs(), x @ v8
        mags = (q.abs() @ (k.abs() * ks[:, None]).T * a.scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
        outs.append(want)
        bounds.append(2.0 ** -8 * want.abs() + (2 * (D + 4) * 2.0 ** -24 * mags + 2.0 ** -17 + chain * 2.0 ** -24) * size + off @ v8.abs())
    return torch.stack(outs, 1), torch.stack(bounds, 1)


@pytest.mark.parametrize("splits", [0, 1, 128])
@pytest.mark.parametrize("case", [([1], [30011], 12, 2, 128, 64, 0), ([1], [100003], 16, 2, 64, 16, 0), ([1] * 3, [8000, 20011, 33], 28, 4, 128, 16, 0),
                                  ([1], [50000], 12, 2, 128, 64, 16385)], ids=lambda c: f"{len(c[0])}x{max(c[1])}-{c[4]}-w{c[6]}")
def test_no_share_of_a_long_context_is_lost(ops, forced, case, splits):  # noqa: F811
    forced(splits=splits, clusters=False if splits > 8 else True)
    a = Attend(*case)
    halves_that_cancel(a)
    got = a.run(ops).double().view(a.q.shape)
    for b, n in enumerate(a.lens):
        chain = n / 4 + 140
        want, bound = sharp(a, b, chain)
        off = (got[b:b + 1] - want).abs()
        assert bool((off <= bound).all()), float((off / bound).max())
        if n < 1000:
            continue
        # what is lost without 1 / 128 of the keys that are seen is seen
        first = max(0, n - a.window) if a.window else 0
        lost, _ = sharp(a, b, chain, slice(first, first + (n - first) // 128))
        assert bool(((lost - want).abs() > bound).any(-1).all())


@pytest.mark.parametrize("row_tiles,splits", [(0, 0), (1, 1), (2, 1), (1, 2), (1, 4), (1, 8)])
@pytest.mark.parametrize("case", [([70], [16011], 12, 2, 128, 64, 0), ([1, 40, 90], [5, 9000, 4100], 14, 2, 64, 16, 0),
                                  ([64], [20000], 6, 2, 128, 16, 8200)], ids=lambda c: f"{len(c[0])}x{max(c[1])}-{c[4]}-w{c[6]}")
def test_no_share_of_a_portions_long_context_is_lost(ops, forced, case, row_tiles, splits):  # noqa: F811
    forced(row_tiles=row_tiles, portion_splits=splits)
    a = Attend(*case)
    halves_that_cancel(a)
    got = a.run(ops).double().view(a.q.shape)
    t = 0
    for b, n in enumerate(a.lens):
        want, bound = sharp(a, b, n)
        off = (got[t:t + a.q_lens[b]] - want).abs()
        assert bool((off <= bound).all()), float((off / bound).max())
        if n > 1000:
            first = max(0, n - a.window) if a.window else 0        # (a turn's 128 keys)
            lost, _ = sharp(a, b, n, slice(first + 1024, first + 1152))
            assert bool(((lost - want).abs() > bound).any(-1).all())
        t += a.q_lens[b]


@pytest.mark.parametrize("case", [([1] * 8, [2048 - 37 * i for i in range(8)], 12, 2, 128, 64, 0), ([1, 1, 130, 2], [99, 640, 463, 150], 28, 4, 128, 16, 0),
                                  ([90, 7], [1500, 20], 14, 2, 64, 32, 70)], ids=["singles", "mixed", "window"])
@pytest.mark.parametrize("splits,portion_splits", [(1, 1), (4, 2), (8, 8)])
def test_the_same_bits_whatever_the_longest_context_with_the_same_cuts(ops, forced, case, splits, portion_splits):  # noqa: F811
    """A captured step is launched for the longest context that the engine allows.  That may change how many blocks cut a request's keys, and so the
    order of the sums; nothing else."""
    forced(row_tiles=1, splits=splits, portion_splits=portion_splits)
    a, b = Attend(*case), Attend(*case, limit=40000)
    b.tables = torch.cat([b.tables, torch.zeros((b.tables.shape[0], 600), dtype=torch.int32, device="cuda")], 1).contiguous()
    assert torch.equal(a.run(ops), b.run(ops))
