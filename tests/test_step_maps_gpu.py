"""A step's maps made on the GPU against the same made by hand: whole numbers, so equal or wrong."""

import pytest
import torch

from tests import plain_q8 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def ops():
    from turingserve_b200 import kernels
    kernels.use(None)
    return kernels.ops()


def run(ops, requests, updates, tables, page, T, W):
    dev = [torch.tensor(x, dtype=torch.int32, device=DEV).contiguous() for x in (requests, updates or torch.empty((0, 4)).tolist())]
    if not updates:
        dev[1] = torch.empty((0, 4), dtype=torch.int32, device=DEV)
    B, G = len(requests[0]), tables.shape[0]
    on = tables.clone().to(DEV)
    new = lambda *s: torch.full(s, -77, dtype=torch.int32, device=DEV)  # noqa: E731
    out = [new(B + 1), new(B), new(T), new(T), new(G, T), new(G, B, W)]
    ops.step_maps(dev[0], dev[1], on, page, *out)
    want = plain.maps(dev[0].cpu(), dev[1].cpu(), tables, page, T, W)
    for got, w in zip([*out, on], want):
        assert torch.equal(got.cpu(), torch.as_tensor(w, dtype=torch.int32).view(got.shape))
    return out, on


def tables_of(G, R, P, seed=0):
    return torch.randint(1, 1 << 20, (G, R, P), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)


@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("B", [1, 8, 129, 300])
def test_single_tokens(ops, B, page):
    g = torch.Generator().manual_seed(B + page)
    rows = torch.randperm(B + 3, generator=g)[:B].tolist()
    start = torch.randint(0, 40 * page, (B,), generator=g).tolist()
    run(ops, [rows, start, [1] * B], [], tables_of(1, B + 3, 41, B), page, B, 41)


def test_portions_padding_and_updates(ops):
    tables = tables_of(2, 9, 50)
    requests = [[3, 0, -1, -1, 8, 5], [63, 0, 0, 0, 17, 100], [1, 1, 1, 1, 640, 33]]
    updates = [[0, 3, 4, 9], [1, 3, 4, 8], [0, 8, 2, 77], [1, 8, 40, 5], [0, 1, 0, 3], [1, 7, 49, 2]]      # rows out of the step among them
    out, on = run(ops, requests, updates, tables, 16, 677, 50)
    assert out[4][0, 1].item() == int(on[0, 0, 0]) * 16 and out[4][:, 2:4].eq(-1).all()


def test_a_later_update_of_the_same_place_holds(ops):
    updates = [[0, 1, 2, 10], [0, 1, 2, 11], [0, 0, 0, 4], [0, 1, 2, 12], [0, 0, 0, 5]]
    _, on = run(ops, [[1], [20], [20]], updates, tables_of(1, 3, 8), 8, 20, 8)
    assert on[0, 1, 2].item() == 12 and on[0, 0, 0].item() == 5


@pytest.mark.parametrize("n", [40, 513, 1300])
def test_updates_in_any_order(ops, n):
    """Many updates, places twice and more among them, a row's far from each other, rows in the step and not; more than a block holds at once."""
    g = torch.Generator().manual_seed(n)
    updates = torch.stack([torch.randint(0, 2, (n,), generator=g), torch.randint(0, 6, (n,), generator=g), torch.randint(0, 50, (n,), generator=g),
                           torch.randint(1, 9999, (n,), generator=g)], 1)
    run(ops, [[4, 1, -1], [300, 17, 0], [90, 1, 1]], updates.tolist(), tables_of(2, 6, 50), 8, 92, 50)
    ascending = sorted(updates.tolist(), key=lambda u: (u[1], u[0], u[2]))
    run(ops, [[4, 1, -1], [300, 17, 0], [90, 1, 1]], ascending, tables_of(2, 6, 50), 8, 92, 50)


def test_narrow_and_wide_block_tables(ops):
    for W in (1, 3, 8, 20):
        run(ops, [[1, 0], [20, 0], [12, 5]], [], tables_of(3, 2, 8), 8, 17, W)


def test_lengths_of_zero(ops):
    run(ops, [[1, 0, 2], [5, 0, 3], [0, 4, 0]], [[0, 0, 0, 6]], tables_of(1, 3, 4), 4, 4, 4)


def test_captured_and_replayed(ops):
    """A replay takes what its arrays hold then."""
    tables = tables_of(1, 5, 30).to(DEV)
    start = tables.clone()
    req = torch.tensor([[2, 4], [15, 7], [1, 1]], dtype=torch.int32, device=DEV)
    upd = torch.tensor([[0, 2, 0, 3]], dtype=torch.int32, device=DEV)
    new = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    out = [new(3), new(2), new(2), new(2), new(1, 2), new(1, 2, 30)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.step_maps(req, upd, tables, 16, *out)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.step_maps(req, upd, tables, 16, *out)
    for i in range(3):
        req[1] += 9
        upd[0, 2:] = torch.tensor([i + 1, 100 + i], dtype=torch.int32)
        tables.copy_(start)
        g.replay()
        want = plain.maps(req.cpu(), upd.cpu(), start, 16, 2, 30)
        for got, w in zip([*out, tables], want):
            assert torch.equal(got.cpu(), torch.as_tensor(w, dtype=torch.int32).view(got.shape))


def test_a_builders_steps_are_the_same_from_the_gpu_and_from_the_host():
    """Requests that come, grow, are thrown out and come back on other slots; a full group, a window, a window that keeps first tokens;
    eager steps, and steps padded into an arena of their own; more new pages at once than the arena brings."""
    import random

    from turingserve_b200 import kernels
    from turingserve_b200.cache import CacheManager, RunNeeds
    from turingserve_b200.engine.batch import StepEntry, StepInputBuilder
    from turingserve_b200.parts.base import CacheNeed

    kernels.use(None)
    rng = random.Random(3)
    page, width = 8, 40
    needs = [RunNeeds(CacheNeed(1, 8), None), RunNeeds(CacheNeed(1, 8, 20), None), RunNeeds(CacheNeed(1, 8, 17, keep_first=9), None)]
    cache = CacheManager(needs, page, 400, 6, torch.bfloat16, "cuda")
    on, off = (StepInputBuilder(cache, 90, 7, width, "cuda") for _ in range(2))
    off.tables, on.device_map_rows = None, 1
    assert on.tables is not None
    arenas = [torch.zeros(b.capacity, dtype=torch.int32, device="cuda") for b in (on, off)]
    live = []

    def compare(entries, **kw):
        steps = [b.build(entries, arena=a if kw else None, **kw) for b, a in zip((on, off), arenas)]
        x, y = steps
        for name in ("input_ids", "positions", "token_request", "q_start", "seq_lens", "state_slots", "sample_rows", "feedback_rows",
                     "feedback_src"):
            assert torch.equal(getattr(x, name), getattr(y, name)), name
        for name in ("num_tokens", "num_requests", "num_decode", "q_lens", "starts", "max_q_len", "max_seq_len", "streaming_decode"):
            assert getattr(x, name) == getattr(y, name), name
        assert (x.host_ids is None) == (y.host_ids is None) and (x.host_ids is None or (x.host_ids == y.host_ids).all())
        for a, b in zip(x.groups, y.groups):
            assert torch.equal(a.block_tables, b.block_tables) and torch.equal(a.slot_mapping, b.slot_mapping)
            assert a.table_width == b.table_width and a.block_tables.is_contiguous() and a.slot_mapping.is_contiguous()

    for turn in range(120):
        on.device_map_rows = rng.choice([1, 1, 1, 4])               # (steps that the host lays out leave the GPU's tables behind)
        while len(live) < 6 and rng.random() < 0.7:
            live.append(cache.admit(f"r{turn}-{len(live)}"))
        entries = []
        for rc in rng.sample(live, rng.randint(1, len(live))) if live else []:
            n = 1 if rng.random() < 0.7 else rng.randint(2, 14)
            if rc.num_tokens + n > page * width:
                continue
            entries.append(StepEntry(rc, [rng.randint(0, 99) for _ in range(n)], [n - 1] if rng.random() < 0.8 else [],
                                     feedback=rng.randint(0, 5) if n == 1 and rng.random() < 0.3 else None))
        if not entries:
            continue
        for e in entries:
            cache.grow(e.cache, len(e.tokens))
        if rng.random() < 0.3:
            on.max_updates = 0 if rng.random() < 0.5 else on.max_updates
        compare(entries)
        if sum(len(e.tokens) == 1 for e in entries) + 1 <= 7 - sum(len(e.tokens) != 1 for e in entries):
            on.device_map_rows = 1
            compare(entries, fixed_width=width, pad_requests=7 - len(entries))
        for e in entries:
            cache.advance(e.cache, len(e.tokens))
        for rc in list(live):
            if rng.random() < 0.08 or rc.num_tokens > page * width - 20:
                live.remove(rc)
                cache.release(rc)
    cache.check()
