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
