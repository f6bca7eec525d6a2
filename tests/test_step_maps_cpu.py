"""Which steps take their maps from the GPU's page tables, without a GPU."""

import pytest
import torch

from turingserve_b200.cache import CacheManager, RunNeeds
from turingserve_b200.engine.batch import StepEntry, StepInputBuilder
from turingserve_b200.parts.base import CacheNeed


def builder_and_steps(lengths, max_pages, page=4):
    cache = CacheManager([RunNeeds(CacheNeed(1, 8), None)], page, 200, 16, torch.float32, "cpu")
    b = StepInputBuilder(cache, 64, 16, max_pages, "cpu")
    b.tables = torch.zeros((1, 16, max_pages), dtype=torch.int32)       # as a builder on a GPU has them
    entries = []
    for i, n in enumerate(lengths):
        rc = cache.admit(str(i))
        cache.grow(rc, n)
        cache.advance(rc, n)
        cache.grow(rc, 1)
        entries.append(StepEntry(rc, [1], [0]))
    return cache, b, entries


class FromTheGpu(Exception):
    pass


@pytest.mark.parametrize("longest,on_gpu", [(31, True), (32, False), (60, False)])
def test_a_request_of_more_pages_than_the_tables_have_columns(monkeypatch, longest, on_gpu):
    """Sixteen requests, one of which has ``longest`` tokens before its new one; tables of 8 pages of 4."""
    _, b, entries = builder_and_steps([5] * 15 + [longest], 8)

    def refuse(*a, **kw):
        raise FromTheGpu
    monkeypatch.setattr(b, "_build_on_device", refuse)
    if on_gpu:
        with pytest.raises(FromTheGpu):
            b.build(entries)
        return
    step = b.build(entries)
    table = entries[-1].cache.tables[0]
    assert step.groups[0].slot_mapping[-1] == table[longest // 4] * 4 + longest % 4
    assert step.groups[0].block_tables[-1].tolist() == table


@pytest.mark.parametrize("rows,on_gpu", [(1, False), (4, False), (5, False), (6, True), (16, True)])
def test_steps_of_few_rows_come_from_the_host(monkeypatch, rows, on_gpu):
    """(a step of one to four requests is no faster with its maps from the GPU; padding rows count)"""
    _, b, entries = builder_and_steps([5] * max(1, rows - 2), 8)
    took = []
    monkeypatch.setattr(b, "_build_on_device", lambda *a, **kw: took.append(True))
    b.build(entries, pad_requests=rows - len(entries))
    assert bool(took) == on_gpu
