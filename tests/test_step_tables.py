"""CPU checks of what a StepContext keeps about the block tables of a step."""
import gc
import weakref

import pytest
import torch


@pytest.fixture
def ctx(pkg, monkeypatch):
    """A StepContext without a GPU, whose slots are copies of the table that they were made for."""
    layer = pkg.s6_layer
    monkeypatch.setattr(layer._lib, 'call', lambda *a: None)
    monkeypatch.setattr(layer._lib, 'stream', lambda *a: 0)
    monkeypatch.setattr(layer, 'slot_mapping', lambda ctx, table, block: (table.clone(), block))
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32)
    return layer.StepContext(torch.tensor([5, 9]), i32(0, 1, 2), i32(6, 10), 1, 2, {}, 1.0, None)


def test_tables_at_one_address_are_told_apart(ctx):
    table = torch.arange(24, dtype=torch.int32).view(4, 6)
    for view in (table, table[::2], table[:, :3], table[:2], table.as_strided((2, 6), (3, 1)), table):
        for block in (16, 32):
            slots, of = ctx.slots(view, block)
            assert torch.equal(slots, view) and of == block
            assert ctx.slots(view, block)[0] is slots            # once per step
    whole, narrow = ctx.block_table(table), ctx.block_table(table[:, :3])
    assert whole.shape == (2, 6) and narrow.shape == (2, 3) and ctx.block_table(table) is whole


def test_a_table_that_was_seen_keeps_its_place(ctx):
    """A gathered table that only the call knew must not make room for another one at the same address."""
    tables = [torch.full((2, 3), 7, dtype=torch.int32) for _ in range(2)]
    refs = [weakref.ref(t) for t in tables]
    ctx.slots(tables[0], 16)
    ctx.block_table(tables[1])
    del tables
    gc.collect()
    assert all(r() is not None for r in refs)
