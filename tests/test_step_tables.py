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


@pytest.mark.parametrize('rows', [1, 2, 3, 5])
def test_tables_of_fewer_rows_than_requests(pkg, monkeypatch, rows):
    """The kernels index a table by a token's request and do not know how many rows it has; padding counts as the last request."""
    layer = pkg.s6_layer
    monkeypatch.setattr(layer._lib, 'call', lambda *a: None)
    monkeypatch.setattr(layer._lib, 'stream', lambda *a: 0)
    i32 = lambda *a: torch.tensor(a, dtype=torch.int32)
    ctx = layer.StepContext(torch.tensor([5, 33, 0, 8, 0, 0]), i32(0, 1, 2, 4, 4), i32(6, 34, 9, 0), 2, 6, {}, 1.0, None)
    ctx.token_requests, ctx.valid = torch.tensor([0, 1, 2, 2, 3, 3]), torch.tensor([1, 1, 1, 1, 0, 0]).bool()
    table = torch.arange(100, 100 + 3 * rows, dtype=torch.int32).view(rows, 3)

    def call(name, bt, *args):
        if name == 'hla_s6_slot_mapping':
            stride, cols, requests, valid, pos, T, block, slots, _ = args
            for t in range(T):
                assert not valid[t] or requests[t] < rows, (t, int(requests[t]))
                slots[t] = bt[requests[t], pos[t] // block] * block + pos[t] % block if valid[t] else -1
        else:
            stride, rows_, cols, requests, T, out, _, _ = args
            assert (requests < rows_).all()
            out.copy_(bt[requests])

    monkeypatch.setattr(layer._lib, 'ptr', lambda t: t)
    monkeypatch.setattr(layer._lib, 'call', call)
    want = [100 * 16 + 5, (103 + 2) * 16 + 1, 106 * 16, 106 * 16 + 8, -1, -1]
    assert ctx.slots(table, 16).tolist() == [w if r < rows else -1 for w, r in zip(want, (0, 1, 2, 2, 3, 3))]
    gathered = ctx.block_table(table)
    assert gathered.shape == (6, 3) and torch.equal(gathered[0], table[0])
