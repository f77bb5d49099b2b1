"""CPU checks of whole exact caches and of pools of pages: the plain pool by hand, how rows are cut, refusals before any launch."""
import copy

import numpy as np
import pytest
import torch

from pool_ref import Pool


@pytest.fixture(scope='module')
def ec(pkg):
    return pkg.exact_cache


@pytest.fixture(scope='module')
def pg(pkg):
    return pkg.pages


def test_a_pool_by_hand():
    p = Pool.empty(10, 4, 4, 3, reserved=1)
    assert p.extend([5, 0, 0, 0]) == ([True] * 4, [{}] * 4) and p.tables[0] == [1, 2, -1]
    assert p.fork([0, 0, 1, 2], [1, 1, 2, 3]) == [True, False, False, False]       # twice; a parent among the children
    assert p.fork([0], [2]) == [True] and p.refs[:4] == [1, 3, 3, 0] and p.lengths == [5, 5, 5, 0]
    ok, pairs = p.extend([6, 9, 5, 0])
    assert ok == [True] * 4 and pairs == [{1: (2, 3)}, {1: (2, 4)}, {}, {}]
    assert p.tables[:3] == [[1, 3, -1], [1, 4, 5], [1, 2, -1]] and p.refs == [1, 3, 1, 1, 1, 1, 0, 0, 0, 0]
    p.check(1)
    assert p.extend([6, 9, 13, 12]) [0] == [True, True, False, True] and p.tables[3] == [6, 7, 8]   # 13 rows fit no table
    p.release([1, 3, 7, 1], [9, 1, 0, 4])
    assert p.tables[1] == [1, -1, -1] and p.lengths == [6, 4, 5, 1] and p.tables[3] == [6, -1, -1]
    p.check(1)
    ok, pairs = p.extend([6, 4, 5, 1], [0, 0, 0, 0])
    assert ok == [True] * 4 and pairs == [{0: (1, 4)}, {0: (1, 5)}, {0: (1, 7)}, {}] and p.refs[1] == 0
    p.check(1)
    assert p.compact() == ([7], [1]) and p.tables[2] == [1, 2, -1]
    p.check(1)


def test_requests_wait_in_order():
    p = Pool.empty(5, 4, 4, 3)
    ok, _ = p.extend([8, 12, 0, 4])
    assert ok == [True, True, True, False] and p.tables[3] == [-1] * 3    # two, three, none, and none are left
    p = Pool.empty(4, 4, 4, 3)
    ok, _ = p.extend([8, 12, 0, 4])
    assert ok == [True, False, True, False] and p.lengths == [8, 0, 0, 0]   # the last one does not overtake


def test_new_pools(pg):
    for pages, reserved in ((0, 0), (1, 0), (31, 1), (32, 0), (33, 33), (70, 40)):
        p = pg.new_pool(pages, 16, 3, 33, 'cpu', reserved)
        want = Pool.empty(pages, 16, 3, 3, reserved)
        assert p.tables.tolist() == want.tables and p.refs.tolist() == want.refs and p.lengths.tolist() == [0] * 3
        assert p.free.dtype == torch.int32 and (p.free.numpy() == want.words()).all() and p.block == 16
    for args in ((4, 0, 1, 1), (4, 16, -1, 1), (4, 16, 8193, 1), (4, 16, 1, -1)):
        with pytest.raises(ValueError, match='no pool'):
            pg.new_pool(*args, 'cpu')
    with pytest.raises(ValueError, match='no pool'):
        pg.new_pool(4, 16, 1, 1, 'cpu', reserved=5)


def test_a_pool_keeps_its_tensors(pg):
    """Operators hold the addresses: a tensor of a pool is not exchanged, and a copy of a pool has tensors of its own."""
    pool = pg.new_pool(5, 4, 2, 12, 'cpu')
    with pytest.raises(AttributeError, match='written into'):
        pool.lengths = torch.zeros(2, dtype=torch.int32)
    other = copy.deepcopy(pool)
    other.lengths[0] = 3
    assert pool.lengths.tolist() == [0, 0] and other._args[4] == other.lengths.data_ptr() != pool.lengths.data_ptr()


def test_how_rows_are_cut(ec):
    """Two workgroups per CU between the KV heads; a workgroup per group for short rows and for very many groups."""
    assert ec.row_shares(8160, 16, 16, 256) == 32 and ec.row_shares(131000, 16, 8, 256) == 64
    assert ec.row_shares(4096, 1024, 16, 256) == 32 and ec.row_shares(10 ** 6, 1, 1, 256) == 512
    assert ec.row_shares(131000, 10 ** 6, 8, 256) == 0 and ec.row_shares(1024, 4, 4, 256) == 0 and ec.row_shares(0, 4, 4, 256) == 0
    assert ec.row_shares(1025, 4, 4, 256) == 128 and ec.row_shares(1536, 128, 8, 256) == 0 and ec.row_shares(1537, 128, 8, 256) == 64
    assert ec.row_shares(4096, 3000, 3000, 256) == 1


def test_which_steps_are_grouped(ec):
    """A group of tokens for every CU, eight heads at most; a workgroup per token of a group where requests are short."""
    assert ec._turns(2048, 1, 16, 256, 512) == 4 and ec._turns(2048, 4, 8, 256, 512) == 4 and ec._turns(2048, 8, 8, 256, 512) == 2
    assert ec._turns(256, 1, 16, 256, 8) == 16 and ec._turns(255, 1, 16, 256, 8) == 16 and ec._turns(240, 1, 16, 256, 8) == 0
    assert ec._turns(10 ** 5, 9, 16, 256, 512) == 0 and ec._turns(0, 1, 16, 256, 0) == 0 and ec._turns(300, 5, 8, 256, 8) == 3


def test_host_tensors_are_refused(ec, pg):
    i32, rows, cache = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, 64, dtype=torch.bfloat16), \
        torch.zeros(2, 2, 16, 128, dtype=torch.bfloat16)
    pool = pg.new_pool(4, 16, 1, 32, 'cpu')
    for call in (lambda: ec.store_rows(rows, rows, i32.long(), cache), lambda: ec.attention(rows, cache, i32[None], i32, 1.0, 16),
                 lambda: pg.release_requests(pool, i32), lambda: pg.fork_requests(pool, i32, i32),
                 lambda: pg.extend_requests(pool, i32), lambda: pg.compact_pages(pool), lambda: pg.copy_pages(cache, i32, i32)):
        with pytest.raises(RuntimeError, match='GPU only'):
            call()


def test_entry_points_check_before_they_launch(pkg):
    lib = pkg._lib

    def call(name, at):
        args = [None if t is lib.P else 0 for t in lib.SIGNATURES[name]]
        for i, v in at.items():
            args[i] = v
        lib.call(name, *args)

    def refused(name, good, changes, error=ValueError):
        for change, match in changes:
            with pytest.raises(error, match=match):
                call(name, {**good, **change})

    attention = {0: 16, 1: 1, 2: 8, 3: 64, 4: 512, 5: 64, 6: 16, 8: 2, 9: 4096, 10: 128, 11: 256, 12: 16, 13: 2, 14: 16, 15: 1, 16: 1,
                 17: 1, 19: 16, 28: 16, 29: 512, 30: 64, 31: 16}
    refused('hla_s6_exact_attention', attention, [
        ({1: -1}, 'token count'), ({3: 96}, 'head dim'), ({8: 0}, 'KV heads'), ({8: 3}, '8 query heads over 3'), ({2: 1}, 'query heads'),
        ({12: 0}, 'block size'), ({13: 0}, 'page count'), ({6: 8}, 'aligned'), ({9: 4097}, 'multiples of 16'), ({11: 255}, 'multiples of 16'),
        ({10: 64}, 'overlap'), ({11: 64}, 'overlap'), ({24: -1}, 'shares'), ({24: 1025}, 'shares'), ({20: -1}, 'window'),
        ({22: 16}, 'scales'), ({23: 16}, 'scales'), ({17: 0}, 'table rows'), ({0: None}, 'null pointer'), ({14: None}, 'null pointer'),
        ({19: None}, 'null pointer'), ({28: None}, 'null pointer'), ({31: None}, 'null pointer'), ({4: 4}, 'aligned'), ({0: 8}, 'aligned'),
        ({30: 4}, 'aligned'), ({1: 2 ** 30, 17: 2 ** 30}, 'too many rows'), ({24: 2, 26: 8, 27: 10 ** 6}, 'aligned'),
        ({24: 2, 25: 1, 26: 16, 27: 10 ** 6}, 'groups of tokens'), ({25: 1, 2: 18}, 'groups of tokens'), ({25: 17}, 'groups of tokens'),
        ({25: -1}, 'groups of tokens')])
    refused('hla_s6_exact_attention', attention, [({24: 2, 26: 16, 27: 10}, 'workspace'), ({24: 2, 27: 10 ** 6}, 'workspace')], RuntimeError)
    call('hla_s6_exact_attention', {**attention, 1: 0, 0: None})      # no tokens, nothing to do
    store = {0: 16, 1: 128, 2: 64, 3: 16, 4: 128, 5: 64, 6: 1, 7: 2, 8: 64, 9: 16, 12: 16, 14: 4096, 15: 128, 16: 256, 17: 16, 18: 2}
    refused('hla_s6_exact_store', store, [
        ({6: -1}, 'token count'), ({8: 32}, 'head dim'), ({0: None}, 'null pointer'), ({9: None}, 'null pointer'), ({1: 132}, 'aligned'),
        ({3: 24}, 'aligned'), ({10: 16}, 'scales'), ({12: 4}, 'aligned'), ({15: 64}, 'overlap')])
    pool = {0: 16, 1: 4, 2: 2, 3: 4, 4: 16, 5: 16, 6: 8, 7: 16, 8: 16}
    bad = [({2: -1}, 'request count'), ({2: 8193}, 'request count'), ({3: -1}, 'table width'), ({6: -1}, 'page count'),
           ({6: 2 ** 31}, 'page count'), ({8: 0}, 'block size'), ({4: None}, 'null lengths'), ({0: None}, 'null tables'),
           ({5: None}, 'null page state'), ({7: None}, 'null page state'), ({1: 3}, 'overlap')]
    refused('hla_s6_pool_release', {**pool, 9: 16, 11: 1}, bad + [({11: -1}, 'list'), ({9: None}, 'list')])
    refused('hla_s6_pool_fork', {**pool, 9: 16, 10: 16, 11: 1, 12: 16}, bad + [
        ({11: -1}, 'lists'), ({11: 8193}, 'lists'), ({9: None}, 'lists'), ({10: None}, 'lists'), ({12: None}, 'lists')])
    refused('hla_s6_pool_extend', {**pool, 9: 16, 11: 16, 12: 16, 13: 16}, bad + [
        ({9: None}, 'null pointer'), ({11: None}, 'null pointer'), ({12: None}, 'null pointer'), ({10: 16}, 'null pointer'),
        ({10: 16, 14: 16, 1: 2 ** 30, 3: 2 ** 30}, 'too many table entries')])
    refused('hla_s6_pool_compact', {**pool, 9: 16, 10: 16, 11: 16}, bad + [({9: None}, 'null pointer'), ({11: None}, 'null pointer')])
    refused('hla_s6_copy_pages', {0: 16, 1: 1, 2: 64, 3: 64, 4: 4, 5: 16, 6: 16, 7: 1}, [
        ({1: -1}, 'negative'), ({4: -1}, 'negative'), ({7: -1}, 'negative'), ({2: 60}, 'overlap'), ({0: None}, 'null pointer'),
        ({5: None}, 'null pointer'), ({3: 2 ** 46, 2: 2 ** 46}, 'too long')])
