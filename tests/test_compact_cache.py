"""CPU checks of the compact cache: the plain restatement of its format, split counts, and refusals before any launch."""
import numpy as np
import pytest
import torch

import compact_ref as C


@pytest.fixture(scope='module')
def cc(pkg):
    return pkg.compact_cache


@pytest.mark.parametrize('w', [128, 256, 512, 1024])
def test_a_tile_has_a_place_for_every_byte(w):
    at = np.concatenate([np.concatenate(C.addresses(w, x)) for x in range(16)])
    assert sorted(at.tolist()) == list(range(17 * w))


def test_rounding_by_hand():
    row = np.zeros(32)
    row[:9] = [7, 0.25, 0.75, -2.5, 5, 3.5, -0.26, 1.75, 1.25]     # scale 1: 7 goes to 6
    code, scale = C.quantise(row[None])
    assert scale.tolist() == [[127]]
    assert C.values(code, scale)[0, :9].tolist() == [6, 0, 1, -2, 4, 4, -0.5, 2, 1]
    row[0] = 7.5                                                   # nearer to 8: scale 2
    code, scale = C.quantise(row[None])
    assert scale.tolist() == [[128]] and C.values(code, scale)[0, :5].tolist() == [8, 0, 1, -2, 4]
    row[0] = np.inf
    code, scale = C.quantise(row[None])
    assert scale.tolist() == [[255]] and np.isnan(C.values(code, scale)).all()


def test_stored_rows_come_back():
    rng = np.random.default_rng(0)
    cache = np.full((3, 2, 17 * 128), 255, np.uint8)
    rows = rng.standard_normal((40, 256))
    slots = rng.permutation(96)[:40]
    C.store(cache, rows[:, :128], rows[:, 128:], slots)
    got = C.load(cache, slots)
    # half of the widest gap (2 of 6) to either side of a value, in a block whose largest is at least 3.5 of its scale
    assert (np.abs(got - rows) <= np.repeat(np.abs(rows.reshape(40, 8, 32)).max(-1), 32, -1) / 3.5).all()


def test_selection_by_hand():
    w = np.array([[5, 1, 1, 7, 1, 9, 2, 0]], np.float32)
    pos = np.arange(8, dtype=np.int32)[None]
    left, ow, op, source, target = C.select(w, pos, [8], [4], [7])
    assert left.tolist() == [4] and op[0].tolist() == [0, 5, 7, 3, -1, -1, -1, -1]     # 0, 3, 5 by weight, 7 protected
    assert ow[0].tolist() == [5, 9, 0, 7, 0, 0, 0, 0]
    assert source[0].tolist() == [5, 7, -1, -1] and target[0].tolist() == [1, 2, -1, -1]
    _, _, op, _, _ = C.select(w, pos, [8], [5], [99])
    assert op[0, :5].tolist() == [0, 1, 6, 3, 5] or op[0, :5].tolist() == [0, 1, 5, 3, 6]   # of the ones, row 1 stays


def test_split_counts(cc):
    assert cc.kv_splits(8160, 64, 256, 512) == 8 and cc.kv_splits(8160, 64, 256, 256) == 8
    assert cc.kv_splits(32736, 8, 256, 512) == 64
    assert cc.kv_splits(128, 64, 256, 512) == 1
    assert cc.kv_splits(992, 1, 256, 512) == 32             # a small step: two slots per 64 keys
    assert cc.kv_splits(10 ** 6, 1, 256, 256) == 512
    assert cc.kv_splits(8160, 8, 256, 512) == 32 and cc.kv_splits(8160, 8, 256, 1024) == 64 and cc.kv_splits(8160, 1, 256, 512) == 128
    assert cc.kv_splits(8160, 4096, 256, 512) == 1 and cc.kv_splits(8160, 100, 256, 512) == 4


def test_how_steps_run(cc):
    assert cc.history_shape(8160, 64, 64, 256, 512) == (1, 8)            # single tokens
    assert cc.history_shape(8160, 2048, 4, 256, 512) == (3, 1)           # large chunks
    assert cc.history_shape(8160, 2048, 4, 256, 256) == (2, 1) and cc.history_shape(8160, 2048, 4, 256, 1024) == (2, 1)
    assert cc.history_shape(8160, 2048, 32, 256, 512) == (2, 1)
    assert cc.history_shape(8160, 64, 4, 256, 512) == (2, 8) and cc.history_shape(8160, 255, 4, 256, 512) == (2, 4)
    assert cc.history_shape(2000, 64, 4, 256, 512)[0] == 1 and cc.history_shape(8160, 2048, 4, 256, 128) == (1, 1)
    assert cc.history_shape(8160, 0, 0, 256, 512)[0] == 1


def test_cache_shape(cc):
    assert cc.cache_shape(10, 32, 512) == (10, 2, 17 * 512)
    for args in ((10, 24, 512), (10, 0, 512), (10, 16, 384)):
        with pytest.raises(ValueError):
            cc.cache_shape(*args)


def test_host_tensors_are_refused(cc):
    cache, rows, i32 = torch.zeros(2, 1, 17 * 128, dtype=torch.uint8), torch.zeros(1, 128, dtype=torch.bfloat16), \
        torch.zeros(1, dtype=torch.int32)
    for call in (lambda: cc.store_rows(rows, rows, i32.long(), cache), lambda: cc.load_rows(cache, i32[None], i32, 4),
                 lambda: cc.history_attention(rows[None].expand(1, 16, 128), cache, i32[None], i32, 1.0, 4),
                 lambda: cc.attention_weights(rows[None].expand(1, 16, 128), cache, i32[None], i32, i32, torch.zeros(16, 1), 1.0,
                                              torch.zeros(1, 4)),
                 lambda: cc.select_rows(torch.zeros(1, 4), i32[None], i32, 2, i32),
                 lambda: cc.move_rows(cache, i32[None], cc.Eviction(i32, i32, i32, i32[None], i32[None]))):
        with pytest.raises(RuntimeError, match='GPU only'):
            call()


def test_entry_points_check_before_they_launch(pkg):
    lib = pkg._lib

    def call(name, **at):
        args = [None if t is lib.P else 0 for t in lib.SIGNATURES[name]]
        for i, v in at.items():
            args[int(i[1:])] = v
        lib.call(name, *args)

    page = 17 * 128
    store = dict(_4=1, _5=128, _7=16, _8=page, _9=16, _10=2)       # tokens, width, cache, page stride, block, pages
    for change, match in ((dict(_5=384), 'width'), (dict(_9=24), 'block size'), (dict(_10=0), 'empty cache'), (dict(_7=8), 'aligned'),
                          (dict(_8=page - 16), 'apart'), (dict(_4=-1), 'token count'), ({}, 'null pointer')):
        with pytest.raises(ValueError, match=match):
            call('hla_s6_compact_store', **{**store, **change})
    load = dict(_0=16, _1=128, _2=page, _3=16, _4=2, _12=1, _13=4)
    for change, match in ((dict(_12=70000), 'request count'), (dict(_1=96), 'width'), ({}, 'null pointer'),
                          (dict(_8=16, _14=16, _5=16, _15=8, _16=8), 'apart'), (dict(_8=16, _14=8, _5=16, _16=256), 'aligned')):
        with pytest.raises(ValueError, match=match):
            call('hla_s6_compact_load', **{**load, **change})
    history = dict(_0=16, _1=1, _2=16, _3=128, _6=16, _7=page, _8=16, _9=2, _10=16, _12=1, _13=1, _15=16, _17=1, _22=1, _24=16, _27=16)
    for change, match in ((dict(_2=8), 'heads'), (dict(_3=64), 'width'), (dict(_17=0), 'num_kv_splits'), (dict(_17=1025), 'num_kv_splits'),
                          (dict(_13=0), 'table rows'), (dict(_0=None), 'null pointer'), (dict(_27=None), 'null pointer'), (dict(_4=4), 'aligned'),
                          (dict(_22=2), 'tokens per group'), (dict(_3=256, _7=2 * page, _22=3), 'tokens per group'),
                          (dict(_17=2, _18=16, _19=10 ** 6, _20=16, _21=3), 'split plan')):
        with pytest.raises(ValueError, match=match):
            call('hla_s6_compact_history', **{**history, **change})
    with pytest.raises(RuntimeError, match='workspace overflow'):
        call('hla_s6_compact_history', **{**history, '_17': 2, '_18': 16, '_19': 10})
    weights = dict(_0=16, _1=1, _2=16, _3=128, _6=16, _7=1, _8=page, _10=16, _11=2, _12=16, _14=1, _15=16, _16=1, _17=16, _18=16, _20=16,
                   _21=4, _22=4, _23=64)
    for change, match in ((dict(_2=1), 'heads'), (dict(_16=70000), 'request count'), (dict(_21=3), 'overlap'), (dict(_23=100), 'multiple of 64'),
                          (dict(_24=65), 'shares'), (dict(_18=None), 'null pointer'), (dict(_7=0, _9=12), 'aligned')):
        with pytest.raises(ValueError, match=match):
            call('hla_s6_attention_weights', **{**weights, **change})
    with pytest.raises(RuntimeError, match='workspace'):
        call('hla_s6_attention_weights', **{**weights, '_24': 2})
    select = dict(_0=16, _1=8, _2=16, _3=8, _4=16, _5=1, _6=8, _7=4, _9=16, _10=16, _11=16, _12=16, _13=16, _14=16)
    for change, match in ((dict(_7=-1), 'budget'), (dict(_1=7), 'overlap'), (dict(_4=None), 'null pointer'), (dict(_13=None), 'null list')):
        with pytest.raises(ValueError, match=match):
            call('hla_s6_select_rows', **{**select, **change})
    move = dict(_0=16, _1=128, _2=1, _3=page, _5=16, _6=2, _7=16, _9=1, _10=16, _11=16, _12=4, _13=4, _14=1)
    for change, match in ((dict(_14=-1), 'request count'), (dict(_12=3), 'overlap'), (dict(_10=None), 'null pointer'), (dict(_1=192), 'width')):
        with pytest.raises(ValueError, match=match):
            call('hla_s6_move_rows', **{**move, **change})
