"""Whole exact caches on the GPU: results do not depend on how rows and tokens are dealt to workgroups. Tolerances are those of
``test_gpu_exact_cache``."""
import math

import numpy as np
import pytest
import torch

from s6util import dev_i32, dev_i64
from test_gpu_exact_cache import Cache, attend, check, query

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ec(pkg):
    return pkg.exact_cache


@pytest.mark.parametrize('bad', [math.nan, math.inf])
@pytest.mark.parametrize('shares', [None, 0, 1, 8, 1024])
def test_rows_of_no_weight_whose_values_are_not_finite(ec, shares, bad):
    """A stretch of rows with scores of -inf: 0 * NaN and 0 * inf are NaN where the token has other rows, in a share of their own
    (with 1024 shares of 128 rows) as in one with others; a token that has nothing else gives 0 and -inf."""
    n = [1000, 1000, 300]
    c = Cache(80, n, 2, 128, 16)
    q = query(81, 3, 4, 128)
    q[:, :, 0] = 1
    for r, rows, kv_head in ((0, range(256, 384), 1), (1, range(0, 16), 0), (2, range(300), 1)):
        for j in rows:
            page, at = int(c.table[r, j // 16]), j % 16
            c.cache[page, :, at, 0] = -math.inf
            c.cache[page, kv_head, at, 128:] = bad
    o, lse = attend(ec, q, c, n, shares=shares)
    assert torch.isnan(o[0, 2:]).all() and torch.isnan(o[1, :2]).all()
    assert torch.isfinite(o[0, :2]).all() and torch.isfinite(o[1, 2:]).all() and torch.isfinite(lse[:, :2]).all()
    assert (o[2] == 0).all() and torch.isneginf(lse[:, 2]).all()
    c.rows[0], c.rows[1] = torch.cat((c.rows[0][:256], c.rows[0][384:])), c.rows[1][16:]
    for t, heads in ((0, slice(0, 2)), (1, slice(2, 4))):
        part = Cache.__new__(Cache)
        part.h, part.rows = 1, [c.rows[t][:, heads.start // 2:heads.stop // 2]]
        check(o[t:t + 1, heads].contiguous(), lse[heads, t:t + 1], q[t:t + 1, heads], part, [0], [c.rows[t].shape[0]], 128 ** -0.5)


# ---- tokens alone beside chunks -----------------------------------------------------------------------------------------

@pytest.fixture
def in_shares(ec, monkeypatch):
    """Tokens alone are cut in shares whatever the length of their rows; the ``(shares, grouped)`` of the calls."""
    calls, call = [], ec._call

    def record(name, device, *args):
        calls.append(args[24:26])
        return call(name, device, *args)

    monkeypatch.setattr(ec, 'LONG_ROWS', 0)
    monkeypatch.setattr(ec, '_call', record)
    return calls


def mixed_step(lens, order):
    """Requests and lengths of a step: ``lens[r]`` tokens at the end of the ``n[r]`` rows of every request."""
    n = [300, 40, 1700, 900, 33, 2500]
    requests = sum(([r] * lens[r] for r in order), [])
    ctx = sum(([n[r] - lens[r] + i + 1 for i in range(lens[r])] for r in order), [])
    return n, requests, ctx


@pytest.mark.parametrize('e4m3', [False, True])
@pytest.mark.parametrize('kv_heads,G,d,block', [(2, 1, 128, 16), (128, 1, 128, 16), (1, 2, 64, 24), (43, 3, 128, 32), (1, 4, 256, 16),
                                               (26, 5, 64, 16), (2, 8, 128, 1)])
@pytest.mark.parametrize('window,turns', [(0, 4), (21, 2), (0, 16)])
def test_tokens_alone_beside_chunks(ec, in_shares, monkeypatch, kv_heads, G, d, block, e4m3, window, turns):
    """At both ends of a step, between chunks and one behind the other; a request that lies there twice; tokens without rows, of which
    one hides a neighbour of the same request; a chunk whose last token lies in the next group."""
    monkeypatch.setattr(ec, '_turns', lambda *a: turns)
    n, requests, ctx = mixed_step([33, 40, 1, 5, 20, 1], (5, 0, 2, 1, 3, 4))
    requests, ctx = requests + [2, 0, 5, 5, 5, 2, 3], ctx + [1000, 250, 2000, 0, 2100, 0, 850]
    requests, ctx = requests + [4, 4, 1, 5], ctx + [0, 0, -3, 2222]
    c = Cache(G + d, n, kv_heads, d, block, e4m3)
    q = query(G, len(ctx), kv_heads * G, d)
    o, lse = ec.attention(q, c.cache, c.table, dev_i32(np.array(ctx)), d ** -0.5, max(n), dev_i64(np.array(requests)), window,
                          c.k_scale, c.v_scale, max_query_len=40)
    assert in_shares == [(max(1, 512 // kv_heads), turns)]
    check(o, lse, q, c, requests, ctx, d ** -0.5, window)


@pytest.mark.parametrize('lens,order', [([1, 1, 1, 1, 1, 1], range(6)), ([64, 1, 64, 64, 32, 64], (0, 2, 3, 5, 4)),
                                        ([1, 1, 1, 1, 1, 300], (0, 1, 2, 5, 3, 4))])
def test_steps_of_one_kind(ec, in_shares, monkeypatch, lens, order):
    """Nothing but tokens alone, nothing but chunks, and a replayed graph whose lengths make one of the other."""
    monkeypatch.setattr(ec, '_turns', lambda *a: 3)
    n, requests, ctx = mixed_step(lens, order)
    c = Cache(90, n, 4, 128, 16)
    q, table_rows, lengths = query(91, len(ctx), 8, 128), dev_i64(np.array(requests)), dev_i32(np.array(ctx))
    ws = ec.s6_ops.S6Workspace(8, 128, 2 * 128 + 10)
    call = lambda: ec.attention(q, c.cache, c.table, lengths, 0.1, max(n), table_rows, max_query_len=max(4, *lens), workspace=ws)
    monkeypatch.setattr(ec, '_most_alone', lambda *a: 1)
    check(*call(), q, c, requests, ctx, 0.1)
    assert in_shares == [(128, 3)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, lse = call()
    for seed in (1, 2, 3):
        rng = np.random.default_rng(seed)
        now = np.where(rng.random(len(ctx)) < 0.5, 0, ctx)
        rows = rng.integers(0, 6, len(ctx)) if seed == 3 else np.array(requests)
        now = np.minimum(now, np.array(n)[rows])
        lengths.copy_(dev_i32(now))
        table_rows.copy_(dev_i64(rows))
        graph.replay()
        check(o, lse, q, c, rows, now.tolist(), 0.1)
        eager = call()
        torch.cuda.synchronize()
        assert torch.equal(eager[0], o) and torch.equal(eager[1], lse)


def test_many_tokens_alone(ec, in_shares, monkeypatch):
    """More of them than are listed, or joined, at a time; a workspace that is too small for them is left alone."""
    monkeypatch.setattr(ec, '_turns', lambda *a: 2)
    rng = np.random.default_rng(5)
    n = rng.integers(1, 400, 1500).tolist() + [700]
    lens = [1] * 1500 + [600]
    order = rng.permutation(1501).tolist()
    requests = sum(([r] * lens[r] for r in order), [])
    ctx = sum(([n[r] - lens[r] + i + 1 for i in range(lens[r])] for r in order), [])
    c = Cache(92, n, 2, 64, 16)
    q = query(93, len(ctx), 16, 64)
    ws = ec.s6_ops.S6Workspace(16, 64, 10)
    ws.ensure(q.device).fill_(math.nan)
    o, lse = ec.attention(q, c.cache, c.table, dev_i32(np.array(ctx)), 0.125, max(n), dev_i64(np.array(requests)), max_query_len=600,
                          workspace=ws)
    assert in_shares == [(256, 2)] and torch.isnan(ws.buffer).all()
    some = [t for t in range(len(ctx)) if requests[t] != 1500 or t % 20 == 0]
    check(o[some], lse[:, some], q[some], c, [requests[t] for t in some], [ctx[t] for t in some], 0.125)


def test_attend_exact_in_groups(pkg, ec, monkeypatch):
    """A prompt, a chunk on a history and single tokens through the layer's call and a pool's tables, rows stored by it."""
    calls, call = [], ec._call
    monkeypatch.setattr(ec, '_call', lambda name, device, *args: (calls.append((name, *args[24:26])), call(name, device, *args))[1])
    layer, ops = pkg.s6_layer, pkg.s6_ops
    n, lens, block = [4200, 300, 700, 5000], [1, 300, 200, 1], 16
    c = Cache(94, n, 16, 128, block)
    pos = np.concatenate([np.arange(n[r] - lens[r], n[r]) for r in range(4)] + [[0, 0]])
    T = len(pos)
    table = torch.zeros(60, c.table.shape[1], dtype=torch.int32, device='cuda')
    table[:4] = c.table
    ctx = layer.StepContext(torch.as_tensor(pos, device='cuda'), dev_i32(np.concatenate(([0], np.cumsum(lens)))), dev_i32(np.array(n)),
                            max(lens), T, {}, 0.09, ops.HIP_BACKENDS, max_seqlen_k=max(n))
    k, v, q = (torch.randn(T, 16, 128, generator=torch.Generator('cuda').manual_seed(95 + i), device='cuda').to(torch.bfloat16)
               for i in range(3))
    t, requests = 0, []
    for r in range(4):
        c.rows[r][n[r] - lens[r]:] = torch.cat((k[t:t + lens[r]], v[t:t + lens[r]]), -1).double()
        requests, t = requests + [r] * lens[r], t + lens[r]
    o = layer.attend_exact(q, k, v, c.cache, table, ctx)
    assert [x for x in calls if x[0] == 'hla_s6_exact_attention'] == [('hla_s6_exact_attention', 32, 16)]
    assert (o[T - 2:] == 0).all()
    lengths = (pos + 1).tolist()
    _, lse = ec.attention(q[:T - 2], c.cache, c.table, dev_i32(np.array(lengths[:T - 2])), 0.09, max(n), dev_i64(np.array(requests)), shares=0)
    some = [0, T - 3] + list(range(1, T - 3, 23))
    check(o[some], lse[:, some], q[some], c, [requests[t] for t in some], [lengths[t] for t in some], 0.09)


def test_a_long_row_among_many_tokens(ec):
    """By the rule in shares, of which some end inside one of several short rows."""
    n = np.random.default_rng(6).integers(0, 300, 300).tolist()
    n[200] = 20000
    c = Cache(96, n, 16, 64, 16)
    q = query(97, 300, 16, 64)
    assert ec.row_shares(20000, 300 * 16, 16) == 32
    o, lse = attend(ec, q, c, n)
    check(o, lse, q, c, range(300), n, 0.125)


def test_two_pools_in_a_step(pkg):
    """Layers on pools of their own, whose rows of the step are gathered anew for every call."""
    layer, ops = pkg.s6_layer, pkg.s6_ops
    g = torch.Generator(device='cuda').manual_seed(98)
    n = [40, 25, 1]
    ctx = layer.StepContext(torch.tensor([39, 24, 0], device='cuda'), dev_i32(np.arange(4)), dev_i32(np.array(n)), 1, 3, {}, 0.1,
                            ops.HIP_BACKENDS, max_seqlen_k=40)
    live = torch.tensor([5, 2, 0], device='cuda')
    for tables in (torch.arange(18, dtype=torch.int32, device='cuda').view(6, 3), torch.arange(17, -1, -1, dtype=torch.int32, device='cuda').view(6, 3)):
        cache = torch.randn(18, 2, 16, 128, generator=g, device='cuda').to(torch.bfloat16)
        q, k, v = (torch.randn(3, 2, 64, generator=g, device='cuda').to(torch.bfloat16) for _ in range(3))
        want = cache.clone()
        for t, r in enumerate(live.tolist()):
            want[tables[r, (n[t] - 1) // 16].long(), :, (n[t] - 1) % 16] = torch.cat((k[t], v[t]), -1)
        layer.attend_exact(q, k, v, cache, tables[live], ctx)
        assert torch.equal(cache, want)


def test_attend_exact_refuses_tables_before_it_stores(pkg):
    layer, ops = pkg.s6_layer, pkg.s6_ops
    ctx = layer.StepContext(torch.tensor([3, 4], device='cuda'), dev_i32(np.arange(3)), dev_i32(np.array([4, 5])), 1, 2, {}, 0.1,
                            ops.HIP_BACKENDS, max_seqlen_k=5)
    cache = query(99, 4, 2 * 16, 128).view(4, 2, 16, 128)
    before, rows = cache.clone(), query(100, 2, 2, 64)
    table = torch.arange(4, dtype=torch.int32, device='cuda').view(2, 2)
    for bad, error in ((table.long(), ValueError), (table.t(), ValueError), (table[0], ValueError), (table[:0], ValueError),
                       (table.cpu(), RuntimeError)):
        with pytest.raises(error):
            layer.attend_exact(rows, rows, rows, cache, bad, ctx)
        assert torch.equal(cache, before)
    o = layer.attend_exact(rows, rows, rows, cache, table[:1], ctx)       # the second request has no row: it stores nothing
    before[0, :, 3] = torch.cat((rows[0], rows[0]), -1)
    assert torch.equal(cache, before) and torch.isfinite(o).all()
