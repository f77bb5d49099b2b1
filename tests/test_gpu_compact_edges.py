"""The compact latent cache, its accounts and evictions at the edges: lengths that change within a step, rows that read as
NaN, padding tokens, long walks of one workgroup, mixed steps. Oracle and bounds are those of test_gpu_compact_cache.py."""
import math

import numpy as np
import pytest
import torch

import compact_ref as C
from s6util import FakeLatentLayer, dev_bf16, dev_i32, dev_i64, host_f32, random_bits
from test_gpu_compact_cache import HALF, SCALE, Pool, check_attention, dev_u8, host_u8, layer_step, want_account
from oracle import bf16

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def cc(pkg):
    return pkg.compact_cache


class Layer:
    """One layer of a step: chunks of requests of given contexts over a compact cache and the bf16 cache of the same values,
    with an exact window."""

    def __init__(self, pkg, ops, rng, contexts, chunk, w, block=16):
        self.pkg, self.ops, self.contexts, self.chunk, self.w, self.block = pkg, ops, contexts, chunk, w, block
        self.rng, H, D = rng, 16, 128
        T = len(contexts) * chunk
        self.pool = Pool(rng, [c + chunk for c in contexts], w, block)
        self.table = dev_i32(self.pool.table)
        pages = len(self.pool.cache)
        self.exact = dev_bf16(random_bits(rng, (pages, H, block, 2 * D)))
        self.q_lat = dev_bf16(random_bits(rng, (T, H, w), 1.4 * math.sqrt(128 / w)))
        self.q_rope, self.k_rope, self.v = (dev_bf16(random_bits(rng, (T, H, D))) for _ in range(3))
        B = dev_bf16(random_bits(rng, (H, w, D), 1 / math.sqrt(w)))
        self.layer = FakeLatentLayer(B, B, [B], [B])
        self.layer.rank1 = self.layer.rank = w

    @property
    def compact(self):
        return dev_u8(self.pool.cache)

    @property
    def plain(self):
        pages, block = len(self.pool.cache), self.block
        every = np.nan_to_num(C.load(self.pool.cache, np.arange(pages * block)))
        return torch.from_numpy(every.reshape(pages, 1, block, 2 * self.w)).to(torch.bfloat16).cuda()

    def step(self):
        return layer_step(self.pkg, self.ops, self.rng, self.contexts, self.chunk, None, self.w)[0]

    def attend(self, cache, ctx, **kw):
        return self.pkg.s6_layer.attend(self.layer, 0, self.q_lat, self.q_rope, self.k_rope, self.v, cache, self.table, None, None,
                                        ctx, (self.exact, self.table), **kw)


# ---- lengths -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('compact', [True, False])
@pytest.mark.parametrize('w,chunk', [(512, 1), (256, 3)])
def test_lengths_may_change_within_a_step(pkg, ops, w, chunk, compact):
    """One StepContext, layers whose caches keep different numbers of rows: each attends to its own."""
    rng = np.random.default_rng(w + chunk)
    x = Layer(pkg, ops, rng, [600, 90, 1200, 333], chunk, w)
    cache = x.compact if compact else x.plain
    ctx = x.step()
    full = ctx.ctx_latent.clone()
    for turn, lengths in enumerate((full // 9, full, full // 2, torch.flip(full, (0,)).minimum(full))):
        if turn % 2:
            ctx.ctx_latent = lengths
        else:
            ctx.ctx_latent.copy_(lengths)
        fresh = x.step()
        fresh.ctx_latent.copy_(lengths)
        assert torch.equal(x.attend(cache, ctx), x.attend(cache, fresh)), turn


# ---- rows that read as NaN ------------------------------------------------------------------------------------------

@pytest.mark.parametrize('where', ['key', 'value'])
@pytest.mark.parametrize('chunk,shape', [(1, None), (3, None), (20, None), (20, (1, 1)), (20, (2, 1)), (20, (2, 3)), (20, (3, 1))])
def test_attend_passes_nan_on(cc, pkg, ops, monkeypatch, chunk, shape, where):
    """A NaN in a request's latent rows makes its output NaN, with an account and without, and no other's. A NaN key makes the
    request's account NaN as well; with a NaN value the weights are what they were."""
    rng = np.random.default_rng(chunk)
    if shape:
        monkeypatch.setattr(cc, 'history_shape', lambda *a: shape)
    contexts, w, block = [300, 200, 90], 512, 16
    x = Layer(pkg, ops, rng, contexts, chunk, w, block)
    M = 300 + chunk
    clean_account = torch.zeros(3, M, device='cuda')
    clean = x.attend(x.compact, x.step(), weights=clean_account)
    rows = x.pool.rows(1)[[77]]
    rows[0, 40 if where == 'key' else w + 40] = np.nan
    C.store(x.pool.cache, rows[:, :w], rows[:, w:], C.slots_of(x.pool.table[1], block, 78)[[77]])
    account = torch.zeros(3, M, device='cuda')
    bad = slice(chunk, 2 * chunk)
    for out in (x.attend(x.compact, x.step(), weights=account), x.attend(x.compact, x.step())):
        assert torch.isnan(out[bad]).all()
        for good in (slice(0, chunk), slice(2 * chunk, 3 * chunk)):
            assert (out[good].float() - clean[good].float()).abs().max() <= 4 * HALF * clean.float().abs().max()
    assert torch.equal(account[[0, 2]], clean_account[[0, 2]])
    behind = contexts[1] - 32
    assert (account[1, behind:] == 0).all()
    if where == 'key':
        assert torch.isnan(account[1, :behind]).all()
    else:
        assert torch.equal(account[1], clean_account[1])


def test_merged_lse(ops):
    """merge_states with its lse: empty sides (-inf, and +inf as the window kernels of others mark them), both, rows of padding,
    NaN. Bounds: an output rounds to bf16 once (half a step: 2^-8) over fp32 weights (2^-20)."""
    rng = np.random.default_rng(6)
    T, H, D = 9, 16, 128
    a, b = (random_bits(rng, (T, H, D)) for _ in range(2))
    la, lb = (rng.standard_normal((H, T)).astype(np.float32) * 3 for _ in range(2))
    la[:, 1], lb[:, 2], la[:, 3], lb[:, 4], la[:, 5], lb[:, 5] = -np.inf, -np.inf, np.inf, np.inf, -np.inf, np.inf
    a[5], b[5] = 0, 0
    la[:, 6], a[6] = np.nan, bf16.from_f32(np.full((H, D), np.nan, np.float32))
    invalid = np.arange(T) == 8
    out, lse = ops.merge_states(dev_bf16(a), torch.from_numpy(la).cuda(), dev_bf16(b), torch.from_numpy(lb).cuda(),
                                torch.from_numpy(invalid).cuda(), 'hip', return_lse=True)
    plain = ops.merge_states(dev_bf16(a), torch.from_numpy(la).cuda(), dev_bf16(b), torch.from_numpy(lb).cuda(),
                             torch.from_numpy(invalid).cuda(), 'hip')
    assert torch.equal(out.view(torch.int16), plain.view(torch.int16))
    assert torch.isnan(out[6]).all() and torch.isnan(lse[:, 6]).all()
    for t in (0, 1, 2, 3, 4, 5, 7, 8):
        x, y = (np.where(np.isinf(l[:, t]) | invalid[t], -np.inf, l[:, t]).astype(np.float64) for l in (la, lb))
        top = np.maximum(np.maximum(x, y), -1e30)
        p, r = np.exp(x - top), np.exp(y - top)
        total = p + r
        with np.errstate(divide='ignore'):
            want_lse = np.where(total > 0, top + np.log(total), -np.inf)
        total = np.maximum(total, 1e-300)
        want = (p / total)[:, None] * bf16.to_f32(a[t]) + (r / total)[:, None] * bf16.to_f32(b[t])
        size = (p / total)[:, None] * np.abs(bf16.to_f32(a[t])) + (r / total)[:, None] * np.abs(bf16.to_f32(b[t]))
        assert (np.abs(host_f32(out[t]) - want) <= HALF * np.abs(want) + 2.0 ** -20 * size).all(), t
        got = lse[:, t].cpu().numpy()
        assert (np.isneginf(got) == np.isneginf(want_lse)).all(), t
        fine = np.isfinite(want_lse)
        assert (np.abs(got[fine] - want_lse[fine]) <= 2.0 ** -20 * (1 + np.abs(want_lse[fine]))).all(), t


@pytest.mark.parametrize('shape', [(1, 1), (1, 3), (2, 1), (2, 3), (3, 1)])
def test_nan_rows_reach_the_tokens_that_see_them(cc, monkeypatch, shape):
    """Every form of a chunk: NaN outputs and lse for tokens whose rows hold one, and neighbours of the same request whose rows
    end before it are exact."""
    monkeypatch.setattr(cc, 'history_shape', lambda *a: shape)
    rng = np.random.default_rng(77)
    n, chunk, w = [300, 130], [19, 14], 512
    p = Pool(rng, n, w, 16)
    req = np.repeat([0, 1], chunk)
    ctx = np.array(n)[req]
    ctx[[0, 3, 4, 9, 18]] = 150, 149, 7, 0, 64
    clean = {0: p.rows(0), 1: p.rows(1)}
    for part in (0, 1):
        rows = clean[0][[150 + part]].copy()
        rows[0, part * w:(part + 1) * w] = np.nan     # a key, and behind it a value
        C.store(p.cache, rows[:, :w], rows[:, w:], C.slots_of(p.table[0], 16, 300)[[150 + part]])
    q = random_bits(rng, (len(req), 16, w), 0.5)
    start = dev_i32(np.concatenate(([0], np.cumsum(chunk))))
    o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE, 300,
                                  token_requests=dev_i64(req), query_start_loc=start, max_query_len=19)
    bad = (req == 0) & (ctx > 150)
    assert torch.isnan(o[torch.from_numpy(bad)]).all() and torch.isnan(lse[:, torch.from_numpy(bad)]).all()
    keep = np.flatnonzero(~bad)
    check_attention(host_f32(o)[keep], host_f32(lse)[:, keep], bf16.to_f32(q)[keep], lambda t: clean[req[keep[t]]], ctx[keep])


@pytest.mark.parametrize('scale', [-SCALE, 0.0])
def test_chunks_at_any_scale(cc, monkeypatch, scale):
    """A negative scale, and none: the smallest scores count most, or all rows alike."""
    monkeypatch.setattr(cc, 'history_shape', lambda *a: (3, 1))
    rng = np.random.default_rng(79)
    p = Pool(rng, [90], 512, 16)
    q = random_bits(rng, (11, 16, 512), 0.5)
    o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32([90] * 11), scale, 90,
                                  token_requests=dev_i64([0] * 11), query_start_loc=dev_i32([0, 11]), max_query_len=11)
    for t in range(11):
        want, want_lse, size = C.attention(bf16.to_f32(q)[t].astype(np.float64), p.rows(0), scale)
        d = 514 * 2.0 ** -24 * abs(scale) * (np.abs(bf16.to_f32(q)[t]).astype(np.float64) @ np.abs(p.rows(0)[:, :512]).T).max()
        bound = HALF * (size * 1.01 + np.abs(want)) + (math.expm1(2 * d) + 2.0 ** -20) * size
        assert (np.abs(host_f32(o)[t] - want) <= bound).all()
        assert (np.abs(host_f32(lse)[:, t] - want_lse) <= d + 2.0 ** -20 + 2.0 ** -22 * np.abs(want_lse)).all()


def test_rows_with_nan_refusals(ops):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device='cuda')
    call = lambda w=512, splits=1, group=4, scale=1.0: ops.history_attention_kv(
        z(2, 16, w), z(4, 1, 16, w), z(4, 1, 16, w), z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32), scale, splits,
        ops.S6Workspace(16, 1024, 8), None, None, 'hip', tokens_per_group=group, nan_rows=True)
    assert torch.isneginf(call()[1]).all()
    for kw in (dict(w=1024), dict(w=128), dict(splits=2), dict(group=1), dict(group=2), dict(scale=0.0), dict(scale=-1.0)):
        with pytest.raises(ValueError, match='rows with NaN'):
            call(**kw)


@pytest.mark.parametrize('shape', [(1, 1), (2, 1), (3, 1)])
def test_tokens_outside_the_chunks_have_rows_too(cc, monkeypatch, shape):
    """Tokens in front of the first chunk and behind the last one that name a request attend to its first ctx rows, in every
    form: none reads memory that nothing was written to (which holds NaN here)."""
    monkeypatch.setattr(cc, 'history_shape', lambda *a: shape)
    rng = np.random.default_rng(78)
    n, w = [210, 64, 33], 512
    p = Pool(rng, n, w, 16)
    req = np.array([2, 0] + [0] * 9 + [1] * 5 + [0, 2, 2])
    start, ctx = dev_i32([2, 11, 16, 16]), np.array(n)[req]
    ctx[2:11] = 90                                             # behind it the request's rows are needed by others alone
    q = random_bits(rng, (len(req), 16, w), 0.5)
    args = (dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE, 210)
    used = [torch.full((3 * 14, 1, 16, 2 * w), float('nan'), dtype=torch.bfloat16, device='cuda') for _ in range(4)]
    del used
    o, lse = cc.history_attention(*args, token_requests=dev_i64(req), query_start_loc=start, max_query_len=9)
    check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), lambda t: p.rows(req[t]), ctx)


# ---- accounts ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('compact', [True, False])
@pytest.mark.parametrize('w,chunk', [(256, 1), (1024, 1), (512, 1), (128, 40), (512, 40), (1024, 40)])
def test_tokens_with_an_infinite_lse_add_nothing(cc, w, chunk, compact):
    """Whatever their queries and the rows hold."""
    rng = np.random.default_rng(w + chunk)
    n, block = [150, 60], 16
    p = Pool(rng, n, w, block)
    T = 2 * chunk
    q = random_bits(rng, (T, 16, w), 1.4 * math.sqrt(128 / w))
    lse = rng.standard_normal((16, T)).astype(np.float32) + 8
    empty = chunk + chunk // 2                                  # a token of request 1
    lse[:, empty] = np.where(np.arange(16) % 2, np.inf, -np.inf)
    q[empty, :, ::5] = bf16.from_f32(np.array([np.nan], np.float32))[0]
    q[empty, 3] = bf16.from_f32(np.array([np.inf], np.float32))[0]
    req, ctx = np.repeat([0, 1], chunk), np.repeat(n, chunk)
    cache = dev_u8(p.cache)
    if not compact:
        every = C.load(p.cache, np.arange(len(p.cache) * block))
        cache = torch.from_numpy(every.reshape(len(p.cache), 1, block, 2 * w)).to(torch.bfloat16).cuda()
    start = rng.random((2, 150)).astype(np.float32)
    clean = bf16.to_f32(q).copy()
    clean[empty] = 0
    want, bound = want_account(start, clean, p.rows, w, lse, req, ctx, 150)
    got = cc.attention_weights(dev_bf16(q), cache, dev_i32(p.table), dev_i32([0, chunk, T]), dev_i32(ctx),
                               torch.from_numpy(lse).cuda(), SCALE, torch.from_numpy(start).cuda()).cpu().numpy()
    assert (np.abs(got - want) <= bound).all()
    assert chunk > 1 or (got[1] == start[1]).all()


@pytest.mark.parametrize('chunk', [1, 64])
def test_rows_behind_the_requests_keep_their_bits(cc, chunk):
    """Accounts behind a request's rows, and of requests without tokens: -0 stays -0, a NaN keeps its payload."""
    rng = np.random.default_rng(chunk)
    n, w, M = [100, 0, 40, 16], 256, 130
    p = Pool(rng, n, w, 16)
    T = 2 * chunk
    assert cc.account_shape(T, 4, M, 256, w)[0] == 0 if chunk == 1 else cc.account_shape(T, 4, M, 256, w)[0] > 1
    req = np.repeat([0, 2], chunk)                              # requests 1 and 3 have no tokens
    bits = np.where(rng.random((4, M)) < 0.5, 0x80000000, 0x7f812345).astype(np.uint32)
    account = torch.from_numpy(bits.view(np.int32)).cuda().view(torch.float32)
    cc.attention_weights(dev_bf16(random_bits(rng, (T, 16, w))), dev_u8(p.cache), dev_i32(p.table),
                         dev_i32([0, chunk, chunk, T, T]), dev_i32(np.array(n)[req]), torch.zeros(16, T, device='cuda'), SCALE, account)
    got = account.view(torch.int32).cpu().numpy().view(np.uint32)
    for r, rows in enumerate([100, 0, 40, 0]):
        assert (got[r, rows:] == bits[r, rows:]).all(), r


# ---- operands ------------------------------------------------------------------------------------------------------

def test_plans_of_other_kinds(cc, ops):
    """A plan of another type is refused; one whose chunk and slots would overflow stays inside the rows."""
    rng = np.random.default_rng(17)
    n, w, S = [200, 77], 256, 3
    p = Pool(rng, n, w, 16)
    q = random_bits(rng, (2, 16, w))
    args = (dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(n), SCALE)
    plan = ops.split_plan(dev_i32(n), p.table.shape[1] * 16, S)
    for bad in (plan.long(), plan.float(), plan[None], plan.repeat_interleave(2)[::2]):
        with pytest.raises(ValueError, match='plan'):
            cc.history_attention(*args, 200, num_kv_splits=S, plan=bad)
        with pytest.raises(ValueError, match='plan'):
            cc.history_partials(*args, S, ops.S6Workspace(16, w, 8), plan=bad)
    items = (len(plan) - 3) // 2
    rows, slots = np.full(items, -1), np.zeros(items)
    rows[:6], slots[:6] = [0, 1, 0, 1, 0, 1], [0, 0, 2, 2, 1, 1]
    for chunk in (2 ** 31 - 1, 2 ** 30, 13):                   # slot 0 holds whole rows; 2 * chunk passes 32 bits
        made = dev_i32(np.concatenate(([chunk, S, S], rows, slots)))
        o, lse = cc.history_attention(*args, 200, num_kv_splits=S, plan=made)
        check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), p.rows, n)


def test_a_workspace_of_another_device_is_refused(cc, ops):
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device='cuda')
    ws = ops.S6Workspace(16, 256, 8)
    ws.ensure('cpu')
    args = (z(2, 16, 256), z(4, 1, 17 * 256, dtype=torch.uint8), z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32), SCALE)
    with pytest.raises(RuntimeError, match='GPU only'):
        cc.history_attention(*args, 48, num_kv_splits=4, workspace=ws)
    with pytest.raises(RuntimeError, match='GPU only'):
        cc.history_partials(*args, 4, ws)
    cc.history_attention(*args, 48, num_kv_splits=1, workspace=ws)     # needs none


def test_a_large_step_without_requests(cc):
    """query_start_loc of no request: all tokens lie outside the chunks, and attend to the rows that they name."""
    rng = np.random.default_rng(18)
    p = Pool(rng, [33], 512, 16)
    T = 2100
    q = random_bits(rng, (T, 16, 512), 0.5)
    assert cc.history_shape(33, T, 1, 256, 512)[0] == 3
    o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32([33] * T), SCALE, 33,
                                  token_requests=dev_i64([0] * T), query_start_loc=dev_i32([0]), max_query_len=T)
    some = [0, 1, 1050, T - 1]
    check_attention(host_f32(o[some]), host_f32(lse[:, some]), bf16.to_f32(q)[some], lambda t: p.rows(0), [33] * 4)


# ---- eviction beside an exact window ----------------------------------------------------------------------------------

@pytest.mark.parametrize('compact', [True, False])
def test_eviction_beside_a_window_in_a_ragged_batch(cc, compact):
    """Requests with none, few, exactly W and many rows above the budget, shorter than the window, with pages of the others in
    their unused table entries: rows go where at least W are to go, and the W rows behind follow them in order."""
    rng = np.random.default_rng(19)
    W, top, w, block = 32, 64, 256, 16
    n = np.array([64, 69, 95, 96, 97, 300, 0, 40, 128])        # rows behind the window's
    p = Pool(rng, n + W, w, block)
    p.table[6, 2:] = p.table[5, :len(p.table[6]) - 2]           # beyond its 32 rows: pages of request 5
    p.table[7, 5:] = p.table[8, :len(p.table[7]) - 5]
    R, M = len(n), 300
    if compact:
        cache = dev_u8(p.cache)
    else:
        every = np.nan_to_num(C.load(p.cache, np.arange(len(p.cache) * block)))
        cache = torch.from_numpy(every.reshape(len(p.cache), 1, block, 2 * w)).to(torch.bfloat16).cuda()
    before = [p.rows(r) for r in range(R)]
    table, lengths = dev_i32(p.table), dev_i32(n)
    account = torch.rand(R, M, device='cuda')
    positions = torch.arange(M, dtype=torch.int32, device='cuda').repeat(R, 1)
    budget = torch.where(lengths >= top + W, top, lengths)
    e = cc.select_rows(account, positions, lengths, budget, lengths)
    cc.move_rows(cache, table, e)
    i, gone = torch.arange(W, dtype=torch.int32, device='cuda'), (e.lengths < lengths)[:, None]
    source, target = (torch.where(gone, x[:, None] + i, -1) for x in (lengths, e.lengths))
    cc.move_rows(cache, table, cc.Eviction(None, None, None, source, target))
    assert e.lengths.tolist() == [64, 69, 95, 64, 64, 64, 0, 40, 64]
    got = host_u8(cache) if compact else host_f32(cache).reshape(-1, 2 * w)
    for r in range(R):
        b = int(e.lengths[r])
        kept = np.concatenate((e.positions[r, :b].cpu().numpy(), n[r] + np.arange(W)))
        slots = C.slots_of(p.table[r], block, b + W)
        assert ((C.load(got, slots) if compact else got[slots]) == before[r][kept]).all(), r
        assert b == n[r] or kept[:b].max() < n[r] and len(set(kept)) == b + W
        assert b < n[r] or (kept == np.arange(b + W)).all()


# ---- long walks ----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize('shape', [(1, 1), (2, 1)])
@pytest.mark.parametrize('width,block', [(128, 16), (256, 48), (512, 16), (1024, 32)])
def test_one_workgroup_walks_past_its_page_look_ups(cc, monkeypatch, width, block, shape):
    """A wave looks up the pages of 32 steps at a time (4096 rows, with two tokens 2048 at width 512, and 1024 rows at 1024):
    rows of more than two look-ups in one slot, in scattered pages, and rows that end with a look-up."""
    if shape[0] == 2 and width == 128:
        shape = (1, 1)                                          # (no form for two tokens there)
    monkeypatch.setattr(cc, 'history_shape', lambda *a: shape)
    rng = np.random.default_rng(width)
    n = [8192 + 73, 4096, 2049] if width < 1024 else [4096 + 73, 2048, 1025]
    p = Pool(rng, n, width, block)
    req = np.array([0, 0, 1, 1, 2])
    ctx = np.array(n)[req]
    q = random_bits(rng, (5, 16, width), 1.4 * math.sqrt(128 / width))
    rows = [p.rows(r) for r in range(3)]
    for length in (2, 1):                                       # rows that tokens share, and rows that stream past the caches
        o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE, max(n),
                                      token_requests=dev_i64(req), max_query_len=length, num_kv_splits=1)
        check_attention(host_f32(o), host_f32(lse), bf16.to_f32(q), lambda t: rows[req[t]], ctx)


@pytest.mark.parametrize('compact', [True, False])
@pytest.mark.parametrize('width,keys', [(128, 1024), (256, 4096), (512, 1024), (512, 4096), (1024, 2048), (1024, 64)])
def test_accounts_of_many_rows_per_workgroup(cc, monkeypatch, width, keys, compact):
    """Single tokens, requests of two and three tokens and of none in the kernel that streams K, over rows that fill the places
    a wave looks up, and end in the middle."""
    monkeypatch.setattr(cc, 'account_shape', lambda *a: (0, keys))
    rng = np.random.default_rng(width + keys)
    n, chunk = [4100, 1030, 16, 333], [1, 3, 0, 2]
    p = Pool(rng, n, width, 16)
    cache = dev_u8(p.cache)
    if not compact:
        every = C.load(p.cache, np.arange(len(p.cache) * 16))
        cache = torch.from_numpy(every.reshape(len(p.cache), 1, 16, 2 * width)).to(torch.bfloat16).cuda()
    req = np.repeat(np.arange(4), chunk)
    ctx = np.array(n)[req]
    ctx[2] = 517
    q = random_bits(rng, (6, 16, width), 1.4 * math.sqrt(128 / width))
    lse = rng.standard_normal((16, 6)).astype(np.float32) + 8
    start = rng.random((4, 4100)).astype(np.float32)
    rows = [p.rows(r) for r in range(4)]
    want, bound = want_account(start, bf16.to_f32(q), lambda r: rows[r], width, lse, req, ctx, 4100)
    got = cc.attention_weights(dev_bf16(q), cache, dev_i32(p.table), dev_i32(np.concatenate(([0], np.cumsum(chunk)))), dev_i32(ctx),
                               torch.from_numpy(lse).cuda(), SCALE, torch.from_numpy(start).cuda()).cpu().numpy()
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())


# ---- steps that mix chunks and single tokens ----------------------------------------------------------------------------

@pytest.mark.parametrize('chunk', [9, 10])
@pytest.mark.parametrize('width', [256, 512])
def test_accounts_of_mixed_steps(cc, width, chunk):
    """Eight single tokens and one chunk, on both sides of the rule that picks the kernel."""
    rng = np.random.default_rng(width + chunk)
    n = [40, 300, 17, 1, 0, 64, 130, 222, 180]
    count = [1] * 8 + [chunk]
    T = sum(count)
    assert (cc.account_shape(T, 9, 300, 256, width)[0] == 0) == (chunk == 9)
    p = Pool(rng, n, width, 16)
    req = np.repeat(np.arange(9), count)
    ctx = np.array(n)[req]
    q = random_bits(rng, (T, 16, width), 1.4 * math.sqrt(128 / width))
    lse = rng.standard_normal((16, T)).astype(np.float32) + 8
    start = rng.random((9, 300)).astype(np.float32)
    want, bound = want_account(start, bf16.to_f32(q), p.rows, width, lse, req, ctx, 300)
    got = cc.attention_weights(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(np.concatenate(([0], np.cumsum(count)))),
                               dev_i32(ctx), torch.from_numpy(lse).cuda(), SCALE, torch.from_numpy(start).cuda()).cpu().numpy()
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize('singles,chunk,width,n', [(100, 412, 256, 60), (100, 412, 512, 60), (30, 100, 512, 4200), (7, 2057, 512, 50)])
def test_history_of_mixed_steps(cc, singles, chunk, width, n):
    """Single tokens and one chunk in the forms that their numbers on average ask for: two tokens a workgroup, in splits, expanded."""
    rng = np.random.default_rng(singles)
    R, T = singles + 1, singles + chunk
    kind, splits = cc.history_shape(n, T, R, 256, width)
    assert (kind, splits > 1) == {60: (2, False), 4200: (2, True), 50: (3, False)}[n]
    lengths = rng.integers(0, 41, R)
    lengths[0], lengths[singles] = n, n - 3
    p = Pool(rng, lengths, width, 16)
    count = [1] * singles + [chunk]
    req = np.repeat(np.arange(R), count)
    ctx = lengths[req]
    q = random_bits(rng, (T, 16, width), 1.4 * math.sqrt(128 / width))
    o, lse = cc.history_attention(dev_bf16(q), dev_u8(p.cache), dev_i32(p.table), dev_i32(ctx), SCALE, n,
                                  token_requests=dev_i64(req), query_start_loc=dev_i32(np.concatenate(([0], np.cumsum(count)))),
                                  max_query_len=chunk)
    some = np.concatenate((np.arange(singles + 2), [T - 2, T - 1]))
    last = p.rows(singles)
    check_attention(host_f32(o[some]), host_f32(lse[:, some]), bf16.to_f32(q)[some],
                    lambda t: last if req[some[t]] == singles else p.rows(req[some[t]]), ctx[some])


@pytest.mark.parametrize('w,contexts,chunk,kind', [(256, [330, 90, 20, 600], 130, 2), (512, [330, 90, 20, 600], 130, 2),
                                                   (512, [330, 90, 20, 600], 512, 3), (512, [4200, 4100], 17, 2)])
def test_attend_in_every_form(cc, pkg, ops, monkeypatch, w, contexts, chunk, kind):
    """s6_layer.attend over a compact cache against the bf16 cache of the same values at sizes that take two tokens a workgroup,
    split and not, and the expanded form; bounds as in test_attend_over_a_compact_cache."""
    rng = np.random.default_rng(w + chunk)
    taken, shape = [], cc.history_shape
    monkeypatch.setattr(cc, 'history_shape', lambda *a: taken.append(shape(*a)) or taken[-1])
    x = Layer(pkg, ops, rng, contexts, chunk, w)
    M, R = max(contexts) + chunk, len(contexts)
    a1, a2 = torch.zeros(R, M, device='cuda'), torch.zeros(R, M, device='cuda')
    cache, plain = x.compact, x.plain
    want = x.attend(plain, x.step()).float()
    for got in (x.attend(cache, x.step()), x.attend(cache, x.step(), weights=a1), x.attend(plain, x.step(), weights=a2)):
        assert (got.float() - want).abs().max() <= 4 * HALF * want.abs().max()
        assert (got.float() - want).norm() <= 2 * HALF * want.norm()
    assert {k for k, _ in taken} == {kind}
    assert torch.allclose(a1, a2, rtol=2.0 ** -10, atol=1e-6)
