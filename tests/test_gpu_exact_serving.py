"""Pools of pages, exact caches and the latent caches in one serving run: prompts, samples that fork off them, decode steps,
requests that finish, compaction, and eviction of latent rows in pages that were shared."""
import numpy as np
import pytest
import torch

from s6util import dev_i32

pytestmark = pytest.mark.gpu
H, KH, D, BLOCK, R, W = 8, 4, 128, 16, 10, 128
SCALE = D ** -0.5
HALF = 2.0 ** -8


class Serving:
    """A pool, an exact bf16 and an e4m3 cache and a compact latent one on its pages; what every request has written, on the host side
    of the test, by position."""

    def __init__(self, pkg, seed):
        self.pkg, self.g = pkg, torch.Generator(device='cuda').manual_seed(seed)
        pages = 150
        self.pool = pkg.pages.new_pool(pages, BLOCK, R, 40 * BLOCK, 'cuda', reserved=1)
        exact = torch.full((pages, BLOCK, KH, 2 * D), float('nan'), device='cuda')
        self.exact, self.e4m3 = exact.to(torch.bfloat16).transpose(1, 2), exact.to(torch.float8_e4m3fn).transpose(1, 2)
        self.scale = torch.rand(KH, generator=self.g, device='cuda') / 64 + 0.01
        self.latent = torch.full(pkg.compact_cache.cache_shape(pages, BLOCK, W), 255, dtype=torch.uint8, device='cuda')
        self.rows = [[] for _ in range(R)]      # (key, value, latent row) per position

    def noise(self, *shape):
        return torch.randn(*shape, generator=self.g, device='cuda').to(torch.bfloat16)

    def copy(self, moves):
        for cache in (self.exact, self.e4m3, self.latent):
            self.pkg.pages.copy_pages(cache, moves.source, moves.target)

    def step(self, counts):
        """``counts[r]`` new tokens of every request."""
        n = np.asarray([len(x) for x in self.rows])
        e = self.pkg.pages.extend_requests(self.pool, dev_i32(n + counts))
        assert e.ok.all()
        self.copy(e)
        live = [r for r in range(R) if counts[r]]
        lens, T = [int(counts[r]) for r in live], int(counts.sum())
        table = self.pool.tables[torch.tensor(live, device='cuda')]
        pad = 2
        positions = np.concatenate([np.arange(n[r], n[r] + counts[r]) for r in live] + [np.zeros(pad, np.int64)])
        ops, layer, cc = self.pkg.s6_ops, self.pkg.s6_layer, self.pkg.compact_cache
        ctx = layer.StepContext(torch.as_tensor(positions, device='cuda'), dev_i32(np.concatenate(([0], np.cumsum(lens)))),
                                dev_i32(n[live] + np.asarray(lens)), max(lens), T + pad, {}, SCALE, ops.HIP_BACKENDS,
                                max_seqlen_k=int((n + counts).max()))
        q, k, v = self.noise(T + pad, H, D), self.noise(T + pad, KH, D), self.noise(T + pad, KH, D)
        lat = self.noise(T + pad, 2 * W)
        cc.store_rows(lat[:, :W], lat[:, W:], ctx.slots(table, BLOCK), self.latent)
        got = layer.attend_exact(q, k, v, self.exact, table, ctx)
        got8 = layer.attend_exact(q, k, v, self.e4m3, table, ctx, self.scale, self.scale)
        q_lat = self.noise(T + pad, 16, W)
        counts_now = ctx.row_counts
        hist, _ = cc.history_attention(q_lat, self.latent, table, counts_now, SCALE, int((n + counts).max()), ctx.token_requests)
        t = 0
        for r in live:
            for _ in range(int(counts[r])):
                self.rows[r].append((k[t], v[t], lat[t]))
                self.check(r, q[t], got[t], got8[t])
                t += 1
        assert (got[T:] == 0).all() and (got8[T:] == 0).all() and (hist[T:] == 0).all()
        return live, table, q_lat, hist, counts_now

    def check(self, r, q, *outs):
        k, v = (torch.stack([row[i] for row in self.rows[r]]).double().repeat_interleave(H // KH, 1) for i in (0, 1))
        for got, eight in zip(outs, (False, True)):
            if eight:
                s = self.scale.double().repeat_interleave(H // KH)[:, None]
                k, v = ((x / s).clamp(-448, 448).float().to(torch.float8_e4m3fn).double() * s for x in (k, v))
            p = torch.softmax((q.double() * k).sum(-1) * SCALE, 0)[..., None]
            want, size = (p * v).sum(0), (p * v.abs()).sum(0)
            # half a step of the output; of an e4m3 row, a quotient that fp32 rounds to the other side of a tie (rare) moves one value
            # by a step of 2^-3: at most the weight of its row
            bound = HALF * want.abs() + 2.0 ** -14 * size + (p.amax(0) * v.abs().amax(0) / 8 if eight else 0)
            assert ((got.double() - want).abs() <= bound).all(), (r, eight)

    def fork(self, parents, children):
        ok = self.pkg.pages.fork_requests(self.pool, dev_i32(np.asarray(parents)), dev_i32(np.asarray(children)))
        assert ok.all()
        for p, c in zip(parents, children):
            self.rows[c] = list(self.rows[p])

    def release(self, requests):
        self.pkg.pages.release_requests(self.pool, dev_i32(np.asarray(requests)))
        for r in requests:
            self.rows[r] = []


@pytest.mark.parametrize('seed', [0, 1])
def test_a_serving_run(pkg, seed):
    s = Serving(pkg, seed)
    s.step(np.array([100, 64, 33, 0, 0, 0, 0, 0, 0, 0]))        # prompts
    s.fork([0, 0, 1, 2, 2], [3, 4, 5, 6, 7])                    # samples, some on a page that is not full
    for _ in range(3):
        s.step(np.array([1, 0, 1, 1, 1, 1, 1, 1, 0, 0]))
    s.release([0, 4])
    s.fork([3], [8])
    s.step(np.array([40, 1, 0, 3, 0, 1, 1, 17, 1, 0]))          # a new prompt beside decoding and short chunks
    used = int((s.pool.refs > 0).sum())
    s.copy(pkg.pages.compact_pages(s.pool))
    assert (s.pool.refs[:used] > 0).all() and (s.pool.refs[used:] == 0).all()
    s.step(np.array([1, 1, 1, 1, 0, 1, 1, 1, 1, 0]))
    lengths = [len(x) for x in s.rows]
    assert s.pool.lengths.tolist() == lengths

    # latent rows are evicted: the pages of every request its own first, then the best rows to the front, then pages given back
    pg, cc = pkg.pages, pkg.compact_cache
    e = pg.extend_requests(s.pool, s.pool.lengths, torch.zeros_like(s.pool.lengths))
    assert e.ok.all()
    s.copy(e)
    assert int(s.pool.refs.max()) == 1
    M = max(lengths)
    account = torch.rand(R, M, generator=s.g, device='cuda')
    positions = torch.arange(M, dtype=torch.int32, device='cuda').expand(R, M).contiguous()
    keep = cc.select_rows(account, positions, s.pool.lengths, 50, s.pool.lengths - 8)
    before = cc.load_rows(s.latent, s.pool.tables, s.pool.lengths, M)
    cc.move_rows(s.latent, s.pool.tables, keep)
    pg.release_requests(s.pool, torch.arange(R, dtype=torch.int32, device='cuda'), keep.lengths)
    assert s.pool.lengths.tolist() == [min(50, n) for n in lengths]
    assert int((s.pool.refs > 0).sum()) == 1 + sum(-(-min(50, n) // BLOCK) for n in lengths)
    after = cc.load_rows(s.latent, s.pool.tables, s.pool.lengths, M)
    for r in range(R):
        n = min(50, lengths[r])
        assert torch.equal(after[r, :n], before[r, keep.positions[r, :n].long()])


def test_history_of_a_shared_latent_cache(pkg):
    """Samples on one prompt's pages read the same latent rows as requests with pages of their own."""
    s = Serving(pkg, 3)
    s.step(np.array([90, 0, 0, 0, 0, 0, 0, 0, 0, 0]))
    s.fork([0, 0], [1, 2])
    live, table, q, hist, counts = s.step(np.array([1, 1, 1, 0, 0, 0, 0, 0, 0, 0]))
    own = pkg.pages.new_pool(60, BLOCK, 3, 40 * BLOCK, 'cuda')
    assert pkg.pages.extend_requests(own, dev_i32(np.asarray([91] * 3))).ok.all()
    other = torch.full(pkg.compact_cache.cache_shape(60, BLOCK, W), 255, dtype=torch.uint8, device='cuda')
    for r in range(3):
        rows = torch.stack([x[2] for x in s.rows[r]])
        at = torch.arange(91, device='cuda')
        slots = own.tables[r].long()[at // BLOCK] * BLOCK + at % BLOCK
        pkg.compact_cache.store_rows(rows[:, :W], rows[:, W:], slots, other)
    want, _ = pkg.compact_cache.history_attention(q[:3], other, own.tables, counts[:3].contiguous(), SCALE, 91)
    assert torch.equal(want, hist[:3])


def test_attend_exact_takes_rows_that_are_there(pkg):
    """Without k and v the caller has written the rows; a profiling step has none; ``row_counts`` follows positions."""
    s = Serving(pkg, 4)
    s.step(np.array([20, 7, 0, 0, 0, 0, 0, 0, 0, 0]))
    layer, ops = pkg.s6_layer, pkg.s6_ops
    pos = torch.tensor([19, 6, 0], device='cuda')
    ctx = layer.StepContext(pos, dev_i32(np.asarray([0, 1, 2])), dev_i32(np.asarray([20, 7])), 1, 3, {}, SCALE, ops.HIP_BACKENDS)
    assert ctx.row_counts.tolist() == [20, 7, 0] and ctx.row_counts.dtype == torch.int32
    q = s.noise(3, H, D)
    out = layer.attend_exact(q, None, None, s.exact, s.pool.tables, ctx)
    out8 = layer.attend_exact(q, None, None, s.e4m3, s.pool.tables, ctx, s.scale, s.scale)
    s.check(0, q[0], out[0], out8[0])
    s.check(1, q[1], out[1], out8[1])
    assert (out[2] == 0).all()
    profile = layer.StepContext(pos, None, None, 1, 3, {}, SCALE, ops.HIP_BACKENDS)
    assert (layer.attend_exact(q, None, None, s.exact, s.pool.tables, profile) == 0).all()
