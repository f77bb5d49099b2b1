"""Pools of pages on the GPU against the plain pool, and the copies against indexing: whole numbers and bytes, all equal."""
import numpy as np
import pytest
import torch

from pool_ref import Pool, held
from s6util import dev_i32

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def pg(pkg):
    return pkg.pages


def up(pg, pool, stride=0):
    """The device pool of a plain one; ``stride``: unused columns between the rows of its tables."""
    tables = np.asarray(pool.tables, np.int32).reshape(len(pool.tables), -1)
    wide = torch.full((tables.shape[0], tables.shape[1] + stride), 77, dtype=torch.int32, device='cuda')
    wide[:, :tables.shape[1]] = dev_i32(tables)
    return pg.Pool(wide[:, :tables.shape[1]], dev_i32(np.asarray(pool.lengths)), dev_i32(np.asarray(pool.refs)),
                   torch.from_numpy(pool.words().copy()).cuda(), pool.block)


def same(dev, pool):
    assert dev.lengths.tolist() == list(pool.lengths)
    assert dev.refs.tolist() == pool.refs
    assert dev.tables.tolist() == pool.tables
    assert (dev.free.cpu().numpy() == pool.words()).all()


def lists(got, pairs, R, cols, full):
    """The copy lists of an extension as the plain one has them."""
    want = np.full((2, R, cols), -1, np.int32)
    for r, p in enumerate(pairs):
        for c, pair in p.items():
            want[:, r, c] = pair
    if not full:
        assert all(len(p) <= 1 for p in pairs)
        want = want.max(-1) if cols else np.full((2, R), -1, np.int32)
    assert (got.source.cpu().numpy() == want[0]).all() and (got.target.cpu().numpy() == want[1]).all()


SHAPES = [  # requests, rows at most, block, spare pages
    (1, 1, 16, 0), (3, 40, 16, 5), (20, 300, 16, 40), (64, 500, 48, 200), (7, 33, 1, 100), (1500, 60, 16, 3000), (40, 5000, 8, 2000)]


@pytest.mark.parametrize('R,rows,block,spare', SHAPES)
def test_release(pg, R, rows, block, spare):
    rng = np.random.default_rng(R)
    n = rng.integers(0, rows + 1, R).tolist()
    cols = held(rows, block) + 1
    pool = Pool.random(rng, n, block, cols, sum(held(x, block) for x in n) + spare + 1, 0.4)
    pool.check()
    dev = up(pg, pool, 3)
    for k in range(3):
        requests = rng.integers(-1, R + 1, R // 2 + 1).tolist()       # repeated ones and numbers outside the pool among them
        lengths = None if k == 2 else rng.integers(-2, rows + block, len(requests)).tolist()
        pool.release(requests, lengths)
        pg.release_requests(dev, dev_i32(np.asarray(requests)), None if lengths is None else dev_i32(np.asarray(lengths)))
        same(dev, pool)
        pool.check()


@pytest.mark.parametrize('R,rows,block,spare', SHAPES)
def test_fork(pg, R, rows, block, spare):
    rng = np.random.default_rng(R + 1)
    n = [x if rng.random() < 0.5 else 0 for x in rng.integers(0, rows + 1, R).tolist()]
    pool = Pool.random(rng, n, block, held(rows, block) + 1, sum(held(x, block) for x in n) + spare + 1)
    dev = up(pg, pool)
    for _ in range(3):
        count = R + 3
        parents, children = (rng.integers(-1, R + 1, count).tolist() for _ in range(2))
        ok = pg.fork_requests(dev, dev_i32(np.asarray(parents)), dev_i32(np.asarray(children)))
        assert ok.tolist() == pool.fork(parents, children)
        same(dev, pool)
    empty, full = [r for r in range(R) if not pool.lengths[r]], [r for r in range(R) if pool.lengths[r]]
    if empty and full:       # every empty request from any other
        parents = rng.choice(full, len(empty)).tolist()
        ok = pg.fork_requests(dev, dev_i32(np.asarray(parents)), dev_i32(np.asarray(empty)))
        assert ok.all() and all(pool.fork(parents, empty))
        same(dev, pool)
        pool.check()


@pytest.mark.parametrize('full', [False, True])
@pytest.mark.parametrize('R,rows,block,spare', SHAPES)
def test_extend(pg, R, rows, block, spare, full):
    """Steps of single rows and of many, with and without enough pages; with rows that are to be rewritten."""
    rng = np.random.default_rng(R + 2 + full)
    n = rng.integers(0, rows + 1, R).tolist()
    cols = held(rows, block) + 2
    pool = Pool.random(rng, n, block, cols, sum(held(x, block) for x in n) + spare + 1, 0.6, reserved=1)
    pool.check(1)
    dev = up(pg, pool, 1)
    for step in range(6):
        more = rng.integers(0, (1, 2, block, 3 * block)[step % 4] + 1, R) + (step % 4 == 0)
        lengths = (np.asarray(pool.lengths) + more - (rng.random(R) < 0.2) * 7).tolist()
        if step == 4:
            lengths[R // 2] = 1 << 30
        write_from = rng.integers(-3, rows + 1, R).tolist() if full else None
        ok, pairs = pool.extend(lengths, write_from)
        got = pg.extend_requests(dev, dev_i32(np.asarray(lengths)), None if write_from is None else dev_i32(np.asarray(write_from)))
        assert got.ok.tolist() == ok
        lists(got, pairs, R, cols, full)
        same(dev, pool)
        pool.check(1)
        if step == 3:
            gone = rng.permutation(R)[:R // 3].tolist()
            pool.release(gone)
            pg.release_requests(dev, dev_i32(np.asarray(gone)))


def test_lengths_of_the_pool_itself(pg):
    """The pool's own lengths as an argument: what they were before the call."""
    rng = np.random.default_rng(9)
    pool = Pool.random(rng, [100, 20, 64, 7], 16, 8, 40)
    dev = up(pg, pool)
    order = [2, 0, 3, 1]
    pool.release(order, list(pool.lengths))
    pg.release_requests(dev, dev_i32(np.asarray(order)), dev.lengths)
    same(dev, pool)
    ok, _ = pool.extend(list(pool.lengths), list(pool.lengths))
    got = pg.extend_requests(dev, dev.lengths, dev.lengths)
    assert got.ok.tolist() == ok and (got.source == -1).all()
    same(dev, pool)


def test_parts_of_the_lengths(pg):
    """Arguments that lie on the pool's lengths, entries apart from those that they are for: what they were before the call."""
    rng = np.random.default_rng(10)
    n = rng.integers(0, 400, 300).tolist()
    pool = Pool.random(rng, n, 16, 30, sum(held(x, 16) for x in n) + 6000, 0.3)
    dev = up(pg, pool)
    order = list(range(299))
    pool.release(order, list(pool.lengths[1:]))
    pg.release_requests(dev, dev_i32(np.asarray(order)), dev.lengths[1:])
    same(dev, pool)
    for full in (False, True):
        long = torch.cat([dev.lengths, dev_i32(np.asarray([90]))])
        dev = pg.Pool(dev.tables, long[:-1], dev.refs, dev.free, dev.block)
        want, start = list(pool.lengths[1:]) + [90], [0] * 300 if full else None
        ok, pairs = pool.extend(want, start)
        got = pg.extend_requests(dev, long[1:], torch.zeros_like(dev.lengths) if full else None)
        assert got.ok.tolist() == ok
        lists(got, pairs, 300, 30, full)
        same(dev, pool)


def test_pages_run_out(pg):
    """The first request that asks for more than there is waits, and those behind it that ask for any."""
    pool = Pool.empty(10, 4, 6, 8)
    dev = up(pg, pool)
    for lengths in ([8, 12, 20, 4, 0, 0], [8, 12, 20, 0, 0, 4], [32, 12, 0, 0, 0, 0], [8, 32, 1, 0, 0, 0], [9, 12, 0, 0, 0, 20]):
        got = pg.extend_requests(dev, dev_i32(np.asarray(lengths)))
        ok, _ = pool.extend(lengths)
        assert got.ok.tolist() == ok
        same(dev, pool)
    assert not pool.free()
    assert not pg.extend_requests(dev, dev.lengths + 30).ok[pool.lengths.index(0)]


def test_a_large_pool(pg):
    """As many pages as a node's caches have, requests of thousands of pages; more words of bits than threads."""
    rng = np.random.default_rng(5)
    n = rng.integers(20000, 131000, 24).tolist()
    pages = sum(held(x, 16) for x in n) + 90000
    pool = Pool.random(rng, n, 16, held(131072, 16), pages, 0.2)
    dev = up(pg, pool)
    gone = [3, 9, 20, 21]
    pool.release(gone, [0, 5, 17000, 1 << 20])
    pg.release_requests(dev, dev_i32(np.asarray(gone)), dev_i32(np.asarray([0, 5, 17000, 1 << 20])))
    lengths = [min(131072, x + 5000) for x in pool.lengths]
    ok, pairs = pool.extend(lengths)
    got = pg.extend_requests(dev, dev_i32(np.asarray(lengths)))
    assert got.ok.tolist() == ok and all(ok)
    lists(got, pairs, len(n), held(131072, 16), False)
    same(dev, pool)
    movers, holes = pool.compact()
    moves = pg.compact_pages(dev)
    k = len(movers)
    assert k > 1000 and moves.source[:k].tolist() == movers and moves.target[:k].tolist() == holes and (moves.source[k:] == -1).all()
    same(dev, pool)


@pytest.mark.parametrize('R,rows,block,spare', SHAPES)
def test_compact(pg, R, rows, block, spare):
    rng = np.random.default_rng(R + 4)
    n = rng.integers(0, rows + 1, R).tolist()
    for reserved in (0, 3):
        pool = Pool.random(rng, n, block, held(rows, block) + 1, sum(held(x, block) for x in n) + spare + reserved, 0.3, reserved)
        pool.release(rng.permutation(R)[:R // 3].tolist())
        dev = up(pg, pool, 2)
        movers, holes = pool.compact()
        moves = pg.compact_pages(dev)
        k, N = len(movers), len(pool.refs)
        assert moves.source.tolist() == movers + [-1] * (N // 2 - k) and moves.target.tolist() == holes + [-1] * (N // 2 - k)
        same(dev, pool)
        pool.check(reserved)
        used = sum(x > 0 for x in pool.refs)
        assert all(pool.refs[:used]) and not any(pool.refs[used:])
        again = pg.compact_pages(dev)
        assert (again.source == -1).all() and (again.target == -1).all()
        same(dev, pool)


def test_a_pool_without_pages(pg):
    pool = pg.new_pool(0, 16, 2, 32, 'cuda')
    assert pg.extend_requests(pool, dev_i32(np.asarray([0, 5]))).ok.tolist() == [True, False]
    assert pg.compact_pages(pool).source.shape == (0,)
    pg.release_requests(pool, dev_i32(np.asarray([0, 1])))
    pool = pg.new_pool(5, 16, 0, 32, 'cuda')
    assert pg.extend_requests(pool, dev_i32(np.zeros(0))).ok.shape == (0,) and pg.compact_pages(pool).source.tolist() == [-1, -1]
    pool = pg.new_pool(5, 16, 2, 0, 'cuda')
    assert pg.extend_requests(pool, dev_i32(np.asarray([0, 1]))).ok.tolist() == [True, False]
    assert pg.extend_requests(pool, dev_i32(np.asarray([0, 1])), dev_i32(np.asarray([0, 0]))).ok.tolist() == [True, False]


@pytest.mark.parametrize('shape,dtype,odd', [((50, 1, 16, 1024), torch.bfloat16, False), ((50, 1, 17 * 128), torch.uint8, False),
                                            ((50, 16, 16, 256), torch.bfloat16, False), ((40, 3, 5), torch.uint8, True),
                                            ((40, 7), torch.int32, True), ((30,), torch.float32, True),
                                            ((20, 2, 16, 128), torch.float8_e4m3fn, False), ((12, 1, 16, 20000), torch.bfloat16, True)])
@pytest.mark.parametrize('count', [1, 7, 5000])
def test_copies(pg, shape, dtype, odd, count):
    """Pages of every size, aligned or not, in lists that are full or nearly empty, of one cache and of many."""
    g = torch.Generator(device='cuda').manual_seed(count)
    N = shape[0]
    bytes_ = torch.Size(shape).numel() * torch.empty(0, dtype=dtype).element_size()
    caches = [torch.randint(0, 256, (bytes_,), dtype=torch.uint8, generator=g, device='cuda').view(dtype).view(shape)
              for _ in range(1 if count == 7 else 5)]
    if len(shape) == 4 and shape[1] > 1:
        caches = [c.transpose(1, 2) for c in caches]
    perm = torch.randperm(N, generator=g, device='cuda').to(torch.int32)
    pairs = min(count, N // 2)
    source, target = torch.full((2, count), -1, dtype=torch.int32, device='cuda')
    at = torch.randperm(count, generator=g, device='cuda')[:pairs]
    source[at], target[at] = perm[:pairs], perm[N - pairs:]
    if count == 5000:
        source[at[0]], target[at[1]], source[at[2]], target[at[3]] = N, -3, 1 << 30, N       # numbers outside: skipped
        target[at[4]] = source[at[4]]
    good = (source >= 0) & (source < N) & (target >= 0) & (target < N)
    raw = lambda c: (c.transpose(1, 2) if len(shape) == 4 and shape[1] > 1 else c).contiguous().view(-1).view(torch.uint8).view(N, -1)
    want = [raw(c).clone() for c in caches]
    for w in want:
        w[target[good].long()] = w[source[good].long()]
    pg.copy_pages(caches, source, target)
    assert all(torch.equal(raw(c), w) for c, w in zip(caches, want))


def test_copies_of_caches_in_larger_tensors(pg):
    big = torch.randint(0, 256, (20, 3, 512), dtype=torch.uint8, device='cuda')
    want = big.clone()
    want[[3, 4], 1] = want[[7, 11], 1]
    pg.copy_pages(big[:, 1], dev_i32(np.asarray([7, 11])), dev_i32(np.asarray([3, 4])))
    assert torch.equal(big, want)
    many = [torch.randint(0, 256, (6, 64), dtype=torch.uint8, device='cuda') for _ in range(300)]     # more than one launch takes
    was = [m.clone() for m in many]
    pg.copy_pages(many, dev_i32(np.asarray([[5], [0]])), dev_i32(np.asarray([[1], [2]])))
    assert all(torch.equal(m[1], w[5]) and torch.equal(m[2], w[0]) and torch.equal(m[3:], w[3:]) for m, w in zip(many, was))
    pg.copy_pages([], dev_i32(np.asarray([0])), dev_i32(np.asarray([1])))


def test_refusals(pg):
    pool, one = pg.new_pool(8, 16, 2, 64, 'cuda'), dev_i32(np.asarray([0]))
    two = dev_i32(np.asarray([0, 1]))
    for call, match in ((lambda: pg.release_requests(pool, one.long()), 'requests'), (lambda: pg.release_requests(pool, one, two), 'lengths'),
                        (lambda: pg.fork_requests(pool, one, two), 'children'), (lambda: pg.extend_requests(pool, one), 'lengths'),
                        (lambda: pg.extend_requests(pool, two, one), 'write_from'),
                        (lambda: pg.Pool(pool.tables, one, pool.refs, pool.free, 16), 'lengths'),
                        (lambda: pg.Pool(pool.tables, pool.lengths, torch.zeros(40, dtype=torch.int32, device='cuda'), pool.free, 16), 'free'),
                        (lambda: pg.Pool(pool.tables.t(), pool.lengths, pool.refs, pool.free, 16), 'tables'),
                        (lambda: pg.Pool(pool.tables, pool.lengths, torch.zeros(16, dtype=torch.int32, device='cuda')[::2], pool.free, 16),
                         'contiguous'),
                        (lambda: pg.Pool(pool.tables, pool.lengths.long(), pool.refs, pool.free, 16), 'lengths'),
                        (lambda: pg.Pool(pool.tables, pool.lengths, pool.refs, pool.free, 0), 'no pool')):
        with pytest.raises(ValueError, match=match):
            call()
    for call in (lambda: pg.fork_requests(pool, one, one.cpu()), lambda: pg.Pool(pool.tables, pool.lengths.cpu(), pool.refs, pool.free, 16)):
        with pytest.raises(RuntimeError):
            call()
    c = torch.zeros(8, 4, 6, device='cuda')
    for caches, a, b, match in (([c, c[:4]], one, one, 'one shape'), ([c, c.half()], one, one, 'one shape'), (c[:, :, :5], one, one, 'dense'),
                                (c[:, ::2], one, one, 'dense'), (c[:1].expand(8, 4, 6), one, one, 'apart'), (c, one, two, 'one shape'),
                                (c, one.long(), one.long(), 'int32')):
        with pytest.raises(ValueError, match=match):
            pg.copy_pages(caches, a, b)


def test_replayed_graphs(pg):
    """A captured turn of a pool (release, fork, extend, copies), replayed; the plain pool goes along."""
    rng = np.random.default_rng(8)
    pool = Pool.random(rng, [100, 37, 64, 0, 0, 0, 0], 16, 12, 60)
    dev = up(pg, pool)
    cache = torch.randint(0, 256, (60, 512), dtype=torch.uint8, device='cuda')
    children, parents = [3, 4, 5, 6], [0, 1, 2, 0]
    kids, mums, target = dev_i32(np.asarray(children)), dev_i32(np.asarray(parents)), dev_i32(np.asarray([100, 37, 64, 101, 38, 65, 120]))

    def turn():
        pg.release_requests(dev, kids)
        ok = pg.fork_requests(dev, mums, kids)
        e = pg.extend_requests(dev, target)
        pg.copy_pages(cache, e.source, e.target)
        return ok, e

    def plain():
        pool.release(children)
        assert all(pool.fork(parents, children))
        return pool.extend(target.tolist())

    turn()
    plain()
    torch.cuda.synchronize()
    same(dev, pool)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ok, e = turn()
    for lengths in ([100, 37, 64, 101, 38, 65, 120], [101, 37, 70, 150, 38, 65, 180], [101, 40, 70, 102, 300, 71, 102]):
        target.copy_(dev_i32(np.asarray(lengths)))
        graph.replay()
        want, pairs = plain()
        assert ok.all() and e.ok.tolist() == want
        lists(e, pairs, 7, 12, False)
        same(dev, pool)
        for p in pairs:
            for a, b in p.values():
                assert torch.equal(cache[a], cache[b])
