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
