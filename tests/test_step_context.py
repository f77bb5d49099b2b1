"""CPU checks of what a StepContext keeps about its latent lengths, and of how much scratch a step may take (the GPU side:
test_gpu_compact_edges.py)."""
import contextlib

import pytest
import torch


@pytest.fixture
def step(pkg, monkeypatch):
    """A StepContext without a GPU: plans are the lengths that they were made for."""
    made = []

    def split_plans(ctx, cap, splits, query_start_loc=None):
        made.append(ctx.tolist())
        return [(s, ctx.tolist()) for s in splits]

    monkeypatch.setattr(pkg.s6_ops, 'split_plans', split_plans)
    monkeypatch.setattr(pkg.s6_layer._lib, 'call', lambda *a: None)
    monkeypatch.setattr(pkg.s6_layer._lib, 'stream', lambda *a: 0)

    def make():
        i32 = lambda *a: torch.tensor(a, dtype=torch.int32)
        ctx = pkg.s6_layer.StepContext(torch.tensor([5, 9]), i32(0, 1, 2), i32(6, 10), 1, 2, {}, 1.0, None, num_kv_splits=4)
        ctx.ctx_latent.copy_(i32(5, 0))
        return ctx, made
    return make


@pytest.mark.parametrize('mode', [contextlib.nullcontext, torch.no_grad, torch.inference_mode])
def test_plans_follow_the_lengths(step, mode):
    with mode():
        ctx, made = step()
        assert ctx.split_plan(4, 64) == (4, [5, 0]) and ctx.empty_latent.tolist() == [False, True]
        assert ctx.split_plan(4, 64) == (4, [5, 0]) and len(made) == 1     # once per step
        ctx.ctx_latent[:] = 7                                              # in place
        assert ctx.split_plan(4, 64) == (4, [7, 7]) and ctx.empty_latent.tolist() == [False, False]
        ctx.ctx_latent = torch.tensor([0, 3], dtype=torch.int32)           # assigned
        assert ctx.split_plan(4, 64) == (4, [0, 3]) and ctx.empty_latent.tolist() == [True, False]
        assert ctx.split_plan(4, 128) == (4, [0, 3])
        ctx.ctx_latent.add_(1)
        assert ctx.split_plan(4, 64) == (4, [1, 4]) and ctx.empty_latent.tolist() == [False, False]
        assert ctx.split_plan(4, 128) == (4, [1, 4])


def test_scratch_of_expanded_rows_is_bounded(pkg):
    shape = pkg.compact_cache.history_shape
    assert shape(32736, 2048, 4, 256, 512) == (3, 1) and shape(32768, 2048, 4, 256, 512) == (3, 1)
    assert shape(32769, 2048, 4, 256, 512) == (2, 1) and shape(32736, 16384, 32, 256, 512) == (2, 1)
    assert shape(131072, 4096, 1, 256, 512) == (3, 1) and shape(131073, 4096, 1, 256, 512) == (2, 1)
    assert shape(300, 4096, 0, 256, 512) == (2, 1)             # no requests: nothing to expand
