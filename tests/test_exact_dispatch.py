"""CPU checks of how ``exact_cache.attention`` deals a step to workgroups, from host numbers alone; nothing is launched."""
import pytest
import torch


@pytest.fixture
def dealt(pkg, monkeypatch):
    """``(shares, grouped, shared_rows)`` of a call with 256 CUs."""
    ec = pkg.exact_cache
    calls = []
    monkeypatch.setattr(ec, '_same_device', lambda *a: None)
    monkeypatch.setattr(ec, '_call', lambda name, device, *args: calls.append(args))
    monkeypatch.setattr(ec._lib, 'device_cus', lambda index: 256)

    def dealt(tokens, requests, kv_heads, group, longest, max_query_len=None, per_request=True, **more):
        cache = torch.empty(4, kv_heads, 16, 128, dtype=torch.bfloat16)
        q = torch.empty(tokens, kv_heads * group, 64, dtype=torch.bfloat16)
        table = torch.empty(requests, -(-longest // 16), dtype=torch.int32)
        ec.attention(q, cache, table, torch.zeros(tokens, dtype=torch.int32), 1.0, longest,
                     torch.zeros(tokens, dtype=torch.int64) if per_request else None, max_query_len=max_query_len, **more)
        args = calls.pop()
        return args[24], args[25], args[32]

    return dealt


def test_who_reads_the_same_rows(dealt):
    """A table with rows to spare says nothing about the tokens of a request where the caller does."""
    assert dealt(64, 1, 8, 4, 8160, 64)[2] == 1 and dealt(64, 256, 8, 4, 8160, 64)[2] == 1
    assert dealt(64, 1, 8, 4, 8160)[2] == 1 and dealt(64, 64, 8, 4, 8160)[2] == 0
    assert dealt(64, 64, 8, 4, 8160, 1)[2] == 0 and dealt(130, 64, 8, 4, 8160, 1)[2] == 0      # (padding)
    assert dealt(64, 64, 8, 4, 8160, per_request=False)[2] == 0 and dealt(64, 64, 8, 4, 8160, 64, per_request=False)[2] == 0


def test_requests_of_a_step(dealt):
    """Nor how many requests there are: one that takes max_query_len of the tokens leaves few to others."""
    assert dealt(4000, 1, 16, 1, 4000, 4000)[1] == 4 and dealt(4000, 256, 16, 1, 4000, 4000)[1] == 4
    assert dealt(4016, 256, 16, 1, 4000, 4000)[1] == 4 and dealt(576, 65, 16, 1, 4000, 512)[1] == 16
    assert dealt(256, 32, 16, 1, 4000, 8)[1] == 16 and dealt(256, 1000, 16, 1, 4000, 8)[1] == 16


def test_tokens_alone_beside_chunks(dealt, pkg):
    """Shares for tokens alone beside groups, where there can be any and rows are long."""
    most = pkg.exact_cache._most_alone
    assert most(2048, 4, 512) == 0 and most(2049, 5, 512) == 1 and most(513, 2, 512) == 1 and most(4000, 256, 4000) == 0
    assert most(576, 65, 512) == 64 and most(576, 300, 512) == 64 and most(100, 4, 512) == 0 and most(12, 4, 8) == 2
    assert dealt(513, 2, 8, 4, 131000, 512)[:2] == (64, 4) and dealt(4016, 17, 16, 1, 8160, 4000)[:2] == (32, 4)
    assert dealt(513, 2, 8, 4, 4095, 512)[:2] == (0, 4) and dealt(2048, 4, 16, 1, 8160, 512)[:2] == (0, 4)
    assert dealt(513, 2, 8, 4, 131000)[:2] == (64, 4) and dealt(513, 1, 8, 4, 131000)[:2] == (0, 4)
    assert dealt(513, 2, 8, 4, 131000, 512, shares=3)[:2] == (3, 0) and dealt(64, 2, 8, 4, 131000, 63)[:2] == (64, 0)


def test_a_long_row_among_many_groups(dealt):
    """Many groups take a workgroup each only as long as none of them takes much longer than the others together."""
    assert dealt(256, 256, 16, 1, 131000, 1)[0] == 32 and dealt(256, 256, 16, 1, 8160, 1)[0] == 32
    assert dealt(256, 256, 16, 1, 4096, 1)[0] == 0 and dealt(256, 256, 16, 1, 4097, 1)[0] == 32
    assert dealt(512, 512, 16, 1, 8192, 1)[0] == 0 and dealt(512, 512, 16, 1, 131000, 1)[0] == 32
