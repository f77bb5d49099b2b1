"""CPU checks of what whole exact caches and pools of pages refuse because a launch cannot hold it: 2^32 threads and more."""
import pytest


@pytest.fixture(scope='module')
def refused(pkg):
    lib = pkg._lib

    def refused(name, arguments, match):
        args = [None if t is lib.P else 0 for t in lib.SIGNATURES[name]]
        for i, v in arguments.items():
            args[i] = v
        with pytest.raises(ValueError, match=match):
            lib.call(name, *args)

    return refused


#: 1 token of 8 query heads over 2 KV heads, d = 64
ATTENTION = {0: 16, 1: 1, 2: 8, 3: 64, 4: 512, 5: 64, 6: 16, 8: 2, 9: 4096, 10: 128, 11: 256, 12: 16, 13: 2, 14: 16, 15: 1, 16: 1, 17: 1,
             19: 16, 28: 16, 29: 512, 30: 64, 31: 16}


@pytest.mark.parametrize('what', [
    {1: 2 ** 23, 17: 2 ** 23},                                              # a workgroup per token and KV head: 2^24
    {1: 2 ** 21, 17: 2 ** 21, 24: 4, 26: 16, 27: 10 ** 9},                  # shares: few workgroups, but 2^24 to join the parts
    {1: 2 ** 20, 2: 1024, 8: 128, 10: 128, 11: 2 ** 14, 17: 2 ** 20, 25: 16},   # groups of 4 tokens, 16 workgroups for each: 2^29
    {1: 2 ** 19, 2: 2 ** 13, 8: 2 ** 10, 10: 128, 11: 2 ** 17, 17: 2 ** 19, 25: 16},   # (more than 32 bits count)
    {1: 2 ** 15, 2: 2 ** 16, 8: 2 ** 16, 10: 128, 11: 2 ** 23, 17: 2 ** 15}])
def test_attention_of_too_many_rows(refused, what):
    refused('hla_s6_exact_attention', {**ATTENTION, **what}, 'too many rows')


def test_lists_that_are_too_long(refused):
    store = {0: 16, 1: 128, 2: 64, 3: 16, 4: 128, 5: 64, 7: 2, 8: 64, 9: 16, 12: 16, 14: 4096, 15: 128, 16: 256, 17: 16, 18: 2}
    for tokens in (2 ** 27, 2 ** 31 - 1):       # 32 threads each
        refused('hla_s6_exact_store', {**store, 6: tokens}, 'too many rows')
    pool = {0: 16, 1: 4, 2: 2, 3: 4, 4: 16, 5: 16, 6: 8, 7: 16, 8: 16, 9: 16}
    for count in (2 ** 24, 2 ** 31 - 1):
        refused('hla_s6_pool_release', {**pool, 11: count}, 'too long')
    for page, count in ((64, 2 ** 30), (2 ** 38, 1), (2 ** 37, 2), (2 ** 45, 2 ** 40), (64, 2 ** 63 - 1), (2 ** 62, 2 ** 62)):
        refused('hla_s6_copy_pages', {0: 16, 1: 1, 2: page, 3: page, 4: 4, 5: 16, 6: 16, 7: count}, 'too long')
