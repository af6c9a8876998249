"""Which calls of the paged cache's budget are served, and by which kernels, without
a GPU: by their workspaces and by what they refuse."""

import ctypes

import pytest

from test_kv_abi import cache, queries


def weigh_workspace(engine, c, q, longest=0):
    return engine._L().mlxvs_kv_weigh_workspace(ctypes.byref(c), ctypes.byref(q), longest)


@pytest.mark.parametrize("requests", [1, 2, 40])
def test_a_cache_without_pages_has_no_prompts(engine, requests):
    # the kernel of prompts (the one that needs a workspace) reads some key in
    # place of an absent one
    q = queries(tokens=5000, requests=requests, columns=320, table_stride=320)
    assert weigh_workspace(engine, cache(), q) > 0
    assert weigh_workspace(engine, cache(pages=0, keys=None, values=None), q) == 0
    assert weigh_workspace(engine, cache(pages=0), q) == 0


@pytest.mark.parametrize("requests,held", [(512, 1 << 20), (4_096, 1 << 17), (300_000, 1 << 20),
                                           (2_000_000, 5 * 64)])
def test_weights_of_single_tokens_in_wide_tables(engine, requests, held):
    # what attention over the same cache serves, whatever the table has room for
    q = queries(tokens=requests, requests=requests, columns=held // 64, table_stride=held // 64)
    c = cache(heads=8, page_size=64)
    lib = engine._L()
    assert weigh_workspace(engine, c, q) >= 0, lib.mlxvs_last_error()
    assert weigh_workspace(engine, c, q, 1_000) >= 0
    assert lib.mlxvs_kv_attend_workspace(ctypes.byref(c), ctypes.byref(q), 0, 1_000) >= 0
    # prompts beside them
    q = queries(tokens=requests + 300, requests=requests, columns=5, table_stride=5)
    assert weigh_workspace(engine, c, q) > 0


def test_weights_of_too_many_requests(engine):
    # a workgroup of 256 threads for each request and head: past 2^32
    q = queries(tokens=2_200_000, requests=2_200_000)
    assert weigh_workspace(engine, cache(heads=8), q) == -1
    assert b"too many tokens" in engine._L().mlxvs_last_error()
    assert weigh_workspace(engine, cache(heads=1 << 16), queries(
        tokens=9, q_heads=1 << 16, requests=(1 << 31) - 1, columns=1 << 22, table_stride=1 << 22)) == -1
    assert weigh_workspace(engine, cache(heads=8), queries(tokens=0, requests=0)) == 0
    assert weigh_workspace(engine, cache(heads=8), queries(tokens=9, requests=0)) >= 0


@pytest.mark.parametrize("tokens,requests,held,longest,dealt", [
    (64, 64, 8_192, 0, False),        # 4 million keys in 8 heads
    (256, 256, 4_096, 0, True),       # 8 million
    (256, 256, 1 << 17, 4_032, False),
    (256, 256, 1 << 17, 4_096, True),
    (32, 32, 1 << 20, 0, False), (33, 33, 1 << 20, 0, True),  # (up to 32 rows are few)
    (200, 512, 4_096, 0, True),       # fewer tokens than rows
    (200, 512, 2_047, 2_000, False),
    (1_024, 1_024, 4_096, 0, True), (1_025, 1_025, 4_096, 0, False),  # (the plan takes too long)
    (3, 2, 64, 0, True), (2, 2, 64, 0, False), (0, 512, 1 << 17, 0, False)])
def test_which_requests_are_dealt(engine, tokens, requests, held, longest, dealt):
    # the device finds the prompts among them (and needs a workspace) where single tokens
    # could take long, or where there are more of them than rows of the table
    columns = -(-held // 64)
    q = queries(tokens=tokens, requests=requests, columns=columns, table_stride=columns)
    need = weigh_workspace(engine, cache(heads=8, page_size=64), q, longest)
    assert need > 0 if dealt else need == 0
    # (64 rows of Q are a tile: more query heads than that are always taken one by one)
    q = queries(tokens=tokens, requests=requests, columns=columns, table_stride=columns, q_heads=8 * 65)
    assert weigh_workspace(engine, cache(heads=8, page_size=64), q, longest) == 0


@pytest.mark.parametrize("group", [33, 64])
def test_single_tokens_of_many_query_heads_are_not_dealt(engine, group):
    # one token's rows are no prompt: there has to be another one
    c = cache(heads=8, page_size=64)
    for tokens, dealt in ((1, False), (2, True)):
        q = queries(tokens=tokens, requests=512, columns=64, table_stride=64, q_heads=8 * group)
        assert (weigh_workspace(engine, c, q) > 0) == dealt
