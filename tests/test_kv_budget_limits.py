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
