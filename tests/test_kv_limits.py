"""How large a call of the paged key-value cache may be, without a GPU: what the
launches have room for is not refused, and what they have not is."""

import pytest

from test_kv_abi import INTERNAL, INVALID, cache, queries, select


@pytest.mark.parametrize("tokens,columns,requests,rc", [
    (600_000, 5, 2, INTERNAL),             # by tiles of 16 tokens: 600,000 workgroups
    (2_000_000, 5, 2_000_000, INTERNAL),   # a row a workgroup: 16 million
    (2_200_000, 5, 2_200_000, INVALID),    # 17.6 million of 256 threads: past 2^32
    (16_000_000, 5, 2, INTERNAL),
    (400_000, 9_000, 400_000, INVALID),    # 71 parts each
    (500_000, 1_025, 500_000, INTERNAL)])
def test_selections_of_many_rows(engine, tokens, columns, requests, rc):
    import mlxvs_amd._hip as hip

    if hip.device_count() > 0:
        pytest.skip("a GPU is present: the addresses are nobody's")
    lib = engine._L()
    q = queries(tokens=tokens, columns=columns, table_stride=columns, requests=requests)
    assert select(lib, cache(heads=8), q) == rc, lib.mlxvs_last_error()
