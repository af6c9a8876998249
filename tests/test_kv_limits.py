"""How large a call of the paged key-value cache may be, without a GPU: what the
launches have room for is not refused, and what they have not is."""

import ctypes

import pytest

from test_kv_abi import INTERNAL, INVALID, attend, cache, queries, select


@pytest.fixture(autouse=True)
def no_gpu():
    import mlxvs_amd._hip as hip

    if hip.device_count() > 0:
        pytest.skip("a GPU is present: the addresses are nobody's")


@pytest.mark.parametrize("tokens,columns,requests,rc", [
    (600_000, 5, 2, INTERNAL),             # by tiles of 16 tokens: 600,000 workgroups
    (2_000_000, 5, 2_000_000, INTERNAL),   # a row a workgroup: 16 million
    (2_200_000, 5, 2_200_000, INVALID),    # 17.6 million of 256 threads: past 2^32
    (16_000_000, 5, 2, INTERNAL),
    (400_000, 9_000, 400_000, INVALID),    # 71 parts each
    (500_000, 1_025, 500_000, INTERNAL)])
def test_selections_of_many_rows(engine, tokens, columns, requests, rc):
    lib = engine._L()
    q = queries(tokens=tokens, columns=columns, table_stride=columns, requests=requests)
    assert select(lib, cache(heads=8), q) == rc, lib.mlxvs_last_error()


@pytest.mark.parametrize("tokens,rc", [(1, INTERNAL), (1024, INTERNAL), (10_000_000, INTERNAL),
                                       (33_000_000, INTERNAL), (34_000_000, INVALID)])
def test_appends_of_many_tokens(engine, tokens, rc):
    # by 16 tokens and a head a workgroup: 16.8 million at most
    lib = engine._L()
    assert lib.mlxvs_kv_append_device(ctypes.byref(cache(heads=8)), 4096, 64, 64, 4096, 64, 64, 4096,
                                      tokens, None) == rc, lib.mlxvs_last_error()


@pytest.mark.parametrize("tokens,requests,rc", [
    (600_000, 600_000, INTERNAL),       # single tokens of short requests: a row a workgroup
    (2_200_000, 2_200_000, INVALID),    # 17.6 million
    (2_200_000, 3, INTERNAL)])          # prompts share workgroups
def test_attention_of_many_tokens(engine, tokens, requests, rc):
    q = queries(tokens=tokens, requests=requests, q_heads=32, token_stride=2048)
    lib = engine._L()
    assert attend(lib, cache(heads=8), q) == rc, lib.mlxvs_last_error()


@pytest.mark.parametrize("tokens_held,longest,keys", [
    (1 << 20, 0, 4096),        # a million places: 256 parts of 8 kv heads
    (1 << 18, 0, 2048),
    (1 << 20, 1 << 20, 16384),  # the caller says that they are taken
    (1 << 20, 16_000, 512)])
def test_parts_of_a_single_token_in_a_wide_table(engine, tokens_held, longest, keys):
    lib = engine._L()
    c = cache(heads=8, page_size=64, dim=128)
    q = queries(tokens=1, q_heads=32, columns=tokens_held // 64, table_stride=tokens_held // 64)
    size = lib.mlxvs_kv_attend_workspace(ctypes.byref(c), ctypes.byref(q), 0, longest)
    parts = -(-(min(tokens_held, longest) if longest else tokens_held) // keys)
    assert size == 32 * parts * (128 + 2) * 4
