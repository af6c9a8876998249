"""The paged key-value cache's C ABI without a GPU: what the entries refuse, and
that a valid call reports the missing GPU instead of falling back."""

import ctypes

import pytest

INVALID, INTERNAL = 1, 3


def structs():
    from mlxvs_amd import kvcache

    return kvcache._Cache, kvcache._Queries


P = 4096  # any 16-byte aligned address: nothing is read before the checks pass


def cache(**k):
    C, _ = structs()
    f = dict(keys=P, values=P, summaries=P, scales=P, pages=4, heads=2, page_size=16, dim=64, type=1)
    f.update(k)
    return C(*[f[n] for n, _ in C._fields_])


def queries(**k):
    _, Q = structs()
    f = dict(q=P, token_stride=512, head_stride=64, tokens=3, q_heads=8, columns=5, table=P,
             table_stride=5, requests=2, token_request=P, positions=P)
    f.update(k)
    return Q(*[f[n] for n, _ in Q._fields_])


def attend(lib, c, q, blocks=None, n=0, scale=0.125, longest=0, out=P, work=None, size=0):
    return lib.mlxvs_kv_attend_device(ctypes.byref(c), ctypes.byref(q), blocks, n, scale, longest,
                                      out, None, work, size, None)


def select(lib, c, q, n=4, first=1, last=1, blocks=P):
    return lib.mlxvs_kv_select_device(ctypes.byref(c), ctypes.byref(q), n, first, last, blocks,
                                      None, 0, None)


@pytest.mark.parametrize("bad", [
    dict(page_size=24), dict(page_size=8), dict(page_size=512), dict(page_size=0), dict(dim=60),
    dict(dim=0), dict(dim=264), dict(heads=0), dict(pages=-1), dict(pages=1 << 31), dict(keys=None),
    dict(values=None), dict(keys=P + 2), dict(scales=None), dict(type=2)])
def test_caches_that_are_refused(engine, bad):
    lib = engine._L()
    for call in (attend, select):
        assert call(lib, cache(**bad), queries()) == INVALID
        assert b"[mlxvs" in lib.mlxvs_last_error()
    assert lib.mlxvs_kv_append_device(ctypes.byref(cache(**bad)), P, 64, 64, P, 64, 64, P, 3,
                                      None) == INVALID
    assert lib.mlxvs_kv_attend_workspace(ctypes.byref(cache(**bad)), ctypes.byref(queries()), 0,
                                         0) == -1


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(q=P + 8), dict(token_stride=12), dict(head_stride=4), dict(tokens=-1),
    dict(q_heads=7), dict(q_heads=0), dict(q_heads=1), dict(columns=-1), dict(table=None),
    dict(columns=1 << 28, table_stride=1 << 28), dict(table_stride=4), dict(requests=-1),
    dict(token_request=None), dict(positions=None), dict(tokens=1 << 31)])
def test_queries_that_are_refused(engine, bad):
    lib = engine._L()
    for call in (attend, select):
        assert call(lib, cache(), queries(**bad)) == INVALID
        assert b"[mlxvs::kv_" in lib.mlxvs_last_error()


def test_arguments_that_are_refused(engine):
    lib = engine._L()
    c, q = cache(), queries()
    for k in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(longest=-1),
              dict(out=None), dict(out=P + 8), dict(n=4), dict(blocks=P, n=0), dict(blocks=P, n=257)):
        assert attend(lib, c, q, **k) == INVALID, k
    for k in (dict(n=0), dict(n=257), dict(first=-1), dict(last=0), dict(first=3, last=2),
              dict(blocks=None)):
        assert select(lib, c, q, **k) == INVALID, k
    assert select(lib, cache(summaries=None, scales=None), q) == INVALID
    # a workspace that a call needs and does not get
    long = queries(tokens=1, columns=4096, table_stride=4096)
    need = lib.mlxvs_kv_attend_workspace(ctypes.byref(c), ctypes.byref(long), 0, 0)
    assert need > 0
    assert attend(lib, c, long) == INVALID and b"workspace" in lib.mlxvs_last_error()
    assert attend(lib, c, long, work=P, size=need - 1) == INVALID
    for a in ((None, 64, 64, P, 64, 64, P, 3), (P, 60, 64, P, 64, 64, P, 3),
              (P, 64, 64, P + 4, 64, 64, P, 3), (P, 64, 64, P, 64, 64, None, 3),
              (P, 64, 64, P, 64, 64, P, -1)):
        assert lib.mlxvs_kv_append_device(ctypes.byref(c), *a, None) == INVALID
    assert lib.mlxvs_kv_attend_device(None, ctypes.byref(q), None, 0, 1.0, 0, P, None, None, 0,
                                      None) == INVALID
    assert lib.mlxvs_kv_attend_device(ctypes.byref(c), None, None, 0, 1.0, 0, P, None, None, 0,
                                      None) == INVALID


def plan(lib, **k):
    f = dict(past=P, fresh=P, requests=3, table=P, stride=5, columns=5, free=P, count=9, cursor=P,
             page=16, tokens=8, slots=P, who=P, where=P, starts=P, lengths=P + 12, first=P, out=P + 4)
    f.update(k)
    return lib.mlxvs_kv_plan_device(*f.values(), None)


@pytest.mark.parametrize("bad", [
    dict(past=None), dict(fresh=None), dict(requests=-1), dict(table=None), dict(stride=4),
    dict(columns=-1), dict(columns=1 << 28, stride=1 << 28), dict(free=None), dict(count=-1),
    dict(cursor=None), dict(page=15), dict(tokens=-1), dict(slots=None), dict(who=None),
    dict(where=None), dict(starts=None), dict(lengths=None), dict(first=None), dict(out=None),
    dict(out=P), dict(lengths=P), dict(lengths=P + 8)])
def test_plans_that_are_refused(engine, bad):
    lib = engine._L()
    assert plan(lib, **bad) == INVALID
    assert b"[mlxvs::kv_plan]" in lib.mlxvs_last_error()


def test_no_fallback_without_a_gpu(engine):
    import mlxvs_amd._hip as hip

    if hip.device_count() > 0:
        pytest.skip("a GPU is present")
    lib = engine._L()
    for rc in (plan(lib), attend(lib, cache(), queries()), select(lib, cache(), queries())):
        assert rc == INTERNAL
        assert b"no HIP device" in lib.mlxvs_last_error()
    with pytest.raises(ValueError, match="GPU tensor"):
        import torch

        t = torch.zeros(1, dtype=torch.int32)
        engine.kv_plan(t, t, t[None], t, t, 16, 4)


def test_workspace_of_calls_without_tokens(engine):
    lib = engine._L()
    none = queries(tokens=0, q=None, token_request=None, positions=None)
    assert lib.mlxvs_kv_attend_workspace(ctypes.byref(cache()), ctypes.byref(none), 0, 0) == 0
    assert lib.mlxvs_kv_select_workspace(ctypes.byref(cache()), ctypes.byref(none), 4) == 0
    assert attend(lib, cache(), none) == 0 and select(lib, cache(), none) == 0
