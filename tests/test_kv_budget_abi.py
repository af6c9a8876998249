"""The budget's entries of the paged key-value cache without a GPU: what they
refuse, the frequencies of positions, and that a valid call reports the missing
GPU."""

import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest

import kv_budget_oracle
from test_kv_abi import INTERNAL, INVALID, P, cache, queries


def lib_of(engine):
    return engine._L()


def rotary(**k):
    from mlxvs_amd import kvcache

    f = dict(turns=P, dim=64, rotated=32, layout=0, magnitude=1.0, type=1)
    f.update(k)
    return kvcache._Rotary(*[f[n] for n, _ in kvcache._Rotary._fields_])


def heads(**k):
    from mlxvs_amd import kvcache

    f = dict(x=P, token_stride=512, head_stride=64, heads=8, norm=None, norm_type=0, out=P,
             out_token_stride=512, out_head_stride=64)
    f.update(k)
    return kvcache._Heads(*[f[n] for n, _ in kvcache._Heads._fields_])


def rotate(lib, rot=None, q=None, k=None, tokens=3, positions=P, who=None, evicted=None,
           requests=0, eps=1e-6):
    ref = lambda x: None if x is None else ctypes.byref(x)  # noqa: E731
    return lib.mlxvs_kv_rotate_device(ref(rot), ref(q), ref(k), tokens, positions, who, evicted,
                                      requests, eps, None)


def weigh(lib, c=None, q=None, starts=P, lse=P, scale=0.125, decay=1.0, longest=0, mass=P, slots=80,
          work=P, size=1 << 30):
    return lib.mlxvs_kv_weigh_device(ctypes.byref(c or cache()), ctypes.byref(q or queries()), starts,
                                     lse, scale, decay, longest, mass, slots, work, size, None)


def keep(lib, **k):
    f = dict(mass=P, requests=2, heads=2, slots=80, lengths=P, n=16, first=1, recent=1, above=16,
             kept=P, work=P, size=1 << 40)
    f.update(k)
    return lib.mlxvs_kv_keep_device(*f.values(), None)


def compact(lib, c=None, work=P, size=1 << 20, **k):
    f = dict(table=P, stride=5, columns=5, requests=2, lengths=P, kept=P, n=16, free=P, count=9,
             cursor=P, mass=P, slots=80, lengths_out=P + 64, cursor_out=P + 128)
    f.update(k)
    return lib.mlxvs_kv_compact_device(ctypes.byref(c or cache()), *f.values(), work, size, None)


@pytest.mark.parametrize("bad", [
    dict(dim=60), dict(dim=0), dict(dim=264), dict(rotated=33), dict(rotated=66), dict(rotated=-2),
    dict(turns=None), dict(layout=2), dict(magnitude=math.inf), dict(type=2)])
def test_rotations_that_are_refused(engine, bad):
    lib = lib_of(engine)
    assert rotate(lib, rotary(**bad), heads(), heads()) == INVALID
    assert b"[mlxvs" in lib.mlxvs_last_error()


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(out=None), dict(x=P + 8), dict(norm=P + 8), dict(out=P + 2), dict(token_stride=12),
    dict(head_stride=4), dict(out_token_stride=20), dict(heads=-1), dict(norm_type=2),
    dict(out=P * 2, out_head_stride=0), dict(out=P * 2, out_token_stride=64),
    dict(out_token_stride=1024), dict(token_stride=1024)])
def test_heads_that_are_refused(engine, bad):
    lib = lib_of(engine)
    assert rotate(lib, rotary(), heads(**bad), None) == INVALID
    assert rotate(lib, rotary(), heads(), heads(**bad)) == INVALID
    assert b"[mlxvs" in lib.mlxvs_last_error()


def test_rotations_with_other_arguments_that_are_refused(engine):
    lib = lib_of(engine)
    for k in (dict(positions=None), dict(tokens=-1), dict(tokens=1 << 31), dict(eps=-1.0),
              dict(eps=math.nan), dict(evicted=P), dict(requests=-1)):
        assert rotate(lib, rotary(), heads(), heads(), **k) == INVALID, k
    assert rotate(lib, None, heads(), heads()) == INVALID


@pytest.mark.parametrize("bad", [
    dict(rotated=3), dict(rotated=-2), dict(rotated=258), dict(base=1.0), dict(base=math.inf),
    dict(scaling=1, factor=0.5), dict(scaling=1, factor=math.nan), dict(scaling=4),
    dict(scaling=2, rotated=2, factor=2.0), dict(scaling=3, factor=2.0, context=0.0),
    dict(frequencies=None), dict(magnitude=None), dict(scaling=2, factor=1e300)])
def test_frequencies_that_are_refused(engine, bad):
    lib = lib_of(engine)
    f = dict(rotated=8, base=10000.0, scaling=0, factor=1.0, context=4096.0,
             frequencies=(ctypes.c_double * 128)(), magnitude=ctypes.byref(ctypes.c_float()))
    f.update(bad)
    assert lib.mlxvs_kv_rotary_frequencies(*f.values()) == INVALID
    assert b"[mlxvs" in lib.mlxvs_last_error()


@pytest.mark.parametrize("rotated", [2, 4, 64, 128, 256])
@pytest.mark.parametrize("scaling,kind", [(None, 0), ("linear", 1), ("base", 2), ("ramp", 3)])
def test_frequencies(engine, rotated, scaling, kind):
    lib = lib_of(engine)
    if scaling == "base" and rotated == 2:
        pytest.skip("no base to scale")
    f, gain = (ctypes.c_double * 128)(), ctypes.c_float()
    assert lib.mlxvs_kv_rotary_frequencies(rotated, 10000.0, kind, 8.0, 4096.0, f,
                                           ctypes.byref(gain)) == 0
    want, g = kv_budget_oracle.frequencies(rotated, 10000.0, scaling, 8.0, 4096.0)
    # (a few operations in 64 bits, one of them a power)
    np.testing.assert_allclose(f[:rotated // 2], want, rtol=2.0 ** -48)
    assert abs(gain.value - g) <= g * 2.0 ** -24
    # turns: the same numbers over a full circle, in 2^-64 of a turn.  pi to 30
    # digits; a double over it in 64 bits of mantissa: off by 2^-62 of the turns.
    turns = (ctypes.c_uint64 * 128)()
    assert lib.mlxvs_kv_rotary_turns(f, rotated // 2, turns) == 0
    pi = Fraction(3141592653589793238462643383279, 10 ** 30)
    for x, t in zip(f[:rotated // 2], turns):
        exact = Fraction(x) / (2 * pi)
        assert abs(Fraction(t, 1 << 64) - exact) <= exact / (1 << 62) + Fraction(1, 1 << 64)


def test_turns_of_other_frequencies(engine):
    lib = lib_of(engine)

    def turns(x):
        t = ctypes.c_uint64(77)
        rc = lib.mlxvs_kv_rotary_turns(ctypes.byref(ctypes.c_double(x)), 1, ctypes.byref(t))
        return rc, t.value / 2.0 ** 64

    # whole turns are left out, negative ones count from the other side
    for x, want in ((0.0, 0.0), (math.pi, 0.5), (-math.pi / 2, 0.75), (7 * math.pi, 0.5)):
        rc, got = turns(x)
        assert rc == 0 and abs((got - want + 0.5) % 1.0 - 0.5) < 2.0 ** -50, (x, got)
    assert turns(-1e-300) == (0, 0.0)  # a whole turn, rounded
    for x in (math.inf, math.nan, 1e6):
        assert turns(x)[0] == INVALID
    assert lib.mlxvs_kv_rotary_turns(None, 1, P) == INVALID
    assert lib.mlxvs_kv_rotary_turns(None, 129, None) == INVALID
    assert lib.mlxvs_kv_rotary_turns(None, 0, None) == 0


def test_weights_that_are_refused(engine):
    lib = lib_of(engine)
    for k in (dict(starts=None), dict(lse=None), dict(mass=None), dict(scale=0.0),
              dict(scale=math.inf), dict(decay=-0.1), dict(decay=1.5), dict(decay=math.nan),
              dict(longest=-1), dict(slots=79), dict(c=cache(dim=60)), dict(c=cache(page_size=24)),
              dict(q=queries(q_heads=7)), dict(q=queries(positions=None)),
              dict(q=queries(table_stride=4)), dict(q=queries(q=P + 8))):
        assert weigh(lib, **k) == INVALID, k
        assert b"[mlxvs::kv_weigh]" in lib.mlxvs_last_error()
    # a prompt's workspace
    q = queries(tokens=5000, columns=320, table_stride=320)
    need = lib.mlxvs_kv_weigh_workspace(ctypes.byref(cache()), ctypes.byref(q), 0)
    assert need > 0
    for k in (dict(work=None), dict(size=need - 1), dict(work=P + 4)):
        assert weigh(lib, q=q, slots=5120, **k) == INVALID
        assert b"workspace" in lib.mlxvs_last_error()
    assert lib.mlxvs_kv_weigh_workspace(ctypes.byref(cache()), ctypes.byref(queries(requests=3)), 0) == 0
    assert lib.mlxvs_kv_weigh_workspace(ctypes.byref(cache()), ctypes.byref(q), -1) == -1


@pytest.mark.parametrize("bad", [
    dict(mass=None), dict(lengths=None), dict(kept=None), dict(requests=-1), dict(heads=0),
    dict(slots=-1), dict(slots=1 << 31), dict(n=0), dict(first=-1), dict(recent=-1),
    dict(first=9, recent=8), dict(above=15), dict(requests=1 << 26, heads=64)])
def test_budgets_that_are_refused(engine, bad):
    lib = lib_of(engine)
    assert keep(lib, **bad) == INVALID
    assert b"[mlxvs::kv_keep]" in lib.mlxvs_last_error()


def test_budgets_of_long_rows_need_a_workspace(engine):
    lib = lib_of(engine)
    assert lib.mlxvs_kv_keep_workspace(2, 2, 30_000) == 0
    assert lib.mlxvs_kv_keep_workspace(2, 2, -1) == -1
    need = lib.mlxvs_kv_keep_workspace(2, 2, 100_000)
    assert need > 0
    for k in (dict(work=None), dict(size=need - 1), dict(work=P + 8)):
        assert keep(lib, slots=100_000, **k) == INVALID
        assert b"workspace" in lib.mlxvs_last_error()


@pytest.mark.parametrize("bad", [
    dict(table=None), dict(stride=4), dict(columns=-1), dict(requests=-1), dict(lengths=None),
    dict(kept=None), dict(n=0), dict(free=None), dict(count=-1), dict(cursor=None), dict(slots=79),
    dict(lengths_out=None), dict(cursor_out=None), dict(cursor_out=P), dict(lengths_out=P + 4),
    dict(lengths_out=P - 4), dict(work=None), dict(size=0), dict(work=P + 8),
    dict(c=cache(page_size=24)), dict(c=cache(scales=None))])
def test_cuts_that_are_refused(engine, bad):
    lib = lib_of(engine)
    assert compact(lib, **bad) == INVALID
    assert b"[mlxvs::kv_compact]" in lib.mlxvs_last_error()
    assert lib.mlxvs_kv_compact_workspace(ctypes.byref(cache()), 5, 2, 0) == -1


def test_calls_without_work(engine):
    lib = lib_of(engine)
    assert rotate(lib, rotary(), heads(), heads(), tokens=0, positions=None) == 0
    assert rotate(lib, rotary(), heads(heads=0), None) == 0
    none = queries(tokens=0, q=None, positions=None, token_request=None)
    assert weigh(lib, q=none, starts=None, lse=None, mass=None) == 0
    assert keep(lib, requests=0, mass=None, lengths=None, kept=None) == 0


def test_no_fallback_without_a_gpu(engine):
    import mlxvs_amd._hip as hip

    if hip.device_count() > 0:
        pytest.skip("a GPU is present: the addresses are nobody's")
    lib = lib_of(engine)
    for rc in (rotate(lib, rotary(), heads(), heads(norm=P)),
               rotate(lib, rotary(rotated=0, turns=None), heads(out=P * 4), None),
               weigh(lib), weigh(lib, q=queries(token_request=None)), keep(lib), compact(lib),
               compact(lib, mass=None, slots=0)):
        assert rc == INTERNAL
        assert b"no HIP device" in lib.mlxvs_last_error()
    with pytest.raises(ValueError, match="device must be a GPU"):
        engine.Rotary(64, device="cpu")
