"""The operators that keep a paged key-value cache within a budget, on the GPU
against their restatement in NumPy (kv_budget_oracle.py): lists, moved values,
summaries, pages and lengths equal, computed numbers within bounds that follow from
their roundings.

With u the unit roundoff of the rows' type (2^-8 for bfloat16, 2^-11 for float16) a
rotated value is rounded once, u |y|; what is computed before that in float32 is off
by some 2^-24 of its terms, sines and cosines by 2^-19 (an angle's 2^-32 of a turn,
its conversion 2^-26 of a turn, 9e-8, and the instruction's own), a norm's factor by
(dim + 8) 2^-24: |y - exact| <= u |y| + (2^-18 + (dim + 8) 2^-24) terms.

A mass sums terms exp(x), x = scale q.k - lse.  A float32 product of dim terms is
off by (dim + 2) 2^-24 of scale sum |q_i k_i| (`reach`), x by 2 2^-24 (|scale q.k| +
|lse|) more, the exponential by 2^-22 and its factor by 2^-23 |x|; sums of n terms by
n 2^-24 of them.  The oracle adds that up (err, in 2^-24).
"""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv_budget_oracle as want_of  # noqa: E402
from test_gpu_kv import DTYPES, UNIT, dev, f32  # noqa: E402

pytestmark = pytest.mark.gpu


# ---- rotate -------------------------------------------------------------------


def check_rotate(engine, q, k, pos, dtype, *, norms=(None, None), eps=1e-6, who=None, evicted=None,
                 out=None, **how):
    dim = q.shape[2]
    rot = engine.Rotary(dim, **how)
    text = np.asarray(pos, np.int64)
    if evicted is not None:
        inside = (np.asarray(who) >= 0) & (np.asarray(who) < len(evicted)) & (text >= 0)
        text = np.where(inside, text + np.asarray(evicted)[np.clip(who, 0, len(evicted) - 1)], text)
    before = [None if x is None else f32(x) for x in (q, k)]
    held = [None if w is None else f32(w) for w in norms]
    got = rot.rotate(q, k, dev(pos, torch.int32), q_norm=norms[0], k_norm=norms[1], eps=eps,
                     requests=None if who is None else dev(who, torch.int32),
                     evicted=None if evicted is None else dev(evicted, torch.int32), out=out)
    for x, w, y in zip(before, held, got):
        if x is None:
            assert y is None
            continue
        exact, size = want_of.rotate(x, text, np.array(rot.frequencies), rot.magnitude, rot.layout, w,
                                     eps)
        off = np.abs(y.double().cpu().numpy() - exact)
        bound = UNIT[dtype] * np.abs(exact) + (2.0 ** -18 + (dim + 8) * 2.0 ** -24) * size + 2.0 ** -24
        assert (off <= bound).all(), float((off - bound).max())
    return got


def rows(rng, tokens, heads, dim, dtype):
    return dev(rng.standard_normal((tokens, heads, dim), np.float32)).to(DTYPES[dtype])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dim,rotated", [(8, 8), (64, 64), (72, 40), (80, 80), (80, 32), (96, 24),
                                         (128, 128), (128, 2), (128, 0), (192, 96), (256, 256),
                                         (248, 246), (200, 176)])
def test_rotation_of_heads(engine, dim, rotated, layout, dtype):
    rng = np.random.default_rng(dim + rotated)
    pos = rng.integers(0, 100_000, 37)
    pos[5], pos[6], pos[-1] = 0, 1, -1
    check_rotate(engine, rows(rng, 37, 7, dim, dtype), rows(rng, 37, 3, dim, dtype), pos, dtype,
                 rotated=rotated, layout=layout)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("dim,rotated", [(8, 8), (64, 64), (72, 40), (80, 32), (96, 24), (128, 128),
                                         (256, 256), (248, 160)])
def test_norm_and_rotation(engine, dim, rotated, layout, dtype):
    rng = np.random.default_rng(dim * rotated)
    wide = torch.float32 if dim % 16 else DTYPES[dtype]
    norms = [dev(1 + 0.3 * rng.standard_normal(dim)).to(t) for t in (wide, DTYPES[dtype])]
    q, k = rows(rng, 21, 5, dim, dtype), rows(rng, 21, 5, dim, dtype)
    q[3] = 0  # (nothing to divide by but eps)
    check_rotate(engine, q, k, rng.integers(0, 9000, 21), dtype, rotated=rotated, layout=layout,
                 norms=norms, eps=1e-5)
    odd = dev(1 + 0.3 * rng.standard_normal(dim + 1)).to(wide)[1:]
    check_rotate(engine, q, k, rng.integers(0, 9000, 21), dtype, rotated=rotated, layout=layout,
                 norms=(None, odd))


@pytest.mark.parametrize("tokens,q_heads,kv_heads", [(1, 1, 1), (1, 32, 8), (3, 33, 1), (64, 9, 3),
                                                     (2000, 2, 2), (700, 40, 8), (5000, 1, 0)])
def test_rotation_of_few_and_many(engine, tokens, q_heads, kv_heads):
    rng = np.random.default_rng(tokens)
    k = rows(rng, tokens, kv_heads, 128, "bf16") if kv_heads else None
    check_rotate(engine, rows(rng, tokens, q_heads, 128, "bf16"), k, np.arange(tokens), "bf16")


@pytest.mark.parametrize("scaling", [None, "linear", "base", "ramp"])
def test_scaled_positions_far_away(engine, scaling):
    rng = np.random.default_rng(5)
    pos = np.array([0, 1, 4095, 4096, 131_071, 10 ** 6, 10 ** 9, 2 ** 31 - 1])
    check_rotate(engine, rows(rng, 8, 2, 128, "f16"), rows(rng, 8, 1, 128, "f16"), pos, "f16",
                 scaling=scaling, factor=16.0, context=8192)


def test_positions_of_requests_that_lost_tokens(engine):
    rng = np.random.default_rng(6)
    pos = np.array([5, 9, -1, 2 ** 31 - 1, 100, 7])
    who = np.array([0, 1, 1, 2, 3, -1])  # (3 and -1: no request)
    check_rotate(engine, rows(rng, 6, 3, 64, "f16"), rows(rng, 6, 3, 64, "f16"), pos, "f16", who=who,
                 evicted=[1000, 0, 2 ** 31 - 1])


def test_own_frequencies(engine):
    rng = np.random.default_rng(7)
    check_rotate(engine, rows(rng, 9, 2, 32, "bf16"), None, np.arange(9) * 1000, "bf16", rotated=6,
                 frequencies=[1.0, -0.25, 100.5], magnitude=0.5)


@pytest.mark.parametrize("layout", ["halves", "pairs"])
@pytest.mark.parametrize("rotated", [128, 72, 20])
def test_rotation_in_place_of_slices_of_a_projection(engine, layout, rotated):
    rng = np.random.default_rng(8)
    fused = rows(rng, 50, 14, 128, "bf16")
    kept = fused.clone()
    q, k = fused[:, :8], fused[:, 8:11]
    norms = [dev(1 + 0.1 * rng.standard_normal(128)).to(torch.bfloat16)] * 2
    got = check_rotate(engine, q, k, np.arange(50) * 77, "bf16", rotated=rotated, layout=layout,
                       norms=norms, out=(q, k))
    assert got[0] is q and got[1] is k
    assert torch.equal(fused[:, 11:], kept[:, 11:])
    again = engine.Rotary(128, rotated=rotated, layout=layout).rotate(
        kept[:, :8], kept[:, 8:11], dev(np.arange(50) * 77, torch.int32), q_norm=norms[0],
        k_norm=norms[1])
    assert torch.equal(again[0], q) and torch.equal(again[1], k)


def test_rotation_of_any_strides(engine):
    rng = np.random.default_rng(9)
    wide = rows(rng, 31, 10, 200, "f16")
    for q in (wide[:, 2:7, 3:131], wide[::2, :, 40:168], wide.transpose(0, 1)[:, :10, :128],
              wide[:1, :1, :128].expand(31, 4, 128)):
        pos = np.arange(len(q))
        check_rotate(engine, q, q[:, :1], pos, "f16")
    out = torch.zeros(5, 31, 128, dtype=torch.float16, device="cuda")
    q = wide[:, :5, :128]
    check_rotate(engine, q, None, np.arange(31), "f16", out=(out.transpose(0, 1), None))
    with pytest.raises(ValueError, match="aligned"):
        engine.Rotary(128).rotate(q, None, dev(np.arange(31), torch.int32),
                                  out=(wide[:, :5, 3:131], None))
    with pytest.raises(ValueError, match="overlap"):
        engine.Rotary(128).rotate(q, None, dev(np.arange(31), torch.int32),
                                  out=(out[:1, :1].expand(31, 5, 128), None))


def test_rotation_of_values_that_are_not_finite(engine):
    # a head that holds them is its own affair, and what passes is not touched
    x = torch.ones(2, 3, 64, dtype=torch.bfloat16, device="cuda")
    x[0, 1, 60], x[1, 2, 63] = math.inf, math.nan
    y, _ = engine.Rotary(64, rotated=32).rotate(x, None, dev([3, 4], torch.int32))
    assert torch.equal(y[..., 32:].nan_to_num(7), x[..., 32:].nan_to_num(7))
    assert y[..., :32].isfinite().all()


def test_rotation_without_tokens_or_keys(engine):
    rot = engine.Rotary(64)
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    a, b = rot.rotate(q, q[:, :2], torch.empty(0, dtype=torch.int32, device="cuda"))
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)


def test_rotation_refuses(engine):
    rot = engine.Rotary(64)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")
    for bad in (dict(q=q.float()), dict(q=q[..., :32]), dict(q=q.cpu()), dict(k=q[:2]),
                dict(k=q.half()), dict(positions=pos.long()), dict(positions=pos[:2]),
                dict(q_norm=q[0, 0, :32]), dict(q_norm=q[0, 0].half()), dict(k=None, k_norm=q[0, 0]),
                dict(evicted=pos), dict(evicted=pos, requests=pos[:1]), dict(eps=-1.0),
                dict(out=q), dict(out=(q[:2], q)), dict(out=(q, q.half()))):
        a = dict(q=q, k=q, positions=pos)
        a.update(bad)
        with pytest.raises(ValueError, match="mlxvs"):
            rot.rotate(a.pop("q"), a.pop("k"), a.pop("positions"), **a)
    for bad in (dict(dim=60), dict(dim=64, rotated=3), dict(dim=64, layout="other"),
                dict(dim=64, scaling="other"), dict(dim=64, frequencies=[1.0]),
                dict(dim=64, scaling="linear", factor=0.0), dict(dim=64, magnitude=math.nan),
                dict(dim=4, rotated=4), dict(dim=64, scaling="ramp", frequencies=[1.0] * 32)):
        with pytest.raises(ValueError, match="mlxvs"):
            engine.Rotary(**bad)


def test_a_gradient_that_is_asked_for_is_an_error(engine):
    rot = engine.Rotary(64)
    q = torch.randn(3, 4, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    y, z = rot.rotate(q, q.detach()[:, :1], pos)
    plain, _ = rot.rotate(q.detach(), None, pos)
    assert torch.equal(y, plain)
    with pytest.raises(RuntimeError, match="no gradient"):
        y.float().sum().backward()
    with pytest.raises(ValueError, match="gradient"):
        rot.rotate(q, None, pos, out=(q.detach(), None))
    with torch.no_grad():
        assert not rot.rotate(q, None, pos)[0].requires_grad


# ---- weigh -------------------------------------------------------------------


class Step:
    """A cache, and the tokens of a step over it."""

    def __init__(self, engine, lengths, counts, *, page=16, heads=2, group=3, dim=64, dtype="bf16",
                 seed=0, spare=0, fill=math.nan):
        rng = np.random.default_rng(seed)
        held = [-(-n // page) for n in lengths]
        cols, pages = max(held + [1]) + spare, sum(held) + 3
        self.cache = engine.PagedKVCache.empty(pages, heads, page, dim, dtype=DTYPES[dtype])
        ids = rng.permutation(pages)
        table = np.full((len(lengths), cols), -1)
        keys = np.full((pages, heads, page, dim), fill, np.float32)  # what nobody wrote
        at = 0
        for r, n in enumerate(lengths):
            table[r, :held[r]] = ids[at:at + held[r]]
            at += held[r]
            for p in range(n):
                keys[table[r, p // page], :, p % page] = rng.standard_normal((heads, dim))
        self.cache.keys.copy_(dev(keys))
        self.cache.values.copy_(dev(rng.standard_normal(self.cache.values.shape, np.float32)))
        self.table = dev(table, torch.int32)
        self.starts = dev(np.concatenate([[0], np.cumsum(counts)]), torch.int32)
        where = np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, counts)] + [[]])
        who = np.repeat(np.arange(len(lengths)), counts)
        self.positions, self.requests = dev(where, torch.int32), dev(who, torch.int32)
        self.q = dev(1.5 * rng.standard_normal((len(where), heads * group, dim))).to(DTYPES[dtype])
        self.mass = dev(rng.random((len(lengths), heads, cols * page)), torch.float32)
        self.scale = 1.0 / math.sqrt(dim)

    def attend(self, **k):
        _, self.lse = self.cache.attend(self.q, self.table, self.requests, self.positions, lse=True, **k)
        return self

    def check(self, decay=1.0, scale=None, **k):
        before = self.mass.cpu().numpy()
        scale = scale or self.scale
        want, err = want_of.weigh(f32(self.q), f32(self.cache.keys), self.table.cpu().numpy(),
                                  self.starts.cpu().numpy(), self.positions.cpu().numpy(),
                                  self.lse.double().cpu().numpy(), before, scale, decay)
        self.cache.weigh(self.q, self.table, self.starts, self.positions, self.lse, self.mass,
                         scale=scale, decay=decay, **k)
        got = self.mass.double().cpu().numpy()
        bound = err * 2.0 ** -24 + 1e-37
        # (what stays as it was may be anything)
        same = (got == want) | (np.isnan(got) & np.isnan(want))
        with np.errstate(invalid="ignore"):
            bad = ~same & ~(np.abs(got - want) <= bound)
        assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5])
        return got


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page,dim,heads,group", [(16, 64, 2, 4), (64, 128, 3, 1), (32, 80, 1, 5),
                                                  (128, 8, 2, 16), (256, 256, 2, 3), (16, 192, 1, 17),
                                                  (64, 96, 2, 7)])
def test_weights_of_single_tokens(engine, page, dim, heads, group, dtype):
    lengths = [1, 2, page, page + 1, 300, 0, 257]
    Step(engine, lengths, [min(1, n) for n in lengths], page=page, dim=dim, heads=heads, group=group,
         dtype=dtype, seed=dim).attend().check()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page,dim,heads,group", [(16, 64, 2, 4), (64, 128, 1, 8), (32, 80, 2, 1),
                                                  (256, 256, 1, 2), (128, 72, 1, 3), (16, 192, 1, 5)])
def test_weights_of_prompts(engine, page, dim, heads, group, dtype):
    # whole prompts, a chunk at the end, one token, none, all of it but one
    Step(engine, [70, 200, 33, 40, 129], [70, 45, 1, 0, 128], page=page, dim=dim, heads=heads,
         group=group, dtype=dtype, seed=dim).attend().check()


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 130])
def test_weights_of_prompts_of_any_length(engine, tokens):
    s = Step(engine, [tokens + 9, tokens], [tokens, tokens], heads=1, group=2, seed=tokens).attend()
    got = s.check()
    # each query head hands out 1
    total = got[1, 0, :tokens].sum()
    assert abs(total - 2 * tokens) <= 2 * tokens * 2.0 ** -10


@pytest.mark.parametrize("lengths,counts,heads,group,dim", [
    ([900, 40, 5], [900, 1, 5], 1, 4, 64), ([1000, 700, 0, 600], [500, 700, 0, 2], 1, 3, 16),
    ([300], [300], 2, 16, 128), ([300], [299], 1, 24, 256), ([700], [650], 1, 2, 192)])
def test_weights_of_prompts_in_pieces(engine, lengths, counts, heads, group, dim):
    # more rows than one workgroup goes through
    Step(engine, lengths, counts, page=64, heads=heads, group=group, dim=dim,
         seed=len(lengths)).attend().check(decay=0.5)


@pytest.mark.parametrize("group", [32, 33, 63, 64, 65, 130])
def test_weights_of_many_query_heads_of_a_key(engine, group):
    Step(engine, [150, 20, 90], [40, 1, 90], heads=1, group=group, dim=32, seed=group).attend().check()


def test_weights_of_a_batch_that_is_one_request_s(engine):
    # no more tokens than requests, all of them one request's
    counts = [0, 0, 21] + [0] * 20
    Step(engine, [30, 0, 300] + [5] * 20, counts, heads=1, group=2, dim=16, seed=5).attend().check()
    Step(engine, [30, 0, 300], [0, 0, 3], heads=2, group=24, dim=96, seed=6).attend().check()


@pytest.mark.parametrize("most", [1, 3])
def test_weights_of_many_requests(engine, most):
    rng = np.random.default_rng(most)
    lengths = rng.integers(0, 40, 1_100)
    lengths[[7, 1_099]] = 300, 290
    counts = np.minimum(lengths, rng.integers(0, most + 1, 1_100))
    counts[1_099] = 200 if most > 1 else 1
    Step(engine, lengths, counts, heads=1, group=2, dim=16, seed=most).attend().check()


@pytest.mark.parametrize("group", [1, 4, 33])
def test_weights_of_requests_with_few_and_many_rows(engine, group):
    # 20 requests, dealt to two kernels: 1 to 33 rows, prompts, none
    counts = [1, 8, 9, 31, 32, 33, 0, 70, 1, 1, 2, 3, 4, 5, 6, 7, 8, 9, 0, 1]
    lengths = [n + 13 * i for i, n in enumerate(counts)]
    s = Step(engine, lengths, counts, heads=2, group=group, dim=48, seed=group).attend()
    s.positions[s.starts[5]:s.starts[6]] = -1  # (one was not admitted)
    s.positions[s.starts[2]:s.starts[3]] = -1
    s.check(decay=0.5)


@pytest.mark.parametrize("longest", [0, 1, 1_000])
def test_weights_of_prompts_of_other_sizes_together(engine, longest):
    # units of many sizes, keys that few of the tokens see, masked tiles in between
    Step(engine, [1_290, 700, 256, 5, 999], [290, 513, 256, 1, 130], page=32, heads=2, group=3, dim=64,
         spare=2, seed=longest).attend().check(longest=longest, decay=0.25)


def test_weights_on_two_streams_at_once(engine):
    steps = [Step(engine, [900, 400], [600, 1], page=64, heads=2, group=4, dim=128, seed=i).attend()
             for i in range(2)]
    want = []
    for s in steps:
        want.append(s.mass.clone())
        s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, want[-1])
    streams = [torch.cuda.Stream() for _ in steps]
    masses = [[s.mass.clone() for _ in range(10)] for s in steps]
    torch.cuda.synchronize()
    for i in range(10):
        for s, stream, m in zip(steps, streams, masses):
            with torch.cuda.stream(stream):
                s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, m[i])
    torch.cuda.synchronize()
    assert all(torch.equal(x, w) for m, w in zip(masses, want) for x in m)


def test_weights_in_a_captured_graph(engine):
    # other tokens, lengths and keys at every replay: units of other sizes and numbers
    s = Step(engine, [800, 500, 300], [300, 1, 20], page=64, heads=2, group=3, dim=64, seed=1).attend()
    start, mass = s.mass.clone(), s.mass.clone()
    s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, mass.clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, mass)
    tokens = len(s.q)
    for counts in ([300, 1, 20], [0, 0, 300], [1, 320, 0], [107, 107, 107], [0, 0, 0]):
        starts = np.concatenate([[0], np.cumsum(counts)])
        where = np.concatenate([np.arange(n - m, n) for n, m in zip([800, 500, 300], counts)]
                               + [[-1] * (tokens - sum(counts))])
        s.starts.copy_(dev(starts, torch.int32))
        s.positions.copy_(dev(where, torch.int32))
        s.requests.copy_(dev(list(np.repeat([0, 1, 2], counts)) + [-1] * (tokens - sum(counts)),
                             torch.int32))
        lse = s.cache.attend(s.q, s.table, s.requests, s.positions, lse=True)[1]
        s.lse.copy_(lse)
        mass.copy_(start)
        graph.replay()
        torch.cuda.synchronize()
        want = start.clone()
        s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, want)
        assert torch.equal(mass, want), counts
        s.mass.copy_(start)
        s.check()


def test_weights_decay_and_begin_anew(engine):
    for decay in (0.0, 0.5, 1.0):
        s = Step(engine, [50, 90, 7], [3, 1, 7], seed=3)
        s.mass[:, :, 60:80] = math.inf
        if decay == 0.0:
            s.mass[0, 0, :40] = math.nan  # (not read)
        s.attend()
        s.mass[2] = math.nan              # (a new request's row was another's)
        last = s.mass.clone()
        if decay == 0.0:
            s.mass[0, 0, :40] = 5.0
            want = s.check(decay=0.0)
            s.mass.copy_(last)
            s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, s.mass, decay=0.0)
            got = s.mass.double().cpu().numpy()
            assert np.array_equal(got, want, equal_nan=True)
        else:
            s.mass[1, :, 60:80] = 3.0
            s.mass[2] = 9.0
            s.check(decay=decay)


def test_weights_of_absent_pages_and_odd_lists(engine):
    s = Step(engine, [100, 64, 64], [20, 1, 64], seed=4)
    s.table[0, 2], s.table[1, 1], s.table[2, 0] = -1, 10 ** 6, -5
    s.attend().check()
    # requests that were not admitted have positions of -1
    s.positions[20] = -1
    s.check()
    # tokens past the batch, starts out of order: nothing is read or written outside
    for starts in ([0, 20, 500, 85], [-7, 20, 20, 30], [50, 10, 85, 85]):
        s.starts.copy_(dev(starts, torch.int32))
        s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, s.mass)


def test_weights_of_a_table_wider_than_its_requests(engine):
    for longest in (0, 5, 70, 1000):
        Step(engine, [70, 40], [4, 1], spare=37, seed=longest).attend().check(longest=longest)


def test_weights_of_long_requests_and_a_larger_scale(engine):
    s = Step(engine, [1500, 777], [1, 2], page=64, heads=1, group=2, dim=64, seed=8)
    s.attend(scale=0.5).check(scale=0.5)


def test_weights_far_from_the_largest(engine):
    # scores over a range of hundreds: most probabilities are 0, none is more than 1
    s = Step(engine, [200], [20], dtype="f16", seed=9)
    s.q *= 40
    got = s.attend().check()
    assert got[0, :, :200].sum() <= 20 * 6 * (1 + 2.0 ** -8) + 180 * 2


def test_weights_of_queries_that_are_not_finite(engine):
    s = Step(engine, [40, 50], [3, 50], seed=10).attend()
    clean = s.mass.clone()
    s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, clean)
    s.q[3 + 49, 0, 0] = math.nan  # the last token of the second request: kv head 0
    s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, s.mass)
    assert s.mass[1, 0, :50].isnan().all()
    assert torch.equal(s.mass[0], clean[0]) and torch.equal(s.mass[1, 1], clean[1, 1])


def test_weights_are_the_same_every_time(engine):
    s = Step(engine, [300, 200, 150], [150, 1, 150], group=4, seed=11).attend()
    first = s.mass.clone()
    s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, first)
    for longest in (0, 300, 32):
        again = s.mass.clone()
        s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, again, longest=longest)
        assert torch.equal(first, again)


def test_weights_of_strided_queries(engine):
    s = Step(engine, [90, 60], [30, 1], dim=128, seed=12).attend()
    want = s.mass.clone()
    s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, want)
    wide = torch.zeros(31, 10, 144, dtype=s.q.dtype, device="cuda")
    for view in (wide[:, 2:8, 8:136], wide[:, 2:8, 5:133]):
        view.copy_(s.q)
        mass = s.mass.clone()
        s.cache.weigh(view, s.table, s.starts, s.positions, s.lse, mass)
        assert torch.equal(mass, want)


def test_weights_refuse(engine):
    s = Step(engine, [20, 30], [2, 3]).attend()
    for bad in (dict(q=s.q[:, :3]), dict(q=s.q.float()), dict(starts=s.starts[:2]),
                dict(starts=s.starts.long()), dict(positions=s.positions[:2]), dict(lse=s.lse[:, :2]),
                dict(lse=s.lse.half()), dict(mass=s.mass[:, :, :16]), dict(mass=s.mass[:1]),
                dict(mass=s.mass.double()), dict(mass=s.mass.cpu()), dict(decay=2.0),
                dict(decay=math.nan), dict(scale=0.0), dict(longest=-1), dict(table=s.table.long())):
        a = dict(q=s.q, table=s.table, starts=s.starts, positions=s.positions, lse=s.lse, mass=s.mass)
        a.update(bad)
        with pytest.raises(ValueError, match="mlxvs"):
            s.cache.weigh(a.pop("q"), a.pop("table"), a.pop("starts"), a.pop("positions"),
                          a.pop("lse"), a.pop("mass"), **a)


# ---- keep ----------------------------------------------------------------------


def small_cache(engine, heads=2, page=16, dim=16):
    return engine.PagedKVCache.empty(1, heads, page, dim)


def check_keep(engine, mass, lengths, n, first=1, recent=1, above=None):
    mass = np.asarray(mass, np.float32)
    got = small_cache(engine, mass.shape[1]).keep(dev(mass), dev(lengths, torch.int32), n, first=first,
                                                  recent=recent, above=above)
    want = want_of.keep(mass, lengths, n, first, recent, n if above is None else above)
    assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("slots", [1, 2, 63, 64, 65, 1000, 1024, 1025, 4097])
def test_budgets_of_rows_of_any_length(engine, slots):
    rng = np.random.default_rng(slots)
    mass = rng.lognormal(0, 2, (4, 2, slots))
    lengths = [slots, max(0, slots - 1), slots // 2, 0]
    for n in sorted({1, 2, max(1, slots // 3), max(1, slots - 1), slots, slots + 5}):
        first, recent = min(4, n // 2), min(7, n // 3)
        check_keep(engine, mass, lengths, n, first, recent)


@pytest.mark.parametrize("slots,n", [(20_000, 5_000), (33_000, 150), (65_536, 65_000), (70_000, 300), (70_000, 69_999),
                                     (140_001, 40_000)])
def test_budgets_of_long_rows(engine, slots, n):
    rng = np.random.default_rng(slots)
    mass = rng.lognormal(0, 2, (2, 1, slots))
    mass[:, :, rng.integers(0, slots, slots // 10)] = 0.0
    check_keep(engine, mass, [slots, slots * 3 // 4], n, 4, 128)


def test_budgets_where_masses_are_equal(engine):
    rng = np.random.default_rng(1)
    for values in ([0.0], [0.0, -0.0], [1.0, 2.0], [3.0, 3.0000002], [1e-40, 0.0, -1e-40]):
        mass = rng.choice(np.array(values, np.float32), (3, 2, 777))
        for n in (1, 64, 100, 776):
            check_keep(engine, mass, [777, 500, 101], n, 0, 0)
            check_keep(engine, mass, [777, 500, 101], n, min(n, 3), max(0, min(n - 3, 50)))


def test_budgets_of_masses_that_are_not_finite(engine):
    rng = np.random.default_rng(2)
    mass = rng.standard_normal((3, 2, 300)).astype(np.float32)
    mass[:, :, ::3] = math.nan
    mass[:, :, 1::7] = math.inf
    mass[:, :, 2::11] = -math.inf
    mass[1, 1, :] = -math.nan
    mass[2, 0, :] = np.finfo(np.float32).min
    for n in (5, 40, 150, 250, 299):
        check_keep(engine, mass, [300, 300, 290], n, 2, 3)


def test_budgets_above_which_requests_are_cut(engine):
    rng = np.random.default_rng(3)
    mass = rng.random((5, 2, 100))
    check_keep(engine, mass, [100, 64, 65, 10, 80], 20, 2, 5, above=64)
    check_keep(engine, mass, [100, 21, 20, 19, 1000], 20, 20, 0)  # (1000: more than the slots)
    check_keep(engine, mass, [100, 21, 20, -3, 0], 20, 0, 20)
    check_keep(engine, mass, [100, 21, 20, 19, 0], 20, 13, 7)


def test_budgets_refuse(engine):
    c, mass = small_cache(engine), torch.zeros(2, 2, 50, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    for bad in (dict(mass=mass[:, :1]), dict(mass=mass.half()), dict(mass=mass[..., ::2]),
                dict(lengths=lengths[:1]), dict(lengths=lengths.long()), dict(n=0), dict(n=-2),
                dict(first=-1), dict(recent=11), dict(above=9)):
        a = dict(mass=mass, lengths=lengths, n=10)
        a.update(bad)
        with pytest.raises(ValueError, match="mlxvs"):
            c.keep(a.pop("mass"), a.pop("lengths"), a.pop("n"), **a)
    assert c.keep(mass[:0], lengths[:0], 4).shape == (0, 2, 4)


# ---- compact -------------------------------------------------------------------


def lists(rng, lengths, heads, n, whole=()):
    out = np.full((len(lengths), heads, n), -1, np.int32)
    for r, length in enumerate(lengths):
        if length > n and r not in whole:
            for h in range(heads):
                out[r, h] = np.sort(rng.choice(length, n, replace=False))
    return out


def check_compact(engine, lengths, kept, *, page=16, dim=64, dtype="bf16", seed=0, spare=0, cursor=None,
                  room=9, mass=True, summaries=True, fill=None, out=None, absent=()):
    rng = np.random.default_rng(seed)
    requests, heads, n = kept.shape
    held = [-(-m // page) for m in lengths]
    cols, pages = max(held + [1]) + spare, sum(held) + 4
    cache = engine.PagedKVCache.empty(pages, heads, page, dim, dtype=DTYPES[dtype], summaries=summaries)
    cache.keys.copy_(dev(rng.standard_normal(cache.keys.shape, np.float32)))
    cache.values.copy_(dev(rng.standard_normal(cache.values.shape, np.float32)))
    if fill is not None:
        cache.keys[rng.integers(0, pages, 3), 0, 1, 0] = fill
    if summaries:
        cache.summaries.fill_(77)
        cache.scales.fill_(-5.0)
    ids = rng.permutation(pages)
    wide = np.full((requests, cols + 2), -1, np.int32)
    at = 0
    for r in range(requests):
        wide[r, :held[r]] = ids[at:at + held[r]]
        at += held[r]
    for r, c in absent:
        wide[r, c] = -1
    free = rng.permutation(at + room).astype(np.int32)
    cursor = at if cursor is None else cursor
    m = rng.random((requests, heads, (cols + 1) * page), np.float32) if mass else None
    t, f, dm = dev(wide), dev(free), None if m is None else dev(m)
    before = dict(keys=cache.keys.view(torch.int16).cpu().numpy().copy(),
                  values=cache.values.view(torch.int16).cpu().numpy().copy())
    args = (cache.summaries.cpu().numpy(), cache.scales.cpu().numpy()) if summaries else (None, None)
    want = want_of.compact(f32(cache.keys), f32(cache.values), *args, wide[:, :cols], lengths, kept,
                           free, cursor, m)
    bits = want_of.compact(before["keys"], before["values"], None, None, wide[:, :cols], lengths, kept,
                           free, cursor, m)
    got = cache.compact(t[:, :cols], dev(lengths, torch.int32), dev(kept), f, dev([cursor], torch.int32),
                        mass=dm, out=out)
    assert np.array_equal(got.lengths.cpu().numpy(), want["lengths"])
    assert np.array_equal(got.cursor.cpu().numpy(), want["cursor"])
    assert np.array_equal(f.cpu().numpy(), want["free"])
    assert np.array_equal(t.cpu().numpy(), wide)
    assert np.array_equal(cache.keys.view(torch.int16).cpu().numpy(), bits["keys"])
    assert np.array_equal(cache.values.view(torch.int16).cpu().numpy(), bits["values"])
    if mass:
        assert np.array_equal(dm.cpu().numpy(), want["mass"])
    if summaries:
        assert np.array_equal(cache.summaries.cpu().numpy(), want["summaries"])
        np.testing.assert_allclose(cache.scales.cpu().numpy(), want["scales"], rtol=2.0 ** -22)
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("page,dim", [(16, 64), (32, 80), (64, 128), (128, 8), (256, 72), (16, 256),
                                      (64, 192), (128, 128)])
def test_cuts_of_requests(engine, page, dim, dtype):
    rng = np.random.default_rng(page + dim)
    lengths = [700, 300, 10, 0, 161, 512]
    check_compact(engine, lengths, lists(rng, lengths, 2, 160), page=page, dim=dim, dtype=dtype,
                  seed=dim)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 300, 511])
def test_cuts_to_any_number(engine, n):
    rng = np.random.default_rng(n)
    lengths = [512, n + 1, n, max(0, n - 1)]
    check_compact(engine, lengths, lists(rng, lengths, 2, n), seed=n)
    check_compact(engine, lengths, lists(rng, lengths, 1, n), page=64, dim=8, seed=n)


def test_cuts_that_keep_ends_and_middles(engine):
    a = np.arange
    for rows_ in ([a(100), a(100, 200), a(50, 150)], [a(0, 200, 2), np.r_[0:99, 199], np.r_[0, 101:200]],
                  [np.r_[0:64, 128:164], np.r_[0:65, 100:135], np.r_[0:50, 150:200]]):
        kept = np.stack([np.stack([x, y]) for x, y in zip(rows_, rows_[1:] + rows_[:1])]).astype(np.int32)
        check_compact(engine, [200, 200, 200], kept, page=32)
        check_compact(engine, [200, 200, 200], kept, page=64, mass=False, summaries=False)


def test_cuts_of_one_long_request(engine):
    rng = np.random.default_rng(5)
    for n, page in ((3000, 16), (100, 64), (4999, 128), (2500, 256)):
        check_compact(engine, [5000], lists(rng, [5000], 2, n), page=page, dim=16, seed=n)


def test_cuts_that_the_free_list_has_no_room_for(engine):
    rng = np.random.default_rng(6)
    lengths = [100, 60, 33, 40, 90]
    kept = lists(rng, lengths, 2, 32)
    # the second request's pages do not fit, nor does any later one's
    for cursor in (0, 4, 5, 6, 7, 8, 11, 12, 13, 30):
        check_compact(engine, lengths, kept, cursor=cursor)
    # a request cut within its last page gives nothing back: always
    check_compact(engine, [40, 36], lists(rng, [40, 36], 2, 34), cursor=0)
    # a cursor past the list, or before it
    for cursor in (200, -1):
        check_compact(engine, [100, 40, 36], lists(rng, [100, 40, 36], 2, 34), cursor=cursor, room=0)


def test_requests_that_are_not_cut(engine):
    rng = np.random.default_rng(7)
    lengths = [100, 90, 20, 21]
    check_compact(engine, lengths, lists(rng, lengths, 2, 20, whole=(0,)))
    check_compact(engine, lengths, np.full((4, 2, 20), -1, np.int32))
    # longer than the table's row: something is wrong with it
    kept = lists(rng, [100, 90], 2, 20)
    c = engine.PagedKVCache.empty(20, 2, 16, 64)
    t = dev(np.arange(12).reshape(2, 6), torch.int32)
    got = c.compact(t, dev([97, 90], torch.int32), dev(kept), dev(np.arange(20), torch.int32),
                    dev([12], torch.int32))
    assert got.lengths.tolist() == [97, 20] and got.cursor.tolist() == [8]


def test_cuts_with_pages_that_are_absent(engine):
    rng = np.random.default_rng(8)
    lengths = [200, 100]
    check_compact(engine, lengths, lists(rng, lengths, 2, 64), absent=[(0, 3), (0, 1), (1, 5)])


def test_cuts_of_keys_that_are_not_finite(engine):
    rng = np.random.default_rng(9)
    lengths = [200, 100]
    for fill in (math.inf, math.nan):
        check_compact(engine, lengths, lists(rng, lengths, 2, 64), fill=fill)


def test_cuts_of_many_requests(engine):
    rng = np.random.default_rng(10)
    lengths = rng.integers(0, 60, 1500)
    check_compact(engine, lengths, lists(rng, lengths, 1, 20), dim=8, seed=1)


def test_cuts_without_requests_and_refusals(engine):
    c = engine.PagedKVCache.empty(9, 2, 16, 64)
    i = dict(dtype=torch.int32, device="cuda")
    t, free, cur = torch.zeros(0, 4, **i), torch.arange(9, **i), torch.tensor([5], **i)
    got = c.compact(t, torch.zeros(0, **i), torch.zeros(0, 2, 8, **i), free, cur)
    assert got.lengths.numel() == 0 and got.cursor.tolist() == [5]
    t, n, kept = torch.zeros(2, 4, **i), torch.zeros(2, **i), torch.full((2, 2, 8), -1, **i)
    mass = torch.zeros(2, 2, 64, device="cuda")
    for bad in (dict(table=t.long()), dict(lengths=n[:1]), dict(kept=kept[:1]), dict(kept=kept[..., :0]),
                dict(kept=kept.long()), dict(free=free.long()), dict(cursor=free[:2]),
                dict(mass=mass[..., :63].contiguous()), dict(mass=mass.half()), dict(out=(n, cur)),
                dict(out=engine.KvCompact(n, torch.zeros(1, **i))),
                dict(out=engine.KvCompact(n.clone(), cur))):
        a = dict(table=t, lengths=n, kept=kept, free=free, cursor=cur)
        a.update(bad)
        with pytest.raises(ValueError, match="mlxvs"):
            c.compact(a.pop("table"), a.pop("lengths"), a.pop("kept"), a.pop("free"), a.pop("cursor"), **a)


def test_cuts_give_the_pages_back_that_a_plan_took(engine):
    i = dict(dtype=torch.int32, device="cuda")
    c = engine.PagedKVCache.empty(40, 2, 16, 64)
    table, free = torch.full((3, 20), -1, **i), torch.randperm(40, device="cuda").int()
    plan = engine.kv_plan(torch.zeros(3, **i), torch.tensor([200, 17, 100], **i), table, free,
                          torch.zeros(1, **i), 16, 320)
    assert plan.cursor.tolist() == [13 + 2 + 7]
    kept = lists(np.random.default_rng(0), [200, 17, 100], 2, 30)
    n, cur = c.compact(table, plan.lengths, dev(kept), free, plan.cursor)
    assert n.tolist() == [30, 17, 30] and cur.tolist() == [6]
    assert sorted(free[6:].tolist() + table[0, :2].tolist() + table[1, :2].tolist()
                  + table[2, :2].tolist()) == list(range(40))
    # every page is in the list or in one row, also after the next step
    plan = engine.kv_plan(n, torch.tensor([100, 300, 3], **i), table, free, cur, 16, 403)
    owned = [table[r, c_].item() for r, m in enumerate(plan.lengths.tolist()) for c_ in range(-(-m // 16))]
    assert plan.first.min() >= 0 and sorted(owned + free[plan.cursor.item():].tolist()) == list(range(40))


# ---- together ------------------------------------------------------------------


def test_a_cache_within_a_budget(engine):
    # requests grow a token a step over a budget and are cut to it; what the cache
    # answers is what attention over the kept tokens at their own positions is
    from mlxvs_amd import PagedKVCache

    rng = np.random.default_rng(1)
    heads, group, dim, page, budget, above = 2, 2, 64, 16, 40, 56
    i = dict(dtype=torch.int32, device="cuda")
    cache = PagedKVCache.empty(30, heads, page, dim)
    rot = engine.Rotary(dim, rotated=48, layout="pairs")
    norm = dev(1 + 0.2 * rng.standard_normal(dim)).to(torch.bfloat16)
    table, free = torch.full((3, 8), -1, **i), torch.randperm(30, device="cuda").int()
    lengths, cursor = torch.zeros(3, **i), torch.zeros(1, **i)
    evicted, mass = torch.zeros(3, **i), torch.full((3, heads, 8 * page), math.nan, device="cuda")
    texts = [[[] for _ in range(heads)] for _ in range(3)]  # (rotated key, value) of what is held
    cuts = 0
    for step in range(30):
        new = [50, 30, 3] if step == 0 else [1, 1, 7] if step % 2 else [1, 0, 1]
        plan = engine.kv_plan(lengths, torch.tensor(new, **i), table, free, cursor, page, 90)
        q, k, v = (rows(rng, 90, n, dim, "bf16") for n in (heads * group, heads, heads))
        q, k = rot.rotate(q, k, plan.positions, q_norm=norm, k_norm=norm, requests=plan.requests,
                          evicted=evicted)
        cache.append(k, v, plan.slots)
        out, lse = cache.attend(q, table, plan.requests, plan.positions, lse=True)
        cache.weigh(q, table, plan.starts, plan.positions, lse, mass, decay=0.9)
        starts = plan.starts.tolist()
        kf, vf, qf, of = (f32(x) for x in (k, v, q, out))
        for r in range(3):
            for t in range(starts[r], starts[r + 1]):
                for h in range(heads):
                    texts[r][h].append((kf[t, h], vf[t, h]))
                    kk = np.stack([x[0] for x in texts[r][h]]).astype(np.float64)
                    vv = np.stack([x[1] for x in texts[r][h]]).astype(np.float64)
                    for g in range(h * group, (h + 1) * group):
                        s = kk @ qf[t, g] / math.sqrt(dim)
                        p = np.exp(s - s.max())
                        # (bf16: weights and the output rounded once each)
                        bound = 2.0 ** -7 * 1.1 * (p @ np.abs(vv) / p.sum()) + 1e-6
                        assert (np.abs(of[t, g] - p @ vv / p.sum()) <= bound).all()
        kept = cache.keep(mass, plan.lengths, budget, first=2, recent=8, above=above)
        lengths, cursor = cache.compact(table, plan.lengths, kept, free, plan.cursor, mass=mass)
        evicted += plan.lengths - lengths
        which = kept.cpu().numpy()
        for r in range(3):
            if which[r, 0, 0] >= 0:
                cuts += 1
                for h in range(heads):
                    texts[r][h] = [texts[r][h][j] for j in which[r, h]]
        held = sum(-(-n // page) for n in lengths.tolist())
        assert cursor.tolist() == [held]
    # (the second request never holds more than 30 + 15 tokens)
    assert cuts >= 4 and evicted[0] > 0 and evicted[1] == 0 and evicted[2] > 0
    # the mass that is left belongs to the tokens that are left
    for r, n in enumerate(lengths.tolist()):
        assert mass[r, :, :n].isfinite().all()


def test_a_captured_step_with_a_budget(engine):
    i = dict(dtype=torch.int32, device="cuda")
    heads, dim, page, budget = 2, 64, 16, 24
    rng = np.random.default_rng(2)
    rot = engine.Rotary(dim)

    def fresh():
        g = torch.Generator(device="cuda").manual_seed(1)
        cache = engine.PagedKVCache.empty(24, heads, page, dim)
        return dict(cache=cache, table=torch.full((2, 6), -1, **i),
                    free=torch.randperm(24, generator=g, device="cuda").int(),
                    lengths=torch.zeros(2, **i), cursor=torch.zeros(1, **i),
                    evicted=torch.zeros(2, **i), mass=torch.zeros(2, heads, 96, device="cuda"),
                    new=torch.ones(2, **i), x=torch.zeros(32, 4 * heads, dim, dtype=torch.bfloat16,
                                                          device="cuda"),
                    out=torch.zeros(32, 2 * heads, dim, dtype=torch.bfloat16, device="cuda"))

    def step(s):
        plan = engine.kv_plan(s["lengths"], s["new"], s["table"], s["free"], s["cursor"], page, 32)
        q, k = rot.rotate(s["x"][:, :2 * heads], s["x"][:, 2 * heads:3 * heads], plan.positions,
                          requests=plan.requests, evicted=s["evicted"])
        s["cache"].append(k, s["x"][:, 3 * heads:], plan.slots)
        out, lse = s["cache"].attend(q, s["table"], plan.requests, plan.positions, lse=True)
        s["cache"].weigh(q, s["table"], plan.starts, plan.positions, lse, s["mass"])
        kept = s["cache"].keep(s["mass"], plan.lengths, budget, first=1, recent=4, above=40)
        n, cur = s["cache"].compact(s["table"], plan.lengths, kept, s["free"], plan.cursor,
                                    mass=s["mass"])
        s["evicted"] += plan.lengths - n
        s["lengths"].copy_(n)
        s["cursor"].copy_(cur)
        s["out"].copy_(out)

    eager, graphed = fresh(), fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    warm = fresh()
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(graphed)
    for n in range(24):
        x = rows(rng, 32, 4 * heads, dim, "bf16")
        new = dev([15 if n % 3 == 0 else 2, 3], torch.int32)
        for s in (eager, graphed):
            s["x"].copy_(x)
            s["new"].copy_(new)
        step(eager)
        graph.replay()
        torch.cuda.synchronize()
        for name in ("lengths", "cursor", "evicted", "free", "table", "mass", "out"):
            assert torch.equal(eager[name], graphed[name]), (n, name)
        for name in ("keys", "values", "summaries", "scales"):
            assert torch.equal(getattr(eager["cache"], name), getattr(graphed["cache"], name)), (n, name)
    assert eager["evicted"].min() > 0


def test_calls_run_on_the_current_stream(engine):
    # each call's inputs are made on another stream just before it
    s = Step(engine, [400, 300], [100, 1], page=64, dim=128, seed=3).attend()
    want = s.mass.clone()
    s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, want)
    rot = engine.Rotary(128)
    turned, _ = rot.rotate(s.q, None, s.positions)
    lengths = dev([400, 300], torch.int32)
    kept = s.cache.keep(want, lengths, 100)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        busy = torch.randn(2048, 2048, device="cuda")
        for _ in range(20):
            busy = busy @ busy * 1e-3
        mass, q = s.mass + 0.0 * busy[0, 0].nan_to_num(), s.q * 1
        mass = s.mass.clone()
        s.cache.weigh(q, s.table, s.starts, s.positions, s.lse, mass)
        again, _ = rot.rotate(q, None, s.positions)
        kept2 = s.cache.keep(mass, lengths, 100)
    stream.synchronize()
    assert torch.equal(mass, want) and torch.equal(again, turned) and torch.equal(kept, kept2)


def test_the_example_within_a_budget(engine):
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parent.parent / "examples" / "paged_cache.py"
    spec = importlib.util.spec_from_file_location("paged_cache", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    lengths, close, ms = example.run(requests=3, context=900, steps=70, blocks=4, budget=256)
    # (prompts of 593 and 886 tokens cut to 256, and again after 64; one of 300 after 20)
    assert lengths == [256 + 50, 256 + 6, 256 + 6] and math.isfinite(close) and ms > 0
    assert example.run(requests=2, context=100, steps=3, blocks=4, budget=1)[0] == [53, 4]


def test_budgets_of_numbers_past_32_bits(engine):
    c = engine.PagedKVCache.empty(1, 2, 16, 64)
    mass, lengths = torch.rand(1, 2, 64, device="cuda"), dev([50], torch.int32)
    assert (c.keep(mass, lengths, 8, above=2 ** 33) == -1).all()
    for k in (dict(first=2 ** 32), dict(recent=2 ** 32 + 1)):
        with pytest.raises(ValueError, match="below 2"):
            c.keep(mass, lengths, 8, **k)


def test_offsets_past_32_bits_of_rows(engine):
    # places 2^30 values apart
    rng = np.random.default_rng(0)
    room = torch.empty(5 * 2 ** 29 + 1024, dtype=torch.bfloat16, device="cuda")
    q, k = rows(rng, 3, 4, 64, "bf16"), rows(rng, 3, 2, 64, "bf16")
    far = room.as_strided((3, 4, 64), (2 ** 30, 64, 1))
    far_k = room.as_strided((3, 2, 64), (2 ** 30, 64, 1), 512)
    far.copy_(q)
    far_k.copy_(k)
    pos = dev([5, 70_000, 2 ** 31 - 1], torch.int32)
    for rotated in (64, 20):
        rot = engine.Rotary(64, rotated=rotated)
        want = rot.rotate(q, k, pos)
        got = rot.rotate(far, far_k, pos)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    rot.rotate(far, far_k, pos, out=(far, far_k))
    assert torch.equal(far, want[0]) and torch.equal(far_k, want[1])


def test_offsets_past_32_bits_of_a_cache(engine):
    # the same step over pages at both ends of a cache of more than 2^31 values
    heads, page, dim = 8, 64, 128
    lengths, counts = [500, 300], [200, 1]
    pages = 2 ** 31 // (heads * page * dim) + 40
    near = Step(engine, lengths, counts, page=page, heads=heads, group=2, dim=dim, seed=2).attend()
    cache = engine.PagedKVCache.empty(pages, heads, page, dim)
    held = near.cache.keys.shape[0]
    for name in ("keys", "values", "summaries", "scales"):
        getattr(cache, name)[pages - held:].copy_(getattr(near.cache, name))
    table = torch.where(near.table >= 0, near.table + (pages - held), near.table)
    for n in (201, 2):  # prompts, and a token each
        s = near
        if n == 2:
            s = Step(engine, lengths, [1, 1], page=page, heads=heads, group=2, dim=dim, seed=2).attend()
        want, mass = s.mass.clone(), s.mass.clone()
        s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, want)
        cache.weigh(s.q, table, s.starts, s.positions, s.lse, mass)
        assert len(s.q) == n and torch.equal(mass, want)
    kept = near.cache.keep(want, dev(lengths, torch.int32), 130)
    i = dict(dtype=torch.int32, device="cuda")
    for c, t, m in ((near.cache, near.table, want), (cache, table, mass)):
        free = torch.full((40,), -7, **i)
        out = c.compact(t, dev(lengths, torch.int32), kept, free, dev([30], torch.int32), mass=m)
        assert out.lengths.tolist() == [130, 130] and out.cursor.tolist() == [30 - 5 - 2]
    assert torch.equal(mass, want)
    for name in ("keys", "values", "summaries", "scales"):
        a, b = getattr(cache, name)[pages - held:], getattr(near.cache, name)
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name


def test_offsets_past_32_bits_of_masses(engine):
    requests, heads, slots = 4_200, 8, 65_536
    c = engine.PagedKVCache.empty(1, heads, 16, 64)
    mass = torch.empty(requests, heads, slots, device="cuda")
    lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")
    lengths[-1] = 6_000
    row = torch.rand(1, heads, slots, device="cuda")
    mass[-1].copy_(row[0])
    want = c.keep(row, lengths[-1:], 100)
    got = c.keep(mass, lengths, 100)
    assert torch.equal(got[-1], want[0]) and (got[:-1] == -1).all()
