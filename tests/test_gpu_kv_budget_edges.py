"""The paged cache's budget at its edges, on the GPU: caches without pages, batches
and rows of the largest kernels, wide tables, tensors written in place.  Bounds as
in test_gpu_kv_budget.py."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_gpu_kv import dev  # noqa: E402
from test_gpu_kv_budget import Step  # noqa: E402

pytestmark = pytest.mark.gpu


def weights(s, mass, decay=1.0):
    """float64 (mass, err) of a Step: kv_budget_oracle.weigh's sums and bounds in
    products over all keys of a request, for many of them."""
    keys, table = s.cache.keys, s.table.long()
    pages, heads, page, d = keys.shape
    out, err = mass.double(), torch.zeros(mass.shape, dtype=torch.float64, device="cuda")
    starts, positions = s.starts.tolist(), s.positions.tolist()
    most, group = table.shape[1] * page, s.q.shape[1] // heads
    for r in range(len(table)):
        a, b = starts[r], starts[r + 1]
        if a == b or positions[a] < 0:
            continue
        first, n = positions[a], min(positions[b - 1] + 1, most)
        p = torch.arange(n, device="cuda")
        pid = table[r, p // page]
        there = (pid >= 0) & (pid < pages)
        k = keys[torch.where(there, pid, 0), :, p % page].double().permute(1, 2, 0).contiguous()
        got, off, sees = (torch.zeros(heads, n, dtype=torch.float64, device="cuda") for _ in range(3))
        step = max(1, (1 << 25) // (heads * group * n))
        for t in range(a, b, step):
            u = min(b, t + step)
            x = s.q[t:u].double().unflatten(1, (heads, group)).transpose(0, 1).flatten(1, 2)
            lse = s.lse[t:u].double().unflatten(1, (heads, group)).transpose(0, 1).flatten(1, 2)[..., None]
            see = (s.positions[t:u, None] >= p).repeat_interleave(group, 0)
            score = x @ k * s.scale
            e = torch.where(see, torch.exp(score - lse), 0.0)
            w = e * ((d + 4) * (x.abs() @ k.abs()) * s.scale + 4 * (score.abs() + lse.abs()) + 16)
            got += e.sum(1)
            off += torch.where(see, w, 0.0).sum(1)
            sees += see.sum(0)
        off = torch.where(there, off + sees * got, 0.0)
        got = torch.where(there, got, 0.0)
        before = torch.where(p < first, decay * out[r, :, :n], 0.0) if decay else torch.zeros_like(got)
        out[r, :, :n] = before + got
        err[r, :, :n] = off + 2 * before.abs() + 2 * got.abs()
    return out, err


def check_weights(s, decay=1.0, **how):
    want, err = weights(s, s.mass, decay)
    again = s.mass.clone()
    s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, s.mass, decay=decay, **how)
    s.cache.weigh(s.q, s.table, s.starts, s.positions, s.lse, again, decay=decay, **how)
    bad = ~((s.mass.double() - want).abs() <= err * 2.0 ** -24 + 1e-37)
    assert not bad.any(), (bad.nonzero()[:5], s.mass[bad][:5], want[bad][:5])
    assert torch.equal(s.mass, again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts", [[40, 3], [1, 1]])
def test_weights_of_a_cache_without_pages(engine, counts, dtype):
    # no key gets anything: what was there decays, the step's own keys start from zero
    c = engine.PagedKVCache.empty(0, 2, 16, 64, dtype=dtype)
    i = dict(dtype=torch.int32, device="cuda")
    tokens, past = sum(counts), [7, 20]
    positions = torch.tensor([p + t for p, n in zip(past, counts) for t in range(n)], **i)
    starts = torch.tensor([0, counts[0], tokens], **i)
    q = torch.randn(tokens, 6, 64, device="cuda").to(dtype)
    lse = torch.full((tokens, 6), -math.inf, device="cuda")
    for table in (torch.full((2, 5), -1, **i), torch.zeros(2, 5, **i)):
        mass = torch.rand(2, 2, 80, device="cuda")
        want = mass.clone()
        for r in range(2):
            want[r, :, :past[r]] *= 0.5
            want[r, :, past[r]:past[r] + counts[r]] = 0
        c.weigh(q, table, starts, positions, lse, mass, decay=0.5)
        assert torch.equal(mass, want)


@pytest.mark.parametrize("longest", [0, 100, 1_800])
def test_weights_of_more_keys_than_a_call_has_workgroups_for(engine, longest):
    # 70 x 64 rows of keys, 3 workgroups of 256 keys each; and one for each of 300 x 64
    rng = np.random.default_rng(longest)
    lengths = rng.integers(1, 1_800, 70)
    lengths[[3, 69]] = 1_800, 769
    s = Step(engine, lengths, [1] * 70, page=64, heads=64, group=1, dim=8, spare=30, seed=1).attend()
    check_weights(s, decay=0.5, longest=longest)
    lengths = rng.integers(0, 600, 300)
    counts = np.minimum(lengths, rng.integers(0, 2, 300))
    check_weights(Step(engine, lengths, counts, page=64, heads=64, group=2, dim=8, seed=2).attend(),
                  longest=longest)


def test_weights_of_few_tokens_beside_prompts_in_many_keys(engine):
    # 20 x 64 rows, 6 workgroups of 256 keys each for the requests of up to 32 rows
    lengths = [2_500, 1_537, 1, 40, 0, 1_900] + [300 + 7 * i for i in range(14)]
    counts = [1, 32, 1, 40, 0, 33] + [i % 3 for i in range(14)]
    check_weights(Step(engine, lengths, counts, page=64, heads=64, group=1, dim=8, spare=9,
                       seed=3).attend(), decay=0.5)


@pytest.mark.parametrize("group,dim,dtype", [(1, 8, "bf16"), (3, 72, "f16"), (40, 24, "f16"),
                                             (64, 16, "bf16")])
def test_weights_of_a_prompt_among_idle_rows(engine, group, dim, dtype):
    # a table with room for 8 million keys: the rows are idle, have a token each, or are
    # few and many tokens', with fewer tokens than rows
    n = 600
    idle = [0] * (n - 1)
    for lengths, counts in (([900] + idle, [n] + idle),
                            ([300] + [20] * 500 + [0] * 99, [77] + [1] * 500 + [0] * 99),
                            ([40] * 10 + [1_300] * 3 + idle[:-11], [2] * 10 + [34, 190, 1] + idle[:-11])):
        s = Step(engine, lengths, counts, page=64, heads=2, group=group, dim=dim, dtype=dtype,
                 spare=-(-8_192 // 64) - -(-max(lengths) // 64), seed=dim).attend()
        assert sum(counts) <= len(lengths) and s.mass.numel() >= 8 << 20
        check_weights(s, decay=0.5)
        s.positions[:s.starts[1].item()] = -1  # (the first one was not admitted)
        check_weights(s)


def step_in_place(engine, requests=2, heads=2, dim=64, page=16):
    """Everything that a step with a budget writes, by name, and the step."""
    i = dict(dtype=torch.int32, device="cuda")
    c = engine.PagedKVCache.empty(20, heads, page, dim)
    t = dict(keys=c.keys, values=c.values, summaries=c.summaries, scales=c.scales,
             table=torch.full((requests, 6), -1, **i), free=torch.arange(20, **i),
             mass=torch.zeros(requests, heads, 6 * page, device="cuda"),
             q=torch.randn(90, 2 * heads, dim, device="cuda").bfloat16(),
             k=torch.randn(90, heads, dim, device="cuda").bfloat16(),
             out=torch.zeros(90, 2 * heads, dim, device="cuda").bfloat16(),
             lengths=torch.zeros(requests, **i), cursor=torch.zeros(1, **i))
    zero = torch.zeros(requests, **i)

    def step():
        plan = engine.kv_plan(zero, torch.tensor([60, 30], **i), t["table"], t["free"],
                              torch.zeros(1, **i), page, 90)
        engine.Rotary(dim).rotate(t["q"], t["k"], plan.positions, out=(t["q"], t["k"]))
        c.append(t["k"], t["k"], plan.slots)
        _, lse = c.attend(t["q"], t["table"], plan.requests, plan.positions, lse=True, out=t["out"])
        c.weigh(t["q"], t["table"], plan.starts, plan.positions, lse, t["mass"])
        kept = c.keep(t["mass"], plan.lengths, 20)
        c.compact(t["table"], plan.lengths, kept, t["free"], plan.cursor, mass=t["mass"],
                  out=engine.KvCompact(t["lengths"], t["cursor"]))

    return t, step


def test_what_is_written_in_place_is_told_to_autograd(engine):
    t, step = step_in_place(engine)
    before = {name: x._version for name, x in t.items()}
    step()
    assert all(x._version > before[name] for name, x in t.items()), before
    assert t["lengths"].tolist() == [20, 20]
    # a backward pass that needs what was there before is an error
    for name in ("keys", "mass", "q", "k", "out"):
        w = torch.ones((), device="cuda", requires_grad=True)
        y = (w * t[name]).sum()
        step()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    # what is only read is not
    t, step = step_in_place(engine)
    q, pos = t["q"], torch.arange(90, dtype=torch.int32, device="cuda")
    at = q._version, pos._version
    engine.Rotary(64).rotate(q, t["k"], pos)
    assert (q._version, pos._version) == at


def test_steps_in_place_in_inference_mode(engine):
    with torch.inference_mode():
        t, step = step_in_place(engine)
        step()
    step()  # (tensors made there have no versions)
    assert t["lengths"].tolist() == [20, 20]


def test_masses_that_want_a_gradient(engine):
    s = Step(engine, [20, 30], [2, 3]).attend()
    args = s.q, s.table, s.starts, s.positions, s.lse
    want = s.mass.clone()
    s.cache.weigh(*args, want)
    lengths, kept = dev([20, 30], torch.int32), s.cache.keep(want, dev([20, 30], torch.int32), 9)
    free, cursor = dev(np.arange(9), torch.int32), dev([5], torch.int32)
    mass = s.mass.clone().requires_grad_()
    for m in (mass, mass * 1):
        with pytest.raises(ValueError, match="gradient"):
            s.cache.weigh(*args, m)
        with pytest.raises(ValueError, match="gradient"):
            s.cache.compact(s.table, lengths, kept, free, cursor, mass=m)
        assert torch.equal(m, s.mass)
    with torch.no_grad():
        s.cache.weigh(*args, mass)
    assert torch.equal(mass, want)
    # values are added: no gradient goes back to queries
    again = s.mass.clone()
    s.cache.weigh(s.q.requires_grad_(), *args[1:], again)
    assert torch.equal(again, want) and not again.requires_grad


def test_budget_of_a_row_of_nearly_two_to_the_31_slots(engine):
    # its last part ends at 2^31: ties go to the lowest, marks lie in the first and last parts
    slots = 2 ** 31 - 1
    c = engine.PagedKVCache.empty(1, 1, 16, 16)
    mass = torch.zeros(1, 1, slots, device="cuda")
    marks = [70_000, 2 ** 30 + 1, slots - 65_535, slots - 3]
    mass[0, 0, torch.tensor(marks, device="cuda")] = dev([1.0, 3.0, 2.0, 4.0], torch.float32)
    for length, want in ((slots, [0, 1, 2, *marks, slots - 1]),
                         (slots - 2, [0, 1, 2, *marks]),
                         (slots - 65_536, [0, 1, 2, 3, 4, *marks[:2], slots - 65_537])):
        kept = c.keep(mass, dev([length], torch.int32), len(want), first=1, recent=1)
        assert kept.flatten().tolist() == want, length


def check_keep(engine, mass, lengths, n, first, recent):
    """kept against a stable sort of float64 masses, for long rows."""
    c = engine.PagedKVCache.empty(1, mass.shape[1], 16, 16)
    got = c.keep(dev(mass), dev(lengths, torch.int32), n, first=first, recent=recent).cpu().numpy()
    for r, length in enumerate(lengths):
        for h in range(mass.shape[1]):
            if length <= n:
                assert (got[r, h] == -1).all()
                continue
            # (lexsort's last key counts most: NaN at the end, then the greatest first, then
            # the lowest position)
            x = mass[r, h, first:length - recent].astype(np.float64)
            best = np.lexsort((np.arange(len(x)), -np.nan_to_num(x), np.isnan(x)))
            want = np.concatenate([np.arange(first), first + np.sort(best[:n - first - recent]),
                                   np.arange(length - recent, length)])
            assert np.array_equal(got[r, h], want), (r, h)


@pytest.mark.parametrize("slots,part", [(262_144, 8_192), (262_145, 16_384), (524_288, 16_384),
                                        (524_289, 32_768), (1_048_577, 65_536), (2_500_000, 65_536)])
def test_budgets_of_rows_in_parts_of_any_size(engine, slots, part):
    # ties of the cut over several parts' borders, rows that end within a part or at its
    # border, parts without tokens
    rng = np.random.default_rng(slots)
    mass = rng.integers(0, 40, (4, 1, slots)).astype(np.float32)
    mass[1] = rng.lognormal(0, 2, (1, slots))
    mass[2, :, part - 300:part + 300] = 100.0
    mass[3, :, ::5], mass[3, :, 1::7] = math.nan, -math.inf
    lengths = [slots, slots - 1, 3 * part, part + 1]
    for n in (1, 500, part, part + 7, slots // 2, slots - 2):
        check_keep(engine, mass, lengths, n, min(4, n // 2), min(128, n // 3))


def test_weights_of_more_shares_than_workgroups(engine):
    # 64 heads leave 32 workgroups to each, which take several shares one after another
    s = Step(engine, [2_100, 3_000, 1_500, 700, 4_500], [2_100, 1_000, 1, 700, 300], page=64, heads=64,
             group=1, dim=8, seed=1).attend()
    check_weights(s, decay=0.5)
    s = Step(engine, [1_300, 1_024, 2_000], [1_200, 1_024, 7], page=128, heads=128, group=2, dim=16,
             dtype="f16", seed=2).attend()
    check_weights(s)


@pytest.mark.parametrize("dim", [16, 192])
def test_weights_of_more_chunks_than_the_plan_takes_at_a_time(engine, dim):
    # 14 requests over the same pages: 1,024 chunks of 256 keys and more, some in several
    # shares, the last ones in a pass of their own
    long, page = 20_480, 256
    s = Step(engine, [long], [0], page=page, heads=1, group=2, dim=dim, seed=dim)
    s.cache.keys[:long // page] = torch.randn(long // page, 1, page, dim, device="cuda").bfloat16()
    lengths = np.array([long - 250 * i for i in range(14)])
    counts = np.array([3, 1, 900, 40, 5, 300, 64, 1, 2, 33, 1, 450, 7, 1_200])
    s.table = torch.randperm(long // page, device="cuda").int().expand(14, -1).contiguous()
    s.starts = dev(np.concatenate([[0], np.cumsum(counts)]), torch.int32)
    s.positions = dev(np.concatenate([np.arange(n - m, n) for n, m in zip(lengths, counts)]), torch.int32)
    s.requests = dev(np.repeat(np.arange(14), counts), torch.int32)
    s.q = torch.randn(counts.sum(), 2, dim, device="cuda").bfloat16()
    s.mass = torch.rand(14, 1, long, device="cuda")
    assert sum(-(-n // 256) for n in lengths) > 1_024
    check_weights(s.attend(), decay=0.5)


@pytest.mark.parametrize("bad", [None, 3, [1.0, 2.0], np.zeros((3, 4, 64), np.float32)])
def test_what_is_no_tensor_is_refused(engine, bad):
    rot, s = engine.Rotary(64), Step(engine, [20, 30], [2, 3]).attend()
    q, pos = s.q[:, :, :64], s.positions
    lengths, kept = dev([20, 30], torch.int32), torch.full((2, 2, 4), -1, dtype=torch.int32, device="cuda")
    free, cursor = dev(np.arange(9), torch.int32), dev([5], torch.int32)
    calls = [lambda: rot.rotate(bad, q, pos), lambda: rot.rotate(q, q, bad),
             lambda: rot.rotate(q, q, pos, evicted=pos, requests=bad),
             lambda: s.cache.weigh(bad, s.table, s.starts, pos, s.lse, s.mass),
             lambda: s.cache.weigh(q, bad, s.starts, pos, s.lse, s.mass),
             lambda: s.cache.weigh(q, s.table, bad, pos, s.lse, s.mass),
             lambda: s.cache.weigh(q, s.table, s.starts, bad, s.lse, s.mass),
             lambda: s.cache.weigh(q, s.table, s.starts, pos, bad, s.mass),
             lambda: s.cache.weigh(q, s.table, s.starts, pos, s.lse, bad),
             lambda: s.cache.keep(bad, lengths, 4), lambda: s.cache.keep(s.mass, bad, 4),
             lambda: s.cache.compact(bad, lengths, kept, free, cursor),
             lambda: s.cache.compact(s.table, bad, kept, free, cursor),
             lambda: s.cache.compact(s.table, lengths, bad, free, cursor),
             lambda: s.cache.compact(s.table, lengths, kept, bad, cursor),
             lambda: s.cache.compact(s.table, lengths, kept, free, bad)]
    if bad is not None:
        calls += [lambda: rot.rotate(q, bad, pos), lambda: rot.rotate(q, q, pos, q_norm=bad),
                  lambda: rot.rotate(q, q, pos, k_norm=bad), lambda: rot.rotate(q, q, pos, out=bad),
                  lambda: rot.rotate(q, q, pos, out=(q, bad)),
                  lambda: rot.rotate(q, q, pos, evicted=bad, requests=pos),
                  lambda: s.cache.compact(s.table, lengths, kept, free, cursor, mass=bad),
                  lambda: s.cache.compact(s.table, lengths, kept, free, cursor, out=bad)]
    for call in calls:
        with pytest.raises(ValueError, match="mlxvs::kv_"):
            call()
    # (of no, one or two axes)
    for mass in (s.mass[0, 0, 0], s.mass[0, 0], s.mass[0]):
        with pytest.raises(ValueError, match="mass must be"):
            s.cache.compact(s.table, lengths, kept, free, cursor, mass=mass)
