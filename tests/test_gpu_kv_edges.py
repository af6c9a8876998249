"""The paged key-value cache's operators at their limits: lists that are partly
empty beside other tables, extreme positions and values, moved tensors."""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv_oracle  # noqa: E402
from test_gpu_kv import (DTYPES, check_attend, check_select, dev, f32, make_cache,  # noqa: E402
                         summaries, tables)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("n", [3, 40, 256])
def test_ragged_lists_over_a_view_of_a_wider_table(engine, n, page):
    """The view's spare columns, and the row after its last, name pages too
    (of nothing but NaN): they are nobody's."""
    rng = np.random.default_rng(n + page)
    heads, group, dim, cols, tokens = 64, 8, 32, 9, 40
    cache = make_cache(engine, 2 * cols + 1, heads, page, dim, "bf16", rng)
    cache.keys[-1] = cache.values[-1] = float("nan")
    wide = torch.full((3, 300), 2 * cols, dtype=torch.int32, device="cuda")
    ids = tables(rng, 2 * cols, 2, cols)
    wide[:2, :cols] = dev(ids)
    view = wide[:2, :cols]
    who = (np.arange(tokens) >= 25).astype(np.int32)
    positions = rng.integers(0, cols * page, tokens)
    q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).bfloat16()
    # another call's full lists first: what it leaves in LDS are blocks past this table
    other = engine.PagedKVCache.empty(300, heads, page, dim)
    full = dev(np.tile(np.arange(300 - n, 300), (tokens, heads, 1)), torch.int32)
    other.attend(q, torch.arange(300, dtype=torch.int32, device="cuda")[None],
                 torch.zeros(tokens, dtype=torch.int32, device="cuda"),
                 torch.full((tokens,), 300 * page - 1, dtype=torch.int32, device="cuda"),
                 blocks=full)
    blocks = rng.integers(-2, cols + 3, (tokens, heads, n))
    blocks[:, :, 2:] = np.where(rng.random((tokens, heads, max(0, n - 2))) < 0.9, -1, blocks[:, :, 2:])
    blocks[::3] = -1
    blocks[::3, :, 0] = 0
    got = cache.attend(q, view, dev(who), dev(positions, torch.int32), blocks=dev(blocks, torch.int32))
    assert torch.equal(got, check_attend(cache, "bf16", q, ids, who, positions, blocks=blocks))


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("heads,group,page,dim,tokens",
                         [(2, 4, 16, 64, 6), (1, 3, 64, 80, 1), (64, 8, 64, 64, 40), (64, 4, 16, 128, 40),
                          (64, 16, 32, 40, 26)])
def test_the_largest_position_sees_the_whole_table(engine, heads, group, page, dim, tokens, listed):
    """Beside tokens that see less, whose values past it stay hidden and whose own stay."""
    rng = np.random.default_rng(heads + page)
    cols = 5
    cache = make_cache(engine, 2 * cols, heads, page, dim, "bf16", rng)
    table = tables(rng, 2 * cols, 2, cols)
    who = (np.arange(tokens) % 7 == 3).astype(np.int32)
    positions = rng.integers(0, cols * page, tokens)
    positions[::3] = np.iinfo(np.int32).max - rng.integers(0, 3, len(positions[::3]))
    positions[0] = np.iinfo(np.int32).max
    q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).bfloat16()
    blocks = rng.integers(-1, cols + 1, (tokens, heads, 4)) if listed else None
    if listed:
        blocks[0] = [0, 4, 2, -1]
    got = check_attend(cache, "bf16", q, table, who, positions, blocks=blocks)
    edge = np.minimum(positions, cols * page - 1)
    assert torch.equal(got, check_attend(cache, "bf16", q, table, who, edge, blocks=blocks))


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("heads,group,page,dim,tokens",
                         [(64, 4, 64, 128, 45), (64, 5, 16, 80, 40), (128, 1, 32, 64, 70),
                          (40, 33, 64, 64, 21), (64, 8, 128, 192, 33), (64, 16, 32, 256, 24),
                          (96, 3, 256, 40, 50)])
def test_values_that_are_not_finite_reach_who_sees_them(engine, heads, group, page, dim, tokens, listed):
    """And nobody else: not the neighbours, another request's tokens or idle ones."""
    rng = np.random.default_rng(heads + group)
    cols = 6
    cache = make_cache(engine, 2 * cols, heads, page, dim, "f16", rng)
    table = np.arange(2 * cols, dtype=np.int32).reshape(2, cols)
    who = (np.arange(tokens) % 9 == 4).astype(np.int32)
    positions = np.sort(rng.integers(0, cols * page, tokens))
    positions[5] = -1
    q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).half()
    blocks = rng.integers(-1, cols, (tokens, heads, 3)) if listed else None
    want = check_attend(cache, "f16", q, table, who, positions, blocks=blocks)
    # of request 0, a key in the middle and one of its first block
    bad = [(3 * page + 9, 2, float("inf")), (3 * page + 9, dim - 1, float("nan")),
           (5, 7, float("-inf")), (3 * page + 9, 7, float("inf"))]
    for key, d, x in bad:
        cache.values[key // page, :, d, key % page] = x
    got = cache.attend(q, dev(table), dev(who), dev(positions, torch.int32),
                       blocks=None if blocks is None else dev(blocks, torch.int32))
    got, want = f32(got), f32(want)
    key_in = lambda k: (who == 0)[:, None] & (positions >= k)[:, None] & (  # noqa: E731
        np.ones((tokens, heads), bool) if blocks is None else (blocks == k // page).any(2))
    mid, low = (np.repeat(key_in(k), group, 1) for k in (3 * page + 9, 5))
    want[..., 2][mid] = np.inf
    want[..., dim - 1][mid] = np.nan
    want[..., 7] = np.where(mid & low, np.nan, np.where(mid, np.inf, np.where(low, -np.inf, want[..., 7])))
    assert np.array_equal(got, want, equal_nan=True)


def best_time(call, n=4):
    times = []
    for _ in range(n):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


def test_what_one_infinite_value_costs(engine):
    """A second round over a workgroup's tiles, not one for each of its tokens."""
    rng = np.random.default_rng(4)
    heads, page, dim, cols, tokens = 64, 64, 64, 32, 512
    cache = make_cache(engine, cols, heads, page, dim, "bf16", rng)
    q = dev(rng.standard_normal((tokens, heads, dim), np.float32)).bfloat16()
    table, who = dev(np.arange(cols)[None], torch.int32), dev(np.zeros(tokens), torch.int32)
    positions = dev(np.arange(tokens) + cols * page - tokens, torch.int32)

    def spent():
        return best_time(lambda: cache.attend(q, table, who, positions))

    clean = spent()
    cache.values[0, :, 3, 5] = float("inf")
    # (measured: 2.4 times as long; with a round for each of 64 tokens 53 times)
    assert spent() < 6 * clean


@pytest.mark.parametrize("cols,tokens,heads", [(60, 5, 2), (300, 16, 64), (2300, 2, 2)])
def test_scales_that_are_not_finite_rank_first(engine, cols, tokens, heads):
    """Of either sign, by rows, by tiles and in parts."""
    rng = np.random.default_rng(cols)
    codes, scales = summaries(rng, 400, heads, 32)
    for i, x in enumerate((-np.inf, np.inf, np.nan, -np.inf, -3e38, 3e38)):
        scales[10 + 7 * i] = x
    codes[31], scales[17] = 0, -np.inf
    table = rng.permutation(400)[np.arange(2 * cols) % 400].reshape(2, cols).astype(np.int32)
    who = np.zeros(tokens, int)
    positions = cols * 16 - 1 - 3 * np.arange(tokens)
    q = dev(rng.standard_normal((tokens, heads * 2, 32), np.float32)).bfloat16()
    for n in (4, 9, 40):
        check_select(engine, q, codes, scales, table, who, positions, 16, n)


def test_select_of_more_than_four_million_rows(engine):
    rng = np.random.default_rng(13)
    heads, d, cols, tokens = 8, 16, 6, 530_000
    codes, scales = summaries(rng, 20, heads, d)
    cache = engine.PagedKVCache(torch.empty((20, heads, 16, d), dtype=torch.bfloat16, device="cuda"),
                                torch.empty((20, heads, d, 16), dtype=torch.bfloat16, device="cuda"),
                                dev(codes), dev(scales))
    table = tables(rng, 20, 2, cols)
    q = torch.randn((tokens, heads, d), device="cuda", dtype=torch.bfloat16)
    who = (np.arange(tokens) >= 300_000).astype(np.int32)
    positions = rng.integers(0, cols * 16, tokens).astype(np.int32)
    got = cache.select(q, dev(table), dev(who), dev(positions), 3)
    some = np.r_[:20, 299_990:300_010, 524_280:524_300, tokens - 20:tokens]
    want = kv_oracle.select(f32(q[dev(some)]), codes, scales, table, who[some], positions[some], 16,
                            3, 1, 1)
    assert np.array_equal(got[dev(some)].cpu().numpy(), want)


def test_a_cache_keeps_its_tensors(engine):
    """Other ones are another cache's; memory that has moved is not used."""
    def make():
        return engine.PagedKVCache.empty(4, 2, 16, 64)

    kv = torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(3, device="cuda")
    who = torch.zeros(3, dtype=torch.int32, device="cuda")
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    cache = make()
    for name in ("keys", "values", "summaries", "scales"):
        with pytest.raises(AttributeError):
            setattr(cache, name, getattr(cache, name).clone())
    cache.append(kv, kv, slots)
    for name, move in (("keys", lambda x: x.resize_(40, 2, 16, 64)),
                       ("values", lambda x: x.set_(torch.empty_like(x))),
                       ("summaries", lambda x: x.untyped_storage().resize_(0)),
                       ("scales", lambda x: x.set_(torch.zeros(1, device="cuda")))):
        cache = make()
        cache.append(kv, kv, slots)
        move(getattr(cache, name))
        for call in (lambda: cache.append(kv, kv, slots), lambda: cache.select(kv, table, who, who, 2),
                     lambda: cache.attend(kv, table, who, who)):
            with pytest.raises(ValueError, match="have moved"):
                call()


def test_a_plan_whose_tensors_have_moved(engine):
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    table = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    free, cursor = torch.arange(9, dtype=torch.int32, device="cuda"), torch.zeros_like(one[:1])

    def plan(out=None):
        return engine.kv_plan(0 * one, one, table, free, cursor, 16, 5, out=out)

    out = plan()
    assert plan(out) is out and out.slots.tolist() == [0, 16, -1, -1, -1]
    out.slots.resize_(5000)
    with pytest.raises(ValueError, match="out.slots"):
        plan(out)
    out = plan()
    out.first.set_(torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="out.first"):
        plan(out)
    out = plan()
    other = torch.full((2,), 7, dtype=torch.int32, device="cuda")
    out.first.set_(other)  # (other memory of the right size is as good)
    assert plan(out).first.tolist() == [0, 1] and other.tolist() == [0, 1]
    with pytest.raises(ValueError, match="KvPlan"):
        plan(tuple(out))
    with pytest.raises(ValueError, match="out.slots"):
        plan(engine.KvPlan(*[None] * 7))


def test_a_gradient_that_is_asked_for_is_an_error(engine):
    cache = engine.PagedKVCache.empty(2, 2, 16, 64)
    cache.keys.normal_()
    cache.values.normal_()
    wide = torch.randn((3, 4, 65), device="cuda").bfloat16()
    table = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    who, positions = torch.zeros(3, dtype=torch.int32, device="cuda"), dev([3, 0, -1], torch.int32)
    for q in (wide[..., :64].contiguous(), wide[..., 1:]):  # (the second is copied by the call)
        want, sums = cache.attend(q, table, who, positions, lse=True)
        assert not want.requires_grad and not sums.requires_grad
        leaf = q.detach().requires_grad_()
        got, lse = cache.attend(leaf, table, who, positions, lse=True)
        assert torch.equal(got, want) and torch.equal(lse, sums)
        for loss in (got.float().sum(), lse[0].sum(), cache.attend(leaf, table, who, positions)[0, 0, 0]):
            with pytest.raises(RuntimeError, match="kv_attend. has no gradient"):
                loss.backward()
        assert leaf.grad is None
        with pytest.raises(ValueError, match="wants a gradient"):
            cache.attend(leaf, table, who, positions, out=torch.empty_like(want))
        with torch.no_grad():
            out = torch.empty_like(want)
            assert cache.attend(leaf, table, who, positions, out=out) is out
            assert not out.requires_grad and torch.equal(out, want)
        assert not cache.select(leaf, table, who, positions, 2).requires_grad
    cache.append(wide[:, :2, :64].float().bfloat16().requires_grad_(), wide[:, :2, :64], who.long())
    assert not cache.keys.requires_grad


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("heads,group,page,dim", [(8, 4, 64, 64), (16, 5, 16, 40), (8, 16, 32, 128),
                                                  (16, 1, 256, 24)])
def test_prompts_among_single_tokens(engine, heads, group, page, dim, listed):
    """Tokens of a few prompts and of many requests with one, in a table with idle
    rows: the prompts start and end within spans of tokens that share a workgroup."""
    rng = np.random.default_rng(heads * group + page)
    requests, cols = 300, -(-4096 // page)
    cache = make_cache(engine, 80, heads, page, dim, "bf16", rng)
    table = rng.integers(0, 80, (requests, cols)).astype(np.int32)
    new = np.ones(requests, int)
    new[150:] = 0
    new[[7, 60, 149]] = 121, 203, 70
    held = rng.integers(1, 330, requests)
    held[[7, 60, 149]] += 200
    who = np.repeat(np.arange(requests), new)
    positions = np.concatenate([np.arange(h - n, h) for h, n in zip(held, new)])
    who, positions = np.r_[who, -1, -1, 5], np.r_[positions, -1, -1, 9]
    tokens = len(who)
    q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).bfloat16()
    blocks = rng.integers(-1, 330 // page + 2, (tokens, heads, 4)) if listed else None
    check_attend(cache, "bf16", q, table, who, positions, blocks=blocks)


@pytest.mark.parametrize("rows", [256, 512])
def test_a_prompt_in_a_table_with_idle_rows(engine, rows):
    """Takes not much longer than alone, its tokens sharing wavefronts there too."""
    rng = np.random.default_rng(5)
    cache = make_cache(engine, 64, 8, 64, 128, "bf16", rng)
    tokens = 512
    q = dev(rng.standard_normal((tokens, 32, 128), np.float32)).bfloat16()
    table = dev(rng.permutation(64)[None], torch.int32)
    tall = torch.full((rows, 64), -1, dtype=torch.int32, device="cuda")
    tall[rows // 2] = table
    who = torch.zeros(tokens, dtype=torch.int32, device="cuda")
    positions = dev(np.arange(tokens) + 4096 - tokens, torch.int32)
    alone = cache.attend(q, table, who, positions)
    assert torch.equal(cache.attend(q, tall, who + rows // 2, positions), alone)
    there = who + rows // 2
    # (measured: 162 and 100 us; every token by itself 874)
    assert best_time(lambda: cache.attend(q, tall, there, positions)) \
        < 3 * best_time(lambda: cache.attend(q, table, who, positions))
