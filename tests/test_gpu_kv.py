"""The paged key-value cache on the GPU against its restatement in NumPy
(kv_oracle.py): whole numbers (plans, codes, selected blocks) equal, attention
within bounds that follow from its roundings.

An attention output sums terms p_j v_j / sum p.  With u the unit roundoff of
the cache's type (2^-8 for bfloat16, 2^-11 for float16), each p is rounded to
that type once and the output once; a float32 score is off by at most (d + 2)
2^-24 of scale sum |q_i k_i| (`reach`), which enters p and the sum of p; sums of
n terms in float32 are off by n 2^-24 and the exponential by 2^-20.  So
|out - exact| <= u |out| + (u + 2 (d + 2) 2^-24 reach + 2 n 2^-24 + 2^-20)
attention of |v|, and the logarithm of the sum by (d + 2) 2^-24 reach + n 2^-24
+ 2^-20 + 2^-22 |lse|.
"""

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import kv_oracle  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def dev(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), device="cuda", dtype=dtype)


def f32(x):
    return x.float().cpu().numpy()


# ---- kv_plan -----------------------------------------------------------------


def check_plan(engine, past, fresh, cols, free, cursor, page, tokens, seed=0, spare=0, out=None):
    past, fresh = np.asarray(past, np.int32), np.asarray(fresh, np.int32)
    rng = np.random.default_rng(seed)
    table = rng.integers(1000, 9000, (len(past), cols + spare)).astype(np.int32)
    wide = dev(table)
    view = wide[:, :cols]
    free = np.asarray(free, np.int32)
    got = engine.kv_plan(dev(past), dev(fresh), view, dev(free), dev([cursor], torch.int32), page,
                         tokens, out=out)
    want = kv_oracle.plan(past, fresh, table[:, :cols], free, cursor, page, tokens)
    for name, a in want.items():
        b = (view if name == "table" else getattr(got, name)).cpu().numpy()
        assert np.array_equal(a, b), name
    assert np.array_equal(wide[:, cols:].cpu().numpy(), table[:, cols:])
    return got


@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("requests", [1, 2, 63, 64, 65, 1023, 1024, 1025, 5000])
def test_plan_of_many_requests(engine, requests, page):
    rng = np.random.default_rng(requests + page)
    past = rng.integers(0, 6 * page, requests)
    fresh = rng.choice([0, 1, 1, 1, page, 2 * page + 3], requests)
    free = rng.permutation(4 * requests + 9)
    check_plan(engine, past, fresh, 10, free, 5, page, int(fresh.sum()) + 13, spare=3)


@pytest.mark.parametrize("tokens", [0, 1, 5, 64, 300])
def test_plan_of_fewer_or_more_places_than_tokens(engine, tokens):
    check_plan(engine, [0, 15, 16, 17, 0], [1, 1, 1, 30, 0], 4, np.arange(100, 140), 0, 16, tokens)


def test_plan_at_page_edges(engine):
    past = [0, 0, 0, 15, 15, 16, 16, 31, 32, 63]
    fresh = [0, 16, 17, 1, 2, 0, 1, 1, 16, 1]
    check_plan(engine, past, fresh, 4, np.arange(50), 0, 16, 64)


def test_plan_that_the_free_list_cannot_serve(engine):
    # the second request takes the last two pages; the third needs none, the
    # fourth finds the list empty, and the last needs none
    check_plan(engine, [0, 0, 3, 16, 20], [16, 32, 4, 1, 5], 4, [7, 8, 9], 0, 16, 80)
    # a large request closes the list for the small one behind it
    check_plan(engine, [0, 0, 0], [16, 64, 16], 8, [7, 8, 9], 0, 16, 100)
    # nothing left, a cursor past the list, one before it
    for cursor in (3, 9, -1):
        check_plan(engine, [0, 5], [16, 4], 4, [7, 8, 9], cursor, 16, 20)


def test_plan_with_lengths_that_cannot_be(engine):
    # negative lengths and rows that are too narrow are not admitted, and take
    # nothing from the others
    check_plan(engine, [-1, 5, 60, 64, 0], [3, -2, 5, 0, 64], 4, np.arange(30), 0, 16, 90)
    big = np.iinfo(np.int32).max
    check_plan(engine, [big, 3], [1, 4], 4, np.arange(30), 0, 16, 8)
    check_plan(engine, [0, 0], [0, 0], 0, [], 0, 16, 4)


def test_plan_without_requests(engine):
    p = check_plan(engine, [], [], 3, [1, 2], 1, 16, 5)
    assert p.starts.tolist() == [0] and p.cursor.tolist() == [1]


def test_plan_into_an_earlier_one_and_steps_in_a_row(engine):
    page, cols = 16, 12
    rng = np.random.default_rng(3)
    past, table = np.zeros(7, np.int32), np.full((7, cols), -1, np.int32)
    free = rng.permutation(100).astype(np.int32)
    cursor, cur = 0, dev([0], torch.int32)
    t, p, out = dev(table), dev(past), None
    for step in range(9):
        fresh = rng.integers(0, 20, 7).astype(np.int32)
        want = kv_oracle.plan(past, fresh, table, free, cursor, page, 160)
        got = engine.kv_plan(p, dev(fresh), t, dev(free), cur, page, 160,
                             out=out if step % 2 else None)
        for name in ("slots", "requests", "positions", "starts", "lengths", "first", "cursor"):
            assert np.array_equal(want[name], getattr(got, name).cpu().numpy()), (step, name)
        assert np.array_equal(want["table"], t.cpu().numpy())
        out = got if step % 2 == 0 else None  # (its cursor is the next call's)
        out = out and out._replace(cursor=torch.empty_like(out.cursor))
        past, table, cursor, cur = want["lengths"], want["table"], int(want["cursor"][0]), got.cursor
        p = got.lengths.clone()


# ---- append -------------------------------------------------------------------


def make_cache(engine, pages, heads, page, dim, dtype, rng, fill="normal"):
    c = engine.PagedKVCache.empty(pages, heads, page, dim, dtype=DTYPES[dtype])
    if fill == "normal":
        c.keys.copy_(dev(rng.standard_normal(c.keys.shape, np.float32)))
        c.values.copy_(dev(rng.standard_normal(c.values.shape, np.float32)))
    else:  # what an allocator may leave behind
        c.keys.fill_(fill)
        c.values.fill_(fill)
    c.summaries.fill_(77)
    c.scales.fill_(-5.0)
    return c


def check_append(cache, k, v, slots):
    keys, values = cache.keys.clone(), cache.values.clone()
    codes, scales = cache.summaries.cpu().numpy().copy(), cache.scales.cpu().numpy().copy()
    page = cache.page_size
    cache.append(k, v, dev(np.asarray(slots, np.int64)))
    done = []
    for t, s in enumerate(slots):
        if 0 <= s < len(keys) * page:
            keys[s // page, :, s % page] = k[t]
            values[s // page, :, :, s % page] = v[t]
            if s % page == page - 1:
                done.append(s // page)
    for p in done:
        for h in range(cache.kv_heads):
            codes[p, h], scales[p, h] = kv_oracle.summary(f32(keys[p, h]))
    bits = torch.int16
    assert torch.equal(cache.keys.view(bits), keys.view(bits))
    assert torch.equal(cache.values.view(bits), values.view(bits))
    assert np.array_equal(cache.summaries.cpu().numpy(), codes)
    got = cache.scales.cpu().numpy()
    same = np.isfinite(scales)
    assert np.array_equal(got[~same], scales[~same])
    # two roundings of float32 quotients and products
    assert (np.abs(got[same] - scales[same]) <= 3 * 2.0 ** -24 * np.abs(scales[same])).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,page,dim", [(1, 16, 8), (3, 16, 80), (2, 32, 64), (8, 64, 128),
                                            (5, 128, 72), (2, 256, 256), (1, 64, 248), (4, 16, 96)])
def test_append(engine, heads, page, dim, dtype):
    rng = np.random.default_rng(heads * page + dim)
    cache = make_cache(engine, 9, heads, page, dim, dtype, rng)
    # prompts that start in the middle of a page, single tokens, skipped places
    slots = []
    for first, count in ((2 * page + 5, 2 * page), (6 * page, page), (5 * page - 1, 1)):
        slots += range(first, first + count)
    slots += [-1, 9 * page, 9 * page + 3, 8 * page + 1, -7]
    n = len(slots)
    fused = dev(rng.standard_normal((n, (3 * heads + 1) * dim), np.float32)).to(DTYPES[dtype])
    k = fused[:, heads * dim:2 * heads * dim].view(n, heads, dim)
    v = fused[:, 2 * heads * dim:3 * heads * dim].view(n, heads, dim)
    check_append(cache, k, v, slots)


@pytest.mark.parametrize("tokens", [1, 15, 16, 17, 256, 257, 1024, 1025, 1500])
def test_append_in_any_order(engine, tokens):
    # slots in no order: a page's last slot may come before its others
    rng = np.random.default_rng(tokens)
    cache = make_cache(engine, 130, 2, 16, 64, "bf16", rng)
    slots = rng.permutation(130 * 16)[:tokens].tolist()
    slots[0] = 130 * 16 - 1 if 130 * 16 - 1 not in slots else slots[0]
    k, v = (dev(rng.standard_normal((tokens, 2, 64), np.float32)).bfloat16() for _ in range(2))
    check_append(cache, k, v, slots)


def test_append_none(engine):
    cache = engine.PagedKVCache.empty(2, 2, 16, 64)
    e = torch.empty((0, 2, 64), dtype=torch.bfloat16, device="cuda")
    cache.append(e, e, torch.empty(0, dtype=torch.int64, device="cuda"))
    assert not cache.keys.any() and not cache.summaries.any()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_summaries_of_unusual_pages(engine, dtype):
    rng = np.random.default_rng(5)
    page, dim = 32, 64
    cache = make_cache(engine, 8, 1, page, dim, dtype, rng)
    k = rng.standard_normal((8, page, dim)).astype(np.float32)
    k[0] = 0.0                                   # nothing
    k[1, 3, 7] = np.nan                          # broken
    k[2, 31, 63] = -np.inf
    k[3] = np.where(np.arange(page)[:, None] % 2, 1.0, -1.0)  # sums to nothing
    k[4] *= 2.0 ** -20 if dtype == "f16" else 1e-36  # tiny
    k[5] = 0.0
    k[5, 0, 0] = 6e4 if dtype == "f16" else 3e38
    k[6] = 0.25
    kt = dev(k.reshape(-1, 1, dim)).to(DTYPES[dtype])
    check_append(cache, kt, kt, list(range(8 * page)))
    assert cache.scales[1:3].isinf().all() and not cache.summaries[1:3].any()
    assert not cache.summaries[0].any() and (cache.summaries[6] == 127).all()


def test_append_to_a_cache_without_summaries(engine):
    cache = engine.PagedKVCache.empty(2, 1, 16, 8, summaries=False)
    k = torch.ones((32, 1, 8), dtype=torch.bfloat16, device="cuda")
    cache.append(k, 2 * k, torch.arange(32, device="cuda"))
    assert (cache.keys == 1).all() and (cache.values == 2).all()


def test_append_of_rows_that_are_not_aligned(engine):
    # (the rows are copied first)
    rng = np.random.default_rng(8)
    cache = make_cache(engine, 3, 2, 16, 64, "f16", rng)
    flat = dev(rng.standard_normal(20 * 131 + 1, np.float32)).half()
    k = flat[1:].view(20, 131)[:, 3:131].unflatten(1, (2, 64))
    v = flat[:-1].view(20, 131)[:, :128].unflatten(1, (2, 64)).flip(0)
    check_append(cache, k, v, list(range(10, 30)))


# ---- select -------------------------------------------------------------------


def check_select(engine, q, codes, scales, table, requests, positions, page, n, first=1, last=1):
    pages, heads, d = codes.shape
    shape = (pages, heads, page, d)
    cache = engine.PagedKVCache(torch.empty(shape, dtype=q.dtype, device="cuda"),
                                torch.empty((pages, heads, d, page), dtype=q.dtype, device="cuda"),
                                dev(codes), dev(scales))
    got = cache.select(q, dev(table), dev(requests, torch.int32), dev(positions, torch.int32), n,
                       first=first, last=last).cpu().numpy()
    want = kv_oracle.select(f32(q), codes, scales, table, requests, positions, page, n, first, last)
    assert np.array_equal(got, want)


def summaries(rng, pages, heads, d, spread=3):
    return (rng.integers(-127, 128, (pages, heads, d)).astype(np.int8),
            (2.0 ** rng.uniform(-spread, spread, (pages, heads))).astype(np.float32))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,group,d", [(1, 1, 8), (2, 3, 72), (3, 5, 80), (8, 4, 128),
                                           (2, 20, 64), (1, 2, 256), (1, 7, 248), (4, 16, 16)])
def test_select(engine, heads, group, d, dtype):
    rng = np.random.default_rng(heads * group * d)
    page, cols, requests = 16, 37, 3
    codes, scales = summaries(rng, 150, heads, d)
    table = rng.permutation(150)[:requests * cols].reshape(requests, cols).astype(np.int32)
    # from none to all columns, in any order, with places that hold no token
    positions = np.array([0, 15, 16, 17 * 16 - 1, 592 - 1, 300, -1, 40, 100, 592 - 16, 583])
    who = np.array([0, 1, 2, 0, 1, 2, 0, 1, -1, 1, 3])
    fused = rng.standard_normal((len(who), (heads * group + 1) * d)).astype(np.float32)
    q = dev(fused).to(DTYPES[dtype])[:, d:].view(len(who), heads * group, d)
    for n, first, last in ((1, 0, 1), (4, 1, 1), (16, 2, 3), (36, 1, 1), (37, 1, 1), (64, 5, 8)):
        check_select(engine, q, codes, scales, table, who, positions, page, n, first, last)


@pytest.mark.parametrize("tokens", [1, 16, 40, 130])
def test_select_for_the_tokens_of_prompts(engine, tokens):
    # tokens of one request next to one another, requests of odd counts
    rng = np.random.default_rng(tokens)
    page, heads, d = 32, 2, 128
    codes, scales = summaries(rng, 200, heads, d)
    table = rng.integers(0, 200, (3, 60)).astype(np.int32)
    who = np.sort(rng.integers(0, 3, tokens))
    positions = np.array([1900 - tokens + i - 500 * w for i, w in enumerate(who)])
    q = dev(rng.standard_normal((tokens, heads * 4, d), np.float32)).bfloat16()
    for n in (3, 16, 50):
        check_select(engine, q, codes, scales, table, who, positions, page, n)


@pytest.mark.parametrize("cols,heads,group,d", [(255, 2, 3, 80), (300, 1, 16, 16), (512, 2, 2, 256),
                                                (513, 1, 5, 64), (896, 2, 1, 128), (897, 1, 2, 48),
                                                (300, 1, 2, 72)])
def test_select_for_prompts_among_many_blocks(engine, cols, heads, group, d):
    rng = np.random.default_rng(cols)
    codes, scales = summaries(rng, 950, heads, d)
    scales[5], scales[9] = np.inf, 0.0
    codes[100:200] = codes[100]  # ties
    scales[100:200] = scales[100]
    table = rng.integers(-3, 960, (2, cols)).astype(np.int32)
    tokens = 45
    who = np.repeat([0, 1, 0, 7], [17, 20, 7, 1])
    positions = rng.integers(0, cols * 16, tokens)
    positions[:20] = cols * 16 - 1 - np.arange(20)
    positions[30] = -1
    q = dev(rng.standard_normal((tokens, heads * group, d), np.float32)).half()
    q[3, 0, 1], q[4] = float("inf"), 0.0
    for n in (2, 33, 256):
        check_select(engine, q, codes, scales, table, who, positions, 16, n)


@pytest.mark.parametrize("heads,tokens", [(64, 19), (24, 11)])
@pytest.mark.parametrize("cols,d", [(256, 16), (512, 80), (600, 256), (897, 128), (2048, 64),
                                    (2049, 16)])
def test_select_of_many_rows(engine, cols, d, heads, tokens):
    rng = np.random.default_rng(cols + heads)
    codes, scales = summaries(rng, 300, heads, d)
    scales[7, ::2] = np.inf
    codes[100:140] = codes[100]  # ties
    scales[100:140] = scales[100]
    table = rng.integers(-3, 310, (2, cols)).astype(np.int32)
    who = np.sort(rng.integers(0, 2, tokens))
    who[-2] = 9
    positions = rng.integers(0, 60 * 16, tokens)
    positions[[0, 4]] = cols * 16 - 1, cols * 16 - 17
    positions[7] = -1
    q = dev(rng.standard_normal((tokens, heads * 2, d), np.float32)).bfloat16()
    for n in (2, 48):
        check_select(engine, q, codes, scales, table, who, positions, 16, n)


@pytest.mark.parametrize("cols", [2048, 2049, 4096, 8192, 8193, 9000])
def test_select_among_many_blocks(engine, cols):
    rng = np.random.default_rng(cols)
    codes, scales = summaries(rng, 700, 1, 16)
    table = rng.integers(0, 700, (2, cols)).astype(np.int32)
    q = dev(rng.standard_normal((3, 2, 16), np.float32)).half()
    positions = np.array([cols * 16 - 1, 5000, (cols - 1) * 16])
    for n in (2, 256):
        check_select(engine, q, codes, scales, table, np.array([0, 0, 1]), positions, 16, n)


@pytest.mark.parametrize("heads,group,d", [(9, 2, 80), (3, 3, 72), (8, 1, 256), (1, 2, 128)])
def test_select_among_many_blocks_of_several_heads(engine, heads, group, d):
    rng = np.random.default_rng(heads)
    codes, scales = summaries(rng, 90, heads, d)
    table = rng.integers(-1, 95, (2, 2100)).astype(np.int32)
    q = dev(rng.standard_normal((3, heads * group, d), np.float32)).bfloat16()
    check_select(engine, q, codes, scales, table, np.array([1, 0, 1]),
                 np.array([2100 * 16 - 1, 16 * 16, 2050 * 16]), 16, 11)


@pytest.mark.parametrize("kind", ["a lane's", "equal", "few values", "neighbours", "few pages",
                                  "a stretch"])
def test_select_of_many_rows_wherever_the_best_lie(engine, kind):
    """Tiles of tokens over 512 columns, a lane of a wavefront holding every 64th."""
    rng = np.random.default_rng(12)
    heads, d, cols, tokens = 64, 16, 512, 17
    codes, scales = summaries(rng, cols, heads, d, spread=0.01)
    table = np.arange(cols, dtype=np.int32)[None].copy()
    if kind == "a lane's":         # 8 of 512 by far, then whatever comes
        codes[5::64], scales[5::64] = 100, 1e6
    elif kind == "equal":
        codes[:], scales[:] = 1, 1.0
    elif kind == "few values":     # more equal ones than a wavefront has lanes
        codes[:], scales[:] = rng.integers(0, 3, (cols, heads, 1)), 1.0
    elif kind == "neighbours":     # scores that differ in their last bits
        codes[:] = 127
        scales[:] = np.float32(1) + np.float32(2.0 ** -23) * rng.permutation(cols)[:, None]
    elif kind == "few pages":
        table[0, rng.permutation(cols)[:480]] = -1
    else:                          # the best 100 side by side
        codes[200:300], scales[200:300] = 120, 50.0
    positions = cols * 16 - 1 - rng.integers(0, 700, tokens) * (np.arange(tokens) % 3)
    q = dev(np.abs(rng.standard_normal((tokens, heads, d), np.float32))).bfloat16()
    for n in (2, 16, 32, 33):
        check_select(engine, q, codes, scales, table, np.zeros(tokens, int), positions, 16, n)


def test_select_ties_go_to_the_lowest_block(engine):
    rng = np.random.default_rng(1)
    for kind in range(4):
        codes = rng.integers(-2, 3, (40, 2, 32)).astype(np.int8)
        scales = np.ones((40, 2), np.float32)
        if kind == 1:
            codes[:] = 1                    # all equal
        if kind == 2:
            scales[::2] = 0.0               # zeros of either sign
        if kind == 3:
            codes[:], scales[:] = 0, 0.0
        table = np.arange(40, dtype=np.int32)[None].repeat(2, 0)
        q = dev(rng.standard_normal((4, 4, 32), np.float32)).bfloat16()
        for n in (2, 7, 39):
            check_select(engine, q, codes, scales, table, np.array([0, 1, 0, 1]),
                         np.array([639, 630, 400, 100]), 16, n)


def test_select_with_absent_pages_and_broken_summaries(engine):
    rng = np.random.default_rng(2)
    codes, scales = summaries(rng, 50, 2, 64)
    table = rng.permutation(60).astype(np.int32)[None].repeat(2, 0)  # 50 to 59: none
    table[1, ::3] = -1
    table[1, 30] = np.iinfo(np.int32).max
    scales[7], scales[11, 1], scales[13, 0] = np.inf, np.nan, np.inf
    scales[20], scales[21] = 3e38, 1e-45
    q = dev(rng.standard_normal((6, 4, 64), np.float32)).bfloat16()
    q[4, 1, 3] = float("nan")
    q[5] = 0.0
    positions = np.array([959, 959, 500, 500, 959, 959])
    for n in (3, 12, 45, 60):
        check_select(engine, q, codes, scales, table, np.array([0, 1, 0, 1, 0, 1]), positions, 16, n)


def test_select_of_no_tokens_or_columns(engine):
    rng = np.random.default_rng(2)
    codes, scales = summaries(rng, 5, 1, 8)
    q = torch.zeros((0, 1, 8), dtype=torch.float16, device="cuda")
    none = np.zeros(0, np.int32)
    check_select(engine, q, codes, scales, np.zeros((1, 3), np.int32), none, none, 16, 4)
    q = torch.zeros((2, 1, 8), dtype=torch.float16, device="cuda")
    check_select(engine, q, codes, scales, np.zeros((1, 0), np.int32), np.zeros(2, np.int32),
                 np.array([0, 40]), 16, 4)


# ---- attend -------------------------------------------------------------------


def check_attend(cache, dtype, q, table, requests, positions, blocks=None, scale=None, longest=0):
    d = q.shape[2]
    got, lse = cache.attend(q, dev(table), dev(requests, torch.int32), dev(positions, torch.int32),
                            blocks=None if blocks is None else dev(blocks, torch.int32),
                            scale=scale, longest=longest, lse=True)
    scale = d ** -0.5 if scale is None else scale
    want, sums, weight, reach, n = kv_oracle.attend(
        f32(q), f32(cache.keys), f32(cache.values), table, requests, positions,
        float(np.float32(scale)), blocks)
    u = UNIT[dtype]
    off = (d + 2) * 2.0 ** -24 * reach
    bound = u * np.abs(want) + (u + 2 * off + 2 * n * 2.0 ** -24 + 2.0 ** -20) * weight
    if dtype == "f16":
        bound += 2.0 ** -24  # (its smallest numbers)
    far = np.abs(got.double().cpu().numpy() - want)
    assert (far <= bound).all(), (far / np.maximum(bound, 1e-300)).max()
    lse = lse.double().cpu().numpy()
    none = np.isneginf(sums)
    assert np.array_equal(none, np.isneginf(lse))
    limit = (off + n * 2.0 ** -24 + 2.0 ** -20)[..., 0] + 2.0 ** -22 * np.where(none, 0, np.abs(sums))
    assert (np.abs(lse[~none] - sums[~none]) <= limit[~none]).all()
    assert not got.cpu()[torch.as_tensor(none)].any()
    return got


def tables(rng, pages, requests, cols):
    return rng.permutation(pages)[:requests * cols].reshape(requests, cols).astype(np.int32)


SHAPES = [(1, 1, 16, 8), (2, 3, 16, 80), (8, 4, 64, 128), (2, 5, 32, 96), (1, 20, 16, 64),
          (1, 33, 64, 72), (3, 8, 128, 128), (2, 16, 256, 192), (1, 2, 32, 256), (2, 1, 64, 248)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,group,page,dim", SHAPES)
def test_attend_over_everything(engine, heads, group, page, dim, dtype):
    rng = np.random.default_rng(heads * group * page + dim)
    cols = max(3, 700 // page)
    cache = make_cache(engine, 4 * cols + 1, heads, page, dim, dtype, rng)
    table = tables(rng, 4 * cols + 1, 4, cols)
    # one key, the edges of pages and tiles, everything, idle places
    positions = np.array([0, 1, page - 1, page, 31, 63, 64, cols * page - 1, -1, 2 * page + 5, 9])
    who = np.array([0, 1, 2, 3, 0, 1, 2, 3, 0, -1, 4])
    q = dev(rng.standard_normal((len(who), (heads * group + 1) * dim), np.float32))
    q = q.to(DTYPES[dtype])[:, dim:].view(len(who), heads * group, dim)
    for longest in (0, 1, cols * page):
        check_attend(cache, dtype, q, table, who, positions, longest=longest)
    check_attend(cache, dtype, q[7:8], table, who[7:8], positions[7:8], scale=0.3)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,group,page,dim", SHAPES)
def test_attend_over_listed_blocks(engine, heads, group, page, dim, dtype):
    rng = np.random.default_rng(heads + group * page + dim)
    cols = max(6, 900 // page)
    cache = make_cache(engine, 2 * cols, heads, page, dim, dtype, rng)
    table = tables(rng, 2 * cols, 2, cols)
    tokens = 9
    who = rng.integers(0, 2, tokens)
    positions = rng.integers(0, cols * page, tokens)
    positions[:4] = 0, page, cols * page - 1, -1
    q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).to(DTYPES[dtype])
    for n in (1, 2, 5, 17, 70):
        # ascending lists with the token's own block, as select gives them, and
        # lists in any order with gaps, repeats, later blocks and none at all
        blocks = rng.integers(-2, cols + 2, (tokens, heads, n))
        for t in range(0, tokens, 2):
            for h in range(heads):
                b = np.unique(rng.integers(0, max(1, positions[t] // page + 1), n))
                blocks[t, h] = np.pad(b, (0, n - len(b)), constant_values=-1)
        blocks[-1] = -1
        check_attend(cache, dtype, q, table, who, positions, blocks=blocks)


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attend_of_many_rows(engine, dtype, listed):
    # more rows than are split: a prompt's tokens, heads of more than one tile
    rng = np.random.default_rng(17)
    for heads, group, page, dim, tokens in ((4, 18, 16, 64, 515), (16, 2, 32, 40, 259),
                                            (8, 1, 64, 200, 513)):
        cols = 160 // page + 1
        cache = make_cache(engine, 2 * cols, heads, page, dim, dtype, rng)
        table = tables(rng, 2 * cols, 2, cols)
        who = (np.arange(tokens) > 300).astype(int)
        positions = rng.integers(-1, cols * page, tokens)
        q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).to(DTYPES[dtype])
        blocks = rng.integers(-1, cols, (tokens, heads, 3)) if listed else None
        check_attend(cache, dtype, q, table, who, positions, blocks=blocks)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens", [3, 16, 40])
def test_attend_of_short_prompts(engine, tokens, dtype):
    # few to many tokens for each of the requests, in either kernel
    rng = np.random.default_rng(tokens)
    heads, group, page, dim, requests = 8, 4, 32, 64, 4
    cols = 20
    cache = make_cache(engine, requests * cols, heads, page, dim, dtype, rng)
    table = tables(rng, requests * cols, requests, cols)
    who = np.repeat(np.arange(requests), tokens)
    positions = np.tile(np.arange(tokens), requests) + np.repeat([0, 33, 300, 640 - tokens], tokens)
    q = dev(rng.standard_normal((len(who), heads * group, dim), np.float32)).to(DTYPES[dtype])
    check_attend(cache, dtype, q, table, who, positions)
    blocks = cache.select(q, dev(table), dev(who, torch.int32), dev(positions, torch.int32), 6)
    check_attend(cache, dtype, q, table, who, positions, blocks=blocks.cpu().numpy())


SHARED = [(128, 2, 16, 64, 70), (64, 5, 32, 80, 60), (64, 16, 64, 128, 24), (40, 20, 128, 96, 33),
          (64, 8, 256, 256, 40), (64, 4, 64, 192, 50), (128, 1, 16, 248, 66), (64, 8, 64, 40, 50),
          (96, 3, 32, 128, 60), (64, 7, 16, 128, 40), (32, 33, 16, 96, 25)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,group,page,dim,tokens", SHARED)
def test_attend_of_tokens_that_share_wavefronts(engine, heads, group, page, dim, tokens, dtype):
    # neighbouring tokens of one request, of others, idle ones; everything, lists
    # as select gives them, lists in any order with gaps and repeats
    rng = np.random.default_rng(heads + dim)
    cols = max(3, 200 // page)
    cache = make_cache(engine, 2 * cols + 2, heads, page, dim, dtype, rng)
    table = tables(rng, 2 * cols + 2, 2, cols)
    table[1, 1] = -1  # an absent page
    who = np.repeat([0, 1, 0, 5, 1], [tokens - 15, 5, 4, 1, 5])
    positions = np.minimum(cols * page - 1, np.arange(tokens) * 3 + 7)
    positions[[2, tokens - 3]] = -1
    positions[-1] = 0
    q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).to(DTYPES[dtype])
    check_attend(cache, dtype, q, table, who, positions)
    n = 5
    blocks = np.full((tokens, heads, n), -1)
    for t in range(tokens):
        for h in range(heads):
            b = np.unique(rng.integers(0, max(1, positions[t] // page + 1), n))
            blocks[t, h, :len(b)] = b
    check_attend(cache, dtype, q, table, who, positions, blocks=blocks)
    blocks = rng.integers(-2, cols + 2, (tokens, heads, 9))
    check_attend(cache, dtype, q, table, who, positions, blocks=blocks)


@pytest.mark.parametrize("n", [70, 256])
def test_attend_over_long_lists_of_many_tokens(engine, n):
    rng = np.random.default_rng(n)
    heads, group, page, dim, cols, tokens = 96, 8, 16, 16, 2300, 24
    cache = make_cache(engine, 300, heads, page, dim, "bf16", rng)
    table = rng.integers(0, 300, (2, cols)).astype(np.int32)
    who, positions = np.zeros(tokens, int), rng.integers(30_000, cols * page, tokens)
    q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).bfloat16()
    blocks = np.sort(rng.integers(0, cols, (tokens, heads, n)), 2)
    blocks[::3] = rng.permuted(blocks[::3], axis=2)
    check_attend(cache, "bf16", q, table, who, positions, blocks=blocks)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens", [2, 40])
def test_a_block_that_is_listed_256_times(engine, tokens, dtype):
    rng = np.random.default_rng(tokens)
    heads, group, page, dim, cols = 64, 8, 16, 32, 5
    cache = make_cache(engine, cols, heads, page, dim, dtype, rng)
    table = np.arange(cols, dtype=np.int32)[None]
    q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).to(DTYPES[dtype])
    blocks = np.full((tokens, heads, 256), 3)
    blocks[::2, :, 100:] = rng.integers(0, cols, (1, 1, 156))
    check_attend(cache, dtype, q, table, np.zeros(tokens, int), np.full(tokens, 70), blocks=blocks)


@pytest.mark.parametrize("listed", [False, True])
@pytest.mark.parametrize("page", [16, 64])
def test_what_only_later_tokens_see_does_not_reach_earlier_ones(engine, page, listed):
    rng = np.random.default_rng(page)
    heads, group, dim, cols, tokens = 64, 8, 64, 8, 40
    cache = make_cache(engine, cols, heads, page, dim, "bf16", rng)
    clean = make_cache(engine, cols, heads, page, dim, "bf16", rng)
    clean.keys.copy_(cache.keys)
    clean.values.copy_(cache.values)
    table = np.arange(cols, dtype=np.int32)[None].repeat(2, 0)
    who, positions = np.zeros(tokens, int), np.arange(tokens) + 2 * page
    bad = 2 * page + 17  # (a key that tokens from the 17th on see)
    cache.values[bad // page, :, 5, bad % page] = float("nan")
    cache.values[bad // page, :, 9, bad % page] = float("inf")
    cache.keys[7] = float("nan")
    cache.values[7] = float("nan")
    q = dev(rng.standard_normal((tokens, heads * group, dim), np.float32)).bfloat16()
    blocks = np.tile(np.array([0, 1, 2, 3, 4, 5, 7], np.int32), (tokens, heads, 1)) if listed else None
    want = check_attend(clean, "bf16", q, table, who, positions, blocks=blocks)
    got = cache.attend(q, dev(table), dev(who, torch.int32), dev(positions, torch.int32),
                       blocks=None if blocks is None else dev(blocks))
    assert torch.equal(got[:17], want[:17])
    others = [i for i in range(dim) if i not in (5, 9)]
    assert torch.equal(got[17:][..., others], want[17:][..., others])
    assert got[17:, :, 5].isnan().all() and got[17:, :, 9].isinf().all()


@pytest.mark.parametrize("tokens", [1, 3, 17])
def test_attend_over_a_long_cache(engine, tokens):
    # many parts that are joined; a request much shorter than the longest
    rng = np.random.default_rng(tokens)
    page, heads, group, dim = 64, 2, 4, 64
    cols = 20_011 // page + 1
    cache = make_cache(engine, cols, heads, page, dim, "bf16", rng)
    table = np.stack([rng.permutation(cols), rng.permutation(cols)]).astype(np.int32)
    who = np.arange(tokens) % 2
    positions = np.where(who, 70, 20_010 - np.arange(tokens))
    q = dev(2.0 * rng.standard_normal((tokens, heads * group, dim), np.float32)).bfloat16()
    for longest in (0, 20_011):
        check_attend(cache, "bf16", q, table, who, positions, longest=longest)


@pytest.mark.parametrize("garbage", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("page", [16, 64])
def test_what_masked_places_hold_does_not_count(engine, garbage, page):
    rng = np.random.default_rng(3)
    heads, dim, cols = 2, 128, 6
    for length in (1, 7, page - 1, page, page + 1, 3 * page + 9):
        cache = make_cache(engine, 2 * cols, heads, page, dim, "bf16", rng, fill=garbage)
        table = tables(rng, 2 * cols, 1, cols)
        slots = np.array([table[0, i // page] * page + i % page for i in range(length)])
        k, v = (dev(rng.standard_normal((length, heads, dim), np.float32)).bfloat16()
                for _ in range(2))
        cache.append(k, v, dev(slots, torch.int64))
        q = dev(rng.standard_normal((3, heads * 4, dim), np.float32)).bfloat16()
        clean = make_cache(engine, 2 * cols, heads, page, dim, "bf16", rng, fill=0.0)
        clean.append(k, v, dev(slots, torch.int64))
        who, positions = np.zeros(3, np.int32), np.array([length - 1, 0, -1])
        blocks = np.tile(np.array([3, 0, 5, -1, 1, 2], np.int32), (3, heads, 1))
        for b in (None, blocks):
            want = check_attend(clean, "bf16", q, table, who, positions, blocks=b)
            got = cache.attend(q, dev(table), dev(who, torch.int32), dev(positions, torch.int32),
                               blocks=None if b is None else dev(b))
            assert torch.equal(got, want)


def test_attend_with_absent_pages(engine):
    rng = np.random.default_rng(4)
    for page in (16, 32):
        cache = make_cache(engine, 40, 2, page, 64, "f16", rng)
        table = rng.permutation(60)[:40].astype(np.int32)[None]
        table[0, 5:9] = -1, 40, np.iinfo(np.int32).max, np.iinfo(np.int32).min
        q = dev(rng.standard_normal((4, 4, 64), np.float32)).half()
        who = np.zeros(4, np.int32)
        positions = np.array([40 * page - 1, 9 * page - 2, 6 * page, 100 * page])
        check_attend(cache, "f16", q, table, who, positions)
        blocks = rng.integers(-1, 41, (4, 2, 30))
        check_attend(cache, "f16", q, table, who, positions, blocks=blocks)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_attend_with_scores_far_apart(engine, dtype):
    # one key far above the rest, all far below zero, all equal, and a long tail
    # of small terms that only together count
    rng = np.random.default_rng(6)
    page, dim, cols = 64, 64, 40
    cache = make_cache(engine, cols, 1, page, dim, dtype, rng)
    q = torch.zeros((4, 1, dim), dtype=DTYPES[dtype], device="cuda")
    q[:, 0, 0] = dev([1.0, 1.0, 0.0, 1.0])
    table = np.arange(cols, dtype=np.int32)[None]
    who, positions = np.zeros(4, np.int32), np.full(4, cols * page - 1)
    for fill, one in ((0.0, 100.0), (-200.0, -200.0), (0.0, 0.0), (0.0, 12.0)):
        cache.keys[..., 0] = fill
        cache.keys[17, 0, 33, 0] = one
        check_attend(cache, dtype, q, table, who, positions, scale=1.0)


def test_scores_that_are_not_finite_show(engine):
    cache = engine.PagedKVCache.empty(4, 1, 16, 64)
    cache.keys.normal_()
    cache.values.normal_()
    cache.keys[1, 0, 3, 5] = float("nan")
    q = torch.ones((3, 2, 64), dtype=torch.bfloat16, device="cuda")
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    who = torch.zeros(3, dtype=torch.int32, device="cuda")
    positions = torch.tensor([63, 18, 19], dtype=torch.int32, device="cuda")
    out, lse = cache.attend(q, table, who, positions, lse=True)
    assert out[0].isnan().all() and out[2].isnan().all() and out[1].isfinite().all()
    assert lse[0].isnan().all() and lse[1].isfinite().all()


def test_a_cache_past_32_bits(engine):
    # 6 GiB of keys: byte offsets past 2^32, value offsets past 2^31
    page, heads, dim = 128, 8, 128
    pages = 24_576
    keys = torch.empty((pages, heads, page, dim), dtype=torch.float16, device="cuda")
    values = torch.empty((pages, heads, dim, page), dtype=torch.float16, device="cuda")
    codes = torch.empty((pages, heads, dim), dtype=torch.int8, device="cuda")
    scales = torch.empty((pages, heads), dtype=torch.float32, device="cuda")
    big = engine.PagedKVCache(keys, values, codes, scales)
    small = engine.PagedKVCache.empty(3, heads, page, dim, dtype=torch.float16)
    rng = np.random.default_rng(9)
    n = 3 * page - 5
    k, v = (dev(rng.standard_normal((n, heads, dim), np.float32)).half() for _ in range(2))
    high = np.array([pages - 1, pages - 2, 17_000])
    i = np.arange(n)
    big.append(k, v, dev(high[i // page] * page + i % page))
    small.append(k, v, dev(i))
    q = dev(rng.standard_normal((2, 2 * heads, dim), np.float32)).half()
    who, pos = dev([0, 0], torch.int32), dev([n - 1, 200], torch.int32)
    t_big, t_small = dev(high[None].astype(np.int32)), dev(np.arange(3, dtype=np.int32)[None])
    assert torch.equal(big.attend(q, t_big, who, pos), small.attend(q, t_small, who, pos))
    assert torch.equal(codes[pages - 1], small.summaries[0])
    b = small.select(q, t_small, who, pos, 2)
    assert torch.equal(big.select(q, t_big, who, pos, 2), b)
    assert torch.equal(big.attend(q, t_big, who, pos, blocks=b),
                       small.attend(q, t_small, who, pos, blocks=b))


def test_the_same_queries_over_tables_of_other_heights(engine):
    """How work is split, and with it a call's workspace, goes by the requests
    too: tokens of one request share wavefronts and tiles, those of many do not."""
    rng = np.random.default_rng(77)
    cols, tokens = 80, 128
    cache = make_cache(engine, cols, 8, 64, 16, "bf16", rng)
    q = dev(rng.standard_normal((tokens, 8, 16), np.float32), torch.bfloat16)
    table = tables(rng, cols, 1, cols)
    positions = rng.integers(4000, cols * 64, tokens)
    wide = rng.integers(0, cols, (1, 800)).astype(np.int32)
    lists = []
    for height in (1, tokens, 1):
        check_attend(cache, "bf16", q, np.repeat(table, height, 0), np.arange(tokens) % height,
                     positions)
        lists.append(cache.select(q, dev(np.repeat(wide, height, 0)),
                                  dev(np.arange(tokens) % height, torch.int32),
                                  dev(positions, torch.int32), 12))
    assert torch.equal(lists[0], lists[1]) and torch.equal(lists[0], lists[2])


def test_many_requests_of_a_wide_table(engine):
    """A place for a million tokens in each of 2,048 rows: the workspace and the
    grid go by what the card can use, not by the table's width."""
    rng = np.random.default_rng(78)
    cache = make_cache(engine, 40, 8, 64, 64, "bf16", rng)
    requests, wide = 2048, 16384
    ids = rng.integers(0, 40, (requests, 25)).astype(np.int32)
    table = torch.full((requests, wide), -1, dtype=torch.int32, device="cuda")
    table[:, :25] = dev(ids)
    positions = rng.integers(-1, 1600, requests)
    q = dev(rng.standard_normal((requests, 8, 64), np.float32), torch.bfloat16)
    who = torch.arange(requests, dtype=torch.int32, device="cuda")
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    got = cache.attend(q, table, who, dev(positions, torch.int32))
    assert torch.cuda.max_memory_allocated() - before < 100 << 20
    some = rng.choice(requests, 50, replace=False)
    want = check_attend(cache, "bf16", q[dev(some)], ids, some, positions[some])
    assert torch.allclose(got[dev(some)].float(), want.float(), rtol=2.0 ** -6, atol=2.0 ** -6)


@pytest.mark.parametrize("listed", [False, True])
def test_prompts_over_a_table_without_columns(engine, listed):
    cache = engine.PagedKVCache.empty(2, 8, 64, 64)
    q = torch.ones((700, 8, 64), dtype=torch.bfloat16, device="cuda")
    table = torch.zeros((1, 0), dtype=torch.int32, device="cuda")
    zeros = torch.zeros(700, dtype=torch.int32, device="cuda")
    blocks = torch.zeros((700, 8, 3), dtype=torch.int32, device="cuda") if listed else None
    out, lse = cache.attend(q, table, zeros, zeros, blocks=blocks, lse=True)
    assert not out.any() and lse.isneginf().all()


def test_attend_none(engine):
    cache = engine.PagedKVCache.empty(2, 2, 16, 64)
    e = torch.empty((0, 4, 64), dtype=torch.bfloat16, device="cuda")
    i = torch.empty(0, dtype=torch.int32, device="cuda")
    t = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    out, lse = cache.attend(e, t, i, i, lse=True)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    q = torch.ones((1, 4, 64), dtype=torch.bfloat16, device="cuda")
    one = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = cache.attend(q, t[:, :0], one, one, lse=True)  # no columns
    assert not out.any() and lse.isneginf().all()
    out = cache.attend(q, t[:0], one, one)                    # no requests
    assert not out.any()


# ---- how they run --------------------------------------------------------------


def step_inputs(engine, rng, requests=5, page=16, heads=2, group=4, dim=64, cols=24):
    cache = engine.PagedKVCache.empty(requests * cols, heads, page, dim)
    past = rng.integers(1, (cols - 2) * page, requests).astype(np.int32)
    past[1] = 2 * page - 1  # completes a page
    table = np.full((requests, cols), -1, np.int32)
    free = rng.permutation(requests * cols).astype(np.int32)
    at = 0
    for r in range(requests):
        held = -(-int(past[r]) // page)
        table[r, :held] = free[at:at + held]
        at += held
    t = dev(table)
    who = np.concatenate([np.full(p, r) for r, p in enumerate(past)])
    pos = np.concatenate([np.arange(p) for p in past])
    n = len(pos)
    slots = dev(table[who, pos // page].astype(np.int64) * page + pos % page)
    k, v = (dev(rng.standard_normal((n, heads, dim), np.float32)).bfloat16() for _ in range(2))
    cache.append(k, v, slots)
    new = dev(np.ones(requests, np.int32))
    q = dev(rng.standard_normal((requests, heads * group, dim), np.float32)).bfloat16()
    k1, v1 = (dev(rng.standard_normal((requests, heads, dim), np.float32)).bfloat16()
              for _ in range(2))
    return cache, dev(past), new, t, dev(free), dev([at], torch.int32), q, k1, v1


def one_step(engine, cache, past, new, table, free, cursor, q, k, v, out=None, n=4):
    plan = engine.kv_plan(past, new, table, free, cursor, cache.page_size, len(q), out=out)
    cache.append(k, v, plan.slots)
    blocks = cache.select(q, table, plan.requests, plan.positions, n)
    sparse = cache.attend(q, table, plan.requests, plan.positions, blocks=blocks)
    dense = cache.attend(q, table, plan.requests, plan.positions)
    return plan, blocks, sparse, dense


def test_the_steps_of_a_serving_loop_agree_with_the_oracle(engine):
    rng = np.random.default_rng(21)
    cache, past, new, table, free, cursor, q, k, v = step_inputs(engine, rng)
    plan, blocks, sparse, dense = one_step(engine, cache, past, new, table, free, cursor, q, k, v)
    who, pos, t = (x.cpu().numpy() for x in (plan.requests, plan.positions, table))
    assert np.array_equal(pos, past.cpu().numpy())
    b = kv_oracle.select(f32(q), cache.summaries.cpu().numpy(), cache.scales.cpu().numpy(), t, who,
                         pos, cache.page_size, 4, 1, 1)
    assert np.array_equal(blocks.cpu().numpy(), b)
    assert torch.equal(check_attend(cache, "bf16", q, t, who, pos), dense)
    assert torch.equal(check_attend(cache, "bf16", q, t, who, pos, blocks=b), sparse)


def test_on_another_stream_and_repeatably(engine):
    rng = np.random.default_rng(22)
    inputs = step_inputs(engine, rng)
    want = [x.clone() for x in one_step(engine, *inputs)[1:]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = one_step(engine, *inputs)[1:]
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_in_a_graph(engine):
    rng = np.random.default_rng(23)
    inputs = step_inputs(engine, rng)
    cache, q = inputs[0], inputs[6]
    out = one_step(engine, *inputs)[0]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = one_step(engine, *inputs, out=out)
    for i in range(4):
        q.copy_(dev(rng.standard_normal(tuple(q.shape), np.float32)))
        g.replay()
        torch.cuda.synchronize()
        have = [x.clone() for x in got[1:]]
        want = one_step(engine, *inputs)[1:]
        torch.cuda.synchronize()
        for a, b in zip(have, want):
            assert torch.equal(a, b), i


def test_stage_times(engine):
    rng = np.random.default_rng(24)
    inputs = step_inputs(engine, rng)
    engine.profile(True)
    try:
        one_step(engine, *inputs)
        stages = engine.profile_report()
    finally:
        engine.profile(False)
    for name, count in (("kv_plan", 1), ("kv_append", 1), ("kv_select", 1), ("kv_attend", 2)):
        assert stages[name][0] == count


# ---- refusals ------------------------------------------------------------------


def test_refusals(engine):
    cache = engine.PagedKVCache.empty(4, 2, 16, 64)
    h = torch.float16

    def z(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device="cuda")

    i32, i64 = torch.int32, torch.int64
    q, who, table, kv = z(3, 4, 64), z(3, dtype=i32), z(1, 4, dtype=i32), z(3, 2, 64)
    keys, values = z(4, 2, 16, 64), z(4, 2, 64, 16)
    for make in (
            lambda: engine.PagedKVCache(keys.float(), values.float()),
            lambda: engine.PagedKVCache(keys, values.half()),
            lambda: engine.PagedKVCache(keys, keys),
            lambda: engine.PagedKVCache(keys.cpu(), values.cpu()),
            lambda: engine.PagedKVCache(keys[:, :, ::2], values),
            lambda: engine.PagedKVCache(keys, values, z(4, 2, 64, dtype=torch.int8)),
            lambda: engine.PagedKVCache(keys, values, z(4, 2, 64), z(4, 2)),
            lambda: engine.PagedKVCache.empty(4, 2, 24, 64),
            lambda: engine.PagedKVCache.empty(4, 2, 512, 64),
            lambda: engine.PagedKVCache.empty(4, 2, 16, 60),
            lambda: engine.PagedKVCache.empty(4, 2, 16, 264),
            lambda: cache.append(kv.half(), kv.half(), z(3, dtype=i64)),
            lambda: cache.append(kv, kv[:2], z(3, dtype=i64)),
            lambda: cache.append(kv, kv, z(3, dtype=i32)),
            lambda: cache.append(kv, kv, z(4, dtype=i64)),
            lambda: cache.append(z(3, 3, 64), z(3, 3, 64), z(3, dtype=i64)),
            lambda: cache.append(z(3, 2, 32), z(3, 2, 32), z(3, dtype=i64)),
            lambda: cache.attend(z(3, 3, 64), table, who, who),
            lambda: cache.attend(z(3, 1, 64), table, who, who),
            lambda: cache.attend(q.half(), table, who, who),
            lambda: cache.attend(q.cpu(), table, who, who),
            lambda: cache.attend(q, table.long(), who, who),
            lambda: cache.attend(q, table[0], who, who),
            lambda: cache.attend(q, table, who[:2], who),
            lambda: cache.attend(q, table, who, who.cpu()),
            lambda: cache.attend(q, table, who, who, scale=0.0),
            lambda: cache.attend(q, table, who, who, scale=-1.0),
            lambda: cache.attend(q, table, who, who, scale=float("nan")),
            lambda: cache.attend(q, table, who, who, longest=-1),
            lambda: cache.attend(q, table, who, who, out=z(3, 4, 64, dtype=h)),
            lambda: cache.attend(q, table, who, who, blocks=z(3, 2, 0, dtype=i32)),
            lambda: cache.attend(q, table, who, who, blocks=z(3, 2, 257, dtype=i32)),
            lambda: cache.attend(q, table, who, who, blocks=z(3, 4, 2, dtype=i32)),
            lambda: cache.attend(q, table, who, who, blocks=z(3, 2, 2, dtype=i64)),
            lambda: cache.select(q, table, who, who, 0),
            lambda: cache.select(q, table, who, who, 257),
            lambda: cache.select(q, table, who, who, 4, last=0),
            lambda: cache.select(q, table, who, who, 4, first=-1),
            lambda: cache.select(q, table, who, who, 4, first=3, last=2),
            lambda: engine.PagedKVCache.empty(4, 2, 16, 64, summaries=False).select(
                q, table, who, who, 4),
            lambda: engine.kv_plan(who.cpu(), who, table, who, who[:1], 16, 3),
            lambda: engine.kv_plan(who, who, table, who, who[:1], 16, 3),
            lambda: engine.kv_plan(who[:1], who[:1], table, who, who[:1], 17, 3),
            lambda: engine.kv_plan(who[:1], who[:1], table, who, who[:1], 16, -1),
            lambda: engine.kv_plan(who[:1], who[:1], table, who, who[:2], 16, 3),
            lambda: engine.kv_plan(who[:1].long(), who[:1], table, who, who[:1], 16, 3)):
        with pytest.raises(ValueError, match=r"\[mlxvs::|PagedKVCache"):
            make()
    plan = engine.kv_plan(who[:1], who[:1], table, who, who[:1], 16, 3)
    with pytest.raises(ValueError, match="cursor_out must not be cursor"):
        engine.kv_plan(who[:1], who[:1], table, who, plan.cursor, 16, 3, out=plan)
    with pytest.raises(ValueError, match="out.slots"):
        engine.kv_plan(who[:1], who[:1], table, who, who[:1], 16, 4, out=plan)


def test_tables_whose_rows_overlap_are_refused(engine):
    """A broadcast row, or rows that start within one another: neither is a
    table of so many requests in memory."""
    cache = engine.PagedKVCache.empty(4, 2, 16, 64)
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    who = torch.zeros(3, dtype=torch.int32, device="cuda")
    row = torch.zeros(8, dtype=torch.int32, device="cuda")
    for table in (row[:4].expand(3, 4), row.as_strided((3, 4), (2, 1))):
        for call in (lambda: cache.attend(q, table, who, who),
                     lambda: cache.select(q, table, who, who, 4),
                     lambda: engine.kv_plan(who, who, table, row, row[:1], 16, 3)):
            with pytest.raises(ValueError, match="do not overlap"):
                call()
    for table in (row[:4].expand(1, 4), row.as_strided((2, 1), (4, 7))):  # (one row, one column)
        assert not cache.attend(q, table, who, who).any()


def test_the_example(engine):
    import importlib.util
    from pathlib import Path
    path = Path(__file__).resolve().parent.parent / "examples" / "paged_cache.py"
    spec = importlib.util.spec_from_file_location("paged_cache", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    lengths, close, ms = example.run(requests=3, context=700, steps=5, blocks=16)
    assert lengths == [238, 464, 691] and ms > 0
    # (12 blocks at most: the lists hold everything, and the two answers are two
    # roundings of one sum)
    assert close > 0.999
