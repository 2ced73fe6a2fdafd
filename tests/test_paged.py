"""Batched serving over the paged 8-bit cache on the GPU against restatements in 64 bits (paged_ref.py)."""
import numpy as np
import pytest

import paged_ref as ref
import tachyon_b200 as tb

pytestmark = pytest.mark.gpu
ENDS = tb.REQUEST_ENDS


def words(ctx, a):
    return ctx.upload(np.asarray(a, np.uint32))


# ---- page tables -----------------------------------------------------------------------------------------------------


def a_pool(rng, lengths, page, width, spare):
    need = [-(-int(x) // page) for x in lengths]
    pages = sum(need) + spare
    order = rng.permutation(max(pages, 1)).astype(np.uint32)
    table = np.full((len(lengths), width), 0xDEAD, np.uint32)
    at = 0
    for r, k in enumerate(need):
        table[r, :k] = order[at:at + k]
        at += k
    free = np.full(max(pages, 1), 0xBEEF, np.uint32)
    free[: pages - at] = order[at:pages]
    return table, free, pages - at, max(pages, 1)


def run_plan(ctx, lengths, fresh, table, free, count, page, pages, max_tokens, in_place=False, positions=True):
    n, width = table.shape
    b = {k: words(ctx, v) for k, v in dict(lengths=lengths, fresh=fresh, table=table, free=free, count=[count], starts=np.full(n + 1, 7), refused=[9], scratch=[0]).items()}
    b["slots"], b["positions"] = words(ctx, np.full(max_tokens + 3, 0xABCD)), words(ctx, np.full(max_tokens + 3, 0xABCD))
    b["lengths_out"] = b["lengths"] if in_place else words(ctx, np.full(n, 5))
    b["count_out"] = b["count"] if in_place else words(ctx, [5])
    ctx.page_plan(tb.PagePlan(lengths=b["lengths"].ptr, fresh=b["fresh"].ptr, lengths_out=b["lengths_out"].ptr, table=b["table"].ptr, free_pages=b["free"].ptr,
                              free_count=b["count"].ptr, free_count_out=b["count_out"].ptr, starts=b["starts"].ptr, slots=b["slots"].ptr,
                              positions=b["positions"].ptr if positions else None, refused=b["refused"].ptr, scratch=b["scratch"].ptr, requests=n, width=width, page=page,
                              pages=pages, max_tokens=max_tokens))
    got = {k: v.download(np.uint32) for k, v in b.items()}
    assert got["scratch"][0] == 0
    return got


def check_plan(got, want, table, free, max_tokens):
    n = len(want["slots"])
    assert got["refused"][0] == want["refused"]
    assert np.array_equal(got["lengths_out"][: table.shape[0]], want["lengths"])
    assert got["count_out"][0] == want["count"]
    assert np.array_equal(got["starts"][: table.shape[0] + 1], want["starts"])
    assert np.array_equal(got["table"][: table.size].reshape(table.shape), want["table"])
    assert np.array_equal(got["free"][: free.size], want["free"])
    assert np.array_equal(got["slots"][:n], np.array(want["slots"], np.uint32))
    assert np.array_equal(got["positions"][:n], np.array(want["positions"], np.uint32))
    assert np.all(got["slots"][n: max_tokens + 3] == 0xABCD) and np.all(got["positions"][n: max_tokens + 3] == 0xABCD), "entries past the last token were written"


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("requests,page,longest,most,seed", [(1, 16, 1, 1, 0), (1, 128, 300, 300, 1), (3, 16, 100, 33, 2), (64, 64, 1000, 1, 3), (257, 32, 200, 70, 4),
                                                             (513, 16, 64, 2, 5), (2000, 16, 90, 17, 6), (8192, 32, 40, 3, 7), (5, 16, 9000, 4000, 8)])
def test_plan(ctx, requests, page, longest, most, seed, in_place):
    rng = np.random.default_rng(seed)
    lengths = rng.integers(0, longest, requests).astype(np.uint32)
    fresh = rng.integers(0, most + 1, requests).astype(np.uint32)
    fresh[rng.random(requests) < 0.1] = ENDS
    lengths[rng.random(requests) < 0.1] = 0
    width = -(-(longest + most) // page)
    table, free, count, pages = a_pool(rng, lengths, page, width, spare=int(sum(-(-int(f) // page) + 1 for f in fresh if f != ENDS)) + 3)
    max_tokens = int(sum(int(f) for f in fresh if f != ENDS)) + (seed % 2)
    want = ref.plan(lengths, fresh, table, free, count, page, pages, max_tokens)
    assert want["refused"] == 0
    check_plan(run_plan(ctx, lengths, fresh, table, free, count, page, pages, max_tokens, in_place), want, table, free, max_tokens)


def test_plan_takes_pages_that_this_call_gets_back(ctx):
    """No page is free: a request that grows gets those of the one that ends, the last given back first, and what is left of them lands in the free list."""
    lengths, fresh = np.array([40, 16, 0], np.uint32), np.array([ENDS, 1, 0], np.uint32)
    rng = np.random.default_rng(0)
    table, free, count, pages = a_pool(rng, lengths, 16, 4, spare=0)
    assert count == 0
    want = ref.plan(lengths, fresh, table, free, count, 16, pages, 1)
    assert want["refused"] == 0 and want["count"] == 2 and want["table"][1, 1] == table[0, 2]
    check_plan(run_plan(ctx, lengths, fresh, table, free, count, 16, pages, 1), want, table, free, 1)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("why,lengths,fresh,spare,width,max_tokens", [(1, [16, 16], [1, 1], 1, 4, 9), (2, [60, 3], [5, 1], 9, 4, 9), (2, [0xFFFFFFF0, 3], [0xFFFFFFFE, 1], 9, 4, 9),
                                                                      (2, [65, 3], [ENDS, 1], 9, 4, 9), (4, [3, 3], [5, 5], 9, 4, 9),
                                                                      (5, [16, 16], [16, 17], 1, 4, 9)])
def test_plan_refuses_and_changes_nothing(ctx, why, lengths, fresh, spare, width, max_tokens, in_place):
    lengths, fresh = np.array(lengths, np.uint32), np.array(fresh, np.uint32)
    rng = np.random.default_rng(1)
    table, free, count, pages = a_pool(rng, np.minimum(lengths, width * 16), 16, width, spare)
    want = ref.plan(lengths, fresh, table, free, count, 16, pages, max_tokens)
    got = run_plan(ctx, lengths, fresh, table, free, count, 16, pages, max_tokens, in_place)
    assert got["refused"][0] & why == why
    want["refused"] = got["refused"][0] if why == 2 else want["refused"]
    check_plan(got, want, table, free, max_tokens)


def test_plan_refuses_a_free_list_that_cannot_be(ctx):
    lengths, fresh = np.array([20], np.uint32), np.array([ENDS], np.uint32)
    table, free = np.array([[0, 1]], np.uint32), np.arange(4, dtype=np.uint32)
    assert run_plan(ctx, lengths, fresh, table, free, 3, 16, 4, 1)["refused"][0] == 8  # 3 free + 2 back > 4 pages
    assert run_plan(ctx, lengths, np.array([0], np.uint32), table, free, 5, 16, 4, 1)["refused"][0] == 8


def test_plan_names_no_slot_where_the_table_names_no_page(ctx):
    lengths, fresh = np.array([3, 3], np.uint32), np.array([2, 2], np.uint32)
    table, free = np.array([[99], [1]], np.uint32), np.zeros(4, np.uint32)
    got = run_plan(ctx, lengths, fresh, table, free, 0, 16, 4, 4, positions=False)
    assert list(got["slots"][:4]) == [0xFFFFFFFF, 0xFFFFFFFF, 16 + 3, 16 + 4]
    assert np.all(got["positions"] == 0xABCD)


# ---- the cache -------------------------------------------------------------------------------------------------------


class Cache:
    """A cache on the GPU and its twin on the host."""

    def __init__(self, ctx, pages, kv_heads, page, D, seed, fill=True):
        rng = np.random.default_rng(seed)
        shape = (pages, kv_heads, page, D)
        self.page, self.pages, self.kv_heads, self.D = page, pages, kv_heads, D
        draw = lambda: np.clip(np.rint(rng.standard_normal(shape) * 28), -127, 127).astype(np.int8) if fill else rng.integers(-127, 128, shape).astype(np.int8)  # noqa: E731
        self.k, self.v = draw(), draw()
        self.ks, self.vs = (2.0 ** rng.integers(-7, -3, (pages, kv_heads))).astype(np.float32), (2.0 ** rng.integers(-8, -2, (pages, kv_heads))).astype(np.float32)
        self.dev = [ctx.upload(x) for x in (self.k, self.v, self.ks, self.vs)]

    def pages_of(self, table=None, requests=0, width=0):
        k, v, ks, vs = self.dev
        return tb.Pages(k=k.ptr, v=v.ptr, k_scale=ks.ptr, v_scale=vs.ptr, table=None if table is None else table.ptr, pages=self.pages, page=self.page,
                        kv_heads=self.kv_heads, head_dim=self.D, requests=requests, width=width)

    def download(self):
        k, v, ks, vs = self.dev
        return (k.download(np.int8, self.k.size).reshape(self.k.shape), v.download(np.int8, self.v.size).reshape(self.v.shape),
                ks.download(np.float32, self.ks.size).reshape(self.ks.shape), vs.download(np.float32, self.vs.size).reshape(self.vs.shape))

    def check(self):
        for got, want in zip(self.download(), (self.k, self.v, self.ks, self.vs)):
            assert np.array_equal(got, want)


def append(ctx, cache, k, v, slots, kind=np.float32, token_stride=None, head_stride=None):
    """Rows [tokens][heads][D] at the given strides (rows may overlap: the oracle takes what the memory holds), into the cache and its twin."""
    n, heads, D = k.shape
    token_stride, head_stride = token_stride or heads * D, head_stride or D
    size = (n - 1) * token_stride + (heads - 1) * head_stride + D
    bufs, held = [], []
    for x in (k, v):
        flat = np.full(size, 1e30 if kind == np.float32 else 6e4, kind)
        for t in range(n):
            for h in range(heads):
                flat[t * token_stride + h * head_stride:][:D] = x[t, h]
        bufs.append(ctx.upload(flat))
        at = np.arange(n)[:, None, None] * token_stride + np.arange(heads)[:, None] * head_stride + np.arange(D)
        held.append(flat[at])
    s = words(ctx, slots)
    ctx.cache_append_q8(tb.CacheRows(cache=cache.pages_of(), k=bufs[0].ptr, v=bufs[1].ptr, dtype=tb.F32 if kind == np.float32 else tb.F16, token_stride=token_stride,
                                     head_stride=head_stride, slots=s.ptr, tokens=n))
    ctx.sync()
    ref.append(cache.k, cache.ks, held[0], slots, cache.page)
    ref.append(cache.v, cache.vs, held[1], slots, cache.page)


def run_slots(table_row, first, count, page):
    p = np.arange(first, first + count)
    return np.asarray(table_row)[p // page] * page + p % page


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("D,page,heads", [(64, 16, 1), (128, 64, 8), (256, 32, 2), (512, 128, 3), (64, 128, 5), (128, 16, 2), (512, 16, 1)])
def test_append(ctx, D, page, heads, kind):
    """Three requests: into a page begun before, over several pages, a single token; then single tokens over and over, as decoding appends them.
    The codes and scales are the definition's, exactly, and nothing else is written."""
    rng = np.random.default_rng(D + page)
    cache = Cache(ctx, 40, heads, page, D, 1, fill=False)
    order = rng.permutation(40)
    rows, at = [order[:10], order[10:20], order[20:30]], [page // 2 + 1, 0, page - 1]
    for step, counts in enumerate([(page // 2, 4 * page + 3, 1), (1, 1, 1), (1, 1, 1), (page, 2, 1), (1, 0, 3)]):
        slots = np.concatenate([run_slots(r, a, c, page) for r, a, c in zip(rows, at, counts)])
        n = len(slots)
        grow = 2.0 ** rng.integers(-3, 4, (n, 1, 1))
        k, v = (rng.standard_normal((n, heads, D)) * grow).astype(np.float32), rng.standard_normal((n, heads, D)).astype(np.float32)
        append(ctx, cache, k, v, slots, kind, *((None, None) if step else (heads * D + 24, D + 8)))
        cache.check()
        at = [a + c for a, c in zip(at, counts)]


def test_append_of_many_single_tokens(ctx):
    """More tokens than blocks take one by one: the span of a block holds several runs."""
    heads, D, page, n = 8, 64, 16, 3000
    cache = Cache(ctx, n, heads, page, D, 2, fill=False)
    rng = np.random.default_rng(3)
    slots = rng.permutation(n) * page + rng.integers(0, page, n)
    x = rng.standard_normal((2, n, heads, D)).astype(np.float32)
    append(ctx, cache, x[0], x[1], slots)
    cache.check()


def test_append_of_a_long_chunk(ctx):
    heads, D, page, n = 2, 128, 32, 5000
    cache = Cache(ctx, 200, heads, page, D, 2, fill=False)
    rng = np.random.default_rng(3)
    x = rng.standard_normal((2, n, heads, D)).astype(np.float16)
    append(ctx, cache, x[0], x[1], run_slots(rng.permutation(200), 7, n, page), np.float16)
    cache.check()


def test_append_of_what_is_no_number_and_of_extremes(ctx):
    """Infinities become the ends and set no scale, NaN becomes 0; the smallest and largest f32, zeros, and the borders 127 * 2^e of the scale."""
    heads, D, page = 1, 64, 16
    cache = Cache(ctx, 20, heads, page, D, 5)
    rows = np.zeros((14, heads, D), np.float32)
    rows[0, 0, :3] = [np.inf, -np.inf, np.nan]
    rows[1, 0, :4] = [np.inf, 1.0, np.nan, -2.0]
    rows[2, 0, :2] = [1e-45, -1e-45]
    rows[3, 0, :2] = [3.4028235e38, -3.4e38]
    rows[4, 0, 0] = 127.0
    rows[5, 0, 0] = np.nextafter(np.float32(127), np.float32(200))
    rows[6, 0, 0] = np.nextafter(np.float32(127), np.float32(0))
    rows[8, 0, :3] = [254.0, 1.0, 3.0]  # ties: 0.5 and 1.5 to even
    rows[9, 0, 0] = 2.0**-126
    rows[10, 0, 0] = 127 * 2.0**-126
    rows[11, 0, 0] = np.nextafter(np.float32(127 * 2.0**-126), np.float32(1))
    slots = np.arange(14) * page
    append(ctx, cache, rows, rows, slots)
    cache.check()
    # onto pages begun with zeros, with infinities, with the largest numbers; and zeros onto each
    append(ctx, cache, rows[::-1].copy(), rows, slots + 1)
    cache.check()
    append(ctx, cache, 0 * np.nan_to_num(rows), rows, slots + 2)
    cache.check()


def test_append_skips_slots_past_the_cache(ctx):
    heads, D, page = 2, 128, 16
    cache = Cache(ctx, 4, heads, page, D, 6)
    x = np.random.default_rng(1).standard_normal((6, heads, D)).astype(np.float32)
    append(ctx, cache, x, x, np.array([0xFFFFFFFF, 0, 4 * page, 5, 0xFFFFFFFE, 3 * page + 15], np.uint64))
    got = cache.download()
    for a, b in zip(got, (cache.k, cache.v, cache.ks, cache.vs)):
        assert np.array_equal(a[1:], b[1:])  # page 0 gets two runs in one call, which the header leaves undefined: its neighbours stand
    cache.k, cache.v, cache.ks, cache.vs = got
    append(ctx, cache, x, x, np.array([0xFFFFFFFF, 0, 4 * page, page + 5, 0xFFFFFFFE, 3 * page + 15], np.uint64))
    cache.check()


def test_a_page_that_grows_token_by_token_stays_within_a_step(ctx):
    """Requantising halves codes: however often the maximum rises, a stored number is off by less than its page's final step (1/2 + 1/4 + ... of it)."""
    heads, D, page = 1, 64, 128
    cache = Cache(ctx, 1, heads, page, D, 7)
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((page, heads, D)) * np.exp2(np.linspace(-4, 6, page))[:, None, None]).astype(np.float32)
    for t in range(page):
        append(ctx, cache, x[t:t + 1], x[t:t + 1], np.array([t]))
    cache.check()
    k, _, ks, _ = cache.download()
    assert np.abs(k[0, 0] * ks[0, 0] - x[:, 0]).max() < ks[0, 0]


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("D,page,heads", [(64, 16, 1), (128, 64, 8), (512, 128, 3)])
def test_read(ctx, D, page, heads, kind):
    cache = Cache(ctx, 9, heads, page, D, 9)
    slots = np.random.default_rng(1).integers(0, 9 * page, 50).astype(np.uint64)
    slots[7] = 9 * page  # past the cache: its row is left as it was
    token_stride, head_stride = heads * (D + 8) + 16, D + 8
    bufs = [ctx.upload(np.full(50 * token_stride, 77, kind)) for _ in range(2)]
    ctx.cache_read_q8(tb.CacheRows(cache=cache.pages_of(), k=bufs[0].ptr, v=bufs[1].ptr, dtype=tb.F32 if kind == np.float32 else tb.F16, token_stride=token_stride,
                                   head_stride=head_stride, slots=words(ctx, slots).ptr, tokens=50))
    for buf, codes, scale in ((bufs[0], cache.k, cache.ks), (bufs[1], cache.v, cache.vs)):
        want = np.full(50 * token_stride, 77, kind)
        for t, s in enumerate(slots):
            if s < 9 * page:
                for h in range(heads):
                    want[t * token_stride + h * head_stride:][:D] = (codes[s // page, h, s % page] * scale[s // page, h]).astype(kind)
        assert np.array_equal(buf.download(kind, want.size), want)
    cache.check()


# ---- attention -------------------------------------------------------------------------------------------------------


def attention_bound(want, size, vmax, D, keys, out_f16, p_f16):
    """What the arithmetic may be off by.  A score is a sum of D products in f32 (D / 16 steps, a rounding of 2^-23 of the running
    sum each and some inside a step) of queries exact to 2^-22, and the exponent's argument is rounded again; a relative error e of every
    weight moves the mean by at most 2 e vmax; the weights' sum and products are added up in f32 over keys / 16 steps.  With weights
    in f16 (prefill) each is off by 2^-11 more (2^-25 absolute below f16's normal range, over the keys)."""
    e = size * (2.0**-21 + (D / 16 + 20) * 2.0**-23) + 2.0**-21
    bound = vmax * (2 * e + (keys / 16 + 64) * 2.0**-23)
    if p_f16:
        bound = bound + vmax * (2 * 2.0**-11 + keys * 2.0**-25)
    if out_f16:
        bound = bound + np.abs(want) * 2.0**-11 + 2.0**-25
    return bound + 1e-30


def run_attend(ctx, cache, q, q_kind, table, starts, lengths, window, scale, out_kind, most, prefill=False, scratch=None, extra=2, stride=0, null_starts=False):
    tokens, heads, D = q.shape
    total = tokens + extra
    row = heads * D + stride
    flat = np.zeros((total, row), q_kind)
    flat[:tokens, : heads * D] = q.reshape(tokens, heads * D)
    qd = ctx.upload(flat)
    out = ctx.upload(np.full((total, row), 3, out_kind))
    scratch = scratch or ctx.zeros(ctx.paged_scratch_bytes(D))
    td, sd, ld = words(ctx, table), words(ctx, starts), words(ctx, lengths)
    kind = lambda x: tb.F32 if x == np.float32 else tb.F16  # noqa: E731
    a = tb.PagedAttend(cache=cache.pages_of(td, len(lengths), table.shape[1]), q=qd.ptr, q_dtype=kind(q_kind), q_stride=row, starts=None if null_starts else sd.ptr,
                       lengths=ld.ptr, tokens=tokens if null_starts else total, heads=heads, most=most, window=window, scale=scale, out=out.ptr, out_dtype=kind(out_kind),
                       out_stride=row, scratch=scratch.ptr, scratch_bytes=scratch.nbytes)
    (ctx.prefill_paged_q8 if prefill else ctx.attend_paged_q8)(a)
    got = out.download(out_kind, total * row).reshape(total, row)
    assert not scratch.download(np.uint32, 1024).any(), "the counters were not left zero"
    assert np.all(got[tokens:] == 3) and np.all(got[:, heads * D:] == 3), "rows or columns that no request owns were written"
    return got[:tokens, : heads * D].reshape(tokens, heads, D)


def tables(rng, lengths, page, width, pages):
    """Every request's pages anywhere in the pool, some shared between requests; unused entries name no page."""
    table = np.full((len(lengths), width), 0xFFFFFFFF, np.uint32)
    for r, n in enumerate(lengths):
        k = -(-int(n) // page)
        table[r, :k] = rng.choice(pages, k, replace=pages < k)
    return table


def attend_case(ctx, D, page, kvh, ratio, lengths, new, window, q_kind, out_kind, prefill=False, seed=0, spread=1.0, most=None, **more):
    rng = np.random.default_rng(seed + D + page)
    pages = max(8, -(-max(lengths, default=1) // page) + 3)
    cache = Cache(ctx, pages, kvh, page, D, seed)
    width = max(1, -(-max(lengths) // page)) + 1
    table = tables(rng, lengths, page, width, pages)
    starts = np.concatenate([[0], np.cumsum(new)])
    tokens, heads = int(starts[-1]), kvh * ratio
    q = (rng.standard_normal((tokens, heads, D)) * spread).astype(q_kind)
    scale = 1 / np.sqrt(D)
    got = run_attend(ctx, cache, q, q_kind, table, starts, lengths, window, scale, out_kind, most or max(new), prefill, **more)
    want, size, vmax = ref.attend(q.astype(np.float64), cache.k, cache.ks, cache.v, cache.vs, table, starts, lengths, window, scale, page)
    bound = attention_bound(want, size, vmax, D, max(lengths), out_kind == np.float16, prefill)
    if prefill and q_kind == np.float32:
        bound = bound + 2 * vmax * size * 2.0**-11
    off = np.abs(got.astype(np.float64) - want)
    assert np.all(off <= bound), float((off / bound).max())


@pytest.mark.parametrize("D,page,kvh,ratio", [(64, 16, 1, 1), (64, 128, 3, 7), (128, 16, 8, 4), (128, 64, 2, 8), (256, 32, 2, 4), (256, 64, 1, 2), (512, 128, 2, 4), (512, 16, 1, 8)])
@pytest.mark.parametrize("q_kind,out_kind", [(np.float32, np.float32), (np.float16, np.float16)])
@pytest.mark.parametrize("window", [0, 37])
def test_attend_single_tokens(ctx, D, page, kvh, ratio, window, q_kind, out_kind):
    lengths = [1, 17, 0, 63, 64, 65, 16, 300, 129, 1000]
    attend_case(ctx, D, page, kvh, ratio, lengths, [1] * len(lengths), window, q_kind, out_kind, spread=2.0)


@pytest.mark.parametrize("D,ratio,new", [(64, 4, [1, 4, 0, 3, 2]), (128, 5, [2, 2, 2, 1, 0]), (256, 8, [8, 1, 3, 0, 2]), (512, 16, [1, 2, 4, 4, 1]), (128, 40, [1, 1, 1, 1, 1])])
@pytest.mark.parametrize("window", [0, 3, 100])
def test_attend_a_few_tokens(ctx, D, ratio, new, window):
    """Drafted tokens checked at once, ragged; more query rows than a group of eight."""
    attend_case(ctx, D, 32, 2, ratio, [5, 77, 40, 200, 513], new, window, np.float32, np.float32, seed=3)


@pytest.mark.parametrize("D", [64, 128, 256, 512])
@pytest.mark.parametrize("lengths", [[30000], [9000, 1, 20000, 700], [4096] * 3])
def test_attend_long(ctx, D, lengths):
    """Lines of keys shared by many blocks."""
    attend_case(ctx, D, 64, 2, 4, lengths, [1] * len(lengths), 0, np.float32, np.float32, seed=5)


def test_attend_many_requests(ctx):
    rng = np.random.default_rng(4)
    lengths = list(rng.integers(0, 90, 700))
    attend_case(ctx, 64, 16, 2, 2, lengths, [1] * 700, 0, np.float16, np.float32)


def test_attend_without_starts_and_with_strides(ctx):
    attend_case(ctx, 128, 16, 2, 4, [30, 70, 1], [1, 1, 1], 0, np.float32, np.float16, null_starts=True, extra=0, stride=24)
    attend_case(ctx, 128, 16, 2, 4, [30, 70, 9], [3, 1, 2], 0, np.float16, np.float32, stride=8, most=5)


@pytest.mark.parametrize("prefill", [False, True])
def test_attend_over_bad_pages_and_bad_lengths(ctx, prefill):
    """Entries that name no page hide their positions, lengths past the table end with it, more new tokens than positions see nothing, tokens past `most` are left."""
    rng = np.random.default_rng(11)
    D, page, kvh, ratio, pages = 128, 16, 2, 4, 20
    cache = Cache(ctx, pages, kvh, page, D, 3)
    lengths = [100, 64, 33, 10**9, 2, 5]
    table = rng.integers(0, pages, (6, 8)).astype(np.uint32)
    table[0, [0, 3, 6]] = [pages, 0xFFFFFFFF, 1 << 31]
    table[1, :] = pages
    new = [1, 2, 1, 1, 3, 4]
    starts = np.concatenate([[0], np.cumsum(new)])
    q = rng.standard_normal((int(starts[-1]), kvh * ratio, D)).astype(np.float16)
    got = run_attend(ctx, cache, q, np.float16, table, starts, lengths, 0, 0.1, np.float32, 3, prefill)
    seen = [min(x, 128) for x in lengths]
    want, size, vmax = ref.attend(q.astype(np.float64), cache.k, cache.ks, cache.v, cache.vs, table, starts, seen, 0, 0.1, page)
    # the last request brings four tokens where `most` says three: the first three count as its newest
    t0 = int(starts[5])
    want[t0: t0 + 3] = ref.attend(q[t0: t0 + 3].astype(np.float64), cache.k, cache.ks, cache.v, cache.vs, table[5:6], [0, 3], seen[5:], 0, 0.1, page)[0]
    want[t0 + 3] = 3
    bound = attention_bound(want, size, vmax, D, 128, False, prefill)
    assert np.all(np.abs(got - want) <= bound)
    assert np.all(got[1:3] == 0) and np.all(got[5] == 0)


@pytest.mark.parametrize("prefill", [False, True])
def test_attend_with_starts_that_cannot_be(ctx, prefill):
    """Falling or far starts own no rows or the rows there are; nothing outside is touched."""
    rng = np.random.default_rng(12)
    cache = Cache(ctx, 9, 2, 16, 64, 3)
    q = rng.standard_normal((4, 2, 64)).astype(np.float16)
    table = rng.integers(0, 9, (3, 4)).astype(np.uint32)
    got = run_attend(ctx, cache, q, np.float16, table, [3, 2, 0xFFFFFFFF, 0xFFFFFFFF], [9, 9, 9], 0, 1.0, np.float32, 2, prefill, extra=0)
    want, _, vmax = ref.attend(q.astype(np.float64), cache.k, cache.ks, cache.v, cache.vs, table, [2, 2, 4, 4], [9, 9, 9], 0, 1.0, 16)
    assert np.all(got[:2] == 3) and np.abs(got[2:] - want[2:]).max() <= 2.0**-9 * vmax


def test_attend_scores_far_apart_and_scales_far_apart(ctx):
    """One key decides; value scales of pages lie 2^40 apart, zero pages among them."""
    D, page, kvh = 128, 16, 1
    cache = Cache(ctx, 16, kvh, page, D, 3)
    cache.vs[:, 0] = 2.0 ** np.array([-30, 10, 0, -5, 3, -20, 8, 0, -30, 10, 0, -5, 3, -20, 8, 0])
    cache.vs[4], cache.v[4] = 0, 0
    cache.ks[2], cache.k[2] = 0, 0
    cache.dev[:] = [ctx.upload(x) for x in (cache.k, cache.v, cache.ks, cache.vs)]
    rng = np.random.default_rng(1)
    table = np.arange(16, dtype=np.uint32)[None]
    for spread in (0.01, 1.0, 30.0):
        q = (rng.standard_normal((1, 4, D)) * spread).astype(np.float32)
        got = run_attend(ctx, cache, q, np.float32, table, [0, 1], [250], 0, 1.0, np.float32, 1)
        want, size, vmax = ref.attend(q.astype(np.float64), cache.k, cache.ks, cache.v, cache.vs, table, [0, 1], [250], 0, 1.0, page)
        assert np.all(np.abs(got - want) <= attention_bound(want, size, vmax, D, 250, False, False))


def test_attend_queries_of_any_size(ctx):
    """Queries at both ends of f32 are scaled before they are cut into f16 parts."""
    D, page = 64, 16
    cache = Cache(ctx, 4, 1, page, D, 3)
    rng = np.random.default_rng(1)
    table = np.arange(4, dtype=np.uint32)[None]
    base = rng.standard_normal((1, 2, D)).astype(np.float32)
    for f in (1e-30, 1e-8, 1e8, 1e30):
        q = base * np.float32(f)
        scale = np.float32(1 / f)
        got = run_attend(ctx, cache, q, np.float32, table, [0, 1], [50], 0, scale, np.float32, 1)
        want, size, vmax = ref.attend(q.astype(np.float64), cache.k, cache.ks, cache.v, cache.vs, table, [0, 1], [50], 0, float(scale), page)
        assert np.all(np.abs(got - want) <= attention_bound(want, size, vmax, D, 50, False, False))


@pytest.mark.parametrize("prefill", [False, True])
def test_attend_past_32_bits_of_offset(ctx, prefill):
    """Pages whose codes start past 2^32 bytes into the cache."""
    D, page, kvh, pages = 512, 128, 4, 17000  # 262144 bytes a page: 4.46 GB
    rng = np.random.default_rng(2)
    used = np.array([16999, 0, 16500, 8200], np.uint32)
    small = Cache(ctx, 4, kvh, page, D, 5)
    k, v = ctx.alloc(pages * kvh * page * D), ctx.alloc(pages * kvh * page * D)
    size = kvh * page * D
    ks, vs = np.ones((pages, kvh), np.float32), np.ones((pages, kvh), np.float32)
    for i, u in enumerate(used):
        for buf, codes in ((k, small.k), (v, small.v)):
            part = np.ascontiguousarray(codes[i])
            tb.check(ctx.lib.tb_upload(ctx.handle, buf.ptr + int(u) * size, part.ctypes.data, part.nbytes))
            ctx.sync()
        ks[u], vs[u] = small.ks[i], small.vs[i]
    big = Cache.__new__(Cache)
    big.page, big.pages, big.kv_heads, big.D, big.dev = page, pages, kvh, D, [k, v, ctx.upload(ks), ctx.upload(vs)]
    new = 1 if not prefill else 70
    q = rng.standard_normal((new, 8, D)).astype(np.float16)
    got = run_attend(ctx, big, q, np.float16, used[None], [0, new], [500], 0, 0.05, np.float32, new, prefill)
    want, s, vmax = ref.attend(q.astype(np.float64), small.k, small.ks, small.v, small.vs, np.arange(4, dtype=np.uint32)[None], [0, new], [500], 0, 0.05, page)
    assert np.all(np.abs(got - want) <= attention_bound(want, s, vmax, D, 500, False, prefill))
    x = rng.standard_normal((2, kvh, D)).astype(np.float32)
    rows, back = ctx.upload(x), ctx.zeros(x.nbytes)
    slots = words(ctx, used[:1].astype(np.uint64) * page + np.arange(2))
    ctx.cache_append_q8(tb.CacheRows(cache=big.pages_of(), k=rows.ptr, v=rows.ptr, dtype=tb.F32, token_stride=kvh * D, head_stride=D, slots=slots.ptr, tokens=2))
    ctx.cache_read_q8(tb.CacheRows(cache=big.pages_of(), k=back.ptr, v=back.ptr, dtype=tb.F32, token_stride=kvh * D, head_stride=D, slots=slots.ptr, tokens=2))
    got = back.download(np.float32, x.size).reshape(x.shape)
    assert np.abs(got - x).max() <= np.abs(x).max() * 2.0**-7  # half a step: the step is at most 2 / 127 of the largest


def test_attend_gives_the_same_bits_and_shares_scratch(ctx):
    """Twice the same call, with a call of another shape through the same scratch between them."""
    rng = np.random.default_rng(6)
    scratch = ctx.zeros(max(ctx.paged_scratch_bytes(D) for D in (64, 128, 256, 512)))
    outs = []
    for _ in range(2):
        for D, kvh, lengths in ((128, 2, [5000, 300, 9000]), (512, 1, [7000]), (256, 2, [40] * 9)):
            cache = Cache(ctx, 150, kvh, 64, D, 1)
            table = tables(np.random.default_rng(3), lengths, 64, 150, 150)
            q = np.random.default_rng(4).standard_normal((len(lengths), kvh * 4, D)).astype(np.float32)
            outs.append(run_attend(ctx, cache, q, np.float32, table, np.arange(len(lengths) + 1), lengths, 0, 0.1, np.float32, 1, scratch=scratch))
    for a, b in zip(outs[:3], outs[3:]):
        assert np.array_equal(a, b)
    assert rng is not None


@pytest.mark.parametrize("window", [0x7FFFFFFF, 0x80000000, 0xFFFFFFFF])
def test_attend_windows_past_every_position(ctx, window):
    attend_case(ctx, 64, 16, 1, 2, [100, 7], [2, 1], window, np.float16, np.float32)
    attend_case(ctx, 64, 16, 1, 2, [100, 7], [90, 1], window, np.float16, np.float32, prefill=True)


def test_attend_needs_its_scratch(ctx):
    cache = Cache(ctx, 2, 1, 16, 64, 1)
    small = ctx.zeros(ctx.paged_scratch_bytes(64) - 16)
    with pytest.raises(tb.Error, match="tb_paged_scratch_bytes") as e:
        run_attend(ctx, cache, np.zeros((1, 1, 64), np.float32), np.float32, np.zeros((1, 1), np.uint32), [0, 1], [3], 0, 1.0, np.float32, 1, scratch=small)
    assert e.value.status == 3


@pytest.mark.parametrize("D,page,kvh,ratio", [(64, 16, 2, 2), (128, 64, 2, 4), (256, 32, 1, 4), (256, 64, 2, 8), (512, 128, 1, 4), (128, 16, 1, 7), (64, 128, 1, 1), (128, 32, 1, 64)])
@pytest.mark.parametrize("window", [0, 50])
@pytest.mark.parametrize("q_kind,out_kind", [(np.float16, np.float16), (np.float32, np.float32)])
def test_prefill(ctx, D, page, kvh, ratio, window, q_kind, out_kind):
    """Chunks from a prompt's first token, late in it, ragged, a single token, an idle request."""
    attend_case(ctx, D, page, kvh, ratio, [70, 300, 1, 40, 129], [70, 33, 1, 0, 65], window, q_kind, out_kind, prefill=True)


@pytest.mark.parametrize("D,ratio", [(64, 4), (128, 4), (256, 4), (512, 4), (128, 1)])
@pytest.mark.parametrize("spread", [1.0, 8.0])
def test_prefill_longer(ctx, D, ratio, spread):
    attend_case(ctx, D, 64, 1, ratio, [1500, 260], [200, 257], 0, np.float16, np.float32, prefill=True, spread=spread)


@pytest.mark.parametrize("D,page,kvh,ratio", [(64, 16, 2, 4), (128, 64, 1, 7), (256, 32, 2, 4), (512, 128, 1, 4)])
@pytest.mark.parametrize("window", [0, 1333])
@pytest.mark.parametrize("q_kind,out_kind", [(np.float16, np.float16), (np.float32, np.float32)])
def test_prefill_of_few_rows_behind_many_keys(ctx, D, page, kvh, ratio, window, q_kind, out_kind):
    """Row tiles whose keys are cut into pieces; some see less than there are pieces."""
    attend_case(ctx, D, page, kvh, ratio, [6001, 2111, 40, 5], [60, 7, 33, 5], window, q_kind, out_kind, prefill=True)


def test_prefill_over_pieces_without_pages(ctx):
    """Pieces none of whose keys has a page, in front, in the middle and everywhere; lengths below the number of new tokens."""
    rng = np.random.default_rng(13)
    D, page, kvh, ratio, pages = 128, 64, 1, 4, 70
    cache = Cache(ctx, pages, kvh, page, D, 3)
    lengths, new = [4000, 4000, 4000, 3], [40, 40, 40, 9]
    table = rng.integers(0, pages, (4, 63)).astype(np.uint32)
    table[0, :30] = 0xFFFFFFFF
    table[1, 20:50] = pages
    table[2, :] = 0xFFFFFFFF
    starts = np.concatenate([[0], np.cumsum(new)])
    q = rng.standard_normal((int(starts[-1]), kvh * ratio, D)).astype(np.float16)
    got = run_attend(ctx, cache, q, np.float16, table, starts, lengths, 0, 0.1, np.float32, 40, True)
    want, size, vmax = ref.attend(q.astype(np.float64), cache.k, cache.ks, cache.v, cache.vs, table, starts, lengths, 0, 0.1, page)
    assert np.all(np.abs(got - want) <= attention_bound(want, size, vmax, D, 4000, False, True))
    assert np.all(got[80:120] == 0) and np.all(got[120:126] == 0)


@pytest.mark.parametrize("requests", [128, 129])
def test_prefill_of_many_requests(ctx, requests):
    """Up to 128 requests are ordered by their lengths; idle ones among them."""
    rng = np.random.default_rng(requests)
    lengths, new = rng.integers(20, 700, requests), rng.integers(0, 20, requests)
    attend_case(ctx, 64, 16, 1, 4, lengths.tolist(), new.tolist(), 0, np.float16, np.float32, prefill=True)


@pytest.mark.parametrize("kind,sizes", [(np.float16, (2.0**-20, 2.0**-10, 2.0**10)), (np.float32, (1e-30, 1e-8, 1e8, 1e30))])
def test_prefill_queries_of_any_size(ctx, kind, sizes):
    """f32 queries are scaled before they are rounded, f16 ones are taken as they are, those below the normal range among them."""
    D, page = 64, 16
    cache = Cache(ctx, 4, 1, page, D, 3)
    rng = np.random.default_rng(1)
    table = np.arange(4, dtype=np.uint32)[None]
    base = rng.standard_normal((3, 2, D)).astype(kind)
    for f in sizes:
        q = base * kind(f)
        scale = np.float32(1 / f)
        got = run_attend(ctx, cache, q, kind, table, [0, 3], [50], 0, scale, np.float32, 3, True)
        want, size, vmax = ref.attend(q.astype(np.float64), cache.k, cache.ks, cache.v, cache.vs, table, [0, 3], [50], 0, float(scale), page)
        bound = attention_bound(want, size, vmax, D, 50, False, True) + (2 * vmax * size * 2.0**-11 if kind == np.float32 else 0)
        assert np.all(np.abs(got - want) <= bound)


def test_prefill_gives_the_same_bits_and_shares_scratch(ctx):
    """Twice the same calls through one scratch, a decode step's between them."""
    scratch = ctx.zeros(max(ctx.paged_scratch_bytes(D) for D in (64, 128, 256, 512)))
    outs = []
    for _ in range(2):
        for D, kvh, lengths, new, prefill in ((128, 2, [5000, 300], [50, 200], True), (256, 1, [9000], [1], False), (512, 1, [3000], [9], True), (64, 2, [700] * 9, [70] * 9, True)):
            cache = Cache(ctx, 150, kvh, 64, D, 1)
            table = tables(np.random.default_rng(3), lengths, 64, 150, 150)
            q = np.random.default_rng(4).standard_normal((sum(new), kvh * 4, D)).astype(np.float32)
            outs.append(run_attend(ctx, cache, q, np.float32, table, np.concatenate([[0], np.cumsum(new)]), lengths, 0, 0.1, np.float32, max(new), prefill, scratch=scratch))
    for a, b in zip(outs[:4], outs[4:]):
        assert np.array_equal(a, b)


def test_two_contexts_at_once(ctx):
    """Two streams over the same cache, each with its own scratch, nothing waited for in between."""
    other = tb.Context(0)
    D, kvh, ratio, page = 128, 2, 4, 64
    cache = Cache(ctx, 80, kvh, page, D, 1)
    rng = np.random.default_rng(8)
    lengths, new = [5000, 700, 31], [70, 1, 31]
    table = words(ctx, tables(rng, lengths, page, 80, 80))
    starts, lens = words(ctx, np.concatenate([[0], np.cumsum(new)])), words(ctx, lengths)
    tokens, row = sum(new), kvh * ratio * D
    q = ctx.upload(rng.standard_normal((tokens, row)).astype(np.float16))
    ctx.sync()
    outs = []
    for c in (ctx, other):
        for prefill in (True, False):
            scratch = c.zeros(c.paged_scratch_bytes(D))
            most = max(new) if prefill else 2
            outs.append((c, prefill, [c.zeros(tokens * row * 4) for _ in range(6)], scratch, most))
        c.sync()
    for i in range(6):
        for c, prefill, out, scratch, most in outs:
            a = tb.PagedAttend(cache=cache.pages_of(table, 3, 80), q=q.ptr, q_dtype=tb.F16, q_stride=row, starts=starts.ptr, lengths=lens.ptr, tokens=tokens,
                               heads=kvh * ratio, most=most, window=0, scale=0.1, out=out[i].ptr, out_dtype=tb.F32, out_stride=row, scratch=scratch.ptr,
                               scratch_bytes=scratch.nbytes)
            (c.prefill_paged_q8 if prefill else c.attend_paged_q8)(a)
    got = [[o.download(np.uint32, tokens * row) for o in out] for _, _, out, _, _ in outs]
    for k in range(4):
        for x in got[k]:
            assert np.array_equal(x, got[k % 2][0])
    assert got[0][0].any() and got[1][0].any()


def test_prefill_needs_its_scratch(ctx):
    cache = Cache(ctx, 2, 1, 16, 64, 1)
    small = ctx.zeros(ctx.paged_scratch_bytes(64) - 16)
    with pytest.raises(tb.Error, match="tb_paged_scratch_bytes") as e:
        run_attend(ctx, cache, np.zeros((1, 1, 64), np.float32), np.float32, np.zeros((1, 1), np.uint32), [0, 1], [3], 0, 1.0, np.float32, 1, True, scratch=small)
    assert e.value.status == 3


# ---- logits ----------------------------------------------------------------------------------------------------------


def logits_case(ctx, rows, vocab, kind, history, biases, masked, seed=0, stride=None, offset=0, in_place=False, mask_of=None, without=()):
    rng = np.random.default_rng(seed + vocab)
    stride = stride or vocab
    x = (rng.standard_normal((rows, vocab)) * 4).astype(kind)
    x[0, : min(3, vocab)] = [np.inf, -np.inf, 0.0][: min(3, vocab)]
    flat = np.full(offset + rows * stride + 16, 77, kind)
    for r in range(rows):
        flat[offset + r * stride:][:vocab] = x[r]
    src = ctx.upload(flat)
    dst = src if in_place else ctx.upload(np.full(flat.size, 55, kind))
    size = np.dtype(kind).itemsize
    a = dict(logits=src.ptr + offset * size, out=dst.ptr + offset * size, dtype=tb.F32 if kind == np.float32 else tb.F16, rows=rows, vocab=vocab, stride=stride,
             out_stride=stride)
    keep, h, prompt, total, pen, bt, b, bc, allowed = [], None, None, None, {}, None, None, None, None
    if history:
        h = (rng.random((rows, history)) ** 3 * vocab * 1.02).astype(np.uint32)  # some past the vocabulary
        total = rng.integers(0, history + 1, rows)
        total[0] = history + 5  # past the list's end
        prompt = rng.integers(0, history + 1, rows)
        pen = {k: v for k, v in dict(repetition=rng.uniform(0.8, 1.5, rows), frequency=rng.uniform(-0.5, 0.5, rows), presence=rng.uniform(-0.5, 0.5, rows)).items()
               if k not in without}
        keep += [words(ctx, h), words(ctx, prompt), words(ctx, total)] + [ctx.upload(v.astype(np.float32)) for v in pen.values()]
        a |= dict(history=keep[0].ptr, prompt=keep[1].ptr, total=keep[2].ptr, history_stride=history) | {k: d.ptr for k, d in zip(pen, keep[3:])}
        pen = {k: v.astype(np.float32) for k, v in pen.items()}
    if biases:
        bt = rng.integers(0, vocab + vocab // 20 + 1, (rows, biases)).astype(np.uint32)
        bt[:, biases // 2:] = bt[:, : biases - biases // 2]  # tokens that come twice
        b, bc = rng.standard_normal((rows, biases)).astype(np.float32), rng.integers(0, biases + 1, rows)
        bc[0] = biases
        more = [words(ctx, bt), ctx.upload(b), words(ctx, bc)]
        keep += more
        a |= dict(bias_token=more[0].ptr, bias=more[1].ptr, bias_count=more[2].ptr, bias_stride=biases)
    if masked:
        nwords = -(-vocab // 32)
        allowed = rng.integers(0, 1 << 32, (masked, nwords + 1), dtype=np.uint64).astype(np.uint32)
        allowed[0] = 0  # lets nothing through
        keep.append(words(ctx, allowed))
        a |= dict(allowed=keep[-1].ptr, allowed_stride=nwords + 1, masks=masked)
        if mask_of is not None:
            keep.append(words(ctx, mask_of))
            a |= dict(mask_of=keep[-1].ptr)
    ctx.logits_adjust(tb.Logits(**a))
    got = dst.download(kind, flat.size)
    want = ref.logits(x, h, prompt, total, pen.get("repetition"), pen.get("frequency"), pen.get("presence"), bt, b, bc, allowed, mask_of)
    rest = np.full(flat.size, 77 if in_place else 55, kind)
    for r in range(rows):
        line = got[offset + r * stride:][:vocab].astype(np.float64)
        fine = np.isfinite(want[r])
        assert np.array_equal(line[~fine], want[r][~fine])
        # f32: a quotient, a fused product, a difference and the biases' sums, each 2^-24 of numbers below 64; then the type's own rounding.
        bound = 64 * (biases + 6) * 2.0**-24 + (np.abs(want[r][fine]) * 2.0**-11 + 2.0**-25 if kind == np.float16 else 0)
        assert np.all(np.abs(line[fine] - want[r][fine]) <= bound)
        rest[offset + r * stride:][:vocab] = got[offset + r * stride:][:vocab]
    assert np.array_equal(got, rest), "values outside the rows were written"


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("rows,vocab,history,biases,masked", [(1, 1, 1, 1, 1), (1, 33, 5, 40, 1), (3, 1000, 100, 7, 3), (2, 8191, 3000, 300, 2), (5, 32000, 17, 0, 5), (4, 8193, 0, 33, 0),
                                                              (1, 262144, 2000, 8, 1), (300, 1025, 64, 3, 300), (2, 50257, 0, 0, 2), (2, 4096, 900, 5, 0), (3, 999, 0, 0, 0)])
def test_logits(ctx, rows, vocab, history, biases, masked, kind):
    logits_case(ctx, rows, vocab, kind, history, biases, masked)


@pytest.mark.parametrize("kind", [np.float32, np.float16])
@pytest.mark.parametrize("stride,offset", [(1000, 0), (1003, 0), (1008, 1), (1016, 8)])
def test_logits_strides_in_place_and_partly_given(ctx, stride, offset, kind):
    logits_case(ctx, 4, 999, kind, 50, 9, 4, stride=stride, offset=offset)
    logits_case(ctx, 4, 999, kind, 50, 9, 4, stride=stride, offset=offset, in_place=True)
    logits_case(ctx, 4, 999, kind, 50, 0, 2, stride=stride, offset=offset, mask_of=[1, 0xFFFFFFFF, 0, 2], without=("frequency",))
    logits_case(ctx, 4, 999, kind, 50, 0, 0, stride=stride, offset=offset, without=("repetition", "presence"))
    logits_case(ctx, 4, 999, kind, 50, 0, 0, stride=stride, offset=offset, without=("repetition", "presence", "frequency"))


def test_logits_add_a_tokens_biases_in_the_lists_order(ctx):
    """2^25, 1 and -2^25 on one token, in orders that f32 tells apart; across the 32 lanes that read a stretch of the list and beyond."""
    for order, want in (([2.0**25, 1.0, -(2.0**25)], 0.0), ([2.0**25, -(2.0**25), 1.0], 1.0), ([1.0, 2.0**25, -(2.0**25)], 0.0)):
        for gap in (0, 1, 30, 40):
            token, bias = np.arange(100, 100 + 3 + 2 * gap, dtype=np.uint32), np.zeros(3 + 2 * gap, np.float32)
            token[[0, 1 + gap, 2 + 2 * gap]], bias[[0, 1 + gap, 2 + 2 * gap]] = 7, order
            bufs = [words(ctx, token), ctx.upload(bias), words(ctx, [len(token)]), ctx.zeros(4 * 300), ctx.zeros(4 * 300)]
            ctx.logits_adjust(tb.Logits(logits=bufs[3].ptr, out=bufs[4].ptr, dtype=tb.F32, rows=1, vocab=300, stride=300, out_stride=300, bias_token=bufs[0].ptr,
                                        bias=bufs[1].ptr, bias_count=bufs[2].ptr, bias_stride=len(token)))
            assert bufs[4].download(np.float32, 300)[7] == want


def test_logits_of_a_history_picked_against_the_tables(ctx):
    """Tokens that all fall to one block by its hash, more of them than its table holds: those without room are worked out one by one."""
    rng = np.random.default_rng(5)
    vocab, want = 1 << 20, 9000
    t = np.arange(vocab, dtype=np.uint64)
    top = ((t * 0x9E3779B1) & 0xFFFFFFFF) >> 16
    picked = np.concatenate([t[top < 700][:want], t[top < 700][:300]]).astype(np.uint32)  # the smallest hashes: the first block's of up to 93; some twice
    assert len(picked) == want + 300
    rng.shuffle(picked)
    x = rng.standard_normal((1, vocab)).astype(np.float32)
    bias_token, bias = picked[None, :50].copy(), rng.standard_normal((1, 50)).astype(np.float32)
    n = len(picked)
    bufs = [ctx.upload(x), ctx.zeros(4 * vocab), words(ctx, picked), words(ctx, [4000]), words(ctx, [n])] + [ctx.upload(np.array([v], np.float32)) for v in (1.3, 0.2, 0.1)]
    bufs += [words(ctx, bias_token), ctx.upload(bias), words(ctx, [50])]
    ctx.logits_adjust(tb.Logits(logits=bufs[0].ptr, out=bufs[1].ptr, dtype=tb.F32, rows=1, vocab=vocab, stride=vocab, out_stride=vocab, history=bufs[2].ptr, history_stride=n,
                                prompt=bufs[3].ptr, total=bufs[4].ptr, repetition=bufs[5].ptr, frequency=bufs[6].ptr, presence=bufs[7].ptr, bias_token=bufs[8].ptr,
                                bias=bufs[9].ptr, bias_count=bufs[10].ptr, bias_stride=50))
    f = lambda v: np.array([v], np.float32)  # noqa: E731
    y = ref.logits(x, picked[None], [4000], [n], f(1.3), f(0.2), f(0.1), bias_token, bias, [50], None, None)
    assert np.abs(bufs[1].download(np.float32, vocab)[None] - y).max() <= 64 * 8 * 2.0**-24


def test_logits_with_long_histories_and_a_step_before_that_writes_them(ctx):
    """In place and without a mask only the tokens' kernel runs, right behind a kernel that has written its lists."""
    rng = np.random.default_rng(6)
    rows, vocab, n = 3, 5000, 20000
    h = rng.integers(0, vocab, (rows, n)).astype(np.uint32)
    x = rng.standard_normal((rows, vocab)).astype(np.float32)
    src, dst = ctx.upload(x), ctx.upload(x)
    hd, old = words(ctx, h), words(ctx, np.zeros((rows, n)))
    keep = [words(ctx, [100, 0, n]), words(ctx, [n, n - 7, n]), ctx.upload(np.array([1.1, 1.2, 1.3], np.float32)), ctx.upload(np.array([0.01, 0.02, 0.03], np.float32))]
    # the lists arrive on the stream right before the call, as uint32 "values" through the stream kernel of an unmasked call
    ctx.logits_adjust(tb.Logits(logits=hd.ptr, out=old.ptr, dtype=tb.F32, rows=rows, vocab=n, stride=n, out_stride=n))
    ctx.logits_adjust(tb.Logits(logits=dst.ptr, out=dst.ptr, dtype=tb.F32, rows=rows, vocab=vocab, stride=vocab, out_stride=vocab, history=old.ptr, history_stride=n,
                                prompt=keep[0].ptr, total=keep[1].ptr, repetition=keep[2].ptr, frequency=keep[3].ptr))
    y = ref.logits(x, h, [100, 0, n], [n, n - 7, n], np.array([1.1, 1.2, 1.3], np.float32), np.array([0.01, 0.02, 0.03], np.float32), None, None, None, None, None, None)
    assert np.abs(dst.download(np.float32, x.size).reshape(x.shape) - y).max() <= 64 * 8 * 2.0**-24
    assert src is not None


# ---- together --------------------------------------------------------------------------------------------------------


def test_a_serving_loop(ctx):
    """Five requests through a chunk of prompt, steps of single tokens, one ending and one joining: plan, append, attend, a projection
    to logits (tb_gemm_f16), penalties, and the pick (tb_sample_greedy), all queued without the host reading anything between; every step
    against the restatements."""
    rng = np.random.default_rng(21)
    D, page, kvh, ratio, n, width, pages, vocab = 64, 16, 2, 4, 5, 12, 40, 512
    heads = kvh * ratio
    cache = Cache(ctx, pages, kvh, page, D, 9, fill=False)
    table, free, count = np.zeros((n, width), np.uint32), rng.permutation(pages).astype(np.uint32), pages
    lengths = np.zeros(n, np.uint32)
    most = 40
    maxt = n * most
    d = {k: words(ctx, v) for k, v in dict(lengths=lengths, table=table, free=free, count=[count], starts=np.zeros(n + 1), slots=np.zeros(maxt), positions=np.zeros(maxt),
                                            refused=[0], scratch=[0]).items()}
    scratch, out = ctx.zeros(ctx.paged_scratch_bytes(D)), ctx.zeros(maxt * heads * D * 2)
    head_w = (rng.standard_normal((vocab, heads * D)) * 0.05).astype(np.float16)
    wd, logit, adj = ctx.upload(head_w), ctx.zeros(maxt * vocab * 4), ctx.zeros(maxt * vocab * 4)
    penalties = [ctx.upload(np.full(maxt, x, np.float32)) for x in (1.2, 0.3, 0.1)]
    steps = [[40, 17, 1, 0, 33], [1, 1, 1, 5, 1], [1, ENDS, 1, 1, 0], [1, 20, 1, 1, 1], [1, 1, ENDS, 1, 1], [1, 1, 3, 1, 1]]
    scale = 0.125
    for fresh in steps:
        fresh = np.array(fresh, np.uint32)
        new = [0 if f == ENDS else int(f) for f in fresh]
        tokens = sum(new)
        k, v = rng.standard_normal((tokens, kvh, D)).astype(np.float32), rng.standard_normal((tokens, kvh, D)).astype(np.float32)
        q = (rng.standard_normal((tokens, heads, D)) * 2).astype(np.float16)
        hist = rng.integers(0, vocab, (tokens, 30)).astype(np.uint32)
        fd, kd, vd, qd, hd = words(ctx, fresh), ctx.upload(k), ctx.upload(v), ctx.upload(q), words(ctx, hist)
        zeros, thirty = words(ctx, np.full(tokens, 10)), words(ctx, np.full(tokens, 30))
        pick, state = ctx.zeros(16), ctx.zeros(8)
        ctx.page_plan(tb.PagePlan(lengths=d["lengths"].ptr, fresh=fd.ptr, lengths_out=d["lengths"].ptr, table=d["table"].ptr, free_pages=d["free"].ptr,
                                  free_count=d["count"].ptr, free_count_out=d["count"].ptr, starts=d["starts"].ptr, slots=d["slots"].ptr, positions=d["positions"].ptr,
                                  refused=d["refused"].ptr, scratch=d["scratch"].ptr, requests=n, width=width, page=page, pages=pages, max_tokens=maxt))
        ctx.cache_append_q8(tb.CacheRows(cache=cache.pages_of(), k=kd.ptr, v=vd.ptr, dtype=tb.F32, token_stride=kvh * D, head_stride=D, slots=d["slots"].ptr, tokens=tokens))
        prefill = max(new) > 8
        attend = tb.PagedAttend(cache=cache.pages_of(d["table"], n, width), q=qd.ptr, q_dtype=tb.F16, q_stride=heads * D, starts=d["starts"].ptr, lengths=d["lengths"].ptr,
                                tokens=tokens, heads=heads, most=max(new), window=0, scale=scale, out=out.ptr, out_dtype=tb.F16, out_stride=heads * D, scratch=scratch.ptr,
                                scratch_bytes=scratch.nbytes)
        (ctx.prefill_paged_q8 if prefill else ctx.attend_paged_q8)(attend)
        ctx.gemm_f16(wd, out, tokens, vocab, heads * D, logit, 0)
        ctx.logits_adjust(tb.Logits(logits=logit.ptr, out=adj.ptr, dtype=tb.F32, rows=tokens, vocab=vocab, stride=vocab, out_stride=vocab, history=hd.ptr, history_stride=30,
                                    prompt=zeros.ptr, total=thirty.ptr, repetition=penalties[0].ptr, frequency=penalties[1].ptr, presence=penalties[2].ptr))
        ctx.sample_greedy(adj, vocab, 0.0, 1.0, None, None, pick, state)

        want = ref.plan(lengths, fresh, table, free, count, page, pages, maxt)
        assert want["refused"] == 0 and d["refused"].download(np.uint32, 1)[0] == 0
        lengths, table, free, count = want["lengths"], want["table"], want["free"], want["count"]
        assert np.array_equal(d["lengths"].download(np.uint32, n), lengths) and np.array_equal(d["table"].download(np.uint32, table.size).reshape(table.shape), table)
        ref.append(cache.k, cache.ks, k, want["slots"], page)
        ref.append(cache.v, cache.vs, v, want["slots"], page)
        cache.check()
        o, size, vmax = ref.attend(q.astype(np.float64), cache.k, cache.ks, cache.v, cache.vs, table, want["starts"], lengths, 0, scale, page)
        got = out.download(np.float16, tokens * heads * D).reshape(tokens, heads, D)
        assert np.all(np.abs(got - o) <= attention_bound(o, size, vmax, D, int(lengths.max()), True, prefill))
        x = got.reshape(tokens, -1).astype(np.float64) @ head_w.astype(np.float64).T
        y = ref.logits(x, hist, np.full(tokens, 10), np.full(tokens, 30), np.full(tokens, np.float32(1.2)), np.full(tokens, np.float32(0.3)), np.full(tokens, np.float32(0.1)),
                       None, None, None, None, None)
        a = adj.download(np.float32, tokens * vocab).reshape(tokens, vocab)
        terms = np.abs(got.reshape(tokens, -1).astype(np.float64)) @ np.abs(head_w.astype(np.float64)).T
        assert np.all(np.abs(a - y) <= 1.2 * (1e-5 * terms + 1e-6) + 64 * 8 * 2.0**-24)
        assert state.download(np.uint32, 2)[1] == int(np.argmax(a[0]))
