"""Attention over the paged cache against the softmax in 64 bits, at the sizes and masks where it can go wrong."""
import numpy as np
import pytest

import fixtures as fx
import serving_ref as sr
from smelt_amd import compiler as cc
from smelt_amd import runtime as rt

pytestmark = pytest.mark.gpu
B = cc.bind
ACT = {fx.F16: rt.ACT_F16, fx.BF16: rt.ACT_BF16}


@pytest.fixture(scope="module")
def ctx():
    c = rt.Context()
    yield c
    c.close()


class Case:
    """Operands in slots 1.. of a batch: new tokens n, own keys L (new ones included), a prefix."""

    def __init__(self, ctx, dtype, n, L, heads, kv_heads, dim, page, prefix=0, window=0, pad=0, gap=0, scale=None, seed=0, poison=True, width=None):
        self.__dict__.update(locals())
        rng = fx.rng_for(220, seed + dim + page + sum(L))
        self.sequences = len(n)
        self.offsets = np.concatenate([[0], np.cumsum(n)]).astype(np.int32)
        self.tokens = int(self.offsets[-1]) + pad
        used = [-(-l // page) for l in L]
        front = -(-prefix // page)
        self.width = width or max(1, max(used))
        self.pages = sum(used) + front + 2
        order = rng.permutation(self.pages)
        self.prefix_pages = order[:front].astype(np.int32)
        self.table = np.full((self.sequences, self.width), 2 ** 30, np.int32)       # entries behind a sequence's end name no page
        at = front
        for s, u in enumerate(used):
            self.table[s, :u] = order[at:at + u]
            at += u
        self.qb, q = sr.values(rng, (self.tokens, heads * dim + gap), dtype, 2.0)
        kb, k = sr.values(rng, (self.pages, kv_heads, page, dim), dtype)
        vb, v = sr.values(rng, (self.pages, kv_heads, page, dim), dtype)
        self.kb, self.vb = kb, vb
        if poison:       # infinities and NaN wherever no sequence has written
            owned = np.zeros((self.pages, page), bool)
            for j in range(prefix):
                owned[self.prefix_pages[j // page], j % page] = True
            for s, l in enumerate(L):
                for j in range(l):
                    owned[self.table[s, j // page], j % page] = True
            bad = np.array([0x7E00, 0x7C00, 0xFC00] if dtype == fx.F16 else [0x7FC0, 0x7F80, 0xFF80], np.uint16)
            for x in (kb, vb):
                free = ~owned[:, None, :, None] & np.ones(x.shape, bool)
                x[free] = bad[rng.integers(0, 3, int(free.sum()))]
        self.q = q[:, :heads * dim].reshape(self.tokens, heads, dim)
        self.lens = np.array(L, np.int32)
        self.scale = 1.0 / np.sqrt(dim) if scale is None else scale
        self.out0 = rng.integers(0, 30000, (self.tokens, heads * dim)).astype(np.uint16)

    def load(self):
        c = self.ctx
        c.put(1, self.qb); c.put(2, sr.keys_to_pages(self.kb, self.page)); c.put(3, self.vb); c.put(4, self.table); c.put(5, self.lens); c.put(6, self.offsets)
        c.put(7, self.out0)
        if self.prefix:
            c.put(8, self.prefix_pages); c.put(9, np.array([self.prefix], np.int32))
        em = cc.Emitter(act_dtype=ACT[self.dtype])
        shared = dict(prefix_table=B(8), prefix_len=B(9), prefix_pages=len(self.prefix_pages)) if self.prefix else {}
        em.paged_attention(B(1), B(2), B(3), B(4), B(5), B(6), B(7), self.tokens, self.sequences, self.heads, self.kv_heads, self.dim, self.page, self.pages, self.width,
                           self.scale, window=self.window, q_stride=self.heads * self.dim + self.gap, **shared)
        return em.table_for(c)

    def result(self):
        return self.ctx.read(7, np.uint16, self.out0.size).reshape(self.out0.shape)

    def want(self):
        k, v = sr.wide(self.kb, self.dtype), sr.wide(self.vb, self.dtype)
        return sr.attention(self.q, k, v, self.pages, self.table, self.lens, self.offsets, float(np.float32(self.scale)), self.window, self.prefix_pages, self.prefix)

    def check(self, got):
        y, reach, sharp, count = self.want()
        live = int(self.offsets[-1])
        assert np.array_equal(got[live:], self.out0[live:])                        # rows behind the last sequence
        tol = sr.attention_tolerance(y, reach, sharp, count, self.dim, self.dtype)[:live]
        g = sr.wide(got[:live], self.dtype).reshape(y[:live].shape)
        assert np.array_equal(np.isnan(g), np.isnan(y[:live])) and np.isfinite(g).all()
        off = np.abs(g - y[:live])
        assert np.all(off <= tol), f"{(off / tol).max():.2f} of the tolerance at {np.unravel_index((off / tol).argmax(), off.shape)}"

    def run(self):
        table = self.load()
        self.ctx.interpret_decode(table)
        self.ctx.wait()
        self.check(self.result())
        return self


TYPES = pytest.mark.parametrize("dtype", [fx.F16, fx.BF16], ids=["f16", "bf16"])


@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_one_token_a_sequence(ctx, dtype, dim, page):
    Case(ctx, dtype, [1] * 7, [1, 2, 31, 32, 33, 300, 65], 6, 2, dim, page, pad=2, gap=8).run()


@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("prefix", [1, 40, 200])
def test_shared_prefix(ctx, dtype, dim, page, prefix):
    Case(ctx, dtype, [1, 0, 4, 1, 7], [1, 50, 4, 90, 33], 12, 2, dim, page, prefix=prefix, pad=1).run()


@TYPES
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (5, 1), (8, 8), (24, 4), (33, 1), (64, 2)])
def test_head_layouts(ctx, dtype, heads, kv_heads):
    Case(ctx, dtype, [1, 3, 2], [70, 3, 129], heads, kv_heads, 64, 32, prefix=45).run()


@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page,prefix", [(16, 0), (64, 0), (16, 37), (64, 100), (256, 0)])
def test_prompts(ctx, dtype, dim, page, prefix):
    """Many rows a sequence, behind earlier keys and from nothing."""
    Case(ctx, dtype, [75, 1, 40], [75, 20, 161], 4, 2, dim, page, prefix=prefix).run()


@TYPES
@pytest.mark.parametrize("window", [1, 5, 32, 100])
@pytest.mark.parametrize("prefix", [0, 90])
def test_windows(ctx, dtype, window, prefix):
    """Rows that see no prefix, part of it, one key."""
    Case(ctx, dtype, [1, 9, 1, 50], [1, 30, 200, 64], 4, 2, 64, 16, prefix=prefix, window=window).run()


@TYPES
@pytest.mark.parametrize("prefix", [0, 20])
def test_rows_that_see_nothing(ctx, dtype, prefix):
    """No keys at all; fewer keys than new rows (the first rows stand before key 0)."""
    c = Case(ctx, dtype, [2, 5, 1], [0, 2, 3], 4, 2, 64, 16, prefix=prefix).run()
    if not prefix:
        assert not c.result()[:2].any() and not c.result()[2:5].any()


@TYPES
def test_long_and_short_together(ctx, dtype):
    """One sequence holds most of the keys: its segments are cut over many workgroups and joined."""
    Case(ctx, dtype, [1, 2, 1, 1], [17, 9000, 1, 64], 4, 2, 128, 64, prefix=0, seed=3).run()
    Case(ctx, dtype, [1, 2], [17, 90], 2, 1, 256, 64, prefix=6000, seed=4).run()


@TYPES
def test_many_sequences(ctx, dtype):
    """More sequences than a workgroup has threads, some without rows."""
    rng = fx.rng_for(221, 0)
    n = rng.integers(0, 3, 300)
    L = np.maximum(rng.integers(0, 60, 300), n)
    Case(ctx, dtype, n.tolist(), L.tolist(), 2, 1, 64, 16, prefix=33, pad=3).run()


@TYPES
@pytest.mark.parametrize("scale", [0.0, -0.2, 3.0])
def test_scales(ctx, dtype, scale):
    Case(ctx, dtype, [1, 4], [40, 100], 4, 2, 64, 32, scale=scale, prefix=17).run()


def test_odd_row_strides_of_q(ctx):
    Case(ctx, fx.F16, [1, 3], [40, 70], 3, 3, 64, 32, gap=3).run()


@TYPES
def test_pages_outside_the_pool_are_not_seen(ctx, dtype):
    """A table entry that names no page of the pool hides its keys: the result is the one without them."""
    for page, hidden in ((16, -1), (64, 2 ** 30)):
        c = Case(ctx, dtype, [1, 2], [200, 150], 4, 2, 64, page, prefix=2 * page + 5)
        c.table[0, 1] = hidden
        c.prefix_pages[1] = hidden
        c.run()


def test_lengths_are_cut_to_what_the_tables_hold(ctx):
    c = Case(ctx, fx.F16, [1, 1], [64, 50], 2, 1, 64, 16, prefix=32)
    want = c.load()
    c.ctx.interpret_decode(want); c.ctx.wait()
    first = c.result().copy()
    c.ctx.put(5, np.array([1 << 30, 50], np.int32)); c.ctx.put(9, np.array([1 << 30], np.int32))
    c.ctx.interpret_decode(want); c.ctx.wait()
    assert np.array_equal(c.result()[0], first[0])
    c.ctx.put(5, np.array([-5, 50], np.int32)); c.ctx.put(9, np.array([-1], np.int32))
    c.ctx.interpret_decode(want); c.ctx.wait()
    assert not c.result()[0].any() and c.result()[1].any()


def test_infinities_and_nans_that_are_seen(ctx):
    """A NaN score makes its rows NaN and no others; a score of -inf is a key that is not seen."""
    c = Case(ctx, fx.BF16, [1, 1, 1], [40, 60, 33], 2, 1, 64, 32)
    at = lambda s, j: (c.table[s, j // 32], 0, j % 32)   # noqa: E731
    c.kb[at(0, 5)] = 0x7FC0
    c.kb[at(2, 7)] = 0
    c.kb[at(2, 7)][0] = 0xFF80                             # q0 * -inf
    sign = c.qb[2, :].reshape(2, 64)[:, 0]
    assert np.all(sr.wide(sign, fx.BF16) != 0)
    c.qb[2, 0::64] &= 0x7FFF                               # q0 positive: the score is -inf
    c.q = sr.wide(c.qb, fx.BF16).reshape(3, 2, 64)
    t = c.load()
    c.ctx.interpret_decode(t); c.ctx.wait()
    g = sr.wide(c.result(), fx.BF16)
    assert np.isnan(g[0]).all() and np.isfinite(g[1:]).all()
    y, reach, sharp, count = c.want()
    tol = sr.attention_tolerance(y, reach, np.where(np.isfinite(sharp), sharp, 20.0), count, 64, fx.BF16)
    assert np.all(np.abs(g[1:].reshape(2, 2, 64) - y[1:]) <= tol[1:])


def test_the_same_inputs_give_the_same_bits(ctx):
    c = Case(ctx, fx.BF16, [1, 5, 3, 1], [700, 2000, 64, 1], 8, 2, 128, 64, prefix=900)
    t = c.load()
    c.ctx.interpret_decode(t); c.ctx.wait()
    first = c.result().copy()
    for _ in range(3):
        c.ctx.interpret_decode(t)
    c.ctx.wait()
    assert np.array_equal(first, c.result())


def test_attention_is_refused_where_a_slot_is_short(ctx):
    c = Case(ctx, fx.F16, [1, 2], [40, 70], 4, 2, 64, 16, prefix=20)
    c.load()

    def go(**kw):
        a = dict(q=B(1), k_cache=B(2), v_cache=B(3), page_table=B(4), kv_lens=B(5), offsets=B(6), out=B(7), tokens=3, sequences=2, heads=4, kv_heads=2, head_dim=64, page_size=16,
                 pages=c.pages, pages_per_sequence=c.width, scale=0.1, prefix_table=B(8), prefix_len=B(9), prefix_pages=2)
        em = cc.Emitter()
        em.paged_attention(**{**a, **kw})
        return ctx.interpret_decode(em.table_for(ctx))

    assert go() >= 1 and go(tokens=0) == 0 and go(sequences=0) == 0
    for kw in (dict(tokens=4), dict(pages=c.pages + 1), dict(pages_per_sequence=c.width + 1), dict(sequences=3), dict(prefix_pages=3), dict(out=B(7, 16)), dict(kv_lens=B(5, 4)),
               dict(q_stride=512), dict(k_cache=B(2, 16))):
        with pytest.raises(rt.SmeltHipError, match="needs"):
            go(**kw)
    with pytest.raises(rt.SmeltHipError, match="aligned"):
        go(tokens=1, sequences=1, out=B(7, 2))
    ctx.wait()


def bad_values(case, at, dims):
    """Infinities and NaN among the values of sequence s's own keys at[s], in `dims`."""
    bad = np.array([0x7C00, 0x7E00, 0xFC00] if case.dtype == fx.F16 else [0x7F80, 0x7FC0, 0xFF80], np.uint16)
    for s, keys in enumerate(at):
        for n, j in enumerate(keys):
            page, off = case.table[s, j // case.page], j % case.page
            for m, d in enumerate(dims):
                case.vb[page, :, off, d] = bad[(n + m) % 3]


def check_where_finite(case, got):
    """The result is not finite exactly where the rows that see such a value say so, and right everywhere else."""
    y, reach, sharp, count = case.want()
    live = int(case.offsets[-1])
    tol = sr.attention_tolerance(y, np.where(np.isfinite(reach), reach, 0.0), sharp, count, case.dim, case.dtype)[:live]
    g, y = sr.wide(got[:live], case.dtype).reshape(y[:live].shape), y[:live]
    assert np.array_equal(np.isnan(g), np.isnan(y))
    assert np.array_equal(np.isposinf(g), np.isposinf(y)) and np.array_equal(np.isneginf(g), np.isneginf(y))
    ok = np.isfinite(y)
    assert ok.any() and not ok.all()
    assert np.all(np.abs(g - y)[ok] <= tol[ok])


# rows a sequence: one row tile of 16, of 32, the kernel for many rows; the prefix apart, and with the own keys
@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,prefix", [([3, 2], 0), ([8, 5], 0), ([70, 33], 0), ([3, 2], 45), ([70, 33], 45)])
@pytest.mark.parametrize("window", [0, 40])
def test_infinities_in_keys_that_only_some_rows_see(ctx, dtype, dim, n, prefix, window):
    c = Case(ctx, dtype, n, [n[0] + 90, n[1] + 31], 8, 2, dim, 16, prefix=prefix, window=window, poison=False)
    ends = [int(c.lens[s]) for s in range(2)]
    bad_values(c, [[ends[0] - 1, ends[0] - 2], [ends[1] - 1]], [0, 5, dim - 1])
    table = c.load()
    c.ctx.interpret_decode(table)
    c.ctx.wait()
    check_where_finite(c, c.result())


@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 40])
def test_infinities_in_keys_before_every_rows_window(ctx, dtype, dim, n):
    c = Case(ctx, dtype, [n], [n + 100], 4, 2, dim, 64, window=9, poison=False)
    bad_values(c, [[100 - 9, 100 - 12]], range(dim))       # (the first row's position is 100: it sees keys 92 on)
    c.run()


# the prefix's segments in six parts each (two for every compute unit), and whole (too short to be cut)
@pytest.mark.parametrize("tokens,heads,kv_heads,prefix", [(600, 32, 4, 1700), (300, 64, 64, 200)])
def test_a_prefix_behind_many_sequences(ctx, tokens, heads, kv_heads, prefix):
    Case(ctx, fx.BF16, [1] * tokens, [1 + s % 5 for s in range(tokens)], heads, kv_heads, 64, 64, prefix=prefix, pad=3).run()


@pytest.mark.parametrize("n", [1, 70])
def test_caches_past_four_gigabytes(n):
    """Pages beyond 2^32 bytes and 2^31 values into keys and values, put away and read."""
    dim, kv, heads, page, pages, own = 256, 8, 16, 256, 4200, 300
    places = np.array([4199, 3, 4198], np.int32)
    rng = fx.rng_for(230, n)
    kb, k = sr.values(rng, (own, kv, dim), fx.BF16)
    vb, v = sr.values(rng, (own, kv, dim), fx.BF16)
    qb, q = sr.values(rng, (n, heads, dim), fx.BF16, 2.0)
    j = np.arange(own)
    ctx = rt.Context()
    try:
        ctx.put(1, kb); ctx.put(2, vb); ctx.put(3, j.astype(np.int32)); ctx.put(4, (places[j // page] * page + j % page).astype(np.int32)); ctx.put(5, np.zeros(1))
        ctx.alloc(6, pages * page * kv * dim * 2); ctx.alloc(7, pages * page * kv * dim * 2)
        ctx.put(8, qb); ctx.put(9, places); ctx.put(10, np.array([own], np.int32)); ctx.put(11, np.array([0, n], np.int32)); ctx.alloc(12, n * heads * dim * 2)
        em = cc.Emitter(act_dtype=ACT[fx.BF16])
        em.paged_kv_append(B(1), B(2), B(3), B(4), B(5), B(6), B(7), own, kv, dim, 0, page, pages)
        em.paged_attention(B(8), B(6), B(7), B(9), B(10), B(11), B(12), n, 1, heads, kv, dim, page, pages, len(places), dim ** -0.5)
        ctx.interpret_decode(em.table_for(ctx))
        ctx.wait()
        got = sr.wide(ctx.read(12, np.uint16, n * heads * dim), fx.BF16).reshape(n, heads, dim)
    finally:
        ctx.close()
    # the same sequence in a pool of two pages
    small = [np.zeros((2, kv, page, dim)) for _ in range(2)]
    for x, rows in zip(small, (k, v)):
        x[j // page, :, j % page] = rows
    y, reach, sharp, count = sr.attention(q, *small, 2, np.array([[0, 1]]), [own], [0, n], float(np.float32(dim ** -0.5)), 0, np.zeros(0, np.int32), 0)
    assert np.all(np.abs(got - y) <= sr.attention_tolerance(y, reach, sharp, count, dim, fx.BF16))


# (the reference's differences of 32-bit numbers overflow for rows before key 0, which see nothing either way)
@pytest.mark.filterwarnings("ignore:overflow encountered")
@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,own,prefix", [(80, 70, 0), (200, 190, 0), (60, 20, 0), (90, 70, 3), (20, 15, 0)])
def test_a_window_of_everything_hides_nothing(ctx, dtype, dim, n, own, prefix):
    """The widest window there is, with fewer keys than rows: the result of no window, bit for bit."""
    got = [Case(ctx, dtype, [n, 1], [own, 30], 2, 2, dim, 16, prefix=prefix, window=window).run().result() for window in (2 ** 31 - 1, 0)]
    assert np.array_equal(*got)


def timed(case, table, repeats=5):
    best = np.inf
    for _ in range(repeats):
        case.ctx.interpret_decode(table)
        case.ctx.wait()
        best = min(best, case.ctx.last_gpu_ns() / 1000.0)
    return best


# decoding and a prompt behind a few thousand keys: a row of NaN in q, or in a key that all rows see
@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,own,prefix", [([1, 1, 2], [3000, 40, 700], 0), ([1, 1, 2], [3000, 40, 700], 500), ([300, 70], [2500, 90], 0), ([300, 70], [2500, 90], 500)])
@pytest.mark.parametrize("where", ["q", "k"])
def test_rows_whose_scores_are_nan(ctx, dtype, dim, n, own, prefix, where):
    """They are NaN, the other rows are as they were bit for bit, and the batch takes as long as it did (a row formed a second time takes
    hundreds of times as long)."""
    c = Case(ctx, dtype, n, own, 8, 2, dim, 64, prefix=prefix, poison=False)
    table = c.load()
    clean = timed(c, table)
    before = c.result().copy()
    nan = 0x7E00 if dtype == fx.F16 else 0x7FC0
    if where == "q":
        c.qb[:n[0]] = nan
    else:
        c.kb[c.table[0, 0], :, 2] = nan
    table = c.load()
    took = timed(c, table)
    got, rows = c.result(), slice(0, n[0])
    assert np.isnan(sr.wide(got[rows], dtype)).all()
    assert np.array_equal(got[n[0]:], before[n[0]:])
    assert took < 3 * clean + 50, f"{took:.0f} us, {clean:.0f} before"


# decoding, drafts and a prompt behind a few thousand keys: NaN among the values of a key that all rows see
@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,own,prefix", [([1, 1, 2], [3000, 40, 700], 0), ([5, 1, 2], [3000, 40, 700], 500), ([300, 70], [2500, 90], 0), ([300, 70], [2500, 90], 500)])
@pytest.mark.parametrize("dims", ["all", "one"])
def test_values_of_nan_that_all_rows_see(ctx, dtype, dim, n, own, prefix, dims):
    """The rows that see them say so, in those values; everything else is as it was bit for bit, and the batch does not take tens of times
    as long."""
    c = Case(ctx, dtype, n, own, 8, 2, dim, 64, prefix=prefix, poison=False)
    table = c.load()
    clean = timed(c, table)
    before = c.result().copy()
    c.vb[c.table[0, 0], :, 2, (slice(None) if dims == "all" else 5)] = 0x7E00 if dtype == fx.F16 else 0x7FC0
    table = c.load()
    took = timed(c, table)
    got = sr.wide(c.result(), dtype).reshape(-1, 8, dim)
    hit = np.zeros(got.shape, bool)
    hit[:n[0], :, (slice(None) if dims == "all" else 5)] = True
    assert np.array_equal(np.isnan(got), hit)
    assert np.array_equal(c.result().reshape(hit.shape)[~hit], before.reshape(hit.shape)[~hit])
    assert took < 8 * clean + 500, f"{took:.0f} us, {clean:.0f} before"


@TYPES
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 3, 60])
@pytest.mark.parametrize("bad", [0x7C00, 0xFC00])
def test_an_infinity_whose_probability_is_small(ctx, dtype, dim, n, bad):
    """exp(-20) is no number of fp16 next to the others, but times an infinity it is one."""
    c = Case(ctx, dtype, [n], [n + 80], 4, 2, dim, 16, scale=1.0, poison=False)
    c.qb[:] = 0
    c.qb[:, ::dim] = fx.to_bits(np.float32([1.0]), dtype)[0]
    c.q = sr.wide(c.qb, dtype).reshape(-1, 4, dim)
    c.kb[:] = 0
    at = (c.table[0, 1], slice(None), 7)
    c.kb[at][:, 0] = fx.to_bits(np.float32([-20.0]), dtype)[0]
    c.vb[at][:, 9] = bad if dtype == fx.F16 else (0x7F80 | bad & 0x8000)
    table = c.load()
    ctx.interpret_decode(table)
    ctx.wait()
    check_where_finite(c, c.result())


@TYPES
@pytest.mark.parametrize("dim,n,own,prefix", [(128, [4, 2], [5000, 300], 0), (256, [3, 1], [4000, 90], 700), (64, [90, 40], [3000, 200], 0), (128, [60, 33], [2000, 200], 600)])
def test_infinities_in_long_sequences(ctx, dtype, dim, n, own, prefix):
    """Segments that are cut over several workgroups, some parts of which are formed again."""
    c = Case(ctx, dtype, n, own, 8, 2, dim, 64, prefix=prefix, poison=False, seed=5)
    bad_values(c, [[own[0] - 1, own[0] - 2, 1700], [own[1] - 1]], [0, 5, dim - 1])
    table = c.load()
    ctx.interpret_decode(table)
    ctx.wait()
    check_where_finite(c, c.result())
    first = c.result().copy()
    ctx.interpret_decode(table)
    ctx.wait()
    assert np.array_equal(first, c.result())
