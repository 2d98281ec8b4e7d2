"""Verification of drafted tokens against the definition in 64 bits: tokens and counts have to be equal."""
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


def batch(rng, dtype, rows, vocab, given=False, pad=0, stride=None, greedy=(), near=1.0):
    offsets = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
    total, s = int(offsets[-1]) + pad, len(rows)
    stride = stride or vocab
    tb, t = sr.values(rng, (total, stride), dtype, 2.5)
    db = fx.to_bits((t + rng.normal(0, near, t.shape)).astype(np.float32), dtype)
    drafts = (t[:, :vocab] + 2 * rng.gumbel(size=(total, vocab))).argmax(1).astype(np.int32)
    temperature = rng.uniform(0.4, 1.5, s).astype(np.float32)
    temperature[list(greedy)] = 0.0
    for r in range(total):      # greedy drafts that are sometimes the largest logit
        if rng.random() < 0.5:
            drafts[r] = t[r, :vocab].argmax() if r < offsets[-1] and temperature[np.searchsorted(offsets[1:], r, side="right")] == 0 else drafts[r]
    return dict(offsets=offsets, target=tb, draft=None if given else db, drafts=drafts, ua=rng.random(total).astype(np.float32), us=rng.random(s).astype(np.float32),
                temperature=temperature, vocab=vocab, stride=stride, tokens=np.full(total, -7, np.int32), dtype=dtype)


def load(ctx, c, offset=0):
    ctx.put(1, np.concatenate([np.zeros(offset, np.uint16), c["target"].ravel()]))
    for slot, key in ((3, "drafts"), (4, "offsets"), (5, "ua"), (6, "us"), (7, "temperature"), (8, "tokens")):
        ctx.put(slot, c[key])
    ctx.put(9, np.full(len(c["us"]), -7, np.int32))
    draft = {}
    if c["draft"] is not None:
        ctx.put(2, c["draft"])
        draft = dict(draft=B(2))
    em = cc.Emitter(act_dtype=ACT[c["dtype"]])
    em.verify_drafts(B(1, 2 * offset), B(3), B(4), B(5), B(6), B(7), B(8), B(9), len(c["tokens"]), len(c["us"]), c["vocab"], stride=c["stride"], **draft)
    return em.table_for(ctx)


def result(ctx, c):
    return ctx.read(8, np.int32, len(c["tokens"])), ctx.read(9, np.int32, len(c["us"]))


def want(c):
    t = sr.wide(c["target"], c["dtype"])[:, :c["vocab"]]
    d = None if c["draft"] is None else sr.wide(c["draft"], c["dtype"])[:, :c["vocab"]]
    return sr.verify(t, d, c["drafts"], c["offsets"], c["ua"], c["us"], c["temperature"], c["tokens"])


def check(ctx, c, offset=0):
    ctx.interpret_decode(load(ctx, c, offset))
    ctx.wait()
    got, ref = result(ctx, c), want(c)
    assert np.array_equal(got[1], ref[1]), (got[1], ref[1])
    assert np.array_equal(got[0], ref[0]), np.flatnonzero(got[0] != ref[0])
    return got


TYPES = pytest.mark.parametrize("dtype", [fx.F16, fx.BF16], ids=["f16", "bf16"])


@TYPES
@pytest.mark.parametrize("given", [False, True], ids=["model", "given"])
@pytest.mark.parametrize("vocab,rows", [(1, [1, 2, 3]), (2, [4, 4, 1]), (7, [2] * 9), (1000, [1, 5, 0, 9, 3]), (2048, [3, 3]), (2049, [6]), (32000, [4, 1, 5, 0, 2, 8]), (151936, [5, 2])])
def test_verify(ctx, dtype, given, vocab, rows):
    rng = fx.rng_for(230, vocab + len(rows))
    for k in range(3):
        check(ctx, batch(rng, dtype, rows, vocab, given, pad=k, greedy=[0] if k == 1 else (range(len(rows)) if k == 2 else ()), near=(1.0, 0.2, 3.0)[k]))


def test_all_outcomes_occur(ctx):
    """Between them these batches take every draft, none and some of them."""
    c = batch(fx.rng_for(231, 1), fx.F16, [5] * 60, 500, near=0.3)
    _, counts = check(ctx, c)
    assert set(counts) >= {0, 1, 2, 4}
    c["ua"][:] = 0.0
    tokens, counts = check(ctx, c)
    assert np.all(counts == 4) and np.all(tokens >= 0)
    c["ua"][:] = np.float32(1.0 - 2.0 ** -24)
    c["draft"] = c["target"].copy()                      # p == q: u < 1 takes every draft
    _, counts = check(ctx, c)
    assert np.all(counts == 4)


def test_more_runs_than_threads(ctx):
    """A vocabulary whose runs the last launch walks in several rounds."""
    for given in (False, True):
        c = batch(fx.rng_for(242, int(given)), fx.F16, [2, 1], 540001, given=given)
        check(ctx, c)


@TYPES
def test_more_rows_than_waves(ctx, dtype):
    c = batch(fx.rng_for(232, 0), dtype, [40, 1, 13], 900, near=0.01)
    c["ua"] *= 0.5
    _, counts = check(ctx, c)
    assert counts[0] > 8


@TYPES
def test_odd_strides_and_offsets(ctx, dtype):
    c = batch(fx.rng_for(233, 0), dtype, [3, 4], 5001, stride=5005)
    check(ctx, c)
    check(ctx, c, offset=1)
    check(ctx, batch(fx.rng_for(233, 1), dtype, [3, 4], 5001, given=True, stride=5008))


@TYPES
@pytest.mark.parametrize("greedy", [False, True])
def test_masked_rows(ctx, dtype, greedy):
    """-inf logits (a grammar's mask), whole rows of them, the type's lowest value, NaN and +inf."""
    c = batch(fx.rng_for(234, 0), dtype, [3, 3, 3, 3, 3, 3], 3001, greedy=range(6) if greedy else ())
    ninf, pinf, nan, low = ((0xFC00, 0x7C00, 0x7E00, 0xFBFF) if dtype == fx.F16 else (0xFF80, 0x7F80, 0x7FC0, 0xFF7F))
    t, d = c["target"], c["draft"]
    t[0, 5:] = ninf; t[1, 10:2990] = ninf
    t[3, :] = ninf                                       # nothing may follow: no draft is taken, nothing is drawn
    t[6:9, 7:] = low
    t[9, 100:2000:7] = nan
    t[12, 77] = pinf; t[12, 2500] = pinf
    d[15:18, :] = ninf                                   # a draft model without weights
    c["drafts"][15] = 1
    tokens, counts = check(ctx, c)
    assert counts[1] == 0 and list(tokens[3:6]) == [-1, -1, -1]


def test_drafts_outside_the_vocabulary_are_refused(ctx):
    c = batch(fx.rng_for(235, 0), fx.F16, [3, 3, 3], 400, greedy=[2])
    c["drafts"][0], c["drafts"][3], c["drafts"][6] = -1, 400, 2 ** 31 - 1
    c["ua"][:] = 0
    _, counts = check(ctx, c)
    assert list(counts) == [0, 0, 0]
    c = batch(fx.rng_for(235, 1), fx.F16, [3, 3], 400, given=True)
    c["drafts"][0], c["drafts"][3] = -1, 70000
    assert list(check(ctx, c)[1]) == [0, 0]


def test_edges_of_the_random_numbers(ctx):
    """u_sample 0 draws the first token with a weight, the largest u below 1 one of the last; ties of the largest logit go to the lowest token."""
    for u in (0.0, 1.0 - 2.0 ** -24):
        c = batch(fx.rng_for(236, 0), fx.F16, [1, 2, 1], 6000)
        c["us"][:] = u
        check(ctx, c)
    c = batch(fx.rng_for(236, 1), fx.BF16, [1, 2], 6000, greedy=[0, 1])
    c["target"][0, 4321] = c["target"][0, 123] = c["target"][0, 5999] = fx.to_bits(np.float32([40.0]), fx.BF16)[0]
    c["target"][1, :] = 0
    c["target"][1, 7] = 0x8000                            # -0 equals 0
    c["drafts"][1] = 0
    tokens, counts = check(ctx, c)
    assert tokens[0] == 123 and list(counts) == [0, 1]


@pytest.mark.parametrize("temperature", [1e-30, 1e-3, 50.0, float("inf"), float("nan"), -1.0])
def test_temperatures(ctx, temperature):
    c = batch(fx.rng_for(237, 0), fx.F16, [2, 4], 1500)
    c["temperature"][:] = temperature
    if np.isinf(temperature):
        c["target"][0, 3:900] = 0xFC00
    check(ctx, c)


def test_the_same_inputs_give_the_same_tokens(ctx):
    c = batch(fx.rng_for(238, 0), fx.F16, [5] * 20, 32000)
    t = load(ctx, c)
    first = None
    for _ in range(4):
        ctx.interpret_decode(t); ctx.wait()
        got = result(ctx, c)
        assert first is None or all(np.array_equal(a, b) for a, b in zip(first, got))
        first = got


def test_verify_is_refused_where_a_slot_is_short(ctx):
    c = batch(fx.rng_for(239, 0), fx.F16, [2, 3], 100)
    load(ctx, c)

    def go(**kw):
        a = dict(target=B(1), draft=B(2), draft_tokens=B(3), offsets=B(4), u_accept=B(5), u_sample=B(6), temperature=B(7), tokens=B(8), counts=B(9), rows=5, sequences=2, vocab=100)
        em = cc.Emitter()
        em.verify_drafts(**{**a, **kw})
        return ctx.interpret_decode(em.table_for(ctx))

    assert go() >= 1 and go(rows=0) == 0 and go(sequences=0) == 0
    for kw in (dict(rows=6), dict(sequences=3), dict(vocab=101), dict(stride=130), dict(tokens=B(8, 4)), dict(counts=B(9, 4)), dict(u_sample=B(6, 4)), dict(draft=B(2, 2))):
        with pytest.raises(rt.SmeltHipError, match="needs"):
            go(**kw)
    ctx.wait()


@TYPES
@pytest.mark.parametrize("vocab", [500, 32000])
@pytest.mark.parametrize("flat", [False, True], ids=["normal", "flat"])
def test_a_draft_model_that_is_the_target_leaves_nothing_over(ctx, dtype, vocab, flat):
    """p == q, and a draft that is refused all the same (outside the vocabulary, masked in both rows, u_accept of 1): max(p - q, 0) is zero
    everywhere, so the token is drawn from p."""
    us = [0.0, 0.03, 0.2, 0.37, 0.5, 0.61, 0.8, 0.97, 1.0 - 2.0 ** -24]
    c = batch(fx.rng_for(243, vocab), dtype, [2] * len(us), vocab)
    if flat:
        c["target"][:] = fx.to_bits(np.float32([1.5]), dtype)[0]
    c["target"][:, 17] = 0xFC00 if dtype == fx.F16 else 0xFF80
    c["draft"] = c["target"].copy()
    c["us"][:] = us
    first = c["offsets"][:-1]
    for drafted, u in ((-1, 0.0), (vocab, 0.5), (17, 0.0), (40, 1.0)):
        c["drafts"][first] = drafted
        c["ua"][first] = u
        _, counts = check(ctx, c)
        assert not counts.any()


@TYPES
@pytest.mark.parametrize("vocab", [9, 400, 3000, 32000])
def test_what_a_certain_draft_leaves_over(ctx, dtype, vocab):
    """A looked-up draft that holds all but 2^-60 of the probability and is refused (u_accept of 1): the token is drawn from the others, however
    little they hold; from p where they hold nothing."""
    us = [0.0, 0.1, 0.25, 0.5, 0.77, 1.0 - 2.0 ** -24]
    c = batch(fx.rng_for(244, vocab), dtype, [2] * len(us), vocab, given=True)
    first = c["offsets"][:-1]
    for at in (0, 5, vocab - 1):
        for others in (1.0, 0.0):
            t = sr.wide(c["target"], dtype) - 60.0
            if not others:
                t[first] = -np.inf
            t[first, at] = 0.0
            c["target"] = fx.to_bits(t.astype(np.float32), dtype)
            c["temperature"][:], c["us"][:] = 1.0, us
            c["drafts"][first], c["ua"][first] = at, 1.0
            tokens, counts = check(ctx, c)
            assert not counts.any() and np.all((tokens[first] == at) == (others == 0.0))
            c = batch(fx.rng_for(244, vocab), dtype, [2] * len(us), vocab, given=True)
