"""Rotary positions against the formula in 64 bits."""
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


def run(ctx, dtype, x, positions, table, amplitude, heads, dim, rot, interleaved, x_stride, y_stride, in_place=False, offset=0):
    """x: bits [tokens, x_stride]; `offset` elements in front of the rows."""
    tokens = x.shape[0]
    ctx.put(1, np.concatenate([np.zeros(offset, np.uint16), x.ravel()]))
    ctx.put(3, positions.astype(np.int32)); ctx.put(4, table)
    if not in_place:
        ctx.put(2, np.full(tokens * y_stride + offset, 0x7FFF, np.uint16))    # (a NaN wherever nothing is written)
    out = 1 if in_place else 2
    em = cc.Emitter(act_dtype=ACT[dtype])
    em.rope(B(1, 2 * offset), B(out, 2 * offset), B(3), B(4), tokens, heads, dim, rot, interleaved=interleaved, amplitude=amplitude, x_stride=x_stride, y_stride=y_stride)
    assert ctx.interpret_decode(em.table_for(ctx)) == 1
    ctx.wait()
    return ctx.read(out, np.uint16, tokens * y_stride, offset=2 * offset).reshape(tokens, y_stride)


@pytest.mark.parametrize("dtype", [fx.F16, fx.BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("tokens,heads,dim,rot,gap,offset", [
    (1, 1, 64, 64, 0, 0), (1, 8, 256, 64, 0, 0), (7, 3, 128, 128, 8, 0), (65, 24, 256, 64, 40, 0), (5, 2, 100, 20, 0, 0), (3, 5, 80, 80, 3, 0),
    (2, 1, 2, 2, 0, 0), (33, 4, 128, 96, 0, 1), (9, 1, 1000, 402, 0, 0), (4500, 2, 64, 64, 0, 0), (2, 7, 72, 40, 0, 0)])
def test_rope(ctx, dtype, interleaved, tokens, heads, dim, rot, gap, offset):
    rng = fx.rng_for(200, tokens * dim + rot)
    stride = heads * dim + gap
    bits, x = sr.values(rng, (tokens, stride), dtype)
    positions = rng.integers(0, 1 << 20, tokens)
    positions[0] = 0
    positions[-1] = (1 << 31) - 1 if tokens > 2 else 131071
    table, _ = cc.rope_table(rot, base=500000.0)
    got = run(ctx, dtype, bits, positions, table[:rot // 2], 1.1386, heads, dim, rot, interleaved, stride, heads * dim + 2 * gap, offset=offset)
    want, reach = sr.rope(x[:, :heads * dim].reshape(tokens, heads, dim), positions, table, float(np.float32(1.1386)), rot, interleaved)
    rows = got[:, :heads * dim].reshape(tokens, heads, dim)
    sr.check_rope(rows, want, reach, dtype, "rope")
    assert np.array_equal(rows[..., rot:], bits[:, :heads * dim].reshape(tokens, heads, dim)[..., rot:])
    if gap:
        assert np.all(got[:, heads * dim:] == 0x7FFF)          # what lies between the rows is left alone


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("dim,rot", [(128, 128), (100, 20)])
def test_rope_in_place_equals_apart(ctx, interleaved, dim, rot):
    rng = fx.rng_for(201, dim)
    bits, _ = sr.values(rng, (19, 3 * dim), fx.BF16)
    positions = rng.integers(0, 5000, 19)
    table, _ = cc.rope_table(rot)
    a = run(ctx, fx.BF16, bits, positions, table, 1.0, 3, dim, rot, interleaved, 3 * dim, 3 * dim)
    b = run(ctx, fx.BF16, bits, positions, table, 1.0, 3, dim, rot, interleaved, 3 * dim, 3 * dim, in_place=True)
    assert np.array_equal(a, b)


def test_rope_is_refused_where_a_slot_is_short(ctx):
    ctx.alloc(1, 1000); ctx.alloc(2, 1000); ctx.alloc(3, 400); ctx.alloc(4, 256)

    def go(tokens, **kw):
        em = cc.Emitter()
        em.rope(kw.get("x", B(1)), kw.get("y", B(2)), kw.get("p", B(3)), kw.get("t", B(4)), tokens, 1, 64, 64)
        return ctx.interpret_decode(em.table_for(ctx))

    assert go(7) == 1 and go(0) == 0
    for kw, word in ((dict(tokens=8), "needs 1024 bytes"), (dict(tokens=7, x=B(1, 200)), "needs"), (dict(tokens=7, p=B(3, 380)), "needs"), (dict(tokens=7, t=B(4, 8)), "needs"),
                     (dict(tokens=1, p=B(3, 2)), "aligned"), (dict(tokens=1, x=B(1, 1)), "aligned"), (dict(tokens=1, t=B(9)), "no buffer")):
        with pytest.raises(rt.SmeltHipError, match=word):
            go(**kw)
    ctx.upload_weights(10, np.zeros(1000, np.uint8))
    with pytest.raises(rt.SmeltHipError, match="read-only"):
        go(1, y=B(10))
    ctx.wait()


def test_dynamic_rows_follow_the_sequence_length(ctx):
    rng = fx.rng_for(202, 1)
    bits, x = sr.values(rng, (12, 128), fx.F16)
    table, _ = cc.rope_table(64)
    positions = np.arange(12) + 100
    ctx.put(1, bits); ctx.put(2, np.zeros((12, 128), np.uint16)); ctx.put(3, positions.astype(np.int32)); ctx.put(4, table)
    em = cc.Emitter()
    em.rope(B(1), B(2), B(3), B(4), 12, 2, 64, 64, dynamic=True)
    t = em.table_for(ctx)
    assert ctx.interpret_prefill(t, seq_len=5) == 1 and ctx.interpret_prefill(t, seq_len=0) == 0
    ctx.wait()
    got = ctx.read(2, np.uint16, 12 * 128).reshape(12, 128)
    want, reach = sr.rope(x.reshape(12, 2, 64), positions, table, 1.0, 64, False)
    sr.check_rope(got[:5].reshape(5, 2, 64), want[:5], reach[:5], fx.F16, "five rows")
    assert not got[5:].any()
    with pytest.raises(rt.SmeltHipError, match="needs"):
        ctx.interpret_prefill(t, seq_len=13)
