"""Appending rotated keys and values to the paged cache; slots bound to the caller's memory."""
import ctypes as C

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


@pytest.mark.parametrize("dtype", [fx.F16, fx.BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("tokens,kv_heads,q_heads,dim,rot,page,pages,gap", [
    (1, 1, 0, 64, 64, 16, 1, 0), (1, 2, 8, 256, 64, 64, 5, 0), (64, 4, 24, 256, 64, 64, 40, 0), (37, 3, 6, 128, 128, 16, 9, 8), (130, 2, 0, 128, 0, 32, 6, 0),
    (29, 1, 5, 64, 20, 128, 3, 0), (50, 2, 2, 64, 64, 16, 5, 3), (700, 8, 0, 128, 128, 256, 4, 16), (5000, 1, 1, 64, 64, 16, 400, 0)])
def test_append(ctx, dtype, interleaved, tokens, kv_heads, q_heads, dim, rot, page, pages, gap):
    rng = fx.rng_for(210, tokens + dim + rot)
    row = kv_heads * dim
    kb, k = sr.values(rng, (tokens, row + gap), dtype)
    vb, _ = sr.values(rng, (tokens, row + 2 * gap), dtype)
    qb, q = sr.values(rng, (tokens, q_heads * dim + gap), dtype)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    if tokens > 4:      # nowhere: negative, or behind the pool
        slots[1], slots[3], slots[4] = -1, pages * page, 2 ** 31 - 1
    live = (slots >= 0) & (slots < pages * page)
    positions = rng.integers(0, 200000, tokens).astype(np.int32)
    kc = rng.integers(0, 65536, (pages, kv_heads, dim // 8, page, 8)).astype(np.uint16)
    vc = rng.integers(0, 65536, (pages, kv_heads, page, dim)).astype(np.uint16)
    table, _ = cc.rope_table(max(rot, 2))
    table = table[:rot // 2] if rot else np.zeros(1)
    for slot, a in ((1, kb), (2, vb), (3, positions), (4, slots), (5, table), (6, kc), (7, vc)):
        ctx.put(slot, a)
    em = cc.Emitter(act_dtype=ACT[dtype])
    extra = {}
    if q_heads:
        ctx.put(8, qb); ctx.put(9, np.full((tokens, q_heads * dim), 0x7FFF, np.uint16))
        extra = dict(q=B(8), q_out=B(9), q_heads=q_heads, q_stride=q_heads * dim + gap)
    em.paged_kv_append(B(1), B(2), B(3), B(4), B(5), B(6), B(7), tokens, kv_heads, dim, rot, page, pages, interleaved=interleaved, amplitude=0.75, kv_stride=row + gap,
                       v_stride=row + 2 * gap, **extra)
    assert ctx.interpret_decode(em.table_for(ctx)) == 1
    ctx.wait()
    got_k = ctx.read(6, np.uint16, kc.size).reshape(kc.shape)
    got_v = ctx.read(7, np.uint16, vc.size).reshape(vc.shape)
    want_v = vc.copy()
    at, off = slots[live] // page, slots[live] % page
    want_v[at, :, off] = vb[live, :row].reshape(-1, kv_heads, dim)
    assert np.array_equal(got_v, want_v)
    want, reach = sr.rope(k[:, :row].reshape(tokens, kv_heads, dim), positions, table, 0.75, rot, interleaved)
    placed = sr.keys_from_pages(got_k)[at, :, off]
    sr.check_rope(placed, want[live], reach[live], dtype, "keys")
    assert np.array_equal(placed[..., rot:], kb[live, :row].reshape(-1, kv_heads, dim)[..., rot:])
    rest = np.ones((pages, page), bool)
    rest[at, off] = False
    assert np.array_equal(sr.keys_from_pages(got_k).swapaxes(1, 2)[rest], sr.keys_from_pages(kc).swapaxes(1, 2)[rest])   # other places are untouched
    if q_heads:
        want, reach = sr.rope(q[:, :q_heads * dim].reshape(tokens, q_heads, dim), positions, table, 0.75, rot, interleaved)
        sr.check_rope(ctx.read(9, np.uint16, want.size), want, reach, dtype, "q")


def test_append_is_refused_where_a_slot_is_short(ctx):
    for slot, n in ((1, 512), (2, 512), (3, 8), (4, 8), (5, 256), (6, 16 * 2 * 128 * 2), (7, 16 * 2 * 128 * 2)):
        ctx.alloc(slot, n)

    def go(tokens=2, pages=2, **kw):
        a = dict(k=B(1), v=B(2), positions=B(3), slots=B(4), table=B(5), k_cache=B(6), v_cache=B(7))
        em = cc.Emitter()
        em.paged_kv_append(**{**a, **kw}, tokens=tokens, kv_heads=1, head_dim=128, rotary_dim=64, page_size=16, pages=pages)
        return ctx.interpret_decode(em.table_for(ctx))

    assert go() == 1 and go(tokens=0) == 0
    for kw in (dict(tokens=3), dict(pages=3), dict(k_cache=B(6, 16)), dict(v_cache=B(7, 16)), dict(slots=B(4, 4)), dict(table=B(5, 16)), dict(k=B(1, 16))):
        with pytest.raises(rt.SmeltHipError, match="needs"):
            go(**kw)
    with pytest.raises(rt.SmeltHipError, match="aligned"):
        go(pages=1, k_cache=B(6, 8))
    ctx.wait()


def hip_runtime():
    lib = C.CDLL("libamdhip64.so.7")     # the one the library has loaded
    lib.hipMalloc.argtypes = [C.POINTER(C.c_void_p), C.c_size_t]
    lib.hipFree.argtypes = [C.c_void_p]
    return lib


def test_slots_bound_to_the_callers_memory(ctx):
    hip = hip_runtime()
    p = C.c_void_p()
    nbytes = 1 << 20
    assert hip.hipMalloc(C.byref(p), nbytes) == 0
    try:
        tokens, heads, dim = 9, 2, 64
        bits, x = sr.values(fx.rng_for(211, 1), (tokens, heads * dim), fx.F16)
        table, _ = cc.rope_table(dim)
        positions = np.arange(tokens, dtype=np.int32)
        ctx.bind(20, p.value, bits.nbytes)
        ctx.bind(21, p.value + nbytes - bits.nbytes, bits.nbytes)          # up to the allocation's last byte
        ctx.write(20, bits); ctx.put(3, positions); ctx.put(4, table)
        em = cc.Emitter()
        em.rope(B(20), B(21), B(3), B(4), tokens, heads, dim, dim)
        assert ctx.interpret_decode(em.table_for(ctx)) == 1
        want, reach = sr.rope(x.reshape(tokens, heads, dim), positions, table, 1.0, dim, False)
        sr.check_rope(ctx.read(21, np.uint16, bits.size), want, reach, fx.F16, "bound slots")
        assert ctx.stream() != 0
        # kernels that load whole vectors behind a ragged tail do not take them
        rec = rt.make_record(ctx.pipeline("buffer_copy"), [(20, 0, 0), (2, 1, 0)], [(2, 8)], (1, 1, 1), (64, 1, 1))
        ctx.alloc(2, 4096)
        with pytest.raises(rt.SmeltHipError, match="only the serving operators"):
            ctx.encode_decode(rec)
        with pytest.raises(rt.SmeltHipError, match="behind its allocation"):
            ctx.bind(22, p.value + nbytes - 16, 32)
        host = np.zeros(64, np.uint8)
        with pytest.raises(rt.SmeltHipError, match="not on the context's device"):
            ctx.bind(22, host.ctypes.data, 64)
        for bad in ((22, 0, 64), (22, p.value, 0), (-1, p.value, 64), (1 << 20, p.value, 64)):
            with pytest.raises(rt.SmeltHipError):
                ctx.bind(*bad)
        ctx.release(20); ctx.release(21); ctx.release(21)
        with pytest.raises(rt.SmeltHipError, match="no buffer"):
            ctx.interpret_decode(em.table_for(ctx))
        ctx.alloc(20, 64)                                                   # a slot that was bound can be allocated, and the other way round
        ctx.bind(20, p.value, 64)
        ctx.release(20)
        free_before = ctx.memory_info()[0]
        ctx.alloc(20, 64 << 20); ctx.release(20)
        assert ctx.memory_info()[0] == free_before
    finally:
        ctx.wait()
        hip.hipFree(p)


@pytest.mark.parametrize("dtype", [fx.F16, fx.BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "interleaved"])
@pytest.mark.parametrize("tokens,kv,h,dim,rot,gap", [(1, 2, 8, 64, 64, 0), (2, 4, 24, 256, 64, 0), (64, 2, 8, 128, 128, 16), (29, 1, 5, 64, 20, 3), (1100, 2, 4, 64, 64, 0)])
def test_append_with_q_in_place_within_fused_rows(ctx, dtype, interleaved, tokens, kv, h, dim, rot, gap):
    """Rows [q | k | v] of one buffer: q rotated where it stands, k and v read beside it and left as they were."""
    rng = fx.rng_for(212, tokens + dim + rot)
    page, q_end, k_end, row = 16, h * dim, (h + kv) * dim, (h + 2 * kv) * dim + gap
    pages = -(-tokens // page) + 1
    bits, x = sr.values(rng, (tokens, row), dtype)
    slots, positions = rng.permutation(pages * page)[:tokens].astype(np.int32), rng.integers(0, 200000, tokens).astype(np.int32)
    table, _ = cc.rope_table(rot)
    for slot, a in ((1, bits), (3, positions), (4, slots), (5, table)):
        ctx.put(slot, a)
    ctx.alloc(6, pages * page * kv * dim * 2); ctx.alloc(7, pages * page * kv * dim * 2)
    em = cc.Emitter(act_dtype=ACT[dtype])
    em.paged_kv_append(B(1, 2 * q_end), B(1, 2 * k_end), B(3), B(4), B(5), B(6), B(7), tokens, kv, dim, rot, page, pages, interleaved=interleaved, kv_stride=row, q=B(1), q_out=B(1), q_heads=h,
                       q_stride=row, q_out_stride=row)
    assert ctx.interpret_decode(em.table_for(ctx)) == 1
    ctx.wait()
    got = ctx.read(1, np.uint16, bits.size).reshape(bits.shape)
    assert np.array_equal(got[:, q_end:], bits[:, q_end:])
    want, reach = sr.rope(x[:, :q_end].reshape(tokens, h, dim), positions, table, 1.0, rot, interleaved)
    sr.check_rope(got[:, :q_end], want, reach, dtype, "q")
    at, off = slots // page, slots % page
    assert np.array_equal(ctx.read(7, np.uint16, pages * page * kv * dim).reshape(pages, kv, page, dim)[at, :, off], bits[:, k_end:k_end + kv * dim].reshape(tokens, kv, dim))
    want, reach = sr.rope(x[:, q_end:k_end].reshape(tokens, kv, dim), positions, table, 1.0, rot, interleaved)
    placed = sr.keys_from_pages(ctx.read(6, np.uint16, pages * page * kv * dim).reshape(pages, kv, dim // 8, page, 8))[at, :, off]
    sr.check_rope(placed, want, reach, dtype, "keys")
