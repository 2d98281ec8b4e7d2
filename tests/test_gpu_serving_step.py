"""The serving operators as a step runs them: q|k|v of new tokens -> rotated and put away -> attention behind a shared prefix -> o
projection -> logits -> drafts verified; eager and as a graph whose lengths, positions and pages move on between replays."""
import numpy as np
import pytest

import fixtures as fx
import gpu_harness as gh
import serving_ref as sr
from smelt_amd import compiler as cc
from smelt_amd import runtime as rt

pytestmark = pytest.mark.gpu
B = cc.bind
ACT = {fx.F16: rt.ACT_F16, fx.BF16: rt.ACT_BF16}

HEADS, KV, DIM, ROT, PAGE, PREFIX, VOCAB = 8, 2, 64, 32, 16, 37, 1000
MODEL = 256
(X, QKV_Q, QKV_K, QKV_V, QR, POS, SLOTS, TABLE, KC, VC, PT, LENS, OFFS, PFX, PLEN, ATT, Y, LOGITS, DRAFTS, UA, US, TEMP, TOK, CNT) = range(1, 25)


class Step:
    """A batch of three sequences that each take a few rows a step."""

    def __init__(self, dtype, seed):
        self.dtype = dtype
        self.rng = fx.rng_for(240, seed)
        self.rows = [3, 1, 4]
        self.tokens = sum(self.rows)
        self.width, self.pages = 12, 48
        order = self.rng.permutation(self.pages)
        front = -(-PREFIX // PAGE)
        self.prefix_pages = order[:front].astype(np.int32)
        self.table = order[front:front + 3 * self.width].reshape(3, self.width).astype(np.int32)
        self.lens = [0, 20, 5]
        self.kc, self.vc = (sr.values(self.rng, (self.pages, KV, PAGE, DIM), dtype)[0] for _ in range(2))
        self.freq, _ = cc.rope_table(ROT)
        self.offsets = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)
        lay = cc.Layout()
        self.bank = lay.affine_bank([HEADS * DIM, KV * DIM, KV * DIM], MODEL, 64)
        self.o = lay.affine(VOCAB, HEADS * DIM, 64)
        self.image = np.zeros(lay.total_bytes, np.uint8)
        for k, e in enumerate((*self.bank, self.o)):
            cc.write_affine(self.image, e, *fx.synth_affine(e.rows, e.cols, 64, dtype, config=4, tensor=k + 1))

    def install(self, ctx):
        ctx.upload_weights(0, self.image)
        ctx.put(KC, sr.keys_to_pages(self.kc, PAGE)); ctx.put(VC, self.vc); ctx.put(PT, self.table); ctx.put(PFX, self.prefix_pages); ctx.put(PLEN, np.array([PREFIX], np.int32))
        ctx.put(TABLE, self.freq[:ROT // 2]); ctx.put(OFFS, self.offsets); ctx.put(X, np.zeros((self.tokens, MODEL), np.uint16))
        for slot, n in ((QKV_Q, HEADS * DIM), (QKV_K, KV * DIM), (QKV_V, KV * DIM), (QR, HEADS * DIM), (ATT, HEADS * DIM), (LOGITS, VOCAB)):
            ctx.alloc(slot, self.tokens * n * 2)
        for slot, n in ((POS, self.tokens), (SLOTS, self.tokens), (LENS, 3), (DRAFTS, self.tokens), (UA, self.tokens), (US, 3), (TEMP, 3), (TOK, self.tokens), (CNT, 3)):
            ctx.alloc(slot, n * 4)
        em = cc.Emitter(act_dtype=ACT[self.dtype])
        for e, out in zip(self.bank, (QKV_Q, QKV_K, QKV_V)):
            em.matvec(0, e, B(X), B(out), batch=self.tokens)
        em.paged_kv_append(B(QKV_K), B(QKV_V), B(POS), B(SLOTS), B(TABLE), B(KC), B(VC), self.tokens, KV, DIM, ROT, PAGE, self.pages, q=B(QKV_Q), q_out=B(QR), q_heads=HEADS)
        em.paged_attention(B(QR), B(KC), B(VC), B(PT), B(LENS), B(OFFS), B(ATT), self.tokens, 3, HEADS, KV, DIM, PAGE, self.pages, self.width, DIM ** -0.5,
                           prefix_table=B(PFX), prefix_len=B(PLEN), prefix_pages=len(self.prefix_pages))
        em.matvec(0, self.o, B(ATT), B(LOGITS), batch=self.tokens)
        em.verify_drafts(B(LOGITS), B(DRAFTS), B(OFFS), B(UA), B(US), B(TEMP), B(TOK), B(CNT), self.tokens, 3, VOCAB)
        return em.table_for(ctx)

    def advance(self, ctx):
        """The next step's inputs, as a host writes them."""
        self.lens = [l + n for l, n in zip(self.lens, self.rows)]
        pos = np.concatenate([np.arange(PREFIX + l - n, PREFIX + l) for l, n in zip(self.lens, self.rows)])
        own = np.concatenate([np.arange(l - n, l) for l, n in zip(self.lens, self.rows)])
        seq = np.repeat(np.arange(3), self.rows)
        self.positions, self.slots = pos.astype(np.int32), (self.table[seq, own // PAGE] * PAGE + own % PAGE).astype(np.int32)
        self.x, _ = sr.values(self.rng, (self.tokens, MODEL), self.dtype, 0.5)
        self.drafts = self.rng.integers(0, VOCAB, self.tokens).astype(np.int32)
        self.ua, self.us = (self.rng.random(n).astype(np.float32) for n in (self.tokens, 3))
        self.temp = np.array([0.7, 0.0, 1.1], np.float32)
        for slot, a in ((X, self.x), (POS, self.positions), (SLOTS, self.slots), (LENS, np.array(self.lens, np.int32)), (DRAFTS, self.drafts), (UA, self.ua), (US, self.us), (TEMP, self.temp),
                        (TOK, np.full(self.tokens, -7, np.int32)), (CNT, np.full(3, -7, np.int32))):
            ctx.write(slot, a)

    def read(self, ctx):
        n = self.tokens
        return {k: ctx.read(s, t, c) for k, s, t, c in (("q", QKV_Q, np.uint16, n * HEADS * DIM), ("k", QKV_K, np.uint16, n * KV * DIM), ("v", QKV_V, np.uint16, n * KV * DIM), ("qr", QR, np.uint16, n * HEADS * DIM),
                                                        ("kc", KC, np.uint16, self.kc.size), ("vc", VC, np.uint16, self.vc.size), ("att", ATT, np.uint16, n * HEADS * DIM), ("logits", LOGITS, np.uint16, n * VOCAB),
                                                        ("tokens", TOK, np.int32, n), ("counts", CNT, np.int32, 3))}

    def check(self, got):
        d, n = self.dtype, self.tokens
        assert np.abs(sr.wide(got["q"], d)).max() > 0
        for part, heads in (("q", HEADS), ("k", KV)):
            want, reach = sr.rope(sr.wide(got[part], d).reshape(n, heads, DIM), self.positions, self.freq, 1.0, ROT, False)
            if part == "q":
                sr.check_rope(got["qr"], want, reach, d, "q")
            else:
                kc = sr.keys_from_pages(got["kc"].reshape(self.pages, KV, DIM // 8, PAGE, 8))
                sr.check_rope(kc[self.slots // PAGE, :, self.slots % PAGE], want, reach, d, "k")
        vc = got["vc"].reshape(self.pages, KV, PAGE, DIM)
        assert np.array_equal(vc[self.slots // PAGE, :, self.slots % PAGE], got["v"].reshape(n, KV, DIM))
        y, reach, sharp, count = sr.attention(sr.wide(got["qr"], d).reshape(n, HEADS, DIM), sr.wide(kc, d), sr.wide(vc, d), self.pages, self.table, self.lens, self.offsets,
                                              float(np.float32(DIM ** -0.5)), 0, self.prefix_pages, PREFIX)
        off = np.abs(sr.wide(got["att"], d).reshape(y.shape) - y)
        assert np.all(off <= sr.attention_tolerance(y, reach, sharp, count, DIM, d))
        tokens, counts = sr.verify(sr.wide(got["logits"], d).reshape(n, VOCAB), None, self.drafts, self.offsets, self.ua, self.us, self.temp, np.full(n, -7, np.int32))
        assert np.array_equal(got["tokens"], tokens) and np.array_equal(got["counts"], counts)


@pytest.mark.parametrize("dtype", [fx.F16, fx.BF16], ids=["f16", "bf16"])
def test_steps_eager_and_replayed(dtype):
    ctx, other = rt.Context(), rt.Context()
    try:
        step, twin = Step(dtype, 1), Step(dtype, 1)
        table, twin_table = step.install(ctx), twin.install(other)
        graph, launches = ctx.capture_decode(table)
        # a second graph on the same context and workspace, replayed in between
        single = cc.Emitter(act_dtype=ACT[dtype])
        single.paged_attention(B(QR), B(KC), B(VC), B(PT), B(LENS), B(OFFS), B(ATT), step.tokens, 3, HEADS, KV, DIM, PAGE, step.pages, step.width, DIM ** -0.5)
        graph2, _ = ctx.capture_decode(single.table_for(ctx))
        assert launches >= 7
        for k in range(6):
            step.advance(ctx); twin.advance(other)
            if k % 2:
                ctx.graph_launch(graph2)
            ctx.graph_launch(graph)
            assert other.interpret_decode(twin_table) == launches
            ctx.wait(); other.wait()
            got, eager = step.read(ctx), twin.read(other)
            for part in got:
                assert np.array_equal(got[part], eager[part]), (k, part)
            step.check(got)
        ctx.graph_destroy(graph); ctx.graph_destroy(graph2)
    finally:
        ctx.close(); other.close()


def test_operands_that_lie_between_their_types_places_are_refused_at_launch():
    """The emitter knows no addresses: it takes every offset, the launch refuses those that no load of the operand's type can take."""
    ctx = rt.Context()
    try:
        for slot in range(1, 12):
            ctx.alloc(slot, 1 << 16)
        base = {
            "rope": dict(x=B(1), y=B(2), positions=B(3), table=B(4)),
            "paged_kv_append": dict(k=B(1), v=B(2), positions=B(3), slots=B(4), table=B(5), k_cache=B(6), v_cache=B(7), q=B(8), q_out=B(9)),
            "paged_attention": dict(q=B(1), k_cache=B(2), v_cache=B(3), page_table=B(4), kv_lens=B(5), offsets=B(6), out=B(7), prefix_table=B(8), prefix_len=B(9)),
            "verify_drafts": dict(target=B(1), draft=B(2), draft_tokens=B(3), offsets=B(4), u_accept=B(5), u_sample=B(6), temperature=B(7), tokens=B(8), counts=B(9))}
        rest = {
            "rope": dict(tokens=2, heads=2, head_dim=64, rotary_dim=64),
            "paged_kv_append": dict(tokens=2, kv_heads=1, head_dim=64, rotary_dim=64, page_size=16, pages=2, q_heads=2),
            "paged_attention": dict(tokens=2, sequences=1, heads=2, kv_heads=1, head_dim=64, page_size=16, pages=2, pages_per_sequence=2, scale=0.1, prefix_pages=1),
            "verify_drafts": dict(rows=2, sequences=1, vocab=100)}
        needs = dict(k_cache=16, v_cache=16, out=8, table=8, x=2, y=2, k=2, v=2, q=2, q_out=2, target=2, draft=2)      # (4 where it is not said)
        for op, operands in base.items():
            def go(**kw):
                em = cc.Emitter()
                getattr(em, op)(**{**operands, **rest[op], **kw})
                return ctx.interpret_decode(em.table_for(ctx))

            assert go() >= 1
            for name, b in operands.items():
                align = needs.get(name, 4)
                for off in {align // 2, align - 1} - {0}:
                    with pytest.raises(rt.SmeltHipError, match="aligned"):
                        go(**{name: B(b.slot, off)})
                assert go(**{name: B(b.slot, 2 * align)}) >= 1
        ctx.wait()
    finally:
        ctx.close()
