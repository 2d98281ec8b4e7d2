"""The serving operators between the projections of a layer and behind its lm_head, as measured cases: rotary positions, the paged
key / value cache, attention over it (with a prefix that a batch shares) and the verification of drafted tokens.

`own` false: elementary torch operations.  `own` true: the calls a user makes (records emitted once, slots bound to the tensors,
one interpret call a pass).
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}

# ---- cases ---------------------------------------------------------------------------------------------------------------


def listed():
    return [
        # the q heads of a small model at one token: nothing but latency
        dict(name="rope one token", op="rope", tokens=1, heads=8, dim=256, rot=64, layout="half", scaling="none", far=2048, dtype="f16", gap=0),
        # the q rows of a prompt inside a fused projection's rows, far positions, frequencies scaled in bands
        dict(name="rope prompt", op="rope", tokens=8192, heads=32, dim=128, rot=128, layout="interleaved", scaling="bands", far=131072, dtype="bf16", gap=2048),
        # one decode step of 64 sequences: q rotated, k rotated and k, v put away (one padded row)
        dict(name="append decode", op="append", tokens=64, heads=24, kv_heads=4, dim=256, rot=64, layout="half", scaling="none", far=32768, page=64, pages=2048, skip=1, dtype="bf16", gap=0),
        # a prompt put into pages of 16, k and v only
        dict(name="append prompt", op="append", tokens=8000, heads=0, kv_heads=8, dim=128, rot=128, layout="interleaved", scaling="parts", far=65536, page=16, pages=2048, skip=0, dtype="f16", gap=1024),
        # one token of one sequence with a short past: latency again
        dict(name="attention one token", op="attention", seqs=1, new=1, new_hi=1, own_lo=1000, own_hi=1000, prefix=0, heads=8, kv_heads=2, dim=256, page=64, window=0, pad=0, dtype="f16", gap=0),
        # a decode step of 64 conversations behind one long system prompt
        dict(name="attention shared decode", op="attention", seqs=64, new=1, new_hi=1, own_lo=17, own_hi=1024, prefix=8192, heads=24, kv_heads=4, dim=256, page=64, window=0, pad=0, dtype="bf16", gap=0),
        # drafted tokens of 24 sequences checked in one pass, ragged, pages of 16, two padded rows
        dict(name="attention shared verify", op="attention", seqs=24, new=1, new_hi=8, own_lo=100, own_hi=2000, prefix=2500, heads=32, kv_heads=8, dim=128, page=16, window=0, pad=2, dtype="f16", gap=2048),
        # a few sequences with a very long past of their own
        dict(name="attention long decode", op="attention", seqs=4, new=1, new_hi=1, own_lo=50000, own_hi=65536, prefix=0, heads=24, kv_heads=4, dim=256, page=64, window=0, pad=0, dtype="bf16", gap=0),
        # the next chunk of two prompts behind a shared prefix
        dict(name="attention prompt chunk", op="attention", seqs=2, new=900, new_hi=1024, own_lo=1500, own_hi=2048, prefix=2000, heads=32, kv_heads=8, dim=128, page=64, window=0, pad=0, dtype="bf16", gap=0),
        # one sequence, four drafts
        dict(name="verify one sequence", op="verify", seqs=1, rows_lo=5, rows_hi=5, vocab=151936, drafts="logits", greedy=0, pad=0, dtype="f16"),
        # a batch of ragged drafts from a draft model, a few sequences greedy
        dict(name="verify batch", op="verify", seqs=64, rows_lo=1, rows_hi=8, vocab=248320, drafts="logits", greedy=8, pad=3, dtype="bf16"),
        # drafts looked up in the prompt: no draft probabilities
        dict(name="verify lookup drafts", op="verify", seqs=32, rows_lo=2, rows_hi=6, vocab=151936, drafts="given", greedy=0, pad=0, dtype="f16"),
    ]


def draw(rng):
    def between(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rope", "append", "attention", "attention", "verify"])
    dtype = rng.choice(["f16", "bf16"])
    dim = rng.choice([64, 128, 256])
    if op in ("rope", "append"):
        rot = rng.choice([dim, dim // 2, dim // 4])
        c = dict(op=op, rot=rot, dim=dim, layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "bands", "parts"]), dtype=dtype, far=between(100, 500000))
        if op == "rope":
            return dict(c, tokens=between(1, 8192), heads=rng.randint(1, 32 * 128 // dim), gap=rng.choice([0, 8 * rng.randint(1, 256)]))
        page = rng.choice([16, 32, 64, 128, 256])
        tokens = between(1, 8000)
        return dict(c, tokens=tokens, heads=rng.choice([0, rng.randint(1, 16)]), kv_heads=rng.randint(1, 8 * 128 // dim), page=page, pages=-(-tokens // page) + rng.randint(1, 200),
                    skip=rng.choice([0, 1, 3]) if tokens > 8 else 0, gap=rng.choice([0, 8 * rng.randint(1, 128)]))
    if op == "attention":
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        heads = kv_heads * rng.choice([m for m in (1, 2, 3, 4, 6, 8) if m * kv_heads * dim <= 8192])
        new = rng.choice([1, 1, between(1, 8), between(1, 300)])
        seqs = between(1, 64) if new <= 8 else between(1, 2)
        most = min(60000, int(2.0e8 / (seqs * kv_heads * dim)))
        if new > 8:
            most = min(most, 4000)
        own_hi = max(new, between(1, most))
        prefix = rng.choice([0, between(1, 8000)])
        if new > 8:
            prefix = min(prefix, 2500)
        return dict(op=op, seqs=seqs, new=rng.choice([0, 1, new]) if seqs > 1 else new, new_hi=new, own_lo=max(1, own_hi // rng.choice([1, 2, 50])), own_hi=own_hi, prefix=prefix, heads=heads, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([16, 32, 64, 128, 256]), window=rng.choice([0, 0, 0, between(1, 5000)]), pad=rng.choice([0, 0, 3]), dtype=dtype, gap=rng.choice([0, 8 * rng.randint(1, 256)]))
    rows_hi = rng.randint(1, 8)
    seqs = between(1, 64)
    return dict(op=op, seqs=seqs, rows_lo=rng.randint(0, 1) if seqs > 1 else 1, rows_hi=rows_hi, vocab=rng.choice([32000, 151936, 248320, between(2, 248320)]), drafts=rng.choice(["logits", "given"]),
                greedy=rng.choice([0, seqs // 3, seqs]), pad=rng.choice([0, 2]), dtype=dtype)


# ---- inputs --------------------------------------------------------------------------------------------------------------


def _frequencies(rot, scaling):
    """Radians a position of each rotated pair in 64 bits, and the amplitude of the rotation, for a context of 4 times the 8192
    positions that the plain frequencies (base 10000, or 500000 in bands) were made for."""
    half = rot // 2
    base = 500000.0 if scaling == "bands" else 10000.0
    f = base ** (-np.arange(half, dtype=np.float64) * 2.0 / rot)
    if scaling == "linear":
        return f / 4.0, 1.0
    if scaling == "bands":   # long waves divided by the factor, short ones kept, a linear passage between
        turns = 8192.0 * f / (2.0 * np.pi)
        keep = np.clip((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return keep * f + (1.0 - keep) * f / 4.0, 1.0
    if scaling == "parts":   # the passage runs over the index of the pair, and the scores are sharpened
        lo, hi = (rot * math.log(8192.0 / (n * 2.0 * math.pi)) / (2.0 * math.log(base)) for n in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), rot - 1)
        divide = np.clip((np.arange(half) - lo) / max(hi - lo, 0.001), 0.0, 1.0)
        return divide * f / 4.0 + (1.0 - divide) * f, 0.1 * math.log(4.0) + 1.0
    return f, 1.0


def _normal(gen, shape, dtype, scale=1.0):
    x = torch.empty(shape, dtype=dtype, device="cuda")
    return x.normal_(0.0, scale, generator=gen)


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _spread(lo, hi, count):
    """`count` lengths from lo to hi, the last of them hi: the same ones for every seed."""
    return np.linspace(hi if count == 1 else lo, hi, count).round().astype(np.int64)


def prepare(case, seed):
    rs = np.random.RandomState(seed & 0x7FFFFFFF)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]
    st = dict(case=case)
    if case["op"] in ("rope", "append"):
        T, D = case["tokens"], case["dim"]
        f, st["amplitude"] = _frequencies(case["rot"], case["scaling"])
        st["table"] = torch.from_numpy(f).cuda()
        st["positions"] = _ints(rs.randint(0, case["far"], T))
    if case["op"] == "rope":
        st["x"] = _normal(gen, (T, case["heads"] * D + case["gap"]), dt)
        st["y"] = torch.zeros((T, case["heads"] * D), dtype=dt, device="cuda")
    elif case["op"] == "append":
        HK, H, page, pages = case["kv_heads"], case["heads"], case["page"], case["pages"]
        st["k"] = _normal(gen, (T, HK * D + case["gap"]), dt)
        st["v"] = _normal(gen, (T, HK * D + case["gap"]), dt)
        st["q"] = _normal(gen, (T, H * D + case["gap"]), dt) if H else None
        st["q_out"] = torch.zeros((T, H * D), dtype=dt, device="cuda") if H else None
        # the last page is nobody's: decode tokens go to places all over the pool, prompts fill whole pages in any order
        if T * page <= pages * 8:
            slots = rs.permutation((pages - 1) * page)[:T]
        else:
            order = rs.permutation(pages - 1)[: -(-T // page)]
            slots = (order[:, None] * page + np.arange(page)[None, :]).reshape(-1)[:T]
        if case["skip"]:
            slots[rs.permutation(T)[: case["skip"]]] = -1
        st["slots"] = _ints(slots)
        st["k_cache"] = _normal(gen, (pages, HK, D // 8, page, 8), dt)
        st["v_cache"] = _normal(gen, (pages, HK, page, D), dt)
    elif case["op"] == "attention":
        S, H, HK, D, page = case["seqs"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        n = rs.permutation(_spread(case["new"], case["new_hi"], S))
        cu = np.concatenate([[0], np.cumsum(n)])
        L = np.maximum(rs.permutation(_spread(case["own_lo"], case["own_hi"], S)), n)
        width, prefix_pages = -(-int(max(case["own_hi"], case["new_hi"])) // page), -(-case["prefix"] // page)
        used = -(-L // page)
        pool = int(used.sum()) + prefix_pages + 1
        order = rs.permutation(pool)
        table = np.full((S, width), 0)
        table[np.arange(width)[None, :] < used[:, None]] = order[prefix_pages : prefix_pages + int(used.sum())]
        T = int(cu[-1]) + case["pad"]
        st.update(pages=pool, width=width, prefix_pages=prefix_pages, tokens=T, scale=1.0 / math.sqrt(D))
        st["q"] = _normal(gen, (T, H * D + case["gap"]), dt, 1.5)
        st["k_cache"] = _normal(gen, (pool, HK, D // 8, page, 8), dt)
        st["v_cache"] = _normal(gen, (pool, HK, page, D), dt)
        st["page_table"], st["kv_lens"], st["offsets"] = _ints(table), _ints(L), _ints(cu)
        st["prefix_table"] = _ints(order[:prefix_pages]) if prefix_pages else None
        st["prefix_len"] = _ints([case["prefix"]])
        st["out"] = _normal(gen, (T, H * D), dt, 0.02)
    else:
        S, V = case["seqs"], case["vocab"]
        cu = np.concatenate([[0], np.cumsum(rs.permutation(_spread(case["rows_lo"], case["rows_hi"], S)))])
        R = int(cu[-1]) + case["pad"]
        st.update(rows=R)
        st["target"] = _normal(gen, (R, V), dt, 2.5)
        # a draft model near the target: its logits are the target's and some noise
        st["draft"] = (st["target"] + _normal(gen, (R, V), dt, 1.0)) if case["drafts"] == "logits" else None
        # drafted tokens are likely ones: the best of a few noisy looks at the target
        noisy = st["target"].float() + 2.0 * torch.empty((R, V), device="cuda").exponential_(generator=gen).log_().neg_()
        st["draft_tokens"] = noisy.argmax(1).to(torch.int32)
        del noisy
        st["offsets"] = _ints(cu)
        st["u_accept"] = torch.rand(R, device="cuda", generator=gen)
        st["u_sample"] = torch.rand(S, device="cuda", generator=gen)
        temperature = rs.uniform(0.5, 1.2, S).astype(np.float32)
        temperature[rs.permutation(S)[: case["greedy"]]] = 0.0
        st["temperature"] = torch.from_numpy(temperature).cuda()
        st["tokens"] = torch.full((R,), -7, dtype=torch.int32, device="cuda")
        st["counts"] = torch.full((S,), -7, dtype=torch.int32, device="cuda")
    if own:
        st["plan"] = _Plan(st)
    return st


# ---- the framework's calls -----------------------------------------------------------------------------------------------

_context = None


class _Plan:
    """What a program keeps for a step: the records and the slots that name its buffers."""

    free = list(range(4000))

    def __init__(self, st):
        from smelt_amd import compiler as cc
        from smelt_amd import runtime as rt

        global _context
        if _context is None:
            _context = rt.Context()
        self.ctx, self.slots = _context, []
        case = st["case"]
        em = cc.Emitter(act_dtype=rt.ACT_F16 if case["dtype"] == "f16" else rt.ACT_BF16)

        def b(name):
            t = st[name]
            slot = _Plan.free.pop()
            self.slots.append(slot)
            self.ctx.bind(slot, t.data_ptr(), t.numel() * t.element_size())
            return cc.bind(slot)

        if case["op"] == "rope":
            em.rope(b("x"), b("y"), b("positions"), b("table"), case["tokens"], case["heads"], case["dim"], case["rot"], interleaved=case["layout"] == "interleaved",
                    amplitude=st["amplitude"], x_stride=st["x"].shape[1])
        elif case["op"] == "append":
            q = dict(q=b("q"), q_out=b("q_out"), q_heads=case["heads"], q_stride=st["q"].shape[1]) if case["heads"] else {}
            em.paged_kv_append(b("k"), b("v"), b("positions"), b("slots"), b("table"), b("k_cache"), b("v_cache"), case["tokens"], case["kv_heads"], case["dim"], case["rot"],
                               case["page"], case["pages"], interleaved=case["layout"] == "interleaved", amplitude=st["amplitude"], kv_stride=st["k"].shape[1], **q)
        elif case["op"] == "attention":
            shared = dict(prefix_table=b("prefix_table"), prefix_len=b("prefix_len"), prefix_pages=st["prefix_pages"]) if case["prefix"] else {}
            em.paged_attention(b("q"), b("k_cache"), b("v_cache"), b("page_table"), b("kv_lens"), b("offsets"), b("out"), st["tokens"], case["seqs"], case["heads"], case["kv_heads"],
                               case["dim"], case["page"], st["pages"], st["width"], st["scale"], window=case["window"], q_stride=st["q"].shape[1], **shared)
        else:
            draft = dict(draft=b("draft")) if case["drafts"] == "logits" else {}
            em.verify_drafts(b("target"), b("draft_tokens"), b("offsets"), b("u_accept"), b("u_sample"), b("temperature"), b("tokens"), b("counts"), st["rows"], case["seqs"],
                             case["vocab"], **draft)
        self.table = em.table_for(self.ctx)
        torch.cuda.synchronize()   # the inputs were made on another stream than the context's

    def run(self):
        self.ctx.interpret_decode(self.table)

    def __del__(self):
        for slot in self.slots:
            self.ctx.release(slot)
            _Plan.free.append(slot)


# ---- one pass ------------------------------------------------------------------------------------------------------------


def run(st):
    op = st["case"]["op"]
    if own:
        st["plan"].run()
        if op == "rope":
            return st["y"]
        if op == "append":
            return [st["k_cache"], st["v_cache"]] + ([st["q_out"]] if st["q_out"] is not None else [])
        if op == "attention":
            return st["out"]
        return [st["tokens"], st["counts"]]
    return {"rope": _rope, "append": _append, "attention": _attention, "verify": _verify}[op](st)


def _rotate(x, st, heads):
    """Rows of `heads` heads rotated to their positions, in the type of x."""
    c = st["case"]
    D, R = c["dim"], c["rot"]
    x = x[:, : heads * D].reshape(-1, heads, D).float()
    angle = st["positions"].double()[:, None] * st["table"][None, :]
    cos, sin = ((fn(angle) * st["amplitude"]).float()[:, None, :] for fn in (torch.cos, torch.sin))
    if c["layout"] == "half":
        a, b = x[:, :, : R // 2], x[:, :, R // 2 : R]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin, x[:, :, R:]], 2)
    else:
        a, b = x[:, :, 0:R:2], x[:, :, 1:R:2]
        y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], 3).flatten(2), x[:, :, R:]], 2)
    return y.to(TYPES[c["dtype"]])


def _rope(st):
    return _rotate(st["x"], st, st["case"]["heads"]).flatten(1)


def _append(st):
    c = st["case"]
    HK, D, page = c["kv_heads"], c["dim"], c["page"]
    k = _rotate(st["k"], st, HK)
    v = st["v"][:, : HK * D].reshape(-1, HK, D)
    # a token without a place rewrites what stands in the pool's last place, which is nobody's
    live = st["slots"] >= 0
    slot = torch.where(live, st["slots"], c["pages"] * page - 1).long()
    at, off = slot // page, slot % page
    keep_k, keep_v = st["k_cache"][at, :, :, off], st["v_cache"][at, :, off]
    st["k_cache"][at, :, :, off] = torch.where(live[:, None, None, None], k.reshape(-1, HK, D // 8, 8), keep_k)
    st["v_cache"][at, :, off] = torch.where(live[:, None, None], v, keep_v)
    return [st["k_cache"], st["v_cache"]] + ([_rotate(st["q"], st, c["heads"]).flatten(1)] if c["heads"] else [])


def _attention(st):
    c = st["case"]
    S, H, HK, D, P, n_max = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["prefix"], max(c["new_hi"], 1)
    G, T = H // HK, st["tokens"]
    cu, L = st["offsets"].long(), st["kv_lens"].long()
    n = cu[1:] - cu[:-1]
    q = st["q"][:, : H * D].reshape(T, HK, G, D)
    i = torch.arange(n_max, device="cuda")
    rows = torch.clamp(cu[:-1, None] + i, max=T - 1)
    q = q[rows].float().permute(0, 2, 3, 1, 4).reshape(S, HK, G * n_max, D)

    def gather(table):
        k, v = st["k_cache"][table.long()], st["v_cache"][table.long()]
        lead = table.dim()
        k = k.transpose(lead + 1, lead + 2).flatten(lead + 2).reshape(v.shape)
        return tuple(x.transpose(lead - 1, lead).flatten(lead, lead + 1).float() for x in (k, v))

    width = int(st["width"]) * c["page"]
    k, v = gather(st["page_table"])
    scores = torch.matmul(q, k.transpose(2, 3))
    if P:
        kp, vp = gather(st["prefix_table"])
        kp, vp = kp[:, :P], vp[:, :P]
        flat = q.transpose(0, 1).reshape(HK, S * G * n_max, D)
        front = torch.matmul(flat, kp.transpose(1, 2)).reshape(HK, S, G * n_max, P).transpose(0, 1)
        scores = torch.cat([front, scores], 3)
    at = (P + L - n)[:, None] + i
    j = torch.arange(P + width, device="cuda")
    seen = (j <= at[:, :, None]) & (j < (P + L)[:, None, None])
    if c["window"]:
        seen &= j > at[:, :, None] - c["window"]
    scores = scores.reshape(S, HK, G, n_max, P + width) * st["scale"]
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(4, keepdim=True)
    w = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = w.sum(4, keepdim=True)
    w = w.reshape(S, HK, G * n_max, P + width)
    out = torch.matmul(w[..., P:], v)
    if P:
        flat = w[..., :P].transpose(0, 1).reshape(HK, S * G * n_max, P)
        out += torch.matmul(flat, vp).reshape(HK, S, G * n_max, D).transpose(0, 1)
    out = out.reshape(S, HK, G, n_max, D) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 3, 1, 2, 4).reshape(S, n_max, H * D)
    t = torch.arange(T, device="cuda")
    s = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=S - 1)
    mine = out[s, torch.clamp(t - cu[s], 0, n_max - 1)].to(st["out"].dtype)
    return torch.where((t < cu[-1])[:, None], mine, st["out"])


def _verify(st):
    c = st["case"]
    S, V, R, k_max = c["seqs"], c["vocab"], st["rows"], max(c["rows_hi"], 1)
    cu = st["offsets"].long()
    n = cu[1:] - cu[:-1]
    t = torch.arange(R, device="cuda")
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=S - 1)
    temperature = st["temperature"].double()
    greedy = temperature <= 0
    warm = torch.where(greedy, 1.0, temperature)

    def weights(logits, row, s):
        x = logits[row].double()
        e = torch.exp((x - x.amax(1, keepdim=True)) / warm[s][:, None])
        return e / e.sum(1, keepdim=True)

    token = st["draft_tokens"].long()
    p = weights(st["target"], t, seq).gather(1, token[:, None])[:, 0]
    q = weights(st["draft"], t, seq).gather(1, token[:, None])[:, 0] if st["draft"] is not None else torch.ones_like(p)
    best = st["target"].float().argmax(1)
    ok = torch.where(greedy[seq], token == best, st["u_accept"].double() * q < p)
    # accepted drafts at the front of each sequence
    i = torch.arange(k_max, device="cuda")
    rows = torch.clamp(cu[:-1, None] + i, max=R - 1)
    lead = (ok[rows] & (i < (n - 1)[:, None])).long().cumprod(1).sum(1)
    pick = torch.clamp(cu[:-1] + lead, max=R - 1)
    every = torch.arange(S, device="cuda")
    w = weights(st["target"], pick, every)
    short = lead < n - 1   # a draft was refused: what the target has beyond the draft
    if st["draft"] is not None:
        less = torch.clamp(w - weights(st["draft"], pick, every), min=0.0)
    else:
        less = w.scatter(1, token[pick][:, None], 0.0)
    w = torch.where((short & (less.sum(1) > 0))[:, None], less, w)
    run_sum = w.cumsum(1)
    drawn = torch.searchsorted(run_sum, (st["u_sample"].double() * run_sum[:, -1])[:, None], right=True)[:, 0]
    last = torch.where(w > 0, torch.arange(V, device="cuda"), 0).amax(1)
    drawn = torch.where(greedy, best[pick], torch.minimum(drawn, last))
    back = t - cu[seq]
    tokens = torch.where(back < lead[seq], token, torch.where(back == lead[seq], drawn[seq], -1))
    tokens = torch.where(t < cu[-1], tokens, st["tokens"].long()).to(torch.int32)
    return [tokens, lead.to(torch.int32)]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------


def work(case):
    if case["op"] == "rope":
        moved = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 4 * moved + 4 * case["tokens"], "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    if case["op"] == "append":
        T, D = case["tokens"], case["dim"]
        return {"bytes": T * (4 * D * (2 * case["kv_heads"] + case["heads"]) + 8), "flops": 3 * T * case["rot"] * (case["kv_heads"] + case["heads"])}
    if case["op"] == "attention":
        new = float(_spread(case["new"], case["new_hi"], case["seqs"]).mean())
        keys = float(_spread(case["own_lo"], case["own_hi"], case["seqs"]).mean())
        S, H, HK, D, P, window = (case[k] for k in ("seqs", "heads", "kv_heads", "dim", "prefix", "window"))
        seen = max(keys - new / 2, 0.5) + P
        read_p, read_own = P, keys
        if window:
            seen = min(seen, window)
            read_own = min(keys, window + new)
            read_p = min(P, max(0, window - case["own_lo"]))
        return {"bytes": 4 * HK * D * (read_p + S * read_own) + 4 * S * new * H * D, "flops": 4 * S * new * H * D * seen}
    S, V = case["seqs"], case["vocab"]
    rows = float(_spread(case["rows_lo"], case["rows_hi"], S).sum())
    draft = max(rows - S, 0) if case["drafts"] == "logits" else 0
    return {"bytes": 2 * V * (rows + draft) + 12 * rows, "flops": 4 * V * (rows + draft)}


# ---- the definitions in 64 bits, head by head ----------------------------------------------------------------------------


def _exact_rope(x, positions, table, amplitude, heads, D, R, layout):
    x = x[:, : heads * D].double()
    y = x.clone()
    for d in range(R // 2):
        i, j = (d, d + R // 2) if layout == "half" else (2 * d, 2 * d + 1)
        phase = torch.polar(torch.full_like(positions, amplitude, dtype=torch.float64), positions.double() * table[d])
        for_all = torch.arange(heads, device=x.device) * D
        z = torch.complex(x[:, for_all + i], x[:, for_all + j]) * phase[:, None]
        y[:, for_all + i], y[:, for_all + j] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        return _exact_rope(st["x"], st["positions"], st["table"], st["amplitude"], case["heads"], case["dim"], case["rot"], case["layout"])
    if case["op"] == "append":
        HK, D, page = case["kv_heads"], case["dim"], case["page"]
        args = (st["positions"], st["table"], st["amplitude"])
        k = _exact_rope(st["k"], *args, HK, D, case["rot"], case["layout"])
        slots = st["slots"].cpu().numpy()
        live = torch.from_numpy(np.flatnonzero(slots >= 0)).cuda()
        at, off = (torch.from_numpy(a[slots >= 0].astype(np.int64)).cuda() for a in (slots // page, slots % page))
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        for h in range(HK):
            for d in range(D // 8):
                kc[at, h, d, off] = k[live, h * D + 8 * d : h * D + 8 * d + 8]
            vc[at, h, off] = st["v"][live, h * D : (h + 1) * D].double()
        return [kc, vc] + ([_exact_rope(st["q"], *args, case["heads"], D, case["rot"], case["layout"])] if case["heads"] else [])
    if case["op"] == "attention":
        H, HK, D, P, page = (case[k] for k in ("heads", "kv_heads", "dim", "prefix", "page"))
        cu, lens, out = st["offsets"].tolist(), st["kv_lens"].tolist(), st["out"].double()
        front = st["prefix_table"].long() if P else None
        for s in range(case["seqs"]):
            n = cu[s + 1] - cu[s]
            if n == 0:
                continue
            own_pages = st["page_table"][s, : -(-lens[s] // page)].long()
            position = torch.arange(n, device="cuda") + P + lens[s] - n
            j = torch.arange(P + lens[s], device="cuda")
            hidden = (j[None, :] > position[:, None]) | ((j[None, :] <= position[:, None] - case["window"]) if case["window"] else False)
            for h in range(HK):
                def rows_of(pages, count):
                    kk = st["k_cache"][pages, h].double()   # page, chunk, key, 8
                    return kk.permute(0, 2, 1, 3).reshape(-1, D)[:count], st["v_cache"][pages, h].double().reshape(-1, D)[:count]

                parts = ([rows_of(front, P)] if P else []) + [rows_of(own_pages, lens[s])]
                kk, vv = (torch.cat([x[m] for x in parts]) for m in (0, 1))
                for g in range(h * (H // HK), (h + 1) * (H // HK)):
                    x = (st["q"][cu[s] : cu[s + 1], g * D : (g + 1) * D].double() @ kk.T.contiguous()) * st["scale"]
                    x = x.masked_fill(hidden, -math.inf)
                    w = torch.softmax(x, 1).nan_to_num(0.0)
                    out[cu[s] : cu[s + 1], g * D : (g + 1) * D] = w @ vv
        return out
    cu, V = st["offsets"].tolist(), case["vocab"]
    tokens, counts = st["tokens"].tolist(), []
    draft_tokens, ua, us, temps = (st[k].tolist() for k in ("draft_tokens", "u_accept", "u_sample", "temperature"))
    for s in range(case["seqs"]):
        n, taken = cu[s + 1] - cu[s], 0
        for i in range(n):
            r = cu[s] + i
            x, temp = st["target"][r].double(), temps[s]
            last = i == n - 1
            if temp <= 0:
                first = int((x == x.max()).nonzero()[0, 0])
                ok, choice = first == draft_tokens[r], first
            else:
                p = torch.softmax(x / temp, 0)
                if st["draft"] is not None:
                    q = torch.softmax(st["draft"][r].double() / temp, 0)
                else:
                    q = torch.zeros_like(p)
                    q[draft_tokens[r]] = 1.0
                ok = ua[r] * float(q[draft_tokens[r]]) < float(p[draft_tokens[r]])
                w = p if last else (p - q).clamp(min=0.0)
                if float(w.sum()) == 0:
                    w = p
                total = w.cumsum(0)
                over = (total > us[s] * float(total[-1])).nonzero()
                choice = int(over[0, 0]) if len(over) else int(w.nonzero()[-1, 0])
            if ok and not last:
                tokens[r], taken = draft_tokens[r], taken + 1
                continue
            tokens[r : cu[s + 1]] = [choice] + [-1] * (n - 1 - i)
            break
        counts.append(taken)
    return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32)]
