"""Serving operators without a GPU: pipeline names, what the emitters refuse, frequency tables, the attention's work partition."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from smelt_amd import compiler as cc
from smelt_amd import runtime as rt

HERE = os.path.dirname(os.path.abspath(__file__))
B = cc.bind


@pytest.mark.parametrize("name,symbol", [
    ("rope_half_d256_r64", "smelt_rope_vec_f16"), ("rope_interleaved_d100_r20@bf16", "smelt_rope_vec_bf16"),
    ("paged_kv_append_half_d128_r0_kv8_p16", "smelt_paged_append_vec_f16"),
    ("paged_kv_append_q_interleaved_d64_r64_kv1_p256", "smelt_paged_append_vec_f16"),
    ("paged_attention_d256_h24_kv4_p64", "smelt_attention_stream16_d256_f16"),
    ("paged_attention_shared_d64_h6_kv2_p16@bf16", "smelt_attention_stream16_d64_bf16"),
    ("verify_drafts", "smelt_verify_stats_f16"), ("verify_drafts_given@bf16", "smelt_verify_stats_bf16")])
def test_names_resolve(name, symbol):
    rc, sym, kinds = cc.resolve_pipeline_name(name)
    assert rc == 0 and sym == symbol and set(kinds) <= set("PUF")


@pytest.mark.parametrize("name,code", [
    ("rope_half_d256_r63", -3), ("rope_half_d64_r128", -3), ("rope_half_d64_r0", -3), ("rope_half_d2000_r64", -3), ("rope_d64_r64", -4),
    ("rope_half_d64", -4), ("rope_half_d64_r64_x", -4), ("paged_kv_append_half_d96_r64_kv4_p64", -3),
    ("paged_kv_append_half_d64_r64_kv4_p24", -3), ("paged_kv_append_half_d64_r64_kv0_p16", -3), ("paged_kv_append_half_d64_r64_kv4", -4),
    ("paged_attention_d80_h8_kv8_p16", -3), ("paged_attention_d64_h8_kv3_p16", -3), ("paged_attention_d64_h0_kv1_p16", -3),
    ("paged_attention_d64_h8_kv2_p48", -3), ("paged_attention_d64_h8_kv2_p99999999999", -4), ("paged_attention", -4), ("verify_drafts_x", -4)])
def test_names_refused(name, code):
    assert cc.resolve_pipeline_name(name)[0] == code


def refused(call, *words):
    with pytest.raises(cc.EmitError) as e:
        call()
    for w in words:
        assert w in e.value.message, e.value.message


def test_rope_refusals():
    em = cc.Emitter()
    ok = dict(tokens=4, heads=8, head_dim=64, rotary_dim=64)
    em.rope(B(1), B(2), B(3), B(4), **ok)
    em.rope(B(1), B(1), B(3), B(4), **ok)                                         # in place
    refused(lambda: em.rope(B(1), B(2), B(3), B(4), **{**ok, "heads": 0}), "heads")
    refused(lambda: em.rope(B(1), B(2), B(3), B(4), **{**ok, "tokens": -1}), "negative")
    refused(lambda: em.rope(B(1), B(2), B(3), B(4), x_stride=500, **ok), "stride")
    refused(lambda: em.rope(B(1), B(2), B(3), B(4), y_stride=511, **ok), "stride")
    refused(lambda: em.rope(B(1), B(1), B(3), B(4), x_stride=1024, **ok), "overlaps")
    refused(lambda: em.rope(B(1), B(1, 64), B(3), B(4), **ok), "overlaps")
    refused(lambda: em.rope(B(1), B(3), B(3), B(4), **ok), "overlaps")
    refused(lambda: em.rope(B(1), B(2), B(3), B(4), **{**ok, "rotary_dim": 65}), "rotated")
    refused(lambda: em.rope(B(1), B(2), B(3), B(4), tokens=4, heads=1024, head_dim=1024, rotary_dim=64), "pieces")
    assert len(em.records()) == 2


def test_append_refusals():
    em = cc.Emitter()

    def go(**kw):
        a = dict(k=B(1), v=B(2), positions=B(3), slots=B(4), table=B(5), k_cache=B(6), v_cache=B(7), tokens=3, kv_heads=2, head_dim=64, rotary_dim=32, page_size=16, pages=10)
        em.paged_kv_append(**{**a, **kw})

    go()
    go(q=B(8), q_out=B(8), q_heads=4)
    go(rotary_dim=0)
    refused(lambda: go(q=B(8)), "q without q_out")
    refused(lambda: go(q=B(8), q_out=B(9), q_heads=0), "heads")
    refused(lambda: go(q=B(8), q_out=B(1), q_heads=4), "overlaps")
    refused(lambda: go(pages=0), "pool")
    refused(lambda: go(pages=2 ** 28), "pool")
    refused(lambda: go(kv_stride=100), "stride")
    refused(lambda: go(v_stride=64), "stride")
    refused(lambda: go(v_cache=B(6)), "overlaps")
    refused(lambda: go(k_cache=B(1)), "overlaps")
    refused(lambda: go(head_dim=96), "64, 128 or 256")
    refused(lambda: go(page_size=8), "pages hold")


def test_attention_refusals():
    em = cc.Emitter()

    def go(**kw):
        a = dict(q=B(1), k_cache=B(2), v_cache=B(3), page_table=B(4), kv_lens=B(5), offsets=B(6), out=B(7), tokens=4, sequences=2, heads=8, kv_heads=2, head_dim=128,
                 page_size=64, pages=100, pages_per_sequence=20, scale=0.1)
        em.paged_attention(**{**a, **kw})

    go()
    go(prefix_table=B(8), prefix_len=B(9), prefix_pages=3)
    go(prefix_table=B(8), prefix_len=B(9), prefix_pages=0)
    refused(lambda: go(prefix_table=B(8)), "half a prefix")
    refused(lambda: go(out=B(1)), "overlaps")
    refused(lambda: go(out=B(3)), "overlaps")
    refused(lambda: go(scale=float("inf")), "finite")
    refused(lambda: go(scale=float("nan")), "finite")
    refused(lambda: go(q_stride=1000), "stride")
    refused(lambda: go(pages_per_sequence=0), "page")
    refused(lambda: go(pages=0), "pool")
    refused(lambda: go(heads=7), "multiple")
    refused(lambda: go(window=-1), "negative")
    refused(lambda: go(pages_per_sequence=2 ** 25), "positions")


def test_verify_refusals():
    em = cc.Emitter()

    def go(**kw):
        a = dict(target=B(1), draft_tokens=B(2), offsets=B(3), u_accept=B(4), u_sample=B(5), temperature=B(6), tokens=B(7), counts=B(8), rows=5, sequences=2, vocab=100)
        em.verify_drafts(**{**a, **kw})

    go()
    go(draft=B(9))
    go(draft=B(1))                       # a draft model that is the target
    refused(lambda: go(stride=99), "stride")
    refused(lambda: go(vocab=0), "vocabulary")
    refused(lambda: go(rows=70000), "65535")
    refused(lambda: go(tokens=B(2)), "overlaps")
    refused(lambda: go(counts=B(7)), "overlaps")
    refused(lambda: go(rows=65535, vocab=10 ** 7), "workspace")


def test_table_for_looks_pipelines_up_by_type():
    em = cc.Emitter(act_dtype=rt.ACT_BF16)
    em.rope(B(1), B(2), B(3), B(4), tokens=4, heads=8, head_dim=64, rotary_dim=64)
    em16 = cc.Emitter()
    em16.rope(B(1), B(2), B(3), B(4), tokens=4, heads=8, head_dim=64, rotary_dim=64, dynamic=True)

    class Stub:
        names = ["something else"]

        def pipeline(self, name):
            if name not in self.names:
                self.names.append(name)
            return self.names.index(name)

    ctx = Stub()
    assert [r.pipeline for r in em.table_for(ctx)] == [1] and [r.pipeline for r in em16.table_for(ctx)] == [2]
    assert ctx.names[1:] == ["rope_half_d64_r64@bf16", "rope_half_d64_r64@f16"]
    assert em16.records()[0].constants[0].kind == rt.CONST_SEQ_LEN


@pytest.mark.parametrize("rot", [2, 64, 96, 128])
def test_rope_tables(rot):
    i = np.arange(rot // 2)
    f = 10000.0 ** (-2.0 * i / rot)
    near = dict(rtol=1e-14, atol=0)
    t, a = cc.rope_table(rot)
    assert a == 1.0 and np.allclose(t[:rot // 2], f, **near)
    assert np.allclose(cc.rope_table(rot, kind=cc.ROPE_LINEAR, factor=8.0)[0][:rot // 2], f / 8, **near)
    if rot > 2:
        t = cc.rope_table(rot, kind=cc.ROPE_BASE, factor=8.0)[0]
        assert t[0] == 1.0 and np.isclose(t[-1], f[-1] / 8, rtol=1e-12)
    t, a = cc.rope_table(rot, base=500000.0, kind=cc.ROPE_BANDS, factor=8.0, positions=8192.0, low=1.0, high=4.0)
    g = 500000.0 ** (-2.0 * i / rot)
    turns = 8192.0 * g / (2 * np.pi)
    keep = np.clip((turns - 1.0) / 3.0, 0, 1)
    assert a == 1.0 and np.allclose(t[:rot // 2], keep * g + (1 - keep) * g / 8, rtol=1e-12)
    t, a = cc.rope_table(rot, kind=cc.ROPE_PARTS, factor=4.0, positions=4096.0, low=1.0, high=32.0)
    lo, hi = (rot * np.log(4096.0 / (n * 2 * np.pi)) / (2 * np.log(10000.0)) for n in (32.0, 1.0))
    lo, hi = max(np.floor(lo), 0), min(np.ceil(hi), rot - 1)
    keep = 1 - np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
    assert np.isclose(a, 0.1 * np.log(4.0) + 1, rtol=1e-6) and np.allclose(t[:rot // 2], keep * f + (1 - keep) * f / 4, rtol=1e-12)


def test_rope_table_refusals():
    for kw in (dict(rotary_dim=0), dict(rotary_dim=7), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, kind=9, factor=2.0), dict(rotary_dim=8, kind=cc.ROPE_LINEAR, factor=0.0),
               dict(rotary_dim=8, kind=cc.ROPE_BANDS, factor=2.0, low=4.0, high=4.0), dict(rotary_dim=8, kind=cc.ROPE_PARTS, factor=2.0, positions=0.0),
               dict(rotary_dim=2, kind=cc.ROPE_BASE, factor=2.0), dict(rotary_dim=8, base=float("nan"))):
        with pytest.raises(ValueError):
            cc.rope_table(**kw)


@pytest.fixture(scope="module")
def partition(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("partition") / "libpartition.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", out, os.path.join(HERE, "serving_partition_check.cpp")], check=True)
    lib = C.CDLL(out)
    lib.check_owners.restype = C.c_uint64
    lib.check_owners.argtypes = [C.c_uint32, C.c_uint32, C.c_uint32]
    return lib


WHOLE, OWN, PREFIX = range(3)


def entries(lib, offsets, lens, tokens, group=1, kv_heads=1, shift=4, width=4, prefix=None, prefix_pages=0, part=WHOLE, row_tile=32, window=0):
    offsets, lens = np.array(offsets, np.int32), np.array(lens, np.int32)
    out, tiles, units = np.zeros((len(lens) + 1, 8), np.int64), np.zeros((100000, 2), np.int64), C.c_uint64()
    p = None if prefix is None else C.byref(C.c_int32(prefix))
    i32p, i64p = C.POINTER(C.c_int32), C.POINTER(C.c_int64)
    n = lib.check_entries(offsets.ctypes.data_as(i32p), lens.ctypes.data_as(i32p), len(lens), tokens, group, kv_heads, shift, width, p, prefix_pages, part, row_tile, window,
                          out.ctypes.data_as(i64p), tiles.ctypes.data_as(i64p), C.byref(units))
    keys = ("first", "tokens", "row_tiles", "front", "own", "front_tiles", "tiles", "sequence")
    got = [dict(zip(keys, r)) for r in out[:n].tolist()]
    at = 0
    for e in got:
        e["of_rows"] = [tuple(t) for t in tiles[at:at + e["row_tiles"]].tolist()]
        at += e["row_tiles"]
    assert units.value == kv_heads * sum(hi - lo for e in got for lo, hi in e["of_rows"])
    return got


def test_entries_are_cut_to_what_the_tables_hold(partition):
    # lengths past the table, negative lengths, offsets outside the rows or falling
    e = entries(partition, [0, 3, 3, -5, 900], [1000, 7, -4, 64], tokens=10, group=12, kv_heads=2)
    assert [x["own"] for x in e] == [64, 7, 0, 64] and [x["tokens"] for x in e] == [3, 0, 0, 10]
    assert [x["first"] for x in e] == [0, 3, 3, 0] and [x["tiles"] for x in e] == [2, 1, 0, 2] and [x["row_tiles"] for x in e] == [2, 0, 0, 4]
    # a prefix longer than its table; the prefix entry covers the rows that belong to a sequence
    e = entries(partition, [0, 1, 2], [5, 0], tokens=4, prefix=1 << 30, prefix_pages=3, part=PREFIX)
    assert len(e) == 1 and {k: e[0][k] for k in ("first", "tokens", "row_tiles", "front", "own", "tiles", "sequence")} == dict(
        first=0, tokens=2, row_tiles=1, front=48, own=0, tiles=2, sequence=-1)
    assert e[0]["of_rows"] == [(0, 2)]
    e = entries(partition, [0, 1, 2], [5, 0], tokens=4, prefix=1 << 30, prefix_pages=3, part=OWN)
    assert [x["tiles"] for x in e] == [1, 0] and [x["of_rows"] for x in e] == [[(0, 1)], [(0, 1)]]     # (rows without keys are still written)
    assert entries(partition, [0, 1], [0], tokens=4, prefix=-3, prefix_pages=3, part=PREFIX)[0]["row_tiles"] == 0
    e = entries(partition, [0, 1], [33], tokens=4, prefix=40, prefix_pages=3)
    assert (e[0]["front_tiles"], e[0]["tiles"]) == (2, 4)


@pytest.mark.parametrize("part", [WHOLE, OWN])
@pytest.mark.parametrize("prefix", [0, 1, 31, 32, 33, 100])
@pytest.mark.parametrize("window", [0, 1, 30, 64, 1000])
def test_row_tiles_cover_what_their_rows_see(partition, part, prefix, window):
    """Against the definition, key by key: the key tiles of a row tile are the smallest run that holds every key one of its rows sees."""
    for n, own, group, row_tile in ((1, 1, 1, 32), (1, 100, 6, 32), (70, 70, 1, 32), (70, 200, 3, 128), (40, 33, 2, 32), (9, 0, 4, 32), (300, 310, 4, 256)):
        e = entries(partition, [0, n], [own], tokens=n, group=group, width=64, prefix=prefix, prefix_pages=7, part=part, row_tile=row_tile, window=window)[0]
        assert e["row_tiles"] == -(-n * group // row_tile)
        front = prefix if part == WHOLE else 0
        tile_of = [j // 32 for j in range(front)] + [-(-front // 32) + j // 32 for j in range(own)]
        for r, (lo, hi) in enumerate(e["of_rows"]):
            seen = set()
            for row in range(r * row_tile, min((r + 1) * row_tile, n * group)):
                p = prefix + own - n + row // group
                for k, t in enumerate(tile_of):
                    j = k if part == WHOLE else prefix + k
                    if j <= p and (not window or j > p - window):
                        seen.add(t)
            assert hi > lo >= 0
            if seen:
                assert (lo, hi) == (min(seen), max(seen) + 1), (n, own, group, row_tile, r)
            else:
                assert hi - lo == 1 and (lo < max(e["tiles"], 1))


def test_every_unit_has_one_workgroup(partition):
    for units in (1, 2, 3, 4, 5, 63, 64, 1000, 1021, 4096, 100003):
        for workgroups in (1, 2, 7, 256, 512):
            for least in (1, 4):
                assert partition.check_owners(units, workgroups, least) == 0, (units, workgroups, least)


def test_reciprocal_division_is_exact(partition):
    for d in (1, 2, 3, 5, 7, 12, 17, 24, 96, 100, 255, 256, 1000, 4095, 4097, 65535):
        assert partition.check_reciprocal(d, min(2 ** 32 // max(d, 1) - 1, 70000)) == 0, d


@pytest.mark.parametrize("tokens,group,kv_heads,prefix", [(64, 6, 4, 8192), (1, 1, 1, 1), (24, 4, 8, 2500), (1000, 8, 8, 300), (5, 3, 2, 40), (4096, 6, 4, 65), (700, 16, 1, 100000)])
@pytest.mark.parametrize("row_tile", [16, 32, 128, 256])
@pytest.mark.parametrize("slots", [0, 1, 100, 512])
def test_every_part_of_the_prefix_has_one_workgroup(partition, tokens, group, kv_heads, prefix, row_tile, slots):
    offsets, workgroups, least = np.array([0, tokens], np.int32), 256, 8
    segments = -(-tokens * group // row_tile) * kv_heads
    for rounds in (1, 2):
        grid = -(-max(segments, workgroups * rounds) // 8) * 8          # what the launch has
        parts, jobs = C.c_uint32(), np.zeros((grid, 3), np.int32)
        n = partition.check_jobs(offsets.ctypes.data_as(C.POINTER(C.c_int32)), tokens, 1, group, kv_heads, prefix, row_tile, workgroups, rounds, slots, least, 8, grid,
                                 C.byref(parts), jobs.ctypes.data_as(C.POINTER(C.c_int32)))
        parts = parts.value
        assert n == segments * parts and len({tuple(j) for j in jobs[:n].tolist()}) == n
        assert jobs[:n].min() >= 0 and tuple(jobs[:n].max(0) + 1) == (segments // kv_heads, kv_heads, parts)
        assert parts == 1 or (segments * parts <= min(slots, workgroups * rounds) and -(-prefix // 32) // parts >= least)


def test_a_prefix_of_no_rows_has_no_parts(partition):
    for offsets, prefix in (([0, 0], 100), ([0, 5], 0)):
        parts, jobs = C.c_uint32(7), np.zeros((256, 3), np.int32)
        assert partition.check_jobs(np.array(offsets, np.int32).ctypes.data_as(C.POINTER(C.c_int32)), 5, 1, 2, 2, prefix, 32, 256, 1, 512, 8, 8, 256, C.byref(parts),
                                    jobs.ctypes.data_as(C.POINTER(C.c_int32))) == 0
        assert parts.value == 0


def test_launches_that_are_too_wide_are_refused():
    em = cc.Emitter()
    em.rope(B(1), B(2), B(3), B(4), tokens=30_000_000, heads=1, head_dim=256, rotary_dim=256)
    refused(lambda: em.rope(B(1), B(2), B(3), B(4), tokens=60_000_000, heads=1, head_dim=256, rotary_dim=256), "threads")
    # a workgroup for each of many segments that there can be, whatever the lengths are
    att = dict(q=B(1), k_cache=B(2), v_cache=B(3), page_table=B(4), kv_lens=B(5), offsets=B(6), out=B(7), heads=64, kv_heads=64, head_dim=64, page_size=16, pages=100,
               pages_per_sequence=1, scale=0.1)
    em.paged_attention(**att, tokens=10_000_000, sequences=100)
    refused(lambda: em.paged_attention(**att, tokens=33_000_000, sequences=200_000), "threads")


@pytest.mark.parametrize("part", [WHOLE, OWN])
@pytest.mark.parametrize("prefix", [0, 20])
def test_the_widest_windows_hide_nothing(partition, part, prefix):
    """Windows up to 2^31 - 1, also where rows stand before the first key (fewer keys than rows): the key tiles of no window."""
    for n, own, group, row_tile in ((80, 70, 1, 128), (80, 70, 6, 256), (300, 2, 1, 32), (40, 0, 2, 16), (1, 1, 1, 32), (9, 500, 4, 32)):
        a = dict(offsets=[0, n], lens=[own], tokens=n, group=group, width=64, prefix=prefix, prefix_pages=7, part=part, row_tile=row_tile)
        want = entries(partition, **a)[0]
        for window in (1000, 2 ** 30, 2 ** 31 - n, 2 ** 31 - 2, 2 ** 31 - 1):
            assert entries(partition, **a, window=window)[0] == want, (n, own, group, row_tile, window)


@pytest.mark.parametrize("tokens", [1, 2, 64])
@pytest.mark.parametrize("interleaved", [False, True])
def test_q_is_rotated_in_place_within_fused_rows(tokens, interleaved):
    """Rows [q | k | v] of one projection: q_out may be q itself, or rows elsewhere in the fused ones that no other operand has."""
    em, (h, kv, d) = cc.Emitter(), (8, 2, 64)
    row = (h + 2 * kv) * d

    def go(q_at=0, q_out_at=0, k_at=h * d, v_at=(h + kv) * d, stride=row, q_out_stride=None, q_out_slot=1, **kw):
        em.paged_kv_append(B(1, 2 * k_at), B(1, 2 * v_at), B(3), B(4), B(5), B(6), B(7), tokens=tokens, kv_heads=kv, head_dim=d, rotary_dim=d, page_size=16, pages=10, kv_stride=stride,
                           q=B(1, 2 * q_at), q_out=B(q_out_slot, 2 * q_out_at), q_heads=h, q_stride=stride, q_out_stride=stride if q_out_stride is None else q_out_stride,
                           interleaved=interleaved, **kw)

    go()
    go(q_at=2 * kv * d, q_out_at=2 * kv * d, k_at=0, v_at=kv * d)                  # [k | v | q]
    go(q_at=kv * d, q_out_at=kv * d, k_at=0, v_at=(h + kv) * d)                    # [k | q | v]
    go(stride=row + 8)
    go(stride=2 * row, q_out_at=row)                                              # columns of their own
    refused(lambda: go(k_at=h * d - 1), "overlaps")                               # one value of q is k's
    refused(lambda: go(q_out_at=kv * d), "overlaps")                              # q's rows, but not the same ones
    refused(lambda: go(stride=2 * row, q_out_at=row - 1), "overlaps")
    if tokens > 1:
        refused(lambda: go(q_out_stride=row + 8), "overlaps")
        refused(lambda: go(q_out_at=row), "overlaps")                             # a row down: where later rows of q are
    refused(lambda: go(q_out_slot=6), "overlaps")
    em.rope(B(1), B(1), B(3), B(4), tokens, h, d, d, x_stride=row, y_stride=row)
    em.rope(B(1, 2 * h * d), B(1, 2 * h * d), B(3), B(4), tokens, kv, d, d, x_stride=row, y_stride=row)
    em.rope(B(1, 2 * h * d), B(1, 2 * (h + kv) * d), B(3), B(4), tokens, kv, d, d, x_stride=row, y_stride=row)


def test_rows_overlap_where_they_share_a_byte():
    """What is refused, against the sets of values that the rows hold."""
    em = cc.Emitter()
    dim, seen = 2, set()
    for tokens in (1, 2, 3):
        for heads in (1, 2):
            for stride in range(heads * dim, 8):
                for stride_y in (stride, stride + 1):
                    for x in (0, 13):
                        for y in range(0, 30):
                            rows = [{at + t * s + i for t in range(tokens) for i in range(heads * dim)} for at, s in ((x, stride), (y, stride_y))]
                            overlap = bool(rows[0] & rows[1]) and not (x == y and stride == stride_y)
                            span = [range(min(r), max(r) + 1) for r in rows]
                            if stride != stride_y and span[0][0] <= span[1][-1] and span[1][0] <= span[0][-1]:
                                overlap = True                                     # (different strides: the runs are compared)
                            call = lambda: em.rope(B(1, 2 * x), B(1, 2 * y), B(3), B(4), tokens, heads, dim, dim, x_stride=stride, y_stride=stride_y)   # noqa: E731
                            if overlap:
                                refused(call, "overlaps")
                            else:
                                call()
                            seen.add(overlap)
    assert seen == {False, True}


def test_rope_table_defaults():
    """What each scaling keeps when the caller does not say: 1 to 4 turns of bands, 1 to 32 of parts."""
    same = lambda kind, high: np.array_equal(cc.rope_table(128, kind=kind, factor=4.0)[0], cc.rope_table(128, kind=kind, factor=4.0, positions=8192.0, low=1.0, high=high)[0])   # noqa: E731
    assert same(cc.ROPE_BANDS, 4.0) and not same(cc.ROPE_BANDS, 32.0)
    assert same(cc.ROPE_PARTS, 32.0) and not same(cc.ROPE_PARTS, 4.0)
    assert not np.array_equal(cc.rope_table(128, kind=cc.ROPE_PARTS, factor=4.0, high=8.0)[0], cc.rope_table(128, kind=cc.ROPE_PARTS, factor=4.0)[0])
