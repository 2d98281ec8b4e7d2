"""A slot that is allocated again at its own size keeps its memory: what a captured graph resolved stays valid."""
import numpy as np
import pytest

from smelt_amd import runtime as rt

pytestmark = pytest.mark.gpu


def test_graph_survives_a_slot_allocated_again_at_its_size():
    ctx = rt.Context()
    try:
        n = 1000
        ctx.alloc(1, n * 2); ctx.alloc(2, n * 2)
        rec = rt.make_record(ctx.pipeline("buffer_copy"), [(1, 0, 0), (2, 1, 0)], [(2, n)], (4, 1, 1), (256, 1, 1))
        graph, count = ctx.capture_decode(ctx.table([rec]))
        assert count == 1
        for seed in range(3):
            x = np.arange(n, dtype=np.uint16) * 7 + seed
            others = [s for s in range(3, 12)]
            for s in others:                       # allocations in between take whatever was freed
                ctx.alloc(s, n * 2)
            ctx.put(1, x)
            ctx.alloc(2, n * 2)
            assert not ctx.read(2, np.uint16, n).any()
            ctx.graph_launch(graph); ctx.wait()
            assert np.array_equal(ctx.read(2, np.uint16, n), x), seed
        ctx.graph_destroy(graph)
    finally:
        ctx.close()
