"""Forms of the decode-step kernels that ordinary sizes do not reach: every (rows, width, alignment) of attention on CUDA cores, the
selection whose weights do not fit shared memory, sums over a long run."""
import math

import numpy as np
import pytest
import torch

from decode_ref import HALF, TYPES, Values
from test_gpu_decode_attention import Case
from test_gpu_decode_evict import _case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mace_b200
    c = mace_b200.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 11])
@pytest.mark.parametrize("dim", [18, 32, 50, 64, 99, 128, 131, 256])
def test_attention_on_cuda_cores(ctx, name, group, dim):
    """One, two, four and eight rows a block, rows of up to 32, 64, 128 and 256 values, in words and one by one; on clusters, as runs and alone."""
    ctx.set_option("tensor_cores", 0)
    try:
        Case(ctx, name, [0, 1, 17, 400], 2 * group, 2, dim, 16, seed=dim + group).run().check()
        Case(ctx, name, [1500], group, 1, dim, 20, seed=dim + group, weights=False).run().check()
    finally:
        ctx.set_option("tensor_cores", 1)


@pytest.mark.parametrize("name,dim", [("f16", 18), ("bf16", 50), ("f32", 99), ("f16", 131), ("f32", 160), ("f32", 256), ("bf16", 252)])
@pytest.mark.parametrize("group", [1, 2, 4])
def test_attention_of_rows_that_no_tensor_core_takes(ctx, name, dim, group):
    Case(ctx, name, [700, 3, 0, 90], 2 * group, 2, dim, 16, seed=dim).run().check()


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "special"])
@pytest.mark.parametrize("length,budget,sinks,recent", [(400000, 1234, 4, 100), (330001, 330000, 0, 0), (700003, 300, 0, 300)])
def test_weights_that_no_shared_memory_holds(ctx, kind, length, budget, sinks, recent):
    """More than sixteen CTAs keep: every pass reads them again."""
    call, check = _case(ctx, "f16", [length, 350], 1, 8, 64, budget, sinks, recent, kind, seed=length)
    call()
    check()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("length", [2000, 120000])
def test_sums_over_a_long_run(ctx, name, length):
    """Even logits and positive values, so that every cut goes the same way; 64 sequences of 8 heads on the same pages, so that a run is as long
    as it gets.  A warp of four adds up to length / 64 chunks of 16 slots.  16-bit types: two products each, what an MMA cuts off is below
    2^-23 of the sum.  fp32: a chunk's six products (2^-23 each) by themselves, then a rounding of 2^-24.  Probabilities and their sum: powers of
    two, length / 32 roundings of 2^-24 in a lane.  Values as pairs: 3 x 2^-23 (fp32).  Joined from 8 parts or fewer at 2^-22."""
    dtype = TYPES[name][1]
    page, kv_heads, batch, dim = 64, 8, 64, 64
    pages = -(-length // page)
    rng = np.random.default_rng(length)
    base = torch.from_numpy(rng.uniform(0.9, 1.1, (pages, 1, page, dim)).astype(np.float32)).to(dtype)
    v = base.expand(pages, kv_heads, page, dim).contiguous()
    q = torch.zeros(batch, kv_heads, dim, dtype=dtype)
    dq, dk, dv, out = Values(ctx, q), Values(ctx, torch.zeros_like(v)), Values(ctx, v), Values(ctx, q)
    lse = Values(ctx, torch.zeros(batch, kv_heads))
    table, lengths = ctx.upload(np.tile(np.arange(pages, dtype=np.int32), (batch, 1))), ctx.upload(np.full(batch, length, np.int32))
    ctx.paged_attention(dq, dk, dv, table, lengths, out, batch, kv_heads, kv_heads, dim, pages, page, pages, length, 1.0, TYPES[name][0], lse=lse)
    ctx.sync()
    o = base.reshape(-1, dim)[:length].double().mean(0)
    chunks = length / 64
    rel = (chunks * 2.0 ** -24 + 9 * 2.0 ** -23 if name == "f32" else 2 * chunks * 2.0 ** -23) + 2 * chunks * 2.0 ** -24 + 2.0 ** -22
    assert ((out.get().double() - o).abs() <= o * (rel + HALF[name])).all()
    assert ((lse.get().double() - math.log(length)).abs() <= 2 * chunks * 2.0 ** -24 + 2.0 ** -20).all()
    for x in (dq, dk, dv, out, lse, table, lengths):
        x.free()


def test_two_graphs_share_scratch(ctx):
    """Captured steps of different sizes, one recorded before the scratch memory grew, replayed in turn with eager calls in between."""
    import ctypes as C

    from mace_b200.capi import lib
    L = lib()
    cases = [Case(ctx, "bf16", [3000, 5, 0], 8, 2, 128, 16, seed=1), Case(ctx, "f16", [9000] * 5, 32, 8, 128, 16, seed=2),
             Case(ctx, "f32", [1200, 700], 6, 3, 50, 16, seed=3)]
    graphs = []
    for c in cases:
        c.run()
        assert L.mb_graph_begin(ctx.h) == 0
        c.call()
        graph = C.c_void_p()
        assert L.mb_graph_end(ctx.h, C.byref(graph)) == 0
        graphs.append(graph)
    for _ in range(3):
        for c, graph in zip(cases, graphs):
            for v in (c.out, c.lse):
                ctx.h2d(v.buf, np.full(v.nbytes, 0x7f, np.uint8))
            ctx.h2d(c.w_out.buf, np.full(c.w_out.shape, -5.0, np.float32))
            ctx.sync()
        for graph in graphs[::-1] + graphs:
            assert L.mb_graph_launch(ctx.h, graph) == 0
        cases[0].call()
        ctx.sync()
        for c in cases:
            c.check()
    for graph in graphs:
        L.mb_graph_destroy(ctx.h, graph)
