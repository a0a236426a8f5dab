"""Attention of one token over the paged cache against a 64-bit form."""
import math

import numpy as np
import pytest
import torch

from decode_ref import HALF, TINY, TYPES, Values, attend, paged, tensor

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mace_b200
    c = mace_b200.Context(0)
    yield c
    c.close()


class Case:
    def __init__(self, ctx, name, lengths, heads, kv_heads, dim, page, seed=0, fill=float("nan"), std=2.0, width=None, max_length=None,
                 weights=True, window=0, offset=0, scale=None):
        rng = np.random.default_rng(seed)
        self.ctx, self.name, self.lengths, self.heads, self.kv_heads, self.dim, self.page = ctx, name, lengths, heads, kv_heads, dim, page
        self.window, self.scale = window, 1.0 / math.sqrt(dim) if scale is None else scale
        batch = len(lengths)
        k, v, self.table, self.rows = paged(rng, name, lengths, kv_heads, dim, page, width, fill=fill)
        self.q = tensor(rng, name, batch, heads, dim, std=std)
        self.max_length = max(list(lengths) + [0]) if max_length is None else max_length
        self.stride = max(self.max_length, 1) + 3
        self.pages = k.shape[0]
        self.w_in = rng.random((batch, kv_heads, self.stride)).astype(np.float32) if weights else None
        self.dk, self.dv, self.dq = Values(ctx, k, offset), Values(ctx, v, offset), Values(ctx, self.q, offset)
        self.dt, self.dn = ctx.upload(self.table), ctx.upload(np.array(lengths, np.int32))
        self.out = Values(ctx, torch.full((batch, heads, dim), 9.0, dtype=k.dtype), offset)
        self.lse = Values(ctx, torch.full((batch, heads), 9.0))
        self.dw = ctx.upload(self.w_in) if weights else None
        self.w_out = Values(ctx, torch.full((batch, kv_heads, self.stride), -5.0)) if weights else None

    def call(self, **kw):
        a = dict(lse=self.lse, weights_in=self.dw, weights_out=self.w_out, weights_stride=self.stride, window=self.window)
        a.update(kw)
        self.ctx.paged_attention(self.dq, self.dk, self.dv, self.dt, self.dn, self.out, len(self.lengths), self.heads, self.kv_heads,
                                 self.dim, self.pages, self.page, self.table.shape[1], self.max_length, self.scale, TYPES[self.name][0], **a)

    def run(self, **kw):
        self.call(**kw)
        self.ctx.sync()
        return self

    def check(self, lengths=None):
        """Per logit: dim products and sums, the factor, the exponential and its argument in powers of two: (dim + 16) x 2^-24 of the
        largest logit's terms (16-bit products on the tensor cores are exact, their sums cut off at 2^-23: the same).  A
        probability is off by twice that (its own logit and the sum), and by the sums over slots: a warp adds a quarter of a run at most,
        then warps and runs, each 2^-23 at most.  16-bit probabilities are kept as pairs of values: 2^-16 of them lost with bf16.
        fp32 values on the tensor cores are pairs of tf32 numbers: what a product loses is 2^-20 of it (two remainders cut at 2^-21).
        Then one rounding."""
        group = self.heads // self.kv_heads
        out, lse = self.out.get().double(), self.lse.get().double()
        weights = self.w_out.get().double() if self.w_out is not None else None
        for b, n in enumerate(self.lengths if lengths is None else lengths):
            begin = max(0, n - self.window) if self.window else 0
            k, v = self.rows[b]
            for h in range(self.kv_heads):
                mine = slice(h * group, (h + 1) * group)
                o, l, p, terms, size = attend(self.q[b, mine], k[:n, h], v[:n, h], self.scale, begin)
                logit = (self.dim + 16) * 2.0 ** -23 * (terms + 1) + (2.0 ** -20 * terms if self.name == "f32" else 0)
                rel = 2 * logit + (n / 4 + 150) * 2.0 ** -23 + (2.0 ** -16 if self.name == "bf16" else 2.0 ** -20)
                assert ((out[b, mine] - o).abs() <= size * rel + o.abs() * HALF[self.name] + TINY[self.name] + 1e-30).all()
                if n == 0:
                    assert (lse[b, mine] == -math.inf).all() and (out[b, mine] == 0).all()
                else:
                    assert ((lse[b, mine] - l).abs() <= logit + (n / 4 + 150) * 2.0 ** -23 + l.abs() * 2.0 ** -22).all()
                if weights is not None:
                    want = torch.from_numpy(self.w_in[b, h, :n].astype(np.float64))
                    off = torch.zeros(n, dtype=torch.float64)
                    want[begin:] += p.sum(0)
                    off[begin:] = p.sum(0) * rel
                    assert ((weights[b, h, :n] - want).abs() <= off + want.abs() * 2.0 ** -22).all()
                    assert (weights[b, h, n:] == -5.0).all()


HEADS = [(1, 1), (2, 1), (3, 1), (8, 2), (8, 8), (14, 2), (32, 4), (17, 1), (20, 1), (24, 1), (32, 1), (40, 1), (56, 1)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
@pytest.mark.parametrize("dim", [64, 128])
def test_heads(ctx, name, heads, kv_heads, dim):
    """Groups of one to forty; lengths of zero, one, tile borders; unused rows hold NaN."""
    Case(ctx, name, [0, 1, 15, 16, 17, 63, 64, 65, 200], heads, kv_heads, dim, 16, seed=heads).run().check()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [1, 2, 8, 20, 32, 33, 40, 72, 96, 100, 130, 136, 200, 248, 256])
def test_dims(ctx, name, dim):
    Case(ctx, name, [5, 130], 6, 2, dim, 8, seed=dim, fill=float("inf")).run().check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("page", [1, 3, 16, 20, 100, 1024])
def test_pages(ctx, name, page):
    Case(ctx, name, [333, 1, 100], 4, 2, 64, page, seed=page).run().check()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("batch,heads,kv_heads,dim,longest", [(1, 8, 1, 128, 5000), (2, 4, 4, 64, 3001), (1, 16, 2, 256, 2500), (70, 4, 2, 64, 700)])
def test_long(ctx, name, batch, heads, kv_heads, dim, longest):
    """Many runs per head, joined; sequences far shorter than the longest."""
    rng = np.random.default_rng(longest)
    lengths = [longest] + [int(n) for n in rng.integers(0, longest, batch - 1)]
    Case(ctx, name, lengths, heads, kv_heads, dim, 32, seed=batch).run().check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_many_sequences(ctx, name):
    """More sequences than every block reads the lengths of, short ones and a long one."""
    rng = np.random.default_rng(8)
    lengths = [int(n) for n in rng.integers(0, 20, 1100)]
    lengths[500] = 9000
    Case(ctx, name, lengths, 4, 2, 64, 16, seed=8).run().check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("batch", [127, 128, 129, 300])
def test_ragged_batches(ctx, name, batch):
    """Sequences beyond one round of the blocks' sum over lengths, some empty."""
    rng = np.random.default_rng(batch)
    lengths = [int(n) for n in rng.integers(0, 300, batch)]
    lengths[batch // 3], lengths[-1] = 3000, 0
    Case(ctx, name, lengths, 2, 1, 64, 16, seed=batch, weights=False).run().check()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_on_cuda_cores(ctx, name):
    """The kernel of odd rows serves every row ("tensor_cores" 0)."""
    ctx.set_option("tensor_cores", 0)
    try:
        Case(ctx, name, [0, 1, 100, 1000], 10, 2, 128, 16, seed=3).run().check()
    finally:
        ctx.set_option("tensor_cores", 1)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page,window", [
    (4, 4, 128, 16, 0), (16, 4, 128, 32, 0), (64, 4, 128, 20, 0), (28, 4, 128, 16, 2000), (8, 8, 64, 16, 0), (40, 8, 64, 100, 4001), (160, 8, 64, 64, 0),
    (12, 4, 256, 16, 0), (64, 4, 256, 16, 5000), (6, 6, 120, 16, 0), (7, 7, 99, 16, 0)])
def test_runs_joined_through_memory(ctx, name, heads, kv_heads, dim, page, window):
    """More than fits clusters: runs cut by the lengths, joined by the block that arrives last; empty and short sequences among long ones."""
    Case(ctx, name, [9000, 0, 1, 4000, 8999, 130, 64], heads, kv_heads, dim, page, seed=dim + heads, window=window).run().check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("window", [1, 7, 64, 500, 100000])
def test_window(ctx, name, window):
    Case(ctx, name, [0, 1, 8, 65, 1300], 8, 2, 64, 16, window=window, seed=window).run().check()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_steep_logits(ctx, name):
    """Logits of hundreds, in rising and falling order: the running maximum moves at every step or never again."""
    c = Case(ctx, name, [700, 700], 8, 2, 64, 16, std=1.0, seed=4)
    for order in (1, -1):
        ramp = torch.linspace(-8, 8, 700).flip(0) if order < 0 else torch.linspace(-8, 8, 700)
        for b in range(2):
            k = ramp[:, None, None].expand(700, 2, 64).to(c.rows[b][0].dtype)
            c.rows[b] = (k.contiguous(), c.rows[b][1])
        pool = c.dk.get()
        for b in range(2):
            for j in range(700):
                pool[int(c.table[b, j // 16]), :, j % 16] = c.rows[b][0][j]
        c.dk = Values(c.ctx, pool)
        c.q = torch.full_like(c.q, 4.0)
        c.dq = Values(c.ctx, c.q)
        c.w_out = Values(c.ctx, torch.full((2, 2, c.stride), -5.0))
        c.run().check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_rows_without_a_finite_logit(ctx, name):
    """Every key is -inf along the query: no probability, out 0 and lse -inf, weights as they were."""
    c = Case(ctx, name, [40], 4, 2, 64, 16, seed=2)
    pool = c.dk.get()
    pool[:] = 0
    pool[..., 0] = -math.inf
    c.dk, c.q = Values(c.ctx, pool), torch.zeros_like(c.q)
    c.q[..., 0] = 1.0
    c.q[..., 1:] = 1.0
    c.dq = Values(c.ctx, c.q)
    c.run()
    assert (c.out.get() == 0).all() and (c.lse.get() == -math.inf).all()
    assert np.array_equal(c.w_out.get().numpy()[..., :40], c.w_in[..., :40])


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_single_infinite_keys(ctx, name):
    """A key that is -inf along positive queries leaves its slot without weight; the other slots share theirs as if it were not there."""
    c = Case(ctx, name, [100], 4, 2, 64, 16, seed=5, weights=False)
    c.q = c.q.abs() + 0.5
    c.dq = Values(c.ctx, c.q)
    pool = c.dk.get()
    gone = [3, 17, 40, 99]
    for j in gone:
        pool[int(c.table[0, j // 16]), :, j % 16, 7] = -math.inf
    c.dk = Values(c.ctx, pool)
    c.run()
    stay = [j for j in range(100) if j not in gone]
    c.rows = [tuple(r[stay] for r in c.rows[0])]
    c.check([len(stay)])


def test_nan_in_a_used_slot_stays_in_its_head(ctx):
    for name in ("f32", "bf16"):
        c = Case(ctx, name, [100], 4, 2, 64, 16, seed=2)
        pool = c.dk.get()
        pool[int(c.table[0, 2]), 1, 5, 3] = math.nan
        c.dk = Values(c.ctx, pool)
        c.run()
        out, lse = c.out.get(), c.lse.get()
        assert torch.isnan(out[0, 2:]).all() and torch.isnan(lse[0, 2:]).all()
        assert not torch.isnan(out[0, :2]).any() and not torch.isnan(lse[0, :2]).any()


@pytest.mark.parametrize("name,offset", [("f32", 1), ("bf16", 1), ("f16", 4), ("bf16", 2)])
def test_alignment(ctx, name, offset):
    Case(ctx, name, [77, 300], 8, 2, 64, 16, offset=offset).run().check()


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_strides_of_queries_and_outputs(ctx, name):
    """q from rows that hold keys and values too, out with room between the rows."""
    c = Case(ctx, name, [20, 33, 1], 4, 2, 64, 16, weights=False)
    wide = torch.full((3, 400), 7.0, dtype=c.q.dtype)
    wide[:, :256] = c.q.reshape(3, 256)
    c.dq, flat = Values(ctx, wide), Values(ctx, torch.full((3, 300), 9.0, dtype=c.q.dtype))
    c.out = flat
    c.run(q_stride=400, out_stride=300)
    got = flat.get()
    assert (got[:, 256:] == 9.0).all()
    c.out = Values(ctx, got[:, :256].reshape(3, 4, 64))
    c.check()


def test_weights_alone_and_in_place(ctx):
    """Without weights_in the sums alone; with weights_in == weights_out they are added to what is there; without either, the same out."""
    c = Case(ctx, "bf16", [500, 3], 8, 2, 128, 16).run()
    first, kept = c.w_out.get(), c.out.get()
    c.run(weights_in=None)
    alone = c.w_out.get()
    n = torch.tensor([500, 3])
    for b in range(2):
        assert ((first[b, :, :n[b]] - alone[b, :, :n[b]]) - torch.from_numpy(c.w_in[b, :, :n[b]])).abs().max() < 1e-5
        assert abs(float(alone[b, :, :n[b]].double().sum()) - 8) < 1e-3      # every query head gives a weight of one
    c.w_out = Values(ctx, torch.from_numpy(c.w_in.copy()))
    c.run(weights_in=c.w_out, weights_out=c.w_out)
    for b in range(2):
        assert torch.equal(c.w_out.get()[b, :, :n[b]], first[b, :, :n[b]])
        assert np.array_equal(c.w_out.get().numpy()[b, :, n[b]:], c.w_in[b, :, n[b]:])
    c.run(weights_in=None, weights_out=None, lse=None)
    assert torch.equal(c.out.get(), kept)


def test_same_result_every_time(ctx):
    """Which block joins the runs changes nothing: no atomics on values."""
    for name in ("f32", "bf16"):
        c = Case(ctx, name, [4000, 100], 8, 2, 128, 16).run()
        first = [v.get() for v in (c.out, c.lse, c.w_out)]
        for _ in range(5):
            c.run()
            assert all(torch.equal(a, v.get()) for a, v in zip(first, (c.out, c.lse, c.w_out)))


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_bad_pages_and_lengths(ctx, name):
    """A page outside the pool counts as slots that are not there, a length beyond what the call allows is cut; both are told at the
    next sync, after which the context works."""
    from mace_b200 import MaceB200Error
    c = Case(ctx, name, [64, 50], 4, 2, 64, 16, seed=3, weights=False)
    for bad in (-1, c.pages, 2 ** 31 - 1, -2 ** 31):
        table = c.table.copy()
        table[0, 1] = bad
        c.dt = ctx.upload(table)
        with pytest.raises(MaceB200Error) as e:
            c.run()
        assert e.value.code == 4 and "outside its range" in str(e.value)
        rows, c.rows = c.rows, list(c.rows)
        c.rows[0] = tuple(torch.cat([r[:16], r[32:]]) for r in rows[0])
        c.lengths = [48, 50]
        c.check()
        c.rows, c.lengths = rows, [64, 50]
    c.dt = ctx.upload(c.table)
    for lengths, used in (([65, 50], [64, 50]), ([-1, 50], [0, 50]), ([64, 2 ** 31 - 1], None)):
        c.dn = ctx.upload(np.array(lengths, np.int32))
        with pytest.raises(MaceB200Error):
            c.run()
        if used:
            c.check(used)
    c.dn = ctx.upload(np.array([64, 50], np.int32))
    c.run().check()


def test_an_empty_table_and_an_empty_batch(ctx):
    c = Case(ctx, "bf16", [0, 0], 4, 2, 64, 16)
    c.run().check()
    c.ctx.paged_attention(c.dq, c.dk, c.dv, c.dt, c.dn, c.out, 0, 4, 2, 64, c.pages, 16, 1, 5, 1.0, 2)
    c.ctx.paged_attention(c.dq, c.dk, c.dv, c.dt, c.dn, c.out, 2, 4, 2, 64, 0, 16, 0, 5, 1.0, 2, lse=c.lse)
    c.ctx.sync()
    assert (c.out.get() == 0).all()


def test_offsets_beyond_32_bits(ctx):
    """Pools of more than 2^32 bytes and 2^31 elements, of which the sequences use the last pages."""
    page, kv_heads, dim = 64, 8, 128
    pages = (1 << 31) // (page * kv_heads * dim) + 8
    c = Case(ctx, "bf16", [130, 64], 16, kv_heads, dim, page, weights=False)
    k, v = c.dk.get(), c.dv.get()
    size = pages * page * kv_heads * dim * 2
    big = [ctx.alloc(size) for _ in range(2)]
    table = c.table.copy()
    at = pages - 1
    for b in range(2):
        for j in range(-(-c.lengths[b] // page)):
            for buf, pool in zip(big, (k, v)):
                row = pool[int(c.table[b, j])].contiguous().view(torch.int16).numpy()

                class At:
                    ptr = buf.ptr + at * row.nbytes
                ctx.h2d(At, row)
            ctx.sync()
            table[b, j] = at
            at -= 1
    c.dk, c.dv = big
    c.dt, c.pages = ctx.upload(table), pages
    c.run().check()
    for buf in big:
        buf.free()


def test_replayed_as_sequences_grow(ctx):
    """A captured step that names the longest sequence is right at every length; a larger call in between, which takes more scratch
    memory, does not take the graph's."""
    c = Case(ctx, "bf16", [600, 600, 600], 8, 2, 64, 16)
    c.run()
    from mace_b200.capi import lib
    import ctypes as C
    L = lib()
    assert L.mb_graph_begin(ctx.h) == 0
    c.call()
    graph = C.c_void_p()
    assert L.mb_graph_end(ctx.h, C.byref(graph)) == 0
    Case(ctx, "f32", [9000] * 4, 64, 8, 128, 16, seed=9).run()
    for lengths in ([600, 1, 77], [0, 599, 256]):
        c.lengths = lengths
        n = np.array(lengths, np.int32)
        ctx.h2d(c.dn, n)
        ctx.h2d(c.w_out.buf, np.full((3, 2, c.stride), -5.0, np.float32))
        ctx.sync()
        assert L.mb_graph_launch(ctx.h, graph) == 0
        ctx.sync()
        c.check()
    L.mb_graph_destroy(ctx.h, graph)


def test_scratch_does_not_grow_inside_a_capture():
    import ctypes as C

    import mace_b200
    from mace_b200.capi import lib
    with mace_b200.Context(0) as ctx:
        c = Case(ctx, "bf16", [3000], 8, 2, 64, 16)
        assert lib().mb_graph_begin(ctx.h) == 0
        with pytest.raises(mace_b200.MaceB200Error) as e:
            c.call()
        assert e.value.code == 4 and "run the sequence once first" in str(e.value)
        graph = C.c_void_p()
        lib().mb_graph_end(ctx.h, C.byref(graph))
        lib().mb_graph_destroy(ctx.h, graph)
        c.run().check()


def test_two_contexts_at_once(ctx):
    """Calls on two contexts' streams that overlap share nothing."""
    import mace_b200
    with mace_b200.Context(0) as other:
        a = Case(ctx, "bf16", [3000, 40], 8, 2, 128, 16, seed=1)
        b = Case(other, "bf16", [2000, 2500], 8, 2, 128, 16, seed=2)
        for _ in range(10):
            a.call()
            b.call()
        ctx.sync()
        other.sync()
        a.check()
        b.check()


def test_refusals(ctx):
    from mace_b200 import MaceB200Error
    c = Case(ctx, "bf16", [10], 4, 2, 64, 16)
    for kw, code in ((dict(window=-1), 1), (dict(weights_stride=5), 1), (dict(weights_out=None), 1), (dict(out_stride=3), 1), (dict(q_stride=-1), 1)):
        if kw.get("out_stride") == 3:
            c2 = Case(ctx, "bf16", [10, 10], 4, 2, 64, 16)
        else:
            c2 = c
        with pytest.raises(MaceB200Error) as e:
            c2.run(**kw)
        assert e.value.code == code, kw
    with pytest.raises(MaceB200Error) as e:
        ctx.paged_attention(c.dq, c.dk, c.dv, c.dt, c.dn, c.out, 1, 4, 2, 264, c.pages, 16, 1, 5, 1.0, 2)
    assert e.value.code == 3
    c.run().check()
