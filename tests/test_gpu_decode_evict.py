"""Eviction by accumulated weight: choices and copies bit for bit."""
import numpy as np
import pytest
import torch

from decode_ref import TYPES, Values, paged

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mace_b200
    c = mace_b200.Context(0)
    yield c
    c.close()


def choose(w, budget, sinks, recent):
    """The kept slots of one head, from the definition."""
    n = len(w)
    if n <= budget:
        return list(range(n))
    between = list(range(sinks, n - recent))
    key = [(-np.inf if np.isnan(w[j]) else float(w[j]), not np.isnan(w[j])) for j in between]
    # heaviest first; NaN behind -inf; of equal ones the lower slot
    order = sorted(range(len(between)), key=lambda i: (-key[i][0], not key[i][1], between[i]))
    return sorted(list(range(sinks)) + [between[i] for i in order[:budget - sinks - recent]] + list(range(n - recent, n)))


def _weights(rng, kind, shape):
    if kind == "spread":
        return np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        return rng.integers(0, 4, shape).astype(np.float32)
    if kind == "equal":
        return np.full(shape, 0.25, np.float32)
    if kind == "close":      # differ in their last bits only
        return (np.float32(1.0).view(np.uint32) + rng.integers(0, 40, shape).astype(np.uint32)).view(np.float32)
    w = rng.standard_normal(shape).astype(np.float32)
    pick = rng.integers(0, 9, shape)
    for i, v in enumerate((np.inf, -np.inf, np.nan, -0.0, 0.0, np.float32(1e-45))):
        w[pick == i] = v
    return w


def _case(ctx, name, lengths, heads, dim, page, budget, sinks, recent, kind="spread", same_lengths=False, same_pool=False, seed=0, stride=None):
    rng = np.random.default_rng(seed)
    batch, longest = len(lengths), max(lengths)
    k, v, table, rows = paged(rng, name, lengths, heads, dim, page, fill=float("nan"))
    stride = longest + 2 if stride is None else stride
    w = _weights(rng, kind, (batch, heads, stride))
    new_width = -(-min(budget, max(longest, 1)) // page)
    dst_pages = batch * new_width + 1
    src_pages = k.shape[0]
    new_table = rng.permutation(dst_pages)[:batch * new_width].reshape(batch, new_width).astype(np.int32)
    if same_pool:     # the new pages lie behind the old ones in one pool
        k, v = (torch.cat([p, torch.full((dst_pages, heads, page, dim), 5.0, dtype=p.dtype)]) for p in (k, v))
        new_table, dst_pages = new_table + src_pages, dst_pages + src_pages
        dk, dv = Values(ctx, k), Values(ctx, v)
        dk2, dv2 = dk, dv
    else:
        dk, dv = Values(ctx, k), Values(ctx, v)
        dk2, dv2 = (Values(ctx, torch.full((dst_pages, heads, page, dim), 5.0, dtype=k.dtype)) for _ in range(2))
    dn = Values(ctx, torch.tensor(lengths, dtype=torch.int32))
    dn2 = dn if same_lengths else Values(ctx, torch.full((batch,), 77, dtype=torch.int32))
    dw, dw2 = ctx.upload(w), Values(ctx, torch.full((batch, heads, budget), -3.0))
    kept = Values(ctx, torch.full((batch, heads, budget), 99, dtype=torch.int32))

    def call():
        ctx.kv_evict(dk, dv, ctx.upload(table), dn, dw, dk2, dv2, ctx.upload(new_table), dn2, dw2, kept, batch, heads, dim, page,
                     src_pages, table.shape[1], dst_pages, new_width, longest, stride, budget, sinks, recent, TYPES[name][0])
        ctx.sync()

    def check():
        got_k, got_v, got, gw = dk2.get(), dv2.get(), kept.get().numpy(), dw2.get().numpy()
        free = torch.ones(dst_pages, heads, page, dtype=torch.bool)
        assert dn2.get().tolist() == [min(n, budget) for n in lengths]
        for b, n in enumerate(lengths):
            for h in range(heads):
                want = choose(w[b, h, :n], budget, sinks, recent)
                m = len(want)
                assert got[b, h, :m].tolist() == want, (b, h)
                assert (got[b, h, m:] == -1).all()
                assert np.array_equal(gw[b, h, :m], w[b, h, want], equal_nan=True) and (gw[b, h, m:] == -3.0).all()
                j = np.arange(m)
                at = torch.from_numpy(new_table[b, j // page].astype(np.int64)), torch.from_numpy(j % page)
                free[at[0], h, at[1]] = False
                assert torch.equal(got_k[at[0], h, at[1]], rows[b][0][want, h])
                assert torch.equal(got_v[at[0], h, at[1]], rows[b][1][want, h])
        if not same_pool:     # rows behind the new lengths stay
            assert (got_k[free] == 5.0).all() and (got_v[free] == 5.0).all()
    return call, check


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "close", "special"])
@pytest.mark.parametrize("budget,sinks,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (64, 4, 16), (100, 100, 0), (100, 0, 100), (99, 50, 49),
                                                 (250, 0, 0), (1000, 3, 5)])
def test_choices(ctx, kind, budget, sinks, recent):
    call, check = _case(ctx, "bf16", [300, 1, 0, 64, 65, 100, 101, 33], 2, 16, 16, budget, sinks, recent, kind, seed=budget)
    call()
    check()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 20), (3, 7), (10, 1), (256, 64), (100, 32), (1, 3)])
def test_rows(ctx, name, dim, page):
    call, check = _case(ctx, name, [130, 40, 77], 3, dim, page, 50, 2, 10, seed=dim)
    call()
    check()


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "special"])
@pytest.mark.parametrize("length,budget", [(5000, 1000), (40000, 39990), (33000, 10), (70001, 30000), (300000, 1234)])
def test_long(ctx, kind, length, budget):
    call, check = _case(ctx, "bf16", [length, 900], 1, 8, 64, budget, 4, min(budget // 2, 100), kind, seed=length)
    call()
    check()


@pytest.mark.parametrize("kind", ["spread", "ties", "special"])
@pytest.mark.parametrize("batch,longest", [(80, 500), (160, 25000)])
def test_more_heads_than_sms(ctx, kind, batch, longest):
    rng = np.random.default_rng(batch)
    lengths = [int(n) for n in rng.integers(0, 300, batch)]
    lengths[3] = longest
    heads = 2 if batch < 148 else 1
    call, check = _case(ctx, "bf16", lengths, heads, 8, 16, 120, 4, 30, kind, seed=batch)
    call()
    check()


def test_lengths_in_place_one_pool_and_twice(ctx):
    call, check = _case(ctx, "f32", [100, 20, 60], 2, 32, 8, 30, 2, 5, same_lengths=True, same_pool=True)
    call()
    check()
    # another context's counters, the same memory: a second call on what the first left
    call, check = _case(ctx, "f32", [100, 20, 60], 2, 32, 8, 30, 2, 5, same_pool=True)
    call()
    call()
    check()


def test_bad_pages_and_lengths(ctx):
    """Rows of a page that a pool lacks are neither read nor written; the next sync says so."""
    from mace_b200 import MaceB200Error
    rng = np.random.default_rng(1)
    k, v, table, rows = paged(rng, "f32", [40, 24], 1, 8, 8)
    w = rng.random((2, 1, 40)).astype(np.float32)
    dst = torch.full((6, 1, 8, 8), 5.0)
    good = np.arange(4, dtype=np.int32).reshape(2, 2)
    dk, dv, dn, dw = Values(ctx, k), Values(ctx, v), ctx.upload(np.array([40, 24], np.int32)), ctx.upload(w)

    def call(src, new, lengths=dn):
        out = [Values(ctx, t) for t in (dst, dst, torch.zeros(2, dtype=torch.int32), torch.zeros(2, 1, 16), torch.zeros(2, 1, 16, dtype=torch.int32))]
        ctx.kv_evict(dk, dv, ctx.upload(src), lengths, dw, out[0], out[1], ctx.upload(new), out[2], out[3], out[4], 2, 1, 8, 8,
                     k.shape[0], src.shape[1], 6, 2, 40, 40, 16, 0, 8, 0)
        return out
    for bad in (-1, 6, 2 ** 31 - 1):
        new = good.copy()
        new[1, 0] = bad
        out = call(table, new)
        with pytest.raises(MaceB200Error) as e:
            ctx.sync()
        assert "outside its range" in str(e.value)
        got = out[0].get()
        assert (got[good[1, 0]] == 5.0).all() and not (got[good[1, 1]] == 5.0).any() and (got[4:] == 5.0).all()
    src = table.copy()
    src[0, :] = k.shape[0]
    out = call(src, good)
    with pytest.raises(MaceB200Error):
        ctx.sync()
    assert (out[0].get()[good[0]] == 5.0).all() and not (out[0].get()[good[1]] == 5.0).any()
    out = call(table, good, ctx.upload(np.array([41, -5], np.int32)))
    with pytest.raises(MaceB200Error):
        ctx.sync()
    assert out[2].get().tolist() == [16, 0]
    call(table, good)
    ctx.sync()


def test_refusals(ctx):
    from mace_b200 import MaceB200Error
    x = Values(ctx, torch.zeros(64))
    y = Values(ctx, torch.zeros(64))

    def call(**kw):
        a = dict(batch=1, kv_heads=1, head_dim=8, page_size=4, src_pages=2, src_max_pages=2, dst_pages=2, dst_max_pages=1, max_length=8,
                 weights_stride=8, budget=4, sinks=1, recent=1, dtype=0)
        a.update(kw)
        ctx.kv_evict(x, x, x, x, x, y, y, x, y, y, y, *a.values())
    for kw in (dict(budget=0, sinks=0, recent=0), dict(sinks=4), dict(recent=-1), dict(budget=5), dict(weights_stride=7), dict(dtype=9),
               dict(page_size=0), dict(batch=-1)):
        with pytest.raises(MaceB200Error) as e:
            call(**kw)
        assert e.value.code == 1, kw
    call(batch=0)
    ctx.sync()


@pytest.mark.parametrize("name,heads,dim,budget,extra", [("bf16", 2, 64, 50, 41), ("f32", 3, 20, 64, 0), ("f16", 1, 128, 300, 7000)])
@pytest.mark.parametrize("same_lengths", [False, True])
def test_weights_as_the_next_step_takes_them(ctx, name, heads, dim, budget, extra, same_lengths):
    """Rows of weights longer than the budget: the kept ones in front, zeros behind, nothing beyond the last row."""
    rng = np.random.default_rng(budget)
    lengths, page = [200, 0, 31, budget, budget + 1, 999], 16
    batch, longest, row = len(lengths), max(lengths), budget + extra
    k, v, table, rows = paged(rng, name, lengths, heads, dim, page)
    w = rng.random((batch, heads, longest)).astype(np.float32)
    width = -(-budget // page)
    new_table = rng.permutation(batch * width).reshape(batch, width).astype(np.int32)
    dk, dv = Values(ctx, k), Values(ctx, v)
    dk2, dv2 = (Values(ctx, torch.full((batch * width, heads, page, dim), 5.0, dtype=k.dtype)) for _ in range(2))
    dn = Values(ctx, torch.tensor(lengths, dtype=torch.int32))
    dn2 = dn if same_lengths else Values(ctx, torch.zeros(batch, dtype=torch.int32))
    dw, dt, dt2 = ctx.upload(w), ctx.upload(table), ctx.upload(new_table)
    dw2, kept = Values(ctx, torch.full((batch * heads * row + 9,), -3.0)), Values(ctx, torch.zeros(batch, heads, budget, dtype=torch.int32))
    ctx.kv_evict(dk, dv, dt, dn, dw, dk2, dv2, dt2, dn2, dw2, kept, batch, heads, dim, page, k.shape[0], table.shape[1], batch * width, width,
                 longest, longest, budget, 4, 10, TYPES[name][0], dst_weights_stride=row)
    ctx.sync()
    got = dw2.get().numpy()
    assert (got[batch * heads * row:] == -3.0).all() and dn2.get().tolist() == [min(n, budget) for n in lengths]
    got = got[:batch * heads * row].reshape(batch, heads, row)
    new_k = dk2.get()
    for b, n in enumerate(lengths):
        for h in range(heads):
            want = choose(w[b, h, :n], budget, 4, 10)
            m = len(want)
            assert kept.get()[b, h, :m].tolist() == want and (kept.get()[b, h, m:] == -1).all()
            assert np.array_equal(got[b, h, :m], w[b, h, want]) and (got[b, h, m:] == 0.0).all()
            j = np.arange(m)
            assert torch.equal(new_k[torch.from_numpy(new_table[b, j // page].astype(np.int64)), h, torch.from_numpy(j % page)], rows[b][0][want, h])


def test_evicted_again_and_again_from_a_graph(ctx):
    """Two evictions, to and fro between two sets of pages and of weights, captured once and replayed: attention's weights need no
    rearranging in between."""
    import ctypes as C

    from mace_b200.capi import lib
    L = lib()
    rng = np.random.default_rng(3)
    batch, heads, kv_heads, dim, page, room, budget, name = 3, 4, 2, 64, 16, 96, 40, "f32"
    lengths = [90, 41, 17]
    width = room // page
    pages = 2 * batch * width
    tables = rng.permutation(pages).reshape(2, batch, width).astype(np.int32)
    k, v = (torch.from_numpy(rng.standard_normal((pages, kv_heads, page, dim)).astype(np.float32)) for _ in range(2))
    w = np.zeros((batch, kv_heads, room), np.float32)
    for b, n in enumerate(lengths):
        w[b, :, :n] = rng.random((kv_heads, n))
    q = torch.from_numpy(rng.standard_normal((batch, heads, dim)).astype(np.float32))
    dk, dv, dq, out = Values(ctx, k), Values(ctx, v), Values(ctx, q), Values(ctx, q)
    dn, dt = Values(ctx, torch.tensor(lengths, dtype=torch.int32)), [ctx.upload(t) for t in tables]
    dw = [Values(ctx, torch.from_numpy(w)), Values(ctx, torch.full((batch, kv_heads, room), -1.0))]
    kept = Values(ctx, torch.zeros(batch, kv_heads, budget, dtype=torch.int32))

    def attend(i):
        ctx.paged_attention(dq, dk, dv, dt[i], dn, out, batch, heads, kv_heads, dim, pages, page, width, room, 0.125, 0, weights_in=dw[i],
                            weights_out=dw[i], weights_stride=room)

    def evict(i, n):
        ctx.kv_evict(dk, dv, dt[i], dn, dw[i], dk, dv, dt[1 - i], dn, dw[1 - i], kept, batch, kv_heads, dim, page, pages, width, pages, width,
                     room, room, n, 2, 5, 0, dst_weights_stride=room)

    def both():
        attend(0)
        evict(0, budget)
        attend(1)
        evict(1, budget - 8)

    # the same by hand
    def host(times):
        rows = [[[(k[torch.from_numpy(tables[0][b][j // page:j // page + 1].astype(np.int64))[0], h, j % page],
                   v[torch.from_numpy(tables[0][b][j // page:j // page + 1].astype(np.int64))[0], h, j % page], float(w[b, h, j]))
                  for j in range(lengths[b])] for h in range(kv_heads)] for b in range(batch)]
        for step in range(2 * times):
            for b in range(batch):
                for h in range(kv_heads):
                    r = rows[b][h]
                    keys = torch.stack([x[0] for x in r]).double()
                    p = torch.softmax(q[b, 2 * h:2 * h + 2].double() @ keys.T * 0.125, 1).sum(0)
                    r = [(x[0], x[1], x[2] + float(y)) for x, y in zip(r, p)]
                    rows[b][h] = [r[j] for j in choose(np.array([x[2] for x in r]), budget - 8 * (step % 2), 2, 5)]
        return rows

    def check(times):
        rows = host(times)
        got_k, got_w, n = dk.get(), dw[0].get().numpy(), dn.get().tolist()
        for b in range(batch):
            for h in range(kv_heads):
                r = rows[b][h]
                assert n[b] == len(r)
                for j, x in enumerate(r):
                    assert torch.equal(got_k[int(tables[0][b][j // page]), h, j % page], x[0])
                # fp32: (dim + 16) roundings of a logit of at most 8 or so, twice, for each of the steps
                assert np.allclose(got_w[b, h, :len(r)], [x[2] for x in r], rtol=0, atol=2 * times * 2 * (dim + 16) * 8 * 2.0 ** -23)
                assert (got_w[b, h, len(r):] == 0.0).all()

    both()
    ctx.sync()
    check(1)
    assert L.mb_graph_begin(ctx.h) == 0
    both()
    graph = C.c_void_p()
    assert L.mb_graph_end(ctx.h, C.byref(graph)) == 0
    for _ in range(3):
        assert L.mb_graph_launch(ctx.h, graph) == 0
    ctx.sync()
    check(4)
    L.mb_graph_destroy(ctx.h, graph)


def test_refusals_of_strided_weights(ctx):
    from mace_b200 import MaceB200Error
    x, y = Values(ctx, torch.zeros(64)), Values(ctx, torch.zeros(64))
    for stride in (0, -1, 3, 2 ** 31):
        with pytest.raises(MaceB200Error) as e:
            ctx.kv_evict(x, x, x, x, x, y, y, x, y, y, y, 1, 1, 8, 4, 2, 2, 2, 1, 8, 8, 4, 1, 1, 0, dst_weights_stride=stride)
        assert e.value.code == 1 and "dst_weights_stride" in str(e.value)
    with pytest.raises(MaceB200Error) as e:     # the rows' tail reaches into weights
        class Before:
            ptr = x.ptr - 16
        ctx.kv_evict(x, x, x, x, x, y, y, x, y, Before, y, 1, 1, 8, 4, 2, 2, 2, 1, 8, 8, 4, 1, 1, 0, dst_weights_stride=8)
    assert e.value.code == 1 and "dst_weights" in str(e.value)
