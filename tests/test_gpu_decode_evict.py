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
