"""Rotary positions and the way into the paged cache against 64-bit forms."""
import numpy as np
import pytest
import torch

from decode_ref import HALF, TINY, TYPES, Values, tensor, turn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mace_b200
    c = mace_b200.Context(0)
    yield c
    c.close()


def _freq(dim, base=10000.0):
    return base ** (-2.0 * np.arange(dim // 2) / max(dim, 1))


def _bound(want, size, name):
    """The angle's fraction of a turn is rounded to 24 bits (2 pi x 2^-25 = 1.9e-7), sincospif is within 2^-22, the factor, two
    products and a sum round once each (5 x 2^-24): less than 2^-20 of the terms' magnitudes.  Then one rounding to the type."""
    return size * 2.0 ** -20 * (1 + HALF[name]) + np.abs(want) * HALF[name] + TINY[name]


def _check(got, want, size, name):
    got = got.double().numpy()
    assert (np.abs(got - want) <= _bound(want, size, name)).all()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rotary", [
    (1, 1, 2, 2), (1, 32, 128, 128), (3, 5, 64, 64), (7, 3, 80, 32), (130, 2, 96, 64), (300, 1, 256, 256), (5, 4, 36, 10), (9, 2, 33, 12),
    (4, 3, 16, 0), (2, 64, 192, 128), (1, 1, 7, 6), (1000, 7, 24, 24)])
def test_rope(ctx, name, interleaved, tokens, heads, dim, rotary):
    rng = np.random.default_rng(tokens * 1000 + dim)
    x = tensor(rng, name, tokens, heads, dim)
    positions = rng.integers(0, 1 << 20, tokens).astype(np.int32)
    positions[0], positions[-1] = 0, 2 ** 31 - 1
    freq = _freq(rotary)
    dx, dy, dp, df = Values(ctx, x), Values(ctx, torch.full_like(x, 7)), ctx.upload(positions), ctx.upload(freq)
    for inverse, magnitude in ((False, 1.0), (True, 1.25)):
        ctx.rope(dx, dy, dp, df, tokens, heads, dim, rotary, TYPES[name][0], interleaved=interleaved, inverse=inverse, magnitude=magnitude)
        want, size = turn(x, positions, freq, magnitude, rotary, interleaved, inverse)
        got = dy.get()
        _check(got[..., :rotary], want[..., :rotary], size[..., :rotary], name)
        assert torch.equal(got[..., rotary:], x[..., rotary:])   # copied bit for bit
    # in place
    ctx.rope(dx, dx, dp, df, tokens, heads, dim, rotary, TYPES[name][0], interleaved=interleaved, inverse=True, magnitude=1.25)
    assert torch.equal(dx.get(), got)


@pytest.mark.parametrize("name,offset", [("f32", 1), ("bf16", 1), ("f16", 2), ("bf16", 4)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strides_and_alignment(ctx, name, offset, interleaved):
    """Heads inside rows that hold more, the output with tokens inside heads, starts that are not 16-byte aligned; what lies between
    the output's rows stays."""
    rng = np.random.default_rng(offset)
    tokens, heads, dim, rotary = 5, 3, 16, 8
    wide = tensor(rng, name, tokens, 77)
    x = torch.as_strided(wide, (tokens, heads, dim), (77, 20, 1))
    positions, freq = rng.integers(0, 5000, tokens).astype(np.int32), _freq(rotary)
    out = torch.full((heads, tokens, dim + 4), 3.0, dtype=TYPES[name][1])
    dx, dy, dp, df = Values(ctx, wide, offset), Values(ctx, out, offset), ctx.upload(positions), ctx.upload(freq)
    ctx.rope(dx, dy, dp, df, tokens, heads, dim, rotary, TYPES[name][0], x_strides=(77, 20), y_strides=(dim + 4, tokens * (dim + 4)),
             interleaved=interleaved)
    want, size = turn(x, positions, freq, 1.0, rotary, interleaved)
    got = dy.get()
    _check(got[..., :dim].permute(1, 0, 2), want, size, name)
    assert (got[..., dim:] == 3.0).all()


@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_inverse_is_the_gradient(ctx, interleaved):
    """d(sum g y) / dx by central differences of the 64-bit form, which is linear, so that a step of 1 gives it to rounding."""
    rng = np.random.default_rng(3)
    tokens, heads, dim, rotary = 2, 2, 12, 8
    x, g = tensor(rng, "f32", tokens, heads, dim), tensor(rng, "f32", tokens, heads, dim)
    positions, freq = np.array([5, 123456], np.int32), _freq(rotary)
    dg, dx, dp, df = Values(ctx, g), Values(ctx, torch.zeros_like(g)), ctx.upload(positions), ctx.upload(freq)
    ctx.rope(dg, dx, dp, df, tokens, heads, dim, rotary, TYPES["f32"][0], interleaved=interleaved, inverse=True, magnitude=1.5)
    want = np.zeros(x.shape)
    gd = g.double().numpy()
    for i in np.ndindex(*x.shape):
        up, down = x.clone().double(), x.clone().double()
        up[i] += 1
        down[i] -= 1
        want[i] = ((turn(up, positions, freq, 1.5, rotary, interleaved)[0] - turn(down, positions, freq, 1.5, rotary, interleaved)[0]) * gd).sum() / 2
    _, size = turn(g, positions, freq, 1.5, rotary, interleaved, True)
    assert (np.abs(dx.get().double().numpy() - want) <= _bound(want, size, "f32") + 1e-13).all()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,rotary,page,interleaved", [
    (1, 1, 1, 16, 16, 1, False), (1, 32, 8, 128, 128, 16, False), (33, 8, 2, 64, 32, 20, True), (70, 3, 3, 40, 40, 7, False),
    (5, 4, 1, 10, 6, 3, True), (12, 7, 7, 256, 256, 64, False)])
def test_append(ctx, name, tokens, heads, kv_heads, dim, rotary, page, interleaved):
    rng = np.random.default_rng(tokens + dim)
    width = (heads + 2 * kv_heads) * dim
    qkv = tensor(rng, name, tokens, width + 8)
    q, k, v = qkv[:, :width].reshape(tokens, -1, dim).split([heads, kv_heads, kv_heads], dim=1)
    pages = -(-tokens // page) + 2
    slots = rng.permutation(pages * page)[:tokens].astype(np.int32)
    if tokens > 4:
        slots[2] = -1      # padding
    positions, freq = rng.integers(0, 100000, tokens).astype(np.int32), _freq(rotary)
    pools = [tensor(rng, name, pages, kv_heads, page, dim) for _ in range(2)]
    dq = Values(ctx, qkv)
    size = qkv.element_size()

    class Part:
        def __init__(self, skip):
            self.ptr = dq.ptr + skip * size
    out = Values(ctx, torch.full((tokens, heads * dim + 4), 5.0, dtype=qkv.dtype))
    dk, dv = (Values(ctx, p) for p in pools)
    dp, ds, df = ctx.upload(positions), ctx.upload(slots), ctx.upload(freq)
    ctx.rope_kv_append(dq, out, Part(heads * dim), Part((heads + kv_heads) * dim), dk, dv, dp, ds, df, tokens, heads, kv_heads, dim,
                       rotary, pages, page, TYPES[name][0], token_strides=(width + 8,) * 3, q_out_stride=heads * dim + 4,
                       interleaved=interleaved, magnitude=0.5)
    ctx.sync()
    want, terms = turn(q, positions, freq, 0.5, rotary, interleaved)
    got = out.get()
    _check(got[:, :heads * dim].reshape(tokens, heads, dim), want, terms, name)
    assert (got[:, heads * dim:] == 5.0).all()
    want, terms = turn(k, positions, freq, 0.5, rotary, interleaved)
    got_k, got_v = dk.get(), dv.get()
    untouched = torch.ones(pages, page, dtype=torch.bool)
    for t, s in enumerate(slots):
        if s < 0:
            continue
        untouched[s // page, s % page] = False
        _check(got_k[s // page, :, s % page], want[t], terms[t], name)
        assert torch.equal(got_v[s // page, :, s % page], v[t])
    for got, had in ((got_k, pools[0]), (got_v, pools[1])):
        assert torch.equal(got.transpose(1, 2)[untouched], had.transpose(1, 2)[untouched])


def test_append_refuses_slots_behind_the_pool(ctx):
    """Such a token is left out, the others are written, and the next sync says so; the context stays usable."""
    from mace_b200 import MaceB200Error
    rng = np.random.default_rng(1)
    k, v, q = (tensor(rng, "f32", 3, 8) for _ in range(3))
    pool = torch.zeros(2, 1, 4, 8)
    dk, dv, dq, out = (Values(ctx, t) for t in (k, v, q, torch.zeros(3, 8)))
    pk, pv = Values(ctx, pool), Values(ctx, pool)
    dp, df = ctx.upload(np.zeros(3, np.int32)), ctx.upload(_freq(8))
    for bad in (8, 2 ** 31 - 1):
        ds = ctx.upload(np.array([1, bad, 6], np.int32))
        ctx.rope_kv_append(dq, out, dk, dv, pk, pv, dp, ds, df, 3, 1, 1, 8, 8, 2, 4, TYPES["f32"][0])
        with pytest.raises(MaceB200Error) as e:
            ctx.sync()
        assert e.value.code == 4 and "outside its range" in str(e.value)
        ctx.sync()
        got = pv.get().reshape(8, 8)
        assert torch.equal(got[1], v[0]) and torch.equal(got[6], v[2]) and (got[[0, 2, 3, 4, 5, 7]] == 0).all()
        assert torch.equal(out.get(), q)      # position 0: unturned


def test_rope_refusals(ctx):
    from mace_b200 import MaceB200Error
    x = Values(ctx, torch.zeros(2, 2, 8))
    f = ctx.upload(_freq(8))
    p = ctx.upload(np.zeros(2, np.int32))
    for change, code in ((dict(rotary_dim=3), 1), (dict(rotary_dim=10), 1), (dict(dtype=3), 1), (dict(heads=0), 1), (dict(tokens=-1), 1),
                         (dict(tokens=1 << 31), 3), (dict(y_strides=(8, 4)), 1)):
        a = dict(tokens=2, heads=2, head_dim=8, rotary_dim=8, dtype=0)
        a.update(change)
        with pytest.raises(MaceB200Error) as e:
            ctx.rope(x, x, p, f, **a)
        assert e.value.code == code, change
    ctx.rope(x, x, p, f, 0, 2, 8, 8, 0)
    ctx.sync()
