"""Attention of one token over the paged cache where the numbers are far apart: a slot that outweighs all others, values at the type's
end, long even sums.  Against the 64-bit form, as in test_gpu_decode_attention.py."""
import math

import numpy as np
import pytest
import torch

from decode_ref import HALF, TINY, TYPES, Values, attend
from test_gpu_decode_attention import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mace_b200
    c = mace_b200.Context(0)
    yield c
    c.close()


def _run(ctx, name, q, k, v, table, lengths, scale, page, weights=False):
    """out, lse and the collected weights (or None) of pools k and v."""
    batch, heads, dim = q.shape
    pages, kv_heads = k.shape[:2]
    dq, dk, dv, out = Values(ctx, q), Values(ctx, k), Values(ctx, v), Values(ctx, torch.zeros_like(q))
    lse, dt, dn = Values(ctx, torch.zeros(batch, heads)), ctx.upload(table), ctx.upload(np.array(lengths, np.int32))
    w = Values(ctx, torch.zeros(batch, kv_heads, max(lengths))) if weights else None
    ctx.paged_attention(dq, dk, dv, dt, dn, out, batch, heads, kv_heads, dim, pages, page, table.shape[1], max(lengths), scale, TYPES[name][0],
                        lse=lse, weights_out=w, weights_stride=max(lengths))
    ctx.sync()
    got = out.get(), lse.get(), w.get() if weights else None
    for x in (dq, dk, dv, out, lse, dt, dn) + ((w,) if weights else ()):
        x.free()
    return got


def _heavy(ctx, name, gap, length, where, heads, kv_heads, dim, page, seed=0):
    """One slot's logit is `gap`, its value zero; all other logits are zero.  What is left are probabilities of e^-gap each.

    All logits but the heavy one are exact; that one is a product with scale log2(e), rounded twice, whose difference from the others
    is rounded once: gap 2^-22; the exponential 2^-22 more, and the same for the sum: (gap + 4) 2^-22 in all.  Sums over slots as in the other
    file ((n / 4 + 150) 2^-23), probabilities 2^-16 of their size (16-bit pairs) or 2^-20 (tf32 pairs), then one rounding."""
    rng = np.random.default_rng(seed + length)
    dtype = TYPES[name][1]
    pages = -(-length // page)
    table = rng.permutation(pages).astype(np.int32)[None]
    k = torch.zeros(pages, kv_heads, page, dim, dtype=dtype)
    # (large, so that 16-bit results keep their bits at small weights)
    v = (1024.0 * (1 + 0.25 * torch.from_numpy(rng.standard_normal((pages, kv_heads, page, dim)).astype(np.float32)))).to(dtype)
    at = int(table[0, where // page]), where % page
    k[at[0], :, at[1]] = gap
    v[at[0], :, at[1]] = 0
    q = torch.ones(1, heads, dim, dtype=dtype)
    out, lse, weights = _run(ctx, name, q, k, v, table, [length], 1.0 / dim, page, weights=True)
    rel = (gap + 4) * 2.0 ** -22 + (length / 4 + 150) * 2.0 ** -23 + (2.0 ** -20 if name == "f32" else 2.0 ** -16)
    rows = torch.from_numpy(table[0].astype(np.int64))
    group = heads // kv_heads
    for h in range(kv_heads):
        kh, vh = (x[rows, h].reshape(-1, dim)[:length] for x in (k, v))
        mine = slice(h * group, (h + 1) * group)
        o, l, p, _, size = attend(q[0, mine], kh, vh, 1.0 / dim)
        assert ((out[0, mine].double() - o).abs() <= size * rel + o.abs() * HALF[name] + TINY[name]).all()
        assert ((lse[0, mine].double() - l).abs() <= rel + l.abs() * 2.0 ** -22).all()
        w = p.sum(0)
        assert ((weights[0, h].double() - w).abs() <= w * (rel + 2.0 ** -22)).all()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("length", [16, 300, 4096])
@pytest.mark.parametrize("gap", [0.5, 10, 14, 16, 16.625, 17, 17.375, 20, 25, 30, 40])
def test_a_slot_that_outweighs_the_others(ctx, name, length, gap):
    for where in (0, length // 2, length - 1):
        _heavy(ctx, name, gap, length, where, 8, 2, 128, 16)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(1, 1, 64, 16), (16, 1, 128, 16), (24, 1, 128, 16), (24, 1, 64, 20), (40, 2, 128, 20),
                                                     (16, 1, 256, 16), (4, 2, 256, 8), (8, 8, 64, 16), (6, 2, 32, 1)])
def test_in_every_form(ctx, name, heads, kv_heads, dim, page):
    for gap in (15, 18, 26, 42):
        _heavy(ctx, name, gap, 777, 5, heads, kv_heads, dim, page)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_runs_joined(ctx, name):
    """Runs of a sequence in blocks of their own: in some of them nothing but the small ones."""
    _heavy(ctx, name, 19, 20000, 3, 32, 16, 128, 16)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_on_cuda_cores(ctx, name):
    ctx.set_option("tensor_cores", 0)
    try:
        for gap in (12, 20, 30):
            _heavy(ctx, name, gap, 500, 0, 8, 2, 64, 16)
    finally:
        ctx.set_option("tensor_cores", 1)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_probabilities_of_every_size(ctx, name):
    """Logits from 0 down to -100, values that grow as the probabilities fall (as far as the type goes), so that every slot is part of the
    result.  A logit is its key times scale log2(e): 2^-23 of it, and 2^-24 of its distance from the maximum, in the exponent."""
    length, dim, page, rng = 201, 64, 16, np.random.default_rng(4)
    dtype = TYPES[name][1]
    j = rng.permutation(length)
    pages = -(-length // page)
    keys, values = torch.zeros(pages * page, dim), torch.zeros(pages * page, dim)
    keys[:length] = torch.from_numpy(-j / 2.0)[:, None]
    top = 60000.0 if name == "f16" else 1e30
    size = torch.from_numpy(np.minimum(np.exp(j / 2.0), top) * rng.uniform(0.5, 1.0, length))
    values[:length] = size.float()[:, None]
    k, v = (x.to(dtype).view(pages, 1, page, dim) for x in (keys, values))
    q = torch.ones(1, 4, dim, dtype=dtype)
    out, lse, _ = _run(ctx, name, q, k, v, np.arange(pages, dtype=np.int32)[None], [length], 1.0 / dim, page)
    o, l, _, terms, size = attend(q[0], k.view(-1, dim)[:length], v.view(-1, dim)[:length], 1.0 / dim)
    rel = (terms + 4) * 2.0 ** -22 + (length / 4 + 150) * 2.0 ** -23 + (2.0 ** -20 if name == "f32" else 2.0 ** -16)
    assert ((out[0].double() - o).abs() <= size * rel + o.abs() * HALF[name]).all()
    assert ((lse[0].double() - l).abs() <= rel + l.abs() * 2.0 ** -22).all()
    assert math.isfinite(float(lse.sum()))


def _single(ctx, name, value, length, dim, page):
    """One slot of a sequence has `value` and -value in turn, the others zeros; logits of zero."""
    dtype = TYPES[name][1]
    pages = -(-length // page)
    k, v = (torch.zeros(pages, 1, page, dim, dtype=dtype) for _ in range(2))
    at = length // 2
    v[at // page, 0, at % page] = torch.tensor([value, -value]).repeat(dim // 2).to(dtype)
    q = torch.ones(1, 4, dim, dtype=dtype)
    out, _, _ = _run(ctx, name, q, k, v, np.arange(pages, dtype=np.int32)[None], [length], 1.0, page)
    o = v[at // page, 0, at % page].double() / length
    # the probability is a quotient of exact numbers: what the product loses of its two factors, the division and the rounding
    assert ((out[0].double() - o).abs() <= o.abs() * (2.0 ** -20 if name == "f32" else 2.0 ** -16) + o.abs() * HALF[name] * 1.01).all()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 20), (256, 16)])
def test_a_single_value_at_the_types_end(ctx, name, dim, page):
    """The largest finite values, which the nearest number of fewer bits would make infinite."""
    top = torch.finfo(TYPES[name][1]).max
    for value in (top, top * (1 - 2.0 ** -12), top * (1 - 2.0 ** -11), top / 2):
        for length in (1, 16, 40, 1000):
            _single(ctx, name, value, length, dim, page)


def _even(ctx, name, values, length, heads, kv_heads, dim, page, tensor_cores=True):
    """Every slot has the same logit: the result is the values' mean, whatever their sum would be."""
    dtype = TYPES[name][1]
    pages = -(-length // page)
    k = torch.zeros(pages, kv_heads, page, dim, dtype=dtype)
    v = values(pages * page).to(dtype)[:, None, None].expand(-1, kv_heads, dim).reshape(pages, page, kv_heads, dim).transpose(1, 2).contiguous()
    q = torch.ones(1, heads, dim, dtype=dtype)
    ctx.set_option("tensor_cores", int(tensor_cores))
    try:
        out, lse, _ = _run(ctx, name, q, k, v, np.arange(pages, dtype=np.int32)[None], [length], 1.0, page)
    finally:
        ctx.set_option("tensor_cores", 1)
    rows = v.transpose(1, 2).reshape(-1, kv_heads, dim)[:length].double()
    o, size = rows.mean(0)[0, 0], rows.abs().mean(0)[0, 0]
    # probabilities are a power of two; sums over slots as ever, of products that lose 2^-20 or nothing
    assert ((out.double() - o).abs() <= size * ((length / 4 + 150) * 2.0 ** -23 + 2.0 ** -20) + o.abs() * HALF[name] * 1.01).all()
    assert ((lse.double() - math.log(length)).abs() <= 2.0 ** -20).all()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("length", [2, 17, 300, 9000, 60000])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (24, 1, 64, 20), (1, 1, 256, 16), (3, 3, 50, 7)])
def test_values_whose_sum_no_float_holds(ctx, name, length, heads, kv_heads, dim, page):
    """All values are near the type's largest, of one sign and of both."""
    top = float(torch.finfo(TYPES[name][1]).max)
    _even(ctx, name, lambda n: torch.full((n,), top * 0.99), length, heads, kv_heads, dim, page)
    _even(ctx, name, lambda n: torch.full((n,), top * 0.99).where(torch.arange(n) % 3 > 0, torch.tensor(-top)), length, heads, kv_heads, dim, page)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_values_whose_sum_no_float_holds_on_cuda_cores(ctx, name):
    top = float(torch.finfo(TYPES[name][1]).max)
    for length in (2, 300, 9000):
        _even(ctx, name, lambda n: torch.full((n,), top * 0.99), length, 8, 2, 128, 16, tensor_cores=False)


@pytest.mark.parametrize("name,heads,kv_heads,dim,page", [("bf16", 8, 1, 128, 16), ("f16", 8, 2, 64, 16), ("f32", 4, 1, 128, 16), ("f32", 4, 2, 64, 20),
                                                          ("f32", 4, 1, 256, 16), ("bf16", 16, 8, 256, 16), ("bf16", 4, 1, 50, 16)])
@pytest.mark.parametrize("length", [1000, 1025, 2048, 4097, 9000, 17000, 40000])
def test_few_heads_and_long_sequences(ctx, name, heads, kv_heads, dim, page, length):
    """Either side of where a head's slots outgrow a cluster, with and without weights."""
    for weights in (False, True):
        Case(ctx, name, [length], heads, kv_heads, dim, page, seed=length, weights=weights).run().check()
