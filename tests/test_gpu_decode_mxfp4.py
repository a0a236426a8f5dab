"""4-bit microscaled floating point against its definition in 64 bits: codes and scales bit for bit, products by a derived bound."""
import numpy as np
import pytest
import torch

from decode_ref import HALF, TINY, TYPES, Values, pack, quantize_mx, tensor, tile_scales, values_mx

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mace_b200
    c = mace_b200.Context(0)
    yield c
    c.close()


def _quantize(ctx, x, name, stride=None, offset=0):
    from mace_b200 import capi
    rows, cols = x.shape
    wide = x
    if stride is not None:
        wide = torch.full((rows, stride), 99.0, dtype=x.dtype)
        wide[:, :cols] = x
    dx = Values(ctx, wide, offset)
    blocks = -(-cols // 32)
    nq, ns = rows * blocks * 16, capi.mxfp4_scale_bytes(rows, cols)
    dq, ds = ctx.upload(np.full(nq + 16, 0xab, np.uint8)), ctx.upload(np.full(ns + 16, 0xab, np.uint8))
    ctx.quantize_mxfp4(dx, dq, ds, rows, cols, TYPES[name][0], stride=stride)
    q, s = ctx.download(dq, (nq + 16,), np.uint8), ctx.download(ds, (ns + 16,), np.uint8)
    assert (q[nq:] == 0xab).all() and (s[ns:] == 0xab).all()
    return dq, ds, q[:nq].reshape(rows, -1), s[:ns]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,stride,offset", [
    (1, 1, None, 0), (1, 32, None, 0), (3, 33, None, 0), (130, 100, None, 0), (128, 256, None, 0), (257, 640, 641, 0), (5, 1000, 1008, 1),
    (2, 4096, None, 0), (129, 31, 40, 8), (6, 2048, None, 0), (7, 2049, 2056, 0), (3, 3999, None, 1), (3, 6000, 6008, 0), (2, 8192, None, 0),
    (5, 9000, None, 0), (2, 20000, None, 0)])
def test_quantize_and_back(ctx, name, rows, cols, stride, offset):
    rng = np.random.default_rng(rows + cols)
    x = tensor(rng, name, rows, cols) * torch.from_numpy(np.exp2(rng.integers(-9, 9, (rows, 1)))).to(TYPES[name][1])
    dq, ds, q, s = _quantize(ctx, x, name, stride, offset)
    codes, scales = quantize_mx(x.double().numpy())
    assert np.array_equal(s, tile_scales(scales))
    assert np.array_equal(q, pack(codes))
    y = Values(ctx, torch.full((rows, (stride or cols)), 3.0, dtype=x.dtype), offset)
    ctx.dequantize_mxfp4(dq, ds, y, rows, cols, TYPES[name][0], stride=stride)
    got = y.get()
    want = torch.from_numpy(values_mx(codes, scales)[:, :cols]).to(x.dtype)   # exact in every type within its range
    assert torch.equal(got[:, :cols], want)
    assert (got[:, cols:] == 3.0).all()


def test_quantize_every_border(ctx):
    """Ties of every pair of neighbours and their fp32 neighbours, both signs, at every scale; maxima between 4 and 8 units."""
    mid = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.999999], np.float32)
    v = np.concatenate([mid, np.nextafter(mid, np.float32(0)), np.nextafter(mid, np.float32(9))])
    v = np.concatenate([v, -v, [0.0, -0.0]]).astype(np.float32)
    v = v[np.abs(v) < 8]
    rows = []
    for e in list(range(-149, -100)) + [-60, 0, 60, 120, 125]:
        for i in range(0, len(v), 31):
            block = np.zeros(32, np.float32)
            block[1:1 + len(v[i:i + 31])] = v[i:i + 31]
            block[0] = 4.0      # the exponent of the block
            with np.errstate(over="ignore", under="ignore"):
                row = np.ldexp(block.astype(np.float64), e).astype(np.float32)
            if np.isfinite(row).all():
                rows.append(row)
    x = np.stack(rows)
    _, _, q, s = _quantize(ctx, torch.from_numpy(x), "f32")
    codes, scales = quantize_mx(x.astype(np.float64))
    assert np.array_equal(s, tile_scales(scales))
    assert np.array_equal(q, pack(codes))


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
def test_quantize_special_values(ctx, name):
    x = torch.zeros(6, 96, dtype=TYPES[name][1])
    x[0, 40] = float("inf")
    x[1, 3] = float("nan")
    x[2, 95] = -float("inf")
    x[3, :32] = torch.finfo(x.dtype).max
    x[4, :32] = torch.finfo(x.dtype).tiny
    x[5, 1] = -0.0
    x[:3, 64] = 1.0
    dq, ds, q, s = _quantize(ctx, x, name)
    codes, scales = quantize_mx(x.double().numpy())
    assert scales[0, 1] == scales[1, 0] == scales[2, 2] == 255
    assert np.array_equal(s, tile_scales(scales)) and np.array_equal(q, pack(codes))
    y = Values(ctx, torch.zeros_like(x))
    ctx.dequantize_mxfp4(dq, ds, y, 6, 96, TYPES[name][0])
    got = y.get()
    want = torch.from_numpy(values_mx(codes, scales)).to(x.dtype)
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(1.0), want.nan_to_num(1.0))


def test_dequantize_every_scale(ctx):
    """Scales 0 .. 255 (255: NaN) times every code: 2^-127 is a subnormal number, 6 times 2^127 an infinity."""
    codes = np.tile(np.arange(16, dtype=np.uint8), (256, 2))
    scales = np.arange(256, dtype=np.uint8)[:, None]
    dq, ds = ctx.upload(pack(codes)), ctx.upload(tile_scales(scales))
    y = Values(ctx, torch.zeros(256, 32))
    ctx.dequantize_mxfp4(dq, ds, y, 256, 32, TYPES["f32"][0])
    with np.errstate(over="ignore"):
        want = values_mx(codes, scales).astype(np.float32)
    assert np.array_equal(y.get().numpy(), want, equal_nan=True)


def _random_mx(rng, rows, cols, low=110, high=140):
    blocks = -(-cols // 32)
    codes = rng.integers(0, 16, (rows, blocks * 32)).astype(np.uint8)
    codes[:, cols:] = 0
    return codes, rng.integers(low, high, (rows, blocks)).astype(np.uint8)


def _gemm(ctx, a, b, bias, name, stride=None, offset=0, tensor_cores=1):
    (ac, as_), (bc, bs) = a, b
    M, N, K = ac.shape[0], bc.shape[0], ac.shape[1]
    bufs = [ctx.upload(v) for v in (pack(ac), tile_scales(as_), pack(bc), tile_scales(bs))]
    db = ctx.upload(bias) if bias is not None else None
    out = Values(ctx, torch.full((M, stride or N), 3.0, dtype=TYPES[name][1]), offset)
    ctx.set_option("tensor_cores", tensor_cores)
    try:
        ctx.gemm_mxfp4(*bufs, out, M, N, K, TYPES[name][0], bias=db, stride=stride)
        ctx.sync()
    finally:
        ctx.set_option("tensor_cores", 1)
    got = out.get()
    for v in bufs + [out]:
        v.free()
    assert (got[:, N:] == 3.0).all()
    return got[:, :N]


def _check(got, a, b, bias, name, cores=False):
    """Products are exact.  On CUDA cores K sums round once each (2^-24 of at most the magnitudes' sum); on the tensor cores one
    instruction adds 64 of the depth and is cut off by at most 2^-23 of the magnitudes, and runs of the depth join with one rounding
    each.  Then the bias and the type."""
    av, bv = values_mx(*a), values_mx(*b)
    K = av.shape[1]
    want, size = av @ bv.T, np.abs(av) @ np.abs(bv).T
    if bias is not None:
        want, size = want + bias.astype(np.float64), size + np.abs(bias)
    steps = K * 2.0 ** -24 if cores else (K / 64 + 12) * 2.0 ** -23
    bound = size * (steps + 2.0 ** -23) * (1 + HALF[name]) + np.abs(want) * HALF[name] + TINY[name]
    assert (np.abs(got.double().numpy() - want) <= bound).all()


SHAPES = [(1, 1, 1), (1, 16, 32), (1, 4096, 4096), (3, 130, 100), (16, 333, 777), (17, 128, 64), (128, 128, 128), (129, 127, 300), (200, 1000, 513),
          (64, 4099, 256), (513, 640, 1024), (40, 8192, 160), (300, 260, 4096), (1000, 1000, 96),
          (2500, 2100, 160), (2563, 2305, 700), (4097, 1280, 64), (5000, 2300, 4128), (3000, 4224, 2080)]


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm(ctx, name, M, N, K):
    rng = np.random.default_rng(M * 7 + N + K)
    # fp16's range: scales that keep the sums small
    low = 116 if name == "f16" else 110
    a, b = _random_mx(rng, M, K, low, 128), _random_mx(rng, N, K, low, 128)
    bias = rng.standard_normal(N).astype(np.float32) if (M + N) % 2 else None
    got = _gemm(ctx, a, b, bias, name, stride=N + 3 if M % 3 == 0 else None, offset=1 if M == 129 else 0)
    _check(got, a, b, bias, name)


@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (65, 70, 100), (130, 64, 320)])
def test_gemm_on_cuda_cores(ctx, M, N, K):
    rng = np.random.default_rng(M)
    a, b = _random_mx(rng, M, K), _random_mx(rng, N, K)
    bias = rng.standard_normal(N).astype(np.float32)
    _check(_gemm(ctx, a, b, bias, "f32", tensor_cores=0), a, b, bias, "f32", cores=True)


@pytest.mark.parametrize("M,N,K", [(1, 128, 256), (20, 130, 512), (300, 520, 256), (2400, 2200, 512)])
def test_gemm_every_code_and_scale_has_its_place(ctx, M, N, K):
    """One non-zero block of one row of each operand: every other result is zero, that one is the block's product.  A scale or code
    that is taken from another row, block or half gives another power of two."""
    rng = np.random.default_rng(N)
    for _ in range(6):
        a, b = _random_mx(rng, M, K, 120, 121), _random_mx(rng, N, K, 120, 121)
        a[1][:] = rng.integers(100, 150, a[1].shape)
        b[1][:] = rng.integers(100, 150, b[1].shape)
        m, n, k = int(rng.integers(M)), int(rng.integers(N)), int(rng.integers(K))
        only = np.zeros_like(a[0])
        only[m, k] = 2                      # 1.0
        other = np.zeros_like(b[0])
        other[n, k] = 6                     # 4.0
        got = _gemm(ctx, (only, a[1]), (other, b[1]), None, "f32").double().numpy()
        want = np.zeros((M, N))
        want[m, n] = 4.0 * 2.0 ** (int(a[1][m, k // 32]) + int(b[1][n, k // 32]) - 254)
        assert np.array_equal(got, want)


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(20, 132, 512), (300, 516, 96), (300, 518, 96), (3, 130, 1024)])
@pytest.mark.parametrize("pad,offset", [(0, 0), (0, 1), (0, 2), (1, 0), (2, 0), (4, 4)])
def test_gemm_rows_of_every_alignment(ctx, name, M, N, K, pad, offset):
    """Stores of one, two and four values: the same bits, and nothing between the rows."""
    rng = np.random.default_rng(N)
    a, b = _random_mx(rng, M, K, 116, 128), _random_mx(rng, N, K, 116, 128)
    bias = rng.standard_normal(N).astype(np.float32)
    got = _gemm(ctx, a, b, bias, name, stride=N + pad, offset=offset)
    _check(got, a, b, bias, name)
    assert torch.equal(got, _gemm(ctx, a, b, bias, name))


def test_gemm_nan_scale_and_empty_sum(ctx):
    rng = np.random.default_rng(5)
    a, b = _random_mx(rng, 20, 200), _random_mx(rng, 140, 200)
    a[1][7, 3] = 255
    b[1][100, 0] = 255
    got = _gemm(ctx, a, b, None, "f32").numpy()
    nan = np.zeros((20, 140), bool)
    nan[7, :] = nan[:, 100] = True
    assert np.array_equal(np.isnan(got), nan)
    # K = 0: the bias, or zero
    out = Values(ctx, torch.full((3, 5), 9.0))
    bias = ctx.upload(np.arange(5, dtype=np.float32))
    none = Values(ctx, torch.zeros(4))
    ctx.gemm_mxfp4(none, none, none, none, out, 3, 5, 0, 0, bias=bias)
    assert torch.equal(out.get(), torch.arange(5.0).expand(3, 5))


def test_refusals(ctx):
    from mace_b200 import MaceB200Error

    class Odd:
        def __init__(self, v):
            self.ptr = v.ptr + 4
    x = Values(ctx, torch.zeros(64, 64))
    with pytest.raises(MaceB200Error) as e:
        ctx.quantize_mxfp4(x, Odd(x), x, 4, 32, 0)
    assert e.value.code == 1
    with pytest.raises(MaceB200Error) as e:
        ctx.dequantize_mxfp4(x, x, x, 4, 32, 0, stride=31)
    assert e.value.code == 1
    with pytest.raises(MaceB200Error) as e:
        ctx.gemm_mxfp4(x, x, x, Odd(x), x, 4, 4, 32, 0)
    assert e.value.code == 1
    with pytest.raises(MaceB200Error) as e:
        ctx.gemm_mxfp4(x, x, x, x, x, 4, 4, 32, 5)
    assert e.value.code == 1
