"""Decode-step operators on tensors of more than 2^31 elements and 2^32 bytes: the first rows, those where an offset passes 31 and 32 bits, and
the last ones are right.  (What lies between is whatever the allocation held.)"""
import numpy as np
import pytest
import torch

from decode_ref import TYPES, Values, pack, quantize_mx, tensor, tile_scales, turn, values_mx
from test_gpu_decode_mxfp4 import _check as check_product
from test_gpu_decode_mxfp4 import _random_mx
from test_gpu_decode_rope import _check as check_turn
from test_gpu_decode_rope import _freq

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mace_b200
    c = mace_b200.Context(0)
    yield c
    c.close()


class _At:
    def __init__(self, buf, skip):
        self.ptr = buf.ptr + skip


def _put(ctx, buf, skip, values):
    raw = values.contiguous().view(torch.uint8).numpy()
    ctx.h2d(_At(buf, skip), raw)
    ctx.sync()


def _take(ctx, buf, skip, *shape, dtype):
    size = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
    return torch.from_numpy(ctx.download(_At(buf, skip), (size,), np.uint8)).view(dtype).reshape(shape)


def test_quantize_and_back(ctx):
    from mace_b200 import capi
    rng = np.random.default_rng(1)
    rows, cols = 66000, 65536                      # 4.3e9 values
    samples = [0, 1, 32767, 32768, 65535, 65536, rows - 1]
    x, y = (ctx.alloc(rows * cols * 2) for _ in range(2))
    codes, scales = ctx.alloc(rows * cols // 2), ctx.alloc(capi.mxfp4_scale_bytes(rows, cols))
    data = {r: tensor(rng, "bf16", 1, cols) for r in samples}
    for r, v in data.items():
        _put(ctx, x, r * cols * 2, v)
    ctx.quantize_mxfp4(x, codes, scales, rows, cols, TYPES["bf16"][0])
    ctx.dequantize_mxfp4(codes, scales, y, rows, cols, TYPES["bf16"][0])
    ctx.sync()
    for r, v in data.items():
        q, s = quantize_mx(v.double().numpy())
        assert np.array_equal(_take(ctx, codes, r * cols // 2, cols // 2, dtype=torch.uint8).numpy(), pack(q)[0])
        tile = _take(ctx, scales, r // 128 * (cols // 128) * 512, cols // 128, 512, dtype=torch.uint8).numpy()
        at = r % 32 * 16 + r // 32 % 4 * 4
        assert np.array_equal(tile[:, at:at + 4].reshape(-1), s[0])
        assert torch.equal(_take(ctx, y, r * cols * 2, 1, cols, dtype=torch.bfloat16), torch.from_numpy(values_mx(q, s)).to(torch.bfloat16))
    for b in (x, y, codes, scales):
        b.free()


@pytest.mark.parametrize("M,N,stride", [(66000, 33001, 33001), (1030, 300, 1 << 22), (9, 300, 1 << 29)])
def test_product(ctx, M, N, stride):
    rng = np.random.default_rng(M)
    K = 96
    a, b = _random_mx(rng, M, K, 116, 128), _random_mx(rng, N, K, 116, 128)
    bufs = [ctx.upload(v) for v in (pack(a[0]), tile_scales(a[1]), pack(b[0]), tile_scales(b[1]))]
    out = ctx.alloc(((M - 1) * stride + N) * 2)
    ctx.gemm_mxfp4(*bufs, out, M, N, K, TYPES["f16"][0], stride=stride)
    ctx.sync()
    picks = sorted({0, M - 1, *(min(M - 1, (1 << p) // stride + d) for p in (31, 32) for d in (-1, 0, 1))})
    got = torch.cat([_take(ctx, out, m * stride * 2, 1, N, dtype=torch.float16) for m in picks])
    check_product(got, (a[0][picks], a[1][picks]), b, None, "f16")
    for v in bufs + [out]:
        v.free()


def test_rope_in_place(ctx):
    rng = np.random.default_rng(2)
    tokens, heads, dim, name = 70000, 32, 1024, "bf16"      # 2.3e9 values
    row = heads * dim
    samples = [0, 1, 32767, 32768, 65535, 65536, tokens - 1]
    positions = rng.integers(0, 1 << 20, tokens).astype(np.int32)
    x, dp, df = ctx.alloc(tokens * row * 2), ctx.upload(positions), ctx.upload(_freq(dim))
    data = {t: tensor(rng, name, 1, heads, dim) for t in samples}
    for t, v in data.items():
        _put(ctx, x, t * row * 2, v)
    ctx.rope(x, x, dp, df, tokens, heads, dim, dim, TYPES[name][0])
    ctx.sync()
    for t, v in data.items():
        want, size = turn(v, positions[t:t + 1], _freq(dim), 1.0, dim, False)
        check_turn(_take(ctx, x, t * row * 2, 1, heads, dim, dtype=torch.bfloat16), want, size, name)
    x.free()


PAGE, KV_HEADS, DIM = 64, 8, 128
PAGES = (1 << 31) // (PAGE * KV_HEADS * DIM) + 8     # of 2^16 values each


def test_append(ctx):
    rng = np.random.default_rng(3)
    name = "f16"
    slots = np.array([0, 77, PAGES * PAGE - 1, (PAGES - 5) * PAGE + 3, (1 << 15) * PAGE - 1, (1 << 15) * PAGE, -1], np.int32)
    tokens = len(slots)
    q, k, v = (tensor(rng, name, tokens, h, DIM) for h in (16, KV_HEADS, KV_HEADS))
    dq, dk, dv = (Values(ctx, t) for t in (q, k, v))
    pools = [ctx.alloc(PAGES * PAGE * KV_HEADS * DIM * 2) for _ in range(2)]
    positions = rng.integers(0, 100000, tokens).astype(np.int32)
    ctx.rope_kv_append(dq, dq, dk, dv, *pools, ctx.upload(positions), ctx.upload(slots), ctx.upload(_freq(DIM)), tokens, 16, KV_HEADS, DIM, DIM,
                       PAGES, PAGE, TYPES[name][0])
    ctx.sync()
    want, size = turn(k, positions, _freq(DIM), 1.0, DIM, False)
    for t, s in enumerate(slots):
        if s < 0:
            continue
        for h in range(KV_HEADS):
            at = ((int(s) // PAGE * KV_HEADS + h) * PAGE + int(s) % PAGE) * DIM * 2
            check_turn(_take(ctx, pools[0], at, 1, DIM, dtype=torch.float16), want[t, h:h + 1], size[t, h:h + 1], name)
            assert torch.equal(_take(ctx, pools[1], at, DIM, dtype=torch.float16), v[t, h])
    for b in pools:
        b.free()


def test_evict(ctx):
    """From the source pool's last pages into the destination's."""
    from test_gpu_decode_evict import choose
    rng = np.random.default_rng(4)
    lengths, budget = [200, 70], 100
    src, dst = ([ctx.alloc(PAGES * PAGE * KV_HEADS * DIM * 2) for _ in range(2)] for _ in range(2))
    table = np.array([[PAGES - 1, 5, PAGES - 2, PAGES - 6], [PAGES - 3, PAGES - 4, -1, -1]], np.int32)
    new = np.array([[PAGES - 1, PAGES - 7], [0, PAGES - 2]], np.int32)
    pages = {int(p): [tensor(rng, "bf16", KV_HEADS, PAGE, DIM) for _ in range(2)] for p in table.reshape(-1) if p >= 0}
    size = KV_HEADS * PAGE * DIM * 2
    for p, kv in pages.items():
        for buf, x in zip(src, kv):
            _put(ctx, buf, p * size, x)
    w = rng.random((2, KV_HEADS, 200)).astype(np.float32)
    kept, weights = Values(ctx, torch.zeros(2, KV_HEADS, budget, dtype=torch.int32)), Values(ctx, torch.zeros(2, KV_HEADS, budget))
    n = Values(ctx, torch.zeros(2, dtype=torch.int32))
    ctx.kv_evict(*src, ctx.upload(table), ctx.upload(np.array(lengths, np.int32)), ctx.upload(w), *dst, ctx.upload(new), n, weights, kept, 2, KV_HEADS, DIM,
                 PAGE, PAGES, 4, PAGES, 2, 200, 200, budget, 4, 20, TYPES["bf16"][0])
    ctx.sync()
    got = {int(p): [_take(ctx, buf, int(p) * size, KV_HEADS, PAGE, DIM, dtype=torch.bfloat16) for buf in dst] for p in new.reshape(-1)}
    for b, length in enumerate(lengths):
        for h in range(KV_HEADS):
            want = choose(w[b, h, :length], budget, 4, 20)
            assert kept.get()[b, h, :len(want)].tolist() == want
            for j, s in enumerate(want):
                for i in range(2):
                    assert torch.equal(got[int(new[b, j // PAGE])][i][h, j % PAGE], pages[int(table[b, s // PAGE])][i][h, s % PAGE])
    for b in src + dst:
        b.free()
