"""Plain 64-bit forms of the decode-step operators, from their definitions, and what the tests of them share."""
import math

import numpy as np
import torch

from mace_b200 import capi

TYPES = {"f32": (capi.F32, torch.float32), "f16": (capi.F16, torch.float16), "bf16": (capi.BF16, torch.bfloat16)}
# half a step of a type, relative to the value; and half its smallest subnormal
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}


class Values:
    """A host tensor of one of the types, on the device."""

    def __init__(self, ctx, tensor, offset=0):
        """offset: elements between the allocation's start and the tensor (alignments other than the allocator's)."""
        self.ctx, self.shape, self.dtype = ctx, tuple(tensor.shape), tensor.dtype
        raw = tensor.contiguous().reshape(-1).view(torch.uint8).numpy()
        skip = offset * tensor.element_size()
        self.buf = ctx.upload(np.concatenate([np.zeros(skip, np.uint8), raw, np.zeros(16, np.uint8)]))
        self.ptr, self.nbytes = self.buf.ptr + skip, raw.nbytes
        self.skip = skip

    def get(self):
        raw = self.ctx.download(self.buf, (self.skip + self.nbytes,), np.uint8)[self.skip:]
        return torch.from_numpy(raw.copy()).view(self.dtype).reshape(self.shape)

    def free(self):
        self.buf.free()


def tensor(rng, name, *shape, std=1.0):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * np.float32(std)).to(TYPES[name][1])


def turn(x, positions, freq, magnitude, rotary, interleaved, inverse=False):
    """Rotary positions of x [tokens][heads][dim] in 64 bits, and the sum of its terms' magnitudes."""
    x = x.double().numpy()
    angle = positions.astype(np.float64)[:, None] * freq * (-1.0 if inverse else 1.0)
    c, s = np.cos(angle)[:, None, :], np.sin(angle)[:, None, :]
    y, size = x.copy(), np.abs(x)
    a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, rotary // 2), slice(rotary // 2, rotary))
    y[..., a] = magnitude * (x[..., a] * c - x[..., b] * s)
    y[..., b] = magnitude * (x[..., a] * s + x[..., b] * c)
    size[..., a] = size[..., b] = abs(magnitude) * (np.abs(x[..., a]) + np.abs(x[..., b]))
    return y, size


def attend(q, k, v, scale, begin=0):
    """One head's queries [g][dim] over keys and values [n][dim]: out, lse, p, the largest logit's terms and the values' weighted
    magnitudes, all in 64 bits."""
    q, k, v = q.double(), k.double()[begin:], v.double()[begin:]
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.full((q.shape[0],), -math.inf, dtype=torch.float64), torch.zeros(q.shape[0], 0), 0.0, torch.zeros_like(q)
    s = scale * (q @ k.T)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    terms = float((abs(scale) * (q.abs() @ k.abs().T)).max())
    return p @ v, lse, p, terms, p @ v.abs()


def paged(rng, name, lengths, kv_heads, dim, page, width=None, spare=2, fill=None):
    """Random pools and a table for sequences of these lengths: (k pool, v pool, table, [per sequence (k, v) of [n][kv_heads][dim]]).
    fill: what the rows that no sequence uses hold."""
    each = [-(-n // page) for n in lengths]
    width = max(each + [1]) if width is None else width
    pages = sum(each) + spare
    order = rng.permutation(pages)
    table = np.full((len(lengths), width), -1, np.int32)
    k, v = (tensor(rng, name, pages, kv_heads, page, dim) for _ in range(2))
    used = torch.zeros(pages, page, dtype=torch.bool)
    at = 0
    for b, n in enumerate(each):
        table[b, :n] = order[at:at + n]
        at += n
        for j in range(n):
            used[int(table[b, j]), :min(page, lengths[b] - j * page)] = True
    if fill is not None:
        hole = ~used[:, None, :, None].expand_as(k)
        k[hole], v[hole] = fill, fill
    rows = [tuple(pool[torch.from_numpy(table[b, :each[b]].astype(np.int64))].permute(0, 2, 1, 3).reshape(-1, kv_heads, dim)[:lengths[b]]
                  for pool in (k, v)) for b in range(len(lengths))]
    return k, v, table, rows


GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize_mx(x):
    """Rows of 4-bit codes (uint8 each) and scales [rows][blocks] of a 64-bit array, from the definition."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    full = np.zeros((rows, blocks * 32))
    full[:, :cols] = x
    v = full.reshape(rows, blocks, 32)
    top = np.abs(v).max(-1)
    bad = ~np.isfinite(v).all(-1)
    top = np.where(bad, 0.0, top)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1 - 2, -127)
    e = np.maximum(e, -127)
    a = np.where(bad[..., None], 0.0, np.abs(v)) / np.exp2(e.astype(np.float64))[..., None]
    d = np.abs(a[..., None] - GRID)
    # the nearest; of two as near the even code
    code = np.where(d == d.min(-1, keepdims=True), np.arange(8) % 2, 9).argmin(-1).astype(np.uint8)
    code = np.where(np.signbit(v), code | 8, code)
    code = np.where(bad[..., None], 0, code).astype(np.uint8)
    code.reshape(rows, -1)[:, cols:] = 0
    return code.reshape(rows, -1), np.where(bad, 255, e + 127).astype(np.uint8)


def pack(codes):
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def tile_scales(scales):
    rows, blocks = scales.shape
    tr, tb = -(-rows // 128), -(-blocks // 4)
    out = np.zeros(tr * tb * 512, np.uint8)
    r, b = np.meshgrid(np.arange(rows), np.arange(blocks), indexing="ij")
    out[(r // 128 * tb + b // 4) * 512 + r % 32 * 16 + r // 32 % 4 * 4 + b % 4] = scales
    return out


def values_mx(codes, scales):
    """What codes and scales stand for, in 64 bits."""
    v = np.where(codes & 8, -GRID[codes & 7], GRID[codes & 7]).reshape(*scales.shape, 32)
    unit = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127.0))
    return (v * unit[..., None]).reshape(codes.shape)
