"""The decode-step operators as a program runs them: a transformer layer with 4-bit weights on a paged cache, prompt, steps, eviction,
steps, eager and replayed from a graph.  Every operator's output is checked against the 64-bit form of what it was given."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from decode_ref import HALF, TINY, TYPES, Values, attend, pack, quantize_mx, tensor, tile_scales, turn, values_mx

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mace_b200
    c = mace_b200.Context(0)
    yield c
    c.close()


class Layer:
    """Projections to queries, keys and values, attention, output projection, and the cache of `batch` sequences."""

    def __init__(self, ctx, name, batch, hidden, heads, kv_heads, dim, page, room, seed=0):
        from mace_b200 import capi
        rng = np.random.default_rng(seed)
        self.ctx, self.name, self.type, self.dtype = ctx, name, TYPES[name][0], TYPES[name][1]
        self.batch, self.hidden, self.heads, self.kv_heads, self.dim, self.page = batch, hidden, heads, kv_heads, dim, page
        self.width = (heads + 2 * kv_heads) * dim
        self.wqkv, self.wout = (self._weights(tensor(rng, "f32", n, k, std=k ** -0.5)) for n, k in ((self.width, hidden), (hidden, heads * dim)))
        self.freq_host, self.magnitude = capi.rope_frequencies(dim, scaling=capi.ROPE_RAMP, factor=4.0, original_length=256.0)
        self.freq = ctx.upload(self.freq_host)
        self.width_pages = -(-room // page)
        self.pages = 2 * batch * self.width_pages + 1
        order = rng.permutation(self.pages)[:2 * batch * self.width_pages].astype(np.int32)
        self.tables = order.reshape(2, batch, self.width_pages)       # before and behind an eviction
        self.current, self.room = 0, room
        zero = torch.zeros(self.pages, kv_heads, page, dim, dtype=self.dtype)
        self.k, self.v = Values(ctx, zero), Values(ctx, zero)
        self.table = [ctx.upload(t) for t in self.tables]
        self.lengths = np.zeros(batch, np.int32)
        self.dn = ctx.upload(self.lengths)
        self.weights = [ctx.upload(np.zeros((batch, kv_heads, room), np.float32)) for _ in range(2)]
        self.buffers = {}

    def _weights(self, w):
        from mace_b200 import capi
        rows, cols = w.shape
        x = Values(self.ctx, w)
        q, s = self.ctx.alloc(rows * -(-cols // 32) * 16), self.ctx.alloc(capi.mxfp4_scale_bytes(rows, cols))
        self.ctx.quantize_mxfp4(x, q, s, rows, cols, capi.F32)
        self.ctx.sync()
        return q, s, values_mx(*quantize_mx(w.double().numpy()))

    def prepare(self, tokens):
        """Buffers of a call of so many tokens."""
        from mace_b200 import capi
        if tokens not in self.buffers:
            ctx = self.ctx
            t = lambda *shape: Values(ctx, torch.zeros(*shape, dtype=self.dtype))  # noqa: E731
            inner = self.heads * self.dim
            self.buffers[tokens] = dict(
                x=t(tokens, self.hidden), qkv=t(tokens, self.width), q=t(tokens, inner), o=t(tokens, inner), y=t(tokens, self.hidden),
                lse=Values(ctx, torch.zeros(tokens, self.heads)), positions=ctx.upload(np.zeros(tokens, np.int32)), slots=ctx.upload(np.zeros(tokens, np.int32)),
                xq=ctx.alloc(tokens * self.hidden // 2), xs=ctx.alloc(capi.mxfp4_scale_bytes(tokens, self.hidden)),
                oq=ctx.alloc(tokens * inner // 2), os=ctx.alloc(capi.mxfp4_scale_bytes(tokens, inner)))
        return self.buffers[tokens]

    def project_and_append(self, tokens):
        b, ctx = self.buffers[tokens], self.ctx
        ctx.quantize_mxfp4(b["x"], b["xq"], b["xs"], tokens, self.hidden, self.type)
        ctx.gemm_mxfp4(b["xq"], b["xs"], self.wqkv[0], self.wqkv[1], b["qkv"], tokens, self.width, self.hidden, self.type)
        size = b["qkv"].nbytes // (tokens * self.width)

        class At:
            def __init__(self, skip):
                self.ptr = b["qkv"].ptr + skip * size
        ctx.rope_kv_append(b["qkv"], b["q"], At(self.heads * self.dim), At((self.heads + self.kv_heads) * self.dim), self.k, self.v, b["positions"],
                           b["slots"], self.freq, tokens, self.heads, self.kv_heads, self.dim, self.dim, self.pages, self.page, self.type,
                           token_strides=(self.width,) * 3, magnitude=self.magnitude)

    def attend_and_project(self):
        b, ctx, n = self.buffers[self.batch], self.ctx, self.batch
        w = self.weights[self.current]
        ctx.paged_attention(b["q"], self.k, self.v, self.table[self.current], self.dn, b["o"], n, self.heads, self.kv_heads, self.dim, self.pages,
                            self.page, self.width_pages, self.room, 1 / math.sqrt(self.dim), self.type, lse=b["lse"], weights_in=w, weights_out=w,
                            weights_stride=self.room)
        ctx.quantize_mxfp4(b["o"], b["oq"], b["os"], n, self.heads * self.dim, self.type)
        ctx.gemm_mxfp4(b["oq"], b["os"], self.wout[0], self.wout[1], b["y"], n, self.hidden, self.heads * self.dim, self.type)

    def slots_of(self, sequence, first, count):
        j = np.arange(first, first + count)
        return self.tables[self.current][sequence][j // self.page] * self.page + j % self.page

    def send(self, tokens, x, positions, slots):
        b = self.buffers[tokens]
        raw = x.contiguous().view(torch.uint8).numpy()
        for dst, arr in ((b["x"], raw), (b["positions"], np.asarray(positions, np.int32)), (b["slots"], np.asarray(slots, np.int32)),
                         (self.dn, self.lengths)):
            self.ctx.h2d(dst, np.ascontiguousarray(arr))
        self.ctx.sync()

    # ---- checks: every stage from what it was given ----
    def check_product(self, x, weights, y):
        v = values_mx(*quantize_mx(x.double().numpy()))
        want, size = v @ weights.T, np.abs(v) @ np.abs(weights).T
        # (as in the tests of the product: 64 of the depth an instruction)
        bound = size * (x.shape[1] / 64 + 12) * 2.0 ** -23 * 1.01 + np.abs(want) * HALF[self.name] + TINY[self.name]
        assert (np.abs(y.double().numpy() - want) <= bound).all()

    def check_turn(self, x, got, positions):
        want, size = turn(x, np.asarray(positions), self.freq_host, self.magnitude, self.dim, False)
        bound = size * 2.0 ** -20 * 1.01 + np.abs(want) * HALF[self.name] + TINY[self.name]
        assert (np.abs(got.double().numpy() - want) <= bound).all()

    def cache(self, sequence, n):
        pages = torch.from_numpy(self.tables[self.current][sequence][:-(-n // self.page)].astype(np.int64))
        return tuple(p.get()[pages].permute(0, 2, 1, 3).reshape(-1, self.kv_heads, self.dim)[:n] for p in (self.k, self.v))

    def check_append(self, tokens, positions, slots):
        b = self.buffers[tokens]
        qkv = b["qkv"].get()
        self.check_product(b["x"].get(), self.wqkv[2], qkv)
        q, k, v = qkv.view(tokens, -1, self.dim).split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        self.check_turn(q, b["q"].get().view(tokens, self.heads, self.dim), positions)
        s = torch.from_numpy(np.asarray(slots, np.int64))
        there = s >= 0
        at = s[there] // self.page, s[there] % self.page
        self.check_turn(k[there], self.k.get()[at[0], :, at[1]], np.asarray(positions)[there.numpy()])
        assert torch.equal(self.v.get()[at[0], :, at[1]], v[there])

    def check_attention(self, before):
        b, group = self.buffers[self.batch], self.heads // self.kv_heads
        q, o = b["q"].get().view(self.batch, self.heads, self.dim), b["o"].get().view(self.batch, self.heads, self.dim).double()
        after = self.ctx.download(self.weights[self.current], before.shape, np.float32)
        for i, n in enumerate(self.lengths):
            k, v = self.cache(i, int(n))
            for h in range(self.kv_heads):
                mine = slice(h * group, (h + 1) * group)
                want, _, p, terms, size = attend(q[i, mine], k[:, h], v[:, h], 1 / math.sqrt(self.dim))
                rel = 2 * ((self.dim + 16) * 2.0 ** -23 + 2.0 ** -20) * (terms + 1) + (n / 4 + 150) * 2.0 ** -23 + 2.0 ** -16
                assert ((o[i, mine] - want).abs() <= size * rel + want.abs() * HALF[self.name] + 1e-30).all()
                got = torch.from_numpy(after[i, h, :n].astype(np.float64))
                had = torch.from_numpy(before[i, h, :n].astype(np.float64))
                assert ((got - had - p.sum(0)).abs() <= p.sum(0) * rel + got.abs() * 2.0 ** -22).all()
            assert np.array_equal(after[i, :, n:], before[i, :, n:])
        self.check_product(b["o"].get(), self.wout[2], b["y"].get())


@pytest.mark.parametrize("name", ["bf16", "f16", "f32"])
def test_layer(ctx, name):
    batch, page, room = 3, 16, 160
    layer = Layer(ctx, name, batch, 256, 8, 2, 64, page, room)
    rng = np.random.default_rng(7)
    # prompts of different lengths in one call, padded to the longest: the padding has no slot
    prompts = np.array([90, 41, 1], np.int32)
    tokens = batch * int(prompts.max())
    positions = np.tile(np.arange(prompts.max()), batch)
    slots = np.concatenate([np.concatenate([layer.slots_of(i, 0, n), np.full(prompts.max() - n, -1)]) for i, n in enumerate(prompts)])
    layer.prepare(tokens)
    layer.prepare(batch)
    layer.send(tokens, tensor(rng, name, tokens, 256), positions, slots)
    layer.project_and_append(tokens)
    ctx.sync()
    layer.check_append(tokens, positions, slots)
    layer.lengths = prompts.copy()
    seen = prompts.copy()       # tokens of each sequence so far: the next one's position
    graph = None
    from mace_b200.capi import lib
    L = lib()

    def step(check=True, replay=None):
        x = tensor(rng, name, batch, 256)
        slots = np.concatenate([layer.slots_of(i, int(n), 1) for i, n in enumerate(layer.lengths)])
        layer.lengths = (layer.lengths + 1).astype(np.int32)
        layer.send(batch, x, seen, slots)
        before = ctx.download(layer.weights[layer.current], (batch, 2, room), np.float32)
        if replay is None:
            layer.project_and_append(batch)
            layer.attend_and_project()
        else:
            assert L.mb_graph_launch(ctx.h, replay) == 0
        ctx.sync()
        if check:
            layer.check_append(batch, seen, slots)
            layer.check_attention(before)
        seen[:] += 1

    for _ in range(3):
        step()
    # the same step as a graph: lengths, positions, slots and inputs change in device memory
    assert L.mb_graph_begin(ctx.h) == 0
    layer.project_and_append(batch)
    layer.attend_and_project()
    graph = C.c_void_p()
    assert L.mb_graph_end(ctx.h, C.byref(graph)) == 0
    for i in range(20):
        step(check=i in (0, 19), replay=graph)
    # eviction to half of the longest, into the other pages; weights and lengths go with it
    budget, sinks, recent = 56, 2, 10
    w = ctx.download(layer.weights[0], (batch, 2, room), np.float32)
    old = [layer.cache(i, int(n)) for i, n in enumerate(layer.lengths)]
    packed = Values(ctx, torch.zeros(batch, 2, budget))
    kept = Values(ctx, torch.zeros(batch, 2, budget, dtype=torch.int32))
    ctx.kv_evict(layer.k, layer.v, layer.table[0], layer.dn, layer.weights[0], layer.k, layer.v, layer.table[1], layer.dn, packed, kept, batch, 2,
                 64, page, layer.pages, layer.width_pages, layer.pages, layer.width_pages, room, room, budget, sinks, recent, layer.type)
    ctx.sync()
    from test_gpu_decode_evict import choose
    lengths = np.minimum(layer.lengths, budget).astype(np.int32)
    assert ctx.download(layer.dn, (batch,), np.int32).tolist() == lengths.tolist()
    layer.current = 1
    fresh = np.zeros((batch, 2, room), np.float32)
    for i, n in enumerate(layer.lengths):
        now = layer.cache(i, int(lengths[i]))
        for h in range(2):
            want = choose(w[i, h, :n], budget, sinks, recent)
            assert kept.get()[i, h, :len(want)].tolist() == want
            for a, b in zip(old[i], now):
                assert torch.equal(a[want, h], b[:, h])
            fresh[i, h, :len(want)] = w[i, h, want]
        assert np.array_equal(packed.get().numpy()[i, :, :lengths[i]], fresh[i, :, :lengths[i]])
    ctx.h2d(layer.weights[1], fresh)
    ctx.sync()
    layer.lengths = lengths
    for _ in range(3):
        step()
    L.mb_graph_destroy(ctx.h, graph)


def test_quantized_weights_match_the_host_form(ctx):
    """What Layer's checks rest on: codes and scales of the device are those of the 64-bit form."""
    rng = np.random.default_rng(2)
    w = tensor(rng, "f32", 200, 96)
    q, s = ctx.alloc(200 * 3 * 16), ctx.alloc(2 * 512)
    ctx.quantize_mxfp4(Values(ctx, w), q, s, 200, 96, 0)
    codes, scales = quantize_mx(w.double().numpy())
    assert np.array_equal(ctx.download(q, (200, 48), np.uint8), pack(codes))
    assert np.array_equal(ctx.download(s, (1024,), np.uint8), tile_scales(scales))
