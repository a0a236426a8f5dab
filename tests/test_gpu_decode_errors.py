"""What a failed call of a decode-step operator leaves behind: nothing."""
import math

import numpy as np
import pytest
import torch

from decode_ref import Values
from test_gpu_decode_attention import Case

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    import mace_b200
    c = mace_b200.Context(0)
    yield c
    c.close()


def test_scratch_that_cannot_be_had_is_not_the_next_calls_error(ctx):
    """Attention with weights wants 4 bytes per query head and slot; more than the device has is refused, and the calls behind it are as
    they were (one of them asks the runtime for the last error after its launch)."""
    from mace_b200 import MaceB200Error
    c = Case(ctx, "bf16", [100, 3], 8, 2, 64, 16, seed=1)
    length = 1 << 28
    with pytest.raises(MaceB200Error) as e:   # 2^4 sequences x 2^8 heads x 2^28 slots: 4 TiB (no pointer is followed before that)
        ctx.paged_attention(c.dq, c.dk, c.dv, c.dt, c.dn, c.out, 16, 256, 256, 64, c.pages, 16, length // 16, length, 1.0, 2, weights_out=c.w_out,
                            weights_stride=length)
    assert e.value.code == 2
    x = np.arange(96 * 40, dtype=np.float32).reshape(1, 96, 40)
    dx, dy = ctx.upload(x), ctx.alloc(x.nbytes)
    ctx.transpose2d_batched(dx, dy, 1, 96, 40, 4)
    ctx.sync()
    assert np.array_equal(ctx.download(dy, (1, 40, 96), np.float32), x.transpose(0, 2, 1))
    c.run().check()


def test_memory_that_cannot_be_had_is_not_the_next_calls_error(ctx):
    from mace_b200 import MaceB200Error
    with pytest.raises(MaceB200Error) as e:
        ctx.alloc(1 << 42)
    assert e.value.code == 2
    x = np.arange(64, dtype=np.float32).reshape(1, 8, 8)
    dx, dy = ctx.upload(x), ctx.alloc(x.nbytes)
    ctx.transpose2d_batched(dx, dy, 1, 8, 8, 4)
    ctx.sync()
    assert np.array_equal(ctx.download(dy, (1, 8, 8), np.float32), x.transpose(0, 2, 1))


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_attention_over_a_pool_without_pages(ctx, name):
    """Null pools: empty sequences are served, others have pages that are not there."""
    from mace_b200 import MaceB200Error
    c = Case(ctx, name, [40, 0, 700], 8, 2, 64, 16, seed=6)

    class Nowhere:
        ptr = None
    c.dk = c.dv = Nowhere
    c.pages = 0
    with pytest.raises(MaceB200Error) as e:
        c.run()
    assert e.value.code == 4 and "outside its range" in str(e.value)
    assert (c.out.get() == 0).all() and (c.lse.get() == -math.inf).all()
    for b, n in enumerate(c.lengths):
        assert np.array_equal(c.w_out.get().numpy()[b, :, :n], c.w_in[b, :, :n])
    c.dn = ctx.upload(np.zeros(3, np.int32))
    c.run()
    assert (c.out.get() == 0).all()


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lengths,heads,kv_heads,dim,page", [([500, 3, 0, 1000], 8, 2, 64, 16), ([30000, 77], 40, 1, 128, 20), ([9000] * 6, 64, 4, 128, 16),
                                                             ([700] * 3, 6, 2, 50, 16), ([20] * 1100, 4, 2, 64, 16)])
def test_attention_in_place(ctx, name, lengths, heads, kv_heads, dim, page):
    """out == q, on clusters, as runs and in one block: heads are written when no block reads their queries any more."""
    c = Case(ctx, name, lengths, heads, kv_heads, dim, page, seed=3)
    for _ in range(3):
        c.out = c.dq = Values(ctx, c.q)
        c.run().check()


def test_attention_in_place_with_another_stride_is_refused(ctx):
    from mace_b200 import MaceB200Error
    c = Case(ctx, "bf16", [20, 33], 4, 2, 64, 16)
    c.out = c.dq
    with pytest.raises(MaceB200Error) as e:
        c.run(q_stride=300)
    assert e.value.code == 1 and "in place" in str(e.value)


def test_the_widest_rotation(ctx):
    """rotary_dim as large as the header allows, and one pair more."""
    from decode_ref import TYPES, tensor, turn
    from mace_b200 import MaceB200Error
    from test_gpu_decode_rope import _check, _freq
    rng = np.random.default_rng(9)
    name, tokens = "f32", 2
    for rotary, append in ((12288, False), (12290, False), (12286, True), (12288, True)):
        x = tensor(rng, name, tokens, 1, rotary)
        positions = np.array([3, 100000], np.int32)
        dx, dy, dp, df = Values(ctx, x), Values(ctx, x), ctx.upload(positions), ctx.upload(_freq(rotary))
        pools = [ctx.alloc(2 * rotary * 4) for _ in range(2)]

        def call():
            if append:
                ctx.rope_kv_append(dx, dy, dx, dx, *pools, dp, ctx.upload(np.array([1, 0], np.int32)), df, tokens, 1, 1, rotary, rotary, 1, 2, TYPES[name][0])
            else:
                ctx.rope(dx, dy, dp, df, tokens, 1, rotary, rotary, TYPES[name][0])
            ctx.sync()
        if rotary == (12288 if append else 12290):
            with pytest.raises(MaceB200Error) as e:
                call()
            assert e.value.code == 3
            continue
        call()
        want, size = turn(x, positions, _freq(rotary), 1.0, rotary, False)
        _check(dy.get(), want, size, name)


@pytest.mark.parametrize("name,dim,code", [("bf16", 511, 0), ("bf16", 512, 0), ("bf16", 513, 3), ("f32", 513, 3), ("bf16", 4096, 0), ("bf16", 4104, 3)])
def test_the_widest_rows_of_eviction(ctx, name, dim, code):
    from mace_b200 import MaceB200Error
    from test_gpu_decode_evict import _case
    run, check = _case(ctx, name, [30, 9], 1, dim, 4, 10, 1, 2, seed=dim)
    if code:
        with pytest.raises(MaceB200Error) as e:
            run()
        assert e.value.code == code
    else:
        run()
        check()
