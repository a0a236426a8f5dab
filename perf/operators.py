"""Operators of a language model's decode step, through the framework's device context (mace_b200.capi).

  rope       rotary positions on a tensor of heads: both pair layouts, a part of the head, scaled frequencies,
             the inverse rotation (its gradient)
  append     rotary positions on a step's queries and keys, keys and values written into a paged cache
  attention  one new token per sequence over the paged cache, with the log-sum-exp and, where asked for, the
             attention weight that each slot has collected
  evict      the heaviest slots of each head's cache kept, in order, in other pages
  linear     a layer in 4-bit microscaled floating point: activations quantised, product with the kept weights
  quantize   to 4-bit microscaled floating point and back

A case is one configuration; listed() the ones to watch, draw() any other of the same ranges.  With own false run()
computes the same results from elementary torch operations in 32 bits (angles in 64).
"""
import functools
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LARGEST_BYTES = 1.05e9
LARGEST_FLOPS = 2.7e11


def listed():
    return [
        # a long prompt's queries on their way into attention
        {"name": "rope_prompt", "op": "rope", "type": "bf16", "tokens": 8192, "heads": 32, "dim": 128, "rotary": 128,
         "interleaved": False, "inverse": False, "scaled": False, "far": 8192},
        # a fine-tuning step's gradient: a part of each head in pairs, positions far beyond the first training length
        {"name": "rope_gradient", "op": "rope", "type": "f32", "tokens": 777, "heads": 12, "dim": 80, "rotary": 32,
         "interleaved": True, "inverse": True, "scaled": True, "far": 1000000},
        # the tokens of one decode step of 32 requests
        {"name": "append_step", "op": "append", "type": "bf16", "tokens": 32, "heads": 32, "kv_heads": 8, "dim": 128,
         "rotary": 128, "page": 16, "interleaved": False, "scaled": False, "far": 8192},
        # a prompt's keys and values entering the cache, odd in number, scaled frequencies
        {"name": "append_prompt", "op": "append", "type": "f16", "tokens": 5001, "heads": 32, "kv_heads": 4, "dim": 96,
         "rotary": 64, "page": 32, "interleaved": True, "scaled": True, "far": 131072},
        # one request's token: nothing to hide latency behind
        {"name": "attention_one", "op": "attention", "type": "bf16", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 16, "longest": 1000, "ragged": False, "weights": False},
        # a full batch of requests at different lengths, some just begun
        {"name": "attention_batch", "op": "attention", "type": "bf16", "batch": 64, "heads": 64, "kv_heads": 8,
         "dim": 128, "page": 32, "longest": 8192, "ragged": True, "weights": False},
        # two long documents, collecting the weights that eviction goes by
        {"name": "attention_long", "op": "attention", "type": "f16", "batch": 2, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "longest": 120001, "ragged": False, "weights": True},
        # prompts cut to a quarter before decoding starts
        {"name": "evict_prompt", "op": "evict", "type": "bf16", "batch": 16, "kv_heads": 8, "dim": 128, "page": 32,
         "longest": 8192, "budget": 2048, "sinks": 4, "recent": 256, "ragged": True},
        # one long cache of fp32 values, cut by a few hundred slots as it fills
        {"name": "evict_long", "op": "evict", "type": "f32", "batch": 1, "kv_heads": 4, "dim": 64, "page": 16,
         "longest": 33333, "budget": 33000, "sinks": 1, "recent": 1000, "ragged": False},
        # one token through a layer's weights
        {"name": "linear_token", "op": "linear", "type": "bf16", "m": 1, "n": 4096, "k": 4096, "bias": False},
        # a prompt of odd length through a layer's weights
        {"name": "linear_prompt", "op": "linear", "type": "bf16", "m": 4099, "n": 8192, "k": 4096, "bias": True},
        # a layer's weights brought to 4 bits when a model is loaded
        {"name": "quantize_weights", "op": "quantize", "type": "bf16", "m": 8192, "k": 8192},
    ]


def _log(rng, low, high, step=1):
    """A whole number from low to high, spread over its logarithm, a multiple of step."""
    return max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))) / step)) * step)


def _draw_once(rng):
    op = rng.choice(["rope", "append", "attention", "attention", "evict", "linear", "linear", "quantize"])
    c = {"op": op, "type": rng.choice(["f32", "f16", "bf16", "bf16"])}
    if op in ("rope", "append"):
        c["tokens"] = _log(rng, 1, 8192)
        if op == "rope":
            c["heads"] = _log(rng, 1, 64)
        else:
            c["kv_heads"] = rng.choice([1, 2, 4, 8, 10])
            c["heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 7, 8])
            c["page"] = rng.choice([8, 16, 20, 32, 64])
        c["dim"] = 2 * rng.randint(8, 128) if rng.random() < 0.4 else rng.choice([64, 96, 128, 256])
        c["rotary"] = c["dim"] if rng.random() < 0.6 else 2 * rng.randint(1, c["dim"] // 2)
        c["interleaved"], c["scaled"] = rng.random() < 0.5, rng.random() < 0.4
        if op == "rope":
            c["inverse"] = rng.random() < 0.3
        c["far"] = _log(rng, 100, 1000000)
    elif op in ("attention", "evict"):
        c["batch"] = _log(rng, 1, 64)
        c["kv_heads"] = rng.choice([1, 2, 4, 8, 12])
        c["dim"] = 8 * rng.randint(4, 32) if rng.random() < 0.4 else rng.choice([64, 128, 128, 256])
        c["page"] = rng.choice([8, 16, 16, 20, 32, 64, 128])
        c["longest"] = _log(rng, 1 if op == "attention" else 16, 120000)
        c["ragged"] = rng.random() < 0.6
        if op == "attention":
            c["heads"] = c["kv_heads"] * rng.choice([1, 1, 2, 3, 4, 6, 7, 8, 8, 16, 20])
            c["weights"] = rng.random() < 0.4
        else:
            c["budget"] = max(8, int(c["longest"] * rng.uniform(0.05, 1.0)))
            c["sinks"], c["recent"] = rng.choice([0, 1, 4]), int(c["budget"] * rng.uniform(0.0, 0.5))
    else:
        step = rng.choice([1, 32, 128])
        c["m"], c["k"] = _log(rng, 1, 8192), _log(rng, 32, 8192, step)
        if op == "linear":
            c["n"], c["bias"] = _log(rng, 32, 8192, rng.choice([1, 16, 128])), rng.random() < 0.5
    return c


def draw(rng):
    while True:
        case = _draw_once(rng)
        w = work(case)
        if w["flops"] <= LARGEST_FLOPS and w["bytes"] <= LARGEST_BYTES:
            return case


# ---- inputs -------------------------------------------------------------------------------

class _Dev:
    """A torch tensor where the binding expects a device buffer."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.ptr = tensor.data_ptr()


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, dtype, *shape, std=1.0):
    out = torch.empty(shape, device="cuda", dtype=dtype)
    return out.normal_(0.0, std, generator=g)


def _integers(g, low, high, *shape):
    return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int32)


def _frequencies(c):
    """Radians per position of each pair, and the factor on the rotated values.  Scaled: turns that the first
    training length (8192) does not complete are slowed eightfold, the fast ones stay, those between are mixed."""
    i = torch.arange(c["rotary"] // 2, dtype=torch.float64, device="cuda")
    freq = 10000.0 ** (-2.0 * i / c["rotary"])
    if not c["scaled"]:
        return freq, 1.0
    turns = 8192.0 * freq / (2.0 * math.pi)
    kept = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return freq * kept + freq / 8.0 * (1.0 - kept), 0.1 * math.log(8.0) + 1.0


def _lengths(c, g):
    batch, longest = c["batch"], c["longest"]
    if not c["ragged"]:
        return [longest] * batch
    share = torch.rand(batch, generator=g, device="cuda").cpu().tolist()
    lengths = [max(1, int(longest * s)) for s in share]
    lengths[0] = longest
    return lengths


def _tables(g, pages_each, width):
    """A table of pages for each sequence, pages handed out in random order; and how many the pool has."""
    pages = sum(pages_each) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(pages_each), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages_each):
        table[b, :n] = order[at:at + n]
        at += n
    return table, pages


def _pool(c, g, pages):
    shape = (pages, c["kv_heads"], c["page"], c["dim"])
    return _normal(g, TYPES[c["type"]], *shape), _normal(g, TYPES[c["type"]], *shape)


def _tiled_scales(scales):
    """Scales [rows][blocks] of 32 values as the product takes them: tiles of 128 rows by 4 blocks, in each of which
    a row's four scales lie at (row % 32) * 16 + (row / 32) * 4; absent rows and blocks hold 0."""
    rows, blocks = scales.shape
    tr, tb = -(-rows // 128), -(-blocks // 4)
    full = torch.zeros((tr * 128, tb * 4), dtype=torch.uint8, device="cuda")
    full[:rows, :blocks] = scales
    return full.view(tr, 4, 32, tb, 4).permute(0, 3, 2, 1, 4).contiguous()


def _weights_4bit(g, n, k):
    """A layer's weights in 4 bits: packed codes, low half first, in rows of whole blocks, and E8M0 scales."""
    blocks = -(-k // 32)
    codes = torch.randint(0, 16, (n, blocks * 32), generator=g, device="cuda", dtype=torch.uint8)
    codes[:, k:] = 0
    # magnitudes 4 and 6 lead a block, as its largest value's exponent sets the scale
    codes[:, ::32] |= 6
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scales = torch.randint(118, 123, (n, blocks), generator=g, device="cuda", dtype=torch.uint8)
    return packed.contiguous(), scales


def prepare(case, seed):
    c, g, op, dtype = case, _generator(seed), case["op"], TYPES[case["type"]]
    s = {"case": c}
    if op == "rope":
        s["x"] = _normal(g, dtype, c["tokens"], c["heads"], c["dim"])
        s["y"] = torch.empty_like(s["x"])
        s["positions"] = _integers(g, 0, c["far"], c["tokens"])
        s["freq"], s["magnitude"] = _frequencies(c)
    elif op == "append":
        t, d = c["tokens"], c["dim"]
        # queries, keys and values side by side, as the projection in front leaves them
        s["qkv"] = _normal(g, dtype, t, (c["heads"] + 2 * c["kv_heads"]) * d)
        s["q_out"] = torch.empty((t, c["heads"], d), dtype=dtype, device="cuda")
        pages = -(-t // c["page"]) + 5
        s["k_cache"], s["v_cache"] = _pool(c, g, pages)
        s["slots"] = torch.randperm(pages * c["page"], generator=g, device="cuda")[:t].to(torch.int32)
        s["positions"] = _integers(g, 0, c["far"], t)
        s["freq"], s["magnitude"] = _frequencies(c)
        s["qkv_parts"] = _split_qkv(c, s["qkv"])
    elif op == "attention":
        lengths = _lengths(c, g)
        width = -(-c["longest"] // c["page"])
        s["table"], pages = _tables(g, [-(-n // c["page"]) for n in lengths], width)
        s["k_cache"], s["v_cache"] = _pool(c, g, pages)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        # queries whose logits spread over a few units, so that some slots carry most of the weight
        s["q"] = _normal(g, dtype, c["batch"], c["heads"], c["dim"], std=2.0)
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty((c["batch"], c["heads"]), device="cuda")
        if c["weights"]:
            s["w_in"] = torch.rand((c["batch"], c["kv_heads"], c["longest"]), generator=g, device="cuda")
            s["w_out"] = torch.zeros_like(s["w_in"])
    elif op == "evict":
        lengths = _lengths(c, g)
        width = -(-c["longest"] // c["page"])
        s["table"], pages = _tables(g, [-(-n // c["page"]) for n in lengths], width)
        s["k_cache"], s["v_cache"] = _pool(c, g, pages)
        s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        kept_pages = -(-c["budget"] // c["page"])
        s["new_table"], pages = _tables(g, [kept_pages] * c["batch"], kept_pages)
        s["k_new"], s["v_new"] = _pool(c, g, pages)
        # collected weights spread over orders of magnitude; a part has collected nothing and ties at zero
        shape = (c["batch"], c["kv_heads"], c["longest"])
        w = torch.exp(2.0 * _normal(g, torch.float32, *shape) - 4.0)
        s["w_in"] = w * (torch.rand(shape, generator=g, device="cuda") > 0.1)
        shape = (c["batch"], c["kv_heads"], c["budget"])
        s["w_out"] = torch.zeros(shape, device="cuda")
        s["kept"] = torch.empty(shape, dtype=torch.int32, device="cuda")
        s["new_lengths"] = torch.empty(c["batch"], dtype=torch.int32, device="cuda")
    else:
        m, k = c["m"], c["k"]
        # activations and weights alike have columns that stand out
        s["x"] = _normal(g, dtype, m, k) * (1.0 + 15.0 * (torch.rand(k, generator=g, device="cuda") > 0.99)).to(dtype)
        blocks = -(-k // 32)
        s["xq"] = torch.empty((m, blocks * 16), dtype=torch.uint8, device="cuda")
        s["xs"] = torch.empty((-(-m // 128), -(-blocks // 4), 32, 4, 4), dtype=torch.uint8, device="cuda")
        if op == "linear":
            s["wq"], s["scales"] = _weights_4bit(g, c["n"], k)
            s["ws"] = _tiled_scales(s["scales"])
            s["bias"] = _normal(g, torch.float32, c["n"]) if c["bias"] else None
            s["y"] = torch.empty((m, c["n"]), dtype=dtype, device="cuda")
        else:
            s["y"] = torch.empty_like(s["x"])
    s["dev"] = {name: _Dev(v) for name, v in s.items() if isinstance(v, torch.Tensor)}
    if op == "append":
        s["dev"].update({name: _Dev(v) for name, v in zip("qkv", s["qkv_parts"])})
    torch.cuda.synchronize()
    return s


def _split_qkv(c, qkv):
    return qkv.view(c["tokens"], -1, c["dim"]).split([c["heads"], c["kv_heads"], c["kv_heads"]], dim=1)


# ---- the framework's calls ----------------------------------------------------------------

@functools.lru_cache(maxsize=None)
def _context():
    """The program's one device context: its operators run in order on one stream."""
    from mace_b200 import capi
    return capi.Context(0)


@functools.lru_cache(maxsize=None)
def _type(name):
    from mace_b200 import capi
    return {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16}[name]


def _run_own(c, s):
    ctx, d, op, dtype = _context(), s["dev"], c["op"], _type(c["type"])
    if op == "rope":
        ctx.rope(d["x"], d["y"], d["positions"], d["freq"], c["tokens"], c["heads"], c["dim"], c["rotary"], dtype,
                 interleaved=c["interleaved"], inverse=c["inverse"], magnitude=s["magnitude"])
        return s["y"]
    if op == "append":
        row = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        ctx.rope_kv_append(d["q"], d["q_out"], d["k"], d["v"], d["k_cache"], d["v_cache"], d["positions"], d["slots"],
                           d["freq"], c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["rotary"],
                           s["k_cache"].shape[0], c["page"], dtype, token_strides=(row, row, row),
                           interleaved=c["interleaved"], magnitude=s["magnitude"])
        return s["q_out"], s["k_cache"], s["v_cache"]
    if op == "attention":
        ctx.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["table"], d["lengths"], d["out"], c["batch"],
                            c["heads"], c["kv_heads"], c["dim"], s["k_cache"].shape[0], c["page"], s["table"].shape[1],
                            c["longest"], 1.0 / math.sqrt(c["dim"]), dtype, lse=d["lse"], weights_in=d.get("w_in"),
                            weights_out=d.get("w_out"), weights_stride=c["longest"])
        return (s["out"], s["lse"]) + ((s["w_out"],) if c["weights"] else ())
    if op == "evict":
        ctx.kv_evict(d["k_cache"], d["v_cache"], d["table"], d["lengths"], d["w_in"], d["k_new"], d["v_new"],
                     d["new_table"], d["new_lengths"], d["w_out"], d["kept"], c["batch"], c["kv_heads"], c["dim"],
                     c["page"], s["k_cache"].shape[0], s["table"].shape[1], s["k_new"].shape[0],
                     s["new_table"].shape[1], c["longest"], c["longest"], c["budget"], c["sinks"], c["recent"], dtype)
        return s["kept"], s["new_lengths"], s["w_out"], s["k_new"], s["v_new"]
    ctx.quantize_mxfp4(d["x"], d["xq"], d["xs"], c["m"], c["k"], dtype)
    if op == "linear":
        ctx.gemm_mxfp4(d["xq"], d["xs"], d["wq"], d["ws"], d["y"], c["m"], c["n"], c["k"], dtype, bias=d.get("bias"))
    else:
        ctx.dequantize_mxfp4(d["xq"], d["xs"], d["y"], c["m"], c["k"], dtype)
    return s["y"]


# ---- the plain form -----------------------------------------------------------------------

def _rotate(x, positions, freq, magnitude, rotary, interleaved, inverse, dtype):
    angle = positions.double()[:, None, None] * freq
    cos, sin = angle.cos().float() * magnitude, angle.sin().float() * (-magnitude if inverse else magnitude)
    r = x[..., :rotary].float()
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = r[..., :rotary // 2], r[..., rotary // 2:]
        r = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((r.to(dtype), x[..., rotary:]), -1)


def _heads_of(cache, table):
    """The cache's rows of each sequence and head in order: [batch][kv heads][slots][dim]."""
    rows = cache[table.clamp(min=0)]
    return rows.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_attention(c, s):
    n = c["longest"]
    k = _heads_of(s["k_cache"], s["table"])[:, :, :n].float()
    v = _heads_of(s["v_cache"], s["table"])[:, :, :n].float()
    there = (torch.arange(n, device="cuda") < s["lengths"][:, None])[:, None, None, :]
    q = s["q"].float().view(c["batch"], c["kv_heads"], -1, c["dim"])
    logits = torch.matmul(q, k.transpose(-1, -2)) * (1.0 / math.sqrt(c["dim"]))
    logits = torch.where(there, logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    p = e / total
    out = torch.matmul(p, torch.where(there.squeeze(2)[..., None], v, 0.0))
    lse = (top + torch.log(total)).view(c["batch"], c["heads"])
    out = out.view(c["batch"], c["heads"], c["dim"]).to(s["q"].dtype)
    if not c["weights"]:
        return out, lse
    return out, lse, torch.where(there.squeeze(2), s["w_in"] + p.sum(2), s["w_out"])


def _plain_evict(c, s):
    n, budget = c["longest"], c["budget"]
    slot = torch.arange(n, device="cuda")
    length = s["lengths"][:, None, None]
    rank = torch.where((slot < c["sinks"]) | (slot >= length - c["recent"]), math.inf, s["w_in"])
    rank = torch.where(slot < length, rank, -math.inf)
    first = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    kept = torch.sort(torch.where(first < length, first, n), dim=-1).values
    if kept.shape[-1] < budget:   # no sequence is as long as the budget
        kept = torch.cat((kept, kept.new_full((*kept.shape[:2], budget - kept.shape[-1]), n)), -1)
    there = kept < n
    at = torch.where(there, kept, 0)
    new_lengths = s["lengths"].clamp(max=budget)
    weights = torch.where(there, s["w_in"].gather(-1, at), s["w_out"])
    page = torch.gather(s["table"][:, None, :].expand(-1, c["kv_heads"], -1), -1, at // c["page"]).long()
    head = torch.arange(c["kv_heads"], device="cuda")[None, :, None]
    to = torch.arange(budget, device="cuda")
    to_page = s["new_table"][:, to // c["page"]].long()[:, None, :].expand(-1, c["kv_heads"], -1)
    where_to = (to_page, head.expand_as(to_page), (to % c["page"]).expand_as(to_page))
    caches = []
    for old, new in ((s["k_cache"], s["k_new"]), (s["v_cache"], s["v_new"])):
        rows = old[page, head, at % c["page"]]
        new[where_to] = torch.where(there[..., None], rows, new[where_to])
        caches.append(new)
    return torch.where(there, kept, -1).to(torch.int32), new_lengths, weights, *caches


def _quantized(x, k):
    """x in blocks of 32 as the 4-bit values it is held in, each times its block's power of two, in 32 bits."""
    blocks = -(-k // 32)
    x = torch.nn.functional.pad(x.float(), (0, blocks * 32 - k)).view(-1, blocks, 32)
    exponent = torch.frexp(x.abs().amax(-1, keepdim=True)).exponent - 3
    a = torch.ldexp(x.abs(), -exponent)
    magnitude = (0.5 * ((a > 0.25).float() + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5) + (a >= 3.5)
                 + 2.0 * (a > 5.0))
    return torch.copysign(torch.ldexp(magnitude, exponent), x).view(-1, blocks * 32)


def _dequantized(packed, scales):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device="cuda")
    codes = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).int()
    values = torch.where(codes >= 8, -grid[codes & 7], grid[codes & 7])
    rows, blocks = scales.shape
    return torch.ldexp(values.view(rows, blocks, 32), scales.int()[..., None] - 127).view(rows, -1)


def _run_plain(c, s):
    op, dtype = c["op"], TYPES[c["type"]]
    if op == "rope":
        return _rotate(s["x"], s["positions"], s["freq"], s["magnitude"], c["rotary"], c["interleaved"], c["inverse"],
                       dtype)
    if op == "append":
        q, k, v = s["qkv_parts"]
        turn = (s["positions"], s["freq"], s["magnitude"], c["rotary"], c["interleaved"], False, dtype)
        slots = s["slots"].long()
        page, at = slots // c["page"], slots % c["page"]
        s["k_cache"][page, :, at] = _rotate(k, *turn)
        s["v_cache"][page, :, at] = v
        return _rotate(q, *turn), s["k_cache"], s["v_cache"]
    if op == "attention":
        return _plain_attention(c, s)
    if op == "evict":
        return _plain_evict(c, s)
    x = _quantized(s["x"], c["k"])
    if op == "quantize":
        return x[:, :c["k"]].to(dtype)
    y = torch.matmul(x, _dequantized(s["wq"], s["scales"]).t())
    return (y if s["bias"] is None else y + s["bias"]).to(dtype)


def run(state):
    return _run_own(state["case"], state) if own else _run_plain(state["case"], state)


# ---- the definition in 64 bits ------------------------------------------------------------

def _exact_turn(x, positions, freq, magnitude, rotary, interleaved, inverse):
    """Each pair as a complex number, turned."""
    first, second = (torch.arange(rotary // 2, device="cuda") * step + start for step, start in
                     (((2, 0), (2, 1)) if interleaved else ((1, 0), (1, rotary // 2))))
    x = x.double()
    angle = torch.outer(positions.double(), freq) * (-1.0 if inverse else 1.0)
    turned = torch.polar(torch.full_like(angle, magnitude), angle)[:, None, :]
    z = torch.complex(x[..., first], x[..., second]) * turned
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_attention(c, s):
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros(c["batch"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    lse = torch.full((c["batch"], c["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    weights = s["w_out"].double() if c["weights"] else None
    for b, n in enumerate(s["lengths"].tolist()):
        pages = s["table"][b, :-(-n // c["page"])].long()
        for h in range(c["kv_heads"]):
            k = s["k_cache"][pages, h].reshape(-1, c["dim"])[:n].double()
            v = s["v_cache"][pages, h].reshape(-1, c["dim"])[:n].double()
            mine = slice(h * group, (h + 1) * group)
            logits = s["q"][b, mine].double() @ k.T / math.sqrt(c["dim"])
            lse[b, mine] = torch.logsumexp(logits, -1)
            p = torch.exp(logits - lse[b, mine, None])
            out[b, mine] = p @ v
            if c["weights"]:
                weights[b, h, :n] = s["w_in"][b, h, :n].double() + p.sum(0)
    return (out, lse, weights) if c["weights"] else (out, lse)


def _exact_quantized(x, k):
    """The nearest value of each block's grid, the one with an even code where two are as near."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device="cuda")
    even_first = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7], device="cuda")
    y = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for at in range(0, k, 32):
        v = x[:, at:at + 32].double()
        top = v.abs().amax(-1, keepdim=True)
        # (a power of two can come out just below its logarithm)
        power = torch.floor(torch.log2(top))
        power = power + (torch.exp2(power + 1.0) <= top).double() - (torch.exp2(power) > top).double()
        unit = torch.where(top > 0.0, torch.exp2(power - 2.0), 1.0)
        near = ((v.abs() / unit)[..., None] - grid[even_first]).abs().argmin(-1)
        y[:, at:at + 32] = torch.sign(v) * grid[even_first[near]] * unit
    return y


def exact(case, seed):
    c, s = case, prepare(case, seed)
    op = c["op"]
    if op == "rope":
        return _exact_turn(s["x"], s["positions"], s["freq"], s["magnitude"], c["rotary"], c["interleaved"],
                           c["inverse"])
    if op == "append":
        q, k, v = s["qkv_parts"]
        turn = (s["positions"], s["freq"], s["magnitude"], c["rotary"], c["interleaved"], False)
        cache, turned = s["k_cache"].double(), _exact_turn(k, *turn)
        slots = s["slots"].long()
        cache[slots // c["page"], :, slots % c["page"]] = turned
        return _exact_turn(q, *turn), cache, None
    if op == "attention":
        return _exact_attention(c, s)
    if op == "evict":
        return None   # choices and copies
    x = _exact_quantized(s["x"], c["k"])
    if op == "quantize":
        return x
    codes = torch.empty((c["n"], s["wq"].shape[1] * 2), dtype=torch.long, device="cuda")
    codes[:, 0::2], codes[:, 1::2] = s["wq"].long() % 16, s["wq"].long() // 16
    # magnitude codes 0 .. 7: a subnormal step of a half, then a bit of mantissa under each exponent
    m, e = (codes % 2).double(), (codes % 8) // 2
    w = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * torch.exp2(e.double() - 1.0))
    w = w * (1.0 - 2.0 * (codes // 8).double())
    w = w * torch.exp2(s["scales"].double() - 127.0).repeat_interleave(32, 1)
    y = x @ w[:, :c["k"]].T
    return y if s["bias"] is None else y + s["bias"].double()


# ---- what a pass cannot do without --------------------------------------------------------

def work(case):
    """Inputs read and outputs written once; two operations for a multiplication and its addition."""
    c, op = case, case["op"]
    size = 4 if c["type"] == "f32" else 2
    if op == "rope":
        values = c["tokens"] * c["heads"] * c["dim"]
        return {"bytes": 2 * values * size + 4 * c["tokens"] + 4 * c["rotary"],
                "flops": 3 * c["tokens"] * c["heads"] * c["rotary"]}
    if op == "append":
        heads = c["heads"] + 2 * c["kv_heads"]
        return {"bytes": 2 * c["tokens"] * heads * c["dim"] * size + 8 * c["tokens"] + 4 * c["rotary"],
                "flops": 3 * c["tokens"] * (c["heads"] + c["kv_heads"]) * c["rotary"]}
    if op in ("attention", "evict"):
        # ragged lengths are uniform up to the longest
        slots = c["longest"] * (1 + 0.5 * (c["batch"] - 1) if c["ragged"] else c["batch"])
        if op == "attention":
            heads = 2 * c["batch"] * c["heads"] * c["dim"] * size + 4 * c["batch"] * c["heads"]
            each = 2 * c["dim"] * size + (8 if c["weights"] else 0)
            return {"bytes": slots * (c["kv_heads"] * each + 4.0 / c["page"]) + heads,
                    "flops": 4 * slots * c["heads"] * c["dim"]}
        kept = slots
        if slots > 0:
            share = min(1.0, c["budget"] / c["longest"])
            # the mean of min(length, budget) over uniform lengths; the first sequence has the longest
            rest = c["longest"] * (share - 0.5 * share * share) if c["ragged"] else c["longest"] * share
            kept = c["longest"] * share + (c["batch"] - 1) * rest
        return {"bytes": c["kv_heads"] * (4 * slots + kept * (4 * c["dim"] * size + 8)), "flops": slots * c["kv_heads"]}
    m, k = c["m"], c["k"]
    if op == "quantize":
        return {"bytes": 2 * m * k * size + m * k * 17 / 16, "flops": 2 * m * k}
    return {"bytes": m * k * size + c["n"] * k * 17 / 32 + m * c["n"] * size + (4 * c["n"] if c["bias"] else 0),
            "flops": 2 * m * c["n"] * k}
