"""What a step of a served decoder does between its quantized products.

  append  kv_append_rotary, kv_gather: a step's queries and keys are rotated by
          their positions, keys and values quantized into their slots of the
          4-bit cache, and read back as the values that the cache now stands for;
  attend  kv_attention_scored: attention over that cache with scores capped by
          a tanh, a bias that falls with distance, or a prefix that every
          query sees (one token per request, a few, a prompt, or a mixture);
  route   moe_route_grouped: experts chosen by sigmoid or softmax scores with a
          bias for balance, out of the best groups, their weights, and the rows
          sorted by expert.

Cache of one layer, all 32-bit words (W = head_dim / 8, G = head_dim / group):
  k_q  [blocks, heads, block_size, W]          value j of word w: dim 8 w + j
  k_sb [blocks, heads, block_size, G]          scale | bias << 16, both T
  v_q  [blocks, heads, block_size / 4, W, 4]   as k_q, four tokens interleaved
  v_sb [blocks, heads, block_size / 4, G, 4]
"""
import math
import random

import torch

own = False

TORCH_T = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
NONE = -1  # a slot that is none (0xffffffff)


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------

def _append(name, tokens, heads, kv_heads, dim, gs, block, dtype, rotary, base, interleaved=False, magnitude=1.0,
            first=0, requests=1, padding=0):
    """rotary: dimensions that rotate, with frequencies base ** (-2 i / rotary); first: the tokens before (of one
    request, or the most of any of several that add a token or a few each); padding: tokens without a slot."""
    return {"name": name, "op": "append", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "gs": gs,
            "block": block, "dtype": dtype, "rotary": rotary, "base": base, "interleaved": interleaved,
            "magnitude": magnitude, "first": first, "requests": requests, "padding": padding}


def _attend(name, seqs, q, past, heads, kv_heads, dim, gs, block, dtype, cap=0.0, slopes=False, prefix=False,
            causal=True, window=0, decode=0.0, idle=0, even=False, mix=0):
    """q, past: largest query count and largest length cached before them (log-uniform from 1, or all the largest
    if even); decode: the share of requests with one query; idle: requests without any; prefix: each request's
    first keys are seen by all of its queries."""
    return {"name": name, "op": "attend", "seqs": seqs, "q": q, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "gs": gs, "block": block, "dtype": dtype, "cap": cap, "slopes": slopes, "prefix": prefix,
            "causal": causal, "window": window, "decode": decode, "idle": idle, "even": even, "mix": mix}


def _route(name, tokens, experts, top_k, dtype, sigmoid, bias, groups=1, top_groups=1, group_best=1, normalize=True,
           scale=1.0):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "sigmoid": sigmoid, "bias": bias, "groups": groups, "top_groups": top_groups, "group_best": group_best,
            "normalize": normalize, "scale": scale}


def listed():
    return [
        # One token of one request of a small model (14 heads of 64 over 2): latency.
        _append("append_token", 1, 14, 2, 64, 64, 16, "bf16", 64, 1e6, first=390),
        # A decode step of 61 requests at lengths all over the range, padded to 64.
        _append("append_decode", 64, 32, 8, 128, 64, 16, "bf16", 128, 1e6, first=16384, requests=61, padding=3),
        # A chunk of a long prompt, far from its start, in small groups; cosines and sines scaled as long contexts do.
        _append("append_prompt", 8191, 32, 8, 128, 32, 64, "f16", 128, 5e5, magnitude=1.1875, first=100000),
        # Wide heads of which a quarter rotates, neighbours paired: a prompt of odd length.
        _append("append_partial", 1501, 16, 4, 256, 128, 32, "bf16", 64, 1e4, interleaved=True),
        # One token of one request, scores capped: latency.
        _attend("attend_token", 1, 1, 390, 14, 2, 64, 64, 16, "bf16", cap=50.0, even=True),
        # 48 requests decoded together in a window, wide heads, capped.
        _attend("attend_batch", 48, 1, 8192, 16, 8, 256, 64, 16, "bf16", cap=50.0, window=4096, mix=3),
        # Three very long requests whose scores fall with distance, small groups, fp16, a drafted token each.
        _attend("attend_slopes", 3, 2, 60001, 32, 8, 128, 32, 64, "f16", slopes=True, even=True),
        # A prompt's second half over a cache that holds the first, capped.
        _attend("attend_prompt", 1, 4096, 4096, 32, 8, 128, 64, 64, "bf16", cap=30.0, even=True),
        # Prompts whose prefix all their tokens see, decoded tokens and an idle request in one step, an odd group of
        # heads, scores that fall with distance.
        _attend("attend_mixed", 13, 1500, 3000, 28, 4, 128, 64, 16, "bf16", slopes=True, prefix=True, decode=0.4,
                idle=1, mix=5),
        # A decode step's router: sigmoid scores, a bias, the best groups.
        _route("route_decode", 16, 256, 8, "bf16", True, True, 8, 4, 2, True, 2.5),
        # The same for a prompt, in fp32 as routers compute.
        _route("route_prompt", 8191, 256, 8, "f32", True, True, 8, 4, 2, True, 2.5),
        # Softmax scores, groups of 20 by their best expert, weights as they are.
        _route("route_softmax", 1500, 160, 6, "f32", False, False, 8, 3, 1, False, 16.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """A case of the same ranges."""
    op = rng.choices(["append", "attend", "route"], weights=[3, 6, 3])[0]
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        size = rng.choice([n for n in (2, 3, 4, 8, 13, 16, 20, 32, 64) if groups * n <= 512 and groups * n >= 4])
        best = rng.choice([1, 2])
        kept = rng.randint(max(1, groups // 4), groups)
        top_k = rng.randint(1, min(16, kept * size))
        return _unnamed(_route("", _log_int(rng, 1, 8191), groups * size, top_k, rng.choice(["f32", "bf16", "f16"]),
                               rng.random() < 0.7, rng.random() < 0.7, groups, kept, best, rng.random() < 0.7,
                               rng.choice([1.0, 2.5, 16.0])))
    mix = rng.randrange(1 << 20)
    block = rng.choice([16, 16, 32, 64, 128])
    dim = rng.choice([64, 128, 128, 256])
    gs = rng.choice([g for g in (32, 64, 64, 128) if dim % g == 0])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 6, 7, 8])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op == "append":
        tokens = _log_int(rng, 1, min(8191, 8191 * 32 * 128 // (heads * dim)))
        requests = rng.choice([1, min(tokens, 61)])
        return _unnamed(_append("", tokens, heads, kv_heads, dim, gs, block, dtype,
                                rng.choice([dim, dim, dim // 2, dim // 4]), rng.choice([1e4, 5e5, 1e6]),
                                rng.random() < 0.3, rng.choice([1.0, 1.0, 1.1875]), _log_int(rng, 1, 120000), requests,
                                rng.randint(0, tokens // 8)))
    kind = rng.choice(["token", "token", "batch", "batch", "drafts", "prompt", "mixed"])
    score = dict(zip(("cap", "slopes", "prefix"), rng.choice([(30.0, False, False), (50.0, False, False),
                                                              (0.0, True, False), (0.0, False, True),
                                                              (30.0, True, False), (50.0, False, True),
                                                              (0.0, True, True)])))
    score["window"] = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
    score["causal"] = score["prefix"] or rng.random() < 0.85
    shape = (heads, kv_heads, dim, gs, block, dtype)
    if kind == "token":
        c = _attend("", 1, 1, _log_int(rng, 1, 120001), *shape, even=True, **score)
    elif kind == "batch":
        c = _attend("", _log_int(rng, 2, 64), 1, _log_int(rng, 16, 16384), *shape, idle=rng.choice([0, 1]), mix=mix,
                    **score)
    elif kind == "drafts":
        c = _attend("", _log_int(rng, 1, 32), rng.randint(2, 12), _log_int(rng, 16, 16384), *shape, mix=mix, **score)
    elif kind == "prompt":
        c = _attend("", 1, _log_int(rng, 13, 4096), _log_int(rng, 1, 4096), *shape, even=True, mix=mix, **score)
    else:
        c = _attend("", _log_int(rng, 2, 24), _log_int(rng, 13, 1500), _log_int(rng, 16, 8192), *shape,
                    decode=rng.choice([0.3, 0.7]), idle=rng.choice([0, 1, 2]), mix=mix, **score)
    limit = _cost(next(x for x in listed() if x["name"] == "attend_prompt"))  # no drawn case costs more
    while _cost(c) > limit:
        c["past"] = max(1, int(c["past"] * 0.7))
        c["q"] = max(1, int(c["q"] * 0.85))
        c["seqs"] = max(1, int(c["seqs"] * 0.85))
    return _unnamed(c)


def _unnamed(c):
    return {k: v for k, v in c.items() if k != "name"}


def _cost(c):
    """Seconds, at round rates."""
    w = work(c)
    return w["bytes"] / 4e12 + w["flops"] / 5e14


# --------------------------------------------------------------------------
# Shapes of a case
# --------------------------------------------------------------------------

def _attend_lengths(c):
    """(queries, keys, prefix) of each request; the queries are its newest keys."""
    rng, q, kv, prefix = random.Random(c["mix"]), [], [], []
    for i in range(c["seqs"]):
        n = c["q"] if c["even"] else 1 if rng.random() < c["decode"] else _log_int(rng, 1, c["q"])
        past = c["past"] if c["even"] else _log_int(rng, 1, c["past"])
        share = rng.random()
        if i < c["idle"]:
            n = 0
        q.append(n)
        kv.append(past + n)
        prefix.append(int(share * (past + n)) if c["prefix"] else 0)
    return q, kv, prefix


def _visible(c, n_q, n_kv, prefix):
    """Query-key pairs of one request, and its keys that any query sees."""
    if n_q == 0:
        return 0, 0
    pairs, first, last = 0, n_kv, 0
    for i in range(n_q):
        pos = n_kv - n_q + i
        lo = max(0, pos - c["window"] + 1) if c["window"] else 0
        hi = max(pos + 1, prefix) if c["causal"] else n_kv
        pairs += max(hi - lo, 0)
        first, last = min(first, lo), max(last, hi)
    return pairs, max(last - first, 0)


def work(case):
    """Bytes and operations a pass cannot do without."""
    c = case
    if c["op"] == "route":
        n, rows = c["tokens"] * c["experts"], c["tokens"] * c["top_k"]
        return {"bytes": n * (4 if c["dtype"] == "f32" else 2) + 20 * rows + 4 * (2 * c["experts"] + 1),
                "flops": 8 * n + 8 * rows}
    packed = c["kv_heads"] * (c["dim"] // 2 + 4 * (c["dim"] // c["gs"]))
    if c["op"] == "append":
        n, row, rot = c["tokens"], c["dim"] * 2, c["rotary"] * (c["heads"] + c["kv_heads"])
        # Queries in and out, keys and values in, packed out and in again, dense out.
        return {"bytes": n * (2 * c["heads"] * row + 4 * c["kv_heads"] * row + 4 * packed + 12),
                "flops": n * (3 * rot + 40 * c["rotary"] // 2 + 2 * c["kv_heads"] * c["dim"] * 8)}
    lengths = list(zip(*_attend_lengths(c)))
    seen = [_visible(c, *n) for n in lengths]
    return {"bytes": 2 * packed * sum(k for _, k in seen) + 4 * c["heads"] * c["dim"] * sum(n[0] for n in lengths) +
                     4 * sum(-(-k // c["block"]) for _, k in seen) + 12 * c["seqs"],
            "flops": (4 * c["dim"] + 4) * c["heads"] * sum(p for p, _ in seen)}


# --------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------

def _quantized(x, gs):
    """Values 0..15 and the scale and bias of each group of x[n, heads, dim],
    with a group that holds an Inf or NaN as 0 * 0 + NaN.  Scales are rounded
    to T; a group's lowest value is its bias."""
    g = x.float().reshape(x.shape[0], x.shape[1], -1, gs)
    lo, hi = g.amin(-1), g.amax(-1)
    span = hi - lo
    bad = ~torch.isfinite(span)
    s = torch.where(bad, torch.zeros_like(span), span / 15.0).to(x.dtype)
    b = torch.where(bad, torch.full_like(lo, float("nan")), lo).to(x.dtype)
    sf = s.float()[..., None]
    q = torch.round((g - lo[..., None]) / torch.where(sf == 0, torch.ones_like(sf), sf)).clamp(0, 15)
    q = torch.where((sf == 0) | bad[..., None], torch.zeros_like(q), q)
    return q.to(torch.int32).reshape(x.shape), s, b


def _bits(t):
    return t.view(torch.int16).to(torch.int32) & 0xFFFF


def _store(cache, c, slots, q, s, b, which):
    """Writes quantized rows into their slots, in the cache's layout."""
    n, h = slots.numel(), c["kv_heads"]
    shift = torch.arange(0, 32, 4, device="cuda", dtype=torch.int64)
    words = (q.reshape(n, h, -1, 8).to(torch.int64) << shift).sum(-1)
    words = torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)
    sb = _bits(s) | (_bits(b) << 16)
    blk, off = (slots // c["block"])[:, None], (slots % c["block"])[:, None]
    head = torch.arange(h, device="cuda")[None, :]
    if which == "k":
        cache["k_q"][blk, head, off], cache["k_sb"][blk, head, off] = words, sb
    else:
        cache["v_q"][blk, head, off // 4, :, off % 4] = words
        cache["v_sb"][blk, head, off // 4, :, off % 4] = sb


def _empty_cache(c, blocks, g):
    """A cache as a running server has it: what ended requests left in it, or
    memory that was never written (NaN scales)."""
    h, w, n, bs = c["kv_heads"], c["dim"] // 8, c["dim"] // c["gs"], c["block"]
    nan = 0x7FC07FC0 if c["dtype"] == "bf16" else 0x7E007E00
    words = lambda *shape: torch.randint(-2**31, 2**31, shape, dtype=torch.int32, device="cuda", generator=g)
    return {"k_q": words(blocks, h, bs, w), "v_q": words(blocks, h, bs // 4, w, 4),
            "k_sb": torch.full((blocks, h, bs, n), nan, dtype=torch.int32, device="cuda"),
            "v_sb": torch.full((blocks, h, bs // 4, n, 4), nan, dtype=torch.int32, device="cuda")}


def _keys(c, n, g, size):
    """Keys: some channels carry most of the size, as rotary models' do."""
    x = torch.empty(n, c["kv_heads"], c["dim"], device="cuda").normal_(0.0, 1.0, generator=g)
    return (x * size).to(TORCH_T[c["dtype"]])


def _channel_sizes(c, g):
    size = torch.empty(c["kv_heads"], c["dim"], device="cuda").normal_(0.0, 0.4, generator=g).exp()
    size[:, 5::37] *= 6.0
    return size * 0.8


def _fill(cache, c, slots, g):
    """Keys and values of earlier tokens into the slots given."""
    size = _channel_sizes(c, g)
    for at in range(0, slots.numel(), 16384):
        part = slots[at:at + 16384]
        _store(cache, c, part, *_quantized(_keys(c, part.numel(), g, size), c["gs"]), "k")
        _store(cache, c, part, *_quantized(_keys(c, part.numel(), g, 0.7), c["gs"]), "v")


def _values(case, seed):
    """The case's inputs as torch tensors, a function of the seed alone."""
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    if c["op"] == "route":
        n, e = c["tokens"], c["experts"]
        # Some experts are liked by all tokens; the bias holds them back.
        liked = torch.empty(e, device="cuda").normal_(0.0, 0.7, generator=g)
        logits = torch.empty(n, e, device="cuda").normal_(0.0, 1.3, generator=g) + liked - 1.0
        v = {"logits": logits.to(TORCH_T[c["dtype"]])}
        if c["bias"]:
            v["bias"] = torch.empty(e, device="cuda").normal_(0.0, 0.02, generator=g) - 0.1 * liked
        return v
    bs = c["block"]
    if c["op"] == "append":
        n, h, d = c["tokens"], c["kv_heads"], c["dim"]
        blocks = -(-n // bs) + 5
        order = torch.randperm(blocks, device="cuda", generator=g)
        row = torch.arange(n, device="cuda")
        slots = order[row // bs] * bs + row % bs
        size = _channel_sizes(c, g)
        qkv = torch.empty(n, c["heads"] + 2 * h, d, dtype=TORCH_T[c["dtype"]], device="cuda")
        qkv.normal_(0.0, 1.0, generator=g)
        qkv[:, c["heads"]:c["heads"] + h] = _keys(c, n, g, size)
        qkv[:, c["heads"] + h:] = _keys(c, n, g, 0.7)
        if c["requests"] == 1:
            positions = c["first"] + row
        else:  # a token or a few of each request
            start = torch.randint(0, c["first"] + 1, (c["requests"],), device="cuda", generator=g)
            request = row * c["requests"] // n
            positions = start[request] + row - (request * n + c["requests"] - 1) // c["requests"]
        pad = torch.randperm(n, device="cuda", generator=g)[:c["padding"]]
        slots[pad] = NONE
        positions[pad] = 0
        exponent = torch.arange(0, c["rotary"], 2, device="cuda", dtype=torch.float64) / c["rotary"]
        return {"cache": _empty_cache(c, blocks, g), "qkv": qkv, "slots": slots.to(torch.int32),
                "positions": positions.to(torch.int32), "frequencies": (c["base"] ** -exponent).float()}
    q, kv, prefix = _attend_lengths(c)
    width = max(-(-k // bs) for k in kv) + 2
    used = sum(-(-k // bs) for k in kv)
    blocks = used + 3
    cache = _empty_cache(c, blocks, g)
    order = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    table = torch.full((c["seqs"], width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, k in enumerate(kv):
        n = -(-k // bs)
        table[i, :n] = order[at:at + n]
        row = torch.arange(k, device="cuda")
        _fill(cache, c, table[i].long()[row // bs] * bs + row % bs, g)
        at += n
    starts = [0]
    for n in q:
        starts.append(starts[-1] + n)
    # Queries are the first heads of the fused projection's rows; some heads look sharply.
    qkv = torch.empty(starts[-1], c["heads"] + 2 * c["kv_heads"], c["dim"], dtype=torch.float32, device="cuda")
    qkv.normal_(0.0, 0.8, generator=g)
    sharp = torch.empty(c["heads"], 1, device="cuda").normal_(0.0, 0.5, generator=g).exp()
    qkv[:, :c["heads"]] *= sharp
    v = {"cache": cache, "qkv": qkv.to(TORCH_T[c["dtype"]]), "table": table, "starts": ints(starts),
         "kv_lens": ints(kv)}
    if c["prefix"]:
        v["prefix"] = ints(prefix)
    if c["slopes"]:
        head = torch.arange(1, c["heads"] + 1, device="cuda", dtype=torch.float32)
        v["slopes"] = torch.exp2(-8.0 * head / c["heads"])
    return v


_PROGRAM = {}  # the device and the command session of this program


def _program():
    """The session is on torch's stream."""
    from cider_press_amd.kernels import Device

    if "dev" not in _PROGRAM:
        _PROGRAM["dev"] = Device.system_default()
    stream = torch.cuda.current_stream().cuda_stream
    if stream not in _PROGRAM:
        _PROGRAM[stream] = _PROGRAM["dev"].wrap_stream(stream)
    return _PROGRAM["dev"], _PROGRAM[stream]


class _Memory:
    """A library buffer as torch sees it."""

    TYPES = {"bf16": "<u2", "f16": "<u2", "u32": "<i4", "f32": "<f4"}

    def __init__(self, buf):
        self.buf = buf
        self.__cuda_array_interface__ = {"shape": (len(buf),), "typestr": self.TYPES[buf.dtype],
                                         "data": (buf.ptr, False), "strides": None, "version": 2}


def _view(buf, *shape):
    t = torch.as_tensor(_Memory(buf), device="cuda")
    return (t.view(TORCH_T[buf.dtype]) if buf.dtype in TORCH_T else t).reshape(shape)


def prepare(case, seed):
    c, v = case, _values(case, seed)
    if not own:
        return {"case": c, "v": v}
    from cider_press_amd.kernels import kv as kkv

    dev, cmds = _program()
    buf, out = {}, {}
    names = {t: label for label, t in TORCH_T.items()}

    def load(label, t):
        buf[label] = dev.alloc_buffer(t.numel(), "u32" if t.dtype == torch.int32 else names[t.dtype])
        _view(buf[label], *t.shape).copy_(t)

    def output(label, dtype, *shape):
        buf[label] = dev.alloc_buffer(math.prod(shape), dtype)
        out[label] = _view(buf[label], *shape)
        out[label].zero_()

    for label, t in v.items():
        if label != "cache":
            load(label, t)
    if c["op"] == "route":
        for label in ("experts", "scores", "lhs", "rhs", "inv"):
            output(label, "f32" if label == "scores" else "u32", c["tokens"] * c["top_k"])
        output("offsets", "u32", c["experts"] + 1)
    else:
        t = v["cache"]
        cache = kkv.KvCache(dev, c["dtype"], t["k_q"].shape[0], c["block"], c["kv_heads"], c["dim"], c["gs"])
        for label in ("k_q", "k_sb", "v_q", "v_sb"):
            _view(getattr(cache, label), *t[label].shape).copy_(t[label])
        buf["cache"] = cache
        if c["op"] == "attend":
            output("out", c["dtype"], v["qkv"].shape[0], c["heads"], c["dim"])
            buf["max"] = [max(n) for n in _attend_lengths(c)]
        else:
            output("q", c["dtype"], c["tokens"], c["heads"], c["dim"])
            for label in ("k", "v"):
                output(label, c["dtype"], c["tokens"], c["kv_heads"], c["dim"])
            h, d, n = c["heads"] * c["dim"], c["kv_heads"] * c["dim"], len(buf["qkv"])
            buf["k_in"], buf["v_in"] = buf["qkv"].slice(h, n - h), buf["qkv"].slice(h + d, n - h - d)
    torch.cuda.synchronize()
    return {"case": c, "buf": buf, "out": out}


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------

def run(state):
    if not own:
        return {"append": _plain_append, "attend": _plain_attend,
                "route": _plain_route}[state["case"]["op"]](state["case"], state["v"])
    from cider_press_amd.kernels import kv as kkv, moe as kmoe

    c, b = state["case"], state["buf"]
    _, cmds = _program()
    if c["op"] == "route":
        kmoe.moe_route_grouped(cmds, b["logits"], c["tokens"], c["experts"], c["top_k"], c["normalize"], b["experts"],
                               b["scores"], b["lhs"], b["rhs"], b["inv"], b["offsets"], sigmoid=c["sigmoid"],
                               bias=b.get("bias"), n_groups=c["groups"], top_groups=c["top_groups"],
                               group_best=c["group_best"], scale=c["scale"])
        return state["out"]
    strides = ((c["heads"] + 2 * c["kv_heads"]) * c["dim"], c["dim"])
    if c["op"] == "attend":
        kkv.kv_attention_scored(cmds, b["cache"], b["qkv"], b["table"], len(b["table"]) // c["seqs"], b["starts"],
                                b["kv_lens"], b["out"], state["out"]["out"].shape[0], c["heads"], c["seqs"],
                                b["max"][0], b["max"][1], 1.0 / math.sqrt(c["dim"]), causal=c["causal"],
                                window=c["window"], softcap=c["cap"], slopes=b.get("slopes"),
                                prefix_lens=b.get("prefix"), q_strides=strides)
    else:
        kkv.kv_append_rotary(cmds, b["cache"], b["qkv"], b["k_in"], b["v_in"], b["slots"], b["positions"],
                             b["frequencies"], b["q"], c["tokens"], c["heads"], interleaved=c["interleaved"],
                             magnitude=c["magnitude"], q_strides=strides, k_strides=strides, v_strides=strides)
        kkv.kv_gather(cmds, b["cache"], b["slots"], c["tokens"], b["k"], b["v"])
    return state["out"]


def _plain_rotate(c, v, x):
    """x[tokens, heads, dim] rotated, in 64 bits (far positions; what lies next to a rounding's border decides a
    quantized value), rounded to 32 and then to T, as the cache's append takes keys."""
    half = c["rotary"] // 2
    angle = (v["positions"].double()[:, None] * v["frequencies"].double()[None, :])[:, None, :]
    cos, sin = torch.cos(angle) * c["magnitude"], torch.sin(angle) * c["magnitude"]
    turn, rest = x[..., :c["rotary"]].double(), x[..., c["rotary"]:]
    if c["interleaved"]:
        a, b = turn[..., 0::2], turn[..., 1::2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turn[..., :half], turn[..., half:]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y.float().to(x.dtype), rest], -1)


def _plain_append(c, v):
    t, h = TORCH_T[c["dtype"]], c["kv_heads"]
    live = (v["slots"] >= 0)[:, None, None]
    q = _plain_rotate(c, v, v["qkv"][:, :c["heads"]])
    out = {"q": torch.where(live, q, torch.zeros_like(q))}
    keys = _plain_rotate(c, v, v["qkv"][:, c["heads"]:c["heads"] + h])
    for label, x in (("k", keys), ("v", v["qkv"][:, c["heads"] + h:])):
        q, s, b = _quantized(x, c["gs"])
        q = q.float().reshape(*q.shape[:2], -1, c["gs"])
        y = (q * s.float()[..., None] + b.float()[..., None]).reshape(c["tokens"], h, c["dim"])
        out[label] = torch.where(live, y, torch.zeros_like(y)).to(t)
    return out


def _plain_rows(c, cache, slots):
    """Keys and values in the slots given, as 32-bit floats."""
    blk, off = (slots // c["block"])[:, None], (slots % c["block"])[:, None]
    head = torch.arange(c["kv_heads"], device="cuda")[None, :]
    shift = torch.arange(0, 32, 4, device="cuda", dtype=torch.int32)
    rows = []
    for words, sb in ((cache["k_q"][blk, head, off], cache["k_sb"][blk, head, off]),
                      (cache["v_q"][blk, head, off // 4, :, off % 4], cache["v_sb"][blk, head, off // 4, :, off % 4])):
        s = sb.to(torch.int16).view(TORCH_T[c["dtype"]]).float()
        b = (sb >> 16).to(torch.int16).view(TORCH_T[c["dtype"]]).float()
        q = ((words[..., None] >> shift) & 15).float().reshape(*s.shape, c["gs"])
        rows.append((q * s[..., None] + b[..., None]).reshape(slots.numel(), c["kv_heads"], c["dim"]))
    return rows


def _plain_attend(c, v):
    bs, h, d = c["block"], c["kv_heads"], c["dim"]
    group = c["heads"] // h
    q_all = v["qkv"][:, :c["heads"]]
    out = torch.zeros(q_all.shape, dtype=TORCH_T[c["dtype"]], device="cuda")
    at = 0
    for i, (n_q, n, prefix) in enumerate(zip(*_attend_lengths(c))):
        if n_q == 0:
            continue
        key = torch.arange(n, device="cuda")
        k, x = _plain_rows(c, v["cache"], v["table"][i].long()[key // bs] * bs + key % bs)
        k, x = k.permute(1, 2, 0).contiguous(), x.transpose(0, 1).contiguous()  # [h, d, n], [h, n, d]
        step = max(1, (1 << 27) // (n * c["heads"]))
        for lo in range(0, n_q, step):
            m = min(step, n_q - lo)
            q = q_all[at + lo:at + lo + m].float().reshape(m, h, group, d).permute(1, 0, 2, 3)
            score = torch.matmul(q.reshape(h, m * group, d), k) * (1.0 / math.sqrt(d))
            if c["cap"]:
                score = c["cap"] * torch.tanh(score / c["cap"])
            pos = (n - n_q + lo + torch.arange(m, device="cuda")).repeat_interleave(group)[:, None]
            if c["slopes"]:
                slope = v["slopes"].reshape(h, 1, group).expand(h, m, group).reshape(h, m * group, 1)
                score = score + slope * (key[None, :] - pos).float()
            seen = torch.ones(m * group, n, dtype=torch.bool, device="cuda")
            if c["causal"]:
                seen &= (key[None, :] <= pos) | (key[None, :] < prefix)
            if c["window"]:
                seen &= key[None, :] > pos - c["window"]
            score = torch.where(seen[None], score, torch.full_like(score, -math.inf))
            top = score.amax(-1, keepdim=True)
            p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
            total = p.sum(-1, keepdim=True)
            y = torch.matmul(p, x) / torch.where(total == 0, torch.ones_like(total), total)
            out[at + lo:at + lo + m] = y.reshape(h, m, group, d).permute(1, 0, 2, 3).reshape(m, c["heads"], d)
        at += n_q
    return {"out": out}


def _plain_route(c, v):
    """In 64 bits: a choice between near scores is a whole number."""
    n, e, k, groups = c["tokens"], c["experts"], c["top_k"], c["groups"]
    x = v["logits"].double()
    if c["sigmoid"]:
        s = 1.0 / (1.0 + torch.exp(-x))
    else:
        p = torch.exp(x - x.amax(-1, keepdim=True))
        s = p / p.sum(-1, keepdim=True)
    choice = s + v["bias"].double() if c["bias"] else s
    if groups > 1:
        best = choice.reshape(n, groups, -1).sort(-1, descending=True).values[..., :c["group_best"]].sum(-1)
        kept = best.sort(dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        hidden = torch.ones(n, groups, dtype=torch.bool, device="cuda").scatter_(1, kept, False)
        choice = choice.masked_fill(hidden.repeat_interleave(e // groups, 1), -math.inf)
    pick = choice.sort(dim=-1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, pick)
    if c["normalize"]:
        w = w / w.sum(-1, keepdim=True)
    rows = pick.flatten()
    order = rows.sort(stable=True).indices
    inv = torch.empty_like(order)
    inv[order] = torch.arange(n * k, device="cuda")
    starts = torch.searchsorted(rows[order].contiguous(), torch.arange(e + 1, device="cuda"))
    i32 = lambda t: t.to(torch.int32)
    return {"experts": i32(rows), "scores": (w * c["scale"]).flatten().float(), "lhs": i32(order // k),
            "rhs": i32(rows[order]), "inv": i32(inv), "offsets": i32(starts)}


# --------------------------------------------------------------------------
# The same from the definition, in 64 bits
# --------------------------------------------------------------------------

def _exact_values(c, words, sb):
    """scale * q + bias of packed words [..., W] and constants [..., G]."""
    nibbles = words.contiguous().view(torch.uint8)
    q = torch.stack([nibbles & 15, nibbles >> 4], -1).double().flatten(-2)
    q = q.reshape(*sb.shape, c["gs"])
    pair = sb.contiguous().view(TORCH_T[c["dtype"]]).double().reshape(*sb.shape, 2)
    return (q * pair[..., :1] + pair[..., 1:]).flatten(-2)


def _exact_cache(c, cache):
    """Words and constants of every row, [slots, heads, W or G], of the keys, then of the values."""
    for words, sb in ((cache["k_q"], cache["k_sb"]),
                      (cache["v_q"].transpose(3, 4).flatten(2, 3), cache["v_sb"].transpose(3, 4).flatten(2, 3))):
        yield words.transpose(1, 2).flatten(0, 1), sb.transpose(1, 2).flatten(0, 1)


def _exact_turn(c, v, x):
    """x rotated: each pair a complex number times magnitude * e^(i angle)."""
    r, h = c["rotary"], c["rotary"] // 2
    angle = torch.outer(v["positions"].double(), v["frequencies"].double())[:, None]
    turn = torch.polar(torch.full_like(angle, c["magnitude"]), angle)
    y = x.double().clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if c["interleaved"] else (slice(0, h), slice(h, r))
    z = torch.complex(y[..., first], y[..., second]) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    c, v = case, _values(case, seed)
    if c["op"] == "route":
        return _exact_route(c, v)
    if c["op"] == "append":
        skip = v["slots"] < 0
        out = {"q": _exact_turn(c, v, v["qkv"][:, :c["heads"]])}
        h = c["heads"] + c["kv_heads"]
        # The cache takes keys in T.
        keys = _exact_turn(c, v, v["qkv"][:, c["heads"]:h]).float().to(TORCH_T[c["dtype"]])
        for label, x in (("k", keys), ("v", v["qkv"][:, h:])):
            x = x.double().unflatten(-1, (-1, c["gs"]))
            lo = x.min(-1, keepdim=True).values
            s = ((x.max(-1, keepdim=True).values - lo) / 15).to(TORCH_T[c["dtype"]]).double()
            q = ((x - lo) / s).nan_to_num(0.0, 0.0, 0.0).round().clamp(0, 15)
            out[label] = (q * s + lo).flatten(-2)
        for y in out.values():
            y[skip] = 0
        return out
    rows = list(_exact_cache(c, v["cache"]))
    out = torch.zeros(v["qkv"].shape[0], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    n_q, n_kv, prefix = _attend_lengths(c)
    group, first = c["heads"] // c["kv_heads"], 0
    for i in range(c["seqs"]):
        n, m = n_kv[i], n_q[i]
        slots = (v["table"][i].long()[:, None] * c["block"] + torch.arange(c["block"], device="cuda")).flatten()[:n]
        for head in range(c["heads"] if m else 0):
            if head % group == 0:
                k, x = (_exact_values(c, words[slots, head // group], sb[slots, head // group]) for words, sb in rows)
            for lo in range(0, m, 1024):
                hi = min(m, lo + 1024)
                score = v["qkv"][first + lo:first + hi, head].double() @ k.t() / math.sqrt(c["dim"])
                if c["cap"]:
                    score = torch.tanh_(score.div_(c["cap"])).mul_(c["cap"])
                ahead = torch.arange(n, device="cuda") - torch.arange(n - m + lo, n - m + hi, device="cuda")[:, None]
                if c["slopes"]:
                    score += ahead * v["slopes"][head].double()
                hidden = torch.zeros_like(score, dtype=torch.bool)
                if c["causal"]:
                    hidden |= ahead > 0
                    hidden[:, :prefix[i]] = False
                if c["window"]:
                    hidden |= ahead <= -c["window"]
                score.masked_fill_(hidden, -math.inf)
                out[first + lo:first + hi, head] = torch.softmax(score, -1).nan_to_num(0.0) @ x
        first += m
    return {"out": out}


def _exact_route(c, v):
    """Pick by pick."""
    n, e, groups = c["tokens"], c["experts"], c["groups"]
    x = v["logits"].double()
    s = torch.sigmoid(x) if c["sigmoid"] else torch.softmax(x, -1)
    choice = s + v["bias"].double() if c["bias"] else s.clone()
    token = torch.arange(n, device="cuda")

    def take(values):
        """The lowest index of each row's largest value, which is taken out."""
        index = torch.arange(values.shape[1], device="cuda")
        top = values.max(1, keepdim=True).values
        at = torch.where(values == top, index, values.shape[1]).min(1).values
        values[token, at] = -math.inf
        return at, top[:, 0]

    if groups > 1:
        best = torch.zeros(n, groups, dtype=torch.float64, device="cuda")
        for i in range(groups):
            part = choice[:, i * (e // groups):(i + 1) * (e // groups)].clone()
            for _ in range(c["group_best"]):
                best[:, i] += take(part)[1]
        lost = torch.ones(n, groups, dtype=torch.bool, device="cuda")
        for _ in range(c["top_groups"]):
            lost[token, take(best)[0]] = False
        choice[lost[:, torch.arange(e, device="cuda") * groups // e]] = -math.inf
    pick = torch.stack([take(choice)[0] for _ in range(c["top_k"])], 1)
    w = s[token[:, None], pick] * c["scale"]
    if c["normalize"]:
        w = w / s[token[:, None], pick].sum(1, keepdim=True)
    # Rows in the order of (expert, row), counted.
    rows = pick.flatten()
    key = rows * rows.numel() + torch.arange(rows.numel(), device="cuda")
    order = key.argsort()
    inv = order.argsort()
    counts = torch.zeros(e + 1, dtype=torch.int64, device="cuda")
    counts.scatter_add_(0, rows + 1, torch.ones_like(rows))
    i32 = lambda t: t.to(torch.int32)
    return {"experts": i32(rows), "scores": w.flatten(), "lhs": i32(order // c["top_k"]), "rhs": i32(rows[order]),
            "inv": i32(inv), "offsets": i32(counts.cumsum(0))}
