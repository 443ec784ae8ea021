"""Operators of a key/value cache held in 4 bits, as a serving program calls them.

Around the quantized linear layers of a model, a program that serves it keeps
the keys and values of every running request.  Here they are held in the
affine 4-bit format of the weights (x = scale * q + bias per group along the
head dimension), in blocks that a table assigns to requests:

  plan    kv_release, kv_plan: blocks of finished requests go back to the
          free list; from the requests' lengths follow the blocks that a step
          adds to the block table, and each new token's slot and position;
  append  kv_append, kv_gather: a step's keys and values are quantized into
          their slots, and read back as the values that the cache now stands
          for;
  gather  kv_gather: cached rows read back as dense T, as a program does that
          hands a cached prefix on;
  attend  kv_attention: softmax attention of a step's queries over the cache
          (one token per request, a few, a prompt, or a mixture of them).

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

TORCH_T = {"bf16": torch.bfloat16, "f16": torch.float16}
NONE = -1  # a slot that is none (0xffffffff)


# --------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------

def _plan(name, seqs, block, cached, new, decode, finished, cap, mix):
    """cached, new: largest lengths (log-uniform from 1); decode: the share of
    requests that add one token; finished: the share that ended; cap: the
    step's slots (unused ones stay padding)."""
    return {"name": name, "op": "plan", "seqs": seqs, "block": block, "cached": cached, "new": new, "decode": decode,
            "finished": finished, "cap": cap, "mix": mix}


def _rows(name, op, tokens, kv_heads, dim, gs, block, dtype, heads=0, padding=0):
    """heads: query heads of the fused projection that k and v are slices of;
    padding: tokens without a slot."""
    return {"name": name, "op": op, "tokens": tokens, "kv_heads": kv_heads, "dim": dim, "gs": gs, "block": block,
            "dtype": dtype, "heads": heads, "padding": padding}


def _attend(name, seqs, q, past, heads, kv_heads, dim, gs, block, dtype, causal=True, window=0, decode=0.0, idle=0,
            even=False, mix=0):
    """q, past: largest query count and largest length cached before them
    (log-uniform from 1, or all the largest if even); decode: the share of
    requests with one query; idle: requests without any."""
    return {"name": name, "op": "attend", "seqs": seqs, "q": q, "past": past, "heads": heads, "kv_heads": kv_heads,
            "dim": dim, "gs": gs, "block": block, "dtype": dtype, "causal": causal, "window": window,
            "decode": decode, "idle": idle, "even": even, "mix": mix}


def listed():
    return [
        # A decode step of 64 requests: one token each, a block now and then.
        _plan("plan_decode", 64, 16, 8192, 1, 1.0, 0.0, 64, 1),
        # A step of a busy server: prompts beside decodes, some requests ended, padded to a fixed size.
        _plan("plan_mixed", 700, 32, 16384, 3000, 0.8, 0.15, 65536, 2),
        # The keys and values of 64 decoded tokens, slices of the fused projection, three of them padding.
        _rows("append_decode", "append", 64, 8, 128, 64, 16, "bf16", heads=32, padding=3),
        # The keys and values of a long prompt, in small groups.
        _rows("append_prompt", "append", 8191, 8, 128, 32, 64, "f16", heads=32),
        # A short cached prefix of a small model read back (2 heads of 64).
        _rows("gather_prefix", "gather", 333, 2, 64, 64, 16, "bf16"),
        # A long prefix read back.
        _rows("gather_long", "gather", 65536, 8, 128, 64, 32, "bf16"),
        # One token of one request of a small model (14 heads of 64 over 2): latency.
        _attend("attend_token", 1, 1, 390, 14, 2, 64, 64, 16, "bf16", even=True),
        # 48 requests decoded together, lengths all over the range.
        _attend("attend_batch", 48, 1, 8192, 32, 8, 128, 64, 16, "bf16", mix=3),
        # Three very long requests in small groups, fp16.
        _attend("attend_long", 3, 1, 120001, 32, 8, 128, 32, 64, "f16", even=True),
        # Several tokens per request at once (drafted tokens to verify), wide heads, a window.
        _attend("attend_drafts", 16, 5, 6000, 16, 4, 256, 128, 32, "bf16", window=1024, mix=4),
        # A prompt's second half over a cache that holds the first.
        _attend("attend_prompt", 1, 4096, 4096, 32, 8, 128, 64, 64, "bf16", even=True),
        # Chunks of prompts, decoded tokens and idle requests in one step, an odd group of heads, fp16.
        _attend("attend_mixed", 13, 1500, 5000, 28, 4, 128, 64, 16, "f16", decode=0.5, idle=2, mix=5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """A case of the same ranges."""
    op = rng.choices(["plan", "append", "gather", "attend"], weights=[2, 2, 2, 7])[0]
    mix = rng.randrange(1 << 20)
    block = rng.choice([16, 16, 32, 64, 128])
    if op == "plan":
        seqs = _log_int(rng, 1, 700)
        new = rng.choice([1, _log_int(rng, 2, 3000)])
        return _unnamed(_plan("", seqs, block, _log_int(rng, 16, 16384), new, rng.choice([0.0, 0.5, 0.9]),
                              rng.choice([0.0, 0.2]), _log_int(rng, seqs, 65536), mix))
    dim = rng.choice([64, 128, 128, 256])
    gs = rng.choice([g for g in (32, 64, 64, 128) if dim % g == 0])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 6, 7, 8])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if op != "attend":
        most = 8191 if op == "append" else 65536 * 8 * 128 // (kv_heads * dim)
        tokens = _log_int(rng, 1, min(most, 65536))
        return _unnamed(_rows("", op, tokens, kv_heads, dim, gs, block, dtype, heads=rng.choice([0, heads]),
                              padding=rng.randint(0, tokens // 8)))
    kind = rng.choice(["token", "token", "batch", "batch", "drafts", "prompt", "mixed"])
    window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
    causal = rng.random() < 0.85
    if kind == "token":
        c = _attend("", 1, 1, _log_int(rng, 1, 120001), heads, kv_heads, dim, gs, block, dtype, causal, window,
                    even=True)
    elif kind == "batch":
        c = _attend("", _log_int(rng, 2, 64), 1, _log_int(rng, 16, 16384), heads, kv_heads, dim, gs, block, dtype,
                    causal, window, idle=rng.choice([0, 1]), mix=mix)
    elif kind == "drafts":
        c = _attend("", _log_int(rng, 1, 32), rng.randint(2, 12), _log_int(rng, 16, 16384), heads, kv_heads, dim, gs,
                    block, dtype, causal, window, mix=mix)
    elif kind == "prompt":
        c = _attend("", 1, _log_int(rng, 13, 4096), _log_int(rng, 1, 4096), heads, kv_heads, dim, gs, block, dtype,
                    causal, window, even=True)
    else:
        c = _attend("", _log_int(rng, 2, 24), _log_int(rng, 13, 1500), _log_int(rng, 16, 8192), heads, kv_heads, dim,
                    gs, block, dtype, causal, window, decode=rng.choice([0.3, 0.7]), idle=rng.choice([0, 1, 2]),
                    mix=mix)
    limit = _cost(listed()[10])  # the prompt: no drawn case costs more
    while _cost(c) > limit:
        c["past"] = max(1, int(c["past"] * 0.7))
        c["q"] = max(1, int(c["q"] * 0.85))
        c["seqs"] = max(1, int(c["seqs"] * 0.85))
    return _unnamed(c)


def _unnamed(c):
    return {k: v for k, v in c.items() if k != "name"}


def _cost(c):
    """Of an attention case: seconds, at round rates."""
    w = work(c)
    return w["bytes"] / 4e12 + w["flops"] / 5e14


# --------------------------------------------------------------------------
# Shapes of a case
# --------------------------------------------------------------------------

def _plan_lengths(c):
    """(cached, new, finished) of each request."""
    rng, cached, new, finished = random.Random(c["mix"]), [], [], []
    for _ in range(c["seqs"]):
        n = 1 if rng.random() < c["decode"] else _log_int(rng, 1, c["new"])
        have = 0 if n > 1 and rng.random() < 0.5 else _log_int(rng, 1, c["cached"])
        end = rng.random() < c["finished"]
        cached.append(have)
        new.append(0 if end else n)
        finished.append(int(end))
    while sum(new) > c["cap"]:  # what a step does not hold waits
        new[new.index(max(new))] //= 2
    return cached, new, finished


def _attend_lengths(c):
    """(queries, keys) of each request; the queries are its newest keys."""
    rng, q, kv = random.Random(c["mix"]), [], []
    for i in range(c["seqs"]):
        n = c["q"] if c["even"] else 1 if rng.random() < c["decode"] else _log_int(rng, 1, c["q"])
        past = c["past"] if c["even"] else _log_int(rng, 1, c["past"])
        if i < c["idle"]:
            n = 0
        q.append(n)
        kv.append(past + n)
    return q, kv


def _visible(c, n_q, n_kv):
    """Query-key pairs of one request, and its keys that any query sees."""
    if n_q == 0:
        return 0, 0
    pairs, first = 0, n_kv
    w = c["window"] or n_kv + 1
    for i in range(n_q):
        pos = n_kv - n_q + i
        lo, hi = max(0, pos - w + 1), (pos + 1 if c["causal"] else n_kv)
        pairs += hi - lo
        first = min(first, lo)
    return pairs, n_kv - first


def work(case):
    """Bytes and operations a pass cannot do without."""
    c = case
    if c["op"] == "plan":
        cached, new, finished = _plan_lengths(c)
        blocks = sum(-(-(h + n) // c["block"]) for h, n in zip(cached, new))
        return {"bytes": 4 * (8 * c["seqs"] + 2 * c["cap"] + 2 * blocks), "flops": 4 * c["cap"]}
    dense = c["kv_heads"] * c["dim"] * 2
    packed = c["kv_heads"] * (c["dim"] // 2 + 4 * (c["dim"] // c["gs"]))
    if c["op"] in ("append", "gather"):
        n = c["tokens"]
        # Keys and values: dense in (append), packed in or out, dense out.
        return {"bytes": 2 * n * (packed + dense) + 4 * n + (2 * n * (dense + packed) if c["op"] == "append" else 0),
                "flops": 2 * n * c["kv_heads"] * c["dim"] * (6 if c["op"] == "append" else 2)}
    q, kv = _attend_lengths(c)
    seen = [_visible(c, a, b) for a, b in zip(q, kv)]
    return {"bytes": 2 * packed * sum(k for _, k in seen) + 4 * c["heads"] * c["dim"] * sum(q) +
                     4 * sum(-(-k // c["block"]) for _, k in seen) + 8 * c["seqs"],
            "flops": 4 * c["dim"] * c["heads"] * sum(p for p, _ in seen)}


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
    if c["op"] == "plan":
        cached, new, finished = _plan_lengths(c)
        bs = c["block"]
        width = max(-(-(h + n) // bs) for h, n in zip(cached, new)) + 3
        have = [-(-h // bs) for h in cached]
        need = sum(max(0, -(-(h + n) // bs) - k) for h, n, k in zip(cached, new, have))
        ids = torch.randperm(sum(have) + need + 17, device="cuda", generator=g).to(torch.int32)
        table = torch.full((c["seqs"], width), -1, dtype=torch.int32, device="cuda")
        column = torch.arange(width, device="cuda")[None, :]
        table[column < ints(have)[:, None]] = ids[:sum(have)]
        free = torch.full((ids.numel(),), -1, dtype=torch.int32, device="cuda")
        free[:need + 17] = ids[sum(have):]
        return {"finished": ints(finished), "lens": ints(cached), "new": ints(new), "table": table, "free": free,
                "free_count": ints([need + 17])}
    bs = c["block"]
    if c["op"] in ("append", "gather"):
        n, h, d = c["tokens"], c["kv_heads"], c["dim"]
        blocks = -(-n // bs) + 5
        order = torch.randperm(blocks, device="cuda", generator=g)
        row = torch.arange(n, device="cuda")
        slots = order[row // bs] * bs + row % bs
        cache = _empty_cache(c, blocks, g)
        out = {"cache": cache}
        if c["op"] == "gather":
            _fill(cache, c, slots, g)
        else:
            size = _channel_sizes(c, g)
            qkv = torch.empty(n, c["heads"] + 2 * h, d, dtype=TORCH_T[c["dtype"]], device="cuda")
            qkv.normal_(0.0, 1.0, generator=g)
            qkv[:, c["heads"]:c["heads"] + h] = _keys(c, n, g, size)
            qkv[:, c["heads"] + h:] = _keys(c, n, g, 0.7)
            out["qkv"] = qkv
        pad = torch.randperm(n, device="cuda", generator=g)[:c["padding"]]
        slots[pad] = NONE
        out["slots"] = slots.to(torch.int32)
        return out
    q, kv = _attend_lengths(c)
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
    return {"cache": cache, "qkv": qkv.to(TORCH_T[c["dtype"]]), "table": table, "starts": ints(starts),
            "kv_lens": ints(kv)}


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

    TYPES = {"bf16": "<u2", "f16": "<u2", "u32": "<i4"}

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

    def load(label, t):
        dtype = "u32" if t.dtype == torch.int32 else c["dtype"]
        buf[label] = dev.alloc_buffer(t.numel(), dtype)
        _view(buf[label], *t.shape).copy_(t)

    def output(label, dtype, *shape):
        buf[label] = dev.alloc_buffer(math.prod(shape), dtype)
        out[label] = _view(buf[label], *shape)

    for label, t in v.items():
        if label != "cache":
            load(label, t)
    if c["op"] == "plan":
        out["table"], out["free"] = (_view(buf[k], *v[k].shape) for k in ("table", "free"))
        for label, n in (("lens_out", c["seqs"]), ("released", 1), ("starts", c["seqs"] + 1), ("kv_lens", c["seqs"]),
                         ("slots", c["cap"]), ("positions", c["cap"]), ("left", 1)):
            output(label, "u32", n)
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
            for label in ("k", "v"):
                output(label, c["dtype"], c["tokens"], c["kv_heads"], c["dim"])
            if c["op"] == "append":
                h, d = c["heads"] * c["dim"], c["kv_heads"] * c["dim"]
                n = len(buf["qkv"])
                buf["k_in"], buf["v_in"] = buf["qkv"].slice(h, n - h), buf["qkv"].slice(h + d, n - h - d)
    torch.cuda.synchronize()
    return {"case": c, "buf": buf, "out": out}


# --------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------

def run(state):
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "gather": _plain_gather,
                "attend": _plain_attend}[state["case"]["op"]](state["case"], state["v"])
    from cider_press_amd.kernels import kv as kkv

    c, b = state["case"], state["buf"]
    _, cmds = _program()
    if c["op"] == "plan":
        width = len(b["table"]) // c["seqs"]
        kkv.kv_release(cmds, b["finished"], b["lens"], b["table"], width, c["block"], b["free"], b["free_count"],
                       b["lens_out"], b["released"])
        kkv.kv_plan(cmds, b["lens_out"], b["new"], b["table"], width, c["block"], b["free"], b["released"],
                    b["starts"], b["kv_lens"], b["slots"], b["positions"], b["left"])
    elif c["op"] == "attend":
        row = (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        kkv.kv_attention(cmds, b["cache"], b["qkv"], b["table"], len(b["table"]) // c["seqs"], b["starts"],
                         b["kv_lens"], b["out"], state["out"]["out"].shape[0], c["heads"], c["seqs"], b["max"][0],
                         b["max"][1], 1.0 / math.sqrt(c["dim"]), causal=c["causal"], window=c["window"],
                         q_strides=(row, c["dim"]))
    else:
        if c["op"] == "append":
            strides = ((c["heads"] + 2 * c["kv_heads"]) * c["dim"], c["dim"])
            kkv.kv_append(cmds, b["cache"], b["k_in"], b["v_in"], b["slots"], c["tokens"], k_strides=strides,
                          v_strides=strides)
        kkv.kv_gather(cmds, b["cache"], b["slots"], c["tokens"], b["k"], b["v"])
    return state["out"]


def _plain_plan(c, v):
    bs, width = c["block"], v["table"].shape[1]
    column = torch.arange(width, device="cuda")[None, :]
    lens, table, free = v["lens"].long(), v["table"].long(), v["free"].long()
    # Blocks of finished requests go on top of the free ones, in the requests' order.
    done = v["finished"] != 0
    back = table[done[:, None] & (column < ((lens + bs - 1) // bs)[:, None])]
    released = v["free_count"].long() + back.numel()
    free = free.clone()
    free[v["free_count"].long() + torch.arange(back.numel(), device="cuda")] = back
    lens = torch.where(done, torch.zeros_like(lens), lens)
    # New blocks come from the top.
    new = v["new"].long()
    kv = lens + new
    have, want = (lens + bs - 1) // bs, (kv + bs - 1) // bs
    first = torch.cumsum(want - have, 0) - (want - have)
    fresh = (column >= have[:, None]) & (column < want[:, None])
    index = released - 1 - (first[:, None] + column - have[:, None])
    table = torch.where(fresh, free[index.clamp(0, free.numel() - 1)], table)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), torch.cumsum(new, 0)])
    token = torch.arange(c["cap"], device="cuda")
    seq = torch.searchsorted(starts[1:], token, right=True).clamp(max=c["seqs"] - 1)
    live = token < starts[-1]
    pos = torch.where(live, lens[seq] + token - starts[seq], torch.zeros_like(token))
    slot = torch.where(live, table[seq, pos // bs] * bs + pos % bs, torch.full_like(token, NONE))
    i32 = lambda t: t.to(torch.int32)
    return {"table": i32(table), "free": i32(free), "lens_out": i32(lens), "released": i32(released),
            "starts": i32(starts), "kv_lens": i32(kv), "slots": i32(slot), "positions": i32(pos),
            "left": i32(released - (want - have).sum())}


def _plain_append(c, v):
    t, h = TORCH_T[c["dtype"]], c["kv_heads"]
    out = {}
    for label, at in (("k", c["heads"]), ("v", c["heads"] + h)):
        q, s, b = _quantized(v["qkv"][:, at:at + h], c["gs"])
        q = q.float().reshape(*q.shape[:2], -1, c["gs"])
        x = (q * s.float()[..., None] + b.float()[..., None]).reshape(c["tokens"], h, c["dim"])
        out[label] = torch.where((v["slots"] >= 0)[:, None, None], x, torch.zeros_like(x)).to(t)
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


def _plain_gather(c, v):
    slots = v["slots"].long()
    live = (slots >= 0)[:, None, None]
    t, out = TORCH_T[c["dtype"]], {"k": [], "v": []}
    for at in range(0, c["tokens"], 16384):
        for label, x in zip(("k", "v"), _plain_rows(c, v["cache"], slots[at:at + 16384].clamp(min=0))):
            out[label].append(torch.where(live[at:at + 16384], x, torch.zeros_like(x)).to(t))
    return {label: torch.cat(parts) for label, parts in out.items()}


def _plain_attend(c, v):
    bs, h, d = c["block"], c["kv_heads"], c["dim"]
    group = c["heads"] // h
    q_all = v["qkv"][:, :c["heads"]]
    out = torch.zeros(q_all.shape, dtype=TORCH_T[c["dtype"]], device="cuda")
    at = 0
    for i, (n_q, n) in enumerate(zip(*_attend_lengths(c))):
        if n_q == 0:
            continue
        key = torch.arange(n, device="cuda")
        k, x = _plain_rows(c, v["cache"], v["table"][i].long()[key // bs] * bs + key % bs)
        k, x = k.permute(1, 2, 0).contiguous(), x.transpose(0, 1).contiguous()  # [h, d, n], [h, n, d]
        step = max(1, (1 << 28) // (n * c["heads"]))
        for lo in range(0, n_q, step):
            m = min(step, n_q - lo)
            q = q_all[at + lo:at + lo + m].float().reshape(m, h, group, d).permute(1, 0, 2, 3)
            score = torch.matmul(q.reshape(h, m * group, d), k) * (1.0 / math.sqrt(d))
            pos = (n - n_q + lo + torch.arange(m, device="cuda")).repeat_interleave(group)[:, None]
            seen = torch.ones(m * group, n, dtype=torch.bool, device="cuda")
            if c["causal"]:
                seen &= key[None, :] <= pos
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


def exact(case, seed):
    c, v = case, _values(case, seed)
    if c["op"] == "plan":
        return _exact_plan(c, v)
    if c["op"] == "append":
        out = {}
        for label, at in (("k", c["heads"]), ("v", c["heads"] + c["kv_heads"])):
            x = v["qkv"][:, at:at + c["kv_heads"]].double().unflatten(-1, (-1, c["gs"]))
            lo = x.min(-1, keepdim=True).values
            s = ((x.max(-1, keepdim=True).values - lo) / 15).to(TORCH_T[c["dtype"]]).double()
            q = ((x - lo) / s).nan_to_num(0.0, 0.0, 0.0).round().clamp(0, 15)
            y = (q * s + lo).flatten(-2)
            y[v["slots"] < 0] = 0
            out[label] = y
        return out
    rows = list(_exact_cache(c, v["cache"]))
    if c["op"] == "gather":
        slots = v["slots"].long()
        out = {}
        for label, (words, sb) in zip(("k", "v"), rows):
            out[label] = _exact_values(c, words[slots.clamp(min=0)], sb[slots.clamp(min=0)])
            out[label][slots < 0] = 0
        return out
    out = torch.zeros(v["qkv"].shape[0], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    n_q, n_kv = _attend_lengths(c)
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
                ahead = torch.arange(n, device="cuda") - torch.arange(n - m + lo, n - m + hi, device="cuda")[:, None]
                hidden = torch.zeros_like(score, dtype=torch.bool)
                if c["causal"]:
                    hidden |= ahead > 0
                if c["window"]:
                    hidden |= ahead <= -c["window"]
                score.masked_fill_(hidden, -math.inf)
                out[first + lo:first + hi, head] = torch.softmax(score, -1).nan_to_num(0.0) @ x
        first += m
    return {"out": out}


def _exact_plan(c, v):
    """Request by request, on lists."""
    bs = c["block"]
    table, free, lens = v["table"].tolist(), v["free"].tolist(), v["lens"].tolist()
    top = v["free_count"].item()
    for i, end in enumerate(v["finished"].tolist()):
        if end:
            for block in table[i][:-(-lens[i] // bs)]:
                free[top] = block
                top += 1
            lens[i] = 0
    released, starts, kv, slots, positions = top, [0], [], [], []
    for i, n in enumerate(v["new"].tolist()):
        for p in range(lens[i], lens[i] + n):
            if p % bs == 0:
                top -= 1
                table[i][p // bs] = free[top]
            positions.append(p)
            slots.append(table[i][p // bs] * bs + p % bs)
        kv.append(lens[i] + n)
        starts.append(len(slots))
    rest = c["cap"] - len(slots)
    t = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return {"table": t(table), "free": t(free), "lens_out": t(lens), "released": t([released]), "starts": t(starts),
            "kv_lens": t(kv), "slots": t(slots + [NONE] * rest), "positions": t(positions + [0] * rest),
            "left": t([top])}
