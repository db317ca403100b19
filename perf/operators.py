"""The quantised key/value cache and the attention around it, as measured cases.

Four operators, in their plain form (elementary torch operations in 32 bits) and as calls of
``mignon_ai_b200.kv``:

* ``write``  rows of keys and values are quantised into a cache of 4 or 8 bits and read back;
* ``read``   positions of the cache's sessions are read back as rows;
* ``attend`` one query token per session over its cached positions, with a sliding window and a
  few first positions that stay visible;
* ``window`` causal attention of whole segments with the same mask, before anything is quantised.

The quantiser, for one row x of one head (float32 arithmetic, each step rounded):
  center = bf16(0.5 max x + 0.5 min x),  half = max(max x - center, center - min x),
  scale = half * (1/15 or 1/127) rounded up to bfloat16 (0 where half < 2^-100),
  m = the odd integer in [-15, 15] (4 bits) or the integer in [-127, 127] (8 bits) that is next to
  (x - center) / scale; the row reads back as center + scale * m.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one decode step's keys and values of 4096 sessions of the 4-head, 128-wide attention model
        _write("write-step-f32-4bit", segs=4096, rows=1, heads=4, dim=32, bits=4, slots=128, sinks=0, dtype="f32"),
        # prompts of uneven length going into the cache of a grouped-head model
        _write("write-prompts-bf16-4bit", segs=250, rows=511, heads=8, dim=128, bits=4, slots=512, sinks=0, dtype="bf16"),
        # one long session read back before its next prompt is processed
        _read("read-long-bf16-4bit", segs=1, rows=65536, heads=8, dim=128, bits=4, slots=65536, sinks=0, dtype="bf16"),
        # many short sessions read back, uneven lengths
        _read("read-short-f32-8bit", segs=500, rows=128, heads=4, dim=48, bits=8, slots=128, sinks=4, dtype="f32"),
        # one session of the 4-head, 128-wide model: the latency of a single token
        _attend("attend-one-f32-4bit", sessions=1, q_heads=4, heads=4, dim=32, bits=4, slots=128, sinks=0, window=64,
                wraps=0, dtype="f32"),
        # a decode step of 4096 sessions of that model
        _attend("attend-4096-f32-4bit", sessions=4096, q_heads=4, heads=4, dim=32, bits=4, slots=128, sinks=0,
                window=64, wraps=0, dtype="f32"),
        # sessions kept to a window by a ring behind four pinned first positions, all wrapped
        _attend("attend-ring-f16-8bit", sessions=257, q_heads=6, heads=6, dim=64, bits=8, slots=1028, sinks=4,
                window=1000, wraps=1, dtype="f16"),
        # a batch of long sessions of uneven length, grouped heads
        _attend("attend-64-bf16-4bit", sessions=64, q_heads=32, heads=8, dim=128, bits=4, slots=8192, sinks=0, window=0,
                wraps=0, dtype="bf16"),
        # one very long session: little to batch, the context itself is the work
        _attend("attend-long-bf16-4bit", sessions=1, q_heads=32, heads=8, dim=128, bits=4, slots=262144, sinks=0,
                window=0, wraps=0, dtype="bf16"),
        # one short prompt: latency
        _window("window-one-f32", segs=1, q_rows=48, past=0, q_heads=4, heads=4, dim=32, window=64, sinks=0,
                dtype="f32"),
        # prompts of 16 to 64 tokens of the 6-head, 384-wide model
        _window("window-prompts-f32", segs=2000, q_rows=64, past=0, q_heads=6, heads=6, dim=64, window=64, sinks=0,
                dtype="f32"),
        # a long document under a window with four sink positions
        _window("window-long-bf16", segs=1, q_rows=8192, past=0, q_heads=32, heads=8, dim=128, window=1024, sinks=4,
                dtype="bf16"),
    ]


def _write(name, **c):
    return dict({"name": name} if name else {}, op="write", **c)


def _read(name, **c):
    return dict({"name": name} if name else {}, op="read", **c)


def _attend(name, **c):
    return dict({"name": name} if name else {}, op="attend", **c)


def _window(name, **c):
    return dict({"name": name} if name else {}, op="window", **c)


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("write", "read", "attend", "window"))
    dtype = rng.choice(("f32", "f16", "bf16"))
    dim = rng.choice((32, 48, 64, 80, 96, 128))
    heads = rng.choice((1, 2, 3, 4, 6, 8))
    bits = rng.choice((4, 8))
    if op in ("write", "read"):
        segs = _spread(rng, 1, 4096)
        rows = _spread(rng, 1, max(1, min(65536, 64_000_000 // (segs * heads * dim))))
        sinks = rng.choice((0, 0, 1, 4, 7))
        # a cache longer than the segments, or (for sessions kept to a window) shorter than them
        slots = sinks + max(8, rng.choice((rows, rows + rng.randint(1, 100), (rows + 1) // 2)))
        make = _write if op == "write" else _read
        return make(None, segs=segs, rows=rows, heads=heads, dim=dim, bits=bits, slots=slots, sinks=sinks, dtype=dtype)
    group = rng.choice((1, 1, 2, 3, 4, 5, 8, 11))
    window = 0 if rng.random() < 0.4 else 1
    sinks = rng.choice((0, 0, 1, 4, 33)) if window else 0
    if op == "attend":
        sessions = _spread(rng, 1, 4096)
        most = max(64, min(262144, 250_000_000 // (sessions * heads * dim * max(1, group // 2))))
        slots = sinks + _spread(rng, 16, most)
        window = rng.randint(1, slots - sinks) if window else 0
        return _attend(None, sessions=sessions, q_heads=heads * group, heads=heads, dim=dim, bits=bits, slots=slots,
                       sinks=sinks, window=window, wraps=rng.choice((0, 1)), dtype=dtype)
    segs = _spread(rng, 1, 1000)
    rows = _spread(rng, 1, max(8, min(8192, int(math.sqrt(1.0e9 / (segs * heads * group))))))
    past = rng.choice((0, 0, rng.randint(1, rows)))
    window = _spread(rng, 1, rows + past) if window else 0
    return _window(None, segs=segs, q_rows=rows, past=past, q_heads=heads * group, heads=heads, dim=dim, window=window,
                   sinks=sinks, dtype=dtype)


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _lengths(g, n, most):
    """n lengths spread evenly from `most` down to a quarter of it, in the seed's order."""
    lens = most - torch.arange(n, device="cuda") * (most - max(1, most // 4)) // max(1, n - 1)
    return lens[torch.randperm(n, generator=g, device="cuda")].int()


def _starts(lens):
    return torch.cat([lens.new_zeros(1), lens.cumsum(0, dtype=torch.int32)])


def _keys(g, shape, dtype):
    """Keys as models have them: a few channels of each head carry an offset far above the rest."""
    x = torch.randn(shape, generator=g, device="cuda")
    off = torch.randn(shape[-2:], generator=g, device="cuda")
    return x.add_(torch.where(off.abs() > 1.8, 3 * off, 0.3 * off)).to(dtype)


def _values(g, shape, dtype):
    """Values: normal, the size of a token's values varying from token to token."""
    size = torch.exp(0.5 * torch.randn((*shape[:-2], 1, 1), generator=g, device="cuda"))
    return torch.randn(shape, generator=g, device="cuda").mul_(size).to(dtype)


def _inputs(case, seed):
    """The rows of a case, its positions and its queries: what is made from the seed."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {}
    dtype, heads, dim = _DTYPES[case["dtype"]], case["heads"], case["dim"]
    if case["op"] in ("write", "read"):
        n, most = case["segs"], case["rows"]
        lens = _lengths(g, n, most)
        # where a write starts in its session: anywhere the session has room for, 0 for reads
        room = max(0, case["slots"] - most) if case["op"] == "write" else 0
        s["pos0"] = torch.randint(0, room + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["lens"], s["start"] = s["pos0"] + lens, _starts(lens)
        s["n_rows"] = int(s["start"][-1])
        shape = (s["n_rows"], heads, dim)
    elif case["op"] == "attend":
        n, slots, sinks = case["sessions"], case["slots"], case["sinks"]
        ring = slots - sinks
        # wrapped sessions have seen one to four times what their ring holds; the others fill part of it
        more = torch.randint(0, 3 * ring + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
        s["lens"] = slots + more if case["wraps"] else _lengths(g, n, slots)
        s["base"] = torch.clamp(s["lens"] - ring, min=sinks)  # the first position that the ring holds
        s["q"] = torch.randn((n, case["q_heads"], dim), generator=g, device="cuda").to(dtype)
        shape = (n, slots, heads, dim)  # the pinned positions, then the ring's in order
    else:
        n, rows, past = case["segs"], case["q_rows"], case["past"]
        q_lens = _lengths(g, n, rows)
        s["q_start"], s["k_start"] = _starts(q_lens), _starts(q_lens + past)
        s["q"] = torch.randn((int(s["q_start"][-1]), case["q_heads"], dim), generator=g, device="cuda").to(dtype)
        shape = (int(s["k_start"][-1]), heads, dim)
    s["k"], s["v"] = _keys(g, shape, dtype), _values(g, shape, dtype)
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if case["op"] == "window" or (case["op"] == "write" and not own):
        return s
    # what a serving program holds between calls is a cache: the framework's handle, filled by its own
    # writes, or the plain form's tensors of codes, scales and centers
    if not own:
        s["cache"] = [_quantise(s[x], case["bits"]) for x in "kv"]
    else:
        from mignon_ai_b200 import kv
        sessions = case["sessions"] if case["op"] == "attend" else case["segs"]
        s["cache"] = kv.KvCache(sessions, case["heads"], case["dim"], case["slots"], bits=case["bits"],
                                sinks=case["sinks"])
        if case["op"] == "read":
            s["cache"].write(s["k"], s["v"], s["pos0"], s["start"])
        elif case["op"] == "attend":
            for lo, hi, pos0 in ((0, case["sinks"], torch.zeros_like(s["base"])),
                                 (case["sinks"], case["slots"], s["base"])):
                start = torch.arange(sessions + 1, device="cuda", dtype=torch.int32) * (hi - lo)
                s["cache"].write(*(s[x][:, lo:hi].reshape(-1, case["heads"], case["dim"]) for x in "kv"), pos0, start)
    if case["op"] != "write":  # the rows are the cache's from here on
        del s["k"], s["v"]
    return s


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _own_write(s):
    s["cache"].write(s["k"], s["v"], s["pos0"], s["start"])
    return s["cache"].read(s["pos0"], s["lens"], s["start"], n_rows=s["n_rows"], dtype=s["k"].dtype)


def _own_read(s):
    return s["cache"].read(s["pos0"], s["lens"], s["start"], n_rows=s["n_rows"], dtype=_DTYPES[s["case"]["dtype"]])


def _own_attend(s):
    return s["cache"].attend(s["q"], s["lens"], window=s["case"]["window"])


def _own_window(s):
    from mignon_ai_b200 import kv
    c = s["case"]
    return kv.window_attention(s["q"], s["k"], s["v"], s["q_start"], s["k_start"], window=c["window"], sinks=c["sinks"])


_own = {"write": _own_write, "read": _own_read, "attend": _own_attend, "window": _own_window}


def _quantise(x, bits):
    """(m int8, scale, center) of rows [..., dim], scale and center float32 [..., 1]."""
    x = x.float()
    hi, lo = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    center = (0.5 * hi + 0.5 * lo).bfloat16().float()
    half = torch.maximum(hi - center, center - lo)
    step = half * torch.tensor(1 / 15 if bits == 4 else 1 / 127, dtype=torch.float32, device=x.device)
    scale = ((step.view(torch.int32) + 0xFFFF) & -65536).view(torch.float32)
    scale = torch.where(half < 2.0 ** -100, torch.zeros_like(scale), scale)
    inv = torch.where(scale > 0, torch.ones_like(scale) / scale, torch.zeros_like(scale))
    t = (x - center) * inv
    m = 2 * torch.floor(0.5 * t).clamp(-8, 7) + 1 if bits == 4 else torch.round(t).clamp(-127, 127)
    return m.to(torch.int8), scale, center


def _value(code):
    m, scale, center = code
    return center + scale * m.float()


def _held(s):
    """Which rows are still in the cache after the whole segment was written: first positions that are
    pinned, and those that the ring has not overwritten since."""
    c = s["case"]
    at = torch.arange(s["n_rows"], device="cuda", dtype=torch.int32)
    seg = torch.searchsorted(s["start"], at, right=True) - 1
    pos = s["pos0"][seg] + at - s["start"][seg]
    return ((pos < c["sinks"]) | (pos >= s["lens"][seg] - (c["slots"] - c["sinks"])))[:, None, None]


def _plain_rows(s, codes):
    held, dtype = _held(s), _DTYPES[s["case"]["dtype"]]
    k, v = codes
    return torch.where(held, _value(k), 0.0).to(dtype), torch.where(held, _value(v), 0.0).to(dtype)


def _plain_write(s):
    return _plain_rows(s, (_quantise(s["k"], s["case"]["bits"]), _quantise(s["v"], s["case"]["bits"])))


def _plain_read(s):
    return _plain_rows(s, s["cache"])


def _softmax(x, seen):
    """Weights over the last axis of the places that `seen` shows; zero where it shows none."""
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _cached_positions(s):
    """[sessions, slots] positions of the cached rows, and which of them the query sees."""
    c = s["case"]
    i = torch.arange(c["slots"], device="cuda")[None]
    pos = torch.where(i < c["sinks"], i, s["base"][:, None] + i - c["sinks"])
    lens = s["lens"][:, None]
    seen = pos < lens
    if c["window"]:
        seen &= (pos < c["sinks"]) | (pos >= lens - c["window"])
    return pos, seen


def _plain_attend(s):
    c = s["case"]
    (k, v), q = s["cache"], s["q"].float()
    n, heads, dim = c["sessions"], c["heads"], c["dim"]
    q = q.view(n, heads, -1, dim) * (1 / math.sqrt(dim))
    seen = _cached_positions(s)[1][:, None, None]
    w = _softmax(q @ _value(k).permute(0, 2, 3, 1), seen)  # [n, heads, group, slots]
    return (w @ _value(v).transpose(1, 2)).reshape(n, c["q_heads"], dim).to(s["q"].dtype)


def _padded(x, start, most):
    """Rows [n, most, heads, dim] of ragged segments (the last row repeated past each end), in 32 bits."""
    at = torch.minimum(start[:-1, None] + torch.arange(most, device="cuda"), start[-1] - 1)
    return x[at].float()


def _plain_window(s):
    c = s["case"]
    n, most, heads, dim, past = c["segs"], c["q_rows"], c["heads"], c["dim"], c["past"]
    q = _padded(s["q"], s["q_start"], most).view(n, most, heads, -1, dim).permute(0, 2, 3, 1, 4)
    k, v = (_padded(s[x], s["k_start"], most + past).transpose(1, 2)[:, :, None] for x in "kv")
    i = torch.arange(most, device="cuda")[:, None] + past  # positions of the queries
    j = torch.arange(most + past, device="cuda")[None]
    seen = j <= i
    if c["window"]:
        seen &= (j < c["sinks"]) | (j > i - c["window"])
    w = _softmax(q * (1 / math.sqrt(dim)) @ k.transpose(-1, -2), seen)
    o = (w @ v).permute(0, 3, 1, 2, 4).reshape(n, most, c["q_heads"], dim)
    real = torch.arange(most, device="cuda") < (s["q_start"][1:] - s["q_start"][:-1])[:, None]
    return o[real].to(s["q"].dtype)


_plain = {"write": _plain_write, "read": _plain_read, "attend": _plain_attend, "window": _plain_window}


# ------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ------------------------------------------------------------------------------------------------
def _mean_length(most):
    return (most + max(1, most // 4)) / 2


def _seen(rows, past, window, sinks):
    """Pairs of a query and a key it sees, in a segment of `rows` queries after `past` positions."""
    total = rows * past + rows * (rows + 1) / 2
    if window:
        hidden = max(0, rows + past - window - sinks)  # keys hidden from the last query
        first = max(0, past + 1 - window - sinks)      # and from the first
        total -= (hidden * (hidden + 1) - first * max(0, first - 1)) / 2 if hidden else 0
    return total


def work(case):
    heads, dim, size = case["heads"], case["dim"], _BYTES[case["dtype"]]
    if case["op"] in ("write", "read"):
        rows = case["rows"] + (case["segs"] - 1) * _mean_length(case["rows"])
        values = 2 * rows * heads * dim
        code = values * case["bits"] / 8 + 2 * rows * heads * 4  # codes, and a scale and center of 16 bits each
        if case["op"] == "read":
            return {"bytes": code + values * size, "flops": 2 * values}
        return {"bytes": 2 * code + 2 * values * size, "flops": 8 * values}
    if case["op"] == "attend":
        longest = case["slots"]
        held = case["sessions"] * longest if case["wraps"] else longest + (case["sessions"] - 1) * _mean_length(longest)
        if case["window"]:
            held = min(held, case["sessions"] * (case["window"] + case["sinks"]))
        code = 2 * held * heads * (dim * case["bits"] / 8 + 4)
        io = 2 * case["sessions"] * case["q_heads"] * dim * size
        return {"bytes": code + io, "flops": 4 * held * case["q_heads"] * dim}
    rows, past = case["q_rows"], case["past"]
    total = rows + (case["segs"] - 1) * _mean_length(rows)
    pairs = _seen(rows, past, case["window"], case["sinks"])
    pairs += (case["segs"] - 1) * _seen(_mean_length(rows), past, case["window"], case["sinks"])
    io = (2 * total * case["q_heads"] + 2 * (total + case["segs"] * past) * heads) * dim * size
    return {"bytes": io, "flops": 4 * pairs * case["q_heads"] * dim}


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _r32(x):
    return x.to(torch.float32).to(torch.float64)


def _exact_rows(x, bits):
    """What rows read back as: the quantiser's steps, each computed in 64 bits and rounded where its
    definition rounds."""
    x = x.double()
    hi, lo = x.max(-1, keepdim=True).values, x.min(-1, keepdim=True).values
    center = _r32(_r32(0.5 * hi) + _r32(0.5 * lo)).to(torch.float32).to(torch.bfloat16).double()
    half = torch.maximum(_r32(hi - center), _r32(center - lo))
    levels = 15 if bits == 4 else 127
    step = _r32(half * _r32(torch.tensor(1.0 / levels, dtype=torch.float64, device=x.device)))
    # bfloat16's spacing at `step`: eight bits from the leading one on
    gap = torch.exp2(torch.floor(torch.log2(torch.clamp(step, min=1e-300))) - 7)
    scale = torch.where(half < 2.0 ** -100, 0.0, torch.ceil(step / gap) * gap)
    t = torch.where(scale > 0, _r32(_r32(x - center) * _r32(1.0 / torch.clamp(scale, min=1e-300))), 0.0)
    if bits == 4:
        m = 2.0 * torch.clamp(torch.floor(t / 2), -8, 7) + 1
    else:
        m = torch.clamp(torch.round(t), -127, 127)
    return center + scale * m


def _exact_attention(q, k, v, seen):
    """softmax(q k / sqrt(dim)) v over the places of `seen`, [rows, dim] each."""
    w = torch.exp(torch.nn.functional.log_softmax((q @ k.T / math.sqrt(q.shape[-1])).masked_fill(~seen, -math.inf), -1))
    return torch.where(seen.any(-1, keepdim=True), torch.nan_to_num(w) @ v, 0.0)


def exact(case, seed):
    s = _inputs(case, seed)
    heads, dim, bits = case["heads"], case["dim"], case.get("bits")
    group = case.get("q_heads", heads) // heads
    if case["op"] in ("write", "read"):
        out = []
        start, pos0 = s["start"].long(), s["pos0"].long()
        counts = start[1:] - start[:-1]
        seg = torch.repeat_interleave(torch.arange(case["segs"], device="cuda"), counts)
        pos = pos0[seg] + torch.arange(len(seg), device="cuda") - start[seg]
        gone = (pos >= case["sinks"]) & (pos + case["slots"] - case["sinks"] < (pos0 + counts)[seg])
        for x in (s["k"], s["v"]):
            y = torch.cat([_exact_rows(part, bits) for part in x.split(16384)])
            y[gone] = 0
            out.append(y)
        return tuple(out)
    if case["op"] == "attend":
        out = torch.zeros((case["sessions"], case["q_heads"], dim), dtype=torch.float64, device="cuda")
        if case["sessions"] * heads > 20000:
            return None
        for b in range(case["sessions"]):
            n, base = int(s["lens"][b]), int(s["base"][b])
            pos = torch.cat([torch.arange(case["sinks"], device="cuda"),
                             base + torch.arange(case["slots"] - case["sinks"], device="cuda")])
            seen = pos < n
            if case["window"]:
                seen &= (pos < case["sinks"]) | (pos > n - 1 - case["window"])
            k, v = _exact_rows(s["k"][b], bits), _exact_rows(s["v"][b], bits)
            for h in range(heads):
                rows = slice(h * group, (h + 1) * group)
                out[b, rows] = _exact_attention(s["q"][b, rows].double(), k[:, h], v[:, h], seen[None].expand(group, -1))
        return out
    if case["segs"] * case["q_heads"] > 20000:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    q_start, k_start = s["q_start"].tolist(), s["k_start"].tolist()
    for b in range(case["segs"]):
        q, k, v = (s[x][a[b]:a[b + 1]].double() for x, a in (("q", q_start), ("k", k_start), ("v", k_start)))
        i = torch.arange(len(q), device="cuda")[:, None] + len(k) - len(q)
        j = torch.arange(len(k), device="cuda")[None]
        seen = (j <= i) & ((j < case["sinks"]) | (i - j < case["window"]) if case["window"] else True)
        for h in range(case["q_heads"]):
            out[q_start[b]:q_start[b + 1], h] = _exact_attention(q[:, h], k[:, h // group], v[:, h // group], seen)
    return out
