"""Plain restatements, in 64 bits, of the quantised cache and the attention around it."""
import math

import torch


def r32(x):
    return x.to(torch.float32).to(torch.float64)


def quantise(x, bits):
    """(m, scale, center) of rows [..., dim] in 64 bits: the quantiser's steps, each rounded to
    float32 where its definition rounds (64 bits hold every float32 step exactly enough for that).
    A row that is not all finite has scale NaN."""
    x = x.double()
    hi, lo = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    center = r32(r32(0.5 * hi) + r32(0.5 * lo)).bfloat16().double()
    half = torch.maximum(r32(hi - center), r32(center - lo))
    levels = 15 if bits == 4 else 127
    step = r32(half * r32(torch.tensor(1.0 / levels, dtype=torch.float64)))
    gap = torch.exp2(torch.floor(torch.log2(step.clamp(min=1e-300))) - 7)  # bfloat16's spacing at step
    scale = torch.where(half < 2.0 ** -100, 0.0, torch.ceil(step / gap) * gap)
    t = torch.where(scale > 0, r32(r32(x - center) * r32(1 / scale.clamp(min=1e-300))), 0.0)
    m = 2 * torch.floor(t / 2).clamp(-8, 7) + 1 if bits == 4 else torch.round(t).clamp(-127, 127)
    bad = ~(torch.isfinite(x).all(-1, keepdim=True) & torch.isfinite(scale) & torch.isfinite(center))
    scale = torch.where(bad, float("nan"), scale)
    return m, scale, torch.where(bad, 0.0, center)


def value(x, bits):
    m, scale, center = quantise(x, bits)
    return center + scale * m


def attention(q, k, v, seen, scale=None):
    """softmax(scale q k) v of rows q [n, dim] over the keys that seen [n, keys] shows; zero for a
    row that is shown none. Keys and values that are not shown are not touched."""
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    out = torch.zeros((q.shape[0], v.shape[-1]), dtype=torch.float64)
    for i in range(q.shape[0]):
        idx = torch.nonzero(seen[i])[:, 0]
        if len(idx):
            out[i] = torch.softmax(scale * (k[idx].double() @ q[i].double()), 0) @ v[idx].double()
    return out


def held(pos, length, slots, sinks):
    return 0 <= pos < length and (pos < sinks or pos >= length - (slots - sinks))
