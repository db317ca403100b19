"""A decoder's attention layers served from the quantised key/value cache.

Prompts of uneven length run through window attention and go into the cache; then every session
decodes token by token from it; then each gets a second prompt, for which its cached past is read back.
The layers are random (a residual stream of `heads * dim`, projections to queries, keys and values):
the point is how the calls follow one another. A second pass with the cache in float32 (plain torch)
says how far the quantised cache moves the result.

    python examples/quantised_cache.py --bits 4 --sessions 64
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from mignon_ai_b200 import kv  # noqa: E402


class Layer:
    """One attention layer's weights, and its keys and values of every session."""

    def __init__(self, g, q_heads, heads, dim, sessions, slots, bits, sinks, dtype):
        width = q_heads * dim
        self.q_heads, self.heads, self.dim = q_heads, heads, dim
        self.proj = (torch.randn((width, (q_heads + 2 * heads) * dim), generator=g, device="cuda") * width ** -0.5).to(dtype)
        self.out = (torch.randn((width, width), generator=g, device="cuda") * width ** -0.5).to(dtype)
        self.cache = kv.KvCache(sessions, heads, dim, slots, bits=bits, sinks=sinks)

    def split(self, x):
        """Queries, keys and values of rows x: views of one projection, as they come."""
        y = torch.nn.functional.rms_norm(x, x.shape[-1:]) @ self.proj
        y = y.unflatten(1, (self.q_heads + 2 * self.heads, self.dim))
        return y[:, :self.q_heads], y[:, self.q_heads:-self.heads], y[:, -self.heads:]

    def add(self, x, attended):
        return x + attended.flatten(1) @ self.out


def starts(lens):
    return torch.cat([lens.new_zeros(1), lens.cumsum(0, dtype=torch.int32)])


def prompt(layers, x, start, window, sinks):
    """First prompts: positions from 0 on."""
    for layer in layers:
        q, k, v = layer.split(x)
        x = layer.add(x, kv.window_attention(q, k, v, start, window=window, sinks=sinks))
        layer.cache.write(k, v, torch.zeros_like(start[1:]), start)
    return x


def decode(layers, x, lens, window):
    """One token per session, at position lens; lens + 1 positions are there afterwards."""
    for layer in layers:
        q, k, v = layer.split(x)
        layer.cache.write(k, v, lens)
        x = layer.add(x, layer.cache.attend(q, lens + 1, window=window))
    return x


def follow_up(layers, x, start, lens, window, sinks):
    """Second prompts: the cached past comes back in front of the new keys and values."""
    rows = start[1:] - start[:-1]
    both = starts(lens + rows)
    n = int(both[-1])
    new = torch.cat([torch.arange(int(a + p), int(b), device="cuda") for a, b, p in zip(both[:-1], both[1:], lens)])
    for layer in layers:
        q, k, v = layer.split(x)
        past_k, past_v = layer.cache.read(torch.zeros_like(lens), lens, both, n_rows=n, dtype=x.dtype)
        past_k[new], past_v[new] = k, v  # positions past lens came back as zeros: the new rows' places
        x = layer.add(x, kv.window_attention(q, past_k, past_v, start, both, window=window, sinks=sinks))
        layer.cache.write(k, v, lens, start)
    return x


def plain(layers, x, window, sinks):
    """One session's whole run in one pass, its keys and values kept in float32: the last row's output."""
    x = x.float()
    i, j = torch.arange(len(x), device="cuda")[:, None], torch.arange(len(x), device="cuda")[None]
    seen = (j <= i) & ((j < sinks) | (j > i - window) if window else True)
    for layer in layers:
        proj, out = layer.proj.float(), layer.out.float()
        y = (torch.nn.functional.rms_norm(x, x.shape[-1:]) @ proj).unflatten(1, (-1, layer.dim))
        q, k, v = y[:, :layer.q_heads], y[:, layer.q_heads:-layer.heads], y[:, -layer.heads:]
        k, v = (t.repeat_interleave(layer.q_heads // layer.heads, 1) for t in (k, v))
        s = torch.einsum("ihd,jhd->hij", q, k) * layer.dim ** -0.5
        w = torch.softmax(s.masked_fill(~seen, float("-inf")), -1)
        x = x + torch.einsum("hij,jhd->ihd", w, v).flatten(1) @ out
    return x


def run(sessions=64, layers=2, q_heads=8, heads=2, dim=64, bits=4, prompt_rows=96, steps=16, second=24, window=0, sinks=0,
        slots=0, dtype=torch.bfloat16, seed=0):
    """Returns the final rows of each session's second prompt, the plain float32 ones of the first four
    sessions, and the seconds that the decode steps took."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    slots = slots or prompt_rows + steps + second
    stack = [Layer(g, q_heads, heads, dim, sessions, slots, bits, sinks, dtype) for _ in range(layers)]
    width = q_heads * dim
    first = torch.randint(1, prompt_rows + 1, (sessions,), generator=g, device="cuda", dtype=torch.int32)
    start, second_start = starts(first), torch.arange(sessions + 1, device="cuda", dtype=torch.int32) * second
    rows = [torch.randn((int(n), width), generator=g, device="cuda").to(dtype) for n in (start[-1], second_start[-1])]
    tokens = torch.randn((steps, sessions, width), generator=g, device="cuda").to(dtype)

    prompt(stack, rows[0], start, window, sinks)
    lens = first.clone()
    torch.cuda.synchronize()
    began = time.perf_counter()
    for x in tokens:
        decode(stack, x, lens, window)
        lens += 1
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    got = follow_up(stack, rows[1], second_start, lens, window, sinks)
    for layer in stack:
        layer.cache.check()

    want = []
    for b in range(min(4, sessions)):
        x = torch.cat([rows[0][start[b]:start[b + 1]], tokens[:, b], rows[1][second * b:second * (b + 1)]])
        want.append(plain(stack, x, window, sinks)[-second:])
    for layer in stack:
        layer.cache.close()
    return got.view(sessions, second, width), torch.stack(want), took


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--sessions", type=int, default=64)
    ap.add_argument("--bits", type=int, choices=(4, 8), default=4)
    ap.add_argument("--window", type=int, default=0)
    ap.add_argument("--sinks", type=int, default=0)
    ap.add_argument("--steps", type=int, default=16)
    a = ap.parse_args()
    got, want, took = run(sessions=a.sessions, bits=a.bits, window=a.window, sinks=a.sinks, steps=a.steps)
    off = ((got[:len(want)].float() - want).norm() / want.norm()).item()
    print(f"{a.sessions} sessions, {a.bits} bits: {a.steps * a.sessions / took:.0f} tokens/s decoded, "
          f"second prompts {off:.3%} from a float32 cache")


if __name__ == "__main__":
    main()
