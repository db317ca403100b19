"""The quantised key/value cache and window attention against plain 64-bit restatements.

Tolerances, as fractions of the largest visible |value| of the head:
  float32   2e-5: float32 sums of up to 128 products, scores up to about 30 in size, whose error of
            a few 1e-7 each the exponential turns into the same relative error of a weight;
  float16   2^-10, bfloat16 2^-7: half a unit in the last place (2^-11 and 2^-8 of the output at
            most), as much again for weights rounded to the type, and a factor of two.
What is read back is compared exactly, after the rounding to its type.
"""
import math

import pytest
import torch

import kv_ref as ref

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOL = {"f32": 2e-5, "f16": 2.0 ** -10, "bf16": 2.0 ** -7}
DEV = torch.device("cuda:0")


@pytest.fixture(scope="module")
def kv():
    from mignon_ai_b200 import kv as module
    return module


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def rows(g, n, heads, dim, dtype, size=1.0):
    """Rows with a large offset on some dimensions and sizes that differ from row to row."""
    x = torch.randn((n, heads, dim), generator=g) * torch.exp(torch.randn((n, heads, 1), generator=g))
    x[..., :: max(1, dim // 3)] += 4
    return (x * size).to(DTYPES[dtype])


def starts(lens):
    return [sum(lens[:i]) for i in range(len(lens) + 1)]


def close(got, want, vmax, dtype, what=""):
    err = (got.double().cpu() - want).abs().max().item() if want.numel() else 0.0
    assert torch.isfinite(got).all(), what
    assert err <= TOL[dtype] * vmax, f"{what}: {err:.3g} > {TOL[dtype] * vmax:.3g}"


# ------------------------------------------------------------------------------------------------
# Write and read
# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
def test_reads_back_the_quantised_rows(kv, dtype, bits, dim):
    g = gen(dim + bits)
    lens, heads = [1, 37, 0, 5, 64, 3], 3
    pos0 = [2, 0, 5, 63, 1, 0]
    n = sum(lens)
    k, v = rows(g, n, heads, dim, dtype), rows(g, n, heads, dim, dtype)
    cache = kv.KvCache(6, heads, dim, 70, bits=bits)
    start = ints(starts(lens))
    cache.write(k.to(DEV), v.to(DEV), ints(pos0), start)
    rk, rv = cache.read(ints(pos0), ints([p + l for p, l in zip(pos0, lens)]), start, n_rows=n, dtype=DTYPES[dtype])
    for x, y in ((k, rk), (v, rv)):
        # center + scale * m is rounded once to float32, then to the type
        assert torch.equal(ref.value(x, bits).float().to(DTYPES[dtype]), y.cpu())
    cache.check()
    cache.close()


@pytest.mark.parametrize("bits", [4, 8])
def test_values_are_within_the_stated_distance(kv, bits):
    g = gen(1)
    k = rows(g, 300, 2, 64, "f32")
    cache = kv.KvCache(300, 2, 64, 1, bits=bits)
    cache.write(k.to(DEV), k.to(DEV), ints([0] * 300))
    rk, _ = cache.read(ints([0] * 300), ints([1] * 300))
    scale = ref.quantise(k, bits)[1]
    err = (rk.cpu().double() - k.double()).abs()
    assert (err <= scale * (1 if bits == 4 else 0.5) * (1 + 1e-5) + k.abs().double() * 2.0 ** -22).all()


@pytest.mark.parametrize("sinks", [0, 1, 4, 7])
@pytest.mark.parametrize("slots", [8, 9, 33])
def test_the_ring_keeps_the_last_positions_and_the_sinks(kv, slots, sinks):
    g = gen(slots)
    heads, dim, total = 2, 32, 71
    k, v = rows(g, total, heads, dim, "f32"), rows(g, total, heads, dim, "f32")
    cache = kv.KvCache(3, heads, dim, slots, bits=8, sinks=sinks)
    done = 0
    for step in (1, 5, 1, 1, 40, 2, 21):  # pieces longer and shorter than the ring
        cache.write(k[done:done + step].to(DEV), v[done:done + step].to(DEV), ints([done]), ints([0, step]), ints([1]))
        done += step
        rk, rv = cache.read(ints([0]), ints([done]), ints([0, total]), n_rows=total, sessions=ints([1]))
        want = torch.tensor([ref.held(p, done, slots, sinks) for p in range(total)])[:, None, None]
        assert torch.equal(torch.where(want, ref.value(k, 8).float(), 0.0), rk.cpu())
        assert torch.equal(torch.where(want, ref.value(v, 8).float(), 0.0), rv.cpu())
    # the other sessions are untouched
    rk, _ = cache.read(ints([0, 0]), ints([0, 0]), ints([0, 5, 10]), n_rows=10, sessions=ints([0, 2]))
    assert not rk.any()
    cache.check()


def test_special_rows(kv):
    """Constant rows, zeros, tiny, huge and non-finite ones."""
    k = torch.ones((9, 1, 32))
    k[0] = 0
    k[1] = 3.3333333
    k[2] *= 1e-38 * torch.arange(32)
    k[3] = torch.linspace(-3e38, 3e38, 32)
    k[4, 0, 3] = float("inf")
    k[5, 0, 31] = float("nan")
    k[6, 0, 0] = -float("inf")
    k[7] = 3.4e38  # past bfloat16's largest value
    k[8] = -2.0 ** -99 * torch.arange(32)
    for bits in (4, 8):
        cache = kv.KvCache(9, 1, 32, 4, bits=bits)
        cache.write(k.to(DEV), k.to(DEV), ints([0] * 9))
        rk, rv = cache.read(ints([0] * 9), ints([1] * 9))
        want = ref.value(k, bits).float()
        assert torch.equal(rk.cpu().nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))
        assert torch.equal(rk.cpu().isnan(), want.isnan())
        assert torch.equal(rk.isnan(), rv.isnan())
        # row 3's step overflows in linspace, so that row holds infinities too
        assert rk[[3, 4, 5, 6, 7]].isnan().all() and not rk[[0, 1, 2, 8]].isnan().any()
        assert not rk[0].any()


def test_strided_rows(kv):
    """Keys and values as slices of one projection, with a stride that is not a multiple of 16 bytes."""
    g = gen(5)
    heads, dim, n = 2, 48, 21
    for width in (2 * heads * dim, 2 * heads * dim + 1):
        both = torch.randn((n, width), generator=g).to(DEV)
        k = both[:, -2 * heads * dim:-heads * dim].unflatten(1, (heads, dim))
        v = both[:, -heads * dim:].unflatten(1, (heads, dim))
        cache = kv.KvCache(1, heads, dim, n)
        cache.write(k, v, ints([0]), ints([0, n]))
        out = torch.full((n, 2, heads, dim + 3), 9.0, device=DEV)
        cache.read(ints([0]), ints([n]), ints([0, n]), out=(out[:, 0, :, :dim], out[:, 1, :, :dim]))
        assert torch.equal(out[:, 0, :, :dim].cpu(), ref.value(k.cpu(), 4).float())
        assert torch.equal(out[:, 1, :, :dim].cpu(), ref.value(v.cpu(), 4).float())
        assert (out[..., dim:] == 9).all()


def test_rows_outside_the_segments_and_bad_indexes(kv):
    heads, dim = 1, 16
    x = torch.randn((6, heads, dim), device=DEV)
    cache = kv.KvCache(2, heads, dim, 8, bits=8)
    # rows 0 and 5 belong to no segment; segment 1 names a session that does not exist
    cache.write(x, x, ints([0, 0]), ints([1, 3, 5]), ints([1, 2]))
    with pytest.raises(Exception, match="out of range"):
        cache.check()
    cache.check()  # cleared
    rk, _ = cache.read(ints([0, -1]), ints([2, 2]), ints([1, 3, 5]), n_rows=6, sessions=ints([1, 1]))
    with pytest.raises(Exception, match="out of range"):
        cache.check()
    want = torch.zeros((6, heads, dim))
    want[1:3] = ref.value(x[1:3].cpu(), 8).float()
    assert torch.equal(rk.cpu(), want)
    out = cache.attend(x[:3], ints([2, 2, 2]), sessions=ints([1, 5, -1]))
    assert not out[1:].any() and out[0].any()
    with pytest.raises(Exception, match="out of range"):
        cache.check()


# ------------------------------------------------------------------------------------------------
# Attention over the cache
# ------------------------------------------------------------------------------------------------
def attend_case(kv, dtype, bits, dim, heads, group, slots, sinks, window, lens, sessions=None, seed=0, q_size=1.0):
    g = gen(seed)
    n = len(lens)
    n_sess = n if sessions is None else max(sessions) + 1
    order = list(range(n)) if sessions is None else sessions
    cache = kv.KvCache(n_sess, heads, dim, slots, bits=bits, sinks=sinks)
    q = (torch.randn((n, heads * group, dim), generator=g) * q_size).to(DTYPES[dtype])
    ks = [rows(g, l, heads, dim, dtype) for l in lens]
    vs = [rows(g, l, heads, dim, dtype) for l in lens]
    for b in range(n):
        if lens[b]:
            cache.write(ks[b].to(DEV), vs[b].to(DEV), ints([0]), ints([0, lens[b]]), ints([order[b]]))
    got = cache.attend(q.to(DEV), ints(lens), sessions=None if sessions is None else ints(sessions), window=window)
    cache.check()
    for b in range(n):
        l = lens[b]
        seen = torch.tensor([ref.held(p, l, slots, sinks) and (not window or p < sinks or p > l - 1 - window)
                             for p in range(l)], dtype=torch.bool)
        for h in range(heads):
            k, v = ref.value(ks[b][:, h], bits), ref.value(vs[b][:, h], bits)
            want = ref.attention(q[b, h * group:(h + 1) * group], k, v, seen[None].expand(group, -1))
            close(got[b, h * group:(h + 1) * group], want, v[seen].abs().max().item() if seen.any() else 1.0, dtype, (b, h))
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [16, 32, 48, 64, 80, 96, 112, 128])
def test_attend_types_and_widths(kv, dtype, bits, dim):
    attend_case(kv, dtype, bits, dim, 2, 1, 200, 0, 0, [1, 200, 63, 64, 65, 0, 31, 33, 129], seed=dim)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 9, 16, 17])
@pytest.mark.parametrize("dtype,bits", [("f32", 4), ("bf16", 8)])
def test_attend_groups(kv, group, dtype, bits):
    attend_case(kv, dtype, bits, 64, 2, group, 150, 0, 0, [150, 1, 77], seed=group)


@pytest.mark.parametrize("slots,sinks,window,lens", [
    (8, 0, 0, [1, 7, 8, 9, 100]), (64, 4, 0, [3, 4, 5, 63, 64, 65, 66, 300]), (65, 64, 1, [64, 65, 66, 200]),
    (200, 0, 1, [1, 2, 200, 450]), (200, 3, 64, [1, 64, 67, 68, 200, 201, 399]), (300, 70, 100, [300, 301, 170, 1000]),
    (1, 0, 0, [1, 2, 3]), (130, 1, 500, [129, 130, 131, 4000])])
@pytest.mark.parametrize("bits", [4, 8])
def test_attend_rings_sinks_and_windows(kv, slots, sinks, window, lens, bits):
    attend_case(kv, "f32", bits, 32, 1, 2, slots, sinks, window, lens, seed=slots)


def test_attend_long_sessions(kv):
    """One and three long sessions: the positions of an item are split and joined."""
    for n, dtype in ((1, "f32"), (3, "bf16")):
        attend_case(kv, dtype, 4, 64, 1, 4, 9000, 4, 0, [9000, 8191, 5][:n], seed=n)
        attend_case(kv, dtype, 8, 128, 1, 1, 9000, 4, 5000, [8999, 20000, 4500][:n], seed=n)


def test_attend_sessions_in_any_order(kv):
    attend_case(kv, "bf16", 4, 64, 2, 2, 100, 0, 0, [50, 100, 7], sessions=[4, 0, 2])


def test_attend_sharp_scores(kv):
    """Large queries: one position takes almost all the weight, the running maximum changes often."""
    attend_case(kv, "f32", 8, 64, 1, 3, 500, 0, 0, [500, 321], q_size=4.0, seed=3)


def test_attend_ignores_what_is_hidden(kv):
    """Non-finite rows outside the window, and past the length, reach no output."""
    heads, dim, n = 1, 64, 200
    g = gen(9)
    k, v = rows(g, n, heads, dim, "f32"), rows(g, n, heads, dim, "f32")
    clean = kv.KvCache(1, heads, dim, n, bits=4)
    clean.write(k.to(DEV), v.to(DEV), ints([0]), ints([0, n]))
    dirty = kv.KvCache(1, heads, dim, n, bits=4)
    k[:90] = float("nan")
    v[:90] = float("inf")
    v[150:] = float("nan")
    k[150:] = -float("inf")
    dirty.write(k.to(DEV), v.to(DEV), ints([0]), ints([0, n]))
    q = torch.randn((1, 3, dim), generator=g).to(DEV)
    a, b = (c.attend(q, ints([150]), window=60) for c in (clean, dirty))
    assert torch.isfinite(b).all() and torch.equal(a, b)
    assert dirty.attend(q, ints([200]), window=60).isnan().all()  # what is visible is not ignored


def test_attend_strides_and_streams(kv):
    g = gen(11)
    heads, dim, n = 2, 32, 40
    cache = kv.KvCache(n, heads, dim, 16, bits=8)
    x = torch.randn((n, 3 * 4 * dim + 1), generator=g).to(DEV)
    q = x[:, 1:1 + 4 * dim].unflatten(1, (4, dim))
    k, v = torch.randn((n, heads, dim), device=DEV), torch.randn((n, heads, dim), device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.write(k, v, ints([0] * n))
        out = torch.empty((n, 5, dim + 1), device=DEV)[:, :4, :dim]
        cache.attend(q, ints([1] * n), out=out)
    torch.cuda.current_stream().wait_stream(side)
    want = ref.value(v.cpu(), 8).repeat_interleave(2, 1)  # one visible position: its value
    close(out, want, want.abs().max().item(), "f32")


# ------------------------------------------------------------------------------------------------
# Window attention
# ------------------------------------------------------------------------------------------------
def window_case(kv, dtype, dim, heads, group, q_lens, past, window, sinks, seed=0, q=None, k=None, v=None, size=1.0):
    g = gen(seed)
    k_lens = [max(0, l + p) for l, p in zip(q_lens, past)]
    nq, nk = sum(q_lens), sum(k_lens)
    q = (torch.randn((nq, heads * group, dim), generator=g) * size).to(DTYPES[dtype]) if q is None else q
    k = rows(g, nk, heads, dim, dtype) if k is None else k
    v = rows(g, nk, heads, dim, dtype) if v is None else v
    qs, ks = starts(q_lens), starts(k_lens)
    got = kv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), ints(qs), ints(ks), window=window, sinks=sinks)
    for b in range(len(q_lens)):
        kb, vb = k[ks[b]:ks[b + 1]], v[ks[b]:ks[b + 1]]
        i = torch.arange(q_lens[b])[:, None] + k_lens[b] - q_lens[b]
        j = torch.arange(k_lens[b])[None]
        seen = (j <= i) & (torch.ones_like(j, dtype=torch.bool) if not window else (j < sinks) | (j > i - window))
        for h in range(heads * group):
            vh = vb[:, h // group]
            want = ref.attention(q[qs[b]:qs[b + 1], h], kb[:, h // group], vh, seen)
            fine = vh[torch.isfinite(vh)].double()
            close(got[qs[b]:qs[b + 1], h], want, fine.abs().max().item() if fine.numel() else 1.0, dtype, (b, h))
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [1, 7, 16, 32, 48, 64, 80, 96, 100, 128, 192, 256])
def test_window_types_and_widths(kv, dtype, dim):
    window_case(kv, dtype, dim, 2, 1, [1, 130, 0, 17, 64], [0] * 5, 0, 0, seed=dim)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 11])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_window_groups(kv, group, dtype):
    window_case(kv, dtype, 64, 2, group, [33, 1, 150], [0, 5, 40], 0, 0, seed=group)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (5, 1), (64, 0), (64, 4), (100, 33), (128, 128), (129, 200), (1000, 3)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_window_masks(kv, window, sinks, dtype):
    window_case(kv, dtype, 32, 1, 2, [300, 64, 1, 129], [0, 100, 400, 257], window, sinks, seed=window)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_window_queries_without_keys(kv, dtype):
    """More queries than keys: the first ones lie before every key and see nothing."""
    got = window_case(kv, dtype, 64, 1, 2, [40, 3, 5], [-10, -3, -9], 16, 0)
    assert not got[:10].any() and not got[40:].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_window_ignores_what_is_hidden(kv, dtype):
    """Infinities, NaN and the type's lowest value in keys and values that a row does not see."""
    g = gen(2)
    n, dim = 200, 64
    k, v = rows(g, 3 * n, 1, dim, dtype), rows(g, 3 * n, 1, dim, dtype)
    low = torch.finfo(DTYPES[dtype]).min
    for x, bad in ((k, low), (v, float("nan"))):
        x[:n] = bad          # the segment before
        x[2 * n - 1:] = bad  # the last key of the middle segment, and the segment after
    v[n + 5], k[n + 5] = float("inf"), float("nan")  # behind the window of every query but the first
    q = torch.randn((3 * n, 2, dim), generator=g).to(DTYPES[dtype])
    s = ints([0, n, 2 * n, 3 * n])
    got = kv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), s, s, window=30, sinks=2)
    middle = slice(n + 36, 2 * n - 1)  # rows that see neither
    i = torch.arange(n)[:, None]
    j = torch.arange(n)[None]
    seen = (j <= i) & ((j < 2) | (j > i - 30))
    for h in range(2):
        want = ref.attention(q[n:2 * n, h], k[n:2 * n, 0], v[n:2 * n, 0], seen)[36:n - 1]
        close(got[middle, h], want, 100.0 if dtype == "f32" else 50.0, dtype)
    assert got[2 * n - 1].isnan().all()


def test_window_strides_and_one_segment(kv):
    """Slices of one projection (16-byte aligned and not), no starts given, outputs in place of queries."""
    g = gen(4)
    n, heads, group, dim = 70, 2, 2, 64
    for dtype in ("f32", "bf16"):
        for odd in (0, 1):
            x = torch.randn((n, (heads * group + 2 * heads) * dim + odd), generator=g).to(DTYPES[dtype])
            q = x[:, odd:odd + heads * group * dim].unflatten(1, (heads * group, dim))
            k = x[:, odd + heads * group * dim:odd + (heads * group + heads) * dim].unflatten(1, (heads, dim))
            v = x[:, odd + (heads * group + heads) * dim:].unflatten(1, (heads, dim))
            xd = x.to(DEV)
            qd = xd[:, odd:odd + heads * group * dim].unflatten(1, (heads * group, dim))
            kd = xd[:, odd + heads * group * dim:odd + (heads * group + heads) * dim].unflatten(1, (heads, dim))
            vd = xd[:, odd + (heads * group + heads) * dim:].unflatten(1, (heads, dim))
            got = kv.window_attention(qd, kd, vd, window=20, scale=0.3)
            i, j = torch.arange(n)[:, None], torch.arange(n)[None]
            seen = (j <= i) & (j > i - 20)
            for h in range(heads * group):
                want = ref.attention(q[:, h], k[:, h // group], v[:, h // group], seen, scale=0.3)
                close(got[:, h], want, v.float().abs().max().item(), dtype)


def test_window_long_segment(kv):
    """Rows of a long segment, checked where they can go wrong: ends of tiles, first and last rows."""
    g = gen(6)
    n, dim = 3000, 128
    for dtype in ("bf16", "f32"):
        q = torch.randn((n, 4, dim), generator=g).to(DTYPES[dtype])
        k, v = rows(g, n, 2, dim, dtype), rows(g, n, 2, dim, dtype)
        for window, sinks in ((0, 0), (700, 4)):
            got = kv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), window=window, sinks=sinks)
            for i in (0, 1, 63, 127, 128, 129, 700, 704, 705, 1500, 2047, 2048, 2999):
                j = torch.arange(n)
                seen = (j <= i) & ((j < sinks) | (j > i - window) if window else torch.ones(n, dtype=torch.bool))
                for h in range(4):
                    want = ref.attention(q[i:i + 1, h], k[:, h // 2], v[:, h // 2], seen[None])
                    close(got[i:i + 1, h], want, v.float().abs().max().item(), dtype, (i, h))


def test_window_segments_out_of_range_are_skipped(kv):
    q = torch.randn((20, 1, 64), device=DEV).bfloat16()
    k = torch.randn((20, 1, 64), device=DEV).bfloat16()
    out = torch.full_like(q, 5.0)
    kv.window_attention(q, k, k, ints([0, 10, 20]), ints([0, 10, 21]), out=out)
    assert (out[10:] == 5).all() and (out[:10] != 5).any()


# ------------------------------------------------------------------------------------------------
# Together
# ------------------------------------------------------------------------------------------------
def test_a_second_prompt_after_reading_back(kv):
    """Prompt, cache, decode token, read back, second prompt: the rows equal those of one pass over
    the same (quantised) keys and values."""
    g = gen(8)
    heads, dim, n1, n2 = 2, 64, 90, 31
    k, v = rows(g, n1 + n2, heads, dim, "bf16").to(DEV), rows(g, n1 + n2, heads, dim, "bf16").to(DEV)
    q = torch.randn((n2, 4, dim), generator=g).bfloat16().to(DEV)
    cache = kv.KvCache(1, heads, dim, 256, bits=8)
    cache.write(k[:n1], v[:n1], ints([0]), ints([0, n1]))
    pk, pv = cache.read(ints([0]), ints([n1]), ints([0, n1]), n_rows=n1, dtype=torch.bfloat16)
    got = kv.window_attention(q, torch.cat([pk, k[n1:]]), torch.cat([pv, v[n1:]]), ints([0, n2]), ints([0, n1 + n2]), window=50)
    hat = lambda x: torch.cat([ref.value(x[:n1].cpu(), 8).float().bfloat16(), x[n1:].cpu()])
    i, j = torch.arange(n2)[:, None] + n1, torch.arange(n1 + n2)[None]
    for h in range(4):
        want = ref.attention(q[:, h].cpu(), hat(k)[:, h // 2], hat(v)[:, h // 2], (j <= i) & (j > i - 50))
        close(got[:, h], want, v.float().abs().max().item(), "bf16")


def test_calls_can_be_captured(kv):
    """A decode step (write, attend) as a CUDA graph, replayed with new contents."""
    heads, dim, n = 2, 64, 5
    cache = kv.KvCache(n, heads, dim, 32, bits=4)
    q, k, v = (torch.randn((n, h, dim), device=DEV) for h in (4, heads, heads))
    pos, lens = ints([0] * n), ints([1] * n)
    cache.write(k, v, pos)
    out = cache.attend(q, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(k, v, pos)
        cache.attend(q, lens, out=out)
        pos += 1
        lens += 1
    ks, vs = [], []
    for _ in range(40):
        k.copy_(torch.randn_like(k))
        v.copy_(torch.randn_like(v))
        ks.append(k.cpu().clone())
        vs.append(v.cpu().clone())
        graph.replay()
    for b in range(n):
        for h in range(4):
            kk = torch.stack([ref.value(x[b, h // 2], 4) for x in ks[-32:]])
            vv = torch.stack([ref.value(x[b, h // 2], 4) for x in vs[-32:]])
            want = ref.attention(q[b, h:h + 1].cpu(), kk, vv, torch.ones((1, 32), dtype=torch.bool))
            close(out[b, h:h + 1], want, vv.abs().max().item(), "f32")
    del graph


def test_the_same_inputs_give_the_same_bits(kv):
    g = gen(12)
    cache = kv.KvCache(2, 2, 64, 6000, bits=4)
    k, v = rows(g, 12000, 2, 64, "bf16").to(DEV), rows(g, 12000, 2, 64, "bf16").to(DEV)
    cache.write(k, v, ints([0, 0]), ints([0, 6000, 12000]))
    q = torch.randn((2, 8, 64), generator=g).to(DEV)
    first = cache.attend(q, ints([6000, 5000]))
    for _ in range(5):
        assert torch.equal(first, cache.attend(q, ints([6000, 5000])))
    first = kv.window_attention(k, k, v, ints([0, 6000, 12000]), window=100)
    assert torch.equal(first, kv.window_attention(k, k, v, ints([0, 6000, 12000]), window=100))


def test_head_major_rows(kv):
    """Rows as views of [heads, rows, dim] tensors: the head stride above the row stride."""
    g = gen(13)
    heads, group, dim, n = 2, 2, 64, 90
    for dtype in ("f32", "bf16"):
        x = [torch.randn((h, n, dim), generator=g).to(DTYPES[dtype]).to(DEV).transpose(0, 1) for h in (heads * group, heads, heads)]
        got = kv.window_attention(*x, window=33, sinks=2)
        cache = kv.KvCache(1, heads, dim, n, bits=8)
        cache.write(x[1], x[2], ints([0]), ints([0, n]))
        rk, rv = cache.read(ints([0]), ints([n]), ints([0, n]), n_rows=n)
        one = cache.attend(x[0][n - 1:], ints([n]))
        q, k, v = (y.cpu() for y in x)
        assert torch.equal(rk.cpu(), ref.value(k, 8).float()) and torch.equal(rv.cpu(), ref.value(v, 8).float())
        i, j = torch.arange(n)[:, None], torch.arange(n)[None]
        seen = (j <= i) & ((j < 2) | (j > i - 33))
        for h in range(heads * group):
            vmax = v.float().abs().max().item()
            close(got[:, h], ref.attention(q[:, h], k[:, h // group], v[:, h // group], seen), vmax, dtype)
            want = ref.attention(q[n - 1:, h], ref.value(k, 8)[:, h // group], ref.value(v, 8)[:, h // group], seen[:1] | True)
            close(one[:, h], want, vmax, dtype)


def test_places_far_into_a_large_cache(kv):
    """Places more than 2^32 bytes into the cache, and positions above 2^30."""
    g = gen(14)
    heads, dim, slots = 8, 128, 1 << 20
    cache = kv.KvCache(3, heads, dim, slots, bits=8, sinks=3)
    assert cache.memory.numel() > 1 << 32
    ring = slots - 3
    for first in (slots - 70, 3 + ring * 1025 - 40):  # up to the cache's last place; across the ring's end
        k, v = rows(g, 64, heads, dim, "bf16"), rows(g, 64, heads, dim, "bf16")
        q = torch.randn((1, heads, dim), generator=g).bfloat16()
        cache.write(k.to(DEV), v.to(DEV), ints([first]), ints([0, 64]), ints([2]))
        rk, rv = cache.read(ints([first]), ints([first + 64]), ints([0, 64]), n_rows=64, sessions=ints([2]))
        assert torch.equal(rk.cpu(), ref.value(k, 8).float()) and torch.equal(rv.cpu(), ref.value(v, 8).float())
        got = cache.attend(q.to(DEV), ints([first + 64]), sessions=ints([2]), window=64)
        cache.check()
        for h in range(heads):  # the three first positions are zeros: codes of nothing written
            kk, vv = (torch.cat([torch.zeros((3, dim), dtype=torch.float64), ref.value(y, 8)[:, h]]) for y in (k, v))
            want = ref.attention(q[:, h], kk, vv, torch.ones((1, 67), dtype=torch.bool))
            close(got[:, h], want, vv.abs().max().item(), "bf16", h)


def test_a_cache_in_the_librarys_own_memory(kv):
    """mc_kv_open without memory: the library allocates and frees it."""
    import ctypes
    from mignon_ai_b200 import _lib
    h, spec = ctypes.c_void_p(), kv._Spec(3, 2, 64, 4, 100, 4)
    _lib.check(_lib.lib().mc_kv_open(0, ctypes.byref(spec), None, None, ctypes.byref(h)))
    cache = kv.KvCache(3, 2, 64, 100, sinks=4)
    theirs, cache._h = cache._h, h  # the wrapper around the other handle
    x = torch.randn((3, 2, 64), device=DEV)
    cache.write(x, x, ints([0, 5, 99]))
    rk, _ = cache.read(ints([0, 5, 99]), ints([1, 6, 100]))
    assert torch.equal(rk.cpu(), ref.value(x.cpu(), 4).float())
    cache._h = theirs
    _lib.check(_lib.lib().mc_kv_close(h))
    cache.close()


@pytest.mark.parametrize("call", ["dtype", "shape", "device", "ints", "groups", "window", "scale", "stride"])
def test_refusals(kv, call):
    cache = kv.KvCache(2, 2, 32, 8)
    x = torch.randn((2, 2, 32), device=DEV)
    with pytest.raises((ValueError, TypeError, RuntimeError)):
        if call == "dtype":
            cache.write(x.double(), x.double(), ints([0, 0]))
        elif call == "shape":
            cache.write(x[:, :1], x[:, :1], ints([0, 0]))
        elif call == "device":
            cache.write(x.cpu(), x.cpu(), ints([0, 0]))
        elif call == "ints":
            cache.write(x, x, ints([0, 0]).long())
        elif call == "groups":
            cache.attend(torch.randn((2, 3, 32), device=DEV), ints([1, 1]))
        elif call == "window":
            cache.attend(x, ints([1, 1]), window=-1)
        elif call == "scale":
            kv.window_attention(x, x, x, scale=float("nan"))
        else:
            cache.write(x.transpose(1, 2).contiguous().transpose(1, 2), x, ints([0, 0]))


@pytest.mark.parametrize("dim", [32, 128])
def test_window_float32_does_not_drift_over_long_rows(kv, dim):
    """Rows of thousands of keys stay at float32's accuracy: within 2^-20 of the result in the 2-norm,
    sixteen of its roundings, as sums that round to nearest stay; sums cut off at every step do not."""
    g = gen(dim)
    n, last = 8192, 64
    q = torch.randn((last, 1, dim), generator=g)
    k, v = torch.randn((n, 1, dim), generator=g), torch.randn((n, 1, dim), generator=g)
    got = kv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV), ints([0, last]), ints([0, n])).cpu().double()
    i, j = torch.arange(last)[:, None] + n - last, torch.arange(n)[None]
    want = ref.attention(q[:, 0], k[:, 0], v[:, 0], j <= i)
    assert (got[:, 0] - want).norm() <= 2.0 ** -20 * want.norm()
