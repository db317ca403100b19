"""Corner calls of the quantised key/value cache and window attention, against plain 64-bit
restatements. Tolerances are those of the ordinary cases unless a test derives its own."""
import contextlib
import ctypes

import pytest
import torch

import kv_ref as ref
from test_gpu_kv import DEV, DTYPES, close, gen, ints, kv, rows, starts, window_case  # noqa: F401 (kv: a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim", [("f32", 64), ("f16", 64), ("bf16", 64), ("f16", 24), ("f32", 192)])
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 50])
def test_windows_near_the_largest_number(kv, dtype, dim, window):
    """A window that shows everything, with queries before the first key: their positions are negative."""
    window_case(kv, dtype, dim, 1, 2, [40, 3, 150, 70], [-10, -3, -100, 20], window, 3)


def test_calls_without_rows(kv):
    """Empty batches, whose tensors have no address: nothing to do, and nothing is done."""
    cache = kv.KvCache(2, 2, 32, 8)
    x = torch.randn((2, 2, 32), device=DEV)
    cache.write(x, x, ints([0, 0]))
    none = ints([])
    cache.write(x[:0], x[:0], none)
    cache.write(x[:0], x[:0], none, sessions=none)
    cache.write(x[:0], x[:0], none, ints([0]))
    cache.write(x[:0], x[:0], ints([0, 0]), ints([0, 0, 0]))
    for sessions in (None, none):
        assert cache.attend(x[:0], none, sessions=sessions).shape == (0, 2, 32)
        assert cache.read(none, none, sessions=sessions)[0].shape == (0, 2, 32)
    assert cache.read(none, none, ints([0]), n_rows=0)[1].shape == (0, 2, 32)
    assert cache.read(ints([0]), ints([1]), ints([0, 0]), n_rows=0)[1].shape == (0, 2, 32)
    assert kv.window_attention(x[:0], x, x, ints([0]), ints([0])).shape == (0, 2, 32)
    assert kv.window_attention(x[:0], x[:0], x[:0]).shape == (0, 2, 32)
    rk, _ = cache.read(ints([0, 0]), ints([1, 1]))
    assert torch.equal(rk.cpu(), ref.value(x.cpu(), 4).float())
    cache.check()
    # the library alone takes null arrays where there is nothing in them
    L, r = cache._lib, ctypes.byref(kv._Rows(None, 64, 32))
    assert L.mc_kv_write_dev(cache._h, r, r, 0, 0, None, None, None, 0, None) == 0
    assert L.mc_kv_read_dev(cache._h, r, r, 0, 0, None, None, None, None, 0, None) == 0
    assert L.mc_kv_attend_dev(cache._h, r, r, 0, 2, None, None, 0, 0, 1.0, None) == 0
    # and none where there is something
    assert L.mc_kv_write_dev(cache._h, r, r, 0, 1, None, None, None, 1, None) == 1
    assert L.mc_kv_attend_dev(cache._h, r, r, 0, 2, None, None, 1, 0, 1.0, None) == 1


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_of_no_segment_at_all(kv, dtype):
    """A read of rows without any segment: all of them come back as zeros."""
    cache = kv.KvCache(2, 2, 32, 8)
    some = ints([0, 0])
    out = torch.full((2, 70, 2, 32), 9.0, dtype=DTYPES[dtype], device=DEV)
    k, v = (ctypes.byref(kv._Rows(x.data_ptr(), 64, 32)) for x in out)
    code = {"f32": 0, "bf16": 2}[dtype]
    assert cache._lib.mc_kv_read_dev(cache._h, k, v, code, 70, some.data_ptr(), None, some.data_ptr(), some.data_ptr(), 0, None) == 0
    torch.cuda.synchronize()
    assert not out.any()


@pytest.mark.parametrize("dtype,bits", [("f32", 8), ("bf16", 4)])
@pytest.mark.parametrize("lens,n_rows", [
    ([4, 16], 10), ([300, 40, 0, 30], 330), ([9, 5], 3), ([1, 1, 3], 3), ([1, 1, 1, 9], 4), ([7, 10 ** 9], 20)])
def test_starts_past_the_rows(kv, dtype, bits, lens, n_rows):
    """Starts that go beyond the rows there are: segments that fit are written and read, rows of the others
    come back as zeros, and the cache reports it. Few and many rows a segment."""
    heads, dim, g = 3, 48, gen(7)
    n = len(lens)
    start = starts(lens)
    x = rows(g, n_rows, heads, dim, dtype)
    cache = kv.KvCache(n, heads, dim, 301, bits=bits)
    cache.write(x.to(DEV), x.to(DEV), ints([0] * n), ints(start))
    with pytest.raises(Exception, match="out of range"):
        cache.check()
    out = tuple(torch.full((n_rows, heads, dim), 9.0, dtype=DTYPES[dtype], device=DEV) for _ in range(2))
    cache.read(ints([0] * n), ints([300] * n), ints(start), out=out)
    with pytest.raises(Exception, match="out of range"):
        cache.check()
    want = torch.zeros(x.shape)
    for b in range(n):
        if start[b + 1] <= n_rows:
            want[start[b]:start[b + 1]] = ref.value(x[start[b]:start[b + 1]], bits).float()
    for y in out:
        assert torch.equal(y.cpu(), want.to(DTYPES[dtype]))


@pytest.mark.parametrize("start,n_rows", [([-2, 4, 10], 10), ([-9, -1, 10], 3), ([0, 6, 3, 12], 12), ([3, 2], 5), ([3, 2], 1)])
def test_starts_below_the_rows_or_out_of_order(kv, start, n_rows):
    """Negative or decreasing starts are reported too."""
    n = len(start) - 1
    cache = kv.KvCache(n, 1, 16, 16, bits=8)
    x = torch.randn((n_rows, 1, 16), device=DEV)
    cache.write(x, x, ints([0] * n), ints(start))
    with pytest.raises(Exception, match="out of range"):
        cache.check()
    out = (torch.full_like(x, 9.0), torch.full_like(x, 9.0))
    cache.read(ints([0] * n), ints([0] * n), ints(start), out=out)
    with pytest.raises(Exception, match="out of range"):
        cache.check()
    assert not out[0].any() and not out[1].any()  # sessions without positions: zeros, whoever's the row is


@pytest.mark.parametrize("dtype,dim,group", [("f32", 64, 2), ("bf16", 64, 2), ("f16", 128, 3), ("f16", 24, 2), ("f32", 192, 2),
                                             ("bf16", 64, 1)])
def test_outputs_in_place_of_the_queries(kv, dtype, dim, group):
    """out=q, with a hidden NaN and infinity that make rows be computed a second time, and a visible one."""
    g, n, heads = gen(dim), 300, 2
    q = torch.randn((n, heads * group, dim), generator=g).to(DTYPES[dtype]).to(DEV)
    k, v = rows(g, n, heads, dim, dtype), rows(g, n, heads, dim, dtype)
    v[100, 0] = float("nan")
    v[150, 1, 3] = float("inf")
    k[290, 1] = float("nan")
    want = kv.window_attention(q, k.to(DEV), v.to(DEV), window=20, sinks=2)
    kv.window_attention(q, k.to(DEV), v.to(DEV), window=20, sinks=2, out=q)
    bad = want.isnan()
    assert bad[100:120, :group].all() and not bad[120:, :group].any() and not bad[:100].any() and bad[290:, group:].all()
    assert torch.equal(q.isnan(), bad) and torch.equal(q.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))


@pytest.mark.parametrize("slots", [70, 9000])
def test_attend_in_place_of_the_queries(kv, slots):
    g = gen(slots)
    cache = kv.KvCache(3, 2, 64, slots, bits=8)
    k = rows(g, 3 * slots, 2, 64, "bf16").to(DEV)
    cache.write(k, k.flip(0), ints([0] * 3), ints([0, slots, 2 * slots, 3 * slots]))
    q = torch.randn((3, 10, 64), generator=g).bfloat16().to(DEV)
    lens = ints([slots, slots // 2, 1])
    want = cache.attend(q, lens)
    assert cache.attend(q, lens, out=q) is q and torch.equal(q, want)


def test_window_segments_out_of_range_are_reported(kv):
    """Bad starts of window attention: skipped, and reported by a check that needs no cache, once."""
    x = {d: torch.randn((20, 1, d), device=DEV) for d in (64, 192)}
    with contextlib.suppress(Exception):
        kv.check()  # of what ran before
    for dim, dtype in ((64, torch.float32), (64, torch.bfloat16), (192, torch.float32)):
        y = x[dim].to(dtype)
        for q_start, k_start in (([0, 10, 20], [0, 10, 21]), ([0, 10, 21], [0, 10, 20]), ([-1, 10, 20], [0, 10, 20]),
                                 ([0, 12, 10], [0, 10, 20]), ([0] * 999 + [25], [0] * 999 + [20])):
            kv.window_attention(y, y, y, ints(q_start), ints(k_start))
            with pytest.raises(Exception, match="out of range"):
                kv.check()
            kv.check()
        kv.window_attention(y, y, y, ints([0, 10, 20]), ints([0, 10, 20]))
        kv.check(0)
    # a cache's own check is about its own indexes
    cache = kv.KvCache(1, 1, 64, 4)
    kv.window_attention(x[64], x[64], x[64], ints([0, 21]))
    cache.check()
    with pytest.raises(Exception, match="out of range"):
        kv.check()


def test_a_wait_that_ran_out_is_reported_and_cleared(kv):
    """The error word of a wait that gave up: reported once, with or without a cache, and what is computed after
    the report is what it was before. A call in between may give up, but ends."""
    L, g = cache_lib(), gen(21)
    q = torch.randn((2000, 8, 128), generator=g).bfloat16().to(DEV)
    k, v = rows(g, 2000, 2, 128, "bf16").to(DEV), rows(g, 2000, 2, 128, "bf16").to(DEV)
    cache = kv.KvCache(1, 2, 128, 2000, bits=4)
    cache.write(k, v, ints([0]), ints([0, 2000]))
    lens = ints([2000])
    calls = lambda: (kv.window_attention(q, k, v), cache.attend(q[:1], lens))
    before = calls()
    for check in (kv.check, cache.check):
        assert L.mc_selftest_kv_wait_timeout(0) == 0
        calls()
        with pytest.raises(Exception, match="gave up"):
            check()
        check()
        assert all(torch.equal(x, y) for x, y in zip(before, calls()))
        kv.check()


def cache_lib():
    from mignon_ai_b200 import _lib
    L = _lib.lib()
    L.mc_selftest_kv_wait_timeout.restype = ctypes.c_int
    L.mc_selftest_kv_wait_timeout.argtypes = [ctypes.c_int]
    return L


@pytest.mark.parametrize("dtype,most", [("f16", 2.0 ** -8), ("bf16", 2.0 ** -7)])
@pytest.mark.parametrize("at", [0, 40000, 65536])
def test_window_small_weights_add_up(kv, dtype, most, at):
    """One key far above 65,536 others of equal weight, exp(-16.25) of its own or 1.47 * 2^-24, whose share of
    the output is 0.0057. A float16 weight may be off by 2^-25 of 2^7 times its maximum's, 0.27 % of such a
    weight, and the output by 2^-11 of itself; bfloat16 ones by 2^-9 and 2^-9."""
    n, dim = 65537, 64
    q, k, v = torch.zeros((3, 1, dim)), torch.zeros((n, 1, dim)), torch.ones((n, 1, dim))
    q[..., 5] = 1
    k[at, 0, 5] = 16.25
    v[at] = 0
    t = DTYPES[dtype]
    got = kv.window_attention(q.to(t).to(DEV), k.to(t).to(DEV), v.to(t).to(DEV), ints([0, 3]), ints([0, n]), scale=1.0)[-1]
    share = 65536 * torch.exp(torch.tensor(-16.25, dtype=torch.float64))
    want = share / (1 + share)
    assert (got.double().cpu() - want).abs().max() <= most * want


@pytest.mark.parametrize("dtype,dim", [("f16", 24), ("bf16", 24), ("f32", 24), ("f16", 64), ("bf16", 64), ("f32", 64), ("f32", 192)])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_window_queries_that_are_not_finite(kv, dtype, dim, what):
    """A NaN among a query's elements, or an infinity that meets a positive key, makes its row NaN, and no other."""
    g = gen(3)
    q = torch.randn((90, 2, dim), generator=g).to(DTYPES[dtype])
    k, v = rows(g, 90, 1, dim, dtype).abs() + 1, rows(g, 90, 1, dim, dtype)
    q[7, 0, 2] = q[70, 1, dim - 1] = what
    got = kv.window_attention(q.to(DEV), k.to(DEV), v.to(DEV))
    bad = torch.zeros((90, 2), dtype=torch.bool)
    bad[7, 0] = bad[70, 1] = True
    assert torch.equal(got.isnan().all(-1).cpu(), bad) and torch.equal(got.isnan().any(-1).cpu(), bad)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("q_size,k_size", [(3e38, 1e-25), (5e37, 1e-20), (1e-36, 1e20), (1e-42, 1e25)])
def test_attend_queries_of_any_size(kv, dtype, bits, q_size, k_size):
    """Queries near the ends of the type's range, with keys and a scale that bring the scores back to a few."""
    g, n, dim, group = gen(5), 150, 64, 3
    q = (torch.rand((1, group, dim), generator=g).double() * 2 - 1).mul(q_size).to(DTYPES[dtype])
    k = rows(g, n, 1, dim, dtype, size=k_size)
    v = rows(g, n, 1, dim, dtype)
    cache = kv.KvCache(1, 1, dim, n, bits=bits)
    cache.write(k.to(DEV), v.to(DEV), ints([0]), ints([0, n]))
    scale = 0.1 / (q_size * k_size)
    got = cache.attend(q.to(DEV), ints([n]), scale=scale)
    scale = torch.tensor(scale, dtype=torch.float32).double().item()  # as the call takes it
    want = ref.attention(q[0], ref.value(k, bits)[:, 0], ref.value(v, bits)[:, 0], torch.ones((group, n), dtype=torch.bool), scale)
    close(got[0], want, v.float().abs().max().item(), dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [1, 3, 8])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_attend_queries_that_are_not_finite(kv, dtype, group, what):
    """A query with a NaN or an infinity gives NaN, whatever the signs it meets, and no other row does."""
    g, n, dim = gen(group), 100, 64
    for center in (-3.0, 3.0, 0.0):
        k = (torch.randn((n, 1, dim), generator=g) * 0.1 + center).to(DTYPES[dtype])
        k[:, 0, 2] = center + 1  # above each row's center
        cache = kv.KvCache(2, 1, dim, n, bits=8)
        cache.write(torch.cat([k, k]).to(DEV), torch.cat([k, k]).to(DEV), ints([0, 0]), ints([0, n, 2 * n]))
        q = torch.randn((2, group, dim), generator=g).to(DTYPES[dtype])
        q[1, group - 1, 2] = what
        got = cache.attend(q.to(DEV), ints([n, n])).isnan().cpu()
        want = torch.zeros((2, group), dtype=torch.bool)
        want[1, group - 1] = True
        assert torch.equal(got.all(-1), want) and torch.equal(got.any(-1), want)


def test_queries_whose_rows_overlap(kv):
    """Rows that share elements (every position of one long row), and rows repeated by a stride of zero: the
    outputs are rows of their own."""
    g = gen(15)
    k, v = rows(g, 40, 1, 64, "f32").to(DEV), rows(g, 40, 1, 64, "f32").to(DEV)
    cache = kv.KvCache(40, 1, 64, 4, bits=8)
    cache.write(k, v, ints([0] * 40))
    q = torch.randn(103, generator=g).to(DEV).unfold(0, 64, 1)[:, None]
    again = torch.randn((1, 1, 64), generator=g).to(DEV).expand(40, 2, 64)
    for x in (q, again):
        assert torch.equal(kv.window_attention(x, k, v), kv.window_attention(x.contiguous(), k, v))
        assert torch.equal(cache.attend(x, ints([1] * 40)), cache.attend(x.contiguous(), ints([1] * 40)))


def test_numbers_that_do_not_fit(kv):
    """Whole numbers beyond 32 bits are refused, not cut."""
    cache = kv.KvCache(2, 2, 32, 8)
    x = torch.randn((2, 2, 32), device=DEV)
    cache.write(x, x, ints([0, 0]))
    for n in (2 ** 32, 2 ** 32 + 1, 2 ** 31, -2 ** 32 + 1):
        for call in (lambda: cache.attend(x, ints([1, 1]), window=n), lambda: kv.window_attention(x, x, x, window=n),
                     lambda: kv.window_attention(x, x, x, sinks=n), lambda: kv.KvCache(2, 2, 32, n),
                     lambda: kv.KvCache(2, 2, 32, 8, sinks=n), lambda: kv.KvCache(2, 2, 32, 8, bits=n + 4),
                     lambda: kv.KvCache(n, 2, 32, 8)):
            with pytest.raises((ValueError, RuntimeError)):
                call()


def test_rows_beyond_32_bits(kv):
    """More rows, or heads, than the library counts (one row seen many times): refused, not cut."""
    cache = kv.KvCache(2, 1, 32, 8)
    many = torch.zeros((1, 1, 32), device=DEV).expand(2 ** 32 + 2, 1, 32)
    heads = torch.zeros((2, 1, 32), device=DEV).expand(2, 2 ** 32 + 1, 32)
    x = torch.zeros((2, 1, 32), device=DEV)
    for call in (lambda: cache.write(many, many, ints([0, 0]), ints([0, 1, 2])),
                 lambda: cache.read(ints([0, 0]), ints([0, 0]), ints([0, 1, 2]), out=(many, many)),
                 lambda: cache.attend(heads, ints([0, 0]), out=heads),
                 lambda: kv.window_attention(x, many, many, ints([0, 2]))):
        with pytest.raises(ValueError, match="32 bits"):
            call()
