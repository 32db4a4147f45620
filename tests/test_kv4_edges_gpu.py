"""The 4-bit paged KV cache at inputs on the edge of what it takes."""
import math

import pytest
import torch

import kv4_ref as R
import kv4_tight as T
from test_kv4_gpu import BF, FP, _dev, _run, _setup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("count", [-1, -4, -(1 << 31)])
def test_page_release_with_a_negative_count(dip, count):
    """It counts as an empty list: nothing is written before the list."""
    room = _dev([77] * 8 + [-1] * 6 + [77] * 4)
    free, fc = room[8:14], _dev([count])
    lens, table = _dev([33, 5]), _dev([[4, 9, 2, -1], [7, -1, -1, -1]])
    dip.page_release(_dev([True, False], torch.bool), lens, table, free, fc, 16)
    assert room.tolist() == [77] * 8 + [4, 9, 2, -1, -1, -1] + [77] * 4
    assert fc.tolist() == [3] and lens.tolist() == [0, 5]
    assert table.tolist() == [[-1] * 4, [7, -1, -1, -1]]


def test_page_release_past_the_capacity(dip):
    room = _dev([77] * 2 + [3, -1] + [77] * 4)
    free, fc = room[2:4], _dev([1])
    lens, table = _dev([33]), _dev([[4, 9, 2]])
    dip.page_release(_dev([True], torch.bool), lens, table, free, fc, 16)
    assert room.tolist() == [77, 77, 3, 4] + [77] * 4 and fc.tolist() == [2]


def _scaled_keys(seed, L, n, H, hkv, D, P, dtype, size):
    """Queries of `size` over keys of 1 / size, so that the scores are ordinary ones."""
    gen = torch.Generator().manual_seed(seed)
    k = (torch.randn(L, hkv, D, generator=gen) / size).to(dtype)
    v = torch.randn(L, hkv, D, generator=gen).to(dtype)
    pages = -(-L // P)
    cache = torch.zeros(pages, hkv, R.page_bytes(P, D), dtype=torch.uint8)
    R.put(cache, P, D, dtype, torch.arange(L), k, v)
    q = (torch.randn(n, H, D, generator=gen) * size).to(dtype)
    return q, cache.cuda(), torch.arange(pages, dtype=torch.int32, device="cuda").view(1, pages)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n", [3, 40, 300])
@pytest.mark.parametrize("dtype,size", [(BF, 1.0), (BF, 2.0 ** 40), (BF, 2.0 ** -40), (FP, 2.0 ** -12)])
def test_non_finite_queries_stay_where_they_are(dip, dtype, size, n, bad):
    """A query with a NaN or an infinity gives NaN; its neighbours' results are their own."""
    L, H, D, P = 400, 8, 64, 16
    q, cache, table = _scaled_keys(n, L, n, H, 2, D, P, dtype, size)
    hit = [(1, 0), (n - 1, 5), (n // 2, 7)]
    for t, h in hit:
        q[t, h, 11] = bad
    q = q.cuda()
    out, lse = dip.kv4_attention(q, cache, table, _dev([L]), _dev([0, n]), n)
    picks = sorted({0, 1, n // 2, n - 1})
    for t, h in hit:
        assert out[t, h].isnan().all() and lse[t, h].isnan()
        q[t, h], out[t, h], lse[t, h] = 0, 0, 0
    ref = T.rows(q, cache, table, [L], [0, n], P, dtype, picks)
    for t, h in hit:
        for x in ref.values():
            x[picks.index(t), h] = 0
        lse[t, h] = -math.inf
    T.check(out[picks], lse[picks], ref, dtype)


@pytest.mark.parametrize("n", [1, 3, 40, 300])
@pytest.mark.parametrize("size", [2.0 ** 119, 2.0 ** 123, 2.0 ** -118])
@pytest.mark.parametrize("scale", [None, -0.25])
def test_queries_over_the_whole_range_of_bf16(dip, size, n, scale):
    """Queries near either end of bf16's range, keys such that the scores are ordinary."""
    L, H, D, P = 400, 8, 64, 16
    q, cache, table = _scaled_keys(n, L, n, H, 2, D, P, BF, size)
    q = q.cuda()
    out, lse = dip.kv4_attention(q, cache, table, _dev([L]), _dev([0, n]), n, scale=scale)
    picks = sorted({0, n // 2, n - 1})
    ref = T.rows(q, cache, table, [L], [0, n], P, BF, picks, scale=scale)
    assert ref["lse"].isfinite().all() and ref["lse"].abs().max() < 100
    T.check(out[picks], lse[picks], ref, BF)


@pytest.mark.parametrize("qs", [[1, 1], [3, 20], [90, 200], [1, 100]])
@pytest.mark.parametrize("first,after", [(1, 0), (7, 3)])
def test_tokens_of_no_request(dip, qs, first, after):
    """Tokens before the first request's and after the last one's: zeros and -inf."""
    lens, P = [300, 250], 16
    q, cache, table, cu = _setup(3, lens, qs, 8, 2, 64, P, BF)
    n = cu[-1]
    wide = torch.randn(first + n + after, 8, 64, generator=torch.Generator().manual_seed(1)).to(BF)
    wide[first:first + n] = q
    junk = torch.full_like(wide, 7.0).cuda()      # leaves something in the allocator's blocks
    del junk
    out, lse = _run(dip, wide, cache, table, lens, [x + first for x in cu])
    R.check(out[first:first + n], lse[first:first + n], R.attention(q, cache, table, lens, cu, P, BF), BF)
    for part in (slice(0, first), slice(first + n, None)):
        assert not out[part].any() and lse[part].isinf().all()


@pytest.mark.parametrize("n,chunk", [(8193, 0), (16384, 0), (20000, 0), (16390, 300)])
def test_more_requests_than_a_launch_takes(dip, n, chunk):
    """Requests on both sides of every launch's border, chunks among them; tokens of no request
    at both ends."""
    gen = torch.Generator().manual_seed(n)
    P, D, hkv, H, pages, first, after = 16, 64, 1, 2, 40, 3, 2
    cache = R.random_cache(gen, pages, hkv, P, D, FP).cuda()
    table = torch.randint(0, pages, (n, 30), generator=gen, dtype=torch.int32).cuda()
    lens = torch.randint(0, 48, (n,), generator=gen).tolist()
    qs = [1] * n
    for r in (5, 8191, 8192, n - 1) if chunk else ():
        lens[r], qs[r] = 400, chunk
    cu = [first]
    for x in qs:
        cu.append(cu[-1] + x)
    q = torch.randn(cu[-1] + after, H, D, generator=gen).to(FP).cuda()
    out, lse = dip.kv4_attention(q, cache, table, _dev(lens), _dev(cu), max(qs))
    for part in (slice(0, first), slice(cu[-1], None)):
        assert not out[part].any() and lse[part].isinf().all()
    for r in sorted({0, 1, 4, 5, 6, 8190, 8191, 8192, n - 2, n - 1} | set(range(100, n, 997))):
        L, m = lens[r], qs[r]
        ref = T.rows(q[cu[r]:cu[r + 1]], cache, table[r:r + 1], [L], [0, m], P, FP, [0, m - 1])
        sel = [cu[r], cu[r] + m - 1]
        T.check(out[sel], lse[sel], ref, FP)


@pytest.mark.parametrize("cu,max_q", [
    ([0, 5, 3, 20], 17), ([0, 20, 0, 20], 20), ([0, 200, 100, 200], 200), ([20, 10, 5, 0], 1),
    ([0, 200] * 40, 200), ([0, 3] * 500, 1), ([0, 200] * 4, 1),
])
@pytest.mark.parametrize("D", [64, 128])
def test_a_descending_cu_q_is_refused(dip, cu, max_q, D):
    """It is known on the device only: zeros, and the device error word."""
    n = len(cu) - 1
    lens = [300] * n
    q, cache, table, _ = _setup(n, [300], [200], 8, 2, D, 64, BF)
    ws = dip.kv4_workspace("cuda")
    args = (q.cuda(), cache.cuda(), table.cuda().repeat(n, 1))
    take = torch.ops.dip_b200.take_device_error
    assert take() == 0
    out, lse = dip.kv4_attention(*args, _dev(lens), _dev(cu), max_q, workspace=ws)
    assert take() == 2
    assert not out.any() and lse.isinf().all()
    good = [0, 200]
    out, lse = dip.kv4_attention(args[0], args[1], table.cuda(), _dev([300]), _dev(good), 200, workspace=ws)
    ref = R.attention(q, cache, table, [300], good, 64, BF)
    R.check(out, lse, ref, BF)
    assert take() == 0
