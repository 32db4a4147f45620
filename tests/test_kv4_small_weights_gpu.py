"""Many small softmax weights below one large one (an attention sink): each is far below the
largest, together they are half of the sum and carry the values' means."""
import pytest
import torch

import kv4_ref as R
import kv4_tight as T

pytestmark = pytest.mark.gpu
BF, FP = torch.bfloat16, torch.float16


def _sink(seed, L, hkv, D, P, dtype, gap):
    """A cache of L tokens on the GPU whose first key scores about `gap` nats above the rest
    for queries along `e`, values with means of their channels."""
    gen = torch.Generator("cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    e = rnd(hkv, D).sign()
    k = 0.2 * rnd(L, hkv, D)
    k[0] = e * gap / (4 * D ** 0.5)              # q = 4 e + noise, scores / sqrt(D)
    v = rnd(L, hkv, D) + rnd(hkv, D)
    pages = -(-L // P)
    cache = torch.zeros(pages, hkv, R.page_bytes(P, D), dtype=torch.uint8, device="cuda")
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    pos = torch.arange(L, device="cuda")
    torch.ops.dip_b200.kv4_append(k.to(dtype), v.to(dtype), table.long()[pos // P] * P + pos % P, cache)
    return gen, e, cache, table


def _queries(gen, e, n, G, dtype):
    hkv, D = e.shape
    q = 4 * e.repeat_interleave(G, 0) + 0.1 * torch.randn(n, hkv * G, D, generator=gen, device="cuda")
    return q.to(dtype)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("L,n,hkv,G,D,gap", [
    (32768, 2400, 8, 8, 64, 11.5),      # whole tiles: as many as go without cuts
    (32768, 1200, 16, 8, 128, 11.5),
    (32768, 256, 8, 8, 128, 11.5),      # tiles in long parts
    (131072, 300, 8, 8, 64, 12.5),
    (131072, 1, 4, 8, 128, 12.5),       # one token, one request
])
def test_sink_chunk(dip, dtype, L, n, hkv, G, D, gap):
    gen, e, cache, table = _sink(L + n, L, hkv, D, 64, dtype, gap)
    q = _queries(gen, e, n, G, dtype)
    out, lse = dip.kv4_attention(q, cache, table[None], _i32([L]), _i32([0, n]), n)
    picks = sorted({0, n // 3, n - 1})
    ref = T.rows(q, cache, table[None], [L], [0, n], 64, dtype, picks)
    T.check(out[picks], lse[picks], ref, dtype)


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("D,nreq,q_len", [(64, 222, 1), (128, 222, 1), (128, 60, 2)])
def test_sink_decode_batch(dip, dtype, D, nreq, q_len):
    """So many requests (of the same pages) that one warp takes whole contexts."""
    L, hkv, G = 32768, 8, 8 // q_len
    gen, e, cache, table = _sink(D, L, hkv, D, 64, dtype, 11.5)
    n = nreq * q_len
    q = _queries(gen, e, n, G, dtype)
    cu = list(range(0, n + 1, q_len))
    tab = table[None].repeat(nreq, 1)
    out, lse = dip.kv4_attention(q, cache, tab, _i32([L] * nreq), _i32(cu), q_len)
    picks = [0, n // 2, n - 1]
    ref = T.rows(q, cache, tab, [L] * nreq, cu, 64, dtype, picks)
    T.check(out[picks], lse[picks], ref, dtype)


@pytest.mark.parametrize("dtype,size", [(BF, 1.0), (BF, 2.0 ** 100), (BF, -2.0 ** 120), (FP, -60000.0)])
@pytest.mark.parametrize("n", [1, 40, 200])
def test_rows_of_equal_values(dip, dtype, size, n):
    """Value rows whose channels are all equal (scale 0), of any size: the result is a mean of them."""
    L, hkv, G, D, P = 1500, 2, 4, 64, 16
    gen, e, cache, table = _sink(n, L, hkv, D, P, dtype, 2.0)
    q = _queries(gen, e, n, G, dtype)
    pos = torch.arange(L, device="cuda")
    k = torch.randn(L, hkv, D, generator=gen, device="cuda").to(dtype)
    v = (size * (0.5 + 0.5 * torch.rand(L, hkv, 1, generator=gen, device="cuda"))).to(dtype)
    dip.kv4_append(k, v.expand(L, hkv, D), table.long()[pos // P] * P + pos % P, cache)
    out, lse = dip.kv4_attention(q, cache, table[None], _i32([L]), _i32([0, n]), n)
    picks = sorted({0, n // 2, n - 1})
    ref = T.rows(q, cache, table[None], [L], [0, n], P, dtype, picks)
    T.check(out[picks], lse[picks], ref, dtype)
