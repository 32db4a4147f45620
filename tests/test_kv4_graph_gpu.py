"""A KV4Cache step on a stream other than the one that made the cache, and captured."""
import pytest
import torch

import kv4_ref as R
import kv4_tight as T
from test_kv4_gpu import BF

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 30])
def test_capture_after_a_warm_up_on_another_stream(dip, n):
    """The other stream waits for the one whose fills the cache and the inputs are."""
    gen = torch.Generator().manual_seed(n)
    B, H, hkv, D, P, steps = 3, 8, 2, 64, 16, 5
    c = dip.KV4Cache(1, 60, hkv, D, B, 256, P, BF)
    k, v, q = (torch.randn(steps + 1, B * n, h, D, generator=gen).to(BF).cuda() for h in (hkv, hkv, H))
    ks, vs, qs = (torch.zeros_like(x[0]) for x in (k, v, q))
    new = torch.full((B,), n, dtype=torch.int32, device="cuda")

    def put(t):
        for dst, src in ((ks, k), (vs, v), (qs, q)):
            dst.copy_(src[t])

    def step():
        c.extend(new, B * n, n)
        c.append(0, ks, vs)
        return c.attend(0, qs)

    put(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = step()
    for t in range(1, steps + 1):
        put(t)
        g.replay()
    L = n * (steps + 1)
    assert c.lens.tolist() == [L] * B and c.status.item() == 0
    for b in range(B):      # every token of request b in the order of the steps
        rows = torch.stack([k[:, b * n:(b + 1) * n].flatten(0, 1), v[:, b * n:(b + 1) * n].flatten(0, 1)])
        page = c.block_table[b, :-(-L // P)].long()
        kc, vc, _, _ = (x.transpose(1, 2).flatten(0, 1)[:L] for x in R.parts(c.layers[0][page], P, D, BF))
        assert torch.equal(kc, R.quantise(rows[0])[0]) and torch.equal(vc, R.quantise(rows[1])[0])
    cu = [b * n for b in range(B + 1)]
    picks = list(range(0, B * n, 7))
    ref = T.rows(qs, c.layers[0], c.block_table, [L] * B, cu, P, BF, picks)
    T.check(out[picks], lse[picks], ref, BF)
