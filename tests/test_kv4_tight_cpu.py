"""The close bounds of the attention tests see the roundings that the kernels do not make."""
import pytest
import torch

import kv4_ref as R
import kv4_tight as T

BF, FP = torch.bfloat16, torch.float16


def _attend(dtype, q_scale, key=None, weight=None, value=None, query=None):
    """Attention in 64 bits with roundings planted in it -> out, lse, reference."""
    gen = torch.Generator().manual_seed(5)
    P, D, H, hkv, L, n = 16, 128, 4, 2, 700, 20
    cache = R.random_cache(gen, -(-L // P), hkv, P, D, dtype)
    table = torch.arange(-(-L // P), dtype=torch.int32).view(1, -1)
    q = (q_scale * torch.randn(n, H, D, generator=gen)).to(dtype)
    ref = T.rows(q, cache, table, [L], [0, n], P, dtype, list(range(n)), causal=False)

    def cut(x, to):
        return x if to is None else x.to(to).double()

    kc, vc, kp, vp = (x.transpose(1, 2).flatten(0, 1)[:L].double() for x in R.parts(cache, P, D, dtype))
    out, lse = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, dtype=torch.float64)
    for h in range(H):
        j = h // (H // hkv)
        k = cut(kc[:, j] * kp[:, j, :1] + kp[:, j, 1:], key)
        v = cut(vc[:, j] * vp[:, j, :1] + vp[:, j, 1:], value)
        s = cut(q[:, h].double(), query) @ k.T / D ** 0.5
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - top)
        if weight == "kernel":      # p scale in fp16, of codes about zero, the rest in full
            w = (p * vp[:, j, 0]).to(FP).double()
            o = w @ (vc[:, j] - 8) + (p @ (vp[:, j, 1] + 8 * vp[:, j, 0]))[:, None]
        else:
            o = cut(p, weight) @ v
        out[:, h] = (o / p.sum(-1, keepdim=True)).to(dtype).double()
        lse[:, h] = top[:, 0] + p.sum(-1).log()
    return out, lse, ref


@pytest.mark.parametrize("q_scale", [1.0, 3.0, 12.0])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_what_the_kernels_round_is_inside(dtype, q_scale):
    T.check(*_attend(dtype, q_scale), dtype)
    T.check(*_attend(dtype, q_scale, weight="kernel"), dtype)


@pytest.mark.parametrize("dtype,planted", [
    (BF, dict(key=BF)), (BF, dict(key=FP)), (BF, dict(value=BF)), (BF, dict(weight=BF)),
    (FP, dict(key=BF)), (FP, dict(key=FP)), (FP, dict(value=BF)), (FP, dict(weight=BF)),
    (FP, dict(query=BF)),
])
def test_other_roundings_are_outside(dtype, planted):
    """At flat scores or at peaked ones, where single rows weigh."""
    seen = 0
    for q_scale in (1.0, 3.0, 12.0):
        out, lse, ref = _attend(dtype, q_scale, **planted)
        try:
            T.check(out, lse, ref, dtype)
        except AssertionError:
            seen += 1
    assert seen
