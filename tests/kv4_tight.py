"""Bounds for the attention over the 4-bit paged cache that follow from what its kernels
round, and 64-bit values of chosen rows on the GPU (long contexts).

What is rounded, to first order, for a row with weights p_t (sum 1), value steps s_t,
codes c_t, mins m_t over L positions:

* scores: products of codes and queries are exact, summed in fp32 by at most 128 terms in
  eight steps of the tensor cores, each of which may cut off 2^-22 of the sum of the terms'
  sizes: 2^-19 sabs with sabs = scale * sum |q| |k|; the pairs' four fp32 roundings, the
  exponential and the reference it is taken from: 2^-21 (sabs + |lse| + 32).  ds, doubled
  for safety.
* weights p_t s_t: once to fp16, 2^-11 of each at most, and 2^-24 where they are
  subnormal (twice 2^-25: a tile's weights may be rescaled after they were rounded) against
  a largest weight of at least 2^5: 2^-29 of the largest, of codes within 8 of the middle,
  for each of L positions.
* fp32 sums: at most L / 16 + 64 steps, each of which cuts off at most 2^-23.
* the result, once: u of it."""
import math

import torch

import kv4_ref as R


def unit(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11


def rows(q, cache, table, kv_lens, cu_q, P, dtype, picks, causal=True, scale=None):
    """For the query tokens `picks`, in 64 bits on the tensors' device: a dict of out, lse,
    sabs, length and the sums of the bounds, each [picks, heads(, D)]."""
    T, H, D = q.shape
    hkv = cache.shape[1]
    G = H // hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    z = dict(dtype=torch.float64, device=q.device)
    n = len(picks)
    res = {"out": torch.zeros(n, H, D, **z), "dev": torch.zeros(n, H, D, **z),
           "dev2": torch.zeros(n, H, D, **z), "size": torch.zeros(n, H, D, **z),
           "lse": torch.full((n, H), -math.inf, **z), "sabs": torch.zeros(n, H, **z),
           "top": torch.zeros(n, H, **z), "len": torch.zeros(n, H, **z)}
    kc, vc, kp, vp = None, None, None, None
    held = None
    for i, t in enumerate(picks):
        r = max(x for x in range(len(kv_lens)) if cu_q[x] <= t)
        L, new = kv_lens[r], cu_q[r + 1] - cu_q[r]
        if held != r:
            page = table[r, :-(-L // P)].long()
            kc, vc, kp, vp = (x.transpose(1, 2).flatten(0, 1)[:L] for x in
                              R.parts(cache[page], P, D, dtype))     # [L, hkv, ...]
            held = r
        lim = L - new + (t - cu_q[r]) + 1 if causal else L
        if lim <= 0:
            continue
        for j in range(hkv):
            hs = slice(j * G, (j + 1) * G)
            ks, km = kp[:lim, j].unbind(-1)
            vs, vm = vp[:lim, j].unbind(-1)
            c = vc[:lim, j].double()
            k = kc[:lim, j] * ks[:, None] + km[:, None]
            qd = q[t, hs].double()
            s = qd @ k.T * scale
            lse = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[:, None])
            w = p * vs
            res["out"][i, hs] = p @ (c * vs[:, None] + vm[:, None])
            res["dev"][i, hs] = w @ (c - 8).abs()
            res["dev2"][i, hs] = w.square() @ (c - 8).square()
            res["size"][i, hs] = w @ (c + 8) + (p @ vm.abs())[:, None]
            res["lse"][i, hs] = lse
            res["sabs"][i, hs] = (qd.abs() @ (kc[:lim, j] * ks[:, None] + km.abs()[:, None]).T
                                  * abs(scale)).amax(-1)
            res["top"][i, hs] = w.amax(-1)
            res["len"][i, hs] = lim
    return res


def check(out, lse, ref, dtype):
    """Elementwise, and each row's root mean square: the roundings of the result are uniform
    (u / sqrt 3 at most), those of the weights independent (2^-11 each at most)."""
    out, lse = out.double(), lse.double()
    u = unit(dtype)
    some = ref["len"] > 0
    assert not out[~some].any() and lse[~some].isinf().all()
    fin = torch.where(some, ref["lse"], 0.0).abs()
    ds = 2 * (2.0 ** -19 * ref["sabs"] + 2.0 ** -21 * (ref["sabs"] + fin + 32))
    acc = (ref["len"] / 16 + 64) * 2.0 ** -23
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-38
    rest = ((torch.expm1(2 * ds) + 2 * acc)[..., None] * ref["size"]
            + (ref["len"] * 8 * 2.0 ** -29 * ref["top"])[..., None] + tiny)
    err = (out - ref["out"]).abs()
    bound = u * ref["out"].abs() + 2.0 ** -11 * ref["dev"] + rest
    bad = (err - bound).max()
    assert bool((err <= bound).all()), f"out off by {err.max():.3e}, past the bound by {bad:.3e}"
    off = (lse - ref["lse"]).abs()[some]
    assert bool((off <= (ds + acc + 2.0 ** -22 * (1 + fin))[some]).all()), f"lse off by {off.max():.3e}"
    rms = err.square().mean(-1).sqrt()
    want = (u * u / 3 * ref["out"].square() + 2.0 ** -22 * ref["dev2"]).mean(-1).sqrt()
    lim = 1.5 * want + rest.amax(-1)
    assert bool((rms <= lim).all()), f"a row's rms error is {(rms / lim).max():.2f} of its limit"
