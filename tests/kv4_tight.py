"""Bounds for the attention over the 4-bit paged cache that follow from what its kernels
round, and 64-bit values of chosen rows on the GPU (long contexts).

What is rounded, to first order, for a row with weights p_t (sum 1), value steps s_t,
codes c_t, mins m_t over L positions:

* scores: products of codes and queries are exact, summed in fp32 in eight steps of the
  tensor cores that cut off 2^-23 of the sum so far each, which lies within four root sums of
  squares of its terms and its end; then the pairs' and the reference's roundings, 2^-22 of
  the parts' sizes together.  ds, doubled for safety.
* weights p_t s_t: once to fp16, 2^-11 of each at most, and 2^-24 where they are
  subnormal (twice 2^-25: a tile's weights may be rescaled after they were rounded) against
  a largest weight of at least 2^5: 2^-29 of the largest, of codes within 8 of the middle,
  for each of L positions.
* fp32 sums: at most L / 16 + 64 steps, each of which cuts off at most 2^-23.
* the result, once: half an ulp of it."""
import math

import torch

import kv4_ref as R


def unit(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11


def rows(q, cache, table, kv_lens, cu_q, P, dtype, picks, causal=True, scale=None):
    """For the query tokens `picks`, in 64 bits on the tensors' device: a dict of out, lse,
    length and what the bounds are made of, each [picks, heads(, D)]."""
    T, H, D = q.shape
    hkv = cache.shape[1]
    G = H // hkv
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    z = dict(dtype=torch.float64, device=q.device)
    n = len(picks)
    res = {"out": torch.zeros(n, H, D, **z), "dev": torch.zeros(n, H, D, **z),
           "dev2": torch.zeros(n, H, D, **z), "size": torch.zeros(n, H, D, **z),
           "lse": torch.full((n, H), -math.inf, **z), "sum": torch.zeros(n, H, **z),
           "part": torch.zeros(n, H, **z), "spread": torch.zeros(n, H, D, **z),
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
            v = c * vs[:, None] + vm[:, None]
            o = res["out"][i, hs]
            res["spread"][i, hs] = ((p.square() @ v.square()) - 2 * o * (p.square() @ v)
                                    + o.square() * p.square().sum(-1, keepdim=True)).clamp(min=0)
            res["sum"][i, hs] = ((qd.square() @ (kc[:lim, j] * ks[:, None]).square().T).sqrt().amax(-1)
                                 * abs(scale))
            mins = qd.sum(-1, keepdim=True).abs() * km.abs() * abs(scale)
            res["part"][i, hs] = s.abs().amax(-1) + mins.amax(-1)
            res["top"][i, hs] = w.amax(-1)
            res["len"][i, hs] = lim
    return res


def check(out, lse, ref, dtype):
    """Elementwise, and the rows' root mean squares against what uniform roundings of the
    result, independent ones of the scores and one large one of a weight make: each row's up to
    sqrt(3) of it (channels of few values, as rows that attend to one token have, may all be
    rounded by half an ulp), that of 64 rows or more up to 1 on average (a mean of roots is below
    the root of the mean)."""
    out, lse = out.double(), lse.double()
    u = unit(dtype)
    some = ref["len"] > 0
    assert not out[~some].any() and lse[~some].isinf().all()
    fin = torch.where(some, ref["lse"], 0.0).abs()
    ds = 2 * (8 * 2.0 ** -23 * (4 * ref["sum"] + ref["part"]) + 2.0 ** -22 * (ref["part"] + fin + 16))
    steps = ref["len"] / 16
    tiny = 2.0 ** -24 if dtype == torch.float16 else 1e-38
    small = (ref["len"] * 8 * 2.0 ** -29 * ref["top"])[..., None] + tiny
    rest = (torch.expm1(2 * ds) + 2 * (steps + 64) * 2.0 ** -23)[..., None] * ref["size"] + small
    err = (out - ref["out"]).abs()
    bound = u * ref["out"].abs() + 2.0 ** -11 * ref["dev"] + rest
    bad = (err - bound).max()
    assert bool((err <= bound).all()), f"out off by {err.max():.3e}, past the bound by {bad:.3e}"
    off = (lse - ref["lse"]).abs()[some]
    room = (ds + (steps + 64) * 2.0 ** -23 + 2.0 ** -22 * (1 + fin))[some]
    assert bool((off <= room).all()), f"lse off by {off.max():.3e}, {(off / room).max():.2f} of its room"
    least = 2.0 ** -14 if dtype == torch.float16 else 2.0 ** -126
    ulp = 2 * u * torch.exp2(torch.floor(torch.log2(ref["out"].abs().clamp(min=least))))
    var = ulp.square() / 12 + 2.0 ** -22 * ref["dev2"] + (2 * ds).square()[..., None] * ref["spread"]
    want = var.mean(-1).sqrt()
    rest = (small + ((steps + 4) * 2.0 ** -24)[..., None] * ref["size"]).amax(-1)
    ratio = (err.square().mean(-1).sqrt() - rest)[some] / want[some]
    if ratio.numel() == 0:
        return
    assert ratio.max() <= 1.74, f"a row's rms error is {ratio.max():.2f} of what is expected"
    if ratio.numel() >= 64:
        assert ratio.mean() <= 1.0, f"the rows' rms errors are {ratio.mean():.2f} of what is expected"
