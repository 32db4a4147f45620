"""Decoder layers around the DIP MLP: int4 projections, the 4-bit paged KV cache and
attention over it, and the pruned MLP, for a ragged batch of requests.

Per layer and token (pre-norm, unit norm weights, no positional encoding):

    x += W_o attend(W_qkv norm(x)),    x += DIP-MLP(norm(x))

The reference replaces the MLP of its host model only (dip_stream_predispatch.py:218-289)
and leaves the rest to it; these layers run the library's operators together as a serving
loop would: one page_extend a step, then append and attention in every layer.  Weights
are synthetic (seeded, quantised int4 g128 as make_layer's).

    python -m dip_b200.decoder          # ragged prompts, then decode steps from a graph
"""
from __future__ import annotations

import torch
import torch.nn.functional as F

from .batch import batched_dip_layer
from .fastpath import _TC_MAX_ROWS, dense_mlp, tc_down_ok, tc_linear_ok
from .kv4 import KV4Cache
from .qlinear import QuantLinear, dequantize
from .stack import RMS_EPS, StackConfig, make_layer


def _quant_linear(in_f: int, out_f: int, gen, device) -> QuantLinear:
    lin = QuantLinear(in_f, out_f).to(device)
    w = torch.randn(out_f, in_f, generator=gen, device=device) * in_f ** -0.5
    lin.qweight, lin.scales = torch.ops.dip_b200.quantize_int4(w.to(torch.bfloat16))
    return lin


class DipDecoder:
    """A stack of decoder layers over one KV4Cache.

    step() takes the new tokens of every request at once (their hidden states side by
    side, requests in order) and returns the layers' output for them: decode with one
    token a request, prompts and chunks of prompts with more, any mix of them."""

    def __init__(self, cfg: StackConfig, heads: int, kv_heads: int, head_dim: int,
                 max_requests: int, max_tokens: int, num_pages: int, page_size: int = 64,
                 device="cuda:0"):
        self.cfg, self.heads, self.kv_heads, self.head_dim = cfg, heads, kv_heads, head_dim
        gen = torch.Generator(device=device).manual_seed(cfg.seed * 7919 + 17)
        self.qkv = [_quant_linear(cfg.hidden, (heads + 2 * kv_heads) * head_dim, gen, device)
                    for _ in range(cfg.n_layers)]
        self.out = [_quant_linear(heads * head_dim, cfg.hidden, gen, device)
                    for _ in range(cfg.n_layers)]
        self.mlp = [make_layer(cfg, l, device) for l in range(cfg.n_layers)]
        self.cache = KV4Cache(cfg.n_layers, num_pages, kv_heads, head_dim, max_requests,
                              max_tokens, page_size, torch.bfloat16, device)
        self._mlp_ws = torch.zeros(
            torch.ops.dip_b200.mlp_workspace_bytes(cfg.hidden, cfg.inter, cfg.k), dtype=torch.uint8,
            device=device)

    def _norm(self, x: torch.Tensor) -> torch.Tensor:
        # norm(x + x) with four times the epsilon: powers of two throughout, so x's own norm to the bit
        return torch.ops.dip_b200.residual_rmsnorm(x, x, 4 * RMS_EPS)

    def _mlp(self, L: dict, x: torch.Tensor, dense: bool) -> torch.Tensor:
        args = (L["gate_qw"], L["gate_sc"], L["up_qw"], L["up_sc"], L["down_t_qw"], L["down_t_sc"])
        hidden, k = self.cfg.hidden, self.cfg.k
        if dense:
            y = dense_mlp(*args, x)
            if y is None:   # shapes that the GEMMs do not take
                w = [dequantize(args[i], args[i + 1]) for i in (0, 2, 4)]
                y = (F.silu(F.linear(x, w[0])) * F.linear(x, w[1])) @ w[2]
            return y
        tc = tc_linear_ok(hidden, x) and tc_down_ok(self.cfg.inter, hidden, x)
        gemv = hidden % 1024 == 0 and hidden <= 5120   # what the batched GEMV takes
        ys = []
        for b in x.split(_TC_MAX_ROWS):
            if tc and (b.shape[0] >= 16 or not gemv):
                ys.append(batched_dip_layer(L, b, k, "tc")[0])
            elif gemv:
                ys.append(batched_dip_layer(L, b, k, "gather")[0])
            else:   # token by token
                ys += [torch.ops.dip_b200.mlp_decode(*args, t, k, self._mlp_ws)[0][None] for t in b]
        return ys[0] if len(ys) == 1 else torch.cat(ys)

    def step(self, x: torch.Tensor, new_lens: torch.Tensor, max_q: int | None = None,
             dense: bool = False) -> torch.Tensor:
        """x [tokens, hidden] bf16, new_lens int32 [requests] on the GPU (their sum is
        tokens, or less where x is padded); max_q bounds one request's new tokens.

        The MLP is pruned for every token, each by its own channels, so that what a
        request gets does not depend on the requests and tokens that share its step.
        dense: this step's tokens take all channels, as the reference's modules run
        prompts (dip_stream_predispatch.py:206-215)."""
        T, c = x.shape[0], self.cache
        h, kv, d = self.heads, self.kv_heads, self.head_dim
        c.extend(new_lens, T, max_q)
        for l in range(self.cfg.n_layers):
            qkv = self.qkv[l](self._norm(x)).view(T, h + 2 * kv, d)
            c.append(l, qkv[:, h:h + kv], qkv[:, h + kv:])
            att, _ = c.attend(l, qkv[:, :h])
            x = x + self.out[l](att.view(T, h * d))
            x = x + self._mlp(self.mlp[l], self._norm(x), dense)
        return x

    def release(self, done: torch.Tensor) -> None:
        """Ends the requests with done[r] (bool on the GPU): their pages are free again."""
        self.cache.release(done)


def main() -> None:
    cfg = StackConfig(n_layers=2, seed=1)          # hidden 5120, intermediate 25600
    prompts, steps = [700, 33, 2500, 1], 32
    dev = torch.device("cuda", 0)
    dec = DipDecoder(cfg, heads=64, kv_heads=8, head_dim=128, max_requests=len(prompts),
                     max_tokens=4096, num_pages=96, device=dev)
    gen = torch.Generator(device=dev).manual_seed(3)
    lens = torch.tensor(prompts, dtype=torch.int32, device=dev)
    x = torch.randn(sum(prompts), cfg.hidden, generator=gen, device=dev).to(torch.bfloat16)
    y = dec.step(x, lens, max(prompts), dense=True)
    last = y[dec.cache.cu_q[1:].long() - 1]        # the prompts' last tokens
    one = torch.ones_like(lens)
    tok = last.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tok.copy_(dec.step(tok, one, 1))           # warm-up, a decode step of its own
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tok.copy_(dec.step(tok, one, 1))
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    for _ in range(steps):
        graph.replay()
    b.record()
    torch.cuda.synchronize()
    print(f"{len(prompts)} requests, {cfg.n_layers} layers: {a.elapsed_time(b) / steps * 1e3:.1f} us "
          f"a decode step, lengths {dec.cache.lens.tolist()}, {dec.cache.free_count.item()} pages free")
    dec.release(torch.ones(len(prompts), dtype=torch.bool, device=dev))
    print(f"released: {dec.cache.free_count.item()} pages free")


if __name__ == "__main__":
    main()
