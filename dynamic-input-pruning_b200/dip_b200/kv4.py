"""The 4-bit paged KV cache: page bookkeeping, append, read and attention.

What a decode step runs around the DIP MLP.  Keys and values are held in 4 bits
(0.53 bytes an element with the pairs, a head of 128): per token and head

    min = min x,  scale = round16((max x - min) / 15),
    code = round((x - min) / scale),                      x ~ code * scale + min

in pages of 16, 32, 64 or 128 tokens; block table, slot map and lengths live on
the GPU, so a step needs no host synchronisation and can be captured in a CUDA
graph.  The reference keeps its host model's 16-bit cache (the DIP modules replace
the MLP only), so there is no counterpart to cite.

`KV4Cache` holds the whole state of a model; the functions are its parts.
"""
from __future__ import annotations

import math

import torch

from ._lib import load_ops

load_ops()


def kv4_page_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one KV head's part of a page."""
    n = torch.ops.dip_b200.kv4_page_bytes(page_size, head_dim)
    if n == 0:
        raise ValueError(f"page_size must be 16, 32, 64 or 128 and head_dim 64 or 128, got "
                         f"{page_size} and {head_dim}")
    return n


def kv4_workspace(device) -> torch.Tensor:
    """Zeroed workspace for kv4_attention: one for each stream that runs it."""
    return torch.zeros(torch.ops.dip_b200.kv4_attention_workspace_bytes(), dtype=torch.uint8,
                       device=device)


def page_extend(lens, new_lens, block_table, free_list, free_count, page_size: int,
                num_tokens: int):
    """Grows request r from lens[r] to lens[r] + new_lens[r] tokens.

    Takes pages from the top of the free list (free_list[free_count - 1] first),
    enters them into block_table [n, max_blocks] in place and returns
    (lens, cu_q [n + 1], slots [num_tokens], free_count, status [1]): the new
    lengths, the requests' first new tokens, each new token's slot (-1 past the
    sum of new_lens), the pages left.  status 0; else nothing was taken and all
    slots are -1: > 0 pages too few, -1 num_tokens too small, -2 a request longer
    than its block table row."""
    return torch.ops.dip_b200.page_extend.default(lens, new_lens, block_table, free_list,
                                                  free_count, page_size, num_tokens)


def page_release(done, lens, block_table, free_list, free_count, page_size: int) -> None:
    """Gives the pages of the requests with done[r] back, in place: their table
    entries become -1, their lengths 0."""
    torch.ops.dip_b200.page_release_.default(done, lens, block_table, free_list, free_count,
                                             page_size)


def kv4_append(k, v, slots, cache) -> None:
    """Quantises k, v [tokens, kv_heads, head_dim] (bf16 or fp16, any token and
    head strides) into cache at slots [tokens]; slots outside it (-1) are skipped."""
    torch.ops.dip_b200.kv4_append.default(k, v, slots, cache)


def kv4_read(cache, slots, head_dim: int, dtype=torch.bfloat16):
    """The keys and values that the rows at slots stand for, [tokens, kv_heads,
    head_dim] each; zeros for slots outside the cache."""
    return torch.ops.dip_b200.kv4_read.default(cache, slots, head_dim, dtype)


def kv4_attention(q, cache, block_table, kv_lens, cu_q, max_q: int, scale: float | None = None,
                  causal: bool = True, workspace=None):
    """q [tokens, heads, head_dim] over the cache -> (out like q, lse [tokens, heads]).

    Request r's queries q[cu_q[r]:cu_q[r+1]] are the last of its kv_lens[r] cached
    tokens; cu_q ascends (else no query is served and take_device_error() gives 2).  scale defaults to 1 / sqrt(head_dim).  max_q bounds the query tokens
    of one request; it only chooses the kernel.  A query that sees nothing, or of no
    request, gets zeros and lse -inf.  Without a workspace (kv4_workspace) each call makes one."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return torch.ops.dip_b200.kv4_attention.default(q, cache, block_table, kv_lens, cu_q, max_q,
                                                    scale, causal, workspace)


class KV4Cache:
    """A model's 4-bit paged KV cache: one block table and free list for all its
    layers, one cache tensor a layer.

    A step is `extend` once, then `append` and `attend` in every layer; `release`
    when requests end.  All of it runs on the current stream without host
    synchronisation (`status` is read by the caller when it wants to know)."""

    def __init__(self, n_layers: int, num_pages: int, kv_heads: int, head_dim: int,
                 max_requests: int, max_tokens: int, page_size: int = 64,
                 dtype=torch.bfloat16, device="cuda:0"):
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"dtype must be bfloat16 or float16, got {dtype}")
        part = kv4_page_bytes(page_size, head_dim)
        self.page_size, self.head_dim, self.dtype = page_size, head_dim, dtype
        i32 = dict(dtype=torch.int32, device=device)
        # zeroed: unwritten rows stand for 0
        self.layers = torch.zeros(n_layers, num_pages, kv_heads, part, dtype=torch.uint8,
                                  device=device)
        self.block_table = torch.full((max_requests, -(-max_tokens // page_size)), -1, **i32)
        self.lens = torch.zeros(max_requests, **i32)
        self.free_list = torch.arange(num_pages - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), num_pages, **i32)
        self.workspace = kv4_workspace(device)
        self.cu_q = self.slots = self.status = None
        self.max_q = 0

    def extend(self, new_lens, num_tokens: int, max_q: int | None = None) -> None:
        """Makes room for new_lens[r] more tokens of every request (int32 on the
        GPU, 0 for an idle one); num_tokens is their sum, or a bound on it when the
        step is padded; max_q bounds the largest of them (default num_tokens)."""
        self.cu_q, self.slots, self.status = torch.ops.dip_b200.page_extend_.default(
            self.lens, new_lens, self.block_table, self.free_list, self.free_count,
            self.page_size, num_tokens)
        self.max_q = num_tokens if max_q is None else max_q

    def append(self, layer: int, k, v) -> None:
        """The step's new keys and values [num_tokens, kv_heads, head_dim] of a layer."""
        if k.dtype != self.dtype:
            raise TypeError(f"the cache holds {self.dtype}, got {k.dtype}")
        kv4_append(k, v, self.slots, self.layers[layer])

    def attend(self, layer: int, q, scale: float | None = None, causal: bool = True):
        """The step's queries [num_tokens, heads, head_dim] over the layer's cache."""
        if q.dtype != self.dtype:
            raise TypeError(f"the cache holds {self.dtype}, got {q.dtype}")
        return kv4_attention(q, self.layers[layer], self.block_table, self.lens, self.cu_q,
                             self.max_q, scale, causal, self.workspace)

    def release(self, done) -> None:
        """Frees the pages of the requests with done[r] (bool on the GPU)."""
        page_release(done, self.lens, self.block_table, self.free_list, self.free_count,
                     self.page_size)
