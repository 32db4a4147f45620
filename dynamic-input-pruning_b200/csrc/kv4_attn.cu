// kv4_attn.cu — attention of new tokens over the 4-bit paged cache.
//
// Request r has kv_len tokens in the cache, of which its n = cu_q[r+1] - cu_q[r]
// query tokens are the last n; query i of it (causal) sees the positions
// <= kv_len - n + i, else all of them:
//   s_t = scale * sum_d q_d K_td,  out_d = sum_t softmax(s)_t V_td,
//   lse = log sum_t exp(s_t);   no visible position: out = 0, lse = -inf.
#include <algorithm>
#include <cmath>

#include "kv4_attn.cuh"

using namespace dip;

// Up to this many query rows a KV head the decode kernel is faster, which reads the cache
// once for eight; the prefill kernel's cost hardly depends on them.  Decode / prefill, us:
// 16 contexts of 900 to 9000 tokens, 8 heads of 128: 145 / 191 at 64 rows, 174 / 191 at 80,
// 203 / 194 at 96, 262 / 196 at 128; 60 of 500: 80 / 118, 94 / 118, 109 / 120, 133 / 122; one
// of 60000: 123 / 123 at 72, 154 / 122 at 96, 199 / 122 at 128.
static constexpr int kDecodeRows = 80;

extern "C" size_t dip_kv4_attention_workspace_bytes(void) {
  // the decode kernel's counters, zero between calls, then parts, which one kernel after the other uses
  return kv4_decode_counter_bytes() + std::max(kv4_decode_part_bytes(), kv4_prefill_part_bytes());
}

extern "C" int dip_kv4_attention(const dip_kv4_attn_t* p, void* workspace, size_t workspace_bytes,
                                 dip_stream_t stream) {
  if (!p || p->num_tokens < 0 || p->nreq < 0 || p->kv_heads < 1 || p->heads < 1 ||
      p->max_blocks < 0 || p->num_pages < 0 || p->max_q < 0 ||
      (p->dtype != DIP_BF16 && p->dtype != DIP_FP16))
    return DIP_ERR_ARG;
  if (p->heads % p->kv_heads || !std::isfinite(p->scale)) return DIP_ERR_ARG;
  const int pl = kv4_page_log2(p->page_size);
  if (pl < 0 || (p->head_dim != 64 && p->head_dim != 128) || p->heads > 65535 ||
      p->num_tokens > 0x7fffffffLL || p->nreq > (1 << 20))
    return DIP_ERR_UNSUPPORTED;
  if (p->num_tokens == 0) return DIP_OK;
  if (!p->q || !p->out || !p->cu_q || !workspace || !aligned16(p->q) || !aligned16(p->out) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255))
    return DIP_ERR_ARG;
  if (p->nreq > 0 && (!p->kv_lens || (p->max_blocks > 0 && !p->block_table))) return DIP_ERR_ARG;
  if (p->num_pages > 0 && (!p->cache || !aligned16(p->cache))) return DIP_ERR_ARG;
  if ((p->q_token_stride | p->q_head_stride) & 7) return DIP_ERR_ARG;
  if (workspace_bytes < dip_kv4_attention_workspace_bytes()) return DIP_ERR_WORKSPACE;
  AttnArgs a = {};
  a.q = (const uint16_t*)p->q;
  a.q_ts = p->q_token_stride;
  a.q_hs = p->q_head_stride;
  a.cache = (const uint8_t*)p->cache;
  a.g = {(int)p->kv_heads, (int)p->head_dim, pl, kv4_part_bytes(p->page_size, p->head_dim),
         p->num_pages};
  a.max_blocks = p->max_blocks;
  a.num_tokens = (int)p->num_tokens;
  a.heads = (int)p->heads;
  a.group = (int)(p->heads / p->kv_heads);
  a.causal = p->causal != 0;
  a.scale = p->scale;
  a.out = (uint16_t*)p->out;
  a.lse = p->lse;
  a.err = error_word_ptr();
  if (!a.err) return launch_status(cudaErrorUnknown);
  const bool f16 = p->dtype == DIP_FP16;
  cudaStream_t st = (cudaStream_t)stream;
  uint8_t* parts = static_cast<uint8_t*>(workspace) + kv4_decode_counter_bytes();
  const int64_t max_q = std::min(p->max_q, p->num_tokens);
  const bool few = max_q * a.group <= kDecodeRows;
  // Every CTA of either kernel goes through all the requests' lengths, so the requests are
  // taken kMaxReq at a time: 65536 single tokens in one launch took 335 ms, 2^20 would take a
  // minute and a half.
  int64_t r0 = 0;
  do {
    a.kv_lens = p->kv_lens + r0;
    a.cu_q = p->cu_q + r0;
    a.table = p->block_table + r0 * p->max_blocks;
    a.nreq = (int)std::min<int64_t>(p->nreq - r0, kMaxReq);
    a.pad = (r0 == 0 ? 1 : 0) | (r0 + a.nreq == p->nreq ? 2 : 0);
    a.max_rows = few ? 0x7fffffff : kDecodeRows;
    int rc;
    // mostly long chunks, or more work than the decode kernel can number: the prefill kernel
    // alone, which takes any; a mixed batch: each request by its kernel
    if ((!few && p->num_tokens * 4 >= p->nreq * max_q) || !kv4_decode_fits(a)) {
      a.max_rows = 0x7fffffff;
      rc = kv4_prefill(a, f16, 0, true, parts, st);
    } else {
      rc = kv4_decode(a, f16, workspace, parts, st);
      if (!rc && !few) rc = kv4_prefill(a, f16, kDecodeRows, false, parts, st);
    }
    if (rc) return rc;
    r0 += a.nreq;
  } while (r0 < p->nreq);
  return DIP_OK;
}
