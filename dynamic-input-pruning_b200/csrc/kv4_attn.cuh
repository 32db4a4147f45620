// kv4_attn.cuh — what the attention kernels over the 4-bit paged cache share.
#pragma once
#include <atomic>

#include "kv4_common.cuh"

namespace dip {

struct AttnArgs {
  const uint16_t* q;
  int64_t q_ts, q_hs;
  const uint8_t* cache;
  Kv4Geom g;
  const int32_t* table;
  int64_t max_blocks;
  const int32_t* kv_lens;
  const int32_t* cu_q;
  int nreq;
  int num_tokens;
  int heads, group, causal;
  float scale;
  uint16_t* out;
  float* lse;
  unsigned* err;
  int max_rows;   // decode kernel: requests with more query rows a KV head are left out
  int pad;        // tokens of no request that are zeroed: 1 those before the requests', 2 those after
};

constexpr int kMaxReq = 8192;       // requests a launch
constexpr int kMaxKv = 0x7fff0000;  // token numbers past a context's end stay 32-bit

// Raises a kernel's dynamic shared memory limit, once a device.
template <auto kern>
inline cudaError_t attn_smem(int bytes) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  const cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
  const cudaError_t r = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (r == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return r;
}

// Request r: first query token, query tokens (clamped to the call's), visible cache length.
struct AttnReq {
  int tok0, n, kv;
  bool bad;  // cu_q descends: the sums of n that both kernels count with are not bounded then
};
__device__ __forceinline__ AttnReq attn_req(const AttnArgs& a, int r) {
  AttnReq q;
  q.tok0 = max(a.cu_q[r], 0);
  q.n = max(min(a.cu_q[r + 1], a.num_tokens) - q.tok0, 0);
  q.bad = a.cu_q[r + 1] < a.cu_q[r];
  q.kv = (int)min((int64_t)min(max(a.kv_lens[r], 0), kMaxKv), a.max_blocks << a.g.p_log2);
  return q;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// Tokens of no request, before the first one's and after the last one's: [0, first) and
// [last, num_tokens).
struct AttnPad {
  int first, last;
};
__device__ __forceinline__ AttnPad attn_pad(const AttnArgs& a) {
  if (a.nreq == 0) return {0, 0};
  const int first = min(max(a.cu_q[0], 0), a.num_tokens);
  const int last = max(min(a.cu_q[a.nreq], a.num_tokens), first);
  return {a.pad & 1 ? first : 0, a.pad & 2 ? last : a.num_tokens};
}
// Their zeros and -inf, by the whole grid.
template <int D>
__device__ __forceinline__ void attn_zero_pad(const AttnArgs& a, const AttnPad& pad, int threads) {
  const int n = pad.first + (a.num_tokens - pad.last);
  for (int x = blockIdx.x; x < n; x += gridDim.x) {
    const int64_t t = x < pad.first ? x : pad.last + (x - pad.first);
    for (int i = threadIdx.x; i < a.heads * D / 8; i += threads)
      reinterpret_cast<uint4*>(a.out + t * a.heads * D)[i] = make_uint4(0, 0, 0, 0);
    if (a.lse)
      for (int i = threadIdx.x; i < a.heads; i += threads) a.lse[t * a.heads + i] = -INFINITY;
  }
}

bool kv4_decode_fits(const AttnArgs& a);
int kv4_decode(const AttnArgs& a, bool f16, void* counters, void* parts, cudaStream_t st);
size_t kv4_decode_counter_bytes();
size_t kv4_decode_part_bytes();
// Requests with more than min_rows query rows a KV head; zero_pad: also the tokens of no request.
int kv4_prefill(const AttnArgs& a, bool f16, int min_rows, bool zero_pad, void* parts, cudaStream_t st);
size_t kv4_prefill_part_bytes();

// As mbar_wait with the poll limit already read (spin_limit is a load from global memory).
__device__ __forceinline__ bool mbar_wait_lim(uint64_t* bar, uint32_t parity, uint32_t limit,
                                              unsigned* err) {
  for (uint32_t i = 0; i < limit; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  atomicOr(err, kErrTimeout);
  return false;
}

// For copies and products that are on their way when a wait has run out: they write to, or
// read, memory that is another block's after this one's exit, so they are waited for with
// the library's own limit, whatever the caller set.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < kSpinLimit; ++i)
    if (mbar_try_wait(bar, parity)) return;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The weights p scale_V are held in fp16, against a reference that puts the largest near
// 2^kPeak when it moves, which it does when one reaches 2^15.  Below 2^-14 fp16 loses bits
// and below 2^-25 all of them, while the sums l and b keep the whole p: a weight is off by
// 2^-25 at most, n of them by n 2^-25 against a largest of 2^(kPeak - 1) or more, so the
// result by n 2^-27 of the largest weight's scale_V (codes within 8 of the middle), 2^-10
// of a quantisation step behind 131072 tokens.  With the largest at 2^-8, all of fp16 from
// 1 up idle, an attention sink 12 nats above 131072 others lost a third of the output.
constexpr float kPeak = 6.f;
// Scale a value row's weight is taken with: its own, but with room for the sums where it is
// 0 (equal values, whose codes are 0: any scale stands for them) or next to it.  p stays
// below 2^95, p min below 2^35.
constexpr float kScaleMin = 0x1p-80f;
__device__ __forceinline__ float weight_scale(float s, float mn) {
  return fmaxf(fmaxf(s, fabsf(mn) * 0x1p-20f), kScaleMin);
}
// Largest of weights (two a word, none negative), and whether one reached 2^15 (or is not
// finite).
__device__ __forceinline__ uint32_t weight_max(uint32_t m, uint32_t a, uint32_t b) {
  return __vimax3_u16x2(m, a, b);
}
__device__ __forceinline__ bool weight_high(uint32_t m) { return ((m + 0x08000800u) & 0x80008000u) != 0; }

}  // namespace dip
