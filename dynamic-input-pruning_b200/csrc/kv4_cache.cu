// kv4_cache.cu — keys and values into and out of the 4-bit paged cache.
//
//   append:  min = min_d x_d,  scale = round16((max_d x_d - min) / 15),
//            code_d = round((x_d - min) / scale), ties to even, at most 15
//   read:    x_d = round16(code_d * scale + min)
//
// min is exact in the 16-bit type (it is one of the inputs); the codes are
// taken against the ROUNDED scale, so the rounding of the scale costs no
// accuracy beyond the step itself.  A vector that holds an infinity or a NaN,
// or whose range overflows fp32, is stored as (NaN, NaN) and reads back as NaN.
// Both are bound by HBM and close behind it by issue, so a lane takes 16 channels of a
// row (two 16-byte words, half a row apart): what is done once a row is shared by them.
// A warp takes kKvBatch x 32 lanes of one token's key and value rows, all loads first.
// Measured, 65521 tokens, 8 heads of 128, bf16 (340 MB each way): append 88 us, 3.9 TB/s;
// read 58 us, 5.9 TB/s or 90 % of a measured 6.5 TB/s copy.  64 tokens: 2 us each, launch.
#include <cfloat>

#include "kv4_common.cuh"

namespace dip {

constexpr int kKvThreads = 256;
// Rows a lane.  Append and read of 65521 tokens with one 173 us, two 144, four 136 to 142;
// of 4093 tokens of 8 heads of 64, whose rows do not fill four, 13.3, 13.3 and 15.3.
constexpr int kKvBatch = 2;

__device__ __forceinline__ uint32_t kv4_min2(uint32_t a, uint32_t b, bool f16) {
  uint32_t r;  // NaN if either is
  if (f16) asm("min.NaN.f16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  else asm("min.NaN.bf16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// (lo, hi) -> two 16-bit values, one rounding each.
template <bool F16>
__device__ __forceinline__ uint32_t kv4_pack2(float lo, float hi) {
  uint32_t y;
  if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(y) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}

// x / y for finite x and y with y's reciprocal r in range: the product with the
// reciprocal and one correction by the exact remainder (Markstein 1990), which leaves a quotient
// that fp32 can hold (a tie between two codes is one) exact.
__device__ __forceinline__ float kv4_div(float x, float y, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, y, x), r, q);
}

// Codes of eight channels against (s, mn): adding magic rounds the quotient to an
// integer, ties to even, in the low bits of the sum.
template <bool F16>
__device__ __forceinline__ uint32_t kv4_codes(const uint4& raw, float s, float inv, float mn) {
  const float magic = 12582912.f;  // 1.5 * 2^23
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  uint32_t acc = 0;
  if (s >= 0x1p-100f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float q = kv4_div(h16_to_f32<F16>(i & 1 ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu) - mn, s, inv);
      if (F16) q = fminf(q, 15.f);  // a subnormal scale may be rounded down by half
      acc += __float_as_uint(q + magic) << (4 * i);
    }
    acc -= 0x4B400000u * 0x11111111u;  // the magic number's bits, shifted and summed
  } else {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const uint32_t p = i < 2 ? w[0] : i < 4 ? w[1] : i < 6 ? w[2] : w[3];
      const float x = h16_to_f32<F16>(i & 1 ? p >> 16 : p & 0xFFFFu);
      acc |= (uint32_t)fminf(rintf(__fdiv_rn(x - mn, s)), 15.f) << (4 * i);
    }
  }
  return acc;
}

// Item = (token, batch) of items = tokens * nb.
template <bool F16, int D>
__global__ void __launch_bounds__(kKvThreads)
kv4_append_kernel(const uint16_t* __restrict__ k, int64_t k_ts, int64_t k_hs,
                  const uint16_t* __restrict__ v, int64_t v_ts, int64_t v_hs,
                  const int64_t* __restrict__ slots, unsigned items, unsigned nb, Kv4Geom g,
                  uint8_t* __restrict__ cache) {
  constexpr int LPR = D / 16;      // lanes a row
  constexpr int RPW = 32 / LPR;    // rows a step of the warp
  const int lane = threadIdx.x & 31, sub = lane % LPR;
  const unsigned item = blockIdx.x * (kKvThreads / 32) + (threadIdx.x >> 5);
  pdl_wait();
  pdl_launch_dependents();
  if (item >= items) return;
  const unsigned t = item / nb;
  const int row0 = (int)(item - t * nb) * kKvBatch * RPW + lane / LPR;
  const int64_t slot = slots[t];
  uint4 raw[kKvBatch][2];
#pragma unroll
  for (int i = 0; i < kKvBatch; ++i) {  // rows: the heads' keys, then their values
    const int row = row0 + i * RPW;
    const bool is_v = row >= g.hkv;
    const int h = is_v ? row - g.hkv : row;
    if (row < 2 * g.hkv) {
      const uint16_t* src = (is_v ? v + t * v_ts + h * v_hs : k + t * k_ts + h * k_hs) + sub * 8;
      raw[i][0] = *reinterpret_cast<const uint4*>(src);
      raw[i][1] = *reinterpret_cast<const uint4*>(src + D / 2);
    }
  }
  const int64_t page = slot >> g.p_log2;
  if (slot < 0 || page >= g.num_pages) return;
  const int P = 1 << g.p_log2, off = (int)(slot & (P - 1));
  uint8_t* base = cache + page * g.hkv * g.page_bytes;
#pragma unroll
  for (int i = 0; i < kKvBatch; ++i) {
    const int row = row0 + i * RPW;
    const bool in = row < 2 * g.hkv, is_v = row >= g.hkv;
    const int h = is_v ? row - g.hkv : row;
    // (min, -max) of the row in one word: negated values' minimum is the maximum's negative
    uint32_t lo[2], hi[2];
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const uint4 w = raw[i][y];
      const uint32_t neg = 0x80008000u;
      lo[y] = kv4_min2(kv4_min2(w.x, w.y, F16), kv4_min2(w.z, w.w, F16), F16);
      hi[y] = kv4_min2(kv4_min2(w.x ^ neg, w.y ^ neg, F16), kv4_min2(w.z ^ neg, w.w ^ neg, F16), F16);
    }
    lo[0] = kv4_min2(lo[0], lo[1], F16);
    hi[0] = kv4_min2(hi[0], hi[1], F16);
    uint32_t m = kv4_min2(__byte_perm(lo[0], hi[0], 0x5410), __byte_perm(lo[0], hi[0], 0x7632), F16);
#pragma unroll
    for (int o = 1; o < LPR; o <<= 1) m = kv4_min2(m, __shfl_xor_sync(0xffffffffu, m, o), F16);
    const float mn = h16_to_f32<F16>(m & 0xFFFFu), mx = -h16_to_f32<F16>(m >> 16);
    const bool bad = !(mx - mn <= FLT_MAX);  // NaN, infinity or a range past fp32
    const uint32_t s16 = f32_to_h16<F16>(mx - mn >= 0x1p-90f ? kv4_div(mx - mn, 15.f, 1.f / 15.f)
                                                         : __fdiv_rn(mx - mn, 15.f));
    const float s = h16_to_f32<F16>(s16);
    uint32_t codes[2] = {0, 0};
    if (!bad && s > 0.f) {
      const float inv = __fdividef(1.f, s);
      codes[0] = kv4_codes<F16>(raw[i][0], s, inv, mn);
      codes[1] = kv4_codes<F16>(raw[i][1], s, inv, mn);
    }
    if (in) {
      uint8_t* part = base + h * g.page_bytes;
      uint32_t* dst = reinterpret_cast<uint32_t*>(part + (is_v ? P * (D / 2) : 0) + off * (D / 2)) + sub;
      dst[0] = codes[0];
      dst[D / 16] = codes[1];
      if (sub == 0) {
        const uint32_t pair = bad ? 0x7FFF7FFFu : (s16 | (m << 16));
        *reinterpret_cast<uint32_t*>(part + P * D + (is_v ? 4 * P : 0) + off * 4) = pair;
      }
    }
    __syncwarp();
  }
}

template <bool F16, int D>
__global__ void __launch_bounds__(kKvThreads)
kv4_read_kernel(const uint8_t* __restrict__ cache, const int64_t* __restrict__ slots, unsigned items,
                unsigned nb, Kv4Geom g, uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
  constexpr int LPR = D / 16, RPW = 32 / LPR;
  const int lane = threadIdx.x & 31, sub = lane % LPR;
  const unsigned item = blockIdx.x * (kKvThreads / 32) + (threadIdx.x >> 5);
  pdl_wait();
  pdl_launch_dependents();
  if (item >= items) return;
  const unsigned t = item / nb;
  const int row0 = (int)(item - t * nb) * kKvBatch * RPW + lane / LPR;
  const int64_t slot = slots[t], page = slot >> g.p_log2;
  const bool held = slot >= 0 && page < g.num_pages;
  const int P = 1 << g.p_log2, off = (int)(slot & (P - 1));
  const uint8_t* base = cache + (held ? page : 0) * g.hkv * g.page_bytes;
  uint32_t codes[kKvBatch][2], pair[kKvBatch];
#pragma unroll
  for (int i = 0; i < kKvBatch; ++i) {
    const int row = row0 + i * RPW;
    const bool is_v = row >= g.hkv;
    codes[i][0] = codes[i][1] = pair[i] = 0;  // a slot outside the cache reads as zeros
    if (held && row < 2 * g.hkv) {
      const uint8_t* part = base + (is_v ? row - g.hkv : row) * g.page_bytes;
      const uint32_t* src = reinterpret_cast<const uint32_t*>(part + (is_v ? P * (D / 2) : 0) + off * (D / 2)) + sub;
      codes[i][0] = src[0];
      codes[i][1] = src[D / 16];
      pair[i] = *reinterpret_cast<const uint32_t*>(part + P * D + (is_v ? 4 * P : 0) + off * 4);
    }
  }
#pragma unroll
  for (int i = 0; i < kKvBatch; ++i) {
    const int row = row0 + i * RPW;
    if (row < 2 * g.hkv) {
      const bool is_v = row >= g.hkv;
      const float s = h16_to_f32<F16>(pair[i] & 0xFFFFu), m = h16_to_f32<F16>(pair[i] >> 16);
      uint16_t* dst = (is_v ? v : k) + ((int64_t)t * g.hkv + (is_v ? row - g.hkv : row)) * D + sub * 8;
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t even = codes[i][y] & 0x0F0F0F0Fu, odd = (codes[i][y] >> 4) & 0x0F0F0F0Fu;
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // 2^23 + code, exact; byte e holds channels 2 e and 2 e + 1
          const float a = __uint_as_float(__byte_perm(even, kF32Magic, 0x7540 + e)) - 8388608.f;
          const float b = __uint_as_float(__byte_perm(odd, kF32Magic, 0x7540 + e)) - 8388608.f;
          w[e] = kv4_pack2<F16>(fmaf(a, s, m), fmaf(b, s, m));
        }
        *reinterpret_cast<uint4*>(dst + y * (D / 2)) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
}

// Batches a token, and warps in all.
static unsigned kv4_batches(int hkv, int d) {
  const int rows = kKvBatch * 32 / (d / 16);
  return (unsigned)((2 * hkv + rows - 1) / rows);
}

static int kv4_check(int64_t tokens, int64_t hkv, int64_t d, int dtype, const void* cache,
                     int64_t num_pages, int64_t page, Kv4Geom* g) {
  if (tokens < 0 || hkv < 1 || num_pages < 0 || (dtype != DIP_BF16 && dtype != DIP_FP16))
    return DIP_ERR_ARG;
  if (kv4_page_log2(page) < 0 || (d != 64 && d != 128) || hkv > 65535) return DIP_ERR_UNSUPPORTED;
  if (tokens > 0 && num_pages > 0 && (!cache || !aligned16(cache))) return DIP_ERR_ARG;
  if (tokens > 0 && tokens > 0xffffffffLL / kv4_batches((int)hkv, (int)d) - 8) return DIP_ERR_UNSUPPORTED;
  *g = {(int)hkv, (int)d, kv4_page_log2(page), kv4_part_bytes(page, d), num_pages};
  return DIP_OK;
}

static dim3 kv4_grid(int64_t items) {
  return dim3((unsigned)((items + kKvThreads / 32 - 1) / (kKvThreads / 32)));
}

}  // namespace dip

using namespace dip;

extern "C" size_t dip_kv4_page_bytes(int64_t page_size, int64_t head_dim) {
  if (kv4_page_log2(page_size) < 0 || (head_dim != 64 && head_dim != 128)) return 0;
  return (size_t)kv4_part_bytes(page_size, head_dim);
}

extern "C" int dip_kv4_append(const void* k, int64_t k_token_stride, int64_t k_head_stride,
                              const void* v, int64_t v_token_stride, int64_t v_head_stride,
                              const int64_t* slots, int64_t num_tokens, int64_t kv_heads,
                              int64_t head_dim, int dtype, void* cache, int64_t num_pages,
                              int64_t page_size, dip_stream_t stream) {
  Kv4Geom g;
  const int st = kv4_check(num_tokens, kv_heads, head_dim, dtype, cache, num_pages, page_size, &g);
  if (st) return st;
  if (num_tokens == 0 || num_pages == 0) return DIP_OK;
  if (!k || !v || !slots || !aligned16(k) || !aligned16(v)) return DIP_ERR_ARG;
  if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) return DIP_ERR_ARG;
  const unsigned nb = kv4_batches(g.hkv, g.d);
  const unsigned items = (unsigned)(num_tokens * nb);
  auto go = [&](auto kern) {
    return launch_status(launch(kern, kv4_grid(items), dim3(kKvThreads), 0,
                                (cudaStream_t)stream, (const uint16_t*)k, k_token_stride,
                                k_head_stride, (const uint16_t*)v, v_token_stride, v_head_stride,
                                slots, items, nb, g, (uint8_t*)cache));
  };
  if (dtype == DIP_FP16)
    return g.d == 64 ? go(kv4_append_kernel<true, 64>) : go(kv4_append_kernel<true, 128>);
  return g.d == 64 ? go(kv4_append_kernel<false, 64>) : go(kv4_append_kernel<false, 128>);
}

extern "C" int dip_kv4_read(const void* cache, int64_t num_pages, int64_t page_size,
                            const int64_t* slots, int64_t num_tokens, int64_t kv_heads,
                            int64_t head_dim, int dtype, void* k, void* v, dip_stream_t stream) {
  Kv4Geom g;
  const int st = kv4_check(num_tokens, kv_heads, head_dim, dtype, cache, num_pages, page_size, &g);
  if (st) return st;
  if (num_tokens == 0) return DIP_OK;
  if (!k || !v || !slots || !aligned16(k) || !aligned16(v)) return DIP_ERR_ARG;
  const unsigned nb = kv4_batches(g.hkv, g.d);
  const unsigned items = (unsigned)(num_tokens * nb);
  auto go = [&](auto kern) {
    return launch_status(launch(kern, kv4_grid(items), dim3(kKvThreads), 0,
                                (cudaStream_t)stream, (const uint8_t*)cache, slots, items, nb, g,
                                (uint16_t*)k, (uint16_t*)v));
  };
  if (dtype == DIP_FP16)
    return g.d == 64 ? go(kv4_read_kernel<true, 64>) : go(kv4_read_kernel<true, 128>);
  return g.d == 64 ? go(kv4_read_kernel<false, 64>) : go(kv4_read_kernel<false, 128>);
}
