// kv4_decode.cu — attention over the 4-bit paged cache for few query rows:
// decode (one token a request) and short verification chunks.
//
// The query rows of one request that share a KV head are N-columns of the
// tensor-core products, the cache rows their M (K = channels, then tokens), so
// codes enter as the A operand straight from the packed words:
//   S^T[token, row] = sum_d code_K[token, d] q[row, d]
//   s = scale_K * S^T + min_K * sum_d q,     p = 2^(c s - m)
//   O^T[d, row]     = sum_token (code_V - 8)[token, d] (p scale_V)[token, row]
//   out = (O + sum p (min_V + 8 scale_V)) / sum p
// (codes about zero, so that the rounding of a weight weighs no more than its value:
// the -8 comes from the sum of the rounded weights).
// A code 0..15 left in the low bits of a 16-bit lane IS the fp16 subnormal
// code * 2^-24 (its neighbour nibble, masked in place, code * 2^-20), which the
// tensor cores multiply exactly: one AND for two codes, no bias to subtract.
// The powers of two go into q (and its row's softmax factor) and into O's rows.
// q is held in fp16 scaled by a power of two a row (exact for bf16 and fp16
// elements down to 2^-24 of the row's largest).  The reference M of a row's
// exponentials is not the largest score but the largest c s + log2 scale_V, less
// kPeak: the weights p scale_V that enter the second product in fp16 peak near
// 2^kPeak whatever the values' size, and M, l = sum p, b = sum p (min_V + 8 scale_V) and O are
// rescaled only when a weight reaches 2^15: a maximum of the packed weights and a vote a
// unit, and no reduction over lanes on the usual path.  (What fp16 loses of small weights:
// at kPeak.)  Sums, statistics, pairs and accumulators are fp32.
//
// Work: the (request, KV head, row block) items are cut into units of 64 cache
// tokens and laid end to end, each item led by kOvh units that stand for its fixed
// cost; every warp takes an equal contiguous stretch, so ragged and single long
// contexts fill the GPU alike, and runs through it on its own: there is no barrier
// between the segments of a stretch.  An item inside one stretch is written
// directly.  The parts of a split item are (m, l, b, O): a warp's last segment is
// joined with its neighbours' of the same item in shared memory when the CTA is
// done, a tail (the part with the item's end) goes to the workspace at once, and
// the CTA that completes an item's count of parts joins them in fixed order.
// Bound by HBM (0.53 bytes a cached element); every warp streams its own units into
// a ring of shared memory, one bulk copy a page (a page of one head is contiguous).
// Measured, 64/8 heads of 128, bf16: one context of 131071 tokens 44 us, 3.3 TB/s or 50 %
// of a measured copy (the stream itself 25 us, 5.7 TB/s; the rest plan, first units and the
// joins); 64 contexts of 17 to 16384 44 us; one of 700 10 us with the launch.  256 contexts
// of 1 to 2048, 8 heads of 64, fp16: 30 us, by the items' fixed latency.  16 x 5 tokens of
// 40/8 heads behind 900 to 9000: 56 us, by unpacking for each of four row blocks.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kv4_attn.cuh"

namespace dip {

constexpr int kUnit = 64;        // cache tokens a unit
constexpr int kOvh = 2;          // an item's fixed cost in units (queries, first reference, result)
constexpr int kDecFineReq = 2048;  // requests with a prefix sum each; above, every fourth has one
constexpr int kDecInfoReq = 1024;  // requests whose lengths are kept in shared memory
constexpr float kNone = -1e30f;     // reference of a row that has seen no position

template <int D>
struct DecCfg {
  // Query rows a block, the tensor cores' N.  Two N-tiles a warp halve the reads and the
  // unpacking of more rows, but take the registers of a second accumulator: 25 rows over
  // 16 contexts of 900 to 9000 tokens 76 us against 59 us for four blocks of eight.
  static constexpr int rows = 8;
  static constexpr int W = 12;                         // warps (168 registers a thread)
  static constexpr int threads = W * 32;
  static constexpr int S = D == 128 ? 2 : 3;           // ring stages a warp
  static constexpr int stage = kUnit * (D + 8);
  static constexpr int slot = rows * (D + 4);          // floats of a part: row (m, l, b, -, O)
  // open parts, scan, finishes | barriers | next chunks | lengths | prefix sums | rings (also slots)
  static constexpr int o_bar = 1280;
  static_assert((3 * W * 8 + 1) * 4 <= o_bar, "tables");
  static constexpr int o_next = o_bar + W * S * 8;
  static constexpr int o_info = o_next + W * 64;
  static int o_ring(int nreq) {
    return (o_info + std::min(nreq, kDecInfoReq) * 12 + std::min(nreq + 1, kDecFineReq + 1) * 4 + 127) & ~127;
  }
  static int smem(int nreq) { return o_ring(nreq) + W * S * stage; }
  static_assert(S * stage >= slot * 4, "a part fits a ring");
  static_assert(o_info + kDecInfoReq * 12 + (kDecFineReq + 1) * 4 + 128 + W * S * stage <= 227 * 1024,
                "shared memory");
};

__device__ __forceinline__ uint32_t movmatrix_t(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
template <bool F16>
__device__ __forceinline__ void pair_f32(uint32_t p, float& s, float& m) {
  if (F16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p));
    s = f.x;
    m = f.y;
  } else {
    s = __uint_as_float(p << 16);
    m = __uint_as_float(p & 0xFFFF0000u);
  }
}
// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// A stretch's piece of one item.
struct DecSeg {
  int r, h, row0;     // request, KV head, first row of the block
  int tok0, n, kv;    // first query token, query tokens, cache length
  int u0, cnt, nu;    // first unit here, units here, units of the item
  int base;           // position of the item's first unit
  int next;           // position of the following segment
};

__device__ __forceinline__ int dec_units(int kv) { return max((kv + kUnit - 1) / kUnit, 1); }

struct DecShared {
  const int* pre;     // positions of the first items of requests 0, 1 << gs, 2 << gs, ...
  const int* info;    // [min(nreq, kDecInfoReq)][3]: tok0, n, kv
  int gs;
  bool few;           // a position a warp: items start at CTA boundaries
};

// Positions an item of nu units takes, and those before its first unit.
template <int D>
__device__ __forceinline__ int dec_len(bool few, int nu) {
  constexpr int W = DecCfg<D>::W;
  return few ? (nu + W - 1) / W * W : nu + kOvh;
}
__device__ __forceinline__ int dec_lead(bool few) { return few ? 0 : kOvh; }

template <int D>
__device__ __forceinline__ int dec_blocks(const AttnArgs& a, int n) {
  const int rows = n * a.group;  // requests with more rows are another kernel's
  return rows > a.max_rows ? 0 : (rows + DecCfg<D>::rows - 1) / DecCfg<D>::rows;
}

// Request r's lengths.
__device__ __forceinline__ void dec_request(const AttnArgs& a, const DecShared& sh, int r, DecSeg& s) {
  s.r = r;
  if (r < kDecInfoReq) {
    s.tok0 = sh.info[3 * r];
    s.n = sh.info[3 * r + 1];
    s.kv = sh.info[3 * r + 2];
  } else {
    const AttnReq q = attn_req(a, r);
    s.tok0 = q.tok0;
    s.n = q.n;
    s.kv = q.kv;
  }
  s.nu = dec_units(s.kv);
}

// The segment at position pos of a stretch that ends at `end`; cnt = 0: none is left.
template <int D>
__device__ __forceinline__ DecSeg dec_seg(const AttnArgs& a, const DecShared& sh, int pos, int end) {
  int lo = 0, hi = (a.nreq + (1 << sh.gs) - 1) >> sh.gs;  // largest entry with pre <= pos
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (sh.pre[m] <= pos) lo = m; else hi = m;
  }
  DecSeg s;
  int base = sh.pre[lo], blocks;
  for (int r = lo << sh.gs;; ++r) {
    dec_request(a, sh, r, s);
    blocks = dec_blocks<D>(a, s.n);
    const int cost = dec_len<D>(sh.few, s.nu) * blocks * a.g.hkv;
    if (sh.gs == 0 || pos < base + cost || r + 1 >= a.nreq) break;
    base += cost;
  }
  const int rel = pos - base;
  const int len = dec_len<D>(sh.few, s.nu);
  const int item = rel / len;
  s.h = item / blocks;
  s.row0 = (item - s.h * blocks) * DecCfg<D>::rows;
  s.base = base + item * len + dec_lead(sh.few);
  s.u0 = max(pos - s.base, 0);
  s.cnt = max(min(s.nu, end - s.base) - s.u0, 0);
  s.next = base + (item + 1) * len;
  return s;
}

// The segment after s in the stretch (s.next < end): the items follow one another, so
// no search and no division.
template <int D>
__device__ __forceinline__ void dec_step(const AttnArgs& a, const DecShared& sh, DecSeg& s, int end) {
  s.row0 += DecCfg<D>::rows;
  if (s.row0 >= s.n * a.group) {
    s.row0 = 0;
    if (++s.h == a.g.hkv) {
      s.h = 0;
      do {
        dec_request(a, sh, ++s.r, s);
      } while (dec_blocks<D>(a, s.n) == 0);
    }
  }
  s.base = s.next + dec_lead(sh.few);
  s.u0 = 0;
  s.cnt = max(min(s.nu, end - s.base), 0);
  s.next += dec_len<D>(sh.few, s.nu);
}

// Joined part -> out and lse: four channels of one row.
template <bool F16, int D>
__device__ __forceinline__ void dec_store(const AttnArgs& a, const DecSeg& s, int row, int d4,
                                          float top, float l, float b, float4 o) {
  const int rw = s.row0 + row, i = rw / a.group;
  const int64_t at = (int64_t)(s.tok0 + i) * a.heads + s.h * a.group + (rw - i * a.group);
  const float inv = top == -INFINITY ? 0.f : 1.f / l;
  uint2 v;
  v.x = f32_to_h16<F16>((o.x + b) * inv) | (f32_to_h16<F16>((o.y + b) * inv) << 16);
  v.y = f32_to_h16<F16>((o.z + b) * inv) | (f32_to_h16<F16>((o.w + b) * inv) << 16);
  *reinterpret_cast<uint2*>(a.out + at * D + d4 * 4) = v;
  if (a.lse && d4 == 0) a.lse[at] = top == -INFINITY ? -INFINITY : top * kLn2 + logf(l);
}

// Joins np parts of one (row, four channels), twelve at a time so that their loads
// overlap; src(c) is the row's start in part c.
template <class SRC>
__device__ __forceinline__ float4 dec_join(int np, int d4, SRC src, float& top, float& l, float& b) {
  constexpr int N = 12;
  top = -INFINITY;
  l = b = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int c0 = 0; c0 < np; c0 += N) {
    float4 h[N], v[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c0 + i < np) {
        const float* p = src(c0 + i);
        h[i] = *reinterpret_cast<const float4*>(p);
        v[i] = *reinterpret_cast<const float4*>(p + 4 + d4 * 4);
      } else {
        h[i] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
        v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    float nt = top;
#pragma unroll
    for (int i = 0; i < N; ++i) nt = fmaxf(nt, h[i].x);
    const float ref = nt == -INFINITY ? 0.f : nt;
    const float f = ex2(top - ref);
    l *= f; b *= f;
    o.x *= f; o.y *= f; o.z *= f; o.w *= f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float g = ex2(h[i].x - ref);
      l = fmaf(h[i].y, g, l);
      b = fmaf(h[i].z, g, b);
      o.x = fmaf(v[i].x, g, o.x);
      o.y = fmaf(v[i].y, g, o.y);
      o.z = fmaf(v[i].z, g, o.z);
      o.w = fmaf(v[i].w, g, o.w);
    }
    top = nt;
  }
  return o;
}

__device__ __forceinline__ int dec_expected(int c0, int c1, int w) { return (c1 - 1) / w - c0 / w + 2; }

template <bool F16, int D>
__global__ void __launch_bounds__(DecCfg<D>::threads, 1)
kv4_decode_kernel(const AttnArgs a, int o_ring, unsigned* __restrict__ counters, float* runs, float* tails) {
  using C = DecCfg<D>;
  constexpr int W = C::W, S = C::S;
  extern __shared__ __align__(128) uint8_t smem[];
  int* desc = reinterpret_cast<int*>(smem);  // [W][8] a warp's open part: base, nu, n, tok0, h, row0
  int* fin = desc + W * 8;                   // [2 W][8] items to finish, the same fields
  int* scan = fin + 2 * W * 8 - 128;         // (before any finish)
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::o_bar) + (threadIdx.x >> 5) * S;
  int* nx = reinterpret_cast<int*>(smem + C::o_next) + (threadIdx.x >> 5) * 16;
  int* info = reinterpret_cast<int*>(smem + C::o_info);
  int* pre = info + min(a.nreq, kDecInfoReq) * 3;
  int* nfin = fin + 2 * W * 8;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < S; ++i) mbar_init(&full[i], 1);
    mbar_fence_init();
  }
  if (tid == 0) *nfin = 0;
  pdl_wait();
  const uint32_t limit = spin_limit(a.err);  // read once, not in every wait
  AttnPad pad = attn_pad(a);
  // ---------------------------------------------------------------- plan
  // exclusive prefix sums of the requests' costs: each thread a run of requests
  const int gs = a.nreq > kDecFineReq ? 2 : 0;
  const int per = (((a.nreq + C::threads - 1) / C::threads) + (1 << gs) - 1) >> gs << gs;
  int sum = 0, aligned = 0;  // costs in the two ways of laying the items out
  bool bad_cu = false;
  for (int i = 0; i < per; ++i) {
    const int r = tid * per + i;
    if (r < a.nreq) {
      const AttnReq q = attn_req(a, r);
      bad_cu |= q.bad;
      if (r < kDecInfoReq) {
        info[3 * r] = q.tok0;
        info[3 * r + 1] = q.n;
        info[3 * r + 2] = q.kv;
      }
      const int items = dec_blocks<D>(a, q.n) * a.g.hkv, nu = dec_units(q.kv);
      sum += dec_len<D>(false, nu) * items;
      aligned += (int)min((long long)dec_len<D>(true, nu) * items, 1LL << 16);
    }
  }
  int inc = sum, inc2 = aligned;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o), t2 = __shfl_up_sync(0xffffffffu, inc2, o);
    if (lane >= o) {
      inc += t;
      inc2 += t2;
    }
  }
  if (lane == 31) {
    scan[warp] = inc;
    scan[16 + warp] = inc2;
  }
  bad_cu = __syncthreads_or(bad_cu);
  int before = inc - sum, before2 = inc2 - aligned, total = 0, total2 = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int t = scan[w], t2 = scan[16 + w];
    if (w < warp) {
      before += t;
      before2 += t2;
    }
    total += t;
    total2 += t2;
  }
  // Few units: one a warp, and items that start at CTA boundaries, so that those of up to
  // W units are joined without leaving their CTA.
  const int workers = (int)gridDim.x * W;
  const DecShared sh = {pre, info, gs, total2 <= workers};
  if (sh.few) {
    before = before2;
    total = total2;
  }
  if (bad_cu) {  // no work, all tokens zeros
    total = 0;
    pad = {0, 0};
    if (blockIdx.x == 0 && tid == 0) atomicOr(a.err, kErrInput);
  }
  const int share = max((total + workers - 1) / workers, 1);
  for (int i = 0; i < per; ++i) {
    const int r = tid * per + i;
    if (r < a.nreq) {
      if ((r & ((1 << gs) - 1)) == 0) pre[r >> gs] = before;
      if (per > 1) {
        DecSeg q;
        dec_request(a, sh, r, q);
        before += dec_len<D>(sh.few, q.nu) * dec_blocks<D>(a, q.n) * a.g.hkv;
      }
    }
  }
  __syncthreads();
  pdl_launch_dependents();

  const int worker = blockIdx.x * W + warp;
  const int first = (int)min((int64_t)worker * share, (int64_t)total), end = min(first + share, total);
  uint8_t* ring = smem + o_ring + warp * (S * C::stage);

  // ---------------------------------------------------------------- feeding the ring
  // A chunk is a run of units of one segment within 32 pages, lane i holding the
  // table entry of its page i.  The next chunk's entries are loaded while this one
  // is fed, so no entry's latency stands between two units.  The walk's state is
  // the same for all lanes and kept in shared memory:
  //   nx: 0 next unit, 1 segment's end, 2.. the segment (r, h, row0, tok0, n, kv, nu, next) |
  //       the next chunk: 12 first unit, 13 end, 14 head, 15 kv
  const int pl = a.g.p_log2, P = 1 << pl;
  int f_u = 0, f_end = 0, f_h = 0, f_kv = 0, f_page = 0;  // the chunk being fed
  int ent = -1, ent_nx = -1;
  auto enter = [&](const DecSeg& s) {  // the walk enters a segment
    nx[0] = s.u0;
    nx[1] = s.u0 + s.cnt;
    nx[2] = s.r;
    nx[3] = s.h;
    nx[4] = s.row0;
    nx[5] = s.tok0;
    nx[6] = s.n;
    nx[7] = s.kv;
    nx[8] = s.nu;
    nx[9] = s.next;
    __syncwarp();
  };
  auto walk = [&]() {  // loads the next chunk; empty (12 == 13): the stretch is done
    if (nx[0] == nx[1] && nx[9] < end) {
      DecSeg s;
      s.r = nx[2]; s.h = nx[3]; s.row0 = nx[4]; s.tok0 = nx[5]; s.n = nx[6]; s.kv = nx[7]; s.nu = nx[8];
      s.next = nx[9];
      __syncwarp();
      dec_step<D>(a, sh, s, end);
      enter(s);
    }
    const int su = nx[0], send = nx[1], h = nx[3], kv = nx[7];
    const int p0 = (su * kUnit) >> pl;
    const int ue = min(send, ((p0 + 32) << pl) / kUnit);
    const int last = (kv - 1) >> pl;  // the context's last page (-1: none)
    ent_nx = su < send && p0 + lane <= last ? a.table[(int64_t)nx[2] * a.max_blocks + p0 + lane] : -1;
    __syncwarp();
    nx[0] = ue;
    nx[12] = su;
    nx[13] = ue;
    nx[14] = h;
    nx[15] = kv;
    __syncwarp();
  };
  auto take = [&]() {  // the next chunk becomes the one being fed
    f_u = nx[12];
    f_end = nx[13];
    f_h = nx[14];
    f_kv = nx[15];
    f_page = (f_u * kUnit) >> pl;
    ent = ent_nx;
    __syncwarp();
  };
  uint32_t badbits = 0;  // four bits a stage: pieces whose page is outside the cache
  const int tp = min(P, kUnit), np = kUnit / tp;  // tokens a piece, pieces a unit
  const int part_bytes = tp * (D + 8);
  int ahead = 0;       // units asked for and not yet waited for
  bool dead = false;   // a wait ran out: nothing is loaded any more, the parts are still joined
  auto feed = [&](int st) {
    if (f_u >= f_end || dead) return;
    ++ahead;
    const int t0 = f_u * kUnit;
    const int e = __shfl_sync(0xffffffffu, ent, ((t0 >> pl) - f_page) + (lane & (np - 1)));
    const bool inside = lane < np && t0 + lane * tp < f_kv;
    const bool ok = inside && e >= 0 && e < a.g.num_pages;
    const uint32_t okm = __ballot_sync(0xffffffffu, ok), bad = __ballot_sync(0xffffffffu, inside && !ok);
    badbits = (badbits & ~(15u << (4 * st))) | (bad << (4 * st));
    if (lane == 0) mbar_arrive_expect_tx(&full[st], __popc(okm) * part_bytes);
    __syncwarp();
    uint8_t* dst = ring + st * C::stage;
    const uint8_t* src = a.cache + ((int64_t)e * a.g.hkv + f_h) * a.g.page_bytes;
    if (P <= kUnit) {
      if (ok) bulk_g2s(dst + lane * part_bytes, src, part_bytes, &full[st]);
    } else if (okm && lane < 4) {  // half a page: a lane each for K, V codes, K, V pairs
      // (with np = 1 every lane holds the page's entry)
      const int half = t0 & (P - 1), pair = lane >> 1, isv = lane & 1;
      const int rb = pair ? 4 : D / 2;
      bulk_g2s(dst + (pair ? kUnit * D : 0) + isv * kUnit * rb,
               src + (pair ? P * D : 0) + isv * P * rb + half * rb, kUnit * rb, &full[st]);
    }
    if (++f_u == f_end) {
      take();
      walk();
    }
  };

  constexpr int KW = D / 32;   // packed words a lane and cache row (K), 2 MMA steps each
  constexpr int MT = D / 16;   // m-tiles of O^T
  constexpr int TT = kUnit / 16;  // tiles of 16 tokens
  const int lr = lane >> 2, lc = lane & 3;
  const int tau = lr ^ ((lr >> 1) & 1);  // cache row of MMA row lr (bank-conflict-free order)
  const int tpl = min(pl, 6);
  int st = 0;
  uint32_t par = 0;
  int fed = 0;  // 1: the first segment's units are on their way
  bool open = false;  // the last segment ends before its item does
  // Row lr of a block's queries; null past the request's rows.
  auto q_row = [&](const DecSeg& s, int x) -> const uint16_t* {
    const int row = s.row0 + x;
    if (row >= s.n * a.group) return nullptr;
    const int i = row / a.group;
    return a.q + (int64_t)(s.tok0 + i) * a.q_ts + (int64_t)(s.h * a.group + row - i * a.group) * a.q_hs;
  };
  DecSeg s = {};
  if (first < end) s = dec_seg<D>(a, sh, first, end);
  while (s.cnt > 0) {
    const int rows_all = s.n * a.group;
    if (!fed) {
      enter(s);
      walk();
    }

    // q as B operand, fp16 scaled by 2^qe a row; the hi-nibble channels by 1/16 more
    uint32_t qf[KW * 4];
    float qsum[2], cf[2];
    int lim[2];
    int minlim = s.kv;
    bool huge;  // queries so large that 2^24 of their rows' factors is taken by the scores
    uint4 raw[KW];
    const uint16_t* qsrc = q_row(s, lr);
#pragma unroll
    for (int w = 0; w < KW; ++w)
      raw[w] = qsrc ? *reinterpret_cast<const uint4*>(qsrc + lc * (KW * 8) + w * 8) : make_uint4(0, 0, 0, 0);
    if (!fed) {  // the first queries are asked for before the stream that would hold them up
      fed = 1;
      take();
      if (f_end - f_u >= S) {  // no chunk ends in these: the next one's entries can wait
#pragma unroll
        for (int i = 0; i < S - 1; ++i) feed(i);
        walk();
      } else {
        walk();
#pragma unroll
        for (int i = 0; i < S - 1; ++i) feed(i);
      }
    }
    {
      float f[KW * 8];
      float mx = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const uint32_t x[4] = {raw[w].x, raw[w].y, raw[w].z, raw[w].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[w * 8 + 2 * j] = h16_to_f32<F16>(x[j] & 0xFFFFu);
          f[w * 8 + 2 * j + 1] = h16_to_f32<F16>(x[j] >> 16);
          mx = fmaxf(mx, fmaxf(fabsf(f[w * 8 + 2 * j]), fabsf(f[w * 8 + 2 * j + 1])));
        }
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      // largest |q| to [2^13, 2^14): products with codes up to 15 * 2^-20 stay small
      const int ex = (int)((__float_as_uint(mx) >> 23) & 255u) - 127;
      const int qe = mx > 0.f && ex < 128 ? min(max(13 - ex, -114), 126) : 0;
      float sg = pow2i(qe);
      if (a.scale < 0.f) sg = -sg;
      if (a.scale == 0.f) sg = 0.f;
      float sum_q = 0.f;
#pragma unroll
      for (int w = 0; w < KW; ++w)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // step 2w: (n0, n4) and (n1, n5); step 2w + 1: (n2, n6) and (n3, n7)
          float lo = f[w * 8 + j] * sg, hi = f[w * 8 + j + 4] * sg;
          if (j & 1) { lo *= 0.0625f; hi *= 0.0625f; }
          const uint32_t p = pack_h2(lo, hi);
          qf[w * 4 + j] = p;
          const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&p));
          sum_q += (b.x + b.y) * ((j & 1) ? 16.f : 1.f);
        }
      sum_q += __shfl_xor_sync(0xffffffffu, sum_q, 1);
      sum_q += __shfl_xor_sync(0xffffffffu, sum_q, 2);
      // the rows of this lane's accumulator columns: 2 lc and 2 lc + 1
      huge = __any_sync(0xffffffffu, qe < -90);
      const float c_row = fmaxf(fabsf(a.scale) * kLog2e * pow2i(-qe) * (huge ? 1.f : 0x1p24f), FLT_MIN);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        qsum[e] = __shfl_sync(0xffffffffu, sum_q, (2 * lc + e) * 4) * 0x1p-24f;
        cf[e] = __shfl_sync(0xffffffffu, a.scale == 0.f ? 1.f : c_row, (2 * lc + e) * 4);
        const int rw = s.row0 + 2 * lc + e;
        int l = s.kv;
        if (a.causal && rw < rows_all) l = s.kv - s.n + rw / a.group + 1;
        lim[e] = l;
        minlim = min(minlim, l);
      }
    }
    minlim = min(minlim, __shfl_xor_sync(0xffffffffu, minlim, 1));
    minlim = min(minlim, __shfl_xor_sync(0xffffffffu, minlim, 2));

    if (s.next < end) {  // the next segment's queries into L1
      DecSeg t = s;
      dec_step<D>(a, sh, t, end);
      const uint16_t* src = q_row(t, lr);
      if (src) asm volatile("prefetch.global.L1 [%0];\n" ::"l"(src + lc * (KW * 8)));
    }

    float o[MT][4];
    float m[2], l[2], b[2], r[2];  // r: sums of the rounded weights
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[e] = kNone;
      l[e] = b[e] = r[e] = 0.f;
    }

#pragma unroll 1
    for (int u = s.u0; u < s.u0 + s.cnt; ++u) {
      __syncwarp();  // the stage before is free
      feed(st == 0 ? S - 1 : st - 1);
      if (!dead) {
        dead = __any_sync(0xffffffffu, !mbar_wait_lim(&full[st], par, limit, a.err));
        if (dead) {
#pragma unroll 1
          for (int i = 0; i < ahead; ++i) {
            const bool round = st + i >= S;
            mbar_drain(&full[st + i - (round ? S : 0)], par ^ (round ? 1u : 0u));
          }
          __syncwarp();
        }
        --ahead;
      }
      const uint8_t* stage = ring + st * C::stage;
      const int tok0 = u * kUnit;
      const uint32_t bad = (badbits >> (4 * st)) & 15u;
      const bool mask = tok0 + kUnit > minlim || bad || huge;
      // tile i's rows: the piece's part, then the rows before it in the piece
      auto at_row = [&](int i, int rb) {
        return stage + ((i * 16) >> tpl) * part_bytes + ((i * 16) & (tp - 1)) * rb;
      };

      // ---- scores
      float sc[TT][4];
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        uint32_t ka[KW], kb[KW];
        const uint8_t* ra = at_row(i, D / 2) + tau * (D / 2) + lc * (KW * 4);
        if (KW == 4) {
          const uint4 x = *reinterpret_cast<const uint4*>(ra);
          const uint4 y = *reinterpret_cast<const uint4*>(ra + 8 * (D / 2));
          ka[0] = x.x; ka[1] = x.y; ka[KW - 2] = x.z; ka[KW - 1] = x.w;
          kb[0] = y.x; kb[1] = y.y; kb[KW - 2] = y.z; kb[KW - 1] = y.w;
        } else {
          const uint2 x = *reinterpret_cast<const uint2*>(ra);
          const uint2 y = *reinterpret_cast<const uint2*>(ra + 8 * (D / 2));
          ka[0] = x.x; ka[1] = x.y;
          kb[0] = y.x; kb[1] = y.y;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[i][e] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const uint32_t xa = ka[w], xb = kb[w], ya = xa >> 8, yb = xb >> 8;
          const uint32_t a0[4] = {xa & 0x000F000Fu, xb & 0x000F000Fu, xa & 0x00F000F0u,
                                  xb & 0x00F000F0u};
          const uint32_t a1[4] = {ya & 0x000F000Fu, yb & 0x000F000Fu, ya & 0x00F000F0u,
                                  yb & 0x00F000F0u};
          mma_f16_16816(sc[i], a0, qf[w * 4], qf[w * 4 + 1]);
          mma_f16_16816(sc[i], a1, qf[w * 4 + 2], qf[w * 4 + 3]);
        }
        // s = scale * S + min * sum q (in units of 2^-24 of the scaled q)
        float ks0, km0, ks1, km1;
        const uint32_t* kp = reinterpret_cast<const uint32_t*>(at_row(i, 4) + tp * D) + tau;
        pair_f32<F16>(kp[0], ks0, km0);
        pair_f32<F16>(kp[8], ks1, km1);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sc[i][e] = fmaf(sc[i][e], ks0, km0 * qsum[e]);
          sc[i][e + 2] = fmaf(sc[i][e + 2], ks1, km1 * qsum[e]);
        }
      }
      float vs[TT][2], vm[TT][2];
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(at_row(i, 4) + tp * (D + 4)) + tau;
#pragma unroll
        for (int x = 0; x < 2; ++x) pair_f32<F16>(vp[8 * x], vs[i][x], vm[i][x]);
      }
      if (mask) {
        const float up = huge ? 0x1p24f : 1.f;
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int at = i * 16 + tau + 8 * x;
            const bool gone = (bad >> ((i * 16) >> tpl)) & 1u;
            if (gone || tok0 + at >= s.kv) vs[i][x] = vm[i][x] = 0.f;  // rows that nobody wrote
#pragma unroll
            for (int e = 0; e < 2; ++e)
              sc[i][e + 2 * x] = gone || tok0 + at >= lim[e] ? -INFINITY : sc[i][e + 2 * x] * up;
            // a non-finite value row reaches the rows that see it only (0 * NaN is NaN)
            if (!(fabsf(vm[i][x]) <= FLT_MAX && vs[i][x] <= FLT_MAX)) {
              vs[i][x] = vm[i][x] = 0.f;
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (sc[i][e + 2 * x] != -INFINITY) l[e] = __int_as_float(0x7fffffff);
            }
          }
      }
#pragma unroll
      for (int i = 0; i < TT; ++i)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          vs[i][x] = weight_scale(vs[i][x], vm[i][x]);
          vm[i][x] = fmaf(8.f, vs[i][x], vm[i][x]);
        }

      // ---- weights p scale_V
      float p[TT][4];
      uint32_t pw[TT][2];
      auto weigh = [&]() {  // true: a weight reached 2^15
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < TT; ++i) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int e = 0; e < 2; ++e) p[i][e + 2 * x] = ex2(fmaf(sc[i][e + 2 * x], cf[e], -m[e]));
            pw[i][x] = pack_h2(p[i][2 * x] * vs[i][x], p[i][2 * x + 1] * vs[i][x]);
          }
          top = weight_max(top, pw[i][0], pw[i][1]);
        }
        return weight_high(top);
      };
      if (__any_sync(0xffffffffu, weigh())) {
        // too large for the rows' references (always so at first)
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = -INFINITY;
#pragma unroll
          for (int i = 0; i < TT; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y)
              x = fmaxf(x, fmaf(sc[i][e + 2 * y], cf[e], __log2f(vs[i][y]) - kPeak));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float nm = fmaxf(m[e], x);
          alpha[e] = ex2(m[e] - nm);
          m[e] = nm;
          l[e] *= alpha[e];
          b[e] *= alpha[e];
          r[e] *= alpha[e];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          o[i][0] *= alpha[0];
          o[i][1] *= alpha[1];
          o[i][2] *= alpha[0];
          o[i][3] *= alpha[1];
        }
        weigh();
      }
#pragma unroll
      for (int i = 0; i < TT; ++i) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[e] += p[i][e] + p[i][e + 2];
          b[e] = fmaf(p[i][e], vm[i][0], fmaf(p[i][e + 2], vm[i][1], b[e]));
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&pw[i][x]));
          r[0] += f.x;
          r[1] += f.y;
          pw[i][x] = movmatrix_t(pw[i][x]);
        }
      }

      // ---- O^T += V^T P^T
      const int ta = (2 * lc) ^ (lc & 1), tb = (2 * lc + 1) ^ (lc & 1);  // tau(2 lc), tau(2 lc + 1)
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        uint32_t va[4][MT / 4];
        const uint8_t* base = at_row(i, D / 2) + tp * (D / 2) + lr * (D / 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint8_t* src = base + ((q & 1 ? tb : ta) + (q & 2 ? 8 : 0)) * (D / 2);
          if (MT == 8) {
            const uint2 x = *reinterpret_cast<const uint2*>(src);
            va[q][0] = x.x;
            va[q][MT / 4 - 1] = x.y;
          } else {
            va[q][0] = *reinterpret_cast<const uint32_t*>(src);
          }
        }
#pragma unroll
        for (int w = 0; w < MT / 4; ++w)
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            // byte y of both tokens: channels 2y (low nibble) and 2y + 1
            constexpr uint32_t kSel[4] = {0x4400u, 0x5511u, 0x6622u, 0x7733u};
            const uint32_t x0 = __byte_perm(va[0][w], va[1][w], kSel[y]);
            const uint32_t x1 = __byte_perm(va[2][w], va[3][w], kSel[y]);
            const uint32_t av[4] = {x0 & 0x000F000Fu, x0 & 0x00F000F0u, x1 & 0x000F000Fu,
                                    x1 & 0x00F000F0u};
            mma_f16_16816(o[w * 4 + y], av, pw[i][0], pw[i][1]);
          }
      }
      if (++st == S) {
        st = 0;
        par ^= 1;
      }
    }

    // ---------------------------------------------------------------- the segment's result
    const bool tail = s.u0 + s.cnt == s.nu;
    const bool whole = tail && s.u0 == 0;
    if (!tail) {
      open = true;
      __syncwarp();  // the ring is free: this was the warp's last segment
      if (lane == 0) {
        int* d = desc + warp * 8;
        d[0] = s.base; d[1] = s.nu; d[2] = s.n; d[3] = s.tok0; d[4] = s.h; d[5] = s.row0;
      }
    }
    // a part: to this warp's ring (its last segment) or the workspace (a tail)
    float* slot = tail ? tails + (size_t)worker * C::slot : reinterpret_cast<float*>(ring);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
          b[e] += __shfl_xor_sync(0xffffffffu, b[e], x);
          r[e] += __shfl_xor_sync(0xffffffffu, r[e], x);
        }
        const int row = 2 * lc + e;
        // (a row of NaN scores has no reference, but l NaN)
        const float top = m[e] == kNone && l[e] == 0.f ? -INFINITY : m[e];
        if (s.row0 + row < rows_all) {
          // O's rows carry 2^-24 (even channels) and 2^-20 (odd ones); the codes' -8
          const float mid = -8.f * r[e];
          float4 v[MT / 2];
#pragma unroll
          for (int i = 0; i < MT; i += 2)
            v[i / 2] = make_float4(fmaf(o[i][e], 0x1p24f, mid), fmaf(o[i][e + 2], 0x1p20f, mid),
                                   fmaf(o[i + 1][e], 0x1p24f, mid), fmaf(o[i + 1][e + 2], 0x1p20f, mid));
          if (whole) {
#pragma unroll
            for (int i = 0; i < MT / 2; ++i)
              dec_store<F16, D>(a, s, row, lr * (MT / 2) + i, top, l[e], b[e], v[i]);
          } else {
            float* dst = slot + row * (D + 4);
            if (lr == 0) *reinterpret_cast<float4*>(dst) = make_float4(top, l[e], b[e], 0.f);
#pragma unroll
            for (int i = 0; i < MT / 2; ++i)
              *reinterpret_cast<float4*>(dst + 4 + (lr * (MT / 2) + i) * 4) = v[i];
          }
        }
      }
    if (tail && !whole) {
      const int c0 = s.base / share, c1 = worker;
      __syncwarp();
      if (lane == 0 && c0 / W != (int)blockIdx.x) {  // else the CTA joins the item at its end
        __threadfence();
        if (atomicAdd(&counters[c0], 1u) == (unsigned)(dec_expected(c0, c1, W) - 1)) {
          __threadfence();
          counters[c0] = 0;
          int* d = fin + atomicAdd(nfin, 1) * 8;
          d[0] = s.base; d[1] = s.nu; d[2] = s.n; d[3] = s.tok0; d[4] = s.h; d[5] = s.row0;
        }
      }
    }
    if (s.next >= end) break;
    dec_step<D>(a, sh, s, end);
  }

  // ---------------------------------------------------------------- open parts of the CTA's warps
  if (lane == 0 && !open) desc[warp * 8] = -1;
  __syncthreads();
  // runs: warps with parts of one item side by side.  Lane w of every warp looks at warp w.
  const int base_w = lane < W ? desc[lane * 8] : -1;
  const int base_b = __shfl_up_sync(0xffffffffu, base_w, 1);
  const bool follows = lane > 0 && base_b == base_w;
  const uint32_t lead = __ballot_sync(0xffffffffu, base_w >= 0 && !follows);
  const uint32_t cont = __ballot_sync(0xffffffffu, base_w >= 0 && follows);
  const int c0_w = base_w / share, c1_w = base_w >= 0 ? (base_w + desc[lane * 8 + 1] - 1) / share : 0;
  // an item that starts and ends in this CTA is joined here, its tail with the run
  const uint32_t here = __ballot_sync(0xffffffffu, c0_w / W == (int)blockIdx.x && c1_w / W == (int)blockIdx.x);
  constexpr int kPer = C::rows * (D / 4);  // (row, four channels) of an item: whole warps
#pragma unroll 1
  for (int phase = 0; phase < 2; ++phase) {
    // 0: the runs; 1: the items whose last part was this CTA's
    const int n = phase ? *nfin : __popc(lead);
#pragma unroll 1
    for (int x = tid; x < n * kPer; x += W * 32) {
      const int e = x / kPer, row = (x % kPer) / (D / 4), d4 = x % (D / 4);
      int w0 = 0, w1 = 0;
      if (!phase) {
        uint32_t m = lead;
        for (int i = 0; i < e; ++i) m &= m - 1;
        w0 = __ffs(m) - 1;
        w1 = w0 + __ffs(~(cont >> (w0 + 1)));
      }
      const int* d = phase ? fin + e * 8 : desc + w0 * 8;
      DecSeg s = {};
      s.base = d[0]; s.nu = d[1]; s.n = d[2]; s.tok0 = d[3]; s.h = d[4]; s.row0 = d[5];
      if (s.row0 + row >= s.n * a.group) continue;
      const int c0 = s.base / share, c1 = (s.base + s.nu - 1) / share;
      const bool whole = phase || ((here >> w0) & 1u);
      // part 0, the ones from part 1 on at equal distances, the tail last
      const float *p0, *p1;
      int stride, np;
      if (phase) {
        const int k0 = c0 / W;
        p0 = runs + (size_t)c0 * C::slot;
        p1 = runs + (size_t)(k0 + 1) * W * C::slot;
        stride = W * C::slot;
        np = dec_expected(c0, c1, W);
      } else {
        p0 = reinterpret_cast<const float*>(smem + o_ring + w0 * (S * C::stage));
        stride = S * C::stage / 4;
        p1 = p0 + stride;
        np = w1 - w0 + (whole ? 1 : 0);
      }
      const float* tail = whole ? tails + (size_t)c1 * C::slot : nullptr;
      auto src = [&](int c) {
        return (c == 0 ? p0 : tail && c == np - 1 ? tail : p1 + (size_t)(c - 1) * stride) + row * (D + 4);
      };
      float top, l, b;
      const float4 o = dec_join(np, d4, src, top, l, b);
      if (whole) {
        dec_store<F16, D>(a, s, row, d4, top, l, b, o);
      } else {
        float* dst = runs + (size_t)(blockIdx.x * W + w0) * C::slot + row * (D + 4);
        if (d4 == 0) *reinterpret_cast<float4*>(dst) = make_float4(top, l, b, 0.f);
        *reinterpret_cast<float4*>(dst + 4 + d4 * 4) = o;
      }
    }
    if (!phase && (lead & ~here)) {  // the same for all threads
      __syncthreads();
      if (warp == 0 && (((lead & ~here) >> lane) & 1u)) {
        __threadfence();  // for all threads' parts, which the barrier ordered before
        if (atomicAdd(&counters[c0_w], 1u) == (unsigned)(dec_expected(c0_w, c1_w, W) - 1)) {
          __threadfence();
          counters[c0_w] = 0;
          int* f = fin + atomicAdd(nfin, 1) * 8;
          for (int i = 0; i < 6; ++i) f[i] = desc[lane * 8 + i];
        }
      }
      __syncthreads();
    }
  }

  attn_zero_pad<D>(a, pad, W * 32);
}

constexpr int kDecMaxCtas = 160;
constexpr int kDecMaxWorkers = kDecMaxCtas * DecCfg<128>::W;
// counters [workers], which stay zero between calls | runs [workers][slot] | tails [workers][slot]
constexpr size_t kDecCounterBytes = (kDecMaxWorkers * 4 + 255) / 256 * 256;
static_assert(kDecCounterBytes <= DIP_KV4_WORKSPACE_ZEROS, "the counters start as zeros");
size_t kv4_decode_counter_bytes() { return kDecCounterBytes; }
size_t kv4_decode_part_bytes() { return 2 * (size_t)kDecMaxWorkers * DecCfg<128>::slot * 4; }

template <bool F16, int D>
static int dec_launch(const AttnArgs& a, void* counters, void* parts, cudaStream_t st) {
  using C = DecCfg<D>;
  auto kern = kv4_decode_kernel<F16, D>;
  const cudaError_t e = attn_smem<kv4_decode_kernel<F16, D>>(227 * 1024);
  if (e != cudaSuccess) return launch_status(e);
  const int grid = std::min(num_sms(), kDecMaxCtas);
  float* runs = static_cast<float*>(parts);
  float* tails = runs + (size_t)kDecMaxCtas * C::W * C::slot;
  return launch_status(launch(kern, dim3(grid), dim3(C::threads), C::smem(a.nreq), st, a,
                              C::o_ring(a.nreq), static_cast<unsigned*>(counters), runs, tails));
}

// Positions are 32-bit: bounded from what the host knows.
bool kv4_decode_fits(const AttnArgs& a) {
  constexpr int rows = DecCfg<128>::rows;
  const int64_t units = (std::min<int64_t>(a.max_blocks << a.g.p_log2, kMaxKv) + kUnit - 1) / kUnit + kOvh + 1;
  const int64_t blocks = std::min((int64_t)a.num_tokens * a.group / rows + a.nreq,
                                  ((int64_t)a.max_rows + rows - 1) / rows * a.nreq);
  return units * a.g.hkv <= (1LL << 30) / std::max<int64_t>(blocks, 1);
}

int kv4_decode(const AttnArgs& a, bool f16, void* counters, void* parts, cudaStream_t st) {
  auto go = [&](auto f, auto d) { return dec_launch<decltype(f)::value, decltype(d)::value>(a, counters, parts, st); };
  using T = std::true_type;
  using F = std::false_type;
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (f16) return a.g.d == 64 ? go(T{}, D64{}) : go(T{}, D128{});
  return a.g.d == 64 ? go(F{}, D64{}) : go(F{}, D128{});
}

}  // namespace dip
