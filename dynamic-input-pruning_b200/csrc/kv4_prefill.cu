// kv4_prefill.cu — attention over the 4-bit paged cache for many query rows
// (prompt chunks), on the 5th-generation tensor cores.
//
// A tile is up to 256 query rows of one request and KV head (rows = query tokens x
// the query heads of the group), two M = 128 blocks that share every dequantised
// key and value tile of 128 cached tokens:
//   S = Q C_K^T,      arg = s_K S + min_K sum q - M,     p = 2^arg
//   O += (p s_V) (C_V - 8),  b += p (min_V + 8 s_V),  l += p,   out = (O + b) / l
// where C are the codes: the products run on the codes themselves, exact in fp16 (a key
// code in the low bits of a 16-bit lane is the subnormal code * 2^-24, its masked
// neighbour nibble code * 2^-20; value codes are made whole numbers about zero, so that
// the rounding of a weight weighs no more than its value, the neighbour nibble's times
// 16; the factor 16 is taken out of the queries and of O's columns), and the pairs
// enter in fp32.  What is rounded: the queries not at all
// (fp16, scaled by one power of two a tile: exact down to 2^-27 of its largest finite one), the
// weights p s_V once to fp16, the result once.  A row's reference M (a whole number, so
// that rescaling is exact) is its largest arg + log2 s_V less kPeak: weights peak
// near 2^kPeak, and M moves only when one reaches 2^15 (then the tile's earlier weights,
// O, b and l are rescaled).  What fp16 loses of small weights: at kPeak.
//
// Warps 0-7: softmax, a warp 32 rows of a block; a thread holds, of each eight columns,
// two of four rows (the 16x256b shape), so that a pair of columns' pairs (32 bytes) is
// read once for four rows.  Warps 8-11: unpack, a lane a cached token, raw codes a tile ahead
// in registers.  Warp 12: issues the MMAs, in the order P0 V, Q0 K, P1 V, Q1 K of
// successive tiles, so that one block's softmax runs under the other's products.
//
// In a call with tokens for fewer than four rounds of tiles, few tiles or a long one among
// them are cut along the keys into parts, each to a slot of the workspace (M, l, O + b of its
// rows in fp32), which a second kernel joins in their order.  32 tokens behind 300000, 64/8
// heads: 0.47 ms (whole 7.02); 2 x 200 behind 30000, 32/4 heads: 0.47 ms (whole 0.72).  A
// launch that cuts nothing pays for the choice (700 fresh tokens 59 and 51 us), so calls with
// more tokens go without, also where one of their contexts is long.
//
// Measured: 4096 tokens behind 4096, 64/8 heads of 128, bf16, 1.12 ms, 0.73 PFLOP/s or
// 44 % of a measured 1.66 PFLOP/s matrix product.  Bound by the softmax warps' latency
// and issue: 4150 of a tile's 5700 cycles in the softmax, 1300 waiting for the block's
// own products (1024 at the tensor cores' rate); and by about eight steps a tile for finding
// it, its queries, the first references, the result.  Slower were: packed fp32 pairs
// (+17 %), 16 softmax warps of half the columns (+12 %), steps of 64 tokens with the
// scores two steps ahead (+6 %: key products of 64 columns read shared memory as often
// as those of 128), register splits between the warps (+6 to 9 %).
// Hidden positions: the weights of rows past the context, of pages outside the cache
// and of those hidden by causality are 0.  A value row with a non-finite pair counts
// as 0 and makes l NaN for the rows that see it, so that it cannot reach the others.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kv4_attn.cuh"

namespace dip {

constexpr int kPfSoft = 8;           // softmax warps, 4 a block
constexpr int kPfThreads = (kPfSoft + 5) * 32;
constexpr int kPfN = 128;            // cached tokens a tile
constexpr int kPfRows = 256;         // query rows a tile
constexpr int kPfSlots = 480;        // parts of split tiles that the workspace holds
constexpr int kPfMinSpan = 4;        // fewest steps of 128 tokens a part
constexpr int kPfPartCost = 8;       // what a part costs beside its steps, in steps (60 x 500 tokens: 8 to 9)
constexpr int kPfWhole = 4;          // rounds of whole tiles from which none is split
constexpr int kPfCuts = 6;           // ways of cutting that are weighed
constexpr float kPfNone = -1e30f;    // reference of a row that has seen no position

template <int D>
struct PfCfg {
  static constexpr int block = 128 * D * 2;       // Q block, K or V tile
  static constexpr int o_k = 2 * block, o_v = 4 * block;
  static constexpr int o_bar = 6 * block;
  // [4] tiles: 4 seen and 4 NaN masks; pairs of two tokens: key (s, s, min, min), value (s, s, min, min)
  static constexpr int o_mask = o_bar + 256;
  static constexpr int o_par = o_mask + 4 * 32;
  static constexpr int o_row = o_par + 4 * kPfN * 16;    // [256] x (sum q, limit; later 1 / l, b / l)
  static constexpr int o_plan = o_row + kPfRows * 8;
  static constexpr int total = o_plan + 1024 + 1024;  // + alignment slack
};

__device__ __forceinline__ void pf_fence_async() {
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
}
__device__ __forceinline__ void pf_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
}
__device__ __forceinline__ void pf_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
}
// Shared memory matrix descriptor, 128-byte swizzle (start, leading and stride byte
// offsets >> 4, version 1, layout type 2).  It moves by x >> 4 when its start moves by x.
__device__ __forceinline__ uint64_t pf_desc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16, fp32 accumulator, fp16 operands, M = 128; B MN-major where b_mn.
__host__ __device__ constexpr uint32_t pf_idesc(int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// One lane of a converged warp, in a form that the compiler knows to be one: an MMA then
// takes two instructions to issue, from a branch on the lane's number fourteen.
__device__ __forceinline__ bool pf_elect() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void pf_mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d), "l"(ad), "l"(bd),
      "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void pf_mma_ts(uint32_t d, uint32_t at, uint64_t bd, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(at), "l"(bd),
      "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void pf_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(
                   smem_u32(bar))
               : "memory");
}
// This warp's 32 lanes x 32 columns.
__device__ __forceinline__ void pf_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void pf_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
// 32 lanes x 16 columns, lanes 0-15 to a, 16-31 to b: registers 4 g, 4 g + 1 are (row lane / 4,
// columns 8 g + 2 (lane % 4) and + 1), 4 g + 2, 4 g + 3 row + 8's.  The wait is part of it: a
// wait of its own that takes the registers as operands costs a move each.
__device__ __forceinline__ void pf_ldf(uint32_t taddr, uint32_t (&a)[8], uint32_t (&b)[8]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n"
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n"
      "tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]), "=r"(a[4]), "=r"(a[5]), "=r"(a[6]), "=r"(a[7]),
        "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]), "=r"(b[4]), "=r"(b[5]), "=r"(b[6]), "=r"(b[7])
      : "r"(taddr), "r"(taddr + (16u << 16))
      : "memory");
}
// The same of 16 lanes.
__device__ __forceinline__ void pf_stf(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.16x256b.x2.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};\n" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
               "r"(taddr)
               : "memory");
}
// 16 lanes x 8 columns of packed pairs: registers 2 g, 2 g + 1 are (row lane / 4, column
// 4 g + lane % 4) and row + 8's.
__device__ __forceinline__ void pf_ldp(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.16x128b.x2.b32 {%0,%1,%2,%3}, [%4];\ntcgen05.wait::ld.sync.aligned;\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void pf_stp(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%4], {%0,%1,%2,%3};\n" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void pf_stp(uint32_t taddr, const uint32_t (&r)[8]) {  // 16 columns
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};\n" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
               "r"(taddr)
               : "memory");
}
__device__ __forceinline__ float pf_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// (lo, hi) -> two 16-bit values, one rounding each.
template <bool F16>
__device__ __forceinline__ uint32_t pf_cvt2(float lo, float hi) {
  uint32_t y;
  if (F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;\n" : "=r"(y) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;\n" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}

// Eight codes of a packed word as fp16 lanes, positions (0,4) (1,5) (2,6) (3,7): code * 2^-24
// at even channels, code * 2^-20 at odd ones.
__device__ __forceinline__ uint4 pf_unpack8(uint32_t w) {
  const uint32_t t = w >> 8;
  return make_uint4(w & 0x000F000Fu, w & 0x00F000F0u, t & 0x000F000Fu, t & 0x00F000F0u);
}

// Eight codes less 8, whole: code - 8 at even channels, 16 (code - 8) at odd ones.
__device__ __forceinline__ uint4 pf_unpack8_mid(uint32_t w) {
  const uint4 c = pf_unpack8(w);
  const __half2 lo = __half2half2(__ushort_as_half(0x6408)), hi = __half2half2(__ushort_as_half(0x6480));
  auto mid = [](uint32_t x, __half2 m) {  // 1024 + x, less 1024 + 8 or 1024 + 128
    x |= 0x64006400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&x), m);
    return *reinterpret_cast<const uint32_t*>(&r);
  };
  return make_uint4(mid(c.x, lo), mid(c.y, hi), mid(c.z, lo), mid(c.w, hi));
}

// Byte offset of (row, 16-byte chunk) in a tile: groups of 8 rows, blocks of 64
// channels, 128-byte rows with their chunks swizzled.  The same bytes serve as a
// K-major (keys, queries) and an MN-major operand (values).
template <int D>
__device__ __forceinline__ uint32_t pf_off(int r, int c) {
  return (r >> 3) * (D * 16) + (c >> 3) * 1024 + (r & 7) * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// What a slot of the workspace holds: a part of a request's tile; slot kPfSlots: r = slots in use.
struct PfMeta {
  int r, tile, part, parts;
};

// A row's lse: M is in powers of two.
__device__ __forceinline__ void pf_lse(const AttnArgs& a, const AttnReq& rq, int h, int row, bool none, float M,
                                       float l) {
  if (!a.lse) return;
  const int i = row / a.group;
  a.lse[(int64_t)(rq.tok0 + i) * a.heads + h * a.group + (row - i * a.group)] =
      none ? -INFINITY : M * kLn2 + logf(l);
}

template <bool F16, int D, bool SPLIT>
__global__ void __launch_bounds__(kPfThreads, 1)
kv4_prefill_kernel(const AttnArgs a, int min_rows, int zero_pad, int ctas, PfMeta* meta, float* parts_out) {
  using C = PfCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::o_bar);
  uint64_t *kfull = bars, *kempty = bars + 2, *vfull = bars + 4, *vempty = bars + 6, *sfull = bars + 8,
           *pready = bars + 10, *odone = bars + 12;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 16);
  uint32_t* masks = reinterpret_cast<uint32_t*>(smem + C::o_mask);
  int* qtop = reinterpret_cast<int*>(bars + 17);   // 16-bit pattern of the tile's largest |q|
  uint64_t *qbar = bars + 18, *drain = bars + 19;
  int* plan = reinterpret_cast<int*>(smem + C::o_plan);           // [2][16] scans, tile, part, work
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform
  pdl_wait();
  const uint32_t limit = spin_limit(a.err);

  // ---------------------------------------------------------------- which tile, which part of its keys
  // Heads fastest, then parts, then tiles with the last (longest) of a request first.
  const int h = blockIdx.x % a.g.hkv, want = blockIdx.x / a.g.hkv;
  auto tiles_of = [&](const AttnReq& q) {
    const int rows = q.n * a.group;
    return rows > min_rows ? (rows + kPfRows - 1) / kPfRows : 0;
  };
  auto steps_of = [](int positions) { return (max(positions, 0) + kPfN - 1) / kPfN; };
  const int per = (a.nreq + kPfThreads - 1) / kPfThreads;
  constexpr int NW = kPfThreads / 32;
  int span = 0x3fffffff;
  if (SPLIT) {
    // Tiles are cut into parts of at most `span` steps, so that neither few tiles nor a long
    // one leave the GPU idle: of some fractions of its even share of all steps the one that
    // should end first: one round if the parts are few, else the share, the parts' cost and
    // half a part at the end.  Eight lanes a request, a lane a cut.
    static_assert(kPfCuts <= 8, "lanes");
    const int k = min(lane & 7, kPfCuts - 1);
    float work = 0.f;
    int longest = 0;
#pragma unroll 1
    for (int r = tid >> 3; r < a.nreq; r += kPfThreads / 8) {
      const AttnReq q = attn_req(a, r);
      const int n = tiles_of(q), last = steps_of(q.kv);
      const int first = a.causal ? steps_of(min(q.kv - q.n + (kPfRows - 1) / a.group + 1, q.kv)) : last;
      work += (float)n * 0.5f * (float)(first + last);
      if (n) longest = max(longest, last);
    }
    work += __shfl_xor_sync(0xffffffffu, work, 8);
    work += __shfl_xor_sync(0xffffffffu, work, 16);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) {
      plan[warp] = __float_as_int(work);
      plan[16 + warp] = longest;
    }
    __syncthreads();
    work = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      work += __int_as_float(plan[w]);
      longest = max(longest, plan[16 + w]);
    }
    work *= a.g.hkv;
    // the first leaves tiles whole
    const int cut = k == 0 ? max(longest, 1)
                           : max((int)fminf(work / ctas * (k == 1 ? 1.06f : 1.03f / k) + 1.f, 1e8f), kPfMinSpan);
    int all = 0, split = 0;  // parts, parts of split tiles
#pragma unroll 1
    for (int r = tid >> 3; r < a.nreq; r += kPfThreads / 8) {
      const AttnReq q = attn_req(a, r);
      const int np = max((steps_of(q.kv) + cut - 1) / cut, 1), n = tiles_of(q) * np;
      all += n;
      if (np > 1) split += n;
    }
    all += __shfl_xor_sync(0xffffffffu, all, 8);
    all += __shfl_xor_sync(0xffffffffu, all, 16);
    split += __shfl_xor_sync(0xffffffffu, split, 8);
    split += __shfl_xor_sync(0xffffffffu, split, 16);
    if (lane < 8) {
      plan[32 + warp * 16 + lane] = all;
      plan[32 + warp * 16 + 8 + lane] = split;
    }
    __syncthreads();
    all = split = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      all += plan[32 + w * 16 + k];
      split += plan[32 + w * 16 + 8 + k];
    }
    const float n = (float)all * a.g.hkv, one = (float)(cut + kPfPartCost);
    float cost = n <= ctas ? one : (work + n * kPfPartCost) / ctas + 0.5f * one;
    if (split > kPfSlots / a.g.hkv) cost = FLT_MAX;
    float best = cost;
#pragma unroll
    for (int o = 4; o; o >>= 1) best = fminf(best, __shfl_xor_sync(0xffffffffu, best, o));
    span = __shfl_sync(0xffffffffu, cut, __ffs(__ballot_sync(0xffffffffu, cost == best)) - 1);
    __syncthreads();
  }
  auto parts_of = [&](const AttnReq& q) { return SPLIT ? max((steps_of(q.kv) + span - 1) / span, 1) : 1; };
  int sum = 0, split = 0;  // parts of this thread's requests; of split tiles
  bool bad_cu = false;
  for (int i = 0; i < per; ++i)
    if (tid * per + i < a.nreq) {
      const AttnReq q = attn_req(a, tid * per + i);
      bad_cu |= q.bad;
      const int np = parts_of(q), n = tiles_of(q) * np;
      sum += n;
      if (np > 1) split += n;
    }
  int inc = sum, inc2 = split;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, inc, o), t2 = __shfl_up_sync(0xffffffffu, inc2, o);
    if (lane >= o) {
      inc += t;
      inc2 += t2;
    }
  }
  if (lane == 31) {
    plan[warp] = inc;
    plan[16 + warp] = inc2;
  }
  if (tid == 0) plan[32] = -1;
  bad_cu = __syncthreads_or(bad_cu);  // then no tile, all tokens zeros
  if (bad_cu && blockIdx.x == 0 && tid == 0) atomicOr(a.err, kErrInput);
  int before = inc - sum, split_before = inc2 - split;
  for (int w = 0; w < warp; ++w) {
    before += plan[w];
    split_before += plan[16 + w];
  }
  if (SPLIT && blockIdx.x == 0 && tid == 0) {
    int all = 0;
    for (int w = 0; w < NW; ++w) all += plan[16 + w];
    meta[kPfSlots].r = bad_cu ? 0 : all * a.g.hkv;
  }
  if (!bad_cu && sum > 0 && want >= before && want < before + sum)
    for (int i = 0; i < per; ++i) {
      const int r = tid * per + i;
      if (r >= a.nreq) break;
      const AttnReq q = attn_req(a, r);
      const int np = parts_of(q), n = tiles_of(q), u = want - before;
      if (u >= 0 && u < n * np) {
        plan[32] = r;
        plan[33] = n - 1 - u / np;
        plan[34] = u % np;
        plan[35] = np;
        plan[36] = (split_before + u) * a.g.hkv + h;  // the part's slot, if there are more
        if (np > 1) meta[plan[36]] = {r, n - 1 - u / np, u % np, np};
      }
      before += n * np;
      if (np > 1) split_before += n * np;
    }
  __syncthreads();
  pdl_launch_dependents();
  if (zero_pad) attn_zero_pad<D>(a, bad_cu ? AttnPad{0, 0} : attn_pad(a), kPfThreads);
  const int r = plan[32];
  if (r < 0) return;
  const AttnReq rq = attn_req(a, r);
  const int row0 = plan[33] * kPfRows;
  const int rows = min(rq.n * a.group - row0, kPfRows);
  const int nblk = rows > 128 ? 2 : 1;
  // the last row's limit bounds the tiles
  const int last_tok = (row0 + rows - 1) / a.group;
  const int maxlim = a.causal ? rq.kv - rq.n + last_tok + 1 : rq.kv;
  const int steps = steps_of(maxlim);
  const int j0 = SPLIT ? (int)((int64_t)steps * plan[34] / plan[35]) : 0;
  const int nt = (SPLIT ? (int)((int64_t)steps * (plan[34] + 1) / plan[35]) : steps) - j0;
  if (SPLIT && tid == 0) plan[38] = j0 * kPfN;
  auto first = [&]() { return SPLIT ? plan[38] : 0; };  // this part's first position

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&kfull[i], 4);
      mbar_init(&kempty[i], 1);
      mbar_init(&vfull[i], 4);
      mbar_init(&vempty[i], 1);
      mbar_init(&sfull[i], 1);
      mbar_init(&pready[i], 4);
      mbar_init(&odone[i], 1);
    }
    mbar_init(qbar, 1);
    mbar_init(drain, 1);
    *qtop = 0;
    mbar_fence_init();
  }
  if (warp == kPfSoft + 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(
                     smem_u32(tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  pf_fence_before();
  __syncthreads();
  pf_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool dead = false;  // a wait ran out: skip the later ones, drain, free TMEM, return
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!dead) dead = !mbar_wait_lim(bar, parity, limit, a.err);
  };
  constexpr uint32_t kO = 256;  // first column of the O accumulators

  // ---------------------------------------------------------------- the tile's queries
  // one power of two for the tile: largest finite |q| to [2^13, 2^14)
  struct RowInfo { float sum; int lim; };  // sum of the scaled q, positions a row sees
  RowInfo* rowinfo = reinterpret_cast<RowInfo*>(smem + C::o_row);
  constexpr int CH = D / 8, RP = 32 / CH;  // chunks a row, rows a load
  // The rows come by bulk copies, a thread a row, to where keys and values will be: loads in
  // registers cost either their latency in every turn of a loop or the fetch of unrolled code
  // (14000 to 20000 cycles a tile, now 5000).
  const uint8_t* raw = smem + C::o_k;
  if (tid < rows) {
    const int qi = (row0 + tid) / a.group;
    if (tid == 0) mbar_arrive_expect_tx(qbar, rows * D * 2);
    bulk_g2s(smem + C::o_k + tid * (D * 2),
             a.q + (int64_t)(rq.tok0 + qi) * a.q_ts + (int64_t)(h * a.group + row0 + tid - qi * a.group) * a.q_hs,
             D * 2, qbar);
  }
  auto q_chunk = [&](int x) {
    return x < rows ? *reinterpret_cast<const uint4*>(raw + x * (D * 2) + (lane % CH) * 16) : make_uint4(0, 0, 0, 0);
  };
  if (warp < 8) {
    wait(qbar, 0);
    uint32_t mx = 0;  // largest |q| as 16-bit patterns, which order as integers
#pragma unroll 4
    for (int i = 0; i < CH; ++i) {
      const uint4 v = q_chunk(warp * 32 + i * RP + lane / CH);
      mx = __vmaxu2(__vmaxu2(mx, __vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu)),
                    __vmaxu2(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
    }
    mx = __reduce_max_sync(0xffffffffu, max(mx & 0xFFFFu, mx >> 16));
    if (lane == 0) atomicMax(qtop, (int)mx);
  }
  __syncthreads();
  constexpr uint32_t kInf = F16 ? 0x7C00u : 0x7F80u;
  if (*qtop >= (int)kInf) {  // a row with an infinity or a NaN: the others' scale is not its own
    __syncthreads();
    if (tid == 0) *qtop = 0;
    __syncthreads();
    if (warp < 8) {
      uint32_t mx = 0;
      auto finite = [&](uint32_t w) {
        const uint32_t lo = w & 0x7FFFu, hi = (w >> 16) & 0x7FFFu;
        mx = max(mx, max(lo < kInf ? lo : 0u, hi < kInf ? hi : 0u));
      };
#pragma unroll 1
      for (int i = 0; i < CH; ++i) {
        const uint4 v = q_chunk(warp * 32 + i * RP + lane / CH);
        finite(v.x);
        finite(v.y);
        finite(v.z);
        finite(v.w);
      }
      mx = __reduce_max_sync(0xffffffffu, mx);
      if (lane == 0) atomicMax(qtop, (int)mx);
    }
    __syncthreads();
  }
  const float qmx = h16_to_f32<F16>((uint32_t)*qtop);
  const int qex = (int)((__float_as_uint(qmx) >> 23) & 255u) - 127;
  const int qe = qmx > 0.f ? min(max(13 - qex, -114), 126) : 0;
  if (warp < 8) {
    uint8_t* qs = smem + (warp >> 2) * C::block;
    const float sg = pf_pow2(qe);
#pragma unroll 2
    for (int i = 0; i < CH; ++i) {
      const int y = warp * 32 + i * RP + lane / CH;
      const uint4 v = q_chunk(y);
      const uint32_t x[4] = {v.x, v.y, v.z, v.w};
      float f[8], sum_q = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[2 * j] = h16_to_f32<F16>(x[j] & 0xFFFFu);
        f[2 * j + 1] = h16_to_f32<F16>(x[j] >> 16);
        f[2 * j] *= sg;
        f[2 * j + 1] *= sg;
        sum_q += f[2 * j] + f[2 * j + 1];
        f[2 * j + 1] *= 0.0625f;  // odd channels: the codes' 16
      }
      *reinterpret_cast<uint4*>(qs + pf_off<D>(y & 127, lane % CH)) =
          make_uint4(pf_cvt2<true>(f[0], f[4]), pf_cvt2<true>(f[1], f[5]), pf_cvt2<true>(f[2], f[6]),
                     pf_cvt2<true>(f[3], f[7]));
#pragma unroll
      for (int o = 1; o < CH; o <<= 1) sum_q += __shfl_xor_sync(0xffffffffu, sum_q, o);
      if (lane % CH == 0)
        rowinfo[y] = {sum_q, a.causal && y < rows ? rq.kv - rq.n + (row0 + y) / a.group + 1 : rq.kv};
    }
    pf_fence_async();
  }
  __syncthreads();

  if (warp < kPfSoft) {
    // ------------------------------------------------------------ softmax
    const int t = warp >> 2;  // block
    if (t < nblk) {
      const int quad = lane >> 2, lc = lane & 3;
      const int lrow = t * 128 + (warp & 3) * 32 + quad;  // this thread's rows: lrow + 8 r
      float qsum[4], M[4], l[4], b[4];
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        qsum[r4] = rowinfo[lrow + r4 * 8].sum;
        M[r4] = kPfNone;
        l[r4] = b[r4] = 0.f;
      }
      const int wlim = rowinfo[t * 128 + (warp & 3) * 32].lim;  // the warp's first row has the smallest
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + lanes + t * 128, to = tmem + lanes + kO + t * D;
#pragma unroll 1
      for (int j = 0; j < nt; ++j) {
        wait(&sfull[t], j & 1);
        pf_fence_after();
        const uint32_t* mk = masks + (j & 3) * 8;
        const float4* par = reinterpret_cast<const float4*>(smem + C::o_par + (j & 3) * (kPfN * 16)) + 2 * lc;
        const bool mask = (mk[0] & mk[1] & mk[2] & mk[3]) != 0xffffffffu ||
                          (mk[4] | mk[5] | mk[6] | mk[7]) || first() + (j + 1) * kPfN > wlim;
        // 16-column chunks between two looks at the weights.  Nothing overlaps across a look,
        // and the weights since the last one stay in registers, which the copy with tests is
        // short of: 2048 tokens behind 6144 took 750 us with one, 749 with two in both copies,
        // 731 with two and one, 1614 (spilled) with four.
        auto chunks = [](auto masked) constexpr { return decltype(masked)::value ? 1 : 2; };
        // 16 N columns from 16 c
        auto chunk = [&](auto masked, int c) {
          constexpr bool MASK = decltype(masked)::value;
          constexpr int N = chunks(masked);
          uint32_t hid[4] = {0, 0, 0, 0};  // bits of 16 hidden columns, from this thread's first
          auto hidden = [&](int c) {
            if (MASK) {
#pragma unroll
              for (int r4 = 0; r4 < 4; ++r4) {
                const int left = rowinfo[lrow + r4 * 8].lim - (first() + j * kPfN + c * 16);
                const uint32_t sh = (c & 1) * 16;
                const uint32_t in = left >= 16 ? 0xffffu : left <= 0 ? 0u : (1u << left) - 1u;
                const uint32_t vis = (mk[c >> 1] >> sh) & in;
                hid[r4] = ~vis >> (2 * lc);
                if ((mk[4 + (c >> 1)] >> sh) & vis) l[r4] = __int_as_float(0x7fffffff);  // a non-finite value row in sight
              }
            }
          };
          // arg of (row r4, group g's two columns), from the columns' key pairs
          auto arg = [&](const uint32_t (&w)[2][8], int r4, int g, const float4& k, float ref, float& x, float& y) {
            const uint32_t* sx = w[r4 >> 1] + 4 * g + 2 * (r4 & 1);
            x = fmaf(__uint_as_float(sx[0]), k.x, fmaf(k.z, qsum[r4], ref));
            y = fmaf(__uint_as_float(sx[1]), k.y, fmaf(k.w, qsum[r4], ref));
            if (MASK) {
              if (hid[r4] & (1u << (8 * g))) x = -INFINITY;
              if (hid[r4] & (2u << (8 * g))) y = -INFINITY;
            }
          };
          uint32_t pk[2][4 * N];
          float lt[4], bt[4];
          auto weigh = [&]() {  // true: a weight reached 2^15
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < N; ++e) {
              uint32_t w[2][8];
              pf_ldf(ts + (c + e) * 16, w[0], w[1]);
              hidden(c + e);
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                const float4 k = par[((c + e) * 2 + g) * 8], v = par[((c + e) * 2 + g) * 8 + 1];
                const bool first = e == 0 && g == 0;
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                  float x, y;
                  arg(w, r4, g, k, -M[r4], x, y);
                  x = ex2(x);
                  y = ex2(y);
                  lt[r4] = first ? x + y : lt[r4] + (x + y);
                  bt[r4] = fmaf(y, v.w, first ? x * v.z : fmaf(x, v.z, bt[r4]));
                  const uint32_t p = pf_cvt2<true>(x * v.x, y * v.y);
                  pk[r4 >> 1][4 * e + 2 * g + (r4 & 1)] = p;
                  if (r4 & 1) top = weight_max(top, p, pk[r4 >> 1][4 * e + 2 * g]);
                }
              }
            }
            return weight_high(top);
          };
          auto rescale = [&]() {
            float nm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, alpha[4];
#pragma unroll 1
            for (int e = 0; e < N; ++e) {
              uint32_t w[2][8];
              pf_ldf(ts + (c + e) * 16, w[0], w[1]);
              hidden(c + e);
#pragma unroll
              for (int g = 0; g < 2; ++g) {
                const float4 k = par[((c + e) * 2 + g) * 8], v = par[((c + e) * 2 + g) * 8 + 1];
                const float l0 = __log2f(v.x) - kPeak, l1 = __log2f(v.y) - kPeak;
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                  float x, y;
                  arg(w, r4, g, k, 0.f, x, y);
                  nm[r4] = fmaxf(nm[r4], fmaxf(x + l0, y + l1));
                }
              }
            }
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
              nm[r4] = fmaxf(nm[r4], __shfl_xor_sync(0xffffffffu, nm[r4], 1));
              nm[r4] = fmaxf(nm[r4], __shfl_xor_sync(0xffffffffu, nm[r4], 2));
              nm[r4] = fmaxf(ceilf(nm[r4]), M[r4]);
              alpha[r4] = M[r4] == kPfNone ? 0.f
                          : nm[r4] - M[r4] >= 126.f ? 0.f : pf_pow2(-(int)(nm[r4] - M[r4]));
              M[r4] = nm[r4];
              l[r4] *= alpha[r4];
              b[r4] *= alpha[r4];
            }
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const __half2 h0 = __float2half2_rn(alpha[2 * hh]), h1 = __float2half2_rn(alpha[2 * hh + 1]);
#pragma unroll 1
              for (int d = 0; d < c; ++d) {  // this tile's weights so far
                uint32_t e[4];
                pf_st_wait();
                pf_ldp(ts + (hh << 20) + d * 8, e);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const __half2 z = __hmul2(*reinterpret_cast<const __half2*>(&e[i]), i & 1 ? h1 : h0);
                  e[i] = *reinterpret_cast<const uint32_t*>(&z);
                }
                pf_stp(ts + (hh << 20) + d * 8, e);
              }
            }
            if (j > 0) {  // the product before this tile's scores is complete (same barrier)
#pragma unroll 1
              for (int d = 0; d < D / 16; ++d) {
                uint32_t e[2][8];
                pf_ldf(to + d * 16, e[0], e[1]);
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
#pragma unroll
                  for (int i = 0; i < 8; ++i)
                    e[hh][i] = __float_as_uint(__uint_as_float(e[hh][i]) * alpha[2 * hh + ((i >> 1) & 1)]);
                  pf_stf(to + (hh << 20) + d * 16, e[hh]);
                }
              }
            }
          };
          // again if a weight is too large for the rows' references (always so at first;
          // once at most: NaN scores stay so)
#pragma unroll 1
          for (int n = 0; __any_sync(0xffffffffu, weigh()) && n == 0; ++n) rescale();
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            l[r4] += lt[r4];
            b[r4] += bt[r4];
          }
          __syncwarp();
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) pf_stp(ts + (hh << 20) + c * 8, pk[hh]);  // over columns already read
        };
        auto tile = [&](auto masked) {
#pragma unroll 1
          for (int c = 0; c < kPfN / 16; c += chunks(masked)) chunk(masked, c);
        };
        // two copies: the tests of a tile with hidden positions cost as much as its arithmetic
        if (mask) tile(std::true_type{});
        else tile(std::false_type{});
        pf_st_wait();
        pf_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&pready[t]);
      }

      // ---- result: per row what takes O to the output, to the threads of the row
      __syncwarp();  // the rows' limits have been read
      float2* rowout = reinterpret_cast<float2*>(rowinfo);
      const int nparts = SPLIT ? plan[35] : 1;  // (not kept in registers meanwhile)
      float* slot = parts_out + (size_t)plan[36] * (kPfRows * (D + 2));
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        float ls = l[r4], bs = b[r4];
        ls += __shfl_xor_sync(0xffffffffu, ls, 1);
        bs += __shfl_xor_sync(0xffffffffu, bs, 1);
        ls += __shfl_xor_sync(0xffffffffu, ls, 2);
        bs += __shfl_xor_sync(0xffffffffu, bs, 2);
        const int x_row = lrow + r4 * 8;
        if (lc == 0) {
          if (nparts > 1) {  // a part: M, l and O + b
            rowout[x_row] = make_float2(1.f, bs);
            *reinterpret_cast<float2*>(slot + x_row * 2) = make_float2(M[r4], ls);
          } else {
            const bool none = M[r4] == kPfNone && ls == 0.f;  // (a row of NaN scores has l NaN)
            const float inv = none ? 0.f : 1.f / ls;
            rowout[x_row] = make_float2(inv, bs * inv);
            if (x_row < rows) pf_lse(a, rq, h, row0 + x_row, none, M[r4], ls);
          }
        }
      }
      __syncwarp();
      const float2 ri = rowout[tid];  // a thread a row
      const bool have = tid < rows;
      const int qi = have ? (row0 + tid) / a.group : 0;
      uint16_t* dst = a.out + ((int64_t)(rq.tok0 + qi) * a.heads + h * a.group +
                               (have ? row0 + tid - qi * a.group : 0)) * D;
      float* pdst = slot + kPfRows * 2 + tid * D;
      if (nt > 0) {
        wait(&odone[t], 0);
        pf_fence_after();
      }
      const float ke = ri.x, ko = ri.x * 0.0625f;
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        uint32_t v[32];
        if (nt > 0) {
          pf_ld32(to + q * 32, v);
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) v[c] = 0;
        }
        if (have) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {  // columns hold channels 0 4 1 5 2 6 3 7 of each eight
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              f[e] = fmaf(__uint_as_float(v[c * 8 + e]), (e >> 1) & 1 ? ko : ke, ri.y);
            if (nparts > 1) {
              float4* d4 = reinterpret_cast<float4*>(pdst + q * 32 + c * 8);
              d4[0] = make_float4(f[0], f[2], f[4], f[6]);
              d4[1] = make_float4(f[1], f[3], f[5], f[7]);
            } else {
              *reinterpret_cast<uint4*>(dst + q * 32 + c * 8) =
                  make_uint4(pf_cvt2<F16>(f[0], f[2]), pf_cvt2<F16>(f[4], f[6]), pf_cvt2<F16>(f[1], f[3]),
                             pf_cvt2<F16>(f[5], f[7]));
            }
          }
        }
        __syncwarp();
      }
    }
  } else if (warp < kPfSoft + 4) {
    // ------------------------------------------------------------ unpack: a lane a token
    const int w = warp - kPfSoft, P = 1 << a.g.p_log2;
    const int32_t* table = a.table + (int64_t)r * a.max_blocks;
    constexpr int NW = D / 32;  // 16-byte words of a row
    uint4 kr[NW], vr[NW];
    uint32_t kp = 0, vp = 0;
    bool seen = false, seen_nx = false;
    const uint8_t* base = nullptr;
    int in = 0, entry = -1;
    auto page_of = [&](int j) {  // this lane's table entry of tile j
      const int tok = first() + j * kPfN + w * 32 + lane;
      return j < nt && tok < rq.kv ? table[tok >> a.g.p_log2] : -1;
    };
    auto locate = [&](int j) {   // tile j's row, from the entry loaded before
      const int tok = first() + j * kPfN + w * 32 + lane;
      seen_nx = entry >= 0 && entry < a.g.num_pages;  // -1 past the context
      in = tok & (P - 1);
      base = a.cache + ((int64_t)(seen_nx ? entry : 0) * a.g.hkv + h) * a.g.page_bytes;
    };
    auto load_k = [&]() {
      kp = vp = 0;
      if (seen_nx) {
        kp = __ldg(reinterpret_cast<const uint32_t*>(base + P * D + in * 4));
        vp = __ldg(reinterpret_cast<const uint32_t*>(base + P * D + 4 * P + in * 4));
#pragma unroll
        for (int x = 0; x < NW; ++x) kr[x] = __ldg(reinterpret_cast<const uint4*>(base + in * (D / 2) + x * 16));
      }
    };
    auto load_v = [&]() {
      if (seen_nx) {
#pragma unroll
        for (int x = 0; x < NW; ++x)
          vr[x] = __ldg(reinterpret_cast<const uint4*>(base + (P + in) * (D / 2) + x * 16));
      }
    };
#pragma unroll
    for (int x = 0; x < NW; ++x) kr[x] = vr[x] = make_uint4(0, 0, 0, 0);
    entry = page_of(0);
    locate(0);
    load_k();
    load_v();
    entry = page_of(1);
    const int trow = w * 32 + lane;
    // (the power of two first: with the rest it may be out of range where the pair brings it back)
    const float fac_q = pf_pow2(-qe), fac_m = a.scale * kLog2e, fac_s = fac_m * 0x1p24f;
#pragma unroll 1
    for (int j = 0; j < nt; ++j) {
      const int st = j & 1;
      seen = seen_nx;
      // pairs in fp32, the keys' times the softmax factors; a hidden token's count as 0
      float ks = h16_to_f32<F16>(kp & 0xFFFFu), km = h16_to_f32<F16>(kp >> 16);
      float vs = h16_to_f32<F16>(vp & 0xFFFFu), vm = h16_to_f32<F16>(vp >> 16);
      const bool bad = seen && !(fabsf(vs) <= FLT_MAX && fabsf(vm) <= FLT_MAX);
      if (!seen) ks = km = 0.f;
      if (!seen || bad) vs = vm = 0.f;
      vs = weight_scale(vs, vm);
      vm = fmaf(8.f, vs, vm);
      const uint32_t seen_m = __ballot_sync(0xffffffffu, seen), bad_m = __ballot_sync(0xffffffffu, bad);
      if (j >= 2) wait(&kempty[st], ((j >> 1) - 1) & 1);
      if (lane == 0) {
        masks[(j & 3) * 8 + w] = seen_m;
        masks[(j & 3) * 8 + 4 + w] = bad_m;
      }
      {
        float* p = reinterpret_cast<float*>(smem + C::o_par + (j & 3) * (kPfN * 16)) + (trow >> 1) * 8 + (trow & 1);
        p[0] = ks * fac_q * fac_s;
        p[2] = km * fac_q * fac_m;
        p[4] = vs;
        p[6] = vm;
      }
      uint8_t* kt = smem + C::o_k + st * C::block;
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        const uint32_t wv[4] = {kr[x].x, kr[x].y, kr[x].z, kr[x].w};
#pragma unroll
        for (int y = 0; y < 4; ++y)
          *reinterpret_cast<uint4*>(kt + pf_off<D>(trow, x * 4 + y)) = pf_unpack8(wv[y]);
      }
      pf_fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kfull[st]);
      locate(j + 1);
      load_k();
      if (j >= 2) wait(&vempty[st], ((j >> 1) - 1) & 1);
      uint8_t* vt = smem + C::o_v + st * C::block;
#pragma unroll
      for (int x = 0; x < NW; ++x) {
        const uint32_t wv[4] = {vr[x].x, vr[x].y, vr[x].z, vr[x].w};
#pragma unroll
        for (int y = 0; y < 4; ++y)
          *reinterpret_cast<uint4*>(vt + pf_off<D>(trow, x * 4 + y)) = pf_unpack8_mid(wv[y]);
      }
      pf_fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&vfull[st]);
      load_v();
      entry = page_of(j + 2);
    }
  } else if (nt > 0) {
    // ------------------------------------------------------------ MMA issue
    constexpr uint32_t id_s = pf_idesc(kPfN, false), id_o = pf_idesc(D, true);
    const uint64_t q0 = pf_desc(smem_u32(smem), 16, D * 16), k0 = pf_desc(smem_u32(smem + C::o_k), 16, D * 16),
                   v0 = pf_desc(smem_u32(smem + C::o_v), 1024, D * 16);
    auto scores = [&](int t, int st) {
      const uint64_t qd = q0 + t * (C::block >> 4), kd = k0 + st * (C::block >> 4);
      if (pf_elect()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const int o = ((k >> 2) * 1024 + (k & 3) * 32) >> 4;
          pf_mma_ss(tmem + t * 128, qd + o, kd + o, id_s, k > 0);
        }
        pf_commit(&sfull[t]);
      }
      __syncwarp();
    };
    auto product = [&](int t, int st, bool first, uint64_t* done) {
      const uint64_t vd = v0 + st * (C::block >> 4);
      if (pf_elect()) {
#pragma unroll
        for (int k = 0; k < kPfN / 16; ++k)
          pf_mma_ts(tmem + kO + t * D, tmem + t * 128 + k * 8, vd + k * (D * 2), id_o, !first || k > 0);
        if (done) pf_commit(done);
      }
      __syncwarp();
    };
#pragma unroll 1
    for (int j = 0; j < nt; ++j) {
      wait(&kfull[j & 1], (j >> 1) & 1);
      if (__any_sync(0xffffffffu, dead)) break;
#pragma unroll 1
      for (int t = 0; t < nblk; ++t) {
        if (j > 0) {
          if (t == 0) wait(&vfull[(j - 1) & 1], ((j - 1) >> 1) & 1);
          wait(&pready[t], (j - 1) & 1);
          __syncwarp();
          pf_fence_after();
          product(t, (j - 1) & 1, j == 1, t == nblk - 1 ? &vempty[(j - 1) & 1] : nullptr);
        } else {
          __syncwarp();
          pf_fence_after();
        }
        scores(t, j & 1);
      }
      if (pf_elect()) pf_commit(&kempty[j & 1]);
      __syncwarp();
    }
    wait(&vfull[(nt - 1) & 1], ((nt - 1) >> 1) & 1);
#pragma unroll 1
    for (int t = 0; t < nblk; ++t) {
      wait(&pready[t], (nt - 1) & 1);
      __syncwarp();
      pf_fence_after();
      product(t, (nt - 1) & 1, nt == 1, &odone[t]);
    }
  }
  __syncwarp();
  pf_fence_before();
  if (__syncthreads_or(dead) && warp == kPfSoft + 4) {  // queries and products still on their way
    if (pf_elect()) pf_commit(drain);
    mbar_drain(qbar, 0);
    mbar_drain(drain, 0);
    __syncwarp();
  }
  if (warp == kPfSoft + 4) {
    pf_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
  }
}

// The parts of split tiles -> out and lse, in the order of the parts: 32 rows of a tile at a
// time, four channels a thread.
constexpr int kPfJoinRows = 32;
template <bool F16, int D>
__global__ void __launch_bounds__(256) kv4_prefill_join(const AttnArgs a, const PfMeta* __restrict__ meta,
                                                        const float* __restrict__ parts) {
  pdl_wait();
  constexpr int G = kPfRows / kPfJoinRows;
  const int used = meta[kPfSlots].r;
#pragma unroll 1
  for (int at = blockIdx.x; at < used * G; at += gridDim.x) {
    const int slot = at / G;
    const PfMeta m = meta[slot];
    if (m.part != 0) continue;
    const AttnReq rq = attn_req(a, m.r);
    const int h = slot % a.g.hkv, row0 = m.tile * kPfRows;
    const int rows = min(rq.n * a.group - row0, kPfRows);
    const size_t stride = (size_t)a.g.hkv * (kPfRows * (D + 2));
    const float* base = parts + (size_t)slot * (kPfRows * (D + 2));
#pragma unroll 1
    for (int x = threadIdx.x; x < kPfJoinRows * (D / 4); x += 256) {
      const int row = at % G * kPfJoinRows + x / (D / 4), d4 = x % (D / 4);
      if (row >= rows) break;
      float top = kPfNone, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
      for (int i = 0; i < m.parts; ++i) {
        const float2 ml = *reinterpret_cast<const float2*>(base + i * stride + row * 2);
        const float4 v = reinterpret_cast<const float4*>(base + i * stride + kPfRows * 2 + row * D)[d4];
        const float nt = fmaxf(top, ml.x), f = ex2(top - nt), g = ex2(ml.x - nt);
        top = nt;
        l = fmaf(ml.y, g, l * f);
        o.x = fmaf(v.x, g, o.x * f);
        o.y = fmaf(v.y, g, o.y * f);
        o.z = fmaf(v.z, g, o.z * f);
        o.w = fmaf(v.w, g, o.w * f);
      }
      const bool none = top == kPfNone && l == 0.f;
      const float inv = none ? 0.f : 1.f / l;
      const int qi = (row0 + row) / a.group;
      *reinterpret_cast<uint2*>(a.out + ((int64_t)(rq.tok0 + qi) * a.heads + h * a.group + row0 + row - qi * a.group) * D +
                                d4 * 4) =
          make_uint2(pf_cvt2<F16>(o.x * inv, o.y * inv), pf_cvt2<F16>(o.z * inv, o.w * inv));
      if (d4 == 0) pf_lse(a, rq, h, row0 + row, none, top, l);
    }
  }
}

// what the slots hold | parts
constexpr size_t kPfMetaBytes = ((kPfSlots + 1) * sizeof(PfMeta) + 255) / 256 * 256;
size_t kv4_prefill_part_bytes() { return kPfMetaBytes + (size_t)kPfSlots * kPfRows * (128 + 2) * sizeof(float); }

int kv4_prefill(const AttnArgs& a, bool f16, int min_rows, bool zero_pad, void* parts, cudaStream_t st) {
  // an upper bound on the tiles: the lengths are on the device
  const int64_t tiles = ((int64_t)a.num_tokens * a.group + kPfRows - 1) / kPfRows + a.nreq;
  const int64_t grid = tiles * a.g.hkv + kPfSlots;  // and the split ones' parts
  if (grid > 0x7fffffffLL) return DIP_ERR_UNSUPPORTED;
  auto launch_as = [&](auto f, auto d, auto s) {
    constexpr int D = decltype(d)::value;
    auto kern = kv4_prefill_kernel<decltype(f)::value, D, decltype(s)::value>;
    const cudaError_t e = attn_smem<kv4_prefill_kernel<decltype(f)::value, D, decltype(s)::value>>(PfCfg<D>::total);
    if (e != cudaSuccess) return launch_status(e);
    PfMeta* meta = static_cast<PfMeta*>(parts);
    float* slots = reinterpret_cast<float*>(static_cast<uint8_t*>(parts) + kPfMetaBytes);
    int rc = launch_status(launch(kern, dim3((unsigned)(decltype(s)::value ? grid : grid - kPfSlots)), dim3(kPfThreads),
                                  PfCfg<D>::total, st, a, min_rows, (int)zero_pad, num_sms(), meta, slots));
    if (rc == DIP_OK && decltype(s)::value)
      rc = launch_status(launch(kv4_prefill_join<decltype(f)::value, D>, dim3(4 * num_sms()), dim3(256),
                                0, st, a, (const PfMeta*)meta, (const float*)slots));
    return rc;
  };
  // Whole tiles where there are surely many: what a last round leaves idle is little then.
  const bool whole = min_rows == 0 && (int64_t)a.num_tokens * a.group / kPfRows * a.g.hkv >= kPfWhole * num_sms();
  auto go = [&](auto f, auto d) {
    return whole ? launch_as(f, d, std::false_type{}) : launch_as(f, d, std::true_type{});
  };
  using T = std::true_type;
  using F = std::false_type;
  using D64 = std::integral_constant<int, 64>;
  using D128 = std::integral_constant<int, 128>;
  if (f16) return a.g.d == 64 ? go(T{}, D64{}) : go(T{}, D128{});
  return a.g.d == 64 ? go(F{}, D64{}) : go(F{}, D128{});
}

}  // namespace dip
