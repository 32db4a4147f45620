// kv4_pages.cu — page bookkeeping of the paged KV cache on the GPU: pages are
// taken from and given back to a free list, and the block table, slot map and
// lengths of a step are written without the host learning any length.
//
// Request r holds L_r tokens in ceil(L_r / P) pages and grows by n_r.  With
//   need_r = ceil((L_r + n_r) / P) - ceil(L_r / P),  first_r = sum_{s<r} need_s,
//   cu_r = sum_{s<r} n_s
// the j-th new page of request r is free[count - 1 - (first_r + j)], and the
// new token t = cu_r + i has slot table[r][(L_r + i) / P] * P + (L_r + i) % P.
// A few KB: bound by latency (lengths, scan, free list, table, slots one after another) and
// the launch.  64 requests by a token each 11 us a call with its five outputs, of which the
// kernel is about 3.
#include <cooperative_groups.h>

#include "kv4_common.cuh"

namespace dip {

constexpr int kPgThreads = 512;
constexpr int kPgMaxReq = 8192;  // requests whose prefix sums fit shared memory (96 KB)
constexpr int kPgCluster = 8;    // CTAs that share the token range of a large call

// Block-wide exclusive scan of three counters (blockDim = kPgThreads).
struct Int3 {
  long long a, b;
  int bad;
};
__device__ __forceinline__ Int3 pg_scan(Int3 v, Int3* wtot, Int3& tot) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Int3 s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long ta = __shfl_up_sync(0xffffffffu, s.a, o);
    const long long tb = __shfl_up_sync(0xffffffffu, s.b, o);
    if (lane >= o) { s.a += ta; s.b += tb; }
  }
  const int bad = __any_sync(0xffffffffu, v.bad);
  if (lane == 31) wtot[warp] = {s.a, s.b, bad};
  __syncthreads();
  Int3 base = {0, 0, 0};
  tot = {0, 0, 0};
#pragma unroll
  for (int w = 0; w < kPgThreads / 32; ++w) {
    const Int3 t = wtot[w];
    if (w < warp) { base.a += t.a; base.b += t.b; }
    tot.a += t.a;
    tot.b += t.b;
    tot.bad |= t.bad;
  }
  __syncthreads();
  return {base.a + s.a - v.a, base.b + s.b - v.b, 0};
}

// Largest r in [0, n) with pre[r] <= x (pre ascending, pre[0] = 0).
__device__ __forceinline__ int pg_find(const int* pre, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int m = (lo + hi) >> 1;
    if (pre[m] <= x) lo = m; else hi = m;
  }
  return lo;
}

struct PgArgs {
  const int32_t* lens;
  const int32_t* new_lens;
  int nreq, page;
  int32_t* table;
  int64_t max_blocks;
  const int32_t* free_list;
  int64_t free_cap;
  const int32_t* free_count;
  int32_t* lens_out;
  int32_t* cu_q;
  int64_t* slots;
  int64_t num_tokens;
  int32_t* free_count_out;
  int32_t* status;
};

// One cluster.  Every CTA scans all the lengths itself (a few KB from L2) and
// writes its share of the table entries and slots; the cluster barrier stands
// between the last read of the lengths and the first write, so the outputs may
// alias the inputs.  Launch latency bounds the small calls (64 requests), the
// slot stores the large ones.
__global__ void __launch_bounds__(kPgThreads) page_extend_kernel(const PgArgs a) {
  extern __shared__ int pg_smem[];
  int* s_len = pg_smem;                // [nreq] clamped lengths
  int* s_cu = s_len + a.nreq;          // [nreq] first new token
  int* s_first = s_cu + a.nreq;        // [nreq] first new page
  __shared__ Int3 wtot[kPgThreads / 32];
  const int tid = threadIdx.x;
  const int rank = blockIdx.x, nrank = gridDim.x;  // the grid is one cluster
  pdl_wait();
  const long long count = *a.free_count;
  Int3 carry = {0, 0, 0};
  for (int base = 0; base < a.nreq; base += kPgThreads) {
    const int r = base + tid;
    int len = 0, n = 0;
    Int3 v = {0, 0, 0};
    if (r < a.nreq) {
      len = max(a.lens[r], 0);
      n = max(a.new_lens[r], 0);
      const long long before = ((long long)len + a.page - 1) / a.page;
      const long long after = ((long long)len + n + a.page - 1) / a.page;
      v.a = n;
      v.b = after - before;
      v.bad = after > a.max_blocks || (long long)len + n > 0x7fffffffLL;
    }
    Int3 tot;
    const Int3 e = pg_scan(v, wtot, tot);
    if (r < a.nreq) {
      s_len[r] = len;
      s_cu[r] = (int)min(carry.a + e.a, 0x7fffffffLL);
      s_first[r] = (int)min(carry.b + e.b, 0x7fffffffLL);
    }
    carry.a += tot.a;
    carry.b += tot.b;
    carry.bad |= tot.bad;
  }
  // all or nothing: a call that cannot be served changes no length and no page
  int status = 0;
  if (carry.bad) status = -2;
  else if (carry.a > a.num_tokens) status = -1;
  else if (carry.b > count || count > a.free_cap)
    status = (int)min(max(carry.b - count, 1LL), 0x7fffffffLL);
  const bool ok = status == 0;
  if (nrank > 1) cooperative_groups::this_cluster().sync();
  else __syncthreads();
  pdl_launch_dependents();

  if (rank == 0) {
    for (int r = tid; r < a.nreq; r += kPgThreads) {
      const int nx = r + 1 < a.nreq ? s_cu[r + 1] : (int)min(carry.a, 0x7fffffffLL);
      a.lens_out[r] = s_len[r] + (ok ? nx - s_cu[r] : 0);
      a.cu_q[r] = ok ? s_cu[r] : 0;
    }
    if (tid == 0) {
      a.cu_q[a.nreq] = ok ? (int)carry.a : 0;
      *a.free_count_out = (int)(ok ? count - carry.b : count);
      *a.status = status;
    }
  }
  const int64_t step = (int64_t)nrank * kPgThreads;
  const int64_t me = (int64_t)rank * kPgThreads + tid;
  if (ok)
    for (int64_t j = me; j < carry.b; j += step) {
      const int r = pg_find(s_first, a.nreq, (int)j);
      const int64_t col = (s_len[r] + (int64_t)a.page - 1) / a.page + (j - s_first[r]);
      a.table[r * a.max_blocks + col] = a.free_list[count - 1 - j];
    }
  for (int64_t t = me; t < a.num_tokens; t += step) {
    int64_t slot = -1;
    if (ok && t < carry.a) {
      const int r = pg_find(s_cu, a.nreq, (int)t);
      const int len = s_len[r];
      const int pos = len + ((int)t - s_cu[r]);
      const int blk = pos / a.page, before = (int)(((int64_t)len + a.page - 1) / a.page);
      const int32_t pg = blk < before ? a.table[r * a.max_blocks + blk]
                                      : a.free_list[count - 1 - (s_first[r] + (blk - before))];
      if (pg >= 0) slot = (int64_t)pg * a.page + (pos - blk * a.page);
    }
    a.slots[t] = slot;
  }
}

// Gives the pages of the requests with done[r] != 0 back to the free list, in
// request and block order, and sets their lengths to 0.  One CTA.
__global__ void __launch_bounds__(kPgThreads)
page_release_kernel(const uint8_t* done, int nreq, int page, int32_t* lens, int32_t* table,
                    int64_t max_blocks, int32_t* free_list, int64_t free_cap,
                    int32_t* free_count) {
  __shared__ Int3 wtot[kPgThreads / 32];
  __shared__ int s_first[kPgThreads], s_held[kPgThreads];
  const int tid = threadIdx.x;
  pdl_wait();
  int64_t count = max(*free_count, 0);  // a negative count is an empty list
  for (int base = 0; base < nreq; base += kPgThreads) {
    const int r = base + tid;
    int held = 0;
    if (r < nreq && done[r])
      held = (int)min(((int64_t)max(lens[r], 0) + page - 1) / page, max_blocks);
    Int3 tot;
    const Int3 e = pg_scan({held, 0, 0}, wtot, tot);
    s_first[tid] = (int)e.a;
    s_held[tid] = held;
    __syncthreads();
    if (r < nreq && done[r]) lens[r] = 0;
    // a warp a request: its blocks are stored side by side
    for (int i = tid >> 5; i < kPgThreads; i += kPgThreads / 32)
      for (int b = tid & 31; b < s_held[i]; b += 32) {
        int32_t* entry = table + (int64_t)(base + i) * max_blocks + b;
        const int64_t at = count + s_first[i] + b;
        if (at < free_cap) free_list[at] = *entry;
        *entry = -1;
      }
    count += tot.a;
    __syncthreads();
  }
  if (tid == 0) *free_count = (int32_t)min(count, free_cap);
}

}  // namespace dip

using namespace dip;

extern "C" int dip_page_extend(const int32_t* lens, const int32_t* new_lens, int64_t nreq,
                               int64_t page_size, int32_t* block_table, int64_t max_blocks,
                               const int32_t* free_list, int64_t free_cap,
                               const int32_t* free_count, int32_t* lens_out, int32_t* cu_q,
                               int64_t* slots, int64_t num_tokens, int32_t* free_count_out,
                               int32_t* status, dip_stream_t stream) {
  if (nreq < 0 || page_size < 1 || page_size > (1 << 20) || max_blocks < 0 || num_tokens < 0 ||
      num_tokens > 0x7fffffffLL || free_cap < 0 || !free_count || !free_count_out || !status ||
      !cu_q)
    return DIP_ERR_ARG;
  if (nreq > 0 && (!lens || !new_lens || !lens_out || (max_blocks > 0 && !block_table)))
    return DIP_ERR_ARG;
  if ((num_tokens > 0 && !slots) || (free_cap > 0 && !free_list)) return DIP_ERR_ARG;
  if (nreq > kPgMaxReq) return DIP_ERR_UNSUPPORTED;
  const PgArgs a = {lens, new_lens, (int)nreq, (int)page_size, block_table, max_blocks, free_list,
                    free_cap, free_count, lens_out, cu_q, slots, num_tokens, free_count_out, status};
  const size_t smem = (size_t)nreq * 12;
  static_assert(kPgMaxReq * 12 <= 200 * 1024, "prefix sums fit shared memory");
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        page_extend_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPgMaxReq * 12);
    if (e != cudaSuccess) return launch_status(e);
  }
  // a cluster pays for itself once one CTA would store several slots a thread
  const unsigned ncta = num_tokens > 4 * kPgThreads ? kPgCluster : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ncta);
  cfg.blockDim = dim3(kPgThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (ncta > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = ncta;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return launch_status(cudaLaunchKernelEx(&cfg, page_extend_kernel, a));
}

extern "C" int dip_page_release(const uint8_t* done, int64_t nreq, int64_t page_size,
                                int32_t* lens, int32_t* block_table, int64_t max_blocks,
                                int32_t* free_list, int64_t free_cap, int32_t* free_count,
                                dip_stream_t stream) {
  if (nreq < 0 || nreq > (1 << 24) || page_size < 1 || max_blocks < 0 || free_cap < 0 ||
      !free_count)
    return DIP_ERR_ARG;
  if (nreq == 0) return DIP_OK;
  if (!done || !lens || (max_blocks > 0 && !block_table) || (free_cap > 0 && !free_list))
    return DIP_ERR_ARG;
  return launch_status(launch(page_release_kernel, dim3(1), dim3(kPgThreads), 0,
                              (cudaStream_t)stream, done, (int)nreq, (int)page_size, lens,
                              block_table, max_blocks, free_list, free_cap, free_count));
}
