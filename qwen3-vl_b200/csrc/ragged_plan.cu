// Ragged serving step: block tables, slot maps and positions from the
// requests' lengths, on the device.
//
// The reference keeps one contiguous cache per request and one start position
// per call (init_kv_cache, model_fused.py:224-232; the slice assignment of
// forward_layer, :244-246).  Here a step packs q[b] new tokens of each request
// b, which already holds past[b] positions in pages of P positions:
//   cu_q[b]   = sum of q[0..b-1]                  kv_lens[b] = past[b] + q[b]
//   need[b]   = ceil((past + q) / P) - ceil(past / P), taken from the free list
//               in request order: table[b, ceil(past/P) + i] = free[first[b] + i]
//               with first[b] = sum of need[0..b-1]
//   token t of request b (cu_q[b] <= t < cu_q[b+1]): position p = past[b] + t -
//               cu_q[b], slot = table[b, p / P] * P + p % P.
//
// Work split: every CTA scans the B lengths itself (two block scans over at
// most 8192 requests, into shared memory) and then takes its share of the
// tokens and of the new pages by binary search, so there is one launch and no
// grid-wide wait: a token whose page is new reads the free list, not the table
// entry that another CTA may be writing.
//
// Bound by latency: one chain of loads (lengths, then table or list), scans and
// stores.  Measured on B200 in a graph: 8 requests of one token 4.2 us, 1024
// requests with 79718 tokens (1.6 MB written) 7.9 us.
#include "common.cuh"

namespace q3 {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxB = 8192;

struct PlanParams {
  const int32_t* q_lens;
  const int32_t* past;
  int32_t* table;
  int64_t table_stride;
  const int32_t* free_pages;
  const int32_t* free_start;
  const int64_t* delta;
  int32_t* cu_q;
  int32_t* kv_lens;
  int32_t* requests;
  int64_t* positions;
  int64_t* slots;
  int32_t* counts;
  int64_t n_tokens;
  int B, width, page_tokens, n_free;
  int* err;
};

// Exclusive prefix sum of one value per thread over the CTA, in 64 bits;
// `total` gets the sum of all.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* total) {
  __shared__ int64_t warp_sums[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // warp_sums of an earlier scan has been read
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    const int64_t s = warp_sums[w];
    if (w < warp) before += s;
    all += s;
  }
  *total = all;
  return before + x - v;
}

// Index of the last entry of a[0..n] (ascending, a[0] = 0) that is <= t.
__device__ __forceinline__ int find_last(const int32_t* a, int n, int32_t t) {
  int lo = 0, hi = n;  // a[lo] <= t < a[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= t) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) ragged_plan_kernel(PlanParams p) {
  extern __shared__ int32_t sm[];
  int32_t* cu = sm;                // [B + 1]
  int32_t* first = sm + p.B + 1;   // [B + 1] pages taken before request b
  // No early launch of the next kernel: attn_decode_paged reads its table before
  // its own wait, and must not start before this one has written it.
  pdl_wait();
  const int tid = threadIdx.x;
  const int per = (p.B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  const int P = p.page_tokens;
  const int64_t cap = (int64_t)p.width * P;
  int bad = 0;

  int64_t mine = 0, total;
  for (int b = b0; b < b1; ++b) {
    const int q = p.q_lens[b], past = p.past[b];
    if (q < 0 || past < 0) bad = 0x901;
    else if (past > cap) bad = 0x902;  // clamped, with or without new tokens
    mine += max(q, 0);
  }
  int64_t at = block_scan(mine, &total);
  for (int b = b0; b < b1; ++b) {
    cu[b] = (int32_t)min64(at, p.n_tokens);
    at += max(p.q_lens[b], 0);
  }
  if (tid == 0) cu[p.B] = (int32_t)min64(total, p.n_tokens);
  if (blockIdx.x == 0) {
    if (bad) report_timeout(p.err, bad);
    if (tid == 0 && total > p.n_tokens) report_timeout(p.err, 0x904);
  }
  __syncthreads();

  // pages a request holds for its past positions, and those its tokens add
  auto pages = [&](int64_t n) { return (int)((min64(n, cap) + P - 1) / P); };
  auto need = [&](int b) {
    const int64_t past = max(p.past[b], 0);
    return pages(past + cu[b + 1] - cu[b]) - pages(past);
  };
  mine = 0;
  if (p.free_pages)
    for (int b = b0; b < b1; ++b) mine += need(b);
  int64_t taken;
  at = block_scan(mine, &taken);
  if (p.free_pages)
    for (int b = b0; b < b1; ++b) {
      first[b] = (int32_t)min64(at, INT32_MAX);
      at += need(b);
    }
  const int32_t n_new = (int32_t)min64(taken, INT32_MAX);
  if (tid == 0) first[p.B] = n_new;
  __syncthreads();
  // the list's entries not taken by earlier calls
  const int start = p.free_start ? min(max(*p.free_start, 0), p.n_free) : 0;
  const int32_t* fresh = p.free_pages + start;
  const int n_free = p.n_free - start;

  const int gtid = blockIdx.x * kPlanThreads + tid, gsize = gridDim.x * kPlanThreads;
  for (int b = gtid; b <= p.B; b += gsize) {
    p.cu_q[b] = cu[b];
    if (b < p.B)
      p.kv_lens[b] = (int32_t)min64((int64_t)max(p.past[b], 0) + cu[b + 1] - cu[b],
                                    min64(cap, INT32_MAX));
  }
  if (gtid == 0) {
    p.counts[0] = cu[p.B];
    p.counts[1] = n_new;
    if (n_new > n_free) report_timeout(p.err, 0x903);
  }
  for (int i = gtid; i < n_new; i += gsize) {
    const int b = find_last(first, p.B, i);
    const int j = pages(max(p.past[b], 0)) + i - first[b];
    p.table[b * p.table_stride + j] = i < n_free ? fresh[i] : -1;
  }
  const int32_t n_live = cu[p.B];
  for (int64_t t = gtid; t < p.n_tokens; t += gsize) {
    int32_t req = -1;
    int64_t pos = 0, slot = -1;
    if (t < n_live) {
      req = find_last(cu, p.B, (int32_t)t);
      const int64_t past = max(p.past[req], 0);
      pos = past + t - cu[req];
      if (pos < cap) {
        const int j = (int)((uint32_t)pos / (uint32_t)P);
        const int have = p.free_pages ? pages(past) : p.width;
        int pg = -1;
        if (j < have) {
          pg = p.table[req * p.table_stride + j];
        } else {
          const int64_t i = (int64_t)first[req] + j - have;
          if (i < n_free) pg = fresh[i];
        }
        if (pg >= 0) slot = (int64_t)pg * P + (pos - (int64_t)j * P);
        else report_timeout(p.err, 0x903);
      } else {
        report_timeout(p.err, 0x902);
      }
      if (p.delta) pos += p.delta[req];
    }
    p.requests[t] = req;
    p.positions[t] = pos;
    p.slots[t] = slot;
  }
}

}  // namespace
}  // namespace q3

extern "C" int q3_ragged_plan(const int32_t* q_lens, const int32_t* past_lens, int B,
                              int32_t* block_table, int64_t table_stride, int table_width,
                              int page_tokens, const int32_t* free_pages, int n_free,
                              const int32_t* free_start, const int64_t* rope_delta,
                              int64_t n_tokens, int32_t* cu_q, int32_t* kv_lens,
                              int32_t* requests, int64_t* positions, int64_t* slots,
                              int32_t* counts, q3_stream_t stream) {
  using namespace q3;
  Q3_REQUIRE(cu_q && counts && (n_tokens == 0 || (requests && positions && slots)) &&
                 (B == 0 || (q_lens && past_lens && block_table && kv_lens)),
             "q3_ragged_plan: null pointer");
  Q3_REQUIRE(B >= 0 && B <= kPlanMaxB, "q3_ragged_plan: B=%d outside [0, %d]", B, kPlanMaxB);
  Q3_REQUIRE(n_tokens >= 0 && n_tokens < (1ll << 31), "q3_ragged_plan: n_tokens=%lld",
             (long long)n_tokens);
  Q3_REQUIRE(page_tokens > 0 && page_tokens % 64 == 0,
             "q3_ragged_plan: page_tokens=%d must be a positive multiple of 64", page_tokens);
  Q3_REQUIRE(table_width > 0 && table_stride >= table_width,
             "q3_ragged_plan: table width %d, stride %lld", table_width,
             (long long)table_stride);
  Q3_REQUIRE((int64_t)table_width * page_tokens < (1ll << 31),
             "q3_ragged_plan: %d pages of %d positions pass 32-bit lengths", table_width,
             page_tokens);
  Q3_REQUIRE(n_free >= 0 && (free_pages || (n_free == 0 && !free_start)),
             "q3_ragged_plan: free list");
  Q3_REQUIRE(aligned(q_lens, 4) && aligned(past_lens, 4) && aligned(block_table, 4) &&
                 aligned(free_pages, 4) && aligned(free_start, 4) && aligned(rope_delta, 8) &&
                 aligned(cu_q, 4) && aligned(kv_lens, 4) && aligned(requests, 4) && aligned(positions, 8) &&
                 aligned(slots, 8) && aligned(counts, 4),
             "q3_ragged_plan: misaligned pointer");
  const size_t smem = (size_t)2 * (B + 1) * sizeof(int32_t);
  if (smem > 48 * 1024)
    Q3_CUDA_CHECK(cudaFuncSetAttribute(ragged_plan_kernel,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       2 * (kPlanMaxB + 1) * (int)sizeof(int32_t)));
  const int64_t want = (max64(n_tokens, B + 1) + kPlanThreads - 1) / kPlanThreads;
  PlanParams p{q_lens, past_lens, block_table, table_stride, free_pages, free_start, rope_delta,
               cu_q, kv_lens, requests, positions, slots, counts, n_tokens, B, table_width,
               page_tokens, n_free, device_error_word()};
  return launch_ex(ragged_plan_kernel, dim3((unsigned)min64(want, num_sms())),
                   dim3(kPlanThreads), smem, (cudaStream_t)stream, 1, p);
}
