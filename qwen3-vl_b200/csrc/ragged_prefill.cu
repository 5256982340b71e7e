// Ragged serving step: causal attention of packed prompt chunks over the paged
// K/V cache, on the 5th-generation tensor cores (tcgen05 + TMEM).
//
// The S > 1 eager attention of forward_layer (model_fused.py:248-262) for a
// batch whose requests bring different numbers of tokens on different cached
// prefixes (the reference, and attn_prefill_tc.cu, take one start position and
// one length for the batch): query i of request b (packed row cu_q[b] + i) sits
// at position kv_lens[b] - q_len + i and sees positions up to its own,
//   out = softmax(q K^T * scale) V,  head h over K/V head h / G, G = Hq / Hkv;
// a query that sees nothing gives zeros.
//
// An item is up to 256 query rows of one K/V head: T = 128 / G tokens times its
// G heads in each of two 128-row tiles, so one K/V tile serves all of them and
// any G up to 16 fills the tile (rows are (token, head) pairs, laid out by one
// 3-D TMA box).  Warp roles and the TMEM plan are those of the persistent
// variant in attn_prefill_tc.cu: warp 0 streams K and V tiles of 128 keys, warp
// 1 issues S(t) = Q(t) K^T and O(t) += P(t) V alternately for the two tiles, a
// warpgroup per tile runs the softmax, P goes back to TMEM as bf16 in place of
// S, and O is rescaled in place only when a row's maximum has grown by 2^8.
//
// Bound by the tensor pipe and the softmax (4 * 128 flops per visible pair).
// The lengths are only known on the device, so the keys of all items, plus two
// tiles' worth per item for its fixed cost, form one list that is cut into equal
// ranges, one per SM (fewer when the list has fewer tiles than SMs).  A cut inside
// an item goes to the nearest tile boundary, and within 2 tiles of the item's edge
// to the edge (a split costs about as much as a tile; with cuts moved by up to 1/16
// of a range the six-prompt case had 12 % more tiles on one SM than on average).
// Counting keys instead of tiles makes a request's sum a polynomial: with tiles it
// was a floor sum and a search, 16300 against 2900 cycles before the first load at
// 10/2 heads.  An item cut in the middle leaves fp32 pieces (O, base, sum) in the
// workspace and a second kernel joins them in CTA order: a 512-token chunk on a 32k
// cache fills every SM (its 64 items alone would fill 64).
// Measured on B200, 32/8 heads: that chunk 256 to 272 us by device (1065 to 1002
// TFLOP/s at the clock the power cap leaves in a long run, 1.66 GHz and 61 % of the
// tensor pipe under ncu); six prompts of 1100 to 4096 tokens 469 to 486 us (997 to
// 962); four prompts of up to 100 tokens at 4/1 heads 11.4 us.
#include <math.h>

#include "common.cuh"

namespace q3 {
namespace {

constexpr int kD = 128;
constexpr int kM = 128;                   // rows of a query tile
constexpr int kN = 128;                   // keys per K/V tile
constexpr int kThreads = 384;             // TMA, MMA, 2 idle, 2 x 4 softmax warps
// registers per thread: the launch has 168 (65536 / 384 in whole 8s), the first
// warpgroup gives some up and the softmax warpgroups take them; 88 + 2 * 208 =
// 3 * 168
constexpr int kRegsIo = 88;
constexpr int kRegsSoftmax = 208;
constexpr int kQBytes = kM * kD * 2;      // 32 KB per query tile (two 64-dim halves)
constexpr int kKVBytes = kN * kD * 2;     // 32 KB per K or V tile
constexpr int kHalf = kKVBytes / 2;       // one 64-dim half of 128 rows
constexpr int kBox = kHalf / 2;           // 64 rows of it: one TMA box of a page
constexpr int kOffK = 2 * kQBytes;
constexpr int kOffV = kOffK + 2 * kKVBytes;
constexpr int kOffOut = kOffV + 2 * kKVBytes;  // 4 KB per softmax warp: 32 rows x 64 dims
constexpr int kOffBar = kOffOut + 8 * 4096;
constexpr int kSmem = kOffBar + 256 + 1024;
static_assert(kSmem + 1024 <= 227 * 1024, "shared memory (1 KB for the static part)");
constexpr uint32_t kTmemCols = 512;       // S[0] S[1] O[0] O[1], 128 columns each
// a row's base moves when its maximum has grown by more than 2^16: P, l and O are
// relative to the base, so over n keys O may reach n 2^16 |V|, which fp32 holds
// while |V| is below 2^112 / n (2^97 at 32768 keys)
constexpr float kLazyLog2 = 16.0f;
constexpr int kMaxB = 65536;
constexpr int kMaxGrid = 512;
constexpr int kPieceRows = 2 * kM;
constexpr int kItemCost = 2 * kN;         // places of the work list an item takes besides its keys

struct RaggedPrefillParams {
  __nv_bfloat16* out;
  int64_t out_stride;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* cu_q;
  const int32_t* kv_lens;
  float* ws_o;    // [2 * grid][32][256] float4: dims 4i..4i+3 of a row, rows contiguous
  float* ws_ml;   // [2 * grid][2][256]  base (log2 units) and sum
  int4* ws_desc;  // [grid] {request or -1, K/V head, item, last CTA of the item}
  int B, Hkv, G, T, page_tokens, num_pages, capacity, n_tokens, causal;
  float scale_log2;
  int* err;
};

__device__ __forceinline__ bool warp_ok(uint64_t* bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}

// The exponentials of keys 64 * HALF .. + 63 of a row against base m: their bf16
// pairs and the sums of the unrounded values.  All on the MUFU pipe: with a
// quarter of them as polynomials on the FMA pipe the six-prompt case took 561 us
// against 520, measured with an epilogue that has since been replaced.
template <int HALF>
__device__ __forceinline__ void half_exps(const uint32_t (&rr)[kN], float scale_log2, float m,
                                          float2 (&sum)[2], uint32_t (&pk)[32]) {
  const float nbase = m == -INFINITY ? 0.f : -m;
  const float2 sc2 = make_float2(scale_log2, scale_log2);
  const float2 nb2 = make_float2(nbase, nbase);
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const float2 x = ffma2(make_float2(__uint_as_float(rr[HALF * 64 + 2 * i]),
                                       __uint_as_float(rr[HALF * 64 + 2 * i + 1])),
                           sc2, nb2);
    const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
    sum[i & 1] = fadd2(sum[i & 1], e);
    pk[i] = pack_bf16x2(e.x, e.y);
  }
}

// tc_mma_bf16, tc_mma_bf16_ts and tc_commit for one lane of a converged warp
// (`leader` != 0 in that lane), with descriptors as (low, high) words: the high
// word is the same for every operand here (stride 1024 bytes, version 1, 128-byte
// swizzle), the low word is the address and the leading offset.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi,
                                       uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t hi,
                                       uint32_t idesc, uint32_t accumulate, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void commit_if(uint64_t* bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          smem_u32(bar)),
      "r"(leader)
      : "memory");
}

template <int N>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// ---------------------------------------------------------------------------
// The work list.  Request b has n = ceil(q_len / 2T) items per K/V head; item i
// has tiles(i) = max(1, ceil(x / 128)) key tiles, x = the positions its last
// query sees.  An item takes x + kItemCost places in the list: its keys, whose
// sum over items is a polynomial (tiles would be a sum of roundings), and a fixed
// cost (loading its queries, an epilogue and a first tile that moves the base
// take about 5000 cycles; a tile takes about 3200).
// ---------------------------------------------------------------------------
struct Req {
  int q0, q_len, L, past;  // first packed row, queries, cached positions, L - q_len
};
__device__ __forceinline__ Req load_req(const RaggedPrefillParams& p, int b, bool* bad) {
  Req r;
  const int c0 = p.cu_q[b], c1 = p.cu_q[b + 1], L = p.kv_lens[b];
  r.q0 = min(max(c0, 0), p.n_tokens);
  r.q_len = min(max(c1, r.q0), p.n_tokens) - r.q0;
  r.L = min(max(L, 0), p.capacity);
  r.past = r.L - r.q_len;
  if (r.q0 != c0 || r.q0 + r.q_len != c1 || r.L != L) *bad = true;
  return r;
}
__device__ __forceinline__ int n_items(const RaggedPrefillParams& p, const Req& r) {
  return (r.q_len + 2 * p.T - 1) / (2 * p.T);
}
__device__ __forceinline__ int n_tiles(const RaggedPrefillParams& p, const Req& r, int i) {
  const int x = p.causal ? r.past + min(r.q_len, (i + 1) * 2 * p.T) : r.L;
  return x <= kN ? 1 : (x + kN - 1) / kN;
}
// places of item i, and of items [0, i) of one K/V head (a request whose tokens
// outnumber its positions counts as if it had none before them)
__device__ __forceinline__ int weight(const RaggedPrefillParams& p, const Req& r, int i) {
  if (!p.causal) return r.L + kItemCost;
  return max(r.past, 0) + min(r.q_len, (i + 1) * 2 * p.T) + kItemCost;
}
__device__ __forceinline__ int64_t places(const RaggedPrefillParams& p, const Req& r, int n, int i) {
  if (!p.causal) return (int64_t)i * (r.L + kItemCost);
  const int64_t base = (int64_t)max(r.past, 0) + kItemCost;
  const int64_t full = i < n ? i : max(n - 1, 0);  // items that end at (k + 1) * 2T
  const int64_t s = full * base + (int64_t)p.T * full * (full + 1);
  return i > full ? s + base + r.q_len : s;
}
// The item (of n) at place `rem` of one K/V head's items: the root of places(i) =
// rem in fp32, corrected by the exact sums.
__device__ __forceinline__ int item_at(const RaggedPrefillParams& p, const Req& r, int n,
                                       int64_t rem) {
  if (n == 1) return 0;
  const float h = (float)max(r.past, 0) + (float)(kItemCost + p.T), T = (float)p.T;
  const float d = h * h + 4.f * T * (float)rem;
  const float x = p.causal ? __fdividef(d * rsqrtf(d) - h, 2.f * T)
                           : __fdividef((float)rem, (float)(r.L + kItemCost));
  int i = min(max((int)x, 0), n - 1);
  while (i > 0 && places(p, r, n, i) > rem) --i;
  while (i + 1 < n && places(p, r, n, i + 1) <= rem) ++i;
  return i;
}
// A cut at place `pos` of an item of `w` places and nt tiles, as a tile boundary
// 0..nt: the nearest one, and within `snap` tiles of an edge the edge.  Cuts of
// the list are at least a tile apart, so those inside an item stay apart.
__device__ __forceinline__ int cut_tile(int64_t pos, int w, int nt, int snap) {
  if (pos >= w) return nt;
  const int t = min((int)(max64(pos - kItemCost + kN / 2, 0) / kN), nt);
  if (t < snap && 2 * t < nt) return 0;
  return nt - t < snap ? nt : t;
}

struct Piece {
  Req r;
  int b, kvh, item, t0, t1, nt;
  int64_t u;  // place of the item in the list
};
struct Walk {
  Req r;
  int b, kvh, item, n, nt, places, snap;
  int64_t pos, u, left;  // place inside the item, of the item, places left
  __device__ __forceinline__ bool next(const RaggedPrefillParams& p, Piece& w) {
    while (left > 0) {
      if (pos == places) {  // the next item
        u += places;
        pos = 0;
        if (++item == n) {
          item = 0;
          if (++kvh == p.Hkv) {
            kvh = 0;
            bool bad = false;
            do {
              if (++b >= p.B) return false;
              r = load_req(p, b, &bad);
              n = n_items(p, r);
            } while (n == 0);
          }
        }
        nt = n_tiles(p, r, item);
        places = weight(p, r, item);
      }
      const int64_t end = min64(pos + left, places);
      w.t0 = cut_tile(pos, places, nt, snap);
      w.t1 = cut_tile(end, places, nt, snap);
      left -= end - pos;
      pos = end;
      if (w.t0 < w.t1) {
        w.r = r;
        w.b = b;
        w.kvh = kvh;
        w.item = item;
        w.nt = nt;
        w.u = u;
        return true;
      }
    }
    return false;
  }
};

__global__ void __launch_bounds__(kThreads, 1)
    ragged_prefill_kernel(const __grid_constant__ CUtensorMap tmQ,
                          const __grid_constant__ CUtensorMap tmK,
                          const __grid_constant__ CUtensorMap tmV, RaggedPrefillParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const uint32_t s_base = smem_u32(smem);
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + kOffBar);
  uint64_t* q_full = bar + 0;
  uint64_t* k_full = bar + 1;    // [2]
  uint64_t* k_empty = bar + 3;   // [2] MMA commit after S of both tiles
  uint64_t* v_full = bar + 5;    // [2]
  uint64_t* v_empty = bar + 7;   // [2] MMA commit after PV of both tiles
  uint64_t* s_full = bar + 9;    // [tile] S (and the PV before it) complete
  uint64_t* p_full = bar + 11;   // [tile][half] P of 64 keys in TMEM: one arrival per warp
  uint64_t* o_final = bar + 15;  // [tile] the piece's last PV complete
  uint64_t* o_empty = bar + 17;  // [tile] the piece's O read out: one arrival per warp
  uint64_t* q_empty = bar + 19;  // the piece's S MMAs complete
  uint64_t* v_tail = bar + 20;   // copies of a V tile that reaches past the last position
  uint64_t* mma_done = bar + 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar + 23);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  __shared__ int64_t s_warp[kThreads / 32];
  __shared__ Walk s_walk;
  __shared__ int s_row[kM];  // token (low 16 bits) and head of a tile's row

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[2 * i], 4);
      mbar_init(&p_full[2 * i + 1], 4);
      mbar_init(&o_final[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    mbar_init(v_tail, 1);
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    s_walk.left = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // TMEM only after the wait: a kernel before this one may still have to
  // allocate its own on this SM
  pdl_wait();
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  // rows of the query tiles past the last (token, head) pair, which no copy
  // fills: zeros, so that they never move a base
  for (int i = p.T * p.G * 16 + threadIdx.x; i < kM * 16; i += kThreads)
#pragma unroll
    for (int t = 0; t < 2; ++t)
      *reinterpret_cast<uint4*>(smem + t * kQBytes + (i & 1) * (kQBytes / 2) + (i >> 4) * 128 +
                                ((i >> 1) & 7) * 16) = make_uint4(0, 0, 0, 0);
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  if (threadIdx.x < kM) {
    const int tk = threadIdx.x / p.G;
    // rows past the last (token, head) pair: a token past any request's end
    s_row[threadIdx.x] = (int)threadIdx.x < p.T * p.G ? tk | (threadIdx.x - tk * p.G) << 16 : 0x7fff;
  }

  // ---- this CTA's range of the list (every CTA scans the lengths) ----
  const int per = (p.B + kThreads - 1) / kThreads;
  const int b0 = min((int)threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);
  int64_t mine = 0;
  bool bad = false;
  for (int b = b0; b < b1; ++b) {
    const Req r = load_req(p, b, &bad);
    const int n = n_items(p, r);
    mine += places(p, r, n, n);
  }
  mine *= p.Hkv;
  if (bad && blockIdx.x == 0) report_timeout(p.err, 0x931);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) s_warp[warp] = incl;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch();
  const uint32_t tmem = *tmem_slot;
  int64_t before = incl - mine, U = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += s_warp[w];
    U += s_warp[w];
  }
  // CTA k's range [U k / nc, U (k + 1) / nc) by one division of U (in 32 bits
  // where it fits) and remainders below 2^18
  const int c = blockIdx.x;
  const uint32_t nc = (uint32_t)min64(gridDim.x, U / kN);  // CTAs that get places, a tile or more
  const int64_t share = nc == 0 ? 0 : U >> 32 ? U / nc : (int64_t)((uint32_t)U / nc);
  const uint32_t rest = (uint32_t)(U - share * nc);
  auto cut = [&](uint32_t k) { return share * k + (rest * k) / nc; };
  const int64_t u0 = c < (int)nc ? cut(c) : U, u1 = c < (int)nc ? cut(c + 1) : U;
  if (u0 < u1 && before <= u0 && u0 < before + mine) {
    int64_t at = before;
    for (int b = b0; b < b1; ++b) {
      const Req r = load_req(p, b, &bad);
      const int n = n_items(p, r);
      const int64_t per_head = places(p, r, n, n), all = per_head * p.Hkv;
      if (u0 < at + all) {
        const int64_t off = u0 - at;
        const int kvh = (int)(all >> 32 ? off / per_head : (uint32_t)off / (uint32_t)per_head);
        const int64_t rem = off - kvh * per_head;
        const int item = item_at(p, r, n, rem);
        s_walk.r = r;
        s_walk.b = b;
        s_walk.kvh = kvh;
        s_walk.item = item;
        s_walk.n = n;
        s_walk.nt = n_tiles(p, r, item);
        s_walk.places = weight(p, r, item);
        s_walk.snap = (int)min64(share / (8 * kN), 2);
        s_walk.pos = rem - places(p, r, n, item);
        s_walk.u = u0 - s_walk.pos;
        s_walk.left = u1 - u0;
        break;
      }
      at += all;
    }
  }
  __syncthreads();
  Piece w;

  if (warp < 4) {
    regs_dec<kRegsIo>();
    if (warp == 0) {
      Walk walk = s_walk;
      // ------------------------------ TMA producer ------------------------------
      int T = 0, ic = 0, nk = 0, nv = 0, tails = 0;
      bool ok = true;
      if (lane == 0) p.ws_desc[c] = make_int4(-1, 0, 0, 0);
      // (one vote on the flag, which another warp may set between two lanes' reads)
      while (ok && !__any_sync(0xffffffffu, *abort_flag != 0) && walk.next(p, w)) {
        // this lane's 64-key block of 16 tiles at a time: its first row in the pool, or
        // -1 (page_tokens % 64 == 0: a block never straddles); loaded ahead of Q
        auto block_row = [&](int j) {
          const int64_t key = ((int64_t)2 * j + lane) * 64;
          if (key >= w.r.L || 2 * j + lane >= 2 * w.t1) return -1;
          int pg = p.table[w.b * p.table_stride + (uint32_t)key / (uint32_t)p.page_tokens];
          if (pg < 0 || pg >= p.num_pages) {  // recorded, page 0 read in its place
            report_timeout(p.err, 0x932);
            pg = 0;
          }
          return (int)(((int64_t)pg * p.Hkv + w.kvh) * p.page_tokens +
                       (uint32_t)key % (uint32_t)p.page_tokens);
        };
        int row = block_row(w.t0);
        if (ic >= 1 && !warp_ok(q_empty, (ic - 1) & 1, p.err, 0x93b)) { ok = false; break; }
        if (lane == 0) {
          const int rows = p.T * p.G;  // rows of a tile that hold a (token, head) pair
          mbar_arrive_expect_tx(q_full, 2 * 2 * rows * 128);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int tok = w.r.q0 + (2 * w.item + t) * p.T;
            tma_load_3d(smem + t * kQBytes, &tmQ, q_full, 0, w.kvh * p.G, tok, kCacheEvictNormal);
            tma_load_3d(smem + t * kQBytes + kQBytes / 2, &tmQ, q_full, 64, w.kvh * p.G, tok,
                        kCacheEvictNormal);
          }
        }
        ++ic;
        for (int j = w.t0; j < w.t1; ++j, ++T) {
          const int s = T & 1, k = (2 * (j - w.t0)) & 31;
          if (k == 0 && j > w.t0) row = block_row(j);
          // blocks past the last position are masked: any valid rows do
          const int ya = max(__shfl_sync(0xffffffffu, row, k), 0);
          const int yb0 = __shfl_sync(0xffffffffu, row, k + 1);
          const int yb = yb0 < 0 ? ya : yb0;
          if (T >= 2 && !warp_ok(&k_empty[s], ((T >> 1) - 1) & 1, p.err, 0x933)) { ok = false; break; }
          if (lane == 0) {
            uint8_t* dk = smem + kOffK + s * kKVBytes;
            mbar_arrive_expect_tx(&k_full[s], kKVBytes);
            tma_load_2d(dk, &tmK, &k_full[s], 0, ya, kCacheEvictNormal);
            tma_load_2d(dk + kBox, &tmK, &k_full[s], 0, yb, kCacheEvictNormal);
            tma_load_2d(dk + kHalf, &tmK, &k_full[s], 64, ya, kCacheEvictNormal);
            tma_load_2d(dk + kHalf + kBox, &tmK, &k_full[s], 64, yb, kCacheEvictNormal);
          }
          nk = T + 1;
          if (T >= 2 && !warp_ok(&v_empty[s], ((T >> 1) - 1) & 1, p.err, 0x934)) { ok = false; break; }
          const int valid = w.r.L - j * kN;  // keys of the tile that exist, if below 128
          uint64_t* vb = valid < kN ? v_tail : &v_full[s];
          uint8_t* dv = smem + kOffV + s * kKVBytes;
          if (lane == 0) {
            mbar_arrive_expect_tx(vb, kKVBytes);
            tma_load_2d(dv, &tmV, vb, 0, ya, kCacheEvictNormal);
            tma_load_2d(dv + kBox, &tmV, vb, 0, yb, kCacheEvictNormal);
            tma_load_2d(dv + kHalf, &tmV, vb, 64, ya, kCacheEvictNormal);
            tma_load_2d(dv + kHalf + kBox, &tmV, vb, 64, yb, kCacheEvictNormal);
          }
          if (valid < kN) {
            // V rows past the last position hold whatever the page held before
            // (NaN included) and 0 * V must be 0: they become zeros here, before
            // the MMA warp is told of the tile
            ++tails;
            if (!warp_ok(v_tail, (tails - 1) & 1, p.err, 0x935)) { ok = false; break; }
            const int v0 = max(valid, 0);
            for (int i = lane; i < (kN - v0) * 16; i += 32)  // 16-byte pieces of both halves
              *reinterpret_cast<uint4*>(dv + ((i >> 3) & 1) * kHalf + (v0 + (i >> 4)) * 128 +
                                        (i & 7) * 16) = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[s]);
          }
          nv = T + 1;
        }
        if (w.t0 == 0 && w.t1 < w.nt) {
          // the item goes on in the next CTAs: find the last of them
          int last = c;
          for (uint32_t k0 = c + 1; k0 < nc; k0 += 32) {
            const uint32_t k = k0 + lane;
            const bool in =
                k < nc && cut_tile(cut(min(k, nc)) - w.u, walk.places, w.nt, walk.snap) < w.nt;
            const int n = __popc(__ballot_sync(0xffffffffu, in));
            last += n;
            if (n < 32) break;
          }
          if (lane == 0) p.ws_desc[c] = make_int4(w.b, w.kvh, w.item, last);
        }
      }
      if (!ok) *abort_flag = 1;
      // The copies this warp issued land before the CTA exits.  They have when all went
      // well; when a wait ran out, here or in another warp, the last ones of each
      // barrier may not have.
      if (lane == 0) {
        if (ic > 0) mbar_wait(q_full, (ic - 1) & 1, nullptr, 0);
        for (int j = max(0, nk - 2); j < nk; ++j)
          mbar_wait(&k_full[j & 1], (j >> 1) & 1, nullptr, 0);
        for (int j = max(0, nv - 2); j < nv; ++j)
          mbar_wait(&v_full[j & 1], (j >> 1) & 1, nullptr, 0);
        if (tails > 0) mbar_wait(v_tail, (tails - 1) & 1, nullptr, 0);
      }
    } else if (warp == 1) {
      // ------------------------------ MMA issuer --------------------------------
      // One thread for both tiles, in turn: S(t) of the next keys goes out behind
      // P V(t), so the tiles stay half a period apart and one tile's softmax runs
      // under the other's MMAs.  (A thread per tile let them fall into step, both
      // in softmax and then both waiting for the tensor pipe: 5500 cycles per
      // K/V tile.)
      // The whole warp runs the loop and every MMA is predicated on one elected
      // lane: control flow and descriptors stay warp-uniform, so the descriptor
      // words live in uniform registers (a lane-0 branch issued an MMA every 96
      // cycles; one takes 64).
      Walk walk = s_walk;
      constexpr uint32_t idesc_s = umma_idesc_bf16(kM, kN);
      constexpr uint32_t idesc_o = umma_idesc_bf16_bmn(kM, kD);
      const uint32_t leader = elect_one();
      const uint32_t base = __shfl_sync(0xffffffffu, s_base, 0);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint32_t lo_q = (uint32_t)umma_desc_k_sw128(base);
      const uint32_t lo_k = (uint32_t)umma_desc_k_sw128(base + kOffK);
      const uint32_t lo_v = (uint32_t)umma_desc_mn_sw128(base + kOffV, kHalf, 1024u);
      auto issue_s = [&](uint32_t stage, int t) {
        const uint32_t dq = lo_q + t * (kQBytes >> 4), dk = lo_k + stage * (kKVBytes >> 4);
        const uint32_t tS = tm + t * kN;
#pragma unroll
        for (int ks = 0; ks < kD / 16; ++ks)
          mma_ss(tS, dq + ((ks >> 2) * (kQBytes / 2) >> 4) + 2 * (ks & 3),
                 dk + ((ks >> 2) * kHalf >> 4) + 2 * (ks & 3), kDescHi, idesc_s, ks != 0, leader);
        commit_if(&s_full[t], leader);
      };
      // keys 64 * half .. + 63 of a tile
      auto issue_pv = [&](uint32_t stage, int t, int half, uint32_t accumulate) {
        const uint32_t dv = lo_v + stage * (kKVBytes >> 4) + half * (4 * 2048 >> 4);
        const uint32_t dp = tm + t * kN + half * 32, tO = tm + 2 * kN + t * kD;
        mma_ts(tO, dp, dv, kDescHi, idesc_o, accumulate, leader);
#pragma unroll
        for (int ks = 1; ks < 4; ++ks)
          mma_ts(tO, dp + ks * 8, dv + (ks * 2048 >> 4), kDescHi, idesc_o, 1u, leader);
      };
      bool ok = true;
      uint32_t T = 0, ic = 0;
      while (ok && walk.next(p, w)) {
        const int n_kb = __shfl_sync(0xffffffffu, w.t1 - w.t0, 0);
        ok = !__any_sync(0xffffffffu, *abort_flag != 0) &&
             warp_ok(q_full, ic & 1, p.err, 0x936) &&
             warp_ok(&k_full[T & 1], (T >> 1) & 1, p.err, 0x937);
        if (!ok) break;
        tc_fence_after();
        issue_s(T & 1, 0);
        issue_s(T & 1, 1);
        commit_if(&k_empty[T & 1], leader);
        if (n_kb == 1) commit_if(q_empty, leader);
        for (int j = 0; ok && j < n_kb; ++j, ++T) {
          ok = warp_ok(&v_full[T & 1], (T >> 1) & 1, p.err, 0x938);
          if (!ok) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            ok = ok &&
                 (j > 0 || ic == 0 || warp_ok(&o_empty[t], (ic - 1) & 1, p.err, 0x93a)) &&
                 warp_ok(&p_full[2 * t], T & 1, p.err, 0x939);
            if (!ok) break;
            tc_fence_after();
            issue_pv(T & 1, t, 0, j > 0 ? 1u : 0u);
            ok = warp_ok(&p_full[2 * t + 1], T & 1, p.err, 0x939);
            if (!ok) break;
            tc_fence_after();
            issue_pv(T & 1, t, 1, 1u);
            if (t == 1) commit_if(&v_empty[T & 1], leader);
            if (j + 1 < n_kb) {
              if (t == 0) ok = warp_ok(&k_full[(T + 1) & 1], ((T + 1) >> 1) & 1, p.err, 0x937);
              if (!ok) break;
              tc_fence_after();
              issue_s((T + 1) & 1, t);
              if (t == 1) {
                commit_if(&k_empty[(T + 1) & 1], leader);
                if (j + 2 == n_kb) commit_if(q_empty, leader);  // the piece's last S MMAs
              }
            } else {
              commit_if(&o_final[t], leader);
            }
          }
        }
        ++ic;
      }
      if (!ok) *abort_flag = 1;
      // every MMA issued above has completed before TMEM is released
      commit_if(mma_done, leader);
      warp_ok(mma_done, 0, nullptr, 0);
    }
  } else {
    // -------------------------------- softmax ---------------------------------
    regs_inc<kRegsSoftmax>();
    Walk walk = s_walk;
    const int t = (warp >> 2) - 1;  // query tile
    const int quarter = warp & 3;   // TMEM lane quarter of this warp
    const int row = quarter * 32 + lane;
    const int tok_in = row / p.G;
    const bool row_used = row < p.T * p.G;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_col = tmem + lane_off + t * kN;
    const uint32_t o_col = tmem + lane_off + 2 * kN + t * kD;
    bool ok = true;
    uint32_t T = 0, ic = 0;
    while (ok && walk.next(p, w)) {
      const int n_kb = w.t1 - w.t0;
      const int tile_tok = (2 * w.item + t) * p.T;
      const int tok = tile_tok + tok_in;
      const bool live = row_used && tok < w.r.q_len;
      // the last position this row sees, and the fewest any row of the tile sees
      const int see = !live ? -1 : p.causal ? w.r.past + tok : w.r.L - 1;
      const int see_min = p.causal ? min(w.r.past + tile_tok, w.r.L - 1) : w.r.L - 1;
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < n_kb; ++j, ++T) {
        ok = !__any_sync(0xffffffffu, *abort_flag != 0) && warp_ok(&s_full[t], T & 1, p.err, 0x93c);
        if (!ok) break;
        tc_fence_after();
        uint32_t rr[kN];  // raw scores; scaling is folded into the exponent's FMA
#pragma unroll
        for (int cc = 0; cc < kN / 32; ++cc)
          tmem_ld_32cols(s_col + cc * 32, *reinterpret_cast<uint32_t(*)[32]>(&rr[cc * 32]));
        tc_wait_ld();
        const int kbase = (w.t0 + j) * kN;
        if (kbase + kN - 1 > see_min) {
          const int lim = see - kbase;  // the last key this row sees
#pragma unroll
          for (int cc = 0; cc < kN / 32; ++cc) {
            const int n = lim - cc * 32;
            const uint32_t seen = n >= 31 ? 0xffffffffu : n < 0 ? 0u : (2u << n) - 1u;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((seen >> i) & 1)) rr[cc * 32 + i] = __float_as_uint(-INFINITY);
          }
        }
        // P = 2^(S scale - base).  The first 64 keys' exponentials are taken
        // against the old base while the tile's maximum is still being found, and
        // taken again in a tile that moves the base: an item's first, and one
        // where the maximum has grown by 2^16.  (No branch around them: the
        // compiler overlaps them with the maximum.)
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[32];
        half_exps<0>(rr, p.scale_log2, m_used, sum, pk);
        float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kN; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            mq[q] = max3f(mq[q], __uint_as_float(rr[i + 2 * q]), __uint_as_float(rr[i + 2 * q + 1]));
        const float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]));
        // scale > 0, so the maximum of the scaled scores is the scaled maximum
        const float m_new = fmaxf(m_used, mx * p.scale_log2);
        const bool move = m_new > m_used + kLazyLog2;  // -inf + 16 = -inf
        if (__any_sync(0xffffffffu, move)) {
          const bool rescale = move && j > 0 && m_used != -INFINITY;
          const float corr = rescale ? ex2_approx(m_used - m_new) : 1.f;
          if (move) {
            l *= ex2_approx(m_used - m_new);  // m_used = -inf: l is 0 and stays 0
            m_used = m_new;
          }
          sum[0] = sum[1] = make_float2(0.f, 0.f);
          half_exps<0>(rr, p.scale_log2, m_used, sum, pk);
          if (__any_sync(0xffffffffu, rescale)) {
            // O holds the piece's tiles before j, complete (covered by the commit
            // of this S): move it to the new base before this PV adds to it
#pragma unroll 1
            for (int cc = 0; cc < kD / 16; ++cc) {
              uint32_t r16[16];
              tmem_ld_16cols(o_col + cc * 16, r16);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                r16[i] = __float_as_uint(__uint_as_float(r16[i]) * corr);
              tmem_st_16cols(o_col + cc * 16, r16);
            }
          }
        }
        tmem_st_32cols(s_col, pk);  // P in place of S: 64 keys in 32 columns
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t]);
        half_exps<1>(rr, p.scale_log2, m_used, sum, pk);
        tmem_st_32cols(s_col + 32, pk);
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + 1]);
        l += (sum[0].x + sum[1].x) + (sum[0].y + sum[1].y);
      }
      ok = ok && warp_ok(&o_final[t], ic & 1, p.err, 0x93d);
      if (!ok) break;
      tc_fence_after();
      if (w.t0 == 0 && w.t1 == w.nt) {
        const float inv = l > 0.f ? 1.f / l : 0.f;
        // 64 dims of the warp's 32 rows at a time through shared memory, so that
        // eight lanes write 128 bytes of a row (a thread writing its own row
        // touched 32 lines per store: 5000 cycles per item)
        uint8_t* stage = smem + kOffOut + (warp - 4) * 4096;
        const int r4 = lane >> 3, u8 = lane & 7;
        const int n_tok = min(w.r.q_len - tile_tok, p.T);  // tokens of the tile
        __nv_bfloat16* dst =
            p.out + (int64_t)(w.r.q0 + tile_tok) * p.out_stride + (int64_t)w.kvh * p.G * kD;
#pragma unroll
        for (int hd = 0; hd < 2; ++hd) {
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            uint32_t r32[32];
            tmem_ld_32cols(o_col + hd * 64 + cc * 32, r32);
            tc_wait_ld();
#pragma unroll
            for (int d = 0; d < 4; ++d) {
              uint4 u;
              u.x = pack_bf16x2(__uint_as_float(r32[8 * d]) * inv, __uint_as_float(r32[8 * d + 1]) * inv);
              u.y = pack_bf16x2(__uint_as_float(r32[8 * d + 2]) * inv,
                                __uint_as_float(r32[8 * d + 3]) * inv);
              u.z = pack_bf16x2(__uint_as_float(r32[8 * d + 4]) * inv,
                                __uint_as_float(r32[8 * d + 5]) * inv);
              u.w = pack_bf16x2(__uint_as_float(r32[8 * d + 6]) * inv,
                                __uint_as_float(r32[8 * d + 7]) * inv);
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((cc * 4 + d) ^ (lane & 7)) << 4)) = u;
            }
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + r4, rt = quarter * 32 + r;  // row of the warp, of the tile
            const uint4 u =
                *reinterpret_cast<const uint4*>(stage + r * 128 + ((u8 ^ (r & 7)) << 4));
            const int tk = s_row[rt] & 0xffff, hh = s_row[rt] >> 16;
            if (tk < n_tok)
              *reinterpret_cast<uint4*>(dst + tk * p.out_stride + hh * kD + hd * 64 + u8 * 8) = u;
          }
          __syncwarp();
        }
      } else {
        // a piece of an item: O relative to m_used, the base and the sum.  A
        // piece that began inside its item has the even slot.
        const int64_t slot = 2 * c + (w.t0 == 0 ? 1 : 0);
        const int r256 = t * kM + row;
        if (live) {
          p.ws_ml[(slot * 2) * kPieceRows + r256] = m_used;
          p.ws_ml[(slot * 2 + 1) * kPieceRows + r256] = l;
        }
        float4* dst = reinterpret_cast<float4*>(p.ws_o) + slot * 32 * kPieceRows + r256;
#pragma unroll
        for (int cc = 0; cc < kD / 32; ++cc) {
          uint32_t r32[32];
          tmem_ld_32cols(o_col + cc * 32, r32);
          tc_wait_ld();
          if (live) {
#pragma unroll
            for (int d = 0; d < 8; ++d)
              dst[(cc * 8 + d) * kPieceRows] =
                  make_float4(__uint_as_float(r32[4 * d]), __uint_as_float(r32[4 * d + 1]),
                              __uint_as_float(r32[4 * d + 2]), __uint_as_float(r32[4 * d + 3]));
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_empty[t]);
      ++ic;
    }
    if (!ok) *abort_flag = 1;
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the pieces of the item that CTA c left unfinished: slots 2c+1, 2(c+1),
// ..., 2*last, in that order.  Eight CTAs per item, 16 dims each.  With few pieces
// (two is the usual case) a thread takes one of the 256 rows; with many pieces of
// few rows (nine queries on a 17k cache) the warps share the pieces of 32 rows at
// a time: 50 -> 21 us for that call, whose 130 pieces a thread took one by one.
constexpr int kJoinD4 = 4;      // float4 columns (of 32) at a time
constexpr int kJoinWarps = 8;
// the workspace slot of piece i of the item that CTA c left unfinished
__device__ __forceinline__ int64_t piece_slot(int c, int i) {
  return i == 0 ? 2 * c + 1 : 2 * (c + i);
}
struct JoinRow {
  int c, first, step, n, r256;  // pieces first, first + step, ... below n of row r256
};
// The row's maximum over the pieces, and sums and dims 4 d40 .. relative to it.
// Loads of two pieces are issued before any is used (four take 126 registers,
// and CTAs without an item then leave more slowly).
constexpr int kJoinBatch = 2;
__device__ __forceinline__ float join_max(const RaggedPrefillParams& p, const JoinRow& j) {
  float M = -INFINITY;
  for (int i0 = j.first; i0 < j.n; i0 += kJoinBatch * j.step) {
    float m[kJoinBatch];
#pragma unroll
    for (int u = 0; u < kJoinBatch; ++u) {
      const int i = min(i0 + u * j.step, j.n - 1);  // the last again: no change
      m[u] = p.ws_ml[piece_slot(j.c, i) * 2 * kPieceRows + j.r256];
    }
#pragma unroll
    for (int u = 0; u < kJoinBatch; ++u) M = fmaxf(M, m[u]);
  }
  return M;
}
__device__ __forceinline__ float join_sum(const RaggedPrefillParams& p, const JoinRow& j, float M,
                                          int d40, float4 (&a)[kJoinD4]) {
#pragma unroll
  for (int k = 0; k < kJoinD4; ++k) a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
  for (int i0 = j.first; i0 < j.n; i0 += kJoinBatch * j.step) {
    float m[kJoinBatch], li[kJoinBatch];
    float4 x[kJoinBatch][kJoinD4];
#pragma unroll
    for (int u = 0; u < kJoinBatch; ++u) {
      const int i = i0 + u * j.step;
      const int64_t slot = piece_slot(j.c, min(i, j.n - 1));
      const float* ml = p.ws_ml + slot * 2 * kPieceRows + j.r256;
      m[u] = i < j.n ? ml[0] : -INFINITY;
      li[u] = ml[kPieceRows];
      const float4* src =
          reinterpret_cast<const float4*>(p.ws_o) + (slot * 32 + d40) * kPieceRows + j.r256;
#pragma unroll
      for (int k = 0; k < kJoinD4; ++k) x[u][k] = src[k * kPieceRows];
    }
#pragma unroll
    for (int u = 0; u < kJoinBatch; ++u) {
      const float f = m[u] == -INFINITY ? 0.f : ex2_approx(m[u] - M);
      // a piece of which the row sees nothing, or none; but a NaN score, which no
      // maximum shows, has made its piece's sum and O NaN, and the row is NaN
      if (f == 0.f && li[u] == li[u]) continue;
      l = fmaf(f, li[u], l);
#pragma unroll
      for (int k = 0; k < kJoinD4; ++k) {
        a[k].x = fmaf(f, x[u][k].x, a[k].x);
        a[k].y = fmaf(f, x[u][k].y, a[k].y);
        a[k].z = fmaf(f, x[u][k].z, a[k].z);
        a[k].w = fmaf(f, x[u][k].w, a[k].w);
      }
    }
  }
  return l;
}
__device__ __forceinline__ void join_store(__nv_bfloat16* dst, const float4 (&a)[kJoinD4],
                                           float l) {
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int k = 0; k < kJoinD4; k += 2) {
    uint4 u;
    u.x = pack_bf16x2(a[k].x * inv, a[k].y * inv);
    u.y = pack_bf16x2(a[k].z * inv, a[k].w * inv);
    u.z = pack_bf16x2(a[k + 1].x * inv, a[k + 1].y * inv);
    u.w = pack_bf16x2(a[k + 1].z * inv, a[k + 1].w * inv);
    *reinterpret_cast<uint4*>(dst + k * 4) = u;
  }
}
__global__ void __launch_bounds__(kJoinWarps * 32) ragged_prefill_join(RaggedPrefillParams p) {
  __shared__ float s_m[kJoinWarps][32], s_l[kJoinWarps][32];
  __shared__ float4 s_acc[kJoinWarps][kJoinD4][32];
  pdl_launch();
  pdl_wait();
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int d40 = blockIdx.y * kJoinD4;
  const int4 d = p.ws_desc[c];
  if (d.x < 0) return;
  const int n = d.w - c + 1;
  bool bad = false;
  const Req r = load_req(p, d.x, &bad);
  // rows of query tile t that hold a token of the request
  auto live_rows = [&](int t) {
    return max(min(r.q_len - (2 * d.z + t) * p.T, p.T), 0) * p.G;
  };
  auto out_of = [&](int r256) {
    const int t = r256 / kM, row = r256 - t * kM, tok_in = row / p.G;
    return p.out + (int64_t)(r.q0 + (2 * d.z + t) * p.T + tok_in) * p.out_stride +
           (int64_t)(d.y * p.G + row - tok_in * p.G) * kD + d40 * 4;
  };
  float4 a[kJoinD4];
  // A thread with its row's n pieces takes about 430 n cycles (its loads wait in
  // turn); eight warps take 54 n + 1500 for each of the blocks of 32 live rows.
  const int blocks = (live_rows(0) + 31) / 32 + (live_rows(1) + 31) / 32;
  if (blocks * (n + 28) >= 8 * n) {
    const int r256 = threadIdx.x;
    if (r256 % kM >= live_rows(r256 / kM)) return;
    const JoinRow j{c, 0, 1, n, r256};
    const float l = join_sum(p, j, join_max(p, j), d40, a);
    join_store(out_of(r256), a, l);
    return;
  }
#pragma unroll 1
  for (int r0 = 0; r0 < kPieceRows; r0 += 32) {  // lane = row
    const int live = live_rows(r0 / kM) - r0 % kM;
    if (live <= 0) continue;
    const JoinRow j{c, warp, kJoinWarps, n, r0 + lane};
    s_m[warp][lane] = join_max(p, j);
    __syncthreads();
    float M = s_m[0][lane];
#pragma unroll
    for (int i = 1; i < kJoinWarps; ++i) M = fmaxf(M, s_m[i][lane]);
    s_l[warp][lane] = join_sum(p, j, M, d40, a);
#pragma unroll
    for (int k = 0; k < kJoinD4; ++k) s_acc[warp][k][lane] = a[k];
    __syncthreads();
    if (warp == 0 && lane < live) {  // the warps' sums in order
      float l = s_l[0][lane];
#pragma unroll
      for (int i = 1; i < kJoinWarps; ++i) {
        l += s_l[i][lane];
#pragma unroll
        for (int k = 0; k < kJoinD4; ++k) {
          const float4 x = s_acc[i][k][lane];
          a[k].x += x.x;
          a[k].y += x.y;
          a[k].z += x.z;
          a[k].w += x.w;
        }
      }
      join_store(out_of(r0 + lane), a, l);
    }
    __syncthreads();
  }
}

int prefill_grid() { return (int)min64(num_sms(), kMaxGrid); }

size_t prefill_ws(size_t* off_ml, size_t* off_desc) {
  const size_t slots = 2 * (size_t)prefill_grid();
  size_t n = slots * kPieceRows * kD * 4;
  *off_ml = n;
  n += slots * kPieceRows * 8;
  *off_desc = n;
  return n + prefill_grid() * sizeof(int4);
}

}  // namespace
}  // namespace q3

extern "C" size_t q3_attn_prefill_ragged_workspace_bytes(void) {
  size_t a, b;
  return q3::prefill_ws(&a, &b);
}

extern "C" int q3_attn_prefill_ragged(const void* q, int64_t q_stride, const void* k_pages,
                                      const void* v_pages, void* out, int64_t out_stride,
                                      int64_t n_tokens, int B, int Hq, int Hkv, int head_dim,
                                      const int32_t* block_table, int64_t table_stride,
                                      int table_width, int page_tokens, int64_t num_pages,
                                      const int32_t* cu_q, const int32_t* kv_lens, int causal,
                                      float scale, void* workspace, size_t workspace_bytes,
                                      q3_stream_t stream) {
  using namespace q3;
  Q3_REQUIRE(head_dim == kD, "q3_attn_prefill_ragged: head_dim must be 128 (got %d)", head_dim);
  Q3_REQUIRE(n_tokens >= 0 && n_tokens < (1ll << 31) - 256 && B >= 0 && B <= kMaxB && Hq > 0 &&
                 Hkv > 0 && Hkv <= 1024 && Hq % Hkv == 0,
             "q3_attn_prefill_ragged: bad shape n=%lld B=%d Hq=%d Hkv=%d", (long long)n_tokens, B,
             Hq, Hkv);
  if (Hq / Hkv > 16)
    return fail(Q3_ERR_UNSUPPORTED, "q3_attn_prefill_ragged: Hq/Hkv=%d above 16", Hq / Hkv);
  if (B == 0 || n_tokens == 0) return Q3_OK;
  Q3_REQUIRE(q && k_pages && v_pages && out && block_table && cu_q && kv_lens && workspace,
             "q3_attn_prefill_ragged: null pointer");
  Q3_REQUIRE(page_tokens > 0 && page_tokens % 64 == 0,
             "q3_attn_prefill_ragged: page_tokens=%d must be a positive multiple of 64",
             page_tokens);
  Q3_REQUIRE(table_width > 0 && table_stride >= table_width && num_pages > 0 &&
                 num_pages < (1ll << 31) &&
                 (int64_t)table_width * page_tokens < (1ll << 31) - 256,
             "q3_attn_prefill_ragged: table width %d, stride %lld, %lld pages", table_width,
             (long long)table_stride, (long long)num_pages);
  Q3_REQUIRE(num_pages * Hkv * page_tokens < (1ll << 31),
             "q3_attn_prefill_ragged: the pool is too large for 32-bit TMA rows");
  Q3_REQUIRE(q_stride >= (int64_t)Hq * kD && out_stride >= (int64_t)Hq * kD &&
                 q_stride % 8 == 0 && out_stride % 8 == 0,
             "q3_attn_prefill_ragged: row strides must cover a row and be multiples of 8");
  Q3_REQUIRE(scale > 0.f && scale < INFINITY, "q3_attn_prefill_ragged: scale must be positive");
  Q3_REQUIRE(aligned(q, 16) && aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(out, 16) &&
                 aligned(block_table, 4) && aligned(cu_q, 4) && aligned(kv_lens, 4) &&
                 aligned(workspace, 16),
             "q3_attn_prefill_ragged: misaligned pointer");
  size_t off_ml, off_desc;
  const size_t need = prefill_ws(&off_ml, &off_desc);
  Q3_REQUIRE(workspace_bytes >= need, "q3_attn_prefill_ragged: workspace of %zu bytes, need %zu",
             workspace_bytes, need);
  const int G = Hq / Hkv, T = kM / G;
  CUtensorMap tq, tk, tv;
  int rc = make_tmap_3d_heads(&tq, q, n_tokens, Hq, q_stride, T, G);
  if (rc) return rc;
  const int64_t rows = num_pages * Hkv * page_tokens;
  rc = make_tmap_2d(&tk, k_pages, rows, kD, 64, 64);
  if (rc) return rc;
  rc = make_tmap_2d(&tv, v_pages, rows, kD, 64, 64);
  if (rc) return rc;
  static bool attr_set[64] = {false};
  int dev = 0;
  Q3_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    Q3_CUDA_CHECK(cudaFuncSetAttribute(ragged_prefill_kernel,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  uint8_t* ws = (uint8_t*)workspace;
  RaggedPrefillParams p{(__nv_bfloat16*)out, out_stride, block_table, table_stride, cu_q, kv_lens,
                        (float*)ws, (float*)(ws + off_ml), (int4*)(ws + off_desc), B, Hkv, G, T,
                        page_tokens, (int)num_pages, table_width * page_tokens, (int)n_tokens,
                        causal ? 1 : 0, scale * 1.4426950408889634f, device_error_word()};
  const dim3 grid((unsigned)prefill_grid());
  rc = launch_ex(ragged_prefill_kernel, grid, dim3(kThreads), kSmem, (cudaStream_t)stream, 1, tq,
                 tk, tv, p);
  if (rc) return rc;
  return launch_ex(ragged_prefill_join, dim3(grid.x, kD / 4 / kJoinD4), dim3(kJoinWarps * 32), 0,
                   (cudaStream_t)stream, 1, p);
}
