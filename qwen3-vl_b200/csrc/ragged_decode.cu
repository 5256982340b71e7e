// Ragged serving step: attention of one new token per request, each request
// over its own length of the paged K/V cache.
//
// The S = 1 eager attention of forward_layer (model_fused.py:248-262) for a
// batch whose requests have different lengths (the reference, and the paged
// kernel of attn_decode.cu, take one length for the whole batch):
//   out[b, h] = softmax(q[b, h] . K_b^T * scale) V_b over positions
//   [0, kv_lens[b]), K/V head h / (Hq / Hkv), position t in page
//   table[b, t / page_tokens]; a request of length 0 gives zeros.
// With cu_q the requests' rows are packed: request b's is cu_q[b], and a request that
// brings no token in this step has none.
// One pass with a running maximum and sum (fp32, log2 units):
//   m' = max(m, s),  l' = l 2^(m-m') + 2^(s-m'),  o' = o 2^(m-m') + 2^(s-m') v.
//
// Bound by HBM: every K/V row of a request is read once, for all Hq / Hkv
// query heads of its K/V head.  The lengths are only known on the device, so
// the work is split there: the 64-position tiles of all (request, K/V head)
// pairs form one list, and CTA c of G takes tiles [U c / G, U (c+1) / G), which
// may begin and end inside a pair.  Equal bytes per SM whatever the lengths
// (32 requests of 257 to 32768 positions or one of 700), where one CTA or one
// fixed number of splits per pair leaves SMs idle behind the longest request.
// A pair inside one CTA is written directly; the pieces of a pair that spans
// CTAs go to the workspace in fp32 and a second kernel joins them in a fixed
// order.  The second kernel costs about 2 us; the last-arriving-CTA join that would
// save it was slower in attn_decode.cu, and its counters would tie the workspace to
// one stream.
//
// A producer warp streams K and V tiles by TMA into a ring of 32 KB stages; four
// consumer warps take 16 positions of each: S = Q K^T by mma.sync with the pair's
// query heads as the rows (8, or 16 when Hq / Hkv > 8), the softmax above per
// row, O += P V with P rounded to bf16 (at most 2^-8 of each p, independent per key;
// the sum l takes the unrounded p).  With values of mixed sign the output shrinks as
// the average of these errors does, so they stay beside the output's own rounding:
// relative error against 64 bits 0.0019 on the long requests below, where an fp32
// form has 0.0016.
// Measured on B200: 32 requests of 257 to 32768 positions, 32/8 heads, 885 MB:
// 133 to 136 us, 6.5 to 6.7 TB/s (1.0 of a copy, which also writes; two tiles a
// step: with one 140, and then with eight consumer warps 149); 8 requests in a 2048
// bucket 10.2 us, of which the 24 MB take 3.5; one request of 700 positions, 4/1
// heads, 5.7 us, about half of it the chain lengths -> table -> first tile and 2 us
// the join.
#include <math.h>

#include <type_traits>

#include "common.cuh"

namespace q3 {
namespace {

constexpr int kD = 128;
constexpr int kTile = 64;                     // positions per stage
constexpr int kHalf = kTile * 128;            // one 64-dim box of a tile (8 KB)
constexpr int kStage = 4 * kHalf;             // K lo/hi + V lo/hi (32 KB)
constexpr int kConsumers = 4;                 // consumer warps, 16 positions of a tile each
constexpr int kThreads = (kConsumers + 1) * 32;
constexpr int kMaxB = 65536;

// WIDE: Hq / Hkv in 9..16 (both row halves of the MMA's A operand are used)
template <bool WIDE>
struct Cfg {
  static constexpr int kRows = WIDE ? 16 : 8;
  static constexpr int kStages = 6;
  static constexpr int kOffMerge = kStages * kStage;
  static constexpr int kMergeBytes = kConsumers * kRows * (kD + 2) * 4;
  static constexpr int kOffBar = kOffMerge + kMergeBytes;
  static constexpr int kSmem = kOffBar + 2 * kStages * 8 + 1024;  // + alignment slack
};
static_assert(Cfg<false>::kSmem <= 227 * 1024 && Cfg<true>::kSmem <= 227 * 1024, "shared memory");

struct RaggedDecodeParams {
  const __nv_bfloat16* q;
  int64_t q_stride;
  __nv_bfloat16* out;
  int64_t out_stride;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* kv_lens;
  float* ws_acc;   // [2 * grid][G][128] unnormalised pieces
  float* ws_ml;    // [2 * grid][G][2]   running max (log2 units) and sum
  // [grid] of the pair that goes on behind CTA c's range: {its row of out * Hkv + its
  // K/V head, its last CTA}; of one that began before it, if the split join will
  // look: {-2 - (its first CTA), its last CTA}; else {-1, -1}
  int2* ws_desc;
  int B, Hkv, G, page_tokens, num_pages, capacity, split;
  float scale_log2;
  int* err;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// Byte offset of 16-byte chunk c (0..15) of row r in a tile's K or V half pair.
__device__ __forceinline__ uint32_t kv_at(int r, int c) {
  return (c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// x / l; 0 where l is 0: every score of the row passed fp32's lowest value, no key
// counts, and the row is zeros as one that sees no key.  A NaN sum stays NaN.
__device__ __forceinline__ float over_sum(float x, float l) { return l == 0.f ? 0.f : x / l; }

// Row of request b in q and out: b, or with packed rows cu_q[b].  A type of its own,
// so that the other form does not pay for it (8 requests in a 2048 bucket 10.3 us,
// 10.7 with the choice made at run time).
template <bool PACKED>
struct Rows {
  __device__ __forceinline__ int find(int b, int*) const { return b; }
  __device__ __forceinline__ int at(int b) const { return b; }
};
template <>
struct Rows<true> {
  const int32_t* cu_q;  // [B + 1]
  int n;                // packed rows
  // -1 without a token.  More than one, or rows outside the packed ones, are not
  // for this call (0x925).
  __device__ __forceinline__ int find(int b, int* bad) const {
    const int first = cu_q[b], end = cu_q[b + 1];
    if (first == end) return -1;
    if (first < 0 || first >= n || end != first + 1) {
      *bad = 0x925;
      return -1;
    }
    return first;
  }
  // of a request that has tiles
  __device__ __forceinline__ int at(int b) const { return cu_q[b]; }
};

// Length of request b, inside what its table row can hold; 0 without a token.
template <bool PACKED>
__device__ __forceinline__ int req_len(const RaggedDecodeParams& p, const Rows<PACKED>& rows, int b,
                                       int* bad) {
  const int L = p.kv_lens[b];
  if (PACKED && rows.find(b, bad) < 0) return 0;
  if (L < 0 || L > p.capacity) *bad = 0x921;
  return min(max(L, 0), p.capacity);
}

// The pieces of a CTA's range, in order: pair (b, kvh), tiles [t0, t1) of nt.
struct Piece {
  int b, kvh, t0, t1, nt, L;
};
struct Walk {
  int b, kvh, tile, nt, L;
  int64_t left;
  template <bool PACKED>
  __device__ __forceinline__ bool next(const RaggedDecodeParams& p, const Rows<PACKED>& rows,
                                       Piece& w) {
    if (left <= 0) return false;
    int bad = 0;
    while (tile >= nt) {  // the next pair that has tiles
      tile = 0;
      if (nt > 0 && ++kvh < p.Hkv) break;
      kvh = 0;
      if (++b >= p.B) return false;
      L = req_len(p, rows, b, &bad);
      nt = (L + kTile - 1) / kTile;
    }
    w.b = b;
    w.kvh = kvh;
    w.t0 = tile;
    w.nt = nt;
    w.L = L;
    const int64_t n = min64(left, nt - tile);
    w.t1 = tile + (int)n;
    tile = w.t1;
    left -= n;
    return true;
  }
};

template <bool WIDE, bool PACKED>
__global__ void __launch_bounds__(kThreads, 1)
    ragged_decode_kernel(const __grid_constant__ CUtensorMap tmK,
                         const __grid_constant__ CUtensorMap tmV, RaggedDecodeParams p,
                         Rows<PACKED> rows) {
  using C = Cfg<WIDE>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  float* sm_o = reinterpret_cast<float*>(smem + C::kOffMerge);  // [warp][row][128]
  float* sm_ml = sm_o + kConsumers * C::kRows * kD;             // [warp][row][2]
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* empty = full + C::kStages;
  __shared__ int64_t s_warp[kThreads / 32];
  __shared__ int s_start[4];  // b, tile inside the request's Hkv * nt, nt, L

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kConsumers);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  pdl_launch();
  pdl_wait();

  // ---- this CTA's range of the tile list (every CTA scans the lengths) ----
  const int c = blockIdx.x;
  uint32_t nc;  // CTAs that get tiles
  int64_t share;
  uint32_t rest;
  // CTA k's range [U k / nc, U (k + 1) / nc) by one division of U (in 32 bits
  // where it fits) and remainders below 2^18
  auto divide = [&](int64_t U) {
    nc = (uint32_t)min64(gridDim.x, U);
    share = nc == 0 ? 0 : U >> 32 ? U / nc : (int64_t)((uint32_t)U / nc);
    rest = (uint32_t)(U - share * nc);
  };
  auto cut = [&](uint32_t k) { return share * k + (rest * k) / nc; };
  Walk walk;
  int64_t u0 = 0, off = 0;
  int bad = 0;  // error code of a request this thread looked at
  walk.b = p.B;
  walk.nt = walk.L = walk.kvh = walk.tile = 0;
  walk.left = 0;
  if (p.B <= 32) {
    // one request per lane: every warp scans for itself
    walk.L = lane < p.B ? req_len(p, rows, lane, &bad) : 0;
    walk.nt = (walk.L + kTile - 1) / kTile;
    const int64_t mine = (int64_t)walk.nt * p.Hkv;
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const int64_t U = __shfl_sync(0xffffffffu, incl, 31);
    divide(U);
    __syncthreads();  // barriers are initialised
    if (c < (int)nc) {
      u0 = cut(c);
      walk.left = cut(c + 1) - u0;
      const int src = __ffs(__ballot_sync(0xffffffffu, u0 < incl)) - 1;
      off = u0 - __shfl_sync(0xffffffffu, incl - mine, src);
      walk.L = __shfl_sync(0xffffffffu, walk.L, src);
      walk.nt = __shfl_sync(0xffffffffu, walk.nt, src);
      walk.b = src;
    }
  } else {
    const int per = (p.B + kThreads - 1) / kThreads;
    const int b0 = min((int)threadIdx.x * per, p.B), b1 = min(b0 + per, p.B);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += (req_len(p, rows, b, &bad) + kTile - 1) / kTile;
    mine *= p.Hkv;
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    int64_t before = incl - mine, U = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += s_warp[w];
      U += s_warp[w];
    }
    divide(U);
    if (c < (int)nc) {
      u0 = cut(c);
      walk.left = cut(c + 1) - u0;
      if (before <= u0 && u0 < before + mine) {  // one thread's requests
        int64_t at = before;
        for (int b = b0; b < b1; ++b) {
          const int L = req_len(p, rows, b, &bad), nt = (L + kTile - 1) / kTile;
          const int64_t n = (int64_t)nt * p.Hkv;
          if (u0 < at + n) {
            s_start[0] = b;
            s_start[1] = (int)(u0 - at);
            s_start[2] = nt;
            s_start[3] = L;
            break;
          }
          at += n;
        }
      }
    }
    __syncthreads();
    if (c < (int)nc) {
      walk.b = s_start[0];
      off = s_start[1];
      walk.nt = s_start[2];
      walk.L = s_start[3];
    }
  }
  if (bad && c == 0) report_timeout(p.err, bad);
  if (walk.left > 0) {
    walk.kvh = (int)((uint32_t)off / (uint32_t)walk.nt);
    walk.tile = (int)off - walk.kvh * walk.nt;
  }
  Piece w;

  if (warp == kConsumers) {
    // ------------------------------ TMA producer ------------------------------
    int it = 0;
    bool ok = true;
    int64_t u = u0;  // first tile of the piece in the list
    if (lane == 0) p.ws_desc[c] = make_int2(-1, -1);
    while (ok && walk.next(p, rows, w)) {
      int pages = 0;  // this lane's entry of 32 tiles' pages
      for (int t = w.t0; t < w.t1; ++t, ++it) {
        const int k = (t - w.t0) & 31;
        if (k == 0) {
          const int tl = t + lane;
          if (tl < w.t1) {
            // a 64-position tile never straddles pages (page_tokens % 64 == 0)
            pages = p.table[w.b * p.table_stride + (uint32_t)tl * kTile / (uint32_t)p.page_tokens];
            if (pages < 0 || pages >= p.num_pages) {  // recorded, page 0 read in its place
              report_timeout(p.err, 0x922);
              pages = 0;
            }
          }
        }
        const int pg = __shfl_sync(0xffffffffu, pages, k);
        const int s = it % C::kStages;
        if (lane == 0) {
          if (it >= C::kStages &&
              !mbar_wait(&empty[s], ((it / C::kStages) - 1) & 1, p.err, 0x923)) {
            ok = false;
          } else {
            const int y = (int)(((int64_t)pg * p.Hkv + w.kvh) * p.page_tokens +
                                (uint32_t)t * kTile % (uint32_t)p.page_tokens);
            uint8_t* st = smem + s * kStage;
            mbar_arrive_expect_tx(&full[s], kStage);
            tma_load_2d(st, &tmK, &full[s], 0, y, kCacheEvictFirst);
            tma_load_2d(st + kHalf, &tmK, &full[s], 64, y, kCacheEvictFirst);
            tma_load_2d(st + 2 * kHalf, &tmV, &full[s], 0, y, kCacheEvictFirst);
            tma_load_2d(st + 3 * kHalf, &tmV, &full[s], 64, y, kCacheEvictFirst);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
      }
      if (w.t1 < w.nt && (w.t0 == 0 || p.split)) {
        // the pair goes on in the next CTAs (this is the CTA's last piece): its
        // first and last CTA have the largest k with cut(k) <= its first, last tile
        auto holder = [&](int from, int64_t tile) {
          int at = from;
          for (uint32_t k0 = from + 1; k0 < nc; k0 += 32) {
            const uint32_t k = k0 + lane;
            const int n = __popc(__ballot_sync(0xffffffffu, k < nc && cut(k) <= tile));
            at += n;
            if (n < 32) break;
          }
          return at;
        };
        const int64_t first = u - w.t0;
        const int last = holder(c, first + w.nt - 1);
        const int id = w.t0 == 0 ? rows.at(w.b) * p.Hkv + w.kvh : -2 - holder(0, first);
        if (lane == 0) p.ws_desc[c] = make_int2(id, last);
      }
      u += w.t1 - w.t0;
    }
    // the copies issued land before the CTA may exit (the consumers wait for
    // every one of them unless a wait ran out, theirs or this warp's)
    if (lane == 0)
      for (int i = max(0, it - C::kStages); i < it; ++i)
        mbar_wait(&full[i % C::kStages], (i / C::kStages) & 1, nullptr, 0);
  } else {
    // ------------------------------- consumers --------------------------------
    const int band = warp;
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = smem_u32(smem);
    bool ok = true;
    int it = 0;
    while (walk.next(p, rows, w)) {
      // Q as the A operand: row g (and g + 8) = query head kvh * G + row
      uint32_t qf[8][WIDE ? 4 : 2];
      {
        const __nv_bfloat16* qh =
            p.q + rows.at(w.b) * p.q_stride + (int64_t)(w.kvh * p.G) * kD + 2 * t4;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
          for (int e = 0; e < (WIDE ? 4 : 2); ++e) {
            // registers: (row g, k lo), [row g+8, k lo], (row g, k hi), [row g+8, k hi]
            const int row = WIDE ? g + 8 * (e & 1) : g;
            const int col = ks * 16 + 8 * (WIDE ? (e >> 1) : e);
            qf[ks][e] = row < p.G ? *reinterpret_cast<const uint32_t*>(qh + row * kD + col) : 0u;
          }
      }
      float o[16][WIDE ? 4 : 2];
#pragma unroll
      for (int i = 0; i < 16; ++i)
#pragma unroll
        for (int e = 0; e < (WIDE ? 4 : 2); ++e) o[i][e] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

      // NT tiles in one step: two are independent work for a warp that has its
      // scheduler to itself
      auto step = [&](auto nt_c, int t) {
        constexpr int NT = decltype(nt_c)::value;
        uint32_t sK[NT];
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const int s = (it + u) % C::kStages;
          if (ok)
            ok = __all_sync(0xffffffffu,
                            mbar_wait(&full[s], ((it + u) / C::kStages) & 1, p.err, 0x924));
          sK[u] = ring + s * kStage;
        }
        if (!ok) return;
        // ---- S = Q K^T: 16 rows x 16 positions of each tile (two n-tiles of 8) ----
        float sc[NT][2][4];
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[u][j][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
          for (int u = 0; u < NT; ++u) {
            uint32_t kf[4];
            const int r = band * 16 + (lane & 7) + ((lane >> 4) << 3);
            ldsm4(kf, sK[u] + kv_at(r, ks * 2 + ((lane >> 3) & 1)));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              if constexpr (WIDE)
                mma_bf16_16816(sc[u][j], qf[ks][0], qf[ks][1], qf[ks][2], qf[ks][3], kf[2 * j],
                               kf[2 * j + 1]);
              else
                mma_bf16_16816(sc[u][j], qf[ks][0], 0u, qf[ks][1], 0u, kf[2 * j], kf[2 * j + 1]);
            }
          }
        const int pos0 = t * kTile + band * 16;  // of the first tile
        const bool tail = pos0 + (NT - 1) * kTile + 16 > w.L;
        if (tail) {
          // V rows past the end hold whatever the page held before: 0 * V must
          // be 0, so this warp's rows there become zeros (the ring's next copy
          // into the stage is ordered behind the fence and the release below)
          const uint32_t sV = sK[NT - 1] + 2 * kHalf;
#pragma unroll
          for (int i = lane; i < 16 * 16; i += 32) {
            const int r = band * 16 + (i >> 4);
            if ((t + NT - 1) * kTile + r >= w.L)
              asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(sV + kv_at(r, i & 15)),
                           "r"(0u)
                           : "memory");
          }
          __syncwarp();
        }
        // ---- running max and sum per row; P as the A operand of P V ----
        uint32_t pa[NT][4];
#pragma unroll
        for (int hh = 0; hh < (WIDE ? 2 : 1); ++hh) {
          float x[NT][4];
          float mx = -INFINITY;
#pragma unroll
          for (int u = 0; u < NT; ++u) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int pos = pos0 + u * kTile + j * 8 + 2 * t4 + e;
                x[u][j * 2 + e] = pos < w.L ? sc[u][j][hh * 2 + e] * p.scale_log2 : -INFINITY;
              }
            mx = fmaxf(mx, fmaxf(fmaxf(x[u][0], x[u][1]), fmaxf(x[u][2], x[u][3])));
          }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m[hh], mx);
          const float base = m_new == -INFINITY ? 0.f : m_new;
          const float corr = ex2_approx(m[hh] - base);
          float rs = 0.f;
#pragma unroll
          for (int u = 0; u < NT; ++u) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[u][e] = ex2_approx(x[u][e] - base);
              rs += x[u][e];
            }
            pa[u][hh] = pack_bf16x2(x[u][0], x[u][1]);
            pa[u][2 + hh] = pack_bf16x2(x[u][2], x[u][3]);
          }
          l[hh] = l[hh] * corr + rs;
          m[hh] = m_new;
#pragma unroll
          for (int d = 0; d < 16; ++d) {
            o[d][hh * 2] *= corr;
            o[d][hh * 2 + 1] *= corr;
          }
        }
        // ---- O += P V ----
#pragma unroll
        for (int ip = 0; ip < 8; ++ip)
#pragma unroll
          for (int u = 0; u < NT; ++u) {
            uint32_t vf[4];
            const int r = band * 16 + (lane & 7) + (((lane >> 3) & 1) << 3);
            ldsm4t(vf, sK[u] + 2 * kHalf + kv_at(r, ip * 2 + (lane >> 4)));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float(&oo)[WIDE ? 4 : 2] = o[2 * ip + j];
              if constexpr (WIDE) {
                mma_bf16_16816(oo, pa[u][0], pa[u][1], pa[u][2], pa[u][3], vf[2 * j],
                               vf[2 * j + 1]);
              } else {
                float d4[4] = {oo[0], oo[1], 0.f, 0.f};
                mma_bf16_16816(d4, pa[u][0], 0u, pa[u][2], 0u, vf[2 * j], vf[2 * j + 1]);
                oo[0] = d4[0];
                oo[1] = d4[1];
              }
            }
          }
        if (tail) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0)
#pragma unroll
          for (int u = 0; u < NT; ++u) mbar_arrive(&empty[(it + u) % C::kStages]);
      };
      int t = w.t0;
      for (; t + 1 < w.t1; t += 2, it += 2) step(std::integral_constant<int, 2>(), t);
      if (t < w.t1) {
        step(std::integral_constant<int, 1>(), t);
        ++it;
      }

      // ---- merge the warps; write the output or this CTA's piece ----
#pragma unroll
      for (int hh = 0; hh < (WIDE ? 2 : 1); ++hh) {
        float ls = l[hh];
        ls += __shfl_xor_sync(0xffffffffu, ls, 1);
        ls += __shfl_xor_sync(0xffffffffu, ls, 2);
        const int row = g + 8 * hh;
        if (row < p.G) {
          float* dst = sm_o + (warp * C::kRows + row) * kD;
#pragma unroll
          for (int d = 0; d < 16; ++d)
            *reinterpret_cast<float2*>(dst + d * 8 + 2 * t4) =
                make_float2(o[d][hh * 2], o[d][hh * 2 + 1]);
          if (t4 == 0)
            *reinterpret_cast<float2*>(sm_ml + (warp * C::kRows + row) * 2) =
                make_float2(m[hh], ls);
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
      const bool whole = w.t0 == 0 && w.t1 == w.nt;
      // a piece that ends this CTA's range but not its pair has the odd slot
      // unless it also began inside the pair
      const int slot = 2 * c + (w.t0 == 0 ? 1 : 0);
      for (int idx = threadIdx.x; idx < p.G * (kD / 4); idx += kConsumers * 32) {
        const int row = idx / (kD / 4), d = idx % (kD / 4) * 4;
        float2 ml[kConsumers];
        float4 x[kConsumers];
#pragma unroll
        for (int i = 0; i < kConsumers; ++i) {
          ml[i] = *reinterpret_cast<const float2*>(sm_ml + (i * C::kRows + row) * 2);
          x[i] = *reinterpret_cast<const float4*>(sm_o + (i * C::kRows + row) * kD + d);
        }
        float M = ml[0].x;
#pragma unroll
        for (int i = 1; i < kConsumers; ++i) M = fmaxf(M, ml[i].x);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        float ls = 0.f;
#pragma unroll
        for (int i = 0; i < kConsumers; ++i) {
          const float f = ml[i].x == -INFINITY ? 0.f : ex2_approx(ml[i].x - M);
          a.x = fmaf(f, x[i].x, a.x);
          a.y = fmaf(f, x[i].y, a.y);
          a.z = fmaf(f, x[i].z, a.z);
          a.w = fmaf(f, x[i].w, a.w);
          ls = fmaf(f, ml[i].y, ls);
        }
        if (whole) {
          const float inv = over_sum(1.0f, ls);
          *reinterpret_cast<uint2*>(p.out + rows.at(w.b) * p.out_stride +
                                    (int64_t)(w.kvh * p.G + row) * kD + d) =
              make_uint2(pack_bf16x2(a.x * inv, a.y * inv), pack_bf16x2(a.z * inv, a.w * inv));
        } else {
          *reinterpret_cast<float4*>(p.ws_acc + ((int64_t)slot * p.G + row) * kD + d) = a;
          if (d == 0)
            *reinterpret_cast<float2*>(p.ws_ml + ((int64_t)slot * p.G + row) * 2) =
                make_float2(M, ls);
        }
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
    }
    // requests with nothing cached: zeros
    const int Hq = p.Hkv * p.G;
    for (int b = c; b < p.B; b += gridDim.x) {
      const int row = rows.find(b, &bad);
      if (row >= 0 && p.kv_lens[b] <= 0)
        for (int i = threadIdx.x; i < Hq * kD / 8; i += kConsumers * 32)
          reinterpret_cast<uint4*>(p.out + row * p.out_stride)[i] = make_uint4(0, 0, 0, 0);
    }
  }
}

constexpr int kMaxGrid = 512;
// Few long requests leave pairs of up to a piece per SM, which one CTA would take
// warp by warp.  Above kFewPieces the CTAs of a pair's first kJoinParts CTAs take 16
// dims each and a warp eight pieces at a time.  Launched (SPLIT) for up to a pair per
// 8 SMs when the table can hold more than kFewPieces tiles: one request of 3000,
// 8000, 30000 positions, 4/1 heads, 7.0, 9.5, 11.7 -> 5.9, 7.1, 8.7 us, two of 11312,
// 6/1, 12.2 -> 8.4; one of 700, with few pieces all the same, 5.4 -> 5.5.  Twelve
// requests of 3000 have 13 pieces a pair: 8.1 us without the split, 8.8 with it.
constexpr int kFewPieces = 16;
constexpr int kJoinParts = 8;
template <int W>
__device__ __forceinline__ void join_many(const RaggedDecodeParams& p, int c0, int n, int part,
                                          int row) {
  __shared__ float2 s_ml[W];
  __shared__ float s_acc[W][kD / kJoinParts];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, d0 = part * (kD / kJoinParts);
  float M = -INFINITY, l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
  for (int i = warp * 8 + (lane >> 2); i < n; i += W * 8) {
    const int64_t piece = (int64_t)(i == 0 ? 2 * c0 + 1 : 2 * (c0 + i)) * p.G + row;
    const float2 ml = *reinterpret_cast<const float2*>(p.ws_ml + piece * 2);
    const float4 x =
        *reinterpret_cast<const float4*>(p.ws_acc + piece * kD + d0 + (lane & 3) * 4);
    const float m_new = fmaxf(M, ml.x);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float f0 = ex2_approx(M - base), f1 = ex2_approx(ml.x - base);
    M = m_new;
    l = fmaf(f1, ml.y, l * f0);
    a.x = fmaf(f1, x.x, a.x * f0);
    a.y = fmaf(f1, x.y, a.y * f0);
    a.z = fmaf(f1, x.z, a.z * f0);
    a.w = fmaf(f1, x.w, a.w * f0);
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {  // the lanes that hold the same dims
    const float m_new = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float f = ex2_approx(M - (m_new == -INFINITY ? 0.f : m_new));
    M = m_new;
    l *= f;
    l += __shfl_xor_sync(0xffffffffu, l, o);
    a = make_float4(a.x * f, a.y * f, a.z * f, a.w * f);
    a.x += __shfl_xor_sync(0xffffffffu, a.x, o);
    a.y += __shfl_xor_sync(0xffffffffu, a.y, o);
    a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
    a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
  }
  if (lane < 4) *reinterpret_cast<float4*>(&s_acc[warp][lane * 4]) = a;
  if (lane == 0) s_ml[warp] = make_float2(M, l);
  __syncthreads();
  if (threadIdx.x < kD / kJoinParts) {
    float Ma = -INFINITY;
    for (int i = 0; i < W; ++i) Ma = fmaxf(Ma, s_ml[i].x);
    float x = 0.f, ls = 0.f;
    for (int i = 0; i < W; ++i) {
      const float f = s_ml[i].x == -INFINITY ? 0.f : ex2_approx(s_ml[i].x - Ma);
      x = fmaf(f, s_acc[i][threadIdx.x], x);
      ls = fmaf(f, s_ml[i].y, ls);
    }
    const int pair = p.ws_desc[c0].x, r = pair / p.Hkv, kvh = pair - r * p.Hkv;
    p.out[r * p.out_stride + (int64_t)(kvh * p.G + row) * kD + d0 + threadIdx.x] =
        f2bf(over_sum(x, ls));
  }
}
// Joins the pieces of the pair whose first piece ends CTA c's range: pieces
// 2c+1, 2(c+1), 2(c+2), ..., 2*last.  One CTA per (c, query head of the pair), of
// four warps with more than 8 heads per K/V head, so that more of the grid waits on
// the SMs beside the first kernel (3 short requests at 32/2 heads 7.6 -> 6.8 us; 16
// long ones at 24/2 20.0 -> 20.6), and for the same reason it is kept to 32 registers
// (with 40 the case of 32 long requests took 3 us longer).
template <int W, bool SPLIT>  // warps
__global__ void __launch_bounds__(W * 32) ragged_decode_join(RaggedDecodeParams p) {
  __shared__ float2 s_ml[W];
  __shared__ __align__(16) float s_acc[W][kD];
  pdl_launch();
  pdl_wait();
  const int c = blockIdx.x, row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int2 d = p.ws_desc[c];
  if (SPLIT ? d.x == -1 : d.x < 0) return;
  if constexpr (SPLIT) {
    const int c0 = d.x < 0 ? -2 - d.x : c;
    if (d.y - c0 + 1 > kFewPieces) {
      if (c - c0 < kJoinParts) join_many<W>(p, c0, d.y - c0 + 1, c - c0, row);
      return;
    }
    if (c != c0) return;
  }
  const int n = d.y - c + 1;  // pieces, at most the first kernel's grid
  // a warp's pieces against a running maximum, then the warps'
  float M = -INFINITY, l = 0.f;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp; i < n; i += W) {
    const int64_t piece = (int64_t)(i == 0 ? 2 * c + 1 : 2 * (c + i)) * p.G + row;
    const float2 ml = *reinterpret_cast<const float2*>(p.ws_ml + piece * 2);
    const float4 x = *reinterpret_cast<const float4*>(p.ws_acc + piece * kD + lane * 4);
    const float m_new = fmaxf(M, ml.x);
    // -inf where every score of the pieces so far passed fp32's lowest value
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float f0 = ex2_approx(M - base), f1 = ex2_approx(ml.x - base);
    M = m_new;
    l = fmaf(f1, ml.y, l * f0);
    a.x = fmaf(f1, x.x, a.x * f0);
    a.y = fmaf(f1, x.y, a.y * f0);
    a.z = fmaf(f1, x.z, a.z * f0);
    a.w = fmaf(f1, x.w, a.w * f0);
  }
  *reinterpret_cast<float4*>(&s_acc[warp][lane * 4]) = a;
  if (lane == 0) s_ml[warp] = make_float2(M, l);
  __syncthreads();
  if (threadIdx.x < kD) {
    float Ma = -INFINITY;
#pragma unroll
    for (int i = 0; i < W; ++i) Ma = fmaxf(Ma, s_ml[i].x);
    float x = 0.f, ls = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const float f = s_ml[i].x == -INFINITY ? 0.f : ex2_approx(s_ml[i].x - Ma);
      x = fmaf(f, s_acc[i][threadIdx.x], x);
      ls = fmaf(f, s_ml[i].y, ls);
    }
    const int r = d.x / p.Hkv, kvh = d.x - r * p.Hkv;
    p.out[r * p.out_stride + (int64_t)(kvh * p.G + row) * kD + threadIdx.x] =
        f2bf(over_sum(x, ls));
  }
}

int decode_grid() { return (int)min64(num_sms(), kMaxGrid); }

size_t decode_ws(int G, size_t* off_ml, size_t* off_desc) {
  const size_t slots = 2 * (size_t)decode_grid();
  size_t n = slots * G * kD * 4;
  *off_ml = n;
  n += slots * G * 8;
  *off_desc = n;
  return n + decode_grid() * sizeof(int2);
}

// Both entry points (a kernel of each width); messages name the first.
template <bool PACKED>
int decode_ragged(const void* q, int64_t q_stride, const void* k_pages, const void* v_pages,
                  void* out, int64_t out_stride, int64_t n_rows, int B, int Hq, int Hkv,
                  int head_dim, const int32_t* block_table, int64_t table_stride, int table_width,
                  int page_tokens, int64_t num_pages, const int32_t* kv_lens, float scale,
                  void* workspace, size_t workspace_bytes, Rows<PACKED> rows_of_q,
                  q3_stream_t stream) {
  Q3_REQUIRE(head_dim == kD, "q3_attn_decode_ragged: head_dim must be 128 (got %d)", head_dim);
  Q3_REQUIRE(B >= 0 && B <= kMaxB && Hq > 0 && Hkv > 0 && Hkv <= 1024 && Hq % Hkv == 0,
             "q3_attn_decode_ragged: bad shape B=%d Hq=%d Hkv=%d", B, Hq, Hkv);
  if (Hq / Hkv > 16)
    return fail(Q3_ERR_UNSUPPORTED, "q3_attn_decode_ragged: Hq/Hkv=%d above 16", Hq / Hkv);
  if (B == 0 || n_rows == 0) return Q3_OK;
  Q3_REQUIRE(q && k_pages && v_pages && out && block_table && kv_lens && workspace,
             "q3_attn_decode_ragged: null pointer");
  Q3_REQUIRE(page_tokens > 0 && page_tokens % kTile == 0,
             "q3_attn_decode_ragged: page_tokens=%d must be a positive multiple of %d",
             page_tokens, kTile);
  Q3_REQUIRE(table_width > 0 && table_stride >= table_width && num_pages > 0 &&
                 num_pages < (1ll << 31) &&
                 (int64_t)table_width * page_tokens < (1ll << 31),
             "q3_attn_decode_ragged: table width %d, stride %lld, %lld pages", table_width,
             (long long)table_stride, (long long)num_pages);
  Q3_REQUIRE((int64_t)table_width * page_tokens / kTile * Hkv < (1ll << 31),
             "q3_attn_decode_ragged: %d pages of %d positions and %d K/V heads pass 32-bit tiles",
             table_width, page_tokens, Hkv);
  Q3_REQUIRE(num_pages * Hkv * page_tokens < (1ll << 31),
             "q3_attn_decode_ragged: the pool is too large for 32-bit TMA rows");
  Q3_REQUIRE(q_stride >= (int64_t)Hq * kD && out_stride >= (int64_t)Hq * kD &&
                 q_stride % 2 == 0 && out_stride % 8 == 0,
             "q3_attn_decode_ragged: row strides");
  Q3_REQUIRE(aligned(q, 4) && aligned(k_pages, 16) && aligned(v_pages, 16) && aligned(out, 16) &&
                 aligned(block_table, 4) && aligned(kv_lens, 4) && aligned(workspace, 16),
             "q3_attn_decode_ragged: misaligned pointer");
  const int G = Hq / Hkv;
  size_t off_ml, off_desc;
  const size_t need = decode_ws(G, &off_ml, &off_desc);
  Q3_REQUIRE(workspace_bytes >= need, "q3_attn_decode_ragged: workspace of %zu bytes, need %zu",
             workspace_bytes, need);
  CUtensorMap tk, tv;
  const int64_t rows = num_pages * Hkv * page_tokens;
  int rc = make_tmap_2d(&tk, k_pages, rows, kD, kTile, 64);
  if (rc) return rc;
  rc = make_tmap_2d(&tv, v_pages, rows, kD, kTile, 64);
  if (rc) return rc;
  uint8_t* ws = (uint8_t*)workspace;
  const int split = (int64_t)B * Hkv * 8 <= decode_grid() &&
                    (int64_t)table_width * page_tokens > kFewPieces * kTile;
  RaggedDecodeParams p{(const __nv_bfloat16*)q, q_stride, (__nv_bfloat16*)out, out_stride,
                       block_table, table_stride, kv_lens, (float*)ws, (float*)(ws + off_ml),
                       (int2*)(ws + off_desc), B, Hkv, G, page_tokens, (int)num_pages,
                       table_width * page_tokens, split, scale * 1.4426950408889634f,
                       device_error_word()};
  static bool attr_set[64] = {false};
  int dev = 0;
  Q3_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !attr_set[dev]) {
    Q3_CUDA_CHECK(cudaFuncSetAttribute(ragged_decode_kernel<false, PACKED>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg<false>::kSmem));
    Q3_CUDA_CHECK(cudaFuncSetAttribute(ragged_decode_kernel<true, PACKED>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Cfg<true>::kSmem));
    if (dev >= 0 && dev < 64) attr_set[dev] = true;
  }
  const dim3 grid((unsigned)decode_grid());
  rc = G > 8 ? launch_ex(ragged_decode_kernel<true, PACKED>, grid, dim3(kThreads), Cfg<true>::kSmem,
                         (cudaStream_t)stream, 1, tk, tv, p, rows_of_q)
             : launch_ex(ragged_decode_kernel<false, PACKED>, grid, dim3(kThreads), Cfg<false>::kSmem,
                         (cudaStream_t)stream, 1, tk, tv, p, rows_of_q);
  if (rc) return rc;
  auto join = G > 8 ? (split ? ragged_decode_join<4, true> : ragged_decode_join<4, false>)
                    : (split ? ragged_decode_join<8, true> : ragged_decode_join<8, false>);
  return launch_ex(join, dim3(grid.x, (unsigned)G), dim3(G > 8 ? 128 : 256), 0,
                   (cudaStream_t)stream, 1, p);
}

}  // namespace
}  // namespace q3

extern "C" size_t q3_attn_decode_ragged_workspace_bytes(int Hq, int Hkv) {
  if (Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Hq / Hkv > 16) return 0;
  size_t a, b;
  return q3::decode_ws(Hq / Hkv, &a, &b);
}

extern "C" int q3_attn_decode_ragged(const void* q, int64_t q_stride, const void* k_pages,
                                     const void* v_pages, void* out, int64_t out_stride, int B,
                                     int Hq, int Hkv, int head_dim, const int32_t* block_table,
                                     int64_t table_stride, int table_width, int page_tokens,
                                     int64_t num_pages, const int32_t* kv_lens, float scale,
                                     void* workspace, size_t workspace_bytes,
                                     q3_stream_t stream) {
  return q3::decode_ragged(q, q_stride, k_pages, v_pages, out, out_stride, B, B, Hq, Hkv, head_dim,
                           block_table, table_stride, table_width, page_tokens, num_pages, kv_lens,
                           scale, workspace, workspace_bytes, q3::Rows<false>{}, stream);
}

extern "C" int q3_attn_decode_ragged_packed(
    const void* q, int64_t q_stride, const void* k_pages, const void* v_pages, void* out,
    int64_t out_stride, int64_t n_tokens, int B, int Hq, int Hkv, int head_dim,
    const int32_t* block_table, int64_t table_stride, int table_width, int page_tokens,
    int64_t num_pages, const int32_t* cu_q, const int32_t* kv_lens, float scale, void* workspace,
    size_t workspace_bytes, q3_stream_t stream) {
  using namespace q3;
  Q3_REQUIRE(n_tokens >= 0 && n_tokens * max64(Hkv, 1) < (1ll << 31),
             "q3_attn_decode_ragged_packed: n_tokens=%lld, %d K/V heads pass 32-bit rows",
             (long long)n_tokens, Hkv);
  Q3_REQUIRE(B == 0 || n_tokens == 0 || (cu_q && aligned(cu_q, 4)),
             "q3_attn_decode_ragged_packed: cu_q is null or misaligned");
  return decode_ragged(q, q_stride, k_pages, v_pages, out, out_stride, n_tokens, B, Hq, Hkv,
                       head_dim, block_table, table_stride, table_width, page_tokens, num_pages,
                       kv_lens, scale, workspace, workspace_bytes,
                       Rows<true>{cu_q, (int)n_tokens}, stream);
}
