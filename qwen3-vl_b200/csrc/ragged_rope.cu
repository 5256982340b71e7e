// Ragged serving step: per-head QK-RMSNorm, 3-axis interleaved rotary
// positions and the K/V rows to their page slots, for packed tokens.
//
// Replaces AttentionBlock.forward after the QKV matmul (model_fused.py:107-129)
// with the cache slice assignment (:244-246) and, for images and video, the
// M-RoPE tables (transformers 5.5.0 modeling_qwen3_vl.py:352-386) for a batch
// whose tokens sit at positions of their own:
//   n = x * rsqrt(mean(x^2) + eps) * w            per head of 128, q and k
//   a_j = pos[axis(j)] * inv_freq[j]              j < 64; axis h for j % 3 == 1
//                                                 and j < 3 sec_h, w for j % 3
//                                                 == 2 and j < 3 sec_w, else t
//   out_j = n_j cos a_j - n_{j+64} sin a_j,  out_{j+64} = n_{j+64} cos a_j + n_j sin a_j
// in fp32 with one rounding to bf16 at the end (the table-driven kernels of
// rope.cu keep the reference's bf16 tables and rounding points; here there is
// no table, and every rounding left out makes the result closer to the
// formula).  The angle is a 53-bit product reduced by whole turns in fp64
// before the fp32 sine and cosine: an fp32 product is off by 4e-3 rad at
// position 10^5.
//
// Bound by HBM: each qkv row is read once, each q, k, v row written once.  A warp
// takes one token (or, when there are few tokens, a part of its heads) and waits
// for no other warp: each lane computes two of the 64 angles and the warp shares
// them.  Eight lanes own one head row; lane l holds dims 8l..8l+7 and their
// rotation partners 64+8l..64+8l+7, so the rotation needs no shuffle, and the
// factors w_j cos a_j, w_{j+64} sin a_j, w_{j+64} cos a_j, w_j sin a_j of its dims
// stay in registers for all heads.
#include <math.h>

#include "common.cuh"

namespace q3 {
namespace {

constexpr int kRD = 128;
constexpr int kRWarps = 2;   // per CTA
// Quads of rows whose loads are in flight together.  16384 tokens of 32 + 2 x 8
// heads, 403 MB: 70.6 us (5.7 TB/s, 0.88 of a copy) with 4 quads, 75 with 8
// (fewer warps fit), 80 with 3, 90 with 1; 8 warps per CTA 73; a CTA of 256
// threads sharing the angles of 4 tokens 83, the same fed by bulk copies into a
// shared-memory ring 95 (a barrier per stage).  The qkv rows are read for the last
// time here, so their loads are marked to leave L2 first: with plain loads the case
// takes 67.4 us, but 7593 tokens of 16/2 heads 20.8 for 19.9 and 4076 of 8/8 11.6 for
// 10.9, because less of q, k and v is then still in L2.
constexpr int kRUnroll = 4;

struct RaggedRopeParams {
  const __nv_bfloat16* qkv;
  int64_t qkv_stride;
  const __nv_bfloat16* qw;
  const __nv_bfloat16* kw;
  const int64_t* pos;
  int64_t pos_stride;  // between axes; 0: one axis for all three
  const float* inv_freq;
  const int64_t* slots;
  __nv_bfloat16* q_out;
  int64_t q_stride;
  __nv_bfloat16* k_pages;
  __nv_bfloat16* v_pages;
  int64_t n_slots;
  int n, parts, Hq, Hkv, page_tokens, sec_h, sec_w;
  float eps;
  int* err;
};

// Eight bf16 values as four fp32 pairs, and back.
__device__ __forceinline__ void unpack8(const uint4& u, float2 (&v)[4]) {
  v[0] = unpack_bf16x2(u.x);
  v[1] = unpack_bf16x2(u.y);
  v[2] = unpack_bf16x2(u.z);
  v[3] = unpack_bf16x2(u.w);
}
__device__ __forceinline__ uint4 pack8(const float2 (&v)[4]) {
  return make_uint4(pack_bf16x2(v[0].x, v[0].y), pack_bf16x2(v[1].x, v[1].y),
                    pack_bf16x2(v[2].x, v[2].y), pack_bf16x2(v[3].x, v[3].y));
}
__device__ __forceinline__ float2 fmul2(float2 a, float2 b) {
  return ffma2(a, b, make_float2(-0.f, -0.f));
}

// A lane's factors: a' = rs (a ac + b bs), b' = rs (b bc + a as).
struct Factors {
  float2 ac[4], bs[4], bc[4], as[4];
};
__device__ __forceinline__ void make_factors(const __nv_bfloat16* w, int l, const float2 (&cs)[4],
                                             const float2 (&sn)[4], Factors& f) {
  float2 wa[4], wb[4];
  unpack8(reinterpret_cast<const uint4*>(w)[l], wa);
  unpack8(reinterpret_cast<const uint4*>(w)[8 + l], wb);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f.ac[i] = fmul2(wa[i], cs[i]);
    f.bc[i] = fmul2(wb[i], cs[i]);
    f.as[i] = fmul2(wa[i], sn[i]);
    f.bs[i] = fmul2(wb[i], make_float2(-sn[i].x, -sn[i].y));
  }
}
// Norm and rotation of the row that this lane's group of eight holds.
__device__ __forceinline__ void norm_rotate(uint4& lo, uint4& hi, const Factors& f, float eps) {
  float2 a[4], b[4];
  unpack8(lo, a);
  unpack8(hi, b);
  float2 q = ffma2(b[0], b[0], fmul2(a[0], a[0]));
#pragma unroll
  for (int i = 1; i < 4; ++i) q = ffma2(a[i], a[i], ffma2(b[i], b[i], q));
  float ss = q.x + q.y;
  ss += __shfl_xor_sync(0xffffffffu, ss, 1);
  ss += __shfl_xor_sync(0xffffffffu, ss, 2);
  ss += __shfl_xor_sync(0xffffffffu, ss, 4);
  const float rs = rsqrtf(ss * (1.0f / kRD) + eps);
  const float2 rs2 = make_float2(rs, rs);
  float2 oa[4], ob[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    oa[i] = fmul2(rs2, ffma2(a[i], f.ac[i], fmul2(b[i], f.bs[i])));
    ob[i] = fmul2(rs2, ffma2(b[i], f.bc[i], fmul2(a[i], f.as[i])));
  }
  lo = pack8(oa);
  hi = pack8(ob);
}

__global__ void __launch_bounds__(kRWarps * 32) qkv_norm_rope_ragged_kernel(RaggedRopeParams p) {
  // No early launch of the next kernel: one that reads cache rows before its own
  // wait (attn_decode_paged streams old rows) must not start before these are
  // written.
  pdl_wait();
  const int lane = threadIdx.x & 31, l = lane & 7, grp = lane >> 3;
  const int64_t unit = (int64_t)blockIdx.x * kRWarps + (threadIdx.x >> 5);
  if (unit >= (int64_t)p.n * p.parts) return;
  const int t = (int)(unit / p.parts), part = (int)(unit - (int64_t)t * p.parts);
  const int64_t slot = p.slots[t];
  if (slot < 0 || slot >= p.n_slots) {  // the whole warp
    if (slot != -1 && lane == 0) report_timeout(p.err, 0x911);
    return;
  }
  // this part's heads, in quads: of q, and of k and v together
  const int nq = (p.Hq + 3) / 4, nkv = (2 * p.Hkv + 3) / 4;
  const int q0 = nq * part / p.parts * 4, q1 = min(nq * (part + 1) / p.parts * 4, p.Hq);
  const int k0 = nkv * part / p.parts * 4, k1 = min(nkv * (part + 1) / p.parts * 4, 2 * p.Hkv);
  const uint4* src = reinterpret_cast<const uint4*>(p.qkv + (int64_t)t * p.qkv_stride) + l;

  uint4 lo[kRUnroll], hi[kRUnroll];
  auto load_q = [&](int base) {
#pragma unroll
    for (int u = 0; u < kRUnroll; ++u) {
      const int h = min(base + 4 * u + grp, p.Hq - 1);
      lo[u] = __ldcs(src + h * 16);
      hi[u] = __ldcs(src + h * 16 + 8);
    }
  };
  if (q0 < q1) load_q(q0);
  // angles j = lane and lane + 32, as half turns (a / pi) reduced to [-1, 1]
  float cv[2], sv[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = lane + 32 * i;
    const int axis = (j % 3 == 1 && j < 3 * p.sec_h) ? 1 : (j % 3 == 2 && j < 3 * p.sec_w) ? 2 : 0;
    double h = (double)p.pos[axis * p.pos_stride + t] * (double)p.inv_freq[j] *
               0.31830988618379067154;
    h -= 2.0 * rint(0.5 * h);
    sincospif((float)h, &sv[i], &cv[i]);
  }
  // angles 8l .. 8l+7: lanes 8 (l & 3) .. + 7, the first or the second of theirs
  float2 cs[4], sn[4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int from = (8 * l + i) & 31;
    const float c0 = __shfl_sync(0xffffffffu, cv[0], from), c1 = __shfl_sync(0xffffffffu, cv[1], from);
    const float s0 = __shfl_sync(0xffffffffu, sv[0], from), s1 = __shfl_sync(0xffffffffu, sv[1], from);
    (i & 1 ? cs[i >> 1].y : cs[i >> 1].x) = l < 4 ? c0 : c1;
    (i & 1 ? sn[i >> 1].y : sn[i >> 1].x) = l < 4 ? s0 : s1;
  }

  Factors f;
  make_factors(p.qw, l, cs, sn, f);
  uint4* dst = reinterpret_cast<uint4*>(p.q_out + (int64_t)t * p.q_stride) + l;
  for (int base = q0; base < q1; base += 4 * kRUnroll) {
    if (base > q0) load_q(base);
#pragma unroll
    for (int u = 0; u < kRUnroll; ++u) {
      const int h = base + 4 * u + grp;
      if (base + 4 * u >= q1) break;
      norm_rotate(lo[u], hi[u], f, p.eps);
      if (h < q1) {
        dst[h * 16] = lo[u];
        dst[h * 16 + 8] = hi[u];
      }
    }
  }
  make_factors(p.kw, l, cs, sn, f);
  const uint32_t pg = (uint32_t)slot / (uint32_t)p.page_tokens;
  const int64_t kv = ((int64_t)pg * p.Hkv * p.page_tokens +
                      ((uint32_t)slot - pg * (uint32_t)p.page_tokens)) * kRD;
  for (int base = k0; base < k1; base += 4 * kRUnroll) {
#pragma unroll
    for (int u = 0; u < kRUnroll; ++u) {
      const int h = p.Hq + min(base + 4 * u + grp, 2 * p.Hkv - 1);
      lo[u] = __ldcs(src + h * 16);
      hi[u] = __ldcs(src + h * 16 + 8);
    }
#pragma unroll
    for (int u = 0; u < kRUnroll; ++u) {
      const int h = base + 4 * u + grp;
      if (base + 4 * u >= k1) break;
      if (base + 4 * u < p.Hkv) {  // a key row among the four
        uint4 a = lo[u], b = hi[u];
        norm_rotate(a, b, f, p.eps);
        if (h < p.Hkv) {
          lo[u] = a;
          hi[u] = b;
        }
      }
      if (h < k1) {
        const bool is_v = h >= p.Hkv;
        uint4* row = reinterpret_cast<uint4*>((is_v ? p.v_pages : p.k_pages) + kv +
                                              (int64_t)(is_v ? h - p.Hkv : h) * p.page_tokens * kRD);
        row[l] = lo[u];
        row[8 + l] = hi[u];
      }
    }
  }
}

}  // namespace
}  // namespace q3

extern "C" int q3_qkv_norm_rope_ragged(const void* qkv, int64_t qkv_stride, const void* q_norm_w,
                                       const void* k_norm_w, const int64_t* positions,
                                       int64_t pos_axis_stride, const float* inv_freq,
                                       const int64_t* slots, void* q_out, int64_t q_stride,
                                       void* k_pages, void* v_pages, int64_t n_tokens, int Hq,
                                       int Hkv, int head_dim, int page_tokens, int64_t num_pages,
                                       int sec_h, int sec_w, float eps, q3_stream_t stream) {
  using namespace q3;
  Q3_REQUIRE(head_dim == kRD, "q3_qkv_norm_rope_ragged: head_dim must be 128 (got %d)", head_dim);
  Q3_REQUIRE(n_tokens >= 0 && n_tokens < (1ll << 31) && Hq > 0 && Hkv > 0 && Hq <= 1024 &&
                 Hkv <= 1024 && page_tokens > 0 && num_pages > 0 && num_pages < (1ll << 31),
             "q3_qkv_norm_rope_ragged: bad shape n=%lld Hq=%d Hkv=%d", (long long)n_tokens, Hq,
             Hkv);
  Q3_REQUIRE(num_pages * page_tokens < (1ll << 31),
             "q3_qkv_norm_rope_ragged: %lld pages of %d positions pass 32-bit slots",
             (long long)num_pages, page_tokens);
  Q3_REQUIRE(sec_h >= 0 && sec_w >= 0 && 3 * sec_h <= kRD / 2 + 2 && 3 * sec_w <= kRD / 2 + 2,
             "q3_qkv_norm_rope_ragged: mrope sections exceed head_dim/2");
  if (n_tokens == 0) return Q3_OK;
  Q3_REQUIRE(qkv && q_norm_w && k_norm_w && positions && inv_freq && slots && q_out && k_pages &&
                 v_pages,
             "q3_qkv_norm_rope_ragged: null pointer");
  Q3_REQUIRE(qkv_stride >= (int64_t)(Hq + 2 * Hkv) * kRD && qkv_stride % 8 == 0 &&
                 q_stride >= (int64_t)Hq * kRD && q_stride % 8 == 0,
             "q3_qkv_norm_rope_ragged: row strides must cover a row and be multiples of 8");
  Q3_REQUIRE(aligned(qkv, 16) && aligned(q_norm_w, 16) && aligned(k_norm_w, 16) &&
                 aligned(positions, 8) && aligned(inv_freq, 4) && aligned(slots, 8) &&
                 aligned(q_out, 16) && aligned(k_pages, 16) && aligned(v_pages, 16),
             "q3_qkv_norm_rope_ragged: misaligned pointer");
  // heads of a token split over warps while that still fills idle SMs
  int parts = 1;
  while (parts < 8 && n_tokens * parts < (int64_t)num_sms() * kRWarps && parts * 4 < Hq) parts *= 2;
  RaggedRopeParams p{(const __nv_bfloat16*)qkv, qkv_stride, (const __nv_bfloat16*)q_norm_w,
                     (const __nv_bfloat16*)k_norm_w, positions, pos_axis_stride, inv_freq, slots,
                     (__nv_bfloat16*)q_out, q_stride, (__nv_bfloat16*)k_pages,
                     (__nv_bfloat16*)v_pages, num_pages * page_tokens, (int)n_tokens, parts, Hq,
                     Hkv, page_tokens, sec_h, sec_w, eps, device_error_word()};
  const int64_t ctas = (n_tokens * parts + kRWarps - 1) / kRWarps;
  return launch_ex(qkv_norm_rope_ragged_kernel, dim3((unsigned)ctas), dim3(kRWarps * 32), 0,
                   (cudaStream_t)stream, 1, p);
}
