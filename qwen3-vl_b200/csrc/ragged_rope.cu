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
// Bound by HBM: each qkv row is read once, each q, k, v row written once.
// Eight lanes own one head row; lane l holds dims 8l..8l+7 and their rotation
// partners 64+8l..64+8l+7 (two 16-byte loads), so the rotation needs no
// shuffle and a pair shares one cosine and sine.  A CTA takes a few tokens: 64
// threads per token compute the angles once for all heads.
#include <math.h>

#include "common.cuh"

namespace q3 {
namespace {

constexpr int kRD = 128;
constexpr int kRThreads = 256;
constexpr int kRRows = kRThreads / 8;  // head rows per CTA pass

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
  int n, Hq, Hkv, page_tokens, sec_h, sec_w;
  float eps;
  int* err;
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y), c = unpack_bf16x2(u.z),
               d = unpack_bf16x2(u.w);
  v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  v[4] = c.x; v[5] = c.y; v[6] = d.x; v[7] = d.y;
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                    pack_bf16x2(v[6], v[7]));
}

template <int TPC>
__global__ void __launch_bounds__(kRThreads) qkv_norm_rope_ragged_kernel(RaggedRopeParams p) {
  __shared__ __align__(16) float s_cos[TPC][64];
  __shared__ __align__(16) float s_sin[TPC][64];
  __shared__ int64_t s_kv[TPC];  // element offset of (slot, KV head 0); -1: skip the token
  pdl_launch();
  pdl_wait();
  const int t0 = blockIdx.x * TPC;
  const int H = p.Hq + 2 * p.Hkv;
  if (threadIdx.x < TPC) {
    const int t = t0 + threadIdx.x;
    int64_t off = -1;
    if (t < p.n) {
      const int64_t slot = p.slots[t];
      if (slot >= 0 && slot < p.n_slots) {
        const uint32_t pg = (uint32_t)slot / (uint32_t)p.page_tokens;
        off = ((int64_t)pg * p.Hkv * p.page_tokens +
               ((uint32_t)slot - pg * (uint32_t)p.page_tokens)) * kRD;
      } else if (slot != -1) {
        report_timeout(p.err, 0x911);
      }
    }
    s_kv[threadIdx.x] = off;
  }
  for (int i = threadIdx.x; i < TPC * 64; i += kRThreads) {
    const int tt = i >> 6, j = i & 63, t = t0 + tt;
    if (t < p.n) {
      const int axis = (j % 3 == 1 && j < 3 * p.sec_h) ? 1 : (j % 3 == 2 && j < 3 * p.sec_w) ? 2 : 0;
      // half turns: an angle a is a / pi of them, reduced to [-1, 1]
      double h = (double)p.pos[axis * p.pos_stride + t] * (double)p.inv_freq[j] *
                 0.31830988618379067154;
      h -= 2.0 * rint(0.5 * h);
      float sn, cs;
      sincospif((float)h, &sn, &cs);
      s_cos[tt][j] = cs;
      s_sin[tt][j] = sn;
    }
  }
  __syncthreads();

  const int l = threadIdx.x & 7, row0 = threadIdx.x >> 3;
  const uint4 qw0 = reinterpret_cast<const uint4*>(p.qw)[l];
  const uint4 qw1 = reinterpret_cast<const uint4*>(p.qw)[8 + l];
  const uint4 kw0 = reinterpret_cast<const uint4*>(p.kw)[l];
  const uint4 kw1 = reinterpret_cast<const uint4*>(p.kw)[8 + l];
  const int rows = TPC * H;
  // the loop runs by whole warps (4 rows each): the shuffles stay converged
  for (int base = 0; base < rows; base += kRRows) {
    const int r = base + row0;
    const int tt = r / H, h = r - tt * H;
    const int64_t kv = r < rows ? s_kv[min(tt, TPC - 1)] : -1;
    const bool live = kv >= 0;
    uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
    if (live) {
      const uint4* src = reinterpret_cast<const uint4*>(p.qkv + (int64_t)(t0 + tt) * p.qkv_stride +
                                                        (int64_t)h * kRD);
      lo = src[l];
      hi = src[8 + l];
    }
    const bool is_v = h >= p.Hq + p.Hkv;
    float a[8], b[8];
    unpack8(lo, a);
    unpack8(hi, b);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(a[i], a[i], fmaf(b[i], b[i], ss));
    ss += __shfl_xor_sync(0xffffffffu, ss, 1);
    ss += __shfl_xor_sync(0xffffffffu, ss, 2);
    ss += __shfl_xor_sync(0xffffffffu, ss, 4);
    if (!live) continue;
    if (!is_v) {
      const bool is_q = h < p.Hq;
      const float rs = 1.0f / sqrtf(ss * (1.0f / kRD) + p.eps);
      float wa[8], wb[8];
      unpack8(is_q ? qw0 : kw0, wa);
      unpack8(is_q ? qw1 : kw1, wb);
      float oa[8], ob[8];
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 c = *reinterpret_cast<const float4*>(&s_cos[tt][l * 8 + i]);
        const float4 s = *reinterpret_cast<const float4*>(&s_sin[tt][l * 8 + i]);
        const float cc[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float na = a[i + e] * rs * wa[i + e], nb = b[i + e] * rs * wb[i + e];
          oa[i + e] = fmaf(na, cc[e], -nb * sn[e]);
          ob[i + e] = fmaf(nb, cc[e], na * sn[e]);
        }
      }
      lo = pack8(oa);
      hi = pack8(ob);
    }
    __nv_bfloat16* dst;
    if (h < p.Hq)
      dst = p.q_out + (int64_t)(t0 + tt) * p.q_stride + (int64_t)h * kRD;
    else if (!is_v)
      dst = p.k_pages + kv + (int64_t)(h - p.Hq) * p.page_tokens * kRD;
    else
      dst = p.v_pages + kv + (int64_t)(h - p.Hq - p.Hkv) * p.page_tokens * kRD;
    reinterpret_cast<uint4*>(dst)[l] = lo;
    reinterpret_cast<uint4*>(dst)[8 + l] = hi;
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
                 Hkv <= 1024 && page_tokens > 0 && num_pages > 0,
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
  RaggedRopeParams p{(const __nv_bfloat16*)qkv, qkv_stride, (const __nv_bfloat16*)q_norm_w,
                     (const __nv_bfloat16*)k_norm_w, positions, pos_axis_stride, inv_freq, slots,
                     (__nv_bfloat16*)q_out, q_stride, (__nv_bfloat16*)k_pages,
                     (__nv_bfloat16*)v_pages, num_pages * page_tokens, (int)n_tokens, Hq, Hkv,
                     page_tokens, sec_h, sec_w, eps, device_error_word()};
  cudaStream_t st = (cudaStream_t)stream;
  if (n_tokens <= 4 * (int64_t)num_sms())
    return launch_ex(qkv_norm_rope_ragged_kernel<1>, dim3((unsigned)n_tokens), dim3(kRThreads), 0,
                     st, 1, p);
  return launch_ex(qkv_norm_rope_ragged_kernel<4>, dim3((unsigned)((n_tokens + 3) / 4)),
                   dim3(kRThreads), 0, st, 1, p);
}
