// Head norm and rotation of a prompt chunk (or a decode position) in one pass:
// the fused q|k|v projection output [tokens, (Hq + 2 Hkv) D] becomes
//   q, k   y = fp16((x * rsqrt(mean(x^2) + eps)) * w), then rotate-half RoPE
//          fp16(y cos + rot(y) sin), products and sum rounded to fp32 separately
//   v      copied
// each contiguous, as the attention and the ring append take them.  New
// component: the reference's patched Qwen3 layer runs the head norms and the
// rotation as separate torch ops (qextract/patch.py:73-87 swaps only the layer
// norms).  The order of the sum of squares and every rounding equal
// qx_fused_rmsnorm over the heads followed by torch's x * cos + rot * sin in
// fp32, so the result is bit-identical to that sequence.
//
// Bound: HBM for a chunk (each value read and written once), launch latency
// for one token.  D / 8 lanes hold one head (16 bytes each: full sectors), so
// the sum is a butterfly over them and the rotation's partner (i +- D/2) sits
// D / 16 lanes away.  A CTA stays on one token: its cos / sin rows and the norm
// weights are read once into registers and serve HPL heads per lane group,
// whose loads are all in flight before the first is used.  2048 tokens of 32 + 2 x 8
// heads of 128: 12.3 us, 4.3 TB/s (8.0 at the copy rate; 10.5 in a graph of such calls), by
// load latency and issue (67 %).  The norm's products two an instruction, the sine negated once instead of the
// partner: 12.7 before; with six heads a lane group 14.5, with 256 threads 14.9, a root
// and a division for each head in every lane 13.9 (before that).  One token: 1.3 us.
#include <algorithm>

#include "qx_b200.h"
#include "qx_common.cuh"

namespace qx {
namespace nrope {

constexpr int THREADS = 128;

struct Params {
  const uint4* qkv;
  const uint4* qw;
  const uint4* kw;
  const float* cosr;  // [rope_rows][D]
  const float* sinr;
  uint4* q;
  uint4* k;
  uint4* v;
  int64_t rope_rows;  // token t of the call reads row t % rope_rows
  int hq, hkv;
  float eps;
};

// two fp32 products an instruction, each rounded as the scalar one
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 x, x, y;\n"
      "mov.b64 {%0, %1}, x; }"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

template <int D, int HPL>
__global__ void __launch_bounds__(THREADS) qk_norm_rope_kernel(const Params p) {
  pdl_trigger();
  constexpr int LPH = D / 8;          // lanes per head
  constexpr int HPP = THREADS / LPH;  // heads per pass of the CTA
  const int64_t tok = blockIdx.x;
  const int l = threadIdx.x % LPH;
  const int h0 = blockIdx.y * (HPP * HPL) + threadIdx.x / LPH;
  const int heads = p.hq + 2 * p.hkv;
  pdl_wait();
  const uint4 wq = __ldg(p.qw + l), wk = __ldg(p.kw + l);
  const uint4* src = p.qkv + tok * heads * LPH + l;
  uint4 x[HPL];
#pragma unroll
  for (int i = 0; i < HPL; ++i) {
    const int h = h0 + i * HPP;
    x[i] = h < heads ? src[int64_t(h) * LPH] : make_uint4(0u, 0u, 0u, 0u);
  }
  float c[8], s[8];
  {
    const int64_t row = tok % p.rope_rows;
    const float4* cr = reinterpret_cast<const float4*>(p.cosr + row * D + l * 8);
    const float4* sr = reinterpret_cast<const float4*>(p.sinr + row * D + l * 8);
    const float4 c0 = cr[0], c1 = cr[1], s0 = sr[0], s1 = sr[1];
    c[0] = c0.x, c[1] = c0.y, c[2] = c0.z, c[3] = c0.w, c[4] = c1.x, c[5] = c1.y, c[6] = c1.z, c[7] = c1.w;
    s[0] = s0.x, s[1] = s0.y, s[2] = s0.z, s[3] = s0.w, s[4] = s1.x, s[5] = s1.y, s[6] = s1.z, s[7] = s1.w;
  }
  if (l < LPH / 2)  // first half of the head: its partner enters negated
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j] = -s[j];
  const int vfirst = p.hq + p.hkv, warp_h = h0 - (threadIdx.x % 32) / LPH;
  float ss[HPL];
#pragma unroll
  for (int i = 0; i < HPL; ++i) {
    const uint32_t xd[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    ss[i] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 t = h2_to_f2(xd[j]);
      ss[i] = fmaf(t.x, t.x, ss[i]);
      ss[i] = fmaf(t.y, t.y, ss[i]);
    }
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss[i] += __shfl_xor_sync(0xffffffffu, ss[i], o);
  }
  // the root and the division once: lane i of a group does head i's
  float root = ss[0];
#pragma unroll
  for (int i = 1; i < HPL; ++i) root = l == i ? ss[i] : root;
  root = 1.0f / sqrtf(root * (1.0f / D) + p.eps);
#pragma unroll
  for (int i = 0; i < HPL; ++i) {
    const int h = h0 + i * HPP;
    const float r = HPL == 1 ? root : __shfl_sync(0xffffffffu, root, i, LPH);
    if (warp_h + i * HPP >= vfirst) {  // the warp's heads are values, or past the last
      if (h < heads) p.v[(tok * p.hkv + (h - vfirst)) * LPH + l] = x[i];
      continue;
    }
    const uint32_t xd[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    const uint4 w = h < p.hq ? wq : wk;
    const uint32_t wd[4] = {w.x, w.y, w.z, w.w};
    uint32_t yd[4], od[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = h2_to_f2(xd[j]), g = h2_to_f2(wd[j]);
      const float2 n = mul2(mul2(f, make_float2(r, r)), g);
      const __half2 y = __floats2half2_rn(n.x, n.y);
      yd[j] = *reinterpret_cast<const uint32_t*>(&y);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t pd = __shfl_xor_sync(0xffffffffu, yd[j], LPH / 2);
      const float2 y = h2_to_f2(yd[j]), t = h2_to_f2(pd);
      // (one at a time: two products and a sum of pairs come out fused, with other roundings)
      const __half2 o =
          __floats2half2_rn(__fadd_rn(__fmul_rn(y.x, c[2 * j]), __fmul_rn(t.x, s[2 * j])),
                            __fadd_rn(__fmul_rn(y.y, c[2 * j + 1]), __fmul_rn(t.y, s[2 * j + 1])));
      od[j] = *reinterpret_cast<const uint32_t*>(&o);
    }
    if (h < p.hq)
      p.q[(tok * p.hq + h) * LPH + l] = make_uint4(od[0], od[1], od[2], od[3]);
    else if (h < vfirst)
      p.k[(tok * p.hkv + (h - p.hq)) * LPH + l] = make_uint4(od[0], od[1], od[2], od[3]);
    else if (h < heads)
      p.v[(tok * p.hkv + (h - vfirst)) * LPH + l] = x[i];
  }
}

template <int D>
cudaError_t launch(const Params& p, int64_t tokens, cudaStream_t st) {
  constexpr int HPP = THREADS / (D / 8);
  const int heads = p.hq + 2 * p.hkv;
  const int passes = (heads + HPP - 1) / HPP;
  // One pass per CTA spreads few tokens over the SMs; with enough tokens to
  // fill them, three passes share the rotation row and keep three loads in flight.
  if (tokens * passes <= 4 * int64_t(device_sm_count()))
    return launch_pdl(qk_norm_rope_kernel<D, 1>, dim3(unsigned(tokens), unsigned(passes)), dim3(THREADS), 0, st, p);
  return launch_pdl(qk_norm_rope_kernel<D, 3>, dim3(unsigned(tokens), unsigned((passes + 2) / 3)), dim3(THREADS), 0,
                    st, p);
}

}  // namespace nrope
}  // namespace qx

using namespace qx;

extern "C" int qx_qk_norm_rope(const void* qkv, int64_t tokens, int q_heads, int kv_heads, int head_dim,
                               const void* q_norm_w, const void* k_norm_w, float eps, const float* cos,
                               const float* sin, int64_t rope_rows, void* q_out, void* k_out, void* v_out,
                               qx_stream_t stream) {
  QX_REQUIRE(tokens >= 0 && q_heads > 0 && kv_heads > 0, "qk_norm_rope: bad sizes tokens=%lld heads q=%d kv=%d",
             (long long)tokens, q_heads, kv_heads);
  QX_REQUIRE(head_dim == 64 || head_dim == 128 || head_dim == 256, "qk_norm_rope: head_dim=%d must be 64, 128 or 256",
             head_dim);
  if (tokens == 0) return QX_OK;
  QX_REQUIRE(tokens < (int64_t(1) << 31), "qk_norm_rope: tokens=%lld too large", (long long)tokens);
  QX_REQUIRE(int64_t(q_heads) + 2 * int64_t(kv_heads) <= 65535, "qk_norm_rope: too many heads");
  QX_REQUIRE(rope_rows >= 1 && tokens % rope_rows == 0,
             "qk_norm_rope: %lld rotation rows do not divide %lld tokens", (long long)rope_rows, (long long)tokens);
  QX_REQUIRE(qkv && q_norm_w && k_norm_w && cos && sin && q_out && k_out && v_out, "qk_norm_rope: null pointer");
  QX_REQUIRE(aligned(qkv, 16) && aligned(q_norm_w, 16) && aligned(k_norm_w, 16) && aligned(cos, 16) &&
                 aligned(sin, 16) && aligned(q_out, 16) && aligned(k_out, 16) && aligned(v_out, 16),
             "qk_norm_rope: tensors must be 16-byte aligned");
  nrope::Params p{};
  p.qkv = static_cast<const uint4*>(qkv);
  p.qw = static_cast<const uint4*>(q_norm_w);
  p.kw = static_cast<const uint4*>(k_norm_w);
  p.cosr = cos;
  p.sinr = sin;
  p.q = static_cast<uint4*>(q_out);
  p.k = static_cast<uint4*>(k_out);
  p.v = static_cast<uint4*>(v_out);
  p.rope_rows = rope_rows;
  p.hq = q_heads;
  p.hkv = kv_heads;
  p.eps = eps;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (head_dim) {
    case 64: QX_CUDA_TRY(nrope::launch<64>(p, tokens, st), "qk_norm_rope: launch"); break;
    case 128: QX_CUDA_TRY(nrope::launch<128>(p, tokens, st), "qk_norm_rope: launch"); break;
    default: QX_CUDA_TRY(nrope::launch<256>(p, tokens, st), "qk_norm_rope: launch"); break;
  }
  return check_launch("qk_norm_rope");
}
