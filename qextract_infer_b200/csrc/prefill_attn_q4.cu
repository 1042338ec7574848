// Prefill attention of a prompt chunk over the 4-bit ring KV cache (format:
// kv4.cuh) and over the chunk's own fp16 keys and values, before the chunk is
// appended.  The mask is qx_prefill_attention's: key kp is visible to query p
// iff kp <= p and (kp < sink or kp > p - window); the ring's slots sit at the
// positions its write rule gives them.  New component (the reference gathers
// the cache, qextract/kv_cache.py:96-112, and attends over the copy).
//
// Flash-attention form: one CTA = 4 warps = 64 query positions of one query
// head; key tiles of 64 (ring slots made fp16 on the way to shared memory,
// then the chunk's), S = Q K^T and O += P V on mma.sync with an online softmax.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "kv4.cuh"
#include "qx_b200.h"

namespace qx {
namespace pattn4 {

constexpr int WARPS = 4, THREADS = WARPS * 32, QROWS = WARPS * 16, KT = 64;

struct Params {
  const __half* q;   // [B][n][Hq][D]
  const __half* kn;  // [B][n][Hkv][D]
  const __half* vn;
  const unsigned char* kc;
  const uint16_t* kp;
  const unsigned char* vc;
  const uint16_t* vp;
  __half* out;
  const int64_t* counts;
  int64_t count, cap;
  int n, hq, hkv, G, sink, window;
  float scale_log2;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Where the ring's tokens stand relative to the chunk's first position c0.
struct Ring {
  int valid;    // slots that hold a token
  int newest;   // ring index (slot - sink) of position c0 - 1; -1: none
  int sinks;    // chunk keys below this index are sinks
  __device__ Ring(int64_t c0, int sink, int window) {
    valid = kv4::valid_slots(c0, sink, window);
    newest = c0 > sink ? int((c0 - 1 - sink) % window) : -1;
    sinks = c0 >= sink ? 0 : int(sink - c0);
  }
  // is the token of `slot` (< valid) visible to chunk row `row`?
  __device__ bool sees(int slot, int row, int sink, int window) const {
    if (slot < sink) return true;
    int age = newest - (slot - sink);  // 0: position c0 - 1
    if (age < 0) age += window;
    return -1 - age > row - window;
  }
  // is the chunk's key `j` visible to row `row`?
  __device__ bool sees_new(int j, int row, int window) const { return j <= row && (j < sinks || j > row - window); }
};

// One value of the ring: K (which = 0) or V, dimension d of storage row `row`.
template <int D, int NG>
__device__ float ring_value(const Params& p, int which, int64_t row, int d) {
  constexpr int NI = D / 32;
  const int j = d >> 3, e = d & 7, c = j & 3, i = j >> 2;
  const int at = which == 0 ? 2 * (c * NI + i) + (e & 1) : (2 * c + (e & 1)) * NI + i;
  const uint16_t* codes = reinterpret_cast<const uint16_t*>(which == 0 ? p.kc : p.vc);
  const uint32_t w = (which == 0 ? p.kp : p.vp)[row * NG + d * NG / D];
  const int code = (codes[row * (D / 4) + at] >> (4 * (e >> 1))) & 15;
  return __half2float(__ushort_as_half(uint16_t(w & 0xFFF0u))) * float(code - int(w & 15u));
}

// A row whose result is not finite, done again by one warp over its visible keys
// alone: in a tile product a hidden key's weight 0 times an infinite or NaN value
// is NaN.  Two passes (maximum; weights and sums), plain fp32.
template <int D, int NG>
__device__ __noinline__ void redo_row(const Params& p, const Ring& ring, int b, int h, int row, int lane) {
  constexpr int E = D / 32;
  const int kvh = h / p.G;
  const int64_t base = (int64_t(b) * p.hkv + kvh) * p.cap;
  const int64_t at = ((int64_t(b) * p.n + row) * p.hq + h) * D + lane;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) q[e] = __half2float(p.q[at + 32 * e]) * p.scale_log2, acc[e] = 0.f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int t = 0; t <= ring.valid + row; ++t) {
      const bool old = t < ring.valid;
      const int j = t - ring.valid;
      if (old ? !ring.sees(t, row, p.sink, p.window) : !ring.sees_new(j, row, p.window)) continue;
      const int64_t fresh = ((int64_t(b) * p.n + (old ? 0 : j)) * p.hkv + kvh) * D + lane;
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e)
        s = fmaf(q[e], old ? ring_value<D, NG>(p, 0, base + t, lane + 32 * e) : __half2float(p.kn[fresh + 32 * e]), s);
      s = warp_sum(s);
      if (pass == 0) {
        m = fmaxf(m, s);
        continue;
      }
      const float w = exp2f(s - m);
      l += w;
#pragma unroll
      for (int e = 0; e < E; ++e)
        acc[e] = fmaf(w, old ? ring_value<D, NG>(p, 1, base + t, lane + 32 * e) : __half2float(p.vn[fresh + 32 * e]),
                      acc[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) p.out[at + 32 * e] = __float2half_rn(acc[e] / l);
}

template <int D, int NG>
__global__ void __launch_bounds__(THREADS) prefill_attn_q4_kernel(const Params p) {
  pdl_trigger();
  constexpr int NI = D / 32, LPR = D / 8, ROWB = D * 2;
  __shared__ __align__(128) unsigned char s_k[KT * ROWB], s_v[KT * ROWB];
  auto swz = [](int r, int ch) { return uint32_t(r * ROWB + ((ch ^ (r & 7)) << 4)); };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int h = blockIdx.y, b = blockIdx.z, kvh = h / p.G;
  const int r0 = blockIdx.x * QROWS;
  const int rowA = r0 + warp * 16 + g, rowB = rowA + 8;
  pdl_wait();
  const Ring ring(kv4::count_of(p.counts, p.count, b), p.sink, p.window);
  const int last = min(p.n, r0 + QROWS) - 1;
  const int ncache = (ring.valid + KT - 1) / KT;
  const int ntiles = ncache + last / KT + 1;
  const uint32_t ks = smem_u32(s_k), vs = smem_u32(s_v);
  const int64_t base = (int64_t(b) * p.hkv + kvh) * p.cap;

  uint32_t qa[D / 16][4];
  {
    const bool okA = rowA < p.n, okB = rowB < p.n;
    const __half* qA = p.q + ((int64_t(b) * p.n + (okA ? rowA : 0)) * p.hq + h) * D;
    const __half* qB = p.q + ((int64_t(b) * p.n + (okB ? rowB : 0)) * p.hq + h) * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const int d0 = kk * 16 + 2 * c;
      qa[kk][0] = okA ? *reinterpret_cast<const uint32_t*>(qA + d0) : 0u;
      qa[kk][1] = okB ? *reinterpret_cast<const uint32_t*>(qB + d0) : 0u;
      qa[kk][2] = okA ? *reinterpret_cast<const uint32_t*>(qA + d0 + 8) : 0u;
      qa[kk][3] = okB ? *reinterpret_cast<const uint32_t*>(qB + d0 + 8) : 0u;
    }
  }
  float o[D / 8][4];
#pragma unroll
  for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  float m_r[2] = {-INFINITY, -INFINITY}, l_r[2] = {0.f, 0.f};
  const int mi = lane >> 3, ri = lane & 7;

  for (int t = 0; t < ntiles; ++t) {
    __syncthreads();
    const bool cache = t < ncache;
    const int k0 = cache ? t * KT : (t - ncache) * KT;
    for (int idx = tid; idx < KT * LPR; idx += THREADS) {
      const int r = idx / LPR, ch = idx % LPR;
      uint4 kv = make_uint4(0u, 0u, 0u, 0u), vv = kv;
      if (cache) {
        if (k0 + r < ring.valid) {
          const int64_t row = base + k0 + r;
          const int cc = ch & 3, i = ch >> 2;
          const uint16_t* vr = reinterpret_cast<const uint16_t*>(p.vc) + row * (2 * LPR);
          const uint32_t kw = *(reinterpret_cast<const uint32_t*>(p.kc) + row * LPR + cc * NI + i);
          const uint32_t vw = uint32_t(vr[2 * cc * NI + i]) | (uint32_t(vr[(2 * cc + 1) * NI + i]) << 16);
          const uint32_t kq = p.kp[row * NG + i * NG / NI], vq = p.vp[row * NG + i * NG / NI];
          uint32_t w[4];
          kv4::dequant_word(kw, kv4::group_scale(kq | (kq << 16)), w);
          kv = make_uint4(w[0], w[1], w[2], w[3]);
          kv4::dequant_word(vw, kv4::group_scale(vq | (vq << 16)), w);
          vv = make_uint4(w[0], w[1], w[2], w[3]);
        }
      } else if (k0 + r < p.n) {
        const int64_t off = ((int64_t(b) * p.n + k0 + r) * p.hkv + kvh) * D + ch * 8;
        kv = *reinterpret_cast<const uint4*>(p.kn + off);
        vv = *reinterpret_cast<const uint4*>(p.vn + off);
      }
      *reinterpret_cast<uint4*>(s_k + swz(r, ch)) = kv;
      *reinterpret_cast<uint4*>(s_v + swz(r, ch)) = vv;
    }
    __syncthreads();
    float s[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
      for (int j2 = 0; j2 < 4; ++j2) {
        uint32_t bk[4];
        ldsm_x4(bk, ks + swz(j2 * 16 + 8 * (mi >> 1) + ri, 2 * kk + (mi & 1)));
        mma_16816(s[2 * j2], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], bk[0], bk[1]);
        mma_16816(s[2 * j2 + 1], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], bk[2], bk[3]);
      }
    }
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
#pragma unroll
      for (int e1 = 0; e1 < 2; ++e1) {
        const int key = k0 + j * 8 + 2 * c + e1;
        bool vA, vB;
        if (cache) {
          vA = key < ring.valid && ring.sees(key, rowA, p.sink, p.window);
          vB = key < ring.valid && ring.sees(key, rowB, p.sink, p.window);
        } else {
          vA = key < p.n && ring.sees_new(key, rowA, p.window);
          vB = key < p.n && ring.sees_new(key, rowB, p.window);
        }
        s[j][e1] = vA ? s[j][e1] * p.scale_log2 : -INFINITY;
        s[j][2 + e1] = vB ? s[j][2 + e1] * p.scale_log2 : -INFINITY;
        mx0 = fmaxf(mx0, s[j][e1]);
        mx1 = fmaxf(mx1, s[j][2 + e1]);
      }
    }
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    const float mn0 = fmaxf(m_r[0], mx0), mn1 = fmaxf(m_r[1], mx1);
    const float mb0 = mn0 == -INFINITY ? 0.f : mn0, mb1 = mn1 == -INFINITY ? 0.f : mn1;
    const float al0 = exp2f(m_r[0] - mb0), al1 = exp2f(m_r[1] - mb1);
    m_r[0] = mn0;
    m_r[1] = mn1;
    float ls0 = 0.f, ls1 = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s[j][0] = exp2f(s[j][0] - mb0 + 14.f);
      s[j][1] = exp2f(s[j][1] - mb0 + 14.f);
      s[j][2] = exp2f(s[j][2] - mb1 + 14.f);
      s[j][3] = exp2f(s[j][3] - mb1 + 14.f);
      ls0 += s[j][0] + s[j][1];
      ls1 += s[j][2] + s[j][3];
    }
    l_r[0] = l_r[0] * al0 + ls0;
    l_r[1] = l_r[1] * al1 + ls1;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      o[j][0] *= al0;
      o[j][1] *= al0;
      o[j][2] *= al1;
      o[j][3] *= al1;
    }
#pragma unroll
    for (int kq = 0; kq < 4; ++kq) {
      const uint32_t pa0 = pack_h2(s[2 * kq][0], s[2 * kq][1]);
      const uint32_t pa1 = pack_h2(s[2 * kq][2], s[2 * kq][3]);
      const uint32_t pa2 = pack_h2(s[2 * kq + 1][0], s[2 * kq + 1][1]);
      const uint32_t pa3 = pack_h2(s[2 * kq + 1][2], s[2 * kq + 1][3]);
#pragma unroll
      for (int jj = 0; jj < D / 16; ++jj) {
        uint32_t bv[4];
        ldsm_x4_t(bv, vs + swz(kq * 16 + 8 * (mi & 1) + ri, 2 * jj + (mi >> 1)));
        mma_16816(o[2 * jj], pa0, pa1, pa2, pa3, bv[0], bv[1]);
        mma_16816(o[2 * jj + 1], pa0, pa1, pa2, pa3, bv[2], bv[3]);
      }
    }
  }
  uint32_t redo = 0;  // bit r: row r of the warp's 16
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    l_r[k] += __shfl_xor_sync(0xffffffffu, l_r[k], 1);
    l_r[k] += __shfl_xor_sync(0xffffffffu, l_r[k], 2);
    const int row = k ? rowB : rowA;
    const float inv = 1.f / l_r[k];
    bool fine = true;
#pragma unroll
    for (int j = 0; j < D / 8; ++j) {
      const float x = o[j][2 * k] * inv, y = o[j][2 * k + 1] * inv;
      fine = fine && fabsf(x) <= 65504.f && fabsf(y) <= 65504.f;
      if (row < p.n)
        *reinterpret_cast<uint32_t*>(p.out + ((int64_t(b) * p.n + row) * p.hq + h) * D + 8 * j + 2 * c) = pack_h2(x, y);
    }
    const uint32_t bad = __ballot_sync(0xffffffffu, !fine && row < p.n);
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if ((bad >> (4 * r)) & 15u) redo |= 1u << (8 * k + r);
  }
  __syncwarp();
  for (; redo; redo &= redo - 1) redo_row<D, NG>(p, ring, b, h, r0 + warp * 16 + __ffs(redo) - 1, lane);
}

template <int D, int NG>
cudaError_t launch(const Params& p, int batch, cudaStream_t st) {
  return launch_pdl(prefill_attn_q4_kernel<D, NG>, dim3((p.n + QROWS - 1) / QROWS, p.hq, batch), dim3(THREADS), 0, st, p);
}

}  // namespace pattn4
}  // namespace qx

using namespace qx;

extern "C" size_t qx_prefill_attention_q4_workspace_size(int batch, int n, int q_heads, int kv_heads, int head_dim,
                                                         int sink, int window) {
  (void)batch, (void)n, (void)q_heads, (void)kv_heads, (void)head_dim, (void)sink, (void)window;
  return 0;
}

extern "C" int qx_prefill_attention_q4(const void* q, const void* k_new, const void* v_new, const void* k_codes,
                                       const void* k_params, const void* v_codes, const void* v_params, void* out,
                                       int batch, int n, int q_heads, int kv_heads, int head_dim, int group, int sink,
                                       int window, int64_t count, const int64_t* counts, float softmax_scale,
                                       void* workspace, size_t workspace_bytes, qx_stream_t stream) {
  (void)workspace, (void)workspace_bytes;
  const int rc = kv4::check_ring("prefill_attention_q4", batch, kv_heads, head_dim, group, sink, window);
  if (rc != QX_OK) return rc;
  QX_REQUIRE(n >= 0 && q_heads > 0 && q_heads % kv_heads == 0 && q_heads / kv_heads <= 16,
             "prefill_attention_q4: bad sizes n=%d heads q=%d kv=%d (a group of 1 to 16)", n, q_heads, kv_heads);
  QX_REQUIRE(batch <= 65535 && kv_heads <= 65535 && n < (1 << 26), "prefill_attention_q4: batch, heads or chunk too large");
  QX_REQUIRE(counts || count >= 0, "prefill_attention_q4: negative count");
  if (batch == 0 || n == 0) return QX_OK;
  QX_REQUIRE(q && k_new && v_new && k_codes && k_params && v_codes && v_params && out,
             "prefill_attention_q4: null pointer");
  QX_REQUIRE(aligned(q, 16) && aligned(k_new, 16) && aligned(v_new, 16) && aligned(k_codes, 16) &&
                 aligned(v_codes, 16) && aligned(k_params, 16) && aligned(v_params, 16) && aligned(out, 16),
             "prefill_attention_q4: tensors must be 16-byte aligned");
  pattn4::Params p{};
  p.q = static_cast<const __half*>(q);
  p.kn = static_cast<const __half*>(k_new);
  p.vn = static_cast<const __half*>(v_new);
  p.kc = static_cast<const unsigned char*>(k_codes);
  p.kp = static_cast<const uint16_t*>(k_params);
  p.vc = static_cast<const unsigned char*>(v_codes);
  p.vp = static_cast<const uint16_t*>(v_params);
  p.out = static_cast<__half*>(out);
  p.counts = counts;
  p.count = count;
  p.cap = kv4::capacity(sink, window);
  p.n = n;
  p.hq = q_heads;
  p.hkv = kv_heads;
  p.G = q_heads / kv_heads;
  p.sink = sink;
  p.window = window;
  p.scale_log2 = (softmax_scale > 0.f ? softmax_scale : 1.0f / sqrtf(float(head_dim))) * 1.4426950408889634f;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (head_dim == 64)
    e = group == 32 ? pattn4::launch<64, 2>(p, batch, st) : pattn4::launch<64, 1>(p, batch, st);
  else
    e = group == 32   ? pattn4::launch<128, 4>(p, batch, st)
        : group == 64 ? pattn4::launch<128, 2>(p, batch, st)
                      : pattn4::launch<128, 1>(p, batch, st);
  QX_CUDA_TRY(e, "prefill_attention_q4: launch");
  return check_launch("prefill_attention_q4");
}
