// Decode attention over the 4-bit ring KV cache (format: kv4.cuh): one query
// token per sequence, grouped-query heads, every valid slot.
//   out[h] = sum_t softmax_t(scale q[h] . K[t]) V[t],  K, V = s (c - z)
// New component (the reference has no attention kernel; semantics: HF Qwen3
// eager attention over the cache's valid slots, whose order does not matter).
//
// Both products run on the tensor cores with the cache as the A operand
// (mma.sync m16n8k16: 16 tokens or 16 head dimensions by 8 query heads), so a
// KV head's group of up to 8 query heads fills the N side (two N tiles up to
// 16).  tcgen05 would need 128 rows of M: the cache rows would have to pass
// through shared memory as fp16, four times their bytes, for a product whose
// arithmetic is a small part of the time.
//   S^T = K Q^T   the codes enter as fp16 subnormals: a mask of a 32-bit word
//                 is the pair c 2^-24 (or 16 c 2^-24, whose q comes divided by
//                 16), exact, one instruction a pair.  Scale and zero point act
//                 on the fp32 accumulator per token and group:
//                 s (sum q c - z sum q).
//   O^T = V^T P^T the token sits on the K side, so V's scale cannot act on the
//                 accumulator; the pairs are made exact fp16 s (c - z) in three
//                 instructions.  P^T comes from S^T's accumulator layout by
//                 movmatrix, in fp16 scaled by 2^14 (its subnormals then start
//                 at weights of 2^-28 of the largest), summed in fp32.
// The online softmax keeps a running maximum and sum per warp and head in fp32.
//
// Loads go from global memory straight to the MMA fragments (the format puts
// each lane's share of a row side by side), one step of 32 tokens ahead; no
// shared memory until the four warps of a CTA join their results.  A warp takes
// every (4 nsplit)-th step; with more than one split the CTAs write fp32 partial
// results and a second kernel joins them.
#include <algorithm>
#include <cmath>

#include "kv4.cuh"
#include "qx_b200.h"

namespace qx {
namespace dattn4 {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int STEP = 32;          // tokens per warp step
constexpr float PSHIFT = 14.f;    // P in fp16 carries 2^14
constexpr int MAX_SPLITS = 64;

struct Params {
  const __half* q;
  const unsigned char* kc;
  const uint16_t* kp;
  const unsigned char* vc;
  const uint16_t* vp;
  __half* out;
  float* part_o;   // [batch][q_heads][nsplit][D]
  float2* part_ml;  // [batch][q_heads][nsplit]
  const int64_t* counts;
  int64_t count, cap;
  int hq, hkv, G, sink, window, nsplit;
  float scale_log2;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
template <int WORDS>
__device__ __forceinline__ void load_words(const void* p, uint32_t (&w)[WORDS]) {
  if constexpr (WORDS == 4) {
    const uint4 v = ldg_stream_v4(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (WORDS == 2) {
    const uint2 v = __ldcs(static_cast<const uint2*>(p));
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = __ldcs(static_cast<const unsigned*>(p));
  }
}

// what a lane holds of 16 tokens: K rows g and g + 8 (a quarter of each), V of
// tokens 2c, 2c + 1, 2c + 8, 2c + 9 (an eighth of each), and their params
template <int D, int NG>
struct Frag {
  static constexpr int NI = D / 32;
  static constexpr int KPW = NG > 2 ? 2 : 1;  // 32-bit words of a K row's params
  uint32_t k[2][NI];
  uint32_t v[4][NI / 2];
  uint32_t kp[2][KPW];
  uint32_t vp[2][NG];  // token pairs (2c, 2c + 1) and (2c + 8, 2c + 9)

  __device__ __forceinline__ void load(const unsigned char* kc, const uint16_t* kpar, const unsigned char* vc,
                                       const uint16_t* vpar, int64_t row0, int g, int c) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t row = row0 + g + 8 * r;
      load_words<NI>(kc + row * (D / 2) + c * (D / 8), k[r]);
      const uint16_t* pp = kpar + row * NG;
      if constexpr (NG == 1)
        kp[r][0] = __ldcs(pp);
      else
        load_words<KPW>(pp, kp[r]);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t)
      load_words<NI / 2>(vc + (row0 + 2 * c + (t & 1) + (t >> 1) * 8) * (D / 2) + g * (D / 16), v[t]);
#pragma unroll
    for (int t = 0; t < 2; ++t) load_words<NG>(vpar + (row0 + 2 * c + t * 8) * NG, vp[t]);
  }
  __device__ __forceinline__ uint32_t kparam(int r, int grp) const {
    return NG == 1 ? kp[r][0] : (grp & 1) ? kp[r][grp >> 1] >> 16 : kp[r][grp >> 1] & 0xFFFFu;
  }
  // the pair's params of one group: token 2c in the low half
  __device__ __forceinline__ uint32_t vparam(int t, int grp) const {
    if constexpr (NG == 1) return vp[t][0];
    return prmt(vp[t][grp >> 1], vp[t][NG / 2 + (grp >> 1)], (grp & 1) ? 0x7632u : 0x5410u);
  }
};

template <int D, int NG, int NT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 3 : 2) decode_attn_q4_kernel(const Params p) {
  pdl_trigger();
  constexpr int NI = D / 32, IPG = NI / NG;  // 32-value blocks of a row, and of a group
  constexpr int SROW = D + 1;                // odd: the column writes below meet no bank twice
  __shared__ float s_o[WARPS][8 * NT][SROW];
  __shared__ float s_m[WARPS][8 * NT], s_l[WARPS][8 * NT];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int64_t base = (int64_t(b) * p.hkv + kvh) * p.cap;
  const unsigned char* kc = p.kc + base * (D / 2);
  const unsigned char* vc = p.vc + base * (D / 2);
  const uint16_t* kp = p.kp + base * NG;
  const uint16_t* vp = p.vp + base * NG;
  pdl_wait();
  const int valid = kv4::valid_slots(kv4::count_of(p.counts, p.count, b), p.sink, p.window);
  const int steps = (valid + STEP - 1) / STEP, stride = p.nsplit * WARPS;
  int step = split * WARPS + warp;

  Frag<D, NG> nxt[2];
  if (step < steps)
#pragma unroll
    for (int u = 0; u < 2; ++u) nxt[u].load(kc, kp, vc, vp, int64_t(step) * STEP + u * 16, g, c);

  // Q^T fragments: head g (of N tile nt), values 32 i + 8 c ..; a head is scaled by
  // the power of two that brings its largest value to [2^10, 2^11), undone in
  // hf: the second pair of each k step is divided by 16 (its codes come
  // multiplied by 16), which then costs no bits that count.
  uint32_t qb[NT][NI][4];
  float qs[NT][NG][2];  // 2^-24 sum of the scaled q over a group, of heads 2c, 2c + 1
  float hf[NT][2];      // accumulator -> log2 domain
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int h = nt * 8 + g;
    uint4 v[NI];
    float top = 0.f, sum[NG];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      v[i] = make_uint4(0u, 0u, 0u, 0u);
      if (h < p.G)
        v[i] = *reinterpret_cast<const uint4*>(p.q + ((int64_t(b) * p.hq + int64_t(kvh) * p.G + h) * D + 32 * i + 8 * c));
      const uint32_t d[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = h2_to_f2(d[e]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = top > 0.f && top <= 65504.f ? int(__float_as_uint(top) >> 23) - 127 : 10;
    const float up = __uint_as_float(uint32_t(127 + 10 - ex) << 23), down = __uint_as_float(uint32_t(127 + ex - 10) << 23);
#pragma unroll
    for (int n = 0; n < NG; ++n) sum[n] = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const uint32_t d[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float2 f = h2_to_f2(d[e]);
        f.x *= up;
        f.y *= up;
        sum[i / IPG] += f.x + f.y;
        qb[nt][i][e] = (e & 1) ? pack_h2(f.x * 0.0625f, f.y * 0.0625f) : pack_h2(f.x, f.y);
      }
    }
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 1);
      sum[n] += __shfl_xor_sync(0xffffffffu, sum[n], 2);
      qs[nt][n][0] = __shfl_sync(0xffffffffu, sum[n], 8 * c) * 0x1p-24f;
      qs[nt][n][1] = __shfl_sync(0xffffffffu, sum[n], 8 * c + 4) * 0x1p-24f;
    }
    const float k = down * 0x1p24f * p.scale_log2;
    hf[nt][0] = __shfl_sync(0xffffffffu, k, 8 * c);
    hf[nt][1] = __shfl_sync(0xffffffffu, k, 8 * c + 4);
  }

  float o[NI][2][NT][4];
#pragma unroll
  for (int i = 0; i < NI; ++i)
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) o[i][f][nt][0] = o[i][f][nt][1] = o[i][f][nt][2] = o[i][f][nt][3] = 0.f;
  float m_r[NT][2], l_r[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m_r[nt][0] = m_r[nt][1] = -INFINITY, l_r[nt][0] = l_r[nt][1] = 0.f;

  for (; step < steps; step += stride) {
    Frag<D, NG> cur[2] = {nxt[0], nxt[1]};
    if (step + stride < steps)
#pragma unroll
      for (int u = 0; u < 2; ++u) nxt[u].load(kc, kp, vc, vp, int64_t(step + stride) * STEP + u * 16, g, c);
    const int left = valid - step * STEP;  // tokens of this step that exist

    // scores: rows g, g + 8 (e >> 1) by heads 2c, 2c + 1 (e & 1)
    float s[2][NT][4];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) s[u][nt][0] = s[u][nt][1] = s[u][nt][2] = s[u][nt][3] = 0.f;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
        for (int i = n * IPG; i < (n + 1) * IPG; ++i) {
          const uint32_t w0 = cur[u].k[0][i], w1 = cur[u].k[1][i], h0 = w0 >> 8, h1 = w1 >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_16816(acc[nt], w0 & 0x000F000Fu, w1 & 0x000F000Fu, w0 & 0x00F000F0u, w1 & 0x00F000F0u, qb[nt][i][0],
                      qb[nt][i][1]);
            mma_16816(acc[nt], h0 & 0x000F000Fu, h1 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x00F000F0u, qb[nt][i][2],
                      qb[nt][i][3]);
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t w = cur[u].kparam(r, n);
          const float sc = __half2float(__ushort_as_half(uint16_t(w & 0xFFF0u)));
          const float z = float(w & 15u);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            s[u][nt][2 * r] = fmaf(sc, fmaf(-z, qs[nt][n][0], acc[nt][2 * r]), s[u][nt][2 * r]);
            s[u][nt][2 * r + 1] = fmaf(sc, fmaf(-z, qs[nt][n][1], acc[nt][2 * r + 1]), s[u][nt][2 * r + 1]);
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][nt][e] *= hf[nt][e & 1];  // to the log2 domain
    }
    if (left < STEP) {  // the last step: slots past the valid ones may hold anything
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (u * 16 + g + 8 * (e >> 1) >= left) s[u][nt][e] = -INFINITY;
        // scale 0: P is 0 there, and 0 times a NaN would not be
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int t0 = u * 16 + 8 * t + 2 * c;
          const uint32_t keep = (t0 < left ? 0xFFFFu : 0u) | (t0 + 1 < left ? 0xFFFF0000u : 0u);
          if constexpr (NG == 1) {
            cur[u].vp[t][0] &= keep;
          } else {
#pragma unroll
            for (int n = 0; n < NG; ++n) cur[u].vp[t][n] &= n < NG / 2 ? (keep & 0xFFFFu) * 0x10001u : (keep >> 16) * 0x10001u;
          }
        }
      }
    }
    // online softmax
    bool grew = false;
    float alpha[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float mx = fmaxf(fmaxf(s[0][nt][k], s[0][nt][2 + k]), fmaxf(s[1][nt][k], s[1][nt][2 + k]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m_r[nt][k], mx), mb = mn == -INFINITY ? 0.f : mn;
        alpha[nt][k] = ex2(m_r[nt][k] - mb);
        grew = grew || mn != m_r[nt][k];
        m_r[nt][k] = mn;
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            s[u][nt][2 * r + k] = ex2(s[u][nt][2 * r + k] - mb + PSHIFT);
            sum += s[u][nt][2 * r + k];
          }
        l_r[nt][k] = fmaf(l_r[nt][k], alpha[nt][k], sum);
      }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            o[i][f][nt][0] *= alpha[nt][0];
            o[i][f][nt][1] *= alpha[nt][1];
            o[i][f][nt][2] *= alpha[nt][0];
            o[i][f][nt][3] *= alpha[nt][1];
          }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        pb[nt][0] = transpose8x8(pack_h2(s[u][nt][0], s[u][nt][1]));
        pb[nt][1] = transpose8x8(pack_h2(s[u][nt][2], s[u][nt][3]));
      }
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const kv4::GroupScale ga = kv4::group_scale(cur[u].vparam(0, n)), gb = kv4::group_scale(cur[u].vparam(1, n));
#pragma unroll
        for (int i = n * IPG; i < (n + 1) * IPG; ++i) {
          const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
          uint32_t va[4], vb[4];
          kv4::dequant_word(prmt(cur[u].v[0][i / 2], cur[u].v[1][i / 2], sel), ga, va);
          kv4::dequant_word(prmt(cur[u].v[2][i / 2], cur[u].v[3][i / 2], sel), gb, vb);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_16816(o[i][0][nt], va[0], va[1], vb[0], vb[1], pb[nt][0], pb[nt][1]);
            mma_16816(o[i][1][nt], va[2], va[3], vb[2], vb[3], pb[nt][0], pb[nt][1]);
          }
        }
      }
    }
  }

  // the warps' results to shared memory, joined per (head, value)
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float l = l_r[nt][k];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      const int h = nt * 8 + 2 * c + k;
      if (g == 0) s_m[warp][h] = m_r[nt][k], s_l[warp][h] = l;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            s_o[warp][h][32 * i + 8 * (g >> 1) + 2 * (2 * f + r) + (g & 1)] = o[i][f][nt][2 * r + k];
    }
  __syncthreads();
  for (int idx = tid; idx < p.G * D; idx += THREADS) {
    const int h = idx / D, d = idx % D;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) m = fmaxf(m, s_m[w][h]);
    const float mb = m == -INFINITY ? 0.f : m;
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float a = ex2(s_m[w][h] - mb);
      acc = fmaf(a, s_o[w][h][d], acc);
      l = fmaf(a, s_l[w][h], l);
    }
    const int64_t row = int64_t(b) * p.hq + int64_t(kvh) * p.G + h;
    if (p.nsplit == 1) {
      p.out[row * D + d] = __float2half_rn(valid > 0 ? acc / l : 0.f);
    } else {
      p.part_o[(row * p.nsplit + split) * D + d] = acc;
      if (d == 0) p.part_ml[row * p.nsplit + split] = make_float2(m, l);
    }
  }
}

// joins the splits of one (sequence, query head): one warp
template <int D>
__global__ void __launch_bounds__(32) decode_attn_q4_merge_kernel(const float* __restrict__ part_o,
                                                                  const float2* __restrict__ part_ml,
                                                                  __half* __restrict__ out, const int64_t* counts,
                                                                  int64_t count, int hq, int nsplit) {
  pdl_trigger();
  pdl_wait();
  constexpr int E = D / 32;
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  float m = -INFINITY;
  for (int s = lane; s < nsplit; s += 32) m = fmaxf(m, part_ml[row * nsplit + s].x);
  m = warp_max(m);
  const float mb = m == -INFINITY ? 0.f : m;
  float acc[E], l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  for (int s = 0; s < nsplit; ++s) {
    const float2 ml = part_ml[row * nsplit + s];
    const float a = ex2(ml.x - mb);
    l = fmaf(a, ml.y, l);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(a, part_o[(row * nsplit + s) * D + e * 32 + lane], acc[e]);
  }
  const bool some = kv4::count_of(counts, count, int(row / hq)) > 0;
#pragma unroll
  for (int e = 0; e < E; ++e) out[row * D + e * 32 + lane] = __float2half_rn(some ? acc[e] / l : 0.f);
}

// CTAs that split a KV head's slots: as many as keep every SM's three CTAs busy,
// as long as each warp has a step
inline int splits(int batch, int kv_heads, int valid) {
  const int pairs = batch * kv_heads;
  const int want = (device_sm_count() * 3 + pairs - 1) / pairs;
  const int most = (valid + STEP * WARPS - 1) / (STEP * WARPS);
  return std::max(1, std::min({want, most, MAX_SPLITS}));
}

inline size_t workspace_for(int batch, int q_heads, int head_dim, int nsplit) {
  return nsplit == 1 ? 0 : size_t(batch) * q_heads * nsplit * (size_t(head_dim) * sizeof(float) + sizeof(float2));
}

template <int D, int NG, int NT>
cudaError_t launch(const Params& p, int batch, cudaStream_t st) {
  return launch_pdl(decode_attn_q4_kernel<D, NG, NT>, dim3(unsigned(p.nsplit), unsigned(p.hkv), unsigned(batch)),
                    dim3(THREADS), 0, st, p);
}
template <int D, int NG>
cudaError_t launch(const Params& p, int batch, cudaStream_t st) {
  return p.G <= 8 ? launch<D, NG, 1>(p, batch, st) : launch<D, NG, 2>(p, batch, st);
}

}  // namespace dattn4
}  // namespace qx

using namespace qx;

extern "C" size_t qx_decode_attention_q4_workspace_size(int batch, int q_heads, int kv_heads, int head_dim, int sink,
                                                        int window) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128) ||
      sink < 0 || window < 1 || kv4::capacity(sink, window) >= (int64_t(1) << 30))
    return 0;
  return dattn4::workspace_for(batch, q_heads, head_dim, dattn4::splits(batch, kv_heads, sink + window));
}

extern "C" int qx_decode_attention_q4(const void* q, const void* k_codes, const void* k_params, const void* v_codes,
                                      const void* v_params, void* out, int batch, int q_heads, int kv_heads,
                                      int head_dim, int group, int sink, int window, int64_t count,
                                      const int64_t* counts, float softmax_scale, void* workspace,
                                      size_t workspace_bytes, qx_stream_t stream) {
  const int rc = kv4::check_ring("decode_attention_q4", batch, kv_heads, head_dim, group, sink, window);
  if (rc != QX_OK) return rc;
  QX_REQUIRE(q_heads > 0 && q_heads % kv_heads == 0 && q_heads / kv_heads <= 16,
             "decode_attention_q4: bad heads q=%d kv=%d (a group of 1 to 16)", q_heads, kv_heads);
  QX_REQUIRE(batch <= 65535 && kv_heads <= 65535, "decode_attention_q4: batch or heads too large");
  QX_REQUIRE(counts || count >= 0, "decode_attention_q4: negative count");
  if (batch == 0) return QX_OK;
  QX_REQUIRE(q && k_codes && k_params && v_codes && v_params && out, "decode_attention_q4: null pointer");
  QX_REQUIRE(aligned(q, 16) && aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(k_params, 16) &&
                 aligned(v_params, 16) && aligned(out, 16),
             "decode_attention_q4: tensors must be 16-byte aligned");
  // the split is chosen for what the ring can hold, whether the counts are known here or not: the
  // same ring always sums in the same order
  const int nsplit = dattn4::splits(batch, kv_heads, sink + window);
  const size_t need = dattn4::workspace_for(batch, q_heads, head_dim, nsplit);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(QX_ERR_WORKSPACE, "decode_attention_q4: workspace needs %zu bytes, 16-byte aligned", need);
  dattn4::Params p{};
  p.q = static_cast<const __half*>(q);
  p.kc = static_cast<const unsigned char*>(k_codes);
  p.kp = static_cast<const uint16_t*>(k_params);
  p.vc = static_cast<const unsigned char*>(v_codes);
  p.vp = static_cast<const uint16_t*>(v_params);
  p.out = static_cast<__half*>(out);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + int64_t(batch) * q_heads * nsplit * head_dim);
  p.counts = counts;
  p.count = count;
  p.cap = kv4::capacity(sink, window);
  p.hq = q_heads;
  p.hkv = kv_heads;
  p.G = q_heads / kv_heads;
  p.sink = sink;
  p.window = window;
  p.nsplit = nsplit;
  p.scale_log2 = (softmax_scale > 0.f ? softmax_scale : 1.0f / sqrtf(float(head_dim))) * 1.4426950408889634f;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (head_dim == 64)
    e = group == 32 ? dattn4::launch<64, 2>(p, batch, st) : dattn4::launch<64, 1>(p, batch, st);
  else
    e = group == 32   ? dattn4::launch<128, 4>(p, batch, st)
        : group == 64 ? dattn4::launch<128, 2>(p, batch, st)
                      : dattn4::launch<128, 1>(p, batch, st);
  QX_CUDA_TRY(e, "decode_attention_q4: launch");
  if (nsplit > 1) {
    const dim3 grid(unsigned(batch) * unsigned(q_heads));
    if (head_dim == 64)
      e = launch_pdl(dattn4::decode_attn_q4_merge_kernel<64>, grid, dim3(32), 0, st,
                     static_cast<const float*>(p.part_o), static_cast<const float2*>(p.part_ml), p.out, counts, count,
                     q_heads, nsplit);
    else
      e = launch_pdl(dattn4::decode_attn_q4_merge_kernel<128>, grid, dim3(32), 0, st,
                     static_cast<const float*>(p.part_o), static_cast<const float2*>(p.part_ml), p.out, counts, count,
                     q_heads, nsplit);
    QX_CUDA_TRY(e, "decode_attention_q4: merge launch");
  }
  return check_launch("decode_attention_q4");
}
