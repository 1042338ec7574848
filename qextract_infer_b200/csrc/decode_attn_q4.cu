// Decode attention over the 4-bit ring KV cache (format: kv4.cuh): one query
// token per sequence, grouped-query heads, every valid slot.
//   out[h] = sum_t softmax_t(scale q[h] . K[t]) V[t],  K, V = s (c - z)
// New component (the reference has no attention kernel; semantics: HF Qwen3
// eager attention over the cache's valid slots, whose order does not matter).
//
// Both products run on the tensor cores with the cache as the A operand
// (mma.sync m16n8k16: 16 tokens or 16 head dimensions by 8 query heads), so a
// KV head's group of up to 8 query heads fills the N side (two N tiles up to
// 16).  tcgen05 takes 128 rows of M: for V^T P^T those are head dimensions, so the
// cache's rows would have to be turned over in shared memory as fp16, four times their
// bytes.  For K Q^T they are tokens, and A could come from TMEM, a token a lane: not built.
// The codes enter as fp16 subnormals: a mask of a 32-bit word is the pair c 2^-24
// (or 16 c 2^-24), exact, one instruction a pair.
//   S^T = K Q^T   sum q c per group; then s (sum q c - z sum q) per token in fp32.  The
//                 q of the codes that come as 16 c are divided by 16.
//   O^T = V^T P^T the token sits on the K side, so the scale goes to the weight:
//                 P s in fp16 per group.  The codes come as c - 8 (one more instruction
//                 a pair, exact), and sum P s (z - 8) is taken off in fp32: with c and z
//                 the two sums of a long context are far larger than their difference
//                 (131072 slots: relative error 5.9e-4 instead of 2.8e-4; it costs 1.9
//                 of 39.5 us for 32 sequences x 4096 slots).  P^T comes from S^T's
//                 accumulator layout by movmatrix.
// The online softmax keeps a running reference and sum per warp and head in fp32.
// The reference is the largest score, to 2^4, plus the exponent of the largest value
// scale so far, and P carries 2^10: P s stays below 2^15 and its fp16 subnormals
// start below 2^-24 of the largest.
//
// What bounds it: where the work fills the GPU (32 sequences x 4096 slots: 37.0 us, 3.9
// TB/s; one of 131072: 41.2 us), neither HBM nor a pipe is full: issue 59 %, the integer
// pipe 50 %, the tensor pipe 24 %, DRAM 45 %.  A scheduler has two warps, each a chain of
// masks, products and exponentials, and they do not cover each other's latencies (of an
// issue 0.67 waits for a fixed latency, 0.31 for a pipe).  So the next step's scores are computed next to
// this step's weights and values (45 -> 44 us for 131072 slots), the zero points' terms
// run on the FMA pipe (one more product each for them: 40 instead of 37.6 us, both with
// c unshifted), and V is not made exact fp16 (three instructions a pair: 46 us).  For one
// sequence of 4096 slots the launch, the first loads and the join are most of the time
// (7.5 us).
//
// Each warp streams its steps of 32 tokens through a ring of its own in shared
// memory (STAGES deep, cp.async) and reads the fragments from there; the format puts
// each lane's share of a row side by side.  (Loaded from global memory straight into
// the fragments, one step ahead, the bytes in flight hung on the registers: 84 us for
// one sequence of 131072 slots.  Four bulk copies a step onto an mbarrier were no
// faster, 46.8 against 45.5 us for 32 sequences x 4096 slots, and have waits to bound.)
//
// The work is cut into units of 128 tokens of one (sequence, KV head), and the CTAs,
// as many as are resident at once, take equal runs of units in order, whatever pair
// they belong to (a grid of (split, KV head, sequence) at its best split: 41 against
// 39.9 us for 32 sequences x 4096 slots, 58 against 48 for one of 131072).  The warps of
// a CTA take a unit's four steps and join their results of a pair in shared memory; a
// pair that one CTA did whole is finished there, the others' fp32 results are joined
// by a second kernel (the results of CTA i for pair j are number i + j: in the order
// of the runs each next one has a larger i or a larger j).
// Where a cluster of at most 16 CTAs a pair leaves each CTA at most FEW units, the
// clusters do the pairs instead and join through distributed shared memory: no second
// kernel, no scratch and no look at the other sequences' counts (one sequence of 4096
// slots 7.2 against 8.3 us as runs, seven of up to 1005 and 5 heads 5.7 against 8.1).
//
// Row g of an MMA is token g ^ (g / 2 & 1) of its eight: neighbouring rows, and the
// rows that four quads read together, then lie in different halves of the banks.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "kv4.cuh"
#include "qx_b200.h"

namespace qx {
namespace dattn4 {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int STEP = 32;          // tokens per warp step
constexpr float GROW = 4.f;       // log2 growth of the largest score that the reference follows
constexpr float PSHIFT = 14.f - GROW;  // what P carries: P s stays below 2^15
constexpr int UNIT = WARPS * STEP;  // tokens
constexpr int STAGES = 3;
constexpr int MAX_CLUSTER = 16;
constexpr int FEW = 4;            // units of a CTA up to which a pair is a cluster's

// bytes of a stage: codes of K and V, params of K and V
template <int D, int NG>
struct Stage {
  static constexpr int CODES = STEP * D / 2, PARAMS = STEP * NG * 2, BYTES = 2 * (CODES + PARAMS);
};
// shared memory: the ring of every warp, then the warps' results
template <int D, int NG, int NT>
struct Smem {
  static constexpr int RING = WARPS * STAGES * Stage<D, NG>::BYTES;
  static constexpr int BYTES = RING + WARPS * 8 * NT * (D + 1 + 2) * 4;
};

struct Params {
  const __half* q;
  const unsigned char* kc;
  const uint16_t* kp;
  const unsigned char* vc;
  const uint16_t* vp;
  __half* out;
  float* part_o;    // [piece][G][D]
  float2* part_ml;  // [piece][G]
  const int64_t* counts;
  int64_t count, cap;
  int batch, hq, hkv, G, sink, window;
  int ctas;     // of the first kernel
  int cluster;  // CTAs of a pair, where a cluster does it; 0: the CTAs take runs of units
  float scale_log2;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ int valid_of(const Params& p, int b) {
  return kv4::valid_slots(kv4::count_of(p.counts, p.count, b), p.sink, p.window);
}
__device__ __forceinline__ int units_of(const Params& p, int b) { return (valid_of(p, b) + UNIT - 1) / UNIT; }
// first unit of CTA i
__device__ __forceinline__ int first_unit(int total, int i, int ctas) {
  return ctas > 0 ? int(int64_t(total) * i / ctas) : 0;
}
// the CTA that has unit u: the last one whose first unit is at most u
__device__ __forceinline__ int cta_of(int u, int total, int ctas) { return int((int64_t(u + 1) * ctas - 1) / total); }

// With a count for each sequence: how the units of all KV heads lie, found by a whole
// block of T threads from the counts.  total: all of them; b, first: the sequence that
// unit `u(total)` lies in and its first unit, or of sequence `want` where that is not
// negative.  Up to T sequences take one pass over the counts.
template <int T, class U>
__device__ void place(const Params& p, int want, U u, int& total, int& b, int& first) {
  __shared__ int s_warp[T / 32], s_b, s_first;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int head = tid < p.batch ? units_of(p, tid) * p.hkv : 0;  // of the first T sequences
  int rest = 0;
  for (int i = T + tid; i < p.batch; i += T) rest += units_of(p, i) * p.hkv;
  total = 0;
  if (p.batch > T) {
    rest = __reduce_add_sync(0xffffffffu, rest);
    if (lane == 0) s_warp[warp] = rest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 32; ++w) total += s_warp[w];
    __syncthreads();
  }
  int at = 0;
  for (int b0 = 0, before = 0;; b0 += T) {
    const int mine = b0 == 0 ? head : b0 + tid < p.batch ? units_of(p, b0 + tid) * p.hkv : 0;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    if (lane == 31) s_warp[warp] = upto;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int w = 0; w < T / 32; ++w) {
      if (w < warp) upto += s_warp[w];
      all += s_warp[w];
    }
    if (b0 == 0) {
      total += all;
      at = u(total);
    }
    upto += before;
    const bool here = want >= 0 ? b0 + tid == want : upto - mine <= at && at < upto;
    if (here) s_b = b0 + tid, s_first = upto - mine;
    before += all;
    __syncthreads();
    if ((want >= 0 ? want < b0 + T : at < before) || b0 + T >= p.batch) break;
  }
  b = s_b;
  first = s_first;
}

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
__device__ __forceinline__ void load_words(const unsigned char* p, uint32_t (&w)[WORDS]) {  // shared memory
  if constexpr (WORDS == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (WORDS == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// the params of one token: NG 16-bit words
template <int NG>
struct RowParams {
  static constexpr int W = NG > 2 ? 2 : 1;
  uint32_t w[W];
  __device__ __forceinline__ void load(const unsigned char* p) {
    if constexpr (NG == 1)
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    else
      load_words<W>(p, w);
  }
};
// a row's zero points less OFF, as fp16 (exactly)
template <int NG, int OFF>
__device__ __forceinline__ void zeros_of(const RowParams<NG>& p, uint32_t (&z)[RowParams<NG>::W]) {
#pragma unroll
  for (int i = 0; i < RowParams<NG>::W; ++i)
    z[i] = hsub2_u32(lop3_and_or(p.w[i], 0x000F000Fu, 0x64006400u), 0x64006400u + OFF * 0x10001u);
}
// a pair of codes less 8, as fp16 times 2^-24, from the low and from the high four bits of its bytes
__device__ __forceinline__ uint32_t mid(uint32_t w) { return hsub2_u32(w & 0x000F000Fu, 0x00080008u); }
__device__ __forceinline__ uint32_t mid16(uint32_t w) { return hsub2_u32(w & 0x00F000F0u, 0x00800080u); }

// one of them, and the scale, of group `grp`
template <int NG>
__device__ __forceinline__ float zero_of(const uint32_t (&z)[RowParams<NG>::W], int grp) {
  const float2 f = h2_to_f2(z[NG == 1 ? 0 : grp >> 1]);
  return NG > 1 && (grp & 1) ? f.y : f.x;
}
template <int NG>
__device__ __forceinline__ float scale_of(const RowParams<NG>& p, int grp) {
  const uint32_t w = NG == 1 ? p.w[0] : (grp & 1) ? p.w[grp >> 1] >> 16 : p.w[grp >> 1];
  return __half2float(__ushort_as_half(uint16_t(w & 0xFFF0u)));
}

// What the registers allow: at D = 128 two CTAs of up to 255 registers a thread are faster than three of 168 (32
// sequences x 4096 slots 37.6 against 40.0 us, one of 131072 42.3 against 46.1, measured with codes unshifted).
constexpr int ctas_per_sm(int head_dim, int n_tiles) { return head_dim == 64 && n_tiles == 1 ? 3 : 2; }

template <int D, int NG, int NT>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(D, NT)) decode_attn_q4_kernel(const __grid_constant__ Params p) {
  pdl_trigger();
  constexpr int NI = D / 32, IPG = NI / NG;  // 32-value blocks of a row, and of a group
  constexpr int SROW = D + 1;                // odd: the column writes below meet no bank twice
  using St = Stage<D, NG>;
  using Sm = Smem<D, NG, NT>;
  extern __shared__ __align__(128) unsigned char smem[];
  float (*s_o)[8 * NT][SROW] = reinterpret_cast<float (*)[8 * NT][SROW]>(smem + Sm::RING);
  float (*s_m)[8 * NT] = reinterpret_cast<float (*)[8 * NT]>(s_o + WARPS);
  float (*s_l)[8 * NT] = s_m + WARPS;
  // a cluster's CTA keeps its result for the others where its rings were
  float* c_o = reinterpret_cast<float*>(smem);
  float2* c_ml = reinterpret_cast<float2*>(c_o + 8 * NT * D);
  static_assert(8 * NT * (D + 2) * 4 <= Sm::RING, "the result fits the rings");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const unsigned char* ring = smem + warp * STAGES * St::BYTES;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  pdl_wait();
  // this CTA's units [u, u_end), and the sequence and its first unit that u lies in
  int b, first, units = 0, u, u_end;
  if (p.cluster) {
    const int pair = blockIdx.x / p.cluster, rank = blockIdx.x - pair * p.cluster;
    b = pair / p.hkv;
    first = 0;
    units = units_of(p, b);
    const int at = (pair - b * p.hkv) * units;
    u = at + units * rank / p.cluster;
    u_end = at + units * (rank + 1) / p.cluster;
  } else {
    int total;
    if (p.counts) {
      place<THREADS>(p, -1, [&](int all) { return first_unit(all, min(int(blockIdx.x), min(p.ctas, all) - 1), min(p.ctas, all)); },
                     total, b, first);
    } else {
      units = units_of(p, 0);
      total = units * p.hkv * p.batch;
    }
    const int n = min(p.ctas, total);  // CTAs with work: none of them has an empty run
    if (int(blockIdx.x) >= n) return;
    u = first_unit(total, blockIdx.x, n);
    u_end = first_unit(total, blockIdx.x + 1, n);
    if (p.counts) {
      units = units_of(p, b);
    } else {
      b = u / (units * p.hkv);
      first = b * units * p.hkv;
    }
  }

  // a step's rows to stage st, 16 bytes a lane and copy; they all lie in the storage: it has a multiple of 64
  auto fetch = [&](int st, int64_t row) {
    const uint32_t dst = ring_at + st * St::BYTES + lane * 16;
    const unsigned char *kc = p.kc + row * (D / 2) + lane * 16, *vc = p.vc + row * (D / 2) + lane * 16;
#pragma unroll
    for (int i = 0; i < St::CODES / 512; ++i) {
      copy16(dst + i * 512, kc + i * 512);
      copy16(dst + St::CODES + i * 512, vc + i * 512);
    }
    const int l = lane & 15;  // params: K's by the first half of the warp, V's by the second
    if (l < St::PARAMS / 16)
      copy16(ring_at + st * St::BYTES + 2 * St::CODES + (lane >> 4) * St::PARAMS + l * 16,
             reinterpret_cast<const unsigned char*>((lane >> 4 ? p.vp : p.kp) + row * NG) + l * 16);
  };
  // this lane's places in a stage: MMA row g is token tg of its eight
  const int tg = g ^ ((g >> 1) & 1), odd = c & 1;
  const int at_k = tg * (D / 2) + c * (D / 8), at_p = 2 * St::CODES + tg * NG * 2;
  const int at_v[2] = {St::CODES + (2 * c + odd) * (D / 2) + g * (D / 16), St::CODES + (2 * c + 1 - odd) * (D / 2) + g * (D / 16)};

  // a pair (sequence b, KV head kvh), or the part of it that is this CTA's: units off .. off + len
  int kvh, off, len, valid, steps, step;
  int64_t row0;
  uint4 q_raw[NT][NI];
  auto begin = [&] {
    kvh = p.cluster ? blockIdx.x / p.cluster - b * p.hkv : (u - first) / units;  // (a cluster's CTA may have no unit)
    off = u - first - kvh * units;
    len = min(units - off, u_end - u);
    valid = valid_of(p, b);
    steps = min((valid + STEP - 1) / STEP, (off + len) * WARPS);
    row0 = (int64_t(b) * p.hkv + kvh) * p.cap;
    step = off * WARPS + warp;
    // the queries first: the first scores wait for them
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < NI; ++i)
        q_raw[nt][i] = nt * 8 + g < p.G
                           ? __ldg(reinterpret_cast<const uint4*>(
                                 p.q + ((int64_t(b) * p.hq + int64_t(kvh) * p.G + nt * 8 + g) * D + 32 * i + 8 * c)))
                           : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < STAGES; ++i) {
      if (step + i * WARPS < steps) fetch(i, row0 + int64_t(step + i * WARPS) * STEP);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  begin();
  while (true) {
  // Q^T fragments: head g (of N tile nt), values 32 i + 8 c ..; a head is scaled by
  // the power of two that brings its largest value to [2^4, 2^5), undone in hf: the
  // second pair of each k step is divided by 16, which then costs no bits that count,
  // and the sum over a group stays within fp16.
  uint32_t qb[NT][NI][4];
  float qz[NT][NG][2];  // minus 2^-24 the sum of the scaled q over a group, of heads 2c, 2c + 1
  float hf[NT][2];      // accumulator -> log2 domain, of heads 2c, 2c + 1
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float top = 0.f, sum[NG];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const uint32_t d[4] = {q_raw[nt][i].x, q_raw[nt][i].y, q_raw[nt][i].z, q_raw[nt][i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = h2_to_f2(d[e]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = top > 0.f && top <= 65504.f ? int(__float_as_uint(top) >> 23) - 127 : 4;
    const float up = __uint_as_float(uint32_t(127 + 4 - ex) << 23), down = __uint_as_float(uint32_t(127 + ex - 4) << 23);
#pragma unroll
    for (int n = 0; n < NG; ++n) sum[n] = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const uint32_t d[4] = {q_raw[nt][i].x, q_raw[nt][i].y, q_raw[nt][i].z, q_raw[nt][i].w};
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
      qz[nt][n][0] = __shfl_sync(0xffffffffu, sum[n], 8 * c) * -0x1p-24f;
      qz[nt][n][1] = __shfl_sync(0xffffffffu, sum[n], 8 * c + 4) * -0x1p-24f;
    }
    const float k = down * 0x1p24f * p.scale_log2;
    hf[nt][0] = __shfl_sync(0xffffffffu, k, 8 * c);
    hf[nt][1] = __shfl_sync(0xffffffffu, k, 8 * c + 4);
  }

  float o[NI][2][NT][4], oz[NG][NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int f = 0; f < 2; ++f) o[i][f][nt][0] = o[i][f][nt][1] = o[i][f][nt][2] = o[i][f][nt][3] = 0.f;
#pragma unroll
    for (int n = 0; n < NG; ++n) oz[n][nt][0] = oz[n][nt][1] = 0.f;
  }
  // m_r: the score and vexp: the exponent (of its bits, biased) of the value scale that the
  // weights refer to
  float m_r[NT][2], l_r[NT][2], shift[NT][2];
  int vexp = 0;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) m_r[nt][0] = m_r[nt][1] = -INFINITY, l_r[nt][0] = l_r[nt][1] = shift[nt][0] = shift[nt][1] = 0.f;
  // scores of a stage's step, over hf: rows g, g + 8 (e >> 1) by heads 2c, 2c + 1 (e & 1)
  auto scores = [&](const unsigned char* at, float (&s)[2][NT][4]) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t kc[2][NI];
      RowParams<NG> kp[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        load_words<NI>(at + at_k + (u * 16 + 8 * r) * (D / 2), kc[r]);
        kp[r].load(at + at_p + (u * 16 + 8 * r) * NG * 2);
      }
      uint32_t kz[2][RowParams<NG>::W];
#pragma unroll
      for (int r = 0; r < 2; ++r) zeros_of<NG, 0>(kp[r], kz[r]);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        float acc[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) acc[nt][0] = acc[nt][1] = acc[nt][2] = acc[nt][3] = 0.f;
#pragma unroll
        for (int i = n * IPG; i < (n + 1) * IPG; ++i) {
          const uint32_t w0 = kc[0][i], w1 = kc[1][i], h0 = w0 >> 8, h1 = w1 >> 8;
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
          const float sc = scale_of<NG>(kp[r], n), z = zero_of<NG>(kz[r], n);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 2; ++k)
            {
              const float a = fmaf(z, qz[nt][n][k], acc[nt][2 * r + k]);
              s[u][nt][2 * r + k] = n == 0 ? sc * a : fmaf(sc, a, s[u][nt][2 * r + k]);
            }
        }
      }
    }
  };
  float s[2][NT][4];
  asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
  __syncwarp();
  scores(ring, s);
  for (int st = 0, next = 1; step < steps; step += WARPS, st = next, next = next + 1 == STAGES ? 0 : next + 1) {
    const int left = valid - step * STEP;  // tokens of this step that exist
    const unsigned char* at = ring + st * St::BYTES;
    // the value scales of tokens g, g + 8, and the exponent of the largest
    float vs[2][2][NG];
    uint32_t vz[2][2][RowParams<NG>::W];
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        RowParams<NG> vp;
        vp.load(at + at_p + St::PARAMS + (u * 16 + 8 * r) * NG * 2);
        // a slot past the valid ones may hold anything: scale 0, for P is 0 there, and 0 times a NaN would not be
        if (left < STEP && u * 16 + tg + 8 * r >= left) vp = RowParams<NG>{};
#pragma unroll
        for (int n = 0; n < NG; ++n) vs[u][r][n] = scale_of<NG>(vp, n);
        zeros_of<NG, 8>(vp, vz[u][r]);
#pragma unroll
        for (int w = 0; w < RowParams<NG>::W; ++w) top = __vmaxu2(top, vp.w[w]);
      }
    if (left < STEP) {
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (u * 16 + tg + 8 * (e >> 1) >= left) s[u][nt][e] = -INFINITY;
    }
    // The reference (a score, m_r, and the exponent of the largest value scale, vexp) follows
    // only where a score passes m_r by 2^GROW or a scale passes vexp; m_r starts at minus infinity.
    float mx[NT][2];
    bool grew = (max(top >> 16, top & 0xFFFFu) >> 10) > uint32_t(vexp);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        mx[nt][k] = fmaxf(fmaxf(s[0][nt][k], s[0][nt][2 + k]), fmaxf(s[1][nt][k], s[1][nt][2 + k])) * hf[nt][k];
        grew = grew || mx[nt][k] > m_r[nt][k] + GROW;
      }
    if (__any_sync(0xffffffffu, grew)) {
      // (of the finite scales: a NaN's exponent would cost the other groups' weights their bits)
      float largest = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
          for (int n = 0; n < NG; ++n) largest = fmaxf(largest, vs[u][r][n]);
      const int e_new = max(vexp, int(__reduce_max_sync(0xffffffffu, __float_as_uint(largest)) >> 23) - 112);
      const float e_shift = float(e_new - vexp);
      vexp = e_new;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float alpha[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float m = mx[nt][k];
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          m = fmaxf(m, m_r[nt][k]);
          const float mb = m == -INFINITY ? 0.f : m;
          alpha[k] = ex2(m_r[nt][k] - mb - e_shift);
          m_r[nt][k] = m;
          l_r[nt][k] *= alpha[k];
          shift[nt][k] = PSHIFT + 14.f - float(vexp) - mb;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
          for (int i = 0; i < NI; ++i) {
            o[i][0][nt][e] *= alpha[e & 1];
            o[i][1][nt][e] *= alpha[e & 1];
          }
#pragma unroll
          for (int n = 0; n < NG; ++n)
            if (e < 2) oz[n][nt][e] *= alpha[e];
        }
      }
    }
    // the next step's scores, next to this step's weights and values (past the last step: of whatever the stage
    // holds, and not used)
    float s_next[2][NT][4];
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncwarp();
    scores(ring + next * St::BYTES, s_next);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            s[u][nt][2 * r + k] = ex2(fmaf(s[u][nt][2 * r + k], hf[nt][k], shift[nt][k]));
            l_r[nt][k] += s[u][nt][2 * r + k];
          }
    // O^T += V^T (P s)^T
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      uint32_t vc[4][NI / 2];
#pragma unroll
      for (int t = 0; t < 4; ++t) load_words<NI / 2>(at + at_v[t & 1] + (u * 16 + (t >> 1) * 8) * (D / 2), vc[t]);
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint32_t ps = pack_h2(s[u][nt][2 * r] * vs[u][r][n], s[u][nt][2 * r + 1] * vs[u][r][n]);
            const float2 f = h2_to_f2(ps);  // the rounded weights, so that c and z meet the same ones
            const float z = zero_of<NG>(vz[u][r], n);
            oz[n][nt][0] = fmaf(f.x, z, oz[n][nt][0]);
            oz[n][nt][1] = fmaf(f.y, z, oz[n][nt][1]);
            pb[nt][r] = transpose8x8(ps);
          }
#pragma unroll
        for (int i = n * IPG; i < (n + 1) * IPG; ++i) {
          const uint32_t sel = (i & 1) ? 0x7632u : 0x5410u;
          const uint32_t a = prmt(vc[0][i / 2], vc[1][i / 2], sel), ah = a >> 8;
          const uint32_t d = prmt(vc[2][i / 2], vc[3][i / 2], sel), dh = d >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {  // rows g: (c - 8) 2^-24, rows g + 8: 16 (c - 8) 2^-24
            mma_16816(o[i][0][nt], mid(a), mid16(a), mid(d), mid16(d), pb[nt][0], pb[nt][1]);
            mma_16816(o[i][1][nt], mid(ah), mid16(ah), mid(dh), mid16(dh), pb[nt][0], pb[nt][1]);
          }
        }
      }
    }
    __syncwarp();  // every lane has read the stage
    if (step + STAGES * WARPS < steps) fetch(st, row0 + int64_t(step + STAGES * WARPS) * STEP);
    asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][nt][e] = s_next[u][nt][e];
  }

  // the next pair's loads start before this one's results are joined
  const bool whole = len == units, more = u + len < u_end;
  const int64_t row = int64_t(b) * p.hq + int64_t(kvh) * p.G;                             // of the result
  const int64_t piece = (int64_t(blockIdx.x) + int64_t(b) * p.hkv + kvh) * p.G;  // of the partial results
  u += len;
  if (more) {
    if (off + len == units && kvh == p.hkv - 1) {  // the next sequence with tokens
      first += units * p.hkv;
      do units = units_of(p, ++b);
      while (units == 0);
    }
    begin();
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
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        oz[n][nt][k] += __shfl_xor_sync(0xffffffffu, oz[n][nt][k], 4);
        oz[n][nt][k] += __shfl_xor_sync(0xffffffffu, oz[n][nt][k], 8);
        oz[n][nt][k] += __shfl_xor_sync(0xffffffffu, oz[n][nt][k], 16);
      }
      if (g == 0) s_m[warp][h] = m_r[nt][k] + float(vexp), s_l[warp][h] = l;
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            s_o[warp][h][32 * i + 8 * (g >> 1) + 2 * (2 * f + r) + (g & 1)] =
                fmaf(o[i][f][nt][2 * r + k], r ? 0x1p20f : 0x1p24f, -oz[i / IPG][nt][k]);
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
    if (p.cluster > 1) {
      c_o[idx] = acc;
      if (d == 0) c_ml[h] = make_float2(m, l);
    } else if (whole) {
      p.out[(row + h) * D + d] = __float2half_rn(units > 0 ? acc / l : 0.f);
    } else {
      p.part_o[(piece + h) * D + d] = acc;
      if (d == 0) p.part_ml[piece + h] = make_float2(m, l);
    }
  }
  if (!more) break;
  __syncthreads();  // read: the next results may come
  }
  if (p.cluster > 1) {
    // every CTA of the pair joins its share of the (head, value)s, in rank order
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int pair = blockIdx.x / p.cluster, rank = blockIdx.x - pair * p.cluster;
    for (int idx = rank * THREADS + tid; idx < p.G * D; idx += p.cluster * THREADS) {
      const uint32_t at_o = static_cast<uint32_t>(__cvta_generic_to_shared(c_o + idx));
      const uint32_t at_m = static_cast<uint32_t>(__cvta_generic_to_shared(c_ml + idx / D));
      float x[MAX_CLUSTER], m[MAX_CLUSTER], l[MAX_CLUSTER], top = -INFINITY;
#pragma unroll
      for (int r = 0; r < MAX_CLUSTER; ++r) {
        m[r] = -INFINITY, l[r] = x[r] = 0.f;
        if (r >= p.cluster) continue;
        uint32_t a, b2;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(at_o), "r"(r));
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b2) : "r"(at_m), "r"(r));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[r]) : "r"(a) : "memory");
        asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(m[r]), "=f"(l[r]) : "r"(b2) : "memory");
      }
#pragma unroll
      for (int r = 0; r < MAX_CLUSTER; ++r) top = fmaxf(top, m[r]);
      const float mb = top == -INFINITY ? 0.f : top;
      float acc = 0.f, sum = 0.f;
#pragma unroll
      for (int r = 0; r < MAX_CLUSTER; ++r) {
        const float w = ex2(m[r] - mb);
        acc = fmaf(w, x[r], acc);
        sum = fmaf(w, l[r], sum);
      }
      p.out[(int64_t(b) * p.hq + int64_t(pair - b * p.hkv) * p.G) * D + idx] = __float2half_rn(units > 0 ? acc / sum : 0.f);
    }
    // (and none leaves while another reads it)
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// Joins the pieces of one (sequence, query head): four values a thread, T / (D / 4)
// parts that take the pieces in turn; zeros where a sequence has no token.  With the
// count known on the host, which pieces those are is found before the first kernel
// ends.  (One value a thread, the pieces looked up after it: 39.3 against 37.2 us for 32
// sequences x 4096 slots, 43.4 against 41.5 for one of 131072, of which the join is now 1.8.)
template <int D, int T>
__global__ void __launch_bounds__(T) decode_attn_q4_merge_kernel(const __grid_constant__ Params p) {
  constexpr int LANES = D / 4, PARTS = T / LANES;
  pdl_trigger();
  __shared__ float4 s_acc[PARTS][LANES];
  __shared__ float2 s_ml[PARTS];
  const int b = blockIdx.x / p.hq, h = blockIdx.x - b * p.hq, kvh = h / p.G;
  const int lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
  int units, first = 0, total = 0, i0 = 0, i1 = 0;
  auto pieces = [&] {  // the CTAs of the first and of the last unit
    const int n = min(p.ctas, total);
    i0 = cta_of(first + kvh * units, total, n);
    i1 = cta_of(first + kvh * units + units - 1, total, n);
  };
  if (p.counts) {
    pdl_wait();
    units = units_of(p, b);
    if (units > 0) {
      int at = b;
      place<T>(p, b, [](int) { return 0; }, total, at, first);
      pieces();
    }
  } else {
    units = units_of(p, b);
    total = units * p.hkv * p.batch;
    first = b * units * p.hkv;
    if (units > 0) pieces();
    pdl_wait();
  }
  uint2* out = reinterpret_cast<uint2*>(p.out + (int64_t(b) * p.hq + h) * D) + lane;
  if (units == 0) {
    if (part == 0) *out = make_uint2(0u, 0u);
    return;
  }
  if (i0 == i1) return;  // one CTA's: finished there
  const int64_t base = (int64_t(b) * p.hkv + kvh) * p.G + (h - kvh * p.G);  // piece i at base + i G
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 0.f;
  auto add = [&](float2 ml, float4 v) {
    const float top = fmaxf(m, ml.x), mb = top == -INFINITY ? 0.f : top;
    const float a = ex2(m - mb), c = ex2(ml.x - mb);
    m = top;
    l = fmaf(l, a, c * ml.y);
    acc.x = fmaf(acc.x, a, c * v.x);
    acc.y = fmaf(acc.y, a, c * v.y);
    acc.z = fmaf(acc.z, a, c * v.z);
    acc.w = fmaf(acc.w, a, c * v.w);
  };
  constexpr int AHEAD = 4;  // pieces whose loads are in flight together
  for (int i = i0 + part; i <= i1; i += PARTS * AHEAD) {
    float2 ml[AHEAD];
    float4 v[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int64_t at = base + int64_t(min(i + k * PARTS, i1)) * p.G;
      ml[k] = p.part_ml[at];
      v[k] = reinterpret_cast<const float4*>(p.part_o + at * D)[lane];
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (i + k * PARTS <= i1) add(ml[k], v[k]);
  }
  if constexpr (PARTS > 1) {
    s_acc[part][lane] = acc;
    if (lane == 0) s_ml[part] = make_float2(m, l);
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int k = 1; k < PARTS; ++k) add(s_ml[k], s_acc[k][lane]);
  }
  const float inv = 1.f / l;
  *out = make_uint2(pack_h2(acc.x * inv, acc.y * inv), pack_h2(acc.z * inv, acc.w * inv));
}

// CTAs of the first kernel: those resident at once, or one a unit of what the ring
// can hold.  Not of what it holds, so that a call sums in the same order whether
// its counts are known on the host or not.
inline int64_t units_most(int batch, int kv_heads, int sink, int window) {
  return (kv4::capacity(sink, window) + UNIT - 1) / UNIT * batch * kv_heads;
}
inline int ctas(int batch, int q_heads, int kv_heads, int head_dim, int sink, int window) {
  const int most = device_sm_count() * ctas_per_sm(head_dim, q_heads / kv_heads > 8 ? 2 : 1);
  return int(std::min<int64_t>(most, units_most(batch, kv_heads, sink, window)));
}
// CTAs of a pair where clusters do the pairs, else 0: a power of two, as many as are
// resident at once for all pairs and have a unit each
inline int cluster_of(int batch, int q_heads, int kv_heads, int head_dim, int sink, int window) {
  const int64_t units = (kv4::capacity(sink, window) + UNIT - 1) / UNIT, pairs = int64_t(batch) * kv_heads;
  const int most = device_sm_count() * ctas_per_sm(head_dim, q_heads / kv_heads > 8 ? 2 : 1);
  int c = 1;
  while (c < MAX_CLUSTER && c < units && pairs * (2 * c) <= most) c *= 2;
  return (units + c - 1) / c <= FEW && pairs * c < (int64_t(1) << 31) ? c : 0;
}
inline size_t workspace_for(int batch, int q_heads, int kv_heads, int head_dim, int n, int cluster) {
  if (cluster) return 0;
  return (size_t(n) + size_t(batch) * kv_heads) * (q_heads / kv_heads) * (size_t(head_dim) * sizeof(float) + sizeof(float2));
}

template <int D, int NG, int NT>
cudaError_t launch(const Params& p, cudaStream_t st) {
  {
    static std::mutex mu;
    static bool done[64] = {};
    int dev = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
    std::lock_guard<std::mutex> lk(mu);
    if (!done[dev]) {
      const cudaError_t a = cudaFuncSetAttribute(decode_attn_q4_kernel<D, NG, NT>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, Smem<D, NG, NT>::BYTES);
      if (a != cudaSuccess) return a;
      const cudaError_t c = cudaFuncSetAttribute(decode_attn_q4_kernel<D, NG, NT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      if (c != cudaSuccess) return c;
      done[dev] = true;
    }
  }
  if (p.cluster) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(p.batch) * unsigned(p.hkv) * unsigned(p.cluster));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = Smem<D, NG, NT>::BYTES;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(p.cluster);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = g_pdl_enabled.load(std::memory_order_relaxed) ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, decode_attn_q4_kernel<D, NG, NT>, p);
  }
  const cudaError_t e = launch_pdl(decode_attn_q4_kernel<D, NG, NT>, dim3(unsigned(p.ctas)), dim3(THREADS),
                                   Smem<D, NG, NT>::BYTES, st, p);
  // where the runs end with pairs, known here without per-sequence counts, every pair is one CTA's
  if (e != cudaSuccess || (!p.counts && p.count > 0 && p.batch * p.hkv % p.ctas == 0)) return e;
  const dim3 grid(unsigned(p.batch) * unsigned(p.hq));
  // many pieces a pair (one sequence: 32 and more) are shared out to 16 warps; of a few, one warp does a head; past
  // 128 sequences four, which look through the counts
  if (p.ctas >= int64_t(8) * p.batch * p.hkv) return launch_pdl(decode_attn_q4_merge_kernel<D, 512>, grid, dim3(512), 0, st, p);
  if (p.batch > 128) return launch_pdl(decode_attn_q4_merge_kernel<D, 128>, grid, dim3(128), 0, st, p);
  return launch_pdl(decode_attn_q4_merge_kernel<D, 32>, grid, dim3(32), 0, st, p);
}
template <int D, int NG>
cudaError_t launch(const Params& p, cudaStream_t st) {
  return p.G <= 8 ? launch<D, NG, 1>(p, st) : launch<D, NG, 2>(p, st);
}

}  // namespace dattn4
}  // namespace qx

using namespace qx;

extern "C" size_t qx_decode_attention_q4_workspace_size(int batch, int q_heads, int kv_heads, int head_dim, int sink,
                                                        int window) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || (head_dim != 64 && head_dim != 128) ||
      sink < 0 || window < 1 || kv4::capacity(sink, window) >= (int64_t(1) << 30))
    return 0;
  return dattn4::workspace_for(batch, q_heads, kv_heads, head_dim,
                               dattn4::ctas(batch, q_heads, kv_heads, head_dim, sink, window),
                               dattn4::cluster_of(batch, q_heads, kv_heads, head_dim, sink, window));
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
  QX_REQUIRE(counts || kv4::count_fits(count), "decode_attention_q4: count=%lld", (long long)count);
  if (batch == 0) return QX_OK;
  QX_REQUIRE(q && k_codes && k_params && v_codes && v_params && out, "decode_attention_q4: null pointer");
  QX_REQUIRE(aligned(q, 16) && aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(k_params, 16) &&
                 aligned(v_params, 16) && aligned(out, 16),
             "decode_attention_q4: tensors must be 16-byte aligned");
  QX_REQUIRE(dattn4::units_most(batch, kv_heads, sink, window) < (int64_t(1) << 31) && int64_t(batch) * q_heads < (int64_t(1) << 31),
             "decode_attention_q4: batch x heads x slots too large");
  const int n = dattn4::ctas(batch, q_heads, kv_heads, head_dim, sink, window);
  const int cluster = dattn4::cluster_of(batch, q_heads, kv_heads, head_dim, sink, window);
  const size_t need = dattn4::workspace_for(batch, q_heads, kv_heads, head_dim, n, cluster);
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
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t(n) + int64_t(batch) * kv_heads) * (q_heads / kv_heads) * head_dim);
  p.counts = counts;
  p.count = count;
  p.cap = kv4::capacity(sink, window);
  p.hq = q_heads;
  p.hkv = kv_heads;
  p.G = q_heads / kv_heads;
  p.sink = sink;
  p.window = window;
  p.batch = batch;
  p.ctas = n;
  p.cluster = cluster;
  p.scale_log2 = (softmax_scale > 0.f ? softmax_scale : 1.0f / sqrtf(float(head_dim))) * 1.4426950408889634f;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (head_dim == 64)
    e = group == 32 ? dattn4::launch<64, 2>(p, st) : dattn4::launch<64, 1>(p, st);
  else
    e = group == 32   ? dattn4::launch<128, 4>(p, st)
        : group == 64 ? dattn4::launch<128, 2>(p, st)
                      : dattn4::launch<128, 1>(p, st);
  QX_CUDA_TRY(e, "decode_attention_q4: launch");
  return check_launch("decode_attention_q4");
}
