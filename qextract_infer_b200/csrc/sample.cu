// Sampling: one token for each row of fp16 logits from one given number u in [0, 1).
//
//   order    tokens stand by their logit, the largest first, equal ones by index
//   weight   w = exp((l - max l) / T), in 64 bits
//   kept     the first top_k; of these the shortest run from the front with at least
//            top_p of their weight; of these the ones with w >= min_p: always a run
//            from the front, n tokens with the weight M
//   drawn    the first token at which the running sum of the weights exceeds u M
//
// fp16 logits have 65536 values, so the order is one of values and not of tokens: a
// row becomes a histogram over the values in descending order (d, 0 the largest), and
// everything above is a question about prefix sums over it.  Weights are computed once
// for each value that occurs.  They are summed as integers, w 2^43 rounded: the sums do
// not depend on how they are split, a token's border is off by at most 2^-44 of the
// largest weight for each token before it, and 2^19 of them stay below 2^62.
//
// A cluster of C CTAs takes a row.  Each CTA counts a slice of it in its own histogram
// (16-bit counters, 128 KB of shared memory), then owns 1 / C of the values: it adds
// their counters of all CTAs through distributed shared memory, and the prefix sums run
// over threads, warps and CTAs.  Whoever owns the border in question (the k-th token,
// top_p of the weight, u of the weight) tells all CTAs.
#include <mutex>

#include "qx_b200.h"
#include "qx_common.cuh"

namespace qx {
namespace smp {

constexpr int THREADS = 1024, WARPS = THREADS / 32;
constexpr int VALUES = 65536;
constexpr int HIST_BYTES = VALUES * 2;
constexpr int SLICE_MAX = 65528;  // logits of a CTA: a 16-bit counter holds them all
constexpr int FRAC = 43;
constexpr unsigned NONE = ~0u;
typedef unsigned long long u64;

struct Params {
  const __half* logits;
  const float* u;
  const float *temperature, *top_p, *min_p;  // a row's own, or NULL: the call's
  const int64_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int64_t top_k_all;
  int64_t* tokens;
  float* logprobs;
  int vocab, slice;
};

template <int C>
struct Shared {
  u64 warp_mass[WARPS];
  unsigned warp_count[WARPS];
  // written by the cluster's CTAs
  unsigned top[C], count[C];
  u64 mass[C];
  u64 k_mass, p_mass, m_mass[C];
  unsigned p_n, m_n[C];
  unsigned pick, pick_nth;
  // this CTA's
  unsigned top_here, m_here, found;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t at_rank(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void tell(const unsigned* p, int rank, unsigned v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at_rank(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void tell(const u64* p, int rank, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at_rank(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_sync() {
  cluster_arrive();
  cluster_wait();
}

// the place of a logit's bits among all values, the largest first; NaN and -inf: NONE
__device__ __forceinline__ unsigned place_of(unsigned bits) {
  if (bits == 0x8000u) bits = 0u;  // the zeros are one value
  if ((bits & 0x7FFFu) > 0x7C00u || bits == 0xFC00u) return NONE;
  return (bits & 0x8000u) ? bits : 0x7FFFu - bits;
}
__device__ __forceinline__ double value_at(unsigned place) {
  const unsigned bits = (place & 0x8000u) ? place : 0x7FFFu - place;
  return double(__half2float(__ushort_as_half(static_cast<unsigned short>(bits))));
}

struct Weights {
  double top, temperature;
  unsigned place;
  bool top_is_inf;
  // logarithm of a value's weight
  __device__ __forceinline__ double log_of(unsigned d) const {
    if (d == place) return 0.0;
    return top_is_inf ? -INFINITY : (value_at(d) - top) / temperature;
  }
  __device__ __forceinline__ double of(unsigned d) const { return exp(log_of(d)); }
};
__device__ __forceinline__ u64 fixed(double w) { return u64(__double2ull_rn(w * double(u64(1) << FRAC))); }

template <int C>
__global__ void __launch_bounds__(THREADS, 1) sample_kernel(const Params p) {
  constexpr int OWN = VALUES / (C * THREADS);  // values of a thread
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned* const hist = reinterpret_cast<unsigned*>(smem);
  Shared<C>& s = *reinterpret_cast<Shared<C>*>(smem + HIST_BYTES);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / C, rank = blockIdx.x % C;
  pdl_trigger();

  for (int i = tid; i < HIST_BYTES / 16; i += THREADS) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0u, 0u, 0u, 0u);
  if (tid == 0) {
    s.pick = s.top_here = s.m_here = s.p_n = NONE;
    for (int r = 0; r < C; ++r) s.m_n[r] = NONE;
  }
  __syncthreads();
  cluster_arrive();
  pdl_wait();

  // ---- count the slice
  const unsigned short* const slice = reinterpret_cast<const unsigned short*>(p.logits) + int64_t(row) * p.vocab + int64_t(rank) * p.slice;
  const int len = max(0, min(p.slice, p.vocab - rank * p.slice));
  unsigned top = NONE;
  auto count = [&](unsigned bits) {
    const unsigned d = place_of(bits);
    if (d == NONE) return;
    atomicAdd(hist + (d >> 1), d & 1 ? 0x10000u : 1u);
    top = min(top, d);
  };
  const int head = min(len, int((16u - (uint32_t(reinterpret_cast<uintptr_t>(slice)) & 15u)) & 15u) >> 1);
  const int vectors = (len - head) >> 3;
  for (int i = tid; i < vectors; i += THREADS) {
    const uint4 v = __ldcg(reinterpret_cast<const uint4*>(slice + head) + i);
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      count(w[e] & 0xFFFFu);
      count(w[e] >> 16);
    }
  }
  const int rest = len - 8 * vectors;  // the ends that no aligned vector covers
  if (tid < rest) count(__ldcg(slice + (tid < head ? tid : tid + 8 * vectors)));
  top = __reduce_min_sync(0xffffffffu, top);
  if (lane == 0) atomicMin(&s.top_here, top);
  __syncthreads();
  cluster_wait();  // every CTA has started
  if (tid < C) tell(&s.top[rank], tid, s.top_here);
  cluster_sync();

  // ---- the counters of the values that this CTA owns, of all CTAs
  const unsigned first = unsigned(rank * THREADS + tid) * OWN;
  unsigned c[OWN];
#pragma unroll
  for (int i = 0; i < OWN; ++i) c[i] = 0;
#pragma unroll
  for (int r = 0; r < C; ++r) {
    const uint32_t at = at_rank(hist + first / 2, (rank + r) % C);
#pragma unroll
    for (int i = 0; i < OWN; i += 8) {
      uint32_t w[4];
      asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "r"(at + 2 * i)
                   : "memory");
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[i + 2 * e] += w[e] & 0xFFFFu;
        c[i + 2 * e + 1] += w[e] >> 16;
      }
    }
  }
  Weights weights;
  weights.place = s.top[0];
  for (int r = 1; r < C; ++r) weights.place = min(weights.place, s.top[r]);
  if (weights.place == NONE) {  // nothing to draw from
    if (rank == 0 && tid == 0) {
      p.tokens[row] = -1;
      p.logprobs[row] = -INFINITY;
    }
    cluster_sync();  // nobody reads this CTA's histogram any more
    return;
  }
  weights.top = value_at(weights.place);
  weights.top_is_inf = isinf(weights.top);
  const float t_row = p.temperature ? p.temperature[row] : p.temperature_all;
  const bool greedy = !(t_row > 0.f);
  weights.temperature = greedy ? 1.0 : double(t_row);
  const float p_row = p.top_p ? p.top_p[row] : p.top_p_all, m_row = p.min_p ? p.min_p[row] : p.min_p_all;
  const double min_p = m_row > 0.f ? fmin(double(m_row), 1.0) : 0.0;

  // ---- prefix sums of counts and weights
  unsigned n_here = 0;
  u64 mass_here = 0;
#pragma unroll
  for (int i = 0; i < OWN; ++i)
    if (c[i]) {
      n_here += c[i];
      mass_here += c[i] * fixed(weights.of(first + i));
    }
  unsigned n_before = n_here;
  u64 before = mass_here;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned n = __shfl_up_sync(0xffffffffu, n_before, o);
    const u64 m = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) {
      n_before += n;
      before += m;
    }
  }
  if (lane == 31) {
    s.warp_count[warp] = n_before;
    s.warp_mass[warp] = before;
  }
  n_before -= n_here;
  before -= mass_here;
  __syncthreads();
  {
    unsigned n = s.warp_count[lane], n_all = n;
    u64 m = s.warp_mass[lane], m_all = m;
    if (lane >= warp) n = 0, m = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      n += __shfl_xor_sync(0xffffffffu, n, o);
      m += __shfl_xor_sync(0xffffffffu, m, o);
      n_all += __shfl_xor_sync(0xffffffffu, n_all, o);
      m_all += __shfl_xor_sync(0xffffffffu, m_all, o);
    }
    n_before += n;
    before += m;
    if (tid < C) {
      tell(&s.count[rank], tid, n_all);
      tell(&s.mass[rank], tid, m_all);
    }
  }
  cluster_sync();
  unsigned kept = 0;
  u64 kept_mass = 0;
  for (int r = 0; r < C; ++r) {
    if (r < rank) {
      n_before += s.count[r];
      before += s.mass[r];
    }
    kept += s.count[r];
    kept_mass += s.mass[r];
  }

  // ---- top-k (every thread of the cluster takes the same branches)
  const int64_t k_row = greedy ? 1 : p.top_k ? p.top_k[row] : p.top_k_all;
  if (k_row > 0 && k_row < int64_t(kept)) {
    kept = unsigned(k_row);
    if (n_before < kept && kept <= n_before + n_here) {
      unsigned left = kept - n_before;
      u64 m = before;
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const unsigned take = min(left, c[i]);
        if (take) m += take * fixed(weights.of(first + i));
        left -= take;
      }
      for (int r = 0; r < C; ++r) tell(&s.k_mass, r, m);
    }
    cluster_sync();
    kept_mass = s.k_mass;
  }

  // ---- top-p and min-p
  if (!greedy && (p_row < 1.f || min_p > 0.0)) {
    if (p_row < 1.f) {
      const u64 want = max(u64(1), min(kept_mass, u64(ceil(fmax(double(p_row), 0.0) * double(kept_mass)))));
      if (before < want && want <= before + mass_here) {
        unsigned n = n_before;
        u64 m = before;
        bool found = false;
#pragma unroll
        for (int i = 0; i < OWN; ++i)
          if (c[i] && !found) {
            const u64 w = fixed(weights.of(first + i));
            found = want <= m + c[i] * w;
            const unsigned take = found ? unsigned((want - m + w - 1) / w) : c[i];
            n += take;
            m += take * w;
          }
        for (int r = 0; r < C; ++r) {
          tell(&s.p_n, r, n);
          tell(&s.p_mass, r, m);
        }
      }
    }
    if (min_p > 0.0) {  // where the first value stands that is too light
      unsigned n = n_before;
      u64 m = before;
      bool found = false;
#pragma unroll
      for (int i = 0; i < OWN; ++i)
        if (c[i] && !found) {
          const double w = weights.of(first + i);
          found = !(w >= min_p);
          if (!found) {
            n += c[i];
            m += c[i] * fixed(w);
          }
        }
      if (!found) n = NONE;
      const unsigned least = __reduce_min_sync(0xffffffffu, n);
      if (lane == 0) atomicMin(&s.m_here, least);
      __syncthreads();
      if (found && n == s.m_here)
        for (int r = 0; r < C; ++r) {
          tell(&s.m_n[rank], r, n);
          tell(&s.m_mass[rank], r, m);
        }
    }
    cluster_sync();
    if (s.p_n < kept) kept = s.p_n, kept_mass = s.p_mass;
    for (int r = 0; r < C; ++r)
      if (s.m_n[r] < kept) kept = s.m_n[r], kept_mass = s.m_mass[r];
  }

  // ---- draw: whoever owns the border finds the value, its number among the equal
  // ones, and the CTA whose slice holds it
  {
    const float u_row = p.u[row];
    const double x = u_row > 0.f ? double(u_row) * double(kept_mass) : 0.0;
    const u64 want = x < double(kept_mass) ? min(u64(x), kept_mass - 1) : kept_mass - 1;
    if (before <= want && want < before + mass_here) {
      u64 m = before;
      unsigned place = 0, nth = 0;
      bool found = false;
#pragma unroll
      for (int i = 0; i < OWN; ++i)
        if (c[i] && !found) {
          const u64 w = fixed(weights.of(first + i));
          if (want < m + c[i] * w) {
            found = true;
            place = first + i;
            nth = unsigned((want - m) / w);
          }
          m += c[i] * w;
        }
      p.logprobs[row] = float(weights.log_of(place) - log(double(kept_mass) / double(u64(1) << FRAC)));
      for (int r = 0; r < C; ++r) {
        uint32_t w;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(w) : "r"(at_rank(hist + (place >> 1), r)) : "memory");
        const unsigned there = place & 1 ? w >> 16 : w & 0xFFFFu;
        if (nth < there) {
          tell(&s.pick_nth, r, nth);
          tell(&s.pick, r, place);
          break;
        }
        nth -= there;
      }
    }
  }
  cluster_sync();
  const unsigned pick = s.pick;
  if (pick == NONE) return;
  // ---- the pick_nth-th logit of that value in the slice, in index order: a warp counts a
  // run of it, the warp that holds the one looks again
  const unsigned nth = s.pick_nth;
  const int run = (len + THREADS - 1) / THREADS * 32;
  const int begin = min(len, warp * run), end = min(len, begin + run);
  unsigned n = 0;
  for (int i = begin + lane; i < end; i += 32) n += place_of(__ldcg(slice + i)) == pick;
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if (lane == 0) s.warp_count[warp] = n;
  __syncthreads();
  unsigned ahead = 0;
  for (int w = 0; w < warp; ++w) ahead += s.warp_count[w];
  if (nth < ahead || nth >= ahead + n) return;
  for (int i = begin; i < end; i += 32) {
    const bool is = i + lane < end && place_of(__ldcg(slice + i + lane)) == pick;
    const unsigned all = __ballot_sync(0xffffffffu, is);
    if (is && ahead + __popc(all & ((1u << lane) - 1)) == nth) p.tokens[row] = int64_t(rank) * p.slice + i + lane;
    ahead += __popc(all);
  }
}

template <int C>
int launch(const Params& p, int batch, cudaStream_t st) {
  constexpr int SMEM = HIST_BYTES + int(sizeof(Shared<C>));
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  QX_CUDA_TRY(cudaGetDevice(&dev), "sample_logits: cudaGetDevice");
  QX_REQUIRE(dev >= 0 && dev < 64, "sample_logits: device index %d unsupported", dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!done[dev]) {
      QX_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM),
                  "sample_logits: set smem limit");
      done[dev] = true;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(batch) * C);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = g_pdl_enabled.load(std::memory_order_relaxed) ? 2 : 1;
  QX_CUDA_TRY(cudaLaunchKernelEx(&cfg, sample_kernel<C>, p), "sample_logits: launch");
  return check_launch("sample_logits");
}

}  // namespace smp
}  // namespace qx

using namespace qx;

extern "C" int qx_sample_logits(const void* logits, const float* u, const float* temperature, const int64_t* top_k,
                                const float* top_p, const float* min_p, float temperature_all, int64_t top_k_all,
                                float top_p_all, float min_p_all, int64_t* tokens, float* logprobs, int batch, int vocab,
                                qx_stream_t stream) {
  constexpr int C = 8;
  QX_REQUIRE(batch >= 0 && vocab > 0, "sample_logits: bad sizes batch=%d vocab=%d", batch, vocab);
  QX_REQUIRE(vocab <= C * smp::SLICE_MAX, "sample_logits: vocab=%d is above %d", vocab, C * smp::SLICE_MAX);
  QX_REQUIRE(int64_t(batch) * C <= 0x7fffffffLL, "sample_logits: batch=%d is too large", batch);
  if (batch == 0) return QX_OK;
  QX_REQUIRE(logits && u && tokens && logprobs, "sample_logits: null pointer");
  QX_REQUIRE(aligned(logits, 2) && aligned(u, 4) && aligned(temperature, 4) && aligned(top_k, 8) && aligned(top_p, 4) &&
                 aligned(min_p, 4) && aligned(tokens, 8) && aligned(logprobs, 4),
             "sample_logits: a tensor is not aligned to its type");
  smp::Params p{};
  p.logits = static_cast<const __half*>(logits);
  p.u = u;
  p.temperature = temperature;
  p.top_k = top_k;
  p.top_p = top_p;
  p.min_p = min_p;
  p.temperature_all = temperature_all;
  p.top_k_all = top_k_all;
  p.top_p_all = top_p_all;
  p.min_p_all = min_p_all;
  p.tokens = tokens;
  p.logprobs = logprobs;
  p.vocab = vocab;
  p.slice = ((vocab + C - 1) / C + 7) / 8 * 8;
  return smp::launch<C>(p, batch, reinterpret_cast<cudaStream_t>(stream));
}
