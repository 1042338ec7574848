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
// (16-bit counters, 128 KB of shared memory) and tells all which groups of 8 values occur.
// The groups that occur anywhere are dealt out in order, as many to each CTA, one to a
// thread, which adds their counters of all CTAs through distributed shared memory; the
// prefix sums run over threads, warps and CTAs.  Whoever owns the border in question
// (the k-th token, top_p of the weight, u of the weight) tells all CTAs: its warp looks
// at the thread's values again, a lane a value.
//
// Bound by a chain of latencies, not by bytes: measured 11.8 us for one row of 151936 (16
// CTAs), 12.2 for 7 rows of 32003, 16.7 to 17.4 for 32 rows of 151936 (4 CTAs a row, 0.58
// TB/s; their bytes alone 1.35); of these 0.2 to 0.6 for the CTA's decision after each exchange.  Of the 32 rows' time a third is loading and counting, then
// come the exchange of what occurs, the counters and weights, and a border 1 to 1.5 us each: the
// owner's warp, a send, and the wait of all.
#include <mutex>

#include "qx_b200.h"
#include "qx_common.cuh"

namespace qx {
namespace smp {

// threads of a CTA, by the CTAs of a row (us of 512 / 1024: a row of 32003 by 8 12.9 / 13.7, 32 rows of 151936
// by 4 23.6 / 18.9)
constexpr int threads_of(int c) { return c >= 8 ? 512 : 1024; }
constexpr int VALUES = 65536;
constexpr int HIST_BYTES = VALUES * 2;
constexpr int GROUP = 8, GROUPS = VALUES / GROUP, WORDS = GROUPS / 32;  // values that are counted, joined and weighed together
// logits of a CTA: they stay in shared memory, and a 16-bit counter holds them all
constexpr int slice_max(int c) { return c == 16 ? 32768 : c == 8 ? 43008 : 45056; }
constexpr int VOCAB_MAX = 524224;
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
  unsigned test_waits;
};

constexpr int RUNS = slice_max(4) / 256;  // of 256 logits in the largest slice

enum Exchange { USED, TOTALS, TOP_K, LIMITS, PICK, EXCHANGES };

template <int C>
struct Shared {
  u64 done[EXCHANGES];  // mbarriers: what the cluster sends for this exchange has arrived
  // written by the cluster's CTAs
  alignas(16) u64 total[C][2];  // tokens and weight of each CTA's values
  alignas(16) u64 p_run[2];     // tokens and weight of the run that top_p leaves
  alignas(16) u64 m_run[C][2];  // those before the first value of each CTA that is too light for min_p
  u64 k_mass, pick;
  alignas(16) unsigned used[C][WORDS];  // of each CTA: which groups occur
  unsigned top[C];
  // this CTA's
  alignas(16) unsigned mine[WORDS];  // its row of `used`
  unsigned any[WORDS];               // the groups that occur in the row
  unsigned short upto[WORDS];        // how many of them up to a word's end
  unsigned short words_upto[WORDS / 32];
  u64 warp_mass[threads_of(C) / 32];
  unsigned warp_count[threads_of(C) / 32];
  unsigned top_here, m_here, found, found_nth;
  unsigned run[RUNS];
};

// Sticky device-side error word of this file's kernel (QX_DEVERR_* bits), merged into
// qx_get_device_error.
static __device__ unsigned g_sample_error = 0;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t at_rank(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
// Sends to CTA `rank` and counts the bytes on its barrier there: an exchange costs a
// store's way and no barrier of the cluster (which took up to 2 us here).
__device__ __forceinline__ void send(const u64* p, const u64* done, int rank, u64 a) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(at_rank(p, rank)),
               "l"(a), "r"(at_rank(done, rank))
               : "memory");
}
__device__ __forceinline__ void send(const unsigned* p, const u64* done, int rank, unsigned a) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(at_rank(p, rank)),
               "r"(a), "r"(at_rank(done, rank))
               : "memory");
}
__device__ __forceinline__ void send(const u64* p, const u64* done, int rank, u64 a, u64 b) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(at_rank(p, rank)),
               "l"(a), "l"(b), "r"(at_rank(done, rank))
               : "memory");
}
__device__ __forceinline__ void send(const unsigned* p, const u64* done, int rank, const uint4& a) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at_rank(p, rank)),
               "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(at_rank(done, rank))
               : "memory");
}
__device__ __forceinline__ void expect(const u64* done, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(done)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

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

// Weights of a row's values.  exp((v - top) / T) = 2^n e^f with n the nearest integer to
// (v - top) log2(e) / T and |f| <= ln(2) / 2; e^f by its Taylor series to f^12 (the
// next term is below 2^-52).  Conversions between doubles and integers are slow: both
// here are a sum with a number that is so large that the integer stands in the sum's
// low bits, rounded to the nearest.
// A thread's values are neighbours and equally spaced, so their weights are a
// geometric sequence: two exponentials, then a product each (measured at 32 values a
// thread: an exponential each 8300 cycles a row).  Every use of a weight makes it by the
// same products, so its integer is the same everywhere.
struct Weights {
  double top, scale;
  unsigned place;

  // 2^y, 0 below half a unit of the sums
  static __device__ __forceinline__ double power(double y) {
    constexpr double BIG = 6755399441055744.0;  // 1.5 x 2^52
    if (!(y > -45.0)) return 0.0;
    const double big = y + BIG;
    const double f = (y - (big - BIG)) * 0.69314718055994530942;
    double e = 1.0 / 479001600.0;
    e = fma(e, f, 1.0 / 39916800.0);
    e = fma(e, f, 1.0 / 3628800.0);
    e = fma(e, f, 1.0 / 362880.0);
    e = fma(e, f, 1.0 / 40320.0);
    e = fma(e, f, 1.0 / 5040.0);
    e = fma(e, f, 1.0 / 720.0);
    e = fma(e, f, 1.0 / 120.0);
    e = fma(e, f, 1.0 / 24.0);
    e = fma(e, f, 1.0 / 6.0);
    e = fma(e, f, 0.5);
    e = fma(e, f, 1.0);
    e = fma(e, f, 1.0);
    return __hiloint2double(__double2hiint(e) + __double2loint(big) * (1 << 20), __double2loint(e));  // e 2^n
  }
  // the weight of the first of a thread's values that is not above the top (only those occur), and
  // what each of the values behind it has of the one before it
  __device__ __forceinline__ void start(unsigned first, double& w, double& ratio) const {
    const unsigned d = max(first, place);
    w = d == place ? 1.0 : power((value_at(d) - top) * scale);
    ratio = power((value_at(first + 1) - value_at(first)) * scale);
  }
  // w: the weight of place d - 1 (or what start gave) -> that of place d
  __device__ __forceinline__ void next(unsigned first, unsigned d, double ratio, double& w) const {
    if (d > first && d > place) w *= ratio;
  }
};
__device__ __forceinline__ u64 fixed(double w) {  // w 2^FRAC <= 2^43
  constexpr double BIG = 4503599627370496.0;  // 2^52
  return u64(__double_as_longlong(fma(w, double(u64(1) << FRAC), BIG))) & ((u64(1) << 52) - 1);
}

// A row as aligned groups of 8 logits; places outside the row read as -inf
struct Row {
  const unsigned short* at;  // the first logit
  int shift;                 // its place in its aligned group
  int vocab;
  // starts the copy of group i into shared memory
  __device__ __forceinline__ void fetch(int i, uint4* to) const {
    const int first = 8 * i - shift;
    if (first >= 0 && first + 8 <= vocab) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(at + first) : "memory");
      return;
    }
    unsigned short* const v = reinterpret_cast<unsigned short*>(to);
#pragma unroll 1
    for (int e = 0; e < 8; ++e) {
      const int k = first + e;
      v[e] = k >= 0 && k < vocab ? __ldcg(at + k) : 0xFC00u;
    }
  }
};
__device__ __forceinline__ uint32_t hadd2_u32(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t hmax2_u32(uint32_t a, uint32_t b) {  // the number, where one is NaN
  uint32_t d;
  asm("max.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// the larger half of a pair and its place
__device__ __forceinline__ unsigned top_of(uint32_t pair) {
  const uint32_t m = hmax2_u32(pair, pair >> 16);
  return place_of(m & 0xFFFFu);
}

// A message did not come in time: the row's token is undefined and says so.
static __device__ __noinline__ void give_up(int64_t* token, float* logprob) {
  cluster_leave_late();
  if (threadIdx.x == 0) {
    *token = -1;
    *logprob = -INFINITY;
  }
}

template <int C>
__global__ void __launch_bounds__(threads_of(C), 1) sample_kernel(const __grid_constant__ Params p) {
  constexpr int THREADS = threads_of(C), WARPS = THREADS / 32;
  constexpr int Q = GROUPS / (C * THREADS), OWN = Q * GROUP;  // groups and values of a thread, at most
  static_assert(Q >= 1 && OWN <= 32 && THREADS >= WORDS, "a thread's share");
  extern __shared__ __align__(16) unsigned char smem[];
  unsigned* const hist = reinterpret_cast<unsigned*>(smem);
  uint4* const slice = reinterpret_cast<uint4*>(smem + HIST_BYTES);
  Shared<C>& s = *reinterpret_cast<Shared<C>*>(smem + HIST_BYTES + 2 * p.slice);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = blockIdx.x / C, rank = blockIdx.x % C;
  pdl_trigger();
  auto wait_for = [&](int exchange) {
    return exchange_wait(smem_u32(&s.done[exchange]), p.test_waits, exchange, rank, &g_sample_error);
  };
  // whether any warp of the CTA has waited in vain
  auto late = [&](int exchange) { return __syncthreads_or(!wait_for(exchange)); };

  if (tid == 0) {
    s.top_here = s.m_here = NONE;
    s.found = s.found_nth = 0;
    for (int i = 0; i < EXCHANGES; ++i)
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(smem_u32(&s.done[i])) : "memory");
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  cluster_arrive();
  pdl_wait();
  Row logits;
  logits.at = reinterpret_cast<const unsigned short*>(p.logits) + int64_t(row) * p.vocab;
  logits.shift = int(uint32_t(reinterpret_cast<uintptr_t>(logits.at)) & 15u) >> 1;
  logits.vocab = p.vocab;
  const int first_group = rank * (p.slice / 8);
  const int groups = max(0, min(p.slice / 8, (p.vocab + logits.shift + 7) / 8 - first_group));
  // the slice, a thread's own groups (nobody else reads them before a barrier)
  for (int i = tid; i < groups; i += THREADS) logits.fetch(first_group + i, slice + i);
  asm volatile("cp.async.commit_group;" ::: "memory");
  const float u_row = p.u[row], t_row = p.temperature ? p.temperature[row] : p.temperature_all;
  const float p_row = p.top_p ? p.top_p[row] : p.top_p_all, m_row = p.min_p ? p.min_p[row] : p.min_p_all;
  const bool greedy = !(t_row > 0.f);
  const int64_t k_row = greedy ? 1 : p.top_k ? p.top_k[row] : p.top_k_all;
  const double min_p = !greedy && m_row > 0.f ? fmin(double(m_row), 1.0) : 0.0;
  Weights weights;
  weights.scale = greedy ? 1.0 : 1.44269504088896340736 / double(t_row);

  for (int i = tid; i < HIST_BYTES / 16; i += THREADS) reinterpret_cast<uint4*>(hist)[i] = make_uint4(0u, 0u, 0u, 0u);
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();

  // ---- count the slice
  // A slice's logits matter only up to its own k-th largest, and that is not below the
  // k-th largest of the threads' largest ones: a search over places, 16 of them together, a
  // count of the block each of 12 steps.  Without top_p nothing lighter than min_p matters (beside the slice's
  // largest, all the more beside the row's).  Either leaves few logits to count.
  unsigned last = 0xFBFFu;  // the last place that is counted
  const bool by_k = k_row > 0 && k_row <= THREADS / 2, by_min = min_p > 0.0 && !(p_row < 1.f);
  if (by_k || by_min) {
    uint32_t best = 0xFC00FC00u;
    for (int i = tid; i < groups; i += THREADS) {
      const uint4 v = slice[i];
      best = hmax2_u32(best, hmax2_u32(hmax2_u32(v.x, v.y), hmax2_u32(v.z, v.w)));
    }
    const unsigned mine = top_of(best);
    if (by_k) {
      unsigned low = 0;  // the first of the 16 places that the k_row-th of the threads' tops is among
#pragma unroll 1
      for (unsigned bit = 0x8000u; bit >= 16; bit >>= 1)
        if (__syncthreads_count(mine < low + bit) < int(k_row)) low += bit;
      last = min(last, low + 15);
    }
    if (by_min) {
      const unsigned warp_top = __reduce_min_sync(0xffffffffu, mine);
      if (lane == 0) atomicMin(&s.top_here, warp_top);
      __syncthreads();
      const unsigned seen = s.top_here;
      if (seen > 0x3FFu && seen != NONE) {
        // (logf and not __logf, whose error beside 1 is absolute: high temperatures would multiply it past the margin)
        const float seen_at = float(value_at(seen)), down = t_row * -logf(float(min_p));
        const float rounded = seen_at - down - 1e-3f * (1.f + fabsf(seen_at) + down);
        last = min(last, place_of(__half_as_ushort(__float2half_rd(rounded))));  // (NONE where it is -inf)
      }
    }
  }
  uint32_t best = 0xFC00FC00u;
  {
    const unsigned span = last - 0x3FFu;  // places before 0x3FF (+inf) are NaN, those behind 0xFBFF -inf and NaN
#pragma unroll 1
    for (int i = tid; i < groups; i += THREADS) {
      const uint4 v = slice[i];
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      const uint32_t all = hmax2_u32(hmax2_u32(v.x, v.y), hmax2_u32(v.z, v.w));
      best = hmax2_u32(best, all);
      if ((by_k || by_min) && top_of(all) > last) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = hadd2_u32(w[e], 0u);  // the zeros are one value
        const uint32_t d = x ^ (~prmt(x, 0u, 0xBB99u) & 0x7FFF7FFFu);  // place_of of both halves
        const unsigned lo = d & 0xFFFFu, hi = d >> 16;
        if (lo - 0x3FFu <= span) atomicAdd(hist + (lo >> 1), lo & 1 ? 0x10000u : 1u);
        if (hi - 0x3FFu <= span) atomicAdd(hist + (hi >> 1), hi & 1 ? 0x10000u : 1u);
      }
    }
  }
  const unsigned warp_top = __reduce_min_sync(0xffffffffu, top_of(best));
  if (lane == 0) atomicMin(&s.top_here, warp_top);
  __syncthreads();
  cluster_wait();  // every CTA has started
  if (tid == 0) expect(&s.done[USED], C * (4 + 4 * WORDS));
#pragma unroll
  for (int i = 0; i < GROUPS / THREADS; ++i) {
    const uint4 v = reinterpret_cast<const uint4*>(hist)[i * THREADS + tid];
    const unsigned used = __ballot_sync(0xffffffffu, (v.x | v.y | v.z | v.w) != 0u);
    if (lane == 0) s.mine[i * WARPS + warp] = used;
  }
  __syncthreads();
  // what was counted before the __syncthreads is seen by whoever receives from these threads
  if (tid < C * (WORDS / 4)) asm volatile("fence.acq_rel.cluster;" ::: "memory");
  if (tid < C) send(&s.top[rank], &s.done[USED], tid, s.top_here);
  for (int i = tid; i < C * (WORDS / 4); i += THREADS)
    send(&s.used[rank][i % (WORDS / 4) * 4], &s.done[USED], i / (WORDS / 4), reinterpret_cast<const uint4*>(s.mine)[i % (WORDS / 4)]);
  const bool have_used = wait_for(USED);
  weights.place = s.top[0];
  for (int r = 1; r < C; ++r) weights.place = min(weights.place, s.top[r]);
  weights.top = value_at(weights.place);
  // (beside +inf nothing has weight, whatever the temperature)
  if (isinf(weights.top)) weights.top = 1e300, weights.scale = 1.0;

  // ---- the groups that occur, dealt out in order, the same number to each CTA: one to a thread, Q where
  // they are more than its threads.  (By equal shares of all values one CTA had most of those that occur.)
  if (tid < WORDS) {
    unsigned any = 0;
#pragma unroll
    for (int r = 0; r < C; ++r) any |= s.used[r][tid];
    s.any[tid] = any;
    unsigned n = __popc(any);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned t = __shfl_up_sync(0xffffffffu, n, o);
      if (lane >= o) n += t;
    }
    s.upto[tid] = n;
    if (lane == 31) s.words_upto[warp] = n;
  }
  if (__syncthreads_or(!have_used)) {
    give_up(p.tokens + row, p.logprobs + row);
    return;
  }
  if (weights.place == NONE) {  // nothing to draw from
    if (rank == 0 && tid == 0) {
      p.tokens[row] = -1;
      p.logprobs[row] = -INFINITY;
    }
    cluster_arrive();  // nobody reads this CTA's histogram any more
    cluster_wait();
    return;
  }
  unsigned occur = 0, words_before[WORDS / 32];
#pragma unroll
  for (int i = 0; i < WORDS / 32; ++i) words_before[i] = occur, occur += s.words_upto[i];
  const unsigned deal = (occur + C - 1) / C;  // to a CTA
  const int share = Q > 1 && deal > THREADS ? Q : 1;
  unsigned first[Q];  // values of the thread's groups
  unsigned c[OWN];
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    const unsigned nth = tid * share + k, slot = rank * deal + nth;
    first[k] = 0;
#pragma unroll
    for (int i = 0; i < GROUP; ++i) c[k * GROUP + i] = 0;
    if (k >= share || nth >= deal || slot >= occur) continue;
    // the word: of 32 words together, then of those
    unsigned block = 0, left = slot;
#pragma unroll
    for (int i = 1; i < WORDS / 32; ++i)
      if (slot >= words_before[i]) block = i, left = slot - words_before[i];
    unsigned word = 0;  // the first with more than `left` up to its end
#pragma unroll
    for (int i = 16; i; i >>= 1)
      if (s.upto[block * 32 + word + i - 1] <= left) word += i;
    if (word) left -= s.upto[block * 32 + word - 1];
    word += block * 32;
    unsigned bits = s.any[word], bit = 0;
#pragma unroll
    for (int i = 16; i; i >>= 1) {
      const unsigned low = __popc(bits & ((1u << i) - 1));
      if (left >= low) left -= low, bits >>= i, bit += i;
    }
    first[k] = (word * 32 + bit) * GROUP;
    // its counters of all CTAs
    uint32_t there[C][4];
#pragma unroll
    for (int r = 0; r < C; ++r) {
#pragma unroll
      for (int e = 0; e < 4; ++e) there[r][e] = 0u;
      if (s.used[r][word] >> bit & 1)
        asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(there[r][0]), "=r"(there[r][1]), "=r"(there[r][2]), "=r"(there[r][3])
                     : "r"(at_rank(hist + first[k] / 2, r))
                     : "memory");
    }
#pragma unroll
    for (int i = 0; i < GROUP / 2; ++i)
#pragma unroll
      for (int r = 0; r < C; ++r) {
        c[k * GROUP + 2 * i] += there[r][i] & 0xFFFFu;
        c[k * GROUP + 2 * i + 1] += there[r][i] >> 16;
      }
  }

  // ---- prefix sums of counts and weights; of those heavy enough for min_p, and whether some are not
  unsigned n_here = 0, n_heavy = 0;
  u64 mass_here = 0, mass_heavy = 0;
  bool light = false;
  double start[Q], ratio[Q];  // the groups' first weights, and what each has of the one before it
#pragma unroll
  for (int k = 0; k < Q; ++k) {
    start[k] = ratio[k] = 0.0;
    if (first[k] == 0) continue;  // no group (the first one's places are NaN and do not occur)
    weights.start(first[k], start[k], ratio[k]);
    double w = start[k];
#pragma unroll
    for (int i = 0; i < GROUP; ++i) {
      const unsigned n = c[k * GROUP + i];
      weights.next(first[k], first[k] + i, ratio[k], w);
      if (n) {
        n_here += n;
        mass_here += n * fixed(w);
        light |= !(w >= min_p);
        if (!light) n_heavy = n_here, mass_heavy = mass_here;
      }
    }
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
  if (warp == 0) {
    const unsigned n_own = lane < WARPS ? s.warp_count[lane] : 0u;
    const u64 m_own = lane < WARPS ? s.warp_mass[lane] : 0u;
    unsigned n = n_own;
    u64 m = m_own;
#pragma unroll
    for (int o = 1; o < WARPS; o <<= 1) {
      const unsigned n2 = __shfl_up_sync(0xffffffffu, n, o);
      const u64 m2 = __shfl_up_sync(0xffffffffu, m, o);
      if (lane >= o) {
        n += n2;
        m += m2;
      }
    }
    if (lane < WARPS) {
      s.warp_count[lane] = n - n_own;
      s.warp_mass[lane] = m - m_own;
    }
    n = __shfl_sync(0xffffffffu, n, WARPS - 1);
    m = __shfl_sync(0xffffffffu, m, WARPS - 1);
    if (lane == 0) expect(&s.done[TOTALS], C * 16);
    if (lane < C) send(s.total[rank], &s.done[TOTALS], lane, n, m);
  }
  __syncthreads();
  n_before += s.warp_count[warp];
  before += s.warp_mass[warp];
  if (late(TOTALS)) {
    give_up(p.tokens + row, p.logprobs + row);
    return;
  }
  unsigned kept = 0;
  u64 kept_mass = 0;
#pragma unroll
  for (int r = 0; r < C; ++r) {
    if (r < rank) {
      n_before += unsigned(s.total[r][0]);
      before += s.total[r][1];
    }
    kept += unsigned(s.total[r][0]);
    kept_mass += s.total[r][1];
  }

  // Three borders: of the first top_k tokens, of top_p of their weight, of u of the weight
  // kept.  Each lies among the values of one thread of the cluster; in its warp, lane i < OWN
  // looks at the thread's value i, and the one that has the border tells all CTAs.  (One
  // loop and not three pieces of code: every instruction is fetched for one use.)
  const bool cut_k = k_row > 0 && k_row < int64_t(kept), cut_p = !greedy && p_row < 1.f;
  if (cut_k) kept = unsigned(k_row);
#pragma unroll 1
  for (int border = TOP_K; border <= PICK; ++border) {
    u64 want = 0;  // the border lies behind this much weight (TOP_K: behind kept - 1 tokens)
    if (border == TOP_K) {
      if (!cut_k) continue;
      if (tid == 0) expect(&s.done[TOP_K], 8);
    } else if (border == LIMITS) {
      if (!cut_p && !(min_p > 0.0)) continue;
      if (tid == 0) expect(&s.done[LIMITS], (cut_p ? 16 : 0) + (min_p > 0.0 ? 16 * C : 0));
      want = max(u64(1), min(kept_mass, u64(ceil(fmax(double(p_row), 0.0) * double(kept_mass))))) - 1;
      if (min_p > 0.0) {  // where the first value stands that is too light
        const unsigned n = light ? n_before + n_heavy : NONE;
        const unsigned least = __reduce_min_sync(0xffffffffu, n);
        if (lane == 0) atomicMin(&s.m_here, least);
        __syncthreads();
        if (s.m_here == NONE ? tid == 0 : light && n == s.m_here)
#pragma unroll 1
          for (int r = 0; r < C; ++r) send(s.m_run[rank], &s.done[LIMITS], r, n, before + mass_heavy);
      }
    } else {
      if (tid == 0) expect(&s.done[PICK], 8);
      const double x = u_row > 0.f ? double(u_row) * double(kept_mass) : 0.0;
      want = x < double(kept_mass) ? min(u64(x), kept_mass - 1) : kept_mass - 1;
    }
    bool here = before <= want && want < before + mass_here;
    if (border == TOP_K) here = n_before < kept && kept <= n_before + n_here;
    if (border == LIMITS) here = here && cut_p;
    const unsigned who = __ballot_sync(0xffffffffu, here);
    if (who) {
      const int o = __ffs(who) - 1;
      unsigned from = __shfl_sync(0xffffffffu, first[0], o), count = 0;
      if (Q > 1) {
        const unsigned second = __shfl_sync(0xffffffffu, first[Q - 1], o);
        if (lane >= GROUP) from = second;
      }
      double w, r;
      // (kept from the sums, when it was chosen: one row of 151936 11.8 us instead of 12.2, 7 of 32003 12.0 instead of 12.7; where a
      // thread has 64 registers, made again: 32 rows 17.4 instead of 17.7)
      if constexpr (THREADS <= 512) {
        w = __shfl_sync(0xffffffffu, start[0], o), r = __shfl_sync(0xffffffffu, ratio[0], o);
        if (Q > 1) {
          const double w2 = __shfl_sync(0xffffffffu, start[Q - 1], o), r2 = __shfl_sync(0xffffffffu, ratio[Q - 1], o);
          if (lane >= GROUP) w = w2, r = r2;
        }
      } else {
        weights.start(from, w, r);
      }
#pragma unroll
      for (int i = 0; i < OWN; ++i) {
        const unsigned t = __shfl_sync(0xffffffffu, c[i], o);
        if (lane == i) count = t;
        if (i < GROUP && i <= (lane & (GROUP - 1))) weights.next(from, from + i, r, w);
      }
      const u64 each = count ? fixed(w) : 0;
      unsigned n = count;
      u64 m = count * each;
#pragma unroll
      for (int i = 1; i < OWN; i <<= 1) {
        const unsigned n2 = __shfl_up_sync(0xffffffffu, n, i);
        const u64 m2 = __shfl_up_sync(0xffffffffu, m, i);
        if (lane >= i) {
          n += n2;
          m += m2;
        }
      }
      n += __shfl_sync(0xffffffffu, n_before, o) - count;  // before this lane's value
      m += __shfl_sync(0xffffffffu, before, o) - count * each;
      const bool found = border == TOP_K ? n < kept && kept <= n + count : m <= want && want < m + count * each;
      const int f = __ffs(__ballot_sync(0xffffffffu, found)) - 1;
      // the tokens of the value before the border: want less m in units of its weight (a count
      // is below 2^19, so the quotient in fp32 is off by one at most)
      unsigned nth = kept - n;
      if (border != TOP_K && found) {
        const u64 x = want - m;
        nth = unsigned(__fdividef(float(x), float(each)));
        if (nth * each > x) --nth;
        if ((nth + 1) * each <= x) ++nth;
      }
      const unsigned place = __shfl_sync(0xffffffffu, from + (lane & (GROUP - 1)), f);
      n = __shfl_sync(0xffffffffu, n, f);
      nth = __shfl_sync(0xffffffffu, nth, f);
      const u64 upto = __shfl_sync(0xffffffffu, m + nth * each, f), one = __shfl_sync(0xffffffffu, each, f);
      // lane r tells CTA r
      if (border == TOP_K) {
        if (lane < C) send(&s.k_mass, &s.done[TOP_K], lane, upto);
      } else if (border == LIMITS) {
        if (lane < C) send(s.p_run, &s.done[LIMITS], lane, n + nth + 1, upto + one);
      } else {  // the CTA that holds the token learns which, the others that it is not theirs
        uint32_t mine = 0;
        if (lane < C) {
          asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(mine) : "r"(at_rank(hist + (place >> 1), lane)) : "memory");
          mine = place & 1 ? mine >> 16 : mine & 0xFFFFu;
        }
        unsigned all = mine;
#pragma unroll
        for (int i = 1; i < C; i <<= 1) {
          const unsigned t = __shfl_up_sync(0xffffffffu, all, i);
          if (lane >= i) all += t;
        }
        const bool holds = all - mine <= nth && nth < all;
        if (lane < C) send(&s.pick, &s.done[PICK], lane, holds ? u64(nth - (all - mine)) << 32 | place : u64(NONE));
        if (lane == 0) {
          const double away = place == weights.place ? 0.0 : (value_at(place) - weights.top) * weights.scale * 0.69314718055994530942;
          p.logprobs[row] = float(away - log(double(kept_mass) / double(u64(1) << FRAC)));
        }
      }
    }
    if (border == PICK) break;
    if (late(border)) {
      give_up(p.tokens + row, p.logprobs + row);
      return;
    }
    if (border == TOP_K) kept_mass = s.k_mass;
    if (border == LIMITS) {
      if (cut_p && s.p_run[0] < kept) kept = unsigned(s.p_run[0]), kept_mass = s.p_run[1];
      if (min_p > 0.0)
#pragma unroll 1
        for (int r = 0; r < C; ++r)
          if (s.m_run[r][0] < kept) kept = unsigned(s.m_run[r][0]), kept_mass = s.m_run[r][1];
    }
  }
  if (late(PICK)) {
    give_up(p.tokens + row, p.logprobs + row);
    return;
  }
  const unsigned pick = unsigned(s.pick);
  if (pick == NONE) return;
  // ---- the logit of that value and number in the slice, in index order: counted in runs
  // of 256 logits (a load of a warp), then within the run that holds it
  const __half value = __ushort_as_half(static_cast<unsigned short>((pick & 0x8000u) ? pick : 0x7FFFu - pick));
  const __half2 pattern = __halves2half2(value, value);
  auto matches = [&](int group) {  // equal as numbers: the zeros' sign does not count
    const uint4 v = slice[group];
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
    unsigned mask = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      mask |= __heq2_mask(*reinterpret_cast<const __half2*>(&w[e]), pattern) & (1u << 2 * e | 0x20000u << 2 * e);
    return (mask | mask >> 16) & 0xFFu;
  };
#pragma unroll 2
  for (int i = tid; i - lane < groups; i += THREADS) {
    const unsigned n = __reduce_add_sync(0xffffffffu, i < groups ? __popc(matches(i)) : 0u);
    if (lane == 0) s.run[i / 32] = n;
  }
  __syncthreads();
  const int runs = (groups + 31) / 32;
  if (warp == 0) {
    unsigned left = unsigned(s.pick >> 32);
    for (int i = 0; i < runs; i += 32) {
      unsigned upto = i + lane < runs ? s.run[i + lane] : 0u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
      }
      const unsigned past = __ballot_sync(0xffffffffu, left < upto);
      if (past) {
        const int r = __ffs(past) - 1;
        const unsigned ahead = r ? __shfl_sync(0xffffffffu, upto, r ? r - 1 : 0) : 0u;
        if (lane == 0) {
          s.found = i + r;
          s.found_nth = left - ahead;
        }
        break;
      }
      left -= __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  __syncthreads();
  if (warp != 0) return;
  const int group = int(s.found) * 32 + lane;
  unsigned mask = unsigned(group) < unsigned(groups) ? matches(group) : 0u;
  unsigned upto = __popc(mask);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned t = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += t;
  }
  const unsigned ahead = upto - __popc(mask), nth = s.found_nth;
  if (nth >= ahead && nth < upto) {
    for (unsigned k = ahead; k < nth; ++k) mask &= mask - 1;
    p.tokens[row] = 8 * int64_t(first_group + group) - logits.shift + __ffs(mask) - 1;
  }
}

template <int C>
constexpr int smem_bytes(int slice) {
  return HIST_BYTES + 2 * slice + int(sizeof(Shared<C>));
}
inline int slice_of(int vocab, int c) {  // (a row may begin up to 7 places into a group of 8)
  return ((vocab + 7 + c - 1) / c + 255) / 256 * 256;
}

struct Launch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
};
template <int C>
void configure(Launch& l, int slice, int batch, cudaStream_t st) {
  l.cfg.gridDim = dim3(unsigned(batch) * C);
  l.cfg.blockDim = dim3(threads_of(C));
  l.cfg.dynamicSmemBytes = size_t(smem_bytes<C>(slice));
  l.cfg.stream = st;
  l.at[0].id = cudaLaunchAttributeClusterDimension;
  l.at[0].val.clusterDim.x = C;
  l.at[0].val.clusterDim.y = l.at[0].val.clusterDim.z = 1;
  l.at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  l.at[1].val.programmaticStreamSerializationAllowed = 1;
  l.cfg.attrs = l.at;
  l.cfg.numAttrs = g_pdl_enabled.load(std::memory_order_relaxed) ? 2 : 1;
}

// Prepares the kernel on the current device, once; how many clusters run on it at the same time.
template <int C>
int prepare(int* clusters) {
  static_assert(smem_bytes<C>(slice_max(C)) <= 227 * 1024, "shared memory of the largest slice");
  static std::mutex mu;
  static int fit[64] = {};
  int dev = 0;
  QX_CUDA_TRY(cudaGetDevice(&dev), "sample_logits: cudaGetDevice");
  QX_REQUIRE(dev >= 0 && dev < 64, "sample_logits: device index %d unsupported", dev);
  std::lock_guard<std::mutex> lk(mu);
  if (fit[dev] == 0) {
    QX_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<C>(slice_max(C))),
                "sample_logits: set smem limit");
    if (C > 8)
      QX_CUDA_TRY(cudaFuncSetAttribute(sample_kernel<C>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1),
                  "sample_logits: allow clusters of 16");
    Launch l;
    configure<C>(l, slice_max(C), 1, nullptr);
    l.cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, sample_kernel<C>, &l.cfg) != cudaSuccess) {
      cudaGetLastError();  // a device that has no room for clusters of this size: none of them
      n = 0;
    }
    fit[dev] = n > 0 ? n : -1;
  }
  *clusters = fit[dev];
  return QX_OK;
}

template <int C>
int launch(Params& p, int batch, cudaStream_t st) {
  p.slice = slice_of(p.vocab, C);
  Launch l;
  configure<C>(l, p.slice, batch, st);
  QX_CUDA_TRY(cudaLaunchKernelEx(&l.cfg, sample_kernel<C>, p), "sample_logits: launch");
  return check_launch("sample_logits");
}

// The largest cluster with which the whole batch runs at once (7 rows by 16 CTAs, 15 by 8, 32 by 4 on a B200 of
// 148 SMs), else 4.  Measured when it was chosen, at 151936 tokens, us by 16 / 8 / 4 CTAs: 1 row 12.6 / 12.7 / 15.6, 7 rows
// 12.2 / 13.1 / 16.0, 8 rows 22.4 / 13.2 / 15.9, 16 rows 33 / 24 / 16.1, 64 rows 108 / 58 / 32.
int choose(Params& p, int batch, cudaStream_t st) {
  int at16 = 0, at8 = 0, at4 = 0;
  if (const int rc = prepare<16>(&at16); rc != QX_OK) return rc;
  if (const int rc = prepare<8>(&at8); rc != QX_OK) return rc;
  if (const int rc = prepare<4>(&at4); rc != QX_OK) return rc;
  if (batch <= at16 || slice_of(p.vocab, 8) > slice_max(8)) return launch<16>(p, batch, st);
  if (batch <= at8 || slice_of(p.vocab, 4) > slice_max(4)) return launch<8>(p, batch, st);
  return launch<4>(p, batch, st);
}

}  // namespace smp

int sample_device_error(unsigned* code, int reset) {
  QX_CUDA_TRY(cudaMemcpyFromSymbol(code, smp::g_sample_error, sizeof(unsigned)), "get_device_error: read");
  if (reset) {
    const unsigned zero = 0;
    QX_CUDA_TRY(cudaMemcpyToSymbol(smp::g_sample_error, &zero, sizeof(unsigned)), "get_device_error: reset");
  }
  return QX_OK;
}

}  // namespace qx

using namespace qx;

extern "C" int qx_sample_logits(const void* logits, const float* u, const float* temperature, const int64_t* top_k,
                                const float* top_p, const float* min_p, float temperature_all, int64_t top_k_all,
                                float top_p_all, float min_p_all, int64_t* tokens, float* logprobs, int batch, int vocab,
                                qx_stream_t stream) {
  QX_REQUIRE(batch >= 0 && vocab > 0, "sample_logits: bad sizes batch=%d vocab=%d", batch, vocab);
  QX_REQUIRE(vocab <= smp::VOCAB_MAX, "sample_logits: vocab=%d is above %d", vocab, smp::VOCAB_MAX);
  QX_REQUIRE(batch <= 0x7fffffff / 16, "sample_logits: batch=%d is too large", batch);
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
  p.test_waits = g_test_waits.load(std::memory_order_relaxed);
  return smp::choose(p, batch, reinterpret_cast<cudaStream_t>(stream));
}
