// Prefill attention of a prompt chunk over the 4-bit ring KV cache (format:
// kv4.cuh) and over the chunk's own fp16 keys and values, before the chunk is
// appended.  The mask is qx_prefill_attention's: key kp is visible to query p
// iff kp <= p and (kp < sink or kp > p - window); the ring's slots sit at the
// positions its write rule gives them.  New component (the reference gathers
// the cache, qextract/kv_cache.py:96-112, and attends over the copy).
//
// Flash-attention form on the tcgen05 tensor cores.  A CTA owns 256 rows of one
// KV head in two tiles of 128; a row is (query position, query head of the
// group), positions outermost, so the group's heads share every key tile and
// the rows of a CTA see nearly the same keys.  Tiles of 128 keys: the ring's
// that any of its rows sees, then the chunk's up to the last row.
//   warp 0          an elected lane issues tcgen05.mma: S = Q K^T (both operands in
//                   shared memory) and O += P V (P from TMEM).  As the last warp
//                   it lost its issue slots to the others and each of its waits
//                   took 300 clocks longer.
//   warps 1-3       loaders: ring rows are made fp16 (exactly: kv4.cuh) on the
//                   way to the 128-byte-swizzled K (K-major) and V (MN-major)
//                   tiles, the chunk's rows copied; two stages each
//   warps 4-7, 8-11 softmax of row tile 0 and 1, one thread a row: S from TMEM,
//                   the running maximum and sum in fp32, P in fp16 back to
//                   TMEM.  O (fp32, TMEM) is rescaled only when the row's
//                   maximum grew by more than 2^4, so P carries 2^11 at the
//                   maximum last used and at most 2^15; both cancel in O / l.
// The two row tiles alternate: while one's softmax runs, the other's P V and next
// Q K^T do, and P V starts on the first 64 keys while the weights of the other 64 are
// computed (2048-token chunk after 4096 slots 180 -> 172.6 us; on the first
// 32: 176.8, 96: 173.2).  A softmax thread takes its row of S to registers, and P goes over S:
// TMEM holds S/P of both row tiles (256 columns) and O of both (2 D), the SM's 512
// at D = 128.  (Steps of 64 keys with an S, P and O apart overlap more on paper,
// but their products read Q twice as often: shared memory is then the bound, and
// every barrier wait queues behind it: 197 us for the 2048-token chunk.)
// What bounds it (2048 tokens after 4096 slots: 171 us, 804 TFLOP/s, 0.48 of the bf16 rate;
// on another GPU 178): the exponentials take 46 % of the time on their pipe, the products
// 45 % on theirs, issue is 47 %, and with two row tiles, which is what TMEM holds, the chain
// S - softmax - P V leaves each idle in turn; and 256 CTAs are 1.73 waves.  (Two threads a row: 251 us; some exponentials as
// polynomials on the FMA pipe: 204 and more, against 180 then.)
// Few rows (a short chunk after a long context): CTAs split the key tiles and a
// second kernel joins their fp32 results.
// Every wait is bounded (kWaitLimitNs, then QX_DEVERR_MBAR_TIMEOUT; the CTA's
// later waits give up at once).
#include <algorithm>
#include <cmath>
#include <mutex>
#include <type_traits>

#include "kv4.cuh"
#include "qx_b200.h"

namespace qx {
namespace pattn4 {

constexpr int ROWS = 128;        // rows of a tile: tcgen05's M
constexpr int KT = 128;          // keys of a tile
constexpr int STAGES = 2;
constexpr int LOAD_WARPS = 3, SOFTMAX_WARP0 = 1 + LOAD_WARPS, SOFTMAX_WARPS = 8;
constexpr int THREADS = (SOFTMAX_WARP0 + SOFTMAX_WARPS) * 32;
constexpr int GROUPS = KT / 8;  // 8-row groups of a key tile, dealt to the loader warps in turn
constexpr int PASSES = (GROUPS + LOAD_WARPS - 1) / LOAD_WARPS;
static_assert(SOFTMAX_WARP0 % 4 == 0, "a softmax warp's TMEM lanes are 32 (warp % 4) ..");
constexpr int FIRST = 64;        // keys of a tile whose P V starts before the other weights are there
constexpr float GROW = 4.f;      // log2 growth of a row's maximum that O is rescaled for
constexpr float PSHIFT = 11.f;   // P carries 2^11: at most 2^15 with GROW, subnormal below 2^-25 of the maximum
constexpr int MAX_SPLITS = 32;

// barriers (8 bytes each)
enum { FULL_K, EMPTY_K = FULL_K + STAGES, FULL_V = EMPTY_K + STAGES, EMPTY_V = FULL_V + STAGES,
       S_FULL = EMPTY_V + STAGES, P_FULL = S_FULL + 2, P_HALF = P_FULL + 2, PV_DONE = P_HALF + 2, O_FULL = PV_DONE + 2, Q_FULL = O_FULL + 2, NBARS };

template <int D>
struct Smem {
  static constexpr int TILE = ROWS * D * 2;  // bytes of a Q, K or V tile
  static constexpr int Q = 0, K = 2 * TILE, V = K + STAGES * TILE, BARS = V + STAGES * TILE;
  static constexpr int TMEM = BARS + NBARS * 8, GAVE_UP = TMEM + 4, LIST = GAVE_UP + 4;
  static constexpr int BYTES = LIST + 128 + 1024;  // + alignment slack
};

struct Params {
  const __half* q;   // [B][n][Hq][D]
  const __half* kn;  // [B][n][Hkv][D]
  const __half* vn;
  const unsigned char* kc;
  const uint16_t* kp;
  const unsigned char* vc;
  const uint16_t* vp;
  __half* out;
  float4* part_o;   // [nsplit][B][Hkv][strip][D / 4][32 rows]
  float2* part_ml;  // [nsplit][B][Hkv][strip][32 rows]
  const int64_t* counts;
  int64_t count, cap;
  int batch, n, hq, hkv, G, sink, window, nsplit;
  int strips;  // of 32 rows (a softmax warp's): 8 a row block
  float scale_log2;
};

// Sticky device-side error word of this file's kernels (QX_DEVERR_* bits),
// merged into qx_get_device_error.
static __device__ unsigned g_prefill4_error = 0;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(b), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t b) {
  asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(b) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred P; mbarrier.try_wait.parity.acquire.cta.shared::cta.b64 P, [%1], %2; "
      "selp.u32 %0, 1, 0, P; }"
      : "=r"(ok)
      : "r"(b), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __noinline__ void bar_wait_slow(uint32_t b, uint32_t parity, volatile unsigned* gave_up) {
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t0));
  while (!bar_try(b, parity)) {
    if (*gave_up) return;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    if (t - t0 > kWaitLimitNs) {
      *gave_up = 1;
      atomicOr(&g_prefill4_error, QX_DEVERR_MBAR_TIMEOUT);
      return;
    }
  }
}
__device__ __forceinline__ void bar_wait(uint32_t b, uint32_t parity, volatile unsigned* gave_up) {
  if (!bar_try(b, parity)) bar_wait_slow(b, parity, gave_up);
}

// shared-memory operand of 128-byte-swizzled rows (64 values), 8-row atoms 1024 B
// apart, tiles of 64 values `half` bytes apart.  K-major (Q, K): the rows are M
// or N, `half` unused; MN-major (V): the rows are the product's K, `half` steps N.
// Only the low word holds the address.
constexpr uint32_t DESC_HI = 64u | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t half) { return (saddr >> 4) | (half >> 4) << 16; }
// kind::f16 instruction descriptor: D f32, A and B f16, M = 128; MN_B: B is MN-major
template <int N, bool MN_B>
constexpr uint32_t idesc() {
  return (1u << 4) | (MN_B ? 1u << 16 : 0u) | (uint32_t(N >> 3) << 17) | (uint32_t(ROWS >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t id, uint32_t acc) {
  asm volatile(
      "{ .reg .pred p;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p; }" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(id), "r"(acc), "r"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t id, uint32_t acc) {
  asm volatile(
      "{ .reg .pred p;\n .reg .b64 b;\n setp.ne.b32 p, %4, 0;\n mov.b64 b, {%2, %5};\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p; }" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(id), "r"(acc), "r"(DESC_HI)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(b) : "memory");
}
// one lane of a converged warp (the same one every time)
__device__ __forceinline__ bool elected() {
  uint32_t ok;
  asm volatile("{ .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p; }" : "=r"(ok));
  return ok != 0;
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

#define QX_R8(v, i) "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3]), "=f"(v[i + 4]), "=f"(v[i + 5]), "=f"(v[i + 6]), "=f"(v[i + 7])
// Columns of the warp's 32 rows, a row a thread.  Load and wait are one statement:
// between them a value still on its way could be copied or spilled.
__device__ __forceinline__ void tmem_ld64(uint32_t addr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : QX_R8(v, 0), QX_R8(v, 8), QX_R8(v, 16), QX_R8(v, 24), QX_R8(v, 32), QX_R8(v, 40), QX_R8(v, 48), QX_R8(v, 56)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : QX_R8(v, 0), QX_R8(v, 8), QX_R8(v, 16), QX_R8(v, 24)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : QX_R8(v, 0), QX_R8(v, 8)
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const float (&v)[16]) {
  uint32_t u[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) u[i] = __float_as_uint(v[i]);
  tmem_st16(addr, u);
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two fp32 operations an instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{ .reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      "fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x; }"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{ .reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 x, x, y;\n"
      "mov.b64 {%0, %1}, x; }"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));  // NaN if one is
  return d;
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

// The key tiles that some row of [rmin, rmax] (chunk positions) may see, as
// ranges of tile numbers: of the ring's slots the sinks (0), those up to the
// newest token's (1) and those after it (2: older, where the ring has wrapped),
// then of the chunk's keys the sinks (3) and the window (4).  What the ring hides
// from rmin it hides from all; a range starts after the one before it.  And the
// keys [lo, hi) of each part that all of the rows see.  Made once, in shared memory.
struct Tiles {
  int start[5], end[5], lo[5], hi[5], total;

  __device__ void make(const Ring& r, int rmin, int rmax, int sink, int window) {
    const int held = r.valid - sink, last = min(r.newest, held - 1);  // ring tokens (below zero: sinks only)
    const bool some = r.newest >= 0;
    // row p sees ring index w <= newest from newest - window + 2 + p, w > newest from newest + 2 + p
    const int from = r.newest - window + 2;
    const int first[5] = {0, sink + max(0, from + rmin), sink + r.newest + 2 + rmin, 0, max(0, rmin - window + 1)};
    const int stop[5] = {min(r.valid, sink), some ? sink + last + 1 : 0, some ? r.valid : 0, min(r.sinks, rmax + 1), rmax + 1};
    int next = 0;
    total = 0;
    for (int k = 0; k < 5; ++k) {
      if (k == 3) next = 0;
      start[k] = max(next, first[k] / KT);
      end[k] = stop[k] > first[k] ? max(start[k], (stop[k] - 1) / KT + 1) : start[k];
      if (end[k] > start[k]) next = end[k];
      total += end[k] - start[k];
    }
    lo[0] = 0, hi[0] = stop[0];
    lo[1] = sink + max(0, from + rmax), hi[1] = stop[1];
    lo[2] = sink + r.newest + 2 + rmax, hi[2] = stop[2];
    lo[3] = 0, hi[3] = min(r.sinks, rmin + 1);
    lo[4] = max(0, rmax - window + 1), hi[4] = rmin + 1;
    if (lo[1] <= hi[0] && hi[1] > hi[0]) hi[0] = hi[1];  // the sinks and the window meet
    if (lo[4] <= hi[3] && hi[4] > hi[3]) hi[3] = hi[4];
  }
};

// a walk over the list from tile t on
struct Walk {
  int k, tile;
  __device__ Walk(const Tiles& l, int t) : k(0) {
    while (k < 4 && t >= l.end[k] - l.start[k]) {
      t -= l.end[k] - l.start[k];
      ++k;
    }
    tile = l.start[k] + t;
  }
  __device__ void next(const Tiles& l) {
    if (++tile < l.end[k]) return;
    while (++k < 5 && l.start[k] >= l.end[k]) {
    }
    if (k < 5) tile = l.start[k];
  }
  __device__ bool of_ring() const { return k < 3; }
};

// bits of [lo, hi) within [base, base + 32)
__device__ __forceinline__ uint32_t bits(int lo, int hi, int base) {
  lo = min(max(lo - base, 0), 32);
  hi = min(max(hi - base, 0), 32);
  if (hi <= lo) return 0u;
  return (0xFFFFFFFFu >> (32 - (hi - lo))) << lo;  // hi > lo: lo < 32 and the width is 1 to 32
}

// the keys k0 + 32 j .. + 31 that the row at `pos` sees, a bit each
__device__ __forceinline__ uint32_t seen_bits(const Params& p, const Ring& ring, bool of_ring, int k0, int j, int pos) {
  if (of_ring) {
    const int sk = p.sink - k0, nw = sk + ring.newest;  // from the tile's first slot: first ring slot, newest
    const int end = ring.valid - k0;
    return bits(0, min(sk, end), 32 * j) | bits(max(sk, nw - p.window + 2 + pos), min(nw + 1, end), 32 * j) |
           bits(max(nw + 1, nw + 2 + pos), end, 32 * j);
  }
  return bits(0, min(pos + 1, ring.sinks) - k0, 32 * j) | bits(pos - p.window + 1 - k0, pos + 1 - k0, 32 * j);
}

// Has a key that the row at `pos` does not see, in its row block's tiles, a value that is
// not finite, where the row sees no key whose values are all NaN (it is NaN then in
// any case: the rows of a padded sequence's end)?  By one warp.
template <int D, int NG>
__device__ __forceinline__ bool hidden_reached(const Params& p, const Ring& ring, int b, int h, int pos, int lane) {
  const int kvh = h / p.G, row0 = (pos * p.G + h - kvh * p.G) / (2 * ROWS) * (2 * ROWS);
  Tiles tiles;
  tiles.make(ring, row0 / p.G, (min(p.n * p.G, row0 + 2 * ROWS) - 1) / p.G, p.sink, p.window);
  uint32_t reached = 0, gone = 0;
#pragma unroll 1
  for (int k = 0; k < 5; ++k) {
    const bool of_ring = k < 3;
    const int end = tiles.end[k] * KT;
#pragma unroll 1
    for (int k1 = tiles.start[k] * KT; k1 < end; k1 += 32 * 32) {
      // of 32 runs of 32 keys, a lane each: those not all seen, and the row's own key's
      const int mine = k1 + 32 * lane;
      const bool own = !of_ring && mine <= pos && pos < mine + 32;
      uint32_t runs = __ballot_sync(0xffffffffu, mine < end && (own || seen_bits(p, ring, of_ring, mine, 0, pos) != 0xFFFFFFFFu));
#pragma unroll 1
      for (; runs; runs &= runs - 1) {
        const int k0 = k1 + 32 * (__ffs(runs) - 1);
        const uint32_t seen = seen_bits(p, ring, of_ring, k0, 0, pos);
        const int key = k0 + lane;
        bool bad = false, nan = false;  // some value, every value
        if (of_ring && key < ring.valid) {  // a scale that is NaN
          const uint16_t* w = p.vp + ((int64_t(b) * p.hkv + kvh) * p.cap + key) * NG;
          nan = true;
#pragma unroll
          for (int n = 0; n < NG; ++n) {
            bad = bad || w[n] >= 0x7C00u;
            nan = nan && w[n] >= 0x7C00u;
          }
        } else if (!of_ring && key < p.n) {
          const uint4* v = reinterpret_cast<const uint4*>(p.vn + ((int64_t(b) * p.n + key) * p.hkv + kvh) * D);
          uint32_t top = 0, least = 0x7FFF7FFFu;  // of the magnitudes' bits
#pragma unroll 4
          for (int i = 0; i < D / 8; ++i) {
            const uint4 x = __ldg(v + i);
            const uint32_t y[4] = {x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu, x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu};
#pragma unroll
            for (int e = 0; e < 4; ++e) top = __vmaxu2(top, y[e]), least = __vminu2(least, y[e]);
          }
          bad = max(top >> 16, top & 0xFFFFu) >= 0x7C00u;
          nan = min(least >> 16, least & 0xFFFFu) > 0x7C00u;
        }
        reached |= __ballot_sync(0xffffffffu, bad) & ~seen;
        gone |= __ballot_sync(0xffffffffu, nan) & seen;
      }
    }
  }
  return reached && !gone;
}

// A row whose result is not finite: where a hidden key's NaN or infinity has reached it
// (in a tile product its weight 0 times that value is NaN), it is done again by one
// warp over the visible keys alone: two passes (maximum; weights and sums), plain fp32,
// eight keys at a time; writes values [from, to).  (Every such row done again, whoever's
// the NaN, took 340 ms for a 2048-token chunk whose second half is NaN; now 0.6.)  It is
// slow where there are many: a NaN token that the ring evicts during a 2048-token chunk
// over 4096 slots makes the call 86 ms instead of 0.18, one in the middle of a 64-token
// chunk over 131072 slots 474 instead of 0.17.
template <int D, int NG>
__device__ __noinline__ void redo_row(const Params& p, const Ring& ring, int b, int h, int row, int lane, int from, int to) {
  constexpr int E = D / 32, KEYS = 8;
  if (!hidden_reached<D, NG>(p, ring, b, h, row, lane)) return;
  const int kvh = h / p.G;
  const int64_t base = (int64_t(b) * p.hkv + kvh) * p.cap;
  const int64_t at = ((int64_t(b) * p.n + row) * p.hq + h) * D + lane;
  float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) q[e] = __half2float(p.q[at + 32 * e]) * p.scale_log2, acc[e] = 0.f;
  // the ring's slots, or the chunk's keys up to the row's own
  auto keys = [&](auto of_ring, bool maximum) {
    constexpr bool OLD = decltype(of_ring)::value;
    const int end = OLD ? ring.valid : row + 1;
    auto value = [&](int which, int t, int e) {
      if constexpr (OLD)
        return ring_value<D, NG>(p, which, base + t, lane + 32 * e);
      else
        return __half2float((which == 0 ? p.kn : p.vn)[((int64_t(b) * p.n + t) * p.hkv + kvh) * D + lane + 32 * e]);
    };
#pragma unroll 1
    for (int t0 = 0; t0 < end; t0 += KEYS) {
      float x[KEYS][E], s[KEYS];
      bool seen[KEYS];
#pragma unroll
      for (int u = 0; u < KEYS; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = value(0, min(t0 + u, end - 1), e);
#pragma unroll
      for (int u = 0; u < KEYS; ++u) {
        s[u] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s[u] = fmaf(q[e], x[u][e], s[u]);
        s[u] = warp_sum(s[u]);
        seen[u] = t0 + u < end && (OLD ? ring.sees(t0 + u, row, p.sink, p.window) : ring.sees_new(t0 + u, row, p.window));
        if (maximum && seen[u]) m = fmaxf(m, s[u]);
      }
      if (maximum) continue;
#pragma unroll
      for (int u = 0; u < KEYS; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) x[u][e] = value(1, min(t0 + u, end - 1), e);
#pragma unroll
      for (int u = 0; u < KEYS; ++u) {
        const float w = seen[u] ? exp2f(s[u] - m) : 0.f;
        l += w;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = fmaf(w, seen[u] ? x[u][e] : 0.f, acc[e]);
      }
    }
  };
  for (int pass = 0; pass < 2; ++pass) {
    keys(std::true_type{}, pass == 0);
    keys(std::false_type{}, pass == 0);
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (lane + 32 * e >= from && lane + 32 * e < to) p.out[at + 32 * e] = __float2half_rn(acc[e] / l);
}

// A loader lane's share of a key tile: a quarter (c) of rows 8 pass + its own, the
// 8-value blocks 4 i + c, as 16-byte chunks of the swizzled tile.  The rows of
// a warp's store turn are four apart in pairs, so that eight lanes write eight
// different 16-byte columns.
template <int D>
__device__ __forceinline__ void put_block(unsigned char* tile, int row, int c, int i, uint4 v) {
  *reinterpret_cast<uint4*>(tile + (i >> 1) * (KT * 128) + row * 128 + (((4 * (i & 1) + c) ^ (row & 7)) << 4)) = v;
}

// A lane's codes and params of one tile of the ring's keys or values, on their way:
// loaded a tile ahead, stored as fp16 when the stage is free.
template <int D, int NG, bool VALUES>
struct RingTile {
  static constexpr int NI = D / 32, PW = NG == 4 ? 2 : 1;
  uint32_t w[PASSES][NI], pr[PASSES][PW];

  __device__ __forceinline__ void load(const Params& p, int64_t base, int k0, int valid, int warp, int lane) {
    const unsigned char* codes = VALUES ? p.vc : p.kc;
    const uint16_t* params = VALUES ? p.vp : p.kp;
    const int c = lane & 3, q = lane >> 2, r8 = (q >> 1) | ((q & 1) << 2);
#pragma unroll
    for (int s = 0; s < PASSES; ++s) {
      // a free slot reads the last valid one's row (the tile may end behind the storage): with weight 0
      // a NaN there adds nothing to what that row, in the same tile, brings already
      const int64_t row = base + min(k0 + (s * LOAD_WARPS + warp) * 8 + r8, valid - 1);
      if constexpr (NI == 4) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(codes + row * (D / 2)) + c);
        w[s][0] = v.x, w[s][1] = v.y, w[s][2] = v.z, w[s][3] = v.w;
      } else {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(codes + row * (D / 2)) + c);
        w[s][0] = v.x, w[s][1] = v.y;
      }
      if constexpr (NG == 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(params + row * NG));
        pr[s][0] = v.x, pr[s][1] = v.y;
      } else if constexpr (NG == 2) {
        pr[s][0] = __ldg(reinterpret_cast<const uint32_t*>(params + row * NG));
      } else {
        pr[s][0] = __ldg(params + row);
      }
    }
  }
  __device__ __forceinline__ void store(unsigned char* tile, int warp, int lane) const {
    const int c = lane & 3, q = lane >> 2, r8 = (q >> 1) | ((q & 1) << 2);
#pragma unroll
    for (int s = 0; s < PASSES; ++s) {
      if (s * LOAD_WARPS + warp >= GROUPS) break;
      const int row = (s * LOAD_WARPS + warp) * 8 + r8;
#pragma unroll
      for (int n = 0; n < NG; ++n) {
        const uint32_t pair = NG == 1 ? pr[s][0] * 0x10001u : prmt(pr[s][n >> 1], 0u, (n & 1) ? 0x3232u : 0x1010u);
        const kv4::GroupScale gs = kv4::group_scale(pair);
#pragma unroll
        for (int i = n * NI / NG; i < (n + 1) * NI / NG; ++i) {
          const uint32_t word = VALUES ? prmt(w[s][i >> 1], w[s][NI / 2 + (i >> 1)], (i & 1) ? 0x7632u : 0x5410u) : w[s][i];
          uint32_t o[4];
          kv4::dequant_word(word, gs, o);
          put_block<D>(tile, row, c, i, make_uint4(o[0], o[1], o[2], o[3]));
        }
      }
    }
  }
};

// one tile of the chunk's keys or values, rows past the chunk zero
template <int D>
__device__ __forceinline__ void copy_new_tile(const __half* src, int64_t first, int64_t stride, int k0, int n,
                                              uint32_t tile, int warp, int lane) {
  constexpr int LPR = D / 8;
#pragma unroll 4
  for (int r = warp * (32 / LPR) + lane / LPR; r < KT; r += LOAD_WARPS * (32 / LPR)) {
    const int ch = lane % LPR, key = k0 + r;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                     tile + (ch >> 3) * (KT * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4)),
                 "l"(src + first + min(key, n - 1) * stride + ch * 8), "r"(key < n ? 16 : 0));
  }
  asm volatile("cp.async.commit_group;");
}

template <int D, int NG>
__global__ void __launch_bounds__(THREADS, 1) prefill_attn_q4_kernel(const __grid_constant__ Params p) {
  using L = Smem<D>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sb = smem_u32(smem);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  volatile unsigned* gave_up = reinterpret_cast<volatile unsigned*>(smem + L::GAVE_UP);
  auto bar = [&](int i) { return sb + L::BARS + 8 * i; };
  if (tid == 0) {
    *gave_up = 0;
    for (int i = 0; i < STAGES; ++i) {
      bar_init(bar(FULL_K + i), LOAD_WARPS);
      bar_init(bar(EMPTY_K + i), 1);
      bar_init(bar(FULL_V + i), LOAD_WARPS);
      bar_init(bar(EMPTY_V + i), 1);
    }
    for (int x = 0; x < 2; ++x) {
      bar_init(bar(S_FULL + x), 1);
      bar_init(bar(P_FULL + x), 4);
      bar_init(bar(P_HALF + x), 4);
      bar_init(bar(PV_DONE + x), 1);
      bar_init(bar(O_FULL + x), 1);
    }
    bar_init(bar(Q_FULL), SOFTMAX_WARPS);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(sb + L::TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  // only now: a kernel launched early must not take TMEM columns that this one waits for
  pdl_trigger();
  pdl_wait();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + L::TMEM);

  const int split = blockIdx.x % p.nsplit, block = blockIdx.x / p.nsplit;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int rows = p.n * p.G, row0 = block * 2 * ROWS;
  const int last_row = min(rows, row0 + 2 * ROWS) - 1;
  const int rmin = row0 / p.G, rmax = last_row / p.G;
  const int ntile = last_row - row0 >= ROWS ? 2 : 1;  // row tiles with rows
  const Ring ring(kv4::count_of(p.counts, p.count, b), p.sink, p.window);
  Tiles& tiles = *reinterpret_cast<Tiles*>(smem + L::LIST);
  static_assert(sizeof(Tiles) <= 128, "room for the tile list");
  if (tid == 0) tiles.make(ring, rmin, rmax, p.sink, p.window);
  __syncthreads();
  const int t0 = int(int64_t(tiles.total) * split / p.nsplit), t1 = int(int64_t(tiles.total) * (split + 1) / p.nsplit);
  const int T = t1 - t0;
  // TMEM columns: S of row tile x, then its P, at 128 x; its O at 256 + D x

  if (warp >= SOFTMAX_WARP0) {
    // --------------------------------------------------------------- softmax
    const int x = (warp - SOFTMAX_WARP0) >> 2, quad = warp & 3;
    const uint32_t lanes = uint32_t(quad * 32) << 16;
    {  // this warp's 32 rows of Q, D / 8 lanes a row, eight loads in flight
      constexpr int LPR = D / 8, TURNS = LPR;
      const int ch = lane % LPR;
#pragma unroll
      for (int u0 = 0; u0 < TURNS; u0 += 8) {
        uint4 v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int row = row0 + x * ROWS + quad * 32 + (u0 + u) * (32 / LPR) + lane / LPR;
          v[u] = make_uint4(0u, 0u, 0u, 0u);
          if (row < rows) {
            const int pos = row / p.G, hg = row - pos * p.G;
            v[u] = __ldg(reinterpret_cast<const uint4*>(p.q + ((int64_t(b) * p.n + pos) * p.hq + kvh * p.G + hg) * D) + ch);
          }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int tr = quad * 32 + (u0 + u) * (32 / LPR) + lane / LPR;
          *reinterpret_cast<uint4*>(smem + L::Q + x * L::TILE + (ch >> 3) * (ROWS * 128) + tr * 128 +
                                    (((ch & 7) ^ (tr & 7)) << 4)) = v[u];
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(bar(Q_FULL));
    }
    const int row = row0 + x * ROWS + quad * 32 + lane;
    const int pos = min(row, rows - 1) / p.G, hg = min(row, rows - 1) - pos * p.G;
    const int64_t orow = (int64_t(b) * p.n + pos) * p.hq + kvh * p.G + hg;
    float m_used = -INFINITY, l = 0.f;
    const float2 scale2 = make_float2(p.scale_log2, p.scale_log2);
    if (x < ntile) {
      const uint32_t ts = tmem + KT * x + lanes, to = tmem + 2 * KT + x * D + lanes;
      Walk walk(tiles, t0);
      int lo[5], hi[5];
#pragma unroll
      for (int k = 0; k < 5; ++k) lo[k] = tiles.lo[k], hi[k] = tiles.hi[k] - KT;
      for (int it = 0; it < T; ++it) {
        const bool of_ring = walk.of_ring();
        const int k0 = walk.tile * KT;
        walk.next(tiles);
        // does every row see every key of the tile?
        const bool full = of_ring ? (k0 >= lo[0] && k0 <= hi[0]) || (k0 >= lo[1] && k0 <= hi[1]) || (k0 >= lo[2] && k0 <= hi[2])
                                  : (k0 >= lo[3] && k0 <= hi[3]) || (k0 >= lo[4] && k0 <= hi[4]);
        bar_wait(bar(S_FULL + x), it & 1, gave_up);
        fence_after();
        float v[KT];
        tmem_ld64(ts, v);
        tmem_ld64(ts + 64, v + 64);
        if (!full) {  // the keys of the tile that this row sees, a bit each
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t seen = seen_bits(p, ring, of_ring, k0, j, pos);
#pragma unroll
            for (int e = 0; e < 32; ++e) v[32 * j + e] = (seen >> e) & 1u ? v[32 * j + e] : -INFINITY;
          }
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int e = 0; e < KT; e += 2) mx[(e >> 1) & 3] = max3(mx[(e >> 1) & 3], v[e], v[e + 1]);
        const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], -INFINITY) * p.scale_log2;
        const bool grew = top > m_used + GROW;
        if (__any_sync(0xffffffffu, grew)) {
          const float m_new = fmaxf(m_used, top);
          const float mb = m_new == -INFINITY ? 0.f : m_new;
          const float alpha = ex2(m_used - mb);
          m_used = m_new;
          l *= alpha;
          if (it > 0) {  // P V of the tile before has ended: this S was computed after it
            float o[16];
#pragma unroll 1
            for (int j = 0; j < D; j += 16) {
              tmem_ld16(to + j, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= alpha;
              tmem_st16(to + j, o);
            }
          }
        }
        // a NaN or +infinity among the scores makes the row NaN
        const float shift = !(top < INFINITY) ? top - top : PSHIFT - (m_used == -INFINITY ? 0.f : m_used);
        const float2 shift2 = make_float2(shift, shift);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int j = 0; j < KT; j += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float2 t = fma2(make_float2(v[j + e], v[j + e + 1]), scale2, shift2);
            const float2 w = make_float2(ex2(t.x), ex2(t.y));
            sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], w);
            pk[e / 2] = pack_h2(w.x, w.y);
          }
          tmem_st16(ts + j / 2, pk);  // over S, which is in registers
          if (j == FIRST - 32) {  // the products with these keys start
            tmem_st_wait();
            fence_before();
            __syncwarp();
            if (lane == 0) bar_arrive(bar(P_HALF + x));
          }
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        tmem_st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar(P_FULL + x));
      }
      // ------------------------------------------------------------- epilogue
      if (T > 0) {
        bar_wait(bar(O_FULL + x), 0, gave_up);
        fence_after();
      }
      float v[32];
      if (p.nsplit == 1) {
        const float inv = 1.f / l;
        bool fine = true;
#pragma unroll 1
        for (int j = 0; j < D; j += 32) {
          tmem_ld32(to + j, v);
          uint32_t h[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            const float a = v[e] * inv, c = v[e + 1] * inv;
            fine = fine && fabsf(a) <= 65504.f && fabsf(c) <= 65504.f;
            h[e / 2] = pack_h2(a, c);
          }
          if (row < rows)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
              *reinterpret_cast<uint4*>(p.out + orow * D + j + 2 * e) = make_uint4(h[e], h[e + 1], h[e + 2], h[e + 3]);
        }
        // a sum that is not finite has a visible score that is not: the whole row is NaN, and is so already
        uint32_t redo = __ballot_sync(0xffffffffu, !fine && fabsf(l) < INFINITY && row < rows);
        __syncwarp();  // the rows' own lanes have stored them: what all lanes store now comes after
        for (; redo; redo &= redo - 1) {
          const int r = row0 + x * ROWS + quad * 32 + __ffs(redo) - 1;
          redo_row<D, NG>(p, ring, b, kvh * p.G + r % p.G, r / p.G, lane, 0, D);
        }
      } else {
        // a lane a row, so that a warp writes 512 bytes in a row (a row a thread, as in the result, took 2.5 us);
        // strips without rows are left out (33 tokens after 4096 slots 19.4 -> 18.7 us)
        const int64_t strip = ((int64_t(split) * p.batch + b) * p.hkv + kvh) * p.strips + block * 8 + x * 4 + quad;
        p.part_ml[strip * 32 + lane] = make_float2(m_used, l);
        if (T > 0 && row0 + x * ROWS + quad * 32 < rows) {
#pragma unroll 1
          for (int j = 0; j < D; j += 32) {
            tmem_ld32(to + j, v);
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              p.part_o[(strip * (D / 4) + (j + e) / 4) * 32 + lane] = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
          }
        }
      }
    }
  } else if (warp > 0) {
    // --------------------------------------------------------------- loaders
    const int lw = warp - 1;
    const int64_t base = (int64_t(b) * p.hkv + kvh) * p.cap;
    const int64_t first = (int64_t(b) * p.n * p.hkv + kvh) * D, stride = int64_t(p.hkv) * D;
    RingTile<D, NG, false> kr;
    RingTile<D, NG, true> vr;
    Walk walk(tiles, t0);
    bool of_ring = T > 0 && walk.of_ring();
    int k0 = walk.tile * KT;
    if (of_ring) {
      kr.load(p, base, k0, ring.valid, lw, lane);
      vr.load(p, base, k0, ring.valid, lw, lane);
    }
    auto done = [&](int b_full) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bar_arrive(bar(b_full));
    };
    for (int it = 0; it < T; ++it) {
      const int st = it % STAGES;
      unsigned char* kt = smem + L::K + st * L::TILE;
      unsigned char* vt = smem + L::V + st * L::TILE;
      walk.next(tiles);
      const bool next_ring = it + 1 < T && walk.of_ring();
      const int next = walk.tile * KT;
      if (it >= STAGES) bar_wait(bar(EMPTY_K + st), (it / STAGES - 1) & 1, gave_up);
      if (of_ring) {
        kr.store(kt, lw, lane);
        done(FULL_K + st);
        if (next_ring) kr.load(p, base, next, ring.valid, lw, lane);
        if (it >= STAGES) bar_wait(bar(EMPTY_V + st), (it / STAGES - 1) & 1, gave_up);
        vr.store(vt, lw, lane);
        done(FULL_V + st);
        if (next_ring) vr.load(p, base, next, ring.valid, lw, lane);
      } else {
        copy_new_tile<D>(p.kn, first, stride, k0, p.n, smem_u32(kt), lw, lane);
        if (it >= STAGES) bar_wait(bar(EMPTY_V + st), (it / STAGES - 1) & 1, gave_up);
        copy_new_tile<D>(p.vn, first, stride, k0, p.n, smem_u32(vt), lw, lane);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        done(FULL_K + st);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        done(FULL_V + st);
      }
      of_ring = next_ring;
      k0 = next;
    }
  } else {
    // -------------------------------------------------------------- products
    // Every value here is the warp's own: what the products' operands are made of
    // then stays in uniform registers (moved there for each product, from the
    // lanes' registers, they held the issue up: 90 clocks a product instead of 50).
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const int n = __shfl_sync(0xffffffffu, T, 0), nx = __shfl_sync(0xffffffffu, ntile, 0);
    const uint32_t q_lo = desc_lo(sb + L::Q, 16), k_lo = desc_lo(sb + L::K, 16), v_lo = desc_lo(sb + L::V, KT * 128);
    auto scores = [&](int x, int it) {  // S_x = Q_x K^T of tile it
      const uint32_t ql = q_lo + x * (L::TILE >> 4), kl = k_lo + it % STAGES * (L::TILE >> 4);
      if (elected()) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t at = ((k >> 2) * (ROWS * 128) + (k & 3) * 32) >> 4;
          mma_ss(tm + KT * x, ql + at, kl + at, idesc<KT, false>(), k != 0);
        }
        mma_commit(bar(S_FULL + x));
        if (x == nx - 1) mma_commit(bar(EMPTY_K + it % STAGES));
      }
      __syncwarp();
    };
    // O_x += P_x V of tile it, keys [from, to): 16 keys are 8 columns of P and 16 rows of V
    auto values = [&](int x, int it, auto from, auto to) {
      const uint32_t vl = v_lo + it % STAGES * (L::TILE >> 4);
      if (elected()) {
#pragma unroll
        for (int k = from.value / 16; k < to.value / 16; ++k)
          mma_ts(tm + 2 * KT + x * D, tm + KT * x + 8 * k, vl + k * (2048 >> 4), idesc<D, true>(), (it | k) != 0);
        if (to.value == KT) {
          mma_commit(bar(it + 1 < n ? PV_DONE + x : O_FULL + x));
          if (x == nx - 1) mma_commit(bar(EMPTY_V + it % STAGES));
        }
      }
      __syncwarp();
    };
    if (n > 0) {
      bar_wait(bar(Q_FULL), 0, gave_up);
      bar_wait(bar(FULL_K), 0, gave_up);
      fence_after();
      for (int x = 0; x < nx; ++x) scores(x, 0);
    }
    for (int it = 0; it < n; ++it) {
      const int st = it % STAGES, nst = (it + 1) % STAGES;
      bar_wait(bar(FULL_V + st), (it / STAGES) & 1, gave_up);
      for (int x = 0; x < nx; ++x) {
        bar_wait(bar(P_HALF + x), it & 1, gave_up);
        fence_after();
        values(x, it, std::integral_constant<int, 0>{}, std::integral_constant<int, FIRST>{});
        bar_wait(bar(P_FULL + x), it & 1, gave_up);
        fence_after();
        values(x, it, std::integral_constant<int, FIRST>{}, std::integral_constant<int, KT>{});
        if (it + 1 == n) continue;
        if (x == 0) bar_wait(bar(FULL_K + nst), ((it + 1) / STAGES) & 1, gave_up);
        // the next S overwrites P: products with different accumulators need not run in the order of their issue
        bar_wait(bar(PV_DONE + x), it & 1, gave_up);
        fence_after();
        scores(x, it + 1);
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 0) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// Joins the splits of a strip of 32 rows, 32 of its values a block: a lane a row, a
// warp four values, AHEAD splits' loads in flight together.
template <int D, int NG, int AHEAD>
__global__ void __launch_bounds__(256) prefill_attn_q4_merge_kernel(const __grid_constant__ Params p) {
  pdl_trigger();
  pdl_wait();
  __shared__ unsigned s_redo;
  const int part = blockIdx.x % (D / 32), strip32 = blockIdx.x / (D / 32);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c4 = part * 8 + warp, kvh = blockIdx.y, b = blockIdx.z;
  const int64_t of_split = int64_t(p.batch) * p.hkv * p.strips;
  const int64_t strip = (int64_t(b) * p.hkv + kvh) * p.strips + strip32;
  if (threadIdx.x == 0) s_redo = 0;
  __syncthreads();
  const int row = strip32 * 32 + lane;
  if (row < p.n * p.G) {
    float m = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s0 = 0; s0 < p.nsplit; s0 += AHEAD) {
      float2 ml[AHEAD];
      float4 v[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const int64_t at = strip + min(s0 + i, p.nsplit - 1) * of_split;
        ml[i] = p.part_ml[at * 32 + lane];
        v[i] = p.part_o[(at * (D / 4) + c4) * 32 + lane];
        if (s0 + i >= p.nsplit) ml[i] = make_float2(-INFINITY, 0.f);
      }
      float top = m;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, ml[i].x);
      const float w0 = m == -INFINITY ? 0.f : ex2(m - top);
      m = top;
      l *= w0;
      acc.x *= w0, acc.y *= w0, acc.z *= w0, acc.w *= w0;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        if (ml[i].x == -INFINITY) {  // no key there (l is 0): its O was not written, or is void
          l += ml[i].y;              // or only scores that are NaN (l is NaN): so is the row
          continue;
        }
        const float w = ex2(ml[i].x - m);
        l = fmaf(w, ml[i].y, l);
        acc.x = fmaf(w, v[i].x, acc.x);
        acc.y = fmaf(w, v[i].y, acc.y);
        acc.z = fmaf(w, v[i].z, acc.z);
        acc.w = fmaf(w, v[i].w, acc.w);
      }
    }
    const float inv = 1.f / l;
    const float a0 = acc.x * inv, a1 = acc.y * inv, a2 = acc.z * inv, a3 = acc.w * inv;
    const int pos = row / p.G, h = kvh * p.G + row - pos * p.G;
    *reinterpret_cast<uint2*>(p.out + ((int64_t(b) * p.n + pos) * p.hq + h) * D + 4 * c4) =
        make_uint2(pack_h2(a0, a1), pack_h2(a2, a3));
    const bool fine = fabsf(a0) <= 65504.f && fabsf(a1) <= 65504.f && fabsf(a2) <= 65504.f && fabsf(a3) <= 65504.f;
    if (!fine && fabsf(l) < INFINITY) atomicOr(&s_redo, 1u << lane);  // (a sum that is not finite: the row is NaN already)
  }
  __syncthreads();
  unsigned redo = s_redo;
  if (redo == 0) return;
  const Ring ring(kv4::count_of(p.counts, p.count, b), p.sink, p.window);
  for (int i = 0; redo; redo &= redo - 1, ++i) {
    if (i % 8 != warp) continue;
    const int r = strip32 * 32 + __ffs(redo) - 1;
    redo_row<D, NG>(p, ring, b, kvh * p.G + r % p.G, r / p.G, lane, part * 32, part * 32 + 32);
  }
}

// CTAs that split the key tiles of a row block: where the row blocks leave SMs
// idle, as many as fill them with two tiles each, where there are that many (33 tokens
// after 4096 slots, 33 tiles: 17 CTAs 19.4 us, 16 CTAs, one of them with three tiles, 20.3).
// Tiles of what the ring can hold, not of what it holds, so that host and device counts
// sum in the same order: a wide ring's first 33 tokens take 13.3 us, of which 3.8 are
// splits without a tile (9.5 in a ring of 128 slots).
inline int splits(int batch, int n, int G, int kv_heads, int sink, int window) {
  const int64_t ctas = (int64_t(n) * G + 2 * ROWS - 1) / (2 * ROWS) * kv_heads * batch;
  const int64_t tiles = (kv4::capacity(sink, window) + KT - 1) / KT + (n + KT - 1) / KT, most = (tiles + 1) / 2;
  return int(std::max<int64_t>(1, std::min<int64_t>({device_sm_count() / ctas, most, MAX_SPLITS})));
}
inline int strips_of(int n, int G) { return (n * G + 2 * ROWS - 1) / (2 * ROWS) * 8; }
inline size_t workspace_for(int batch, int n, int G, int kv_heads, int head_dim, int nsplit) {
  return nsplit == 1 ? 0
                     : size_t(nsplit) * batch * kv_heads * strips_of(n, G) * 32 * (size_t(head_dim) * sizeof(float) + sizeof(float2));
}

template <int D, int NG>
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
      const cudaError_t a = cudaFuncSetAttribute(prefill_attn_q4_kernel<D, NG>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 Smem<D>::BYTES);
      if (a != cudaSuccess) return a;
      done[dev] = true;
    }
  }
  const int blocks = (p.n * p.G + 2 * ROWS - 1) / (2 * ROWS);
  const cudaError_t e = launch_pdl(prefill_attn_q4_kernel<D, NG>, dim3(unsigned(blocks * p.nsplit), unsigned(p.hkv), unsigned(p.batch)),
                                   dim3(THREADS), Smem<D>::BYTES, st, p);
  if (e != cudaSuccess || p.nsplit == 1) return e;
  // all splits' loads at once where that is few enough (past the last one they are loaded again for nothing: 2 splits
  // 22.3 us for the call with room for 2, 23.7 with 8; 17 splits 17.7 with 18, 18.7 with 8)
  const dim3 grid(unsigned((p.n * p.G + 31) / 32 * (D / 32)), unsigned(p.hkv), unsigned(p.batch));
  if (p.nsplit <= 2) return launch_pdl(prefill_attn_q4_merge_kernel<D, NG, 2>, grid, dim3(256), 0, st, p);
  if (p.nsplit <= 6) return launch_pdl(prefill_attn_q4_merge_kernel<D, NG, 6>, grid, dim3(256), 0, st, p);
  return launch_pdl(prefill_attn_q4_merge_kernel<D, NG, 18>, grid, dim3(256), 0, st, p);
}

}  // namespace pattn4

int prefill4_device_error(unsigned* code, int reset) {
  QX_CUDA_TRY(cudaMemcpyFromSymbol(code, pattn4::g_prefill4_error, sizeof(unsigned)), "get_device_error: read");
  if (reset) {
    const unsigned zero = 0;
    QX_CUDA_TRY(cudaMemcpyToSymbol(pattn4::g_prefill4_error, &zero, sizeof(unsigned)), "get_device_error: reset");
  }
  return QX_OK;
}

}  // namespace qx

using namespace qx;

extern "C" size_t qx_prefill_attention_q4_workspace_size(int batch, int n, int q_heads, int kv_heads, int head_dim,
                                                         int sink, int window) {
  if (batch <= 0 || n <= 0 || n >= (1 << 26) || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads ||
      q_heads / kv_heads > 16 || (head_dim != 64 && head_dim != 128) || sink < 0 || window < 1 ||
      kv4::capacity(sink, window) >= (int64_t(1) << 30))
    return 0;
  return pattn4::workspace_for(batch, n, q_heads / kv_heads, kv_heads, head_dim,
                               pattn4::splits(batch, n, q_heads / kv_heads, kv_heads, sink, window));
}

extern "C" int qx_prefill_attention_q4(const void* q, const void* k_new, const void* v_new, const void* k_codes,
                                       const void* k_params, const void* v_codes, const void* v_params, void* out,
                                       int batch, int n, int q_heads, int kv_heads, int head_dim, int group, int sink,
                                       int window, int64_t count, const int64_t* counts, float softmax_scale,
                                       void* workspace, size_t workspace_bytes, qx_stream_t stream) {
  const int rc = kv4::check_ring("prefill_attention_q4", batch, kv_heads, head_dim, group, sink, window);
  if (rc != QX_OK) return rc;
  QX_REQUIRE(n >= 0 && q_heads > 0 && q_heads % kv_heads == 0 && q_heads / kv_heads <= 16,
             "prefill_attention_q4: bad sizes n=%d heads q=%d kv=%d (a group of 1 to 16)", n, q_heads, kv_heads);
  QX_REQUIRE(batch <= 65535 && kv_heads <= 65535 && n < (1 << 26), "prefill_attention_q4: batch, heads or chunk too large");
  QX_REQUIRE(counts || kv4::count_fits(count), "prefill_attention_q4: count=%lld", (long long)count);
  if (batch == 0 || n == 0) return QX_OK;
  QX_REQUIRE(q && k_new && v_new && k_codes && k_params && v_codes && v_params && out,
             "prefill_attention_q4: null pointer");
  QX_REQUIRE(aligned(q, 16) && aligned(k_new, 16) && aligned(v_new, 16) && aligned(k_codes, 16) &&
                 aligned(v_codes, 16) && aligned(k_params, 16) && aligned(v_params, 16) && aligned(out, 16),
             "prefill_attention_q4: tensors must be 16-byte aligned");
  const int nsplit = pattn4::splits(batch, n, q_heads / kv_heads, kv_heads, sink, window);
  const size_t need = pattn4::workspace_for(batch, n, q_heads / kv_heads, kv_heads, head_dim, nsplit);
  if (need && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(QX_ERR_WORKSPACE, "prefill_attention_q4: workspace needs %zu bytes, 16-byte aligned", need);
  pattn4::Params p{};
  p.q = static_cast<const __half*>(q);
  p.kn = static_cast<const __half*>(k_new);
  p.vn = static_cast<const __half*>(v_new);
  p.kc = static_cast<const unsigned char*>(k_codes);
  p.kp = static_cast<const uint16_t*>(k_params);
  p.vc = static_cast<const unsigned char*>(v_codes);
  p.vp = static_cast<const uint16_t*>(v_params);
  p.out = static_cast<__half*>(out);
  p.part_o = static_cast<float4*>(workspace);
  p.strips = pattn4::strips_of(n, q_heads / kv_heads);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + int64_t(nsplit) * batch * kv_heads * p.strips * 32 * (head_dim / 4));
  p.counts = counts;
  p.count = count;
  p.cap = kv4::capacity(sink, window);
  p.batch = batch;
  p.n = n;
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
    e = group == 32 ? pattn4::launch<64, 2>(p, st) : pattn4::launch<64, 1>(p, st);
  else
    e = group == 32   ? pattn4::launch<128, 4>(p, st)
        : group == 64 ? pattn4::launch<128, 2>(p, st)
                      : pattn4::launch<128, 1>(p, st);
  QX_CUDA_TRY(e, "prefill_attention_q4: launch");
  return check_launch("prefill_attention_q4");
}
