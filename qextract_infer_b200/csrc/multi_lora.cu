// Low-rank adapters of many requests beside a shared projection: sequence b has the
// adapter a = adapters[b] of n (outside 0 .. n - 1: none), and every token of it
//   out = fp16( y + scales[a] (x A[a]) B[a] )
// with y the shared projection's output, A fp16 [n][K][P r] and B fp16 [n][r][N].  The
// columns are P blocks (the parts of a fused projection: q | k | v, gate | up); block j
// takes the ranks j r .. j r + r - 1 of A.
//
// Sequences with the same adapter are a group, and their tokens in order are the
// group's rows.  A cluster of 8 CTAs takes a chunk of a group's rows: 8 rows where
// sequences have few tokens (a decode step), 32 or 64 else (a prompt).  Nothing is sorted or
// prepared: the cluster of sequence b counts the sequences before it that share its
// adapter, which says whether a chunk starts in b, and looks up those after it that
// fill the chunk; clusters without a chunk end at once.  The group's weights are read
// once a cluster, and each of the 8 CTAs reads an eighth of them: it multiplies an eighth
// of K (its part of A), the partial h = x A meet through distributed shared memory, and
// then it does an eighth of the columns (its part of B).
//
// A row's result depends on no other row: the sums are split in the same way wherever a
// row stands.  Where there are few chunks, several clusters take one: each reads all of A
// and makes h, then does its share of the columns.
#include <algorithm>
#include <mutex>

#include "qx_b200.h"
#include "qx_common.cuh"

namespace qx {
namespace mlora {

constexpr int C = 8;  // CTAs of a cluster
constexpr int MAX_PARTS = 4;
constexpr int MAX_RANKS = 256;  // P r
constexpr int MAX_BATCH = 32768;  // a cluster looks through the sequences before its own
constexpr int MAX_SMEM = 225 * 1024;  // dynamic; the rest of 227 KB for the static arrays

struct Params {
  const __half *y, *x, *A, *B;
  const int64_t* adapters;
  const float* scales;
  __half* out;
  int batch, tokens, K, N, rank, ranks, n, parts;
  int edge[MAX_PARTS + 1];  // first column of each block, then N
  int chunks;               // chunks that may start in a sequence
  int fan;                  // clusters of a chunk: each makes h, and does its share of the columns
  int k_slice, k_step;      // K of a CTA, and of one of its steps (multiples of 16)
  int width;                // columns of a CTA
  int a_pitch;              // bytes of a staged row of A: an odd number of 16-byte units
  unsigned test_waits;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// 16 bytes, or zeros where `ok` is false
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// Sticky device-side error word of this file's kernels (QX_DEVERR_* bits), merged into
// qx_get_device_error.
static __device__ unsigned g_lora_error = 0;

__device__ __forceinline__ void bar_init(uint32_t bar) {  // one arrival, that of bar_expect
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\nfence.mbarrier_init.release.cluster;" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// the adapter of sequence b, -1 where it has none
__device__ __forceinline__ int64_t adapter_of(const Params& p, int b, bool fresh) {
  const int64_t a = fresh ? __ldcg(p.adapters + b) : p.adapters[b];
  return a >= 0 && a < p.n ? a : -1;
}

// The chunk of ROWS rows that cluster (b, j) takes of its group.  With `guess` it is found
// while the kernel before may still be writing the adapters: find() reads them, the loads
// of weights that follow from them start, and after the wait for that kernel ask_again()
// reads them once more; changed() compares, behind the work that hides these loads and
// before anything leaves the CTA.  If it says so, find() and all after it is done again.
// Whatever find() reads, its results are the same in all threads, and its rows and adapter
// exist.  (When it was chosen: a launch of one token 5.3 us so, 6.9 with the wait first, 4.9 if the second
// look is left out; of 32 tokens with an adapter each 11.7, 13.2 and 11.0.)
template <int ROWS, int THREADS>
struct Chunk {
  int64_t a;       // the adapter, -1: none
  int n;           // rows, 0: no chunk
  bool settled;    // the kernel before has ended
  unsigned seen;   // a bit for each of up to 32 steps of THREADS sequences: this thread's one has the adapter
  int end;         // sequences looked at
  int64_t again;   // this thread's one of the first step, read again
  bool differs;    // of the others

  __device__ __forceinline__ Chunk(const Params& p, bool guess) : settled(!guess || p.batch > 32 * THREADS) {
    if (settled) pdl_wait();
  }
  __device__ __forceinline__ bool any() const { return n > 0 && a >= 0; }

  // rows: row indexes into x, y and out
  __device__ __forceinline__ void find(const Params& p, int b, int j, int (&rows)[ROWS]) {
    constexpr int WARPS = THREADS / 32;
    __shared__ int s_seq[ROWS + 1], s_count[WARPS];
    __shared__ int64_t s_adapter;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, T = p.tokens;
    const int need = (ROWS - 1) / T + 2;  // sequences that a chunk can reach into, at most ROWS + 1
    const int64_t mine = adapter_of(p, b, settled);
    int before = 0, found = 0, i = 0;
    seen = 0;
    for (; i < p.batch && (i <= b || found < need); i += THREADS) {
      const int q = i + tid;
      const bool same = q < p.batch && (q == b || adapter_of(p, q, settled) == mine);
      if (q == b) s_adapter = mine;
      seen = seen << 1 | same;
      const unsigned after = __ballot_sync(0xffffffffu, same && q >= b);
      if (lane == 0) s_count[warp] = __popc(after);
      before += __syncthreads_count(same && q < b);
      int at = found;
      for (int w = 0; w < WARPS; ++w) {
        if (w == warp && same && q >= b) {
          const int n = at + __popc(after & ((1u << lane) - 1));
          if (n < need) s_seq[n] = q;
        }
        at += s_count[w];
      }
      found = at;
      __syncthreads();
    }
    end = i;
    a = s_adapter;
    const int64_t first = (int64_t(before) * T + ROWS - 1) / ROWS * ROWS + int64_t(j) * ROWS;
    const int64_t here = first - int64_t(before) * T;  // of sequence b's tokens
    n = here >= T ? 0 : int(min(int64_t(ROWS), int64_t(min(found, need)) * T - here));
    if (tid < ROWS && n > 0) {
      const int g = int(here) + min(tid, n - 1);
      rows[tid] = s_seq[g / T] * T + g % T;
    }
    __syncthreads();
  }
  __device__ __forceinline__ void ask_again(const Params& p) {
    if (settled) return;
    const int tid = threadIdx.x;
    if (tid < p.batch) again = __ldcg(p.adapters + tid);
    differs = false;
    for (int i = end - THREADS, step = 0; i > 0; i -= THREADS, ++step)
      differs |= (i + tid < p.batch && adapter_of(p, i + tid, true) == a) != bool(seen >> step & 1);
  }
  __device__ __forceinline__ bool changed(const Params& p) {  // a barrier
    const bool same = int(threadIdx.x) < p.batch && (again >= 0 && again < p.n ? again : -1) == a;
    const bool then = seen >> (end / THREADS - 1) & 1;
    const bool now = __syncthreads_or(!settled && (differs || same != then));
    settled = true;
    return now;
  }
};

// the column block that a column is in
__device__ __forceinline__ int part_of(const Params& p, int column) {
  int part = 0;
#pragma unroll
  for (int i = 1; i < MAX_PARTS; ++i) part += i < p.parts && column >= p.edge[i];
  return part;
}

// ---------------------------------------------------------------- few tokens --
// 8 rows a chunk.  h^T [P r][8] = A^T x^T by mma.sync with A as the 16-row operand (its
// rows are the ranks) and the chunk's rows as the 8 columns: an instruction covers
// 16 ranks x 16 of K for every row.  Then thread by thread 4 columns of a row in fp32.
// Bound by the weights' bytes where every row has its own adapter, else by the chain of
// latencies: adapters, A, x, the exchange, y.  Measured: one token of 4096 x 6144, 3 x 16
// ranks, 5.3 us (its bytes alone 0.1); 32 tokens with an adapter each, 4096 x 24576, 2 x 16
// ranks, 10.9 us, 3.4 TB/s (5.2); there the two phases' loads take turns, as A's place takes
// B's second step: all of B ahead leaves an SM one CTA; asked into L2 ahead, or by bulk copies, it took 7 % more.
namespace few {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int ROWS = 8;
constexpr int A_BYTES = 25600;   // a step's rows of A
constexpr int B_BYTES = 32768;   // a step's columns of B
constexpr int MAX_STEP = 512;    // K of a step

struct Layout {
  int a, a_step, x, x_step, b[2], part, recv, h, done, total;  // byte offsets, bytes of a buffer
  int x_pitch, steps, a_shift, b_shift;  // a row of A in 2^a_shift threads; a step of B has 2^b_shift 4-column pieces
};
__host__ __device__ inline int log2_up(int v) {
  int s = 0;
  while (1 << s < v) ++s;
  return s;
}
inline Layout layout(const Params& p) {
  Layout l;
  l.steps = (p.k_slice + p.k_step - 1) / p.k_step;
  l.x_pitch = p.k_step * 2 + 16;
  l.a_shift = log2_up(p.ranks / 8);
  l.b_shift = std::min(log2_up(B_BYTES / (8 * p.rank) + 1) - 1, log2_up(p.width / 4));  // the largest that fits and is of use
  const int buffers = l.steps > 1 ? 2 : 1;
  int at = 0;
  l.a = at, l.a_step = p.k_step * p.a_pitch + 16;  // + 16: the last tile of 16 ranks may end past the last row
  // when h is done, A's place takes every other step of B
  l.b[1] = at, at += buffers * l.a_step > B_BYTES ? buffers * l.a_step : B_BYTES;
  l.b[0] = at, at += B_BYTES;
  l.x = at, l.x_step = ROWS * l.x_pitch, at += buffers * l.x_step;
  l.part = at, at += 8 * 16 * ROWS * 4 > p.ranks * ROWS * 4 ? 8 * 16 * ROWS * 4 : p.ranks * ROWS * 4;
  l.recv = at, at += C * p.ranks * ROWS * 4;
  l.h = at, at += p.ranks * ROWS * 4;
  l.done = at, at += 16;
  l.total = at;
  return l;
}

__global__ void __launch_bounds__(THREADS, 2) multi_lora_rows_kernel(const __grid_constant__ Params p,
                                                                     const __grid_constant__ Layout l) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int rows[ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % C, cluster = blockIdx.x / C, chunk = cluster / p.fan;
  const int cut = (cluster - chunk * p.fan) * C + rank;  // of the columns
  const int b = chunk / p.chunks;
  pdl_trigger();
  const uint32_t base = smem_u32(smem);
  if (tid == 0) {
    bar_init(base + l.done);
    bar_expect(base + l.done, C * p.ranks * ROWS * 4);
  }
  cluster_arrive();
  // The first columns of B are asked for at once by a few clusters, by more of them behind x, so that the
  // products do not wait for B's bytes too (when it was chosen, us, B first / behind, rank 16, K 4096: one token, 6144
  // columns 5.3 / 5.6; 32 tokens with an adapter each, 4096 columns 9.8 / 9.1, 8192 9.4 / 8.7, 24576 11.6 / 11.4).
  const bool late = gridDim.x > 8 * C;
  Chunk<ROWS, THREADS> at(p, true);
  // this CTA's columns, and its part of K
  const int n0 = min(p.N, cut * p.width), n1 = min(p.N, n0 + p.width);
  const int k0 = rank * p.k_slice, k_end = min(p.K, k0 + p.k_slice);
  const int units = p.ranks / 8;  // 16-byte units of a row of A
  auto load_a = [&](int step) {
    const int c = tid & ((1 << l.a_shift) - 1);
    if (step >= l.steps || c >= units) return;
    int kk = tid >> l.a_shift;
    const int k = k0 + step * p.k_step;
    uint32_t to = base + l.a + (step & 1) * l.a_step + kk * p.a_pitch + c * 16;
    const __half* from = p.A + (at.a * p.K + k + kk) * p.ranks + c * 8;
    const int down = THREADS >> l.a_shift;
    for (; kk < p.k_step; kk += down) {
      const bool ok = k + kk < k_end;
      copy16(to, ok ? from : p.A, ok);
      to += down * p.a_pitch;
      from += down * p.ranks;
    }
  };
  auto load_x = [&](int step) {  // a warp a row
    if (step >= l.steps) return;
    const int k = k0 + step * p.k_step;
    const uint32_t to = base + l.x + (step & 1) * l.x_step + warp * l.x_pitch;
    const __half* from = p.x + int64_t(rows[warp]) * p.K + k;
    for (int c = lane * 8; c < p.k_step; c += 256) {
      const bool ok = warp < at.n && k + c < k_end;
      copy16(to + c * 2, ok ? from + c : p.x, ok);
    }
  };
  const int columns = 4 << l.b_shift;  // of a step of B
  auto load_b = [&](int step) {
    const int eighths = l.b_shift - 1;  // log2 of 8-column pieces
    const int c = tid & ((1 << eighths) - 1), column = n0 + step * columns + c * 8;
    if (column >= n1) return;
    int j = tid >> eighths;
    uint32_t to = base + l.b[step & 1] + (j * columns + c * 8) * 2;
    const __half* from = p.B + (at.a * p.rank + j) * p.N + column;
    const int down = THREADS >> eighths;  // (a step has at most 256 pieces of 8: its ranks are 8 or more)
    for (; j < p.rank; j += down) {
      copy16(to, from, true);
      to += down * columns * 2;
      from += int64_t(down) * p.N;
    }
  };
  // a warp's tiles of 16 ranks, and which of the 16-wide steps along K are its own
  const int tiles = (p.ranks + 15) / 16;
  const int shares = tiles == 1 ? 8 : tiles == 2 ? 4 : tiles <= 4 ? 2 : 1;
  const int g = lane >> 2, q = lane & 3;
  float* const part = reinterpret_cast<float*>(smem + l.part);  // [share][ranks][8]
  float scale = 0.f;
  for (;;) {
    at.find(p, b, chunk - b * p.chunks, rows);
    // (loops, not copies: each instruction here is fetched for one use)
#pragma unroll 1
    for (int when = 0; when < 2; ++when) {
      if (when == 1) pdl_wait();
      if (at.any()) {
#pragma unroll 1
        for (int step = 0; step < 2; ++step) {
          if (when == 0) {
            load_a(step);
          } else {
            load_x(step);
            copy_commit();
          }
        }
        if (late == (when == 1)) load_b(0);
      }
      copy_commit();
    }
    at.ask_again(p);
    if (at.any()) {
      scale = __ldcg(p.scales + at.a);
      float acc[2][4] = {};
      for (int step = 0; step < l.steps; ++step) {
        if (step < 2) copy_wait<2>();  // all but the next step and B
        else copy_wait<1>();
        __syncthreads();
        const uint32_t as = base + l.a + (step & 1) * l.a_step, xs = base + l.x + (step & 1) * l.x_step;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int item = warp + WARPS * i, tile = item % tiles, share = item / tiles;
          if (share < shares) {
            // matrices: (k 0-7, ranks 0-7), (k 0-7, ranks 8-15), (k 8-15, ranks 0-7), (k 8-15, ranks 8-15)
            const uint32_t at = as + ((lane & 7) + 8 * (lane >> 4)) * p.a_pitch + tile * 32 + ((lane >> 3) & 1) * 16;
            const uint32_t xt = xs + g * l.x_pitch + q * 4;
            for (int k = share * 16; k < p.k_step; k += shares * 16) {
              uint32_t w[4];
              ldsm4_t(w, at + k * p.a_pitch);
              mma_16816(acc[i], w[0], w[1], w[2], w[3], lds32(xt + k * 2), lds32(xt + k * 2 + 16));
            }
          }
        }
        __syncthreads();
        if (step + 2 < l.steps) {
          load_a(step + 2);
          load_x(step + 2);
        }
        copy_commit();
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int item = warp + WARPS * i, tile = item % tiles, share = item / tiles;
        const int j = tile * 16 + g;
        if (share < shares) {
          float* to = part + (share * p.ranks + j) * ROWS + 2 * q;
          if (j < p.ranks) *reinterpret_cast<float2*>(to) = make_float2(acc[i][0], acc[i][1]);
          if (j + 8 < p.ranks) *reinterpret_cast<float2*>(to + 8 * ROWS) = make_float2(acc[i][2], acc[i][3]);
        }
      }
    }
    if (!at.changed(p)) break;
    copy_wait<0>();
    __syncthreads();
  }
  const int n = at.n;
  cluster_wait();  // every CTA has started
  if (n == 0) return;  // (every CTA of the cluster)
  if (at.a < 0) {      // no adapter: the rows as they are
    if (p.out == p.y) return;
    for (int m = 0; m < n; ++m) {
      const int64_t row = int64_t(rows[m]) * p.N;
      for (int c = n0 + 8 * tid; c < n1; c += 8 * THREADS)
        *reinterpret_cast<uint4*>(p.out + row + c) = __ldcg(reinterpret_cast<const uint4*>(p.y + row + c));
    }
    return;
  }
  // a step of B that has landed stays where it is; the next takes A's place
  const int b_steps = (n1 - n0 + columns - 1) / columns;
  load_b(1);
  copy_commit();
  // this CTA's partial h to every CTA: thread (4 values, CTA)
  for (int i = tid; i < p.ranks * 2 * C; i += THREADS) {
    const int v = i / C, r = i % C;
    float4 sum = reinterpret_cast<const float4*>(part)[v];
    for (int s = 1; s < shares; ++s) {
      const float4 o = reinterpret_cast<const float4*>(part)[s * p.ranks * 2 + v];
      sum.x += o.x, sum.y += o.y, sum.z += o.z, sum.w += o.w;
    }
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                     at_rank(base + l.recv + (rank * p.ranks * 2 + v) * 16, r)),
                 "f"(sum.x), "f"(sum.y), "f"(sum.z), "f"(sum.w), "r"(at_rank(base + l.done, r))
                 : "memory");
  }
  // thread's first piece of the columns: item (row, 4 columns) of a step
  auto read_y = [&](int step, int item) {
    const int m = item >> l.b_shift, c = n0 + step * columns + (item & ((1 << l.b_shift) - 1)) * 4;
    return m < n && c < n1 ? __ldcg(reinterpret_cast<const uint2*>(p.y + int64_t(rows[m]) * p.N + c)) : make_uint2(0u, 0u);
  };
  uint2 y = read_y(0, tid);
  const bool have_sums = exchange_wait(base + l.done, p.test_waits, 0, rank, &g_lora_error);
  float* const h = reinterpret_cast<float*>(smem + l.h);  // [ranks][8]
  {
    const float* recv = reinterpret_cast<const float*>(smem + l.recv);
    for (int i = tid; i < p.ranks * ROWS; i += THREADS) {
      float sum = 0.f;
#pragma unroll
      for (int r = 0; r < C; ++r) sum += recv[r * p.ranks * ROWS + i];
      h[i] = scale * sum;
    }
  }

  if (__syncthreads_or(!have_sums)) {  // out stays unwritten
    cluster_leave_late();
    return;
  }
  for (int step = 0; step < b_steps; ++step) {
    copy_wait<1>();
    __syncthreads();
    const __half* const w = reinterpret_cast<const __half*>(smem + l.b[step & 1]);
    const int items = n << l.b_shift;
    for (int i = tid; i < items; i += THREADS) {
      const uint2 yv = y;
      y = i + THREADS < items ? read_y(step, i + THREADS) : read_y(step + 1, tid);
      const int m = i >> l.b_shift, c = (i & ((1 << l.b_shift) - 1)) * 4, column = n0 + step * columns + c;
      if (column >= n1) continue;
      const float* hm = h + part_of(p, column) * p.rank * ROWS + m;
      const __half* wc = w + c;
      float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll 8
      for (int j = 0; j < p.rank; ++j) {
        const uint2 bw = *reinterpret_cast<const uint2*>(wc);
        const float2 b01 = h2_to_f2(bw.x), b23 = h2_to_f2(bw.y);
        const float hv = hm[j * ROWS];
        s0 = fmaf(hv, b01.x, s0);
        s1 = fmaf(hv, b01.y, s1);
        s2 = fmaf(hv, b23.x, s2);
        s3 = fmaf(hv, b23.y, s3);
        wc += columns;
      }
      const float2 y01 = h2_to_f2(yv.x), y23 = h2_to_f2(yv.y);
      const __half2 o01 = __floats2half2_rn(y01.x + s0, y01.y + s1), o23 = __floats2half2_rn(y23.x + s2, y23.y + s3);
      *reinterpret_cast<uint2*>(p.out + int64_t(rows[m]) * p.N + column) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&o01), *reinterpret_cast<const uint32_t*>(&o23));
    }
    if (step + 2 < b_steps) {
      __syncthreads();
      load_b(step + 2);
    }
    copy_commit();
  }
}

}  // namespace few

// ------------------------------------------------------------------- a prompt --
// 64 rows a chunk, 32 where that leaves an SM a CTA.  h = x A by mma.sync (a warp: 32 rows,
// a quarter of each step of 64 along K, of 32-row chunks half of the ranks), 64 ranks at a
// time.  CTA i of the cluster adds the partial sums of its eighth of the rows and gives them
// to all as the sum of two fp16 numbers, high (rounded towards zero) and low, of h 2^-e with e
// from the row's largest of that column block: 21 bits (2^-32 of the largest at least) over any fp32
// range, and a second product instead of a rounding of h to 11 bits.  Both have h's sign, and neither
// is zero where h is not: beside an infinity of B the two products are the same infinity (a zero, or a
// low part of the other sign, would make it NaN).  Then a warp takes 32 columns at a time for all rows; the y of the next
// one or two blocks of columns is on its way into shared memory meanwhile (a lane's own
// 16-byte pieces, refilled as they are used).  Within the 32 columns the product's columns
// stand in the order in which a thread gets 8 neighbouring ones, so y and out move 16 bytes
// a lane.
//
// Measured: 2048 tokens of 12288 x 4096, 64 ranks, 37.6 us, 2.3 TB/s (its bytes alone 12.4).
// Of a CTA's 64K cycles h takes 31K (its loads alone 26K: A comes from L2 for each chunk;
// its products alone 17K, 12K of them the rate of mma.sync), waiting for the cluster's
// slowest CTA 9K (256 CTAs on 148 SMs), the columns 12K.  Chunks of 128 rows leave an SM one
// CTA, and of 16 such clusters 15 run at once: 72 us.  999 tokens of 2560 x 9728, 8 ranks:
// 15.9 us, 2.8 TB/s (6.7): launch, five steps along K, the two exchanges, then the columns.
//
// It launches nothing early: with the next call's clusters waiting on the SMs a 2048-token
// chunk took 55.7 us instead of 40.6.  Two CTAs an SM: of clusters of 8 with an SM a CTA
// only 15 run at once.
namespace many {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int STEP = 64;         // K of a step
constexpr int X_PITCH = STEP * 2 + 16;
constexpr int RANKS = 64;        // ranks of a pass over x, and of a step over a block's ranks
constexpr int STAGES = 5;        // steps in the ring
constexpr int GROUP = WARPS;     // 32-column blocks that are staged together
enum Exchange { SUMS, LOW_RANK, EXCHANGES };

// blocks of columns whose y is on its way, by the ranks of a column block
__host__ __device__ constexpr int blocks_ahead(int ranks) { return ranks <= 32 ? 2 : ranks <= 64 ? 1 : 0; }

struct Layout {
  int stage, b_pitch, b_rows, y, recv, hi, lo, h_pitch, factor, done, total;
  int padded;  // ranks of a column block, in whole steps of 16
};
__host__ __device__ inline Layout layout(const Params& p, int ROWS) {
  Layout l;
  l.padded = (p.rank + 15) / 16 * 16;
  l.stage = (ROWS * X_PITCH + STEP * p.a_pitch + 16 + 127) / 128 * 128;
  // the ring of steps; when it is empty, in its place: first the quarters' partial sums, then B's
  // columns, and behind either the low-rank values, which the other CTAs send only when they
  // have this one's sums and so when the ring is empty
  const int here = p.ranks < RANKS ? p.ranks : RANKS;
  const int meet = 4 * ROWS * (here + 4) * 4;
  l.b_pitch = GROUP * 64 + 16;
  l.b_rows = l.padded < RANKS ? l.padded : RANKS;
  // (up to 64 ranks: B of as many blocks of columns as y is ahead, read into registers at
  // once; more: two pieces of B, y as it is needed)
  const int ahead = blocks_ahead(l.padded);
  l.y = (ahead ? ahead : 2) * l.b_rows * l.b_pitch;
  const int b_bytes = l.y + ahead * WARPS * ROWS * 64;
  l.h_pitch = p.parts * l.padded * 2 + 16;
  l.hi = meet > b_bytes ? meet : b_bytes;
  l.lo = l.hi + ROWS * l.h_pitch;
  int at = l.lo + ROWS * l.h_pitch;
  if (STAGES * l.stage > at) at = STAGES * l.stage;
  l.recv = at, at += ROWS * p.ranks * 4;
  l.factor = at, at += ROWS * MAX_PARTS * 4;
  l.done = at, at += EXCHANGES * 8;
  l.total = at;
  return l;
}
// Two values as (high, low) halves; `plain`: within +-2^10, else (a row with an infinity or NaN) only those count
__device__ __forceinline__ void split(float v0, float v1, float down, bool plain, uint32_t& hi, uint32_t& lo) {
  const float s0 = plain ? v0 * down : isfinite(v0) ? 0.f : v0, s1 = plain ? v1 * down : isfinite(v1) ? 0.f : v1;
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(s1), "f"(s0));
  const float2 back = h2_to_f2(hi);
  const __half2 rest = __floats2half2_rn(plain ? s0 - back.x : s0, plain ? s1 - back.y : s1);
  lo = *reinterpret_cast<const uint32_t*>(&rest);
  // what is not zero is at least the smallest number of its sign in both
  const uint32_t sign = (__float_as_uint(v0) >> 16 & 0x8000u) | (__float_as_uint(v1) & 0x80000000u);
  if (v0 != 0.f) {
    if (!(hi & 0x7FFFu)) hi |= (sign & 0x8000u) | 1u;
    if (!(lo & 0x7FFFu)) lo |= (sign & 0x8000u) | 1u;
  }
  if (v1 != 0.f) {
    if (!(hi & 0x7FFF0000u)) hi |= (sign & 0x80000000u) | 0x10000u;
    if (!(lo & 0x7FFF0000u)) lo |= (sign & 0x80000000u) | 0x10000u;
  }
}
// KS: a column block's ranks in steps of 16 (1, 2, up to 4): its B stays in registers for all
// row tiles.  0: more than 64 ranks, 64 at a time, the sums of 64 rows in registers
template <int KS, int ROWS>
__global__ void __launch_bounds__(THREADS, 2) multi_lora_tile_kernel(const __grid_constant__ Params p) {
  constexpr int PAIRS = ROWS / 32, UNITS = RANKS / 8 * PAIRS / 2;  // 32-row tiles; units of 8 ranks that a warp multiplies
  constexpr int OWN = ROWS / C;                                   // rows that this CTA adds up
  constexpr int BLOCK_BYTES = ROWS * 64;                          // of y: the rows of a block of 32 columns
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int rows[ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, q = lane & 3;
  const int rank = blockIdx.x % C, cluster = blockIdx.x / C, chunk = cluster / p.fan;
  const int cut = (cluster - chunk * p.fan) * C + rank;  // of the columns
  const int b = chunk / p.chunks;
  const Layout l = layout(p, ROWS);
  const uint32_t base = smem_u32(smem);
  if (tid == 0) {
    bar_init(base + l.done + 8 * SUMS);
    bar_init(base + l.done + 8 * LOW_RANK);
    bar_expect(base + l.done + 8 * SUMS, C * OWN * p.ranks * 4);
    bar_expect(base + l.done + 8 * LOW_RANK, ROWS * p.parts * (l.padded * 4 + 4));
  }
  __syncthreads();
  cluster_arrive();
  Chunk<ROWS, THREADS> at(p, false);
  at.find(p, b, chunk - b * p.chunks, rows);
  const int n = at.n;
  const int64_t a = at.a;
  if (n == 0 || a < 0) {  // (every CTA of the cluster)
    cluster_wait();
    if (n == 0 || p.out == p.y) return;
    // no adapter: the rows as they are
    const int n0 = min(p.N, cut * p.width), n1 = min(p.N, n0 + p.width);
    for (int m = warp; m < n; m += WARPS) {
      const int64_t row = int64_t(rows[m]) * p.N;
      for (int c = n0 + 8 * lane; c < n1; c += 8 * 32)
        *reinterpret_cast<uint4*>(p.out + row + c) = __ldcg(reinterpret_cast<const uint4*>(p.y + row + c));
    }
    return;
  }
  const float scale = __ldcg(p.scales + a);

  // ---- h of this CTA's part of K
  const int k0 = min(p.K, rank * p.k_slice), k1 = min(p.K, k0 + p.k_slice);
  const int steps = (k1 - k0 + STEP - 1) / STEP;
  // rows 32 pair .. + 31, K 16 quarter .. + 15 of a step, ranks 8 unit .. of a pass
  const int pair = warp % PAIRS, quarter = warp / PAIRS % 4, unit = warp / (4 * PAIRS) * UNITS;
  bool started = false;
  for (int j0 = 0; j0 < p.ranks; j0 += RANKS) {
    const int here = min(RANKS, p.ranks - j0), units = here / 8;
    // a thread's 16-byte pieces of x's and of A's part of a step: from, to, and the first K that
    // they need to exist
    const __half *from_x[PAIRS], *from_a[2];
    uint32_t to_x[PAIRS], to_a[2];
    int at_x[PAIRS], at_a[2];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const int m = (tid >> 3) + 32 * i, c = tid & 7;
      from_x[i] = p.x + int64_t(rows[m]) * p.K + k0 + 8 * c;
      to_x[i] = base + m * X_PITCH + c * 16;
      at_x[i] = m < n ? k0 + 8 * c : 1 << 30;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int id = tid + THREADS * i, kk = id / units, u = id - kk * units;
      from_a[i] = p.A + (a * p.K + k0 + kk) * p.ranks + j0 + 8 * u;
      to_a[i] = base + ROWS * X_PITCH + kk * p.a_pitch + u * 16;
      at_a[i] = kk < STEP ? k0 + kk : -1;
    }
    auto load = [&](int step) {
      if (step < steps) {
        const uint32_t stage = step % STAGES * l.stage;
        const int k = step * STEP;
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
          const bool ok = at_x[i] + k < k1;
          copy16(to_x[i] + stage, ok ? from_x[i] + k : p.x, ok);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (at_a[i] >= 0) {
            const bool ok = at_a[i] + k < k1;
            copy16(to_a[i] + stage, ok ? from_a[i] + int64_t(k) * p.ranks : p.A, ok);
          }
      }
      copy_commit();
    };
    float acc[2][UNITS][4] = {};
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load(s);
    for (int step = 0; step < steps; ++step) {
      copy_wait<STAGES - 2>();
      __syncthreads();
      load(step + STAGES - 1);
      const uint32_t xs = base + step % STAGES * l.stage, as = xs + ROWS * X_PITCH;
      uint32_t xv[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        ldsm4(xv[i], xs + (pair * 32 + i * 16 + (lane & 15)) * X_PITCH + quarter * 32 + (lane >> 4) * 16);
      // two units of 8 ranks a load (past the last unit: what the ring holds there, not used)
#pragma unroll
      for (int t = 0; t < UNITS; t += 2)
        if (unit + t < units) {
          uint32_t w[4];
          ldsm4_t(w, as + (quarter * 16 + (lane & 15)) * p.a_pitch + (unit + t + (lane >> 4)) * 16);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            mma_16816(acc[i][t], xv[i][0], xv[i][1], xv[i][2], xv[i][3], w[0], w[1]);
            if (unit + t + 1 < units) mma_16816(acc[i][t + 1], xv[i][0], xv[i][1], xv[i][2], xv[i][3], w[2], w[3]);
          }
        }
    }
    copy_wait<0>();
    __syncthreads();  // nobody reads the ring any more: the four quarters meet in it
    float* const meet = reinterpret_cast<float*>(smem);  // [quarter][rows][here + 4]
    const int pitch = here + 4;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int t = 0; t < UNITS; ++t)
        if (unit + t < units) {
          float* to = meet + (quarter * ROWS + pair * 32 + i * 16 + g) * pitch + (unit + t) * 8 + 2 * q;
          *reinterpret_cast<float2*>(to) = make_float2(acc[i][t][0], acc[i][t][1]);
          *reinterpret_cast<float2*>(to + 8 * pitch) = make_float2(acc[i][t][2], acc[i][t][3]);
        }
    if (!started) cluster_wait();  // every CTA has started
    started = true;
    __syncthreads();
    for (int i = tid; i < ROWS * (here / 4); i += THREADS) {  // 4 ranks of a row, to the CTA that adds the row up
      const int m = i / (here / 4), j = (i - m * (here / 4)) * 4;
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float4*>(meet + (k * ROWS + m) * pitch + j);
      asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
                       at_rank(base + l.recv + ((rank * OWN + m % OWN) * p.ranks + j0 + j) * 4, m / OWN)),
                   "f"(v[0].x + v[1].x + v[2].x + v[3].x), "f"(v[0].y + v[1].y + v[2].y + v[3].y),
                   "f"(v[0].z + v[1].z + v[2].z + v[3].z), "f"(v[0].w + v[1].w + v[2].w + v[3].w),
                   "r"(at_rank(base + l.done + 8 * SUMS, m / OWN))
                   : "memory");
    }
    __syncthreads();  // the ring is free
  }
  // ---- this CTA's columns: its share of the 32-column blocks (a block is of one part)
  int total = 0;
  for (int i = 0; i < p.parts; ++i) total += (p.edge[i + 1] - p.edge[i] + 31) / 32;
  const int first = int(int64_t(total) * cut / (C * p.fan)), last = int(int64_t(total) * (cut + 1) / (C * p.fan));
  const int groups = (last - first + GROUP - 1) / GROUP;
  // this warp's block of a group: its part, first column and number of columns (0: none)
  struct Block {
    int part, column, columns;
  };
  auto block_of = [&](int group) {
    int block = first + group * GROUP + warp;
    Block at = {0, 0, 0};
    if (block < last) {
      for (;; ++at.part) {
        const int here = (p.edge[at.part + 1] - p.edge[at.part] + 31) / 32;
        if (block < here) break;
        block -= here;
      }
      at.column = p.edge[at.part] + block * 32;
      at.columns = min(32, p.edge[at.part + 1] - at.column);
    }
    return at;
  };
  const int pieces = KS ? 1 : (l.padded + RANKS - 1) / RANKS;  // of a block's ranks
  auto load_b = [&](int step, int buffer) {  // a warp loads the block that it multiplies
    const Block at = block_of(step / pieces);
    if (at.columns > 0) {
      const int j0 = step % pieces * RANKS, j = lane >> 2, c = lane & 3;
      const bool ok = c * 8 < at.columns;
      uint32_t to = base + buffer * l.b_rows * l.b_pitch + warp * 64 + j * l.b_pitch + c * 16;
      const __half* from = p.B + (a * p.rank + j0 + j) * p.N + at.column + c * 8;
      const int64_t down = int64_t(8) * p.N;
      for (int i = j; i < min(RANKS, l.padded - j0); i += 8) {
        const bool exists = ok && j0 + i < p.rank;
        copy16(to, exists ? from : p.B, exists);
        to += 8 * l.b_pitch;
        from += down;
      }
    }
  };
  // lane (g, q): columns column + 8 q .. + 7 of rows 16 t + g and + 8; in shared memory a lane's
  // pieces are a run of the warp's
  constexpr int AHEAD = blocks_ahead(KS * 16);
  constexpr int TILES = ROWS / 16;  // of a block, a commit each
  auto ask_y = [&](const Block& at, int t, int buffer) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int m = t * 16 + e * 8 + g;
      if (8 * q < at.columns && m < n)
        copy16(base + l.y + (buffer * WARPS + warp) * BLOCK_BYTES + ((t * 2 + e) * 32 + lane) * 16,
               p.y + int64_t(rows[m]) * p.N + at.column + 8 * q, true);
    }
  };
  if constexpr (KS > 0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const Block at = block_of(i);
      load_b(i, i);
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        ask_y(at, t, i);
        copy_commit();
      }
    }
  } else {
    load_b(0, 0);
    copy_commit();
    load_b(1, 1);
    copy_commit();
  }
  auto have = [&](int exchange) {
    return exchange_wait(base + l.done + 8 * exchange, p.test_waits, exchange, rank, &g_lora_error);
  };
  if (!have(SUMS)) {  // the partial sums of this CTA's rows; out stays unwritten (no barrier of the CTA lies behind)
    cluster_leave_late();
    return;
  }

  // ---- add them up: a warp a row, a lane 4 ranks
  for (int own = warp; own < OWN; own += WARPS) {
    const float* recv = reinterpret_cast<const float*>(smem + l.recv) + own * p.ranks;
    const int m = rank * OWN + own;
    for (int part = 0; part < p.parts; ++part) {
      float v[MAX_RANKS / 128][4];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < MAX_RANKS / 128; ++i) {
        const int j = 4 * lane + 128 * i;
        v[i][0] = v[i][1] = v[i][2] = v[i][3] = 0.f;
        if (j < p.rank) {
#pragma unroll
          for (int r = 0; r < C; ++r) {
            const float4 o = *reinterpret_cast<const float4*>(recv + r * OWN * p.ranks + part * p.rank + j);
            v[i][0] += o.x, v[i][1] += o.y, v[i][2] += o.z, v[i][3] += o.w;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) top = fmaxf(top, isfinite(v[i][k]) ? fabsf(v[i][k]) : INFINITY);
        }
      }
      top = warp_max(top);
      const bool finite = isfinite(top);
      // 2^e with top 2^-e in [2^9, 2^10); a row with an infinity or NaN keeps only those
      const int e = finite ? max(int(__float_as_uint(top) >> 23) - 127 - 9, -100) : 0;
      const float down = __uint_as_float(uint32_t(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < MAX_RANKS / 128; ++i) {
        const int j = 4 * lane + 128 * i;
        if (j < l.padded) {
          uint32_t hi[2], lo[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) split(v[i][2 * k], v[i][2 * k + 1], down, finite, hi[k], lo[k]);
          const uint32_t at = m * l.h_pitch + (part * l.padded + j) * 2;
#pragma unroll
          for (int r = 0; r < C; ++r) {
            const uint32_t done = at_rank(base + l.done + 8 * LOW_RANK, r);
            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(
                             at_rank(base + l.hi + at, r)),
                         "r"(hi[0]), "r"(hi[1]), "r"(done)
                         : "memory");
            asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(
                             at_rank(base + l.lo + at, r)),
                         "r"(lo[0]), "r"(lo[1]), "r"(done)
                         : "memory");
          }
        }
      }
      if (lane < C)
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(
                         at_rank(base + l.factor + (m * MAX_PARTS + part) * 4, lane)),
                     "r"(__float_as_uint(scale * __uint_as_float(uint32_t(127 + e) << 23))),
                     "r"(at_rank(base + l.done + 8 * LOW_RANK, lane))
                     : "memory");
    }
  }
  if (!have(LOW_RANK)) {
    cluster_leave_late();
    return;
  }

  // ---- the columns
  const float* const factor = reinterpret_cast<const float*>(smem + l.factor);
  auto write = [&](const Block& at, int t, int e, const uint4& yv, const float (&acc)[4][4]) {
    const int m = t * 16 + e * 8 + g;
    const float f = factor[m * MAX_PARTS + at.part];
    const uint32_t yd[4] = {yv.x, yv.y, yv.z, yv.w};
    uint32_t od[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 yf = h2_to_f2(yd[i]);
      const __half2 o = __floats2half2_rn(fmaf(f, acc[i][2 * e], yf.x), fmaf(f, acc[i][2 * e + 1], yf.y));
      od[i] = *reinterpret_cast<const uint32_t*>(&o);
    }
    *reinterpret_cast<uint4*>(p.out + int64_t(rows[m]) * p.N + at.column + 8 * q) = make_uint4(od[0], od[1], od[2], od[3]);
  };
  // B's fragments of 16 ranks: product column g of tile i is column 8 (g / 2) + 2 i + g % 2 of the block
  auto weights = [&](uint32_t bs, int k, uint32_t (&w)[4][2]) {
    const uint32_t sel = g & 1 ? 0x7632u : 0x5410u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t at = bs + (k * 16 + 2 * q) * l.b_pitch + (8 * (g >> 1) + 2 * i) * 2;  // a pair of columns
      w[i][0] = prmt(lds32(at), lds32(at + l.b_pitch), sel);
      w[i][1] = prmt(lds32(at + 8 * l.b_pitch), lds32(at + 9 * l.b_pitch), sel);
    }
  };
  // 16 rows x 16 ranks (from rank `j`, padded, of all) x 32 columns
  auto multiply = [&](int t, int j, const uint32_t (&w)[4][2], float (&acc)[4][4]) {
    const uint32_t at = (t * 16 + (lane & 15)) * l.h_pitch + (j + 8 * (lane >> 4)) * 2;
    uint32_t hi[4], lo[4];
    ldsm4(hi, base + l.hi + at);
    ldsm4(lo, base + l.lo + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      mma_16816(acc[i], hi[0], hi[1], hi[2], hi[3], w[i][0], w[i][1]);
      mma_16816(acc[i], lo[0], lo[1], lo[2], lo[3], w[i][0], w[i][1]);
    }
  };
  for (int group = 0; group < groups; ++group) {
    const Block now = block_of(group);
    const bool mine = 8 * q < now.columns;
    if constexpr (KS > 0) {
      const Block later = block_of(group + AHEAD);
      const int buffer = AHEAD == 1 ? 0 : group & 1;
      // AHEAD blocks of commits are on their way behind the one that is waited for
      copy_wait<TILES * AHEAD - 1>();
      __syncwarp();
      const int ks = l.padded / 16;
      uint32_t w[KS > 0 ? KS : 1][4][2];
      if (now.columns > 0)
#pragma unroll
        for (int k = 0; k < KS; ++k)
          if (k < ks) weights(base + buffer * l.b_rows * l.b_pitch + warp * 64, k, w[k]);
      __syncwarp();
      load_b(group + AHEAD, buffer);
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        copy_wait<TILES * AHEAD - 1>();  // a lane reads its own copies
        uint4 y[2];
#pragma unroll
        for (int e = 0; e < 2; ++e)
          y[e] = *reinterpret_cast<const uint4*>(smem + l.y + (buffer * WARPS + warp) * BLOCK_BYTES + ((t * 2 + e) * 32 + lane) * 16);
        ask_y(later, t, buffer);
        copy_commit();
        if (t * 16 < n && now.columns > 0) {
          float acc[4][4] = {};
#pragma unroll
          for (int k = 0; k < KS; ++k)
            if (k < ks) multiply(t, now.part * l.padded + k * 16, w[k], acc);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (mine && t * 16 + e * 8 + g < n) write(now, t, e, y[e], acc);
        }
      }
    } else {
      float acc[ROWS / 16][4][4] = {};
      for (int piece = 0; piece < pieces; ++piece) {
        const int step = group * pieces + piece;
        copy_wait<1>();
        __syncwarp();
        if (now.columns > 0)
          for (int k = 0; k < min(RANKS, l.padded - piece * RANKS) / 16; ++k) {
            uint32_t w[4][2];
            weights(base + (step & 1) * l.b_rows * l.b_pitch + warp * 64, k, w);
#pragma unroll
            for (int t = 0; t < ROWS / 16; ++t) multiply(t, now.part * l.padded + piece * RANKS + k * 16, w, acc[t]);
          }
        __syncwarp();
        load_b(step + 2, step & 1);
        copy_commit();
      }
#pragma unroll
      for (int t = 0; t < ROWS / 16; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int m = t * 16 + e * 8 + g;
          if (mine && m < n)
            write(now, t, e, __ldcg(reinterpret_cast<const uint4*>(p.y + int64_t(rows[m]) * p.N + now.column + 8 * q)), acc[t]);
        }
    }
  }
}

}  // namespace many

// whether two runs of memory share a byte
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
  return p < q + uintptr_t(b_bytes) && q < p + uintptr_t(a_bytes);
}

// Clusters of a chunk: doubled while a CTA has more than `columns` columns, up to 8 and up to
// `at_once` in all.  Measured (rank 16, K 4096, 24576 columns, us by 1 / 8 clusters a chunk): 8
// tokens 15.9 / 6.0, 16 tokens 20.0 / 9.6, 128 tokens 23.3 / 13.1; one token and 6144 columns: 4.9
// with 1, 5.0 with 2, 5.1 with 4.  The chunks counted are those that may start.  Sequences that share an
// adapter make fewer, and those are not spread: 8 sequences of one token on one adapter take 16.2 us, with an adapter
// each 6.8; 32 on one 19.2, on 4 21.7, with an adapter each 10.9; 64 on 1, 2 or 4 26.
void spread(Params& p, int columns, int at_once) {
  p.fan = 1;
  while (p.fan < 8 && int64_t(p.batch) * p.chunks * p.fan * 2 <= at_once && p.N / (C * p.fan) > columns) p.fan *= 2;
  p.width = ((p.N + C * p.fan - 1) / (C * p.fan) + 7) / 8 * 8;
}

// In all: of the tile kernel those that run at once on a B200 (148 SMs, clusters of 8 CTAs within a GPC) where two
// CTAs fit an SM, and where one does: 33 chunks of 32 rows take 15.7 us, 34 26.2 (rank 8, 2560 x 9728); 15 of
// 3 x 64 ranks 35.2 us, 16 67.9.  Of the other 8: with more, a decode step's next projection, which streams its weights
// meanwhile, finds its SMs taken (the decoder's tok/s with 8 sequences and 8 / 16 / 32 clusters a
// call: 1848 / 1811 / 1759; 16 sequences and 16 / 32: 2470 / 2334; one sequence and 1 / 8: 364 / 368).
constexpr int AT_ONCE_BY_TWO = 33, AT_ONCE = 15, AT_ONCE_FEW = 8;
constexpr int HALF_SMEM = 115000;  // dynamic shared memory of which an SM has room for two

// C CTAs for every cluster of every chunk that may start in a sequence
template <typename... Args>
int launch(void (*kernel)(Args...), int threads, const Params& p, int smem, cudaStream_t st, Args... args) {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  QX_CUDA_TRY(cudaGetDevice(&dev), "multi_lora_add: cudaGetDevice");
  QX_REQUIRE(dev >= 0 && dev < 64, "multi_lora_add: device index %d unsupported", dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!done[dev]) {
      using namespace many;
      const char* what = "multi_lora_add: set smem limit";
      constexpr cudaFuncAttribute limit = cudaFuncAttributeMaxDynamicSharedMemorySize;
      QX_CUDA_TRY(cudaFuncSetAttribute(few::multi_lora_rows_kernel, limit, MAX_SMEM), what);
      for (auto k : {multi_lora_tile_kernel<0, 64>, multi_lora_tile_kernel<1, 64>, multi_lora_tile_kernel<2, 64>,
                     multi_lora_tile_kernel<4, 64>, multi_lora_tile_kernel<1, 32>, multi_lora_tile_kernel<2, 32>,
                     multi_lora_tile_kernel<4, 32>})
        QX_CUDA_TRY(cudaFuncSetAttribute(k, limit, MAX_SMEM), what);
      done[dev] = true;
    }
  }
  QX_REQUIRE(smem <= MAX_SMEM, "multi_lora_add: %d bytes of shared memory needed", smem);
  const int64_t ctas = int64_t(p.batch) * p.chunks * p.fan * C;
  QX_REQUIRE(ctas <= 0x7fffffffLL, "multi_lora_add: %d sequences of %d tokens are too many", p.batch, p.tokens);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = size_t(smem);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = g_pdl_enabled.load(std::memory_order_relaxed) ? 2 : 1;
  QX_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, args...), "multi_lora_add: launch");
  return check_launch("multi_lora_add");
}

// 8-row chunks, for sequences of up to FEW_TOKENS.  Where only one of their CTAs fits an SM (128
// ranks in all and more) the other kernel does them, unless a block has more than 64 ranks, which
// it takes piece by piece.  Measured (a decode step of 1 / 8 / 32 sequences with an adapter each,
// us here / there): 3 x 32 ranks and 6144 columns 8.8 / 12.6, 9.9 / 16.9, 20 / 21.8; 2 x 64
// and 24576 12.5 / 14.2, 24 / 23.7, 73 / 43.5; 2 x 128 26.5 / 34.9, 60.5 / 84, 182 / 245.
constexpr int FEW_TOKENS = 8;

bool plan_few(Params& p, few::Layout* l) {
  using namespace few;
  if (p.tokens > FEW_TOKENS) return false;
  p.chunks = (p.tokens + ROWS - 1) / ROWS;
  const int most = std::min(MAX_STEP, A_BYTES / p.a_pitch / 16 * 16);
  const int steps = (p.k_slice + most - 1) / most;
  p.k_step = ((p.k_slice + steps - 1) / steps + 15) / 16 * 16;
  const int columns = 1024 / int(std::min<int64_t>(ROWS, int64_t(p.batch) * p.tokens));
  spread(p, columns, AT_ONCE_FEW);
  *l = layout(p);
  return l->total <= HALF_SMEM || p.rank > many::RANKS;
}

// Up to SMALL_ROWS rows in all, chunks of 32 rows where they take no more waves of clusters than chunks of 64
// (each sequence counted by itself).  Measured, us by 32 / 64 (2560 x 9728 rank 8 | 4096 x 24576 rank 16 | 12288 x
// 4096 rank 64): one sequence of 320 tokens 11.2 / 12.6 | 18.3 / 19.0 | 20.9 / 22.7, of 1056 15.7 / 21.9 | 29.1 / 43.7
// | 25.6 / 36.4, of 1088 26.2 / 22.0 | 47.3 / 43.7 | 40.2 / 36.5; 100 of 10 tokens with an adapter each 48.2 / 57.7 | 83.7 /
// 100.4 | 79.8 / 106.0, with one 27.4 / 27.3 | 42.4 / 47.7 | 39.1 / 41.8; 20 of 40 with an adapter each 25.8 / 19.8 | 44.4 / 37.2 |
// 40.0 / 33.9.  With more rows sequences that share adapters fill chunks of 64: 48 of 32 tokens, 8 adapters, 29.9 / 25.0 |
// 54.8 / 46.6 | 47.4 / 39.7.
constexpr int SMALL_ROWS = 1152;

// waves of the tile kernel's clusters with chunks of `rows`
int64_t waves(const Params& p, int rows) {
  const int64_t chunks = int64_t(p.batch) * ((p.tokens + rows - 1) / rows);
  const int at_once = many::layout(p, rows).total > HALF_SMEM ? AT_ONCE : AT_ONCE_BY_TWO;
  return (chunks + at_once - 1) / at_once;
}

int launch_many(Params& p, cudaStream_t st) {
  using namespace many;
  const int ks = (p.rank + 15) / 16;
  const int here = std::min(RANKS, p.ranks);
  p.a_pitch = here * 2 + (here / 8 % 2 ? 0 : 16);
  const bool small = int64_t(p.batch) * p.tokens <= SMALL_ROWS && ks <= 4;
  const int rows = small && waves(p, 32) <= waves(p, 64) ? 32 : 64;
  p.chunks = (p.tokens + rows - 1) / rows;
  const int smem = layout(p, rows).total;
  spread(p, 256, smem > HALF_SMEM ? AT_ONCE : AT_ONCE_BY_TWO);
  void (*kernel)(Params);
  if (rows == 32)
    kernel = ks == 1 ? multi_lora_tile_kernel<1, 32> : ks == 2 ? multi_lora_tile_kernel<2, 32> : multi_lora_tile_kernel<4, 32>;
  else
    kernel = ks == 1   ? multi_lora_tile_kernel<1, 64>
             : ks == 2 ? multi_lora_tile_kernel<2, 64>
             : ks <= 4 ? multi_lora_tile_kernel<4, 64>
                       : multi_lora_tile_kernel<0, 64>;
  return launch(kernel, THREADS, p, smem, st, p);
}

}  // namespace mlora

int lora_device_error(unsigned* code, int reset) {
  QX_CUDA_TRY(cudaMemcpyFromSymbol(code, mlora::g_lora_error, sizeof(unsigned)), "get_device_error: read");
  if (reset) {
    const unsigned zero = 0;
    QX_CUDA_TRY(cudaMemcpyToSymbol(mlora::g_lora_error, &zero, sizeof(unsigned)), "get_device_error: reset");
  }
  return QX_OK;
}

}  // namespace qx

using namespace qx;

extern "C" int qx_multi_lora_add(const void* y, const void* x, const void* lora_A, const void* lora_B,
                                 const int64_t* adapters, const float* scales, void* out, int batch, int tokens, int K,
                                 int N, int rank, int num_adapters, const int* splits, int num_splits,
                                 qx_stream_t stream) {
  using namespace mlora;
  QX_REQUIRE(batch >= 0 && tokens >= 0 && K > 0 && N > 0 && num_adapters >= 0,
             "multi_lora_add: bad sizes batch=%d tokens=%d K=%d N=%d adapters=%d", batch, tokens, K, N, num_adapters);
  QX_REQUIRE(batch <= MAX_BATCH, "multi_lora_add: batch=%d is above %d (rows of one adapter go together as [batch, tokens])",
             batch, MAX_BATCH);
  QX_REQUIRE(K % 8 == 0 && N % 8 == 0 && K <= 1 << 30 && N <= 1 << 30,
             "multi_lora_add: K=%d and N=%d must be multiples of 8 and at most 2^30", K, N);
  QX_REQUIRE(num_splits >= 0 && num_splits <= MAX_PARTS && (num_splits == 0 || splits),
             "multi_lora_add: %d column blocks (at most %d)", num_splits, MAX_PARTS);
  Params p{};
  p.parts = num_splits ? num_splits : 1;
  QX_REQUIRE(rank >= 8 && rank % 8 == 0 && rank <= MAX_RANKS / p.parts,
             "multi_lora_add: rank=%d must be a multiple of 8 and at most %d for %d column blocks", rank, MAX_RANKS / p.parts,
             p.parts);
  int64_t at = 0;
  for (int j = 0; j < p.parts; ++j) {
    const int width = num_splits ? splits[j] : N;
    QX_REQUIRE(width > 0 && width % 8 == 0, "multi_lora_add: a block of %d columns (a multiple of 8 needed)", width);
    at += width;
    QX_REQUIRE(at <= N, "multi_lora_add: the column blocks exceed N=%d", N);
    p.edge[j + 1] = int(at);
  }
  QX_REQUIRE(at == N, "multi_lora_add: the column blocks cover %lld of N=%d columns", (long long)at, N);
  const int64_t rows = int64_t(batch) * tokens;
  QX_REQUIRE(rows <= 0x7fffffffLL, "multi_lora_add: %lld rows are too many", (long long)rows);
  if (rows == 0) return QX_OK;
  QX_REQUIRE(y && x && adapters && out, "multi_lora_add: null pointer");
  QX_REQUIRE(num_adapters == 0 || (lora_A && lora_B && scales), "multi_lora_add: null pointer");
  QX_REQUIRE(aligned(y, 16) && aligned(x, 16) && aligned(lora_A, 16) && aligned(lora_B, 16) && aligned(out, 16) &&
                 aligned(adapters, 8) && aligned(scales, 4),
             "multi_lora_add: y, x, lora_A, lora_B and out must be 16-byte aligned");
  const int64_t n_out = rows * N * 2;
  QX_REQUIRE((out == y || !overlap(out, n_out, y, n_out)) && !overlap(out, n_out, x, rows * K * 2) &&
                 !overlap(out, n_out, lora_A, int64_t(num_adapters) * K * rank * p.parts * 2) &&
                 !overlap(out, n_out, lora_B, int64_t(num_adapters) * rank * N * 2) &&
                 !overlap(out, n_out, adapters, int64_t(batch) * 8) && !overlap(out, n_out, scales, int64_t(num_adapters) * 4),
             "multi_lora_add: out may be y, and must not overlap anything else");
  p.y = static_cast<const __half*>(y);
  p.x = static_cast<const __half*>(x);
  p.A = static_cast<const __half*>(lora_A);
  p.B = static_cast<const __half*>(lora_B);
  p.adapters = adapters;
  p.scales = scales;
  p.out = static_cast<__half*>(out);
  p.batch = batch;
  p.tokens = tokens;
  p.K = K;
  p.N = N;
  p.rank = rank;
  p.ranks = rank * p.parts;
  p.n = num_adapters;
  p.test_waits = g_test_waits.load(std::memory_order_relaxed);
  p.a_pitch = p.ranks * 2 + (p.ranks / 8 % 2 ? 0 : 16);
  p.k_slice = ((K + C - 1) / C + 15) / 16 * 16;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  few::Layout l;
  if (plan_few(p, &l)) return launch(few::multi_lora_rows_kernel, few::THREADS, p, l.total, st, p, l);
  return launch_many(p, st);
}
