// Low-rank adapters of many requests beside a shared projection: sequence b has the
// adapter a = adapters[b] of n (outside 0 .. n - 1: none), and every token of it
//   out = fp16( y + scales[a] (x A[a]) B[a] )
// with y the shared projection's output, A fp16 [n][K][P r] and B fp16 [n][r][N].  The
// columns are P blocks (the parts of a fused projection: q | k | v, gate | up); block j
// takes the ranks j r .. j r + r - 1 of A.
//
// Sequences with the same adapter are a group, and their tokens in order are the
// group's rows.  A cluster of 8 CTAs takes a chunk of a group's rows: 8 rows where
// sequences have few tokens (a decode step), 64 else (a prompt).  Nothing is sorted or
// prepared: the cluster of sequence b counts the sequences before it that share its
// adapter, which says whether a chunk starts in b, and looks up those after it that
// fill the chunk; clusters without a chunk end at once.  The group's weights are read
// once a chunk, and each of the 8 CTAs reads an eighth of them: it multiplies an eighth
// of K (its part of A), the partial h = x A meet through distributed shared memory, and
// then it does an eighth of the columns (its part of B).
//
// A row's result depends on no other row: the sums are split in the same way wherever a
// row stands.  Everything that does not come from the kernel before (adapters, A, B,
// scales) is requested before the wait for it.
#include <algorithm>
#include <mutex>

#include "qx_b200.h"
#include "qx_common.cuh"

namespace qx {
namespace mlora {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int C = 8;  // CTAs of a cluster
constexpr int MAX_PARTS = 4;
constexpr int MAX_RANKS = 256;  // P r
constexpr int MAX_SMEM = 226 * 1024;

struct Params {
  const __half *y, *x, *A, *B;
  const int64_t* adapters;
  const float* scales;
  __half* out;
  int batch, tokens, K, N, rank, ranks, n, parts;
  int edge[MAX_PARTS + 1];  // first column of each block, then N
  int chunks;               // clusters of a sequence: the chunks that may start in it
  int k_slice, k_step;      // K of a CTA, and of one of its steps (multiples of 16)
  int a_pitch;              // bytes of a staged row of A: an odd number of 16-byte units
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
__device__ __forceinline__ void ldsm2_t(uint32_t (&r)[2], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];" : "=r"(r[0]), "=r"(r[1]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}

// the adapter of sequence b, -1 where it has none
__device__ __forceinline__ int64_t adapter_of(const Params& p, int b) {
  const int64_t a = p.adapters[b];
  return a >= 0 && a < p.n ? a : -1;
}

// The chunk of ROWS rows that cluster (b, j) takes of its group: row indexes into
// x, y and out; returns their number, 0 where it has no chunk.
template <int ROWS>
__device__ __forceinline__ int find_rows(const Params& p, int b, int j, int64_t mine, int (&rows)[ROWS]) {
  __shared__ int s_seq[ROWS + 1], s_count[WARPS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, T = p.tokens;
  const int need = (ROWS - 1) / T + 2;  // sequences that a chunk can reach into, at most ROWS + 1
  int before = 0, found = 0;
  for (int i = 0; i < p.batch && (i <= b || found < need); i += THREADS) {
    const int q = i + tid;
    const bool same = q < p.batch && adapter_of(p, q) == mine;
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
  const int64_t first = (int64_t(before) * T + ROWS - 1) / ROWS * ROWS + int64_t(j) * ROWS;
  const int64_t here = first - int64_t(before) * T;  // of sequence b's tokens
  if (here >= T) return 0;
  const int64_t n = min(int64_t(ROWS), int64_t(min(found, need)) * T - here);
  if (tid < ROWS) {
    const int g = int(here) + min(tid, int(n) - 1);
    rows[tid] = s_seq[g / T] * T + g % T;
  }
  __syncthreads();
  return int(n);
}

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
namespace few {

constexpr int ROWS = 8;
constexpr int A_BYTES = 25600;   // a step's rows of A
constexpr int B_BYTES = 16384;   // a step's columns of B
constexpr int MAX_STEP = 512;    // K of a step

struct Layout {
  int a, x, b, part, recv, h, total;  // byte offsets
  int x_pitch, b_columns, steps;
};
__host__ __device__ inline Layout layout(const Params& p) {
  Layout l;
  l.steps = (p.k_slice + p.k_step - 1) / p.k_step;
  l.x_pitch = p.k_step * 2 + 16;
  l.b_columns = B_BYTES / (2 * p.rank) / 8 * 8;
  const int buffers = l.steps > 1 ? 2 : 1;
  int at = 0;
  l.a = at, at += buffers * (p.k_step * p.a_pitch + 16);  // + 16: the last tile of 16 ranks may end past the last row
  l.x = at, at += buffers * ROWS * l.x_pitch;
  l.b = at, at += 2 * B_BYTES;
  l.part = at, at += 8 * 16 * ROWS * 4 > p.ranks * 2 * ROWS * 4 ? 8 * 16 * ROWS * 4 : p.ranks * 2 * ROWS * 4;
  l.recv = at, at += C * p.ranks * ROWS * 4;
  l.h = at, at += p.ranks * ROWS * 4;
  l.total = at;
  return l;
}

__global__ void __launch_bounds__(THREADS, 2) multi_lora_rows_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int rows[ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % C, chunk = blockIdx.x / C;
  const int b = chunk / p.chunks;
  pdl_trigger();
  const int64_t a = adapter_of(p, b);
  const int n = a < 0 && p.out == p.y ? 0 : find_rows(p, b, chunk - b * p.chunks, a, rows);
  if (n == 0) {  // (every CTA of the cluster)
    pdl_wait();
    return;
  }
  // this CTA's columns
  const int width = ((p.N + C - 1) / C + 7) / 8 * 8;
  const int n0 = min(p.N, rank * width), n1 = min(p.N, n0 + width);
  if (a < 0) {  // no adapter: the rows as they are
    pdl_wait();
    for (int m = 0; m < n; ++m) {
      const int64_t at = int64_t(rows[m]) * p.N;
      for (int c = n0 + 8 * tid; c < n1; c += 8 * THREADS)
        *reinterpret_cast<uint4*>(p.out + at + c) = __ldcg(reinterpret_cast<const uint4*>(p.y + at + c));
    }
    return;
  }
  cluster_arrive();
  const Layout l = layout(p);
  const uint32_t base = smem_u32(smem);
  const int k0 = rank * p.k_slice;
  const int units = p.ranks / 8;  // 16-byte units of a row of A
  auto load_a = [&](int step) {
    if (step >= l.steps) return;
    const uint32_t to = base + l.a + (step & 1) * (p.k_step * p.a_pitch + 16);
    const int k = k0 + step * p.k_step;
    const __half* from = p.A + (a * p.K + k) * p.ranks;
    for (int i = tid; i < p.k_step * units; i += THREADS) {
      const int kk = i / units, c = i - kk * units;
      const bool ok = k + kk < p.K && step * p.k_step + kk < p.k_slice;
      copy16(to + kk * p.a_pitch + c * 16, ok ? from + i * 8 : p.A, ok);
    }
  };
  auto load_x = [&](int step) {
    if (step >= l.steps) return;
    const uint32_t to = base + l.x + (step & 1) * ROWS * l.x_pitch;
    const int k = k0 + step * p.k_step, per_row = p.k_step / 8;
    for (int i = tid; i < ROWS * per_row; i += THREADS) {
      const int m = i / per_row, c = i - m * per_row;
      const bool ok = m < n && k + 8 * c < p.K && step * p.k_step + 8 * c < p.k_slice;
      copy16(to + m * l.x_pitch + c * 16, ok ? p.x + int64_t(rows[m]) * p.K + k + 8 * c : p.x, ok);
    }
  };
  const int b_steps = (n1 - n0 + l.b_columns - 1) / l.b_columns;
  auto load_b = [&](int step) {
    if (step >= b_steps) return;
    const uint32_t to = base + l.b + (step & 1) * B_BYTES;
    const int c0 = n0 + step * l.b_columns, per_row = min(l.b_columns, n1 - c0) / 8;
    const __half* from = p.B + a * p.rank * p.N + c0;
    for (int i = tid; i < p.rank * per_row; i += THREADS) {
      const int j = i / per_row, c = i - j * per_row;
      copy16(to + (j * l.b_columns + c * 8) * 2, from + int64_t(j) * p.N + c * 8, true);
    }
  };
  load_a(0);
  load_a(1);
  load_b(0);
  load_b(1);
  copy_commit();
  const float scale = p.scales[a];
  pdl_wait();
  load_x(0);
  copy_commit();
  load_x(1);
  copy_commit();

  // a warp's tiles of 16 ranks, and which of the 16-wide steps along K are its own
  const int tiles = (p.ranks + 15) / 16;
  const int shares = tiles == 1 ? 8 : tiles == 2 ? 4 : tiles <= 4 ? 2 : 1;
  float acc[2][4] = {};
  const int g = lane >> 2, q = lane & 3;
  for (int step = 0; step < l.steps; ++step) {
    copy_wait<1>();
    __syncthreads();
    const uint32_t as = base + l.a + (step & 1) * (p.k_step * p.a_pitch + 16), xs = base + l.x + (step & 1) * ROWS * l.x_pitch;
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
  float* const part = reinterpret_cast<float*>(smem + l.part);  // [share][ranks][8]
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
  __syncthreads();
  cluster_wait();  // every CTA has started
  // this CTA's partial h to every CTA: thread (4 values, CTA)
  for (int i = tid; i < p.ranks * 2 * C; i += THREADS) {
    const int v = i / C, r = i % C;
    float4 sum = reinterpret_cast<const float4*>(part)[v];
    for (int s = 1; s < shares; ++s) {
      const float4 o = reinterpret_cast<const float4*>(part)[s * p.ranks * 2 + v];
      sum.x += o.x, sum.y += o.y, sum.z += o.z, sum.w += o.w;
    }
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(
                     at_rank(base + l.recv + (rank * p.ranks * 2 + v) * 16, r)),
                 "f"(sum.x), "f"(sum.y), "f"(sum.z), "f"(sum.w)
                 : "memory");
  }
  cluster_arrive();
  cluster_wait();
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

  for (int step = 0; step < b_steps; ++step) {
    copy_wait<1>();
    __syncthreads();
    const __half* const w = reinterpret_cast<const __half*>(smem + l.b + (step & 1) * B_BYTES);
    const int c0 = n0 + step * l.b_columns, fours = min(l.b_columns, n1 - c0) / 4;
    for (int i = tid; i < fours * n; i += THREADS) {
      const int m = i / fours, c = (i - m * fours) * 4;
      const int64_t at = int64_t(rows[m]) * p.N + c0 + c;
      const uint2 yv = __ldcg(reinterpret_cast<const uint2*>(p.y + at));
      const float* hm = h + part_of(p, c0 + c) * p.rank * ROWS + m;
      float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll 8
      for (int j = 0; j < p.rank; ++j) {
        const uint2 bw = *reinterpret_cast<const uint2*>(w + j * l.b_columns + c);
        const float2 b01 = h2_to_f2(bw.x), b23 = h2_to_f2(bw.y);
        const float hv = hm[j * ROWS];
        s0 = fmaf(hv, b01.x, s0);
        s1 = fmaf(hv, b01.y, s1);
        s2 = fmaf(hv, b23.x, s2);
        s3 = fmaf(hv, b23.y, s3);
      }
      const float2 y01 = h2_to_f2(yv.x), y23 = h2_to_f2(yv.y);
      const __half2 o01 = __floats2half2_rn(y01.x + s0, y01.y + s1), o23 = __floats2half2_rn(y23.x + s2, y23.y + s3);
      *reinterpret_cast<uint2*>(p.out + at) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&o01), *reinterpret_cast<const uint32_t*>(&o23));
    }
    __syncthreads();
    if (step + 2 < b_steps) load_b(step + 2);
    copy_commit();
  }
}

}  // namespace few

// ------------------------------------------------------------------- a prompt --
// 64 rows a chunk.  h [64][P r] = x A by mma.sync (a warp: 16 rows, half of each step of
// 64 along K), 64 ranks at a time.  CTA i of the cluster adds the partial sums of rows
// 8 i .. 8 i + 7 and gives them to all as two fp16 numbers, high and low (22 bits), of
// h 2^-e with e from the row's largest of that column block: any fp32 range, and a
// second product instead of a rounding of h to 11 bits.  Then a warp takes 32 columns
// at a time for all 64 rows.  Within the 32 columns the product's columns stand in the
// order in which a thread gets 8 neighbouring ones, so y and out move 16 bytes a lane.
namespace many {

constexpr int ROWS = 64;
constexpr int STEP = 64;         // K of a step
constexpr int X_PITCH = STEP * 2 + 16;
constexpr int RANKS = 64;        // ranks of a pass over x, and of a step over a block's ranks
constexpr int STAGES = 3;
constexpr int GROUP = WARPS;     // 32-column blocks that are staged together

struct Layout {
  int stage, ring, b, b_pitch, b_rows, recv, hi, lo, h_pitch, factor, total;
  int padded;  // ranks of a column block, in whole steps of 16
};
__host__ __device__ inline Layout layout(const Params& p) {
  Layout l;
  l.padded = (p.rank + 15) / 16 * 16;
  l.stage = ROWS * X_PITCH + STEP * p.a_pitch + 16;
  l.stage = (l.stage + 127) / 128 * 128;
  l.ring = 0;
  l.b = 0;  // after the last step over K, B's columns take the ring's place
  l.b_pitch = GROUP * 64 + 16;
  int at = STAGES * l.stage;
  l.b_rows = l.padded < RANKS ? l.padded : RANKS;
  const int b_bytes = 2 * l.b_rows * l.b_pitch;
  if (b_bytes > at) at = b_bytes;
  l.recv = at, at += C * 8 * p.ranks * 4;
  l.h_pitch = p.parts * l.padded * 2 + 16;
  l.hi = at, at += ROWS * l.h_pitch;
  l.lo = at, at += ROWS * l.h_pitch;
  l.factor = at, at += ROWS * MAX_PARTS * 4;
  l.total = at;
  return l;
}

// KS: a column block's ranks in steps of 16 (1, 2, up to 4): its B stays in registers for the
// four row tiles.  0: more than 64 ranks, 64 at a time, the sums of the row tiles in registers
template <int KS>
__global__ void __launch_bounds__(THREADS, 2) multi_lora_tile_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int rows[ROWS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, q = lane & 3;
  const int rank = blockIdx.x % C, chunk = blockIdx.x / C;
  const int b = chunk / p.chunks;
  pdl_trigger();
  const int64_t a = adapter_of(p, b);
  const int n = a < 0 && p.out == p.y ? 0 : find_rows(p, b, chunk - b * p.chunks, a, rows);
  pdl_wait();
  if (n == 0) return;  // (every CTA of the cluster)
  if (a < 0) {         // no adapter: the rows as they are
    const int width = ((p.N + C - 1) / C + 7) / 8 * 8;
    const int n0 = min(p.N, rank * width), n1 = min(p.N, n0 + width);
    for (int m = warp; m < n; m += WARPS) {
      const int64_t at = int64_t(rows[m]) * p.N;
      for (int c = n0 + 8 * lane; c < n1; c += 8 * 32)
        *reinterpret_cast<uint4*>(p.out + at + c) = __ldcg(reinterpret_cast<const uint4*>(p.y + at + c));
    }
    return;
  }
  cluster_arrive();
  const Layout l = layout(p);
  const uint32_t base = smem_u32(smem);
  const float scale = p.scales[a];

  // ---- h of this CTA's part of K
  const int k0 = min(p.K, rank * p.k_slice), k1 = min(p.K, k0 + p.k_slice);
  const int steps = (k1 - k0 + STEP - 1) / STEP;
  const int row_tile = warp & 3, half = warp >> 2;
  bool started = false;
  for (int j0 = 0; j0 < p.ranks; j0 += RANKS) {
    const int here = min(RANKS, p.ranks - j0), units = here / 8;
    auto load = [&](int step) {
      if (step < steps) {
        const uint32_t to = base + l.ring + step % STAGES * l.stage;
        const int k = k0 + step * STEP;
        for (int i = tid; i < ROWS * (STEP / 8); i += THREADS) {
          const int m = i / (STEP / 8), c = i % (STEP / 8);
          const bool ok = m < n && k + 8 * c < k1;
          copy16(to + m * X_PITCH + c * 16, ok ? p.x + int64_t(rows[m]) * p.K + k + 8 * c : p.x, ok);
        }
        const __half* from = p.A + (a * p.K + k) * p.ranks + j0;
        for (int i = tid; i < STEP * units; i += THREADS) {
          const int kk = i / units, c = i - kk * units;
          const bool ok = k + kk < k1;
          copy16(to + ROWS * X_PITCH + kk * p.a_pitch + c * 16, ok ? from + int64_t(kk) * p.ranks + c * 8 : p.A, ok);
        }
      }
      copy_commit();
    };
    float acc[RANKS / 8][4] = {};
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load(s);
    for (int step = 0; step < steps; ++step) {
      copy_wait<STAGES - 2>();
      __syncthreads();
      load(step + STAGES - 1);
      const uint32_t xs = base + l.ring + step % STAGES * l.stage, as = xs + ROWS * X_PITCH;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int k = half * 32 + kk * 16;
        uint32_t xv[4];
        ldsm4(xv, xs + (row_tile * 16 + (lane & 15)) * X_PITCH + (k + 8 * (lane >> 4)) * 2);
#pragma unroll
        for (int t = 0; t < RANKS / 8; ++t)
          if (t < units) {
            uint32_t w[2];
            ldsm2_t(w, as + (k + (lane & 15)) * p.a_pitch + t * 16);
            mma_16816(acc[t], xv[0], xv[1], xv[2], xv[3], w[0], w[1]);
          }
      }
    }
    copy_wait<0>();
    __syncthreads();  // nobody reads the ring any more: the two halves meet in it
    float* const meet = reinterpret_cast<float*>(smem + l.ring);  // [64][64 + 4]
    if (half == 1) {
#pragma unroll
      for (int t = 0; t < RANKS / 8; ++t)
        if (t < units) {
          float* to = meet + (row_tile * 16 + g) * (RANKS + 4) + t * 8 + 2 * q;
          *reinterpret_cast<float2*>(to) = make_float2(acc[t][0], acc[t][1]);
          *reinterpret_cast<float2*>(to + 8 * (RANKS + 4)) = make_float2(acc[t][2], acc[t][3]);
        }
    }
    if (!started) cluster_wait();  // every CTA has started
    started = true;
    __syncthreads();
    if (half == 0) {  // rows 16 row_tile + g (CTA 2 row_tile) and + 8 (the next): [from][8 rows][ranks]
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t to = at_rank(base + l.recv, 2 * row_tile + e) + ((rank * 8 + g) * p.ranks + j0 + 2 * q) * 4;
        const float* other = meet + (row_tile * 16 + 8 * e + g) * (RANKS + 4) + 2 * q;
#pragma unroll
        for (int t = 0; t < RANKS / 8; ++t)
          if (t < units) {
            const float2 o = *reinterpret_cast<const float2*>(other + t * 8);
            asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to + t * 32), "f"(acc[t][2 * e] + o.x),
                         "f"(acc[t][2 * e + 1] + o.y)
                         : "memory");
          }
      }
    }
    __syncthreads();  // the ring is free
  }
  cluster_arrive();

  // ---- this CTA's columns: an eighth of the 32-column blocks (a block is of one part)
  int total = 0;
  for (int i = 0; i < p.parts; ++i) total += (p.edge[i + 1] - p.edge[i] + 31) / 32;
  const int first = int(int64_t(total) * rank / C), last = int(int64_t(total) * (rank + 1) / C);
  const int groups = (last - first + GROUP - 1) / GROUP;
  // block -> its part, first column and number of columns
  auto block_at = [&](int block, int& part, int& column, int& columns) {
    part = 0;
    for (;; ++part) {
      const int here = (p.edge[part + 1] - p.edge[part] + 31) / 32;
      if (block < here) break;
      block -= here;
    }
    column = p.edge[part] + block * 32;
    columns = min(32, p.edge[part + 1] - column);
  };
  const int pieces = KS ? 1 : (l.padded + RANKS - 1) / RANKS;  // of a block's ranks
  auto load_b = [&](int step) {  // a warp loads the block that it multiplies
    const int block = first + step / pieces * GROUP + warp, j0 = step % pieces * RANKS;
    if (block < last) {
      const uint32_t to = base + l.b + (step & 1) * l.b_rows * l.b_pitch + warp * 64;
      int part, column, columns;
      block_at(block, part, column, columns);
      const __half* from = p.B + a * p.rank * p.N + column;
      for (int i = lane; i < min(RANKS, l.padded - j0) * 4; i += 32) {
        const int j = i >> 2, c = i & 3;
        const bool ok = j0 + j < p.rank && c * 8 < columns;
        copy16(to + j * l.b_pitch + c * 16, ok ? from + int64_t(j0 + j) * p.N + c * 8 : p.B, ok);
      }
    }
    copy_commit();
  };
  load_b(0);
  load_b(1);
  cluster_wait();  // the partial sums of this CTA's 8 rows are here

  // ---- add them up: a warp a row
  {
    const float* recv = reinterpret_cast<const float*>(smem + l.recv) + warp * p.ranks;
    const int m = rank * 8 + warp;
    for (int part = 0; part < p.parts; ++part) {
      float v[MAX_RANKS / 32], top = 0.f;
#pragma unroll
      for (int i = 0; i < MAX_RANKS / 32; ++i) {
        const int j = lane + 32 * i;
        v[i] = 0.f;
        if (j < p.rank) {
#pragma unroll
          for (int r = 0; r < C; ++r) v[i] += recv[r * 8 * p.ranks + part * p.rank + j];
          top = fmaxf(top, isfinite(v[i]) ? fabsf(v[i]) : INFINITY);
        }
      }
      top = warp_max(top);
      const bool finite = isfinite(top);
      // 2^e with top 2^-e in [2^9, 2^10); a row with an infinity or NaN keeps only those
      const int e = finite ? max(int(__float_as_uint(top) >> 23) - 127 - 9, -100) : 0;
      const float down = __uint_as_float(uint32_t(127 - e) << 23);
#pragma unroll
      for (int i = 0; i < MAX_RANKS / 32; ++i) {
        const int j = lane + 32 * i;
        if (j < l.padded) {
          const float s = finite ? v[i] * down : isfinite(v[i]) ? 0.f : v[i];
          const __half hi = __float2half_rn(s);
          const __half lo = finite ? __float2half_rn(s - __half2float(hi)) : __ushort_as_half(0);
          const uint32_t at = m * l.h_pitch + (part * l.padded + j) * 2;
          for (int r = 0; r < C; ++r) {
            asm volatile("st.shared::cluster.u16 [%0], %1;" ::"r"(at_rank(base + l.hi + at, r)), "h"(__half_as_ushort(hi)) : "memory");
            asm volatile("st.shared::cluster.u16 [%0], %1;" ::"r"(at_rank(base + l.lo + at, r)), "h"(__half_as_ushort(lo)) : "memory");
          }
        }
      }
      if (lane < C)
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at_rank(base + l.factor + (m * MAX_PARTS + part) * 4, lane)),
                     "f"(scale * __uint_as_float(uint32_t(127 + e) << 23))
                     : "memory");
    }
  }
  cluster_arrive();
  cluster_wait();

  // ---- the columns
  const float* const factor = reinterpret_cast<const float*>(smem + l.factor);
  // lane (g, q): columns column + 8 q .. + 7 of rows 16 t + g and + 8
  auto read_y = [&](int t, int e, int column) {
    return __ldcg(reinterpret_cast<const uint4*>(p.y + int64_t(rows[t * 16 + e * 8 + g]) * p.N + column + 8 * q));
  };
  auto write = [&](int t, int e, int part, int column, const uint4& y, const float (&acc)[4][4]) {
    const int m = t * 16 + e * 8 + g;
    const float f = factor[m * MAX_PARTS + part];
    const uint32_t yd[4] = {y.x, y.y, y.z, y.w};
    uint32_t od[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 yf = h2_to_f2(yd[i]);
      const __half2 o = __floats2half2_rn(fmaf(f, acc[i][2 * e], yf.x), fmaf(f, acc[i][2 * e + 1], yf.y));
      od[i] = *reinterpret_cast<const uint32_t*>(&o);
    }
    *reinterpret_cast<uint4*>(p.out + int64_t(rows[m]) * p.N + column + 8 * q) = make_uint4(od[0], od[1], od[2], od[3]);
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
    const int block = first + group * GROUP + warp;
    int part = 0, column = 0, columns = 0;
    if (block < last) block_at(block, part, column, columns);
    const bool mine = 8 * q < columns;
    if constexpr (KS > 0) {
      uint4 yv[4][2];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (mine && t * 16 + e * 8 + g < n) yv[t][e] = read_y(t, e, column);
      copy_wait<1>();
      __syncwarp();
      if (columns > 0) {
        const int ks = l.padded / 16;
        uint32_t w[KS][4][2];
#pragma unroll
        for (int k = 0; k < KS; ++k)
          if (k < ks) weights(base + l.b + (group & 1) * l.b_rows * l.b_pitch + warp * 64, k, w[k]);
#pragma unroll
        for (int t = 0; t < 4; ++t)
          if (t * 16 < n) {
            float acc[4][4] = {};
#pragma unroll
            for (int k = 0; k < KS; ++k)
              if (k < ks) multiply(t, part * l.padded + k * 16, w[k], acc);
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (mine && t * 16 + e * 8 + g < n) write(t, e, part, column, yv[t][e], acc);
          }
      }
      __syncwarp();
      load_b(group + 2);
    } else {
      float acc[4][4][4] = {};
      for (int piece = 0; piece < pieces; ++piece) {
        const int step = group * pieces + piece;
        copy_wait<1>();
        __syncwarp();
        if (columns > 0)
          for (int k = 0; k < min(RANKS, l.padded - piece * RANKS) / 16; ++k) {
            uint32_t w[4][2];
            weights(base + l.b + (step & 1) * l.b_rows * l.b_pitch + warp * 64, k, w);
#pragma unroll
            for (int t = 0; t < 4; ++t) multiply(t, part * l.padded + piece * RANKS + k * 16, w, acc[t]);
          }
        __syncwarp();
        load_b(step + 2);
      }
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (mine && t * 16 + e * 8 + g < n) write(t, e, part, column, read_y(t, e, column), acc[t]);
    }
  }
}

}  // namespace many

// whether two runs of memory share a byte
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
  return p < q + uintptr_t(b_bytes) && q < p + uintptr_t(a_bytes);
}

constexpr int FEW_TOKENS = 8;  // tokens of a sequence up to which 8-row chunks do them

// one cluster of C CTAs for every chunk that may start in a sequence
int launch(void (*kernel)(Params), const Params& p, int smem, cudaStream_t st) {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  QX_CUDA_TRY(cudaGetDevice(&dev), "multi_lora_add: cudaGetDevice");
  QX_REQUIRE(dev >= 0 && dev < 64, "multi_lora_add: device index %d unsupported", dev);
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!done[dev]) {
      for (auto k : {few::multi_lora_rows_kernel, many::multi_lora_tile_kernel<0>, many::multi_lora_tile_kernel<1>,
                     many::multi_lora_tile_kernel<2>, many::multi_lora_tile_kernel<4>})
        QX_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM),
                    "multi_lora_add: set smem limit");
      done[dev] = true;
    }
  }
  QX_REQUIRE(smem <= MAX_SMEM, "multi_lora_add: %d bytes of shared memory needed", smem);
  const int64_t ctas = int64_t(p.batch) * p.chunks * C;
  QX_REQUIRE(ctas <= 0x7fffffffLL, "multi_lora_add: %d sequences of %d tokens are too many", p.batch, p.tokens);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(THREADS);
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
  QX_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p), "multi_lora_add: launch");
  return check_launch("multi_lora_add");
}

int launch_few(Params& p, cudaStream_t st) {
  using namespace few;
  p.chunks = (p.tokens + ROWS - 1) / ROWS;
  p.k_slice = ((p.K + C - 1) / C + 15) / 16 * 16;
  const int most = std::min(MAX_STEP, A_BYTES / p.a_pitch / 16 * 16);
  const int steps = (p.k_slice + most - 1) / most;
  p.k_step = ((p.k_slice + steps - 1) / steps + 15) / 16 * 16;
  return launch(multi_lora_rows_kernel, p, layout(p).total, st);
}

int launch_many(Params& p, cudaStream_t st) {
  using namespace many;
  p.chunks = (p.tokens + ROWS - 1) / ROWS;
  p.k_slice = ((p.K + C - 1) / C + 15) / 16 * 16;
  const int here = std::min(RANKS, p.ranks);
  p.a_pitch = here * 2 + (here / 8 % 2 ? 0 : 16);
  const Layout l = layout(p);
  const int ks = l.padded / 16;
  if (ks == 1) return launch(multi_lora_tile_kernel<1>, p, l.total, st);
  if (ks == 2) return launch(multi_lora_tile_kernel<2>, p, l.total, st);
  if (ks <= 4) return launch(multi_lora_tile_kernel<4>, p, l.total, st);
  return launch(multi_lora_tile_kernel<0>, p, l.total, st);
}

}  // namespace mlora
}  // namespace qx

using namespace qx;

extern "C" int qx_multi_lora_add(const void* y, const void* x, const void* lora_A, const void* lora_B,
                                 const int64_t* adapters, const float* scales, void* out, int batch, int tokens, int K,
                                 int N, int rank, int num_adapters, const int* splits, int num_splits,
                                 qx_stream_t stream) {
  using namespace mlora;
  QX_REQUIRE(batch >= 0 && tokens >= 0 && K > 0 && N > 0 && num_adapters >= 0,
             "multi_lora_add: bad sizes batch=%d tokens=%d K=%d N=%d adapters=%d", batch, tokens, K, N, num_adapters);
  QX_REQUIRE(K % 8 == 0 && N % 8 == 0, "multi_lora_add: K=%d and N=%d must be multiples of 8", K, N);
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
  p.a_pitch = p.ranks * 2 + (p.ranks / 8 % 2 ? 0 : 16);
  return tokens <= FEW_TOKENS ? launch_few(p, reinterpret_cast<cudaStream_t>(stream))
                              : launch_many(p, reinterpret_cast<cudaStream_t>(stream));
}
