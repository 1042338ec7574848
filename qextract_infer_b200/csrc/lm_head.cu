// Greedy sampling head: logits = h W (fp16 weights [H, V], V contiguous:
// this rank's vocabulary slice) and, per row, the largest logit and its index,
// in two launches instead of a library GEMV, a reduction and an index add.
//
// Kernel 1: a CTA owns 128 vocabulary columns (4 warps x 32) for every row
// (batch <= 32, one or two 16-row m-tiles).  64-row K tiles of W and of h are
// staged by cp.async (three of them: 62 KB, three CTAs an SM); W fragments come from ldmatrix.trans,
// h fragments from ldmatrix; mma.sync m16n8k16 with fp32 accumulation.  The
// logits are rounded to fp16 (the values a fp16 GEMV stores), and the CTA's
// per-row maximum with its smallest index is written to the workspace.
// Kernel 2: one warp per row reduces the CTAs' candidates in index order
// (ties go to the smallest index) and adds the slice's vocabulary offset.
//
// Whole logits (qx_lm_head_logits): kernel 1 with the fp16 values stored instead of
// compared, 32 rows a launch.
//
// Bound by the weights' bytes: 1 / 17 / 32 rows of 4096 x 151936 take 173 / 177 / 181 us (7.2 to
// 6.9 TB/s; a kernel that only reads them 173; 32 rows among calls of other kernels 189 to 200), of 4096 x 37984
// 48 / 52 / 53 (297 CTAs: one SM has three, the others two); 33 rows and more read them again, 64 rows 372.  With
// more rows a tile's own time counts: addresses that only move on, instead of each piece's own
// (198 instructions a warp and tile at 17 rows, 117 at 16), took 32 rows from 194 to 184 us; h through
// L1, where an SM's CTAs meet and not all CTAs at the same lines of L2, from 184 to 181, of the slice from
// 56.4 to 52.8.
// Measured before that for 1 / 32 rows of 4096 x 151936 and 1 row of 4096 x 37984 (us,
// tiles K x columns): 64 x 256 in two stages 189 / 222 / 59, 32 x 256 in four 208 / 238 / 66, 64 x
// 128 in two 172 / 196 / 59, in three 171 / 188 / 54 (kept), in four (two CTAs an SM) 190 / 208 /
// 63; eight warps of 16 columns 175 / 197 / 51 (48 with four).  The next kernel is let in at the end: earlier, its CTAs
// fill the slots as they come free, three on one SM and one on another (the slice: 54 us, 48 without).
#include <algorithm>
#include <mutex>

#include "qx_b200.h"
#include "qx_common.cuh"

namespace qx {
namespace lmh {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int COLS = 128;                  // vocabulary columns per CTA
constexpr int WCOLS = COLS / WARPS, NJ = WCOLS / 8;  // of a warp, in tiles of 8
constexpr int KT = 64;                     // K rows per tile
constexpr int MAXB = 32;                   // rows (two m-tiles)
constexpr int WROW = COLS * 2;             // bytes of one W tile row (256)
constexpr int W_TILE = KT * WROW;          // 16 KB
constexpr int HROW = KT * 2 + 16;          // bytes of one staged h row (+16: conflict-free ldmatrix)
constexpr int H_TILE = MAXB * HROW;        // 4.5 KB
constexpr int STAGE = W_TILE + H_TILE;
constexpr int STAGES = 3;
constexpr int SMEM = STAGES * STAGE;

struct Cand {
  float v;
  int i;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes));
}
// the same through L1: the SM's CTAs read the same rows of h at about the same time
__device__ __forceinline__ void cp_async16_l1(uint32_t dst, const void* src, int src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N));
}
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
// W tile row r (K), 16-byte chunk ch (8 columns): XOR swizzle over 8 rows
__device__ __forceinline__ uint32_t wswz(int r, int ch) {
  return uint32_t(r * WROW + ((ch ^ (r & 7)) << 4));
}
// larger value wins (never a NaN); equal values: the smaller index.  A row that is all NaN ends as (-inf,
// NOWHERE), which becomes the first index: whoever embeds the token next stays inside the vocabulary
constexpr int NOWHERE = 0x7fffffff;
__device__ __forceinline__ bool better(float v, int i, float bv, int bi) {
  return v > bv || (v == bv && i < bi);
}

// STORE: the logits go to `out` [B, V]; else the CTA's candidates to `part`
template <int MT, bool STORE>
__global__ void __launch_bounds__(THREADS) logits_kernel(const __half* __restrict__ h, const __half* __restrict__ W,
                                                        int B, int H, int V, Cand* __restrict__ part,
                                                        __half* __restrict__ out) {
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Cand s_best[WARPS][MAXB];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * COLS;
  const uint32_t sbase = smem_u32(smem);
  const int ktiles = H / KT;

  // a thread's 16-byte pieces of a tile: W rows tid / 16 + 8 i (64 x 16 pieces in all; those past V and rows past B
  // read as zero), h rows tid / 8 + 16 i (8 pieces each)
  static_assert(THREADS == COLS && THREADS == 16 * (KT / 8), "a thread's pieces stand under one another");
  const int w_col = n0 + (tid % 16) * 8, h_row = tid / 8;
  const int w_bytes = w_col < V ? 16 : 0;  // V % 8 == 0: a piece is all in or all out
  const __half* w_from = W + size_t(tid / 16) * V + (w_bytes ? w_col : 0);
  const size_t w_down = size_t(8) * V;
  const __half* h_from[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) h_from[m] = h + size_t(h_row + 16 * m < B ? h_row + 16 * m : 0) * H + (tid % 8) * 8;
  const uint32_t w_to = sbase + wswz(tid / 16, tid % 16), h_to = sbase + W_TILE + h_row * HROW + (tid % 8) * 16;
  auto issue = [&](int stage) {  // the next tile along K
    const uint32_t at = stage * STAGE;
#pragma unroll
    for (int i = 0; i < KT / 8; ++i) {
      cp_async16(w_to + at + i * 8 * WROW, w_from, w_bytes);
      w_from += w_down;
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      cp_async16_l1(h_to + at + m * 16 * HROW, h_from[m], h_row + 16 * m < B ? 16 : 0);
      h_from[m] += KT;
    }
    cp_async_commit();
  };

  float acc[MT][NJ][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[m][j][0] = acc[m][j][1] = acc[m][j][2] = acc[m][j][3] = 0.f;

  pdl_wait();  // h comes from the previous kernel
#pragma unroll
  for (int i = 0; i < STAGES; ++i) {
    if (i < ktiles) issue(i);
    else cp_async_commit();
  }
  const int mi = lane >> 3, ri = lane & 7;
  // a lane's rows of the fragments: h (rows 0-7 | 8-15) x (k 0-7 | 8-15), W (k 0-7 | 8-15) x (columns 0-7 | 8-15)
  const uint32_t a_at = sbase + W_TILE + ((mi & 1) * 8 + ri) * HROW + (mi >> 1) * 16;
  uint32_t b_at[NJ / 2];
#pragma unroll
  for (int jj = 0; jj < NJ / 2; ++jj)
    b_at[jj] = sbase + ((mi & 1) * 8 + ri) * WROW + (((warp * WCOLS + jj * 16) / 8 + (mi >> 1)) ^ ri) * 16;
  int stage = 0;
  for (int kt = 0; kt < ktiles; ++kt) {
    cp_async_wait<STAGES - 1>();
    __syncthreads();
    const uint32_t at = stage * STAGE;
#pragma unroll
    for (int ks = 0; ks < KT / 16; ++ks) {
      uint32_t a[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) ldsm_x4(a[m], a_at + at + m * 16 * HROW + ks * 32);
#pragma unroll
      for (int jj = 0; jj < NJ / 2; ++jj) {
        uint32_t bw[4];
        ldsm_x4_t(bw, b_at[jj] + at + ks * 16 * WROW);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          mma_16816(acc[m][2 * jj], a[m][0], a[m][1], a[m][2], a[m][3], bw[0], bw[1]);
          mma_16816(acc[m][2 * jj + 1], a[m][0], a[m][1], a[m][2], a[m][3], bw[2], bw[3]);
        }
      }
    }
    __syncthreads();
    if (kt + STAGES < ktiles) issue(stage);
    else cp_async_commit();
    stage = stage == STAGES - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  pdl_trigger();

  if constexpr (STORE) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int hr = 0; hr < 2; ++hr) {  // rows g and g + 8 of the m-tile
        const int row = m * 16 + g + hr * 8;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int col = n0 + warp * WCOLS + j * 8 + 2 * c;
          if (row < B && col < V)  // V % 8 == 0: both columns or none
            *reinterpret_cast<__half2*>(out + size_t(row) * V + col) =
                __floats2half2_rn(acc[m][j][hr * 2], acc[m][j][hr * 2 + 1]);
        }
      }
    return;
  }
  // per row: the fp16-rounded logits' maximum and its smallest index
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int hr = 0; hr < 2; ++hr) {  // rows g and g + 8 of the m-tile
      const int row = m * 16 + g + hr * 8;
      float bv = -INFINITY;
      int bi = NOWHERE;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int col = n0 + warp * WCOLS + j * 8 + 2 * c + e;
          const float v = __half2float(__float2half_rn(acc[m][j][hr * 2 + e]));
          if (col < V && better(v, col, bv, bi)) {
            bv = v;
            bi = col;
          }
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {  // the quad holding the row
        const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
        const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
        if (better(ov, oi, bv, bi)) {
          bv = ov;
          bi = oi;
        }
      }
      if (c == 0 && row < MAXB) s_best[warp][row] = Cand{bv, bi};
    }
  }
  __syncthreads();
  for (int row = tid; row < B; row += THREADS) {
    Cand best = s_best[0][row];
    for (int w = 1; w < WARPS; ++w) {
      const Cand o = s_best[w][row];
      if (better(o.v, o.i, best.v, best.i)) best = o;
    }
    part[size_t(blockIdx.x) * MAXB + row] = best;
  }
}

__global__ void __launch_bounds__(128) argmax_finish_kernel(const Cand* __restrict__ part, int nblk, int B,
                                                             int64_t offset, float* __restrict__ out_val,
                                                             int64_t* __restrict__ out_idx) {
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x * 4 + warp;
  if (row >= B) return;
  float bv = -INFINITY;
  int bi = NOWHERE;
  for (int k = lane; k < nblk; k += 32) {
    const Cand o = part[size_t(k) * MAXB + row];
    if (better(o.v, o.i, bv, bi)) {
      bv = o.v;
      bi = o.i;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    if (better(ov, oi, bv, bi)) {
      bv = ov;
      bi = oi;
    }
  }
  if (lane == 0) {
    out_val[row] = bv;
    out_idx[row] = int64_t(bi == NOWHERE ? 0 : bi) + offset;
  }
}

// shared-memory limits of the kernels on the current device, once
int prepare(const char* what) {
  static std::mutex mu;
  static bool done[64] = {};
  int dev = 0;
  QX_CUDA_TRY(cudaGetDevice(&dev), what);
  QX_REQUIRE(dev >= 0 && dev < 64, "%s: device index %d unsupported", what, dev);
  std::lock_guard<std::mutex> lk(mu);
  if (done[dev]) return QX_OK;
  for (auto kernel : {logits_kernel<1, false>, logits_kernel<2, false>, logits_kernel<1, true>, logits_kernel<2, true>})
    QX_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM), what);
  done[dev] = true;
  return QX_OK;
}

}  // namespace lmh
}  // namespace qx

using namespace qx;

extern "C" size_t qx_lm_head_argmax_workspace_size(int vocab) {
  return vocab > 0 ? size_t((vocab + lmh::COLS - 1) / lmh::COLS) * lmh::MAXB * sizeof(lmh::Cand) : 0;
}

extern "C" int qx_lm_head_argmax(const void* h, const void* weight, int batch, int hidden, int vocab,
                                 int64_t vocab_offset, float* out_val, int64_t* out_idx, void* workspace,
                                 size_t workspace_bytes, qx_stream_t stream) {
  QX_REQUIRE(batch >= 1 && batch <= lmh::MAXB, "lm_head_argmax: batch=%d (1..%d)", batch, lmh::MAXB);
  QX_REQUIRE(hidden > 0 && hidden % lmh::KT == 0, "lm_head_argmax: hidden=%d must be a multiple of %d",
             hidden, lmh::KT);
  QX_REQUIRE(vocab > 0 && vocab % 8 == 0, "lm_head_argmax: vocab=%d must be a multiple of 8", vocab);
  QX_REQUIRE(h && weight && out_val && out_idx, "lm_head_argmax: null pointer");
  QX_REQUIRE(aligned(h, 16) && aligned(weight, 16), "lm_head_argmax: h and weight must be 16-byte aligned");
  const size_t need = qx_lm_head_argmax_workspace_size(vocab);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(QX_ERR_WORKSPACE, "lm_head_argmax: workspace needs %zu bytes, 16-byte aligned", need);
  if (const int rc = lmh::prepare("lm_head_argmax"); rc != QX_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int nblk = (vocab + lmh::COLS - 1) / lmh::COLS;
  auto H = static_cast<const __half*>(h);
  auto Wt = static_cast<const __half*>(weight);
  auto part = static_cast<lmh::Cand*>(workspace);
  QX_CUDA_TRY(launch_pdl(batch <= 16 ? lmh::logits_kernel<1, false> : lmh::logits_kernel<2, false>, dim3(nblk),
                         dim3(lmh::THREADS), lmh::SMEM, st, H, Wt, batch, hidden, vocab, part,
                         static_cast<__half*>(nullptr)),
              "lm_head_argmax: launch");
  QX_CUDA_TRY(launch_pdl(lmh::argmax_finish_kernel, dim3((batch + 3) / 4), dim3(128), 0, st,
                         static_cast<const lmh::Cand*>(part), nblk, batch, vocab_offset, out_val, out_idx),
              "lm_head_argmax: finish launch");
  return check_launch("lm_head_argmax");
}

extern "C" int qx_lm_head_logits(const void* h, const void* weight, void* logits, int batch, int hidden, int vocab,
                                 qx_stream_t stream) {
  QX_REQUIRE(batch >= 0, "lm_head_logits: batch=%d", batch);
  QX_REQUIRE(hidden > 0 && hidden % lmh::KT == 0, "lm_head_logits: hidden=%d must be a multiple of %d", hidden,
             lmh::KT);
  QX_REQUIRE(vocab > 0 && vocab % 8 == 0, "lm_head_logits: vocab=%d must be a multiple of 8", vocab);
  if (batch == 0) return QX_OK;
  QX_REQUIRE(h && weight && logits, "lm_head_logits: null pointer");
  QX_REQUIRE(aligned(h, 16) && aligned(weight, 16) && aligned(logits, 4),
             "lm_head_logits: h and weight must be 16-byte aligned, logits 4-byte");
  if (const int rc = lmh::prepare("lm_head_logits"); rc != QX_OK) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int nblk = (vocab + lmh::COLS - 1) / lmh::COLS;
  for (int64_t r = 0; r < batch; r += lmh::MAXB) {
    const int rows = int(std::min<int64_t>(lmh::MAXB, batch - r));
    QX_CUDA_TRY(launch_pdl(rows <= 16 ? lmh::logits_kernel<1, true> : lmh::logits_kernel<2, true>, dim3(nblk),
                           dim3(lmh::THREADS), lmh::SMEM, st, static_cast<const __half*>(h) + r * hidden,
                           static_cast<const __half*>(weight), rows, hidden, vocab, static_cast<lmh::Cand*>(nullptr),
                           static_cast<__half*>(logits) + r * vocab),
                "lm_head_logits: launch");
  }
  return check_launch("lm_head_logits");
}
