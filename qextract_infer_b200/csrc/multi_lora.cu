// Low-rank adapters of many requests beside a shared projection: sequence b has the
// adapter a = adapters[b] of n (outside 0 .. n - 1: none), and every token of it
//   out = fp16( y + scales[a] (x A[a]) B[a] )
// with y the shared projection's output, A fp16 [n][K][P r] and B fp16 [n][r][N].  The
// columns are P blocks (the parts of a fused projection: q | k | v, gate | up); block j
// takes the ranks j r .. j r + r - 1 of A.
//
// A CTA takes a row: h = x A in fp32, then the row's columns.
#include "qx_b200.h"
#include "qx_common.cuh"

namespace qx {
namespace mlora {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_PARTS = 4;
constexpr int MAX_RANKS = 256;  // P r

struct Params {
  const __half *y, *x, *A, *B;
  const int64_t* adapters;
  const float* scales;
  __half* out;
  int batch, tokens, K, N, rank, ranks, n, parts;
  int edge[MAX_PARTS + 1];  // first column of each block, then N
};

__global__ void __launch_bounds__(THREADS) multi_lora_kernel(const Params p) {
  __shared__ float h[MAX_RANKS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_trigger();
  pdl_wait();
  const int64_t row = blockIdx.x;
  const int64_t a = p.adapters[row / p.tokens];
  const __half* const y = p.y + row * p.N;
  __half* const out = p.out + row * p.N;
  if (a < 0 || a >= p.n) {
    if (out != y)
      for (int c = tid; c < p.N; c += THREADS) out[c] = y[c];
    return;
  }
  const __half* const x = p.x + row * p.K;
  const __half* const A = p.A + a * p.K * p.ranks;
  const __half* const B = p.B + a * p.rank * p.N;
  for (int j = warp; j < p.ranks; j += WARPS) {
    float sum = 0.f;
    for (int k = lane; k < p.K; k += 32) sum = fmaf(__half2float(x[k]), __half2float(A[int64_t(k) * p.ranks + j]), sum);
    sum = warp_sum(sum);
    if (lane == 0) h[j] = sum;
  }
  __syncthreads();
  const float scale = p.scales[a];
  for (int c = tid; c < p.N; c += THREADS) {
    int part = 0;
    while (c >= p.edge[part + 1]) ++part;
    float sum = 0.f;
    for (int j = 0; j < p.rank; ++j) sum = fmaf(h[part * p.rank + j], __half2float(B[int64_t(j) * p.N + c]), sum);
    out[c] = __float2half_rn(fmaf(scale, sum, __half2float(y[c])));
  }
}

// whether two runs of memory share a byte
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
  const uintptr_t p = reinterpret_cast<uintptr_t>(a), q = reinterpret_cast<uintptr_t>(b);
  return p < q + uintptr_t(b_bytes) && q < p + uintptr_t(a_bytes);
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
  QX_CUDA_TRY(launch_pdl(multi_lora_kernel, dim3(unsigned(rows)), dim3(THREADS), 0,
                         reinterpret_cast<cudaStream_t>(stream), p),
              "multi_lora_add: launch");
  return check_launch("multi_lora_add");
}
