// Append to and read-back of the 4-bit ring KV cache (format: kv4.cuh).  The
// slot rules are the fp16 ring's (ring_kv.cu; reference
// csrc/kv_cache/ring_buffer.cu:115-123, 149-173): token at position p goes to
// slot p < sink ? p : sink + (p - sink) % window, later tokens of a chunk win.
//
// Quantisation of a group x (each step the nearest real result, ties to even):
//   lo = min(0, min x), hi = max(0, max x)
//   s = the smallest fp16 number of 7 significant bits >= (hi - lo) / 15
//   z = rint(-lo / s)   (0..15, since -lo <= 15 s)
//   c = clamp(rint(x / s) + z, 0, 15), then one step towards z where
//       |s (c - z)| would pass the largest finite fp16 number
// so |x - s (c - z)| <= s / 2 (clamping loses nothing more: hi <= 15 s + lo).
// A group holding a NaN or an infinity gets the scale NaN: it reads as NaN.
// s is found by rounding up in fp32 (hi - lo, then its fifteenth), to fp16, to 7
// bits: a candidate s and 15 s are numbers of each of those formats, so each step
// keeps which of them are large enough.  x / s (11 bits by 7 bits) is a tie or at
// least 2^-12 away from one: near k + 1/2, x - (k + 1/2) s is a whole multiple of
// the smaller of their units.  So x times the rounded 1 / s (off by less than
// 2^-18) is rounded to a multiple of 2^-13 first: ties become exact ties, and
// nothing else reaches one.
//
// Bound: HBM (2 bytes read per value, 0.53 written; the read-back the reverse).
// Four lanes hold one (token, head) row, lane c the blocks 4 i + c: its codes are
// 16 bytes side by side in the cache (8 at D = 64), a group of 32 is one block of
// each of the four lanes, and a row's loads are all in flight at once.  (With
// D / 8 lanes a row, one block each, and 64-bit index divisions: append of 2048
// tokens x 8 heads and read-back of 4096 slots 29.6 us; now 10.7, two kernels that
// each are one wave.)
#include <algorithm>

#include "kv4.cuh"
#include "qx_b200.h"

namespace qx {
namespace ring4 {

constexpr int THREADS = 256, LANES = 4, ROWS = THREADS / LANES;  // rows of a CTA

struct AppendParams {
  unsigned char* codes[2];
  uint16_t* params[2];
  const __half* fresh[2];
  const int64_t* counts;
  int64_t count, cap;
  int tokens, kv_heads, rows, sink, window;  // rows: tokens * kv_heads, of one sequence
};

// nearest whole number to x / s, ties to even (see above); |x / s| <= 16
__device__ __forceinline__ int nearest(float x, float inv_s) {
  const float t = fmaf(x, inv_s, 1536.f) - 1536.f;  // fp32's step at 1024 .. 2048 is 2^-13
  return __float_as_int(t + 12582912.f) - __float_as_int(12582912.f);
}

template <int D, int GROUP>
__global__ void __launch_bounds__(THREADS) append_kernel(const __grid_constant__ AppendParams p) {
  pdl_trigger();
  pdl_wait();
  constexpr int NI = D / 32, NG = D / GROUP, IPG = NI / NG;
  const int c = threadIdx.x % LANES, b = blockIdx.y, which = blockIdx.z;
  const int r = int(blockIdx.x) * ROWS + int(threadIdx.x) / LANES;
  const int j = r / p.kv_heads, h = r - j * p.kv_heads;
  const int64_t count = kv4::count_of(p.counts, p.count, b), pos = count + j;
  // a ring token that a later one of this chunk replaces is not stored
  const bool keep = r < p.rows && (pos < p.sink || j >= p.tokens - p.window);
  uint4 v[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i)
    v[i] = keep ? __ldg(reinterpret_cast<const uint4*>(p.fresh[which] + (int64_t(b) * p.rows + r) * D) + 4 * i + c)
                : make_uint4(0u, 0u, 0u, 0u);
  uint32_t word[NI], param[NG];
#pragma unroll
  for (int n = 0; n < NG; ++n) {
    __half2 lo2 = __float2half2_rn(0.f), hi2 = lo2;
#pragma unroll
    for (int i = n * IPG; i < (n + 1) * IPG; ++i) {
      const uint32_t d[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const __half2 x = *reinterpret_cast<const __half2*>(&d[e]);
        lo2 = __hmin2_nan(lo2, x);
        hi2 = __hmax2_nan(hi2, x);
      }
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
      lo2 = __hmin2_nan(lo2, __shfl_xor_sync(0xffffffffu, lo2, o));
      hi2 = __hmax2_nan(hi2, __shfl_xor_sync(0xffffffffu, hi2, o));
    }
    const float lo = __half2float(__hmin_nan(__low2half(lo2), __high2half(lo2)));
    const float hi = __half2float(__hmax_nan(__low2half(hi2), __high2half(hi2)));
    const bool fine = lo >= -65504.f && hi <= 65504.f;  // false for a NaN
    const float least = __fdiv_ru(__fsub_ru(hi, lo), 15.f);
    const uint32_t bits = (uint32_t(__half_as_ushort(__float2half_ru(least))) + 15u) & 0xFFF0u;
    const float s = __half2float(__ushort_as_half(uint16_t(bits)));
    const float inv = fine && s > 0.f ? __frcp_rn(s) : 0.f;
    const int z = fine ? nearest(-lo, inv) : 0;
    param[n] = fine ? bits | uint32_t(z) : kv4::NAN_PARAM;
#pragma unroll
    for (int i = n * IPG; i < (n + 1) * IPG; ++i) {
      const uint32_t d[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = h2_to_f2(d[e]);
        int c0 = min(max(nearest(x.x, inv) + z, 0), 15), c1 = min(max(nearest(x.y, inv) + z, 0), 15);
        if (s > 65504.f / 15.f) {  // only then can s (c - z) pass the largest finite number
          if (fabsf(float(c0 - z) * s) > 65504.f) c0 -= c0 > z ? 1 : -1;
          if (fabsf(float(c1 - z) * s) > 65504.f) c1 -= c1 > z ? 1 : -1;
        }
        w |= uint32_t(c0) << (4 * e) | uint32_t(c1) << (4 * e + 16);  // even values low, odd values high
      }
      word[i] = fine ? w : 0u;
    }
  }
  if (!keep) return;
  const int64_t slot = pos < p.sink ? pos : p.sink + (pos - p.sink) % p.window;
  const int64_t row = (int64_t(b) * p.kv_heads + h) * p.cap + slot;
  if (which == 1) {  // values: the even halves side by side, then the odd ones
    uint32_t t[NI];
#pragma unroll
    for (int i = 0; i < NI; i += 2) {
      t[i / 2] = prmt(word[i], word[i + 1], 0x5410u);
      t[NI / 2 + i / 2] = prmt(word[i], word[i + 1], 0x7632u);
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) word[i] = t[i];
  }
  unsigned char* dst = p.codes[which] + row * (D / 2) + c * (D / 8);
  if constexpr (NI == 4)
    *reinterpret_cast<uint4*>(dst) = make_uint4(word[0], word[1], word[2], word[3]);
  else
    *reinterpret_cast<uint2*>(dst) = make_uint2(word[0], word[1]);
  uint16_t* pp = p.params[which] + row * NG;
#pragma unroll
  for (int n = 0; n < NG; ++n)
    if (c == n) pp[n] = uint16_t(param[n]);
}

struct GatherParams {
  const unsigned char* codes[2];
  const uint16_t* params[2];
  __half* out[2];
  int64_t cap;
  int start, kv_heads, rows, sink, window;  // start: the ring's oldest token; rows: valid * kv_heads
};

template <int D, int GROUP>
__global__ void __launch_bounds__(THREADS) gather_kernel(const __grid_constant__ GatherParams p) {
  pdl_trigger();
  pdl_wait();
  constexpr int NI = D / 32, NG = D / GROUP;
  const int c = threadIdx.x % LANES, b = blockIdx.y, which = blockIdx.z;
  const int r = int(blockIdx.x) * ROWS + int(threadIdx.x) / LANES;
  if (r >= p.rows) return;
  const int n = r / p.kv_heads, h = r - n * p.kv_heads;
  int slot = n;
  if (n >= p.sink) {
    slot += p.start;  // below sink + 2 window
    if (slot >= p.sink + p.window) slot -= p.window;
  }
  const int64_t row = (int64_t(b) * p.kv_heads + h) * p.cap + slot;
  const unsigned char* src = p.codes[which] + row * (D / 2) + c * (D / 8);
  uint32_t w[NI], param[NG];
  if constexpr (NI == 4) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(src));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
    const uint2 v = __ldg(reinterpret_cast<const uint2*>(src));
    w[0] = v.x, w[1] = v.y;
  }
#pragma unroll
  for (int g = 0; g < NG; ++g) param[g] = __ldg(p.params[which] + row * NG + g) * 0x10001u;
  uint4* out = reinterpret_cast<uint4*>(p.out[which] + (int64_t(b) * p.rows + r) * D) + c;
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const uint32_t word =
        which == 0 ? w[i] : prmt(w[i >> 1], w[NI / 2 + (i >> 1)], (i & 1) ? 0x7632u : 0x5410u);
    uint32_t o[4];
    kv4::dequant_word(word, kv4::group_scale(param[i * NG / NI]), o);
    out[4 * i] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

template <int D, int GROUP>
cudaError_t launch_append(const AppendParams& p, int batch, cudaStream_t st) {
  return launch_pdl(append_kernel<D, GROUP>, dim3(unsigned((p.rows + ROWS - 1) / ROWS), unsigned(batch), 2),
                    dim3(THREADS), 0, st, p);
}
template <int D, int GROUP>
cudaError_t launch_gather(const GatherParams& p, int batch, cudaStream_t st) {
  return launch_pdl(gather_kernel<D, GROUP>, dim3(unsigned((p.rows + ROWS - 1) / ROWS), unsigned(batch), 2),
                    dim3(THREADS), 0, st, p);
}

}  // namespace ring4
}  // namespace qx

using namespace qx;

extern "C" int64_t qx_ring_q4_slots(int sink, int window) {
  QX_REQUIRE(sink >= 0 && window >= 1, "ring_q4_slots: sink=%d window=%d", sink, window);
  return kv4::capacity(sink, window);
}

extern "C" int qx_ring_append_q4(void* k_codes, void* k_params, void* v_codes, void* v_params, const void* new_k,
                                 const void* new_v, int batch, int tokens, int kv_heads, int head_dim, int group,
                                 int sink, int window, int64_t count, const int64_t* counts, qx_stream_t stream) {
  const int rc = kv4::check_ring("ring_append_q4", batch, kv_heads, head_dim, group, sink, window);
  if (rc != QX_OK) return rc;
  QX_REQUIRE(tokens >= 0 && (counts || kv4::count_fits(count)), "ring_append_q4: tokens=%d count=%lld", tokens, (long long)count);
  if (batch == 0 || tokens == 0) return QX_OK;
  QX_REQUIRE(k_codes && k_params && v_codes && v_params && new_k && new_v, "ring_append_q4: null pointer");
  QX_REQUIRE(aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(k_params, 16) && aligned(v_params, 16) &&
                 aligned(new_k, 16) && aligned(new_v, 16),
             "ring_append_q4: tensors must be 16-byte aligned");
  QX_REQUIRE(batch <= 65535 && int64_t(tokens) * kv_heads < (int64_t(1) << 31) - ring4::ROWS,
             "ring_append_q4: batch=%d or tokens=%d too large", batch, tokens);
  ring4::AppendParams p{};
  p.codes[0] = static_cast<unsigned char*>(k_codes);
  p.codes[1] = static_cast<unsigned char*>(v_codes);
  p.params[0] = static_cast<uint16_t*>(k_params);
  p.params[1] = static_cast<uint16_t*>(v_params);
  p.fresh[0] = static_cast<const __half*>(new_k);
  p.fresh[1] = static_cast<const __half*>(new_v);
  p.counts = counts;
  p.count = count;
  p.rows = tokens * kv_heads;
  p.tokens = tokens;
  p.kv_heads = kv_heads;
  p.sink = sink;
  p.window = window;
  p.cap = kv4::capacity(sink, window);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (head_dim == 64)
    e = group == 32 ? ring4::launch_append<64, 32>(p, batch, st) : ring4::launch_append<64, 64>(p, batch, st);
  else
    e = group == 32   ? ring4::launch_append<128, 32>(p, batch, st)
        : group == 64 ? ring4::launch_append<128, 64>(p, batch, st)
                      : ring4::launch_append<128, 128>(p, batch, st);
  QX_CUDA_TRY(e, "ring_append_q4: launch");
  return check_launch("ring_append_q4");
}

extern "C" int qx_ring_gather_q4(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                                 void* k_out, void* v_out, int batch, int kv_heads, int head_dim, int group, int sink,
                                 int window, int64_t count, qx_stream_t stream) {
  const int rc = kv4::check_ring("ring_gather_q4", batch, kv_heads, head_dim, group, sink, window);
  if (rc != QX_OK) return rc;
  QX_REQUIRE(kv4::count_fits(count), "ring_gather_q4: count=%lld", (long long)count);
  const int valid = kv4::valid_slots(count, sink, window);
  if (batch == 0 || valid == 0) return QX_OK;
  QX_REQUIRE(k_codes && k_params && v_codes && v_params && k_out && v_out, "ring_gather_q4: null pointer");
  QX_REQUIRE(aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(k_params, 16) && aligned(v_params, 16) &&
                 aligned(k_out, 16) && aligned(v_out, 16),
             "ring_gather_q4: tensors must be 16-byte aligned");
  QX_REQUIRE(batch <= 65535 && int64_t(valid) * kv_heads < (int64_t(1) << 31) - ring4::ROWS,
             "ring_gather_q4: batch=%d or %d tokens too large", batch, valid);
  ring4::GatherParams p{};
  p.codes[0] = static_cast<const unsigned char*>(k_codes);
  p.codes[1] = static_cast<const unsigned char*>(v_codes);
  p.params[0] = static_cast<const uint16_t*>(k_params);
  p.params[1] = static_cast<const uint16_t*>(v_params);
  p.out[0] = static_cast<__half*>(k_out);
  p.out[1] = static_cast<__half*>(v_out);
  p.start = count - sink <= window ? 0 : int((count - sink) % window);
  p.rows = valid * kv_heads;
  p.kv_heads = kv_heads;
  p.sink = sink;
  p.window = window;
  p.cap = kv4::capacity(sink, window);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (head_dim == 64)
    e = group == 32 ? ring4::launch_gather<64, 32>(p, batch, st) : ring4::launch_gather<64, 64>(p, batch, st);
  else
    e = group == 32   ? ring4::launch_gather<128, 32>(p, batch, st)
        : group == 64 ? ring4::launch_gather<128, 64>(p, batch, st)
                      : ring4::launch_gather<128, 128>(p, batch, st);
  QX_CUDA_TRY(e, "ring_gather_q4: launch");
  return check_launch("ring_gather_q4");
}
