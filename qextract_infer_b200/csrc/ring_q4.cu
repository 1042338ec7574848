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
// s is found by rounding up in three steps (64-bit quotient to fp32 to fp16 to
// 7 bits), which composes; x / s is the IEEE fp32 quotient of an 11-bit by a
// 7-bit number: one that is no tie is at least 2^-12 away from any (near k + 1/2,
// x - (k + 1/2) s is a whole multiple of the smaller of their units), so its rint
// is the real quotient's.
//
// Bound: HBM (2 bytes read per value, 0.53 written; the read-back the reverse).
// D / 8 lanes hold one (token, head) row, 8 values each: the group's minimum and
// maximum are butterflies over group / 8 lanes.
#include <algorithm>

#include "kv4.cuh"
#include "qx_b200.h"

namespace qx {
namespace ring4 {

constexpr int THREADS = 256;

struct AppendParams {
  uint32_t* codes[2];
  uint16_t* params[2];
  const uint4* fresh[2];
  const int64_t* counts;
  int64_t count, rows;  // rows: batch * tokens * kv_heads
  int tokens, kv_heads, sink, window;
  int64_t cap;
};

// E (low half): codes of the even values of the lane's 8; O (high half): of the odd ones
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], float s, int z) {
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    int k = s > 0.f ? int(rintf(__fdiv_rn(x[e], s))) : 0;
    int c = min(max(k + z, 0), 15);
    k = c - z;
    if (fabsf(float(k) * s) > 65504.f) c -= k > 0 ? 1 : -1;
    w |= uint32_t(c) << ((e >> 1) * 4 + (e & 1) * 16);
  }
  return w;
}

template <int D, int GROUP>
__global__ void __launch_bounds__(THREADS) append_kernel(const AppendParams p) {
  pdl_trigger();
  pdl_wait();
  constexpr int LPR = D / 8;      // lanes per row
  constexpr int LPG = GROUP / 8;  // lanes per group
  constexpr int NI = D / 32;
  const int l = threadIdx.x % LPR;
  const int which = blockIdx.y;
  const int64_t step = int64_t(gridDim.x) * (THREADS / LPR);
  const int64_t first = int64_t(blockIdx.x) * (THREADS / LPR) + threadIdx.x / LPR;
  // every lane of a warp runs every turn (the butterflies need them all)
  const int64_t turns = (p.rows + step - 1) / step;
  for (int64_t turn = 0; turn < turns; ++turn) {
    const int64_t r = first + turn * step;
    const bool in = r < p.rows;
    const int64_t bt = in ? r / p.kv_heads : 0;
    const int h = in ? int(r - bt * p.kv_heads) : 0;
    const int b = int(bt / p.tokens), j = int(bt - int64_t(b) * p.tokens);
    const int64_t count = kv4::count_of(p.counts, p.count, b);
    const int64_t pos = count + j;
    // a ring token that a later one of this chunk replaces is not stored
    const bool keep = in && (pos < p.sink || j >= p.tokens - p.window);
    const uint4 v = keep ? __ldg(p.fresh[which] + r * LPR + l) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t vd[4] = {v.x, v.y, v.z, v.w};
    float x[8], lo = 0.f, hi = 0.f;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = h2_to_f2(vd[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
      fine = fine && fabsf(f.x) <= 65504.f && fabsf(f.y) <= 65504.f;  // false for a NaN
      lo = fminf(lo, fminf(f.x, f.y));
      hi = fmaxf(hi, fmaxf(f.x, f.y));
    }
    int bad = fine ? 0 : 1;
#pragma unroll
    for (int o = LPG / 2; o > 0; o >>= 1) {
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      bad |= __shfl_xor_sync(0xffffffffu, bad, o);
    }
    uint32_t word = 0, param = kv4::NAN_PARAM;
    if (!bad) {
      const float least = __double2float_ru((double(hi) - double(lo)) / 15.0);
      const uint32_t bits = (uint32_t(__half_as_ushort(__float2half_ru(least))) + 15u) & 0xFFF0u;
      const float s = __half2float(__ushort_as_half(uint16_t(bits)));
      const int z = s > 0.f ? int(rintf(__fdiv_rn(-lo, s))) : 0;
      word = quantise8(x, s, z);
      param = bits | uint32_t(z);
    }
    const int c = l & 3, i = l >> 2;
    if (which == 1) {
      // values: the even halves of blocks (i, i + 1) share a word, and the odd ones
      const uint32_t send = (i & 1) ? (word & 0xFFFFu) : (word >> 16);
      const uint32_t got = __shfl_xor_sync(0xffffffffu, send, 4);
      word = (i & 1) ? (got | (word & 0xFFFF0000u)) : ((word & 0xFFFFu) | (got << 16));
    }
    if (!keep) continue;
    const int64_t slot = pos < p.sink ? pos : p.sink + (pos - p.sink) % p.window;
    const int64_t row = (int64_t(b) * p.kv_heads + h) * p.cap + slot;
    const int at = which == 0 ? c * NI + i : ((2 * c + (i & 1)) * NI + (i & ~1)) / 2;
    p.codes[which][row * LPR + at] = word;
    if (l % LPG == 0) p.params[which][row * (D / GROUP) + l / LPG] = uint16_t(param);
  }
}

struct GatherParams {
  const uint16_t* codes[2];
  const uint16_t* params[2];
  uint4* out[2];
  int64_t count, rows;  // rows: batch * valid * kv_heads
  int valid, kv_heads, sink, window;
  int64_t cap;
};

template <int D, int GROUP>
__global__ void __launch_bounds__(THREADS) gather_kernel(const GatherParams p) {
  pdl_trigger();
  pdl_wait();
  constexpr int LPR = D / 8, NI = D / 32;
  const int l = threadIdx.x % LPR, c = l & 3, i = l >> 2;
  const int which = blockIdx.y;
  const int64_t step = int64_t(gridDim.x) * (THREADS / LPR);
  const int64_t f = p.count - p.sink;
  const int64_t start = f <= p.window ? 0 : f % p.window;  // the ring's oldest token
  for (int64_t r = int64_t(blockIdx.x) * (THREADS / LPR) + threadIdx.x / LPR; r < p.rows; r += step) {
    const int64_t bi = r / p.kv_heads;
    const int h = int(r - bi * p.kv_heads);
    const int b = int(bi / p.valid), n = int(bi - int64_t(b) * p.valid);
    const int64_t slot = n < p.sink ? n : p.sink + (start + (n - p.sink)) % p.window;
    const int64_t row = (int64_t(b) * p.kv_heads + h) * p.cap + slot;
    const uint16_t* cr = p.codes[which] + row * (2 * LPR);
    const uint32_t word = which == 0 ? __ldg(reinterpret_cast<const uint32_t*>(cr) + c * NI + i)
                                     : (uint32_t(__ldg(cr + 2 * c * NI + i)) |
                                        (uint32_t(__ldg(cr + (2 * c + 1) * NI + i)) << 16));
    const uint32_t param = __ldg(p.params[which] + row * (D / GROUP) + l / (GROUP / 8));
    uint32_t o[4];
    kv4::dequant_word(word, kv4::group_scale(param | (param << 16)), o);
    p.out[which][r * LPR + l] = make_uint4(o[0], o[1], o[2], o[3]);
  }
}

inline unsigned grid_for(int64_t rows, int lanes_per_row) {
  const int64_t per = THREADS / lanes_per_row;
  return unsigned(std::max<int64_t>(1, std::min<int64_t>((rows + per - 1) / per, int64_t(device_sm_count()) * 16)));
}

template <int D, int GROUP>
cudaError_t launch_append(const AppendParams& p, cudaStream_t st) {
  return launch_pdl(append_kernel<D, GROUP>, dim3(grid_for(p.rows, D / 8), 2), dim3(THREADS), 0, st, p);
}
template <int D, int GROUP>
cudaError_t launch_gather(const GatherParams& p, cudaStream_t st) {
  return launch_pdl(gather_kernel<D, GROUP>, dim3(grid_for(p.rows, D / 8), 2), dim3(THREADS), 0, st, p);
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
  QX_REQUIRE(tokens >= 0 && (counts || count >= 0), "ring_append_q4: tokens=%d count=%lld", tokens, (long long)count);
  if (batch == 0 || tokens == 0) return QX_OK;
  QX_REQUIRE(k_codes && k_params && v_codes && v_params && new_k && new_v, "ring_append_q4: null pointer");
  QX_REQUIRE(aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(k_params, 16) && aligned(v_params, 16) &&
                 aligned(new_k, 16) && aligned(new_v, 16),
             "ring_append_q4: tensors must be 16-byte aligned");
  ring4::AppendParams p{};
  p.codes[0] = static_cast<uint32_t*>(k_codes);
  p.codes[1] = static_cast<uint32_t*>(v_codes);
  p.params[0] = static_cast<uint16_t*>(k_params);
  p.params[1] = static_cast<uint16_t*>(v_params);
  p.fresh[0] = static_cast<const uint4*>(new_k);
  p.fresh[1] = static_cast<const uint4*>(new_v);
  p.counts = counts;
  p.count = count;
  p.rows = int64_t(batch) * tokens * kv_heads;
  p.tokens = tokens;
  p.kv_heads = kv_heads;
  p.sink = sink;
  p.window = window;
  p.cap = kv4::capacity(sink, window);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (head_dim == 64)
    e = group == 32 ? ring4::launch_append<64, 32>(p, st) : ring4::launch_append<64, 64>(p, st);
  else
    e = group == 32   ? ring4::launch_append<128, 32>(p, st)
        : group == 64 ? ring4::launch_append<128, 64>(p, st)
                      : ring4::launch_append<128, 128>(p, st);
  QX_CUDA_TRY(e, "ring_append_q4: launch");
  return check_launch("ring_append_q4");
}

extern "C" int qx_ring_gather_q4(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params,
                                 void* k_out, void* v_out, int batch, int kv_heads, int head_dim, int group, int sink,
                                 int window, int64_t count, qx_stream_t stream) {
  const int rc = kv4::check_ring("ring_gather_q4", batch, kv_heads, head_dim, group, sink, window);
  if (rc != QX_OK) return rc;
  QX_REQUIRE(count >= 0, "ring_gather_q4: negative count");
  const int valid = kv4::valid_slots(count, sink, window);
  if (batch == 0 || valid == 0) return QX_OK;
  QX_REQUIRE(k_codes && k_params && v_codes && v_params && k_out && v_out, "ring_gather_q4: null pointer");
  QX_REQUIRE(aligned(k_codes, 16) && aligned(v_codes, 16) && aligned(k_params, 16) && aligned(v_params, 16) &&
                 aligned(k_out, 16) && aligned(v_out, 16),
             "ring_gather_q4: tensors must be 16-byte aligned");
  ring4::GatherParams p{};
  p.codes[0] = static_cast<const uint16_t*>(k_codes);
  p.codes[1] = static_cast<const uint16_t*>(v_codes);
  p.params[0] = static_cast<const uint16_t*>(k_params);
  p.params[1] = static_cast<const uint16_t*>(v_params);
  p.out[0] = static_cast<uint4*>(k_out);
  p.out[1] = static_cast<uint4*>(v_out);
  p.count = count;
  p.rows = int64_t(batch) * valid * kv_heads;
  p.valid = valid;
  p.kv_heads = kv_heads;
  p.sink = sink;
  p.window = window;
  p.cap = kv4::capacity(sink, window);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (head_dim == 64)
    e = group == 32 ? ring4::launch_gather<64, 32>(p, st) : ring4::launch_gather<64, 64>(p, st);
  else
    e = group == 32   ? ring4::launch_gather<128, 32>(p, st)
        : group == 64 ? ring4::launch_gather<128, 64>(p, st)
                      : ring4::launch_gather<128, 128>(p, st);
  QX_CUDA_TRY(e, "ring_gather_q4: launch");
  return check_launch("ring_gather_q4");
}
