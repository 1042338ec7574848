// The 4-bit ring KV cache: its format and the index rules shared by the
// append, the read-back and the attention kernels.
//
// A layer's storage, keys and values alike:
//   codes  uint8 [batch][kv_heads][cap][D / 2]      two 4-bit codes per byte
//   params u16   [batch][kv_heads][cap][D / group]  one word per group
// cap = sink + window rounded up to 64 slots.  Slots of one KV head are
// contiguous (the attention streams one head's slots; with heads innermost, a
// 32-byte sector of params would hold eight heads' words and seven eighths of
// it would be read for nothing).
//
// A group of `group` consecutive head dimensions (32, 64 or 128) stands for
//   x = s (c - z),  c, z in 0..15
// with s a fp16 number of 7 significant bits.  c - z has 4 bits, so s (c - z)
// has at most 11 and is a fp16 number exactly: the attention multiplies what
// the read-back returns, with no rounding of its own.  The 7-bit s costs at
// most 1/64 of a step and leaves the four low bits of its fp16 word for z, so
// a group takes 16 bits of parameters (4.25 bits a value at group 64).
//
// Order of the codes in a row (halfwords of four codes, low bits first).  An
// 8-value block j = 4 i + c (i < D/32, c < 4) is two halfwords: its even and its
// odd values.  Keys: at halfwords 2 (c NI + i) and + 1, so the lane of an
// MMA quad (c) reads the row's quarter it multiplies with one load and a mask
// of a 32-bit word gives two neighbouring values.  Values: even at 2 c NI + i,
// odd at (2 c + 1) NI + i, so the lanes of an MMA row group (2 c + parity)
// read theirs with one load, each halfword within one group.
#pragma once

#include "qx_common.cuh"

namespace qx {
namespace kv4 {

constexpr int SLOT_ALIGN = 64;
constexpr uint32_t NAN_PARAM = 0x7E00u;  // scale NaN, zero point 0

__host__ __device__ __forceinline__ int64_t capacity(int sink, int window) {
  return (int64_t(sink) + window + SLOT_ALIGN - 1) / SLOT_ALIGN * SLOT_ALIGN;
}

// slots that hold a token after `count` tokens: a prefix of the storage
__host__ __device__ __forceinline__ int valid_slots(int64_t count, int sink, int window) {
  if (count <= 0) return 0;
  if (count <= sink) return int(count);
  const int64_t f = count - sink;
  return sink + int(f < window ? f : window);
}

// what the entry points take as a count of tokens: positions and their sums with a chunk's stay within 64 bits
constexpr int64_t MAX_COUNT = (int64_t(1) << 62) - 1;
inline bool count_fits(int64_t count) { return count >= 0 && count <= MAX_COUNT; }

// tokens written to sequence b: its own count, or the call's.  The host does not see a
// device count: one outside 0 .. MAX_COUNT is taken as the nearer end, so that no position
// wraps to a slot before the storage.
__device__ __forceinline__ int64_t count_of(const int64_t* counts, int64_t count, int b) {
  const int64_t c = counts ? counts[b] : count;
  return c < 0 ? 0 : c < MAX_COUNT ? c : MAX_COUNT;
}

// one halfword pair: bits n of the low half (even values) and of the high half
// (odd values) of `w` -> the fp16 pair (s (c - z)) of values 2n, 2n + 1.
// 0x6400 | c is 1024 + c and 0x5400 | (c << 4) is 64 + c; both differences and
// the product are exact.  zz: (1024 + z) twice, zz4: (64 + z) twice, ss: s twice.
struct GroupScale {
  uint32_t ss, zz, zz4;
};
__device__ __forceinline__ uint32_t hmul2_u32(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// two params words side by side (low and high half) -> their scales and zero points
__device__ __forceinline__ GroupScale group_scale(uint32_t pair) {
  GroupScale g;
  g.ss = pair & 0xFFF0FFF0u;
  g.zz = lop3_and_or(pair, 0x000F000Fu, 0x64006400u);
  g.zz4 = lop3_and_or(pair << 4, 0x00F000F0u, 0x54005400u);
  return g;
}
// the four pairs of a 32-bit word (two halfwords) under the scales of its halves
__device__ __forceinline__ void dequant_word(uint32_t w, const GroupScale& g, uint32_t (&out)[4]) {
  const uint32_t h = w >> 8;
  out[0] = hmul2_u32(hsub2_u32(lop3_and_or(w, 0x000F000Fu, 0x64006400u), g.zz), g.ss);
  out[1] = hmul2_u32(hsub2_u32(lop3_and_or(w, 0x00F000F0u, 0x54005400u), g.zz4), g.ss);
  out[2] = hmul2_u32(hsub2_u32(lop3_and_or(h, 0x000F000Fu, 0x64006400u), g.zz), g.ss);
  out[3] = hmul2_u32(hsub2_u32(lop3_and_or(h, 0x00F000F0u, 0x54005400u), g.zz4), g.ss);
}

// shared argument checks of the entry points; 0 or an error status
inline int check_ring(const char* op, int batch, int kv_heads, int head_dim, int group, int sink, int window) {
  if (batch < 0 || kv_heads <= 0)
    return fail(QX_ERR_INVALID, "%s: bad sizes batch=%d kv_heads=%d", op, batch, kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return fail(QX_ERR_INVALID, "%s: head_dim=%d must be 64 or 128", op, head_dim);
  if ((group != 32 && group != 64 && group != 128) || group > head_dim)
    return fail(QX_ERR_INVALID, "%s: group=%d must be 32, 64 or 128 and at most head_dim=%d", op, group, head_dim);
  if (sink < 0 || window < 1) return fail(QX_ERR_INVALID, "%s: sink=%d window=%d", op, sink, window);
  if (capacity(sink, window) >= (int64_t(1) << 30))
    return fail(QX_ERR_INVALID, "%s: sink + window = %lld slots is too large", op, (long long)sink + window);
  return QX_OK;
}

}  // namespace kv4
}  // namespace qx
