// Layout and arithmetic of the 4-bit K/V cache.
//
// A row (one cached token of one KV head, hd values y) is kept as
//   e   exponent, max|y| in [2^e, 2^(e+1)), held to -40 .. 40 (-40 for a row of zeros): 2^-e and products with it stay
//       inside fp32. Rows of 2^41 and more have z up to 2^16, rows below 2^-40 have z below 1: m and s stay inside fp16.
//       Byte e + 127; 255 marks a row with a non-finite value or one of 2^56 or more: its values are NaN (its codes and
//       scales are zeros, so a masked one adds exactly nothing). Zero bytes, a new pool's, stand for zeros.
//   m, s  per 32 dims of z = y 2^-e: fp16(min z) and fp16((max z - min z) / 15)
//   c   per value: round((z - m) / s) in 0 .. 15; the value it stands for is 2^e (m + s c)
// that is 1.25 hd + 2 bytes for K and V together, against 4 hd in bf16.
//
// 16 rows of one KV head form a block of 20 hd + 32 contiguous bytes (a multiple of 32: whole DRAM sectors, and one
// bulk copy brings a block to shared memory): K codes | V codes | K s [16][hd/32] | K m | V s [hd/32][16] | V m |
// 16 K exponents | 16 V exponents. The order inside the codes is the one in which the attention's tensor-core fragments
// want them, arranged so that a warp's shared-memory loads touch every bank once:
//   K  row r, dim d = 32 i + 8 t + b: nibble b of word (t, i) of the row; a lane's words are contiguous (at hd 256 the
//      two 64-byte halves of odd rows are exchanged)
//   V  row r, dim d = 32 i + 4 g + b: nibble b of 16-bit unit i of the row's chunk g; chunks are exchanged by XOR with
//      bits of r inside each 128 bytes (256 / hd rows)
// and V's s and m of row r sit at slot 4 (r % 8 / 2) + 2 (r / 8) + r % 2: the four rows of a fragment lane adjoin.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kv4.h"
#include "ptx.cuh"

namespace rf {

constexpr int kKv4Mark = 255;
constexpr int kKv4Limit = 40;

template <int HD>
struct Kv4L {
  static constexpr int NG = HD / 32;          // groups of a row
  static constexpr int PER = HD / 32;         // values of a lane when a warp holds a row
  static constexpr int BYTES = 20 * HD + 32;  // a block
  static constexpr int V = 8 * HD, KS = 16 * HD, KM = 17 * HD, VS = 18 * HD, VM = 19 * HD, KE = 20 * HD,
                       VE = 20 * HD + 16;
  // byte of the 32-bit word (t, i) of K row r
  static __host__ __device__ constexpr int k_word(int r, int t, int i) {
    return r * (HD / 2) + 4 * (HD == 256 ? (((i >> 2) ^ (r & 1)) * 16 + t * 4 + (i & 3)) : t * NG + i);
  }
  // byte of chunk g of V row r
  static __host__ __device__ constexpr int v_chunk(int r, int g) {
    constexpr int U = 256 / HD;
    const int flip = HD == 256 ? 2 * ((r >> 1) & 3) : HD == 128 ? 4 * ((r >> 1) & 3) : 8 * ((r >> 2) & 1);
    return V + (r / U) * 128 + ((g + 8 * (r % U)) ^ flip) * (HD / 16);
  }
};
__host__ __device__ constexpr int kv4_slot(int r) { return 4 * ((r & 7) >> 1) + 2 * (r >> 3) + (r & 1); }

// The next kernel of the stream, if launched for it, may start before this one ends / wait until the previous one has ended
// and its stores are seen (nothing to wait for where the launch did not allow an early start). A kernel that starts early
// touches no global memory before its wait: what the previous kernel wrote is seen after it only.
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

__device__ __forceinline__ float kv4_pow2(int e) { return __int_as_float((e + 127) << 23); }

// 2^e of an exponent byte, NaN for a marked row
__device__ __forceinline__ float kv4_size(int byte) {
  return byte == kKv4Mark ? __int_as_float(0x7fffffff) : __int_as_float(byte << 23);
}

// Block base of cache row `row` of KV head g of launch sequence sq; nullptr where the table names no page of the pool.
template <int HD>
__device__ __forceinline__ uint8_t* kv4_block(const Kv4Pages& c, int sq, int g, int row) {
  const int page = __ldg(c.pages[sq] + row / c.page_size);
  if (page < 0 || page >= c.num_pages) return nullptr;
  const long slab = ((long)page * c.hkv + g) * (c.page_size / 16) + (row % c.page_size) / 16;
  return c.pool + slab * Kv4L<HD>::BYTES;
}

__device__ __forceinline__ void kv4_load(const __nv_bfloat16* p, float (&v)[4]) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  v[0] = bf16_lo(u.x), v[1] = bf16_hi(u.x), v[2] = bf16_lo(u.y), v[3] = bf16_hi(u.y);
}
__device__ __forceinline__ void kv4_store(__nv_bfloat16* p, const float (&v)[4]) {
  *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
}

}  // namespace rf
