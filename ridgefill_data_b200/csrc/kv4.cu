// Append to and read from the 4-bit K/V cache (layout: kv4.cuh).
//
// kv4_append_kernel  a warp per row and head (q | k | v), a lane holding hd / 32 consecutive values: head norm and rotation
//                    (q, k), then q goes out in bf16 and k / v rows are quantised into their block.
// kv4_append_rows_kernel  the same for many rows (below).
// kv4_read_kernel    a block of 16 rows to shared memory in 16-byte pieces by 1, 2 or 4 warps, then 8 values a lane: the
//                    numbers that the codes stand for, in fp32 and from there in bf16, whole rows to a store.
//
// Roundings are the bf16 model's (norm and each step of the rotation round to bf16), so a cached key is the 4-bit form
// of the row the bf16 cache would hold. The norm's sum of squares and its root are taken in 64 bits: products of two
// bf16 are exact there, so the row, and with it every code next to a border, does not depend on the order of the sum;
// its products with the root are carried as two 32-bit numbers (46 bits). A query is not quantised: 32 bits.
#include "kv4.cuh"

#include "kernels.h"

#include <algorithm>
#include <stdexcept>

namespace rf {

namespace {

constexpr unsigned kFull = 0xffffffffu;

// Two 32-bit numbers under one instruction, each rounded as alone: half the issue slots, which bound the append.
struct Two {
  uint64_t w;
  __device__ __forceinline__ Two() {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(w) : "f"(a), "f"(b)); }
  __device__ __forceinline__ explicit Two(float a) : Two(a, a) {}
  __device__ __forceinline__ explicit Two(uint32_t bf16_pair) : Two(bf16_lo(bf16_pair), bf16_hi(bf16_pair)) {}
  __device__ __forceinline__ void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(w)); }
};
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(c.w) : "l"(a.w), "l"(b.w), "l"(c.w));
  return c;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(a.w) : "l"(a.w), "l"(b.w));
  return a;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(a.w) : "l"(a.w), "l"(b.w));
  return a;
}
__device__ __forceinline__ Two neg2(Two a) {
  a.w ^= 0x8000000080000000ull;
  return a;
}

// 1 / sqrt(m) to about 50 bits: two Newton steps on the 22 bits of the single-precision root.
__device__ __forceinline__ double inverse_root(double m) {
  if (!(m > 1e-30 && m < 1e30)) return 1.0 / sqrt(m);
  double y = (double)rsqrtf((float)m);
  const double h = 0.5 * m;
  y = y * fma(-h * y, y, 1.5);
  return y * fma(-h * y, y, 1.5);
}

__device__ __forceinline__ uint32_t mul_bf16(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmul2_rn(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t fma_bf16(uint32_t a, uint32_t b, uint32_t c) {
  const __nv_bfloat162 r = __hfma2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b),
                                   *reinterpret_cast<__nv_bfloat162*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t add_bf16(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hadd2_rn(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// |x| of the lower and upper bf16 of a pair in 64 bits, by moving the exponent and the mantissa to their places (the
// special-function unit's conversions would take most of a norm). Zero and subnormals come out as 2^-127 .. 2^-126:
// their squares are nothing beside eps, which the caller holds to 1e-30 and more; infinities and NaN come out finite and
// stay in the row itself.
__device__ __forceinline__ double low_double(uint32_t w) {
  return __hiloint2double((int)((w & 0x7fffu) * 8192u + 0x38000000u), 0);
}
__device__ __forceinline__ double high_double(uint32_t w) {
  return __hiloint2double((int)(__umulhi(w & 0x7fff0000u, 0x20000000u) + 0x38000000u), 0);
}

// 1 / sqrt(mean square + eps) of a key as two floats, and a pair of values times it and the norm weight (mode 0 plain, 1
// zero-centred), rounded to bf16 where the model rounds.
struct Root {
  float rh, rl;
  __device__ __forceinline__ explicit Root(double m) {
    const double inv = inverse_root(m);
    rh = (float)inv, rl = (float)(inv - (double)rh);
  }
  __device__ __forceinline__ uint32_t pair(uint32_t v, uint32_t w, int mode) const {
    Two ph(rh), pl(rl);
    if (mode == 1) {   // (1 + w) r as ph + pl
      const Two h = ph, x(w), wh = add2(x, Two(1.f)), wl = fma2(add2(wh, Two(-1.f)), Two(-1.f), x);
      ph = mul2(h, wh), pl = fma2(pl, wh, fma2(h, wl, fma2(h, wh, neg2(ph))));
    }
    const Two y(v), p = mul2(y, ph);
    float a, b;
    add2(p, fma2(y, pl, fma2(y, ph, neg2(p)))).get(a, b);
    const uint32_t z = pack_bf16x2(a, b);
    return mode == 0 ? mul_bf16(z, w) : z;
  }
};

// The same of a query, which is not quantised, in 32 bits: the arithmetic of head_norm_rope (norm.cu), bit for bit.
__device__ __forceinline__ uint32_t query_pair(float inv, uint32_t v, uint32_t w, int mode) {
  Two y = mul2(Two(v), Two(inv));
  if (mode == 1) y = mul2(y, add2(Two(w), Two(1.f)));
  float a, b;
  y.get(a, b);
  const uint32_t z = pack_bf16x2(a, b);
  return mode == 0 ? mul_bf16(z, w) : z;
}

// NaN where either is
__device__ __forceinline__ uint32_t min_bf16(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmin2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t max_bf16(uint32_t a, uint32_t b) {
  const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The 16 steps of a group whose values lie in [lo, hi], in z = y * size.
struct Steps {
  __half s, m;
  float mf, sf, size;
  __device__ __forceinline__ Steps(float lo, float hi, float size_) : size(size_) {
    // (hi - lo) / 15 correctly rounded: the product with the rounded reciprocal and one correction by the exact
    // remainder (P. Markstein, 1990)
    const float d = hi * size - lo * size, q = d * (1.f / 15.f);
    s = __float2half_rn(fmaf(fmaf(-15.f, q, d), 1.f / 15.f, q));
    mf = __half2float(__float2half_rn(lo * size)) + 0.f;   // + 0: a zero is kept as +0
    m = __float2half_rn(mf);
    sf = __half2float(s);
  }
  // round((z - m) / s) of N values in bf16 pairs, to words of 8: the quotient by an approximate reciprocal and one
  // correction by its remainder (Markstein again), the integer that an fp32 sum with 1.5 2^23 leaves in its low bits.
  // Where s is so small that its own rounding can lead past 0 .. 15, held to them.
  template <int N>
  __device__ __forceinline__ void codes(const uint32_t* pairs, uint32_t* words) const {
    constexpr float kBase = 12582912.f;            // its bits: 0x4b400000
    const float inv = sf == 0.f ? 0.f : __fdividef(1.f, sf);
    Two c[N / 2];
    const Two size2(size), m2(-mf), s2(-sf), inv2(inv);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      const Two d = fma2(Two(pairs[j]), size2, m2), q = mul2(d, inv2);
      c[j] = fma2(fma2(q, s2, d), inv2, q);
    }
    if (sf < 0x1p-13f) {
#pragma unroll
      for (int j = 0; j < N / 2; ++j) {
        float x, y;
        c[j].get(x, y);
        c[j] = Two(fminf(fmaxf(x, 0.f), 15.f), fminf(fmaxf(y, 0.f), 15.f));
      }
    }
    uint32_t base = 0;                             // the sum of the bases by 16^j
#pragma unroll
    for (int j = 0; j < (N < 8 ? N : 8); ++j) base += 0x4b400000u << (4 * j);
#pragma unroll
    for (int x = 0; x < (N + 7) / 8; ++x) words[x] = 0u - base;
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      float x, y;
      add2(c[j], Two(kBase)).get(x, y);
      words[j / 4] += __float_as_uint(x) << (8 * (j & 3));
      words[j / 4] += __float_as_uint(y) << (8 * (j & 3) + 4);
    }
  }
};

// A lane's hd / 32 consecutive values of a row as bf16 pairs.
template <int PER>
struct Row {
  uint32_t w[PER / 2];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    if constexpr (PER == 8) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else if constexpr (PER == 4) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = u.x, w[1] = u.y;
    } else {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    }
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const {
    if constexpr (PER == 8)
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else if constexpr (PER == 4)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint32_t*>(p) = w[0];
  }
  __device__ __forceinline__ float get(int j) const { return j & 1 ? bf16_hi(w[j / 2]) : bf16_lo(w[j / 2]); }
};

// A lane's part of the rotation at one position: its entries of the tables, and the lane of its partners.
template <int PER>
struct Turn {
  Row<PER> c, s;          // s negative in the first half
  int from;
  bool in;

  __device__ __forceinline__ void load(const Kv4AppendArgs& a, int p, int lane) {
    const int h = a.rot / 2, i0 = lane * PER;   // h is a multiple of PER: a lane's values lie on one side of it
    in = i0 < a.rot;
    from = lane;
    if (in) {
      const bool low = i0 < h;
      const int t0 = low ? i0 : i0 - h;
      from = low ? lane + h / PER : lane - h / PER;
      c.load(a.cos + (long)p * h + t0);
      s.load(a.sin + (long)p * h + t0);
#pragma unroll
      for (int j = 0; j < PER / 2; ++j) s.w[j] ^= low ? 0x80008000u : 0u;
    }
  }
  // rotate-half, each product and the sum rounded to bf16 (a sum of two bf16 rounds the same by way of fp32: it is
  // exact there, or too far from its larger term to move it)
  __device__ __forceinline__ void apply(Row<PER>& v) const {
#pragma unroll
    for (int j = 0; j < PER / 2; ++j) {
      const uint32_t x = __shfl_sync(kFull, v.w[j], from);
      const uint32_t y = add_bf16(mul_bf16(v.w[j], c.w[j]), mul_bf16(x, s.w[j]));
      v.w[j] = in ? y : v.w[j];
    }
  }
};

// Head norm of one row of a warp: mode 0 plain, 1 zero-centred.
template <int PER>
__device__ __forceinline__ void norm(Row<PER>& row, const Row<PER>& w, int mode, double eps, bool key) {
  constexpr int HD = 32 * PER;
  if (key) {
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < PER / 2; ++j) {
      const double l = low_double(row.w[j]), h = high_double(row.w[j]);
      ss = fma(h, h, fma(l, l, ss));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
    const Root r(ss * (1.0 / HD) + eps);
#pragma unroll
    for (int j = 0; j < PER / 2; ++j) row.w[j] = r.pair(row.w[j], w.w[j], mode);
  } else {
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) ss = fmaf(row.get(j), row.get(j), ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
    const float inv = rsqrtf(ss / (float)HD + (float)eps);
#pragma unroll
    for (int j = 0; j < PER / 2; ++j) row.w[j] = query_pair(inv, row.w[j], w.w[j], mode);
  }
}

// One row of a warp quantised into row r of its block.
template <int HD, bool IS_V>
__device__ __forceinline__ void put_row(const Row<HD / 32>& row, uint8_t* block, int r, int lane) {
  using L = Kv4L<HD>;
  constexpr int PER = L::PER;
  constexpr int LANES = 32 / PER;   // lanes of a group
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < PER / 2; ++j) top = __vmaxu2(top, row.w[j] & 0x7fff7fffu);
  top = __reduce_max_sync(kFull, max(top & 0xffffu, top >> 16));
  const bool bad = top >= 0x5b80u;   // 2^56 and above, infinities and NaN
  const int e = max(-kKv4Limit, min(kKv4Limit, (int)(top >> 7) - 127));
  Row<PER> v = row;
  if (bad)
#pragma unroll
    for (int j = 0; j < PER / 2; ++j) v.w[j] = 0;
  float lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) lo = fminf(lo, v.get(j)), hi = fmaxf(hi, v.get(j));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(kFull, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(kFull, hi, o));
  }
  const Steps st(lo, hi, kv4_pow2(-e));
  uint32_t codes;
  st.codes<PER>(v.w, &codes);
  const int i = lane / LANES, in = lane % LANES;   // group, lane in it
  if constexpr (!IS_V) {
    if constexpr (PER == 8)
      *reinterpret_cast<uint32_t*>(block + L::k_word(r, in, i)) = codes;
    else if constexpr (PER == 4)
      *reinterpret_cast<uint16_t*>(block + L::k_word(r, in / 2, i) + 2 * (in & 1)) = (uint16_t)codes;
    else
      block[L::k_word(r, in / 4, i) + (in & 3)] = (uint8_t)codes;
  } else {
    if constexpr (PER == 8) {
      *reinterpret_cast<uint16_t*>(block + L::v_chunk(r, 2 * in) + 2 * i) = (uint16_t)codes;
      *reinterpret_cast<uint16_t*>(block + L::v_chunk(r, 2 * in + 1) + 2 * i) = (uint16_t)(codes >> 16);
    } else if constexpr (PER == 4) {
      *reinterpret_cast<uint16_t*>(block + L::v_chunk(r, in) + 2 * i) = (uint16_t)codes;
    } else {
      block[L::v_chunk(r, in / 2) + 2 * i + (in & 1)] = (uint8_t)codes;
    }
  }
  if (in == 0) {
    const int at = IS_V ? i * 16 + kv4_slot(r) : r * L::NG + i;
    reinterpret_cast<__half*>(block + (IS_V ? L::VS : L::KS))[at] = st.s;
    reinterpret_cast<__half*>(block + (IS_V ? L::VM : L::KM))[at] = st.m;
  }
  if (lane == 0) block[(IS_V ? L::VE : L::KE) + r] = (uint8_t)(bad ? kKv4Mark : e + 127);
}

// A warp a row and head. Warps of a block: 8 rows of one head (down 0), or 8 heads of one row (few rows: down 1). Bound by
// latency: a row's load, the tables' entries, two to four reductions across the warp. B200: 16 rows of 24 + 4 heads of 256
// with norms 3.1 us, 128 rows of 32 + 8 heads of 128 3.2 us.
template <int HD>
__global__ void __launch_bounds__(256)
    kv4_append_kernel(const __grid_constant__ Kv4AppendArgs a, int r0, int rows, int down) {
  constexpr int PER = HD / 32;
  allow_next();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = a.hq + 2 * a.c.hkv;
  const int n = down ? blockIdx.x : blockIdx.x * 8 + warp;   // row of this launch
  const int head = down ? blockIdx.y * 8 + warp : blockIdx.y, kh = head - a.hq;
  if (n >= rows || head >= heads) return;
  const int sq = a.T == 1 ? n : n < a.T ? 0 : n / a.T, t = n - sq * a.T;
  const int src_row = r0 * a.T + n;
  Row<PER> v, w;
  v.load(a.src + (long)src_row * a.src_row + lane * PER + (kh < 0 ? head * a.q_stride : a.k_col + kh * HD));
  const bool normed = kh < a.c.hkv && a.norm_mode >= 0;
  if (normed) w.load((kh < 0 ? a.q_norm : a.k_norm) + lane * PER);
  const int first = a.row0 != nullptr ? __ldg(a.row0 + r0 + sq) : a.row0_host;
  const long at = (long)first + t;
  const int row = (int)at;
  const int p = a.pos != nullptr ? __ldg(a.pos + src_row) : a.pos_offset >= 0 ? a.pos_offset + t : row;
  const bool skip = first < 0;
  const bool ok = !skip && at < a.c.rows[sq] && (a.rot == 0 || (p >= 0 && p < a.table_rows));
  uint8_t* block = nullptr;
  if (kh >= 0) {
    if (ok) {
      const int page = a.page_shift >= 0 ? row >> a.page_shift : row / a.c.page_size;
      const int id = __ldg(a.c.pages[sq] + page);
      const int g = kh < a.c.hkv ? kh : kh - a.c.hkv;
      if (id >= 0 && id < a.c.num_pages)
        block = a.c.pool +
                (((long)id * a.c.hkv + g) * (a.c.page_size / 16) + ((row - page * a.c.page_size) >> 4)) * Kv4L<HD>::BYTES;
    }
    if (block == nullptr) {
      if (!skip && lane == 0) record_error(a.err, kErrBadIndex);
      return;
    }
  }
  Turn<PER> turn;
  turn.in = false, turn.from = lane;
  if (ok && a.rot > 0 && kh < a.c.hkv) turn.load(a, p, lane);
  if (normed) norm<PER>(v, w, a.norm_mode, a.eps, kh >= 0);
  if (a.rot > 0 && kh < a.c.hkv) turn.apply(v);
  if (kh < 0) {
    if (!ok)
#pragma unroll
      for (int j = 0; j < PER / 2; ++j) v.w[j] = 0;
    v.store(a.q_out + (long)src_row * a.q_out_row + (long)head * a.q_out_head + lane * PER);
  } else if (kh < a.c.hkv) {
    put_row<HD, false>(v, block, row & 15, lane);
  } else {
    put_row<HD, true>(v, block, row & 15, lane);
  }
}

// Many rows: the queries and the cached rows go their own ways in one launch (kv4_append_rows_kernel).
//
// query_rows            a lane holds 8 values (16 bytes), so a warp's loads and stores are whole sectors whatever the head
//                       size: 256 / hd heads of a row at a time. The rotation's half is whole lanes (rot / 2 a multiple of
//                       8).
// cache_block           a CTA per block of 16 cache rows and 512 / hd heads of K or of V, a warp two rows: a lane holds 16
//                       values (half a group), hd / 16 lanes a head, so what is done once a head or a group is done for all
//                       its heads at once; the block's bytes are put together in shared memory and leave as 16-byte pieces
//                       (row by row they would be 24 partial sectors a row and head). A block that is only partly appended
//                       is written in place, row by row. The rotation's half is whole lanes (rot / 2 a multiple of 16).
//
// Both load the rows, the page's id and the rotation's entries before anything waits for one of them (80 -> 72 us for the
// queries; behind one another each costs a trip to memory with 32 warps an SM to cover it). What is above the bytes is the
// cached rows' arithmetic (16 values of a lane: 190 instructions, 86 of them the codes), a chain that 28 warps an SM do not
// cover: issue slots 61 to 70 % busy, DRAM 30 to 58 %, so neither is at its limit. B200, 16384 rows: 32 q and 8 KV heads of
// 128 72 us (356 MB: 54 at the measured 6.55 TB/s), the KV heads alone 35 (88 MB: 13.5); 24 gated and 4 of 256 with norms
// 109 us (491 MB: 75). Tried: row pieces through a ring of asynchronous copies (equal), the next wave's rows fetched to L2
// ahead (84 us), 3 CTAs an SM of 80 registers (82 us).

// kept out of line: the common cases branch past it
__device__ __noinline__ int divide(int a, int b) { return a / b; }

struct Place {
  int row, p;   // cache row (negative: the sequence is skipped), rotary position
  bool ok;
};
__device__ __forceinline__ Place place(const Kv4AppendArgs& a, int first, int sq, int t, int src_row) {
  Place f;
  const unsigned row = (unsigned)first + t;   // below 2^32: first < 2^31, t < 2^30
  f.p = a.pos != nullptr ? __ldg(a.pos + src_row) : a.pos_offset >= 0 ? a.pos_offset + t : (int)row;
  f.ok = first >= 0 && row < (unsigned)a.c.rows[sq] && (a.rot == 0 || (unsigned)f.p < (unsigned)a.table_rows);
  f.row = first < 0 ? -1 : (int)(row & 0x7fffffffu);
  return f;
}

// A piece of the query rows: a warp takes US rows of YS x 256 / hd heads, their loads in flight together. What is done once
// a row serves as many heads as fit the registers; at hd 64 fewer, since models of such heads have few.
template <int HD>
struct QPiece {
  static constexpr int LANES = HD / 8, HEADS = 32 / LANES, YS = HD == 64 ? 2 : 4, US = 4 / YS;
  static constexpr int ROWS = 8 * US, SET = YS * HEADS;
};

template <int HD, int MODE, bool TURN>
__device__ __forceinline__ void query_rows(const Kv4AppendArgs& a, int r0, int rows, int x, int set) {
  using Q = QPiece<HD>;
  constexpr int LANES = Q::LANES, HEADS = Q::HEADS, YS = Q::YS, US = Q::US;
  const int lane = threadIdx.x & 31, j = lane % LANES;
  const int n0 = x * Q::ROWS + (threadIdx.x >> 5);
  if (n0 >= rows) return;
  const int head = set * Q::SET + lane / LANES;   // and HEADS, 2 HEADS, .. further
  Row<8> v[US][YS], w;
#pragma unroll
  for (int u = 0; u < US; ++u) {
    const int src_row = r0 * a.T + min(n0 + 8 * u, rows - 1);
    const __nv_bfloat16* src = a.src + (long)src_row * a.src_row + 8 * j;
#pragma unroll
    for (int y = 0; y < YS; ++y) v[u][y].load(src + (head + y * HEADS < a.hq ? (head + y * HEADS) * a.q_stride : 0));
  }
  if constexpr (MODE >= 0) w.load(a.q_norm + 8 * j);
  const int h = a.rot / 2, i0 = 8 * j;
  const bool low = i0 < h;
  Turn<8> turn[US];
  Place f[US];
#pragma unroll
  for (int u = 0; u < US; ++u) {
    const int n = min(n0 + 8 * u, rows - 1);
    int sq = 0, t = n;
    if (t >= a.T) sq = divide(n, a.T), t = n - sq * a.T;
    f[u] = place(a, a.row0 != nullptr ? __ldg(a.row0 + r0 + sq) : a.row0_host, sq, t, r0 * a.T + n);
    turn[u].in = i0 < a.rot;
    turn[u].from = !turn[u].in ? lane : low ? lane + h / 8 : lane - h / 8;
    if constexpr (TURN) {
      const long entry = f[u].ok && turn[u].in ? (long)f[u].p * h + (low ? i0 : i0 - h) : 0;
      turn[u].c.load(a.cos + entry);
      turn[u].s.load(a.sin + entry);
    }
  }
#pragma unroll
  for (int u = 0; u < US; ++u) {
    const int n = n0 + 8 * u;
    if (n >= rows) break;
    const int src_row = r0 * a.T + n;
    if constexpr (TURN) {
#pragma unroll
      for (int z = 0; z < 4; ++z) turn[u].s.w[z] ^= low ? 0x80008000u : 0u;
    }
    __nv_bfloat16* dst = a.q_out + (long)src_row * a.q_out_row + (long)head * a.q_out_head + 8 * j;
#pragma unroll
    for (int y = 0; y < YS; ++y) {
      Row<8>& q = v[u][y];
      if constexpr (MODE >= 0) {
        // the sums of the hd / 32 values that a lane holds when a warp takes one head, added across in that order too:
        // the same bits as there
        constexpr int PARTS = 256 / HD, PER = HD / 32;
        float ss[PARTS];
#pragma unroll
        for (int y = 0; y < PARTS; ++y) {
          ss[y] = 0.f;
#pragma unroll
          for (int z = 0; z < PER; ++z) ss[y] = fmaf(q.get(y * PER + z), q.get(y * PER + z), ss[y]);
#pragma unroll
          for (int o = LANES / 2; o > 0; o >>= 1) ss[y] += __shfl_xor_sync(kFull, ss[y], o);
        }
#pragma unroll
        for (int o = PARTS / 2; o > 0; o >>= 1)
#pragma unroll
          for (int y = 0; y < o; ++y) ss[y] += ss[y + o];
        const float inv = rsqrtf(ss[0] / (float)HD + (float)a.eps);
#pragma unroll
        for (int y = 0; y < 4; ++y) q.w[y] = query_pair(inv, q.w[y], w.w[y], MODE);
      }
      if constexpr (TURN) turn[u].apply(q);
      if (!f[u].ok) q.w[0] = q.w[1] = q.w[2] = q.w[3] = 0;
      if (head + y * HEADS < a.hq) q.store(dst + (long)(y * HEADS) * a.q_out_head);
    }
  }
}

// 16 values of a lane in place of Turn: entries of the tables at one position, loaded while the row before is quantised.
struct Turn16 {
  uint4 c[2], s[2];
  int at, from;            // first entry, lane of the partners
  bool inside;
  uint32_t sign;           // -1 in the first half, as bf16 pairs

  __device__ __forceinline__ Turn16(int rot, int lane, int j) {
    const int half = rot / 32;                 // lanes of half the rotated values
    const bool low = j < half;
    inside = j < 2 * half;
    at = !inside ? 0 : 16 * (low ? j : j - half);
    from = !inside ? lane : low ? lane + half : lane - half;
    sign = low ? 0xbf80bf80u : 0x3f803f80u;
  }
  __device__ __forceinline__ void load(const Kv4AppendArgs& a, int p) {
    const long e = (long)p * (a.rot / 2) + at;
    const uint4* cp = reinterpret_cast<const uint4*>(a.cos + e);
    const uint4* sp = reinterpret_cast<const uint4*>(a.sin + e);
    c[0] = __ldg(cp), c[1] = __ldg(cp + 1), s[0] = __ldg(sp), s[1] = __ldg(sp + 1);
  }
  __device__ __forceinline__ void apply(uint32_t (&v)[8]) const {
    const uint32_t cw[8] = {c[0].x, c[0].y, c[0].z, c[0].w, c[1].x, c[1].y, c[1].z, c[1].w};
    const uint32_t sw[8] = {s[0].x, s[0].y, s[0].z, s[0].w, s[1].x, s[1].y, s[1].z, s[1].w};
#pragma unroll
    for (int x = 0; x < 8; ++x) {
      const uint32_t other = __shfl_sync(kFull, v[x], from);
      const uint32_t y = fma_bf16(mul_bf16(other, sw[x]), sign, mul_bf16(v[x], cw[x]));   // a product with +-1 is exact
      v[x] = inside ? y : v[x];
    }
  }
};

// One row of a warp's heads of K (or V), quantised to `block`, its head's block.
template <int HD, bool IS_V>
__device__ __forceinline__ void put_heads(uint32_t (&v)[8], uint8_t* block, bool there, int r, int lane) {
  using L = Kv4L<HD>;
  constexpr int LANES = HD / 16;
  const int j = lane % LANES;                  // lane of its head
  // the group's ends over its two lanes, and from them the head's largest magnitude; NaN is kept on the way
  uint32_t least = v[0], most = v[0];
#pragma unroll
  for (int x = 1; x < 8; ++x) least = min_bf16(least, v[x]), most = max_bf16(most, v[x]);
  least = min_bf16(least, __shfl_xor_sync(kFull, least, 1));
  most = max_bf16(most, __shfl_xor_sync(kFull, most, 1));
  unsigned top = __vmaxu2(least & 0x7fff7fffu, most & 0x7fff7fffu);
  top = max(top & 0xffffu, top >> 16);
#pragma unroll
  for (int o = LANES / 2; o > 1; o >>= 1) top = max(top, __shfl_xor_sync(kFull, top, o));
  const bool bad = top >= 0x5b80u;             // 2^56 and above, infinities and NaN
  if (bad) {
    least = most = 0;
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = 0;
  }
  const int e = max(-kKv4Limit, min(kKv4Limit, (int)(top >> 7) - 127));
  const Steps st(fminf(bf16_lo(least), bf16_hi(least)), fmaxf(bf16_lo(most), bf16_hi(most)), kv4_pow2(-e));
  uint32_t codes[2];
  st.codes<16>(v, codes);
  if (!there) return;
  const int i = j / 2, side = j & 1;
  if constexpr (!IS_V) {
    *reinterpret_cast<uint32_t*>(block + L::k_word(r, 2 * side, i)) = codes[0];
    *reinterpret_cast<uint32_t*>(block + L::k_word(r, 2 * side + 1, i)) = codes[1];
  } else {
#pragma unroll
    for (int x = 0; x < 4; ++x)
      *reinterpret_cast<uint16_t*>(block + L::v_chunk(r, 4 * side + x) + 2 * i) = (uint16_t)(codes[x / 2] >> (16 * (x & 1)));
  }
  // one lane of the group writes s, the other m (hd / 2 halves further)
  __half* params = reinterpret_cast<__half*>(block + (IS_V ? L::VS : L::KS));
  params[(IS_V ? i * 16 + kv4_slot(r) : r * L::NG + i) + side * (HD / 2)] = side ? st.m : st.s;
  if (j == 0) block[(IS_V ? L::VE : L::KE) + r] = (uint8_t)(bad ? kKv4Mark : e + 127);
}

template <int HD, bool IS_V, int MODE, bool TURN>
__device__ __forceinline__ void cache_block(uint8_t* image, const Kv4AppendArgs& a, int r0, int sq, int x, int set) {
  using L = Kv4L<HD>;
  constexpr int LANES = HD / 16, HEADS = 32 / LANES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int head = set * HEADS + lane / LANES;
  const bool there = head < a.c.hkv;
  const int first = a.row0 != nullptr ? __ldg(a.row0 + r0 + sq) : a.row0_host;
  if (first < 0) return;
  const int block0 = first / 16 + x;           // the block of the sequence
  const long behind = (long)block0 * 16 - first;
  if (behind >= a.T || (long)block0 * 16 >= (1l << 31)) return;
  const int t0 = (int)behind;                  // above -16: row r of the block is row t0 + r of the call
  const int src0 = (r0 + sq) * a.T;
  const int per = a.c.page_size / 16;
  const int nth = a.page_shift >= 0 ? block0 >> (a.page_shift - 4) : divide(block0, per);
  int id = -1;
  if (block0 * 16 < a.c.rows[sq]) id = __ldg(a.c.pages[sq] + nth);
  const __nv_bfloat16* src = a.src + a.k_col + ((there ? head : 0) + (IS_V ? a.c.hkv : 0)) * HD + 16 * (lane % LANES);
  uint32_t v[2][8];
  const int p0 = a.pos_offset >= 0 ? a.pos_offset + t0 : block0 * 16;
  int p[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int r = warp + 8 * u, t = t0 + r, src_row = src0 + (t >= 0 && t < a.T ? t : 0);
    const uint4* at = reinterpret_cast<const uint4*>(src + (long)src_row * a.src_row);
    const uint4 y = __ldg(at), z = __ldg(at + 1);
    v[u][0] = y.x, v[u][1] = y.y, v[u][2] = y.z, v[u][3] = y.w, v[u][4] = z.x, v[u][5] = z.y, v[u][6] = z.z, v[u][7] = z.w;
    p[u] = a.pos != nullptr ? __ldg(a.pos + src_row) : p0 + r;
  }
  // every row of the block here, within the table and at a rotary position of the tables: through shared memory
  bool whole = t0 >= 0 && t0 + 16 <= a.T && block0 * 16 < a.c.rows[sq];
  if (whole && a.rot > 0)
    whole = a.pos == nullptr ? p0 <= a.table_rows - 16
                             : __all_sync(kFull, (unsigned)__ldg(a.pos + src0 + t0 + (lane & 15)) < (unsigned)a.table_rows);
  Turn16 turn(a.rot, lane, lane % LANES);
  if constexpr (TURN) turn.load(a, (unsigned)p[0] < (unsigned)a.table_rows ? p[0] : 0);
  const int pitch = per * L::BYTES;            // between KV heads (a page of a head is below 2^31 bytes)
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    if constexpr (MODE >= 0) {
      double ss = 0.0, sh = 0.0;
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const double l = low_double(v[u][x]), h = high_double(v[u][x]);
        ss = fma(l, l, ss), sh = fma(h, h, sh);
      }
      ss += sh;
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
      const Root root(ss * (1.0 / HD) + a.eps);
      const uint4* wp = reinterpret_cast<const uint4*>(a.k_norm + 16 * (lane % LANES));
      const uint4 y = __ldg(wp), z = __ldg(wp + 1);
      const uint32_t w[8] = {y.x, y.y, y.z, y.w, z.x, z.y, z.z, z.w};
#pragma unroll
      for (int x = 0; x < 8; ++x) v[u][x] = root.pair(v[u][x], w[x], MODE);
    }
    if constexpr (TURN) {
      turn.apply(v[u]);
      if (u == 0) turn.load(a, (unsigned)p[1] < (unsigned)a.table_rows ? p[1] : 0);
    }
    const int r = warp + 8 * u, t = t0 + r;
    uint8_t* block = image + (lane / LANES) * L::BYTES;
    if (!whole) {                              // row by row, each where it belongs
      if (t < 0 || t >= a.T) continue;
      if (id < 0 || id >= a.c.num_pages || (a.rot > 0 && (unsigned)p[u] >= (unsigned)a.table_rows)) {
        if (lane == 0) record_error(a.err, kErrBadIndex);
        continue;
      }
      block = a.c.pool + ((long)id * a.c.hkv + head) * pitch + (block0 - nth * per) * L::BYTES;
    }
    put_heads<HD, IS_V>(v[u], block, there, r, lane);
  }
  if (!whole) return;
  __syncthreads();
  if (id < 0 || id >= a.c.num_pages) {
    if (threadIdx.x == 0) record_error(a.err, kErrBadIndex);
    return;
  }
  uint8_t* out = a.c.pool + ((long)id * a.c.hkv + set * HEADS) * pitch + (block0 - nth * per) * L::BYTES;
  // K: codes, s and m, exponents; V: the same, each behind K's
  constexpr int CODES = HD / 2, PARAMS = HD / 8, PIECES = CODES + PARAMS + 1;
  const int heads = min(HEADS, a.c.hkv - set * HEADS);
  for (int y = threadIdx.x; y < heads * PIECES; y += 256) {
    const int h = y / PIECES, piece = y - h * PIECES;
    const int at = piece < CODES            ? (IS_V ? L::V : 0) + 16 * piece
                   : piece < CODES + PARAMS ? (IS_V ? L::VS : L::KS) + 16 * (piece - CODES)
                                            : (IS_V ? L::VE : L::KE);
    *reinterpret_cast<uint4*>(out + (long)h * pitch + at) = *reinterpret_cast<const uint4*>(image + h * L::BYTES + at);
  }
}

// n / d for 32-bit n by a product: m = (2^64 + e) / d with e < d makes it n / d + n e / (d 2^64), less than 1 / d above. (The
// compiler's divisions, one of them in 64 bits, were a twelfth of the kernel's instructions.)
struct Divisor {
  unsigned d;
  unsigned long long m;
  explicit Divisor(unsigned d_ = 1) : d(d_), m(d_ == 1 ? 0 : ~0ull / d_ + 1) {}
  __device__ __forceinline__ unsigned of(unsigned n) const { return m == 0 ? n : (unsigned)__umul64hi(n, m); }
};

// Queries (bound by their bytes) and cached rows (bound by their arithmetic) of one call side by side: CTA i takes a block of
// the cache when i kv / (q + kv) reaches its next whole number, else query rows.
struct AppendPlan {
  Divisor q_sets;              // of the queries: sets of heads
  Divisor kv_sets, spans;      // of the cache: 2 x sets of KV heads, blocks of a sequence
  unsigned long long share;    // 2^32 kv / (q + kv), rounded up: i share / 2^32 counts up to kv
};

template <int HD, int MODE, bool TURN>
__global__ void __launch_bounds__(256, 4)
    kv4_append_rows_kernel(const __grid_constant__ Kv4AppendArgs a, int r0, int rows, const AppendPlan plan) {
  __shared__ __align__(16) uint8_t image[512 / HD * Kv4L<HD>::BYTES];
  allow_next();
  const unsigned i = blockIdx.x, at = (unsigned)(i * plan.share >> 32);
  if ((unsigned)((i + 1) * plan.share >> 32) > at) {
    // kv sets of one block side by side: they share the rows of the source
    const unsigned span = plan.kv_sets.of(at), set = at - span * plan.kv_sets.d;
    const unsigned sq = plan.spans.of(span), x = span - sq * plan.spans.d;
    if (set & 1)
      cache_block<HD, true, -1, false>(image, a, r0, sq, x, set / 2);
    else
      cache_block<HD, false, MODE, TURN>(image, a, r0, sq, x, set / 2);
  } else {
    const unsigned q = i - at, n = plan.q_sets.of(q);
    query_rows<HD, MODE, TURN>(a, r0, rows, n, q - n * plan.q_sets.d);
  }
}

// hd / 64 warps take a block, four rows of 256 values (or as many of shorter rows) each; a CTA 4 warps, 256 / hd blocks. So a
// lane has 8 values whatever the head size. Bound by the bytes, nearly all of them the bf16 rows written: B200, 65536 rows
// of 1024 values (4 x 256, 8 x 128, 16 x 64) 58 us of 54 (353 MB at the measured 6.55 TB/s), 16384 rows 16 us of 13.5; a
// warp a block with hd / 32 values a lane took 59, 66 and 81 us.
template <int HD>
struct ReadPlan {
  static constexpr int WARPS = 4, PER_BLOCK = HD / 64, BLOCKS = WARPS / PER_BLOCK;
};

template <int HD>
__global__ void __launch_bounds__(ReadPlan<HD>::WARPS * 32)
    kv4_read_kernel(const __grid_constant__ Kv4ReadArgs a, int r0, int spans, long tasks) {
  using L = Kv4L<HD>;
  using P = ReadPlan<HD>;
  constexpr int PIECES = L::BYTES / 16, STEP = 32 * P::PER_BLOCK;
  constexpr int LANES = HD / 8, ROWS = 32 / LANES;   // lanes of a row, rows of a warp's step
  __shared__ uint4 held[P::BLOCKS][PIECES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int mine = warp / P::PER_BLOCK, part = warp % P::PER_BLOCK;
  const long task = (long)blockIdx.x * P::BLOCKS + mine;
  int lo = 0, hi = 0, t0 = 0, g = 0, sq = 0;         // rows [lo, hi) of the block, in rows of the output behind t0
  const uint8_t* block = nullptr;
  if (task < tasks) {
    const int x = (int)(task % spans), gs = (int)(task / spans);
    g = gs % a.c.hkv, sq = gs / a.c.hkv;
    const int first = a.row0 != nullptr ? __ldg(a.row0 + r0 + sq) : a.row0_host;
    const long row = first < 0 ? 16l * x : (long)(first / 16 + x) * 16;
    t0 = (int)(row - (first < 0 ? 0 : first));
    lo = max(0, -t0), hi = min(16, a.n - t0);
    if (lo < hi && first >= 0) {
      if (row < a.c.rows[sq]) block = kv4_block<HD>(a.c, sq, g, (int)row);
      if (block == nullptr && part == 0 && lane == 0) record_error(a.err, kErrBadIndex);
    }
  }
  if (block != nullptr) {
#pragma unroll
    for (int j = 0; j < (PIECES + STEP - 1) / STEP; ++j) {
      const int piece = part * 32 + lane + j * STEP;
      if (piece < PIECES) held[mine][piece] = __ldg(reinterpret_cast<const uint4*>(block) + piece);
    }
  }
  __syncthreads();
  const uint8_t* b = reinterpret_cast<const uint8_t*>(held[mine]);
  const int j = lane % LANES, i = j / 4, in = j % 4;
  const long at = (long)(r0 + sq) * a.out_seq + (long)g * a.out_head + (long)t0 * HD + 8 * j;
#pragma unroll
  for (int y = 0; y < 4; ++y) {
    const int r = (4 * part + y) * ROWS + lane / LANES;
    if (r < lo || r >= hi) continue;
    uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (block != nullptr) {
      const uint32_t c[2] = {*reinterpret_cast<const uint32_t*>(b + L::k_word(r, in, i)),
                             *reinterpret_cast<const uint16_t*>(b + L::v_chunk(r, 2 * in) + 2 * i) |
                                 (uint32_t)*reinterpret_cast<const uint16_t*>(b + L::v_chunk(r, 2 * in + 1) + 2 * i) << 16};
      const int at_s[2] = {r * L::NG + i, i * 16 + kv4_slot(r)};
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const Two s(__half2float(reinterpret_cast<const __half*>(b + (x ? L::VS : L::KS))[at_s[x]]));
        const Two m(__half2float(reinterpret_cast<const __half*>(b + (x ? L::VM : L::KM))[at_s[x]]));
        const Two size(kv4_size(b[(x ? L::VE : L::KE) + r]));
        // the codes as numbers: 2^23 + c, put together from bytes, minus 2^23
        const uint32_t even = c[x] & 0x0f0f0f0fu, odd = c[x] >> 4 & 0x0f0f0f0fu;
        uint32_t w[4];
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const Two f(__uint_as_float(__byte_perm(even, 0x4b000000u, 0x7440 + z)),
                      __uint_as_float(__byte_perm(odd, 0x4b000000u, 0x7440 + z)));
          float v0, v1;
          mul2(size, fma2(s, add2(f, Two(-8388608.f)), m)).get(v0, v1);
          w[z] = pack_bf16x2(v0, v1);
        }
        out[x] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    *reinterpret_cast<uint4*>(a.k + at + (long)r * HD) = out[0];
    *reinterpret_cast<uint4*>(a.v + at + (long)r * HD) = out[1];
  }
}

template <int HD, int MODE, bool TURN>
void launch_rows(const Kv4AppendArgs& a, int r0, int seqs, cudaStream_t stream) {
  constexpr int HEADS = 512 / HD;
  const int rows = seqs * a.T;
  using Q = QPiece<HD>;
  const unsigned q_sets = (a.hq + Q::SET - 1) / Q::SET, kv_sets = 2 * ((a.c.hkv + HEADS - 1) / HEADS);
  // blocks that T rows can touch: known exactly for a host row, else one more
  const unsigned spans = a.row0 == nullptr ? (unsigned)(((long)a.row0_host + a.T - 1) / 16 - a.row0_host / 16 + 1)
                                           : (unsigned)(a.T + 14) / 16 + 1;
  const unsigned kv = spans * kv_sets * seqs, grid = (unsigned)((rows + Q::ROWS - 1) / Q::ROWS) * q_sets + kv;
  const AppendPlan plan{Divisor(std::max(q_sets, 1u)), Divisor(kv_sets), Divisor(spans),
                        (((unsigned long long)kv << 32) + grid - 1) / grid};
  kv4_append_rows_kernel<HD, MODE, TURN><<<grid, 256, 0, stream>>>(a, r0, rows, plan);
  count_launch();
}

template <int HD>
void launch_append(Kv4AppendArgs a, int r0, int seqs, cudaStream_t stream) {
  const int heads = a.hq + 2 * a.c.hkv, rows = seqs * a.T;
  a.page_shift = -1;
  for (int j = 4; j < 31; ++j)
    if (a.c.page_size == 1 << j) a.page_shift = j;
  // From 256 rows on, in whole blocks' worth, the kernel for many rows; fewer: a warp a row and head, the shorter way through
  // a row. (32 + 8 heads of 128, many / few: 128 rows 3.5 / 3.3 us, 256 rows 4.1 / 4.7, 1024 rows 6.5 / 12.7; 16 sequences
  // of 8 rows 3.6 / 3.5, of 16 rows 3.9 / 5.0. 24 + 4 heads of 256 with norms: 256 rows 5.3 / 5.2, 1024 rows 10.0 / 12.7.)
  // Rotary dims that are no multiple of 32 stay with a warp a row and head whatever the rows, since half of them is no whole
  // number of the other kernel's lanes. (32 + 8 heads of 64 rotated over 16 / 32 dims: 1024 rows 12.2 / 4.9 us, 16384 rows
  // 168 / 35.)
  if (a.T >= 16 && rows >= 256 && a.rot % 32 == 0) {
    switch ((a.norm_mode + 1) * 2 + (a.rot > 0)) {
      case 0: launch_rows<HD, -1, false>(a, r0, seqs, stream); break;
      case 1: launch_rows<HD, -1, true>(a, r0, seqs, stream); break;
      case 2: launch_rows<HD, 0, false>(a, r0, seqs, stream); break;
      case 3: launch_rows<HD, 0, true>(a, r0, seqs, stream); break;
      case 4: launch_rows<HD, 1, false>(a, r0, seqs, stream); break;
      default: launch_rows<HD, 1, true>(a, r0, seqs, stream); break;
    }
    return;
  }
  if (rows < 8)
    kv4_append_kernel<HD><<<dim3(rows, (heads + 7) / 8), 256, 0, stream>>>(a, r0, rows, 1);
  else
    kv4_append_kernel<HD><<<dim3((rows + 7) / 8, heads), 256, 0, stream>>>(a, r0, rows, 0);
  count_launch();
}

template <int HD>
void launch_read(const Kv4ReadArgs& a, int r0, int spans, long tasks, cudaStream_t stream) {
  using P = ReadPlan<HD>;
  const unsigned ctas = (unsigned)((tasks + P::BLOCKS - 1) / P::BLOCKS);
  kv4_read_kernel<HD><<<ctas, P::WARPS * 32, 0, stream>>>(a, r0, spans, tasks);
}

}  // namespace

void kv4_append(const Kv4AppendArgs& a, int r0, int seqs, cudaStream_t stream) {
  if (seqs <= 0 || a.T <= 0) return;
  switch (a.c.hd) {
    case 64: launch_append<64>(a, r0, seqs, stream); break;
    case 128: launch_append<128>(a, r0, seqs, stream); break;
    case 256: launch_append<256>(a, r0, seqs, stream); break;
    default: throw std::runtime_error("kv4_append: head_dim 64 / 128 / 256");
  }
}

void kv4_read(const Kv4ReadArgs& a, int r0, int seqs, cudaStream_t stream) {
  // blocks that n rows can touch: known exactly for a host row, else one more
  const int spans = a.row0 == nullptr ? (a.row0_host + a.n - 1) / 16 - a.row0_host / 16 + 1 : (a.n + 14) / 16 + 1;
  const long tasks = (long)seqs * spans * a.c.hkv;
  if (tasks <= 0 || a.n <= 0) return;
  switch (a.c.hd) {
    case 64: launch_read<64>(a, r0, spans, tasks, stream); break;
    case 128: launch_read<128>(a, r0, spans, tasks, stream); break;
    case 256: launch_read<256>(a, r0, spans, tasks, stream); break;
    default: throw std::runtime_error("kv4_read: head_dim 64 / 128 / 256");
  }
  count_launch();
}

}  // namespace rf
