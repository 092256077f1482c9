// Decode attention over the 4-bit K/V cache: one query row per sequence.
//
// kv4_attn_kernel     grid (key split, KV head, sequence), 4 warps: split s owns keys [s L, (s + 1) L) of the sequence's
//                     rows 0 .. pos, L depending on pos alone (the same bits alone or batched). A warp streams every
//                     4th block of 16 keys through its own ring of bulk copies; no warp waits for another before the
//                     end, where their states are joined in warp order into the split's partial (max, sum, output).
// kv4_combine_kernel  grid (query head, sequence): the splits' partials in split order, the sum's division, the gate.
//
// Both products run on the tensor cores with the cache as the A operand (16 rows) and the G <= 8 query heads as its 8
// columns, so nothing of a tile is wasted on absent query rows, and with the codes as they are stored: a masked nibble
// of a word is the fp16 number c 2^-24 (or 16 c 2^-24 from the odd nibbles; both exact, subnormal), so eight codes cost
// four ANDs and a shift and no conversion. Scales stay outside the products:
//   S_j = 2^(e_q + e_j) (2^24 sum_i s_ji (C_ji . q_i) + sum_i m_ji Q_i),   Q_i the sum of q over group i
//   O   = 2^24 sum_j C_j (P_j s_ji) + sum_j m_ji P_j
// per 32-dim group i: one fp32 FMA a score and group on the K side, one fp16 multiply of P on the V side. The m sums are
// one more product each (Q_i as two fp16 halves of 22 bits together). P takes the V row's size 2^e_j on the way, so
// the running maximum is over S_j + e_j and P and P s stay inside fp16 whatever the rows' sizes; P is at most 2^14,
// and the maximum is raised only when a score would pass that.
#include "kv4.cuh"

#include "kernels.h"

#include <algorithm>
#include <stdexcept>

namespace rf {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 4;
constexpr float kLow = -1e30f;   // below every score: exp2 of a difference to it is 0, never NaN

__host__ __device__ constexpr int split_keys(int p) { return 256 * (p / (256 * kKv4Splits) + 1); }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ float2 unpack_half(uint32_t x) { return __half22float2(*reinterpret_cast<__half2*>(&x)); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// WORDS consecutive 32-bit words of shared memory
template <int WORDS>
__device__ __forceinline__ void lds(const uint8_t* p, uint32_t* w) {
  if constexpr (WORDS == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else if constexpr (WORDS == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

constexpr float kTop = 14.f;    // P <= 2^14
constexpr float kRoom = 6.f;    // a raised maximum leaves P <= 2^6

template <int HD>
struct Warp {
  using L = Kv4L<HD>;
  static constexpr int NG = L::NG;
  uint32_t q[NG][2][2];    // B fragments of the query heads: group, half (even, odd nibbles' dims), register
  uint32_t qs[2];          // their group sums: high and low halves
  float cs[2];             // per column 2t, 2t + 1: scale log2(e) 2^e_q
  float o[NG][2][4];       // output accumulators: group, tile
  float om[4];             // sums of m P
  float ref[2], l[2];

  // query rows [G, HD] of one KV head, as fp16 q 2^-e_q with max |q| 2^-e_q in [2^9, 2^10)
  __device__ __forceinline__ void load_q(const Kv4AttnArgs& a, const __nv_bfloat16* rows, int G, int lane) {
    const int g = lane >> 2, t = lane & 3;
    float v[NG][8];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      if (g < G) kv4_load<8>(rows + (long)g * a.q_head + 32 * i + 8 * t, v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[i][j]) & 0x7fffffffu);
    }
    top = max(top, __shfl_xor_sync(kFull, top, 1));
    top = max(top, __shfl_xor_sync(kFull, top, 2));
    const bool bad = top >= 0x7f800000u;
    const int e = min(max((int)(top >> 23) - 127, -100), 127) - 9;   // q 2^-e; 2^-100 and below keep fewer bits
    const float down = kv4_pow2(-e / 2), down2 = kv4_pow2(-e - -e / 2);
    float sum[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      sum[i] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] = bad ? 0.f : v[i][j] * down * down2;
        sum[i] += v[i][j];
      }
      sum[i] += __shfl_xor_sync(kFull, sum[i], 1);
      sum[i] += __shfl_xor_sync(kFull, sum[i], 2);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        q[i][h][0] = pack_half(v[i][2 * h], v[i][2 * h + 4]);
        q[i][h][1] = pack_half(v[i][2 * h + 1] * 0.0625f, v[i][2 * h + 5] * 0.0625f);
      }
    }
    float a0 = 0.f, a1 = 0.f;
#pragma unroll
    for (int i = 0; i < NG; i += 2)
      if (i == 2 * t) a0 = sum[i], a1 = sum[i + 1];
    qs[0] = pack_half(a0, a1);
    const float2 hi = unpack_half(qs[0]);
    qs[1] = pack_half(a0 - hi.x, a1 - hi.y);
    // the scale of column g sits in lanes 4 g ..; columns 2t, 2t + 1 belong to this lane's scores
    const float c = bad ? __int_as_float(0x7fffffff) : ldexpf(a.scale_log2, e);
    cs[0] = __shfl_sync(kFull, c, 8 * t);
    cs[1] = __shfl_sync(kFull, c, 8 * t + 4);
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][x][j] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) om[j] = 0.f;
    ref[0] = ref[1] = kLow;
    l[0] = l[1] = 0.f;
  }

  // one block of 16 keys; LAST: only its first `live` rows exist (the others' bytes may be anything)
  template <bool LAST>
  __device__ __forceinline__ void block(const uint8_t* b, int live, int lane) {
    const int g = lane >> 2, t = lane & 3;
    // scores: rows g and g + 8, columns 2t and 2t + 1
    constexpr int KW = NG < 4 ? NG : 4;    // words of one load
    float s[4] = {0.f, 0.f, 0.f, 0.f}, cm[4] = {0.f, 0.f, 0.f, 0.f};
    {
      uint32_t ks[2][NG / 2];
#pragma unroll
      for (int r = 0; r < 2; ++r) lds<NG / 2>(b + L::KS + (g + 8 * r) * NG * 2, ks[r]);
#pragma unroll
      for (int i0 = 0; i0 < NG; i0 += KW) {
        uint32_t w[2][KW];
#pragma unroll
        for (int r = 0; r < 2; ++r) lds<KW>(b + L::k_word(g + 8 * r, t, i0), w[r]);
#pragma unroll
        for (int i = i0; i < i0 + KW; ++i) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t x = w[0][i - i0], y = w[1][i - i0];
          mma_f16(acc, x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, q[i][0][0], q[i][0][1]);
          x >>= 8, y >>= 8;
          mma_f16(acc, x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, q[i][1][0], q[i][1][1]);
          const float2 p0 = unpack_half(ks[0][i / 2]), p1 = unpack_half(ks[1][i / 2]);
          const float s0 = i & 1 ? p0.y : p0.x, s1 = i & 1 ? p1.y : p1.x;
          s[0] = fmaf(s0, acc[0], s[0]);
          s[1] = fmaf(s0, acc[1], s[1]);
          s[2] = fmaf(s1, acc[2], s[2]);
          s[3] = fmaf(s1, acc[3], s[3]);
        }
      }
      uint32_t m0 = 0, m1 = 0;
      if (2 * t < NG) {
        m0 = *reinterpret_cast<const uint32_t*>(b + L::KM + g * NG * 2 + 4 * t);
        m1 = *reinterpret_cast<const uint32_t*>(b + L::KM + (g + 8) * NG * 2 + 4 * t);
      }
      mma_f16(cm, m0, m1, m0, m1, qs[0], qs[1]);
    }
    const int ve0 = b[L::VE + g], ve1 = b[L::VE + g + 8];
    const float kz0 = kv4_size(b[L::KE + g]), kz1 = kv4_size(b[L::KE + g + 8]);
    const float nan = __int_as_float(0x7fffffff);
    const float e0 = ve0 == kKv4Mark ? nan : (float)(ve0 - 127), e1 = ve1 == kKv4Mark ? nan : (float)(ve1 - 127);
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = fmaf(s[j], 16777216.f, cm[j]) * ((j < 2 ? kz0 : kz1) * cs[j & 1]);
      y[j] = x + (j < 2 ? e0 : e1);
      if (LAST && g + (j < 2 ? 0 : 8) >= live) y[j] = -INFINITY;
    }
    const bool over = fmaxf(y[0], y[2]) > ref[0] + kTop || fmaxf(y[1], y[3]) > ref[1] + kTop;
    if (__any_sync(kFull, over)) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = fmaxf(y[c], y[c + 2]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, d));
        m = fmaxf(ref[c], m - kRoom);
        const float f = ex2(ref[c] - m);
        ref[c] = m;
        l[c] *= f;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
          for (int x = 0; x < 2; ++x) o[i][x][c] *= f, o[i][x][c + 2] *= f;
        om[c] *= f, om[c + 2] *= f;
      }
    }
    float p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = ex2(y[j] - ref[j & 1]);
    const float iv0 = __int_as_float((254 - min(ve0, 253)) << 23), iv1 = __int_as_float((254 - min(ve1, 253)) << 23);
    l[0] = fmaf(p[0], iv0, fmaf(p[2], iv1, l[0]));
    l[1] = fmaf(p[1], iv0, fmaf(p[3], iv1, l[1]));
    const uint32_t b0 = transpose_8x8(pack_half(p[0], p[1])), b1 = transpose_8x8(pack_half(p[2], p[3]));
    // values: keys 2t, 2t + 1, 2t + 8, 2t + 9; tile x of group i: dims 32 i + 4 g + 2 x (rows g), + 1 (rows g + 8)
    uint32_t keep0 = kFull, keep1 = kFull;
    if constexpr (LAST) {
      keep0 = (2 * t < live ? 0xffffu : 0u) | (2 * t + 1 < live ? 0xffff0000u : 0u);
      keep1 = (2 * t + 8 < live ? 0xffffu : 0u) | (2 * t + 9 < live ? 0xffff0000u : 0u);
    }
    {
      uint32_t m[2] = {0u, 0u};
      if (g < NG) lds<2>(b + L::VM + g * 32 + 8 * t, m);
      if constexpr (LAST) m[0] &= keep0, m[1] &= keep1;
      mma_f16(om, m[0], 0u, m[1], 0u, b0, b1);
    }
    uint32_t w[4][NG / 2];
#pragma unroll
    for (int j = 0; j < 4; ++j) lds<NG / 2>(b + L::v_chunk(2 * t + (j & 1) + 8 * (j >> 1), g), w[j]);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      uint32_t sc[2];
      lds<2>(b + L::VS + i * 32 + 8 * t, sc);
      if constexpr (LAST) sc[0] &= keep0, sc[1] &= keep1;
      const uint32_t c0 = mul_half2(b0, sc[0]), c1 = mul_half2(b1, sc[1]);
      const unsigned pick = i & 1 ? 0x7632 : 0x5410;
      uint32_t x = __byte_perm(w[0][i / 2], w[1][i / 2], pick), z = __byte_perm(w[2][i / 2], w[3][i / 2], pick);
      mma_f16(o[i][0], x & 0x000f000fu, x & 0x00f000f0u, z & 0x000f000fu, z & 0x00f000f0u, c0, c1);
      x >>= 8, z >>= 8;
      mma_f16(o[i][1], x & 0x000f000fu, x & 0x00f000f0u, z & 0x000f000fu, z & 0x00f000f0u, c0, c1);
    }
  }

  // ref [8], l [8] and the outputs [8][HD] of this warp's keys (columns below G)
  __device__ __forceinline__ void store(float* refs, float* ls, float* out, int G, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[c] += __shfl_xor_sync(kFull, l[c], d);
      if (g == 0) refs[2 * t + c] = ref[c], ls[2 * t + c] = l[c];
    }
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float m = __shfl_sync(kFull, om[c], 4 * i + t);
        float4 v;
        v.x = fmaf(o[i][0][c], 16777216.f, m);
        v.y = fmaf(o[i][0][c + 2], 1048576.f, m);
        v.z = fmaf(o[i][1][c], 16777216.f, m);
        v.w = fmaf(o[i][1][c + 2], 1048576.f, m);
        if (2 * t + c < G) *reinterpret_cast<float4*>(out + (2 * t + c) * HD + 32 * i + 4 * g) = v;
      }
  }
};

template <int HD>
struct Cfg {
  static constexpr int STAGES = HD == 256 ? 3 : 4;
  static constexpr int RING = kWarps * STAGES * Kv4L<HD>::BYTES;
  static constexpr int JOIN = kWarps * 8 * HD * 4;     // the warps' outputs, in the ring's place after the last block
  static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

template <int HD>
__global__ void __launch_bounds__(kWarps * 32) kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a, int r0) {
  using L = Kv4L<HD>;
  constexpr int ST = Cfg<HD>::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kWarps][ST];
  __shared__ float refs[kWarps][8], ls[kWarps][8];
  const int s = blockIdx.x, g = blockIdx.y, sq = blockIdx.z, r = r0 + sq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.hq / a.c.hkv;
  const int p = a.pos[r];
  if (p >= a.c.rows[sq]) {
    if (s == 0 && g == 0 && threadIdx.x == 0) record_error(a.err, kErrBadIndex);
    return;
  }
  if (p < 0) return;
  const int keys = split_keys(p), start = s * keys;
  if (start > p) return;
  const int end = min(start + keys, p + 1);
  // blocks warp, warp + 4, ... of the split; lane x of the first ST drives stage x: its barrier, its copies, the page
  // id of the copy after next
  const int blocks = (end - start + 15) / 16;
  uint8_t* ring = smem + warp * ST * L::BYTES;
  uint64_t* bar = bars[warp];
  int mine = warp + kWarps * lane;                 // the block this lane loads next
  int page = 0;                                    // its page
  bool good = false;
  const int* table = a.c.pages[sq];
  auto issue = [&]() {
    const int row = start + 16 * mine;
    good = page >= 0 && page < a.c.num_pages;
    if (good) {
      const long slab = ((long)page * a.c.hkv + g) * (a.c.page_size / 16) + (row % a.c.page_size) / 16;
      mbar_expect_tx(bar + lane, L::BYTES);
      bulk_load(ring + lane * L::BYTES, a.c.pool + slab * L::BYTES, L::BYTES, bar + lane);
    } else {
      record_error(a.err, kErrBadIndex);
      mbar_arrive(bar + lane);
    }
    mine += kWarps * ST;
    if (mine < blocks) page = __ldg(table + (start + 16 * mine) / a.c.page_size);
  };
  if (lane < ST) {
    mbar_init(bar + lane, 1);
    fence_barrier_init();
    if (mine < blocks) {
      page = __ldg(table + (start + 16 * mine) / a.c.page_size);
      issue();
    }
  }
  __syncwarp();
  Warp<HD> w;
  w.load_q(a, a.q + (long)r * a.q_row + (long)g * G * a.q_head, G, lane);
  int stage = 0, phase = 0;
  for (int k = warp; k < blocks; k += kWarps) {
    if (!__all_sync(kFull, mbar_wait(bar + stage, phase, a.err, kErrTimeoutProducer))) {
      for (int j = 0; j < ST && k < blocks; ++j, k += kWarps) {   // no copy may outlive the CTA
        mbar_wait(bar + stage, phase, a.err, kErrTimeoutDrain);
        if (++stage == ST) stage = 0, phase ^= 1;
      }
      break;
    }
    const uint8_t* b = ring + stage * L::BYTES;
    if (__shfl_sync(kFull, good, stage)) {
      const int live = end - start - 16 * k;
      if (live >= 16)
        w.template block<false>(b, 16, lane);
      else
        w.template block<true>(b, live, lane);
    }
    __syncwarp();
    if (lane == stage && mine < blocks) issue();
    if (++stage == ST) stage = 0, phase ^= 1;
  }
  __syncthreads();                                 // every copy has landed: the ring's memory is free
  float* outs = reinterpret_cast<float*>(smem);
  w.store(refs[warp], ls[warp], outs + warp * 8 * HD, G, lane);
  __syncthreads();
  const long base = (((long)r * a.c.hkv + g) * a.splits + s) * G;
  for (int x = threadIdx.x; x < G * HD; x += kWarps * 32) {
    const int h = x / HD;
    float M = refs[0][h], S = 0.f, O = 0.f;
#pragma unroll
    for (int i = 1; i < kWarps; ++i) M = fmaxf(M, refs[i][h]);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float f = exp2f(refs[i][h] - M);
      S = fmaf(ls[i][h], f, S);
      O = fmaf(outs[i * 8 * HD + x], f, O);
    }
    a.part_o[base * HD + x] = O;
    if (x % HD == 0) a.part_ml[(base + h) * 2] = M, a.part_ml[(base + h) * 2 + 1] = S;
  }
}

__global__ void kv4_combine_kernel(Kv4AttnArgs a, int r0) {
  const int HD = blockDim.x, G = a.hq / a.c.hkv;
  const int h = blockIdx.x, sq = blockIdx.y, r = r0 + sq, e = threadIdx.x;
  const int p = a.pos[r];
  float o = 0.f;
  if (p >= 0 && p < a.c.rows[sq]) {
    const int ns = p / split_keys(p) + 1;
    const long base = ((long)r * a.c.hkv + h / G) * a.splits * G + h % G;
    float M = kLow, S = 0.f;
    for (int s = 0; s < ns; ++s) M = fmaxf(M, a.part_ml[(base + (long)s * G) * 2]);
    for (int s = 0; s < ns; ++s) {
      const long i = base + (long)s * G;
      const float f = exp2f(a.part_ml[i * 2] - M);
      S = fmaf(a.part_ml[i * 2 + 1], f, S);
      o = fmaf(a.part_o[i * HD + e], f, o);
    }
    o = S == 0.f ? 0.f : o / S;
    if (a.gate != nullptr) {
      const float z = __bfloat162float(a.gate[(long)r * a.gate_row + (long)h * a.gate_head + e]);
      o *= 1.f / (1.f + __expf(-z));
    }
  }
  a.out[(long)r * a.out_row + (long)h * HD + e] = __float2bfloat16(o);
}

template <int HD>
void launch(const Kv4AttnArgs& a, int r0, int seqs, cudaStream_t stream) {
  const int G = a.hq / a.c.hkv;
  if (G < 1 || G > 8 || a.hq % a.c.hkv) throw std::runtime_error("kv4_attention: 1 to 8 query heads per KV head");
  static PerDeviceOnce once;
  once([] {
    cudaFuncSetAttribute(kv4_attn_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::SMEM);
  });
  kv4_attn_kernel<HD><<<dim3(a.splits, a.c.hkv, seqs), kWarps * 32, Cfg<HD>::SMEM, stream>>>(a, r0);
  count_launch();
  kv4_combine_kernel<<<dim3(a.hq, seqs), HD, 0, stream>>>(a, r0);
  count_launch();
}

}  // namespace

int kv4_splits(int rows) { return rows <= 0 ? 1 : std::min(kKv4Splits, (rows - 1) / 256 + 1); }

void kv4_attention(const Kv4AttnArgs& a, int r0, int seqs, cudaStream_t stream) {
  if (seqs <= 0) return;
  switch (a.c.hd) {
    case 64: launch<64>(a, r0, seqs, stream); break;
    case 128: launch<128>(a, r0, seqs, stream); break;
    case 256: launch<256>(a, r0, seqs, stream); break;
    default: throw std::runtime_error("kv4_attention: head_dim 64 / 128 / 256");
  }
}

}  // namespace rf
