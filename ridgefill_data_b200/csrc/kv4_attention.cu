// Decode attention over the 4-bit K/V cache: one query row per sequence.
//
// kv4_attn_kernel     grid (key split, KV head, sequence), 4 warps: split s owns keys [s L, (s + 1) L) of the sequence's
//                     rows 0 .. pos, L depending on pos alone (the same bits alone or batched). A warp streams every
//                     4th block of 16 keys through its own ring of bulk copies; no warp waits for another before the
//                     end, where their states are joined in warp order into the split's partial (max, sum, output).
// kv4_combine_kernel  grid (query head, sequence): the splits' partials in a fixed order, the sum's division, the gate. Both
//                     start while the kernel before them ends.
//
// Bound by the cache's bytes: inside a CTA's loop DRAM runs at its rate, and what is above the floor is the CTAs' start (3 us:
// position, page ids, query, first block) and join (1.6 us), which the CTAs that share an SM reach together. B200, L2 flushed
// before the call, join included: four streams behind 128K rows of 8 heads of 128 141 us (680 MB: 104 at the measured 6.55
// TB/s), eight behind up to 32K rows of 4 heads of 256 53 us (147 MB: 22), one behind 16K rows of those 20 us (21 MB: 3.2;
// latency: 8 blocks a warp, one after another). Replayed from a graph over the same inputs, of which L2 keeps a part: 131,
// 47 and 16 us.
//
// Both products run on the tensor cores with the cache as the A operand (16 rows) and the G <= 8 query heads as its 8
// columns, so nothing of a tile is wasted on absent query rows, and with the codes as they are stored: a masked nibble
// of a word is the fp16 number c 2^-24 (or 16 c 2^-24 from the odd nibbles; both exact, subnormal), so eight codes cost
// four ANDs and a shift and no conversion. Scales stay outside the products:
//   S_j = 2^(e_q + e_j) (2^24 sum_i s_ji (C_ji . q_i) + sum_i m_ji Q_i),   Q_i the sum of q over group i
//   O   = 2^24 sum_j C_j (P_j s_ji) + sum_j m_ji P_j
// per 32-dim group i: one fp32 FMA a score and group on the K side, one fp16 multiply of P on the V side. The m sums are
// one more product each (Q_i as two fp16 halves of 22 bits together). P takes the V row's size 2^e_j on the way, so
// the running maximum is over S_j + e_j and P and P s stay inside fp16 whatever the rows' sizes (fit_size sees to the rows
// whose stored exponent is not their size); P is at most 2^14, and the maximum is raised only when a score would pass
// that.
//
// Fewer bits than fp32, since the tensor cores take the codes as fp16 beside an fp16 operand: P is rounded to 11 bits for
// the m sums, P s once more for the codes' (subnormal, and with fewer bits, for keys of small weight in a group whose range
// is small beside its row's largest value), the query's group sums to 22. The sum of weights is of the unrounded P, in fp32,
// as are all accumulators. Next to the output's own rounding to bf16 they are small: over four and eight streams of up to
// 128K rows the outputs lie 0.0005 to 0.001 of their norm from a computation in fp32, whose own distance from 64 bits,
// 0.0011 to 0.0032, grows by 2 % at most.
#include "kv4.cuh"

#include "kernels.h"

#include <algorithm>
#include <stdexcept>

namespace rf {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 4;
constexpr float kLow = -1e30f;   // below every score: exp2 of a difference to it is 0, never NaN

// Keys of a split, at least: a CTA's start and join take 4 us beside 1 us a block of each warp, so short splits cost batches
// (256: eight behind up to 32K rows 52 us against 46) and long ones a single stream (1024: 23 us against 16 behind 16K).
constexpr int kUnit = 512;
constexpr int kTile = 128;         // and a multiple of this: every warp whole runs of blocks

// keys of a split of rows 0 .. p when there may be `splits` of them
__host__ __device__ inline int split_keys(int p, int splits) { return max(kUnit, kTile * (p / (kTile * splits) + 1)); }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// the same with a zero accumulator
__device__ __forceinline__ void mma_f16_new(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
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

// out = o / sum * sigmoid(gate) for 4 dims of a head. A sum of -inf (or NaN) tells of a visible row with non-finite
// values; 0 of no row at all.
__device__ __forceinline__ void finish(const Kv4AttnArgs& a, int r, int col, int h, int e, float4 o, float sum) {
  const float n = sum == 0.f ? 0.f : sum > 0.f && sum < INFINITY ? 1.f / sum : __int_as_float(0x7fffffff);
  float g[4] = {n, n, n, n};
  if (a.gate != nullptr) {
    float z[4];
    kv4_load(a.gate + (long)r * a.gate_row + (long)h * a.gate_head + e, z);
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] = n / (1.f + __expf(-z[j]));
  }
  const float v[4] = {o.x * g[0], o.y * g[1], o.z * g[2], o.w * g[3]};
  kv4_store(a.out + (long)r * a.out_row + col, v);
}

constexpr float kTop = 14.f;    // P <= 2^14
constexpr float kRoom = 6.f;    // a raised maximum leaves P <= 2^6

// The query heads of one KV head as B fragments, shared by the CTA's warps.
template <int HD>
struct Query {
  uint2 q[HD / 32][2][32];   // group, half (of 8 dims of a lane: even and odd nibbles), lane
  float scale[8];            // per column: scale log2(e) 2^e_q
  unsigned top[kWarps][8];
  float part[HD / 32][8];    // group sums by column
};

// The query heads [G, HD] of one KV head as fp16 q 2^-e_q with max |q| 2^-e_q in [2^9, 2^10). All warps, each the groups
// it has loaded.
template <int HD>
struct QueryLoad {
  static constexpr int NG = HD / 32, MINE = (NG + kWarps - 1) / kWarps;
  uint4 raw[MINE];

  __device__ __forceinline__ void load(const Kv4AttnArgs& a, const __nv_bfloat16* rows, int G, int warp, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int i = warp + kWarps * j;
      raw[j] = make_uint4(0u, 0u, 0u, 0u);
      if (g < G && i < NG) raw[j] = *reinterpret_cast<const uint4*>(rows + (long)g * a.q_head + 32 * i + 8 * t);
    }
  }

  // the fragments into s; returns this lane's group sums as halves (high, low). Two barriers.
  __device__ __forceinline__ uint2 prepare(Query<HD>& s, float scale_log2, int warp, int lane) const {
    const int g = lane >> 2, t = lane & 3;
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const unsigned w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
      for (int x = 0; x < 4; ++x) top = __vmaxu2(top, w[x] & 0x7fff7fffu);
    }
    top = max(top & 0xffffu, top >> 16);
    top = max(top, __shfl_xor_sync(kFull, top, 1));
    top = max(top, __shfl_xor_sync(kFull, top, 2));
    if (t == 0) s.top[warp][g] = top;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kWarps; ++j) top = max(top, s.top[j][g]);
    const bool bad = top >= 0x7f80u;   // a row with a non-finite value: zeros, and its scale is NaN
    const int e = min(max((int)(top >> 7) - 127, -100), 127) - 9;   // at 2^-100 and below fewer bits are kept
    const float down = kv4_pow2(-e);
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
      const int i = warp + kWarps * j;
      if (i >= NG) break;
      const unsigned w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
      float v[8], sum = 0.f;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        v[2 * x] = bad ? 0.f : bf16_lo(w[x]) * down;
        v[2 * x + 1] = bad ? 0.f : bf16_hi(w[x]) * down;
        sum += v[2 * x] + v[2 * x + 1];
      }
      sum += __shfl_xor_sync(kFull, sum, 1);
      sum += __shfl_xor_sync(kFull, sum, 2);
      if (t == 0) s.part[i][g] = sum;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        s.q[i][h][lane] = make_uint2(pack_half(v[2 * h], v[2 * h + 4]),
                                     pack_half(v[2 * h + 1] * 0.0625f, v[2 * h + 5] * 0.0625f));
    }
    if (warp == 0 && t == 0) s.scale[g] = bad ? __int_as_float(0x7fffffff) : ldexpf(scale_log2, e);
    __syncthreads();
    float a0 = 0.f, a1 = 0.f;
    if (2 * t < NG) a0 = s.part[2 * t][g], a1 = s.part[2 * t + 1][g];
    const uint32_t hi = pack_half(a0, a1);
    const float2 f = unpack_half(hi);
    return make_uint2(hi, pack_half(a0 - f.x, a1 - f.y));
  }
};

// A V row's exponent byte states its size but for
//   rows of 2^41 and more, whose exponent the cache holds to 40: their z reaches 2^16 and their step 2^13.1, past what P
//   leaves in fp16;
//   rows that nothing was appended to, zeros under the new pool's zero byte: l, in units of 2^-e, would overflow.
// Such rows get their own size in the ring before their block's values are used: large ones z below 2, s and m by a power
// of two (exact, or to 2^-25 of a row of size 1), zeros the smallest size. So in every block P s <= 2^14 (4 / 15), and l
// lies between 2^-56 and 2^54 a key. A marked row (255) misfits too and is left as it is.
// Rows below 2^-40 count as of that size, as the cache holds them: from about 2^-50 on their P s loses bits.
__device__ __forceinline__ bool size_misfits(int byte) { return (unsigned)(byte - (127 - kKv4Limit)) >= 2u * kKv4Limit; }

template <int HD>
__device__ __forceinline__ void fit_size(uint8_t* block, int r) {
  using L = Kv4L<HD>;
  __half* s = reinterpret_cast<__half*>(block + L::VS) + kv4_slot(r);
  __half* m = reinterpret_cast<__half*>(block + L::VM) + kv4_slot(r);
  float top = 0.f;
#pragma unroll 1
  for (int i = 0; i < L::NG; ++i) {
    const float low = __half2float(m[16 * i]), high = fmaf(15.f, __half2float(s[16 * i]), low);
    top = fmaxf(top, fmaxf(fabsf(low), fabsf(high)));
  }
  const int byte = block[L::VE + r];
  if (top == 0.f && byte < 127 - kKv4Limit) block[L::VE + r] = 127 - kKv4Limit;
  if (byte == 127 + kKv4Limit && top >= 2.f) {
    const int up = min((__float_as_int(top) >> 23) - 127, 16);
    const float down = kv4_pow2(-up);
#pragma unroll 1
    for (int i = 0; i < L::NG; ++i) {
      s[16 * i] = __float2half_rn(__half2float(s[16 * i]) * down);
      m[16 * i] = __float2half_rn(__half2float(m[16 * i]) * down);
    }
    block[L::VE + r] = (uint8_t)(byte + up);
  }
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the next copy into the ring
}

// The state of a warp over its keys. Fragment layouts as in mma.cuh: lane (g, t) = (lane / 4, lane % 4).
template <int HD>
struct Warp {
  using L = Kv4L<HD>;
  static constexpr int NG = L::NG;
  static constexpr bool kHold = HD != 256;   // the fragments in registers, or read from shared memory at each use
  uint2 held[kHold ? NG : 1][2];
  const Query<HD>* query;
  int lane_;
  uint2 qs;                // group sums
  float cs[2];             // per column 2t, 2t + 1
  float o[NG][2][4];       // output accumulators: group, tile
  float om[4];             // sums of m P
  float ref[2], l[2];

  __device__ __forceinline__ uint2 q(int i, int h) const {
    if constexpr (kHold) return held[i][h];
    return query->q[i][h][lane_];
  }

  __device__ __forceinline__ void start(const Query<HD>& s, uint2 sums, int lane) {
    query = &s;
    lane_ = lane;
    if constexpr (kHold) {
#pragma unroll
      for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) held[i][h] = s.q[i][h][lane];
    }
    qs = sums;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      cs[c] = s.scale[2 * (lane & 3) + c];
      ref[c] = kLow;
      l[c] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[i][x][j] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) om[j] = 0.f;
  }

  // NB blocks of 16 keys at b; LAST: only the first live[u] rows of block u exist (the others' bytes may be anything)
  template <bool LAST, int NB>
  __device__ __forceinline__ void blocks(uint8_t* b, const int (&live)[NB], int lane) {
    const int g = lane >> 2, t = lane & 3;
    bool misfit = false;
    // scores: rows g and g + 8, columns 2t and 2t + 1; y = score + size of the V row (its byte)
    constexpr int KW = NG < 4 ? NG : 4;    // words of one load
    float y[NB][4], iv[NB][2];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const uint8_t* k = b + u * L::BYTES;
      float s[4], cm[4];
      uint32_t ks[2][NG / 2];
#pragma unroll
      for (int r = 0; r < 2; ++r) lds<NG / 2>(k + L::KS + (g + 8 * r) * NG * 2, ks[r]);
#pragma unroll
      for (int i0 = 0; i0 < NG; i0 += KW) {
        uint32_t w[2][KW];
#pragma unroll
        for (int r = 0; r < 2; ++r) lds<KW>(k + L::k_word(g + 8 * r, t, i0), w[r]);
        // the groups' first products, then their second ones: no product waits for the one just issued
        float acc[KW][4];
#pragma unroll
        for (int j = 0; j < KW; ++j) {
          const uint2 f = q(i0 + j, 0);
          mma_f16_new(acc[j], w[0][j] & 0x000f000fu, w[1][j] & 0x000f000fu, w[0][j] & 0x00f000f0u, w[1][j] & 0x00f000f0u,
                      f.x, f.y);
        }
#pragma unroll
        for (int j = 0; j < KW; ++j) {
          const uint2 f = q(i0 + j, 1);
          const uint32_t x = w[0][j] >> 8, z = w[1][j] >> 8;
          mma_f16(acc[j], x & 0x000f000fu, z & 0x000f000fu, x & 0x00f000f0u, z & 0x00f000f0u, f.x, f.y);
        }
#pragma unroll
        for (int j = 0; j < KW; ++j) {
          const int i = i0 + j;
          const float2 p0 = unpack_half(ks[0][i / 2]), p1 = unpack_half(ks[1][i / 2]);
          const float s0 = i & 1 ? p0.y : p0.x, s1 = i & 1 ? p1.y : p1.x;
#pragma unroll
          for (int x = 0; x < 4; ++x)
            s[x] = i == 0 ? (x < 2 ? s0 : s1) * acc[j][x] : fmaf(x < 2 ? s0 : s1, acc[j][x], s[x]);
        }
      }
      uint32_t m0 = 0, m1 = 0;
      if (2 * t < NG) {
        m0 = *reinterpret_cast<const uint32_t*>(k + L::KM + g * NG * 2 + 4 * t);
        m1 = *reinterpret_cast<const uint32_t*>(k + L::KM + (g + 8) * NG * 2 + 4 * t);
      }
      mma_f16_new(cm, m0, m1, m0, m1, qs.x, qs.y);
      // sizes by their bytes: a marked row's 255 makes the K size infinite (its score 0 x inf = NaN) and the V size's
      // inverse -inf, which the sum keeps (or turns to NaN) and the join answers with NaN
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int ve = k[L::VE + g + 8 * r];
        const float kz = __int_as_float(k[L::KE + g + 8 * r] << 23), e = (float)ve;
        iv[u][r] = __int_as_float((254 - ve) << 23);
        misfit |= size_misfits(ve);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          y[u][2 * r + c] = fmaf(fmaf(s[2 * r + c], 16777216.f, cm[2 * r + c]), kz * cs[c], e);
        if (LAST && g + 8 * r >= live[u]) y[u][2 * r] = y[u][2 * r + 1] = -INFINITY, iv[u][r] = 0.f;
      }
    }
    float top[2];
    auto find_top = [&] {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        top[c] = fmaxf(y[0][c], y[0][c + 2]);
#pragma unroll
        for (int u = 1; u < NB; ++u) top[c] = fmaxf(top[c], fmaxf(y[u][c], y[u][c + 2]));
      }
    };
    find_top();
    if (__any_sync(kFull, misfit || top[0] > ref[0] + kTop || top[1] > ref[1] + kTop)) {
      if (__any_sync(kFull, misfit)) {
        float was[NB][2];
#pragma unroll
        for (int u = 0; u < NB; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) was[u][r] = (float)b[u * L::BYTES + L::VE + g + 8 * r];
        __syncwarp();
        if (lane < 16 * NB) fit_size<HD>(b + (lane >> 4) * L::BYTES, lane & 15);
        __syncwarp();
#pragma unroll
        for (int u = 0; u < NB; ++u)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int ve = b[u * L::BYTES + L::VE + g + 8 * r];
            y[u][2 * r] += (float)ve - was[u][r], y[u][2 * r + 1] += (float)ve - was[u][r];
            if (iv[u][r] != 0.f) iv[u][r] = __int_as_float((254 - ve) << 23);
          }
        find_top();
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float m = top[c];
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
    uint32_t pb[NB][2];
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      float p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[j] = ex2(y[u][j] - ref[j & 1]);
        l[j & 1] = fmaf(p[j], iv[u][j >> 1], l[j & 1]);
      }
      pb[u][0] = transpose_8x8(pack_half(p[0], p[1]));
      pb[u][1] = transpose_8x8(pack_half(p[2], p[3]));
    }
    // values: keys 2t, 2t + 1, 2t + 8, 2t + 9; tile x of group i: dims 32 i + 4 g + 2 x (rows g), + 1 (rows g + 8)
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      const uint8_t* v = b + u * L::BYTES;
      uint32_t keep[2] = {kFull, kFull};
      if constexpr (LAST) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
          keep[r] = (2 * t + 8 * r < live[u] ? 0xffffu : 0u) | (2 * t + 8 * r + 1 < live[u] ? 0xffff0000u : 0u);
      }
      uint32_t m[2] = {0u, 0u};
      if (g < NG) lds<2>(v + L::VM + g * 32 + 8 * t, m);
      if constexpr (LAST) m[0] &= keep[0], m[1] &= keep[1];
      mma_f16(om, m[0], 0u, m[1], 0u, pb[u][0], pb[u][1]);
      uint32_t w[4][NG / 2];
#pragma unroll
      for (int j = 0; j < 4; ++j) lds<NG / 2>(v + L::v_chunk(2 * t + (j & 1) + 8 * (j >> 1), g), w[j]);
#pragma unroll
      for (int i = 0; i < NG; ++i) {
        uint32_t sc[2];
        lds<2>(v + L::VS + i * 32 + 8 * t, sc);
        if constexpr (LAST) sc[0] &= keep[0], sc[1] &= keep[1];
        const uint32_t c0 = mul_half2(pb[u][0], sc[0]), c1 = mul_half2(pb[u][1], sc[1]);
        const unsigned pick = i & 1 ? 0x7632 : 0x5410;
        uint32_t x = __byte_perm(w[0][i / 2], w[1][i / 2], pick), z = __byte_perm(w[2][i / 2], w[3][i / 2], pick);
        mma_f16(o[i][0], x & 0x000f000fu, x & 0x00f000f0u, z & 0x000f000fu, z & 0x00f000f0u, c0, c1);
        x >>= 8, z >>= 8;
        mma_f16(o[i][1], x & 0x000f000fu, x & 0x00f000f0u, z & 0x000f000fu, z & 0x00f000f0u, c0, c1);
      }
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

// Two blocks a step where the registers allow (hd 64, 128: 147 -> 130 us for four streams behind 128K rows; a second chain
// of dependent instructions beside the first); at hd 256 one, with the query's fragments left in shared memory for 3 CTAs
// an SM. The ring holds what 12 to 24 warps an SM keep in flight: 124 to 185 KB.
template <int HD>
struct Cfg {
  static constexpr int NB = HD == 256 ? 1 : 2;          // blocks of a stage
  static constexpr int STAGES = HD == 256 ? 3 : 2;
  static constexpr int CTAS = HD == 256 ? 3 : HD == 128 ? 4 : 6;   // on an SM: its registers bound the compiler's
  static constexpr int RING = kWarps * STAGES * NB * Kv4L<HD>::BYTES;
  static constexpr int JOIN = kWarps * 8 * HD * 4;     // the warps' outputs, in the ring's place after the last block
  static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

template <int HD>
__global__ void __launch_bounds__(kWarps * 32, Cfg<HD>::CTAS)
    kv4_attn_kernel(const __grid_constant__ Kv4AttnArgs a, int r0) {
  using L = Kv4L<HD>;
  constexpr int ST = Cfg<HD>::STAGES, NB = Cfg<HD>::NB;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint64_t bars[kWarps][ST];
  __shared__ float refs[kWarps][8], ls[kWarps][8];
  __shared__ Query<HD> query;
  const int s = blockIdx.x, g = blockIdx.y, sq = blockIdx.z, r = r0 + sq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.hq / a.c.hkv;
  if (lane < ST) mbar_init(bars[warp] + lane, NB);
  fence_barrier_init();
  allow_next();
  wait_previous();      // the previous kernel may have written any of this: rows, queries, positions, tables
  const int p = a.pos[r];
  if (p < 0 || p >= a.c.rows[sq]) {
    if (s > 0) return;
    if (p >= 0 && g == 0 && threadIdx.x == 0) record_error(a.err, kErrBadIndex);
    for (int x = threadIdx.x; x < G * HD / 4; x += kWarps * 32)
      kv4_store(a.out + (long)r * a.out_row + g * G * HD + 4 * x, {0.f, 0.f, 0.f, 0.f});
    return;
  }
  const int keys = split_keys(p, a.most), start = s * keys;
  if (start > p) return;
  const int end = min(start + keys, p + 1);
  // the split's blocks in runs of NB: runs warp, warp + 4, ... Lane x of the first ST NB drives slot x of the ring: its
  // copies, its share of the stage's barrier, and the page id of the copy after next
  const int blocks = (end - start + 15) / 16;
  uint8_t* ring = smem + warp * ST * NB * L::BYTES;
  uint64_t* bar = bars[warp];
  int mine = NB * (warp + kWarps * (lane / NB)) + lane % NB;   // the block this lane loads next: block `in` of page
  const int per = a.c.page_size / 16;                          // `page`, whose id is fetched one turn ahead
  const int first = start / 16 + mine;
  int page = first / per, in = first % per, id = -1;
  const int step = NB * kWarps * ST / per, left = NB * kWarps * ST % per;
  const int* table = a.c.pages[sq];
  const long head = (long)g * per;
  bool good = false;
  auto issue = [&]() {
    uint64_t* full = bar + lane / NB;
    good = mine < blocks;
    if (good && (id < 0 || id >= a.c.num_pages)) {
      record_error(a.err, kErrBadIndex);
      good = false;
    }
    if (good) {
      mbar_expect_tx(full, L::BYTES);
      bulk_load(ring + lane * L::BYTES, a.c.pool + ((long)id * a.c.hkv * per + head + in) * L::BYTES, L::BYTES, full);
    } else {
      mbar_arrive(full);
    }
    mine += NB * kWarps * ST;
    page += step, in += left;
    if (in >= per) in -= per, ++page;
    if (mine < blocks) id = table[page];
  };
  __syncwarp();
  if (lane < ST * NB && mine < blocks) id = table[page];
  QueryLoad<HD> loading;
  loading.load(a, a.q + (long)r * a.q_row + (long)g * G * a.q_head, G, warp, lane);
  if (lane < ST * NB && mine - lane % NB < blocks) issue();
  __syncwarp();
  const uint2 sums = loading.prepare(query, a.scale_log2, warp, lane);
  Warp<HD> w;
  w.start(query, sums, lane);
  int stage = 0, phase = 0;
  for (int k = NB * warp; k < blocks; k += NB * kWarps) {
    if (!__all_sync(kFull, mbar_wait(bar + stage, phase, a.err, kErrTimeoutProducer))) {
      for (int j = 0; j < ST && k < blocks; ++j, k += NB * kWarps) {   // no copy may outlive the CTA
        mbar_wait(bar + stage, phase, a.err, kErrTimeoutDrain);
        if (++stage == ST) stage = 0, phase ^= 1;
      }
      break;
    }
    uint8_t* b = ring + stage * NB * L::BYTES;
    const unsigned loaded = __ballot_sync(kFull, good) >> (stage * NB);
    int live[NB];
    bool full = true;
#pragma unroll
    for (int u = 0; u < NB; ++u) {
      live[u] = loaded >> u & 1 ? end - start - 16 * (k + u) : 0;
      full = full && live[u] >= 16;
    }
    if (full)
      w.template blocks<false, NB>(b, live, lane);
    else
      w.template blocks<true, NB>(b, live, lane);
    __syncwarp();
    if (lane / NB == stage && mine - lane % NB < blocks) issue();
    if (++stage == ST) stage = 0, phase ^= 1;
  }
  __syncthreads();                                 // every copy has landed: the ring's memory is free
  float* outs = reinterpret_cast<float*>(smem);
  w.store(refs[warp], ls[warp], outs + warp * 8 * HD, G, lane);
  __syncthreads();
  const long base = (((long)r * a.c.hkv + g) * a.splits + s) * G;
  const bool only = p < keys;                      // one split holds every row: its join is the output
  if (threadIdx.x < G) {                           // the warps' weights in place of their references
    const int h = threadIdx.x;
    float M = refs[0][h], S = 0.f;
#pragma unroll
    for (int i = 1; i < kWarps; ++i) M = fmaxf(M, refs[i][h]);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float f = ex2(refs[i][h] - M);
      S = fmaf(ls[i][h], f, S);
      refs[i][h] = f;
    }
    ls[0][h] = S;
    if (!only) *reinterpret_cast<float2*>(a.part_ml + (base + h) * 2) = make_float2(M, S);
  }
  __syncthreads();
  for (int x = threadIdx.x; x < G * HD / 4; x += kWarps * 32) {
    const int h = x / (HD / 4);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      const float f = refs[i][h];
      const float4 v = reinterpret_cast<const float4*>(outs + i * 8 * HD)[x];
      sum.x = fmaf(v.x, f, sum.x), sum.y = fmaf(v.y, f, sum.y);
      sum.z = fmaf(v.z, f, sum.z), sum.w = fmaf(v.w, f, sum.w);
    }
    if (only)
      finish(a, r, (g * G) * HD + 4 * x, g * G + h, 4 * x - h * HD, sum, ls[0][h]);
    else
      reinterpret_cast<float4*>(a.part_o + base * HD)[x] = sum;
  }
}

constexpr int kJoin = 8;    // split lanes of the combine: thread (x, y) sums float4 x of splits y, y + kJoin, ...

template <int HD>
__global__ void __launch_bounds__(HD / 4 * kJoin) kv4_combine_kernel(const __grid_constant__ Kv4AttnArgs a, int r0) {
  __shared__ float f[kKv4Splits];
  __shared__ float4 part[kJoin][HD / 4];
  const int G = a.hq / a.c.hkv;
  const int h = blockIdx.x, sq = blockIdx.y, r = r0 + sq;
  const int x = threadIdx.x % (HD / 4), y = threadIdx.x / (HD / 4);
  wait_previous();
  allow_next();
  const int p = a.pos[r];
  if (p >= a.c.rows[sq] || p < kUnit) return;   // no row, or one split: written by it
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  float S = 0.f;
  const int ns = p / split_keys(p, a.most) + 1;
  const long base = ((long)r * a.c.hkv + h / G) * a.splits * G + h % G;
  // every warp finds the largest maximum and the sum; the split's weight for all from the first
  const int lane = threadIdx.x & 31;
  float m[kKv4Splits / 32], l[kKv4Splits / 32], M = kLow;
#pragma unroll
  for (int j = 0; j < kKv4Splits / 32; ++j) {
    const int s = lane + 32 * j;
    const float2 ml = s < ns ? *reinterpret_cast<const float2*>(a.part_ml + (base + (long)s * G) * 2) : make_float2(kLow, 0.f);
    m[j] = ml.x, l[j] = ml.y;
    M = fmaxf(M, m[j]);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(kFull, M, d));
#pragma unroll
  for (int j = 0; j < kKv4Splits / 32; ++j) {
    const float w = exp2f(m[j] - M);
    S = fmaf(l[j], w, S);
    if (threadIdx.x < 32) f[lane + 32 * j] = w;
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) S += __shfl_xor_sync(kFull, S, d);
  __syncthreads();
#pragma unroll 4
  for (int s = y; s < ns; s += kJoin) {
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + (base + (long)s * G) * HD + 4 * x);
    o.x = fmaf(v.x, f[s], o.x), o.y = fmaf(v.y, f[s], o.y), o.z = fmaf(v.z, f[s], o.z), o.w = fmaf(v.w, f[s], o.w);
  }
  part[y][x] = o;
  __syncthreads();
  if (y > 0) return;
#pragma unroll
  for (int j = 1; j < kJoin; ++j) {
    const float4 v = part[j][x];
    o.x += v.x, o.y += v.y, o.z += v.z, o.w += v.w;
  }
  finish(a, r, h * HD + 4 * x, h, 4 * x, o, S);
}

template <int HD>
void launch(const Kv4AttnArgs& a, int r0, int seqs, cudaStream_t stream) {
  const int G = a.hq / a.c.hkv;
  if (G < 1 || G > 8 || a.hq % a.c.hkv) throw std::runtime_error("kv4_attention: 1 to 8 query heads per KV head");
  static PerDeviceOnce once;
  once([] {
    cudaFuncSetAttribute(kv4_attn_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<HD>::SMEM);
  });
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.splits, a.c.hkv, seqs);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = Cfg<HD>::SMEM;
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kv4_attn_kernel<HD>, a, r0) != cudaSuccess)
    throw std::runtime_error("kv4_attention: launch failed");
  count_launch();
  if (a.splits > 1) {
    cfg.gridDim = dim3(a.hq, seqs);
    cfg.blockDim = dim3(HD / 4 * kJoin);
    cfg.dynamicSmemBytes = 0;
    if (cudaLaunchKernelEx(&cfg, kv4_combine_kernel<HD>, a, r0) != cudaSuccess)
      throw std::runtime_error("kv4_attention: launch of the join failed");
    count_launch();
  }
}

}  // namespace

// As many splits as the KV heads of one long sequence need to fill the GPU once (148 SMs of Cfg::CTAS each), in steps of 32
// from 64 to kKv4Splits: by the model's shape alone, so the split of a sequence does not depend on the batch. (One
// sequence behind 128K rows of 4 heads of 256: 64 splits 47 us, 111 45 us; four behind 128K rows of 8 heads of 128: 64
// splits 130 us, 74 133 us.)
int kv4_most_splits(int hd, int hkv) {
  const int slots = 148 * (hd == 256 ? Cfg<256>::CTAS : hd == 128 ? Cfg<128>::CTAS : Cfg<64>::CTAS);
  return std::max(64, std::min(kKv4Splits, slots / hkv / 32 * 32));
}

int kv4_splits(int rows, int hd, int hkv) {
  return rows <= 0 ? 1 : std::min(kv4_most_splits(hd, hkv), (rows - 1) / kUnit + 1);
}

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
