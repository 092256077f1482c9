// Append to and read from the 4-bit K/V cache (layout: kv4.cuh).
//
// kv4_append_kernel  one warp per (row, q head | k head | v head), a lane holding hd / 32 consecutive values: head norm
//                    and rotation (q, k), then q goes out in bf16 and k / v rows are quantised into their block.
// kv4_read_kernel    one warp per (row, KV head): the values the codes stand for, rounded once to bf16.
//
// Roundings are the bf16 model's (norm and each step of the rotation round to bf16), so a cached key is the 4-bit form
// of the row the bf16 cache would hold. The norm's sum of squares and its root are taken in 64 bits: products of two
// bf16 are exact there, so the row, and with it every code next to a border, does not depend on the order of the sum.
#include "kv4.cuh"

#include "kernels.h"

#include <stdexcept>

namespace rf {

namespace {

constexpr unsigned kFull = 0xffffffffu;

// Head norm (mode -1 none, 0 plain, 1 zero-centred) and rotate-half RoPE on [0, rot) at position p of one row.
template <int PER>
__device__ __forceinline__ void norm_rope(float (&v)[PER], const __nv_bfloat16* w, const Kv4AppendArgs& a, int p,
                                          int lane) {
  constexpr int HD = 32 * PER;
  const int h = a.rot / 2, i0 = lane * PER;
  float wv[PER], cv[PER], sv[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) wv[j] = cv[j] = sv[j] = 0.f;
  if (a.norm_mode >= 0) kv4_load<PER>(w + i0, wv);
  if (i0 < a.rot) {   // h is a multiple of PER: a lane's values lie on one side of it and inside rot
    const int t0 = i0 < h ? i0 : i0 - h;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      cv[j] = __bfloat162float(a.cos[(long)p * h + t0 + j]);
      sv[j] = __bfloat162float(a.sin[(long)p * h + t0 + j]);
    }
  }
  if (a.norm_mode >= 0) {
    double ss = 0.0;
#pragma unroll
    for (int j = 0; j < PER; ++j) ss += (double)v[j] * (double)v[j];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(kFull, ss, o);
    const double inv = 1.0 / sqrt(ss / HD + a.eps);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const double f = (double)v[j] * inv;
      v[j] = a.norm_mode == 0 ? kv4_bfr(kv4_bfr((float)f) * wv[j]) : kv4_bfr((float)(f * (1.0 + (double)wv[j])));
    }
  }
  if (a.rot > 0) {
    const int loff = h / PER;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const float up = __shfl_down_sync(kFull, v[j], loff);
      const float dn = __shfl_up_sync(kFull, v[j], loff);
      if (i0 + j < a.rot)
        v[j] = i0 + j < h ? kv4_bfr(kv4_bfr(v[j] * cv[j]) + kv4_bfr(-up * sv[j]))
                          : kv4_bfr(kv4_bfr(v[j] * cv[j]) + kv4_bfr(dn * sv[j]));
    }
  }
}

// One row of a warp quantised into row r of its block.
template <int HD, bool IS_V>
__device__ __forceinline__ void put_row(const float (&y)[HD / 32], uint8_t* block, int r, int lane) {
  using L = Kv4L<HD>;
  constexpr int PER = L::PER;
  constexpr int LANES = 32 / PER;   // lanes of a group
  unsigned top = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
  top = __reduce_max_sync(kFull, top);
  const bool bad = top >= 0x5b800000u;   // 2^56 and above, infinities and NaN
  int e = top == 0 ? 0 : (int)(top >> 23) - 127;
  e = max(-kKv4Limit, min(kKv4Limit, e));
  const float size = kv4_pow2(-e);
  float z[PER], lo = INFINITY, hi = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    z[j] = bad ? 0.f : y[j] * size;
    lo = fminf(lo, z[j]);
    hi = fmaxf(hi, z[j]);
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(kFull, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(kFull, hi, o));
  }
  const __half s = __float2half_rn((hi - lo) / 15.f);
  const float mf = __half2float(__float2half_rn(lo)) + 0.f, sf = __half2float(s);   // + 0: a zero is kept as +0
  const __half m = __float2half_rn(mf);
  uint32_t codes = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const float c = sf == 0.f ? 0.f : fminf(fmaxf(rintf((z[j] - mf) / sf), 0.f), 15.f);
    codes |= (uint32_t)c << (4 * j);
  }
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
    reinterpret_cast<__half*>(block + (IS_V ? L::VS : L::KS))[at] = s;
    reinterpret_cast<__half*>(block + (IS_V ? L::VM : L::KM))[at] = m;
  }
  if (lane == 0) block[(IS_V ? L::VE : L::KE) + r] = (uint8_t)(bad ? kKv4Mark : e + 127);
}

template <int HD>
__global__ void __launch_bounds__(256) kv4_append_kernel(Kv4AppendArgs a, int r0, long tasks) {
  constexpr int PER = HD / 32;
  const long task = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (task >= tasks) return;
  const int heads = a.hq + 2 * a.c.hkv;
  const long n = task / heads;             // row of this launch
  const int head = (int)(task % heads);
  const int sq = (int)(n / a.T), t = (int)(n % a.T);
  const long src_row = (long)r0 * a.T + n;
  const int first = a.row0 != nullptr ? __ldg(a.row0 + r0 + sq) : a.row0_host;
  const long row = (long)first + t;
  const int p = a.pos != nullptr ? __ldg(a.pos + src_row) : a.pos_offset >= 0 ? a.pos_offset + t : (int)row;
  const bool skip = first < 0;
  bool ok = !skip && row < a.c.rows[sq] && (a.rot == 0 || (p >= 0 && p < a.table_rows));
  const __nv_bfloat16* src = a.src + src_row * a.src_row;
  if (head < a.hq) {
    float v[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = 0.f;
    if (ok) {
      kv4_load<PER>(src + (long)head * a.q_stride + lane * PER, v);
      norm_rope<PER>(v, a.q_norm, a, p, lane);
    }
    kv4_store<PER>(a.q_out + src_row * a.q_out_row + (long)head * a.q_out_head + lane * PER, v);
  } else {
    const int kh = head - a.hq;
    const int g = kh < a.c.hkv ? kh : kh - a.c.hkv;
    uint8_t* block = ok ? kv4_block<HD>(a.c, sq, g, (int)row) : nullptr;
    if (block == nullptr) {
      if (!skip && lane == 0) record_error(a.err, kErrBadIndex);
      return;
    }
    float v[PER];
    kv4_load<PER>(src + a.k_col + (long)kh * HD + lane * PER, v);
    if (kh < a.c.hkv) {
      norm_rope<PER>(v, a.k_norm, a, p, lane);
      put_row<HD, false>(v, block, (int)row & 15, lane);
    } else {
      put_row<HD, true>(v, block, (int)row & 15, lane);
    }
  }
}

template <int HD>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4ReadArgs a, int r0, long tasks) {
  using L = Kv4L<HD>;
  constexpr int PER = L::PER;
  constexpr int LANES = 32 / PER;
  const long task = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (task >= tasks) return;
  const int t = (int)(task % a.n);
  const int g = (int)(task / a.n % a.c.hkv), sq = (int)(task / a.n / a.c.hkv);
  const int first = a.row0 != nullptr ? __ldg(a.row0 + r0 + sq) : a.row0_host;
  const long row = (long)first + t;
  float kv[PER], vv[PER];
#pragma unroll
  for (int j = 0; j < PER; ++j) kv[j] = vv[j] = 0.f;
  const uint8_t* block = first >= 0 && row < a.c.rows[sq] ? kv4_block<HD>(a.c, sq, g, (int)row) : nullptr;
  if (block != nullptr) {
    const int r = (int)row & 15, i = lane / LANES, in = lane % LANES;
    uint32_t kc, vc;
    if constexpr (PER == 8) {
      kc = *reinterpret_cast<const uint32_t*>(block + L::k_word(r, in, i));
      vc = *reinterpret_cast<const uint16_t*>(block + L::v_chunk(r, 2 * in) + 2 * i) |
           (uint32_t)*reinterpret_cast<const uint16_t*>(block + L::v_chunk(r, 2 * in + 1) + 2 * i) << 16;
    } else if constexpr (PER == 4) {
      kc = *reinterpret_cast<const uint16_t*>(block + L::k_word(r, in / 2, i) + 2 * (in & 1));
      vc = *reinterpret_cast<const uint16_t*>(block + L::v_chunk(r, in) + 2 * i);
    } else {
      kc = block[L::k_word(r, in / 4, i) + (in & 3)];
      vc = block[L::v_chunk(r, in / 2) + 2 * i + (in & 1)];
    }
    const int ka = r * L::NG + i, va = i * 16 + kv4_slot(r);
    const float ks = __half2float(reinterpret_cast<const __half*>(block + L::KS)[ka]);
    const float km = __half2float(reinterpret_cast<const __half*>(block + L::KM)[ka]);
    const float vs = __half2float(reinterpret_cast<const __half*>(block + L::VS)[va]);
    const float vm = __half2float(reinterpret_cast<const __half*>(block + L::VM)[va]);
    const float ke = kv4_size(block[L::KE + r]), ve = kv4_size(block[L::VE + r]);
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      kv[j] = ke * fmaf(ks, (float)(kc >> (4 * j) & 15), km);
      vv[j] = ve * fmaf(vs, (float)(vc >> (4 * j) & 15), vm);
    }
  } else if (first >= 0 && lane == 0) {
    record_error(a.err, kErrBadIndex);
  }
  const long at = (long)(r0 + sq) * a.out_seq + (long)g * a.out_head + (long)t * HD + lane * PER;
  kv4_store<PER>(a.k + at, kv);
  kv4_store<PER>(a.v + at, vv);
}

}  // namespace

void kv4_append(const Kv4AppendArgs& a, int r0, int seqs, cudaStream_t stream) {
  const long tasks = (long)seqs * a.T * (a.hq + 2 * a.c.hkv);
  if (tasks <= 0) return;
  const unsigned blocks = (unsigned)((tasks + 7) / 8);
  switch (a.c.hd) {
    case 64: kv4_append_kernel<64><<<blocks, 256, 0, stream>>>(a, r0, tasks); break;
    case 128: kv4_append_kernel<128><<<blocks, 256, 0, stream>>>(a, r0, tasks); break;
    case 256: kv4_append_kernel<256><<<blocks, 256, 0, stream>>>(a, r0, tasks); break;
    default: throw std::runtime_error("kv4_append: head_dim 64 / 128 / 256");
  }
  count_launch();
}

void kv4_read(const Kv4ReadArgs& a, int r0, int seqs, cudaStream_t stream) {
  const long tasks = (long)seqs * a.n * a.c.hkv;
  if (tasks <= 0) return;
  const unsigned blocks = (unsigned)((tasks + 7) / 8);
  switch (a.c.hd) {
    case 64: kv4_read_kernel<64><<<blocks, 256, 0, stream>>>(a, r0, tasks); break;
    case 128: kv4_read_kernel<128><<<blocks, 256, 0, stream>>>(a, r0, tasks); break;
    case 256: kv4_read_kernel<256><<<blocks, 256, 0, stream>>>(a, r0, tasks); break;
    default: throw std::runtime_error("kv4_read: head_dim 64 / 128 / 256");
  }
  count_launch();
}

}  // namespace rf
