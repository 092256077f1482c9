// Decode attention over the 4-bit K/V cache: one query row per sequence.
//
// kv4_attn_kernel     grid (key split, KV head, sequence), 4 warps: split s owns keys [s L, (s + 1) L) of the sequence's
//                     rows 0 .. pos, L depending on pos alone (the same bits alone or batched). Each warp takes every
//                     4th key: scores of the G query heads, an online softmax and the weighted values in fp32; the
//                     warps' states are joined in warp order into the split's partial (max, sum, output).
// kv4_combine_kernel  grid (query head, sequence): the splits' partials in split order, the sum's division, the gate.
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

template <int HD, int G>
__global__ void __launch_bounds__(kWarps * 32) kv4_attn_kernel(Kv4AttnArgs a, int r0) {
  using L = Kv4L<HD>;
  constexpr int PER = L::PER, LANES = 32 / PER;
  __shared__ float accs[kWarps][G][HD];
  __shared__ float ms[kWarps][G], ls[kWarps][G];
  const int s = blockIdx.x, g = blockIdx.y, sq = blockIdx.z, r = r0 + sq;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int p = a.pos[r];
  if (p >= a.c.rows[sq]) {
    if (s == 0 && g == 0 && threadIdx.x == 0) record_error(a.err, kErrBadIndex);
    return;
  }
  if (p < 0) return;
  const int keys = split_keys(p), start = s * keys, end = min(start + keys, p + 1);
  if (start > p) return;
  float q[G][PER], m[G], l[G], acc[G][PER];
#pragma unroll
  for (int h = 0; h < G; ++h) {
    kv4_load<PER>(a.q + (long)r * a.q_row + (long)(g * G + h) * a.q_head + lane * PER, q[h]);
    m[h] = kLow;
    l[h] = 0.f;
#pragma unroll
    for (int j = 0; j < PER; ++j) acc[h][j] = 0.f;
  }
  for (int key = start + warp; key < end; key += kWarps) {
    const uint8_t* block = kv4_block<HD>(a.c, sq, g, key);
    if (block == nullptr) {
      if (lane == 0) record_error(a.err, kErrBadIndex);
      continue;
    }
    const int row = key & 15, i = lane / LANES, in = lane % LANES;
    uint32_t kc, vc;
    if constexpr (PER == 8) {
      kc = *reinterpret_cast<const uint32_t*>(block + L::k_word(row, in, i));
      vc = *reinterpret_cast<const uint16_t*>(block + L::v_chunk(row, 2 * in) + 2 * i) |
           (uint32_t)*reinterpret_cast<const uint16_t*>(block + L::v_chunk(row, 2 * in + 1) + 2 * i) << 16;
    } else if constexpr (PER == 4) {
      kc = *reinterpret_cast<const uint16_t*>(block + L::k_word(row, in / 2, i) + 2 * (in & 1));
      vc = *reinterpret_cast<const uint16_t*>(block + L::v_chunk(row, in) + 2 * i);
    } else {
      kc = block[L::k_word(row, in / 4, i) + (in & 3)];
      vc = block[L::v_chunk(row, in / 2) + 2 * i + (in & 1)];
    }
    const int ka = row * L::NG + i, va = i * 16 + kv4_slot(row);
    const float ks = __half2float(reinterpret_cast<const __half*>(block + L::KS)[ka]);
    const float km = __half2float(reinterpret_cast<const __half*>(block + L::KM)[ka]);
    const float vs = __half2float(reinterpret_cast<const __half*>(block + L::VS)[va]);
    const float vm = __half2float(reinterpret_cast<const __half*>(block + L::VM)[va]);
    const float ke = kv4_size(block[L::KE + row]), ve = kv4_size(block[L::VE + row]);
    float kf[PER], vf[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      kf[j] = ke * fmaf(ks, (float)(kc >> (4 * j) & 15), km);
      vf[j] = ve * fmaf(vs, (float)(vc >> (4 * j) & 15), vm);
    }
#pragma unroll
    for (int h = 0; h < G; ++h) {
      float d = 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) d = fmaf(q[h][j], kf[j], d);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(kFull, d, o);
      const float x = d * a.scale_log2;
      const float mn = fmaxf(m[h], x);
      const float corr = exp2f(m[h] - mn), pj = exp2f(x - mn);
      l[h] = fmaf(l[h], corr, pj);
#pragma unroll
      for (int j = 0; j < PER; ++j) acc[h][j] = fmaf(pj, vf[j], acc[h][j] * corr);
      m[h] = mn;
    }
  }
#pragma unroll
  for (int h = 0; h < G; ++h) {
    if (lane == 0) ms[warp][h] = m[h], ls[warp][h] = l[h];
#pragma unroll
    for (int j = 0; j < PER; ++j) accs[warp][h][lane * PER + j] = acc[h][j];
  }
  __syncthreads();
  const long base = (((long)r * a.c.hkv + g) * a.splits + s) * G;
  for (int t = threadIdx.x; t < G * HD; t += kWarps * 32) {
    const int h = t / HD, e = t % HD;
    float M = kLow, S = 0.f, O = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) M = fmaxf(M, ms[w][h]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2f(ms[w][h] - M);
      S = fmaf(ls[w][h], f, S);
      O = fmaf(accs[w][h][e], f, O);
    }
    a.part_o[(base + h) * HD + e] = O;
    if (e == 0) a.part_ml[(base + h) * 2] = M, a.part_ml[(base + h) * 2 + 1] = S;
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
  const dim3 grid(a.splits, a.c.hkv, seqs);
  switch (a.hq / a.c.hkv) {
#define RF_KV4_CASE(G) case G: kv4_attn_kernel<HD, G><<<grid, kWarps * 32, 0, stream>>>(a, r0); break;
    RF_KV4_CASE(1) RF_KV4_CASE(2) RF_KV4_CASE(3) RF_KV4_CASE(4) RF_KV4_CASE(5) RF_KV4_CASE(6) RF_KV4_CASE(7)
    RF_KV4_CASE(8)
#undef RF_KV4_CASE
    default: throw std::runtime_error("kv4_attention: 1 to 8 query heads per KV head");
  }
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
