// Python bindings of the 4-bit K/V cache (kv4.h). Everything a kernel indexes by is checked here for type,
// device, layout and extent; positions and page ids, which live in device memory, are checked by the kernels.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <string>

#include "kv4.h"

torch::Tensor& err_word(int dev);   // bindings.cpp: the per-device error word

namespace {

using at::Tensor;
using OptT = c10::optional<Tensor>;

cudaStream_t cur() { return at::cuda::getCurrentCUDAStream().stream(); }
__nv_bfloat16* bf(const Tensor& t) { return reinterpret_cast<__nv_bfloat16*>(t.data_ptr()); }
bool small(int64_t stride) { return stride >= 0 && stride < (1ll << 31); }
bool aligned(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// Numbers reach a message as std::to_string: streaming one faults where the compiler's libstdc++ is not torch's.
void need(const Tensor& t, at::ScalarType st, const Tensor& like, const char* name) {
  TORCH_CHECK(t.device() == like.device(), name, " is on ", t.device().str(), ", the pool on ", like.device().str());
  TORCH_CHECK(t.scalar_type() == st, name, " has dtype ", t.scalar_type(), ", expected ", st);
}

// Whether some element of t lies `shift` elements behind another one of t (behind itself: not when `same`), dim after dim from
// the widest stride, at the multiples that the inner dims (together `inner` elements wide at most) can make up for.
bool meets(const Tensor& t, const std::vector<int64_t>& dims, size_t at, int64_t inner, int64_t shift, bool same) {
  if (at == dims.size()) return shift == 0 && !same;
  const int64_t stride = t.stride(dims[at]), last = t.size(dims[at]) - 1;   // last > 0
  if (stride == 0) return true;
  inner -= last * stride;
  const auto down = [&](int64_t x) { return x >= 0 ? x / stride : -((-x + stride - 1) / stride); };
  for (int64_t x = std::max(-last, -down(inner - shift)); x <= std::min(last, down(shift + inner)); ++x)
    if (meets(t, dims, at + 1, inner, shift - x * stride, same && x == 0)) return true;
  return false;
}

// Rows that a call writes into given outputs must share no element: t's own, or those of t and of a second output of t's
// strides.
void need_apart(const Tensor& t, const char* op, const OptT& second = c10::nullopt) {
  if (t.numel() == 0) return;
  std::vector<int64_t> dims;
  int64_t inner = 0;
  for (int64_t d = 0; d < t.dim(); ++d)
    if (t.size(d) > 1) dims.push_back(d), inner += (t.size(d) - 1) * t.stride(d);
  std::sort(dims.begin(), dims.end(), [&](int64_t x, int64_t y) { return t.stride(x) > t.stride(y); });
  const int64_t shift = second.has_value() ? ((const char*)second->data_ptr() - (const char*)t.data_ptr()) / t.element_size() : 0;
  TORCH_CHECK(!meets(t, dims, 0, inner, shift, !second.has_value()), op,
              ": an output's rows lie on each other (several of its elements at one memory location)");
}

// pool and page tables of every sequence -> the launch's part of them
struct Cache {
  Tensor pool;
  std::vector<Tensor> pages;
  int hd, hkv, page_size, num_pages;

  Cache(Tensor p, std::vector<Tensor> t, const char* op) : pool(std::move(p)), pages(std::move(t)) {
    TORCH_CHECK(pool.scalar_type() == at::kByte && pool.dim() == 4 && pool.is_contiguous() &&
                    aligned(pool),
                op, ": the pool is a contiguous uint8 tensor [pages, kv_heads, page_size / 16, 20 head_dim + 32]");
    hd = (int)((pool.size(3) - 32) / 20);
    TORCH_CHECK((hd == 64 || hd == 128 || hd == 256) && pool.size(3) == 20 * hd + 32, op,
                ": head_dim 64, 128 or 256 (blocks of 20 head_dim + 32 bytes)");
    TORCH_CHECK(pool.size(0) > 0 && pool.size(1) > 0 && pool.size(1) <= 65535 && pool.size(2) > 0 &&
                    pool.size(0) < (1 << 30) && pool.size(2) * pool.size(3) < (1ll << 31),
                op, ": empty or oversized pool");
    num_pages = (int)pool.size(0);
    hkv = (int)pool.size(1);
    page_size = (int)pool.size(2) * 16;
    for (const Tensor& t : pages) {
      need(t, at::kInt, pool, "pages");
      TORCH_CHECK(t.dim() == 1 && t.is_contiguous(), op, ": a page table is a contiguous int32 vector");
    }
  }

  // rows of a sequence: at most 2^30, so a split's first row fits an int
  int64_t rows(size_t r) const { return std::min<int64_t>(pages[r].numel() * page_size, 1ll << 30); }

  // the last check before a launch, so that every other refusal holds on any device
  void on_gpu(const char* op) const { TORCH_CHECK(pool.is_cuda(), op, ": the cache must be on a CUDA device"); }

  int* err() const { return err_word(pool.get_device()).data_ptr<int>(); }

  rf::Kv4Pages part(int64_t r0, int n) const {
    rf::Kv4Pages c{};
    c.pool = pool.data_ptr<uint8_t>();
    c.num_pages = num_pages;
    c.page_size = page_size;
    c.hkv = hkv;
    c.hd = hd;
    for (int s = 0; s < n; ++s) {
      c.pages[s] = pages[r0 + s].data_ptr<int>();
      c.rows[s] = (int)rows(r0 + s);
    }
    return c;
  }
};

// row0: an int32 vector with one row per sequence, or (absent) the host value of the only sequence
const int* first_rows(const OptT& row0, int64_t host, const Cache& c, int64_t T, const char* op) {
  if (row0.has_value()) {
    need(*row0, at::kInt, c.pool, "row0");
    TORCH_CHECK(row0->dim() == 1 && row0->is_contiguous() && row0->numel() == (int64_t)c.pages.size(), op,
                ": one row0 per sequence");
    return row0->data_ptr<int>();
  }
  TORCH_CHECK(c.pages.size() == 1, op, ": a host row0 serves one sequence");
  TORCH_CHECK(host >= 0 && host <= c.rows(0) - T, op, ": rows ", std::to_string(host), " .. ",
              std::to_string(static_cast<int64_t>(static_cast<uint64_t>(host) + T)), " of a cache that holds ",
              std::to_string(c.rows(0)));
  return nullptr;
}

// -> the rotated q rows (q_out when given), undefined without q heads
OptT kv4_append(Tensor src, Tensor pool, std::vector<Tensor> pages, OptT row0, int64_t row0_host, int64_t hq, bool gated,
                OptT q_norm, OptT k_norm, int64_t norm_mode, double eps, OptT cos, OptT sin, int64_t rot, OptT pos,
                int64_t pos_offset, OptT q_out) {
  const Cache c(pool, std::move(pages), "kv4.append");
  const int64_t R = (int64_t)c.pages.size();
  need(src, at::kBFloat16, c.pool, "src");
  // each number's own range before a product or sum of it, which may pass 64 bits
  const int64_t qw = hq >= 0 && hq <= 65535 ? hq * c.hd * (gated ? 2 : 1) : 0;
  TORCH_CHECK(src.dim() == 2 && src.stride(1) == 1 && hq >= 0 && hq <= 65535 && hq + 2 * c.hkv <= 65535 &&
                  src.size(1) >= qw + 2 * (int64_t)c.hkv * c.hd,
              "kv4.append: rows [*, q heads | k heads | v heads], up to 65535 heads");
  TORCH_CHECK(aligned(src) && (src.size(0) <= 1 || src.stride(0) % 8 == 0) && small(src.stride(0)),
              "kv4.append: 16-byte aligned rows");
  TORCH_CHECK(R > 0 && src.size(0) % R == 0, "kv4.append: the same number of rows for every sequence");
  const int64_t T = src.size(0) / R;
  TORCH_CHECK(T < (1 << 30), "kv4.append: too many rows");
  rf::Kv4AppendArgs a{};
  a.row0 = first_rows(row0, row0_host, c, T, "kv4.append");
  a.row0_host = (int)row0_host;
  TORCH_CHECK(norm_mode >= -1 && norm_mode <= 1, "kv4.append: norm_mode -1, 0 or 1");
  if (norm_mode >= 0) {
    TORCH_CHECK(eps >= 1e-30 && eps <= 1e30, "kv4.append: a norm's eps lies between 1e-30 and 1e30");
    TORCH_CHECK(k_norm.has_value() && (hq == 0 || q_norm.has_value()), "kv4.append: norm weights");
    for (const OptT* w : {&q_norm, &k_norm})
      if (w->has_value()) {
        need(**w, at::kBFloat16, c.pool, "norm weight");
        TORCH_CHECK((*w)->is_contiguous() && (*w)->numel() == c.hd && aligned(**w), "kv4.append: norm weights [head_dim]");
      }
    a.q_norm = q_norm.has_value() ? bf(*q_norm) : nullptr;
    a.k_norm = bf(*k_norm);
  }
  TORCH_CHECK(rot >= 0 && rot <= c.hd && rot % (c.hd / 16) == 0, "kv4.append: rotary dims a multiple of head_dim / 16");
  if (rot > 0) {
    TORCH_CHECK(cos.has_value() && sin.has_value(), "kv4.append: RoPE tables");
    for (const OptT* t : {&cos, &sin}) {
      need(**t, at::kBFloat16, c.pool, "RoPE table");
      TORCH_CHECK((*t)->dim() == 2 && (*t)->is_contiguous() && (*t)->size(1) == rot / 2 && aligned(**t) &&
                      (*t)->size(0) == cos->size(0) && (*t)->size(0) < (1ll << 31) && (T == 0 || (*t)->size(0) > 0),
                  "kv4.append: RoPE tables [positions, rot / 2] of one position or more");
    }
    a.cos = bf(*cos);
    a.sin = bf(*sin);
    a.table_rows = (int)cos->size(0);
  }
  a.pos_offset = pos_offset < 0 ? -1 : (int)pos_offset;
  if (pos.has_value()) {
    need(*pos, at::kInt, c.pool, "pos");
    TORCH_CHECK(pos->dim() == 1 && pos->is_contiguous() && pos->numel() == src.size(0), "kv4.append: one position a row");
    a.pos = pos->data_ptr<int>();
  } else if (pos_offset >= 0) {
    TORCH_CHECK(R == 1 && pos_offset < (1ll << 31) - T, "kv4.append: pos_offset serves one sequence");
  }
  if (rot > 0 && !pos.has_value() && !row0.has_value())
    TORCH_CHECK((pos_offset < 0 ? row0_host : pos_offset) + T <= a.table_rows,
                "kv4.append: positions past the RoPE tables' ", std::to_string(a.table_rows));
  if (hq == 0) q_out = c10::nullopt;
  if (hq > 0) {
    const bool given = q_out.has_value();
    if (!given) q_out = at::empty({src.size(0), hq, c.hd}, src.options());
    need(*q_out, at::kBFloat16, c.pool, "q_out");
    TORCH_CHECK(q_out->dim() == 3 && q_out->size(0) == src.size(0) && q_out->size(1) == hq && q_out->size(2) == c.hd &&
                    q_out->stride(2) == 1 && small(q_out->stride(0)) && small(q_out->stride(1)) &&
                    q_out->stride(0) % 8 == 0 && q_out->stride(1) % 8 == 0 && aligned(*q_out),
                "kv4.append: q_out [rows, q heads, head_dim], 16-byte aligned");
    if (given) need_apart(*q_out, "kv4.append");
    a.q_out = bf(*q_out);
    a.q_out_row = (int)q_out->stride(0);
    a.q_out_head = (int)q_out->stride(1);
  }
  TORCH_CHECK(src.size(0) * (hq + 2 * c.hkv) < (1ll << 31), "kv4.append: too many rows");
  if (T == 0) return q_out;
  a.src = bf(src);
  a.src_row = (int)src.stride(0);
  a.T = (int)T;
  a.hq = (int)hq;
  a.q_stride = c.hd * (gated ? 2 : 1);
  a.k_col = (int)qw;
  a.norm_mode = (int)norm_mode;
  a.eps = eps;
  a.rot = (int)rot;
  c.on_gpu("kv4.append");
  a.err = c.err();
  c10::cuda::CUDAGuard guard(c.pool.device());
  for (int64_t r0 = 0; r0 < R; r0 += rf::kKv4Seqs) {
    const int n = (int)std::min<int64_t>(rf::kKv4Seqs, R - r0);
    a.c = c.part(r0, n);
    rf::kv4_append(a, (int)r0, n, cur());
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return q_out;
}

// -> k, v [sequences, kv_heads, n, head_dim], or without the first dim (single)
std::tuple<Tensor, Tensor> kv4_read(Tensor pool, std::vector<Tensor> pages, OptT row0, int64_t row0_host, int64_t n,
                                    bool single, OptT k_out, OptT v_out) {
  const Cache c(pool, std::move(pages), "kv4.read");
  const int64_t R = (int64_t)c.pages.size();
  TORCH_CHECK(k_out.has_value() == v_out.has_value(), "kv4.read: both of k and v, or neither");
  TORCH_CHECK(n >= 0 && n < (1ll << 31) - 64 && (n / 16 + 2) * c.hkv < (1ll << 31) / rf::kKv4Seqs,
              "kv4.read: a number of rows from 0 to what a launch takes");
  TORCH_CHECK(!single || R == 1, "kv4.read: one sequence");
  const auto opts = c.pool.options().dtype(at::kBFloat16);
  const int64_t lead = single ? 1 : 0;
  std::vector<int64_t> shape{R, c.hkv, n, c.hd};
  if (single) shape.erase(shape.begin());
  Tensor k = k_out.has_value() ? *k_out : at::empty(shape, opts), v = v_out.has_value() ? *v_out : at::empty(shape, opts);
  for (const Tensor* t : {&k, &v}) {
    need(*t, at::kBFloat16, c.pool, "k / v");
    TORCH_CHECK(t->sizes() == at::IntArrayRef(shape), "kv4.read: k and v [sequences, kv_heads, rows, head_dim]");
    TORCH_CHECK(t->numel() == 0 || (t->stride(3 - lead) == 1 && t->stride(2 - lead) == c.hd && t->stride(1 - lead) % 8 == 0 &&
                                    (single || t->stride(0) % 8 == 0) && t->strides() == k.strides() && aligned(*t)),
                "kv4.read: k and v rows head_dim apart, 16-byte aligned, the same strides");
    if (k_out.has_value()) need_apart(*t, "kv4.read");
  }
  if (k_out.has_value()) need_apart(k, "kv4.read", v);
  rf::Kv4ReadArgs a{};
  if (R == 0) return {k, v};
  a.row0 = first_rows(row0, row0_host, c, n, "kv4.read");
  if (n == 0) return {k, v};
  a.row0_host = (int)row0_host;
  a.n = (int)n;
  a.k = bf(k);
  a.v = bf(v);
  a.out_seq = single ? 0 : k.stride(0);
  a.out_head = k.stride(1 - lead);
  c.on_gpu("kv4.read");
  a.err = c.err();
  c10::cuda::CUDAGuard guard(c.pool.device());
  for (int64_t r0 = 0; r0 < R; r0 += rf::kKv4Seqs) {
    const int m = (int)std::min<int64_t>(rf::kKv4Seqs, R - r0);
    a.c = c.part(r0, m);
    rf::kv4_read(a, (int)r0, m, cur());
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return {k, v};
}

Tensor kv4_attention(Tensor q, Tensor pool, std::vector<Tensor> pages, Tensor pos, double scale, OptT gate,
                     int64_t gate_head, OptT out_given) {
  const Cache c(pool, std::move(pages), "kv4.attention");
  const int64_t R = (int64_t)c.pages.size();
  need(q, at::kBFloat16, c.pool, "q");
  need(pos, at::kInt, c.pool, "pos");
  TORCH_CHECK(q.dim() == 3 && q.size(0) == R && q.size(2) == c.hd && q.stride(2) == 1 && q.stride(1) % 8 == 0 &&
                  (R <= 1 || q.stride(0) % 8 == 0) && aligned(q),
              "kv4.attention: q [sequences, q heads, head_dim], 16-byte aligned");
  const int64_t hq = q.size(1);
  TORCH_CHECK(hq % c.hkv == 0 && hq / c.hkv >= 1 && hq / c.hkv <= 8, "kv4.attention: 1 to 8 query heads per KV head, not ",
              std::to_string(hq), " over ", std::to_string(c.hkv));
  TORCH_CHECK(pos.dim() == 1 && pos.is_contiguous() && pos.numel() == R, "kv4.attention: one position per sequence");
  Tensor out = out_given.has_value() ? *out_given : at::empty({R, hq * c.hd}, q.options());
  need(out, at::kBFloat16, c.pool, "out");
  TORCH_CHECK(out.dim() == 2 && out.size(0) == R && out.size(1) == hq * c.hd && out.stride(1) == 1 && aligned(out) &&
                  (R <= 1 || out.stride(0) % 8 == 0),
              "kv4.attention: out [sequences, q heads * head_dim], 16-byte aligned");
  if (out_given.has_value()) need_apart(out, "kv4.attention");
  rf::Kv4AttnArgs a{};
  if (gate.has_value()) {
    need(*gate, at::kBFloat16, c.pool, "gate");
    TORCH_CHECK(gate->dim() == 2 && gate->size(0) == R && gate->stride(1) == 1 && gate_head >= 0 && gate_head % 8 == 0 &&
                    (hq == 1 || gate_head <= gate->size(1)) && gate->size(1) >= (hq - 1) * gate_head + c.hd && aligned(*gate) &&
                    (R <= 1 || gate->stride(0) % 8 == 0),
                "kv4.attention: gate rows whose head h starts at column h * gate_head, 16-byte aligned");
    a.gate = bf(*gate);
    a.gate_row = gate->stride(0);
    a.gate_head = gate_head;
  }
  if (R == 0) return out;
  c.on_gpu("kv4.attention");
  int64_t most = 1;
  for (int64_t r = 0; r < R; ++r) most = std::max(most, c.rows(r));
  const int64_t S = rf::kv4_splits((int)most, c.hd, c.hkv);
  // the splits' outputs, maxima and sums: this call's own, so calls on other streams and graphs share nothing
  Tensor parts;
  if (S > 1) parts = at::empty({R * S * hq * (c.hd + 2)}, q.options().dtype(at::kFloat));
  a.q = bf(q);
  a.q_row = q.stride(0);
  a.q_head = q.stride(1);
  a.hq = (int)hq;
  a.pos = pos.data_ptr<int>();
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.out = bf(out);
  a.out_row = out.stride(0);
  a.splits = (int)S;
  a.most = rf::kv4_most_splits(c.hd, c.hkv);
  a.part_o = S > 1 ? parts.data_ptr<float>() : nullptr;
  a.part_ml = S > 1 ? a.part_o + R * S * hq * c.hd : nullptr;
  a.err = c.err();
  c10::cuda::CUDAGuard guard(c.pool.device());
  for (int64_t r0 = 0; r0 < R; r0 += rf::kKv4Seqs) {
    const int n = (int)std::min<int64_t>(rf::kKv4Seqs, R - r0);
    a.c = c.part(r0, n);
    rf::kv4_attention(a, (int)r0, n, cur());
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  return out;
}

}  // namespace

void register_kv4(pybind11::module_& m) {
  m.def("kv4_append", &kv4_append);
  m.def("kv4_read", &kv4_read);
  m.def("kv4_attention", &kv4_attention);
}
