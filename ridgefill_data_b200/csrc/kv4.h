// A paged K/V cache held in 4 bits: append (head norm + RoPE + quantisation), read back, decode attention (kv4.cu,
// kv4_attention.cu). The storage layout is in kv4.cuh.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace rf {

constexpr int kKv4Seqs = 64;   // sequences of one launch (their page tables travel in the kernel arguments)

struct Kv4Pages {
  uint8_t* pool;                  // [num_pages, hkv, page_size / 16, 20 hd + 32]
  int num_pages, page_size, hkv, hd;
  const int* pages[kKv4Seqs];     // page table of each sequence
  int rows[kKv4Seqs];             // rows its pages hold
};

struct Kv4AppendArgs {
  Kv4Pages c;
  const __nv_bfloat16* src;       // [R * T, *] projected rows: q heads (each [q | gate] when gated) | k heads | v heads
  int src_row;
  int T;                          // rows a sequence
  int hq, q_stride;               // q heads (0: no q), elements between their starts
  int k_col;                      // column of the first k head (the v heads follow the k heads)
  const __nv_bfloat16* q_norm;    // [hd], norm_mode >= 0
  const __nv_bfloat16* k_norm;
  int norm_mode;                  // -1 none, 0 plain RMSNorm, 1 zero-centred
  double eps;
  const __nv_bfloat16* cos;       // [table_rows, rot / 2]
  const __nv_bfloat16* sin;
  int rot, table_rows;
  const int* row0;                // [R] cache row of each sequence's first row (negative: the sequence is skipped), or
  int row0_host;                  // nullptr: this row for the only sequence
  const int* pos;                 // [R * T] rotary positions, or nullptr: pos_offset + the row's index (pos_offset >= 0),
  int pos_offset;                 // or the cache row (pos_offset < 0)
  __nv_bfloat16* q_out;           // rotated q rows
  int q_out_row, q_out_head;
  int page_shift;                 // log2 of the page size, -1 when it is no power of two (set by the launch)
  int* err;
};
void kv4_append(const Kv4AppendArgs& a, int r0, int seqs, cudaStream_t stream);

struct Kv4ReadArgs {
  Kv4Pages c;
  const int* row0;                // [R] or nullptr: row0_host
  int row0_host;
  int n;                          // rows a sequence
  __nv_bfloat16* k;               // [R, hkv, n, hd] (any sequence and head pitch, row pitch hd)
  __nv_bfloat16* v;
  long out_seq, out_head;
  int* err;
};
void kv4_read(const Kv4ReadArgs& a, int r0, int seqs, cudaStream_t stream);

constexpr int kKv4Splits = 128;   // key splits per (sequence, KV head), at most
struct Kv4AttnArgs {
  Kv4Pages c;
  const __nv_bfloat16* q;         // [R, hq, hd] rotated query rows
  long q_row, q_head;
  int hq;
  const int* pos;                 // [R] last visible cache row of each sequence (negative: none, the output is zero)
  float scale_log2;               // softmax scale times log2(e)
  const __nv_bfloat16* gate;      // optional: gate of (row, head h) at gate + row * gate_row + h * gate_head
  long gate_row, gate_head;
  __nv_bfloat16* out;             // [R, hq * hd]
  long out_row;
  int splits;                     // splits the longest sequence's rows can need (the launch's grid)
  int most;                       // splits a sequence may have (kv4_most_splits)
  float* part_o;                  // [R, hkv, splits, G, hd]
  float* part_ml;                 // [R, hkv, splits, G, 2]
  int* err;
};
int kv4_most_splits(int hd, int hkv);
int kv4_splits(int rows, int hd, int hkv);   // splits that a sequence of `rows` cache rows needs at most
void kv4_attention(const Kv4AttnArgs& a, int r0, int seqs, cudaStream_t stream);

}  // namespace rf
