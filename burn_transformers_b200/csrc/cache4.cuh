// A cache held in 4 bits.  A page of one key head is a record of 68 x dim bytes:
//   key codes   [64 positions][dim / 2]     channel c of a row: nibble c % 2 (0: the lower) of byte c / 2
//   value codes [64 positions][dim / 2]
//   key scales  [64 positions][dim / 32]    a byte for 32 channels
//   value scales[64 positions][dim / 32]
// A nibble n with the scale byte b stands for (n - 8) s(b), s(b) = 2^((b >> 3) - 20) (1 + (b & 7) / 8); b = 255 stands for NaN.
// n - 8 has at most 4 significant bits and s has 4, so that every value is a bfloat16 exactly: what reads the cache needs no
// rounding of its own.  s(b)'s bfloat16 bits are the byte shifted and moved by a constant; its range, 2^-20 to 3,584, holds values
// up to 25,088 (larger ones are held as that) and steps down to 2^-20.
#pragma once
#include "common.cuh"

namespace bt {

constexpr int C4_PAGE = 64;

__host__ __device__ constexpr int c4_record(int dim) { return 68 * dim; }
__host__ __device__ constexpr int c4_value_codes(int dim) { return 32 * dim; }
__host__ __device__ constexpr int c4_key_scales(int dim) { return 64 * dim; }
__host__ __device__ constexpr int c4_value_scales(int dim) { return 66 * dim; }

// A byte's scale in 32 bits.
__device__ __forceinline__ float c4_scale(unsigned b) {
  return b == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float((b << 20) + (107u << 23));
}

// The pages of a layer and of a step's sequences.
struct Cache4View {
  unsigned char* pool;          // [n_pages][n_kv_heads][record]
  long long n_pages;
  const int* table;             // [sequences][table_stride]; position p's page: entry (p / 64) % table_len
  int table_stride, table_len;
  int n_kv_heads;
  int* status;
};

// The record of (page entry, key head); an entry outside the pool is reported and page 0 stands in for it.
__device__ __forceinline__ const unsigned char* c4_page(const Cache4View& c, int seq, int page_of_seq, int kv_head, int dim) {
  int page = c.table[(long long)seq * c.table_stride + page_of_seq % c.table_len];
  if (page < 0 || page >= c.n_pages) {
    if (c.status) atomicExch(c.status, 9);
    page = 0;
  }
  return c.pool + ((long long)page * c.n_kv_heads + kv_head) * c4_record(dim);
}

// A sequence's new tokens: rows t0 .. t0 + n_new - 1 of the step, which has n_tokens.
__device__ __forceinline__ void c4_new_tokens(const int* seq_start, int seq, int n_tokens, int& t0, int& n_new) {
  t0 = max(0, seq_start[seq]);
  n_new = min(seq_start[seq + 1], n_tokens) - t0;
}

// A sequence's length before the step.  One that no sequence has is reported and taken for 0: positions, and with them the places in
// the table, are never negative.
__device__ __forceinline__ int c4_past(const int* past_len, int seq, int* status) {
  const int past = past_len[seq];
  if ((unsigned)past <= 1u << 30) return past;
  if (status) atomicExch(status, 9);
  return 0;
}

// Which keys the query at `pos` sees: `kept` first ones (0 .. kept - 1) and the run lo .. pos, which does not overlap them.
__device__ __forceinline__ void c4_seen(int pos, int window, int keep_first, int& kept, int& lo) {
  lo = window > 0 ? max(0, pos - window + 1) : 0;
  kept = min(window > 0 ? keep_first : 0, lo);
}

}  // namespace bt
