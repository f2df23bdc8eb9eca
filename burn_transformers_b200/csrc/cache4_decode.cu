// Attention over a 4-bit cache (cache4.cuh) for steps that bring few tokens a sequence: bfloat16 queries, heads of 64 or 128 channels.
//
// A block serves one (sequence, key head) and 8 or 16 columns: the query heads that share the key head, for each new token.  Each of its
// warps takes pages of the visible run by itself, through a ring of its own (a page of a key head is one record: one bulk copy), so
// that no barrier stands between pages.  With the keys on the 16 rows of an mma.sync tile and the columns on its 8:
//   S^T = K q^T   a lane's 16 (8) bytes of a key row are 32 (16) channels in a row; the contraction may take the channels in any order, so
//                 that the codes go to the tensor cores as they come out of the word (nibbles i and i + 4), and the queries are put in
//                 that order once;
//   O^T = V^T P^T a lane takes the same bytes of two keys and pairs their nibbles; the rows of a score tile are keys in such an order
//                 that the weights, transposed by movmatrix, meet their keys' values.
// Two codes become their bfloat16 values by a shift, a logical operation and a multiply-add (cache4_codes.cuh), without rounding.
// Maximum, sum and products are 32-bit; the weights are rounded to bfloat16 for the second product, whose operands have 16 bits, as the
// other attention kernels of this library do: results are 1.7e-3 to 1.8e-3 off 64 bits, of which rounding the result is 1.6e-3 to 1.75e-3.
//
// What bounds it: a page takes a warp a chain of dependent steps (1.45 us by itself, 3.2 beside eleven others, 0.27 a page and
// multiprocessor), and 168 registers allow 12 warps; the integer pipe, which takes the codes apart (7 operations for a word of eight), is
// active 53 to 64 % of the time, memory 60 % (64 sequences of 1,000 to 8,000 tokens, 32 heads over 8 of 128: 81 us, 3.9 TB/s).  Half precision,
// which needs 5 operations for a word, came to the same; 16 warps of 128 registers, fed in half pages so that their rings fit, to 7 us more.
// A block has 4 to 12 warps and the run is cut into `n_splits` pieces as the caller's model of their cost says (kernels.py); the
// pieces' results (maximum, sum, weighted values) are joined in order by a second kernel.
// Keys that a column does not see get the weight 0 exactly, and what lies in a page past the sequence's end (any bytes) is never
// multiplied; a value filed as NaN reaches the columns that see its key and no other.
#include "cache4.cuh"
#include "cache4_codes.cuh"
#include "decode_mma.cuh"

namespace bt {

constexpr int C4D_MOST_WARPS = 12;        // of a block, by the registers of a multiprocessor (with 16 columns: 8)
constexpr int C4D_WAIT_LIMIT = 1 << 20;

struct Cache4DecodeParams {
  const __nv_bfloat16* q;
  long long q_row;
  __nv_bfloat16* out;
  const int *seq_start, *past_len;
  int n_tokens, n_heads, group, col_blocks, max_new, slots;
  int sorted;                  // the longest sequences go first
  float scale_log2;
  int window, keep_first;
  float* part;                 // [unit][split][columns][HD], then [unit][split][columns][2]
  long long part_ml;           // where the second begins
};

constexpr int C4D_MOST_SLOTS = 8;        // pages of a warp's ring

__device__ __forceinline__ unsigned c4d_transpose(unsigned v) {
  unsigned d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(v));
  return d;
}

__device__ __forceinline__ float c4d_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;\n" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// A block's sequence: the rank-th, or the one with the rank-th longest run of keys, where blocks wait for others to end: a long sequence
// that is begun late is waited for.  64 sequences of 1,000 to 8,000 tokens in any order: 81 us; in their own order 79 where the longest happen to
// come first, 97 where they come last, 110 to 115 where they are mixed (128 of 500 to 2,000: 60; 56, 60, 64).  Every thread takes some
// sequences and counts those that go before; what the block needs of its own is asked for meanwhile.
// Up to 128 sequences are sorted; of more a thread would count several, for which no form has been made and timed.  They go in their own order:
// 160 of 1,000 to 8,000 take 170 us falling, 190 rising, 210 mixed, 256 of 500 to 4,000 153, 159 and 171.
constexpr int C4D_SORTED = 128;
struct C4dSequence {
  int seq, past, t0, n_new;
};
__device__ __forceinline__ C4dSequence c4d_sequence(const Cache4DecodeParams& p, int n_seqs, int rank, int* status) {
  C4dSequence at;
  if (!p.sorted) {
    at.seq = rank;
    at.past = c4_past(p.past_len, rank, status);
    c4_new_tokens(p.seq_start, rank, p.n_tokens, at.t0, at.n_new);
    return at;
  }
  __shared__ __align__(16) int s_key[C4D_SORTED];      // no two alike
  __shared__ C4dSequence s_at;
  const int tid = threadIdx.x, threads = blockDim.x;
  for (int i = tid; i < C4D_SORTED; i += threads) {
    int past = i < n_seqs ? max(p.past_len[i], 0) : 0;
    if (p.window > 0) past = min(past, p.window);
    s_key[i] = i < n_seqs ? min(past, (1 << 23) - 1) * C4D_SORTED + (C4D_SORTED - i) : 0;
  }
  __syncthreads();
  for (int i = tid; i < n_seqs; i += threads) {
    at.seq = i;
    at.past = c4_past(p.past_len, i, status);
    c4_new_tokens(p.seq_start, i, p.n_tokens, at.t0, at.n_new);
    const int mine = s_key[i];
    int before[4] = {0, 0, 0, 0};
#pragma unroll 8
    for (int j = 0; j < n_seqs; j += 4) {
      const int4 other = *reinterpret_cast<const int4*>(&s_key[j]);
      before[0] += other.x > mine;
      before[1] += other.y > mine;
      before[2] += other.z > mine;
      before[3] += other.w > mine;
    }
    if (before[0] + before[1] + before[2] + before[3] == rank) s_at = at;
  }
  __syncthreads();
  return s_at;
}

template <bool V>
struct C4dFlag {
  static constexpr bool value = V;
};

template <int HD, int NT>
__global__ void __launch_bounds__(NT == 1 ? 384 : 256, 1)
cache4_decode_kernel(Cache4DecodeParams p, Cache4View c) {
  constexpr int REC = c4_record(HD), G = HD / 32;
  constexpr int KW = HD / 32;            // 32-bit words of a key row a lane holds
  constexpr int VW = HD / 64;            // of a value row
  constexpr int MT = HD / 16;
  constexpr int COLS = 8 * NT;
  extern __shared__ __align__(128) unsigned char c4d_raw[];
  __shared__ __align__(8) unsigned long long s_full[C4D_MOST_WARPS][C4D_MOST_SLOTS];
  __shared__ float s_ml[C4D_MOST_WARPS][COLS][2];
  __shared__ int s_failed;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, q = lane & 3;
  const int n_warps = (int)blockDim.x >> 5;
  const int split = blockIdx.x, n_splits = gridDim.x;
  const int kv_head = (int)blockIdx.y / p.col_blocks, col0 = (int)blockIdx.y % p.col_blocks * COLS;
  const C4dSequence at_seq = c4d_sequence(p, gridDim.z, blockIdx.z, c.status);
  const int seq = at_seq.seq, past = at_seq.past, t0 = at_seq.t0, n_new = at_seq.n_new;
  const int n_cols = n_new * p.group - col0;
  if (n_cols <= 0) return;
  const int pos_first = past + col0 / p.group, pos_last = past + min(n_new * p.group - 1, col0 + COLS - 1) / p.group;
  // the pages that any column sees: kept ones before the window's, then the window's
  const int lo = p.window > 0 ? max(0, pos_first - p.window + 1) : 0;
  const int pg_lo = lo / C4_PAGE, pg_hi = pos_last / C4_PAGE;
  const int kept_only = p.window > 0 ? min((min(p.keep_first, pos_last + 1) + C4_PAGE - 1) / C4_PAGE, pg_lo) : 0;
  const int n_pages = kept_only + pg_hi - pg_lo + 1;
  const int per = (n_pages + n_splits - 1) / n_splits;
  const int first = split * per, mine = min(n_pages, first + per) - first;
  const long long unit = (long long)seq * gridDim.y + blockIdx.y;
  if (mine <= 0) return;                 // (the join counts the pieces in the same way)
  auto page_at = [&](int i) { return i < kept_only ? i : pg_lo + (i - kept_only); };

  if (lane == 0) {
    for (int s = 0; s < p.slots; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(ds_smem(&s_full[warp][s])));
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (tid == 0) s_failed = 0;
  __syncthreads();
  unsigned char* ring = c4d_raw + warp * p.slots * REC;
  const int count = mine > warp ? (mine - warp + n_warps - 1) / n_warps : 0;      // this warp's pages: first + warp + n_warps i
  // records of this warp's next 32 pages, one a lane
  auto record_of = [&](int i) { return c4_page(c, seq, page_at(first + warp + n_warps * min(i, count - 1)), kv_head, HD); };
  const unsigned char* next = count > 0 ? record_of(lane) : nullptr;
  auto ask = [&](int slot, const unsigned char* rec) {      // (one lane)
    const unsigned bar = ds_smem(&s_full[warp][slot]);
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"((unsigned)REC) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n" ::"r"(
                     ds_smem(ring + slot * REC)),
                 "l"(rec), "r"((unsigned)REC), "r"(bar)
                 : "memory");
  };
  if (lane < min(p.slots, count)) ask(lane, next);

  // the queries, column g (+ 8) of the second operand: this lane's channels in the order in which codes leave a word
  unsigned qf[NT][KW][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int col = 8 * n + g;
    uint4 raw[HD / 32];
#pragma unroll
    for (int w = 0; w < KW; ++w) raw[w] = make_uint4(0, 0, 0, 0);
    if (col < n_cols) {
      const int token = (col0 + col) / p.group, head = kv_head * p.group + (col0 + col) % p.group;
      const uint4* src = reinterpret_cast<const uint4*>(p.q + (t0 + token) * p.q_row + (long long)head * HD + q * (HD / 4));
#pragma unroll
      for (int w = 0; w < KW; ++w) raw[w] = src[w];
    }
    if (p.scale_log2 <= 0.f) {        // from here on the largest product has the largest weight
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const unsigned f = p.scale_log2 < 0.f ? 0xbf80bf80u : 0u;      // -1 or 0
        raw[w] = make_uint4(c4_fma2(raw[w].x, f, 0x80008000u), c4_fma2(raw[w].y, f, 0x80008000u), c4_fma2(raw[w].z, f, 0x80008000u),
                            c4_fma2(raw[w].w, f, 0x80008000u));
      }
    }
#pragma unroll
    for (int w = 0; w < KW; ++w) {
      qf[n][w][0] = __byte_perm(raw[w].x, raw[w].z, 0x5410);      // channels 0, 4
      qf[n][w][1] = __byte_perm(raw[w].x, raw[w].z, 0x7632);      // 1, 5
      qf[n][w][2] = __byte_perm(raw[w].y, raw[w].w, 0x5410);      // 2, 6
      qf[n][w][3] = __byte_perm(raw[w].y, raw[w].w, 0x7632);      // 3, 7
    }
  }
  // this lane's columns of a score tile: 2q, 2q + 1 (+ 8)
  int pos[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) pos[n][e] = past + min(col0 + 8 * n + 2 * q + e, n_new * p.group - 1) / p.group;
  float m[NT][2], l[NT][2], acc[NT][MT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      m[n][e] = -INFINITY;
      l[n][e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][i][e] = 0.f;
  }
  const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  const int kg = (g >> 1) + 4 * (g & 1);      // the key on row g of a tile of 16 (row g + 8: 8 further)
  const C4Bits bits;
  // One page of keys and values.  PLAIN: every column sees all of it, and no scale stands for NaN.
  auto page = [&](auto plain, const unsigned char* rec, int key0, bool whole) {
    constexpr bool PLAIN = decltype(plain)::value;
    // ---- scores of its 64 keys ----
    float s[NT][4][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][t][e] = 0.f;
      unsigned w[2][KW], s2[2], sh[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = 16 * t + 8 * h + kg;
        const unsigned char* row = rec + key * (HD / 2) + q * (HD / 8);
        if constexpr (KW == 4) {
          const uint4 v = *reinterpret_cast<const uint4*>(row);
          w[h][0] = v.x; w[h][1] = v.y; w[h][2] = v.z; w[h][3] = v.w;
        } else {
          const uint2 v = *reinterpret_cast<const uint2*>(row);
          w[h][0] = v.x; w[h][1] = v.y;
        }
        const unsigned b = rec[c4_key_scales(HD) + key * G + q * G / 4];
        s2[h] = PLAIN || b != 255u ? c4_scale_twice(b) : 0x7fc07fc0u;
        sh[h] = c4_shift(s2[h]);
      }
#pragma unroll
      for (int k = 0; k < KW; ++k) {
        unsigned x[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          x[h][0] = c4_fma2(c4_pair<0>(w[h][k], bits), s2[h], sh[h]);
          x[h][1] = c4_fma2(c4_pair<1>(w[h][k], bits), s2[h], sh[h]);
          x[h][2] = c4_fma2(c4_pair<2>(w[h][k], bits), s2[h], sh[h]);
          x[h][3] = c4_fma2(c4_pair<3>(w[h][k], bits), s2[h], sh[h]);
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          ds_mma(s[n][t], x[0][0], x[1][0], x[0][1], x[1][1], qf[n][k][0], qf[n][k][1]);
          ds_mma(s[n][t], x[0][2], x[1][2], x[0][3], x[1][3], qf[n][k][2], qf[n][k][3]);
        }
      }
    }
    // ---- which of them a column sees; maximum, weights ----
    auto seen = [&](int key, int at) { return key <= at && (p.window <= 0 || key > at - p.window || key < p.keep_first); };
    if (!PLAIN && !whole) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!seen(key0 + 16 * t + 8 * (e >> 1) + kg, pos[n][e & 1])) s[n][t][e] = -INFINITY;
    }
    unsigned pt[NT][4][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float use[2];
      bool grown = false;
      float top[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[e] = fmaxf(s[n][0][e], s[n][0][e + 2]);
#pragma unroll
        for (int t = 1; t < 4; ++t) top[e] = c4d_max3(top[e], s[n][t][e], s[n][t][e + 2]);
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 4));
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 8));
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 16)) * scale;
        grown |= top[e] > m[n][e];
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float m_new = fmaxf(m[n][e], top[e]);
          const float alpha = ds_exp2(m[n][e] - (m_new == -INFINITY ? 0.f : m_new));      // 0 for a column that had seen nothing yet
          m[n][e] = m_new;
          l[n][e] *= alpha;
#pragma unroll
          for (int k = 0; k < MT; ++k) {
            acc[n][k][e] *= alpha;
            acc[n][k][e + 2] *= alpha;
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) use[e] = m[n][e] == -INFINITY ? 0.f : -m[n][e];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = ds_exp2(fmaf(s[n][t][e], scale, use[e & 1]));
          l[n][e & 1] += w[e];
        }
        pt[n][t][0] = c4d_transpose(ds_pack(w[0], w[1]));
        pt[n][t][1] = c4d_transpose(ds_pack(w[2], w[3]));
      }
    }
    // ---- weighted values: a lane's keys of a tile are q, q + 4, q + 8, q + 12 ----
    bool odd = false;                       // a value of NaN among this lane's
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      unsigned w[4][VW], b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = 16 * t + q + 4 * j;
        const unsigned char* row = rec + c4_value_codes(HD) + key * (HD / 2) + g * (HD / 16);
        if constexpr (VW == 2) {
          const uint2 v = *reinterpret_cast<const uint2*>(row);
          w[j][0] = v.x; w[j][1] = v.y;
        } else {
          w[j][0] = *reinterpret_cast<const unsigned*>(row);
        }
        b[j] = rec[c4_value_scales(HD) + key * G + g * G / 8];
      }
      unsigned s01 = c4_scale_pair(b[0], b[1]), s23 = c4_scale_pair(b[2], b[3]);
      if (!PLAIN) {
        unsigned v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool past_end = !whole && key0 + 16 * t + q + 4 * j > pos_last;
          v[j] = c4_scale_bits(b[j]);
          if ((!whole && b[j] == 255u) || past_end) {      // (NaN is seen to below; what lies past the end is not there)
            v[j] = 0u;
            odd |= !past_end;
          }
        }
        s01 = v[0] | v[1] << 16;
        s23 = v[2] | v[3] << 16;
      }
      const unsigned h01 = c4_shift(s01), h23 = c4_shift(s23);
#pragma unroll
      for (int k = 0; k < VW; ++k)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const unsigned a = __byte_perm(w[0][k], w[1][k], half ? 0x7632 : 0x5410), d = __byte_perm(w[2][k], w[3][k], half ? 0x7632 : 0x5410);
          unsigned x[4], y[4];
          x[0] = c4_fma2(c4_pair<0>(a, bits), s01, h01);
          x[1] = c4_fma2(c4_pair<1>(a, bits), s01, h01);
          x[2] = c4_fma2(c4_pair<2>(a, bits), s01, h01);
          x[3] = c4_fma2(c4_pair<3>(a, bits), s01, h01);
          y[0] = c4_fma2(c4_pair<0>(d, bits), s23, h23);
          y[1] = c4_fma2(c4_pair<1>(d, bits), s23, h23);
          y[2] = c4_fma2(c4_pair<2>(d, bits), s23, h23);
          y[3] = c4_fma2(c4_pair<3>(d, bits), s23, h23);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            ds_mma(acc[n][4 * k + 2 * half], x[0], x[1], y[0], y[1], pt[n][t][0], pt[n][t][1]);
            ds_mma(acc[n][4 * k + 2 * half + 1], x[2], x[3], y[2], y[3], pt[n][t][0], pt[n][t][1]);
          }
        }
    }
    if (!PLAIN && !whole && __any_sync(0xffffffffu, odd)) {      // the columns that see a key whose values are NaN
      for (int key = 0; key < C4_PAGE; ++key) {
        if (rec[c4_value_scales(HD) + key * G + g * G / 8] != 255u) continue;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (seen(key0 + key, pos[n][e])) {
#pragma unroll
              for (int k = 0; k < MT; ++k) acc[n][k][e] = acc[n][k][e + 2] = NAN;
            }
      }
    }
  };
  bool ok = true;
  int slot = 0;
  unsigned parity = 0;
  for (int i = 0; i < count; ++i) {
    const int key0 = page_at(first + warp + n_warps * i) * C4_PAGE;
    const unsigned char* rec = ring + slot * REC;
    {
      const unsigned bar = ds_smem(&s_full[warp][slot]);
      bool landed = false;
      for (int t = 0; t < C4D_WAIT_LIMIT && !landed; ++t) {
        unsigned done;
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
            : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        landed = done != 0;
      }
      ok = __all_sync(0xffffffffu, landed);
      if (!ok) break;
    }
    const bool whole = key0 + C4_PAGE - 1 <= pos_first &&
                       (p.window <= 0 || key0 > pos_last - p.window || key0 + C4_PAGE <= p.keep_first);
    bool nan = false;                       // among the page's scales?  (128 G bytes)
#pragma unroll
    for (int j = 0; j < G; ++j) nan |= c4_has_255(*reinterpret_cast<const unsigned*>(rec + c4_key_scales(HD) + 4 * (lane + 32 * j)));
    if (whole && !__any_sync(0xffffffffu, nan))
      page(C4dFlag<true>(), rec, key0, true);
    else
      page(C4dFlag<false>(), rec, key0, whole);
    const int then = i + p.slots;           // the page that comes into this slot
    if (then < count) {
      __syncwarp();
      const unsigned long long rec_next = __shfl_sync(0xffffffffu, (unsigned long long)next, then & 31);
      if (lane == 0) {
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        ask(slot, reinterpret_cast<const unsigned char*>(rec_next));
      }
      if ((then & 31) == 31) next = record_of(then + 1 + lane);
    }
    if (++slot == p.slots) {
      slot = 0;
      parity ^= 1u;
    }
  }
  if (!ok) {
    s_failed = 1;
    let_copies_land();
  }
  // ---- the warps' results, joined in shared memory (over the rings) ----
  float* s_acc = reinterpret_cast<float*>(c4d_raw);      // [warp][column][HD]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
      l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
      if (g == 0) {
        s_ml[warp][8 * n + 2 * q + e][0] = m[n][e];
        s_ml[warp][8 * n + 2 * q + e][1] = l[n][e];
      }
    }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float* row = s_acc + (warp * COLS + 8 * n + 2 * q + e) * HD + g * (HD / 8);
#pragma unroll
      for (int k = 0; k < MT; ++k) {      // tile k: channels 2k, 2k + 1 of this lane's
        row[2 * k] = acc[n][k][e];
        row[2 * k + 1] = acc[n][k][e + 2];
      }
    }
  __syncthreads();
  if (s_failed && tid == 0 && c.status) atomicExch(c.status, 10);
  for (int i = tid; i < COLS * HD; i += (int)blockDim.x) {
    const int col = i / HD, d = i % HD;
    if (col >= n_cols) break;
    float top = -INFINITY, sum = 0.f, o = 0.f;
    for (int w = 0; w < n_warps; ++w) top = fmaxf(top, s_ml[w][col][0]);
    const float use = top == -INFINITY ? 0.f : top;
    for (int w = 0; w < n_warps; ++w) {
      const float weight = ds_exp2(s_ml[w][col][0] - use);
      sum += s_ml[w][col][1] * weight;
      o += s_acc[(w * COLS + col) * HD + d] * weight;
    }
    if (s_failed) sum = NAN;
    if (n_splits == 1) {
      const int token = (col0 + col) / p.group, head = kv_head * p.group + (col0 + col) % p.group;
      p.out[((long long)(t0 + token) * p.n_heads + head) * HD + d] = __float2bfloat16_rn(o / sum);
    } else {
      const long long at = (unit * n_splits + split) * COLS + col;
      p.part[at * HD + d] = o;
      if (d == 0) {
        p.part[p.part_ml + 2 * at] = top;
        p.part[p.part_ml + 2 * at + 1] = sum;
      }
    }
  }
}

// Joins the pieces of a column of a (sequence, key head), in an order that the number of pieces alone sets.  A block a column: the pieces'
// maxima and sums at once, then a thread a channel and every GROUPS-th piece, then the groups' sums.
constexpr int C4J_MOST = 1024;      // pieces at most
template <int HD, int NT, int GROUPS>
__global__ void __launch_bounds__(HD * GROUPS)
cache4_join_kernel(Cache4DecodeParams p, int n_splits) {
  constexpr int COLS = 8 * NT, THREADS = HD * GROUPS;
  __shared__ float s_weight[C4J_MOST], s_sum[GROUPS][HD], scratch[33];
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.z, kv_head = (int)blockIdx.y / p.col_blocks, col0 = (int)blockIdx.y % p.col_blocks * COLS, col = blockIdx.x;
  int t0, n_new;
  c4_new_tokens(p.seq_start, seq, p.n_tokens, t0, n_new);
  if (col0 + col >= n_new * p.group) return;
  const int past = c4_past(p.past_len, seq, nullptr);
  const int pos_first = past + col0 / p.group, pos_last = past + min(n_new * p.group - 1, col0 + COLS - 1) / p.group;
  const int pg_lo = (p.window > 0 ? max(0, pos_first - p.window + 1) : 0) / C4_PAGE;
  const int kept_only = p.window > 0 ? min((min(p.keep_first, pos_last + 1) + C4_PAGE - 1) / C4_PAGE, pg_lo) : 0;
  const int n_pages = kept_only + pos_last / C4_PAGE - pg_lo + 1;
  const int per = (n_pages + n_splits - 1) / n_splits, used = (n_pages + per - 1) / per;
  const long long at0 = ((long long)seq * gridDim.y + blockIdx.y) * n_splits * COLS + col;
  const int tid = threadIdx.x, d = tid % HD, group = tid / HD;
  float top = -INFINITY;
  for (int s = tid; s < used; s += THREADS) {
    const float m = p.part[p.part_ml + 2 * (at0 + (long long)s * COLS)];
    s_weight[s] = m;
    top = fmaxf(top, m);
  }
  top = block_max(top, scratch);
  const float use = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int s = tid; s < used; s += THREADS) {
    const float w = ds_exp2(s_weight[s] - use);
    s_weight[s] = w;
    sum += p.part[p.part_ml + 2 * (at0 + (long long)s * COLS) + 1] * w;
  }
  sum = block_sum(sum, scratch);      // (every weight is in shared memory when it returns)
  float o = 0.f;
#pragma unroll 4
  for (int s = group; s < used; s += GROUPS) o += p.part[(at0 + (long long)s * COLS) * HD + d] * s_weight[s];
  s_sum[group][d] = o;
  __syncthreads();
  if (group != 0) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) o += s_sum[i][d];
  const int token = (col0 + col) / p.group, head = kv_head * p.group + (col0 + col) % p.group;
  p.out[((long long)(t0 + token) * p.n_heads + head) * HD + d] = __float2bfloat16_rn(o / sum);
}

template <int HD, int NT>
static int launch_c4d(Cache4DecodeParams p, const Cache4View& c, int n_seqs, int n_splits, int n_warps, cudaStream_t stream) {
  // the rings: the blocks that share a multiprocessor, as many as their registers allow and the call has, share its shared memory
  constexpr int MOST = NT == 1 ? 12 : 8, WHOLE = 222 * 1024;
  BT_CHECK(n_warps >= 1 && n_warps <= MOST, "cache4_attention: %d warps a block (1 to %d)", n_warps, MOST);
  const long long blocks = (long long)n_splits * c.n_kv_heads * p.col_blocks * n_seqs;
  const int sms = sm_count() > 0 ? sm_count() : 148;
  int side = (int)(blocks <= sms ? 1 : blocks <= 2ll * sms ? 2 : 3);
  if (side > MOST / n_warps) side = MOST / n_warps;
  // blocks that wait for others to end
  p.sorted = blocks > (long long)side * sms && n_seqs > 1 && n_seqs <= C4D_SORTED;
  p.slots = (WHOLE / side - 2048) / (n_warps * c4_record(HD));
  if (p.slots > C4D_MOST_SLOTS) p.slots = C4D_MOST_SLOTS;
  const size_t smem = (size_t)n_warps * p.slots * c4_record(HD);
  static_assert(2 * c4_record(HD) >= (int)sizeof(float) * 8 * NT * HD && WHOLE / 3 - 2048 >= 2 * 4 * c4_record(HD), "the joined results outgrow the rings");
  auto kern = cache4_decode_kernel<HD, NT>;
  static SharedMemoryAllowance allowed;
  BT_CHECK(allow_shared_memory(allowed, kern, smem), "cache4_attention: cannot reserve %zu bytes of shared memory", smem);
  const dim3 grid(n_splits, c.n_kv_heads * p.col_blocks, n_seqs);
  BT_PDL_OK("cache4_decode", launch_pdl(kern, grid, dim3(n_warps * 32), smem, stream, 1, p, c));
  if (n_splits > 1) {
    const dim3 columns(p.group * p.max_new < 8 * NT ? p.group * p.max_new : 8 * NT, c.n_kv_heads * p.col_blocks, n_seqs);
    if (n_splits <= 16)
      BT_PDL_OK("cache4_join", launch_pdl(cache4_join_kernel<HD, NT, 1>, columns, dim3(HD), 0, stream, 1, p, n_splits));
    else
      BT_PDL_OK("cache4_join", launch_pdl(cache4_join_kernel<HD, NT, 4>, columns, dim3(HD * 4), 0, stream, 1, p, n_splits));
  }
  return 0;
}

}  // namespace bt

// Arguments as bt_cache4_attention (bfloat16).  max_new * (n_heads / n_kv_heads) columns a key head go in blocks of 8 or 16.
// scratch: 32-bit words for more than one split: n_seqs * n_kv_heads * column blocks * splits * columns * (dim + 2).
extern "C" int bt_cache4_decode(const void* q, long long q_row, void* out, const void* pool, long long n_pages, const int* table,
                                int table_stride, int table_len, int* status, const int* seq_start, const int* past_len, int n_tokens, int n_seqs,
                                int max_new, int n_heads, int n_kv_heads, int dim, float scale, int window, int keep_first, int n_splits,
                                int n_warps, float* scratch, long long scratch_floats, cudaStream_t stream) {
  using namespace bt;
  BT_CHECK(dim == 64 || dim == 128, "cache4_attention: the kernel for few tokens takes heads of 64 or 128 channels, not %d", dim);
  BT_CHECK(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0, "cache4_attention: %d query heads cannot share %d key heads", n_heads, n_kv_heads);
  BT_CHECK(n_pages > 0 && table != nullptr && table_len > 0 && n_seqs >= 0 && max_new >= 0 && window >= 0 && keep_first >= 0,
           "cache4_attention: bad sizes pages=%lld table_len=%d sequences=%d window=%d kept=%d", n_pages, table_len, n_seqs, window, keep_first);
  auto at16 = [](const void* x) { return (unsigned long long)x % 16 == 0; };
  BT_CHECK(at16(pool) && at16(q) && q_row % 8 == 0, "cache4_attention: pool and query rows must lie on 16-byte boundaries");
  if (n_seqs == 0 || max_new == 0 || n_tokens == 0) return 0;
  const int group = n_heads / n_kv_heads;
  const long long cols = (long long)max_new * group;
  const int nt = cols <= 8 ? 1 : 2, blocks = (int)((cols + 8 * nt - 1) / (8 * nt));
  BT_CHECK(n_seqs <= 65535 && (long long)n_kv_heads * blocks <= 65535 && n_splits >= 1 && n_splits <= C4J_MOST,
           "cache4_attention: grid too large");
  const long long parts = (long long)n_seqs * n_kv_heads * blocks * n_splits * 8 * nt;
  BT_CHECK(n_splits == 1 || (scratch != nullptr && scratch_floats >= parts * (dim + 2)),
           "cache4_attention: %d splits need %lld floats of scratch", n_splits, parts * (dim + 2));
  const Cache4DecodeParams p{(const __nv_bfloat16*)q, q_row, (__nv_bfloat16*)out, seq_start, past_len, n_tokens, n_heads, group, blocks, max_new, 0, 0,
                             scale * 1.4426950408889634f, window, keep_first, scratch, parts * dim};
  const Cache4View c{(unsigned char*)pool, n_pages, table, table_stride, table_len, n_kv_heads, status};
  if (dim == 64) return nt == 1 ? launch_c4d<64, 1>(p, c, n_seqs, n_splits, n_warps, stream) : launch_c4d<64, 2>(p, c, n_seqs, n_splits, n_warps, stream);
  return nt == 1 ? launch_c4d<128, 1>(p, c, n_seqs, n_splits, n_warps, stream) : launch_c4d<128, 2>(p, c, n_seqs, n_splits, n_warps, stream);
}
