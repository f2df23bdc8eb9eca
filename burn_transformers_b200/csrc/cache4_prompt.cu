// Attention over a 4-bit cache (cache4.cuh) for steps that bring many tokens a sequence, on the fifth-generation tensor cores:
// bfloat16 queries, heads of 64 or 128 channels.
//
// A block serves one (sequence, key head) and 256 rows (or 128): row r is query head r % group of new token r / group, so that heads which
// share a key head share its keys, however many new tokens there are.  The rows are two tiles of 128 (rows of the tensor memory), and the
// visible pages go by in steps of one (64 keys), staged two at a time.  Sixteen warps:
//   0-3, 4-7  softmax, a thread a row of tile 0 or 1: a step's scores from tensor memory into registers, running maximum and sum in
//         32-bit, weights as bfloat16 (that product's operands have 16 bits: results are 1.9e-3 to 2.2e-3 off 64 bits, 1.6e-3 of it by their own
//         rounding) back over the scores they were made of, from where P V takes them.  The output accumulates in
//         tensor memory and is rescaled only when a row's maximum has outgrown the one its weights are formed with by more than 2^8;
//   12, 13  issue S = Q K^T and O += P V, each for its tile of rows.  Scores lie in two sets of columns: a step's are formed while the
//         softmax is at the step before;
//   8-10, 11, 14 and 15  take the keys' and the values' codes apart: a lane reads 16 bytes (32 channels, one scale) of the next tile ahead,
//         turns them into the exact bfloat16 values (cache4_codes.cuh) and stores them where the products read them.  A word of eight
//         codes leaves as channels 0 4 1 5 2 6 3 7; the queries are stored in the same order, and the result's registers renamed.
// What bounds it is the products of 64 columns: they take a tensor core as long as ones of 128 (69 cycles for 16 channels, measured), so
// that a step of 256 rows takes it 1,500 cycles of the 1,860 it lasts; the exponentials take 1,024 of the special-function units'.
// Products of whole tiles of 128 keys are cheaper, but their scores and weights fill the tensor memory: each tile's next scores then
// wait for its last product and the softmax for both, which came to the same for long prompts (2 x 4,096 tokens, 32 heads over 8 of
// 128: 328 us, 331 here: 830 TFLOP/s), and short ones also step over tiles of which they see half (8 x 257 behind a window of
// 1,024: 82 us, 70 here).  One issuer for both tiles of rows: 376.  Taking the tiles apart beforehand, for all blocks of rows at once:
// 316, but 91 for the short ones.  Where rows and heads do not fill the GPU the keys are cut into `n_splits` runs of pages, whose
// results a second kernel joins in order.
//
// Masked keys get the weight 0 exactly.  A value filed as NaN reaches the rows that see its key and no other: in a page that every row
// of the block sees it is multiplied as it is; in the few others (eleven at most: five on the diagonal, as many at the window's far edge, the
// last kept one) it is multiplied as 0 and noted, and the rows look at the notes at the end.
// All hand-overs go through mbarriers; every wait is bounded, and one that runs out sets the status word.
#include "attention_tcgen05.cuh"
#include "cache4.cuh"
#include "cache4_codes.cuh"

namespace bt {

constexpr int C4P_THREADS = 512;
constexpr int C4P_EDGES = 12;           // pages that not every row of a block sees: at most 11

struct Cache4PromptParams {
  const __nv_bfloat16* q;
  long long q_row;
  __nv_bfloat16* out;
  const int *seq_start, *past_len;
  int n_tokens, n_heads, group, rows;     // rows a block: 128 or 256
  float scale_log2;
  int window, keep_first;
  float* part;                 // [unit][split][rows][HD], then [unit][split][rows][2]
  long long part_ml;
  int sorted;                  // the blocks with the most pages go first
};

template <int HD>
struct C4pShape {
  static constexpr int TILE = HD / 64 * 2 * TA_BOX_BYTES;        // 128 rows of a head
  static constexpr size_t SMEM = (size_t)6 * TILE;               // two tiles of queries, two stages of keys and of values
};

// The pages that a block's rows see, and how they are cut: the same for the attention and the kernel that joins.
struct C4pRun {
  int past, pos_first, pos_last, kept_only, pg_lo, n_pages, per;
  __device__ C4pRun(int past_, int n_new, int row0, int rows, int group, int window, int keep_first, int n_splits) : past(past_) {
    pos_first = past + row0 / group;
    pos_last = past + min(n_new * group - 1, row0 + rows - 1) / group;
    const int lo = window > 0 ? max(0, pos_first - window + 1) : 0;
    pg_lo = lo / C4_PAGE;
    kept_only = window > 0 ? min((min(keep_first, pos_last + 1) + C4_PAGE - 1) / C4_PAGE, pg_lo) : 0;
    n_pages = kept_only + pos_last / C4_PAGE - pg_lo + 1;
    per = (n_pages + n_splits - 1) / n_splits;
  }
  __device__ int page_at(int i) const { return i < kept_only ? i : pg_lo + (i - kept_only); }
};

// 32 channels of a row of keys or values (16 bytes of codes, one scale) as bfloat16, to their places in a tile.
__device__ __forceinline__ void c4p_place(unsigned char* tile, int r, int chunk, const uint4& raw, unsigned scale, const C4Bits& bits) {
  const unsigned s2 = scale | scale << 16, shift = c4_shift(s2);
  unsigned char* dst = tile + chunk / 2 * (2 * TA_BOX_BYTES) + r * 128;
  const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint4 v = make_uint4(c4_fma2(c4_pair<0>(w[k], bits), s2, shift), c4_fma2(c4_pair<1>(w[k], bits), s2, shift),
                               c4_fma2(c4_pair<2>(w[k], bits), s2, shift), c4_fma2(c4_pair<3>(w[k], bits), s2, shift));
    *reinterpret_cast<uint4*>(dst + ((((chunk & 1) * 4 + k) ^ (r & 7)) << 4)) = v;
  }
}

__device__ __forceinline__ void c4p_bar_arrive_warp(unsigned long long* bar, int lane) {
  __syncwarp();
  if (lane == 0) ta_bar_arrive(bar);
}

// A block's sequence and tile of rows: in their order, the last rows (which see the most) first, or, where blocks wait for others to end, those
// that see the most pages first: a long block that is begun late is waited for.  8 portions of 200 tokens behind 100 to 4,000: 84 us, in their
// own order 110 to 127.  Prompts without a past are in a good order already (2 of 1,024, 12 heads of 64: 18.0, sorted 20.1).
// Up to 128 pairs of sequence and tile are sorted, a thread a pair; more go in their own order: 40 portions of 200 behind 100 to 4,000 (160 pairs) take
// 435 us with the longest first, 468 in any other order, 64 of them 693 and 720.
constexpr int C4P_SORTED = 128;
__device__ __forceinline__ int2 c4p_place_of(const Cache4PromptParams& p, int seq, int n_seqs) {
  const int tiles = gridDim.y;
  if (!p.sorted) return make_int2(seq, tiles - 1 - (int)blockIdx.y);
  __shared__ __align__(16) int s_key[C4P_SORTED];      // no two alike
  __shared__ int s_pick;
  const int tid = threadIdx.x, rank = (int)blockIdx.y * n_seqs + seq, items = n_seqs * tiles;
  int mine = 0;
  if (tid < C4P_SORTED) {
    if (tid < items) {
      const int s = tid / tiles, row0 = tid % tiles * p.rows;
      int t0, n_new, pages = 0;
      c4_new_tokens(p.seq_start, s, p.n_tokens, t0, n_new);
      if (n_new * p.group > row0) pages = max(0, C4pRun(c4_past(p.past_len, s, nullptr), n_new, row0, p.rows, p.group, p.window, p.keep_first, 1).n_pages);
      mine = min(pages, (1 << 23) - 1) * C4P_SORTED + C4P_SORTED - tid;
    }
    s_key[tid] = mine;
  }
  __syncthreads();
  if (tid < items) {
    int before = 0;
#pragma unroll 8
    for (int j = 0; j < items; j += 4) {
      const int4 other = *reinterpret_cast<const int4*>(&s_key[j]);
      before += (other.x > mine) + (other.y > mine) + (other.z > mine) + (other.w > mine);
    }
    if (before == rank) s_pick = tid;
  }
  __syncthreads();
  return make_int2(s_pick / tiles, s_pick % tiles);
}

template <int HD>
__global__ void __launch_bounds__(C4P_THREADS, 1)
cache4_prompt_kernel(Cache4PromptParams p, Cache4View c) {
  constexpr int TILE = C4pShape<HD>::TILE, CH = HD / 32, ISSUER = 12;
  extern __shared__ __align__(1024) unsigned char c4p_raw[];
  __shared__ __align__(8) unsigned long long bars[20];
  __shared__ unsigned s_nan[C4P_EDGES][CH][2];      // a bit a key of a page that not every row sees
  __shared__ int s_edge_key[C4P_EDGES], s_edges;
  __shared__ unsigned s_tmem;
  __shared__ int failed;
  unsigned char *Qs = c4p_raw, *Ks = Qs + 2 * TILE, *Vs = Ks + 2 * TILE;
  unsigned long long *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6;      // [stage]
  unsigned long long *s_full = bars + 8, *p_ready = bars + 12, *o_done = bars + 16;      // [tile of rows][step parity]

  const int kv_head = (int)blockIdx.x % c.n_kv_heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  pdl_trigger();
  pdl_wait();
  const int2 place = c4p_place_of(p, (int)blockIdx.x / c.n_kv_heads, (int)gridDim.x / c.n_kv_heads);
  const int seq = place.x, tile = place.y;
  int t0, n_new;
  c4_new_tokens(p.seq_start, seq, p.n_tokens, t0, n_new);
  const int row0 = tile * p.rows;
  const int n_rows = min(p.rows, n_new * p.group - row0);
  if (n_rows <= 0) return;
  const C4pRun run(c4_past(p.past_len, seq, c.status), n_new, row0, p.rows, p.group, p.window, p.keep_first, (int)gridDim.z);
  // steps of a page each; two in a row are a tile of the stages
  const int page0 = (int)blockIdx.z * run.per, n_steps = min(run.n_pages, page0 + run.per) - page0, n_tiles = (n_steps + 1) / 2;
  if (n_steps <= 0) return;
  if ((ta_smem(c4p_raw) & 1023u) != 0) {      // the swizzled layouts need the alignment: refuse rather than compute nonsense
    if (tid == 0 && c.status) atomicExch(c.status, 10);
    return;
  }
  const int n_sub = n_rows > TA_BQ ? 2 : 1;      // tiles of rows

  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      ta_bar_init(&k_full[s], 3);
      ta_bar_init(&k_empty[s], n_sub);
      ta_bar_init(&v_full[s], 3);
      ta_bar_init(&v_empty[s], n_sub);
    }
    for (int s = 0; s < 4; ++s) {
      ta_bar_init(&s_full[s], 1);
      ta_bar_init(&p_ready[s], 4);
      ta_bar_init(&o_done[s], 1);
    }
    failed = 0;
    s_edges = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (tid < C4P_EDGES * CH * 2) (&s_nan[0][0][0])[tid] = 0u;
  if (warp == ISSUER) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(ta_smem(&s_tmem)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
  }
  // queries: 16-byte pieces of 8 channels, into the order in which codes leave a word; rows past the last are zero
  for (int i = tid; i < n_sub * TA_BQ * (HD / 8); i += C4P_THREADS) {
    const int r = i / (HD / 8), piece = i % (HD / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < n_rows) {
      const int token = (row0 + r) / p.group, head = kv_head * p.group + (row0 + r) % p.group;
      v = *reinterpret_cast<const uint4*>(p.q + (t0 + token) * p.q_row + (long long)head * HD + piece * 8);
    }
    const uint4 w = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                               __byte_perm(v.y, v.w, 0x7632));
    unsigned char* dst = Qs + r / TA_BQ * TILE + piece / 8 * (2 * TA_BOX_BYTES) + r % TA_BQ * 128;
    *reinterpret_cast<uint4*>(dst + (((piece & 7) ^ (r & 7)) << 4)) = w;
  }
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  ta_fence_before();
  __syncthreads();
  ta_fence_after();
  const unsigned tmem = s_tmem, tmem_o = tmem + 256;      // S of both tiles of rows, two steps each (64 columns, the weights over the first 32); O

  // registers: 512 threads x 128 at launch are 2 x 128 x 176 + 2 x 128 x 80
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;\n");
    // ---- softmax: a thread a row; warp w reaches the lanes of quarter w % 4 ----
    const int sub = warp >> 2, r = (warp & 3) * 32 + lane;
    if (sub < n_sub) {
      const int row = min(row0 + sub * TA_BQ + r, n_new * p.group - 1), pos = run.past + row / p.group;
      const int at_first = run.past + (row0 + sub * TA_BQ) / p.group;
      const int at_last = run.past + min(n_new * p.group - 1, row0 + sub * TA_BQ + TA_BQ - 1) / p.group;
      const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
      const unsigned my_s = tmem + (unsigned)(sub * TA_BK) + lanes, my_o = tmem_o + (unsigned)(sub * HD) + lanes;
      const float scale = p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
      float m = -INFINITY, l = 0.f;      // the reference maximum (base 2, scaled) and the sum of weights formed with it
      bool ok = true;
#pragma unroll 1
      for (int j = 0; j < n_steps; ++j) {
        const int key0 = run.page_at(page0 + j) * C4_PAGE;
        const bool whole = key0 + 63 <= at_first && (p.window <= 0 || key0 > at_last - p.window || key0 + 64 <= p.keep_first);
        ok = __all_sync(0xffffffffu, ta_bar_wait(&s_full[2 * sub + (j & 1)], (j >> 1) & 1));
        if (!ok) break;                  // (uniform in the warp; the others run into their own bounds)
        ta_fence_after();
        unsigned a[2][32];
        ta_ld32_issue(my_s + 64u * (j & 1), a[0]);
        ta_ld32_issue(my_s + 64u * (j & 1) + 32u, a[1]);
        ta_ld_wait(a[0], a[1]);
        if (p.scale_log2 <= 0.f) {       // from here on the largest score has the largest weight
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < 32; ++i) a[q][i] = p.scale_log2 < 0.f ? a[q][i] ^ 0x80000000u : __float_as_uint(__uint_as_float(a[q][i]) * 0.f);
        }
        if (!whole) {                    // a bit a key
          const int lo = (p.window > 0 ? max(0, pos - p.window + 1) : 0) - key0, hi = pos - key0;
          const int kept = p.window > 0 ? min(p.keep_first, pos + 1) - key0 : 0;
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const int first = lo - 32 * q, last = hi - 32 * q, below = kept - 32 * q;
            unsigned seen = last >= 31 ? 0xffffffffu : last < 0 ? 0u : (2u << last) - 1u;
            seen &= first <= 0 ? 0xffffffffu : first > 31 ? 0u : 0xffffffffu << first;
            seen |= below >= 32 ? 0xffffffffu : below <= 0 ? 0u : (1u << below) - 1u;
#pragma unroll
            for (int i = 0; i < 32; ++i) a[q][i] = (seen >> i) & 1u ? a[q][i] : __float_as_uint(-INFINITY);
          }
        }
        float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};      // (four chains side by side)
#pragma unroll
        for (int i = 0; i < 16; i += 2)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            t4[q] = ta_max3(t4[q], __uint_as_float(a[q >> 1][(q & 1) * 16 + i]), __uint_as_float(a[q >> 1][(q & 1) * 16 + i + 1]));
        const float top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * scale;
        const bool grown = top > m + TS_GROWTH || (m == -INFINITY && top > -INFINITY);
        if (__any_sync(0xffffffffu, grown)) {
          const float m_new = grown ? top : m;
          const float alpha = grown ? ta_exp2(m - m_new) : 1.f;      // 0 for a row that had seen nothing yet
          l *= alpha;
          m = m_new;
          if (j > 0) {                   // the products before must have been added
            ok = __all_sync(0xffffffffu, ta_bar_wait(&o_done[2 * sub + ((j - 1) & 1)], ((j - 1) >> 1) & 1));
            if (!ok) break;
            ta_fence_after();
#pragma unroll 1
            for (int q = 0; q < HD; q += 32) {
              unsigned o[32];
              ta_ld32_issue(my_o + (unsigned)q, o);
              ta_ld_wait1(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              ta_st32(my_o + (unsigned)q, o);
            }
          }
        }
        const float m_use = m == -INFINITY ? 0.f : m;
        const unsigned long long scale2 = ta_two(__float_as_uint(scale), __float_as_uint(scale));
        const unsigned long long shift2 = ta_two(__float_as_uint(-m_use), __float_as_uint(-m_use));
        unsigned long long sum[4] = {0ull, 0ull, 0ull, 0ull};
        unsigned w[32];
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            unsigned x, y;
            ta_halves(ta_fma2(ta_two(a[q][i], a[q][i + 1]), scale2, shift2), x, y);
            x = __float_as_uint(ta_exp2(__uint_as_float(x)));
            y = __float_as_uint(ta_exp2(__uint_as_float(y)));
            sum[(i >> 1) & 3] = ta_add2(sum[(i >> 1) & 3], ta_two(x, y));
            w[q * 16 + (i >> 1)] = ta_pack(__uint_as_float(x), __uint_as_float(y));
          }
        ta_st32(my_s + 64u * (j & 1), w);
        {
          unsigned x, y;
          ta_halves(ta_add2(ta_add2(sum[0], sum[1]), ta_add2(sum[2], sum[3])), x, y);
          l += __uint_as_float(x) + __uint_as_float(y);
        }
        ta_st_wait();
        ta_fence_before();
        c4p_bar_arrive_warp(&p_ready[2 * sub + (j & 1)], lane);
      }
      if (ok) ok = __all_sync(0xffffffffu, ta_bar_wait(&o_done[2 * sub + ((n_steps - 1) & 1)], ((n_steps - 1) >> 1) & 1));
      ta_fence_after();
      if (!ok) {
        failed = 1;
      } else {
        // channels whose values are NaN for a key that this row sees, but were multiplied as 0
        unsigned lost = 0;
        auto look = [&](int key0, int word, unsigned bits) {
          while (bits) {
            const int key = key0 + 32 * (word & 1) + __ffs(bits) - 1;
            bits &= bits - 1;
            if (key <= pos && (p.window <= 0 || key > pos - p.window || key < p.keep_first)) lost |= 1u << (word >> 1);
          }
        };
        const int edges = *(volatile int*)&s_edges;
        for (int e = 0; e < edges; ++e)
          for (int j = 0; j < CH * 2; ++j) look(s_edge_key[e], j, s_nan[e][j >> 1][j & 1]);
        const bool mine = sub * TA_BQ + r < n_rows;
        const bool cut = gridDim.z > 1;
        const float inv = cut ? 1.f : 1.f / l;
        const int token = row / p.group, head = kv_head * p.group + row % p.group;
        __nv_bfloat16* dst = p.out + ((long long)(t0 + token) * p.n_heads + head) * HD;
        const long long unit = (((long long)(seq * c.n_kv_heads + kv_head) * gridDim.y + tile) * gridDim.z + blockIdx.z) * p.rows + sub * TA_BQ + r;
        float* part = p.part + unit * HD;
#pragma unroll 1
        for (int q = 0; q < CH; ++q) {
          unsigned raw[32];
          ta_ld32_issue(my_o + 32u * q, raw);
          ta_ld_wait1(raw);
          if (!mine) continue;
          const float f = (lost >> q) & 1u ? NAN : inv;
#pragma unroll
          for (int i = 0; i < 32; i += 8) {      // columns 0 .. 7 are the channels 0 4 1 5 2 6 3 7
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = __uint_as_float(raw[i + (j < 4 ? 2 * j : 2 * j - 7)]) * f;
            if (cut) {
              reinterpret_cast<float4*>(part + 32 * q + i)[0] = make_float4(o[0], o[1], o[2], o[3]);
              reinterpret_cast<float4*>(part + 32 * q + i)[1] = make_float4(o[4], o[5], o[6], o[7]);
            } else {
              *reinterpret_cast<uint4*>(dst + 32 * q + i) =
                  make_uint4(ta_pack(o[0], o[1]), ta_pack(o[2], o[3]), ta_pack(o[4], o[5]), ta_pack(o[6], o[7]));
            }
          }
        }
        if (cut && mine) {
          p.part[p.part_ml + 2 * unit] = m;
          p.part[p.part_ml + 2 * unit + 1] = l;
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;\n");
    if (warp != ISSUER && warp != ISSUER + 1) {
      // ---- takes the codes apart: warps 8-10 the keys', 11, 14 and 15 the values'.  A warp's read is 16 bytes a lane of SPAN rows in a row (a
      // unit); eight lanes of a store cover eight rows' same piece ----
      constexpr int SPAN = 32 / CH, UNITS = TA_BK / SPAN;
      constexpr int step = 3;
      const bool values = warp > 10;
      const int who = !values ? warp - 8 : warp == 11 ? 0 : warp - 13;
      constexpr int MOST = (UNITS + 2) / 3;      // units of a warp
      const int chunk = (lane >> 3) % CH, sub_row = (lane & 7) + 8 * ((lane >> 3) / CH);
      unsigned char* const stage0 = values ? Vs : Ks;
      unsigned long long *const full = values ? v_full : k_full, *const empty = values ? v_empty : k_empty;
      const int codes_at = (values ? c4_value_codes(HD) : 0) + chunk * 16, scales_at = (values ? c4_value_scales(HD) : c4_key_scales(HD)) + chunk;
      const C4Bits bits;
      // the records of the next 32 pages, one a lane (behind the last: the last again), and a bit a page that not every row sees
      unsigned long long records;
      unsigned narrow, narrow_now;
      auto look_up = [&](int j) {
        const int page = run.page_at(page0 + min(j, n_steps - 1)), key0 = page * C4_PAGE;
        records = (unsigned long long)c4_page(c, seq, page, kv_head, HD);
        const bool whole = key0 + C4_PAGE - 1 <= run.pos_first && (p.window <= 0 || key0 > run.pos_last - p.window || key0 + C4_PAGE <= p.keep_first);
        narrow = __ballot_sync(0xffffffffu, !whole && j < n_steps);
      };
      look_up(lane);
      uint4 raw[MOST];
      unsigned sc[MOST];
      auto fetch = [&](int it) {
        const unsigned char* rec0 = reinterpret_cast<const unsigned char*>(__shfl_sync(0xffffffffu, records, (2 * it) & 31));
        const unsigned char* rec1 = reinterpret_cast<const unsigned char*>(__shfl_sync(0xffffffffu, records, (2 * it + 1) & 31));
        narrow_now = narrow >> ((2 * it) & 31) & 3u;
        if ((it & 15) == 15) look_up(2 * it + 2 + lane);
#pragma unroll
        for (int j = 0; j < MOST; ++j) {
          const int unit = j * step + who;
          if (unit >= UNITS) continue;           // (the same in the warp)
          const int r = SPAN * unit + sub_row, in_page = r % C4_PAGE;
          const unsigned char* rec = SPAN * unit < C4_PAGE ? rec0 : rec1;
          raw[j] = *reinterpret_cast<const uint4*>(rec + codes_at + in_page * (HD / 2));
          sc[j] = rec[scales_at + in_page * CH];
        }
      };
      int edges = 0;
      bool ok = true;
      fetch(0);
#pragma unroll 1
      for (int it = 0; it < n_tiles; ++it) {
        const int s = it & 1;
        const unsigned now = narrow_now;
        if (values && now && who == 0 && lane == 0) {
          const int page = run.page_at(page0 + 2 * it + ((now & 1u) ? 0 : 1)), more = now == 3u ? 1 : 0;
          s_edge_key[min(edges, C4P_EDGES - 1)] = page * C4_PAGE;
          if (more) s_edge_key[min(edges + 1, C4P_EDGES - 1)] = run.page_at(page0 + 2 * it + 1) * C4_PAGE;
          *(volatile int*)&s_edges = min(edges + 1 + more, C4P_EDGES);
        }
        if (it >= 2) ok = __all_sync(0xffffffffu, ta_bar_wait(&empty[s], ((it >> 1) - 1) & 1));
        if (!ok) break;
#pragma unroll
        for (int j = 0; j < MOST; ++j) {
          const int unit = j * step + who;
          if (unit >= UNITS) continue;
          const int r = SPAN * unit + sub_row;
          const int half = SPAN * unit < C4_PAGE ? 0 : 1;
          unsigned sb = c4_scale_bits(sc[j]);
          if (values && (now >> half & 1u) && sc[j] == 255u) {
            sb = 0u;
            atomicOr(&s_nan[min(edges + (half & (int)now), C4P_EDGES - 1)][chunk][r / 32 & 1], 1u << (r & 31));
          }
          c4p_place(stage0 + s * TILE, r, chunk, raw[j], sb, bits);
        }
        if (values) edges += __popc(now);
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
        c4p_bar_arrive_warp(&full[s], lane);
        if (it + 1 < n_tiles) fetch(it + 1);
      }
      if (!ok) failed = 1;
    }
    if (warp == ISSUER || (warp == ISSUER + 1 && n_sub > 1)) {
      // ---- issuers, one a tile of rows.  Instruction descriptors: 32-bit accumulator, bfloat16 operands, M = 128; S: N = 64, both K-major;
      // P V: N = HD, the first operand in tensor memory, the second MN-major ----
      const unsigned idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(64 >> 3) << 17) | ((unsigned)(TA_BQ >> 4) << 24);
      const unsigned idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((unsigned)(HD >> 3) << 17) | ((unsigned)(TA_BQ >> 4) << 24);
      const unsigned long long desc_q = ta_desc(Qs, 16), desc_k = ta_desc(Ks, 16), desc_v = ta_desc(Vs, 2 * TA_BOX_BYTES);
      const int sub = warp - ISSUER;
      // S of step j's 64 keys (half j % 2 of their tile's rows) into the columns of its parity
      auto scores = [&](int j) {
        if (ta_elect()) {
          const unsigned long long dq = desc_q + (unsigned long long)(sub * (TILE >> 4));
          const unsigned long long dk = desc_k + (unsigned long long)(((j >> 1) & 1) * (TILE >> 4) + (j & 1) * (TA_BOX_BYTES >> 4));
#pragma unroll
          for (int k = 0; k < HD / 16; ++k) {      // 16 channels: 32 bytes further along the row, a box further every 64
            const unsigned long long step = (k / 4) * (2 * TA_BOX_BYTES >> 4) + 2 * (k % 4);
            ta_mma(tmem + (unsigned)(sub * TA_BK + (j & 1) * 64), dq + step, dk + step, idesc_s, k > 0 ? 1u : 0u);
          }
          ta_commit(&s_full[2 * sub + (j & 1)]);
          if ((j & 1) || j + 1 == n_steps) ta_commit(&k_empty[(j >> 1) & 1]);
        }
        __syncwarp();
      };
      auto mix = [&](int j) {             // P V: 16 keys further are 8 columns of P, 16 rows of V
        if (ta_elect()) {
          const unsigned long long dv = desc_v + (unsigned long long)(((j >> 1) & 1) * (TILE >> 4) + (j & 1) * (TA_BOX_BYTES >> 4));
#pragma unroll
          for (int i = 0; i < 4; ++i)
            ta_mma_tmem(tmem_o + (unsigned)(sub * HD), tmem + (unsigned)(sub * TA_BK + (j & 1) * 64) + 8u * i,
                        dv + (unsigned long long)(i * (16 * 128 >> 4)), idesc_o, (j > 0 || i > 0) ? 1u : 0u);
          ta_commit(&o_done[2 * sub + (j & 1)]);
          if ((j & 1) || j + 1 == n_steps) ta_commit(&v_empty[(j >> 1) & 1]);
        }
        __syncwarp();
      };
      // P V of a step when its weights are there (and the values); then, when that product is done, the scores two steps ahead, whose
      // columns its weights held (and their keys are there).  The softmax has the step between to work on meanwhile.
      bool ok = true;
      for (int j = -2; j < n_steps && ok; ++j) {
        if (j >= 0) {
          ok = __all_sync(0xffffffffu, ta_bar_wait(&v_full[(j >> 1) & 1], (j >> 2) & 1) && ta_bar_wait(&p_ready[2 * sub + (j & 1)], (j >> 1) & 1));
          if (!ok) break;
          ta_fence_after();
          mix(j);
        }
        if (j + 2 < n_steps) {
          ok = __all_sync(0xffffffffu, ta_bar_wait(&k_full[((j + 2) >> 1) & 1], ((j + 2) >> 2) & 1) &&
                                           (j < 0 || ta_bar_wait(&o_done[2 * sub + (j & 1)], (j >> 1) & 1)));
          if (!ok) break;
          ta_fence_after();
          scores(j + 2);
        }
      }
      if (!ok && lane == 0) failed = 1;
    }
  }
  ta_fence_before();
  __syncthreads();
  if (failed) let_copies_land();
  if (warp == ISSUER) {
    ta_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
  }
  if (tid == 0 && failed && c.status) atomicExch(c.status, 10);
}

// Joins the runs of keys of a block's rows: a warp a row, a lane HD / 32 channels; weights of 32 runs at once, values in the runs' order.
constexpr int C4P_JOIN_WARPS = 8;
template <int HD>
__global__ void __launch_bounds__(32 * C4P_JOIN_WARPS)
cache4_prompt_join_kernel(Cache4PromptParams p, int n_kv_heads, int row_tiles, int n_splits) {
  constexpr int CH = HD / 32;
  pdl_trigger();
  pdl_wait();
  const int kv_head = (int)blockIdx.y % n_kv_heads, seq = (int)blockIdx.y / n_kv_heads, lane = threadIdx.x & 31;
  const int place = (int)blockIdx.x * C4P_JOIN_WARPS + ((int)threadIdx.x >> 5);
  const int tile = place / p.rows, r = place % p.rows, row0 = tile * p.rows, row = row0 + r;
  int t0, n_new;
  c4_new_tokens(p.seq_start, seq, p.n_tokens, t0, n_new);
  if (row >= n_new * p.group) return;
  const C4pRun run(c4_past(p.past_len, seq, nullptr), n_new, row0, p.rows, p.group, p.window, p.keep_first, n_splits);
  const int used = (run.n_pages + run.per - 1) / run.per;
  const long long unit0 = ((long long)blockIdx.y * row_tiles + tile) * n_splits * p.rows + r;      // run s: p.rows further
  const float2* ml = reinterpret_cast<const float2*>(p.part + p.part_ml);
  float top = -INFINITY;
  for (int s = lane; s < used; s += 32) top = fmaxf(top, ml[unit0 + (long long)s * p.rows].x);
  top = warp_max(top);
  const float use = top == -INFINITY ? 0.f : top;
  float sum = 0.f, o[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) o[i] = 0.f;
  for (int s0 = 0; s0 < used; s0 += 32) {
    float weight = 0.f;
    if (s0 + lane < used) {
      const float2 mine = ml[unit0 + (long long)(s0 + lane) * p.rows];
      weight = ta_exp2(mine.x - use);
      sum += mine.y * weight;
    }
    const int count = min(32, used - s0);
#pragma unroll 4
    for (int s = 0; s < count; ++s) {
      const float* part = p.part + (unit0 + (long long)(s0 + s) * p.rows) * HD + lane * CH;
      const float w = __shfl_sync(0xffffffffu, weight, s);
      float x[CH];
      if constexpr (CH == 4)
        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(part);
      else
        *reinterpret_cast<float2*>(x) = *reinterpret_cast<const float2*>(part);
#pragma unroll
      for (int i = 0; i < CH; ++i) o[i] = fmaf(x[i], w, o[i]);
    }
  }
  sum = warp_sum(sum);
  const int token = row / p.group, head = kv_head * p.group + row % p.group;
  unsigned* dst = reinterpret_cast<unsigned*>(p.out + ((long long)(t0 + token) * p.n_heads + head) * HD + lane * CH);
  if constexpr (CH == 4)
    *reinterpret_cast<uint2*>(dst) = make_uint2(ta_pack(o[0] / sum, o[1] / sum), ta_pack(o[2] / sum, o[3] / sum));
  else
    *dst = ta_pack(o[0] / sum, o[1] / sum);
}

template <int HD>
static int launch_c4p(const Cache4PromptParams& p, const Cache4View& c, int n_seqs, int row_tiles, int n_splits, cudaStream_t stream) {
  constexpr size_t smem = C4pShape<HD>::SMEM;
  auto kern = cache4_prompt_kernel<HD>;
  static SharedMemoryAllowance allowed;
  BT_CHECK(allow_shared_memory(allowed, kern, smem), "cache4_attention: cannot reserve %zu bytes of shared memory", smem);
  BT_PDL_OK("cache4_prompt", launch_pdl(kern, dim3(n_seqs * c.n_kv_heads, row_tiles, n_splits), dim3(C4P_THREADS), smem, stream, 1, p, c));
  if (n_splits > 1)
    BT_PDL_OK("cache4_prompt_join", launch_pdl(cache4_prompt_join_kernel<HD>, dim3(row_tiles * (p.rows / C4P_JOIN_WARPS), n_seqs * c.n_kv_heads),
                                               dim3(32 * C4P_JOIN_WARPS), 0, stream, 1, p, c.n_kv_heads, row_tiles, n_splits));
  return 0;
}

}  // namespace bt

// Arguments as bt_cache4_attention (bfloat16).  scratch: 32-bit words for more than one split: n_seqs * n_kv_heads * row tiles (of `rows` rows:
// max_new * (n_heads / n_kv_heads)) * splits * rows * (dim + 2).  behind_others: there are sequences whose new tokens are not their first.
extern "C" int bt_cache4_prompt(const void* q, long long q_row, void* out, const void* pool, long long n_pages, const int* table,
                                int table_stride, int table_len, int* status, const int* seq_start, const int* past_len, int n_tokens, int n_seqs,
                                int max_new, int n_heads, int n_kv_heads, int dim, float scale, int window, int keep_first, int n_splits,
                                int rows, float* scratch, long long scratch_floats, int behind_others, cudaStream_t stream) {
  using namespace bt;
  BT_CHECK(rows == 128 || rows == 256, "cache4_attention: %d rows a block (128 or 256)", rows);
  BT_CHECK(dim == 64 || dim == 128, "cache4_attention: the kernel for many tokens takes heads of 64 or 128 channels, not %d", dim);
  BT_CHECK(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0, "cache4_attention: %d query heads cannot share %d key heads", n_heads, n_kv_heads);
  BT_CHECK(n_pages > 0 && table != nullptr && table_len > 0 && n_seqs >= 0 && max_new >= 0 && window >= 0 && keep_first >= 0,
           "cache4_attention: bad sizes pages=%lld table_len=%d sequences=%d window=%d kept=%d", n_pages, table_len, n_seqs, window, keep_first);
  auto at16 = [](const void* x) { return (unsigned long long)x % 16 == 0; };
  BT_CHECK(at16(pool) && at16(q) && at16(out) && q_row % 8 == 0, "cache4_attention: pool, queries and results must lie on 16-byte boundaries");
  if (n_seqs == 0 || max_new == 0 || n_tokens == 0) return 0;
  const int group = n_heads / n_kv_heads;
  BT_CHECK((long long)max_new * group < (1ll << 30), "cache4_attention: %d new tokens of %d heads are too many", max_new, group);
  const int row_tiles = (int)(((long long)max_new * group + rows - 1) / rows);
  const long long units = (long long)n_seqs * n_kv_heads;
  BT_CHECK(units <= 65535 && row_tiles <= 65535 && n_splits >= 1 && n_splits <= 65535, "cache4_attention: grid too large (%lld sequences' heads, %d tiles of rows)",
           units, row_tiles);
  const long long parts = units * row_tiles * n_splits * rows;
  BT_CHECK(n_splits == 1 || (scratch != nullptr && at16(scratch) && scratch_floats >= parts * (dim + 2)),
           "cache4_attention: %d splits need %lld floats of scratch on a 16-byte boundary", n_splits, parts * (dim + 2));
  const Cache4PromptParams p{(const __nv_bfloat16*)q, q_row, (__nv_bfloat16*)out, seq_start, past_len, n_tokens, n_heads, group, rows,
                             scale * 1.4426950408889634f, window, keep_first, scratch, parts * dim,
                             behind_others && n_splits == 1 && units * row_tiles > (sm_count() > 0 ? sm_count() : 148) &&
                                 n_seqs * (long long)row_tiles <= C4P_SORTED};
  const Cache4View c{(unsigned char*)pool, n_pages, table, table_stride, table_len, n_kv_heads, status};
  if (dim == 64) return launch_c4p<64>(p, c, n_seqs, row_tiles, n_splits, stream);
  return launch_c4p<128>(p, c, n_seqs, row_tiles, n_splits, stream);
}
