// Attention over a 4-bit cache (cache4.cuh) for every case, in 32-bit arithmetic: 32-bit and bfloat16 queries, heads of any multiple of
// 32 channels up to 256, shared key heads, a window with kept first positions.
//
// A block serves one (sequence, key head) and up to 8 rows: row r is query head r % group of new token r / group.  With the keys that any
// of its rows sees numbered in a row (kept first ones, then the window's run), it walks them in tiles of 256: a thread takes two keys' codes
// apart and forms their scores for all rows, the block each row's maximum and sum (a running softmax), then a thread mixes its share of
// the tile's values for four channels of all rows.  Keys that a row does not see have the weight 0 and their values are left out, so that
// what lies there (NaN) does not matter.
//
// What bounds it is the 32-bit multiply-adds and the reading of queries and weights from shared memory beside them; one row a block takes a
// code apart for each multiply-add, eight for eight: two prompts of 4,096 tokens, 32 heads over 8 of 128, in 32 bits, take 13.5 ms (20 TFLOP/s;
// one row a block and one key a thread: 78), one sequence of 32,766 108 us.  Where rows and heads do not fill the GPU the keys are cut into pieces, whose results a
// second kernel joins in order.
#include "cache4.cuh"

namespace bt {

constexpr int C4S_THREADS = 128, C4S_KEYS = 2, C4S_TILE = C4S_KEYS * C4S_THREADS;

struct Cache4AnyParams {
  const void* q;
  long long q_row;
  void* out;
  const int *seq_start, *past_len;
  int n_tokens, n_heads, group, dim;
  float scale;
  int window, keep_first, pieces;
  float* part;                 // [unit][piece][row][dim], then [unit][piece][row][2]
  long long part_ml;
};

// A block's rows and the keys that any of them sees.
struct C4Any {
  int t0, n_rows, row0, past, kept, lo, n_keys;
  __device__ C4Any(const Cache4AnyParams& p, int seq, int row_block, int rows, int* status) {
    int n_new;
    c4_new_tokens(p.seq_start, seq, p.n_tokens, t0, n_new);
    row0 = row_block * rows;
    n_rows = min(rows, n_new * p.group - row0);
    past = c4_past(p.past_len, seq, status);
    const int first = past + row0 / p.group, last = past + (row0 + max(n_rows, 1) - 1) / p.group;
    int none;
    c4_seen(first, p.window, p.keep_first, none, lo);
    kept = min(p.window > 0 ? min(p.keep_first, last + 1) : 0, lo);
    n_keys = kept + last - lo + 1;
  }
  __device__ int key(int i) const { return i < kept ? i : lo + (i - kept); }
};

// A code as a number: 2^23 + n by its bits, less 2^23 + 8.
__device__ __forceinline__ float c4_number(unsigned code) { return __uint_as_float(0x4b000000u | code) - 8388616.f; }

template <typename T, int ROWS>
__global__ void __launch_bounds__(C4S_THREADS)
cache4_attention_kernel(Cache4AnyParams p, Cache4View c) {
  __shared__ __align__(16) float s_q[ROWS][256];
  __shared__ __align__(16) float s_p[C4S_TILE][ROWS];
  __shared__ const unsigned char* s_rec[C4S_TILE];
  __shared__ int s_in[C4S_TILE];
  __shared__ float s_red[2][C4S_THREADS / 32][ROWS];
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, dim = p.dim, seq = blockIdx.z, kv_head = blockIdx.y;
  const int piece = (int)blockIdx.x % p.pieces, row_block = (int)blockIdx.x / p.pieces;
  const C4Any at(p, seq, row_block, ROWS, c.status);
  if (at.n_rows <= 0) return;
  const int per = (at.n_keys + p.pieces - 1) / p.pieces, begin = piece * per, end = min(at.n_keys, begin + per);
  if (begin >= end) return;
  for (int i = tid; i < ROWS * dim; i += C4S_THREADS) {
    const int r = i / dim, d = i % dim, row = at.row0 + r;
    float x = 0.f;
    if (r < at.n_rows)
      x = to_float(reinterpret_cast<const T*>(p.q)[(at.t0 + row / p.group) * p.q_row + (long long)(kv_head * p.group + row % p.group) * dim + d]);
    s_q[r][d] = x;
  }
  // this thread's four channels, and which share of a tile's keys it mixes
  const int quads = dim / 4, shares = C4S_THREADS / quads, share = tid / quads, d0 = tid % quads * 4;
  float m[ROWS], l[ROWS], acc[4][ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i][r] = 0.f;
  }
  for (int first = begin; first < end; first += C4S_TILE) {
    const int count = min(C4S_TILE, end - first);
    float score[C4S_KEYS][ROWS];
    unsigned sees[C4S_KEYS];             // a bit a row
    __syncthreads();           // (the tile before has been mixed; the queries are there)
    const uint4* codes[C4S_KEYS];
    const unsigned char* scales[C4S_KEYS];
#pragma unroll
    for (int k = 0; k < C4S_KEYS; ++k) {
      const int j = min(tid + k * C4S_THREADS, count - 1);      // (a thread without a key of its own takes the last)
      const int key = at.key(first + j), in_page = key % C4_PAGE;
      const unsigned char* rec = c4_page(c, seq, key / C4_PAGE, kv_head, dim);
      if (tid + k * C4S_THREADS < count) {
        s_rec[j] = rec;
        s_in[j] = in_page;
      }
      codes[k] = reinterpret_cast<const uint4*>(rec + in_page * (dim / 2));
      scales[k] = rec + c4_key_scales(dim) + in_page * (dim / 32);
      sees[k] = 0u;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        score[k][r] = 0.f;
        const int pos = at.past + (at.row0 + r) / p.group;
        if (tid + k * C4S_THREADS < count && r < at.n_rows && key <= pos && (p.window <= 0 || key > pos - p.window || key < p.keep_first))
          sees[k] |= 1u << r;
      }
    }
    for (int g = 0; g < dim / 32; ++g) {
      unsigned w[C4S_KEYS][4];
      float part[C4S_KEYS][ROWS];
#pragma unroll
      for (int k = 0; k < C4S_KEYS; ++k) {
        const uint4 raw = codes[k][g];
        w[k][0] = raw.x; w[k][1] = raw.y; w[k][2] = raw.z; w[k][3] = raw.w;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) part[k][r] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 32; e += 4) {
        float x[C4S_KEYS][4];
#pragma unroll
        for (int k = 0; k < C4S_KEYS; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) x[k][i] = c4_number(w[k][e >> 3] >> (4 * ((e & 7) + i)) & 15u);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float4 q = *reinterpret_cast<const float4*>(&s_q[r][32 * g + e]);
#pragma unroll
          for (int k = 0; k < C4S_KEYS; ++k)
            part[k][r] = fmaf(x[k][0], q.x, fmaf(x[k][1], q.y, fmaf(x[k][2], q.z, fmaf(x[k][3], q.w, part[k][r]))));
        }
      }
#pragma unroll
      for (int k = 0; k < C4S_KEYS; ++k) {
        const float s = c4_scale(scales[k][g]);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) score[k][r] = fmaf(part[k][r], s, score[k][r]);
      }
    }
    // each row's maximum over the tile (a maximum passes over NaN; the weight and the sum keep it)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < C4S_KEYS; ++k) {
        score[k][r] *= p.scale;
        if (sees[k] >> r & 1u) top = fmaxf(top, score[k][r]);
      }
      top = warp_max(top);
      if (lane == 0) s_red[0][warp][r] = top;
    }
    __syncthreads();
    float keep[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float m_new = m[r], sum = 0.f;
#pragma unroll
      for (int i = 0; i < C4S_THREADS / 32; ++i) m_new = fmaxf(m_new, s_red[0][i][r]);
#pragma unroll
      for (int k = 0; k < C4S_KEYS; ++k) {
        const bool mine = sees[k] >> r & 1u;
        const float weight = !mine || (m_new == -INFINITY && score[k][r] == score[k][r]) ? 0.f : expf(score[k][r] - m_new);
        sum += weight;
        // (a key that this row does not see: its values are left out, by a weight that no other has)
        s_p[tid + k * C4S_THREADS][r] = mine ? weight : -1.f;
      }
      keep[r] = m[r] == -INFINITY ? 0.f : expf(m[r] - m_new);
      m[r] = m_new;
      sum = warp_sum(sum);
      if (lane == 0) s_red[1][warp][r] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < C4S_THREADS / 32; ++i) sum += s_red[1][i][r];
      l[r] = l[r] * keep[r] + sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i][r] *= keep[r];
    }
    if (share < shares) {
#pragma unroll 2
      for (int j = share; j < count; j += shares) {
        const unsigned char* rec = s_rec[j];
        const int in_page = s_in[j];
        const unsigned n = *reinterpret_cast<const unsigned short*>(rec + c4_value_codes(dim) + in_page * (dim / 2) + d0 / 2);
        const float s = c4_scale(rec[c4_value_scales(dim) + in_page * (dim / 32) + d0 / 32]);
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = c4_number(n >> (4 * i) & 15u) * s;
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
          const float w = s_p[j][r];
          if (w >= 0.f || w != w) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i][r] = fmaf(w, v[i], acc[i][r]);
          }
        }
      }
    }
  }
  // the shares of a channel, joined in order (over the queries)
  float(*s_acc)[256] = s_q;
  for (int from = 1; from < shares; ++from) {
    __syncthreads();
    if (share == from) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r) *reinterpret_cast<float4*>(&s_acc[r][d0]) = make_float4(acc[0][r], acc[1][r], acc[2][r], acc[3][r]);
    }
    __syncthreads();
    if (share == 0) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i][r] += s_acc[r][d0 + i];
    }
  }
  if (share != 0) return;
  const long long unit = ((long long)seq * gridDim.y + kv_head) * ((int)gridDim.x / p.pieces) + row_block;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (r >= at.n_rows) continue;
    const int row = at.row0 + r;
    const long long place = (unit * p.pieces + piece) * ROWS + r;
    T* dst = reinterpret_cast<T*>(p.out) + ((long long)(at.t0 + row / p.group) * p.n_heads + kv_head * p.group + row % p.group) * dim + d0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p.pieces == 1)
        dst[i] = from_float<T>(acc[i][r] / l[r]);
      else
        p.part[place * dim + d0 + i] = acc[i][r];
    }
    if (p.pieces > 1 && d0 == 0) {
      p.part[p.part_ml + 2 * place] = m[r];
      p.part[p.part_ml + 2 * place + 1] = l[r];
    }
  }
}

// Joins a row's pieces in their order: a block a row.
template <typename T, int ROWS>
__global__ void __launch_bounds__(C4S_THREADS)
cache4_attention_join_kernel(Cache4AnyParams p) {
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.z, kv_head = blockIdx.y, row_block = (int)blockIdx.x / ROWS, r = (int)blockIdx.x % ROWS, dim = p.dim;
  const C4Any at(p, seq, row_block, ROWS, nullptr);
  if (r >= at.n_rows) return;
  const int per = (at.n_keys + p.pieces - 1) / p.pieces, used = (at.n_keys + per - 1) / per;
  const long long unit = ((long long)seq * gridDim.y + kv_head) * ((int)gridDim.x / ROWS) + row_block;
  const int row = at.row0 + r;
  for (int d = threadIdx.x; d < dim; d += C4S_THREADS) {
    float top = -INFINITY, sum = 0.f, o = 0.f;
    for (int s = 0; s < used; ++s) {
      const long long place = (unit * p.pieces + s) * ROWS + r;
      const float m = p.part[p.part_ml + 2 * place], l = p.part[p.part_ml + 2 * place + 1], x = p.part[place * dim + d];
      const float m_new = fmaxf(top, m), use = m_new == -INFINITY ? 0.f : m_new;
      const float a = expf(top - use), b = expf(m - use);
      sum = sum * a + l * b;
      o = o * a + x * b;
      top = m_new;
    }
    reinterpret_cast<T*>(p.out)[((long long)(at.t0 + row / p.group) * p.n_heads + kv_head * p.group + row % p.group) * dim + d] = from_float<T>(o / sum);
  }
}

template <typename T, int ROWS>
static int launch_c4s(const Cache4AnyParams& p, const Cache4View& c, int n_seqs, int row_blocks, cudaStream_t stream) {
  BT_PDL_OK("cache4_attention", launch_pdl(cache4_attention_kernel<T, ROWS>, dim3(row_blocks * p.pieces, c.n_kv_heads, n_seqs), dim3(C4S_THREADS), 0,
                                           stream, 1, p, c));
  if (p.pieces > 1)
    BT_PDL_OK("cache4_attention_join", launch_pdl(cache4_attention_join_kernel<T, ROWS>, dim3(row_blocks * ROWS, c.n_kv_heads, n_seqs),
                                                  dim3(C4S_THREADS), 0, stream, 1, p));
  return 0;
}

}  // namespace bt

// q: rows of n_heads heads of `dim` channels, `q_row` elements apart; out: [tokens][n_heads * dim].  dtype: 0 32-bit, 1 bfloat16.  rows: 1
// or 8 a block.  scratch, 32-bit words for more than one piece: n_seqs * n_kv_heads * row blocks * pieces * rows * (dim + 2).
extern "C" int bt_cache4_attention(const void* q, long long q_row, void* out, const void* pool, long long n_pages, const int* table,
                                   int table_stride, int table_len, int* status, const int* seq_start, const int* past_len, int n_tokens,
                                   int n_seqs, int max_new, int n_heads, int n_kv_heads, int dim, float scale, int window, int keep_first,
                                   int pieces, int rows, float* scratch, long long scratch_floats, int dtype, cudaStream_t stream) {
  using namespace bt;
  BT_CHECK(dim > 0 && dim <= 256 && dim % 32 == 0, "cache4_attention: heads of %d channels; the 4-bit cache takes multiples of 32 up to 256", dim);
  BT_CHECK(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads <= 65535,
           "cache4_attention: %d query heads cannot share %d key heads", n_heads, n_kv_heads);
  BT_CHECK(n_pages > 0 && table != nullptr && table_len > 0 && n_seqs >= 0 && max_new >= 0 && window >= 0 && keep_first >= 0,
           "cache4_attention: bad sizes pages=%lld table_len=%d sequences=%d window=%d kept=%d", n_pages, table_len, n_seqs, window, keep_first);
  BT_CHECK((unsigned long long)pool % 16 == 0, "cache4_attention: the pool must start on a 16-byte boundary");
  BT_CHECK(n_seqs <= 65535, "cache4_attention: %d sequences are too many for one launch", n_seqs);
  BT_CHECK(dtype == kF32 || dtype == kBF16, "cache4_attention: unknown element type %d", dtype);
  BT_CHECK((rows == 1 || rows == 8) && pieces >= 1, "cache4_attention: %d rows a block, %d pieces", rows, pieces);
  if (n_seqs == 0 || max_new == 0 || n_tokens == 0) return 0;
  const int group = n_heads / n_kv_heads;
  const long long blocks = ((long long)max_new * group + rows - 1) / rows;
  BT_CHECK(blocks * rows * pieces < (1ll << 31), "cache4_attention: %d new tokens of %d heads in %d pieces are too many", max_new, group, pieces);
  const long long parts = (long long)n_seqs * n_kv_heads * blocks * pieces * rows;
  BT_CHECK(pieces == 1 || (scratch != nullptr && scratch_floats >= parts * (dim + 2)), "cache4_attention: %d pieces need %lld floats of scratch",
           pieces, parts * (dim + 2));
  const Cache4AnyParams p{q, q_row, out, seq_start, past_len, n_tokens, n_heads, group, dim, scale, window, keep_first, pieces, scratch, parts * dim};
  const Cache4View c{(unsigned char*)pool, n_pages, table, table_stride, table_len, n_kv_heads, status};
  if (dtype == kF32)
    return rows == 1 ? launch_c4s<float, 1>(p, c, n_seqs, (int)blocks, stream) : launch_c4s<float, 8>(p, c, n_seqs, (int)blocks, stream);
  return rows == 1 ? launch_c4s<__nv_bfloat16, 1>(p, c, n_seqs, (int)blocks, stream) : launch_c4s<__nv_bfloat16, 8>(p, c, n_seqs, (int)blocks, stream);
}
