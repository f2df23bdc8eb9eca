// Attention over a 4-bit cache (cache4.cuh) for every case: 32-bit and bfloat16 queries, heads of any multiple of 32 channels up to
// 256, shared key heads, a window with kept first positions.
//
// A block is one (query, head).  With the visible keys numbered in a row (kept first ones, then the window's run), it walks them in
// tiles of 128: a thread forms the score of one key, the block the tile's maximum and sum (32-bit, running maximum and sum of a
// softmax over the tiles), then a thread mixes the tile's values for one channel.  Keys that are not visible are never read.
#include "cache4.cuh"

namespace bt {

constexpr int C4S_THREADS = 128;

template <typename T>
__global__ void __launch_bounds__(C4S_THREADS)
cache4_attention_kernel(const T* __restrict__ q, long long q_row, T* __restrict__ out, Cache4View c, const int* __restrict__ seq_start,
                        const int* __restrict__ past_len, int n_heads, int dim, float scale, int window, int keep_first) {
  __shared__ float s_q[256], s_p[C4S_THREADS], scratch[33];
  __shared__ long long s_row[C4S_THREADS];       // the record of each key of the tile, and its place in the page
  pdl_trigger();
  pdl_wait();
  const int seq = blockIdx.z, head = blockIdx.y;
  const int t0 = seq_start[seq], n_new = seq_start[seq + 1] - t0, i = blockIdx.x;
  if (i >= n_new) return;
  const int pos = past_len[seq] + i, kv_head = head / (n_heads / c.n_kv_heads), tid = threadIdx.x;
  int kept, lo;
  c4_seen(pos, window, keep_first, kept, lo);
  const int n_keys = kept + pos - lo + 1;
  for (int d = tid; d < dim; d += C4S_THREADS) s_q[d] = to_float(q[(t0 + i) * q_row + (long long)head * dim + d]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
  for (int first = 0; first < n_keys; first += C4S_THREADS) {
    float score = -INFINITY;
    const int count = min(C4S_THREADS, n_keys - first);
    if (tid < count) {
      const int j = first + tid, key = j < kept ? j : lo + (j - kept);
      const unsigned char* rec = c4_page(c, seq, key / C4_PAGE, kv_head, dim);
      const int in_page = key % C4_PAGE;
      s_row[tid] = (rec - c.pool) * 64 + in_page;
      const uint4* codes = reinterpret_cast<const uint4*>(rec + in_page * (dim / 2));
      const unsigned char* scales = rec + c4_key_scales(dim) + in_page * (dim / 32);
      score = 0.f;
      for (int g = 0; g < dim / 32; ++g) {
        const uint4 raw = codes[g];
        const unsigned w[4] = {raw.x, raw.y, raw.z, raw.w};
        float part = 0.f;
#pragma unroll
        for (int e = 0; e < 32; ++e) part = fmaf((float)((int)(w[e >> 3] >> (4 * (e & 7)) & 15u) - 8), s_q[32 * g + e], part);
        score = fmaf(part, c4_scale(scales[g]), score);
      }
      score *= scale;
    }
    const float m_new = fmaxf(m, block_max(score, scratch));      // (a maximum passes over NaN; the weight and the sum keep it)
    const float weight = tid >= count ? 0.f : m_new == -INFINITY && score == score ? 0.f : expf(score - m_new);
    s_p[tid] = weight;
    const float keep = m == -INFINITY ? 0.f : expf(m - m_new);
    l = l * keep + block_sum(weight, scratch);
    m = m_new;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int d = tid + h * C4S_THREADS;
      if (d >= dim) continue;
      float sum = 0.f;
      for (int j = 0; j < count; ++j) {
        const int in_page = (int)(s_row[j] & 63);
        const unsigned char* rec = c.pool + (s_row[j] >> 6);
        const unsigned n = rec[c4_value_codes(dim) + in_page * (dim / 2) + d / 2] >> (4 * (d & 1)) & 15u;
        sum = fmaf(s_p[j], (float)((int)n - 8) * c4_scale(rec[c4_value_scales(dim) + in_page * (dim / 32) + d / 32]), sum);
      }
      acc[h] = acc[h] * keep + sum;
    }
    __syncthreads();
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int d = tid + h * C4S_THREADS;
    if (d < dim) out[((long long)(t0 + i) * n_heads + head) * dim + d] = from_float<T>(acc[h] / l);
  }
}

}  // namespace bt

// q: rows of n_heads heads of `dim` channels, `q_row` elements apart; out: [tokens][n_heads * dim].  dtype: 0 32-bit, 1 bfloat16.
extern "C" int bt_cache4_attention(const void* q, long long q_row, void* out, const void* pool, long long n_pages, const int* table,
                                   int table_stride, int table_len, int* status, const int* seq_start, const int* past_len, int n_seqs,
                                   int max_new, int n_heads, int n_kv_heads, int dim, float scale, int window, int keep_first, int dtype,
                                   cudaStream_t stream) {
  using namespace bt;
  BT_CHECK(dim > 0 && dim <= 256 && dim % 32 == 0, "cache4_attention: heads of %d channels; the 4-bit cache takes multiples of 32 up to 256", dim);
  BT_CHECK(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0 && n_heads <= 65535,
           "cache4_attention: %d query heads cannot share %d key heads", n_heads, n_kv_heads);
  BT_CHECK(n_pages > 0 && table != nullptr && table_len > 0 && n_seqs >= 0 && max_new >= 0 && window >= 0 && keep_first >= 0,
           "cache4_attention: bad sizes pages=%lld table_len=%d sequences=%d window=%d kept=%d", n_pages, table_len, n_seqs, window, keep_first);
  BT_CHECK((unsigned long long)pool % 16 == 0, "cache4_attention: the pool must start on a 16-byte boundary");
  BT_CHECK(n_seqs <= 65535, "cache4_attention: %d sequences are too many for one launch", n_seqs);
  BT_CHECK(dtype == kF32 || dtype == kBF16, "cache4_attention: unknown element type %d", dtype);
  if (n_seqs == 0 || max_new == 0) return 0;
  const Cache4View c{(unsigned char*)pool, n_pages, table, table_stride, table_len, n_kv_heads, status};
  const dim3 grid(max_new, n_heads, n_seqs);
  if (dtype == kF32)
    BT_PDL_OK("cache4_attention", launch_pdl(cache4_attention_kernel<float>, grid, dim3(C4S_THREADS), 0, stream, 1, (const float*)q, q_row,
                                             (float*)out, c, seq_start, past_len, n_heads, dim, scale, window, keep_first));
  else
    BT_PDL_OK("cache4_attention", launch_pdl(cache4_attention_kernel<__nv_bfloat16>, grid, dim3(C4S_THREADS), 0, stream, 1,
                                             (const __nv_bfloat16*)q, q_row, (__nv_bfloat16*)out, c, seq_start, past_len, n_heads, dim, scale,
                                             window, keep_first));
  return 0;
}
