// Files a step's keys and values in the pages of a 4-bit cache (cache4.cuh), and reads them back.
//
// A group is 32 channels of one token and head.  Its scale s is the smallest of the format with 7 s >= max |x|, its codes are
// round(x / s), ties to even, at most 7 in size: all decided exactly, so that the result does not depend on how a division rounds.
// A group that holds an infinity or NaN is filed as NaN.  Values beyond what the format holds (25,088) are held as its largest.
//
// Both are bound by memory and, for a decode step, by latency: four lanes share a group, a lane moves 8 channels in 16-byte pieces
// (32-bit inputs: two), and the four bytes of codes beside its neighbours'.  A block takes several tokens, a thread the same 8
// channels of each, so that their loads are in flight together.
#include "cache4.cuh"

namespace bt {

constexpr int C4_THREADS = 256;

struct Cache4Rows {
  long long k_row, k_head, v_row, v_head;      // elements between tokens and between heads
};

template <typename T, bool VEC>
__device__ __forceinline__ void c4_load8(const T* p, float (&x)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_float(p[i]);
  } else if constexpr (sizeof(T) == 2) {
    unpack16(*reinterpret_cast<const uint4*>(p), x);
  } else {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void c4_store8(T* p, const float (&x)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = from_float<T>(x[i]);
  } else if constexpr (sizeof(T) == 2) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);      // (exact: the values have 7 bits)
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
}

// The smallest scale byte with 7 s >= top (finite, not negative); 254 where none has.
__device__ __forceinline__ int c4_scale_byte(float top) {
  // the bits of top / 7 above the third of its fraction are the byte, give or take one for the rounding
  const int near = (int)(__float_as_uint(top * (1.f / 7.f)) >> 20) - 107 * 8 - 1;
  int b = min(max(near, 0), 254);
#pragma unroll
  for (int i = 0; i < 3; ++i) b += b < 254 && 7.f * c4_scale((unsigned)b) < top ? 1 : 0;      // (7 s is exact)
  return b;
}

// round(x / s) + 8, ties to even, in the last four bits.  `inv`: 1 / s rounded.
// bfloat16 x: the corrected quotient is x / s rounded to 24 bits, which is no tie unless x / s is one (x and (k + 1/2) s have 8
// significant bits each, so that they are equal or differ by more than 2^-9 of x).  32-bit x may lie closer to a tie than a quotient
// tells: the rest x - r s, which is exact, says on which side.
template <typename T>
__device__ __forceinline__ unsigned c4_code(float x, float s, float inv) {
  constexpr float kMagic = 12582912.f;         // 1.5 x 2^23: a sum with it rounds to whole numbers
  float r = x * inv;
  r = fmaf(fmaf(-r, s, x), inv, r);
  if constexpr (sizeof(T) == 4) {
    r = rintf(r);
    const float rest = fmaf(-r, s, x), half = 0.5f * s;
    const bool odd = (int)fminf(fmaxf(r, -8.f), 8.f) & 1;
    if (fabsf(rest) > half || (fabsf(rest) == half && odd)) r += rest > 0.f ? 1.f : -1.f;
  }
  return __float_as_uint(r + (kMagic + 8.f)) & 15u;
}

// grid (blocks of tokens, pieces of a token's lanes); a lane: (head, key or value, 8 channels)
template <typename T, bool VEC, int TOKENS>
__global__ void __launch_bounds__(C4_THREADS)
cache4_append_kernel(const T* __restrict__ k, const T* __restrict__ v, Cache4Rows rows, Cache4View c, const int* __restrict__ positions,
                     const int* __restrict__ token_seq, const int* __restrict__ ctx_len, int n_tokens, int n_table, int dim) {
  pdl_trigger();
  pdl_wait();
  const int lane = blockIdx.y * C4_THREADS + threadIdx.x;
  const int eighths = dim / 8;
  const int head = lane / (2 * eighths);
  if (head >= c.n_kv_heads) return;            // (whole groups of four lanes: dim / 8 is a multiple of 4)
  const int which = lane / eighths & 1, at = lane % eighths;
  const unsigned quad = 0xfu << (threadIdx.x & 28);
  const T* src = which ? v + head * rows.v_head : k + head * rows.k_head;
  const long long row = which ? rows.v_row : rows.k_row;
  const int t0 = blockIdx.x * TOKENS;
  float x[TOKENS][8];
  unsigned char* rec[TOKENS];                  // null: not filed
  int in_page[TOKENS];
#pragma unroll
  for (int i = 0; i < TOKENS; ++i)
    if (t0 + i < n_tokens) c4_load8<T, VEC>(src + (t0 + i) * row + at * 8, x[i]);
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    rec[i] = nullptr;
    in_page[i] = 0;
    if (t0 + i >= n_tokens) continue;
    const int seq = token_seq[t0 + i], pos = positions[t0 + i];
    if (seq < 0 || seq >= n_table || pos < 0) {
      if (c.status) atomicExch(c.status, 9);
      continue;
    }
    // (in a ring only the newest positions that it holds are written, so that no two tokens of a step meet)
    if ((long long)pos < (long long)ctx_len[seq] - (long long)c.table_len * C4_PAGE) continue;
    const int page = c.table[(long long)seq * c.table_stride + pos / C4_PAGE % c.table_len];
    if (page < 0 || page >= c.n_pages) {
      if (c.status) atomicExch(c.status, 9);
      continue;
    }
    in_page[i] = pos % C4_PAGE;
    rec[i] = c.pool + ((long long)page * c.n_kv_heads + head) * c4_record(dim);
  }
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    if (rec[i] == nullptr) continue;           // (the same in the four lanes)
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[i][j]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(quad, top, 1));
    top = max(top, __shfl_xor_sync(quad, top, 2));
    const bool fine = top < 0x7f800000u;
    const int b = fine ? c4_scale_byte(__uint_as_float(top)) : 255;
    const float s = c4_scale((unsigned)b), inv = 1.f / s;
    if (b == 254) {                            // the largest scale: what its seventh multiple does not reach stays at it
#pragma unroll
      for (int j = 0; j < 8; ++j) x[i][j] = fminf(fmaxf(x[i][j], -7.f * s), 7.f * s);
    }
    unsigned word = 0;
#pragma unroll
    for (int j = 7; j >= 0; --j) word = word * 16u + c4_code<T>(x[i][j], s, inv);
    if (!fine) word = 0x88888888u;
    *reinterpret_cast<unsigned*>(rec[i] + which * c4_value_codes(dim) + in_page[i] * (dim / 2) + at * 4) = word;
    if ((at & 3) == 0) rec[i][c4_key_scales(dim) + which * (2 * dim) + in_page[i] * (dim / 32) + at / 4] = (unsigned char)b;
  }
}

template <typename T, bool VEC, int TOKENS>
__global__ void __launch_bounds__(C4_THREADS)
cache4_gather_kernel(T* __restrict__ k, T* __restrict__ v, Cache4Rows rows, Cache4View c, const int* __restrict__ positions,
                     const int* __restrict__ token_seq, int n_tokens, int n_table, int dim) {
  pdl_trigger();
  pdl_wait();
  const int lane = blockIdx.y * C4_THREADS + threadIdx.x;
  const int eighths = dim / 8;
  const int head = lane / (2 * eighths), t0 = blockIdx.x * TOKENS;
  if (head >= c.n_kv_heads) return;
  const int which = lane / eighths & 1, at = lane % eighths;
  T* dst = (which ? v + head * rows.v_head : k + head * rows.k_head) + at * 8;
  const long long row = which ? rows.v_row : rows.k_row;
  unsigned word[TOKENS], b[TOKENS];
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    word[i] = 0;
    b[i] = 255u;
    if (t0 + i >= n_tokens) continue;
    const int seq = token_seq[t0 + i], pos = positions[t0 + i];
    int page = -1;
    if (seq >= 0 && seq < n_table && pos >= 0) page = c.table[(long long)seq * c.table_stride + pos / C4_PAGE % c.table_len];
    if (page < 0 || page >= c.n_pages) {
      if (c.status) atomicExch(c.status, 9);
      continue;
    }
    const int in_page = pos % C4_PAGE;
    const unsigned char* rec = c.pool + ((long long)page * c.n_kv_heads + head) * c4_record(dim);
    word[i] = *reinterpret_cast<const unsigned*>(rec + which * c4_value_codes(dim) + in_page * (dim / 2) + at * 4);
    b[i] = rec[c4_key_scales(dim) + which * (2 * dim) + in_page * (dim / 32) + at / 4];
  }
#pragma unroll
  for (int i = 0; i < TOKENS; ++i) {
    if (t0 + i >= n_tokens) break;
    const float s = c4_scale(b[i]);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)((int)(word[i] >> (4 * j) & 15u) - 8) * s;
    c4_store8<T, VEC>(dst + (t0 + i) * row, x);
  }
}

static int c4_check(const char* what, const void* pool, long long n_pages, const int* table, int table_len, int n_tokens, int n_kv_heads,
                    int dim) {
  BT_CHECK(dim > 0 && dim <= 256 && dim % 32 == 0, "%s: heads of %d channels; the 4-bit cache takes multiples of 32 up to 256", what, dim);
  BT_CHECK(n_kv_heads > 0 && n_kv_heads <= 65535 && n_pages > 0 && table != nullptr && table_len > 0 && n_tokens >= 0,
           "%s: bad sizes heads=%d pages=%lld table_len=%d tokens=%d", what, n_kv_heads, n_pages, table_len, n_tokens);
  BT_CHECK((unsigned long long)pool % 16 == 0, "%s: the pool must start on a 16-byte boundary", what);
  return 0;
}

static bool c4_whole(const void* k, const void* v, const Cache4Rows& r, int es) {
  const long long step = 16 / es;
  return ((unsigned long long)k | (unsigned long long)v) % 16 == 0 && r.k_row % step == 0 && r.k_head % step == 0 && r.v_row % step == 0 &&
         r.v_head % step == 0;
}

}  // namespace bt

// k, v: `n_tokens` rows of n_kv_heads heads of `dim` channels, strides in elements.  dtype: 0 32-bit, 1 bfloat16.
extern "C" int bt_cache4_append(const void* k, long long k_row, long long k_head, const void* v, long long v_row, long long v_head,
                                void* pool, long long n_pages, const int* positions, const int* token_seq, const int* ctx_len,
                                const int* table, int n_table, int table_stride, int table_len, int* status, int n_tokens,
                                int n_kv_heads, int dim, int dtype, cudaStream_t stream) {
  using namespace bt;
  if (int rc = c4_check("cache4_append", pool, n_pages, table, table_len, n_tokens, n_kv_heads, dim)) return rc;
  BT_CHECK(dtype == kF32 || dtype == kBF16, "cache4_append: unknown element type %d", dtype);
  if (n_tokens == 0) return 0;
  const Cache4Rows rows{k_row, k_head, v_row, v_head};
  const Cache4View c{(unsigned char*)pool, n_pages, table, table_stride, table_len, n_kv_heads, status};
  const int lanes = n_kv_heads * dim / 4, pieces = (lanes + C4_THREADS - 1) / C4_THREADS;
  const bool vec = c4_whole(k, v, rows, dtype == kF32 ? 4 : 2);
  // several tokens a block once there are enough of them to fill the GPU
  const bool many = (long long)n_tokens * pieces > 4096;
  const int per = many ? 4 : 1;
  const dim3 grid((n_tokens + per - 1) / per, pieces);
#define BT_C4_APPEND(T, VEC, TOK)                                                                                                     \
  BT_PDL_OK("cache4_append", launch_pdl(cache4_append_kernel<T, VEC, TOK>, grid, dim3(C4_THREADS), 0, stream, 1, (const T*)k, (const T*)v, \
                                        rows, c, positions, token_seq, ctx_len, n_tokens, n_table, dim))
#define BT_C4_APPEND_T(T)                                                          \
  if (vec) {                                                                       \
    if (many) BT_C4_APPEND(T, true, 4); else BT_C4_APPEND(T, true, 1);             \
  } else {                                                                         \
    if (many) BT_C4_APPEND(T, false, 4); else BT_C4_APPEND(T, false, 1);           \
  }
  if (dtype == kF32) {
    BT_C4_APPEND_T(float)
  } else {
    BT_C4_APPEND_T(__nv_bfloat16)
  }
#undef BT_C4_APPEND_T
#undef BT_C4_APPEND
  return 0;
}

extern "C" int bt_cache4_gather(void* k, long long k_row, long long k_head, void* v, long long v_row, long long v_head, const void* pool,
                                long long n_pages, const int* positions, const int* token_seq, const int* table, int n_table,
                                int table_stride, int table_len, int* status, int n_tokens, int n_kv_heads, int dim, int dtype,
                                cudaStream_t stream) {
  using namespace bt;
  if (int rc = c4_check("cache4_gather", pool, n_pages, table, table_len, n_tokens, n_kv_heads, dim)) return rc;
  BT_CHECK(dtype == kF32 || dtype == kBF16, "cache4_gather: unknown element type %d", dtype);
  if (n_tokens == 0) return 0;
  const Cache4Rows rows{k_row, k_head, v_row, v_head};
  const Cache4View c{(unsigned char*)pool, n_pages, table, table_stride, table_len, n_kv_heads, status};
  const int lanes = n_kv_heads * dim / 4;
  const bool vec = c4_whole(k, v, rows, dtype == kF32 ? 4 : 2);
  const int pieces = (lanes + C4_THREADS - 1) / C4_THREADS;
  const bool many = (long long)n_tokens * pieces > 4096;
  const dim3 grid(many ? (n_tokens + 3) / 4 : n_tokens, pieces);
#define BT_C4_GATHER(T, VEC, TOK)                                                                                                   \
  BT_PDL_OK("cache4_gather", launch_pdl(cache4_gather_kernel<T, VEC, TOK>, grid, dim3(C4_THREADS), 0, stream, 1, (T*)k, (T*)v, rows, c, \
                                        positions, token_seq, n_tokens, n_table, dim))
#define BT_C4_GATHER_T(T)                                                          \
  if (vec) {                                                                       \
    if (many) BT_C4_GATHER(T, true, 4); else BT_C4_GATHER(T, true, 1);             \
  } else {                                                                         \
    if (many) BT_C4_GATHER(T, false, 4); else BT_C4_GATHER(T, false, 1);           \
  }
  if (dtype == kF32) {
    BT_C4_GATHER_T(float)
  } else {
    BT_C4_GATHER_T(__nv_bfloat16)
  }
#undef BT_C4_GATHER_T
#undef BT_C4_GATHER
  return 0;
}
