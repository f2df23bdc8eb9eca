// Files a step's keys and values in the pages of a 4-bit cache (cache4.cuh), and reads them back.
//
// A group is 32 channels of one token and head.  Its scale s is the smallest of the format with 7 s >= max |x|, its codes are
// round(x / s), ties to even, at most 7 in size: all decided exactly, so that the result does not depend on how a division rounds.
// A group that holds an infinity or NaN is filed as NaN.  Values beyond what the format holds (25,088) are held as its largest.
//
// 8,592 tokens of 8 heads of 128 channels, bfloat16, are filed in 11.5 us (3.9 TB/s; 16.8 with scales by comparison and codes one by one) and
// read back in 7.4 (6.0 TB/s into L2); 64 tokens take 2.1 and 1.9.  Reading back is bound by its stores, a decode step by latency.  Filing of many
// is bound by no unit alone (issue slots 56 % active, integer pipe 43): warps wait for their tokens' places and for the four lanes' maxima.
// Four lanes share a group, a lane moves 8 channels in 16-byte pieces (32-bit inputs: two) and the four bytes of their codes beside its
// neighbours'.  A block takes several tokens, a thread the same 8 channels of each, four of them in flight; where a token's records lie is
// looked up once a block, while the first rows come.  Four tokens a block: 11.3; eight in flight: 12.2.
#include "cache4.cuh"
#include "cache4_codes.cuh"

namespace bt {

constexpr int C4_THREADS = 256, C4_AHEAD = 4;

struct Cache4Rows {
  long long k_row, k_head, v_row, v_head;      // elements between tokens and between heads
};
struct Cache4Where {
  const int *positions, *token_seq, *ctx_len;
  int n_tokens, n_table;
};

// 8 channels as they lie in memory, and as numbers.
template <typename T, bool VEC>
struct C4Row {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      T* x = reinterpret_cast<T*>(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = p[i];
    }
  }
  // the largest of the 8 without their signs, as a 32-bit number's bits (above 0x7f800000: NaN)
  __device__ __forceinline__ unsigned top() const {
    if constexpr (sizeof(T) == 2) {
      const unsigned m = 0x7fff7fffu, a = __vmaxu2(__vmaxu2(v[0].x & m, v[0].y & m), __vmaxu2(v[0].z & m, v[0].w & m));
      return max(a << 16, a & 0xffff0000u);
    } else {
      unsigned t = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) t = max(t, reinterpret_cast<const unsigned*>(v)[i] & 0x7fffffffu);
      return t;
    }
  }
  __device__ __forceinline__ float at(int i) const {
    if constexpr (sizeof(T) == 2) {
      const unsigned w = reinterpret_cast<const unsigned*>(v)[i >> 1];
      return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    } else {
      return __uint_as_float(reinterpret_cast<const unsigned*>(v)[i]);
    }
  }
};

// The smallest scale byte with 7 s >= top (finite, not negative); 254 where none has.  The byte is the bits of top / 7 above the third of
// its fraction, rounded up.  bfloat16: top has 8 significant bits and 7 s at most 7, so that top is 7 s or more than 2^-9 away from it,
// and a seventh that is 2^-11 too small takes either to its place.  32-bit: from what may be one too low, by comparing (7 s is exact).
template <typename T>
__device__ __forceinline__ int c4_scale_byte(float top) {
  if constexpr (sizeof(T) == 2) {
    constexpr float kSeventh = (float)((1.0 - 1.0 / 2048.0) / 7.0);
    return min(max((int)((__float_as_uint(top * kSeventh) + 0xfffffu) >> 20) - 107 * 8, 0), 254);
  }
  const int near = (int)(__float_as_uint(top * (1.f / 7.f)) >> 20) - 107 * 8 - 1;
  int b = min(max(near, 0), 254);
#pragma unroll
  for (int i = 0; i < 3; ++i) b += b < 254 && 7.f * c4_scale((unsigned)b) < top ? 1 : 0;
  return b;
}

// A sum that rounds to whole numbers, ties to even: the bits of round(x / s) + kC4Whole.
constexpr float kC4Round = 12582912.f + 8.f;         // 1.5 x 2^23, and the code of 0
constexpr unsigned kC4Whole = 0x4b400000u;

// 32-bit x may lie closer to a tie than a quotient tells: the rest x - r s, which is exact, says on which side.  `inv`: 1 / s, nearly.
__device__ __forceinline__ unsigned c4_code(float x, float s, float inv) {
  float r = x * inv;
  r = rintf(fmaf(fmaf(-r, s, x), inv, r));
  const float rest = fmaf(-r, s, x), half = 0.5f * s;
  const bool odd = (int)fminf(fmaxf(r, -8.f), 8.f) & 1;
  if (fabsf(rest) > half || (fabsf(rest) == half && odd)) r += rest > 0.f ? 1.f : -1.f;
  return __float_as_uint(r + kC4Round);
}

// Two bfloat16 x at once.  x / s is a tie or 2^-9 away from one at least (8 significant bits over 4, 7 at most), so that a quotient rounded to
// whole multiples of 2^-11, by adding 1.5 x 2^12, is as good as the exact one, and 1 / s may be a step off.
__device__ __forceinline__ void c4_codes2(float x, float y, float inv, unsigned& cx, unsigned& cy) {
  constexpr float kFine = 6144.f;
  asm("{\n .reg .b64 v, i, f, c;\n mov.b64 v, {%2, %3};\n mov.b64 i, {%4, %4};\n mov.b64 f, {%5, %5};\n mov.b64 c, {%6, %6};\n"
      " fma.rn.f32x2 v, v, i, f;\n add.rn.f32x2 v, v, c;\n mov.b64 {%0, %1}, v;\n}\n"
      : "=r"(cx), "=r"(cy) : "f"(x), "f"(y), "f"(inv), "f"(kFine), "f"(kC4Round - kFine));
}

// Eight channels' codes, the first lowest, each plus kC4Whole; x is taken into +-7 s first if it is to be `bounded`.
template <typename T, bool VEC>
__device__ __forceinline__ unsigned c4_word(const C4Row<T, VEC>& x, float s, bool bounded) {
  const float most = 7.f * s;
  unsigned word = 0;
  if constexpr (sizeof(T) == 2) {
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
#pragma unroll
    for (int j = 6; j >= 0; j -= 2) {
      unsigned a, b;
      if (bounded)
        c4_codes2(fminf(fmaxf(x.at(j), -most), most), fminf(fmaxf(x.at(j + 1), -most), most), inv, a, b);
      else
        c4_codes2(x.at(j), x.at(j + 1), inv, a, b);
      word = (word * 16u + b) * 16u + a;
    }
  } else {
    const float inv = __frcp_rn(s);
#pragma unroll
    for (int j = 7; j >= 0; --j) word = word * 16u + c4_code(bounded ? fminf(fmaxf(x.at(j), -most), most) : x.at(j), s, inv);
  }
  return word;
}

// Where the tokens t0 .. of a block lie: the byte offset of their page in the pool and their place in it, -1 for one that is not there.
template <int TOKENS>
__device__ __forceinline__ void c4_look_up(const Cache4View& c, const Cache4Where& at, int t0, int dim, bool ring, long long* s_page, int* s_row) {
  const int tid = threadIdx.y * blockDim.x + threadIdx.x;
  if (tid < TOKENS && t0 + tid < at.n_tokens) {
    const int seq = at.token_seq[t0 + tid], pos = at.positions[t0 + tid];
    long long page = -1;
    bool bad = seq < 0 || seq >= at.n_table || pos < 0;
    // (in a ring only the newest positions that it holds are written, so that no two tokens of a step meet)
    if (!bad && !(ring && (long long)pos < (long long)at.ctx_len[seq] - (long long)c.table_len * C4_PAGE)) {
      int entry = pos / C4_PAGE;
      if (entry >= c.table_len) entry %= c.table_len;
      page = c.table[(long long)seq * c.table_stride + entry];
      if (page < 0 || page >= c.n_pages) {
        bad = true;
        page = -1;
      }
    }
    if (bad && c.status) atomicExch(c.status, 9);
    s_page[tid] = page < 0 ? -1 : page * c.n_kv_heads * c4_record(dim);
    s_row[tid] = pos % C4_PAGE;
  }
}

// block (lanes of a head: keys' pieces of 8 channels, then values'; heads); grid (blocks of tokens, blocks of heads)
template <typename T, bool VEC, int TOKENS>
__global__ void __launch_bounds__(C4_THREADS)
cache4_append_kernel(const T* __restrict__ k, const T* __restrict__ v, Cache4Rows rows, Cache4View c, Cache4Where where, int dim) {
  __shared__ long long s_page[TOKENS];
  __shared__ int s_row[TOKENS];
  pdl_trigger();
  pdl_wait();
  const int eighths = dim / 8, which = (int)threadIdx.x >= eighths, at = (int)threadIdx.x - which * eighths;
  const int head = blockIdx.y * blockDim.y + threadIdx.y, t0 = blockIdx.x * TOKENS;
  const bool mine = head < c.n_kv_heads;
  const long long row = which ? rows.v_row : rows.k_row;
  const T* src = (which ? v + head * rows.v_head : k + head * rows.k_head) + at * 8;
  constexpr int AHEAD = TOKENS < C4_AHEAD ? TOKENS : C4_AHEAD;
  C4Row<T, VEC> x[AHEAD];
  auto fetch = [&](int first) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (mine && t0 + first + i < where.n_tokens) x[i].load(src + (t0 + first + i) * row);
  };
  fetch(0);
  c4_look_up<TOKENS>(c, where, t0, dim, true, s_page, s_row);
  __syncthreads();
  if (!mine) return;                           // (whole groups of four lanes: dim / 8 is a multiple of 4)
  const unsigned quad = 0xfu << ((threadIdx.y * blockDim.x + threadIdx.x) & 28);
  unsigned char* const codes = c.pool + (long long)head * c4_record(dim) + which * c4_value_codes(dim) + at * 4;
  unsigned char* const scales = c.pool + (long long)head * c4_record(dim) + c4_key_scales(dim) + which * (2 * dim) + at / 4;
#pragma unroll
  for (int first = 0; first < TOKENS; first += AHEAD) {
    if (first > 0) fetch(first);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int t = first + i;
      if (t0 + t >= where.n_tokens || s_page[t] < 0) continue;      // (the same in the four lanes)
      unsigned top = x[i].top();
      top = max(top, __shfl_xor_sync(quad, top, 1));
      top = max(top, __shfl_xor_sync(quad, top, 2));
      const bool fine = top < 0x7f800000u;
      const int b = fine ? c4_scale_byte<T>(__uint_as_float(top)) : 255;
      const float s = c4_scale((unsigned)b);
      // the largest scale: what its seventh multiple does not reach stays at it
      unsigned word = b == 254 ? c4_word(x[i], s, true) : c4_word(x[i], s, false);
      word = fine ? word - 0x11111111u * kC4Whole : 0x88888888u;
      *reinterpret_cast<unsigned*>(codes + s_page[t] + s_row[t] * (dim / 2)) = word;
      if ((at & 3) == 0) scales[s_page[t] + s_row[t] * (dim / 32)] = (unsigned char)b;
    }
  }
}

template <typename T, bool VEC, int TOKENS>
__global__ void __launch_bounds__(C4_THREADS)
cache4_gather_kernel(T* __restrict__ k, T* __restrict__ v, Cache4Rows rows, Cache4View c, Cache4Where where, int dim) {
  __shared__ long long s_page[TOKENS];
  __shared__ int s_row[TOKENS];
  pdl_trigger();
  pdl_wait();
  const int eighths = dim / 8, which = (int)threadIdx.x >= eighths, at = (int)threadIdx.x - which * eighths;
  const int head = blockIdx.y * blockDim.y + threadIdx.y, t0 = blockIdx.x * TOKENS;
  c4_look_up<TOKENS>(c, where, t0, dim, false, s_page, s_row);
  __syncthreads();
  if (head >= c.n_kv_heads) return;
  const unsigned char* const codes = c.pool + (long long)head * c4_record(dim) + which * c4_value_codes(dim) + at * 4;
  const unsigned char* const scales = c.pool + (long long)head * c4_record(dim) + c4_key_scales(dim) + which * (2 * dim) + at / 4;
  const long long row = which ? rows.v_row : rows.k_row;
  T* dst = (which ? v + head * rows.v_head : k + head * rows.k_head) + at * 8 + t0 * row;
  const C4Bits bits;
  unsigned word[TOKENS], b[TOKENS];
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    word[t] = 0;
    b[t] = 255u;
    if (t0 + t < where.n_tokens && s_page[t] >= 0) {
      word[t] = *reinterpret_cast<const unsigned*>(codes + s_page[t] + s_row[t] * (dim / 2));
      b[t] = scales[s_page[t] + s_row[t] * (dim / 32)];
    }
  }
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    if (t0 + t >= where.n_tokens) break;
    const unsigned s = c4_scale_bits(b[t]), s2 = s | s << 16, shift = c4_shift(s2);
    const unsigned p0 = c4_fma2(c4_pair<0>(word[t], bits), s2, shift), p1 = c4_fma2(c4_pair<1>(word[t], bits), s2, shift);
    const unsigned p2 = c4_fma2(c4_pair<2>(word[t], bits), s2, shift), p3 = c4_fma2(c4_pair<3>(word[t], bits), s2, shift);
    // a pair is channels i and i + 4
    const uint4 y = make_uint4(__byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632), __byte_perm(p2, p3, 0x7632));
    if constexpr (sizeof(T) == 2 && VEC) {
      *reinterpret_cast<uint4*>(dst) = y;
    } else {
      float x[8];
      unpack16(y, x);
      if constexpr (VEC) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) dst[j] = from_float<T>(x[j]);
      }
    }
    dst += row;
  }
}

// Blocks of one token up to here, of eight above: fewer would leave multiprocessors idle.
constexpr int C4_MANY = 2048;

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
  const Cache4Where where{positions, token_seq, ctx_len, n_tokens, n_table};
  const bool vec = c4_whole(k, v, rows, dtype == kF32 ? 4 : 2);
  const dim3 block(dim / 4, C4_THREADS / (dim / 4));
  const int pieces = (n_kv_heads + (int)block.y - 1) / (int)block.y;
  const bool many = (long long)n_tokens * pieces > C4_MANY;
#define BT_C4_APPEND(T, VEC, TOK)                                                                                                         \
  BT_PDL_OK("cache4_append", launch_pdl(cache4_append_kernel<T, VEC, TOK>, dim3((n_tokens + TOK - 1) / TOK, pieces), block, 0, stream, 1, \
                                        (const T*)k, (const T*)v, rows, c, where, dim))
#define BT_C4_APPEND_T(T)                                                          \
  if (vec) {                                                                       \
    if (many) BT_C4_APPEND(T, true, 8); else BT_C4_APPEND(T, true, 1);             \
  } else {                                                                         \
    if (many) BT_C4_APPEND(T, false, 8); else BT_C4_APPEND(T, false, 1);           \
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
  const Cache4Where where{positions, token_seq, nullptr, n_tokens, n_table};
  const bool vec = c4_whole(k, v, rows, dtype == kF32 ? 4 : 2);
  const dim3 block(dim / 4, C4_THREADS / (dim / 4));
  const int pieces = (n_kv_heads + (int)block.y - 1) / (int)block.y;
  const bool many = (long long)n_tokens * pieces > C4_MANY;
#define BT_C4_GATHER(T, VEC, TOK)                                                                                                         \
  BT_PDL_OK("cache4_gather", launch_pdl(cache4_gather_kernel<T, VEC, TOK>, dim3((n_tokens + TOK - 1) / TOK, pieces), block, 0, stream, 1, \
                                        (T*)k, (T*)v, rows, c, where, dim))
#define BT_C4_GATHER_T(T)                                                          \
  if (vec) {                                                                       \
    if (many) BT_C4_GATHER(T, true, 8); else BT_C4_GATHER(T, true, 1);             \
  } else {                                                                         \
    if (many) BT_C4_GATHER(T, false, 8); else BT_C4_GATHER(T, false, 1);           \
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
