// Norms of a step's query and key heads and their rotation by position, in one pass over the projections.
//
// Per token and head: y = x / sqrt(mean(x^2) + eps) * weight (one weight for all query heads, one for all key heads; without
// weights x as it is), then pairs of the first `rot` channels, (i, i + rot / 2) or (2i, 2i + 1), turned by pos * f_i with cosine and
// sine times `size`.  Sums and products are 32-bit, rounded once.  Angles: pos * f_i is formed in 64 bits and taken into one turn
// there, so that far positions lose nothing by the product (in 32 bits it is off by pos * f / 2^24: 0.06 at position 10^6).  The frequencies
// come as 32-bit numbers: where they were rounded to that, the angle of f itself is off by up to pos / 2^25, 0.03 there.
//
// Bound by memory: every channel is read and written once.  A warp takes one token and some of its heads.  Its lanes form the token's cosines
// and sines once, in shared memory, and a lane keeps what its eight pairs are multiplied by in registers; it holds 16 channels of a head
// (the two pieces of 8 that turn into one another, or 16 in a row), so that nothing but the norm's sum goes between lanes.  How many
// heads a warp takes: all of them when there are enough tokens to fill the GPU, as few as fit its lanes when there are not.
// 16,384 tokens of 32 + 8 heads of 128 channels, bfloat16: 63 us, 5.3 TB/s (with factors formed for every head and single
// multiply-adds: 94); 8 tokens: 2.3.
#include "common.cuh"

namespace bt {

constexpr int QN_WARPS = 8;

struct QnParams {
  const void* src;
  void* dst;
  long long src_row, dst_row;          // elements between tokens
  const int* positions;
  const float* freq;                   // [rot / 2]
  const float *q_weight, *k_weight;    // [dim] or null
  int n_tokens, n_heads, n_vecs;       // n_vecs: query heads and key heads, side by side
  int dim, rot;
  int vecs_per_warp, warps_per_token;
  float eps, size;
  int interleaved, normed;
};

__device__ __forceinline__ float2 qn_turn(int pos, float f, float size) {
  double t = (double)pos * (double)f * 0.31830988618379067154;      // half turns
  t -= 2.0 * rint(0.5 * t);
  float s, c;
  sincospif((float)t, &s, &c);
  return make_float2(c * size, s * size);
}

// 16 channels of a lane, in two pieces of 8 as they lie in memory.
template <typename T>
struct QnRaw {
  uint4 v[sizeof(T)];
  __device__ __forceinline__ void load(const T* a, const T* b) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      v[i] = reinterpret_cast<const uint4*>(a)[i];
      v[i + sizeof(T) / 2] = reinterpret_cast<const uint4*>(b)[i];
    }
  }
  __device__ __forceinline__ void store(T* a, T* b) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
      reinterpret_cast<uint4*>(a)[i] = v[i];
      reinterpret_cast<uint4*>(b)[i] = v[i + sizeof(T) / 2];
    }
  }
  __device__ __forceinline__ float at(int i) const {      // i: 0 .. 15
    if constexpr (sizeof(T) == 2) {
      const unsigned w = reinterpret_cast<const unsigned*>(v)[i >> 1];
      return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
    } else {
      return __uint_as_float(reinterpret_cast<const unsigned*>(v)[i]);
    }
  }
  __device__ __forceinline__ void set(int i, float x, float y) {      // channels i (even), i + 1
    if constexpr (sizeof(T) == 2) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
      reinterpret_cast<unsigned*>(v)[i >> 1] = *reinterpret_cast<const unsigned*>(&h);
    } else {
      reinterpret_cast<unsigned*>(v)[i] = __float_as_uint(x);
      reinterpret_cast<unsigned*>(v)[i + 1] = __float_as_uint(y);
    }
  }
};

// Pairs of 32-bit numbers in one register pair: one instruction for two multiply-adds, each rounded as by itself.
__device__ __forceinline__ unsigned long long qn_two(float a, float b) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ void qn_halves(unsigned long long v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ unsigned long long qn_fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long qn_mul2(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// LANES: lanes a head (a power of two, 16 channels each; those past the head's channels idle).  NEAR: neighbours turn into one another.
// A lane's 16 channels are 8 pairs (u, v) that turn: u' = r (u w_u c - v w_v s), v' = r (v w_v c + u w_u s), r the norm's factor; the products
// of weights with cosines and sines are the same for all heads of a token (queries, then keys).
template <typename T, int LANES, bool NEAR>
__global__ void __launch_bounds__(QN_WARPS * 32, 3)
qk_norm_rotary_kernel(QnParams p) {
  __shared__ float2 s_turn[QN_WARPS][128];
  pdl_trigger();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long job = (long long)blockIdx.x * QN_WARPS + warp;
  const int token = (int)(job / p.warps_per_token), part = (int)(job % p.warps_per_token);
  if (token >= p.n_tokens) return;
  const int pos = p.positions[token];
  // this lane's two pieces of 8 channels: pieces that turn into one another, or (past the turned ones, and for neighbours) in a row
  const int c = lane % LANES, sub = lane / LANES, pairs = NEAR ? 0 : p.rot / 16;
  const bool mine = 16 * c < p.dim, turned = 16 * c < p.rot;
  const int a = c < pairs ? 8 * c : 16 * c, b = c < pairs ? 8 * (c + pairs) : 16 * c + 8;
  const int first = part * p.vecs_per_warp, last = min(p.n_vecs, first + p.vecs_per_warp);
  const T* src = reinterpret_cast<const T*>(p.src) + token * p.src_row;
  T* dst = reinterpret_cast<T*>(p.dst) + token * p.dst_row;
  // the next heads are asked for before the ones at hand are worked on (the first before the angles)
  QnRaw<T> next;
  auto fetch = [&](int v) {
    if (mine && v < last) next.load(src + v * p.dim + a, src + v * p.dim + b);
  };
  fetch(first + sub);
  float2* turn = s_turn[warp];
  for (int i = lane; i < p.rot / 2; i += 32) turn[i] = qn_turn(pos, p.freq[i], p.size);
  __syncwarp();
  // w_u c, -w_v s, w_v c, w_u s of two pairs each
  unsigned long long uc[4], vs[4], vc[4], us[4];
  auto weigh = [&](const float* weight) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      float f[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int i = j + e, u = NEAR ? 16 * c + 2 * i : a + i, v = NEAR ? 16 * c + 2 * i + 1 : b + i;
        const float2 w = turned ? turn[8 * c + i] : make_float2(1.f, 0.f);
        const float wu = p.normed ? weight[u] : 1.f, wv = p.normed ? weight[v] : 1.f;
        f[e][0] = wu * w.x;
        f[e][1] = -wv * w.y;
        f[e][2] = wv * w.x;
        f[e][3] = wu * w.y;
      }
      uc[j / 2] = qn_two(f[0][0], f[1][0]);
      vs[j / 2] = qn_two(f[0][1], f[1][1]);
      vc[j / 2] = qn_two(f[0][2], f[1][2]);
      us[j / 2] = qn_two(f[0][3], f[1][3]);
    }
  };
  const float per_channel = 1.f / (float)p.dim;
  int kind = -1;                       // whose weights those are
  for (int v0 = first; v0 < last; v0 += 32 / LANES) {
    const int v = v0 + sub;
    const bool here = mine && v < last;
    const QnRaw<T> at = next;
    fetch(v + 32 / LANES);
    unsigned long long u2[4], v2[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u2[j] = NEAR ? qn_two(at.at(4 * j), at.at(4 * j + 2)) : qn_two(at.at(2 * j), at.at(2 * j + 1));
      v2[j] = NEAR ? qn_two(at.at(4 * j + 1), at.at(4 * j + 3)) : qn_two(at.at(8 + 2 * j), at.at(8 + 2 * j + 1));
    }
    float r = 1.f;
    if (p.normed) {
      unsigned long long sum2 = 0ull;
#pragma unroll
      for (int j = 0; j < 4; ++j) sum2 = qn_fma2(u2[j], u2[j], qn_fma2(v2[j], v2[j], sum2));
      float x, y;
      qn_halves(sum2, x, y);
      float sum = here ? x + y : 0.f;
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      r = rsqrtf(fmaf(sum, per_channel, p.eps));
    }
    if (!here) continue;
    if (kind != (v >= p.n_heads)) {
      kind = v >= p.n_heads;
      weigh(kind ? p.k_weight : p.q_weight);
    }
    const unsigned long long r2 = qn_two(r, r);
    QnRaw<T> done;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      unsigned long long u = qn_mul2(u2[j], uc[j]), w = qn_mul2(v2[j], vc[j]);
      if (turned) {                    // (elsewhere an infinity beside a zero would become NaN)
        u = qn_fma2(v2[j], vs[j], u);
        w = qn_fma2(u2[j], us[j], w);
      }
      float x0, x1, y0, y1;
      qn_halves(qn_mul2(u, r2), x0, x1);
      qn_halves(qn_mul2(w, r2), y0, y1);
      if (NEAR) {
        done.set(4 * j, x0, y0);
        done.set(4 * j + 2, x1, y1);
      } else {
        done.set(2 * j, x0, x1);
        done.set(8 + 2 * j, y0, y1);
      }
    }
    done.store(dst + v * p.dim + a, dst + v * p.dim + b);
  }
}

// Any head size up to 256, any even `rot`, any alignment: a warp a (token, head), a lane a pair or a channel at a time.
template <typename T>
__global__ void __launch_bounds__(QN_WARPS * 32)
qk_norm_rotary_any_kernel(QnParams p) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long job = (long long)blockIdx.x * QN_WARPS + (threadIdx.x >> 5);
  const int token = (int)(job / p.n_vecs), v = (int)(job % p.n_vecs);
  if (token >= p.n_tokens) return;
  const int pos = p.positions[token], half = p.rot / 2, slots = half + p.dim - p.rot;
  const T* src = reinterpret_cast<const T*>(p.src) + token * p.src_row + (long long)v * p.dim;
  T* dst = reinterpret_cast<T*>(p.dst) + token * p.dst_row + (long long)v * p.dim;
  const float* weight = v < p.n_heads ? p.q_weight : p.k_weight;
  float x[8], y[8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int s = lane + 32 * i;
    x[i] = y[i] = 0.f;
    if (s < half) {
      x[i] = to_float(src[p.interleaved ? 2 * s : s]);
      y[i] = to_float(src[p.interleaved ? 2 * s + 1 : s + half]);
    } else if (s < slots) {
      x[i] = to_float(src[half + s]);
    }
    sum = fmaf(x[i], x[i], fmaf(y[i], y[i], sum));
  }
  const float r = p.normed ? rsqrtf(warp_sum(sum) / (float)p.dim + p.eps) : 1.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int s = lane + 32 * i;
    if (s < half) {
      const int a = p.interleaved ? 2 * s : s, b = p.interleaved ? 2 * s + 1 : s + half;
      const float2 w = qn_turn(pos, p.freq[s], p.size);
      const float u = p.normed ? x[i] * (r * weight[a]) : x[i], z = p.normed ? y[i] * (r * weight[b]) : y[i];
      dst[a] = from_float<T>(u * w.x - z * w.y);
      dst[b] = from_float<T>(z * w.x + u * w.y);
    } else if (s < slots) {
      dst[half + s] = from_float<T>(p.normed ? x[i] * (r * weight[half + s]) : x[i]);
    }
  }
}

template <typename T>
static int launch_qn(QnParams p, bool whole, cudaStream_t stream) {
  if (whole) {
    const int lanes = p.dim <= 16 ? 1 : p.dim <= 32 ? 2 : p.dim <= 64 ? 4 : p.dim <= 128 ? 8 : 16;
    const int side = 32 / lanes, rounds = (p.n_vecs + side - 1) / side;
    // rounds a warp: as many as leave no more warps than run at once (three blocks a multiprocessor)
    long long split = 3ll * QN_WARPS * (sm_count() > 0 ? sm_count() : 148) / p.n_tokens;
    if (split < 1) split = 1;
    if (split > rounds) split = rounds;
    const int per = (int)((rounds + split - 1) / split);
    p.vecs_per_warp = per * side;
    p.warps_per_token = (rounds + per - 1) / per;
    const long long blocks = ((long long)p.n_tokens * p.warps_per_token + QN_WARPS - 1) / QN_WARPS;
    BT_CHECK(blocks < (1ll << 31), "qk_norm_rotary: %d tokens of %d heads are too many for one launch", p.n_tokens, p.n_vecs);
    const dim3 grid((unsigned)blocks), block(QN_WARPS * 32);
#define BT_QN(LANES)                                                                                                                  \
  if (p.interleaved)                                                                                                                  \
    BT_PDL_OK("qk_norm_rotary", launch_pdl(qk_norm_rotary_kernel<T, LANES, true>, grid, block, 0, stream, 1, p));                     \
  else                                                                                                                                \
    BT_PDL_OK("qk_norm_rotary", launch_pdl(qk_norm_rotary_kernel<T, LANES, false>, grid, block, 0, stream, 1, p));                    \
  break
    switch (lanes) {
      case 1: BT_QN(1);
      case 2: BT_QN(2);
      case 4: BT_QN(4);
      case 8: BT_QN(8);
      default: BT_QN(16);
    }
#undef BT_QN
    return 0;
  }
  const long long blocks = ((long long)p.n_tokens * p.n_vecs + QN_WARPS - 1) / QN_WARPS;
  BT_CHECK(blocks < (1ll << 31), "qk_norm_rotary: %d tokens of %d heads are too many for one launch", p.n_tokens, p.n_vecs);
  BT_PDL_OK("qk_norm_rotary", launch_pdl(qk_norm_rotary_any_kernel<T>, dim3((unsigned)blocks), dim3(QN_WARPS * 32), 0, stream, 1, p));
  return 0;
}

}  // namespace bt

// src, dst (which may be the same): rows of n_heads query heads and n_kv_heads key heads of `dim` channels.  dtype: 0 32-bit, 1 bfloat16.
extern "C" int bt_qk_norm_rotary(const void* src, long long src_row, void* dst, long long dst_row, const int* positions, const float* freq,
                                 const float* q_weight, const float* k_weight, int n_tokens, int n_heads, int n_kv_heads, int dim, int rot,
                                 float eps, float size, int interleaved, int dtype, cudaStream_t stream) {
  using namespace bt;
  BT_CHECK(dim > 0 && dim <= 256 && rot >= 0 && rot <= dim && rot % 2 == 0, "qk_norm_rotary: %d turned channels of %d", rot, dim);
  BT_CHECK(n_tokens >= 0 && n_heads >= 0 && n_kv_heads >= 0 && n_heads + n_kv_heads > 0, "qk_norm_rotary: bad sizes tokens=%d heads=%d key heads=%d",
           n_tokens, n_heads, n_kv_heads);
  BT_CHECK((q_weight == nullptr) == (k_weight == nullptr), "qk_norm_rotary: give both weights or neither");
  BT_CHECK(dtype == kF32 || dtype == kBF16, "qk_norm_rotary: unknown element type %d", dtype);
  if (n_tokens == 0) return 0;
  QnParams p{src, dst, src_row, dst_row, positions, freq, q_weight, k_weight, n_tokens, n_heads, n_heads + n_kv_heads, dim, rot, 0, 0, eps,
             size, interleaved, q_weight != nullptr};
  const int step = dtype == kF32 ? 4 : 8;
  auto at16 = [](const void* x) { return (unsigned long long)x % 16 == 0; };
  const bool whole = dim % 16 == 0 && rot % 16 == 0 && src_row % step == 0 && dst_row % step == 0 && at16(src) && at16(dst) && at16(q_weight) &&
                     at16(k_weight);
  if (dtype == kF32) return launch_qn<float>(p, whole, stream);
  return launch_qn<__nv_bfloat16>(p, whole, stream);
}
