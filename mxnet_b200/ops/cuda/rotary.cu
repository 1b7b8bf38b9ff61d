// Rotary position embedding for sm_100a, forward and backward (the backward pass is the rotation by the negative angle).
//
//   pairs (a, b) of a head's first R channels, angle t = position * inv_freq[i]:
//     a' = scale (a cos t - b sin t),   b' = scale (b cos t + a sin t);   channels R.. pass through.
//   pairs are (i, i + R/2) in the half layout and (2 i, 2 i + 1) in the interleaved one.
//
// Bytes bound it: every element is read once and written once.  A block owns a few tokens: it computes their R/2 sines and
// cosines once into shared memory (the product and its reduction to a fraction of a turn in 64 bits, so that a position of
// 10^6 keeps its angle to 1e-10 turns; the sine itself in 32) and applies them to all heads with accesses of up to 16 bytes.
// 8 x 2048 x 20 heads of 128 bf16: 29 us, 5.8 TB/s of the 6.4 TB/s that a copy reaches; with the loads of the next unit under way
// during the arithmetic it took 36 us (registers cost more resident blocks than the overlap gains).
#include "common.cuh"

namespace mxb {

constexpr int kRotThreads = 256;
constexpr int kRotMaxTokens = 16;        // tokens of one block

struct RotaryParams {
  const void* x;
  void* y;                               // contiguous [B, T, H, D]
  const void* pos;
  const void* inv_freq;
  int64_t sb, st, sh;                    // element strides of x
  int64_t pos_sb, pos_st;                // element strides of the positions (batch stride 0: one row for all samples)
  int T, H, D, R;
  int tokens;                            // B * T
  int per_block;
  int units;                             // units of one head: rotated pairs of vectors, then copied vectors
  FastDiv div_t, div_hu, div_u;
  int pos_type;                          // 0 float, 1 double, 2 int32, 3 int64
  int freq64;
  float scale, sign;
};

template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

__device__ __forceinline__ double rot_position(const RotaryParams& p, int64_t i) {
  switch (p.pos_type) {
    case 0: return (double)static_cast<const float*>(p.pos)[i];
    case 1: return static_cast<const double*>(p.pos)[i];
    case 2: return (double)static_cast<const int*>(p.pos)[i];
    default: return (double)static_cast<const long long*>(p.pos)[i];
  }
}

template <typename T, int V, bool kInter>
__global__ void __launch_bounds__(kRotThreads)
rotary_kernel(const RotaryParams p) {
  extern __shared__ float2 table[];      // [per_block][R / 2]: (scale cos, scale sin)
  typedef Pack<T, V> P;
  const int half = p.R >> 1;
  const int tok0 = blockIdx.x * p.per_block;
  const int ntok = min(p.per_block, p.tokens - tok0);
  const int pairs = half / V;            // rotated units of one head
  const int total = ntok * p.H * p.units;
  for (int i = threadIdx.x; i < ntok * half; i += kRotThreads) {
    const int k = i / half, f = i - k * half;
    uint32_t b, t;
    fd_divmod((uint32_t)(tok0 + k), p.div_t, &b, &t);
    const double pos = rot_position(p, (int64_t)b * p.pos_sb + (int64_t)t * p.pos_st);
    const double w = p.freq64 ? static_cast<const double*>(p.inv_freq)[f] : (double)static_cast<const float*>(p.inv_freq)[f];
    double turns = pos * w * 0.15915494309189533577;      // 1 / (2 pi)
    turns -= rint(turns);
    float s, co;
    sincospif((float)(2.0 * turns), &s, &co);
    table[i] = make_float2(co * p.scale, s * p.scale * p.sign);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < total; i += kRotThreads) {
    // unit u of head h of the block's token k
    uint32_t k, rest, h, u, b, t;
    fd_divmod((uint32_t)i, p.div_hu, &k, &rest);
    fd_divmod(rest, p.div_u, &h, &u);
    fd_divmod((uint32_t)tok0 + k, p.div_t, &b, &t);
    const T* x = static_cast<const T*>(p.x) + (int64_t)b * p.sb + (int64_t)t * p.st + (int64_t)h * p.sh;
    T* y = static_cast<T*>(p.y) + ((int64_t)(tok0 + (int)k) * p.H + h) * p.D;
    if ((int)u >= pairs) {
      const int ic = p.R + ((int)u - pairs) * V;
      *reinterpret_cast<P*>(y + ic) = *reinterpret_cast<const P*>(x + ic);
      continue;
    }
    const int ia = kInter ? (int)u * 2 * V : (int)u * V, ib = kInter ? ia + V : ia + half;
    const P a0 = *reinterpret_cast<const P*>(x + ia), c0 = *reinterpret_cast<const P*>(x + ib);
    const float2* tab = table + k * half + u * V;
    P oa, ob;
    if (kInter) {
      float in[2 * V], out[2 * V];
#pragma unroll
      for (int j = 0; j < V; ++j) { in[j] = Cvt<T>::to_f(a0.v[j]); in[V + j] = Cvt<T>::to_f(c0.v[j]); }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 cs = tab[j];
        out[2 * j] = in[2 * j] * cs.x - in[2 * j + 1] * cs.y;
        out[2 * j + 1] = in[2 * j + 1] * cs.x + in[2 * j] * cs.y;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) { oa.v[j] = Cvt<T>::from_f(out[j]); ob.v[j] = Cvt<T>::from_f(out[V + j]); }
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 cs = tab[j];
        const float fa = Cvt<T>::to_f(a0.v[j]), fb = Cvt<T>::to_f(c0.v[j]);
        oa.v[j] = Cvt<T>::from_f(fa * cs.x - fb * cs.y);
        ob.v[j] = Cvt<T>::from_f(fb * cs.x + fa * cs.y);
      }
    }
    *reinterpret_cast<P*>(y + ia) = oa;
    *reinterpret_cast<P*>(y + ib) = ob;
  }
}

template <typename T, int V>
static void rotary_launch(const RotaryParams& p, int interleaved, int grid, size_t smem, cudaStream_t st) {
  if (interleaved) rotary_kernel<T, V, true><<<grid, kRotThreads, smem, st>>>(p);
  else rotary_kernel<T, V, false><<<grid, kRotThreads, smem, st>>>(p);
}

}  // namespace mxb

using namespace mxb;

// x: [B, T, H, D] with element strides (sb, st, sh, 1); y contiguous; pos: [B, T] or one row for all samples (pos_sb = 0);
// inv_freq: [R / 2].  backward != 0 rotates by the negative angle.
MXB_EXPORT int mxb_rotary(int dtype, const void* x, void* y, const void* pos, const void* inv_freq, int64_t B, int T, int H, int D,
                          int R, int64_t sb, int64_t st, int64_t sh, int64_t pos_sb, int64_t pos_st, int pos_type, int freq64,
                          int interleaved, float scale, int backward, void* stream) {
  if (dtype < kF32 || dtype > kBF16 || pos_type < 0 || pos_type > 3) return -1;
  if (B < 1 || T < 1 || H < 1 || D < 1 || D > 1024 || R < 0 || R > D || (R & 1) || H > 4096) return -2;
  if (B * (int64_t)T > 0x3fffffff) return -2;
  RotaryParams p{};
  p.x = x; p.y = y; p.pos = pos; p.inv_freq = inv_freq;
  p.sb = sb; p.st = st; p.sh = sh; p.pos_sb = pos_sb; p.pos_st = pos_st;
  p.T = T; p.H = H; p.D = D; p.R = R; p.tokens = (int)(B * T);
  p.pos_type = pos_type; p.freq64 = freq64; p.scale = scale; p.sign = backward ? -1.f : 1.f;
  const int size = dtype == kF32 ? 4 : 2, vec = 16 / size;
  // the widest unit whose vectors are whole and aligned: head size, rotated half, strides and base addresses are multiples of it
  // (16 x 1024 x 20 heads of 96, 24 rotated, bf16: single elements 112 us, vectors of 4 25 us)
  int V = vec;
  auto fits = [&](int v) {
    const int64_t bytes = (int64_t)v * size;
    return D % v == 0 && (R / 2) % v == 0 && (sb * size) % bytes == 0 && (st * size) % bytes == 0 && (sh * size) % bytes == 0 &&
           (uintptr_t)x % bytes == 0 && (uintptr_t)y % bytes == 0;
  };
  while (V > 1 && !fits(V)) V >>= 1;
  p.units = (R / 2 + (D - R)) / V;
  if (p.units < 1) return -2;
  // one unit for each thread; four where that still leaves every SM four blocks (the table is made once for more of them)
  auto tokens_of = [&](int threads) {
    const int n = threads / (H * p.units);
    return n < 1 ? 1 : (n > kRotMaxTokens ? kRotMaxTokens : n);
  };
  int per = tokens_of(4 * kRotThreads);
  if (p.tokens / per < 4 * sm_count()) per = tokens_of(kRotThreads);
  if (R && per > 8192 / R) per = 8192 / R;               // the table stays within 32 KB (R <= 1024: at least 8 tokens)
  p.per_block = per;
  p.div_t = make_fastdiv((uint32_t)T);
  p.div_hu = make_fastdiv((uint32_t)(H * p.units));
  p.div_u = make_fastdiv((uint32_t)p.units);
  const int grid = (p.tokens + per - 1) / per;
  const size_t smem = (size_t)per * (R / 2) * sizeof(float2);
  cudaStream_t s = (cudaStream_t)stream;
  auto half_types = [&](auto zero) {
    typedef decltype(zero) T;
    if (V == 8) rotary_launch<T, 8>(p, interleaved, grid, smem, s);
    else if (V == 4) rotary_launch<T, 4>(p, interleaved, grid, smem, s);
    else if (V == 2) rotary_launch<T, 2>(p, interleaved, grid, smem, s);
    else rotary_launch<T, 1>(p, interleaved, grid, smem, s);
  };
  if (dtype == kF16) half_types(__half());
  else if (dtype == kBF16) half_types(__nv_bfloat16());
  else if (V == 4) rotary_launch<float, 4>(p, interleaved, grid, smem, s);
  else if (V == 2) rotary_launch<float, 2>(p, interleaved, grid, smem, s);
  else rotary_launch<float, 1>(p, interleaved, grid, smem, s);
  return (int)cudaGetLastError();
}
