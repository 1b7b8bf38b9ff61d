// Log probabilities of given tokens, the entropy of each row and its k most probable tokens, forward and backward.
//
//   m = max x, e_i = exp(x_i - m), total = 1 + r with r the sum over all but one largest element:
//     log p_i = (x_i - m) - log1p(r),   entropy = log1p(r) + w / (1 + r),  w = sum e_i (m - x_i)
//   Every term of r and w is >= 0, so a token that is almost certain keeps the digits of its log probability, and the
//   entropy of a sharp row those of its entropy.
//   backward: with h = dL/dentropy and G = dL/dlogp_token + sum of the alternatives' gradients,
//     dx_i = -p_i (G + h (log p_i + entropy)) + [i = token] dL/dlogp_token + [i = alternative j] dL/dtop_j.
//
// The forward pass reads the logits once and keeps (m, r, w) for each thread, rescaled when the thread's maximum moves.
// Alternatives: the k-th largest of the threads' maxima is a lower bound of the k-th largest element, so only the elements
// of threads whose maximum reaches it (k of them, more with ties) are read a second time, out of cache; a warp keeps its 32
// best as one sorted entry for each lane.  Equal logits rank by the lower index.
#include "common.cuh"

namespace mxb {

constexpr int kLpMaxTop = 32;

struct RowStat { float m, r, w; };       // m = -inf: nothing yet (total 0)

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ RowStat rs_merge(const RowStat& a, const RowStat& b) {
  const bool a_hi = a.m >= b.m;
  const RowStat hi = a_hi ? a : b, lo = a_hi ? b : a;
  if (!(lo.m > -INFINITY)) return {hi.m, hi.r + (lo.r != lo.r ? lo.r : 0.f), hi.w};   // an empty side only passes a NaN on
  const float d = hi.m - lo.m, f = exp2f(-d * kLog2e);
  // f = 0 (a gap beyond the range of exp, such as to a mask of the type's lowest value): d times the total may overflow
  return {hi.m, hi.r + (1.f + lo.r) * f, f > 0.f ? hi.w + f * (lo.w + d * (1.f + lo.r)) : hi.w + 0.f * lo.r};
}

template <int N>
__device__ __forceinline__ void rs_add(RowStat& s, const float (&x)[N]) {
  float cm = x[0];
#pragma unroll
  for (int j = 1; j < N; ++j) cm = fmaxf(cm, x[j]);
  if (cm <= s.m && s.m > -INFINITY) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = s.m - x[j], e = exp2f(-d * kLog2e);
      s.r += e;
      s.w += e > 0.f ? e * d : e;                         // e = 0 covers x = -inf, where e d would be 0 * inf; a NaN stays one
    }
    return;
  }
  if (cm > s.m) {
    if (s.m > -INFINITY) {
      const float d = cm - s.m, f = exp2f(-d * kLog2e), t = 1.f + s.r;
      s.w = f * (s.w + d * t);
      s.r = t * f;
      if (!(f > 0.f)) s.w = f;
    }
    s.m = cm;
    bool one = true;                                      // one element of the maximum is the 1 of the total
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (one && x[j] == cm) { one = false; continue; }
      const float d = cm - x[j], e = exp2f(-d * kLog2e);
      s.r += e;
      s.w += e > 0.f ? e * d : e;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < N; ++j) if (x[j] != x[j]) s.r = x[j];   // nothing but NaN (and -inf) so far
}

// Values in the order of their bits as unsigned numbers; a NaN ranks first.
__device__ __forceinline__ uint32_t lp_order(float v) {
  if (v != v) return 0xffffffffu;
  const uint32_t b = __float_as_uint(v == 0.f ? 0.f : v);     // -0 ties with 0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ uint64_t lp_key(float v, uint32_t index) { return ((uint64_t)lp_order(v) << 32) | (uint32_t)~index; }
__device__ __forceinline__ float lp_value(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  if (u == 0xffffffffu) return NAN;
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// Row of `cols` elements as scalars up to the first 16-byte boundary, vectors, and scalars behind the last one.
template <typename T> struct RowCut {
  static constexpr int V = 16 / sizeof(T);
  int head, vecs, tail0, loose;          // loose = scalars in all: [0, head) and [tail0, cols)
  __device__ __forceinline__ RowCut(const T* x, int cols) {
    head = (int)(((16u - (uint32_t)((uintptr_t)x & 15u)) & 15u) / sizeof(T));
    if (head > cols) head = cols;
    vecs = (cols - head) / V;
    tail0 = head + vecs * V;
    loose = head + (cols - tail0);
  }
  __device__ __forceinline__ int loose_index(int i) const { return i < head ? i : tail0 + (i - head); }
};

// Keeps the 32 largest keys of a warp, one per lane in descending order; `key` is each lane's candidate (0 = none).
__device__ __forceinline__ void warp_insert(uint64_t& list, uint64_t key, int k) {
  const int lane = threadIdx.x & 31;
  while (true) {
    const uint64_t last = __shfl_sync(0xffffffffu, list, k - 1);
    const uint32_t want = __ballot_sync(0xffffffffu, key > last);
    if (!want) return;
    const int src = __ffs(want) - 1;
    const uint64_t c = __shfl_sync(0xffffffffu, key, src);
    const int at = __popc(__ballot_sync(0xffffffffu, list > c));
    const uint64_t up = __shfl_up_sync(0xffffffffu, list, 1);
    if (lane == at) list = c;
    else if (lane > at) list = up;
    if (lane == src) key = 0;
  }
}
// The 32 largest of two descending lists (one entry per lane), descending.
template <typename K>
__device__ __forceinline__ K warp_merge_desc(K a, K b) {
  const int lane = threadIdx.x & 31;
  const K r = __shfl_sync(0xffffffffu, b, 31 - lane);
  a = a > r ? a : r;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const K other = __shfl_xor_sync(0xffffffffu, a, o);
    const bool keep_big = (lane & o) == 0;
    a = ((a > other) == keep_big) ? a : other;
  }
  return a;
}
template <typename K>
__device__ __forceinline__ K warp_sort_desc(K v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int o = size >> 1; o > 0; o >>= 1) {
      const K other = __shfl_xor_sync(0xffffffffu, v, o);
      const bool desc = (lane & size) == 0 || size == 32;
      const bool keep_big = ((lane & o) == 0) == desc;
      v = ((v > other) == keep_big) ? v : other;
    }
  }
  return v;
}

struct LogProbParams {
  const void* x;
  const int64_t* tokens;
  float* log_prob;
  float* entropy;
  float* top_lp;           // [rows, k] or null
  int64_t* top_id;
  float* stat;             // [rows, 3]: m, log1p(r) and the entropy, read by the backward pass (or null)
  int64_t rows;
  int cols, k;
  int64_t ignore;
};

template <typename T>
__global__ void __launch_bounds__(512)
logprob_fwd_kernel(const LogProbParams p) {
  constexpr int V = 16 / sizeof(T);
  __shared__ RowStat red[32];
  __shared__ uint32_t best32[32][32];
  __shared__ uint64_t best64[32][32];
  __shared__ uint16_t winners[1024];
  __shared__ int nwin;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nw = blockDim.x >> 5;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.cols;
    const RowCut<T> cut(x, p.cols);
    const T* body = x + cut.head;
    RowStat s{-INFINITY, 0.f, 0.f};
    if (tid < cut.loose) {
      const float v[1] = {Cvt<T>::to_f(x[cut.loose_index(tid)])};
      rs_add(s, v);
    }
    for (int i = tid; i < cut.vecs; i += blockDim.x) {
      const Vec16<T> a = ld16(body + (int64_t)i * V);
      float v[V];
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = Cvt<T>::to_f(a.v[j]);
      rs_add(s, v);
    }
    RowStat all = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const RowStat b{__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.r, o), __shfl_xor_sync(0xffffffffu, all.w, o)};
      all = rs_merge(all, b);
    }
    if (lane == 0) red[warp] = all;
    uint32_t mine = 0;
    if (p.k) {
      mine = warp_sort_desc(lp_order(s.m));
      best32[warp][lane] = mine;
    }
    if (tid == 0) nwin = 0;
    __syncthreads();
    all = lane < nw ? red[lane] : RowStat{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const RowStat b{__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.r, o), __shfl_xor_sync(0xffffffffu, all.w, o)};
      all = rs_merge(all, b);
    }
    const bool empty = all.m == -INFINITY && all.r == all.r;      // nothing is possible: every log probability is -inf
    if (all.m == INFINITY) all.r = NAN;
    const float lt = log1pf(all.r);
    if (tid == 0) {
      const int64_t t = p.tokens[row];
      float lp;
      if (t == p.ignore) lp = 0.f;
      else if (t < 0 || t >= p.cols) lp = NAN;                    // no such token
      else lp = empty ? -INFINITY : (Cvt<T>::to_f(x[t]) - all.m) - lt;
      p.log_prob[row] = lp;
      const float ent = empty ? 0.f : lt + all.w / (1.f + all.r);
      p.entropy[row] = ent;
      if (p.stat) { p.stat[3 * row] = all.m; p.stat[3 * row + 1] = lt; p.stat[3 * row + 2] = ent; }
    }
    if (p.k) {
      for (int half = 1; half < nw; half <<= 1) {
        if ((warp & (2 * half - 1)) == 0 && warp + half < nw) {
          mine = warp_merge_desc(mine, best32[warp + half][lane]);
          best32[warp][lane] = mine;
        }
        __syncthreads();
      }
      uint32_t bound = best32[0][p.k - 1];
      if (all.r != all.r) bound = 0;                              // a NaN somewhere: look at everything
      if (lp_order(s.m) >= bound) winners[atomicAdd(&nwin, 1)] = (uint16_t)tid;
      __syncthreads();
      uint64_t list = 0;
      const int n = nwin;
      for (int wi = warp; wi < n; wi += nw) {
        const int who = winners[wi];
        {
          uint64_t key = 0;
          if (lane == 0 && who < cut.loose) {
            const int c = cut.loose_index(who);
            const float v = Cvt<T>::to_f(x[c]);
            if (lp_order(v) >= bound) key = lp_key(v, (uint32_t)c);
          }
          warp_insert(list, key, p.k);
        }
        const int rounds = (cut.vecs - who + (int)blockDim.x - 1) / (int)blockDim.x;    // vectors of that thread
        for (int r0 = 0; r0 < rounds; r0 += 32) {
          const int i = who + (r0 + lane) * (int)blockDim.x;
          const bool in = r0 + lane < rounds;
          Vec16<T> a;
          if (in) a = ld16(body + (int64_t)i * V);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            uint64_t key = 0;
            if (in) {
              const float v = Cvt<T>::to_f(a.v[j]);
              if (lp_order(v) >= bound) key = lp_key(v, (uint32_t)(cut.head + i * V + j));
            }
            warp_insert(list, key, p.k);
          }
        }
      }
      best64[warp][lane] = list;
      __syncthreads();
      for (int half = 1; half < nw; half <<= 1) {
        if ((warp & (2 * half - 1)) == 0 && warp + half < nw) {
          list = warp_merge_desc(list, best64[warp + half][lane]);
          best64[warp][lane] = list;
        }
        __syncthreads();
      }
      if (warp == 0 && lane < p.k) {
        const float v = lp_value(list);
        p.top_lp[row * p.k + lane] = empty ? -INFINITY : (v - all.m) - lt;
        p.top_id[row * p.k + lane] = (int64_t)(uint32_t)~(uint32_t)list;
      }
    }
    __syncthreads();                                              // the shared lists belong to the next row now
  }
}

struct LogProbGradParams {
  const void* x;
  void* dx;
  const int64_t* tokens;
  const float* stat;
  const float* g_lp;       // each may be null
  const float* g_ent;
  const float* g_top;
  const int64_t* top_id;
  int64_t rows;
  int cols, k;
  int64_t ignore;
};

template <typename T>
__global__ void __launch_bounds__(512)
logprob_bwd_kernel(const LogProbGradParams p) {
  constexpr int V = 16 / sizeof(T);
  const int tid = threadIdx.x;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.cols;
    T* dx = static_cast<T*>(p.dx) + row * p.cols;
    const float m = p.stat[3 * row], lt = p.stat[3 * row + 1], ent = p.stat[3 * row + 2];
    const int64_t t = p.tokens[row];
    float gl = p.g_lp ? p.g_lp[row] : 0.f;
    if (t == p.ignore) gl = 0.f;
    else if (t < 0 || t >= p.cols) gl = NAN;
    const float h = p.g_ent ? p.g_ent[row] : 0.f;
    float G = gl;
    if (p.g_top) for (int j = 0; j < p.k; ++j) G += p.g_top[row * p.k + j];
    const bool empty = m == -INFINITY && lt == lt;
    auto grad = [&](float v, int c) {
      const float lp = (v - m) - lt;
      const float pr = exp2f(lp * kLog2e);
      float g = pr > 0.f || pr != pr ? -pr * (G + h * (lp + ent)) : 0.f;
      if (empty) g = 0.f;
      return g;
    };
    const RowCut<T> cut(x, p.cols);
    const bool wide = (((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0;
    if (wide) {
      if (tid < cut.loose) {
        const int c = cut.loose_index(tid);
        dx[c] = Cvt<T>::from_f(grad(Cvt<T>::to_f(x[c]), c));
      }
      for (int i = tid; i < cut.vecs; i += blockDim.x) {
        const Vec16<T> a = ld16(x + cut.head + (int64_t)i * V);
        Vec16<T> o;
#pragma unroll
        for (int j = 0; j < V; ++j) o.v[j] = Cvt<T>::from_f(grad(Cvt<T>::to_f(a.v[j]), 0));
        st16(dx + cut.head + (int64_t)i * V, o);
      }
    } else {
      for (int c = tid; c < p.cols; c += blockDim.x) dx[c] = Cvt<T>::from_f(grad(Cvt<T>::to_f(x[c]), c));
    }
    __syncthreads();
    // the few elements with a gradient of their own are rewritten whole, so that each is rounded once
    if (!empty) {
      for (int j = tid; j < 1 + (p.g_top ? p.k : 0); j += blockDim.x) {
        const int64_t c = j == 0 ? t : p.top_id[row * p.k + j - 1];
        if (c < 0 || c >= p.cols) continue;
        float own = 0.f;
        if (c == t && t != p.ignore) own += gl;
        if (p.g_top) for (int q = 0; q < p.k; ++q) if (p.top_id[row * p.k + q] == c) own += p.g_top[row * p.k + q];
        dx[c] = Cvt<T>::from_f(grad(Cvt<T>::to_f(x[c]), (int)c) + own);
      }
    }
  }
}

inline int lp_threads(int cols, int size) {
  const int64_t want = ((int64_t)cols * size + 63) / 64;          // four 16-byte vectors of each thread, while the block grows
  int t = 32;
  while (t < 512 && t < want) t <<= 1;
  return t;
}

}  // namespace mxb

using namespace mxb;

// x: [rows, cols]; tokens: [rows]; top_lp / top_id: [rows, k] (k may be 0); stat: [rows, 3] floats for the backward pass.
MXB_EXPORT int mxb_logprob_forward(int dtype, const void* x, const int64_t* tokens, float* log_prob, float* entropy, float* top_lp,
                                   int64_t* top_id, float* stat, int64_t rows, int cols, int k, int64_t ignore, void* stream) {
  if (rows < 1 || cols < 1 || k < 0 || k > kLpMaxTop || k > cols) return -2;
  LogProbParams p{x, tokens, log_prob, entropy, top_lp, top_id, stat, rows, cols, k, ignore};
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t cap = (int64_t)sm_count() * 64;
  const unsigned grid = (unsigned)(rows < cap ? rows : cap);
  if (dtype == kF32) logprob_fwd_kernel<float><<<grid, lp_threads(cols, 4), 0, st>>>(p);
  else if (dtype == kF16) logprob_fwd_kernel<__half><<<grid, lp_threads(cols, 2), 0, st>>>(p);
  else if (dtype == kBF16) logprob_fwd_kernel<__nv_bfloat16><<<grid, lp_threads(cols, 2), 0, st>>>(p);
  else return -1;
  return (int)cudaGetLastError();
}

// dx: [rows, cols] of the logits' type; g_lp, g_ent: [rows] floats, g_top: [rows, k] floats (each may be null).
MXB_EXPORT int mxb_logprob_backward(int dtype, const void* x, void* dx, const int64_t* tokens, const float* stat,
                                    const float* g_lp, const float* g_ent, const float* g_top, const int64_t* top_id, int64_t rows,
                                    int cols, int k, int64_t ignore, void* stream) {
  if (rows < 1 || cols < 1 || k < 0 || k > kLpMaxTop || k > cols) return -2;
  LogProbGradParams p{x, dx, tokens, stat, g_lp, g_ent, g_top, top_id, rows, cols, k, ignore};
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t cap = (int64_t)sm_count() * 64;
  const unsigned grid = (unsigned)(rows < cap ? rows : cap);
  if (dtype == kF32) logprob_bwd_kernel<float><<<grid, lp_threads(cols, 4), 0, st>>>(p);
  else if (dtype == kF16) logprob_bwd_kernel<__half><<<grid, lp_threads(cols, 2), 0, st>>>(p);
  else if (dtype == kBF16) logprob_bwd_kernel<__nv_bfloat16><<<grid, lp_threads(cols, 2), 0, st>>>(p);
  else return -1;
  return (int)cudaGetLastError();
}
