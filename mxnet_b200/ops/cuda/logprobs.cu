// Log probabilities of given tokens, the entropy of each row and its k most probable tokens, forward and backward.
//
//   m = max x, e_i = exp(x_i - m), total = 1 + r with r the sum over all but one largest element:
//     log p_i = (x_i - m) - log1p(r),   entropy = log1p(r) + w / (1 + r),  w = sum e_i (m - x_i)
//   Every term of r and w is >= 0, so a token that is almost certain keeps the digits of its log probability, and the
//   entropy of a sharp row those of its entropy.
//   backward: with h = dL/dentropy and G = dL/dlogp_token + sum of the alternatives' gradients,
//     dx_i = -p_i (G + h (log p_i + entropy)) + [i = token] dL/dlogp_token + [i = alternative j] dL/dtop_j.
//
// The forward pass reads the logits once; each thread keeps (maximum, sum, weighted sum), moved to a new maximum at most once
// for 64 bytes.  The thread that holds the row's only largest element cannot tell a small rest from that element's 1: its
// few vectors are added up again without it by one warp, out of cache.
// Alternatives: the k-th largest of the threads' maxima is a lower bound of the k-th largest element, so only the elements
// of threads whose maximum reaches it (k of them, more with ties) are read a second time; a warp keeps its 32 best as one
// sorted entry for each lane.  Equal logits rank by the lower index.
// Few rows: a cluster of CTAs shares a row and joins over distributed shared memory.
//
// 4096 x 33278 bf16: forward 62 to 68 us for 273 MB (4.0 to 4.4 TB/s; bound by instructions: 70 % of the issue slots), backward 93 us for 545 MB (5.9 TB/s of the 6.4 a copy reaches).  24 x 131072 fp32 with
// 20 alternatives: 16 us for 12.6 MB, a chain of joins.
#include "common.cuh"

namespace mxb {

constexpr int kLpMaxTop = 32;

struct RowStat { float m, r, w; };       // m = -inf: nothing yet (total 0); otherwise the total is 1 + r

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ RowStat rs_merge(const RowStat& a, const RowStat& b) {
  const bool a_hi = a.m >= b.m;
  const RowStat hi = a_hi ? a : b, lo = a_hi ? b : a;
  if (!(lo.m > -INFINITY)) return hi;
  if (hi.m == INFINITY) return {hi.m, NAN, NAN};
  const float d = hi.m - lo.m, f = exp2f(-d * kLog2e);
  // f = 0 (a gap beyond the range of exp, such as to a mask of the type's lowest value): d times the total may overflow
  return {hi.m, hi.r + (1.f + lo.r) * f, f > 0.f ? hi.w + f * (lo.w + d * (1.f + lo.r)) : hi.w};
}

__device__ __forceinline__ float max_nan(float a, float b) {      // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// 16 bytes of logits as they lie in memory.
template <typename T> struct LpVec;
template <> struct LpVec<float> {
  static constexpr int pairs = 2;
  static __device__ __forceinline__ float top(const uint4& v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  static __device__ __forceinline__ void pair(const uint4& v, int i, float& a, float& b) {
    a = __uint_as_float(i ? v.z : v.x);
    b = __uint_as_float(i ? v.w : v.y);
  }
};
template <> struct LpVec<__half> {
  static constexpr int pairs = 4;
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    const uint32_t m = max2(max2(v.x, v.y), max2(v.z, v.w));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u); }
  static __device__ __forceinline__ void pair(const uint4& v, int i, float& a, float& b) {
    const uint32_t w = i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x;
    b = f.y;
  }
};
template <> struct LpVec<__nv_bfloat16> {
  static constexpr int pairs = 4;
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float top(const uint4& v) {
    const uint32_t m = max2(max2(v.x, v.y), max2(v.z, v.w));
    return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  static __device__ __forceinline__ uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  static __device__ __forceinline__ void pair(const uint4& v, int i, float& a, float& b) {
    const uint32_t w = i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w));
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  }
};

// A thread's share of a row: s = sum of exp(x - m), w = sum of exp(x - m) (x - m), m the largest element (a NaN stays).
constexpr float kFar = -1e4f;            // differences are cut here: exp is 0 there, and 0 * -inf does not arise
struct ThreadStat {
  float m = -INFINITY;
  f32x2 s = 0, w = 0;                    // two sums side by side
  __device__ __forceinline__ void move(float top) {
    const float mn = max_nan(m, top);
    if (mn != m) {
      const float d = fmaxf(m - mn, kFar), f = exp2f(d * kLog2e);
      const f32x2 ff = pack_f2(f, f);
      w = mul_f2(fma_f2(s, pack_f2(d, d), w), ff);
      s = mul_f2(s, ff);
      m = mn;
    }
  }
  // after move(): adds a pair of elements
  __device__ __forceinline__ void add(float a, float b, f32x2 neg_m) {
    float d0, d1, t0, t1;
    unpack_f2(add_f2(pack_f2(a, b), neg_m), d0, d1);
    const f32x2 d = pack_f2(fmaxf(d0, kFar), fmaxf(d1, kFar));
    unpack_f2(mul_f2(d, pack_f2(kLog2e, kLog2e)), t0, t1);
    const f32x2 e = pack_f2(exp2f(t0), exp2f(t1));
    s = add_f2(s, e);
    w = fma_f2(e, d, w);
  }
  __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
};

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
  int share;               // CTAs of a cluster that share a row
  int part;                // elements of each one's part
};

template <typename V> __device__ __forceinline__ V lp_remote(const V* local, uint32_t rank);
template <> __device__ __forceinline__ float lp_remote<float>(const float* local, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
template <> __device__ __forceinline__ uint64_t lp_remote<uint64_t>(const uint64_t* local, uint32_t rank) {
  uint32_t at;
  uint64_t v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void lp_cluster_sync() { asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory"); }

constexpr int kLpThreads = 512, kLpMaxShare = 8;
constexpr int kLpBatch = 4;              // vectors of a thread on their way at once

template <typename T>
__global__ void __launch_bounds__(kLpThreads, 2)
logprob_fwd_kernel(const LogProbParams p) {
  constexpr int V = 16 / sizeof(T);
  typedef LpVec<T> L;
  __shared__ float red_m[16], red_s[16], red_w[16];
  __shared__ int holders, holder;        // threads that hold the maximum, one of them
  __shared__ RowStat part_stat;
  __shared__ uint64_t best[16][32];      // lists of the warps; best[0]: of this CTA
  __shared__ uint16_t winners[kLpThreads];
  __shared__ int nwin;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, nth = blockDim.x, nw = nth >> 5;
  const int rank = blockIdx.x % p.share;
  const int64_t step = gridDim.x / p.share;
  for (int64_t row = blockIdx.x / p.share; row < p.rows; row += step) {
    const T* x = static_cast<const T*>(p.x) + row * p.cols;
    const int from = min(p.cols, rank * p.part), len = min(p.part, p.cols - from);
    const T* xp = x + from;
    const RowCut<T> cut(xp, len);
    const uint4* body = reinterpret_cast<const uint4*>(xp + cut.head);
    ThreadStat t;
    float loose = -INFINITY;
    if (tid < cut.loose) loose = Cvt<T>::to_f(xp[cut.loose_index(tid)]);
    t.move(loose);
    t.add(loose, -INFINITY, pack_f2(-t.base(), -t.base()));
    uint4 next[kLpBatch];                                         // on their way while the batch before is worked on
#pragma unroll
    for (int u = 0; u < kLpBatch; ++u) next[u] = tid + u * nth < cut.vecs ? body[tid + u * nth] : L::none();
    for (int i0 = tid; i0 < cut.vecs; i0 += nth * kLpBatch) {
      uint4 v[kLpBatch];
#pragma unroll
      for (int u = 0; u < kLpBatch; ++u) v[u] = next[u];
#pragma unroll
      for (int u = 0; u < kLpBatch; ++u) next[u] = i0 + (kLpBatch + u) * nth < cut.vecs ? body[i0 + (kLpBatch + u) * nth] : L::none();
      float top = L::top(v[0]);
#pragma unroll
      for (int u = 1; u < kLpBatch; ++u) top = max_nan(top, L::top(v[u]));
      t.move(top);
      const f32x2 neg = pack_f2(-t.base(), -t.base());
#pragma unroll
      for (int u = 0; u < kLpBatch; ++u) {
        if (i0 + u * nth >= cut.vecs) break;
#pragma unroll
        for (int j = 0; j < L::pairs; ++j) {
          float a, b;
          L::pair(v[u], j, a, b);
          t.add(a, b, neg);
        }
      }
    }
    // ---------------------------------------------------------------- the CTA's maximum
    float m = t.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red_m[warp] = m;
    uint32_t mine = 0;
    if (p.k) {
      mine = warp_sort_desc(lp_order(t.m));
      best[warp][lane] = mine;
    }
    if (tid == 0) { nwin = 0; holders = 0; }
    __syncthreads();
    m = red_m[lane < nw ? lane : 0];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    // ---------------------------------------------------------------- its sums; whose thread holds the maximum alone
    const bool holds = t.m == m;
    float s0, s1, w0, w1;
    unpack_f2(t.s, s0, s1);
    unpack_f2(t.w, w0, w1);
    float s = s0 + s1, w = w0 + w1;
    {
      const float d = m == -INFINITY ? 0.f : fmaxf(t.m - m, kFar), f = exp2f(d * kLog2e);
      w = f * (w + d * s);
      s *= f;
    }
    const float s_all = warp_sum(s), w_all = warp_sum(w);         // in w the largest element counts 0: it needs no second look
    if (lane == 0) { red_s[warp] = s_all; red_w[warp] = w_all; }
    if (holds) { atomicAdd(&holders, 1); holder = tid; }          // with several holders any of them will do: it is not used then
    __syncthreads();
    const int n = holders;
    float r = warp_sum(lane < nw ? red_s[lane] : 0.f);
    const float wr = warp_sum(lane < nw ? red_w[lane] : 0.f);
    const bool sure = n == 1 && r < 1.5f;                         // r - 1 has lost digits
    r -= 1.f;
    if (sure) {
      // the sums of all threads but the holder, and the holder's elements again without one of the largest value
      const float others = warp_sum(holds ? 0.f : s);
      __syncthreads();                                            // everyone has read red_s
      if (lane == 0) red_s[warp] = others;
      __syncthreads();
      if (warp == holder >> 5) {
        const int h = holder;
        float again = 0.f;
        bool spent = false;              // some lane before has left its element out
        auto rest = [&](float v, bool skip) {
          if (skip) return;
          again += exp2f(fmaxf(v - m, kFar) * kLog2e);
        };
        if (h < cut.loose) {
          const float v = Cvt<T>::to_f(xp[cut.loose_index(h)]);
          spent = v == m;
          rest(v, lane != 0 || spent);
        }
        const int rounds = (cut.vecs - h + nth - 1) / nth;
        for (int r0 = 0; r0 < rounds; r0 += 32) {
          const int i = h + (r0 + lane) * nth;
          uint4 v = L::none();
          if (r0 + lane < rounds) v = body[i];
          const uint32_t has = __ballot_sync(0xffffffffu, L::top(v) == m);
          bool skip = !spent && has && lane == __ffs(has) - 1;
          spent = spent || has;
#pragma unroll
          for (int j = 0; j < L::pairs; ++j) {
            float a, b;
            L::pair(v, j, a, b);
            const bool sa = skip && a == m;
            if (sa) skip = false;
            rest(a, sa);
            const bool sb = skip && b == m;
            if (sb) skip = false;
            rest(b, sb);
          }
        }
        again = warp_sum(again);
        if (lane == 0) red_s[warp] += again;
      }
      __syncthreads();
      r = warp_sum(lane < nw ? red_s[lane] : 0.f);
    }
    if (warp == 0) {
      RowStat st{m, r, -wr};
      if (m == -INFINITY) st = {-INFINITY, 0.f, 0.f};
      if (m != m || m == INFINITY) st = {INFINITY, NAN, NAN};
      if (lane == 0) part_stat = st;
    }
    // ---------------------------------------------------------------- the CTA's most probable elements
    if (p.k) {
      for (int half = 1; half < nw; half <<= 1) {
        if ((warp & (2 * half - 1)) == 0 && warp + half < nw) {
          mine = warp_merge_desc(mine, (uint32_t)best[warp + half][lane]);
          best[warp][lane] = mine;
        }
        __syncthreads();
      }
      uint32_t bound = (uint32_t)best[0][p.k - 1];
      if (m != m) bound = 0;                                      // a NaN somewhere: look at everything
      if (lp_order(t.m) >= bound || bound == 0) winners[atomicAdd(&nwin, 1)] = (uint16_t)tid;
      __syncthreads();
      uint64_t list = 0;
      const int nwinners = nwin;
      for (int wi = warp; wi < nwinners; wi += nw) {
        const int h = winners[wi];
        {
          uint64_t key = 0;
          if (lane == 0 && h < cut.loose) {
            const int c = cut.loose_index(h);
            const float v = Cvt<T>::to_f(xp[c]);
            if (lp_order(v) >= bound) key = lp_key(v, (uint32_t)(from + c));
          }
          warp_insert(list, key, p.k);
        }
        const int rounds = (cut.vecs - h + nth - 1) / nth;        // vectors of that thread
        for (int r0 = 0; r0 < rounds; r0 += 32) {
          const int i = h + (r0 + lane) * nth;
          const bool in = r0 + lane < rounds;
          uint4 v = L::none();
          if (in) v = body[i];
#pragma unroll
          for (int j = 0; j < L::pairs; ++j) {
            float a, b;
            L::pair(v, j, a, b);
            const uint32_t at = (uint32_t)(from + cut.head + i * V + 2 * j);
            warp_insert(list, in && lp_order(a) >= bound ? lp_key(a, at) : 0, p.k);
            warp_insert(list, in && lp_order(b) >= bound ? lp_key(b, at + 1) : 0, p.k);
          }
        }
      }
      __syncthreads();                                            // everyone has read the bound
      best[warp][lane] = list;
      __syncthreads();
      for (int half = 1; half < nw; half <<= 1) {
        if ((warp & (2 * half - 1)) == 0 && warp + half < nw) {
          list = warp_merge_desc(list, best[warp + half][lane]);
          best[warp][lane] = list;
        }
        __syncthreads();
      }
    }
    // ---------------------------------------------------------------- the row's results
    if (p.share > 1) lp_cluster_sync();
    else __syncthreads();
    if (rank == 0 && warp == 0) {
      // every remote word is asked for before the first is used: a trip to another CTA takes about a microsecond
      RowStat all = part_stat;
      uint64_t list = best[0][lane];
      if (p.share > 1) {
        uint64_t other[kLpMaxShare - 1];
        if (p.k) {
#pragma unroll
          for (int c = 1; c < kLpMaxShare; ++c) other[c - 1] = c < p.share ? lp_remote(&best[0][lane], c) : 0;
        }
        all = {-INFINITY, 0.f, 0.f};
        if (lane < p.share) all = {lp_remote(&part_stat.m, lane), lp_remote(&part_stat.r, lane), lp_remote(&part_stat.w, lane)};
#pragma unroll
        for (int o = 1; o < kLpMaxShare; o <<= 1)
          all = rs_merge(all, {__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.r, o), __shfl_xor_sync(0xffffffffu, all.w, o)});
        if (p.k) {
#pragma unroll
          for (int c = 1; c < kLpMaxShare; ++c) if (c < p.share) list = warp_merge_desc(list, other[c - 1]);
        }
      }
      all.m = __shfl_sync(0xffffffffu, all.m, 0);
      all.r = __shfl_sync(0xffffffffu, all.r, 0);
      all.w = __shfl_sync(0xffffffffu, all.w, 0);
      const bool empty = all.m == -INFINITY;                      // nothing is possible: every log probability is -inf
      const float lt = log1pf(all.r);
      if (lane == 0) {
        const int64_t tok = p.tokens[row];
        float lp;
        if (tok == p.ignore) lp = 0.f;
        else if (tok < 0 || tok >= p.cols) lp = NAN;              // no such token
        else lp = empty ? -INFINITY : (Cvt<T>::to_f(x[tok]) - all.m) - lt;
        p.log_prob[row] = lp;
        const float ent = empty ? 0.f : lt + all.w / (1.f + all.r);
        p.entropy[row] = ent;
        if (p.stat) { p.stat[3 * row] = all.m; p.stat[3 * row + 1] = lt; p.stat[3 * row + 2] = ent; }
      }
      if (lane < p.k) {
        const float v = lp_value(list);
        p.top_lp[row * p.k + lane] = empty ? -INFINITY : (v - all.m) - lt;
        p.top_id[row * p.k + lane] = (int64_t)(uint32_t)~(uint32_t)list;
      }
    }
    if (p.share > 1) lp_cluster_sync();                           // the shared lists belong to the next row now
    else __syncthreads();
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

constexpr int kLpGradThreads = 512, kLpGradBatch = 4;          // vectors of a thread on their way at once
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
    else if (t < 0 || t >= p.cols) gl = gl == 0.f ? 0.f : NAN;   // no such token: only a gradient that asks about it is NaN
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
      for (int i0 = tid; i0 < cut.vecs; i0 += blockDim.x * kLpGradBatch) {
        uint4 a[kLpGradBatch];
#pragma unroll
        for (int u = 0; u < kLpGradBatch; ++u)
          if (i0 + u * (int)blockDim.x < cut.vecs) a[u] = __ldcs(reinterpret_cast<const uint4*>(x + cut.head) + i0 + u * (int)blockDim.x);
#pragma unroll
        for (int u = 0; u < kLpGradBatch; ++u) {
          if (i0 + u * (int)blockDim.x >= cut.vecs) break;
          const Vec16<T>& in = *reinterpret_cast<const Vec16<T>*>(&a[u]);
          Vec16<T> o;
#pragma unroll
          for (int j = 0; j < V; ++j) o.v[j] = Cvt<T>::from_f(grad(Cvt<T>::to_f(in.v[j]), 0));
          __stcs(reinterpret_cast<uint4*>(dx + cut.head) + i0 + u * (int)blockDim.x, *reinterpret_cast<const uint4*>(&o));
        }
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

inline int lp_threads(int cols, int size, int most) {
  const int64_t want = ((int64_t)cols * size + 63) / 64;          // four 16-byte vectors of each thread, while the block grows
  int t = 32;
  while (t < most && t < want) t <<= 1;
  return t;
}

template <typename T>
static int logprob_forward(LogProbParams p, cudaStream_t st) {
  // Rows are shared while that fills no more than two CTAs on every SM and leaves each CTA 16 KB (a part with less has too little
  // to read for the joins it causes).
  p.share = 1;
  while (p.share < kLpMaxShare && p.rows * p.share * 2 <= 2 * sm_count() && (int64_t)p.cols * sizeof(T) / (p.share * 2) >= 16384) p.share <<= 1;
  p.part = p.share == 1 ? p.cols : ((p.cols + p.share - 1) / p.share + 63) / 64 * 64;
  const int64_t cap = (int64_t)sm_count() * 64;
  const int64_t rows = p.rows < cap ? p.rows : cap;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * p.share));
  // Blocks of 128 threads: their joins overlap with the reading of 7 others on the SM (4096 x 33278 bf16: 68 us, 256 threads 72,
  // 512 threads 101); 512 where blocks are too few to overlap (24 x 131072 fp32 in clusters of 8).
  cfg.blockDim = dim3(lp_threads(p.part, sizeof(T), rows * p.share <= 2 * sm_count() ? kLpThreads : 128));
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = p.share; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = p.share > 1 ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, logprob_fwd_kernel<T>, p);
}

}  // namespace mxb

using namespace mxb;

// x: [rows, cols]; tokens: [rows]; top_lp / top_id: [rows, k] (k may be 0); stat: [rows, 3] floats for the backward pass.
MXB_EXPORT int mxb_logprob_forward(int dtype, const void* x, const int64_t* tokens, float* log_prob, float* entropy, float* top_lp,
                                   int64_t* top_id, float* stat, int64_t rows, int cols, int k, int64_t ignore, void* stream) {
  if (rows < 1 || cols < 1 || k < 0 || k > kLpMaxTop || k > cols) return -2;
  LogProbParams p{x, tokens, log_prob, entropy, top_lp, top_id, stat, rows, cols, k, ignore, 1, cols};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == kF32) return logprob_forward<float>(p, st);
  if (dtype == kF16) return logprob_forward<__half>(p, st);
  if (dtype == kBF16) return logprob_forward<__nv_bfloat16>(p, st);
  return -1;
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
  if (dtype == kF32) logprob_bwd_kernel<float><<<grid, lp_threads(cols, 4, kLpGradThreads), 0, st>>>(p);
  else if (dtype == kF16) logprob_bwd_kernel<__half><<<grid, lp_threads(cols, 2, kLpGradThreads), 0, st>>>(p);
  else if (dtype == kBF16) logprob_bwd_kernel<__nv_bfloat16><<<grid, lp_threads(cols, 2, kLpGradThreads), 0, st>>>(p);
  else return -1;
  return (int)cudaGetLastError();
}
