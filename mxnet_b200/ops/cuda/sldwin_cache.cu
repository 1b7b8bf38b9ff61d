// The rolling key/value cache of sliding-window attention for sm_100a: filling it with prompts, and the attention of one
// new token of each sequence over it.
//
// A cache of C rows keeps the first `sinks` positions in place and the last R = C - sinks others in a ring:
//   row(p) = p < sinks ? p : sinks + (p - sinks) mod R.
// Both kernels are bound by the bytes of the keys and values they move.  Filling 16 caches of 4096 x 8 heads of 128 (bf16, 354 MB
// read and written): 51 us, the rate of a copy.  A token for each of 64 sequences over 4100 rows of 8 heads of 128 for 32 query
// heads (bf16, 892 MB): 168 us, 5.3 TB/s of the 6.4 a copy reaches.
#include "common.cuh"

namespace mxb {

struct CacheStride { int64_t b, t, h; };

// ------------------------------------------------------------------------------------------------ fill
struct FillParams {
  const void *k, *v;
  void *kc, *vc;
  const int* valid;                      // [B] or null
  CacheStride sk, sv, skc, svc;
  int B, T, H, D, C, sinks;
  int units;                             // H * D / V
  FastDiv div_units, div_d;              // div_d: D / V
};

constexpr int kFillThreads = 256;

template <typename U, int V>
__global__ void __launch_bounds__(kFillThreads)
cache_fill_kernel(const FillParams p) {
  const int b = blockIdx.y;
  int n = p.valid ? p.valid[b] : p.T;
  n = n < 0 ? 0 : (n > p.T ? p.T : n);
  const int ring = p.C - p.sinks;
  const int ns = min(p.sinks, n), lo = max(p.sinks, n - ring);
  const int keep = ns + max(0, n - lo);
  const int64_t total = (int64_t)keep * p.units;
  for (int64_t e = (int64_t)blockIdx.x * kFillThreads + threadIdx.x; e < total; e += (int64_t)gridDim.x * kFillThreads) {
    int i, u;
    if (total <= 0x7fffffff) {
      uint32_t qi, qu;
      fd_divmod((uint32_t)e, p.div_units, &qi, &qu);
      i = (int)qi; u = (int)qu;
    } else { i = (int)(e / p.units); u = (int)(e - (int64_t)i * p.units); }
    const int pos = i < ns ? i : lo + (i - ns);
    const int row = pos < p.sinks ? pos : p.sinks + (pos - p.sinks) % ring;
    uint32_t h, d;
    fd_divmod((uint32_t)u, p.div_d, &h, &d);
    const int64_t c = (int64_t)d * V;
    const U kv = *reinterpret_cast<const U*>(static_cast<const char*>(p.k) + (b * p.sk.b + pos * p.sk.t + h * p.sk.h + c) * (int64_t)(sizeof(U) / V));
    const U vv = *reinterpret_cast<const U*>(static_cast<const char*>(p.v) + (b * p.sv.b + pos * p.sv.t + h * p.sv.h + c) * (int64_t)(sizeof(U) / V));
    *reinterpret_cast<U*>(static_cast<char*>(p.kc) + (b * p.skc.b + row * p.skc.t + h * p.skc.h + c) * (int64_t)(sizeof(U) / V)) = kv;
    *reinterpret_cast<U*>(static_cast<char*>(p.vc) + (b * p.svc.b + row * p.svc.t + h * p.svc.h + c) * (int64_t)(sizeof(U) / V)) = vv;
  }
}

// ------------------------------------------------------------------------------------------------ step
struct StepParams {
  const void *q, *k, *v;                 // contiguous [B, Hq, D], [B, Hk, D]
  void *kc, *vc;
  void* out;                             // [B, Hq, D]
  const int64_t* pos;                    // [B]: position of the new token; negative = no sequence here
  CacheStride skc, svc;
  int B, Hq, Hk, D, C, window, sinks;    // window: 1 .. C - sinks
  float scale;
};

constexpr int kStepMaxD = 256;

// Keys that a token at `pos` sees, as indexes 0 .. seen - 1: the sinks, then a run of ring rows; the last one is the token itself.
struct StepView {
  int64_t seen, ns, first;               // first: ring row of index ns
  int ring, sinks;
  int64_t row_new;
  __device__ __forceinline__ StepView(const StepParams& p, int64_t pos) {
    ring = p.C - p.sinks;
    sinks = p.sinks;
    if (pos < 0) { seen = ns = first = row_new = 0; return; }
    const int64_t lo = max((int64_t)p.sinks, pos - p.window + 1);
    ns = min((int64_t)p.sinks, pos + 1);
    seen = ns + max((int64_t)0, pos + 1 - lo);
    first = (lo - p.sinks) % ring;
    row_new = pos < p.sinks ? pos : p.sinks + (pos - p.sinks) % ring;
  }
  __device__ __forceinline__ int row(int64_t i) const {
    if (i < ns) return (int)i;
    const int64_t r = first + (i - ns);
    return sinks + (int)(r >= ring ? r - ring : r);
  }
};

// ------------------------------------------------------------------------------------------------ step, general
// A block for each sample and key head, its warps side by side over the keys, channels over the lanes; one query head after
// another.  For fp32 and head sizes that the kernel below does not take.
constexpr int kStepWarps = 8;

template <typename T>
__global__ void __launch_bounds__(kStepWarps * 32)
step_general_kernel(const StepParams p) {
  __shared__ float s_m[kStepWarps], s_l[kStepWarps], s_o[kStepWarps][kStepMaxD];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / p.Hk, hk = blockIdx.x % p.Hk, group = p.Hq / p.Hk;
  const int64_t pos = p.pos[b];
  const StepView view(p, pos);
  T* kc = static_cast<T*>(p.kc) + b * p.skc.b + hk * p.skc.h;
  T* vc = static_cast<T*>(p.vc) + b * p.svc.b + hk * p.svc.h;
  const T* kn = static_cast<const T*>(p.k) + ((int64_t)b * p.Hk + hk) * p.D;
  const T* vn = static_cast<const T*>(p.v) + ((int64_t)b * p.Hk + hk) * p.D;
  if (pos >= 0)
    for (int d = threadIdx.x; d < p.D; d += blockDim.x) { kc[view.row_new * p.skc.t + d] = kn[d]; vc[view.row_new * p.svc.t + d] = vn[d]; }
  const float sc = p.scale * 1.4426950408889634f;
  for (int g = 0; g < group; ++g) {
    const int64_t at = ((int64_t)b * p.Hq + hk * group + g) * p.D;
    const T* q = static_cast<const T*>(p.q) + at;
    float qr[kStepMaxD / 32], acc[kStepMaxD / 32];
#pragma unroll
    for (int c = 0; c < kStepMaxD / 32; ++c) { qr[c] = lane + c * 32 < p.D ? Cvt<T>::to_f(q[lane + c * 32]) : 0.f; acc[c] = 0.f; }
    float m = -INFINITY, l = 0.f;
    for (int64_t i = warp; i < view.seen; i += kStepWarps) {
      const bool own = i == view.seen - 1;
      const int64_t row = view.row(i);
      const T* kr = own ? kn : kc + row * p.skc.t;
      const T* vr = own ? vn : vc + row * p.svc.t;
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < kStepMaxD / 32; ++c) if (lane + c * 32 < p.D) s += qr[c] * Cvt<T>::to_f(kr[lane + c * 32]);
      s = warp_sum(s) * sc;
      const float mn = fmaxf(m, s), mm = mn == -INFINITY ? 0.f : mn, alpha = exp2f(m - mm), w = exp2f(s - mm);
      l = l * alpha + w;
      m = mn;
#pragma unroll
      for (int c = 0; c < kStepMaxD / 32; ++c)
        if (lane + c * 32 < p.D) acc[c] = acc[c] * alpha + w * Cvt<T>::to_f(vr[lane + c * 32]);
    }
    if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
    for (int c = 0; c < kStepMaxD / 32; ++c) if (lane + c * 32 < p.D) s_o[warp][lane + c * 32] = acc[c];
    __syncthreads();
    float mm = -INFINITY, total = 0.f;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) mm = fmaxf(mm, s_m[w]);
    const float base = mm == -INFINITY ? 0.f : mm;
#pragma unroll
    for (int w = 0; w < kStepWarps; ++w) total += s_l[w] * exp2f(s_m[w] - base);
    for (int d = threadIdx.x; d < p.D; d += blockDim.x) {
      float o = 0.f;
#pragma unroll
      for (int w = 0; w < kStepWarps; ++w) o += s_o[w][d] * exp2f(s_m[w] - base);
      static_cast<T*>(p.out)[at + d] = Cvt<T>::from_f(total == 0.f ? 0.f : o / total);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ step, half types
// Bound by the bytes of the visible keys and values: 2 x seen x D x 2 for each key head, which every query head of the group
// shares.  The products run on the tensor cores only because at 8 heads for each byte the fp32 pipe would be the limit.
// A warp takes 16 keys at a time straight from memory into matrix fragments, 16 bytes for each load and no shared memory:
//   S^T[16 keys, 8 heads] = K Q^T: the order of the channels in a dot product is free, so the 8 adjacent channels of a load
//   serve as the elements that two k-steps want of a lane;
//   O^T[D, 8 heads] += V^T P^T: a lane holds 8 adjacent channels of 4 keys; pairs of keys are packed per channel, and the
//   channels of a 16-row tile are the ones that its lanes hold.  P^T turns by one 8 x 8 transpose for each 8 keys.
// The keys of one sample and key head are dealt over the warps of a cluster of CTAs; partial results meet in shared memory,
// then over distributed shared memory: one launch, no workspace, a fixed order of additions.
constexpr float kStepShift = 6.f, kStepLag = 8.f;        // as in the sequence kernels: P is kept 2^6 times its value

template <typename T> __device__ __forceinline__ void mma_16x8x16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16x8x16<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T> __device__ __forceinline__ uint32_t step_pack(float lo, float hi) {
  const T a = Cvt<T>::from_f(lo), b = Cvt<T>::from_f(hi);
  return (uint32_t)*reinterpret_cast<const uint16_t*>(&a) | ((uint32_t)*reinterpret_cast<const uint16_t*>(&b) << 16);
}
__device__ __forceinline__ float ld_cluster_f32(const float* local, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(local)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// blockIdx.x = ((sample, key head, chunk of 8 query heads), rank in the cluster)
template <typename T, int D>
__global__ void __launch_bounds__(256, 2)
step_tc_kernel(const StepParams p, int chunks, int csize) {
  constexpr int C16 = D / 64;                             // 64-channel parts of a row
  extern __shared__ float sm[];                           // [warps][8 heads][D + 2]: partial outputs, then m and l
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int r = lane >> 2, c = lane & 3;
  const int rank = blockIdx.x % csize, unit = blockIdx.x / csize;
  const int chunk = unit % chunks, bh = unit / chunks, b = bh / p.Hk, hk = bh % p.Hk, group = p.Hq / p.Hk;
  const int heads = min(8, group - chunk * 8), h0 = hk * group + chunk * 8;
  const int64_t pos = p.pos[b];
  const StepView view(p, pos);
  T* kc = static_cast<T*>(p.kc) + b * p.skc.b + hk * p.skc.h;
  T* vc = static_cast<T*>(p.vc) + b * p.svc.b + hk * p.svc.h;
  const T* kn = static_cast<const T*>(p.k) + ((int64_t)b * p.Hk + hk) * D;
  const T* vn = static_cast<const T*>(p.v) + ((int64_t)b * p.Hk + hk) * D;
  // The new token's row replaces a position that its ring has passed: nobody reads the old contents.
  if (pos >= 0 && rank == 0 && chunk == 0 && threadIdx.x < D / 4) {
    const int which = threadIdx.x / (D / 8), e = threadIdx.x % (D / 8) * 8;
    st16((which ? vc + view.row_new * p.svc.t : kc + view.row_new * p.skc.t) + e, ld16((which ? vn : kn) + e));
  }
  uint32_t q[D / 16][2];                                  // Q^T fragments: head r, channels in the order of the key loads
#pragma unroll
  for (int m = 0; m < D / 32; ++m) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < heads) v = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + ((int64_t)b * p.Hq + h0 + r) * D + m * 32 + c * 8);
    q[2 * m][0] = v.x; q[2 * m][1] = v.y; q[2 * m + 1][0] = v.z; q[2 * m + 1][1] = v.w;
  }
  float o[4 * C16][4];                                    // tile t of part u: channels 64 u + 8 (row % 8) + 2 t + (row >= 8)
#pragma unroll
  for (int t = 0; t < 4 * C16; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;
  float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};       // heads 2 c and 2 c + 1
  const float sc = p.scale * 1.4426950408889634f;

  const int64_t stride = (int64_t)csize * nw * 16;
  for (int64_t i0 = ((int64_t)rank * nw + warp) * 16; i0 < view.seen; i0 += stride) {
    auto key_row = [&](int64_t i) { return i >= view.seen - 1 ? kn : kc + (int64_t)view.row(i) * p.skc.t; };   // behind the end: the token's own, masked
    auto val_row = [&](int64_t i) { return i >= view.seen - 1 ? vn : vc + (int64_t)view.row(i) * p.svc.t; };
    uint4 k0[D / 32], k1[D / 32], v[4][C16];
    {
      const T *a = key_row(i0 + r) + c * 8, *e = key_row(i0 + r + 8) + c * 8;
#pragma unroll
      for (int m = 0; m < D / 32; ++m) { k0[m] = __ldcs(reinterpret_cast<const uint4*>(a + m * 32)); k1[m] = __ldcs(reinterpret_cast<const uint4*>(e + m * 32)); }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const T* w = val_row(i0 + 2 * c + (x & 1) + (x >> 1) * 8) + r * 8;
#pragma unroll
        for (int u = 0; u < C16; ++u) v[x][u] = __ldcs(reinterpret_cast<const uint4*>(w + u * 64));
      }
    }
    float s[4] = {0.f, 0.f, 0.f, 0.f};                    // (key r, heads 2 c, 2 c + 1), (key r + 8, the same)
#pragma unroll
    for (int m = 0; m < D / 32; ++m) {
      const uint32_t a0[4] = {k0[m].x, k1[m].x, k0[m].y, k1[m].y}, a1[4] = {k0[m].z, k1[m].z, k0[m].w, k1[m].w};
      mma_16x8x16<T>(s, a0, q[2 * m][0], q[2 * m][1]);
      mma_16x8x16<T>(s, a1, q[2 * m + 1][0], q[2 * m + 1][1]);
    }
    const bool in0 = i0 + r < view.seen, in1 = i0 + r + 8 < view.seen;
#pragma unroll
    for (int e = 0; e < 2; ++e) { s[e] = in0 ? s[e] * sc : -INFINITY; s[e + 2] = in1 ? s[e + 2] * sc : -INFINITY; }
    const float t0 = fmaxf(s[0], s[2]), t1 = fmaxf(s[1], s[3]);
    const bool move = t0 > mx[0] + kStepLag || t1 > mx[1] + kStepLag || (mx[0] == -INFINITY && t0 > -INFINITY) || (mx[1] == -INFINITY && t1 > -INFINITY);
    if (__any_sync(0xffffffffu, move)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float t = e ? t1 : t0;
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, d));
        const float mn = fmaxf(mx[e], t), alpha = mn == -INFINITY ? 0.f : exp2f(mx[e] - mn);
        mx[e] = mn;
        sum[e] *= alpha;
#pragma unroll
        for (int x = 0; x < 4 * C16; ++x) { o[x][e] *= alpha; o[x][e + 2] *= alpha; }
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float off = kStepShift - (mx[e] == -INFINITY ? 0.f : mx[e]);
      s[e] = exp2f(s[e] + off);
      s[e + 2] = exp2f(s[e + 2] + off);
      sum[e] += s[e] + s[e + 2];
    }
    const uint32_t b0 = transpose_8x8(step_pack<T>(s[0], s[1])), b1 = transpose_8x8(step_pack<T>(s[2], s[3]));
#pragma unroll
    for (int u = 0; u < C16; ++u) {
      const uint32_t* w0 = reinterpret_cast<const uint32_t*>(&v[0][u]);
      const uint32_t* w1 = reinterpret_cast<const uint32_t*>(&v[1][u]);
      const uint32_t* w2 = reinterpret_cast<const uint32_t*>(&v[2][u]);
      const uint32_t* w3 = reinterpret_cast<const uint32_t*>(&v[3][u]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t a[4] = {__byte_perm(w0[t], w1[t], 0x5410), __byte_perm(w0[t], w1[t], 0x7632), __byte_perm(w2[t], w3[t], 0x5410),
                               __byte_perm(w2[t], w3[t], 0x7632)};
        mma_16x8x16<T>(o[u * 4 + t], a, b0, b1);
      }
    }
  }

  // ------------------------------------------------------------ the warps' parts, then the CTAs'
  constexpr int W = D + 2;
#pragma unroll
  for (int e = 0; e < 2; ++e)
#pragma unroll
    for (int d = 4; d < 32; d <<= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], d);
  float* mine = sm + warp * 8 * W;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    float* at = mine + (2 * c + e) * W;
#pragma unroll
    for (int x = 0; x < 4 * C16; ++x) {
      const int d = (x >> 2) * 64 + r * 8 + (x & 3) * 2;
      at[d] = o[x][e];
      at[d + 1] = o[x][e + 2];
    }
    if (r == 0) { at[D] = mx[e]; at[D + 1] = sum[e]; }
  }
  __syncthreads();
  float* all = sm + nw * 8 * W;                           // this CTA's [8][W]
  for (int e = threadIdx.x; e < 8 * D; e += blockDim.x) {
    const int h = e / D, d = e % D;
    float m = -INFINITY, acc = 0.f, l = 0.f;
    for (int w = 0; w < nw; ++w) m = fmaxf(m, sm[(w * 8 + h) * W + D]);
    const float base = m == -INFINITY ? 0.f : m;
    for (int w = 0; w < nw; ++w) {
      const float f = exp2f(sm[(w * 8 + h) * W + D] - base);
      acc += sm[(w * 8 + h) * W + d] * f;
      l += sm[(w * 8 + h) * W + D + 1] * f;
    }
    all[h * W + d] = acc;
    if (d == 0) { all[h * W + D] = m; all[h * W + D + 1] = l; }
  }
  if (csize > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
  else __syncthreads();
  for (int e = rank * blockDim.x + threadIdx.x; e < heads * D; e += csize * blockDim.x) {
    const int h = e / D, d = e % D;
    float m = -INFINITY, acc = 0.f, l = 0.f;
    for (int k = 0; k < csize; ++k) m = fmaxf(m, ld_cluster_f32(all + h * W + D, k));
    const float base = m == -INFINITY ? 0.f : m;
    for (int k = 0; k < csize; ++k) {
      const float f = exp2f(ld_cluster_f32(all + h * W + D, k) - base);
      acc += ld_cluster_f32(all + h * W + d, k) * f;
      l += ld_cluster_f32(all + h * W + D + 1, k) * f;
    }
    static_cast<T*>(p.out)[((int64_t)b * p.Hq + h0) * D + e] = Cvt<T>::from_f(l == 0.f ? 0.f : acc / l);
  }
  // nobody leaves while others still read its shared memory
  if (csize > 1) asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <typename T, int D>
static int step_tc(const StepParams& p, cudaStream_t st) {
  const int group = p.Hq / p.Hk, chunks = (group + 7) / 8;
  const int64_t units = (int64_t)p.B * p.Hk * chunks;
  const int64_t most = (int64_t)p.sinks + p.window < p.C ? (int64_t)p.sinks + p.window : p.C;      // keys that a token may see
  // A cluster grows while its CTAs leave SMs short of the four that fit one and every warp still has 16 keys to take (512 units of
  // 4100 keys, head size 128: no cluster 176 us, clusters of 2 186 us, of 4 198 us).  Where clusters of 8 give no SM a second CTA,
  // CTAs get 8 warps, and clusters 16 CTAs if keys are many (8 units of 131072 keys: 8 CTAs x 4 warps 370 us, 8 x 8 213 us, 16 x 8
  // 155 us, 16 x 16 170 us).
  int csize = 1, nw = 4;
  while (csize < 8 && units * csize < 3 * (int64_t)sm_count() && most > (int64_t)csize * nw * 16) csize <<= 1;
  if (csize == 8 && units * csize <= 2 * (int64_t)sm_count() && most > 8 * 8 * 16) {
    nw = 8;
    if (units * 16 <= 2 * (int64_t)sm_count() && most > 16 * 8 * 16) csize = 16;
  }
  if (units * csize > 0x7fffffff) return -2;
  const size_t smem = (size_t)(nw + 1) * 8 * (D + 2) * sizeof(float);
  static unsigned long long seen = 0;
  if (auto first = first_on_device(&seen)) {
    const int code = first.take((int)cudaFuncSetAttribute(step_tc_kernel<T, D>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (code) { cudaGetLastError(); return code; }
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(units * csize));
  cfg.blockDim = dim3(nw * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = csize; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, step_tc_kernel<T, D>, p, chunks, csize);
}

}  // namespace mxb

using namespace mxb;

// form: B, T, H, D, C, sinks (0 .. C - 1), then the element strides of batch, position and head of k, v, key cache and value cache.
MXB_EXPORT int mxb_cache_fill(int dtype, const void* k, const void* v, void* kc, void* vc, const int* valid, const int64_t* form,
                              void* stream) {
  if (dtype < kF32 || dtype > kBF16) return -1;
  FillParams p{};
  p.k = k; p.v = v; p.kc = kc; p.vc = vc; p.valid = valid;
  for (int i = 0; i < 6; ++i) if (form[i] < 0 || form[i] > 0x7fffffff) return -2;
  p.B = (int)form[0]; p.T = (int)form[1]; p.H = (int)form[2]; p.D = (int)form[3]; p.C = (int)form[4]; p.sinks = (int)form[5];
  const int64_t* s = form + 6;
  p.sk = {s[0], s[1], s[2]}; p.sv = {s[3], s[4], s[5]}; p.skc = {s[6], s[7], s[8]}; p.svc = {s[9], s[10], s[11]};
  if (p.B < 1 || p.B > 65535 || p.T < 1 || p.H < 1 || p.D < 1 || p.sinks < 0 || p.C <= p.sinks) return -2;
  if ((int64_t)p.H * p.D > (1 << 30)) return -2;
  const int size = dtype == kF32 ? 4 : 2, vec = 16 / size;
  bool wide = p.D % vec == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)kc % 16 == 0 && (uintptr_t)vc % 16 == 0;
  for (int i = 0; i < 12; ++i) wide = wide && (s[i] * size) % 16 == 0;
  const int V = wide ? vec : 1;
  p.units = p.H * p.D / V;
  p.div_units = make_fastdiv((uint32_t)p.units);
  p.div_d = make_fastdiv((uint32_t)(p.D / V));
  const int64_t keep = p.T < p.C ? p.T : p.C;
  const int64_t blocks = (keep * p.units + kFillThreads - 1) / kFillThreads;
  const int64_t cap = ((int64_t)sm_count() * 64 + p.B - 1) / p.B;
  const dim3 grid((unsigned)(blocks < cap ? blocks : (cap < 1 ? 1 : cap)), (unsigned)p.B);
  cudaStream_t st = (cudaStream_t)stream;
  if (wide && size == 2) cache_fill_kernel<uint4, 8><<<grid, kFillThreads, 0, st>>>(p);
  else if (wide) cache_fill_kernel<uint4, 4><<<grid, kFillThreads, 0, st>>>(p);
  else if (size == 2) cache_fill_kernel<uint16_t, 1><<<grid, kFillThreads, 0, st>>>(p);
  else cache_fill_kernel<uint32_t, 1><<<grid, kFillThreads, 0, st>>>(p);
  return (int)cudaGetLastError();
}

// form: B, Hq, Hk, D, C, window (1 .. C - sinks), sinks, then the element strides of batch, row and head of the key and the value cache.
MXB_EXPORT int mxb_sldwin_step(int dtype, const void* q, const void* k, const void* v, void* kc, void* vc, const int64_t* pos, void* out,
                               const int64_t* form, float scale, void* stream) {
  StepParams p{};
  p.q = q; p.k = k; p.v = v; p.kc = kc; p.vc = vc; p.pos = pos; p.out = out;
  for (int i = 0; i < 7; ++i) if (form[i] < 0 || form[i] > 0x7fffffff) return -2;
  p.B = (int)form[0]; p.Hq = (int)form[1]; p.Hk = (int)form[2]; p.D = (int)form[3]; p.C = (int)form[4]; p.window = (int)form[5];
  p.sinks = (int)form[6];
  const int64_t* s = form + 7;
  p.skc = {s[0], s[1], s[2]}; p.svc = {s[3], s[4], s[5]};
  p.scale = scale;
  if (p.B < 1 || p.Hk < 1 || p.Hq < p.Hk || p.Hq % p.Hk || p.D < 1 || p.D > kStepMaxD || p.sinks < 0 || p.C <= p.sinks ||
      p.window < 1 || p.window > p.C - p.sinks || (int64_t)p.B * p.Hk > 0x7fffffff) return -2;
  cudaStream_t st = (cudaStream_t)stream;
  const bool aligned = (uintptr_t)q % 16 == 0 && (uintptr_t)k % 16 == 0 && (uintptr_t)v % 16 == 0 && (uintptr_t)kc % 16 == 0 &&
                       (uintptr_t)vc % 16 == 0 && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0 && s[3] % 8 == 0 && s[4] % 8 == 0 &&
                       s[5] % 8 == 0;
  if (aligned && dtype == kF16 && p.D == 64) return step_tc<__half, 64>(p, st);
  if (aligned && dtype == kF16 && p.D == 128) return step_tc<__half, 128>(p, st);
  if (aligned && dtype == kBF16 && p.D == 64) return step_tc<__nv_bfloat16, 64>(p, st);
  if (aligned && dtype == kBF16 && p.D == 128) return step_tc<__nv_bfloat16, 128>(p, st);
  const unsigned grid = (unsigned)(p.B * p.Hk);
  if (dtype == kF32) step_general_kernel<float><<<grid, kStepWarps * 32, 0, st>>>(p);
  else if (dtype == kF16) step_general_kernel<__half><<<grid, kStepWarps * 32, 0, st>>>(p);
  else if (dtype == kBF16) step_general_kernel<__nv_bfloat16><<<grid, kStepWarps * 32, 0, st>>>(p);
  else return -1;
  return (int)cudaGetLastError();
}
