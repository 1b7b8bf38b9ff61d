// The rolling key/value cache of sliding-window attention for sm_100a: filling it with prompts, and the attention of one
// new token of each sequence over it.
//
// A cache of C rows keeps the first `sinks` positions in place and the last R = C - sinks others in a ring:
//   row(p) = p < sinks ? p : sinks + (p - sinks) mod R.
// Both kernels are bound by the bytes of the keys and values they move.
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

// One warp for each query head of one sample: keys one after another, channels over the lanes.
template <typename T>
__global__ void step_general_kernel(const StepParams p) {
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.x / p.Hk, hk = blockIdx.x % p.Hk, group = p.Hq / p.Hk;
  const int64_t pos = p.pos[b];
  const int ring = p.C - p.sinks;
  const int64_t row_new = pos < p.sinks ? pos : p.sinks + (pos - p.sinks) % ring;
  T* kc = static_cast<T*>(p.kc) + b * p.skc.b + hk * p.skc.h;
  T* vc = static_cast<T*>(p.vc) + b * p.svc.b + hk * p.svc.h;
  const T* kn = static_cast<const T*>(p.k) + ((int64_t)b * p.Hk + hk) * p.D;
  const T* vn = static_cast<const T*>(p.v) + ((int64_t)b * p.Hk + hk) * p.D;
  if (pos >= 0)
    for (int d = threadIdx.x; d < p.D; d += blockDim.x) { kc[row_new * p.skc.t + d] = kn[d]; vc[row_new * p.svc.t + d] = vn[d]; }
  __syncthreads();
  const float sc = p.scale * 1.4426950408889634f;
  const int64_t ns = min((int64_t)p.sinks, pos + 1), lo = max((int64_t)p.sinks, pos - p.window + 1);
  const int64_t seen = pos < 0 ? 0 : ns + max((int64_t)0, pos + 1 - lo);
  const int64_t lo_ring = (lo - p.sinks) % ring;
  for (int g = threadIdx.x >> 5; g < group; g += blockDim.x >> 5) {
    const int64_t at = ((int64_t)b * p.Hq + hk * group + g) * p.D;
    const T* q = static_cast<const T*>(p.q) + at;
    float qr[kStepMaxD / 32], acc[kStepMaxD / 32];
#pragma unroll
    for (int c = 0; c < kStepMaxD / 32; ++c) { qr[c] = lane + c * 32 < p.D ? Cvt<T>::to_f(q[lane + c * 32]) : 0.f; acc[c] = 0.f; }
    float m = -INFINITY, l = 0.f;
    for (int64_t i = 0; i < seen; ++i) {
      int64_t row = i;
      if (i >= ns) { row = lo_ring + (i - ns); row = p.sinks + (row >= ring ? row - ring : row); }
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < kStepMaxD / 32; ++c) if (lane + c * 32 < p.D) s += qr[c] * Cvt<T>::to_f(kc[row * p.skc.t + lane + c * 32]);
      s = warp_sum(s) * sc;
      const float mn = fmaxf(m, s), mm = mn == -INFINITY ? 0.f : mn, alpha = exp2f(m - mm), w = exp2f(s - mm);
      l = l * alpha + w;
      m = mn;
#pragma unroll
      for (int c = 0; c < kStepMaxD / 32; ++c)
        if (lane + c * 32 < p.D) acc[c] = acc[c] * alpha + w * Cvt<T>::to_f(vc[row * p.svc.t + lane + c * 32]);
    }
    const float inv = seen ? 1.f / l : 0.f;
    T* o = static_cast<T*>(p.out) + at;
#pragma unroll
    for (int c = 0; c < kStepMaxD / 32; ++c) if (lane + c * 32 < p.D) o[lane + c * 32] = Cvt<T>::from_f(seen ? acc[c] * inv : 0.f);
  }
}

}  // namespace mxb

using namespace mxb;

// dims: B, T, H, D, C, sinks (0 .. C - 1).  strides: batch, position, head of k, v, key cache, value cache, in elements.
MXB_EXPORT int mxb_cache_fill(int dtype, const void* k, const void* v, void* kc, void* vc, const int* valid, const int* dims,
                              const int64_t* s, void* stream) {
  if (dtype < kF32 || dtype > kBF16) return -1;
  FillParams p{};
  p.k = k; p.v = v; p.kc = kc; p.vc = vc; p.valid = valid;
  p.B = dims[0]; p.T = dims[1]; p.H = dims[2]; p.D = dims[3]; p.C = dims[4]; p.sinks = dims[5];
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

// dims: B, Hq, Hk, D, C, window (1 .. C - sinks), sinks.  strides: batch, row, head of the key and the value cache.
MXB_EXPORT int mxb_sldwin_step(int dtype, const void* q, const void* k, const void* v, void* kc, void* vc, const int64_t* pos, void* out,
                               const int* dims, const int64_t* s, float scale, void* stream) {
  StepParams p{};
  p.q = q; p.k = k; p.v = v; p.kc = kc; p.vc = vc; p.pos = pos; p.out = out;
  p.B = dims[0]; p.Hq = dims[1]; p.Hk = dims[2]; p.D = dims[3]; p.C = dims[4]; p.window = dims[5]; p.sinks = dims[6];
  p.skc = {s[0], s[1], s[2]}; p.svc = {s[3], s[4], s[5]};
  p.scale = scale;
  if (p.B < 1 || p.Hk < 1 || p.Hq < p.Hk || p.Hq % p.Hk || p.D < 1 || p.D > kStepMaxD || p.sinks < 0 || p.C <= p.sinks ||
      p.window < 1 || p.window > p.C - p.sinks || (int64_t)p.B * p.Hk > 0x7fffffff) return -2;
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)(p.B * p.Hk);
  const int group = p.Hq / p.Hk;
  const int threads = 32 * (group < 8 ? group : 8);
  if (dtype == kF32) step_general_kernel<float><<<grid, threads, 0, st>>>(p);
  else if (dtype == kF16) step_general_kernel<__half><<<grid, threads, 0, st>>>(p);
  else if (dtype == kBF16) step_general_kernel<__nv_bfloat16><<<grid, threads, 0, st>>>(p);
  else return -1;
  return (int)cudaGetLastError();
}
