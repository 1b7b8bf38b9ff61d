// Causal attention over a sliding window with sinks for sm_100a, forward and backward.
//
//   query i sees key j when j <= i and (i - j < window or j < sinks); window 0: every j <= i.
//   Rows at or behind valid_length are not there: they see nothing, are seen by nothing, and their outputs and gradients are 0.
//   O = softmax(scale Q K^T) V;  with P the probabilities and delta = rowsum(dO * O):
//   dV = P^T dO,  dS = P * (dO V^T - delta),  dQ = scale dS K,  dK = scale dS^T Q, summed over the query heads of a key head.
//
// Layout [B, T, H, D] with element strides for batch, position and head; Hq a multiple of Hk.  The log-sum-exp of each row is
// kept in units of log2 (fp32 [B, Hq, T]); it is +inf where a row sees nothing, so that its probabilities are 0.
//
// This file holds the general kernels, which serve fp32 and head sizes that the tensor-core kernels do not take.  One
// warp works on one query (or key) row and walks the other side in tiles of 32 rows in shared memory, one lane for each
// row of the tile in the products over channels, one lane for each 32nd channel in the sums over rows.
#include <mutex>

#include "tcgen05.cuh"

namespace mxb {

constexpr int kSwMaxD = 256;
constexpr int kSwWarps = 8;
constexpr float kSwLog2e = 1.4426950408889634f;

struct SwStride { int64_t b, t, h; };

struct SwParams {
  const void *q, *k, *v, *o, *dout;
  void *out, *dq, *dk, *dv;              // contiguous [B, T, H, D]
  float* lse;                            // [B, Hq, T]
  float* delta;                          // [B, Hq, T]
  const int* valid;                      // [B] or null
  SwStride sq, sk, sv, sdo;
  int B, T, Hq, Hk, D;
  int window, sinks;                     // window >= 1; unlimited = T
  float scale;
};

__device__ __forceinline__ int sw_valid(const SwParams& p, int b) {
  int n = p.valid ? p.valid[b] : p.T;
  return n < 0 ? 0 : (n > p.T ? p.T : n);
}
__device__ __forceinline__ bool sw_sees(const SwParams& p, int i, int j) { return j <= i && (i - j < p.window || j < p.sinks); }

// ------------------------------------------------------------------------------------------------ general kernels
// blockIdx.x = (b, h, tile of kSwWarps rows); kMode 0: forward, 1: dQ and delta.
template <typename T, int kMode>
__global__ void __launch_bounds__(kSwWarps * 32)
sw_row_kernel(const SwParams p) {
  extern __shared__ float sm[];
  const int D = p.D, W = D + 1;
  float* sK = sm;
  float* sV = sK + 32 * W;
  float* sQ = sV + 32 * W;               // [kSwWarps][D]
  float* sG = sQ + kSwWarps * D;         // dO rows
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tiles = (p.T + kSwWarps - 1) / kSwWarps;
  const int tile = blockIdx.x % tiles;
  const int bh = blockIdx.x / tiles, b = bh / p.Hq, h = bh % p.Hq, hk = h / (p.Hq / p.Hk);
  const int n = sw_valid(p, b);
  const int i0 = tile * kSwWarps, i = i0 + warp;
  const bool live = i < n;
  const T* k = static_cast<const T*>(p.k) + b * p.sk.b + hk * p.sk.h;
  const T* v = static_cast<const T*>(p.v) + b * p.sv.b + hk * p.sv.h;
  float delta = 0.f, lse = INFINITY;
  if (live) {
    const T* q = static_cast<const T*>(p.q) + b * p.sq.b + i * p.sq.t + h * p.sq.h;
    for (int d = lane; d < D; d += 32) sQ[warp * D + d] = Cvt<T>::to_f(q[d]);
    if (kMode == 1) {
      const T* g = static_cast<const T*>(p.dout) + b * p.sdo.b + i * p.sdo.t + h * p.sdo.h;
      const T* o = static_cast<const T*>(p.o) + (((int64_t)b * p.T + i) * p.Hq + h) * D;
      for (int d = lane; d < D; d += 32) {
        const float gv = Cvt<T>::to_f(g[d]);
        sG[warp * D + d] = gv;
        delta += gv * Cvt<T>::to_f(o[d]);
      }
      delta = warp_sum(delta);
      lse = p.lse[((int64_t)b * p.Hq + h) * p.T + i];
    }
  }
  float acc[kSwMaxD / 32];
#pragma unroll
  for (int c = 0; c < kSwMaxD / 32; ++c) acc[c] = 0.f;
  float m = -INFINITY, l = 0.f;
  const int last = min(i0 + kSwWarps, n) - 1;             // last row of the block that is there
  if (last >= i0) {
    const int first = max(0, i0 - p.window + 1);          // first key of the windows
    const int sink_end = min(p.sinks, last + 1);
    const float sc = p.scale * kSwLog2e;
    for (int j0 = 0; j0 <= last; j0 += 32) {
      if (j0 >= sink_end && j0 + 32 <= first) { j0 = (first / 32) * 32 - 32; continue; }
      __syncthreads();
      for (int e = threadIdx.x; e < 32 * D; e += kSwWarps * 32) {
        const int r = e / D, d = e - r * D, j = j0 + r;
        sK[r * W + d] = j <= last ? Cvt<T>::to_f(k[j * p.sk.t + d]) : 0.f;
        sV[r * W + d] = j <= last ? Cvt<T>::to_f(v[j * p.sv.t + d]) : 0.f;
      }
      __syncthreads();
      if (!live) continue;
      const int j = j0 + lane;
      float s = 0.f, dp = 0.f;
      for (int d = 0; d < D; ++d) s += sQ[warp * D + d] * sK[lane * W + d];
      s = sw_sees(p, i, j) ? s * sc : -INFINITY;
      float w;
      if (kMode == 0) {
        const float mn = fmaxf(m, warp_max(s));
        const float mm = mn == -INFINITY ? 0.f : mn;
        const float alpha = exp2f(m - mm);
        w = s == -INFINITY ? 0.f : exp2f(s - mm);
        l = l * alpha + warp_sum(w);
        m = mn;
#pragma unroll
        for (int c = 0; c < kSwMaxD / 32; ++c) acc[c] *= alpha;
      } else {
        for (int d = 0; d < D; ++d) dp += sG[warp * D + d] * sV[lane * W + d];
        w = s == -INFINITY ? 0.f : exp2f(s - lse) * (dp - delta) * p.scale;
      }
      const float* rows = kMode == 0 ? sV : sK;
      for (int r = 0; r < 32; ++r) {
        const float pr = __shfl_sync(0xffffffffu, w, r);
        if (!sw_sees(p, i, j0 + r)) continue;             // a hidden row may hold anything: it is not even multiplied by 0
#pragma unroll
        for (int c = 0; c < kSwMaxD / 32; ++c) if (lane + c * 32 < D) acc[c] += pr * rows[r * W + lane + c * 32];
      }
    }
  }
  if (i < p.T) {
    const int64_t at = ((int64_t)b * p.Hq + h) * p.T + i;
    const float inv = kMode == 0 ? (l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l)) : 1.f;
    T* out = static_cast<T*>(kMode == 0 ? p.out : p.dq) + (((int64_t)b * p.T + i) * p.Hq + h) * D;
#pragma unroll
    for (int c = 0; c < kSwMaxD / 32; ++c) if (lane + c * 32 < D) out[lane + c * 32] = Cvt<T>::from_f(live ? acc[c] * inv : 0.f);
    if (lane == 0) {
      if (kMode == 0) { if (p.lse) p.lse[at] = live && l > 0.f ? m + log2f(l) : (l == l ? INFINITY : l); }
      else p.delta[at] = live ? delta : 0.f;
    }
  }
}

// dK and dV: blockIdx.x = (b, key head, tile of kSwWarps keys); walks the queries that can see them, head after head.
template <typename T>
__global__ void __launch_bounds__(kSwWarps * 32)
sw_key_kernel(const SwParams p) {
  extern __shared__ float sm[];
  const int D = p.D, W = D + 1;
  float* sQ = sm;
  float* sG = sQ + 32 * W;
  float* sK = sG + 32 * W;               // [kSwWarps][D]
  float* sV = sK + kSwWarps * D;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tiles = (p.T + kSwWarps - 1) / kSwWarps;
  const int tile = blockIdx.x % tiles;
  const int bh = blockIdx.x / tiles, b = bh / p.Hk, hk = bh % p.Hk, group = p.Hq / p.Hk;
  const int n = sw_valid(p, b);
  const int j0 = tile * kSwWarps, j = j0 + warp;
  const bool live = j < n;
  if (live) {
    const T* k = static_cast<const T*>(p.k) + b * p.sk.b + j * p.sk.t + hk * p.sk.h;
    const T* v = static_cast<const T*>(p.v) + b * p.sv.b + j * p.sv.t + hk * p.sv.h;
    for (int d = lane; d < D; d += 32) { sK[warp * D + d] = Cvt<T>::to_f(k[d]); sV[warp * D + d] = Cvt<T>::to_f(v[d]); }
  }
  float ak[kSwMaxD / 32], av[kSwMaxD / 32];
#pragma unroll
  for (int c = 0; c < kSwMaxD / 32; ++c) ak[c] = av[c] = 0.f;
  const int lastk = min(j0 + kSwWarps, n) - 1;
  // queries: from the first key of the tile to the end, or to the last window that reaches the tile
  int64_t end = n;
  if (j0 >= p.sinks) end = min((int64_t)n, (int64_t)lastk + p.window);
  const float sc = p.scale * kSwLog2e;
  if (lastk >= j0) {
    for (int h = hk * group; h < (hk + 1) * group; ++h) {
      const T* q = static_cast<const T*>(p.q) + b * p.sq.b + h * p.sq.h;
      const T* g = static_cast<const T*>(p.dout) + b * p.sdo.b + h * p.sdo.h;
      const float* lse = p.lse + ((int64_t)b * p.Hq + h) * p.T;
      const float* delta = p.delta + ((int64_t)b * p.Hq + h) * p.T;
      for (int i0 = j0; i0 < end; i0 += 32) {
        __syncthreads();
        for (int e = threadIdx.x; e < 32 * D; e += kSwWarps * 32) {
          const int r = e / D, d = e - r * D, i = i0 + r;
          sQ[r * W + d] = i < end ? Cvt<T>::to_f(q[i * p.sq.t + d]) : 0.f;
          sG[r * W + d] = i < end ? Cvt<T>::to_f(g[i * p.sdo.t + d]) : 0.f;
        }
        __syncthreads();
        if (!live) continue;
        const int i = i0 + lane;
        float s = 0.f, dp = 0.f;
        for (int d = 0; d < D; ++d) { s += sK[warp * D + d] * sQ[lane * W + d]; dp += sV[warp * D + d] * sG[lane * W + d]; }
        const bool on = i < end && sw_sees(p, i, j);
        const float pr = on ? exp2f(s * sc - lse[i]) : 0.f;
        const float ds = on ? pr * (dp - delta[i]) * p.scale : 0.f;
        for (int r = 0; r < 32; ++r) {
          const float pv = __shfl_sync(0xffffffffu, pr, r), dv = __shfl_sync(0xffffffffu, ds, r);
          if (i0 + r >= end || !sw_sees(p, i0 + r, j)) continue;
#pragma unroll
          for (int c = 0; c < kSwMaxD / 32; ++c)
            if (lane + c * 32 < D) { av[c] += pv * sG[r * W + lane + c * 32]; ak[c] += dv * sQ[r * W + lane + c * 32]; }
        }
      }
    }
  }
  if (j < p.T) {
    const int64_t at = (((int64_t)b * p.T + j) * p.Hk + hk) * D;
#pragma unroll
    for (int c = 0; c < kSwMaxD / 32; ++c)
      if (lane + c * 32 < D) {
        static_cast<T*>(p.dk)[at + lane + c * 32] = Cvt<T>::from_f(live ? ak[c] : 0.f);
        static_cast<T*>(p.dv)[at + lane + c * 32] = Cvt<T>::from_f(live ? av[c] : 0.f);
      }
  }
}

static size_t sw_smem(int D) { return (size_t)(2 * 32 * (D + 1) + 2 * kSwWarps * D) * sizeof(float); }

template <typename T>
static int sw_general(const SwParams& p, int pass, cudaStream_t st) {
  static unsigned long long seen = 0;
  if (auto first = first_on_device(&seen)) {
    const int most = (int)sw_smem(kSwMaxD);
    int code = first.take(allow_smem(sw_row_kernel<T, 0>, most));
    if (!code) code = first.take(allow_smem(sw_row_kernel<T, 1>, most));
    if (!code) code = first.take(allow_smem(sw_key_kernel<T>, most));
    if (code) return code;
  }
  const int64_t tiles = (p.T + kSwWarps - 1) / kSwWarps;
  const int64_t gq = tiles * p.B * p.Hq, gk = tiles * p.B * p.Hk;
  if (gq > 0x7fffffff) return -2;
  if (pass == 0) sw_row_kernel<T, 0><<<(unsigned)gq, kSwWarps * 32, sw_smem(p.D), st>>>(p);
  else {
    sw_row_kernel<T, 1><<<(unsigned)gq, kSwWarps * 32, sw_smem(p.D), st>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    sw_key_kernel<T><<<(unsigned)gk, kSwWarps * 32, sw_smem(p.D), st>>>(p);
  }
  return (int)cudaGetLastError();
}

static bool sw_shape_ok(const SwParams& p) {
  return p.B >= 1 && p.T >= 1 && p.Hk >= 1 && p.Hq >= p.Hk && p.Hq % p.Hk == 0 && p.D >= 1 && p.D <= kSwMaxD && p.window >= 1 &&
         p.window <= p.T && p.sinks >= 0 && p.sinks <= p.T && p.T <= (1 << 30) && (int64_t)p.B * p.Hq <= 0x7fffffff;
}

// form: B, T, Hq, Hk, D, window (1 .. T), sinks (0 .. T), then the element strides of batch, position and head of q, k, v (and dO in
// the backward pass); channels are adjacent.  A size beyond 32 bits reads as -1, which no check passes.
static SwParams sw_params(const int64_t* form, bool strides, float scale) {
  auto size = [&](int i) { return form[i] > 0x7fffffff ? -1 : (int)form[i]; };
  SwParams p{};
  p.B = size(0); p.T = size(1); p.Hq = size(2); p.Hk = size(3); p.D = size(4); p.window = size(5); p.sinks = size(6);
  if (strides) {
    p.sq = {form[7], form[8], form[9]};
    p.sk = {form[10], form[11], form[12]};
    p.sv = {form[13], form[14], form[15]};
  }
  p.scale = scale;
  return p;
}

#include "sldwin_tc.inl"
#include "sldwin_tc_bwd.inl"

}  // namespace mxb

using namespace mxb;

// The word of host memory in which the kernels of every device report a wait that ran out (null: there is no memory).  It may be
// asked for first inside a stream capture, which forbids allocations unless the thread says that this one is none of its own.
MXB_EXPORT int* mxb_report_word(void) {
  static std::mutex lock;
  static int* word = nullptr;
  std::lock_guard<std::mutex> guard(lock);
  if (!word) {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    void* at = nullptr;
    if (cudaHostAlloc(&at, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped) == cudaSuccess) {
      word = static_cast<int*>(at);
      *word = 0;
    } else cudaGetLastError();
    cudaThreadExchangeStreamCaptureMode(&mode);
  }
  return word;
}

// lse: [B, Hq, T] floats (may be null when no backward pass follows).
MXB_EXPORT int mxb_sldwin_forward(int dtype, const void* q, const void* k, const void* v, const int* valid, void* out, float* lse,
                                  const int64_t* form, float scale, int* error_flag, void* stream) {
  SwParams p = sw_params(form, true, scale);
  p.q = q; p.k = k; p.v = v; p.valid = valid; p.out = out; p.lse = lse;
  if (!sw_shape_ok(p)) return -2;
  cudaStream_t st = (cudaStream_t)stream;
  if (tc_takes(p, dtype)) {
    if (dtype == kF16) return p.D == 64 ? tc_forward<__half, 64>(p, 0, error_flag, st) : tc_forward<__half, 128>(p, 0, error_flag, st);
    return p.D == 64 ? tc_forward<__nv_bfloat16, 64>(p, 1, error_flag, st) : tc_forward<__nv_bfloat16, 128>(p, 1, error_flag, st);
  }
  if (dtype == kF32) return sw_general<float>(p, 0, st);
  if (dtype == kF16) return sw_general<__half>(p, 0, st);
  if (dtype == kBF16) return sw_general<__nv_bfloat16>(p, 0, st);
  return -1;
}

// dq: [B, T, Hq, D], dk and dv: [B, T, Hk, D], contiguous; delta: B (Hq (T + tiles) + Hk tiles) floats of workspace, tiles = ceil(T / 128); parts:
// mxb_sldwin_backward_parts floats of workspace (may be null when that is 0).
MXB_EXPORT int mxb_sldwin_backward(int dtype, const void* q, const void* k, const void* v, const int* valid, const void* o,
                                   const void* dout, const float* lse, float* delta, float* parts, void* dq, void* dk, void* dv,
                                   const int64_t* form, float scale, int* error_flag, void* stream) {
  SwParams p = sw_params(form, true, scale);
  p.q = q; p.k = k; p.v = v; p.valid = valid; p.o = o; p.dout = dout; p.lse = const_cast<float*>(lse); p.delta = delta;
  p.dq = dq; p.dk = dk; p.dv = dv;
  p.sdo = {form[16], form[17], form[18]};
  if (!sw_shape_ok(p)) return -2;
  cudaStream_t st = (cudaStream_t)stream;
  if (tc_takes(p, dtype) && tc_layout_ok(dout, p.sdo, p.B, p.T, p.Hq)) {
    if (dtype == kF16) return p.D == 64 ? tc_backward<__half, 64>(p, parts, 0, error_flag, st) : tc_backward<__half, 128>(p, parts, 0, error_flag, st);
    return p.D == 64 ? tc_backward<__nv_bfloat16, 64>(p, parts, 1, error_flag, st) : tc_backward<__nv_bfloat16, 128>(p, parts, 1, error_flag, st);
  }
  if (dtype == kF32) return sw_general<float>(p, 1, st);
  if (dtype == kF16) return sw_general<__half>(p, 1, st);
  if (dtype == kBF16) return sw_general<__nv_bfloat16>(p, 1, st);
  return -1;
}

// Floats of workspace for sums that come in parts (0 for shapes that only the general kernels take).
MXB_EXPORT int64_t mxb_sldwin_backward_parts(int dtype, const int64_t* form) {
  const SwParams p = sw_params(form, false, 1.f);
  if (!sw_shape_ok(p) || (p.D != 64 && p.D != 128) || (dtype != kF16 && dtype != kBF16)) return 0;
  return dkv_part_floats(p);
}
