// Backward pass of the tensor-core sliding-window attention (included by sldwin_attention.cu inside namespace mxb).
//
// Two kernels, each the owner of what it accumulates, so that no result depends on the order of anything: dQ by query tiles
// (S, dP and dS K: three products per pair of tiles) and dK, dV by key tiles (S^T, dP^T, P^T dO, dS^T Q: four).  The scores
// are formed twice; sharing them would need sums of dQ across CTAs in memory.  In both, four warpgroups share each tile of
// scores (32 columns each: a thread holds its scores and their gradients in registers; two with steps of 64), so that the
// exponentials of a tile take less time than its products.
//
// What bounds it: a step of the dK, dV walk takes 2700 cycles, of which the four products need 2048 at the tensor cores' full rate
// (512 for 128 x 128 x 128) and the chain scores, probabilities, next scores the rest; then the start and the end of each CTA, with
// one CTA on an SM for heads of 128 (shared memory and TMEM are full).
// 2 x 4096, 16 heads over 4 of 128, window 1024, 4 sinks, bf16: dQ 134 us (tensor pipe active 42 %), dK and dV 147 us (61 %).
// Heads of 64 fit twice on an SM in steps of 64, so that one CTA's start and end run under the other's walk (figures at the
// choice of the step, tc_backward).
//
// Range in fp16: probabilities enter the dV product 2^14 times their value (at most 2^14, digits kept down to 2^-28), and dS is
// formed from dO scaled by a power of two f.  f brings the largest dO of the CTA's tiles into [8, 16), so that neither small
// gradients nor a loss scale push dS out of the type's range, and gives way where the values V are large: with M the largest
// |f dP| <= D * 16 * max |V|, a row's delta is a mean of its dP, so |f dS| = P |f dP - f delta| <= 2 P (1 - P) M <= M / 2, and f is
// halved until M < 2^16 (dS up to 2^15, half the type's range).  Values up to 32 (heads of 128) or 64 leave f as it is; larger ones
// take as many of the lowest digits of dS as they add at its top.  Both factors leave with the fp32 sums.  bf16 needs neither.
template <typename T> struct BwdRange { static constexpr bool scaled = false; static constexpr float shift = 0.f, unshift = 1.f; };
template <> struct BwdRange<__half> { static constexpr bool scaled = true; static constexpr float shift = 14.f, unshift = 1.f / 16384.f; };
__device__ __forceinline__ int float_exponent(float a) { return (int)((__float_as_uint(a) >> 23) & 255u) - 127; }      // a in [2^e, 2^(e + 1))
template <int D>
__device__ __forceinline__ float bwd_factor(float gmax, float vmax) {
  const int e = float_exponent(gmax), over = min(float_exponent(vmax), 15) - (D == 128 ? 4 : 5);
  return e < -30 || e > 16 ? 1.f : __uint_as_float((uint32_t)(127 + 3 - e - max(over, 0)) << 23);
}

// Largest |V| of each tile of 128 keys that are there (fp16 alone): blockIdx.x = (sample, key head, tile).  A pass over V ahead of
// the two kernels (16 x 512, 12 heads of 64: 4 us of 65); a maximum taken in the forward pass would cost calls without gradients too.
template <typename T, int D>
__global__ void __launch_bounds__(256)
sw_vmax_kernel(const TcParams p, const T* v, SwStride sv, int tiles) {
  __shared__ float red[8];
  const int kt = blockIdx.x % tiles, bh = blockIdx.x / tiles, b = bh / p.Hk, hk = bh % p.Hk;
  const int rows = min(kTcRows, tc_valid(p, b) - kt * kTcRows);
  const T* at = v + b * sv.b + (int64_t)kt * kTcRows * sv.t + hk * sv.h;
  constexpr int kEach = kTcRows * (D / 8) / 256;          // vectors of a thread, all on their way at once
  Vec16<T> x[kEach];
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int e = threadIdx.x + u * 256, row = e / (D / 8);
    if (row < rows) x[u] = ld16(at + (int64_t)row * sv.t + e % (D / 8) * 8);
  }
  float big = 0.f;
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    if ((threadIdx.x + u * 256) / (D / 8) >= rows) continue;
#pragma unroll
    for (int c = 0; c < 8; ++c) big = fmaxf(big, fabsf(Cvt<T>::to_f(x[u].v[c])));
  }
  big = warp_max(big);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = big;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < 8; ++w) big = fmaxf(big, red[w]);
    p.vmax[blockIdx.x] = big;
  }
}

// Of every 8 pairs of exponentials kBwdPoly go through the polynomial.  What belongs to hidden keys is replaced by 0 afterwards.
constexpr int kBwdPoly = 3;
__device__ __forceinline__ f32x2 bwd_exp(int pair, f32x2 y) {
  float a, b;
  unpack_f2(y, a, b);
  return pair * kBwdPoly % 8 < kBwdPoly ? exp2_poly(a, b) : pack_f2(ex2(a), ex2(b));
}
// 32 columns of a row: x = scores, y = dP  ->  x = P (f dP + neg_delta)
template <typename T>
__device__ __forceinline__ void bwd_ds(uint32_t (&x)[32], const uint32_t (&y)[32], float sc, float neg_lse, float f, float neg_delta) {
  const f32x2 sc2 = pack_f2(sc, sc), l2 = pack_f2(neg_lse, neg_lse), f2 = pack_f2(f, f), d2 = pack_f2(neg_delta, neg_delta);
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    const f32x2 pr = bwd_exp(c >> 1, fma_f2(pack_f2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), sc2, l2));
    const f32x2 dp = pack_f2(__uint_as_float(y[c]), __uint_as_float(y[c + 1]));
    float a, b;
    unpack_f2(mul_f2(pr, BwdRange<T>::scaled ? fma_f2(dp, f2, d2) : add_f2(dp, d2)), a, b);
    x[c] = __float_as_uint(a);
    x[c + 1] = __float_as_uint(b);
  }
}
// 32 columns of a key's row: x = scores  ->  x = P, with the columns' own log-sum-exps
__device__ __forceinline__ void bwd_probs(uint32_t (&x)[32], const float* lse, float sc) {
  const f32x2 sc2 = pack_f2(sc, sc);
#pragma unroll
  for (int c = 0; c < 32; c += 4) {
    const float4 l = *reinterpret_cast<const float4*>(lse + c);   // negated
    float a, b;
    unpack_f2(bwd_exp(c >> 1, fma_f2(pack_f2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), sc2, pack_f2(l.x, l.y))), a, b);
    x[c] = __float_as_uint(a);
    x[c + 1] = __float_as_uint(b);
    unpack_f2(bwd_exp((c >> 1) + 1, fma_f2(pack_f2(__uint_as_float(x[c + 2]), __uint_as_float(x[c + 3])), sc2, pack_f2(l.z, l.w))), a, b);
    x[c + 2] = __float_as_uint(a);
    x[c + 3] = __float_as_uint(b);
  }
}

// ------------------------------------------------------------------------------------------------ dQ
// TMEM columns: S of even tiles | S of odd tiles | dP (128 each) | dQ (D).  dS lies over the S it comes from: each part of the
// columns over its own.
// kKeys: keys of a step.  With 64 of them heads of 64 fit twice on an SM (shared memory, 256 TMEM columns, 320 threads).
template <int D, int kKeys> struct DqForm {
  static_assert(kKeys == 128 || D == 64, "");
  static constexpr int parts = kKeys / 32, rows_warps = 4 * parts, mma = rows_warps, tma = mma + 1, threads = 32 * (mma + 2);
  static constexpr uint32_t tmem_dp = 2 * kKeys, tmem_dq = 3 * kKeys, tmem_cols = kKeys == 64 ? 256 : 512;
  static constexpr uint32_t tile = (D / 64) * kTcHalf, ktile = tile * kKeys / 128;
  static constexpr int kst = 3, vst = 2;
  // delta: [128], then the warps' largest |dO|; sums: [parts][128] pairs, with steps of 128 keys in a stage that two steps leave unused
  static constexpr uint32_t q = 0, g = tile, k = 2 * tile, v = k + kst * ktile, delta = v + vst * ktile,
                            sums = kKeys == 64 ? delta + 1024 : k + 2 * ktile, bars = kKeys == 64 ? sums + parts * 1024 : delta + 1024;
  static constexpr uint32_t total = bars + 256;
};

template <typename T, int D, int kKeys>
__global__ void __launch_bounds__(32 * (kKeys / 8 + 2), kKeys == 64 ? 2 : 1)
sw_dq_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g, const TcParams p, int bf16) {
  typedef DqForm<D, kKeys> L;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* s_delta = reinterpret_cast<float*>(smem + L::delta);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::bars);
  uint64_t *qg_full = bars, *k_full = bars + 1, *k_empty = bars + 4, *v_full = bars + 7, *v_empty = bars + 9, *sd_full = bars + 11,
           *dp_empty = bars + 12, *ds_full = bars + 13, *done = bars + 15, *patch = bars + 16, *drain = bars + 17;
  // ds_full: two, in turn - a warp may be done with its dS of a step before another is with the step before
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 18);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (smem_u32(smem) & 1023u) {                                    // swizzled tiles lie on 1024-byte boundaries
    if (threadIdx.x == 0 && p.error_flag) *static_cast<volatile int*>(p.error_flag) = 1;
    return;
  }
  const int tiles = p.T / kTcRows + (p.T % kTcRows ? 1 : 0);
  const int qt = tiles - 1 - (int)(blockIdx.x / p.items), item = blockIdx.x % p.items;
  const int b = item / p.Hq, h = item % p.Hq, hk = h / (p.Hq / p.Hk);
  const int n = warp_uniform(tc_valid(p, b));
  const int q0 = qt * kTcRows;
  const KeyTiles<kKeys> r(q0, n, p.window, p.sinks);
  const int ntiles = r.count();
  // Rows that see few keys (those whose keys lie in 128 rows, the first query tile's among them) get delta from the sum of P dP
  // instead of from the rounded output, whose rounding is not small beside dP - delta there: such a CTA walks its tiles once for
  // the sums and once more for dQ.
  const int ahead = ntiles <= kTcRows / kKeys ? ntiles : 0, nit = ahead + ntiles;
  auto key_tile = [&](int it) {
    const int j = it < ahead ? it : it - ahead;
    return j < r.ns ? j : r.lo + (j - r.ns);
  };

  if (ntiles == 0) {                                              // rows behind the sequence
    const int rows = min(kTcRows, p.T - q0);
    tc_zero_rows(static_cast<T*>(p.dq) + (((int64_t)b * p.T + q0) * p.Hq + h) * D, rows, D / 8, (int64_t)p.Hq * D / 8);
    for (int e = threadIdx.x; e < rows; e += L::threads) p.delta[((int64_t)b * p.Hq + h) * p.T + q0 + e] = 0.f;
    if (BwdRange<T>::scaled && threadIdx.x == 0) p.gmax[((int64_t)b * p.Hq + h) * tiles + qt] = 0.f;
    return;
  }
  uint32_t tmem = 0;
  if (warp == L::tma) {
    if (lane == 0) {
      mbar_init(qg_full, 1);
      for (int s = 0; s < L::kst; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
      for (int s = 0; s < L::vst; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); }
      mbar_init(sd_full, 1); mbar_init(dp_empty, L::rows_warps); mbar_init(&ds_full[0], L::rows_warps); mbar_init(&ds_full[1], L::rows_warps); mbar_init(done, 1); mbar_init(patch, 1); mbar_init(drain, 1);
      *abort_flag = 0;
    }
    tc_start_loader<L::threads>();
  } else tmem = tc_start<L::threads, L::tmem_cols>(tmem_slot, warp == L::mma);

  if (warp == L::tma) {
    if (lane == 0) {
      mbar_expect_tx(qg_full, 2 * L::tile);
      tc_load_tile<D>(smem + L::q, &map_q, h, q0, b, qg_full);
      tc_load_tile<D>(smem + L::g, &map_g, h, q0, b, qg_full);
    }
    bool ok = true;
    int nk = 0, nv = 0;
    uint32_t patched = 0;
    for (int j = 0; j < nit; ++j) {
      const int sk = j % L::kst, sv = j % L::vst, kt = key_tile(j);
      if (j >= L::kst && !(ok = mbar_wait_warp(&k_empty[sk], (uint32_t)(j / L::kst + 1) & 1u))) break;
      const bool ends = (kt + 1) * kKeys > n && n < p.T;      // the sequence ends inside this tile: dS K must not meet what follows
      uint8_t* tile = smem + L::k + sk * L::ktile;
      if (lane == 0) {
        uint64_t* bar = ends ? patch : &k_full[sk];
        mbar_expect_tx(bar, L::ktile);
        tc_load_tile<D>(tile, &map_k, hk, kt * kKeys, b, bar);
      }
      nk = ends ? j : j + 1;
      if (ends) {
        if (!(ok = mbar_wait_warp(patch, patched++ & 1u))) break;
        tc_clear_rows<D, kKeys>(tile, n - kt * kKeys);
        if (lane == 0) mbar_arrive(&k_full[sk]);
      }
      if (j >= L::vst && !(ok = mbar_wait_warp(&v_empty[sv], (uint32_t)(j / L::vst + 1) & 1u))) break;
      if (lane == 0) {
        mbar_expect_tx(&v_full[sv], L::ktile);
        tc_load_tile<D>(smem + L::v + sv * L::ktile, &map_v, hk, kt * kKeys, b, &v_full[sv]);
      }
      nv = j + 1;
    }
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0) {                                          // no copy may still be under way at the end
        mbar_wait(qg_full, 0);
        for (int s = 0; s < L::kst; ++s) if (nk > s) mbar_wait(&k_full[s], (uint32_t)((nk - 1 - s) / L::kst) & 1u);
        for (int s = 0; s < L::vst; ++s) if (nv > s) mbar_wait(&v_full[s], (uint32_t)((nv - 1 - s) / L::vst) & 1u);
      }
    }
  } else if (warp == L::mma) {
    const uint32_t id_s = make_idesc(bf16, kKeys, 0, 0), id_o = make_idesc(bf16, D, 0, 1);
    const uint64_t dq = make_desc(smem_u32(smem + L::q)), dg = make_desc(smem_u32(smem + L::g)), dk = make_desc(smem_u32(smem + L::k)),
                   dv = make_desc(smem_u32(smem + L::v)), dkm = make_desc_mn(smem_u32(smem + L::k), kTcHalf);
    constexpr uint64_t step = L::ktile >> 4;
    bool ok = mbar_wait_warp(qg_full, 0);
    auto scores = [&](int j) {
      ok = mbar_wait_warp(&k_full[j % L::kst], (uint32_t)(j / L::kst) & 1u);
      tc_fence_after();
      if (ok && elect_one()) tc_scores<D>(tmem + kKeys * (j & 1), dq, dk + (j % L::kst) * step, id_s);
    };
    auto dprobs = [&](int j) {
      ok = mbar_wait_warp(&v_full[j % L::vst], (uint32_t)(j / L::vst) & 1u);
      tc_fence_after();
      if (ok && elect_one()) {
        tc_scores<D>(tmem + L::tmem_dp, dg, dv + (j % L::vst) * step, id_s);
        umma_commit(sd_full);
        umma_commit(&v_empty[j % L::vst]);
      }
    };
    if (ok) scores(0);
    if (ok) dprobs(0);
    if (ok && nit > 1) scores(1);
    for (int j = 0; j < nit && ok; ++j) {
      if (j + 1 < nit) {
        ok = mbar_wait_warp(dp_empty, (uint32_t)j & 1u);        // dP of this tile is in registers
        if (ok) dprobs(j + 1);
        if (!ok) break;
      }
      ok = mbar_wait_warp(&ds_full[j & 1], (uint32_t)(j >> 1) & 1u);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        if (j >= ahead)
          tc_accumulate<2, 0, kKeys / 16>(tmem + L::tmem_dq, tmem + kKeys * (j & 1), dkm + (j % L::kst) * step, id_o, j > ahead ? 1u : 0u);
        umma_commit(&k_empty[j % L::kst]);
      }
      if (j + 2 < nit) scores(j + 2);                        // over S and dS of this tile, read by the product before it
    }
    if (elect_one()) umma_commit(ok ? done : drain);
    if (!ok) { *abort_flag = 1; mbar_wait_warp(drain, 0); }
  } else {
    const int part = warp >> 2, quad = warp & 3;
    const int row = quad * 32 + lane, i = q0 + row;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const bool live = i < n;
    // delta = rowsum(dO * O) while the first products run: a few rows for each warp, whole rows side by side in a load
    constexpr int kLanes = D / 8, kRows = 32 / kLanes, kOwn = kTcRows / L::rows_warps;
    float big = 0.f;
#pragma unroll
    for (int r0 = 0; r0 < kOwn; r0 += kRows) {
      const int rr = warp * kOwn + r0 + lane / kLanes, ch = lane % kLanes * 8;
      float dot = 0.f;
      if (q0 + rr < n) {
        const Vec16<T> a = ld16(static_cast<const T*>(p.o) + (((int64_t)b * p.T + q0 + rr) * p.Hq + h) * D + ch);
        const Vec16<T> g = ld16(static_cast<const T*>(p.dout) + b * p.sdo.b + (int64_t)(q0 + rr) * p.sdo.t + h * p.sdo.h + ch);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float ge = Cvt<T>::to_f(g.v[e]);
          dot += Cvt<T>::to_f(a.v[e]) * ge;
          if (BwdRange<T>::scaled) big = fmaxf(big, fabsf(ge));
        }
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (lane % kLanes == 0) s_delta[rr] = dot;
    }
    if (BwdRange<T>::scaled) {
      big = warp_max(big);
      if (lane == 0) s_delta[128 + warp] = big;
    }
    const float lse = live ? p.lse[((int64_t)b * p.Hq + h) * p.T + i] : INFINITY;
    auto rows_meet = [] {                                         // the lanes of a warp may come one by one
      __syncwarp();
      asm volatile("barrier.sync 1, %0;" ::"n"(32 * L::rows_warps) : "memory");
    };
    rows_meet();
    float delta = s_delta[row];
    float f = 1.f;
    if (BwdRange<T>::scaled) {
#pragma unroll
      for (int w = 0; w < L::rows_warps; ++w) big = fmaxf(big, s_delta[128 + w]);
      if (threadIdx.x == 0) p.gmax[((int64_t)b * p.Hq + h) * tiles + qt] = big;
      // values of all tiles of 128 keys that the walk touches: the sinks', then the windows'
      const float* vmax = p.vmax + ((int64_t)b * p.Hk + hk) * tiles;
      const int from = r.lo * kKeys / kTcRows, to = r.hi * kKeys / kTcRows, front = min((r.ns * kKeys + kTcRows - 1) / kTcRows, from);
      float vbig = 0.f;
      for (int e = lane; e < front + to - from + 1; e += 32) vbig = fmaxf(vbig, vmax[e < front ? e : from + e - front]);
      f = bwd_factor<D>(big, warp_max(vbig));
    }
    if (part == 0 && i < p.T && !ahead) p.delta[((int64_t)b * p.Hq + h) * p.T + i] = delta;
    delta *= f;
    const float out_scale = p.scale / f;
    const float sc = p.scale * kSwLog2e;
    bool ok = true;
    float sum = 0.f, total = 0.f;
    for (int j = 0; j < nit; ++j) {
      const int kt = key_tile(j);
      ok = mbar_wait_warp(sd_full, (uint32_t)j & 1u);
      if (!ok) {
        if (j < ahead) rows_meet();                               // the warps that got through wait there
        break;
      }
      tc_fence_after();
      const uint32_t ts = tmem + kKeys * (j & 1) + 32 * part + lane_off, td = tmem + L::tmem_dp + 32 * part + lane_off;
      uint32_t x[32], y[32];
      tmem_ld32(ts, x);
      tmem_ld32(td, y);
      tmem_wait_ld32(x);
      tmem_wait_ld32(y);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(dp_empty);
      const int k0 = kt * kKeys;
      const bool whole = k0 + kKeys - 1 <= q0 && (q0 + kTcRows - 1 - k0 < p.window || k0 + kKeys <= p.sinks);
      const int base = k0 + 32 * part;
      const uint32_t seen = whole ? 0xffffffffu : tc_seen(i - base, i - p.window - base, p.sinks - 1 - base);
      if (j < ahead) {
#pragma unroll
        for (int c = 0; c < 32; ++c) {
          const bool on = seen >> c & 1u;
          const float pr = on ? ex2(fmaf(__uint_as_float(x[c]), sc, -lse)) : 0.f;
          sum = fmaf(pr, on ? __uint_as_float(y[c]) : 0.f, sum);
          total += pr;
        }
        if (j == ahead - 1) {
          float2* s_sum = reinterpret_cast<float2*>(smem + L::sums);
          s_sum[part * kTcRows + row] = make_float2(sum, total);
          rows_meet();
          sum = total = 0.f;
#pragma unroll
          for (int w = 0; w < L::parts; ++w) { sum += s_sum[w * kTcRows + row].x; total += s_sum[w * kTcRows + row].y; }
          // over the sum of the same P, which is 1 but for the rounding of the log-sum-exp: a row with one key gets that key's dP
          delta = live && total != 0.f ? __fdiv_rn(sum, total) : 0.f;
          if (part == 0 && i < p.T) p.delta[((int64_t)b * p.Hq + h) * p.T + i] = delta;
          delta *= f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ds_full[j & 1]);
        __syncwarp();
        continue;
      }
      bwd_ds<T>(x, y, sc, -lse, f, -delta);
      if (!__all_sync(0xffffffffu, seen == 0xffffffffu)) {
#pragma unroll
        for (int c = 0; c < 32; ++c) if (!(seen & 1u << c)) x[c] = 0u;
      }
      uint32_t pk[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) pk[c] = pack2<T>(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1]));
      tmem_st16(ts, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ds_full[j & 1]);
    }
    if (ok) ok = mbar_wait_warp(done, 0);
    if (!ok) *abort_flag = 1;
    tc_fence_after();
    if (ok && 32 * part < D) {
      T* dst = static_cast<T*>(p.dq) + (((int64_t)b * p.T + i) * p.Hq + h) * D + 32 * part;
      uint32_t o[32];
      tmem_ld32(tmem + L::tmem_dq + 32 * part + lane_off, o);
      tmem_wait_ld32(o);
      if (i < p.T) {
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          uint4 w = make_uint4(0, 0, 0, 0);
          if (live) {
            w.x = pack2<T>(__uint_as_float(o[v * 8]) * out_scale, __uint_as_float(o[v * 8 + 1]) * out_scale);
            w.y = pack2<T>(__uint_as_float(o[v * 8 + 2]) * out_scale, __uint_as_float(o[v * 8 + 3]) * out_scale);
            w.z = pack2<T>(__uint_as_float(o[v * 8 + 4]) * out_scale, __uint_as_float(o[v * 8 + 5]) * out_scale);
            w.w = pack2<T>(__uint_as_float(o[v * 8 + 6]) * out_scale, __uint_as_float(o[v * 8 + 7]) * out_scale);
          }
          *reinterpret_cast<uint4*>(dst + v * 8) = w;
        }
      }
    }
  }
  tc_finish(tmem, L::tmem_cols, warp, L::mma, abort_flag, p.error_flag);
}

// ------------------------------------------------------------------------------------------------ dK, dV
// A CTA owns 128 keys of one key head and walks (query head, query tile): the heads of its part of the group, the tiles whose
// windows reach its keys.  A key tile that holds sinks is seen by all later queries as well: those far tiles go to CTAs of
// their own in chunks, and where keys are few the heads of a group are split over CTAs; such parts are
// written in fp32 and added in a fixed order by a last small kernel.
// TMEM columns: S^T | dP^T (128 each) | dV | dK (D each); P^T over S^T, dS^T over dP^T, each part of the columns over its own.
struct DkvSplit {
  int tiles, near_span;                  // query tiles kt .. kt + near_span reach a key tile by their windows
  int sink_tiles, far_chunks, far_len;   // far CTAs: sink_tiles x far_chunks, of far_len query tiles
  int hsplit;                            // parts of a head group
  int part_tiles;                        // key tiles whose sums come in parts: the first part_tiles
  int items;                             // B * Hk * hsplit
  float* parts;                          // near: [hsplit][B * Hk][part_tiles], far: [hsplit][far_chunks][B * Hk][sink_tiles], each 2 x 128 x D
};
__device__ __forceinline__ float* dkv_near_part(const DkvSplit& s, int64_t bh_all, int hs, int bh, int kt, int D) {
  return s.parts + ((((int64_t)hs * bh_all + bh) * s.part_tiles + kt) * 2) * kTcRows * D;
}
__device__ __forceinline__ float* dkv_far_part(const DkvSplit& s, int64_t bh_all, int hs, int chunk, int bh, int kt, int D) {
  const int64_t near = (int64_t)s.hsplit * bh_all * s.part_tiles;
  return s.parts + ((near + (((int64_t)hs * s.far_chunks + chunk) * bh_all + bh) * s.sink_tiles + kt) * 2) * kTcRows * D;
}

// kQ: query rows of a step.  With 64 of them heads of 64 fit twice on an SM (shared memory, 256 TMEM columns, 352 threads).
template <int D, int kQ> struct DkvForm {
  static_assert(kQ == 128 || D == 64, "");
  static constexpr int parts = kQ / 32, rows_warps = 4 * parts, mma = rows_warps, tma = mma + 1, stats = mma + 2, threads = 32 * (mma + 3);
  static constexpr uint32_t tmem_dp = kQ, tmem_dv = 2 * kQ, tmem_dk = 2 * kQ + D, tmem_cols = kQ == 64 ? 256 : 512;
  static constexpr uint32_t tile = (D / 64) * kTcHalf, qtile = tile * kQ / 128;
  static constexpr int qst = 3, gst = 2;
  static constexpr uint32_t k = 0, v = tile, q = 2 * tile, g = q + qst * qtile, stat = g + gst * qtile, bars = stat + 2048;
  static constexpr uint32_t total = bars + 256;
};

template <typename T, int D, int kQ>
__global__ void __launch_bounds__(32 * (kQ / 8 + 3), kQ == 64 ? 2 : 1)
sw_dkv_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_g, const TcParams p,
                 const DkvSplit sp, int bf16) {
  typedef DkvForm<D, kQ> L;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* s_stat = reinterpret_cast<float*>(smem + L::stat);        // [2 stages][-lse kQ | -delta kQ]
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::bars);
  uint64_t *kv_full = bars, *q_full = bars + 1, *q_empty = bars + 4, *g_full = bars + 7, *g_empty = bars + 9, *st_full = bars + 11,
           *st_empty = bars + 13, *s_full = bars + 15, *dp_full = bars + 16, *p_ready = bars + 17, *ds_ready = bars + 18, *done = bars + 19,
           *patch = bars + 20, *drain = bars + 21;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  float* s_factor = reinterpret_cast<float*>(tmem_slot + 2);
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  if (smem_u32(smem) & 1023u) {                                    // swizzled tiles lie on 1024-byte boundaries
    if (threadIdx.x == 0 && p.error_flag) *static_cast<volatile int*>(p.error_flag) = 1;
    return;
  }
  const int unit = blockIdx.x / sp.items, item = blockIdx.x % sp.items;
  const int hs = item % sp.hsplit, bh = item / sp.hsplit, b = bh / p.Hk, hk = bh % p.Hk;
  const int group = p.Hq / p.Hk, heads = group / sp.hsplit, h_first = hk * group + hs * heads;
  // far chunks, all of them full, start first; near tiles follow from the first key tile, whose walks are the longest
  const int nfar = sp.sink_tiles * sp.far_chunks;
  const bool far = unit < nfar;
  const int kt = far ? unit % sp.sink_tiles : unit - nfar;
  const int chunk = far ? unit / sp.sink_tiles : 0;
  const int n = warp_uniform(tc_valid(p, b));
  const int k0 = kt * kTcRows;
  const int last_q = n > 0 ? (n - 1) / kQ : -1;                    // in steps of kQ queries
  const int from_tile = far ? kt + sp.near_span + 1 + chunk * sp.far_len : kt;
  const int qlo = from_tile * (kTcRows / kQ);
  const int qhi = (int)min((int64_t)last_q, ((int64_t)from_tile + (far ? sp.far_len : sp.near_span + 1)) * (kTcRows / kQ) - 1);
  const int per_head = max(0, qhi - qlo + 1);
  const int nit = k0 < n ? per_head * heads : 0;

  if (nit == 0) {                                                 // keys behind the sequence, or queries that a short one does not have
    if (kt < sp.part_tiles) {
      float* sum = far ? dkv_far_part(sp, (int64_t)p.B * p.Hk, hs, chunk, bh, kt, D) : dkv_near_part(sp, (int64_t)p.B * p.Hk, hs, bh, kt, D);
      tc_zero_rows(sum, 2 * kTcRows, D / 4, D / 4);
    } else {
      const int64_t at = (((int64_t)b * p.T + k0) * p.Hk + hk) * D;
      const int rows = min(kTcRows, p.T - k0);
      tc_zero_rows(static_cast<T*>(p.dk) + at, rows, D / 8, (int64_t)p.Hk * D / 8);
      tc_zero_rows(static_cast<T*>(p.dv) + at, rows, D / 8, (int64_t)p.Hk * D / 8);
    }
    return;
  }
  uint32_t tmem = 0;
  if (warp == L::tma) {
    if (lane == 0) {
      mbar_init(kv_full, 1);
      for (int s = 0; s < L::qst; ++s) { mbar_init(&q_full[s], 1); mbar_init(&q_empty[s], 1); }
      for (int s = 0; s < 2; ++s) { mbar_init(&g_full[s], 1); mbar_init(&g_empty[s], 1); mbar_init(&st_full[s], 1); mbar_init(&st_empty[s], L::rows_warps); }
      mbar_init(s_full, 1); mbar_init(dp_full, 1); mbar_init(p_ready, L::rows_warps); mbar_init(ds_ready, L::rows_warps); mbar_init(done, 1); mbar_init(patch, 1);
      mbar_init(drain, 1);
      *abort_flag = 0;
    }
    tc_start_loader<L::threads>();
  } else tmem = tc_start<L::threads, L::tmem_cols>(tmem_slot, warp == L::mma);

  if (warp == L::tma) {
    if (lane == 0) {
      mbar_expect_tx(kv_full, 2 * L::tile);
      tc_load_tile<D>(smem + L::k, &map_k, hk, k0, b, kv_full);
      tc_load_tile<D>(smem + L::v, &map_v, hk, k0, b, kv_full);
    }
    bool ok = true;
    int nq = 0, ng = 0;
    uint32_t patched = 0;
    for (int it = 0; it < nit && ok; ++it) {
      const int h = h_first + it / per_head, q0 = (qlo + it % per_head) * kQ;
      const int sq = it % L::qst, sg = it % L::gst;
      const bool ends = q0 + kQ > n && n < p.T;            // the sequence ends inside this tile
      uint8_t *tq = smem + L::q + sq * L::qtile, *tg = smem + L::g + sg * L::qtile;
      if (it >= L::qst && !(ok = mbar_wait_warp(&q_empty[sq], (uint32_t)(it / L::qst + 1) & 1u))) break;
      if (lane == 0) {
        uint64_t* bar = ends ? patch : &q_full[sq];
        mbar_expect_tx(bar, ends ? 2 * L::qtile : L::qtile);
        tc_load_tile<D>(tq, &map_q, h, q0, b, bar);
      }
      nq = ends ? it : it + 1;
      if (it >= L::gst && !(ok = mbar_wait_warp(&g_empty[sg], (uint32_t)(it / L::gst + 1) & 1u))) break;
      if (lane == 0) {
        uint64_t* bar = ends ? patch : &g_full[sg];
        if (!ends) mbar_expect_tx(bar, L::qtile);
        tc_load_tile<D>(tg, &map_g, h, q0, b, bar);
      }
      ng = ends ? it : it + 1;
      if (ends) {
        if (!(ok = mbar_wait_warp(patch, patched++ & 1u))) break;
        tc_clear_rows<D, kQ>(tq, n - q0);
        tc_clear_rows<D, kQ>(tg, n - q0);
        if (lane == 0) { mbar_arrive(&q_full[sq]); mbar_arrive(&g_full[sg]); }
      }
    }
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0) {                                          // no copy may still be under way at the end
        mbar_wait(kv_full, 0);
        for (int s = 0; s < L::qst; ++s) if (nq > s) mbar_wait(&q_full[s], (uint32_t)((nq - 1 - s) / L::qst) & 1u);
        for (int s = 0; s < L::gst; ++s) if (ng > s) mbar_wait(&g_full[s], (uint32_t)((ng - 1 - s) / L::gst) & 1u);
      }
    }
  } else if (warp == L::stats) {
    bool ok = true;
    float f = BwdRange<T>::unshift;
    if (BwdRange<T>::scaled) {
      float big = 0.f;
      for (int e = lane; e < nit; e += 32)
        big = fmaxf(big, p.gmax[((int64_t)b * p.Hq + h_first + e / per_head) * sp.tiles + (qlo + e % per_head) / (kTcRows / kQ)]);
      const float up = bwd_factor<D>(warp_max(big), p.vmax[((int64_t)b * p.Hk + hk) * sp.tiles + kt]);
      f *= up;
      if (lane == 0) s_factor[0] = up;
    }
    for (int it = 0; it < nit && ok; ++it) {
      const int h = h_first + it / per_head, q0 = (qlo + it % per_head) * kQ;
      // log-sum-exp and delta of the tile's rows; a row that is not there gets +inf: probability 0
      if (it >= 2 && !(ok = mbar_wait_warp(&st_empty[it & 1], (uint32_t)(it / 2 + 1) & 1u))) break;
      const int64_t at = ((int64_t)b * p.Hq + h) * p.T + q0;
      float* st = s_stat + (it & 1) * 2 * kQ;
#pragma unroll
      for (int e = 0; e < kQ / 32; ++e) {
        const int c = lane + 32 * e;
        st[c] = q0 + c < n ? BwdRange<T>::shift - p.lse[at + c] : -INFINITY;
        st[kQ + c] = q0 + c < n ? -p.delta[at + c] * f : 0.f;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&st_full[it & 1]);
    }
    if (!ok) *abort_flag = 1;
  } else if (warp == L::mma) {
    const uint32_t id_s = make_idesc(bf16, kQ, 0, 0), id_o = make_idesc(bf16, D, 0, 1);
    const uint64_t dk = make_desc(smem_u32(smem + L::k)), dv = make_desc(smem_u32(smem + L::v)), dq = make_desc(smem_u32(smem + L::q)),
                   dg = make_desc(smem_u32(smem + L::g)), dqm = make_desc_mn(smem_u32(smem + L::q), kTcHalf),
                   dgm = make_desc_mn(smem_u32(smem + L::g), kTcHalf);
    constexpr uint64_t step = L::qtile >> 4;
    bool ok = mbar_wait_warp(kv_full, 0);
    auto scores = [&](int it) {
      ok = mbar_wait_warp(&q_full[it % L::qst], (uint32_t)(it / L::qst) & 1u);
      tc_fence_after();
      if (ok && elect_one()) { tc_scores<D>(tmem, dk, dq + (it % L::qst) * step, id_s); umma_commit(s_full); }
    };
    auto dprobs = [&](int it) {
      ok = mbar_wait_warp(&g_full[it % L::gst], (uint32_t)(it / L::gst) & 1u);
      tc_fence_after();
      if (ok && elect_one()) { tc_scores<D>(tmem + L::tmem_dp, dv, dg + (it % L::gst) * step, id_s); umma_commit(dp_full); }
    };
    if (ok) scores(0);
    if (ok) dprobs(0);
    for (int it = 0; it < nit && ok; ++it) {
      ok = mbar_wait_warp(p_ready, (uint32_t)it & 1u);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        tc_accumulate<2, 0, kQ / 16>(tmem + L::tmem_dv, tmem, dgm + (it % L::gst) * step, id_o, it > 0 ? 1u : 0u);
        umma_commit(&g_empty[it % L::gst]);                     // dP of this tile was issued before: dO is done with
      }
      if (it + 1 < nit) scores(it + 1);
      if (!ok) break;
      ok = mbar_wait_warp(ds_ready, (uint32_t)it & 1u);
      if (!ok) break;
      tc_fence_after();
      if (elect_one()) {
        tc_accumulate<2, 0, kQ / 16>(tmem + L::tmem_dk, tmem + L::tmem_dp, dqm + (it % L::qst) * step, id_o, it > 0 ? 1u : 0u);
        umma_commit(&q_empty[it % L::qst]);
      }
      if (it + 1 < nit) dprobs(it + 1);
    }
    if (elect_one()) umma_commit(ok ? done : drain);
    if (!ok) { *abort_flag = 1; mbar_wait_warp(drain, 0); }
  } else {
    const int part = warp >> 2, quad = warp & 3;
    const int row = quad * 32 + lane, j = k0 + row;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t ts = tmem + 32 * part + lane_off, td = tmem + L::tmem_dp + 32 * part + lane_off;
    const float sc = p.scale * kSwLog2e;
    float f = 1.f;                                                // of dO in dS
    bool ok = true;
    for (int it = 0; it < nit; ++it) {
      const int q0 = (qlo + it % per_head) * kQ;
      const float* st = s_stat + (it & 1) * 2 * kQ + 32 * part;
      ok = mbar_wait_warp(&st_full[it & 1], (uint32_t)(it / 2) & 1u) && mbar_wait_warp(s_full, (uint32_t)it & 1u);
      if (!ok) break;
      tc_fence_after();
      uint32_t x[32], y[32];
      tmem_ld32(ts, x);
      tmem_wait_ld32(x);
      const bool whole = k0 + kTcRows - 1 <= q0 && (q0 + kQ - 1 - k0 < p.window || k0 + kTcRows <= p.sinks);
      bwd_probs(x, st, sc);
      if (!whole) {
        // query i = base + c sees key j when c >= j - base, and c < j - base + window or j is a sink
        const int base = q0 + 32 * part;
        const int last = j < p.sinks ? 31 : (int)min((int64_t)31, (int64_t)(j - base) + p.window - 1);
        const uint32_t w = tc_upto(last) & ~tc_upto(j - base - 1);
        if (!__all_sync(0xffffffffu, w == 0xffffffffu)) {
#pragma unroll
          for (int c = 0; c < 32; ++c) if (!(w & 1u << c)) x[c] = 0u;
        }
      }
      uint32_t pk[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) pk[c] = pack2<T>(__uint_as_float(x[2 * c]), __uint_as_float(x[2 * c + 1]));
      tmem_st16(ts, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_ready);
      ok = mbar_wait_warp(dp_full, (uint32_t)it & 1u);
      if (!ok) break;
      tc_fence_after();
      if (BwdRange<T>::scaled && it == 0) f = s_factor[0];
      const float fu = f * BwdRange<T>::unshift;
      const f32x2 fu2 = pack_f2(fu, fu);
      tmem_ld32(td, y);
      tmem_wait_ld32(y);
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const float2 d2 = *reinterpret_cast<const float2*>(st + kQ + c);
        const f32x2 dp = pack_f2(__uint_as_float(y[c]), __uint_as_float(y[c + 1])), nd = pack_f2(d2.x, d2.y);
        float a, b;
        unpack_f2(mul_f2(pack_f2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), BwdRange<T>::scaled ? fma_f2(dp, fu2, nd) : add_f2(dp, nd)), a, b);
        pk[c >> 1] = pack2<T>(a, b);
      }
      tmem_st16(td, pk);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) { mbar_arrive(ds_ready); mbar_arrive(&st_empty[it & 1]); }
    }
    if (ok) ok = mbar_wait_warp(done, 0);
    if (!ok) *abort_flag = 1;
    tc_fence_after();
    if (ok) {
      // the first half of the parts writes dK, each an equal share of the channels, the second dV
      constexpr int kEach = L::parts / 2, kWide = D / kEach;
      const int which = part / kEach, from = part % kEach * kWide;
      const float mul = which == 0 ? p.scale / f : BwdRange<T>::unshift;
      const uint32_t acc = tmem + (which == 0 ? L::tmem_dk : L::tmem_dv) + from + lane_off;
      const bool parts = kt < sp.part_tiles;
      const bool live = j < n;
      float* sum = nullptr;
      if (parts) {
        sum = far ? dkv_far_part(sp, (int64_t)p.B * p.Hk, hs, chunk, bh, kt, D) : dkv_near_part(sp, (int64_t)p.B * p.Hk, hs, bh, kt, D);
        sum += ((int64_t)which * kTcRows + row) * D + from;
      }
      T* dst = static_cast<T*>(which == 0 ? p.dk : p.dv) + (((int64_t)b * p.T + j) * p.Hk + hk) * D + from;
#pragma unroll 1
      for (int c0 = 0; c0 < kWide; c0 += 32) {
        uint32_t o[32];
        tmem_ld32(acc + c0, o);
        tmem_wait_ld32(o);
        if (parts) {
#pragma unroll
          for (int v = 0; v < 8; ++v) {
            float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
            if (live) w = make_float4(__uint_as_float(o[v * 4]) * mul, __uint_as_float(o[v * 4 + 1]) * mul, __uint_as_float(o[v * 4 + 2]) * mul,
                                      __uint_as_float(o[v * 4 + 3]) * mul);
            *reinterpret_cast<float4*>(sum + c0 + v * 4) = w;
          }
        } else if (j < p.T) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (live) {
              w.x = pack2<T>(__uint_as_float(o[v * 8]) * mul, __uint_as_float(o[v * 8 + 1]) * mul);
              w.y = pack2<T>(__uint_as_float(o[v * 8 + 2]) * mul, __uint_as_float(o[v * 8 + 3]) * mul);
              w.z = pack2<T>(__uint_as_float(o[v * 8 + 4]) * mul, __uint_as_float(o[v * 8 + 5]) * mul);
              w.w = pack2<T>(__uint_as_float(o[v * 8 + 6]) * mul, __uint_as_float(o[v * 8 + 7]) * mul);
            }
            *reinterpret_cast<uint4*>(dst + c0 + v * 8) = w;
          }
        }
      }
    }
  }
  tc_finish(tmem, L::tmem_cols, warp, L::mma, abort_flag, p.error_flag);
}

// dK and dV of the key tiles that came in parts: blockIdx.x = (sample and key head, key tile), blockIdx.y a stretch of the tile.
template <typename T, int D>
__global__ void __launch_bounds__(256)
sw_dkv_join_kernel(const TcParams p, const DkvSplit sp) {
  const int kt = blockIdx.x % sp.part_tiles, bh = blockIdx.x / sp.part_tiles, b = bh / p.Hk, hk = bh % p.Hk;
  const int64_t all = (int64_t)p.B * p.Hk;
  for (int e = blockIdx.y * 256 + threadIdx.x; e < 2 * kTcRows * D / 8; e += 256 * gridDim.y) {
    const int at = e * 8, which = at / (kTcRows * D), row = at / D % kTcRows, d = at % D, j = kt * kTcRows + row;
    if (j >= p.T) continue;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto take = [&](const float* part) {
      const float4 u = *reinterpret_cast<const float4*>(part + at), v = *reinterpret_cast<const float4*>(part + at + 4);
      acc[0] += u.x; acc[1] += u.y; acc[2] += u.z; acc[3] += u.w;
      acc[4] += v.x; acc[5] += v.y; acc[6] += v.z; acc[7] += v.w;
    };
    for (int hs = 0; hs < sp.hsplit; ++hs) {
      take(dkv_near_part(sp, all, hs, bh, kt, D));
      if (kt < sp.sink_tiles)
#pragma unroll 4
        for (int c = 0; c < sp.far_chunks; ++c) take(dkv_far_part(sp, all, hs, c, bh, kt, D));
    }
    T* dst = static_cast<T*>(which == 0 ? p.dk : p.dv) + (((int64_t)b * p.T + j) * p.Hk + hk) * D + d;
    Vec16<T> w;
#pragma unroll
    for (int q = 0; q < 8; ++q) w.v[q] = Cvt<T>::from_f(acc[q]);
    st16(dst, w);
  }
}

// ------------------------------------------------------------------------------------------------ host
static DkvSplit dkv_split(const SwParams& p) {
  DkvSplit s{};
  s.tiles = (p.T + kTcRows - 1) / kTcRows;
  s.near_span = (int)(((int64_t)kTcRows - 2 + p.window) / kTcRows);
  if (s.near_span > s.tiles - 1) s.near_span = s.tiles - 1;
  const int far = s.tiles - 1 - s.near_span;             // query tiles behind the windows of the first key tile
  // Fewer CTAs than SMs: the heads of a group are walked side by side instead of one after another.  The sums in parts cost more
  // than a device that is filled better gives once half the SMs have a CTA (16 heads over 4 of 128, window 1024, whole backward
  // pass: 1 x 4096 tokens, 128 CTAs, 164 us, two parts 175 us; 1 x 2048, 64 CTAs, two parts 94 us, four 106 us, one 116 us),
  // unless windows cut hardly any walk short: there the first keys' walks are long and the others fill in (1 x 4096, 8 heads
  // over 1 of 128, no window, 32 CTAs: one part 435 us, two 261, four 173, eight 137).
  const int group = p.Hq / p.Hk;
  const int64_t enough = 4 * (int64_t)s.near_span >= 3 * (int64_t)s.tiles ? sm_count() : sm_count() / 2;
  s.hsplit = 1;
  for (int k = 1; k <= group; ++k)
    if (group % k == 0) { s.hsplit = k; if ((int64_t)p.B * p.Hk * s.tiles * k >= enough) break; }
  s.items = p.B * p.Hk * s.hsplit;
  if (far > 0 && p.sinks > 0) {
    // Chunks as long as a window, twice as long while there are more of them than SMs: each writes 2 x 128 x D sums that are read
    // again.  1 x 32768, 16 heads over 4 of 128, window 128: backward 672 us with chunks of a window, 595 so; 8 x 4096, 12 over 4 of
    // 64: 380 and 343; up to two CTAs for each SM: 620 and 360.
    s.sink_tiles = (p.sinks + kTcRows - 1) / kTcRows;
    s.far_len = s.near_span + 1;
    while (s.far_len < far && (int64_t)s.items * s.sink_tiles * ((far + s.far_len - 1) / s.far_len) > sm_count()) s.far_len *= 2;
    s.far_chunks = (far + s.far_len - 1) / s.far_len;
  }
  s.part_tiles = s.hsplit > 1 ? s.tiles : s.sink_tiles;
  return s;
}

static int64_t dkv_part_floats(const SwParams& p) {
  const DkvSplit s = dkv_split(p);
  return ((int64_t)s.hsplit * p.B * p.Hk * s.part_tiles + (int64_t)s.hsplit * s.far_chunks * p.B * p.Hk * s.sink_tiles) * 2 * kTcRows * p.D;
}

template <typename T, int D, int kKeys>
static int dq_launch(const SwParams& p, const TcParams& t, unsigned grid, int bf16, cudaStream_t st) {
  typedef DqForm<D, kKeys> L;
  CUtensorMap mq, mk, mv, mg;
  int rc = tc_map(&mq, p.q, bf16, p.B, p.T, p.Hq, D, p.sq);
  if (!rc) rc = tc_map(&mk, p.k, bf16, p.B, p.T, p.Hk, D, p.sk, kKeys);
  if (!rc) rc = tc_map(&mv, p.v, bf16, p.B, p.T, p.Hk, D, p.sv, kKeys);
  if (!rc) rc = tc_map(&mg, p.dout, bf16, p.B, p.T, p.Hq, D, p.sdo);
  if (rc) return rc;
  static unsigned long long seen = 0;
  if (auto first = first_on_device(&seen))
    if (int code = first.take(allow_smem(sw_dq_tc_kernel<T, D, kKeys>, L::total))) return code;
  sw_dq_tc_kernel<T, D, kKeys><<<grid, L::threads, L::total, st>>>(mq, mk, mv, mg, t, bf16);
  return (int)cudaGetLastError();
}

template <typename T, int D, int kQ>
static int dkv_launch(const SwParams& p, const TcParams& t, const DkvSplit& s, unsigned grid, int bf16, cudaStream_t st) {
  typedef DkvForm<D, kQ> L;
  CUtensorMap mq, mk, mv, mg;
  int rc = tc_map(&mq, p.q, bf16, p.B, p.T, p.Hq, D, p.sq, kQ);
  if (!rc) rc = tc_map(&mk, p.k, bf16, p.B, p.T, p.Hk, D, p.sk);
  if (!rc) rc = tc_map(&mv, p.v, bf16, p.B, p.T, p.Hk, D, p.sv);
  if (!rc) rc = tc_map(&mg, p.dout, bf16, p.B, p.T, p.Hq, D, p.sdo, kQ);
  if (rc) return rc;
  static unsigned long long seen = 0;
  if (auto first = first_on_device(&seen))
    if (int code = first.take(allow_smem(sw_dkv_tc_kernel<T, D, kQ>, L::total))) return code;
  sw_dkv_tc_kernel<T, D, kQ><<<grid, L::threads, L::total, st>>>(mq, mk, mv, mg, t, s, bf16);
  return (int)cudaGetLastError();
}

template <typename T, int D>
static int tc_backward(const SwParams& p, float* parts, int bf16, int* error_flag, cudaStream_t st) {
  TcParams t = tc_params(p, error_flag);
  t.items = p.B * p.Hq;
  DkvSplit s = dkv_split(p);
  s.parts = parts;
  if (s.part_tiles && (!parts || (uintptr_t)parts % 16)) return -3;
  const int64_t gq = (int64_t)s.tiles * t.items, gk = ((int64_t)s.tiles + (int64_t)s.sink_tiles * s.far_chunks) * s.items;
  if (gq > 0x7fffffff || gk > 0x7fffffff) return -2;
  // Heads of 64: steps of 64 keys or queries and two CTAs on an SM, where there are CTAs for both.  Whole backward pass with such
  // steps for dQ, dK and dV / for dK and dV alone / for neither: 64 x 128, 12 heads 77 / 87 / 99 us, 16 x 512 91 / 105 / 116,
  // 8 x 2048 285 / 306 / 335, 4 x 4096, 16 over 4, window 128 188 / 226 / 234; 1 x 1024, 96 CTAs, dK and dV 44 against 40.
  if constexpr (BwdRange<T>::scaled) {
    sw_vmax_kernel<T, D><<<(unsigned)(s.tiles * p.B * p.Hk), 256, 0, st>>>(t, static_cast<const T*>(p.v), p.sv, s.tiles);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
  }
  int code = D == 64 && gq > sm_count() ? dq_launch<T, 64, 64>(p, t, (unsigned)gq, bf16, st) : dq_launch<T, D, 128>(p, t, (unsigned)gq, bf16, st);
  if (code) return code;
  code = D == 64 && gk > sm_count() ? dkv_launch<T, 64, 64>(p, t, s, (unsigned)gk, bf16, st) : dkv_launch<T, D, 128>(p, t, s, (unsigned)gk, bf16, st);
  if (code || !s.part_tiles) return code;
  sw_dkv_join_kernel<T, D><<<dim3((unsigned)(s.part_tiles * p.B * p.Hk), 2 * kTcRows * D / 8 / 256), 256, 0, st>>>(t, s);
  return (int)cudaGetLastError();
}
