// Sliding-window attention on the tcgen05 tensor cores, head sizes 64 and 128, fp16 and bf16 (included by
// sldwin_attention.cu inside namespace mxb).
//
// Products with both operands in shared memory make scores in TMEM (S = Q K^T and the like); row threads turn them into
// probabilities (or their gradients), written back to TMEM in the operand type over the scores they came from; products
// with the first operand in TMEM accumulate the outputs there.  Nothing of a score passes through shared memory.
// Tiles come by TMA out of strided [B, T, H, D] tensors (4-D maps, 128-byte swizzle, rows behind T read as zeros).
// Every wait is bounded; on expiry the CTA reports through an error word, waits for its copies, frees its TMEM and ends.

constexpr int kTcRows = 128;
constexpr uint32_t kTcHalf = kTcRows * 64 * 2;           // 16 KB: 128 rows x 64 channels, one swizzled box

__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float max3(float a, float b, float c) {      // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max2(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// 2^x on the fp32 pipes, for x <= 2^6: n + f with f in [-1/2, 1/2], 2^f by the degree-4 polynomial of least relative error with
// 2^0 = 1 (2.8e-6, far below the half step of P's type), n added to the exponent.  Arguments are cut at -127, where the bits of 1
// become those of 0: what is hidden weighs nothing, however large its value.  A NaN becomes the largest number, which is
// infinite in half types.
constexpr float kRoundMagic = 12582912.f;                 // 1.5 * 2^23: adding it rounds to a whole number in the low bits
__device__ __forceinline__ f32x2 exp2_poly(float a, float b) {
  const f32x2 x = pack_f2(max2(a, -127.f), max2(b, -127.f)), magic = pack_f2(kRoundMagic, kRoundMagic);
  const f32x2 n = add_f2(x, magic);
  const f32x2 f = add_f2(x, mul_f2(add_f2(n, pack_f2(-kRoundMagic, -kRoundMagic)), pack_f2(-1.f, -1.f)));
  f32x2 y = fma_f2(f, pack_f2(0.009582844f, 0.009582844f), pack_f2(0.055906426f, 0.055906426f));
  y = fma_f2(y, f, pack_f2(0.24024099f, 0.24024099f));
  y = fma_f2(y, f, pack_f2(0.69312418f, 0.69312418f));
  y = fma_f2(y, f, pack_f2(1.f, 1.f));
  float y0, y1, n0, n1;
  unpack_f2(y, y0, y1);
  unpack_f2(n, n0, n1);
  return pack_f2(__uint_as_float(__float_as_uint(y0) + (__float_as_uint(n0) << 23)), __uint_as_float(__float_as_uint(y1) + (__float_as_uint(n1) << 23)));
}

struct TcParams {
  const int* valid;
  const void* o;                         // backward: forward output, contiguous [B, T, Hq, D]
  const void* dout;
  SwStride sdo;
  void *out, *dq, *dk, *dv;              // contiguous
  float* lse;                            // [B, Hq, T]
  float* delta;                          // [B, Hq, T], behind it gmax
  float* gmax;                           // [B, Hq, tiles]: largest |dO| of each query tile (fp16)
  float* vmax;                           // [B, Hk, tiles]: largest |V| of each key tile (fp16)
  int B, T, Hq, Hk, window, sinks;
  int qpair;                             // 1: the two tiles of a CTA are two query heads, 0: two consecutive query tiles
  int items;                             // (sample, head or head pair) combinations
  float scale;
  int* error_flag;
};

__device__ __forceinline__ int tc_valid(const TcParams& p, int b) {
  int n = p.valid ? p.valid[b] : p.T;
  return n < 0 ? 0 : (n > p.T ? p.T : n);
}

// Tiles of kKeys keys that queries [q0, q0 + 128) of a sequence of n tokens see: the first `ns` (sinks) and those from lo to hi.
template <int kKeys>
struct KeyTiles {
  int ns, lo, hi;
  __device__ __forceinline__ KeyTiles(int q0, int n, int window, int sinks) {
    const int last = min(q0 + kTcRows, n) - 1;           // last query that is there
    if (last < q0) { ns = 0; lo = 0; hi = -1; return; }
    hi = last / kKeys;
    const int64_t first = (int64_t)q0 - window + 1;
    lo = first <= 0 ? 0 : (int)(first / kKeys);
    ns = min((min(sinks, last + 1) + kKeys - 1) / kKeys, lo);
  }
  __device__ __forceinline__ bool has(int kt) const { return kt <= hi && (kt >= lo || kt < ns); }
  __device__ __forceinline__ int count() const { return hi < lo ? 0 : ns + hi - lo + 1; }
};
typedef KeyTiles<kTcRows> KeyRange;

// Bits of 32 neighbouring keys that a query sees: keys up to `hi`, of them those behind `gone` and those up to `sink` (indexes
// relative to the first of the 32).
__device__ __forceinline__ uint32_t tc_upto(int last) { return last < 0 ? 0u : (last >= 31 ? 0xffffffffu : 0xffffffffu >> (31 - last)); }
__device__ __forceinline__ uint32_t tc_seen(int hi, int gone, int sink) { return tc_upto(hi) & (~tc_upto(gone) | tc_upto(sink)); }

// One [128 x D] tile: D / 64 boxes on one barrier.
template <int D>
__device__ __forceinline__ void tc_load_tile(uint8_t* dst, const CUtensorMap* map, int h, int t, int b, uint64_t* bar) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c) tma_load_4d(dst + c * kTcHalf, map, c * 64, h, t, b, bar);
}
// Rows [from, kRows) of a tile become zeros (a whole warp): what lies behind a sequence must not reach a sum, not even times 0.
template <int D, int kRows = kTcRows>
__device__ __forceinline__ void tc_clear_rows(uint8_t* tile, int from) {
  const int lane = threadIdx.x & 31;
  for (int c = 0; c < D / 64; ++c)
    for (uint32_t o = (uint32_t)from * 128u + lane * 16u; o < kRows * 128u; o += 512u)
      *reinterpret_cast<uint4*>(tile + c * kTcHalf + o) = make_uint4(0, 0, 0, 0);
  fence_async_smem();
  __syncwarp();
}
// One lane of a converged warp.  The warps that issue MMAs run their loops as a whole and elect a lane only around the
// instructions: their operands then stay in uniform registers, where an issue inside a one-lane branch moves each of them there
// every time (80 cycles for an MMA instead of its 45).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ int warp_uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// S[128, 128] = A B^T over D channels, both tiles row by row in shared memory (descriptors of their first boxes).
template <int D>
__device__ __forceinline__ void tc_scores(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int k = 0; k < D / 16; ++k) {
    const uint64_t o = (uint64_t)((k >> 2) * (kTcHalf >> 4) + 2 * (k & 3));
    umma(tmem_d, a + o, b + o, idesc, k > 0 ? 1u : 0u);
  }
}
// O[128, D] (+)= P[128, 128] V[128, D], k-steps kFrom .. kTo - 1 of 16.  P lies in TMEM, two values to a column, over the scores it
// was made of: a thread's share of kSteps k-steps starts where its 16 kSteps columns of scores did.  V row by row in shared memory.
template <int kSteps, int kFrom = 0, int kTo = 8>
__device__ __forceinline__ void tc_accumulate(uint32_t tmem_d, uint32_t tmem_p, uint64_t v, uint32_t idesc, uint32_t carry) {
#pragma unroll
  for (int k = kFrom; k < kTo; ++k)
    umma_ts(tmem_d, tmem_p + k / kSteps * 16 * kSteps + k % kSteps * 8, v + (uint64_t)k * 128u, idesc, k > 0 ? 1u : carry);
}

// The start of a CTA: the loading warp has set up the barriers and goes on at once, the others meet behind the TMEM allocation.
// It may be at the end of its work before they have met, so the end meets on another barrier.
template <int kThreads>
__device__ __forceinline__ void tc_start_loader() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  fence_async_smem();
  __syncwarp();
  asm volatile("bar.arrive 0, %0;" ::"n"(kThreads) : "memory");
}
template <int kThreads, int kCols = 512>
__device__ __forceinline__ uint32_t tc_start(uint32_t* slot, bool alloc) {
  if (alloc) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  asm volatile("bar.sync 0, %0;" ::"n"(kThreads) : "memory");
  tc_fence_after();
  return warp_uniform(*slot);
}
// `count` rows of `row` 16-byte words become zeros, `pitch` words from one to the next (a whole CTA).
__device__ __forceinline__ void tc_zero_rows(void* dst, int count, int row, int64_t pitch) {
  for (int e = threadIdx.x; e < count * row; e += blockDim.x) static_cast<uint4*>(dst)[e / row * pitch + e % row] = make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ void tc_finish(uint32_t tmem_base, uint32_t cols, int warp, int alloc_warp, volatile int* abort_flag, int* error_flag) {
  tc_fence_before();
  __syncwarp();
  asm volatile("barrier.sync 2, %0;" ::"r"((int)blockDim.x) : "memory");
  if (threadIdx.x == 0 && *abort_flag && error_flag) {
    *static_cast<volatile int*>(error_flag) = 1;         // host memory
    __threadfence_system();
  }
  if (warp == alloc_warp) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(cols) : "memory");
  }
}
// ------------------------------------------------------------------------------------------------ forward
// Warps 0-3 and 4-7: the softmax of query tiles 0 and 1, one thread for each row; warp 8: MMA issue and TMEM; warp 9: TMA;
// warps 10 and 11 complete the warpgroup that gives its registers to the others.
// The two tiles take turns: while one's scores are in the hands of its row threads, the tensor cores work for the other.
// 1 x 8192, 32 heads over 8 of 128, window 2048, 4 sinks, bf16: 240 us, 1.0 PFLOP/s of the 1.66 a library product reaches; tensor
// pipe 53 % active, exponential unit 40 %, issue slots 41 %: a step takes 3400 cycles, of which the four products of the two
// tiles need 2048 at the tensor cores' full rate and the row threads' chain the rest.  Four warpgroups for the two
// tiles (64 columns to a thread) took longer: the halves of a row have to agree on its maximum.  One product narrowed to 32 keys
// for a tile that only holds sinks gains 3 % at windows of 128 and costs 3 % everywhere else: the branch breaks up the
// exponentials.
// TMEM columns: S0 | S1 (128 each; P over the first 64 of its S), O0 | O1 (D each).
// With one tile (kTiles 1, heads of 64) a CTA takes half an SM and the turns are taken by two CTAs.
constexpr int kFwdStages = 2;
template <int D, int kTiles> struct FwdForm {
  static constexpr int threads = 128 * kTiles + 128, per_sm = kTiles == 1 ? 2 : 1;
  // registers: launched with 168 each, 2 x 128 x 224 + 128 x 56 of the 64512; with one tile 128 each, 128 x 200 + 128 x 56 of 32768
  static constexpr int row_regs = kTiles == 1 ? 200 : 224, other_regs = 56;
  static constexpr uint32_t tmem_o = 128 * kTiles, tmem_cols = kTiles == 1 ? 256 : 512;
  static constexpr int mma = 4 * kTiles, tma = mma + 1;            // warps
  static constexpr uint32_t tile = (D / 64) * kTcHalf;
  static constexpr uint32_t q = 0, k = kTiles * tile, v = k + kFwdStages * tile, bars = v + kFwdStages * tile;
  static constexpr uint32_t total = bars + 256 + 1024;
};
// P is kept 2^6 times its value, so that in fp16 a weight keeps its digits down to 2^-20 of the row's largest; the running
// maximum may lag behind by 8 (2^14 in all, far from the type's largest) before the output is rescaled.
constexpr float kPShift = 6.f, kMaxLag = 8.f;
constexpr int kPolyPairs = 2;

// 32 columns of a row: P = 2^(score sc + off), its sums, and its values in the operand type.  Of every 8 pairs kPolyPairs go
// through the polynomial (the MUFU pipe alone takes 1024 cycles for a tile).
template <typename T>
__device__ __forceinline__ void tc_weigh(const uint32_t* x, f32x2 sc2, f32x2 off2, f32x2 (&part)[2], uint32_t (&pk)[16]) {
#pragma unroll
  for (int c = 0; c < 32; c += 2) {
    float e0, e1;
    unpack_f2(fma_f2(pack_f2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), sc2, off2), e0, e1);
    f32x2 e;
    if ((c >> 1) * kPolyPairs % 8 < kPolyPairs) e = exp2_poly(e0, e1);
    else e = pack_f2(ex2(e0), ex2(e1));
    part[c >> 1 & 1] = add_f2(part[c >> 1 & 1], e);
    unpack_f2(e, e0, e1);
    pk[c >> 1] = pack2<T>(e0, e1);
  }
}

template <typename T, int D, int kTiles>
__global__ void __launch_bounds__(128 * kTiles + 128, kTiles == 1 ? 2 : 1)
sw_fwd_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const TcParams p, int bf16) {
  typedef FwdForm<D, kTiles> L;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::bars);
  uint64_t *q_full = bars, *k_full = bars + 2, *k_empty = bars + 4, *v_full = bars + 6, *v_empty = bars + 8, *s_full = bars + 10,
           *p_half = bars + 12, *p_full = bars + 14, *o_full = bars + 16, *patch = bars + 17, *drain = bars + 18;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 19);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  // the last tiles of causal attention are the longest: they start first
  const int tiles = p.T / kTcRows + (p.T % kTcRows ? 1 : 0);
  const bool pair = kTiles == 2 && p.qpair;
  const int qblocks = pair || kTiles == 1 ? tiles : (tiles + 1) / 2;
  const int qb = qblocks - 1 - (int)(blockIdx.x / p.items), item = blockIdx.x % p.items;
  const int hcount = pair ? p.Hq / 2 : p.Hq;
  const int b = item / hcount, h0 = (item % hcount) * (pair ? 2 : 1), hk = h0 / (p.Hq / p.Hk);
  const int n = warp_uniform(tc_valid(p, b));
  const int qa = pair || kTiles == 1 ? qb * kTcRows : qb * 2 * kTcRows;
  const int qstep = pair || kTiles == 1 ? 0 : kTcRows, hstep = pair ? 1 : 0;
  const KeyRange r0(qa, n, p.window, p.sinks), r1(qa + qstep, n, p.window, p.sinks);
  // the union of both: sinks, then [lo of the first, hi of the second]
  const int hi = max(r0.hi, r1.hi), lo = r0.lo, ns = max(r0.ns, min(r1.ns, lo));
  const int ntiles = hi < lo ? 0 : ns + hi - lo + 1;
  auto key_tile = [&](int j) { return j < ns ? j : lo + (j - ns); };

  if (ntiles == 0) {                                              // rows behind the sequence
    for (int s = 0; s < kTiles; ++s) {
      const int q0 = qa + s * qstep, h = h0 + s * hstep, rows = min(kTcRows, p.T - q0);
      if (rows <= 0 || (s == 1 && !qstep && !hstep)) continue;
      tc_zero_rows(static_cast<T*>(p.out) + (((int64_t)b * p.T + q0) * p.Hq + h) * D, rows, D / 8, (int64_t)p.Hq * D / 8);
      if (p.lse) for (int e = threadIdx.x; e < rows; e += L::threads) p.lse[((int64_t)b * p.Hq + h) * p.T + q0 + e] = INFINITY;
    }
    return;
  }
  uint32_t tmem = 0;
  if (warp == L::tma) {
    if (lane == 0) {
      for (int s = 0; s < 2; ++s) {
        mbar_init(&q_full[s], 1); mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1);
        mbar_init(&s_full[s], 1); mbar_init(&p_half[s], 4); mbar_init(&p_full[s], 4);
      }
      mbar_init(o_full, 1); mbar_init(patch, 1); mbar_init(drain, 1);
      *abort_flag = 0;
    }
    tc_start_loader<L::threads>();
  } else tmem = tc_start<L::threads, L::tmem_cols>(tmem_slot, warp == L::mma);

  if (warp == L::tma) {
    // ---------------------------------------------------------------- loads
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::other_regs));
    if (lane == 0) {
      for (int s = 0; s < kTiles; ++s) {
        if ((s ? r1 : r0).count() == 0) continue;
        mbar_expect_tx(&q_full[s], L::tile);
        tc_load_tile<D>(smem + L::q + s * L::tile, &map_q, h0 + s * hstep, qa + s * qstep, b, &q_full[s]);
      }
    }
    bool ok = true;
    int nk = 0, nv = 0;                                         // tiles asked for
    for (int j = 0; j < ntiles; ++j) {
      const int st = j % kFwdStages, kt = key_tile(j);
      const uint32_t ph = (uint32_t)(j / kFwdStages + 1) & 1u;
      if (j >= kFwdStages && !(ok = mbar_wait_warp(&k_empty[st], ph))) break;
      if (lane == 0) {
        mbar_expect_tx(&k_full[st], L::tile);
        tc_load_tile<D>(smem + L::k + st * L::tile, &map_k, hk, kt * kTcRows, b, &k_full[st]);
      }
      nk = j + 1;
      if (j >= kFwdStages && !(ok = mbar_wait_warp(&v_empty[st], ph))) break;
      const bool ends = (kt + 1) * kTcRows > n && n < p.T;      // the sequence ends inside this tile
      uint8_t* tile = smem + L::v + st * L::tile;
      if (lane == 0) {
        uint64_t* bar = ends ? patch : &v_full[st];
        mbar_expect_tx(bar, L::tile);
        tc_load_tile<D>(tile, &map_v, hk, kt * kTcRows, b, bar);
      }
      nv = ends ? j : j + 1;
      if (ends) {                                               // the last tile of the sequence: at most once
        if (!(ok = mbar_wait_warp(patch, 0))) break;
        tc_clear_rows<D>(tile, n - kt * kTcRows);
        if (lane == 0) mbar_arrive(&v_full[st]);
      }
    }
    if (!ok) {
      *abort_flag = 1;
      if (lane == 0) {
        // no copy may still be under way when the CTA's shared memory is given back
        for (int s = 0; s < 2; ++s) {
          if (s < kTiles && (s ? r1 : r0).count()) mbar_wait(&q_full[s], 0);
          if (nk > s) mbar_wait(&k_full[s], (uint32_t)((nk - 1 - s) / kFwdStages) & 1u);
          if (nv > s) mbar_wait(&v_full[s], (uint32_t)((nv - 1 - s) / kFwdStages) & 1u);
        }
      }
    }
  } else if (warp == L::mma) {
    // ---------------------------------------------------------------- products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::other_regs));
    const uint32_t id_s = make_idesc(bf16, 128, 0, 0), id_o = make_idesc(bf16, D, 0, 1);
    const uint64_t dq = make_desc(smem_u32(smem + L::q)), dk = make_desc(smem_u32(smem + L::k)),
                   dv = make_desc_mn(smem_u32(smem + L::v), kTcHalf);
    constexpr uint64_t step = L::tile >> 4;
    bool ok = true;
    uint32_t pphase = 0, started = 0;                           // bit s: of query tile s
    for (int s = 0; s < kTiles && ok; ++s) {
      const KeyRange& r = s ? r1 : r0;
      if (r.count() == 0) continue;
      ok = mbar_wait_warp(&q_full[s], 0);
      if (ok && r.has(key_tile(0))) {
        ok = mbar_wait_warp(&k_full[0], 0);
        tc_fence_after();
        if (ok && elect_one()) { tc_scores<D>(tmem + 128 * s, dq + s * step, dk, id_s); umma_commit(&s_full[s]); }
      }
    }
    if (elect_one()) umma_commit(&k_empty[0]);
    for (int j = 0; j < ntiles && ok; ++j) {
      const int kt = key_tile(j), next = j + 1 < ntiles ? key_tile(j + 1) : -1;
      const int st = j % kFwdStages, sn = (j + 1) % kFwdStages;
      const uint32_t ph = (uint32_t)(j / kFwdStages) & 1u, pn = (uint32_t)((j + 1) / kFwdStages) & 1u;
      ok = mbar_wait_warp(&v_full[st], ph);
#pragma unroll
      for (int s = 0; s < kTiles; ++s) {
        const KeyRange& r = s ? r1 : r0;
        if (ok && r.has(kt)) {
          ok = mbar_wait_warp(&p_half[s], pphase >> s & 1u);
          tc_fence_after();
          if (ok && elect_one()) tc_accumulate<8, 0, 4>(tmem + L::tmem_o + D * s, tmem + 128 * s, dv + st * step, id_o, started >> s & 1u);
          ok = ok && mbar_wait_warp(&p_full[s], pphase >> s & 1u);
          pphase ^= 1u << s;
          tc_fence_after();
          if (ok && elect_one()) tc_accumulate<8, 4, 8>(tmem + L::tmem_o + D * s, tmem + 128 * s, dv + st * step, id_o, 1u);
          started |= 1u << s;
        }
        if (ok && next >= 0 && r.has(next)) {
          if (s == 0 || !r0.has(next)) ok = mbar_wait_warp(&k_full[sn], pn);
          tc_fence_after();
          if (ok && elect_one()) {
            tc_scores<D>(tmem + 128 * s, dq + s * step, dk + sn * step, id_s);
            umma_commit(&s_full[s]);                            // complete only after P V of this tile, issued before it
          }
        }
      }
      if (ok && elect_one()) {
        umma_commit(&v_empty[st]);
        if (next >= 0) umma_commit(&k_empty[sn]);
      }
    }
    if (elect_one()) umma_commit(ok ? o_full : drain);
    if (!ok) { *abort_flag = 1; mbar_wait_warp(drain, 0); }
  } else if (warp > L::tma) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::other_regs));
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::row_regs));
    const int s = warp >> 2, quad = warp & 3;
    const int row = quad * 32 + lane;
    const int q0 = qa + s * qstep, i = q0 + row, h = h0 + s * hstep;
    const KeyRange r = s ? r1 : r0;
    const uint32_t lane_off = (uint32_t)(quad * 32) << 16;
    const uint32_t ts = tmem + 128 * s + lane_off, to = tmem + L::tmem_o + D * s + lane_off;
    const float sc = p.scale * kSwLog2e;
    float m = -INFINITY, l = 0.f;
    uint32_t phase = 0;
    bool ok = true, first = true;
    for (int j = 0; j < ntiles; ++j) {
      const int kt = key_tile(j);
      if (!r.has(kt)) continue;
      ok = mbar_wait_warp(&s_full[s], phase);
      if (!ok) break;
      phase ^= 1u;
      tc_fence_after();
      uint32_t x[128];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld32(ts + 32 * c, x + 32 * c);
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_wait_ld32(x + 32 * c);
      const int k0 = kt * kTcRows;
      const bool whole = k0 + kTcRows - 1 <= q0 && (q0 + kTcRows - 1 - k0 < p.window || k0 + kTcRows <= p.sinks);
      if (!whole) {
#pragma unroll
        for (int c0 = 0; c0 < 128; c0 += 32) {
          const uint32_t w = tc_seen(i - k0 - c0, i - p.window - k0 - c0, p.sinks - 1 - k0 - c0);
          if (__all_sync(0xffffffffu, w == 0xffffffffu)) continue;
#pragma unroll
          for (int c = 0; c < 32; ++c) if (!(w & 1u << c)) x[c0 + c] = 0xff800000u;
        }
      }
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 128; c += 2) mx[c >> 1 & 3] = max3(mx[c >> 1 & 3], __uint_as_float(x[c]), __uint_as_float(x[c + 1]));
      const float mt = max2(m, max3(max2(mx[0], mx[1]), mx[2], mx[3]) * sc);
      const bool move = !(mt <= m + kMaxLag) || m == -INFINITY;
      if (__any_sync(0xffffffffu, move)) {
        const float to_m = move ? (mt < INFINITY ? mt : NAN) : m;            // a score of NaN or +inf makes the row NaN
        const float alpha = move ? (to_m == -INFINITY ? 0.f : ex2(m - to_m)) : 1.f;
        m = to_m;
        l *= alpha;
        if (!first) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld32(to + c, o);
            tmem_wait_ld32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st32(to + c, o);
          }
        }
      }
      first = false;
      const float off = kPShift - (m == -INFINITY ? 0.f : m);
      const f32x2 sc2 = pack_f2(sc, sc), off2 = pack_f2(off, off);
      f32x2 part[2] = {0, 0};
#pragma unroll
      for (int c0 = 0; c0 < 128; c0 += 32) {
        uint32_t pk[16];
        tc_weigh<T>(x + c0, sc2, off2, part, pk);
        tmem_st16(ts + (c0 >> 1), pk);
        if (c0 == 32 || c0 == 96) {                               // the first half of P V starts under the second half's exponentials
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(c0 == 32 ? &p_half[s] : &p_full[s]);
        }
      }
      float l0, l1;
      unpack_f2(add_f2(part[0], part[1]), l0, l1);
      l += l0 + l1;
    }
    if (ok) ok = mbar_wait_warp(o_full, 0);
    if (!ok) *abort_flag = 1;
    tc_fence_after();
    if (ok) {
      const bool live = i < n && r.count() > 0;
      const float inv = live && l != 0.f ? 1.f / l : 0.f;
      T* orow = static_cast<T*>(p.out) + (((int64_t)b * p.T + i) * p.Hq + h) * D;
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        uint32_t o[32];
        if (r.count() > 0) { tmem_ld32(to + c0, o); tmem_wait_ld32(o); }
        if (i < p.T) {
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (live) {
              w.x = pack2<T>(__uint_as_float(o[v * 8]) * inv, __uint_as_float(o[v * 8 + 1]) * inv);
              w.y = pack2<T>(__uint_as_float(o[v * 8 + 2]) * inv, __uint_as_float(o[v * 8 + 3]) * inv);
              w.z = pack2<T>(__uint_as_float(o[v * 8 + 4]) * inv, __uint_as_float(o[v * 8 + 5]) * inv);
              w.w = pack2<T>(__uint_as_float(o[v * 8 + 6]) * inv, __uint_as_float(o[v * 8 + 7]) * inv);
            }
            *reinterpret_cast<uint4*>(orow + c0 + v * 8) = w;
          }
        }
      }
      if (i < p.T && p.lse) p.lse[((int64_t)b * p.Hq + h) * p.T + i] = live && l != 0.f ? m + log2f(l) - kPShift : INFINITY;
    }
  }
  tc_finish(tmem, L::tmem_cols, warp, L::mma, abort_flag, p.error_flag);
}

// ------------------------------------------------------------------------------------------------ host
// 4-D tensor map over [B, T, H, D] with element strides; box = 64 channels x 1 head x `rows` positions.
static int tc_map(CUtensorMap* map, const void* base, int bf16, int B, int T, int H, int D, SwStride s, int rows = kTcRows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return -10;
  auto bytes = [&](int64_t stride, int size) { return size == 1 ? (cuuint64_t)D * 2 : (cuuint64_t)stride * 2; };   // an axis of one entry is never walked
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)B};
  cuuint64_t strides[3] = {bytes(s.h, H), bytes(s.t, T), bytes(s.b, B)};
  cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult rc = fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base),
                         dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return rc == CUDA_SUCCESS ? 0 : -(1000 + (int)rc);
}

// TMA reads from 16-byte boundaries with strides of whole 16 bytes (below 2^40 bytes).
static bool tc_layout_ok(const void* base, const SwStride& s, int B, int T, int H) {
  auto ok = [](int64_t st, int size) { return size == 1 || (st > 0 && st % 8 == 0 && st < (1ll << 38)); };
  return (uintptr_t)base % 16 == 0 && ok(s.b, B) && ok(s.t, T) && ok(s.h, H);
}

// The tensor cores take half types, head sizes 64 and 128 and a positive scale (the running maximum is taken of the unscaled
// scores).  What they do not take runs on the general kernels.
static bool tc_takes(const SwParams& p, int dtype) {
  return (dtype == kF16 || dtype == kBF16) && (p.D == 64 || p.D == 128) && p.scale > 0.f && p.scale < 1e30f &&
         tc_layout_ok(p.q, p.sq, p.B, p.T, p.Hq) && tc_layout_ok(p.k, p.sk, p.B, p.T, p.Hk) && tc_layout_ok(p.v, p.sv, p.B, p.T, p.Hk);
}

static TcParams tc_params(const SwParams& p, int* error_flag) {
  TcParams t{};
  t.valid = p.valid; t.o = p.o; t.dout = p.dout; t.sdo = p.sdo; t.out = p.out; t.dq = p.dq; t.dk = p.dk; t.dv = p.dv;
  t.lse = p.lse; t.delta = p.delta; t.gmax = p.delta + (int64_t)p.B * p.Hq * p.T;
  t.vmax = t.gmax + (int64_t)p.B * p.Hq * ((p.T + kTcRows - 1) / kTcRows);
  t.B = p.B; t.T = p.T; t.Hq = p.Hq; t.Hk = p.Hk; t.window = p.window; t.sinks = p.sinks; t.scale = p.scale; t.error_flag = error_flag;
  return t;
}

template <typename T, int D, int kTiles>
static int tc_forward_launch(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, TcParams& t, int bf16, cudaStream_t st) {
  typedef FwdForm<D, kTiles> L;
  t.qpair = kTiles == 2 && (t.Hq / t.Hk) % 2 == 0;      // two heads over the same keys and the same rows, where heads come in pairs
  t.items = t.B * (t.qpair ? t.Hq / 2 : t.Hq);
  const int64_t tiles = (t.T + kTcRows - 1) / kTcRows;
  const int64_t grid = (t.qpair || kTiles == 1 ? tiles : (tiles + 1) / 2) * t.items;
  if (grid > 0x7fffffff) return -2;
  static unsigned long long seen = 0;
  if (auto first = first_on_device(&seen))
    if (int code = first.take(allow_smem(sw_fwd_tc_kernel<T, D, kTiles>, L::total))) return code;
  sw_fwd_tc_kernel<T, D, kTiles><<<(unsigned)grid, L::threads, L::total, st>>>(mq, mk, mv, t, bf16);
  return (int)cudaGetLastError();
}

template <typename T, int D>
static int tc_forward(const SwParams& p, int bf16, int* error_flag, cudaStream_t st) {
  CUtensorMap mq, mk, mv;
  int rc = tc_map(&mq, p.q, bf16, p.B, p.T, p.Hq, D, p.sq);
  if (!rc) rc = tc_map(&mk, p.k, bf16, p.B, p.T, p.Hk, D, p.sk);
  if (!rc) rc = tc_map(&mv, p.v, bf16, p.B, p.T, p.Hk, D, p.sv);
  if (rc) return rc;
  TcParams t = tc_params(p, error_flag);
  // Heads of 64: one query tile to a CTA and two CTAs on an SM while walks are short and their starts and ends count (64 x 128, 12
  // heads: 24 us against 39; 16 x 512: 33 and 38; 4 x 4096, 16 over 4, window 128: 75 and 82; 8 x 2048, 12 heads, no window: 114
  // and 116); for long walks two tiles that share their keys (4 x 4096, 16 over 4, no window: 218 us against 238).
  if (D == 64 && p.window <= 2048) return tc_forward_launch<T, 64, 1>(mq, mk, mv, t, bf16, st);
  return tc_forward_launch<T, D, 2>(mq, mk, mv, t, bf16, st);
}
