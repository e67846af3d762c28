// out[M, N] = A[M, K] . dequant(Wq[N, K], scales)^T (+ bias) with 4-bit
// weights for tens to hundreds of rows, in one tcgen05 kernel: the weights
// (format: dq4.cu) become bf16 on their way through shared memory and never
// exist in HBM as such.
//
// D^T = W A^T: 128 weight rows are the M side of the MMA and up to 256 rows of A
// the N side, so a few dozen rows do not leave the tensor core idle on padding.
// Per step of 64 or 128 columns of K, eight warps take a tile of codes from a TMA
// ring (256 columns a stage), put code - 8 (exact in bf16: 128 + code is a bit
// pattern) times the scale (one rounding; an f32 scale as two bf16 parts) into
// a swizzled tile, and one thread issues the MMAs against A's tile, which comes
// through a ring of its own. Four warps bring the scales, two stages ahead: 32
// rows' scales are 32 cache lines, and the unpacking warps would wait for them.
// f32 sums in TMEM. Where tiles are few, the CTAs of a cluster take parts of K
// and add their f32 sums in rank order through distributed shared memory.
//
// Measured (groups of 64): 17 to 64 rows x 16,384 x 4,096 33 us, 128 rows 35, 256
// rows 43 to 47 (760 TFLOP/s), 1,001 rows 146 (920). What bounds it below 200
// rows is the unpacking and the hand-over of a step (1.3 us per 256 columns,
// whatever the rows); above, the MMAs (2 us per 256 columns of 256 rows), and
// each CTA's start and end, about 10 us. Steps of 64 columns: taking the codes
// unconverted saved 4 %, a second group of unpacking warps 7 %; four
// accumulators in turn gained nothing.
#include <atomic>

#include "attn_math.cuh"
#include "common.cuh"
#include "kernels.h"

namespace ltxb {

constexpr int DT_GROUPS = 2, DT_WARPS = 8 * DT_GROUPS;  // unpacking: groups of 8 warps take steps in turn
constexpr int DT_SCALERS = 4;  // warps that fetch scales
constexpr int DT_THREADS = 32 * (DT_WARPS + 3 + DT_SCALERS);
constexpr int DT_ROWS = 128;  // weight rows of a CTA
constexpr int DT_WBYTES = DT_ROWS * 128, DT_TILE = DT_ROWS * 128;  // a stage of codes; a bf16 tile of 64 columns
constexpr int DT_MAXM = 256, DT_MAXST = 16;  // rows of A of a CTA, slots of its ring
constexpr int DT_BARS = 1024;
constexpr int DT_SROW = 136;  // a stage's scales: [group][128 rows], padded for the stores' banks
constexpr int DT_SMEM = 227 * 1024 - DT_BARS - 1024;  // rings

struct DtArgs {
  const void* scales;
  const __nv_bfloat16* bias;
  __nv_bfloat16* out;
  int M, N, K, splits;
  int mpad;    // rows of A of a CTA, a multiple of 16
  int wslots, dslots, aslots;  // ring slots: stages of codes, steps of bf16 weights, steps of A
  int shift;   // log2(group / 32)
  int sbytes;  // of a stage's scales
  uint32_t tmem_cols;
};

__device__ __forceinline__ uint32_t bfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}

// A scale's bits, and from them a pair of equal bf16 halves; an f32 scale's
// remainder likewise in `lo`. (Taken apart a stage after the load, which would
// hold the warp up otherwise.)
template <bool BF>
__device__ __forceinline__ uint32_t dt_load(const void* s, size_t i) {
  return BF ? __ldg(reinterpret_cast<const uint16_t*>(s) + i) : __ldg(reinterpret_cast<const uint32_t*>(s) + i);
}
template <bool BF>
__device__ __forceinline__ uint32_t dt_scale(uint32_t v, uint32_t* lo) {
  *lo = 0;
  if (BF) return v | (v << 16);
  const float f = __uint_as_float(v);
  const uint32_t hi = pack_bf16x2(f, f);
  const float rest = f - bf16_lo(hi);
  *lo = pack_bf16x2(rest, rest);
  return hi;
}

// Eight codes -> eight bf16 weights in order.
template <bool BF>
__device__ __forceinline__ uint4 dt_weights(uint32_t w, uint32_t hi, uint32_t lo) {
  uint32_t e[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;  // 128 + codes i, i + 4
  uint32_t r[4] = {__byte_perm(e[0], e[1], 0x5410), __byte_perm(e[2], e[3], 0x5410), __byte_perm(e[0], e[1], 0x7632),
                   __byte_perm(e[2], e[3], 0x7632)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t d = bfma2(r[i], 0x3F803F80u, 0xC308C308u);  // - 136
    r[i] = bfma2(d, hi, BF ? 0x80008000u : bfma2(d, lo, 0x80008000u));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// (Not the .aligned form: that one needs a warp's lanes to come together, and
// they come from loops of unequal length.)
__device__ __forceinline__ void dt_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float4 dt_ld_cluster4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

// STEP: blocks of 64 columns that are handed over together.
template <bool BF, int STEP>
__global__ void __launch_bounds__(DT_THREADS, 1)
    dq4_tc_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmA, const DtArgs p) {
  extern __shared__ uint8_t dt_raw[];
  uint8_t* wring = dt_raw + (-smem_u32(dt_raw) & 1023u);
  uint8_t* tiles = wring + p.wslots * DT_WBYTES;  // bf16 weights
  uint8_t* aring = tiles + p.dslots * STEP * DT_TILE;
  const int ablock = p.mpad * 128, abytes = STEP * ablock;
  uint8_t* sring = aring + p.aslots * abytes;
  uint64_t* bars = reinterpret_cast<uint64_t*>(wring + DT_SMEM);
  uint64_t *wfull = bars, *wempty = bars + 4, *dfull = bars + 8, *done = bars + 12, *afull = bars + 14,
           *mdone = afull + DT_MAXST;  // [kb % 16]: the MMAs of block kb have read both tiles
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 13);
  const int warp = warp_id(), lane = lane_id();
  const int n0 = blockIdx.x * DT_ROWS, rank = blockIdx.y, S = p.splits, m0 = blockIdx.z * p.mpad;
  // stages of 256 columns [s0, s1), steps [kb0, kb1)
  constexpr int SPS = 4 / STEP, COLS = 64 * STEP;
  const int nst = (p.K + 255) / 256, s0 = (int)((long long)rank * nst / S), s1 = (int)((long long)(rank + 1) * nst / S);
  const int kb0 = SPS * s0, kb1 = SPS * s1 < p.K / COLS ? SPS * s1 : p.K / COLS;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&wfull[i], 1 + DT_SCALERS);
      mbar_init(&wempty[i], DT_WARPS);
      mbar_init(&dfull[i], 8);
    }
    for (int i = 0; i < DT_MAXST; ++i) {
      mbar_init(&afull[i], 1);
      mbar_init(&mdone[i], 1);
    }
    mbar_init(done, 1);
    fence_mbar_init();
  }
  if (warp == DT_WARPS + 1) tmem_alloc(tmem_slot, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool ok = true;

  if (warp < DT_WARPS) {
    // ---------------- codes -> bf16: thread (group, row, half) takes 32 of 64 columns ----------------
    const int row = threadIdx.x & 127, half = (threadIdx.x >> 7) & 1, grp = warp >> 3;
    int ds = grp, it = grp;  // slot and number of the step
    uint32_t wph = 0;
    for (int s = s0, ws = 0; s < s1 && ok; ++s) {
      ok = warp_wait(&wfull[ws], wph, 0x331);
      if (!ok) break;
      const uint8_t* srow = sring + ws * p.sbytes + row * (BF ? 4 : 8);
      const uint8_t* wrow = wring + ws * DT_WBYTES + row * 128;
      const int nk = kb1 - SPS * s < SPS ? kb1 - SPS * s : SPS;
#pragma unroll
      for (int i = 0; i < SPS / DT_GROUPS; ++i) {
        const int k = i * DT_GROUPS + grp;
        if (k >= nk) break;
        uint4 r[STEP][4];
#pragma unroll
        for (int t = 0; t < STEP; ++t) {
          const int c = 2 * (k * STEP + t) + half;  // of the stage's eight blocks of 32 columns
          const uint4 w = *reinterpret_cast<const uint4*>(wrow + ((c ^ (row & 7)) << 4));
          const uint8_t* sp = srow + (c >> p.shift) * (DT_SROW * (BF ? 4 : 8));
          const uint32_t hi = *reinterpret_cast<const uint32_t*>(sp), lo = BF ? 0u : *reinterpret_cast<const uint32_t*>(sp + 4);
          r[t][0] = dt_weights<BF>(w.x, hi, lo);
          r[t][1] = dt_weights<BF>(w.y, hi, lo);
          r[t][2] = dt_weights<BF>(w.z, hi, lo);
          r[t][3] = dt_weights<BF>(w.w, hi, lo);
        }
        if (it >= p.dslots) ok = warp_wait(&mdone[(it - p.dslots) % DT_MAXST], ((it - p.dslots) / DT_MAXST) & 1, 0x332);
        if (!ok) break;
        uint8_t* d = tiles + ds * STEP * DT_TILE + row * 128;
#pragma unroll
        for (int t = 0; t < STEP; ++t)
#pragma unroll
          for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(d + t * DT_TILE + (((half * 4 + j) ^ (row & 7)) << 4)) = r[t][j];
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&dfull[ds]);
        it += DT_GROUPS;
        if ((ds += DT_GROUPS) >= p.dslots) ds -= p.dslots;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&wempty[ws]);
      if (++ws == p.wslots) ws = 0, wph ^= 1;
    }
    if (ok) ok = warp_wait(done, 0, 0x333);
  } else if (warp == DT_WARPS) {
    // ---------------- codes ----------------
    if (lane == 0) {
      prefetch_tmap(&tmW);
      uint32_t ph = 1;
      for (int s = s0, ws = 0; s < s1 && ok; ++s) {
        ok = mbar_wait(&wempty[ws], ph, 0x334);
        if (!ok) break;
        mbar_arrive_expect_tx(&wfull[ws], DT_WBYTES);
        tma_load_2d(wring + ws * DT_WBYTES, &tmW, &wfull[ws], s * 128, n0);  // columns past K come as zeros
        if (++ws == p.wslots) ws = 0, ph ^= 1;
      }
    }
  } else if (warp == DT_WARPS + 1) {
    // ---------------- MMAs ----------------
    const uint32_t idesc = idesc_bf16_f32(DT_ROWS, p.mpad);
    const uint32_t w0 = desc_lo(smem_u32(tiles), 1), a0 = desc_lo(smem_u32(aring), 1);
    int ds = 0, as = 0;
    uint32_t ph = 0, aph = 0;
    for (int i = 0; i < kb1 - kb0; ++i) {
      ok = warp_wait(&afull[as], aph, 0x335);
      if (ok) ok = warp_wait(&dfull[ds], ph, 0x336);
      if (!ok) break;
      tc_fence_after();
      const uint32_t dw = w0 + ds * (STEP * DT_TILE >> 4), da = a0 + as * (abytes >> 4);
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < 4 * STEP; ++k)
          mma_ss_lo(tmem, dw + (k >> 2) * (DT_TILE >> 4) + 2 * (k & 3), da + (k >> 2) * (ablock >> 4) + 2 * (k & 3), idesc,
                    (i | k) != 0);
        umma_commit(&mdone[i % DT_MAXST]);
        if (i == kb1 - kb0 - 1) umma_commit(done);
      }
      __syncwarp();
      if (++ds == p.dslots) ds = 0, ph ^= 1;
      if (++as == p.aslots) as = 0, aph ^= 1;
    }
  } else if (warp == DT_WARPS + 2) {
    // ---------------- A ----------------
    if (lane == 0) {
      prefetch_tmap(&tmA);
      uint32_t as = 0;
      for (int i = 0; i < kb1 - kb0; ++i) {
        const int before = i - p.aslots;
        if (before >= 0) ok = mbar_wait(&mdone[before % DT_MAXST], (before / DT_MAXST) & 1, 0x337);
        if (!ok) break;
        mbar_arrive_expect_tx(&afull[as], abytes);
#pragma unroll
        for (int t = 0; t < STEP; ++t)  // rows past M come as zeros
          tma_load_2d(aring + as * abytes + t * ablock, &tmA, &afull[as], (kb0 + i) * COLS + t * 64, m0);
        if (++as == (uint32_t)p.aslots) as = 0;
      }
    }
  } else {
    // ---------------- scales: a quarter of a stage's a warp, loaded two stages ahead ----------------
    const int lg = 3 - p.shift, per = 1 << lg, ng = p.K >> (5 + p.shift);  // groups of a row's stage, of a row
    const int x0 = (warp - DT_WARPS - 3) * 32 + lane;
    uint32_t v[3][8];
    auto fetch = [&](int st, uint32_t (&d)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= per) break;
        const int x = x0 + i * 32 * DT_SCALERS, row = x >> lg, c = (st << lg) + (x & (per - 1));
        const int n = n0 + row < p.N ? n0 + row : p.N - 1;
        d[i] = dt_load<BF>(p.scales, (size_t)n * ng + (c < ng ? c : ng - 1));
      }
    };
    auto put = [&](uint8_t* at, const uint32_t (&d)[8]) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (i >= per) break;
        const int x = x0 + i * 32 * DT_SCALERS, row = x >> lg, c = x & (per - 1);
        uint32_t lo;
        const uint32_t hi = dt_scale<BF>(d[i], &lo);
        if (BF)
          *reinterpret_cast<uint32_t*>(at + (c * DT_SROW + row) * 4) = hi;
        else
          *reinterpret_cast<uint2*>(at + (c * DT_SROW + row) * 8) = make_uint2(hi, lo);
      }
    };
    fetch(s0, v[0]);
    fetch(s0 + 1, v[1]);
    int ws = 0;
    uint32_t ph = 1;
    for (int s = s0; s < s1 && ok; s += 3) {
#pragma unroll
      for (int u = 0; u < 3; ++u) {
        if (s + u >= s1) break;
        fetch(s + u + 2, v[(u + 2) % 3]);
        ok = warp_wait(&wempty[ws], ph, 0x338);
        if (!ok) break;
        put(sring + ws * p.sbytes, v[u]);
        __syncwarp();
        if (lane == 0) mbar_arrive(&wfull[ws]);
        if (++ws == p.wslots) ws = 0, ph ^= 1;
      }
    }
  }
  __syncwarp();
  const bool failed = __syncthreads_or(!ok);
  if (failed && threadIdx.x == 0) {  // (reported in the status word) copies under way land before the rings are given up
    const uint64_t t0 = globaltimer_ns();
    for (int i = 0; i < 4 + DT_MAXST; ++i)
      for (int ph = 0; ph < 2; ++ph)
        while (!mbar_try_wait(smem_u32(i < 4 ? &wfull[i] : &afull[i - 4]), ph) && globaltimer_ns() - t0 < 10000000ull) {
        }
  }

  // ---------------- the sums: a lane has one weight row, registers rows of A ----------------
  float* part = reinterpret_cast<float*>(wring);  // [mpad][DT_ROWS + 4], in the rings' place (all of them consumed)
  if (!failed && warp < DT_WARPS) {
    tc_fence_after();
    const int q = warp & 3, n = q * 32 + lane;
    const bool in = n0 + q * 32 < p.N;  // N is a multiple of 32
    const float bias = S == 1 && p.bias && in ? __bfloat162float(p.bias[n0 + n]) : 0.f;
    for (int cb = (warp >> 2) * 16; cb < p.mpad; cb += 4 * DT_WARPS) {
      uint32_t u[16];
      tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + cb, u);
      tmem_wait_ld();
      if (S > 1) {
#pragma unroll
        for (int e = 0; e < 16; ++e) part[(cb + e) * (DT_ROWS + 4) + n] = __uint_as_float(u[e]);
      } else if (in) {
#pragma unroll
        for (int e = 0; e < 16; e += 2) {  // two lanes trade, so that each stores two neighbouring columns of out
          const float a = __uint_as_float(u[e]) + bias, b = __uint_as_float(u[e + 1]) + bias;
          const float got = __shfl_xor_sync(0xffffffffu, lane & 1 ? a : b, 1);
          const int m = m0 + cb + e + (lane & 1);
          if (m < p.M)
            *reinterpret_cast<uint32_t*>(p.out + (size_t)m * p.N + n0 + (n & ~1)) =
                lane & 1 ? pack_bf16x2(got, b) : pack_bf16x2(a, got);
        }
      }
    }
    tc_fence_before();
  }
  if (S > 1)
    dt_cluster_sync();
  else
    __syncthreads();
  if (warp == DT_WARPS + 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
  if (S == 1) return;
  const int lp = 29 - __clz(DT_ROWS / S);  // this CTA's share: 128 / S weight rows, four a thread
  const int cols = p.M - m0 < p.mpad ? p.M - m0 : p.mpad;
  for (int i = threadIdx.x; i < cols << lp; i += DT_THREADS) {
    const int j = i >> lp, n = ((rank << lp) + (i - (j << lp))) * 4;
    if (failed || n0 + n >= p.N) continue;
    const uint32_t at = smem_u32(part + j * (DT_ROWS + 4) + n);
    float4 x[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) x[r] = r < S ? dt_ld_cluster4(at, r) : make_float4(0.f, 0.f, 0.f, 0.f);
    float4 v = x[0];
#pragma unroll
    for (int r = 1; r < 8; ++r) v.x += x[r].x, v.y += x[r].y, v.z += x[r].z, v.w += x[r].w;
    if (p.bias) {
      const uint2 bb = __ldg(reinterpret_cast<const uint2*>(p.bias + n0 + n));
      v.x += bf16_lo(bb.x), v.y += bf16_hi(bb.x), v.z += bf16_lo(bb.y), v.w += bf16_hi(bb.y);
    }
    *reinterpret_cast<uint2*>(p.out + (size_t)(m0 + j) * p.N + n0 + n) =
        make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  }
  dt_cluster_sync();  // the others have read this CTA's sums
}

// CTAs of a cluster: waves of CTAs times their stages (1.3 us and 0.7 more with
// 256 rows) and about 6 us for starting and ending, with clusters 2 more.
static int dt_splits(int units, int nst, int mpad) {
  const int sms = sm_count();
  const double per = 1.3 + 0.7 * mpad / 256;
  int best = 1;
  double best_t = 0;
  for (int s = 1; s <= 8 && 2 * s <= nst; s *= 2) {
    const double t = ((long long)units * s + sms - 1) / sms * ((nst + s - 1) / s * per + (s > 1 ? 8 : 6));
    if (s == 1 || t < best_t) best = s, best_t = t;
  }
  return best;
}

int dq4_gemm_tc(const void* A, const void* Wq, const void* scales, int scale_bf16, int group, const void* bias, void* out,
                int M, int N, int K, cudaStream_t st) {
  DtArgs p{};
  p.scales = scales;
  p.bias = static_cast<const __nv_bfloat16*>(bias);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.M = M;
  p.N = N;
  p.K = K;
  p.shift = group == 128 ? 2 : group == 64 ? 1 : 0;
  const int chunks = (M + DT_MAXM - 1) / DT_MAXM, tiles = (N + DT_ROWS - 1) / DT_ROWS;
  p.mpad = ((M + chunks - 1) / chunks + 15) / 16 * 16;
  // Steps of 128 columns as long as two of A's fit beside them: a hand-over costs
  // nearly as much for 128 columns as for 64 (128 rows x 16,384 x 4,096: 35 us
  // instead of 41, 36,864 x 4,096: 62 instead of 70).
  const bool two = p.mpad <= 128;
  p.wslots = 3;
  p.dslots = two ? 2 : 3;
  const int step = two ? 2 : 1;
  p.sbytes = (8 >> p.shift) * DT_SROW * (scale_bf16 ? 4 : 8);
  const int fit = (DT_SMEM - p.wslots * (DT_WBYTES + p.sbytes) - p.dslots * step * DT_TILE) / (step * p.mpad * 128);  // 2 or more
  p.aslots = fit < DT_MAXST ? fit : DT_MAXST;
  p.splits = dt_splits(tiles * chunks, (K + 255) / 256, p.mpad);
  p.tmem_cols = 32;
  while ((int)p.tmem_cols < p.mpad) p.tmem_cols *= 2;
  constexpr int bytes = DT_SMEM + DT_BARS + 1024;
  const int which = 2 * scale_bf16 + two;
  auto kern = which == 0 ? dq4_tc_kernel<false, 1> : which == 1 ? dq4_tc_kernel<false, 2> : which == 2 ? dq4_tc_kernel<true, 1> : dq4_tc_kernel<true, 2>;
  static std::atomic<bool> attr[4][kMaxDevices];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return set_error(LTXB_EINVAL, "dq4_gemm: device %d out of range", dev);
  cudaError_t e;
  if (!attr[which][dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return set_cuda_error(e, "dq4_gemm: cudaFuncSetAttribute");
    attr[which][dev].store(true, std::memory_order_release);
  }
  CUtensorMap tw, ta;
  if (int rc = make_tmap_2d(&tw, Wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, K / 2, N, K / 2, 128, DT_ROWS, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  if (int rc = make_tmap_2d(&ta, A, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, K, M, K, 64, p.mpad, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles, p.splits, chunks);
  cfg.blockDim = dim3(DT_THREADS);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute la[1];
  la[0].id = cudaLaunchAttributeClusterDimension;
  la[0].val.clusterDim.x = 1;
  la[0].val.clusterDim.y = p.splits;
  la[0].val.clusterDim.z = 1;
  cfg.attrs = la;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, tw, ta, p);
  launched();
  return e == cudaSuccess ? LTXB_OK : set_cuda_error(e, "dq4_gemm launch");
}

}  // namespace ltxb
