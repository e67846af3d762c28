// Attention of many query rows over a 4-bit cache, on tcgen05: softmax(q k^T)
// v with f16 operands that kv4_prep.cu has laid out, f32 scores, sums and
// accumulators.
//
// The query rows of one sequence and K/V head (its tokens times the G query
// heads that share the head, token-major) are cut into tiles of 256; a CTA
// takes one tile as two 128-row halves A and B that share every 128-key K/V
// tile. The roles, the TMEM layout and the order of the MMAs are those of the
// bf16 kernel (attn_tc.cu): 16 softmax warps (two per row), a TMA warp, an MMA
// warp; S_A S_B | PV_A S_A' | PV_B S_B' | ... with P written over S in TMEM.
// What differs: a row's own scale (its power of two), a row's own last key
// (causal, ragged), tiles found from row_start on the device, f16 in place of
// bf16 for all four operands (P carries 11 bits down to 2^-24 of a row's
// largest weight, see kKtLift: the output's own rounding dominates), and NaN
// scores that must reach the result.
//
// Causal tiles are started from the last (longest) to the first, so the short
// ones fill the end of the grid. With few tiles the keys are split (grid z)
// into f32 states (m, l, O) that a second kernel joins in order.
#define LTXB_LOCAL_STATUS 1  // whole-program device code (no -rdc): own status word
#include <float.h>

#include <atomic>

#include "attn_math.cuh"
#include "kv4.cuh"

namespace ltxb {

constexpr int KT_M = 128, KT_N = 128, KT_D = 128, KT_STAGES = 2;
constexpr int KT_TILE = KT_M * KT_D * 2, KT_HALF = KT_TILE / 2;
constexpr int KT_THREADS = 576;
constexpr int KT_SMEM = 1024 + 2 * KT_TILE + 2 * KT_STAGES * KT_TILE + 256 + (2 * 2 * 2 + 2 * 2) * KT_M * 4;
// P is 2^10 times p = 2^(score - reference), and a warp's references move when a
// score of one of its rows passes it by 2^5: P stays below 2^15 in f16, keeps 11
// bits while p is above 2^-24 and vanishes from 2^-35 on. (As p itself it would
// vanish from 2^-25 on: 131,072 keys there are 2^-8 of a row's weight, and all of
// its result if the heaviest key's V is small. The sum l takes the f32 values.)
// 3,520 x 28,160 tokens, 32 heads: 1,792 us, as without the factor and with moves
// at 2^8 (1,784); 2^11 and moves at 2^4 take 1,824, and 1,887 where a move is one
// row's alone: a warp has 32 rows, each of which grows now and then.
constexpr float kKtRescale = 5.0f, kKtLift = 10.0f, kKtDown = 1.0f / 1024;  // log2 units; 2^-lift
constexpr uint32_t kKtPoly = 0x2020u;  // pairs of 16 whose exp2 runs as the polynomial (2, as in the bf16 kernel)

struct KtArgs {
  Kv4View c;
  Kv4Tc t;
  const float* gate;
  __nv_bfloat16* out;
  int causal;
};

// f16 A and B, f32 accumulator
__host__ __device__ constexpr uint32_t idesc_f16_f32(int M, int N, int b_mn_major) {
  return (1u << 4) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ uint32_t kt_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// maximum that hands on a NaN
__device__ __forceinline__ float nmax3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float nmax(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <bool SPLIT>
__global__ void __launch_bounds__(KT_THREADS, 1)
    kv4_attn_tc_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                       const __grid_constant__ CUtensorMap tmV, const KtArgs args) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * KT_TILE;
  uint8_t* sV = sK + KT_STAGES * KT_TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + KT_STAGES * KT_TILE);
  uint64_t* q_full = bars + 0;
  uint64_t* k_full = bars + 1;
  uint64_t* v_full = bars + 3;
  uint64_t* k_empty = bars + 5;
  uint64_t* v_empty = bars + 7;
  uint64_t* s_full = bars + 9;
  uint64_t* p_full = bars + 11;
  uint64_t* o_done = bars + 13;
  uint64_t* p_half = bars + 15;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 17);
  int* s_tile = reinterpret_cast<int*>(bars + 18);  // sequence, tile
  float* xmax = reinterpret_cast<float*>(bars + 32);
  float* xsum = xmax + 2 * 2 * 2 * KT_M;

  const int warp = warp_id(), lane = lane_id();
  const Kv4View& c = args.c;
  const int G = args.t.G, h = blockIdx.y;

  // ---- which tile: the x-th of all sequences' tiles, each sequence's from its last to its first ----
  if (warp == 0) {
    int left = blockIdx.x, b = -1, tile = 0;
    for (int b0 = 0; b0 < c.batch && b < 0; b0 += 32) {
      int first, count, n = 0;
      if (b0 + lane < c.batch) {
        kv4_rows(c, b0 + lane, &first, &count);
        n = (int)(((long long)count * G + KV4_TC_ROWS - 1) / KV4_TC_ROWS);
      }
      int x = n;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, s);
        if (lane >= s) x += y;
      }
      const uint32_t at = __ballot_sync(0xffffffffu, left < x);
      if (at) {
        const int l = __ffs(at) - 1;
        b = b0 + l;
        tile = __shfl_sync(0xffffffffu, x, l) - 1 - left;
      } else {
        left -= __shfl_sync(0xffffffffu, x, 31);
      }
    }
    if (lane == 0) {
      s_tile[0] = b;
      s_tile[1] = tile;
    }
  }
  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 8);
      mbar_init(&p_half[i], 8);
      mbar_init(&o_done[i], 1);
    }
    fence_mbar_init();
  }
  __syncthreads();
  const int b = s_tile[0];
  if (b < 0) return;  // the grid is an upper bound on the tiles
  int first, count;
  kv4_rows(c, b, &first, &count);
  const int len = kv4_len(c, b);
  const int r0 = s_tile[1] * KV4_TC_ROWS, nrows = count * G;  // rows [r0, r0 + 256) of the sequence's nrows
  const size_t heads_rows = (size_t)c.rows * G;
  const size_t grow0 = (size_t)h * heads_rows + (size_t)first * G + r0;  // row r0 in q16 and the states
  // keys [k0, k0 + 128 nkv) for this CTA; a row sees keys 0 .. last(row)
  auto last_of = [&](int r) { return args.causal ? len - count + r / G : len - 1; };
  const int r_end = r0 + KV4_TC_ROWS < nrows ? r0 + KV4_TC_ROWS : nrows;
  int keys = last_of(r_end - 1) + 1;
  keys = keys < 0 ? 0 : keys > len ? len : keys;
  const int nall = (keys + KT_N - 1) / KT_N;
  const int nsplit = SPLIT ? args.t.splits : 1;
  const int t0 = (int)((long long)blockIdx.z * nall / nsplit);
  const int nkv = (int)((long long)(blockIdx.z + 1) * nall / nsplit) - t0;
  const size_t state0 = (size_t)blockIdx.z * c.heads * heads_rows + grow0;
  if (nkv == 0) {  // nothing to see: zero rows, or an empty state
    for (int r = warp; r < r_end - r0; r += KT_THREADS / 32) {
      if (SPLIT) {
        if (lane == 0) reinterpret_cast<float2*>(args.t.ml_part)[state0 + r] = make_float2(-FLT_MAX, 0.f);
      } else {
        const int tok = (r0 + r) / G, g = (r0 + r) - tok * G;
        reinterpret_cast<uint2*>(args.out)[(((size_t)(first + tok) * c.heads + h) * G + g) * 32 + lane] = make_uint2(0, 0);
      }
    }
    return;
  }
  if (warp == 16 && lane == 0) {
    prefetch_tmap(&tmQ);
    prefetch_tmap(&tmK);
    prefetch_tmap(&tmV);
  }
  if (warp == 17) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // without a causal order each CTA starts at its own key tile, so that the
  // resident CTAs stream different tiles (the order is fixed per CTA)
  const int kv0 = args.causal ? 0 : (int)((long long)blockIdx.x * nkv / gridDim.x);
  auto kv_tile = [&](int i) { const int t = i + kv0; return t0 + (t >= nkv ? t - nkv : t); };

  if (warp == 16) {
    // ---------------- TMA producer ----------------
    if (elect_one()) {
      const int y = (int)grow0;
      mbar_arrive_expect_tx(q_full, 2 * KT_TILE);
      tma_load_2d(sQ, &tmQ, q_full, 0, y);
      tma_load_2d(sQ + KT_HALF, &tmQ, q_full, 64, y);
      tma_load_2d(sQ + KT_TILE, &tmQ, q_full, 0, y + KT_M);
      tma_load_2d(sQ + KT_TILE + KT_HALF, &tmQ, q_full, 64, y + KT_M);
    }
    __syncwarp();
    const int base = (b * c.heads + h) * args.t.tokens;
    for (int j = 0; j < nkv; ++j) {
      const int st = j & 1;
      uint8_t* k = sK + st * KT_TILE;
      uint8_t* v = sV + st * KT_TILE;
      const int krow = base + kv_tile(j) * KT_N;
      if (!warp_wait(&k_empty[st], ((j >> 1) & 1) ^ 1, 0x311)) goto done;
      if (elect_one()) {
        mbar_arrive_expect_tx(&k_full[st], KT_TILE);
        tma_load_2d(k, &tmK, &k_full[st], 0, krow);
        tma_load_2d(k + KT_HALF, &tmK, &k_full[st], 64, krow);
      }
      __syncwarp();
      if (!warp_wait(&v_empty[st], ((j >> 1) & 1) ^ 1, 0x312)) goto done;
      if (elect_one()) {
        mbar_arrive_expect_tx(&v_full[st], KT_TILE);
        tma_load_2d(v, &tmV, &v_full[st], 0, krow);
        tma_load_2d(v + KT_HALF, &tmV, &v_full[st], 64, krow);
      }
      __syncwarp();
    }
  } else if (warp == 17) {
    // ---------------- MMA issuer ----------------
    constexpr uint32_t idesc_s = idesc_f16_f32(KT_M, KT_N, 0);
    constexpr uint32_t idesc_o = idesc_f16_f32(KT_M, KT_D, 1);
    const uint32_t qa = smem_u32(sQ);
    auto issue_s = [&](int tile, int j) {
      const uint32_t klo = desc_lo(smem_u32(sK + (j & 1) * KT_TILE), 1);
      const uint32_t qlo = desc_lo(qa + tile * KT_TILE, 1);
      const uint32_t d = tmem + tile * 128;
      if (elect_one()) {
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t off = ((kk >> 2) * KT_HALF + (kk & 3) * 32) >> 4;
          mma_ss_lo(d, qlo + off, klo + off, idesc_s, kk > 0);
        }
        umma_commit(&s_full[tile]);
      }
      __syncwarp();
    };
    // part 0: the key steps whose P is handed over first (0, 1, 4, 5), part 1: 2, 3, 6, 7
    auto issue_pv = [&](int tile, int j, int part) {
      const uint32_t vlo = desc_lo(smem_u32(sV + (j & 1) * KT_TILE), KT_HALF >> 4);
      const uint32_t d = tmem + 256 + tile * 128, pa = tmem + tile * 128;
      if (elect_one()) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int kk = (i & 1) + (i >> 1) * 4 + part * 2;
          mma_ts_lo(d, pa + kk * 8, vlo + kk * (2048 >> 4), idesc_o, (j | part | i) != 0);
        }
      }
      __syncwarp();
    };
    auto commit = [&](uint64_t* bar) {
      if (elect_one()) umma_commit(bar);
      __syncwarp();
    };
    if (!warp_wait(q_full, 0, 0x313)) goto done;
    if (!warp_wait(&k_full[0], 0, 0x314)) goto done;
    tc_fence_after();
    issue_s(0, 0);
    issue_s(1, 0);
    commit(&k_empty[0]);
    for (int j = 0; j < nkv; ++j) {
      const int st = j & 1;
      const bool more = j + 1 < nkv;
      if (!warp_wait(&v_full[st], (j >> 1) & 1, 0x315)) goto done;
      if (!warp_wait(&p_half[0], j & 1, 0x316)) goto done;
      tc_fence_after();
      issue_pv(0, j, 0);
      if (!warp_wait(&p_full[0], j & 1, 0x317)) goto done;
      tc_fence_after();
      issue_pv(0, j, 1);
      if (more) {
        if (!warp_wait(&k_full[st ^ 1], ((j + 1) >> 1) & 1, 0x318)) goto done;
        tc_fence_after();
        issue_s(0, j + 1);
      } else {
        commit(&o_done[0]);
      }
      if (!warp_wait(&p_half[1], j & 1, 0x319)) goto done;
      tc_fence_after();
      issue_pv(1, j, 0);
      if (!warp_wait(&p_full[1], j & 1, 0x31a)) goto done;
      tc_fence_after();
      issue_pv(1, j, 1);
      commit(&v_empty[st]);
      if (more) {
        issue_s(1, j + 1);
        commit(&k_empty[st ^ 1]);
      } else {
        commit(&o_done[1]);
      }
    }
  } else if (warp < 16) {
    // ---------------- softmax / correction / epilogue ----------------
    const int tile = warp >> 3, hf = (warp >> 2) & 1, qw = warp & 3;
    const int r = qw * 32 + lane;
    const uint32_t bar_id = 1 + tile * 4 + qw;
    const uint32_t lane_off = (uint32_t)(qw * 32) << 16;
    const uint32_t tS = tmem + tile * 128 + lane_off;
    const uint32_t tO = tmem + 256 + tile * 128 + lane_off + hf * 64;
    const int row = r0 + tile * KT_M + r;  // of the sequence's nrows
    const bool row_ok = row < nrows;
    const int last = row_ok ? last_of(row) : len - 1;
    const float2 kvs = args.t.kv_scale[(size_t)b * c.heads + h];
    // scores -> log2 units; kept positive (a masked score is -inf times this), at
    // a size where any product of two f16 rows still counts as zero
    const float cr = fmaxf(row_ok ? args.t.q_scale[grow0 + tile * KT_M + r] * kvs.x : 0.f, 1e-37f);
    float m_ref = -FLT_MAX, l = 0.f;
    bool ok = true;
    auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(bar_id) : "memory"); };
    // every warp of a pair passes the same barriers, also after a timed-out wait
    for (int j = 0; j < nkv; ++j) {
      if (ok && !warp_wait(&s_full[tile], j & 1, 0x31b)) ok = false;
      float* xm = xmax + (((j & 1) * 2 + tile) * 2) * KT_M;
      if (!ok) {
        xm[hf * KT_M + r] = -INFINITY;
        pair_sync();
        continue;
      }
      tc_fence_after();
      uint32_t c0[32], c1[32];
      tmem_ld32(tS + hf * 64, c0);
      tmem_ld32(tS + hf * 64 + 32, c1);
      tmem_wait_ld();
      const int valid = last + 1 - kv_tile(j) * KT_N - hf * 64;  // this row sees this warp's columns < valid
      if (__any_sync(0xffffffffu, valid < 64)) {
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          if (e >= valid) c0[e] = __float_as_uint(-INFINITY);
          if (32 + e >= valid) c1[e] = __float_as_uint(-INFINITY);
        }
      }
      float m4[4] = {__uint_as_float(c0[0]), __uint_as_float(c0[1]), __uint_as_float(c1[0]), __uint_as_float(c1[1])};
#pragma unroll
      for (int e = 1; e < 16; ++e) {
        m4[(2 * e) & 3] = nmax3(m4[(2 * e) & 3], __uint_as_float(c0[2 * e]), __uint_as_float(c0[2 * e + 1]));
        m4[(2 * e + 1) & 3] = nmax3(m4[(2 * e + 1) & 3], __uint_as_float(c1[2 * e]), __uint_as_float(c1[2 * e + 1]));
      }
      const float pm = nmax3(m4[0], m4[1], nmax(m4[2], m4[3]));
      xm[hf * KT_M + r] = pm;
      const uint64_t c2 = pk2(cr, cr);
      uint64_t acc2[2];
      uint32_t pk[16];
      auto exp_chunk = [&](const uint32_t* cv) {
        const uint64_t nm2 = pk2(kKtLift - m_ref, kKtLift - m_ref);
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          float a0, a1, p0, p1;
          up2(fma2(pk2(__uint_as_float(cv[2 * e]), __uint_as_float(cv[2 * e + 1])), c2, nm2), a0, a1);
          if ((kKtPoly >> e) & 1u) {
            ex2_poly2(a0, a1, p0, p1);
          } else {
            p0 = ex2_mufu(a0);
            p1 = ex2_mufu(a1);
          }
          acc2[e & 1] = add2(acc2[e & 1], pk2(p0, p1));
          pk[e] = kt_pack(p0, p1);
        }
      };
      auto hand_over = [&](int ch) {
        tmem_st16(tS + hf * 32 + ch * 16, pk);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(ch == 0 ? &p_half[tile] : &p_full[tile]);
        __syncwarp();  // (the next TMEM access takes the whole warp)
      };
      acc2[0] = acc2[1] = pk2(0.f, 0.f);
      exp_chunk(c0);  // with the current reference; redone below if that moves
      pair_sync();
      const float sm = nmax(pm, xm[(hf ^ 1) * KT_M + r]);
      // a NaN score (the polynomial's clamp would swallow it) stays in the row's sum
      if (sm != sm) l = sm;
      const float cm = sm * cr;
      const bool need = cm > m_ref + kKtRescale;
      if (__any_sync(0xffffffffu, need)) {
        const float m_new = fmaxf(cm, m_ref);  // every row's, once one must (a NaN leaves it)
        const float corr = ex2_mufu(m_ref - m_new);
        m_ref = m_new;
        l *= corr;
        if (j > 0) {
#pragma unroll 1
          for (int cc = 0; cc < 4; ++cc) {
            uint32_t u[16];
            tmem_ld16(tO + cc * 16, u);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(__uint_as_float(u[e]) * corr);
            tmem_st16(tO + cc * 16, u);
          }
        }
        uint32_t s0[32];
        tmem_ld32(tS + hf * 64, s0);
        tmem_wait_ld();
        if (__any_sync(0xffffffffu, valid < 32)) {
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (e >= valid) s0[e] = __float_as_uint(-INFINITY);
        }
        acc2[0] = acc2[1] = pk2(0.f, 0.f);
        exp_chunk(s0);
      }
      hand_over(0);
      exp_chunk(c1);
      hand_over(1);
      {
        float x0, x1, x2, x3;
        up2(acc2[0], x0, x1);
        up2(acc2[1], x2, x3);
        l += (x0 + x1) + (x2 + x3);
      }
    }
    // ---------------- this warp's 64 output columns ----------------
    const bool eok = ok && warp_wait(&o_done[tile], 0, 0x31c);
    float* xs = xsum + tile * 2 * KT_M;
    xs[hf * KT_M + r] = l;
    pair_sync();
    if (eok) {
      tc_fence_after();
      const float lt = l + xs[(hf ^ 1) * KT_M + r];
      // a row that sees none of this CTA's keys has only the masked scores' remains in its sum
      const bool none = last < t0 * KT_N;
      const int tok = row / G, g = row - tok * G;
      const size_t orow = ((size_t)(first + tok) * c.heads + h) * G + g;
      const float gate = (!SPLIT && row_ok && args.gate) ? args.gate[orow] : 1.0f;
      const float f = SPLIT ? kvs.y * kKtDown : none ? 0.f : gate * kvs.y / lt;  // (2^10 is in O and in lt)
      const size_t si = state0 + tile * KT_M + r;
      if (SPLIT && row_ok && hf == 0)
        reinterpret_cast<float2*>(args.t.ml_part)[si] = none ? make_float2(-FLT_MAX, 0.f) : make_float2(m_ref, lt * kKtDown);
#pragma unroll 1
      for (int cc = 0; cc < 2; ++cc) {
        uint32_t u[32];
        tmem_ld32(tO + cc * 32, u);
        tmem_wait_ld();
        if (row_ok) {
#pragma unroll
          for (int e = 0; e < 32; ++e) u[e] = none ? 0u : __float_as_uint(__uint_as_float(u[e]) * f);
          if (SPLIT) {
            uint4* op = reinterpret_cast<uint4*>(args.t.o_part + si * KT_D + hf * 64 + cc * 32);
#pragma unroll
            for (int e = 0; e < 8; ++e) op[e] = make_uint4(u[4 * e], u[4 * e + 1], u[4 * e + 2], u[4 * e + 3]);
          } else {
            uint4* op = reinterpret_cast<uint4*>(args.out + orow * KT_D + hf * 64 + cc * 32);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              op[e] = make_uint4(pack_bf16x2(__uint_as_float(u[8 * e]), __uint_as_float(u[8 * e + 1])),
                                 pack_bf16x2(__uint_as_float(u[8 * e + 2]), __uint_as_float(u[8 * e + 3])),
                                 pack_bf16x2(__uint_as_float(u[8 * e + 4]), __uint_as_float(u[8 * e + 5])),
                                 pack_bf16x2(__uint_as_float(u[8 * e + 6]), __uint_as_float(u[8 * e + 7])));
          }
        }
      }
    }
  }
done:
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// One warp per (row, head): the sum of a row's split states, in split order.
__global__ void __launch_bounds__(256) kv4_tc_join_kernel(const KtArgs a) {
  const int lane = lane_id(), G = a.t.G, H = a.c.heads * G;
  const int n = a.c.rows * H;  // below 2^31 on this path
  const size_t stride = (size_t)n;
  for (int u = blockIdx.x * 8 + warp_id(); u < n; u += gridDim.x * 8) {
    const int row = u / H, hq = u - row * H;
    const int b = kv4_row_seq(a.c, row);
    if (b < 0) continue;
    int first, count;
    kv4_rows(a.c, b, &first, &count);
    if (row < first || row >= first + count) continue;
    const size_t si = (size_t)(hq / G) * a.c.rows * G + (size_t)row * G + hq % G;
    const float2* ml = reinterpret_cast<const float2*>(a.t.ml_part);
    float top = -FLT_MAX;
#pragma unroll 8
    for (int z = 0; z < a.t.splits; ++z) top = fmaxf(top, ml[z * stride + si].x);
    float sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int z = 0; z < a.t.splits; ++z) {
      const float2 s = ml[z * stride + si];
      const float4 x = reinterpret_cast<const float4*>(a.t.o_part + (z * stride + si) * KT_D)[lane];
      if (s.y == 0.f) continue;  // an empty state: its O was not written
      const float f = ex2_mufu(s.x - top);
      sum = fmaf(s.y, f, sum);
      v.x = fmaf(x.x, f, v.x);
      v.y = fmaf(x.y, f, v.y);
      v.z = fmaf(x.z, f, v.z);
      v.w = fmaf(x.w, f, v.w);
    }
    const float f = (sum == 0.f ? 0.f : 1.f / sum) * (a.gate ? a.gate[u] : 1.f);
    reinterpret_cast<uint2*>(a.out)[(size_t)u * 32 + lane] =
        make_uint2(pack_bf16x2(v.x * f, v.y * f), pack_bf16x2(v.z * f, v.w * f));
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Upper bound on the tiles: a partial tile for every sequence that has rows
// (exact without row_start).
static long long kt_tiles(const Kv4View& c, int G) {
  if (!c.row_start) return (long long)c.batch * (((long long)c.per * G + KV4_TC_ROWS - 1) / KV4_TC_ROWS);
  return (long long)c.rows * G / KV4_TC_ROWS + (c.batch < c.rows ? c.batch : c.rows);
}

int kv4_tc_splits(const Kv4View& c, int G) {
  // In key tiles of 128 (1.65 us each here): waves of CTAs times their tiles and
  // about three more for starting and ending, and with splits the f32 states
  // (512 bytes per row, head and split, written and read at 6.5 TB/s, 1e-4 of a
  // tile). 3,520 x 28,160 tokens, 32 heads: 4 splits 1.66 ms, none 1.95; four
  // causal prompts of 1,500 tokens: none 0.13 ms, 8 splits 0.41. Tiles are
  // counted alike with and without row_start: the workspace is sized before
  // that is known.
  const long long tiles = (long long)c.rows * G / KV4_TC_ROWS + (c.batch < c.rows ? c.batch : c.rows);
  const long long units = tiles * c.heads;
  const int nkv = (c.cap + KT_N - 1) / KT_N, sms = sm_count();
  int best = 1;
  double best_t = 0;
  for (int s = 1; s <= 8 && s <= nkv; ++s) {
    const double waves = (double)((units * s + sms - 1) / sms);
    const double t = waves * ((nkv + s - 1) / s + 3) + (s > 1 ? 1e-4 * s * c.rows * G * c.heads : 0.0);
    if (s == 1 || t < best_t) {
      best = s;
      best_t = t;
    }
  }
  return best;
}

template <bool SPLIT>
static int kt_launch(const KtArgs& a, cudaStream_t st) {
  static std::atomic<bool> attr[kMaxDevices];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return set_error(LTXB_EINVAL, "kv4 attention: device %d out of range", dev);
  if (!attr[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kv4_attn_tc_kernel<SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize, KT_SMEM);
    if (e != cudaSuccess) return set_cuda_error(e, "kv4 attention: cudaFuncSetAttribute");
    attr[dev].store(true, std::memory_order_release);
  }
  const int qrows = a.c.heads * a.c.rows * a.t.G, krows = a.c.batch * a.c.heads * a.t.tokens;
  CUtensorMap tq, tk, tv;
  int rc = make_tmap_2d(&tq, a.t.q16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, KT_D, qrows, KT_D, 64, KT_M, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc) rc = make_tmap_2d(&tk, a.t.k16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, KT_D, krows, KT_D, 64, KT_N, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!rc) rc = make_tmap_2d(&tv, a.t.v16, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, KT_D, krows, KT_D, 64, KT_N, CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  kv4_attn_tc_kernel<SPLIT><<<dim3((unsigned)kt_tiles(a.c, a.t.G), a.c.heads, SPLIT ? a.t.splits : 1), KT_THREADS, KT_SMEM, st>>>(
      tq, tk, tv, a);
  launched();
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LTXB_OK : set_cuda_error(e, "kv4 attention launch");
}

int kv4_attention_tc(const Kv4View& c, const Kv4Tc& t, const float* gate, void* out, int causal, cudaStream_t st) {
  const KtArgs a{c, t, gate, static_cast<__nv_bfloat16*>(out), causal};
  if (t.splits == 1) return kt_launch<false>(a, st);
  if (int rc = kt_launch<true>(a, st)) return rc;
  const long long ctas = ((long long)c.rows * c.heads * t.G + 7) / 8, most = 8ll * sm_count();
  kv4_tc_join_kernel<<<(unsigned)(ctas < most ? ctas : most), 256, 0, st>>>(a);
  launched();
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LTXB_OK : set_cuda_error(e, "kv4 attention join launch");
}

cudaError_t kv4_attn_status(uint32_t* v, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(v, g_status, sizeof(*v));
  if (e == cudaSuccess && clear && *v) {
    const uint32_t z = 0;
    e = cudaMemcpyToSymbol(g_status, &z, sizeof(z));
  }
  return e;
}

}  // namespace ltxb
