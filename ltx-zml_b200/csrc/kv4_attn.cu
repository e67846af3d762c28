// Attention of a few query rows over the paged 4-bit K/V cache (decoding and
// short runs of tokens): softmax(q k^T * scale) v with k, v = zero + scale_kv * code.
//
// The codes go to the tensor cores as they are: a nibble alone in the lowest
// mantissa bits of an f16 is the subnormal code * 2^-24, in the next four bits
// code * 2^-20, both exact and without an offset, so one shift and four masks
// unpack eight codes into four operand registers of mma.m16n8k16, and
//   q . (z + s c)       = s sum q c + z sum q
//   sum_t p_t (z + s c) = sum (p s) c + sum p z.
// K: q's values at the first kind of place are held 16 times larger, so that
// both kinds add up in units of 2^-20 (which scores keep, see KA_UNIT). V: the two kinds are rows of their own.
// (Other forms that were measured at 131,009 tokens x 32 heads: 1 + c / 16 with
// the offset taken out by one more MMA, 205 us with 16 tokens a step; c - 8 by
// an f16 FMA a pair, 149; K through the integer MMA with q in two bytes, 136;
// K as e4m3, which runs as f16 with conversions here, 169.)
// Scale and zero thus touch only score-sized data (per group of 32 / 64 / 128).
//
// A warp takes 16 tokens of a page as the M side of the MMA, so up to 8 query
// rows (the query heads that share the K/V head, times the call's tokens) cost
// the same as one: S^T = K Q^T, then O^T = V^T P^T with P^T transposed in
// registers (movmatrix). q enters as f16 after a power of two per row (its 8
// bits stay exact down to 2^-27 of the row's largest value). p s enters as f16
// after a power of two per row, which keeps the largest p s that the row has met
// between 2^9 and 2^15: 11 significant bits down to 2^-23 of that, where bf16
// would keep 8, so the result's own rounding dominates, and nothing from 2^-34
// on. It goes by p s, not by p or s: neither a heavy token of small V nor a large
// V without weight pushes the others out. Row maxima (whole numbers) move only
// when a score passes them by 2^8, or with the powers; sums and accumulators are f32.
//
// Work is split by pages, not by sequence: all (sequence, head, row tile)
// items laid end to end are one line of pages (each item with KA_ITEM more,
// what starting and ending it costs: without them a batch of 64 sequences of 17
// to 8,192 tokens took 173 us instead of 100), each CTA takes an equal piece of
// it, its warps take the pages of an item in turn, and a second kernel joins
// the items that were cut (in page order, so results do not depend on timing).
// Lengths are read on the device only. A warp has room for one (page, head)
// block of its own: the next page's K (codes and pairs, two bulk copies)
// arrives while it works on V, the next V while it works on K, and no barrier
// joins the warps until an item ends.
//
// Measured: 131,009 tokens x 32 heads, groups of 128 (570 MB): 113 to 121 us, 4.9
// TB/s; the loads alone take 95. 64 sequences of 17 to 8,192 tokens, 32 heads over
// 8, groups of 32 (328 MB): 92 us. 8 of 900 to 2,500, 16 rows each: 24 us from L2,
// 31 without. What bounds it is the instructions of a tile (230 per 16 tokens, the
// ALU pipe 59 % busy) under 12 warps an SM; two buffers each for K and V, or 16
// warps, gained nothing. One sequence of 77 tokens: 12 us for both kernels,
// latencies from the lengths to the join.
//
// A token whose V group is stored as NaN, or whose page number is bad, makes
// every row that attends to it NaN and no others: where a page holds tokens
// that some row does not see, they are left out of the product.
#include <float.h>

#include <atomic>

#include "kv4.cuh"

namespace ltxb {

constexpr int KA_OLD = KV4_D + 4;  // floats per row of the warps' O tiles

// Scores are kept in units of 2^20 up to the exponential: a sum of q times K
// holds q (at most 2^11 in its row's unit) times 2^-20, so that no K or zero up
// to bf16's ends overflows it before the row's unit brings it back.
constexpr float KA_UNIT = 1048576.f, KA_PER = 1.f / KA_UNIT;
// The largest power of two that p takes on its way to f16 (p is at most 2^8:
// the product stays a number) and its exponent's field; where it starts.
constexpr float KA_SG_MAX = 6.646139978924579e35f;  // 2^119
constexpr int KA_SG_FIELD = 127 + 119;
// Where the largest p s of a row goes when it moves: 64 sequences of 17 to 8,192
// tokens took 107 us with 8 and 9, 121 with 11 (a move looked at every group's scale then; 92 now).
constexpr int KA_SG_TO = 9;

struct KaArgs {
  Kv4View c;
  const __nv_bfloat16* q;
  size_t ldq;
  const float* gate;   // [rows, H] or null
  __nv_bfloat16* out;  // [rows, H, 128]
  float cs;            // scale * log2(e)
  int G;               // query heads per K/V head
  int causal;
  float* part;         // [2 * CTAs] slots of R * 130 floats: O [R][128], m [R], l [R]
  int4* cut;           // [CTAs] (sequence, row tile, head, last CTA) of the item that starts here and goes on
};

__device__ __forceinline__ float ka_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
// low half = lo, high half = hi, rounded to f16
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// f16 pairs code * 2^-24 (bits 0-3 of both halves) and code * 2^-20 (bits 4-7)
__device__ __forceinline__ uint32_t code_0(uint32_t w) { return w & 0x000F000Fu; }
__device__ __forceinline__ uint32_t code_1(uint32_t w) { return w & 0x00F000F0u; }
// two-wide f32
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void un2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t f2fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t f2add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// One-dimensional bulk copy global -> shared; both ends 16-byte aligned, the
// size a multiple of 16.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// Pages [pa, pb) of (sequence b, row tile rt, head h): an item, or the part
// of it that lies in a CTA's piece of the line of pages.
struct KaSeg {
  int b, rt, h, pa, pb;
  int pages, tiles, len, first, count;  // of sequence b
  int left, lead;                       // places of the CTA's piece from here on, and those before page pa
};
constexpr int KA_ITEM = 10;  // places on the line that an item takes besides its pages

template <int R>
__device__ __forceinline__ void ka_seq(const KaArgs& a, KaSeg& k) {
  k.len = kv4_len(a.c, k.b);
  kv4_rows(a.c, k.b, &k.first, &k.count);
  k.pages = (k.len + KV4_PAGE - 1) / KV4_PAGE;
  k.tiles = k.pages > 0 ? (k.count * a.G + R - 1) / R : 0;
}
// pb from the places that are left; pb <= pa: none for a page
__device__ __forceinline__ void ka_end(KaSeg& k) {
  const int n = k.left - k.lead;
  k.pb = k.pages - k.pa < n ? k.pages : k.pa + n;
}
// The next item of the CTA's piece; false behind its last.
template <int R>
__device__ __forceinline__ bool ka_next(const KaArgs& a, KaSeg& k) {
  k.left -= k.lead + k.pb - k.pa;
  if (k.left <= KA_ITEM) return false;
  k.lead = KA_ITEM;
  k.pa = 0;
  if (++k.h >= a.c.heads) {
    k.h = 0;
    if (++k.rt >= k.tiles) {
      k.rt = 0;
      do {
        if (++k.b >= a.c.batch) return false;
        ka_seq<R>(a, k);
      } while (k.tiles == 0);
    }
  }
  ka_end(k);
  return true;
}

constexpr int KA_WARPS = 4, KA_THREADS = KA_WARPS * 32;
template <int R>
struct KaSmem {
  float o[KA_WARPS][R][KA_OLD];  // the warps' O tiles, joined when an item ends
  float m[KA_WARPS][R], l[KA_WARPS][R];
  uint64_t kfull[KA_WARPS], vfull[KA_WARPS];
  int good[KA_WARPS][2];  // the page number was valid (of even and odd pages)
  // the CTA's item and each warp's loading place: here and not in registers,
  // which the accumulators need
  KaSeg at;
  KaSeg ls[KA_WARPS];
  int lp[KA_WARPS];
  int scan[KA_WARPS], items[KA_WARPS];
  int found[4];
};
template <int R>
constexpr int ka_smem_bytes(int ng) {
  return KA_WARPS * kv4_block(ng) + (int)sizeof(KaSmem<R>) + 128;
}
// CTAs an SM, of 168 registers a thread: with four and 128 registers 131,009
// tokens x 32 heads took 125 us instead of 118
constexpr int KA_PER_SM = 3;

template <int NG, int R>
__global__ void __launch_bounds__(KA_THREADS, KA_PER_SM) kv4_attn_kernel(const KaArgs a) {
  constexpr int NT = R / 8, BLK = kv4_block(NG), NW = KA_WARPS, THREADS = KA_THREADS;
  constexpr int MT = R == 8 ? 4 : 2;        // tiles of 16 tokens whose scores are held at once
  constexpr int PAIRS = KV4_PAGE * 4 * NG;  // bytes of a page's K or V pairs
  extern __shared__ __align__(128) uint8_t ka_raw[];
  // (aligned by an offset: through an integer the pointer would lose its address space)
  uint8_t* ring = ka_raw + (-smem_u32(ka_raw) & 127u);
  KaSmem<R>& sm = *reinterpret_cast<KaSmem<R>*>(ring + NW * BLK);
  const int tid = threadIdx.x, warp = warp_id(), lane = lane_id(), g = lane >> 2, cq = lane & 3;
  const int Hq = a.c.heads * a.G;

  if (tid == 0) {
    for (int i = 0; i < NW; ++i) {
      mbar_init(&sm.kfull[i], 1);
      mbar_init(&sm.vfull[i], 1);
    }
    fence_mbar_init();
    sm.found[0] = -1;
  }
  // ---- this CTA's piece of the line of pages (the host has made sure that it is shorter than 2^31) ----
  auto units = [&](int b, int* items) -> int {
    KaSeg k;
    k.b = b;
    ka_seq<R>(a, k);
    *items = k.tiles * a.c.heads;
    return k.tiles > 0 ? (k.pages + KA_ITEM) * *items : 0;
  };
  int mine = 0, items = 0, n0 = 0;  // n0: pages of the thread's first sequence
  for (int b = tid; b < a.c.batch; b += THREADS) {
    int it;
    const int n = units(b, &it);
    if (b == tid) n0 = n;
    mine += n;
    items += it;
  }
  int upto = mine;  // inclusive over the warp's lanes
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, upto, s);
    if (lane >= s) upto += y;
    items += __shfl_xor_sync(0xffffffffu, items, s);
  }
  if (lane == 31) sm.scan[warp] = upto;
  if (lane == 0) sm.items[warp] = items;
  __syncthreads();
  const int total = sm.scan[0] + sm.scan[1] + sm.scan[2] + sm.scan[3];
  items = sm.items[0] + sm.items[1] + sm.items[2] + sm.items[3];
  // a CTA for every item, or at least a page for every warp of a CTA, within the grid
  int ctas = (total - items * KA_ITEM + NW - 1) / NW;
  if (ctas < items) ctas = items;
  if (ctas > (int)gridDim.x) ctas = gridDim.x;
  // sequences without tokens: their rows attend to nothing and are zero
  for (int b = blockIdx.x; b < a.c.batch; b += gridDim.x) {
    int first, count;
    kv4_rows(a.c, b, &first, &count);
    if (count > 0 && kv4_len(a.c, b) == 0)
      for (long long i = tid; i < (long long)count * Hq * (KV4_D / 8); i += THREADS)
        reinterpret_cast<uint4*>(a.out + (size_t)first * Hq * KV4_D)[i] = make_uint4(0, 0, 0, 0);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if ((int)blockIdx.x >= ctas) {
    if (tid == 0) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }
  // pieces of `each` pages, the first `longer` of one page more
  const int each = total / ctas, longer = total - each * ctas;
  const int u0 = (int)blockIdx.x * each + ((int)blockIdx.x < longer ? (int)blockIdx.x : longer);
  const int u1 = u0 + each + ((int)blockIdx.x < longer ? 1 : 0);
  {  // the sequence that holds u0
    auto found = [&](int b, int d) {
      KaSeg k;
      k.b = b;
      ka_seq<R>(a, k);
      const int item = d / (k.pages + KA_ITEM);
      sm.found[0] = b;
      sm.found[1] = item / a.c.heads;
      sm.found[2] = item % a.c.heads;
      sm.found[3] = d - item * (k.pages + KA_ITEM);
    };
    int base = 0;
    if (a.c.batch <= THREADS) {  // a thread has one sequence, whose place the first scan gives
      for (int w = 0; w < warp; ++w) base += sm.scan[w];
      const int x = base + upto;
      if (n0 > 0 && u0 >= x - n0 && u0 < x) found(tid, u0 - (x - n0));
    } else {
      for (int b0 = 0; base <= u0 && b0 < a.c.batch; b0 += THREADS) {
        int it;
        const int n = b0 + tid < a.c.batch ? units(b0 + tid, &it) : 0;
        int x = n;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, s);
          if (lane >= s) x += y;
        }
        __syncthreads();
        if (lane == 31) sm.scan[warp] = x;
        __syncthreads();
        for (int w = 0; w < warp; ++w) x += sm.scan[w];
        x += base;
        if (n > 0 && u0 >= x - n && u0 < x) found(b0 + tid, u0 - (x - n));
        base += sm.scan[0] + sm.scan[1] + sm.scan[2] + sm.scan[3];
      }
    }
    __syncthreads();
    if (sm.found[0] < 0) {  // only if the lengths changed while this ran
      if (tid == 0) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    if (tid < NW) {
      KaSeg k;
      k.b = sm.found[0];
      k.rt = sm.found[1];
      k.h = sm.found[2];
      const int d = sm.found[3] - KA_ITEM;
      k.pa = d > 0 ? d : 0;
      k.lead = d > 0 ? 0 : -d;
      k.left = u1 - u0;
      ka_seq<R>(a, k);
      ka_end(k);
      sm.ls[tid] = k;
      sm.lp[tid] = k.pa + tid;
      if (tid == 0) sm.at = k;
    }
    __syncthreads();
    if (sm.at.pb <= sm.at.pa) {  // a short piece, all of it before an item's first page
      if (tid == 0) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
  }

  // ---- loads (lane 0): this warp's pages in order; K of the next page, then its V ----
  uint8_t* sk = ring + warp * BLK;       // K codes, K pairs
  uint8_t* sv = sk + KV4_VOFF + PAIRS;   // V codes, V pairs
  int sent = 0, np = -1;         // np: the number of the next page (its table entry is fetched a page ahead)
  bool more = true;
  const uint8_t* src = nullptr;  // the block whose V is still to be fetched; null: a bad page
  auto find = [&]() {            // the next page of this warp
    KaSeg& ls = sm.ls[warp];
    int lp = sm.lp[warp];
    while (lp >= ls.pb) {
      if (!ka_next<R>(a, ls)) {
        more = false;
        return;
      }
      lp = ls.pa + warp;
    }
    sm.lp[warp] = lp + NW;
    const size_t i = (size_t)ls.b * a.c.max_pages + lp;
    np = a.c.table ? __ldg(a.c.table + i) : (int)i;
  };
  auto send_k = [&]() {
    if (!more) return;
    const bool good = (unsigned)np < (unsigned)a.c.n_pages;
    src = good ? kv4_block_at(a.c, np, sm.ls[warp].h, BLK) : nullptr;
    sm.good[warp][sent & 1] = good;
    if (good) {
      mbar_arrive_expect_tx(&sm.kfull[warp], KV4_VOFF + PAIRS);
      bulk_load(sk, src, KV4_VOFF, &sm.kfull[warp]);
      bulk_load(sk + KV4_VOFF, src + KV4_KPAIR, PAIRS, &sm.kfull[warp]);
    } else {
      report_index(LTXB_SITE_KV4_PAGE);
      mbar_arrive(&sm.kfull[warp]);
    }
    ++sent;
    find();
  };
  auto send_v = [&]() {
    if (src) {
      mbar_arrive_expect_tx(&sm.vfull[warp], KV4_VOFF + PAIRS);
      bulk_load(sv, src + KV4_VOFF, KV4_VOFF, &sm.vfull[warp]);
      bulk_load(sv + KV4_VOFF, src + kv4_vpair(NG), PAIRS, &sm.vfull[warp]);
    } else {
      mbar_arrive(&sm.vfull[warp]);
    }
  };
  if (lane == 0) {
    find();
    send_k();
    if (sent > 0) send_v();
  }
  __syncwarp();

  bool ok = true, failed = false, go = true;
  int used = 0;  // pages this warp has done
  while (go) {
    const KaSeg& at = sm.at;
    // ---- a new item: its query rows as f16, sums of q, nothing accumulated ----
    uint32_t qf[NT][16];  // [j][nibbles 0 4, 1 5, 2 6, 3 7 of the lane's word]
    uint64_t qs[NT][NG], rs[NT], l[NT], zs[NT][NG];  // rows 2 c, 2 c + 1: sum q; softmax scale * log2(e) * the row's unit; ...
    float o[NT][8][4], m[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = at.rt * R + t * 8 + g, tok = r / a.G;
      const bool has = tok < at.count;
      const __nv_bfloat16* qp =
          a.q + (size_t)(at.first + (has ? tok : 0)) * a.ldq + (at.h * a.G + (has ? r - tok * a.G : 0)) * KV4_D + 8 * cq;
      uint4 w[4];
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[j] = has ? __ldg(reinterpret_cast<const uint4*>(qp + 32 * j)) : make_uint4(0, 0, 0, 0);
        const uint32_t ws[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = fabsf(bf16_lo(ws[i])), y = fabsf(bf16_hi(ws[i]));
          top = !(x < INFINITY) || !(y < INFINITY) ? NAN : top == top ? fmaxf(top, fmaxf(x, y)) : top;
        }
      }
#pragma unroll
      for (int i = 1; i < 4; i <<= 1) {
        const float y = __shfl_xor_sync(0xffffffffu, top, i);
        top = top != top || y != y ? NAN : fmaxf(top, y);
      }
      int field = 264 - (int)((__float_as_uint(top) >> 23) & 255u);  // the largest value into [2^10, 2^11)
      field = field < 1 ? 1 : field > 249 ? 249 : field;
      const float f = __uint_as_float((uint32_t)field << 23), f16 = 16.f * f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        qf[t][4 * j + 0] = pack_f16x2(bf16_lo(w[j].x) * f16, bf16_lo(w[j].z) * f16);  // dims 0, 4 of the eight
        qf[t][4 * j + 1] = pack_f16x2(bf16_hi(w[j].x) * f, bf16_hi(w[j].z) * f);      // 1, 5
        qf[t][4 * j + 2] = pack_f16x2(bf16_lo(w[j].y) * f16, bf16_lo(w[j].w) * f16);  // 2, 6
        qf[t][4 * j + 3] = pack_f16x2(bf16_hi(w[j].y) * f, bf16_hi(w[j].w) * f);      // 3, 7
      }
      const float back = top == top ? __uint_as_float((uint32_t)(254 - field) << 23) * a.cs : NAN;  // not finite: a NaN row
      rs[t] = f2(__shfl_sync(0xffffffffu, back, 8 * cq), __shfl_sync(0xffffffffu, back, 8 * cq + 4));
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int rc = at.rt * R + t * 8 + 2 * cq + e;
        lim[t][e] = a.causal ? at.len - at.count + rc / a.G : at.len - 1;  // last key the row sees
        m[t][e] = -FLT_MAX * KA_PER;
      }
      l[t] = 0;
#pragma unroll
      for (int x = 0; x < 8; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[t][x][e] = 0.f;
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int y = 0; y < 8 / NG; ++y) {  // rows of 1/16 and 1
          const int i = 2 * (x * (8 / NG) + y);
          mma_f16(s, 0x2C002C00u, 0x2C002C00u, 0x3C003C00u, 0x3C003C00u, qf[t][i], qf[t][i + 1]);
        }
        qs[t][x] = f2(KA_PER * s[0], KA_PER * s[1]);
        zs[t][x] = 0;
      }
    }
    // keys that every row of the tile sees: up to the first row's
    const int all = a.causal ? at.len - at.count + (at.rt * R) / a.G : at.len - 1;
    uint64_t sg[NT];  // rows 2 c, 2 c + 1: p s enters the product as p * sg * s
#pragma unroll
    for (int t = 0; t < NT; ++t) sg[t] = f2(KA_SG_MAX, KA_SG_MAX);
    const int npg = at.pb - at.pa > warp ? (at.pb - at.pa - warp + NW - 1) / NW : 0;
    for (int k = 0; k < npg; ++k, ++used) {
      if (ok) ok = warp_wait(&sm.kfull[warp], used & 1, 0x301);
      if (!ok) break;
      const int page0 = (at.pa + warp + k * NW) * KV4_PAGE;
      const bool good = sm.good[warp][used & 1] != 0;
      const bool whole = good && page0 + KV4_PAGE - 1 <= all;
#pragma unroll 1
      for (int h = 0; h < 4 / MT; ++h) {
        // ---- S^T: MT tiles of 16 tokens x R rows; a lane has tokens g, g + 8, rows 2 c, 2 c + 1 ----
        uint64_t s[MT][NT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int t0 = (h * MT + mt) * 16 + g;
          const uint4 k0 = *reinterpret_cast<const uint4*>(sk + t0 * 64 + cq * 16);
          const uint4 k1 = *reinterpret_cast<const uint4*>(sk + (t0 + 8) * 64 + cq * 16);
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
          const uint32_t* kp = reinterpret_cast<const uint32_t*>(sk + KV4_VOFF) + t0 * NG;
#pragma unroll
          for (int x = 0; x < NG; ++x) {
            float acc[NT][4];
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.f;
#pragma unroll
            for (int y = 0; y < 4 / NG; ++y) {
              const int j = x * (4 / NG) + y;
              const uint32_t a0 = w0[j], a1 = w1[j], b0 = w0[j] >> 8, b1 = w1[j] >> 8;
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                mma_f16(acc[t], code_0(a0), code_0(a1), code_1(a0), code_1(a1), qf[t][4 * j], qf[t][4 * j + 1]);
                mma_f16(acc[t], code_0(b0), code_0(b1), code_1(b0), code_1(b1), qf[t][4 * j + 2], qf[t][4 * j + 3]);
              }
            }
            const uint32_t p0 = kp[x], p1 = kp[8 * NG + x];
            const float s0 = bf16_lo(p0), s1 = bf16_lo(p1), z0 = bf16_hi(p0), z1 = bf16_hi(p1);  // (codes count 2^-20)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const uint64_t y0 = x ? f2fma(f2(z0, z0), qs[t][x], s[mt][t][0]) : f2mul(f2(z0, z0), qs[t][x]);
              const uint64_t y1 = x ? f2fma(f2(z1, z1), qs[t][x], s[mt][t][1]) : f2mul(f2(z1, z1), qs[t][x]);
              s[mt][t][0] = f2fma(f2(s0, s0), f2(acc[t][0], acc[t][1]), y0);
              s[mt][t][1] = f2fma(f2(s1, s1), f2(acc[t][2], acc[t][3]), y1);
            }
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            s[mt][t][0] = f2mul(s[mt][t][0], rs[t]);
            s[mt][t][1] = f2mul(s[mt][t][1], rs[t]);
          }
        }
        __syncwarp();
        if (lane == 0 && (h + 1) * MT == 4) send_k();  // the next page's (its V follows when this page's has been read)
        __syncwarp();
        if (h == 0) ok = warp_wait(&sm.vfull[warp], used & 1, 0x302);
        if (!ok) break;
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(sv + KV4_VOFF) + (h * MT * 16 + g) * NG;
        float svm;
        if (whole) {  // the largest scale: positive bf16 values order like their bits
          uint32_t x = 0;
#pragma unroll
          for (int i = 0; i < 2 * MT * NG; ++i) x = __vmaxu2(x, vp[(i / NG) * 8 * NG + i % NG]);
          svm = bf16_lo(x);
        } else {  // a page that holds tokens some row does not see
          svm = 0.f;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int key = page0 + (h * MT + mt) * 16 + y * 8 + g;
              float bad = good ? 0.f : NAN;  // NaN for a row that sees a token which is not finite
              const bool in = key < at.len && good;
#pragma unroll
              for (int x = 0; x < NG; ++x) {
                const uint32_t p = vp[(mt * 16 + y * 8) * NG + x];
                if (!(fabsf(bf16_lo(p) + bf16_hi(p)) < INFINITY))
                  bad = NAN;
                else if (in)
                  svm = fmaxf(svm, bf16_lo(p));
              }
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                float x0, x1;
                un2(s[mt][t][y], x0, x1);
                x0 = key <= lim[t][0] && key < at.len ? x0 + bad : -INFINITY;
                x1 = key <= lim[t][1] && key < at.len ? x1 + bad : -INFINITY;
                s[mt][t][y] = f2(x0, x1);
              }
            }
        }
        // ---- reference maxima and the powers of p s move only when they must, all rows' then: when a score
        // passes its maximum by 2^8, or some p sg s may pass 2^15 (the lane's largest p times its largest
        // scale, which need not be one token's) ----
        bool move = false;
        float top[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float x0, x1, x2, x3;
            un2(s[mt][t][0], x0, x1);
            un2(s[mt][t][1], x2, x3);
            top[t][0] = mt ? fmax3(top[t][0], x0, x2) : fmaxf(x0, x2);
            top[t][1] = mt ? fmax3(top[t][1], x1, x3) : fmaxf(x1, x3);
          }
          float g0, g1;
          un2(sg[t], g0, g1);
          const float d0 = (top[t][0] - m[t][0]) * KA_UNIT, d1 = (top[t][1] - m[t][1]) * KA_UNIT;
          move = move || d0 > 8.f || d1 > 8.f || ka_ex2(d0) * g0 * svm > 32768.f || ka_ex2(d1) * g1 * svm > 32768.f;
        }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            float c[2], f[2], g2[2], most[2] = {0.f, 0.f};  // most: each row's largest p s, times 2^-20
            int was[2];
            un2(sg[t], g2[0], g2[1]);
            // maxima to the next whole number: sg can grow by the power of two that p loses
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float x = top[t][e];
#pragma unroll
              for (int i = 4; i < 32; i <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, i));
              x = fmaxf(m[t][e], ceilf(x * KA_UNIT) * KA_PER);
              const float d = (x - m[t][e]) * KA_UNIT;
              c[e] = ka_ex2(-d);
              m[t][e] = x;
              was[e] = (int)(__float_as_uint(g2[e]) >> 23) + (int)fminf(d, 512.f);  // field of the sg that leaves O as it is
            }
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                // the token's largest scale (a NaN drops out of the maximum below, as does whatever a p of 0 stands before)
                uint32_t w = 0;
                float x0, x1;
#pragma unroll
                for (int x = 0; x < NG; ++x) w = __vmaxu2(w, vp[(mt * 16 + y * 8) * NG + x]);
                const float sc = KA_PER * bf16_lo(w);
                un2(s[mt][t][y], x0, x1);
                most[0] = fmaxf(most[0], sc * ka_ex2((x0 - m[t][0]) * KA_UNIT));
                most[1] = fmaxf(most[1], sc * ka_ex2((x1 - m[t][1]) * KA_UNIT));
              }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int i = 4; i < 32; i <<= 1) most[e] = fmaxf(most[e], __shfl_xor_sync(0xffffffffu, most[e], i));
              // fields: with sg's at f, p s sg lies in [2^(to + f - 254 + 20), twice that); in [2^KA_SG_TO, twice that) at most from now on
              const int to = (int)(__float_as_uint(most[e]) >> 23);
              int now = was[e] < KA_SG_FIELD ? was[e] : KA_SG_FIELD;
              if (to > 0 && now > 254 - 20 + KA_SG_TO - to) now = 254 - 20 + KA_SG_TO - to;
              now = now < 1 ? 1 : now;
              g2[e] = __uint_as_float((uint32_t)now << 23);
              f[e] = was[e] - now < 127 ? __uint_as_float((uint32_t)(127 - (was[e] - now)) << 23) : 0.f;
            }
            sg[t] = f2(g2[0], g2[1]);
            l[t] = f2mul(l[t], f2(c[0], c[1]));
#pragma unroll
            for (int x = 0; x < NG; ++x) zs[t][x] = f2mul(zs[t][x], f2(c[0], c[1]));
#pragma unroll
            for (int x = 0; x < 8; ++x)
#pragma unroll
              for (int e = 0; e < 4; ++e) o[t][x][e] *= f[e & 1];
          }
        }
        // ---- p, its sums, P^T fragments, O^T += V^T P^T ----
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          uint32_t pb[NT][NG][2];
          uint64_t p2[NT][2], pg[NT][2];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint64_t nm = f2(-KA_UNIT * m[t][0], -KA_UNIT * m[t][1]), un = f2(KA_UNIT, KA_UNIT);
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float x0, x1;
              un2(f2fma(s[mt][t][y], un, nm), x0, x1);
              p2[t][y] = f2(ka_ex2(x0), ka_ex2(x1));
              l[t] = f2add(l[t], p2[t][y]);
              pg[t][y] = f2mul(p2[t][y], sg[t]);
            }
          }
#pragma unroll
          for (int x = 0; x < NG; ++x)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t p = vp[(mt * 16 + y * 8) * NG + x];
              float sc = bf16_lo(p), zv = bf16_hi(p);
              if (!whole) {
                const int key = page0 + (h * MT + mt) * 16 + y * 8 + g;
                if (key >= at.len || !good || !(fabsf(sc + zv) < INFINITY)) sc = zv = 0.f;
              }
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                zs[t][x] = f2fma(p2[t][y], f2(zv, zv), zs[t][x]);
                float x0, x1;
                un2(f2mul(pg[t][y], f2(sc, sc)), x0, x1);
                pb[t][x][y] = transpose8x8(pack_f16x2(x0, x1));
              }
            }
          const uint8_t* vb = sv + (h * MT + mt) * 1024 + lane * 16;
          const uint4 v0 = *reinterpret_cast<const uint4*>(vb), v1 = *reinterpret_cast<const uint4*>(vb + 512);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int x = j * NG / 4;
            const uint32_t sel = (j & 1) ? 0x7632 : 0x5410;
            const uint32_t w0 = __byte_perm(j < 2 ? v0.x : v0.y, j < 2 ? v0.z : v0.w, sel);
            const uint32_t w1 = __byte_perm(j < 2 ? v1.x : v1.y, j < 2 ? v1.z : v1.w, sel);
            const uint32_t a0 = code_0(w0), a1 = code_1(w0), a2 = code_0(w1), a3 = code_1(w1);
            const uint32_t b0 = code_0(w0 >> 8), b1 = code_1(w0 >> 8), b2 = code_0(w1 >> 8), b3 = code_1(w1 >> 8);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              mma_f16(o[t][2 * j], a0, a1, a2, a3, pb[t][x][0], pb[t][x][1]);
              mma_f16(o[t][2 * j + 1], b0, b1, b2, b3, pb[t][x][0], pb[t][x][1]);
            }
          }
        }
      }
      if (!ok) break;
      __syncwarp();
      if (lane == 0 && sent > used + 1) send_v();
      __syncwarp();
    }
    // ---- the item, or this CTA's piece of it, is done: join the warps ----
    if (ok) {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float lt[2], z[NG][2], back[2];
        un2(l[t], lt[0], lt[1]);
        un2(sg[t], back[0], back[1]);  // powers of two: 1 / sg from the exponent's field
        back[0] = __uint_as_float((254u << 23) - __float_as_uint(back[0]));
        back[1] = __uint_as_float((254u << 23) - __float_as_uint(back[1]));
#pragma unroll
        for (int x = 0; x < NG; ++x) un2(zs[t][x], z[x][0], z[x][1]);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int i = 4; i < 32; i <<= 1) {
            lt[e] += __shfl_xor_sync(0xffffffffu, lt[e], i);
#pragma unroll
            for (int x = 0; x < NG; ++x) z[x][e] += __shfl_xor_sync(0xffffffffu, z[x][e], i);
          }
          // a NaN group of any V makes the whole row NaN, not its own dims alone
#pragma unroll
          for (int x = 0; x < NG; ++x) lt[e] += (z[x][e] - z[x][e]) + (o[t][8 / NG * x][e] - o[t][8 / NG * x][e]);
          const int r = t * 8 + 2 * cq + e;
          if (g == 0) {
            sm.m[warp][r] = KA_UNIT * m[t][e];
            sm.l[warp][r] = lt[e];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float zz = z[j * NG / 4][e];
            *reinterpret_cast<float4*>(&sm.o[warp][r][32 * j + 4 * g]) =
                make_float4(fmaf(16777216.f * o[t][2 * j][e], back[e], zz), fmaf(1048576.f * o[t][2 * j][2 + e], back[e], zz),
                            fmaf(16777216.f * o[t][2 * j + 1][e], back[e], zz),
                            fmaf(1048576.f * o[t][2 * j + 1][2 + e], back[e], zz));  // codes count 2^-24 and 2^-20
          }
        }
      }
    }
    failed = __syncthreads_or(!ok);
    if (failed) break;
    const bool ends = at.pb == at.pages, whole_item = ends && at.pa == 0;
    float* slot = a.part + (size_t)(2 * blockIdx.x + (at.pa == 0 ? 1 : 0)) * (R * (KV4_D + 2));
#pragma unroll 1
    for (int r = warp; r < R; r += NW) {
      const int rr = at.rt * R + r, tok = rr / a.G, head = at.h * a.G + (rr - tok * a.G);
      if (tok >= at.count) break;
      const float top = fmaxf(fmaxf(sm.m[0][r], sm.m[1][r]), fmaxf(sm.m[2][r], sm.m[3][r]));
      float sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float f = ka_ex2(sm.m[w][r] - top);
        const float4 x = *reinterpret_cast<const float4*>(&sm.o[w][r][4 * lane]);
        sum = fmaf(sm.l[w][r], f, sum);
        v.x = fmaf(x.x, f, v.x);
        v.y = fmaf(x.y, f, v.y);
        v.z = fmaf(x.z, f, v.z);
        v.w = fmaf(x.w, f, v.w);
      }
      if (whole_item) {
        const size_t orow = (size_t)(at.first + tok) * Hq + head;
        const float f = (sum == 0.f ? 0.f : 1.f / sum) * (a.gate ? __ldg(a.gate + orow) : 1.f);
        *reinterpret_cast<uint2*>(a.out + orow * KV4_D + 4 * lane) =
            make_uint2(pack_bf16x2(v.x * f, v.y * f), pack_bf16x2(v.z * f, v.w * f));
      } else {
        *reinterpret_cast<float4*>(slot + r * KV4_D + 4 * lane) = v;
        if (lane == 0) {
          slot[R * KV4_D + r] = top;
          slot[R * KV4_D + R + r] = sum;
        }
      }
    }
    __syncthreads();  // the O tiles and the item have been read
    if (tid == 0) {
      const KaSeg was = sm.at;
      KaSeg k = was;
      const bool next = ka_next<R>(a, k);
      sm.at = k;
      sm.found[0] = next;
      int4 cut = make_int4(-1, 0, 0, 0);
      if (!next && was.pa == 0 && was.pb != was.pages) {
        // the item's last page on the line of pages, and the CTA that has it
        const int end = u1 - 1 + (was.pages - was.pb), head = longer * (each + 1);
        const int z = end < head ? end / (each + 1) : longer + (end - head) / each;
        // (another number only if lengths changed meanwhile, or rows of sequences overlap: not followed)
        if (z > (int)blockIdx.x && z < ctas) cut = make_int4(was.b, was.rt, was.h, z);
      }
      if (!next) a.cut[blockIdx.x] = cut;
    }
    __syncthreads();
    go = sm.found[0] != 0;
  }
  // a failed wait (reported in the status word) leaves copies under way: let
  // them land before this CTA's shared memory is given up
  if (failed) {
    if (lane == 0 && sent > used) {
      const uint64_t t0 = globaltimer_ns();
      while ((!mbar_try_wait(smem_u32(&sm.kfull[warp]), (sent - 1) & 1) ||
              !mbar_try_wait(smem_u32(&sm.vfull[warp]), used & 1)) &&
             globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    }
    if (tid == 0) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
  }
}

// Joins the pieces of the items that were cut: CTA (x, y) takes rows of the
// item that starts in attention CTA x and goes on to CTA cut[x].w. Its pieces
// are slot 2 x + 1 and slots 2 i, i = x + 1 .. w. Items of many pieces: row y,
// the pieces taken in that order by eight warps in turn, whose sums are added in
// warp order. Items of few (WARP_ROWS): row 8 y + warp, in that order.
template <int R, bool WARP_ROWS>
__global__ void __launch_bounds__(256) kv4_join_kernel(const KaArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float sm_m[8], sm_l[8];
  __shared__ float4 sm_o[8][32];
  const int4 cut = a.cut[blockIdx.x];
  if (cut.x < 0) return;
  const int warp = warp_id(), lane = lane_id(), r = WARP_ROWS ? 8 * blockIdx.y + warp : blockIdx.y;
  int first, count;
  kv4_rows(a.c, cut.x, &first, &count);
  const int rr = cut.y * R + r, tok = rr / a.G;
  if (tok >= count) return;
  const int pieces = cut.w - (int)blockIdx.x + 1;
  constexpr int SLOT = R * (KV4_D + 2);
  auto slot = [&](int i) { return a.part + (size_t)(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * SLOT; };
  float top = -FLT_MAX;
  for (int i = WARP_ROWS ? lane : threadIdx.x; i < pieces; i += WARP_ROWS ? 32 : 256) top = fmaxf(top, slot(i)[R * KV4_D + r]);
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
  if (!WARP_ROWS) {
    if (lane == 0) sm_m[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, sm_m[w]);
  }
  float sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = WARP_ROWS ? 0 : warp; i < pieces; i += WARP_ROWS ? 1 : 8) {
    const float* s = slot(i);
    const float f = ka_ex2(s[R * KV4_D + r] - top);
    const float4 x = *reinterpret_cast<const float4*>(s + r * KV4_D + 4 * lane);
    sum = fmaf(s[R * KV4_D + R + r], f, sum);
    v.x = fmaf(x.x, f, v.x);
    v.y = fmaf(x.y, f, v.y);
    v.z = fmaf(x.z, f, v.z);
    v.w = fmaf(x.w, f, v.w);
  }
  if (!WARP_ROWS) {
    sm_o[warp][lane] = v;
    if (lane == 0) sm_l[warp] = sum;
    __syncthreads();
  }
  if (WARP_ROWS || warp == 0) {
#pragma unroll
    for (int w = 1; w < (WARP_ROWS ? 1 : 8); ++w) {
      const float4 x = sm_o[w][lane];
      sum += sm_l[w];
      v.x += x.x;
      v.y += x.y;
      v.z += x.z;
      v.w += x.w;
    }
    const size_t orow = (size_t)(first + tok) * a.c.heads * a.G + cut.z * a.G + (rr - tok * a.G);
    const float f = (sum == 0.f ? 0.f : 1.f / sum) * (a.gate ? __ldg(a.gate + orow) : 1.f);
    *reinterpret_cast<uint2*>(a.out + orow * KV4_D + 4 * lane) =
        make_uint2(pack_bf16x2(v.x * f, v.y * f), pack_bf16x2(v.z * f, v.w * f));
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Many rows a sequence and K/V head: the tcgen05 kernel over f16 operands in
// the workspace. Below this the page kernel above, whose time grows with every
// 16 rows, is faster than laying the operands out (4 x 16,384 tokens x 8 heads:
// 33 us per 16 rows against 165 for up to 256).
constexpr int KV4_TC_MIN = 80;
constexpr uint64_t KV4_TC_BYTES = 24ull << 30;  // and never for operands beyond this

static uint64_t kv4_tc_layout(const Kv4View& c, int G, Kv4Tc* t, void* ws) {
  uint64_t at = 0;
  uint8_t* base = static_cast<uint8_t*>(ws);
  auto take = [&](uint64_t bytes) {
    uint8_t* p = base ? base + at : nullptr;
    at += (bytes + 255) & ~uint64_t(255);
    return p;
  };
  const uint64_t qr = (uint64_t)c.heads * c.rows * G, bh = (uint64_t)c.batch * c.heads;
  t->G = G;
  t->tokens = (c.cap + 127) / 128 * 128;
  t->chunks = (t->tokens / KV4_PAGE + 15) / 16;
  t->splits = kv4_tc_splits(c, G);
  t->q16 = take(qr * KV4_D * 2);
  t->q_scale = reinterpret_cast<float*>(take(qr * 4));
  t->k16 = take(bh * t->tokens * KV4_D * 2);
  t->v16 = take(bh * t->tokens * KV4_D * 2);
  t->top = reinterpret_cast<float2*>(take(bh * t->chunks * 8));
  t->kv_scale = reinterpret_cast<float2*>(take(bh * 8));
  t->o_part = reinterpret_cast<float*>(take(t->splits > 1 ? t->splits * qr * KV4_D * 4 : 0));
  t->ml_part = reinterpret_cast<float*>(take(t->splits > 1 ? t->splits * qr * 8 : 0));
  return at;
}

// Whether a call takes the tcgen05 path, and its workspace there.
static bool kv4_use_tc(const Kv4View& c, int G, uint64_t* bytes, Kv4Tc* t) {
  if ((int64_t)c.rows * G < (int64_t)KV4_TC_MIN * c.batch || c.cap == 0 || c.batch > 65535 || c.heads > 65535) return false;
  if ((int64_t)c.heads * c.rows * G > INT32_MAX || (int64_t)c.batch * c.heads * ((c.cap + 127ll) / 128 * 128) > INT32_MAX)
    return false;  // TMA coordinates
  *bytes = kv4_tc_layout(c, G, t, nullptr);
  return *bytes <= KV4_TC_BYTES;
}

// Query rows of a tile: 8 where every sequence's rows fit (one n8 tile of
// the MMA), else 16, which unpacks a page once for twice the rows.
static int ka_rows(int rows, int batch, int G) { return (int64_t)rows * G <= 8ll * batch ? 8 : 16; }
// CTAs of a call: as many as the GPU holds at once, or as the capacity can keep
// busy (one per item, a page per warp). Row tiles are bounded alike with and
// without row_start: the workspace is sized before that is known.
static int ka_ctas(const Kv4View& c, int G, int R) {
  const int64_t items = ((int64_t)c.rows * G / R + (c.batch < c.rows ? c.batch : c.rows)) * c.heads;
  const int64_t pages = (c.cap + KV4_PAGE - 1) / KV4_PAGE, most = (int64_t)sm_count() * KA_PER_SM;
  if (items >= most || items * pages / KA_WARPS >= most) return (int)most;
  const int64_t n = (items * pages + KA_WARPS - 1) / KA_WARPS;
  return (int)(n > items ? n : items);
}
constexpr int KA_FEW = 8;  // pieces an item
static uint64_t ka_cut_bytes(int ctas) { return ((uint64_t)ctas * 16 + 255) & ~uint64_t(255); }
static uint64_t ka_workspace(int ctas, int R) { return ka_cut_bytes(ctas) + (uint64_t)ctas * 2 * R * (KV4_D + 2) * 4; }

template <int NG, int R>
static int ka_launch(const KaArgs& a, int ctas, cudaStream_t st) {
  constexpr int bytes = ka_smem_bytes<R>(NG);
  static std::atomic<bool> attr[kMaxDevices];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return set_error(LTXB_EINVAL, "kv4 attention: device %d out of range", dev);
  if (!attr[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(kv4_attn_kernel<NG, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return set_cuda_error(e, "kv4 attention: cudaFuncSetAttribute");
    attr[dev].store(true, std::memory_order_release);
  }
  kv4_attn_kernel<NG, R><<<ctas, KA_THREADS, bytes, st>>>(a);
  launched();
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "kv4 attention launch");
  cudaLaunchConfig_t cfg{};
  // Items of few pieces (on average): a row a warp, and an eighth of the CTAs, most of
  // which find nothing to join. 8 x 1,700 tokens x 8 heads, 16 rows, without L2: 32 us
  // instead of 36; 4 x 4,000, 64 rows: 52 and 60. With 14 pieces an item (131,009 tokens x 32
  // heads) 124 and 122.
  const int64_t tiles = (int64_t)a.c.rows * a.G / R;
  const bool warp_rows = ctas <= KA_FEW * (tiles > a.c.batch ? tiles : a.c.batch) * a.c.heads;
  cfg.gridDim = dim3(ctas, warp_rows ? R / 8 : R);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute la[1];
  la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  la[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = la;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, warp_rows ? kv4_join_kernel<R, true> : kv4_join_kernel<R, false>, a);
  launched();
  return e == cudaSuccess ? LTXB_OK : set_cuda_error(e, "kv4 attention join launch");
}

}  // namespace ltxb

using namespace ltxb;

extern "C" {

uint64_t ltxb_attention_kv4_workspace_bytes(const ltxb_kv4_cache* cache, int rows, int H) {
  Kv4View c;
  Kv4Tc t;
  if (rows <= 0 || H <= 0 || kv4_check(cache, nullptr, 0, "kv4 attention", &c) || H % c.heads || c.batch == 0) return 0;
  c.rows = rows;
  uint64_t bytes;
  if (kv4_use_tc(c, H / c.heads, &bytes, &t)) return bytes;
  const int R = ka_rows(rows, c.batch, H / c.heads);
  return ka_workspace(ka_ctas(c, H / c.heads, R), R);
}

int ltxb_attention_kv4(const ltxb_kv4_cache* cache, const int32_t* row_start, const void* q, int64_t ldq, void* out,
                       const float* gate, int rows, int H, int causal, float scale, void* workspace,
                       uint64_t workspace_bytes, void* stream) {
  KaArgs a{};
  if (int rc = kv4_check(cache, row_start, rows, "kv4 attention", &a.c)) return rc;
  if (H <= 0 || H % cache->kv_heads)
    return set_error(LTXB_EINVAL, "kv4 attention: H = %d is not a multiple of the cache's %d K/V heads", H, cache->kv_heads);
  if (rows == 0) return LTXB_OK;
  if (!q || !out || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15) || ldq % 8)
    return set_error(LTXB_EINVAL, "kv4 attention: q and out must be 16-byte aligned, q's row stride a multiple of 16 bytes");
  if (ldq < (int64_t)H * KV4_D) return set_error(LTXB_EINVAL, "kv4 attention: q's row stride is smaller than H * 128");
  if (reinterpret_cast<uintptr_t>(gate) & 3) return set_error(LTXB_EINVAL, "kv4 attention: gate must be 4-byte aligned");
  if (!(scale == scale) || scale - scale != 0.f) return set_error(LTXB_EINVAL, "kv4 attention: scale must be finite");
  a.G = H / cache->kv_heads;
  const int R = ka_rows(rows, cache->batch, a.G);
  uint64_t need = 0;
  Kv4Tc t{};
  const bool tc = kv4_use_tc(a.c, a.G, &need, &t);
  const int ctas = ka_ctas(a.c, a.G, R);
  if (!tc) need = ka_workspace(ctas, R);
  if (!workspace || workspace_bytes < need)
    return set_error(LTXB_EINVAL, "kv4 attention: workspace of %llu bytes is smaller than the %llu required",
                     (unsigned long long)workspace_bytes, (unsigned long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) & 255) return set_error(LTXB_EINVAL, "workspace must be 256-byte aligned");
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.ldq = (size_t)ldq;
  a.gate = gate;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.cs = scale * 1.4426950408889634f;
  a.causal = causal != 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (tc) {
    kv4_tc_layout(a.c, a.G, &t, workspace);
    t.cs = a.cs;
    if (int rc = kv4_prepare(a.c, t, q, (size_t)ldq, cache->group, st)) return rc;
    return kv4_attention_tc(a.c, t, gate, out, a.causal, st);
  }
  const int64_t tiles = (int64_t)rows * a.G / R + a.c.batch;  // at least the row tiles of all sequences
  if (((int64_t)(a.c.cap + KV4_PAGE - 1) / KV4_PAGE + KA_ITEM) * a.c.heads > INT32_MAX / tiles)
    return set_error(LTXB_EINVAL, "kv4 attention: more than 2^31 pages of work in a call (max_len bounds it)");
  a.cut = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ka_cut_bytes(ctas));
  const int ng = KV4_D / cache->group;
  if (R == 8) {
    if (ng == 1) return ka_launch<1, 8>(a, ctas, st);
    if (ng == 2) return ka_launch<2, 8>(a, ctas, st);
    return ka_launch<4, 8>(a, ctas, st);
  }
  if (ng == 1) return ka_launch<1, 16>(a, ctas, st);
  if (ng == 2) return ka_launch<2, 16>(a, ctas, st);
  return ka_launch<4, 16>(a, ctas, st);
}

}  // extern "C"
