// Attention of a few query rows over the paged 4-bit K/V cache (decoding and
// short runs of tokens): softmax(q k^T * scale) v with k, v = zero + scale_kv * code.
//
// The codes go to the tensor cores as they are. Put in the top mantissa bits
// of a 16-bit float, a code c reads u = 1 + c / 16 exactly, and
//   q . (z + s c)       = 16 s (q . u - 1.5 sum q) + (z + 8 s) sum q
//   sum_t p_t (z + s c) = 16 (sum p s u - 1.5 sum p s) + sum p (z + 8 s)
// (per group of 32 / 64 / 128 dims), so scale and zero touch only score-sized
// data and unpacking costs one shift and one logic operation per two codes.
// The offsets are subtracted where they were added: q's part as the initial
// value of the accumulator, p's part by one more MMA with constant rows 1.5
// over the same rounded p s.
//
// One warp takes 16 tokens of a page as the M side of mma.m16n8k16, so up to
// 8 query rows (the query heads that share the K/V head, times the call's
// tokens) cost the same as one: S^T = K Q^T, then O^T = V^T P^T with P^T
// transposed in registers (movmatrix). K and q enter as bf16 (q is bf16, the
// codes are exact). p s enters as f16 scaled by a power of two that follows
// the largest V scale seen (between 2^3 and 2^7 times p): 11 significant bits
// where bf16 would keep 8, so the result's own rounding dominates. Row maxima
// move only when a score passes them by 2^8; sums and accumulators are f32.
//
// Work is split by pages, not by sequence: all (sequence, head, row tile)
// items laid end to end are one line of pages, each CTA takes an equal piece
// of it, and a second kernel joins the items that were cut (in page order, so
// results do not depend on timing). Lengths are read on the device only.
// A page's block for one head (8.5 - 10 KB) arrives by one bulk copy into a
// ring of KA_STAGES, so 4 CTAs keep about 100 KB per SM in flight.
//
// A token whose V group is stored as NaN, or whose page number is bad, makes
// its score NaN (every row that attends to it becomes NaN) and is left out of
// the product, so that rows which do not attend to it stay finite.
#include <float.h>

#include <atomic>

#include "kv4.cuh"

namespace ltxb {

constexpr int KA_STAGES = 4;
constexpr int KA_THREADS = 128;
constexpr int KA_OLD = KV4_D + 4;  // floats per row of the warps' O tiles

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

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// bf16 pair (1 + c / 16) of nibbles I and I + 4 of w
template <int I>
__device__ __forceinline__ uint32_t code_bf16(uint32_t w) {
  const uint32_t s = I == 0 ? w << 3 : w >> (4 * I - 3);
  return (s & 0x00780078u) | 0x3F803F80u;
}
// f16 pair (1 + c / 16) of nibble I of both halves of w
template <int I>
__device__ __forceinline__ uint32_t code_f16(uint32_t w) {
  const uint32_t s = I < 2 ? w << (6 - 4 * I) : w >> (4 * I - 6);
  return (s & 0x03C003C0u) | 0x3C003C00u;
}

// One-dimensional bulk copy global -> shared; both ends 16-byte aligned, the
// size a multiple of 16.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// A place on the line of pages: page `page` of (sequence b, row tile rt, head h).
struct KaCursor {
  int b, rt, h, page;
  int pages, tiles, len, first, count;  // of sequence b
};

template <int R>
__device__ __forceinline__ void ka_seq(const KaArgs& a, KaCursor& k) {
  k.len = kv4_len(a.c, k.b);
  kv4_rows(a.c, k.b, &k.first, &k.count);
  k.pages = (k.len + KV4_PAGE - 1) / KV4_PAGE;
  k.tiles = k.pages > 0 ? (k.count * a.G + R - 1) / R : 0;
}

template <int R>
__device__ __forceinline__ void ka_next(const KaArgs& a, KaCursor& k) {
  if (++k.page < k.pages) return;
  k.page = 0;
  if (++k.h < a.c.heads) return;
  k.h = 0;
  if (++k.rt < k.tiles) return;
  k.rt = 0;
  do {
    if (++k.b >= a.c.batch) return;
    ka_seq<R>(a, k);
  } while (k.tiles == 0);
}

template <int R>
struct KaSmem {
  uint64_t full[KA_STAGES], empty[KA_STAGES];
  int good[KA_STAGES];  // the stage's page number was valid
  long long scan[4];
  int found[4];
  float m[4][R], l[4][R];
  float o[4][R][KA_OLD];
};
template <int R>
constexpr int ka_smem_bytes(int ng) {
  return KA_STAGES * kv4_block(ng) + (int)sizeof(KaSmem<R>) + 128;
}

template <int NG, int R>
__global__ void __launch_bounds__(KA_THREADS, R == 8 ? 4 : 3) kv4_attn_kernel(const KaArgs a) {
  constexpr int NT = R / 8, BLK = kv4_block(NG);
  extern __shared__ __align__(128) uint8_t ka_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(ka_raw) + 127) & ~uintptr_t(127));
  KaSmem<R>& sm = *reinterpret_cast<KaSmem<R>*>(ring + KA_STAGES * BLK);
  const int tid = threadIdx.x, warp = warp_id(), lane = lane_id(), g = lane >> 2, cq = lane & 3;
  const int Hq = a.c.heads * a.G;

  if (tid == 0) {
    for (int i = 0; i < KA_STAGES; ++i) {
      mbar_init(&sm.full[i], 1);
      mbar_init(&sm.empty[i], 4);
    }
    fence_mbar_init();
  }
  // ---- this CTA's piece [u0, u1) of the line of pages ----
  auto units = [&](int b) -> long long {
    KaCursor k;
    k.b = b;
    ka_seq<R>(a, k);
    return (long long)k.pages * k.tiles * a.c.heads;
  };
  long long mine = 0;
  for (int b = tid; b < a.c.batch; b += KA_THREADS) mine += units(b);
#pragma unroll
  for (int s = 16; s; s >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, s);
  if (lane == 0) sm.scan[warp] = mine;
  if (tid == 0) sm.found[0] = -1;
  __syncthreads();
  const long long total = sm.scan[0] + sm.scan[1] + sm.scan[2] + sm.scan[3];
  const int ctas = total < gridDim.x ? (int)total : (int)gridDim.x;
  // sequences without tokens: their rows attend to nothing and are zero
  for (int b = blockIdx.x; b < a.c.batch; b += gridDim.x) {
    int first, count;
    kv4_rows(a.c, b, &first, &count);
    if (count > 0 && kv4_len(a.c, b) == 0)
      for (long long i = tid; i < (long long)count * Hq * (KV4_D / 8); i += KA_THREADS)
        reinterpret_cast<uint4*>(a.out + (size_t)first * Hq * KV4_D)[i] = make_uint4(0, 0, 0, 0);
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if ((int)blockIdx.x >= ctas) {
    if (tid == 0) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
    return;
  }
  const long long u0 = total * blockIdx.x / ctas, u1 = total * (blockIdx.x + 1) / ctas;
  // the sequence that holds u0: prefix sums over 128 sequences at a time
  KaCursor at;
  {
    long long base = 0;
    for (int b0 = 0;; b0 += KA_THREADS) {
      const long long n = b0 + tid < a.c.batch ? units(b0 + tid) : 0;
      long long x = n;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, s);
        if (lane >= s) x += y;
      }
      __syncthreads();
      if (lane == 31) sm.scan[warp] = x;
      __syncthreads();
      for (int w = 0; w < warp; ++w) x += sm.scan[w];
      x += base;
      if (n > 0 && u0 >= x - n && u0 < x) {
        const long long d = u0 - (x - n);
        KaCursor k;
        k.b = b0 + tid;
        ka_seq<R>(a, k);
        sm.found[0] = k.b;
        sm.found[1] = (int)(d / ((long long)k.pages * a.c.heads));
        sm.found[2] = (int)(d / k.pages % a.c.heads);
        sm.found[3] = (int)(d % k.pages);
      }
      base += sm.scan[0] + sm.scan[1] + sm.scan[2] + sm.scan[3];
      if (base > u0 || b0 >= a.c.batch) break;
    }
    __syncthreads();
    if (sm.found[0] < 0) {  // only if the lengths changed while this ran
      if (tid == 0) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    at.b = sm.found[0];
    at.rt = sm.found[1];
    at.h = sm.found[2];
    at.page = sm.found[3];
    ka_seq<R>(a, at);
  }
  const int n = (int)(u1 - u0);

  // ---- producer (lane 0 of warp 0): page i of this CTA into stage i % KA_STAGES ----
  KaCursor pc = at;
  int sent = 0;
  auto send = [&]() {
    const int st = sent % KA_STAGES;
    const int p = kv4_page(a.c, pc.b, pc.page);
    sm.good[st] = p >= 0;
    if (p >= 0) {
      mbar_arrive_expect_tx(&sm.full[st], BLK);
      bulk_load(ring + st * BLK, kv4_block_at(a.c, p, pc.h, BLK), BLK, &sm.full[st]);
    } else {
      mbar_arrive(&sm.full[st]);
    }
    ++sent;
    if (sent < n) ka_next<R>(a, pc);
  };
  if (tid == 0)
    while (sent < n && sent < KA_STAGES - 1) send();

  bool ok = true, item = false, failed = false;
  uint32_t qf[NT][16];
  float qs[NT][NG][2], o[NT][8][4], o1[NT][NG][4], m[NT][2], l[NT][2], zs[NT][NG][2];
  int lim[NT][2];
  float sig = 1.f, sig_max = 0.f;  // p s is held as p * (s * sig); sig moves when s passes sig_max
  int item_start = 0;              // page of the item this CTA began with
  for (int i = 0; i < n; ++i) {
    if (!item) {  // a new item: its query rows, and nothing accumulated
      item = true;
      item_start = at.page;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int r = at.rt * R + t * 8 + g, tok = r / a.G;
        const bool has = tok < at.count;
        const __nv_bfloat16* src = a.q + (size_t)(at.first + tok) * a.ldq + (at.h * a.G + (r - tok * a.G)) * KV4_D + 8 * cq;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint4 w = has ? __ldg(reinterpret_cast<const uint4*>(src + 32 * j)) : make_uint4(0, 0, 0, 0);
          qf[t][4 * j + 0] = __byte_perm(w.x, w.z, 0x5410);  // dims 0, 4 of the eight
          qf[t][4 * j + 1] = __byte_perm(w.x, w.z, 0x7632);  // 1, 5
          qf[t][4 * j + 2] = __byte_perm(w.y, w.w, 0x5410);  // 2, 6
          qf[t][4 * j + 3] = __byte_perm(w.y, w.w, 0x7632);  // 3, 7
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int rc = at.rt * R + t * 8 + 2 * cq + e, tc = rc / a.G;
          lim[t][e] = a.causal ? at.len - at.count + tc : at.len - 1;  // last key the row sees
          m[t][e] = -FLT_MAX;
          l[t][e] = 0.f;
        }
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][x][e] = 0.f;
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int y = 0; y < 8 / NG; ++y) {
            const int k = x * (8 / NG) + y;
            mma_bf16(s, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u, qf[t][2 * k], qf[t][2 * k + 1]);
          }
          qs[t][x][0] = s[0];
          qs[t][x][1] = s[1];
          zs[t][x][0] = zs[t][x][1] = 0.f;
          o1[t][x][0] = o1[t][x][1] = o1[t][x][2] = o1[t][x][3] = 0.f;
        }
      }
      sig = 1.f;
      sig_max = 0.f;
    }
    const int st = i % KA_STAGES;
    if (ok) ok = warp_wait(&sm.full[st], (i / KA_STAGES) & 1, 0x301);
    if (ok) {
      const uint8_t* blk = ring + st * BLK;
      const int t0 = warp * 16 + g;  // this lane's tokens t0 and t0 + 8 of the page
      const int key0 = at.page * KV4_PAGE + t0, key1 = key0 + 8;
      const int len = at.len;
      const bool good = sm.good[st] != 0;
      // ---- S^T: 16 tokens x R rows ----
      float s[NT][4];
      {
        const uint4 k0 = *reinterpret_cast<const uint4*>(blk + t0 * 64 + cq * 16);
        const uint4 k1 = *reinterpret_cast<const uint4*>(blk + (t0 + 8) * 64 + cq * 16);
        const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
        float acc[NT][NG][4];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < NG; ++x) {
            acc[t][x][0] = acc[t][x][2] = -1.5f * qs[t][x][0];
            acc[t][x][1] = acc[t][x][3] = -1.5f * qs[t][x][1];
          }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int x = j * NG / 4;
          const uint32_t a00 = code_bf16<0>(w0[j]), a10 = code_bf16<0>(w1[j]), a01 = code_bf16<1>(w0[j]),
                         a11 = code_bf16<1>(w1[j]), a02 = code_bf16<2>(w0[j]), a12 = code_bf16<2>(w1[j]),
                         a03 = code_bf16<3>(w0[j]), a13 = code_bf16<3>(w1[j]);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_bf16(acc[t][x], a00, a10, a01, a11, qf[t][4 * j], qf[t][4 * j + 1]);
            mma_bf16(acc[t][x], a02, a12, a03, a13, qf[t][4 * j + 2], qf[t][4 * j + 3]);
          }
        }
        const uint32_t* kp = reinterpret_cast<const uint32_t*>(blk + KV4_KPAIR);
#pragma unroll
        for (int t = 0; t < NT; ++t) s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          const uint32_t p0 = kp[t0 * NG + x], p1 = kp[(t0 + 8) * NG + x];
          const float s0 = bf16_lo(p0) * a.cs, s1 = bf16_lo(p1) * a.cs;
          const float z0 = fmaf(8.f, s0, bf16_hi(p0) * a.cs), z1 = fmaf(8.f, s1, bf16_hi(p1) * a.cs);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            s[t][0] += fmaf(16.f * s0, acc[t][x][0], z0 * qs[t][x][0]);
            s[t][1] += fmaf(16.f * s0, acc[t][x][1], z0 * qs[t][x][1]);
            s[t][2] += fmaf(16.f * s1, acc[t][x][2], z1 * qs[t][x][0]);
            s[t][3] += fmaf(16.f * s1, acc[t][x][3], z1 * qs[t][x][1]);
          }
        }
      }
      // ---- V scales of the two tokens: sv = 16 s, zv = z + 8 s ----
      float sv0[NG], sv1[NG], zv0[NG], zv1[NG], bad0 = 0.f, bad1 = 0.f, svm = 0.f;
      {
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(blk + kv4_vpair(NG));
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          const uint32_t p0 = vp[t0 * NG + x], p1 = vp[(t0 + 8) * NG + x];
          sv0[x] = bf16_lo(p0);
          sv1[x] = bf16_lo(p1);
          zv0[x] = fmaf(8.f, sv0[x], bf16_hi(p0));
          zv1[x] = fmaf(8.f, sv1[x], bf16_hi(p1));
          // a group that is not finite, a page that was not read, a token behind
          // the last one (which the mask takes out): not in the product
          if (key0 >= len || !good || !(fabsf(zv0[x]) < INFINITY)) {
            bad0 = NAN;
            sv0[x] = zv0[x] = 0.f;
          }
          if (key1 >= len || !good || !(fabsf(zv1[x]) < INFINITY)) {
            bad1 = NAN;
            sv1[x] = zv1[x] = 0.f;
          }
          svm = fmaxf(svm, fmaxf(sv0[x], sv1[x]));
        }
      }
      // ---- masks; reference maxima and the V power move only when they must ----
      bool move = svm > sig_max;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int last = lim[t][e] < len - 1 ? lim[t][e] : len - 1;
          s[t][e] = key0 <= last ? s[t][e] + bad0 : -INFINITY;
          s[t][2 + e] = key1 <= last ? s[t][2 + e] + bad1 : -INFINITY;
          move = move || fmaxf(s[t][e], s[t][2 + e]) > m[t][e] + 8.f;
        }
      if (__any_sync(0xffffffffu, move)) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) svm = fmaxf(svm, __shfl_xor_sync(0xffffffffu, svm, k));
        float turn = 1.f;
        if (svm > sig_max) {  // the same in every lane
          // sig = 2^(3 - floor(log2 svm)): s * sig in [8, 16) now, at most 128 before it moves again
          int ex = 257 - (int)(__float_as_uint(svm) >> 23);
          ex = ex > 253 ? 253 : ex < 1 ? 1 : ex;
          const float ns = __uint_as_float((uint32_t)ex << 23);
          turn = ns / sig;
          sig = ns;
          sig_max = 128.f / ns;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(m[t][e], fmaxf(s[t][e], s[t][2 + e]));
#pragma unroll
            for (int k = 4; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
            const float c = ka_ex2(m[t][e] - top);
            m[t][e] = top;
            l[t][e] *= c;
#pragma unroll
            for (int x = 0; x < NG; ++x) zs[t][x][e] *= c;
            f[e] = c * turn;
          }
#pragma unroll
          for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][x][e] *= f[e & 1];
#pragma unroll
          for (int x = 0; x < NG; ++x)
#pragma unroll
            for (int e = 0; e < 4; ++e) o1[t][x][e] *= f[e & 1];
        }
      }
      // ---- p, its sums, and P^T fragments ----
      uint32_t pb[NT][NG][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) p[e] = ka_ex2(s[t][e] - m[t][e & 1]);
        l[t][0] += p[0] + p[2];
        l[t][1] += p[1] + p[3];
#pragma unroll
        for (int x = 0; x < NG; ++x) {
          zs[t][x][0] += fmaf(p[0], zv0[x], p[2] * zv1[x]);
          zs[t][x][1] += fmaf(p[1], zv0[x], p[3] * zv1[x]);
          const float f0 = sv0[x] * sig, f1 = sv1[x] * sig;
          pb[t][x][0] = transpose8x8(pack_f16x2(p[0] * f0, p[1] * f0));
          pb[t][x][1] = transpose8x8(pack_f16x2(p[2] * f1, p[3] * f1));
        }
      }
      // ---- O^T += V^T P^T ----
      {
        const uint8_t* vb = blk + KV4_VOFF + warp * 1024 + lane * 16;
        const uint4 v0 = *reinterpret_cast<const uint4*>(vb), v1 = *reinterpret_cast<const uint4*>(vb + 512);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int x = j * NG / 4;
          const uint32_t sel = (j & 1) ? 0x7632 : 0x5410;
          const uint32_t w0 = __byte_perm(j < 2 ? v0.x : v0.y, j < 2 ? v0.z : v0.w, sel);
          const uint32_t w1 = __byte_perm(j < 2 ? v1.x : v1.y, j < 2 ? v1.z : v1.w, sel);
          const uint32_t a00 = code_f16<0>(w0), a01 = code_f16<1>(w0), a02 = code_f16<2>(w0), a03 = code_f16<3>(w0);
          const uint32_t a10 = code_f16<0>(w1), a11 = code_f16<1>(w1), a12 = code_f16<2>(w1), a13 = code_f16<3>(w1);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma_f16(o[t][2 * j], a00, a01, a10, a11, pb[t][x][0], pb[t][x][1]);
            mma_f16(o[t][2 * j + 1], a02, a03, a12, a13, pb[t][x][0], pb[t][x][1]);
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int x = 0; x < NG; ++x)
            mma_f16(o1[t][x], 0x3E003E00u, 0x3E003E00u, 0x3E003E00u, 0x3E003E00u, pb[t][x][0], pb[t][x][1]);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(&sm.empty[st]);
    if (tid == 0 && sent < n) {  // the stage that page i - 1 has left
      bool fre = true;
      if (i > 0) fre = mbar_wait(&sm.empty[(i - 1) % KA_STAGES], ((i - 1) / KA_STAGES) & 1, 0x302);
      if (fre)
        send();
      else
        ok = false;
    }
    __syncwarp();
    const bool last_page = at.page + 1 == at.pages;
    if (last_page || i + 1 == n) {
      // ---- the item ends here, or this CTA's piece of it: join the warps ----
      failed = __syncthreads_or(!ok);  // also: the last item's tiles have been read
      if (failed) break;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float back = 16.f / sig;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int k = 4; k < 32; k <<= 1) {
            l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], k);
#pragma unroll
            for (int x = 0; x < NG; ++x) zs[t][x][e] += __shfl_xor_sync(0xffffffffu, zs[t][x][e], k);
          }
          const int r = t * 8 + 2 * cq + e;
          if (g == 0) {
            sm.m[warp][r] = m[t][e];
            sm.l[warp][r] = l[t][e];
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int x = j * NG / 4;
            const float c1 = o1[t][x][e], z = zs[t][x][e];
            *reinterpret_cast<float4*>(&sm.o[warp][r][32 * j + 4 * g]) =
                make_float4(fmaf(o[t][2 * j][e] - c1, back, z), fmaf(o[t][2 * j][2 + e] - c1, back, z),
                            fmaf(o[t][2 * j + 1][e] - c1, back, z), fmaf(o[t][2 * j + 1][2 + e] - c1, back, z));
          }
        }
      }
      __syncthreads();
      const bool whole = item_start == 0 && last_page;
      float* slot = a.part + (size_t)(2 * blockIdx.x + (item_start == 0 ? 1 : 0)) * (R * (KV4_D + 2));
#pragma unroll 1
      for (int r = warp; r < R; r += 4) {
        const int rr = at.rt * R + r, tok = rr / a.G, head = at.h * a.G + (rr - tok * a.G);
        if (tok >= at.count) break;
        const float top = fmaxf(fmaxf(sm.m[0][r], sm.m[1][r]), fmaxf(sm.m[2][r], sm.m[3][r]));
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = ka_ex2(sm.m[w][r] - top);
          const float4 x = *reinterpret_cast<const float4*>(&sm.o[w][r][4 * lane]);
          sum = fmaf(sm.l[w][r], f, sum);
          v.x = fmaf(x.x, f, v.x);
          v.y = fmaf(x.y, f, v.y);
          v.z = fmaf(x.z, f, v.z);
          v.w = fmaf(x.w, f, v.w);
        }
        if (whole) {
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
      if (i + 1 == n && tid == 0) {
        int4 cut = make_int4(-1, 0, 0, 0);
        if (item_start == 0 && !last_page) {
          // its last page is page u1 - 1 + (pages - 1 - at.page) of the line
          const long long end = u1 - 1 + (at.pages - 1 - at.page);
          long long z = (end * ctas) / total;
          while (total * (z + 1) / ctas <= end) ++z;
          while (total * z / ctas > end) --z;
          cut = make_int4(at.b, at.rt, at.h, (int)z);
        }
        a.cut[blockIdx.x] = cut;
      }
      item = false;
    }
    if (i + 1 < n) ka_next<R>(a, at);
  }
  // a failed wait (reported in the status word) leaves copies under way: let
  // them land before this CTA's shared memory is given up
  if (tid == 0) {
    const uint64_t t0 = globaltimer_ns();
    for (int i = sent > KA_STAGES ? sent - KA_STAGES : 0; i < sent; ++i)
      while (!mbar_try_wait(smem_u32(&sm.full[i % KA_STAGES]), (i / KA_STAGES) & 1) &&
             globaltimer_ns() - t0 < kWaitLimitNs) {
      }
    if (failed) a.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
  }
}

// Joins the pieces of the items that were cut: CTA (x, y) takes row y of the
// item that starts in attention CTA x and goes on to CTA cut[x].w. Its pieces
// are slot 2 x + 1 and slots 2 i, i = x + 1 .. w, taken in that order by four
// warps in turn, whose sums are added in warp order.
template <int R>
__global__ void __launch_bounds__(128) kv4_join_kernel(const KaArgs a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float sm_m[4], sm_l[4];
  __shared__ float4 sm_o[4][32];
  const int4 cut = a.cut[blockIdx.x];
  if (cut.x < 0) return;
  const int warp = warp_id(), lane = lane_id(), r = blockIdx.y;
  int first, count;
  kv4_rows(a.c, cut.x, &first, &count);
  const int rr = cut.y * R + r, tok = rr / a.G;
  if (tok >= count) return;
  const int pieces = cut.w - (int)blockIdx.x + 1;
  constexpr int SLOT = R * (KV4_D + 2);
  auto slot = [&](int i) { return a.part + (size_t)(2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * SLOT; };
  float top = -FLT_MAX;
  for (int i = threadIdx.x; i < pieces; i += 128) top = fmaxf(top, slot(i)[R * KV4_D + r]);
#pragma unroll
  for (int k = 1; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
  if (lane == 0) sm_m[warp] = top;
  __syncthreads();
  top = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
  float sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp; i < pieces; i += 4) {
    const float* s = slot(i);
    const float f = ka_ex2(s[R * KV4_D + r] - top);
    const float4 x = *reinterpret_cast<const float4*>(s + r * KV4_D + 4 * lane);
    sum = fmaf(s[R * KV4_D + R + r], f, sum);
    v.x = fmaf(x.x, f, v.x);
    v.y = fmaf(x.y, f, v.y);
    v.z = fmaf(x.z, f, v.z);
    v.w = fmaf(x.w, f, v.w);
  }
  sm_o[warp][lane] = v;
  if (lane == 0) sm_l[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    sum = (sm_l[0] + sm_l[1]) + (sm_l[2] + sm_l[3]);
    const float4 x0 = sm_o[0][lane], x1 = sm_o[1][lane], x2 = sm_o[2][lane], x3 = sm_o[3][lane];
    const size_t orow = (size_t)(first + tok) * a.c.heads * a.G + cut.z * a.G + (rr - tok * a.G);
    const float f = (sum == 0.f ? 0.f : 1.f / sum) * (a.gate ? __ldg(a.gate + orow) : 1.f);
    *reinterpret_cast<uint2*>(a.out + orow * KV4_D + 4 * lane) =
        make_uint2(pack_bf16x2(((x0.x + x1.x) + (x2.x + x3.x)) * f, ((x0.y + x1.y) + (x2.y + x3.y)) * f),
                   pack_bf16x2(((x0.z + x1.z) + (x2.z + x3.z)) * f, ((x0.w + x1.w) + (x2.w + x3.w)) * f));
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Many rows a sequence and K/V head: the tcgen05 kernel over f16 operands in
// the workspace. Below this the page kernel above, which reads the cache once
// per 16 rows, is faster than laying the operands out.
constexpr int KV4_TC_MIN = 64;
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
static int ka_ctas(int R) { return sm_count() * (R == 8 ? 4 : 3); }
static uint64_t ka_workspace(int R) {
  const uint64_t n = ka_ctas(R);
  return n * 16 + n * 2 * R * (KV4_D + 2) * 4;
}

template <int NG, int R>
static int ka_launch(const KaArgs& a, cudaStream_t st) {
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
  const int ctas = ka_ctas(R);
  kv4_attn_kernel<NG, R><<<ctas, KA_THREADS, bytes, st>>>(a);
  launched();
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "kv4 attention launch");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas, R);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute la[1];
  la[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  la[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = la;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kv4_join_kernel<R>, a);
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
  return ka_workspace(ka_rows(rows, c.batch, H / c.heads));
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
  if (!tc) need = ka_workspace(R);
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
  a.cut = static_cast<int4*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (size_t)ka_ctas(R) * 16);
  const int ng = KV4_D / cache->group;
  if (R == 8) {
    if (ng == 1) return ka_launch<1, 8>(a, st);
    if (ng == 2) return ka_launch<2, 8>(a, st);
    return ka_launch<4, 8>(a, st);
  }
  if (ng == 1) return ka_launch<1, 16>(a, st);
  if (ng == 2) return ka_launch<2, 16>(a, st);
  return ka_launch<4, 16>(a, st);
}

}  // extern "C"
