// out[M, N] = A[M, K] . dequant(Wq[N, K], scales)^T (+ bias) with 4-bit
// weights: w = (code - 8) * scale, one scale per group of 32, 64 or 128
// columns of a row, two codes a byte (low half the even column).
//
// Few rows (up to DQ4_STREAM_ROWS): bound by the weights' bytes (N K / 2 plus
// scales). The codes go to the tensor cores as they are: a nibble alone in the
// lowest mantissa bits of an f16 is the subnormal code * 2^-24, in the next
// four bits code * 2^-20, both exact, so one shift and four masks unpack eight
// codes into four operand registers of mma.m16n8k16. A's rows enter as f16
// after a power of two per row and 256 columns (16 times larger where they meet
// the first kind of nibble; a bf16 value stays exact down to 2^-27 of the
// largest of the 256), and the accumulator of a group starts from -8 sum x, so
// that
//   sum_k x (c - 8) s = s (sum x c - 8 sum x)
// needs one f32 FMA per group and output. Products are exact, sums f32.
//
// A CTA takes 128 weight rows and 1 / S of K: a producer warp streams [rows x
// 128 bytes] tiles (TMA, 256 columns) through a ring, eight warps take 16 rows
// each, both 128-column blocks of a tile side by side. A's records (its values in the order of the B fragments, the
// groups' sums) come through the same ring from a kernel of their own, which
// runs under this one's start; where a CTA has few values of A (DQ4_OWN), its
// warps make them in shared memory while the ring fills. The S CTAs of a
// cluster add their f32 partials in rank order through distributed shared
// memory. S fills the SMs where N alone does not: the largest power of two up
// to 8 that keeps the CTAs within what the SMs hold at once.
// Measured: 2 x 36,864 x 4,096, groups of 64, f32 scales: 25 us (85 MB, 3.4
// TB/s); 8 x 36,864 x 4,096, groups of 128: 24 us; 16 x 4,096 x 16,384, groups
// of 32: 28 us; 16 x 16,384 x 4,096: 22 us. What bounds it there is the start
// (A's records, first tiles: 3.5 us), the instructions of a tile (the scale
// and start value of every group and output) and their latencies, and where K is
// split (not with 36,864 rows) the cluster's sum (3 us), no longer the bytes. (Four warps of 32 rows each: 27, 27, 42 and 21 us.)
//
// 17 to 1,024 rows (DQ4_TC_ROWS): the tcgen05 kernel of dq4_tc.cu, which makes
// bf16 weights (one rounding: the code and a bf16 scale have up to 11
// significant bits) in shared memory. The way above with four row tiles took 64
// us for 32 x 36,864 x 4,096 (58 there), 73 for 32 x 4,096 x 16,384 (35) and 126
// for 64 x 36,864 x 4,096 (59).
// More rows: the same bf16 weights in the workspace, multiplied by the tcgen05
// GEMM, as for int8 weights. There the two meet: 1,024 rows in the tcgen05 kernel
// and 1,025 here 287 and 316 us (36,864 x 4,096), 164 and 160 (16,384 x 4,096),
// 135 and 148 (4,096 x 16,384); at 2,048 262 and about 245 (16,384 x 4,096).
#include <atomic>

#include "common.cuh"
#include "kernels.h"

namespace ltxb {

constexpr int DQ4_STREAM_ROWS = 16, DQ4_TC_ROWS = 1024;
constexpr int DQ4_WARPS = 8, DQ4_THREADS = 32 * (DQ4_WARPS + 1);
constexpr int DQ4_TILE = 128, DQ4_PER_SM = 2;  // weight rows of a CTA, CTAs an SM
constexpr int DQ4_OWN = 2048;      // values of A (rows x columns of a CTA) that a CTA puts in order itself
constexpr int DQ4_OWN_RECORDS = 8; // 2048 columns

// A's record of 256 columns for NT tiles of 8 rows in shared memory: per block
// of 128 the fragments [tile][word 0 .. 3][lane] of 16 bytes and the
// accumulators' initial values -8 * 2^-20 * sum x, f32 [group][8 NT]; then
// 1 / the rows' powers of two, f32 [8 NT].
__host__ __device__ constexpr int dq4_block(int ng, int nt) { return 2048 * nt + 32 * ng * nt; }
__host__ __device__ constexpr int dq4_record(int ng, int nt) { return 2 * dq4_block(ng, nt) + 32 * nt; }

struct Dq4Args {
  const void* scales;
  const __nv_bfloat16* bias;
  __nv_bfloat16* out;
  const __nv_bfloat16* a;
  const uint8_t* rec;  // [K / 256] records, or null: made from `a` by the CTA
  int M, N, K, splits;
};

__device__ __forceinline__ void dq4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t dq4_pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t dq4_lo(uint32_t w) { return w & 0x000F000Fu; }
__device__ __forceinline__ uint32_t dq4_hi(uint32_t w) { return w & 0x00F000F0u; }

// Word y = 0 .. 3 of lane quarter c in a block of 128 columns covers columns
// dq4_col(y, c) .. + 7 and lies in group y NG / 4 (NG = 128 / group): a quad's
// four words make up 32 columns of one group.
template <int NG>
__device__ __forceinline__ int dq4_col(int y, int c) {
  return NG == 1 ? 32 * c + 8 * y : NG == 2 ? 64 * (y >> 1) + 16 * c + 8 * (y & 1) : 32 * y + 8 * c;
}
// The NG scales of one row and block: one aligned load.
template <int NG, bool BF>
__device__ __forceinline__ void dq4_scales(const void* s, size_t i, float (&v)[NG]) {
  if (BF) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(s) + i * NG;
    if (NG == 1) {
      v[0] = __uint_as_float((uint32_t)__ldg(p) << 16);
    } else if (NG == 2) {
      const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(p));
      v[0] = bf16_lo(w), v[NG - 1] = bf16_hi(w);
    } else {
      const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
      v[0] = bf16_lo(w.x), v[1 % NG] = bf16_hi(w.x), v[2 % NG] = bf16_lo(w.y), v[3 % NG] = bf16_hi(w.y);
    }
  } else {
    const float* p = reinterpret_cast<const float*>(s) + i * NG;
    if (NG == 1) {
      v[0] = __ldg(p);
    } else if (NG == 2) {
      const float2 w = __ldg(reinterpret_cast<const float2*>(p));
      v[0] = w.x, v[NG - 1] = w.y;
    } else {
      const float4 w = __ldg(reinterpret_cast<const float4*>(p));
      v[0] = w.x, v[1 % NG] = w.y, v[2 % NG] = w.z, v[3 % NG] = w.w;
    }
  }
}
__device__ __forceinline__ float dq4_scale(const void* s, int is_bf16, size_t i) {
  return is_bf16 ? __uint_as_float((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(s) + i) << 16)
                 : __ldg(reinterpret_cast<const float*>(s) + i);
}

// One warp: columns [k0, k0 + 256) of the row at `row` (zeros from K on, or
// everywhere if there is no row) into the record `rec`, as row j of the 8 NT.
template <int NG, int NT>
__device__ __forceinline__ void dq4_put(const __nv_bfloat16* __restrict__ row, int k0, int K, int j, uint8_t* rec) {
  const int lane = lane_id(), t = j >> 3, g = j & 7;
  const int k = k0 + 8 * lane;
  const uint4 v = row && k < K ? __ldg(reinterpret_cast<const uint4*>(row + k)) : make_uint4(0, 0, 0, 0);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  // The largest finite value; the group's sum, of values times 2^-8: as they
  // come, 32 of 1.1e37 pass the largest f32. (bf16's last place is 2^-133: exact.)
  float top = 0.f, s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = bf16_lo(w[i]), y = bf16_hi(w[i]);
    if (fabsf(x) < INFINITY) top = fmaxf(top, fabsf(x));
    if (fabsf(y) < INFINITY) top = fmaxf(top, fabsf(y));
    s = fmaf(x, 0.00390625f, fmaf(y, 0.00390625f, s));
  }
#pragma unroll
  for (int i = 1; i < 32; i <<= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    if (i < 16 / NG) s += __shfl_xor_sync(0xffffffffu, s, i);
  }
  int field = 264 - (int)(__float_as_uint(top) >> 23);  // the largest value into [2^10, 2^11)
  field = field < 1 ? 1 : field > 249 ? 249 : field;
  const float f = __uint_as_float((uint32_t)field << 23), f16 = 16.f * f;
  // the lane's eight columns are word y of lane quarter c (a quad's four words of one y make up 32 columns of a group)
  const int q = lane & 15;
  const int y = NG == 1 ? q & 3 : NG == 2 ? 2 * (q >> 3) + (q & 1) : q >> 2;
  const int c = NG == 1 ? q >> 2 : NG == 2 ? (q >> 1) & 3 : q & 3;
  uint8_t* blk = rec + (lane >> 4) * dq4_block(NG, NT);
  *reinterpret_cast<uint4*>(blk + ((t * 4 + y) * 32 + g * 4 + c) * 16) =
      make_uint4(dq4_pack(bf16_lo(v.x) * f16, bf16_lo(v.z) * f16), dq4_pack(bf16_hi(v.x) * f, bf16_hi(v.z) * f),
                 dq4_pack(bf16_lo(v.y) * f16, bf16_lo(v.w) * f16), dq4_pack(bf16_hi(v.y) * f, bf16_hi(v.w) * f));
  if ((lane & (16 / NG - 1)) == 0)
    *reinterpret_cast<float*>(blk + 2048 * NT + ((q / (16 / NG)) * 8 * NT + j) * 4) = s * f * -0.001953125f;  // 2^8 * -8 * 2^-20
  if (lane == 0)
    *reinterpret_cast<float*>(rec + 2 * dq4_block(NG, NT) + j * 4) = __uint_as_float((uint32_t)(254 - field) << 23);
}

// All records of A, a warp each (row of the 8 NT, 256 columns).
template <int NG, int NT>
__global__ void __launch_bounds__(256) dq4_rows_kernel(const __nv_bfloat16* __restrict__ A, int M, int K, int tasks,
                                                       uint8_t* __restrict__ rec) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int n = (K + 255) / 256;
  const int x = blockIdx.x * 8 + warp_id();
  if (x >= tasks) return;
  const int m = x / n, r = x - m * n;
  dq4_put<NG, NT>(m < M ? A + (size_t)m * K : nullptr, r * 256, K, m, rec + (size_t)r * dq4_record(NG, NT));
}

__device__ __forceinline__ void dq4_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// (Not the .aligned form: that one needs a warp's lanes to come together, and
// they come from loops of unequal length.)
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr, uint32_t rank) {
  float4 v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [a];\n\t}"
      : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
      : "r"(addr), "r"(rank)
      : "memory");
  return v;
}

template <int NG, int NT, bool OWN>
struct Dq4Cfg {
  static constexpr int RT = 1, ROWS = 16 * RT * DQ4_WARPS;  // tiles of 16 weight rows a warp; weight rows of a CTA
  static constexpr int WBYTES = ROWS * 128, RECORD = dq4_record(NG, NT);
  static constexpr int STAGE = WBYTES + (OWN ? 0 : (RECORD + 1023) / 1024 * 1024);  // 1 KB: the swizzled tile's alignment
  static constexpr int PER_SM = DQ4_PER_SM;
  static constexpr int STAGES = 4;
  static constexpr int PART = 8 * NT * (ROWS + 4) * 4;
  static constexpr int SMEM = STAGES * STAGE + (OWN ? DQ4_OWN_RECORDS * RECORD : 0) + 1024 + 256;
  static_assert(PART <= STAGES * STAGE, "the partials take the ring's place");
};

template <int NG, int NT, bool BF, bool OWN>
__global__ void __launch_bounds__(DQ4_THREADS, Dq4Cfg<NG, NT, OWN>::PER_SM)
    dq4_stream_kernel(const __grid_constant__ CUtensorMap tmW, const Dq4Args p) {
  using C = Dq4Cfg<NG, NT, OWN>;
  constexpr int RT = C::RT;
  extern __shared__ uint8_t dq4_raw[];
  uint8_t* ring = dq4_raw + (-smem_u32(dq4_raw) & 1023u);
  uint8_t* recs = ring + C::STAGES * C::STAGE;  // OWN: this CTA's records
  uint64_t* full = reinterpret_cast<uint64_t*>(recs + (OWN ? DQ4_OWN_RECORDS * C::RECORD : 0));
  uint64_t* empty = full + C::STAGES;
  const int warp = warp_id(), lane = lane_id(), g = lane >> 2, c = lane & 3;
  // MMA row g stands for weight row pg of eight: the rows whose words a quarter or
  // half of a warp loads together then lie in different banks of the swizzled tile
  const int pg = ((g & 1) << 2) | (g & 2) | (g >> 2);
  const int n0 = blockIdx.x * C::ROWS, rank = blockIdx.y, S = p.splits;
  const int nkb = p.K / 128;
  // whole stages of 256 columns
  const int nst = (nkb + 1) / 2, kb0 = 2 * (int)((long long)rank * nst / S);
  int kb1 = 2 * (int)((long long)(rank + 1) * nst / S);
  if (kb1 > nkb) kb1 = nkb;
  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], DQ4_WARPS);
    }
    fence_mbar_init();
  }
  __syncthreads();
  float tot[RT][NT][4];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < NT; ++t) tot[r][t][0] = tot[r][t][1] = tot[r][t][2] = tot[r][t][3] = 0.f;
  bool ok = true;
  if (warp == DQ4_WARPS) {
    // ---------------- producer ----------------
    const int n = (kb1 - kb0 + 1) / 2;  // stages of two blocks; the last may hold one
    if (lane == 0) {
      prefetch_tmap(&tmW);
      const uint8_t* rec = OWN ? nullptr : p.rec + (size_t)(kb0 / 2) * C::RECORD;
      auto weights = [&](int i) {  // columns past K come as zeros and are not multiplied
        const int st = i % C::STAGES;
        mbar_arrive_expect_tx(&full[st], C::WBYTES + (OWN ? 0 : C::RECORD));
        tma_load_2d(ring + st * C::STAGE, &tmW, &full[st], (kb0 + 2 * i) * 64, n0);
      };
      auto record = [&](int i) {
        const int st = i % C::STAGES;
        if (!OWN) dq4_bulk(ring + st * C::STAGE + C::WBYTES, rec + (size_t)i * C::RECORD, C::RECORD, &full[st]);
      };
      const int head = n < C::STAGES ? n : C::STAGES;
      for (int i = 0; i < head; ++i) weights(i);
      if (!OWN) asm volatile("griddepcontrol.wait;" ::: "memory");  // the weights do not wait for A's records
      for (int i = 0; i < head; ++i) record(i);
      for (int i = head; i < n && ok; ++i) {
        ok = mbar_wait(&empty[i % C::STAGES], (i / C::STAGES - 1) & 1, 0x321);
        if (!ok) break;
        weights(i);
        record(i);
      }
    }
    __syncwarp();
  } else {
    // ---------------- 16 RT weight rows a warp ----------------
    const int wrow = warp * 16 * RT;
    size_t srow[RT][2];  // scale blocks (NG scales) of the lane's rows
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int n = n0 + wrow + r * 16 + e * 8 + pg;
        srow[r][e] = (size_t)(n < p.N ? n : p.N - 1) * nkb + kb0;
      }
    const int nb = kb1 - kb0;
    float sc[2][RT][2][NG], sn[2][RT][2][NG];  // this stage's scales and the next one's
    auto fetch = [&](int i, float (&s)[2][RT][2][NG]) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e) dq4_scales<NG, BF>(p.scales, srow[r][e] + (i + b < nb ? i + b : nb - 1), s[b][r][e]);
    };
    fetch(0, sc);
    if (OWN) {
      const int n = (nb + 1) / 2;
      for (int i = threadIdx.x; i < n * C::RECORD / 16; i += DQ4_WARPS * 32)  // rows past M stay zeros
        reinterpret_cast<uint4*>(recs)[i] = make_uint4(0, 0, 0, 0);
      __syncwarp();  // (the barrier takes whole warps; the loop's last step only some of their lanes)
      named_bar(1, DQ4_WARPS * 32);
#pragma unroll 1
      for (int x = warp; x < n * p.M; x += DQ4_WARPS) {
        const int j = x / n, r = x - j * n;
        dq4_put<NG, NT>(p.a + (size_t)j * p.K, (kb0 + 2 * r) * 128, p.K, j, recs + r * C::RECORD);
      }
      __syncwarp();
      named_bar(1, DQ4_WARPS * 32);
    }
    for (int i = 0; i < nb; i += 2) {
      const int st = (i >> 1) % C::STAGES;
      if (ok) ok = warp_wait(&full[st], ((i >> 1) / C::STAGES) & 1, 0x322);
      if (!ok) break;
      const uint8_t* rec = OWN ? recs + (i >> 1) * C::RECORD : ring + st * C::STAGE + C::WBYTES;
      if (i + 2 < nb) fetch(i + 2, sn);
      const uint8_t* ws = ring + st * C::STAGE;
      float sum[RT][NT][4];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < NT; ++t) sum[r][t][0] = sum[r][t][1] = sum[r][t][2] = sum[r][t][3] = 0.f;
      // The stage's two blocks side by side (independent sums); a block past K
      // has zeros on A's side and takes the last block's scales.
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        float acc[2][RT][NT][4];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const float2 v = *reinterpret_cast<const float2*>(rec + b * dq4_block(NG, NT) + 2048 * NT +
                                                              (x * 8 * NT + t * 8 + 2 * c) * 4);
#pragma unroll
            for (int r = 0; r < RT; ++r) acc[b][r][t][0] = acc[b][r][t][2] = v.x, acc[b][r][t][1] = acc[b][r][t][3] = v.y;
          }
        uint32_t w[2][RT][2][4 / NG];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              // 128-byte rows, 16-byte chunk j of row n at j ^ (n % 8)
              const uint8_t* rp = ws + (wrow + r * 16 + e * 8 + pg) * 128;
              uint32_t(&d)[4 / NG] = w[b][r][e];
              if (NG == 1) {
                const uint4 v = *reinterpret_cast<const uint4*>(rp + (((4 * b + c) ^ pg) << 4));
                d[0] = v.x, d[1 % (4 / NG)] = v.y, d[2 % (4 / NG)] = v.z, d[3 % (4 / NG)] = v.w;
              } else if (NG == 2) {
                const uint2 v = *reinterpret_cast<const uint2*>(rp + (((4 * b + 2 * x + (c >> 1)) ^ pg) << 4) + (c & 1) * 8);
                d[0] = v.x, d[1 % (4 / NG)] = v.y;
              } else {
                d[0] = *reinterpret_cast<const uint32_t*>(rp + (((4 * b + x) ^ pg) << 4) + 4 * c);
              }
            }
#pragma unroll
        for (int yy = 0; yy < 4 / NG; ++yy)
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const int y = x * (4 / NG) + yy;
            uint32_t lo[RT][4], hi[RT][4];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const uint32_t a0 = w[b][r][0][yy], a1 = w[b][r][1][yy], a2 = a0 >> 8, a3 = a1 >> 8;
              lo[r][0] = dq4_lo(a0), lo[r][1] = dq4_lo(a1), lo[r][2] = dq4_lo(a2), lo[r][3] = dq4_lo(a3);
              hi[r][0] = dq4_hi(a0), hi[r][1] = dq4_hi(a1), hi[r][2] = dq4_hi(a2), hi[r][3] = dq4_hi(a3);
            }
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              const uint4 q = *reinterpret_cast<const uint4*>(rec + b * dq4_block(NG, NT) + ((t * 4 + y) * 32 + lane) * 16);
#pragma unroll
              for (int r = 0; r < RT; ++r) {
                dq4_mma(acc[b][r][t], lo[r][0], lo[r][1], hi[r][0], hi[r][1], q.x, q.y);
                dq4_mma(acc[b][r][t], lo[r][2], lo[r][3], hi[r][2], hi[r][3], q.z, q.w);
              }
            }
          }
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int e = 0; e < 4; ++e) sum[r][t][e] = fmaf(acc[b][r][t][e], sc[b][r][e >> 1][x], sum[r][t][e]);
          }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {  // out of the rows' powers of two
        const float2 f = *reinterpret_cast<const float2*>(rec + 2 * dq4_block(NG, NT) + (t * 8 + 2 * c) * 4);
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 4; ++e) tot[r][t][e] = fmaf(sum[r][t][e] * 1048576.f, e & 1 ? f.y : f.x, tot[r][t][e]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int x = 0; x < NG; ++x) sc[b][r][e][x] = sn[b][r][e][x];
    }
  }
  // ---- partials [8 NT columns][ROWS] in the ring's place, added over the cluster in rank order ----
  const bool failed = __syncthreads_or(!ok);
  float* part = reinterpret_cast<float*>(ring);
  if (failed) {  // (reported in the status word) copies under way land before the ring is given up
    if (threadIdx.x == DQ4_WARPS * 32) {
      const uint64_t t0 = globaltimer_ns();
      for (int i = 0; i < C::STAGES; ++i)
        for (int ph = 0; ph < 2; ++ph)
          while (!mbar_try_wait(smem_u32(&full[i]), ph) && globaltimer_ns() - t0 < 10000000ull) {
          }
    }
  } else if (warp < DQ4_WARPS) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          part[(t * 8 + 2 * c + (e & 1)) * (C::ROWS + 4) + warp * 16 * RT + r * 16 + (e >> 1) * 8 + pg] = tot[r][t][e];
  }
  if (S > 1)
    cluster_sync();
  else
    __syncthreads();
  const int lp = 29 - __clz(C::ROWS / S);  // this CTA's share: ROWS / S rows, four a thread
  for (int i = threadIdx.x; i < p.M << lp; i += DQ4_THREADS) {
    const int j = i >> lp, n = ((rank << lp) + (i - (j << lp))) * 4, m = j;
    if (failed || n0 + n >= p.N) continue;
    const float* at = part + j * (C::ROWS + 4) + n;
    float4 v = *reinterpret_cast<const float4*>(at);
    if (S > 1) {
      const uint32_t a = smem_u32(at);
      float4 x[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) x[r] = r < S ? ld_cluster4(a, r) : make_float4(0.f, 0.f, 0.f, 0.f);  // all under way at once
      v = x[0];
#pragma unroll
      for (int r = 1; r < 8; ++r) v.x += x[r].x, v.y += x[r].y, v.z += x[r].z, v.w += x[r].w;
    }
    if (p.bias) {
      const uint2 bb = __ldg(reinterpret_cast<const uint2*>(p.bias + n0 + n));
      v.x += bf16_lo(bb.x), v.y += bf16_hi(bb.x), v.z += bf16_lo(bb.y), v.w += bf16_hi(bb.y);
    }
    *reinterpret_cast<uint2*>(p.out + (size_t)m * p.N + n0 + n) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  }
  if (S > 1) cluster_sync();  // the others have read this CTA's partials
}

// Eight codes (4 bytes) -> 16 bytes of bf16 per thread and step, four steps
// under way: a warp reads and writes whole lines. Bound by 2.5 bytes a weight.
__global__ void __launch_bounds__(256) dq4_expand_kernel(const uint32_t* __restrict__ w, const void* __restrict__ scales,
                                                         int scale_bf16, int shift, size_t n8, uint4* __restrict__ out) {
  const size_t stride = (size_t)gridDim.x * blockDim.x;
  auto put = [&](size_t i, uint32_t v, float s) {
    uint32_t r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      // 2^23 + code and back: exact; (code - 8) * scale is rounded once more to bf16
      const float a = (__uint_as_float(((v >> (8 * k)) & 15u) | 0x4B000000u) - 8388616.f) * s;
      const float b = (__uint_as_float(((v >> (8 * k + 4)) & 15u) | 0x4B000000u) - 8388616.f) * s;
      r[k] = pack_bf16x2(a, b);
    }
    out[i] = make_uint4(r[0], r[1], r[2], r[3]);
  };
  size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x;
  for (; i + 3 * stride < n8; i += 4 * stride) {
    uint32_t v[4];
    float s[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      v[u] = __ldg(w + i + u * stride);
      s[u] = dq4_scale(scales, scale_bf16, (i + u * stride) >> shift);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) put(i + u * stride, v[u], s[u]);
  }
  for (; i < n8; i += stride) put(i, __ldg(w + i), dq4_scale(scales, scale_bf16, i >> shift));
}

// row tiles of 8 of a call
static int dq4_nt(int M) { return M <= 8 ? 1 : 2; }
// CTAs of a cluster: the largest power of two that the SMs hold at once
static int dq4_splits(int N, int K) {
  const int tiles = (N + DQ4_TILE - 1) / DQ4_TILE;
  int S = 1;
  while (S < 8 && (int64_t)tiles * S * 2 <= DQ4_PER_SM * sm_count() && K / 256 >= 2 * S) S *= 2;
  return S;
}
static bool dq4_own(int M, int K, int S) {
  const int cols = ((K + 255) / 256 + S - 1) / S * 256;
  return M <= 8 && cols <= DQ4_OWN_RECORDS * 256 && M * cols <= DQ4_OWN;
}
static uint64_t dq4_records_bytes(int M, int K) {  // for groups of 32, the largest
  return (uint64_t)((K + 255) / 256) * dq4_record(4, dq4_nt(M));
}

template <int NG, int NT, bool BF, bool OWN>
static int dq4_launch(const void* Wq, Dq4Args p, uint8_t* ws, cudaStream_t st) {
  using C = Dq4Cfg<NG, NT, OWN>;
  static std::atomic<bool> attr[kMaxDevices];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= kMaxDevices) return set_error(LTXB_EINVAL, "dq4_gemm: device %d out of range", dev);
  if (!attr[dev].load(std::memory_order_acquire)) {
    cudaError_t e = cudaFuncSetAttribute(dq4_stream_kernel<NG, NT, BF, OWN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e != cudaSuccess) return set_cuda_error(e, "dq4_gemm: cudaFuncSetAttribute");
    attr[dev].store(true, std::memory_order_release);
  }
  const int tiles = (p.N + C::ROWS - 1) / C::ROWS;
  CUtensorMap tm;
  if (int rc = make_tmap_2d(&tm, Wq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, p.K / 2, p.N, p.K / 2, 128, C::ROWS, CU_TENSOR_MAP_SWIZZLE_128B))
    return rc;
  cudaError_t e;
  const int tasks = 8 * NT * ((p.K + 255) / 256);
  if (!OWN) {
    p.rec = ws;
    dq4_rows_kernel<NG, NT><<<(tasks + 7) / 8, 256, 0, st>>>(p.a, p.M, p.K, tasks, ws);
    launched();
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(e, "dq4_gemm rows");
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(tiles, p.splits);
  cfg.blockDim = dim3(DQ4_THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute la[2];
  la[0].id = cudaLaunchAttributeClusterDimension;
  la[0].val.clusterDim.x = 1;
  la[0].val.clusterDim.y = p.splits;
  la[0].val.clusterDim.z = 1;
  la[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  la[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = la;
  // The early start pays while A's kernel is small: 8 x 36,864 x 4,096 24.0 us
  // with it, 25.5 without; 16 x 4,096 x 16,384 (1,024 warps of A's) 33.0 and 27.7.
  cfg.numAttrs = !OWN && tasks <= 512 ? 2 : 1;
  e = cudaLaunchKernelEx(&cfg, dq4_stream_kernel<NG, NT, BF, OWN>, tm, p);
  launched();
  return e == cudaSuccess ? LTXB_OK : set_cuda_error(e, "dq4_gemm launch");
}

template <int NG, bool BF>
static int dq4_stream(const void* Wq, Dq4Args p, void* workspace, cudaStream_t st) {
  const int nt = dq4_nt(p.M);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.splits = dq4_splits(p.N, p.K);
  if (nt == 1)
    return dq4_own(p.M, p.K, p.splits) ? dq4_launch<NG, 1, BF, true>(Wq, p, ws, st) : dq4_launch<NG, 1, BF, false>(Wq, p, ws, st);
  return dq4_launch<NG, 2, BF, false>(Wq, p, ws, st);
}

}  // namespace ltxb

using namespace ltxb;

extern "C" {

uint64_t ltxb_dq4_gemm_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K < 128) return 0;
  if (M > DQ4_TC_ROWS) return (uint64_t)N * K * 2;
  if (M > DQ4_STREAM_ROWS) return 0;
  return dq4_own(M, K, dq4_splits(N, K)) ? 0 : dq4_records_bytes(M, K);
}

int ltxb_dq4_gemm(const void* A, const void* Wq, const void* scales, int scale_dtype, int group, const void* bias,
                  void* out, int M, int N, int K, void* workspace, uint64_t workspace_bytes, void* stream) {
  if (scale_dtype != LTXB_DT_F32 && scale_dtype != LTXB_DT_BF16)
    return set_error(LTXB_EINVAL, "dq4_gemm: scale dtype must be LTXB_DT_F32 or LTXB_DT_BF16");
  if (group != 32 && group != 64 && group != 128) return set_error(LTXB_EINVAL, "dq4_gemm: group must be 32, 64 or 128");
  if (M < 0 || N <= 0 || K <= 0 || N % 32 || K % 128)
    return set_error(LTXB_EINVAL, "dq4_gemm: N must be a multiple of 32 and K of 128 (M %d, N %d, K %d)", M, N, K);
  if (M == 0) return LTXB_OK;
  auto a16 = [](const void* q) { return q && (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
  if (!a16(A) || !a16(Wq) || !a16(scales) || !a16(out) || (reinterpret_cast<uintptr_t>(bias) & 15))
    return set_error(LTXB_EINVAL, "dq4_gemm: A, weights, scales, bias and out must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sb = scale_dtype == LTXB_DT_BF16;
  cudaError_t e;
  const uint64_t need = ltxb_dq4_gemm_workspace_bytes(M, N, K);
  if (need && (!workspace || workspace_bytes < need))
    return set_error(LTXB_EINVAL, "dq4_gemm: workspace of %llu bytes is smaller than the %llu required",
                     (unsigned long long)workspace_bytes, (unsigned long long)need);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return set_error(LTXB_EINVAL, "dq4_gemm: workspace must be 16-byte aligned");
  if (M > DQ4_STREAM_ROWS && M <= DQ4_TC_ROWS)
    return dq4_gemm_tc(A, Wq, scales, sb, group, bias, out, M, N, K, st);
  if (M > DQ4_TC_ROWS) {
    GemmArgs g{};
    g.A = A;
    g.lda = K;
    g.B = workspace;
    g.ldb = K;
    g.M = M;
    g.N = N;
    g.K = K;
    g.epi = EPI_BF16;
    g.bias = bias;
    g.out = out;
    g.ldo = N;
    if (int rc = gemm_check(g, nullptr)) return rc;  // before the expansion is launched
    const size_t n8 = (size_t)N * K / 8;
    const size_t ctas = (n8 + 255) / 256, most = 8 * (size_t)sm_count();
    dq4_expand_kernel<<<(unsigned)(ctas < most ? ctas : most), 256, 0, st>>>(
        static_cast<const uint32_t*>(Wq), scales, sb, group == 128 ? 4 : group == 64 ? 3 : 2, n8, static_cast<uint4*>(workspace));
    launched();
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(e, "dq4_gemm expansion");
    return gemm_tc(g, st);
  }
  Dq4Args p{};
  p.scales = scales;
  p.bias = static_cast<const __nv_bfloat16*>(bias);
  p.out = static_cast<__nv_bfloat16*>(out);
  p.M = M;
  p.N = N;
  p.K = K;
  p.a = static_cast<const __nv_bfloat16*>(A);
  if (group == 128) return sb ? dq4_stream<1, true>(Wq, p, workspace, st) : dq4_stream<1, false>(Wq, p, workspace, st);
  if (group == 64) return sb ? dq4_stream<2, true>(Wq, p, workspace, st) : dq4_stream<2, false>(Wq, p, workspace, st);
  return sb ? dq4_stream<4, true>(Wq, p, workspace, st) : dq4_stream<4, false>(Wq, p, workspace, st);
}

}  // extern "C"
