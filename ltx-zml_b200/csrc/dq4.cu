// out[M, N] = A[M, K] . dequant(Wq[N, K], scales)^T (+ bias) with 4-bit
// weights: w = (code - 8) * scale, one scale per group of 32, 64 or 128
// columns of a row, two codes a byte (low half the even column).
//
// Few rows (up to DQ4_STREAM_ROWS): bound by the weights' bytes (N K / 2 plus
// scales). The codes go to the tensor cores as they are: in the top mantissa
// bits of a bf16 a code c reads u = 1 + c / 16, and
//   sum x (c - 8) s = 16 s (sum x u - 1.5 sum x)
// so unpacking costs one shift and one logic operation per two codes, the
// offset is the accumulator's initial value (one MMA with constant rows
// -1.5), and the scale is applied once per group to f32 sums. The products
// are exact; nothing is rounded before the output.
//
// A warp takes 16 weight rows as the M side of mma.m16n8k16 and up to 8 NT
// rows of A as the N side; the warps of a CTA share the 16 rows and split K.
// Lane 4 g + c loads weight rows g and g + 8, a quarter of each group's
// columns (16, 8 or 4 bytes for groups of 128, 64, 32), and A's row g at the
// same columns: both sides of a contraction may be permuted alike.
//
// More rows: the weights are expanded to bf16 in the workspace (one rounding:
// the code and a bf16 scale have up to 11 significant bits) and multiplied by
// the tcgen05 GEMM, as for int8 weights.
#include <atomic>

#include "common.cuh"
#include "kernels.h"

namespace ltxb {

constexpr int DQ4_THREADS = 256, DQ4_WARPS = 8;
constexpr int DQ4_STREAM_ROWS = 64;

struct Dq4Args {
  const __nv_bfloat16* a;
  const uint8_t* w;
  const void* scales;
  const __nv_bfloat16* bias;
  __nv_bfloat16* out;
  int M, N, K, scale_bf16;
};

__device__ __forceinline__ void dq4_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// bf16 pair (1 + c / 16) of nibbles I and I + 4 of w
template <int I>
__device__ __forceinline__ uint32_t dq4_code(uint32_t w) {
  const uint32_t s = I == 0 ? w << 3 : w >> (4 * I - 3);
  return (s & 0x00780078u) | 0x3F803F80u;
}

// Words y = 0 .. 3 of a lane in a block of 128 columns cover columns
// dq4_col(y) .. + 7 and lie in group y NG / 4 (NG = 128 / group).
template <int NG>
__device__ __forceinline__ int dq4_col(int y, int c) {
  return NG == 1 ? 32 * c + 8 * y : NG == 2 ? 64 * (y >> 1) + 16 * c + 8 * (y & 1) : 32 * y + 8 * c;
}
template <int NG>
__device__ __forceinline__ void dq4_load(const uint8_t* row, int c, uint32_t (&w)[4]) {
  if (NG == 1) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + 16 * c));
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if (NG == 2) {
    const uint2 v0 = __ldg(reinterpret_cast<const uint2*>(row + 8 * c));
    const uint2 v1 = __ldg(reinterpret_cast<const uint2*>(row + 32 + 8 * c));
    w[0] = v0.x, w[1] = v0.y, w[2] = v1.x, w[3] = v1.y;
  } else {
#pragma unroll
    for (int y = 0; y < 4; ++y) w[y] = __ldg(reinterpret_cast<const uint32_t*>(row + 16 * y + 4 * c));
  }
}
__device__ __forceinline__ float dq4_scale(const void* s, int is_bf16, size_t i) {
  return is_bf16 ? __uint_as_float((uint32_t)__ldg(reinterpret_cast<const uint16_t*>(s) + i) << 16)
                 : __ldg(reinterpret_cast<const float*>(s) + i);
}

template <int NG, int NT>
__global__ void __launch_bounds__(DQ4_THREADS) dq4_stream_kernel(const Dq4Args p) {
  __shared__ float red[DQ4_WARPS][16][8 * NT + 1];
  const int warp = warp_id(), lane = lane_id(), g = lane >> 2, c = lane & 3;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 8 * NT;
  const int nkb = p.K / 128;
  const int kb0 = warp * nkb / DQ4_WARPS, kb1 = (warp + 1) * nkb / DQ4_WARPS;
  const uint8_t* w0 = p.w + (size_t)(n0 + g) * (p.K / 2);
  const uint8_t* w1 = w0 + (size_t)8 * (p.K / 2);
  const size_t s0 = (size_t)(n0 + g) * (nkb * NG), s1 = s0 + (size_t)8 * (nkb * NG);
  float tot[NT][4];
#pragma unroll
  for (int t = 0; t < NT; ++t) tot[t][0] = tot[t][1] = tot[t][2] = tot[t][3] = 0.f;
  uint32_t u0[4], u1[4];
  if (kb0 < kb1) {
    dq4_load<NG>(w0 + (size_t)kb0 * 64, c, u0);
    dq4_load<NG>(w1 + (size_t)kb0 * 64, c, u1);
  }
  for (int kb = kb0; kb < kb1; ++kb) {
    uint32_t v0[4], v1[4];
    if (kb + 1 < kb1) {
      dq4_load<NG>(w0 + (size_t)(kb + 1) * 64, c, v0);
      dq4_load<NG>(w1 + (size_t)(kb + 1) * 64, c, v1);
    }
    float f0[NG], f1[NG];
#pragma unroll
    for (int x = 0; x < NG; ++x) {
      f0[x] = 16.f * dq4_scale(p.scales, p.scale_bf16, s0 + kb * NG + x);
      f1[x] = 16.f * dq4_scale(p.scales, p.scale_bf16, s1 + kb * NG + x);
    }
    float acc[NT][NG][4];
    uint32_t b[NT][16];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int m = m0 + t * 8 + g;
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint4 v = m < p.M ? __ldg(reinterpret_cast<const uint4*>(p.a + (size_t)m * p.K + kb * 128 + dq4_col<NG>(y, c)))
                                : make_uint4(0, 0, 0, 0);
        b[t][4 * y + 0] = __byte_perm(v.x, v.z, 0x5410);
        b[t][4 * y + 1] = __byte_perm(v.x, v.z, 0x7632);
        b[t][4 * y + 2] = __byte_perm(v.y, v.w, 0x5410);
        b[t][4 * y + 3] = __byte_perm(v.y, v.w, 0x7632);
      }
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        acc[t][x][0] = acc[t][x][1] = acc[t][x][2] = acc[t][x][3] = 0.f;
#pragma unroll
        for (int y = 0; y < 8 / NG; ++y) {
          const int k = x * (8 / NG) + y;
          dq4_mma(acc[t][x], 0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u, 0xBFC0BFC0u, b[t][2 * k], b[t][2 * k + 1]);
        }
      }
    }
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      const int x = y * NG / 4;
      const uint32_t a00 = dq4_code<0>(u0[y]), a10 = dq4_code<0>(u1[y]), a01 = dq4_code<1>(u0[y]),
                     a11 = dq4_code<1>(u1[y]), a02 = dq4_code<2>(u0[y]), a12 = dq4_code<2>(u1[y]),
                     a03 = dq4_code<3>(u0[y]), a13 = dq4_code<3>(u1[y]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        dq4_mma(acc[t][x], a00, a10, a01, a11, b[t][4 * y], b[t][4 * y + 1]);
        dq4_mma(acc[t][x], a02, a12, a03, a13, b[t][4 * y + 2], b[t][4 * y + 3]);
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int x = 0; x < NG; ++x) {
        tot[t][0] = fmaf(acc[t][x][0], f0[x], tot[t][0]);
        tot[t][1] = fmaf(acc[t][x][1], f0[x], tot[t][1]);
        tot[t][2] = fmaf(acc[t][x][2], f1[x], tot[t][2]);
        tot[t][3] = fmaf(acc[t][x][3], f1[x], tot[t][3]);
      }
#pragma unroll
    for (int y = 0; y < 4; ++y) u0[y] = v0[y], u1[y] = v1[y];
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) red[warp][g + (e >> 1) * 8][t * 8 + 2 * c + (e & 1)] = tot[t][e];
  __syncthreads();
  for (int i = threadIdx.x; i < 16 * 8 * NT; i += DQ4_THREADS) {
    const int n = i & 15, m = i >> 4;
    if (m0 + m >= p.M) break;
    float v = p.bias ? __bfloat162float(p.bias[n0 + n]) : 0.f;
#pragma unroll
    for (int w = 0; w < DQ4_WARPS; ++w) v += red[w][n][m];
    p.out[(size_t)(m0 + m) * p.N + n0 + n] = __float2bfloat16_rn(v);
  }
}

// 32 codes (16 bytes) a thread -> bf16
__global__ void __launch_bounds__(256) dq4_expand_kernel(const uint8_t* __restrict__ w, const void* __restrict__ scales,
                                                         int scale_bf16, int group, size_t n32,
                                                         __nv_bfloat16* __restrict__ out) {
  const int per = group / 32;
  for (size_t i = blockIdx.x * (size_t)blockDim.x + threadIdx.x; i < n32; i += (size_t)gridDim.x * blockDim.x) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(w) + i);
    const float s = dq4_scale(scales, scale_bf16, i / per), o = -8.f * s;
    const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t r[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        r[k] = pack_bf16x2(fmaf((float)((x[j] >> (8 * k)) & 15u), s, o), fmaf((float)((x[j] >> (8 * k + 4)) & 15u), s, o));
      reinterpret_cast<uint4*>(out)[i * 4 + j] = make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
}

template <int NG>
static void dq4_stream(const Dq4Args& p, cudaStream_t st) {
  if (p.M <= 8)
    dq4_stream_kernel<NG, 1><<<dim3(p.N / 16, 1), DQ4_THREADS, 0, st>>>(p);
  else if (p.M <= 16)
    dq4_stream_kernel<NG, 2><<<dim3(p.N / 16, 1), DQ4_THREADS, 0, st>>>(p);
  else
    dq4_stream_kernel<NG, 4><<<dim3(p.N / 16, (p.M + 31) / 32), DQ4_THREADS, 0, st>>>(p);
}

}  // namespace ltxb

using namespace ltxb;

extern "C" {

uint64_t ltxb_dq4_gemm_workspace_bytes(int M, int N, int K) {
  return M > DQ4_STREAM_ROWS && N > 0 && K > 0 ? (uint64_t)N * K * 2 : 0;
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
  if (M > DQ4_STREAM_ROWS) {
    const uint64_t need = ltxb_dq4_gemm_workspace_bytes(M, N, K);
    if (!workspace || workspace_bytes < need)
      return set_error(LTXB_EINVAL, "dq4_gemm: workspace of %llu bytes is smaller than the %llu required",
                       (unsigned long long)workspace_bytes, (unsigned long long)need);
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
    const size_t n32 = (size_t)N * K / 32;
    int grid = (int)((n32 + 255) / 256);
    if (grid > 8 * sm_count()) grid = 8 * sm_count();
    dq4_expand_kernel<<<grid, 256, 0, st>>>(static_cast<const uint8_t*>(Wq), scales, sb, group, n32,
                                            static_cast<__nv_bfloat16*>(workspace));
    launched();
    e = cudaGetLastError();
    if (e != cudaSuccess) return set_cuda_error(e, "dq4_gemm expansion");
    return gemm_tc(g, st);
  }
  Dq4Args p{static_cast<const __nv_bfloat16*>(A), static_cast<const uint8_t*>(Wq), scales,
            static_cast<const __nv_bfloat16*>(bias), static_cast<__nv_bfloat16*>(out), M, N, K, sb};
  if (group == 128)
    dq4_stream<1>(p, st);
  else if (group == 64)
    dq4_stream<2>(p, st);
  else
    dq4_stream<4>(p, st);
  launched();
  e = cudaGetLastError();
  return e == cudaSuccess ? LTXB_OK : set_cuda_error(e, "dq4_gemm");
}

}  // extern "C"
