// Operands of the many-row attention over a 4-bit cache (kv4_attn_tc.cu):
// the query rows and every sequence's K and V as f16 matrices.
//
// f16 keeps 11 significant bits, where bf16 would keep 8 of a cached value's
// 12 and more; its range is met by powers of two: each query row is scaled by
// its own, K and V by one per sequence and head (taken from the scales and
// zeros alone, 6 to 25 % of the cache's bytes), so that the largest value
// lies in [2^14, 2^15]. A bf16 query value is then exact down to 2^-31 of its
// row's largest; below that it is off by at most 2^-39 of it.
//
// Both kernels are bandwidth-bound: 4 bytes per query value, and 136 to 160
// bytes in, 512 out per token and head.
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace ltxb {

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Exponent field of the power of two that takes `top` into [2^14, 2^15).
__device__ __forceinline__ uint32_t kv4_field(float top) {
  const int f = 268 - (int)(__float_as_uint(top) >> 23);
  return (uint32_t)(f < 1 ? 1 : f > 253 ? 253 : f);
}

// CTAs [0, q_ctas): query rows, four (row, head) a warp; the others: the
// largest |K| and |V| that the pairs of 16 pages of one (sequence, head)
// allow (finite groups only).
template <int NG>
__global__ void __launch_bounds__(256) kv4_prep_kernel(const Kv4View c, const Kv4Tc t, const __nv_bfloat16* __restrict__ q,
                                                       size_t ldq, int q_ctas) {
  const int lane = lane_id(), warp = warp_id(), H = c.heads * t.G;
  if ((int)blockIdx.x < q_ctas) {
    // four (row, head) rows a warp and step; rows * H < 2^31 here
    const int n = c.rows * H;
    for (int u0 = ((int)blockIdx.x * 8 + warp) * 4; u0 < n; u0 += q_ctas * 32) {
      uint2 w[4];
      float top[4];
      int row[4], h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int u = u0 + i < n ? u0 + i : n - 1;
        row[i] = u / H;
        h[i] = u - row[i] * H;
        w[i] = __ldg(reinterpret_cast<const uint2*>(q + (size_t)row[i] * ldq + h[i] * KV4_D + lane * 4));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        top[i] = fmaxf(fmaxf(fabsf(bf16_lo(w[i].x)), fabsf(bf16_hi(w[i].x))), fmaxf(fabsf(bf16_lo(w[i].y)), fabsf(bf16_hi(w[i].y))));
#pragma unroll
      for (int s = 1; s < 32; s <<= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], s));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (u0 + i >= n) break;
        const uint32_t field = kv4_field(top[i]);
        // the sign of the softmax scale goes with the row, so that q_scale is positive; a row with an infinity is NaN
        const float f = !(top[i] < INFINITY) ? NAN : t.cs == 0.f ? 0.f : copysignf(__uint_as_float(field << 23), t.cs);
        const int hk = h[i] / t.G;
        const size_t o = ((size_t)hk * c.rows + row[i]) * t.G + (h[i] - hk * t.G);
        reinterpret_cast<uint2*>(t.q16)[o * 32 + lane] = make_uint2(pack_h2(bf16_lo(w[i].x) * f, bf16_hi(w[i].x) * f),
                                                                    pack_h2(bf16_lo(w[i].y) * f, bf16_hi(w[i].y) * f));
        if (lane == 0) t.q_scale[o] = __uint_as_float((254u - field) << 23) * fabsf(t.cs);
      }
    }
    return;
  }
  const int u = blockIdx.x - q_ctas;
  const int chunk = u % t.chunks, bh = u / t.chunks, b = bh / c.heads, h = bh % c.heads;
  int first, count;
  kv4_rows(c, b, &first, &count);
  if (count == 0) return;  // no row reads this sequence
  const int pages = (kv4_len(c, b) + KV4_PAGE - 1) / KV4_PAGE;
  float km = 0.f, vm = 0.f;
  for (int j = chunk * 16 + warp; j < pages && j < chunk * 16 + 16; j += 8) {
    const int p = kv4_page(c, b, j);
    if (p < 0) continue;
    const int left = kv4_len(c, b) - j * KV4_PAGE, words = (left < KV4_PAGE ? left : KV4_PAGE) * NG;
    const uint32_t* kp = reinterpret_cast<const uint32_t*>(kv4_block_at(c, p, h, kv4_block(NG)) + KV4_KPAIR);
    const uint32_t* vp = kp + KV4_PAGE * NG;
    for (int i = lane; i < words; i += 32) {
      const uint32_t a = kp[i], d = vp[i];
      const float ka = fmaxf(fabsf(bf16_hi(a)), fabsf(fmaf(15.f, bf16_lo(a), bf16_hi(a))));
      const float va = fmaxf(fabsf(bf16_hi(d)), fabsf(fmaf(15.f, bf16_lo(d), bf16_hi(d))));
      if (ka < INFINITY) km = fmaxf(km, ka);
      if (va < INFINITY) vm = fmaxf(vm, va);
    }
  }
  __shared__ float2 red[8];
#pragma unroll
  for (int s = 1; s < 32; s <<= 1) {
    km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, s));
    vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, s));
  }
  if (lane == 0) red[warp] = make_float2(km, vm);
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) {
      km = fmaxf(km, red[i].x);
      vm = fmaxf(vm, red[i].y);
    }
    t.top[u] = make_float2(km, vm);
  }
}

// value zero + scale (16 (u - 1)), u = 1 + code / 16, as one FMA: s16 u + o
__device__ __forceinline__ float kv4_u(uint32_t w, int nibble) {
  const uint32_t s = nibble < 5 ? w << (19 - 4 * nibble) : w >> (4 * nibble - 19);
  return __uint_as_float((s & 0x00780000u) | 0x3F800000u);
}

// One CTA per page and head: thread (token, c) the K chunk 16 c of a token,
// thread (octet, c, g) the V unit 4 g + c of an octet. Tokens from the length
// to the next multiple of 128 are zeros; a token whose V holds a group that is
// not finite, or whose page number is bad, gets V = 0 and K = NaN (its score
// then makes the rows that see it NaN, and no others).
template <int NG>
__global__ void __launch_bounds__(256) kv4_expand_kernel(const Kv4View c, const Kv4Tc t) {
  __shared__ float s_f[2];
  __shared__ uint32_t s_bad[2];
  const int h = blockIdx.y, b = blockIdx.z;
  int first, count;
  kv4_rows(c, b, &first, &count);
  if (count == 0) return;
  const int len = kv4_len(c, b);
  // the powers of two of this (sequence, head)
  if (threadIdx.x < 32) {
    const int n = ((len + KV4_PAGE - 1) / KV4_PAGE + 15) / 16;
    float km = 0.f, vm = 0.f;
    for (int i = threadIdx.x; i < n; i += 32) {
      const float2 m = t.top[((size_t)b * c.heads + h) * t.chunks + i];
      km = fmaxf(km, m.x);
      vm = fmaxf(vm, m.y);
    }
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, s));
      vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, s));
    }
    if (threadIdx.x == 0) {
      const uint32_t kf = kv4_field(km), vf = kv4_field(vm);
      s_f[0] = __uint_as_float(kf << 23);
      s_f[1] = __uint_as_float(vf << 23);
      if (blockIdx.x == 0)
        t.kv_scale[(size_t)b * c.heads + h] =
            make_float2(__uint_as_float((254u - kf) << 23), __uint_as_float((254u - vf) << 23));
    }
  }
  __syncthreads();
  const float kf = s_f[0], vf = s_f[1];
  const int pages = (len + 127) / 128 * 2;
  const size_t row0 = ((size_t)b * c.heads + h) * t.tokens;
  for (int j = blockIdx.x; j < pages; j += gridDim.x) {
    const int left = len - j * KV4_PAGE;  // tokens of this page that exist
    const int p = left > 0 ? kv4_page(c, b, j) : -1;
    uint2* kd = reinterpret_cast<uint2*>(t.k16) + (row0 + (size_t)j * KV4_PAGE) * 32;
    uint2* vd = reinterpret_cast<uint2*>(t.v16) + (row0 + (size_t)j * KV4_PAGE) * 32;
    __syncthreads();  // s_bad of the page before is no longer read
    if (threadIdx.x < 2) s_bad[threadIdx.x] = 0;
    __syncthreads();
    const uint8_t* blk = p >= 0 ? kv4_block_at(c, p, h, kv4_block(NG)) : nullptr;
    {
      const int tok = threadIdx.x;  // one warp pair looks at the V pairs of all tokens
      if (p >= 0 && tok < KV4_PAGE && tok < left) {
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(blk + kv4_vpair(NG)) + tok * NG;
        bool bad = false;
#pragma unroll
        for (int x = 0; x < NG; ++x) bad = bad || !(fabsf(fmaf(8.f, bf16_lo(vp[x]), bf16_hi(vp[x]))) < INFINITY);
        if (bad) atomicOr(&s_bad[tok >> 5], 1u << (tok & 31));
      }
    }
    __syncthreads();
    {  // K
      const int tok = threadIdx.x >> 2, cq = threadIdx.x & 3;
      const bool has = p >= 0 && tok < left;
      // NaN also where the page number was bad: its tokens must not be attended to as zeros
      const bool nan = tok < left && (p < 0 || ((s_bad[tok >> 5] >> (tok & 31)) & 1u));
      uint4 w = make_uint4(0, 0, 0, 0);
      if (has) w = *reinterpret_cast<const uint4*>(blk + tok * 64 + cq * 16);
      const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        float s16 = 0.f, o = 0.f;
        if (has) {
          const uint32_t pr = reinterpret_cast<const uint32_t*>(blk + KV4_KPAIR)[tok * NG + x * NG / 4];
          s16 = 16.f * (kf * bf16_lo(pr));
          o = fmaf(kf, bf16_hi(pr), -s16);
        }
        if (nan) o = NAN;
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          r[i] = pack_h2(fmaf(s16, kv4_u(ws[x], 2 * i), o), fmaf(s16, kv4_u(ws[x], 2 * i + 1), o));
        *reinterpret_cast<uint4*>(kd + tok * 32 + x * 8 + cq * 2) = make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
    {  // V
      const int oct = threadIdx.x >> 5, cq = (threadIdx.x >> 3) & 3, g = threadIdx.x & 7;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (p >= 0) w = *reinterpret_cast<const uint4*>(blk + KV4_VOFF + oct * 512 + g * 64 + cq * 16);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int tok = oct * 8 + 2 * cq + e;
        const bool has = p >= 0 && tok < left && !((s_bad[tok >> 5] >> (tok & 31)) & 1u);
        const uint32_t lo = e ? w.z : w.x, hi = e ? w.w : w.y;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          float s16 = 0.f, o = 0.f;
          if (has) {
            const uint32_t pr = reinterpret_cast<const uint32_t*>(blk + kv4_vpair(NG))[tok * NG + x * NG / 4];
            s16 = 16.f * (vf * bf16_lo(pr));
            o = fmaf(vf, bf16_hi(pr), -s16);
          }
          const uint32_t code = (x < 2 ? lo : hi) >> (16 * (x & 1));
          vd[tok * 32 + x * 8 + g] =
              make_uint2(pack_h2(fmaf(s16, kv4_u(code, 0), o), fmaf(s16, kv4_u(code, 1), o)),
                         pack_h2(fmaf(s16, kv4_u(code, 2), o), fmaf(s16, kv4_u(code, 3), o)));
        }
      }
    }
  }
}

int kv4_prepare(const Kv4View& c, const Kv4Tc& t, const void* q, size_t ldq, int group, cudaStream_t st) {
  const int H = c.heads * t.G;
  const long long qw = ((long long)c.rows * H + 31) / 32, most = 8ll * sm_count();
  const int q_ctas = (int)(qw < most ? qw : most);
  const long long grid = q_ctas + (long long)c.batch * c.heads * t.chunks;
  const __nv_bfloat16* qb = static_cast<const __nv_bfloat16*>(q);
  if (group == 128)
    kv4_prep_kernel<1><<<(unsigned)grid, 256, 0, st>>>(c, t, qb, ldq, q_ctas);
  else if (group == 64)
    kv4_prep_kernel<2><<<(unsigned)grid, 256, 0, st>>>(c, t, qb, ldq, q_ctas);
  else
    kv4_prep_kernel<4><<<(unsigned)grid, 256, 0, st>>>(c, t, qb, ldq, q_ctas);
  launched();
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "kv4 attention operands");
  // enough CTAs over the pages to fill the GPU eight deep, at most one a page
  int px = t.tokens / KV4_PAGE;
  const long long want = (8ll * sm_count() * 2 + (long long)c.batch * c.heads - 1) / ((long long)c.batch * c.heads);
  if (px > want) px = (int)want;
  const dim3 eg(px, c.heads, c.batch);
  if (group == 128)
    kv4_expand_kernel<1><<<eg, 256, 0, st>>>(c, t);
  else if (group == 64)
    kv4_expand_kernel<2><<<eg, 256, 0, st>>>(c, t);
  else
    kv4_expand_kernel<4><<<eg, 256, 0, st>>>(c, t);
  launched();
  e = cudaGetLastError();
  return e == cudaSuccess ? LTXB_OK : set_cuda_error(e, "kv4 attention expansion");
}

}  // namespace ltxb
