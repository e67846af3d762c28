// Writing K/V rows into the paged 4-bit cache and reading them back
// (format: kv4.cuh).
//
// Quantiser, per token, head and group of 32 / 64 / 128 values x (bf16):
//   zero = min x, scale = bf16((max x - min x) / 15), code = round((x - zero) / scale),
// ties to even, code 0 where scale is 0. The code is the one of exact
// arithmetic: x - zero is rounded once in f32 and multiplied by 1 / scale,
// and where that product comes within 1e-5 of a half (its error is below
// 16 * 2^-22 = 4e-6) the quotient is taken again in 64 bits. scale is at
// least range / 15 * (1 - 2^-8), so the product stays below 15.06 and needs
// no clamp there.
// A group that holds a NaN or an infinity (or whose range is above the
// largest f32) stores scale = NaN and reads back as NaN.
//
// Both kernels are bandwidth-bound: 512 bytes of bf16 K and V on one side
// and 128 + 8 NG bytes on the other per token and head.
#include "kv4.cuh"

namespace ltxb {

__device__ uint32_t g_index_status = 0;

cudaError_t index_status(uint32_t* v, bool clear) {
  cudaError_t e = cudaMemcpyFromSymbol(v, g_index_status, sizeof(*v));
  if (e == cudaSuccess && clear && *v) {
    const uint32_t z = 0;
    e = cudaMemcpyToSymbol(g_index_status, &z, sizeof(z));
  }
  return e;
}

// bf16x2 minimum / maximum that hand on a NaN
__device__ __forceinline__ uint32_t bmax2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Four codes (a lane's dims 4 L .. 4 L + 3, nibble i = value i) and the
// group's (scale, zero) pair of the 4 bf16 values in `w`; the 8 * (4 / NG)
// lanes of a group agree.
template <int NG>
__device__ __forceinline__ uint32_t kv4_quantise(uint2 w, uint32_t* pair) {
  // (max, -min) as one bf16x2: one shuffle and one maximum per step
  const uint32_t hi = bmax2(w.x, w.y), lo = bmax2(w.x ^ 0x80008000u, w.y ^ 0x80008000u);
  uint32_t mm = bmax2(__byte_perm(hi, lo, 0x5410), __byte_perm(hi, lo, 0x7632));
#pragma unroll
  for (int s = 1; s < 32 / NG; s <<= 1) mm = bmax2(mm, __shfl_xor_sync(0xffffffffu, mm, s));
  const float top = bf16_lo(mm), zero = -bf16_hi(mm);
  const float range = top - zero;
  const float q15 = __fdiv_rn(range, 15.0f);
  const __nv_bfloat16 sb = __float2bfloat16_rn(q15);
  const float scale = __bfloat162float(sb);
  const bool finite = range < INFINITY;  // false for NaN and for infinity
  *pair = finite ? ((mm ^ 0x80000000u) & 0xFFFF0000u) | __bfloat16_as_ushort(sb) : 0x7FFFu;
  const bool tiny = scale < 7.5e-37f;  // 2^-120: 1 / scale would leave f32's range
  const float inv = scale > 0.f ? __frcp_rn(scale) : 0.f;
  const float x[4] = {bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
  uint32_t code = 0;
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = (x[i] - zero) * inv;
    const float m = t + 12582912.0f;  // 1.5 * 2^23: the integer in the low mantissa bits
    far = fmaxf(far, fabsf(t - (m - 12582912.0f)));
    code |= (__float_as_uint(m) & 15u) << (4 * i);
  }
  if ((far > 0.49999f || tiny) && scale > 0.f && finite) {
    code = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const double t = rint(((double)x[i] - (double)zero) / (double)scale);
      code |= (uint32_t)(t > 15.0 ? 15.0 : t) << (4 * i);
    }
  }
  return code;
}

// One warp per row and head: lane L holds dims 4 L .. 4 L + 3 of K and V.
template <int NG>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4View c, const __nv_bfloat16* __restrict__ k,
                                                         size_t ldk, const __nv_bfloat16* __restrict__ v,
                                                         size_t ldv) {
  const int lane = lane_id();
  const long long n = (long long)c.rows * c.heads;
  for (long long u = blockIdx.x * 8ll + warp_id(); u < n; u += gridDim.x * 8ll) {
    const int row = (int)(u / c.heads), h = (int)(u % c.heads);
    const int b = kv4_row_seq(c, row);
    if (b < 0) continue;
    int first, count;
    kv4_rows(c, b, &first, &count);
    const int pos = kv4_len(c, b) - count + (row - first);
    if (row < first || row >= first + count || pos < 0) continue;
    const int page = kv4_page(c, b, pos / KV4_PAGE);
    if (page < 0) continue;
    const uint2 kx = *reinterpret_cast<const uint2*>(k + row * ldk + h * KV4_D + lane * 4);
    const uint2 vx = *reinterpret_cast<const uint2*>(v + row * ldv + h * KV4_D + lane * 4);
    uint32_t kp, vp;
    uint32_t kc = kv4_quantise<NG>(kx, &kp);
    uint32_t vc = kv4_quantise<NG>(vx, &vp);
    uint8_t* blk = const_cast<uint8_t*>(kv4_block_at(c, page, h, kv4_block(NG)));
    const int t = pos % KV4_PAGE;
    // K: lanes 2 m, 2 m + 1 make one word; V: halves j, j + 1 of chunk g
    kc |= __shfl_down_sync(0xffffffffu, kc, 1) << 16;
    vc |= __shfl_down_sync(0xffffffffu, vc, 8) << 16;
    const int j = lane >> 3, cc = (lane >> 1) & 3, g = lane & 7;
    if ((lane & 1) == 0) *reinterpret_cast<uint32_t*>(blk + t * 64 + (cc * 4 + j) * 4) = kc;
    if ((j & 1) == 0)
      *reinterpret_cast<uint32_t*>(blk + KV4_VOFF + (t >> 3) * 512 + g * 64 + ((t & 7) >> 1) * 16 + (t & 1) * 8 +
                                   (j >> 1) * 4) = vc;
    if (lane % (32 / NG) == 0) {
      const int gi = lane / (32 / NG);
      *reinterpret_cast<uint32_t*>(blk + KV4_KPAIR + (t * NG + gi) * 4) = kp;
      *reinterpret_cast<uint32_t*>(blk + kv4_vpair(NG) + (t * NG + gi) * 4) = vp;
    }
  }
}

// The four values of a lane: zero + scale * code in f32, rounded once.
__device__ __forceinline__ float4 kv4_values(uint32_t code, uint32_t pair) {
  const float s = bf16_lo(pair), z = bf16_hi(pair);
  return make_float4(fmaf(s, (float)(code & 15u), z), fmaf(s, (float)((code >> 4) & 15u), z),
                     fmaf(s, (float)((code >> 8) & 15u), z), fmaf(s, (float)((code >> 12) & 15u), z));
}

template <int NG, bool F32>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4View c, void* __restrict__ k_out,
                                                       void* __restrict__ v_out) {
  const int lane = lane_id();
  const long long n = (long long)c.rows * c.heads;
  for (long long u = blockIdx.x * 8ll + warp_id(); u < n; u += gridDim.x * 8ll) {
    const int row = (int)(u / c.heads), h = (int)(u % c.heads);
    const int b = kv4_row_seq(c, row);
    if (b < 0) continue;
    int first, count;
    kv4_rows(c, b, &first, &count);
    const int pos = kv4_len(c, b) - count + (row - first);
    if (row < first || row >= first + count || pos < 0) continue;
    const int page = kv4_page(c, b, pos / KV4_PAGE);
    if (page < 0) continue;
    const uint8_t* blk = kv4_block_at(c, page, h, kv4_block(NG));
    const int t = pos % KV4_PAGE, j = lane >> 3, cc = (lane >> 1) & 3, g = lane & 7, gi = lane / (32 / NG);
    const uint32_t kc = *reinterpret_cast<const uint16_t*>(blk + t * 64 + (cc * 4 + j) * 4 + (lane & 1) * 2);
    const uint32_t vc = *reinterpret_cast<const uint16_t*>(blk + KV4_VOFF + (t >> 3) * 512 + g * 64 +
                                                           ((t & 7) >> 1) * 16 + (t & 1) * 8 + j * 2);
    const float4 kf = kv4_values(kc, *reinterpret_cast<const uint32_t*>(blk + KV4_KPAIR + (t * NG + gi) * 4));
    const float4 vf = kv4_values(vc, *reinterpret_cast<const uint32_t*>(blk + kv4_vpair(NG) + (t * NG + gi) * 4));
    const size_t o = (size_t)u * 32 + lane;
    if (F32) {
      reinterpret_cast<float4*>(k_out)[o] = kf;
      reinterpret_cast<float4*>(v_out)[o] = vf;
    } else {
      reinterpret_cast<uint2*>(k_out)[o] = make_uint2(pack_bf16x2(kf.x, kf.y), pack_bf16x2(kf.z, kf.w));
      reinterpret_cast<uint2*>(v_out)[o] = make_uint2(pack_bf16x2(vf.x, vf.y), pack_bf16x2(vf.z, vf.w));
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

int kv4_check(const ltxb_kv4_cache* c, const int32_t* row_start, int rows, const char* what, Kv4View* out) {
  if (!c) return set_error(LTXB_EINVAL, "%s: no cache", what);
  if (c->group != 32 && c->group != 64 && c->group != 128)
    return set_error(LTXB_EINVAL, "%s: group must be 32, 64 or 128", what);
  if (c->kv_heads <= 0 || c->n_pages <= 0 || c->batch < 0 || c->max_pages < 0 || c->max_len < 0 || rows < 0)
    return set_error(LTXB_EINVAL, "%s: negative size, no K/V heads or no pages", what);
  if (!c->pages || (c->batch > 0 && !c->seq_lens)) return set_error(LTXB_EINVAL, "%s: pages or seq_lens missing", what);
  if (reinterpret_cast<uintptr_t>(c->pages) & 15) return set_error(LTXB_EINVAL, "%s: pages must be 16-byte aligned", what);
  if ((reinterpret_cast<uintptr_t>(c->page_table) | reinterpret_cast<uintptr_t>(c->seq_lens) |
       reinterpret_cast<uintptr_t>(row_start)) & 3)
    return set_error(LTXB_EINVAL, "%s: page_table, seq_lens and row_start must be 4-byte aligned", what);
  if (!c->page_table && (int64_t)c->batch * c->max_pages > c->n_pages)
    return set_error(LTXB_EINVAL, "%s: without a page table the cache needs batch * max_pages pages", what);
  if ((int64_t)c->max_pages * KV4_PAGE > INT32_MAX)
    return set_error(LTXB_EINVAL, "%s: sequences of 2^31 tokens or more", what);
  if (rows > 0 && c->batch == 0) return set_error(LTXB_EINVAL, "%s: rows but no sequences", what);
  if (!row_start && c->batch > 0 && rows % c->batch)
    return set_error(LTXB_EINVAL, "%s: without row_start every sequence has the same number of rows (%d rows, %d sequences)",
                     what, rows, c->batch);
  Kv4View v{};
  v.pages = static_cast<uint8_t*>(c->pages);
  v.table = c->page_table;
  v.lens = c->seq_lens;
  v.row_start = row_start;
  v.n_pages = c->n_pages;
  v.heads = c->kv_heads;
  v.max_pages = c->max_pages;
  v.batch = c->batch;
  v.cap = c->max_pages * KV4_PAGE;
  if (c->max_len > 0 && c->max_len < v.cap) v.cap = c->max_len;
  v.rows = rows;
  v.per = c->batch > 0 ? rows / c->batch : 0;
  *out = v;
  return LTXB_OK;
}

static int kv4_grid(const Kv4View& v) {
  const long long ctas = ((long long)v.rows * v.heads + 7) / 8, most = 8ll * 8 * sm_count();
  return (int)(ctas < most ? ctas : most);
}

}  // namespace ltxb

using namespace ltxb;

extern "C" {

uint64_t ltxb_kv4_block_bytes(int group) {
  if (group != 32 && group != 64 && group != 128) return 0;
  return (uint64_t)kv4_block(KV4_D / group);
}

int ltxb_kv4_append(const ltxb_kv4_cache* cache, const int32_t* row_start, const void* k, int64_t ldk, const void* v,
                    int64_t ldv, int rows, void* stream) {
  Kv4View c;
  if (int rc = kv4_check(cache, row_start, rows, "kv4 append", &c)) return rc;
  if (rows == 0) return LTXB_OK;
  if (!k || !v || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) || (ldk % 8) || (ldv % 8))
    return set_error(LTXB_EINVAL, "kv4 append: k and v must be 16-byte aligned with 16-byte row strides");
  if (ldk < (int64_t)c.heads * KV4_D || ldv < (int64_t)c.heads * KV4_D)
    return set_error(LTXB_EINVAL, "kv4 append: row strides are smaller than kv_heads * 128");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const __nv_bfloat16 *kb = static_cast<const __nv_bfloat16*>(k), *vb = static_cast<const __nv_bfloat16*>(v);
  const int grid = kv4_grid(c);
  if (cache->group == 128)
    kv4_append_kernel<1><<<grid, 256, 0, st>>>(c, kb, ldk, vb, ldv);
  else if (cache->group == 64)
    kv4_append_kernel<2><<<grid, 256, 0, st>>>(c, kb, ldk, vb, ldv);
  else
    kv4_append_kernel<4><<<grid, 256, 0, st>>>(c, kb, ldk, vb, ldv);
  launched();
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LTXB_OK : set_cuda_error(e, "kv4 append");
}

int ltxb_kv4_read(const ltxb_kv4_cache* cache, const int32_t* row_start, void* k_out, void* v_out, int out_dtype,
                  int rows, void* stream) {
  Kv4View c;
  if (int rc = kv4_check(cache, row_start, rows, "kv4 read", &c)) return rc;
  if (out_dtype != LTXB_DT_BF16 && out_dtype != LTXB_DT_F32)
    return set_error(LTXB_EINVAL, "kv4 read: output dtype must be LTXB_DT_BF16 or LTXB_DT_F32");
  if (rows == 0) return LTXB_OK;
  if (!k_out || !v_out || ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15))
    return set_error(LTXB_EINVAL, "kv4 read: outputs must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int grid = kv4_grid(c);
  auto go = [&](auto kern) { kern<<<grid, 256, 0, st>>>(c, k_out, v_out); };
  const bool f = out_dtype == LTXB_DT_F32;
  if (cache->group == 128)
    f ? go(kv4_read_kernel<1, true>) : go(kv4_read_kernel<1, false>);
  else if (cache->group == 64)
    f ? go(kv4_read_kernel<2, true>) : go(kv4_read_kernel<2, false>);
  else
    f ? go(kv4_read_kernel<4, true>) : go(kv4_read_kernel<4, false>);
  launched();
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? LTXB_OK : set_cuda_error(e, "kv4 read");
}

}  // extern "C"
