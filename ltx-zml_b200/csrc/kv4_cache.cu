// Writing K/V rows into the paged 4-bit cache and reading them back
// (format: kv4.cuh).
//
// Quantiser, per token, head and group of 32 / 64 / 128 values x (bf16):
//   zero = min x, scale = bf16((max x - min x) / 15), code = round((x - zero) / scale),
// all of it exact, ties to even, code 0 where scale is 0. A quotient is a product
// with 1 / scale and one Newton step: off by at most 0.5001 units of its last
// place, and a half where it is one (ties are common, both sides having few bits).
// Elsewhere the quotient of an f32 difference d by the 8-bit scale s stays 0.5019
// units away from each half h (h s is an f32 number, so d is a unit or more from
// it: 2^-23 / m(h s) of it, m the mantissa in [1, 2), at most 2 - 2^-7, where half
// a unit of h is 2^-24 / m(h)): it falls on its own side. A difference is an f32
// number unless a value's exponent lies 16 or more below another's; rounding
// it can then only make a tie, never pass one, and what was rounded off decides
// that tie. Such a tie is the larger of the two itself, for it has 8 bits and h s
// has 13, and the smaller is 2^-24 of it or less: zero = -h s, with some x close to
// 0, or x = h s and zero close to 0. A token's K or V whose zero is the one or the
// other is done again with care (8 us of the time below; looking at all values
// for small ones took 11 to 30). scale is at least range / 15 * (1 - 2^-8), so the
// quotient stays below 15.06: no clamp. (scale itself needs no such care: 15 times a
// bf16 midpoint has more than 8 bits and is no sum of one value and a far smaller one.)
// A group that holds a NaN or an infinity (or whose range is above the
// largest f32) stores scale = NaN and reads back as NaN.
//
// Both kernels are bandwidth-bound: 512 bytes of bf16 K and V on one side
// and 128 + 8 NG bytes on the other per token and head. A warp takes the
// call's tokens of one octet (8 positions, the unit of the V layout) of one
// head: 4 KB of K and V rows are under way at once, the codes are put in order
// in shared memory and stored 16 bytes a lane. With one warp per token (4-byte
// stores into 8 sectors for V) writing and reading back 28,160 tokens x 32
// heads took 620 us.
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

// The tokens that unit u of the call covers: octet `o` (positions 8 o ..) of
// sequence b, of which [p0, p1) belong to the call and are row `row0` on; false
// if there are none. Sequence b's units start at row_start[b] / 8 + 2 b, which
// leaves room for its octets however its tokens lie in them.
struct Kv4Octet {
  int b, p0, p1, row0;
};
__device__ __forceinline__ bool kv4_octet(const Kv4View& c, long long u, Kv4Octet* out) {
  auto start = [&](int b) -> long long {
    const int r = c.row_start ? __ldg(c.row_start + b) : b * c.per;
    return (r < 0 ? 0 : r) / 8 + 2ll * b;
  };
  int lo = 0, hi = c.batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start(mid) <= u)
      lo = mid;
    else
      hi = mid;
  }
  int first, count;
  kv4_rows(c, lo, &first, &count);
  const int len = kv4_len(c, lo), begin = len - count;  // position of row `first`; may be negative
  const int from = begin < 0 ? 0 : begin;
  const long long o = from / 8 + (u - start(lo));
  if (count == 0 || u < start(lo) || o * 8 >= len) return false;  // (no rows: its pages are not looked at either)
  out->b = lo;
  out->p0 = (int)(o * 8) < from ? from : (int)(o * 8);
  out->p1 = (int)(o * 8) + 8 < len ? (int)(o * 8) + 8 : len;
  out->row0 = first + out->p0 - begin;
  return true;
}

// two-wide f32
__device__ __forceinline__ uint64_t c2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void c2un(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t c2add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t c2mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t c2fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// Code c of x - zero: where its f32 value over scale is a tie, what was rounded off decides.
__device__ __forceinline__ float kv4_settle(float c, float x, float zero, float scale) {
  const float d = x - zero, b = d - x, off = (x - (d - b)) + (-zero - b);  // x - zero = d + off
  const float rest = fmaf(-scale, c, d), half = 0.5f * scale;
  return rest == half && off > 0.f ? c + 1.f : rest == -half && off < 0.f ? c - 1.f : c;
}

// Whether a group of this pair may hold such ties (a pair of NaN does not).
__device__ __forceinline__ bool kv4_unsettled(uint32_t pair) {
  const float scale = bf16_lo(pair), zero = bf16_hi(pair);
  const float q = __fdiv_rn(-zero, scale);
  return fabsf(q - rintf(q)) == 0.5f || (zero != 0.f && fabsf(zero) * 8388608.f <= 16.f * scale);
}

// Eight codes (nibble i = value i of a lane's eight consecutive dims) and the
// group's (scale, zero) pair; the 16 / NG lanes of a group agree. Without SETTLE
// ties that only rounding made are as they fall.
template <int NG, bool SETTLE>
__device__ __forceinline__ uint32_t kv4_quantise(uint4 v, uint32_t* pair) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  // (max, -min) as one bf16x2: one shuffle and one maximum per step
  const uint32_t hi = bmax2(bmax2(w[0], w[1]), bmax2(w[2], w[3]));
  const uint32_t sign = 0x80008000u;
  const uint32_t lo = bmax2(bmax2(w[0] ^ sign, w[1] ^ sign), bmax2(w[2] ^ sign, w[3] ^ sign));
  uint32_t mm = bmax2(__byte_perm(hi, lo, 0x5410), __byte_perm(hi, lo, 0x7632));
#pragma unroll
  for (int s = 1; s < 16 / NG; s <<= 1) mm = bmax2(mm, __shfl_xor_sync(0xffffffffu, mm, s));
  const float top = bf16_lo(mm), zero = -bf16_hi(mm);
  const float range = top - zero;
  // range / 15, correctly rounded: product with 1 / 15 and one Newton step
  const float r15 = range * (1.f / 15.f);
  const __nv_bfloat16 sb = __float2bfloat16_rn(fmaf(fmaf(-15.f, r15, range), 1.f / 15.f, r15));
  const float scale = __bfloat162float(sb);
  const bool finite = range < INFINITY;  // false for NaN and for infinity
  *pair = finite ? ((mm ^ 0x80000000u) & 0xFFFF0000u) | __bfloat16_as_ushort(sb) : 0x7FFFu;
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
  const uint64_t nz = c2(-zero, -zero), in2 = c2(inv, inv), ns = c2(-scale, -scale), mg = c2(12582912.f, 12582912.f),
                 nm = c2(-12582912.f, -12582912.f);
  float q[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t d = c2add(c2(bf16_lo(w[i]), bf16_hi(w[i])), nz), t = c2mul(d, in2);
    const uint64_t t1 = c2fma(c2fma(ns, t, d), in2, t);
    c2un(c2add(c2add(t1, mg), nm), q[2 * i], q[2 * i + 1]);  // the nearest integers (1.5 * 2^23 added and taken off)
  }
  if (SETTLE) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      q[2 * i] = kv4_settle(q[2 * i], bf16_lo(w[i]), zero, scale);
      q[2 * i + 1] = kv4_settle(q[2 * i + 1], bf16_hi(w[i]), zero, scale);
    }
  }
  uint32_t code[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // four codes as one exact number below 2^16, in the low bits of 1.5 * 2^23
    const float p = fmaf(fmaf(q[4 * h + 3], 16.f, q[4 * h + 2]), 256.f, fmaf(q[4 * h + 1], 16.f, q[4 * h]));
    code[h] = __float_as_uint(p + 12582912.f);
  }
  uint32_t out = __byte_perm(code[0], code[1], 0x5410);
  if (scale < 7.5e-37f || !finite) {  // below 2^-120 1 / scale leaves f32's range: quotients one by one
    out = 0;
    if (scale > 0.f && finite)
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        const float x = __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
        out |= (uint32_t)kv4_settle(fminf(rintf(__fdiv_rn(x - zero, scale)), 15.f), x, zero, scale) << (4 * i);
      }
  }
  return out;
}

// CTA (x, y): octet unit x, heads 8 y + warp. Lane = 16 half + m holds dims
// 8 m .. 8 m + 7 of tokens 2 i + half, i = 0 .. 3 of the octet.
template <int NG>
__global__ void __launch_bounds__(256, 4) kv4_append_kernel(const Kv4View c, const __nv_bfloat16* __restrict__ k,
                                                         size_t ldk, const __nv_bfloat16* __restrict__ v,
                                                         size_t ldv) {
  __shared__ __align__(16) uint8_t codes[8][2][512];
  __shared__ uint32_t pairs[8][4][2][2 * NG];
  const int warp = warp_id(), lane = lane_id(), half = lane >> 4, m = lane & 15;
  const int h = blockIdx.y * 8 + warp;
  if (h >= c.heads) return;
  Kv4Octet oc;
  if (!kv4_octet(c, blockIdx.x, &oc)) return;
  const int base = oc.p0 & ~7, t8 = (base % KV4_PAGE) / 8;  // first position, octet of the page
  const int page = kv4_page(c, oc.b, oc.p0 / KV4_PAGE);     // used after the rows are under way
  uint4 x[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int pos = base + 2 * i + half;
    const bool in = pos >= oc.p0 && pos < oc.p1;
    const size_t row = in ? oc.row0 + (pos - oc.p0) : oc.row0;
    x[0][i] = __ldg(reinterpret_cast<const uint4*>(k + row * ldk + h * KV4_D + 8 * m));
    x[1][i] = __ldg(reinterpret_cast<const uint4*>(v + row * ldv + h * KV4_D + 8 * m));
  }
  if (page < 0) return;
  uint8_t* blk = const_cast<uint8_t*>(kv4_block_at(c, page, h, kv4_block(NG)));
  const int j = m >> 2, cc = m & 3;  // dims 32 j + 8 cc .. + 7
  auto put_k = [&](int t, uint32_t kc) { *reinterpret_cast<uint32_t*>(&codes[warp][0][t * 64 + (cc * 4 + j) * 4]) = kc; };
  auto put_v = [&](int t, uint32_t vc) {  // halves j of chunks 2 cc and 2 cc + 1
    uint8_t* vd = &codes[warp][1][2 * cc * 64 + (t >> 1) * 16 + (t & 1) * 8 + j * 2];
    *reinterpret_cast<uint16_t*>(vd) = (uint16_t)vc;
    *reinterpret_cast<uint16_t*>(vd + 64) = (uint16_t)(vc >> 16);
  };
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 2 * i + half, pos = base + t;
    uint32_t kp, vp;
    put_k(t, kv4_quantise<NG, false>(x[0][i], &kp));
    put_v(t, kv4_quantise<NG, false>(x[1][i], &vp));
    if (m % (16 / NG) == 0) {
      pairs[warp][i][0][lane / (16 / NG)] = kp;
      pairs[warp][i][1][lane / (16 / NG)] = vp;
      if (pos >= oc.p0 && pos < oc.p1) {
        const int at = ((t8 * 8 + t) * NG + m / (16 / NG)) * 4;
        *reinterpret_cast<uint32_t*>(blk + KV4_KPAIR + at) = kp;
        *reinterpret_cast<uint32_t*>(blk + kv4_vpair(NG) + at) = vp;
      }
    }
  }
  __syncwarp();
  // the calls (token pair, K or V) whose groups may hold unsettled ties: a pair or two a lane
  uint32_t again = 0;
#pragma unroll
  for (int u = lane; u < 16 * NG; u += 32)
    if (kv4_unsettled((&pairs[warp][0][0][0])[u])) again |= 1u << (u / (2 * NG));
  again = __reduce_or_sync(0xffffffffu, again);
#pragma unroll 1
  for (; again; again &= again - 1) {
    const int n = __ffs(again) - 1, t = 2 * (n >> 1) + half, pos = base + t;
    const size_t row = pos >= oc.p0 && pos < oc.p1 ? oc.row0 + (pos - oc.p0) : oc.row0;
    uint32_t pair;
    const uint32_t code = kv4_quantise<NG, true>(
        __ldg(reinterpret_cast<const uint4*>((n & 1 ? v + row * ldv : k + row * ldk) + h * KV4_D + 8 * m)), &pair);
    if (n & 1)
      put_v(t, code);
    else
      put_k(t, code);
  }
  __syncwarp();
  const uint4 ko = *reinterpret_cast<const uint4*>(&codes[warp][0][lane * 16]);
  const uint4 vo = *reinterpret_cast<const uint4*>(&codes[warp][1][lane * 16]);
  const int kt = base + (lane >> 2), v0 = base + 2 * (lane & 3);  // tokens of the lane's 16 bytes of K; of V, v0 and v0 + 1
  if (kt >= oc.p0 && kt < oc.p1) *reinterpret_cast<uint4*>(blk + t8 * 512 + lane * 16) = ko;
  uint8_t* vd = blk + KV4_VOFF + t8 * 512 + lane * 16;
  const bool in0 = v0 >= oc.p0 && v0 < oc.p1, in1 = v0 + 1 >= oc.p0 && v0 + 1 < oc.p1;
  if (in0 && in1)
    *reinterpret_cast<uint4*>(vd) = vo;
  else if (in0)
    *reinterpret_cast<uint2*>(vd) = make_uint2(vo.x, vo.y);
  else if (in1)
    *reinterpret_cast<uint2*>(vd + 8) = make_uint2(vo.z, vo.w);
}

// Values zero + scale * code in f32, rounded once, of the N = 4 or 8 codes of
// `code`, stored at `out` (f32 or bf16).
template <int N, bool F32>
__device__ __forceinline__ void kv4_values(uint32_t code, uint32_t pair, void* out, size_t at) {
  const float s = bf16_lo(pair), z = bf16_hi(pair);
  const uint64_t s2 = c2(s, s), z2 = c2(z, z), off = c2(-8388608.f, -8388608.f);
  float f[N];
#pragma unroll
  for (int i = 0; i < N; i += 2) {  // 2^23 + code, exactly
    const uint32_t a = ((code >> (4 * i)) & 15u) | 0x4B000000u, b = ((code >> (4 * i + 4)) & 15u) | 0x4B000000u;
    c2un(c2fma(s2, c2add(c2(__uint_as_float(a), __uint_as_float(b)), off), z2), f[i], f[i + 1]);
  }
  if (F32) {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      *reinterpret_cast<float4*>(reinterpret_cast<float*>(out) + at + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else if (N == 8) {
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(out) + at) =
        make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[N - 4], f[N - 3]), pack_bf16x2(f[N - 2], f[N - 1]));
  } else {
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(out) + at) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
  }
}

template <int NG, bool F32>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4View c, void* __restrict__ k_out,
                                                       void* __restrict__ v_out) {
  const int lane = lane_id(), h = blockIdx.y * 8 + warp_id();
  if (h >= c.heads) return;
  Kv4Octet oc;
  if (!kv4_octet(c, blockIdx.x, &oc)) return;
  const int page = kv4_page(c, oc.b, oc.p0 / KV4_PAGE);
  if (page < 0) return;
  const uint8_t* blk = kv4_block_at(c, page, h, kv4_block(NG));
  const int base = oc.p0 & ~7, t8 = (base % KV4_PAGE) / 8;
  const uint4 kw = *reinterpret_cast<const uint4*>(blk + t8 * 512 + lane * 16);
  const uint4 vw = *reinterpret_cast<const uint4*>(blk + KV4_VOFF + t8 * 512 + lane * 16);
  const uint32_t* kp = reinterpret_cast<const uint32_t*>(blk + KV4_KPAIR) + t8 * 8 * NG;
  const uint32_t* vp = reinterpret_cast<const uint32_t*>(blk + kv4_vpair(NG)) + t8 * 8 * NG;
  const int g = lane >> 2, cq = lane & 3;
  auto at = [&](int pos) { return ((size_t)(oc.row0 + (pos - oc.p0)) * c.heads + h) * KV4_D; };
  if (base + g >= oc.p0 && base + g < oc.p1) {
    const uint32_t w[4] = {kw.x, kw.y, kw.z, kw.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) kv4_values<8, F32>(w[j], kp[g * NG + j * NG / 4], k_out, at(base + g) + 32 * j + 8 * cq);
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int t = 2 * cq + e;
    if (base + t < oc.p0 || base + t >= oc.p1) continue;
    const uint32_t w[2] = {e ? vw.z : vw.x, e ? vw.w : vw.y};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      kv4_values<4, F32>(w[j >> 1] >> (16 * (j & 1)), vp[t * NG + j * NG / 4], v_out, at(base + t) + 32 * j + 4 * g);
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
  if (c->kv_heads > 65535 * 8 || c->batch > (1 << 28)) return set_error(LTXB_EINVAL, "%s: too many heads or sequences", what);
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

// octet units x groups of eight heads
static dim3 kv4_grid(const Kv4View& v) { return dim3(v.rows / 8 + 2 * v.batch, (v.heads + 7) / 8); }

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
  const dim3 grid = kv4_grid(c);
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
  const dim3 grid = kv4_grid(c);
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
