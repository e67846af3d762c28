// The paged 4-bit K/V cache: format constants and device helpers shared by
// the kernels that write, read and attend to it (kv4_cache.cu, kv4_attn.cu,
// kv4_attn_tc.cu).
//
// A page holds KV4_PAGE tokens of every K/V head; one (page, head) block is
//   K codes [64 tokens][64 bytes] | V codes [64][64] | K pairs [64][NG] | V pairs [64][NG]
// with NG = 128 / group (scale, zero) bf16 pairs per token (scale in the low
// half of the 32-bit word); value = zero + scale * code, code in 0 .. 15.
//
// The order of the codes is the order in which a warp's matrix fragments
// need them, so that the attention loads 16 bytes per lane and unpacks
// in place (lane = 4 g + c, g = lane / 4, c = lane % 4):
//   K: dim 32 j + 8 c + i of a token is nibble i of the 32-bit word 4 c + j
//      of its 64 bytes: lane (g, c) takes token g's 16 bytes at 16 c, and
//      word j of the four lanes of a quad covers one 32-dim group;
//   V: dim 32 j + 4 g + i of token 8 o + 2 c + e is nibble i of the 16-bit
//      half j of the 8 bytes at 512 o + 64 g + 16 c + 8 e: lane (g, c) takes
//      the 16 bytes at 512 o + 16 lane, tokens 2 c and 2 c + 1 of an octet.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace ltxb {

constexpr int KV4_PAGE = LTXB_KV4_PAGE;
constexpr int KV4_D = 128;
constexpr int KV4_VOFF = KV4_PAGE * 64;            // V codes
constexpr int KV4_KPAIR = 2 * KV4_VOFF;            // K pairs
__host__ __device__ constexpr int kv4_vpair(int ng) { return KV4_KPAIR + KV4_PAGE * 4 * ng; }
__host__ __device__ constexpr int kv4_block(int ng) { return KV4_KPAIR + 2 * KV4_PAGE * 4 * ng; }

// A cache (ltxb_kv4_cache) and the rows of one call, as the kernels see them.
struct Kv4View {
  uint8_t* pages;
  const int* table;      // [batch, max_pages] or null: page b * max_pages + j
  const int* lens;       // [batch]
  const int* row_start;  // [batch + 1] or null: `per` rows for every sequence
  int n_pages, heads, max_pages, batch, cap, rows, per;
};

// Indexes that the host cannot check (page numbers, lengths) are checked by
// the kernels: a bad one is not followed, and its site is kept in a word of
// its own (not in g_status: a bad page of one caller must not make other
// kernels' waits give up).
#ifdef LTXB_LOCAL_STATUS  // kv4_attn_tc.cu: the operand kernels of the same call have reported
__device__ __forceinline__ void report_index(uint32_t) {}
#else
extern __device__ uint32_t g_index_status;
__device__ __forceinline__ void report_index(uint32_t site) { atomicCAS(&g_index_status, 0u, site); }
#endif

// Tokens of sequence b in the cache, in [0, cap].
__device__ __forceinline__ int kv4_len(const Kv4View& v, int b) {
  const int l = __ldg(v.lens + b);
  if ((unsigned)l <= (unsigned)v.cap) return l;
  report_index(LTXB_SITE_KV4_LEN);
  return l < 0 ? 0 : v.cap;
}

// Physical page of sequence b's page j (j < max_pages), or -1.
__device__ __forceinline__ int kv4_page(const Kv4View& v, int b, int j) {
  const size_t i = (size_t)b * v.max_pages + j;
  const int p = v.table ? __ldg(v.table + i) : (int)i;
  if ((unsigned)p < (unsigned)v.n_pages) return p;
  report_index(LTXB_SITE_KV4_PAGE);
  return -1;
}

// Rows [*first, *first + *count) of the call belong to sequence b.
__device__ __forceinline__ void kv4_rows(const Kv4View& v, int b, int* first, int* count) {
  if (!v.row_start) {
    *first = b * v.per;
    *count = v.per;
    return;
  }
  int s = __ldg(v.row_start + b), e = __ldg(v.row_start + b + 1);
  if (s < 0 || e < s || e > v.rows) {
    report_index(LTXB_SITE_KV4_ROWS);
    s = s < 0 ? 0 : s > v.rows ? v.rows : s;
    e = e < s ? s : e > v.rows ? v.rows : e;
  }
  *first = s;
  *count = e - s;
}

// Sequence of row i (the last one whose rows start at or before i), or -1.
__device__ __forceinline__ int kv4_row_seq(const Kv4View& v, int i) {
  if (!v.row_start) return i / v.per;
  int lo = 0, hi = v.batch;  // row_start[lo] <= i < row_start[hi], if it is in order
  if (i < __ldg(v.row_start) || i >= __ldg(v.row_start + hi)) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(v.row_start + mid) <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ const uint8_t* kv4_block_at(const Kv4View& v, int page, int head, int bytes) {
  return v.pages + ((size_t)page * v.heads + head) * bytes;
}

// ---- many-row attention: operands in the workspace (kv4_prep.cu, kv4_attn_tc.cu) ----
struct Kv4Tc {
  void* q16;         // f16 [heads][rows * G][128]: row `row * G + g` of a K/V head
  float* q_scale;    // [heads][rows * G]: softmax scale * log2(e) / the row's power of two
  void* k16;         // f16 [batch * heads][tokens][128]
  void* v16;
  float2* top;       // [batch * heads][chunks]: largest |K|, |V| of 16 pages
  float2* kv_scale;  // [batch * heads]: 1 / the powers of two of K and V
  float* o_part;     // [splits][heads][rows * G][128], with splits > 1
  float* ml_part;    // [splits][heads][rows * G][2]: reference maximum, sum
  int tokens, chunks, G, splits;
  float cs;          // softmax scale * log2(e)
};
int kv4_prepare(const Kv4View& c, const Kv4Tc& t, const void* q, size_t ldq, int group, cudaStream_t st);
int kv4_attention_tc(const Kv4View& c, const Kv4Tc& t, const float* gate, void* out, int causal, cudaStream_t st);
// rows of a query tile pair, and the K/V splits that fill the GPU
constexpr int KV4_TC_ROWS = 256;
int kv4_tc_splits(const Kv4View& c, int G);

// host side (kv4_cache.cu): argument checks shared by the entry points
int kv4_check(const ltxb_kv4_cache* c, const int32_t* row_start, int rows, const char* what, Kv4View* out);

}  // namespace ltxb
