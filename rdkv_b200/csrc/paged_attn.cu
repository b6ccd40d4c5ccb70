// Attention of the new tokens of a batch of requests over their paged keys and values.
//
// Request i's cache holds kv_len_i tokens, the last n_i = q_start[i+1] - q_start[i] of them new ones: query row j of
// the request stands at position p = kv_len_i - n_i + j and sees key s if s <= p, and, under a window of w tokens,
// s > p - w or s < sinks, and if the page of s is there (a page number outside the pages stands for none):
//   o = sum_s softmax_s(scale * q.k_s) v_s;  a row that sees nothing is zero (record: m = -inf, l = 0).
#include <algorithm>

#include "rdkv_common.cuh"

namespace rdkv {

struct PagedArgs {
  const uint16_t* q; const uint16_t* k; const uint16_t* v;
  int64_t q_tok, q_head;                          // elements
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;
  int n_pages, page, page_log2, H_q, H_kv, g;
  const int32_t* table; int64_t table_stride; int width;
  const int32_t* q_start; const int32_t* kv_lens; int S, T;
  int window, sinks;                              // window 0: everything
  float scale;
  uint16_t* out; int64_t o_tok, o_head; int zero_pad;
  float* rec;                                     // [T][H_q][132] instead of out
};

template <bool BF16>
__device__ __forceinline__ float paged_up(uint16_t x) { return BF16 ? __uint_as_float((uint32_t)x << 16) : h2f(x); }
template <bool BF16>
__device__ __forceinline__ uint16_t paged_down(float x) {
  return BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
}

// One warp per (token, query head), four channels a lane, one key after the other.
template <bool BF16>
__global__ void __launch_bounds__(128)
paged_attn_plain_kernel(const PagedArgs A) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (int64_t)A.T * A.H_q) return;
  const int t = (int)(row / A.H_q), hq = (int)(row - (int64_t)t * A.H_q), h = hq / A.g;
  int lo = 0, hi = A.S;                                      // requests whose first token is at or before t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (A.q_start[mid + 1] <= t) lo = mid + 1; else hi = mid;
  }
  uint16_t* o16 = A.out + (int64_t)t * A.o_tok + (int64_t)hq * A.o_head + 4 * lane;
  float* rec = A.rec + row * RDKV_PARTIAL_STRIDE;
  if (lo >= A.S || A.q_start[lo] > t) {
    if (A.rec == nullptr && A.zero_pad) *reinterpret_cast<uint2*>(o16) = make_uint2(0u, 0u);
    return;
  }
  const int64_t len = min((int64_t)A.kv_lens[lo], (int64_t)A.width << A.page_log2);
  const int64_t pos = (int64_t)A.kv_lens[lo] - (A.q_start[lo + 1] - t);
  float q[4], o[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = paged_up<BF16>(A.q[(int64_t)t * A.q_tok + (int64_t)hq * A.q_head + 4 * lane + e]) * A.scale;
  for (int64_t s = 0; s < len && s <= pos; ++s) {
    if (A.window > 0 && s <= pos - A.window && s >= A.sinks) { s = max((int64_t)A.sinks - 1, pos - A.window); continue; }
    const int id = A.table[lo * A.table_stride + (s >> A.page_log2)];
    if (id < 0 || id >= A.n_pages) continue;
    const int64_t r = s & (A.page - 1);
    const uint16_t* kp = A.k + id * A.k_page + h * A.k_head + r * A.k_row + 4 * lane;
    const uint16_t* vp = A.v + id * A.v_page + h * A.v_head + r * A.v_row + 4 * lane;
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) x = fmaf(q[e], paged_up<BF16>(kp[e]), x);
    x = warp_sum(x);
    x = __shfl_sync(0xffffffffu, x, 0);
    const float n = fmaxf(m, x), a = m == -INFINITY ? 0.f : __expf(m - n), p = __expf(x - n);
    l = fmaf(l, a, p);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = fmaf(o[e], a, p * paged_up<BF16>(vp[e]));
    m = n;
  }
  if (A.rec != nullptr) {
    *reinterpret_cast<float4*>(rec + 4 + 4 * lane) = make_float4(o[0], o[1], o[2], o[3]);
    if (lane == 0) { rec[0] = m; rec[1] = l; rec[2] = 0.f; rec[3] = 0.f; }
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) o16[e] = paged_down<BF16>(l > 0.f || l != l ? o[e] / l : 0.f);
  }
}

}  // namespace rdkv

using namespace rdkv;

extern "C" int64_t rdkv_paged_attention_workspace(int n_requests, int n_tokens, int H_q, int H_kv, int max_new) {
  if (n_requests < 0 || n_tokens < 0 || H_q <= 0 || H_kv <= 0 || max_new < 0) return -1;
  return 0;
}

extern "C" int rdkv_paged_attention(const void* q, int64_t q_tok_stride, int64_t q_head_stride, int dtype, int n_tokens, int H_q,
                                    const void* k_pages, int64_t k_page_stride, int64_t k_head_stride, int64_t k_row_stride,
                                    const void* v_pages, int64_t v_page_stride, int64_t v_head_stride, int64_t v_row_stride,
                                    int n_pages, int H_kv, int page_size, const int32_t* block_tables, int64_t table_stride,
                                    int width, const int32_t* q_start, const int32_t* kv_lens, int n_requests, int max_new,
                                    int window, int sinks, float scale, void* out, int64_t out_tok_stride, int64_t out_head_stride,
                                    int zero_padding, float* out_partial, void* workspace, int64_t workspace_bytes, void* stream) {
  if (n_tokens < 0 || n_requests < 0 || H_q <= 0 || H_kv <= 0 || n_pages < 0 || width < 0 || window < 0 || sinks < 0 || max_new < 0)
    return RDKV_ERR_BAD_ARG;
  if (dtype != RDKV_F16 && dtype != RDKV_BF16) return RDKV_ERR_BAD_ARG;
  if (H_q % H_kv != 0 || H_q / H_kv > MAX_GROUP) return RDKV_ERR_BAD_SHAPE;
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)) != 0) return RDKV_ERR_BAD_SHAPE;
  if (n_tokens == 0) return RDKV_OK;
  if (q == nullptr || q_start == nullptr || (out == nullptr) == (out_partial == nullptr)) return RDKV_ERR_BAD_ARG;
  if (n_requests > 0 && (kv_lens == nullptr || (width > 0 && block_tables == nullptr))) return RDKV_ERR_BAD_ARG;
  if (n_pages > 0 && (k_pages == nullptr || v_pages == nullptr)) return RDKV_ERR_BAD_ARG;
  PagedArgs A = {};
  A.q = (const uint16_t*)q; A.k = (const uint16_t*)k_pages; A.v = (const uint16_t*)v_pages;
  A.q_tok = q_tok_stride; A.q_head = q_head_stride;
  A.k_page = k_page_stride; A.k_head = k_head_stride; A.k_row = k_row_stride;
  A.v_page = v_page_stride; A.v_head = v_head_stride; A.v_row = v_row_stride;
  A.n_pages = n_pages; A.page = page_size; A.H_q = H_q; A.H_kv = H_kv; A.g = H_q / H_kv;
  for (A.page_log2 = 0; (1 << A.page_log2) < page_size; ++A.page_log2) {}
  A.table = block_tables; A.table_stride = table_stride; A.width = width; A.q_start = q_start; A.kv_lens = kv_lens;
  A.S = n_requests; A.T = n_tokens; A.window = window; A.sinks = sinks; A.scale = scale;
  A.out = (uint16_t*)out; A.o_tok = out_tok_stride; A.o_head = out_head_stride; A.zero_pad = zero_padding; A.rec = out_partial;
  const int64_t blocks = ((int64_t)n_tokens * H_q + 3) / 4;
  if (blocks > 0x7fffffffLL) return RDKV_ERR_TOO_LARGE;
  if (dtype == RDKV_BF16) paged_attn_plain_kernel<true><<<(unsigned)blocks, 128, 0, (cudaStream_t)stream>>>(A);
  else paged_attn_plain_kernel<false><<<(unsigned)blocks, 128, 0, (cudaStream_t)stream>>>(A);
  return launch_status();
}
