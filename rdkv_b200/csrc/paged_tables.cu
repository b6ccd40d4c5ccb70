// Block tables and slot maps of a paged cache, from the requests' lengths, in one launch.
//
// Request i holds ctx_i tokens in ceil(ctx_i / P) pages and gets new_i more.  The pages it lacks come from a list
// of free pages, in request order:
//   held_i = ceil(ctx_i / P),  need_i = max(0, min(ceil((ctx_i + new_i) / P), W) - held_i),  base_i = start + sum_{j<i} need_j
//   table[i][held_i + e] = free[base_i + e]   (e < need_i; -1 behind the list's end)
// and new token t of request i, at position p = ctx_i + t - q_start_i, gets slot table[i][p / P] * P + p % P.
//
// Every CTA works out both prefix sums (new tokens, new pages) for itself in shared memory and then writes its share of
// the entries; who owns a token or a page is found by bisection.  So nothing is handed from CTA to CTA: entries of
// the table that are read belong to pages held before, entries that are written to new ones.  Bound by latency:
// two dependent loads, a scan, a bisection, a store (16 requests of one new token 4.3 us, 512 requests with 46 thousand 5.3).
#include <algorithm>

#include "rdkv_common.cuh"

namespace rdkv {

constexpr int TABLES_THREADS = 512;
constexpr int TABLES_MAX_REQUESTS = 16384;       // two prefix sums of 4 bytes a request in shared memory

struct TablesArgs {
  const int32_t* ctx; const int32_t* fresh;      // [S]
  int32_t* table; int64_t table_stride;          // [S][width]
  const int32_t* free_pages; const int32_t* free_start;
  int S, width, n_free, page;
  int64_t n_tokens;
  int64_t* slot_map; int32_t* positions;         // [n_tokens]
  int32_t* q_start; int32_t* kv_lens;            // [S+1], [S]
  int32_t* free_next; int32_t* missing;          // [1]
};

// Inclusive sums of a pair over the block; the pair of the whole block in `all`.
__device__ __forceinline__ void tables_scan(int64_t& a, int64_t& b, int64_t& all_a, int64_t& all_b, int64_t (*s_part)[2]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) { a += x; b += y; }
  }
  if (lane == 31) { s_part[warp][0] = a; s_part[warp][1] = b; }
  __syncthreads();
  all_a = all_b = 0;
  int64_t before_a = 0, before_b = 0;
#pragma unroll
  for (int w = 0; w < TABLES_THREADS / 32; ++w) {
    if (w == warp) { before_a = all_a; before_b = all_b; }
    all_a += s_part[w][0]; all_b += s_part[w][1];
  }
  a += before_a; b += before_b;
}

// Largest i in [0, n] with begin[i] <= x (begin is non-decreasing, begin[0] <= x).
__device__ __forceinline__ int tables_owner(const int32_t* begin, int n, int64_t x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (begin[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(TABLES_THREADS)
paged_tables_kernel(const TablesArgs A) {
  extern __shared__ int32_t tables_smem[];
  __shared__ int64_t s_part[TABLES_THREADS / 32][2];
  __shared__ unsigned long long s_lost;
  int32_t* q_begin = tables_smem;                            // [S+1] new tokens before request i
  int32_t* p_begin = tables_smem + A.S + 1;                  // [S+1] new pages before request i
  const int tid = threadIdx.x, S = A.S;
  const uint32_t page = (uint32_t)A.page;
  const int64_t most = 0x7fffffff;
  if (tid == 0) s_lost = 0ull;
  __syncthreads();

  const int each = (S + TABLES_THREADS - 1) / TABLES_THREADS, i0 = min(S, tid * each), i1 = min(S, i0 + each);
  // pages request i lacks; `lost` counts those its row of the table has no room for
  auto lacks = [&](int64_t c, int64_t n, int64_t* lost) {
    const int64_t held = (c + page - 1) / page, full = (c + n + page - 1) / page;
    *lost = max((int64_t)0, full - max(held, min(full, (int64_t)A.width)));
    return max((int64_t)0, min(full, (int64_t)A.width) - held);
  };
  int64_t tok = 0, pages = 0, lost_sum = 0;
  for (int i = i0; i < i1; ++i) {
    int64_t lost;
    const int64_t c = max(A.ctx[i], 0), n = max(A.fresh[i], 0);
    tok += n; pages += lacks(c, n, &lost);
    lost_sum += lost;
  }
  int64_t tok_end = tok, pages_end = pages, tok_all, pages_all;
  tables_scan(tok_end, pages_end, tok_all, pages_all, s_part);
  int64_t tok_at = tok_end - tok, pages_at = pages_end - pages;
  for (int i = i0; i < i1; ++i) {
    int64_t lost;
    q_begin[i] = (int32_t)min(tok_at, most);
    p_begin[i] = (int32_t)min(pages_at, most);
    const int64_t c = max(A.ctx[i], 0), n = max(A.fresh[i], 0);
    tok_at += n; pages_at += lacks(c, n, &lost);
  }
  if (tid == 0) { q_begin[S] = (int32_t)min(tok_all, most); p_begin[S] = (int32_t)min(pages_all, most); }
  if (blockIdx.x == 0 && lost_sum > 0) atomicAdd(&s_lost, (unsigned long long)lost_sum);
  __syncthreads();

  const int64_t start = A.free_start != nullptr ? (int64_t)max(*A.free_start, 0) : 0;
  const int64_t at = (int64_t)blockIdx.x * TABLES_THREADS + tid, step = (int64_t)gridDim.x * TABLES_THREADS;
  auto free_page = [&](int64_t i) { return i < A.n_free ? A.free_pages[i] : -1; };
  // new pages
  for (int64_t x = at; x < p_begin[S]; x += step) {
    const int i = tables_owner(p_begin, S - 1, x);
    const int64_t e = ((int64_t)max(A.ctx[i], 0) + page - 1) / page + (x - p_begin[i]);
    A.table[(int64_t)i * A.table_stride + e] = free_page(start + x);
  }
  // new tokens, padding behind them
  for (int64_t t = at; t < A.n_tokens; t += step) {
    int64_t slot = -1;
    int32_t pos = 0;
    if (t < q_begin[S]) {
      const int i = tables_owner(q_begin, S - 1, t);
      const uint32_t c = (uint32_t)max(A.ctx[i], 0);
      const int64_t p64 = (int64_t)c + (t - q_begin[i]);
      const uint32_t p = (uint32_t)min(p64, most), e = p / page, held = c / page + (c % page != 0);
      int id = -1;
      if (e < (uint32_t)A.width)
        id = e < held ? A.table[(int64_t)i * A.table_stride + e] : free_page(start + p_begin[i] + (int64_t)(e - held));
      if (id >= 0) slot = (int64_t)id * page + p % page;
      pos = (int32_t)p;
    }
    A.slot_map[t] = slot;
    A.positions[t] = pos;
  }
  for (int64_t i = at; i <= S; i += step) {
    A.q_start[i] = q_begin[i];
    if (i < S) A.kv_lens[i] = (int32_t)min((int64_t)max(A.ctx[i], 0) + max(A.fresh[i], 0), most);
  }
  if (blockIdx.x == 0 && tid == 0) {
    const int64_t end = start + pages_all;
    A.free_next[0] = (int32_t)min(end, (int64_t)A.n_free);
    A.missing[0] = (int32_t)min((int64_t)s_lost + max((int64_t)0, end - max(start, (int64_t)A.n_free)), most);
  }
}

}  // namespace rdkv

using namespace rdkv;

extern "C" int rdkv_paged_tables(const int32_t* ctx_lens, const int32_t* new_lens, int n_requests, int32_t* block_tables,
                                 int64_t table_stride, int width, const int32_t* free_pages, int n_free, const int32_t* free_start,
                                 int page_size, int64_t n_tokens, int64_t* slot_map, int32_t* positions, int32_t* q_start,
                                 int32_t* kv_lens, int32_t* free_next, int32_t* missing, void* stream) {
  if (n_requests < 0 || width < 0 || n_free < 0 || page_size <= 0 || n_tokens < 0 || q_start == nullptr || free_next == nullptr ||
      missing == nullptr)
    return RDKV_ERR_BAD_ARG;
  if (n_requests > 0 && (ctx_lens == nullptr || new_lens == nullptr || kv_lens == nullptr || (width > 0 && block_tables == nullptr)))
    return RDKV_ERR_BAD_ARG;
  if ((n_free > 0 && free_pages == nullptr) || (n_tokens > 0 && (slot_map == nullptr || positions == nullptr))) return RDKV_ERR_BAD_ARG;
  if (width > 0 && n_requests > 1 && table_stride < width) return RDKV_ERR_BAD_SHAPE;
  if (n_requests > TABLES_MAX_REQUESTS || n_tokens > 0x7fffffffLL) return RDKV_ERR_TOO_LARGE;
  TablesArgs A;
  A.ctx = ctx_lens; A.fresh = new_lens; A.table = block_tables; A.table_stride = table_stride; A.free_pages = free_pages;
  A.free_start = free_start; A.S = n_requests; A.width = width; A.n_free = n_free; A.page = page_size; A.n_tokens = n_tokens;
  A.slot_map = slot_map; A.positions = positions; A.q_start = q_start; A.kv_lens = kv_lens; A.free_next = free_next; A.missing = missing;
  const size_t smem = sizeof(int32_t) * 2 * (size_t)(n_requests + 1);
  const cudaError_t e = allow_dynamic_smem_once<paged_tables_kernel>(sizeof(int32_t) * 2 * (TABLES_MAX_REQUESTS + 1));
  if (e != cudaSuccess) { g_last_cuda_error = (int)e; return RDKV_ERR_LAUNCH; }
  const int64_t items = std::max<int64_t>(n_tokens, n_requests + 1);
  const unsigned grid = (unsigned)std::min<int64_t>(148, (items + TABLES_THREADS - 1) / TABLES_THREADS);
  paged_tables_kernel<<<grid, TABLES_THREADS, smem, (cudaStream_t)stream>>>(A);
  return launch_status();
}
