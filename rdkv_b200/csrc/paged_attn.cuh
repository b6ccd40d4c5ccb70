// Attention of the new tokens of a batch of requests over their paged keys and values: what its two kernels share.
//
// Request i's cache holds kv_len_i tokens, the last n_i = q_start[i+1] - q_start[i] of them new ones: query row j of
// the request stands at position p = kv_len_i - n_i + j (also where the tensor has not all of the n_i rows) and sees key s if s <= p, and, under a window of w tokens,
// s > p - w or s < sinks, and if the page of s is there (a page number outside the pages stands for none):
//   o = sum_s softmax_s(scale * q.k_s) v_s;  a row that sees nothing is zero (record: m = -inf, l = 0).
//
// Both kernels cut their work the same way.  An ITEM is (request, group of its new tokens, KV head): the rows (token, query
// head of the KV head) of the group stand one under the other in one tile of the tensor cores.  Its keys come in
// tiles; only tiles that some row of the group can see count (the sinks' tiles, then the window's).  All items in order,
// their tiles one after another and a fixed cost each, make one line of units, which is cut into as many equal parts
// as there are CTAs: long contexts and short ones, chunks and single tokens balance without a plan from the host.
// Every CTA finds its part of the line from the lengths alone (paged_place), so nothing has to be known or copied
// before the launch.  An item that a cut goes through leaves records (m, l, o) of its parts, which a small dependent
// kernel joins in order: the same bits every time.
#pragma once

#include <algorithm>
#include <cstring>

#include "sm100.cuh"

namespace rdkv {

constexpr float PAGED_LOG2E = 1.4426950408889634f, PAGED_LN2 = 0.6931471805599453f;
constexpr int PAGED_SMS = 148;
constexpr int PAGED_CHANNELS = 128;

struct PagedArgs {
  const uint16_t* q; const uint16_t* k; const uint16_t* v;
  int64_t q_tok, q_head;                          // elements
  int64_t k_page, k_head, k_row, v_page, v_head, v_row;
  int n_pages, page, page_log2, H_q, H_kv, g;
  const int32_t* table; int64_t table_stride; int width;
  int cap;                                        // tokens a row of the table has room for
  const int32_t* q_start; const int32_t* kv_lens; int S, T;
  int window, sinks;                              // window 0: everything
  int group;                                      // new tokens of an item
  float scale_log2;                               // scale * log2 e: scores are kept in base 2
  uint16_t* out; int64_t o_tok, o_head; int zero_pad;
  float* rec;                                     // [T][H_q][132] instead of out
  uint32_t wait_ns;                               // how long a wait may take
  // workspace
  int4* place;                                    // [G+1][2] where CTA c starts: request, head, group, tile; the item's tiles, rows, first query row
  int* status;                                    // [G] bits: 1 a wait of the CTA ran out, 2 q_start falls
  float* part;                                    // [2 G][rows of an item][132] records of cut items
};

template <bool BF16>
__device__ __forceinline__ float paged_up(uint16_t x) { return BF16 ? __uint_as_float((uint32_t)x << 16) : h2f(x); }
template <bool BF16>
__device__ __forceinline__ uint32_t paged_pack(float lo, float hi) {   // two values rounded to the 16-bit type
  if (BF16) { const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const uint32_t*>(&v); }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Softmax weights are rounded to the 16-bit type for the second product (its operands have one type, and the values
// have that one): half a step of each weight's own size, against which the total is kept unrounded in 32 bits.  The
// running maximum only moves when a score passes it by more than RAISE (in base 2), so that accumulators are rarely
// rescaled; fp16 weights are 2^LIFT times larger, which keeps all that are over 2^-24 of the largest out of its subnormals.
template <bool BF16> struct PagedWeights { static constexpr float RAISE = 8.f, LIFT = 0.f; };
template <> struct PagedWeights<false> { static constexpr float RAISE = 4.f, LIFT = 10.f; };

int paged_decode_launch(const PagedArgs& A, bool bf16, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st);
int paged_chunk_launch(const PagedArgs& A, bool bf16, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st);
constexpr int PAGED_CHUNK_ROWS = 256, PAGED_CHUNK_CTAS = PAGED_SMS, PAGED_CHUNK_KEYS = 128;
constexpr int PAGED_DECODE_ROWS = 16, PAGED_DECODE_CTAS = 2 * PAGED_SMS, PAGED_DECODE_KEYS = 64;
constexpr int PAGED_STATUS_WORDS = 2 * PAGED_SMS;   // one a CTA, of the larger grid
static_assert(PAGED_STATUS_WORDS % 4 == 0 && PAGED_STATUS_WORDS >= PAGED_DECODE_CTAS && PAGED_STATUS_WORDS >= PAGED_CHUNK_CTAS);

// A pair of 16-bit values: bits 15 and 31 of the result say which of them is not finite (its exponent is all ones: one more carries over).
template <bool BF16>
__device__ __forceinline__ uint32_t paged_exponent_full(uint32_t x) {
  return BF16 ? (x & 0x7F807F80u) + 0x00800080u : (x & 0x7C007C00u) + 0x04000400u;
}
// The pair with zeros in the place of what is not finite.
template <bool BF16>
__device__ __forceinline__ uint32_t paged_finite(uint32_t x) { return x & ~((paged_exponent_full<BF16>(x) >> 15 & 0x00010001u) * 0xFFFFu); }
template <bool BF16>
__device__ __forceinline__ bool paged_not_finite(uint32_t x) { return (paged_exponent_full<BF16>(x) & 0x80008000u) != 0u; }

// x * y + z of pairs of 16-bit values.
template <bool BF16>
__device__ __forceinline__ uint32_t paged_fma2(uint32_t x, uint32_t y, uint32_t z) {
  uint32_t r;
  if (BF16) asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(z));
  else asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(z));
  return r;
}

// ── items ───────────────────────────────────────────────────────────────────
struct PagedRequest { int q0, n, len; };          // first query row, query rows, tokens up to the last row's (at most 0: none is seen)
struct PagedItem {
  int tok0, n_tok;                                // query rows of the group
  int p0;                                         // position of the first (below zero: it sees nothing)
  int hi;                                         // keys [0, hi) are in front of the last one's end
  int t_lo, t_sink, n;                            // tiles [0, t_sink) and from t_lo on: n in all
};

__device__ __forceinline__ PagedRequest paged_request(const PagedArgs& A, int i) {
  PagedRequest r;
  r.q0 = min(max(A.q_start[i], 0), A.T);
  const int end = A.q_start[i + 1], t1 = min(max(end, r.q0), A.T);
  r.n = t1 - r.q0;
  r.len = max(max(A.kv_lens[i], 0) - max(end - A.T, 0), 0);   // (tokens behind the last row there is are not this call's, but they are among kv_lens)
  return r;
}
// Whether q_start falls behind request i (one of a batch's requests; other numbers: no).
__device__ __forceinline__ bool paged_falls(const PagedArgs& A, int i) { return i < A.S && A.q_start[i + 1] < A.q_start[i]; }
__device__ __forceinline__ int paged_groups(const PagedArgs& A, const PagedRequest& r) { return (r.n + A.group - 1) / A.group; }

template <int KEYS>
__device__ __forceinline__ PagedItem paged_item(const PagedArgs& A, const PagedRequest& r, int group) {
  PagedItem it;
  const int j0 = group * A.group;
  it.tok0 = r.q0 + j0;
  it.n_tok = min(A.group, r.n - j0);
  it.p0 = r.len - r.n + j0;
  it.hi = max(0, min(it.p0 + it.n_tok, A.cap));
  const int t_hi = (it.hi + KEYS - 1) / KEYS;
  const int lo = A.window > 0 ? max(0, it.p0 - A.window + 1) : 0;
  it.t_lo = min(lo / KEYS, t_hi);
  it.t_sink = A.window > 0 ? min((min(A.sinks, it.hi) + KEYS - 1) / KEYS, it.t_lo) : 0;
  it.n = it.t_sink + t_hi - it.t_lo;
  return it;
}
__device__ __forceinline__ int paged_tile(const PagedItem& it, int k) { return k < it.t_sink ? k : it.t_lo + k - it.t_sink; }

// ── the line of units ───────────────────────────────────────────────────────
struct PagedPlace { int i, head, group, tile; };  // head = H_kv: the end

struct PagedPlaceScratch { uint32_t part[32], most[32], groups[32]; uint32_t at[2]; int request[2]; int4 found[2], item; };

// Where the part of CTA c of G starts and ends.  All threads of the block (NT, whole warps) call it.  The line goes through
// the heads, in a head through the requests, in a request through its groups.  FIXED: cost of an item besides its tiles; a cut that
// would leave fewer than SNAP tiles of an item on one side is moved to the item's edge.  With no more items than CTAs, and
// none more than WHOLE units over its share, every CTA gets a whole item: a cut costs both its sides an item's records,
// written and read again.  The launcher has seen to it that a head's units fit 31 bits.  (Every launch pays for this code from
// a cold instruction cache: in 64 bits, with two divisions more, it took 7400 cycles.)  Returns false, and the end as both places,
// where q_start falls somewhere: requests would share query rows.
template <int KEYS, int NT, int FIXED, int SNAP, int WHOLE, int G>
__device__ __forceinline__ bool paged_place(const PagedArgs& A, int c, PagedPlaceScratch& s, PagedPlace& from, PagedPlace& to) {
  constexpr uint32_t FALLS = 0x80000000u;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // units of a head of request i, its groups, its costliest item (FALLS: q_start falls there)
  auto units = [&](int i, uint32_t& groups_, uint32_t& most) -> uint32_t {
    PagedRequest r = {0, 0, 0};
    if (i < A.S) r = paged_request(A, i);
    const int groups = paged_groups(A, r);
    groups_ = (uint32_t)groups;
    uint32_t sum = 0;
    most = 0;
    if (groups == 1) sum = most = paged_item<KEYS>(A, r, 0).n + FIXED;
    unsigned many = __ballot_sync(0xffffffffu, groups > 1);   // chunks: the warp's lanes take their groups
    while (many != 0) {
      const int from_lane = __ffs(many) - 1;
      many &= many - 1;
      PagedRequest o;
      o.q0 = __shfl_sync(0xffffffffu, r.q0, from_lane); o.n = __shfl_sync(0xffffffffu, r.n, from_lane);
      o.len = __shfl_sync(0xffffffffu, r.len, from_lane);
      const int n = paged_groups(A, o);
      uint32_t mine = 0, top = 0;
#pragma unroll 1
      for (int x = lane; x < n; x += 32) {
        const uint32_t cost = paged_item<KEYS>(A, o, x).n + FIXED;
        mine += cost; top = max(top, cost);
      }
      mine = __reduce_add_sync(0xffffffffu, mine);
      top = __reduce_max_sync(0xffffffffu, top);
      if (lane == from_lane) { sum = mine; most = top; }
    }
    if (paged_falls(A, i)) most = FALLS;
    return sum;
  };
  auto warp_scan = [&](uint32_t x) {                          // inclusive
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    return x;
  };
  auto block_scan = [&](uint32_t x, uint32_t& all) {          // exclusive
    const uint32_t incl = warp_scan(x);
    __syncthreads();
    if (lane == 31) s.part[warp] = incl;
    __syncthreads();
    uint32_t before = incl - x;
    all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      const uint32_t y = s.part[w];
      before += w < warp ? y : 0u;
      all += y;
    }
    return before;
  };
  if (tid < 2) s.request[tid] = -1;
  uint32_t total = 0, mine = 0, groups = 0, n_groups = 0, most = 0, before = 0, all = 0;
  for (int base = 0; base < A.S; base += NT) {
    uint32_t top;
    mine = units(base + tid, groups, top);
    top = __reduce_max_sync(0xffffffffu, top);
    const uint32_t sum = __reduce_add_sync(0xffffffffu, groups);
    if (base > 0) __syncthreads();                            // (the round before has been read)
    if (lane == 0) { s.most[warp] = top; s.groups[warp] = sum; }
    before = block_scan(mine, all);
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) { most = max(most, s.most[w]); n_groups += s.groups[w]; }
    total += all;
  }
  const bool ordered = most < FALLS;
  const bool whole = (uint64_t)n_groups * A.H_kv <= (uint64_t)G && most <= (uint32_t)((uint64_t)total * A.H_kv / G) + WHOLE;
  // cut e: its head, and its place in the head's line
  int head[2];
  uint32_t cut[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    if (whole) {
      head[e] = n_groups > 0 ? min((c + e) / (int)n_groups, A.H_kv) : A.H_kv;
      cut[e] = (uint32_t)(c + e - head[e] * (int)n_groups);
    } else {
      const int x = (c + e) * A.H_kv;
      head[e] = x / G;
      cut[e] = (uint32_t)((uint64_t)(x - head[e] * G) * total / G);
    }
  }
  if (whole) { total = n_groups; if (A.S <= NT) { mine = groups; before = block_scan(mine, all); } }
  uint32_t run = 0;
  for (int base = 0; base < A.S; base += NT) {
    if (A.S > NT) {
      uint32_t top;
      mine = units(base + tid, groups, top);
      if (whole) mine = groups;
      before = block_scan(mine, all);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (ordered && head[e] < A.H_kv && cut[e] - (run + before) < mine) { s.request[e] = base + tid; s.at[e] = cut[e] - (run + before); }
    run += all;
  }
  __syncthreads();
  if (warp < 2) {                                 // warp e: the group and tile of cut e
    const int i = s.request[warp];
    if (i >= 0) {
      const PagedRequest r = paged_request(A, i);
      const int n_mine = paged_groups(A, r);
      uint32_t left = s.at[warp];
#pragma unroll 1
      for (int x0 = 0;; x0 += 32) {
        const PagedItem it = paged_item<KEYS>(A, r, min(x0 + lane, n_mine - 1));
        const uint32_t cost = x0 + lane < n_mine ? (whole ? 1u : (uint32_t)(it.n + FIXED)) : 0u;
        const uint32_t incl = warp_scan(cost), sum = __shfl_sync(0xffffffffu, incl, 31);
        if (left < sum || x0 + 32 >= n_mine) {
          const uint32_t off = left - (incl - cost);
          if (off < cost) {
            int tile = whole ? 0 : max(0, (int)off - FIXED);
            if (tile < SNAP) tile = 0;
            else if (it.n - tile < SNAP) tile = it.n;
            s.found[warp] = make_int4(i, warp == 0 ? head[0] : head[1], x0 + lane, tile);
            if (warp == 0) s.item = make_int4(it.n, it.n_tok * A.g, it.tok0, 0);
          }
          break;
        }
        left -= sum;
      }
    } else if (lane == 0) {
      s.found[warp] = make_int4(0, A.H_kv, 0, 0);
      if (warp == 0) s.item = make_int4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  const int4 f = s.found[0], t = s.found[1];
  from = {f.x, f.y, f.z, f.w};
  to = {t.x, t.y, t.z, t.w};
  if (tid == 0) {
    A.place[2 * c] = f; A.place[2 * c + 1] = s.item;
    if (c == G - 1) A.place[2 * G] = make_int4(0, A.H_kv, 0, 0);
  }
  return ordered;
}

// The segments of a CTA: runs of tiles of one item.  Every role of the CTA walks them by itself.
struct PagedSegment {
  PagedRequest request;
  PagedItem item;
  int i, head, group, k0, k1;
};
template <int KEYS>
struct PagedWalk {
  PagedPlace at, to;
  PagedRequest r;
  int groups;
  bool done;
  __device__ __forceinline__ PagedWalk(const PagedArgs& A, const PagedPlace& from, const PagedPlace& end) : at(from), to(end), done(false) {
    load(A);
  }
  __device__ __forceinline__ void load(const PagedArgs& A) {
    groups = 0;
    if (at.head < A.H_kv) { r = paged_request(A, at.i); groups = paged_groups(A, r); }
  }
  __device__ __forceinline__ void next_request(const PagedArgs& A) {
    at.group = at.tile = 0;
    if (++at.i == A.S) { at.i = 0; ++at.head; }
    load(A);
  }
  __device__ __forceinline__ bool next(const PagedArgs& A, PagedSegment& s) {
    while (!done && at.head < A.H_kv) {
      if (groups == 0) { next_request(A); continue; }
      const bool last = at.head == to.head && at.i == to.i && at.group == to.group;
      s.request = r; s.i = at.i; s.head = at.head; s.group = at.group;
      s.item = paged_item<KEYS>(A, r, at.group);
      s.k0 = at.tile;
      s.k1 = last ? min(to.tile, s.item.n) : s.item.n;
      const bool some = s.k0 < s.k1 || (s.item.n == 0 && s.k0 == 0 && !last);
      at.tile = 0;
      if (last) done = true;
      else if (++at.group == groups) next_request(A);
      if (some) return true;
    }
    return false;
  }
};

// ── results ─────────────────────────────────────────────────────────────────
// Where a row of a segment goes: the result (normalised, 16 bits), the caller's record, or a record in the workspace.
struct PagedRow { uint16_t* out; float* rec; };
template <int ROWS>
__device__ __forceinline__ PagedRow paged_row(const PagedArgs& A, const PagedSegment& s, int row, int cta) {
  PagedRow d = {nullptr, nullptr};
  if (s.k0 == 0 && s.k1 == s.item.n) {
    const int tok = row / A.g, hq = s.head * A.g + (row - tok * A.g);
    const int64_t t = s.item.tok0 + tok;
    if (A.rec != nullptr) d.rec = A.rec + (t * A.H_q + hq) * RDKV_PARTIAL_STRIDE;
    else d.out = A.out + t * A.o_tok + hq * A.o_head;
  } else {
    d.rec = A.part + ((int64_t)(2 * cta + (s.k0 > 0 ? 0 : 1)) * ROWS + row) * RDKV_PARTIAL_STRIDE;
  }
  return d;
}
// 1 / l, or zero for a row that saw nothing (NaN stays NaN).
__device__ __forceinline__ float paged_over(float l) { return l == 0.f ? 0.f : __fdividef(1.f, l); }

// What values that are not finite add to rows [row0, row1) of a segment, whose results this warp has written.  A weight of zero times such a
// value is NaN, so the products take zero for it at keys that some rows of the item see and others do not.  Here every row that sees
// such a key gets the values themselves added, whose weight is positive: infinities and NaN stay what they are whatever it is.  These
// keys lie in front of the last row and behind the first, or at the window's end: fewer than two of them a new token of the
// item, however long the context, so that the other warps, which wait meanwhile, do so for microseconds.
template <bool BF16, int KEYS, int ROWS>
__device__ __noinline__ void paged_repair(const PagedArgs& A, const PagedSegment& s, int row0, int row1, int cta) {
  const int lane = threadIdx.x & 31, p_first = s.item.p0, p_last = s.item.p0 + s.item.n_tok - 1;
  const int d0 = max(p_first + 1, 0), n1 = max(s.item.hi - d0, 0);
  const int w0 = max(max(p_first - A.window + 1, A.sinks), 0);
  const int n = n1 + (A.window > 0 ? max(min(min(p_last - A.window, p_first), s.item.hi - 1) + 1 - w0, 0) : 0);   // (up to 510: a group has 256 tokens at most)
  auto key_of = [&](int x) { return x < n1 ? d0 + x : w0 + x - n1; };
  auto value = [&](int key) {                                // four channels a lane; zeros where the segment has not the key
    const int t = key / KEYS, k = t < s.item.t_sink ? t : t >= s.item.t_lo ? t - s.item.t_lo + s.item.t_sink : -1;
    if (k < s.k0 || k >= s.k1) return make_uint2(0u, 0u);
    const int id = A.table[s.i * A.table_stride + (key >> A.page_log2)];
    if (id < 0 || id >= A.n_pages) return make_uint2(0u, 0u);
    return *reinterpret_cast<const uint2*>(A.v + id * A.v_page + s.head * A.v_head + (int64_t)(key & (A.page - 1)) * A.v_row + 4 * lane);
  };
  uint32_t found = 0u;                                       // lane w: a bit for each of keys 32 w ... that has such a value
  for (int x0 = 0; x0 < n; x0 += 8) {
    uint2 v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x0 + i < n ? value(key_of(x0 + i)) : make_uint2(0u, 0u);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const bool bad = __any_sync(0xffffffffu, paged_not_finite<BF16>(v[i].x) || paged_not_finite<BF16>(v[i].y));
      if (bad && lane == x0 >> 5) found |= 1u << ((x0 + i) & 31);
    }
  }
  __syncwarp();
  for (int row = row0; row < row1;) {
    const int tok = row / A.g, end = min(row1, (tok + 1) * A.g), pos = p_first + tok;
    float4 add = make_float4(0.f, 0.f, 0.f, 0.f);
    auto plus = [](float& a, float x) { a += fabsf(x) < INFINITY ? 0.f : x; };
    for (int w = 0; 32 * w < n; ++w) {
      uint32_t bits = __shfl_sync(0xffffffffu, found, w);
      while (bits != 0u) {
        const int key = key_of(32 * w + __ffs(bits) - 1);
        bits &= bits - 1;
        if (key > pos || (A.window > 0 && key <= pos - A.window && key >= A.sinks)) continue;
        const uint2 v = value(key);
        plus(add.x, paged_up<BF16>(v.x & 0xFFFF)); plus(add.y, paged_up<BF16>(v.x >> 16));
        plus(add.z, paged_up<BF16>(v.y & 0xFFFF)); plus(add.w, paged_up<BF16>(v.y >> 16));
      }
    }
    const bool mine = add.x != 0.f || add.y != 0.f || add.z != 0.f || add.w != 0.f;
    for (; row < end; ++row) {
      if (!mine) continue;
      const PagedRow d = paged_row<ROWS>(A, s, row, cta);
      if (d.rec != nullptr) {
        float4* at = reinterpret_cast<float4*>(d.rec + 4 + 4 * lane);
        const float4 o = *at;
        *at = make_float4(o.x + add.x, o.y + add.y, o.z + add.z, o.w + add.w);
      } else {
        uint2* at = reinterpret_cast<uint2*>(d.out + 4 * lane);
        const uint2 o = *at;
        *at = make_uint2(paged_pack<BF16>(paged_up<BF16>(o.x & 0xFFFF) + add.x, paged_up<BF16>(o.x >> 16) + add.y),
                         paged_pack<BF16>(paged_up<BF16>(o.y & 0xFFFF) + add.z, paged_up<BF16>(o.y >> 16) + add.w));
      }
    }
  }
}

// Rows that belong to no request (all rows, where q_start falls and nothing was computed), in a result that the call allocated: zeros.
// All threads of the grid.
__device__ __forceinline__ void paged_zero_padding(const PagedArgs& A, int n_threads, bool falls) {
  if (!A.zero_pad || A.rec != nullptr) return;
  const int first = A.S > 0 && !falls ? min(max(A.q_start[0], 0), A.T) : A.T;
  const int end = A.S > 0 && !falls ? min(max(A.q_start[A.S], first), A.T) : A.T;
  const int64_t rows = (int64_t)(first + A.T - end) * A.H_q * 16;           // 16 bytes a step
  for (int64_t x = (int64_t)blockIdx.x * n_threads + threadIdx.x; x < rows; x += (int64_t)gridDim.x * n_threads) {
    const int64_t row = x >> 4, tk = row / A.H_q, hq = row - tk * A.H_q;
    const int64_t t = tk < first ? tk : end + (tk - first);
    *reinterpret_cast<uint4*>(A.out + t * A.o_tok + hq * A.o_head + (x & 15) * 8) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// The CTA's status word (the first CTA also writes those of CTAs that the launch does not have).
__device__ __forceinline__ void paged_report(const PagedArgs& A, int trouble) {
  if (threadIdx.x == 0) A.status[blockIdx.x] = trouble;
  if (blockIdx.x == 0)
    for (int i = gridDim.x + threadIdx.x; i < PAGED_STATUS_WORDS; i += blockDim.x) A.status[i] = 0;
}

// Joins the records of items that a cut went through.  Block (c, y): if the cut in front of CTA c is the first one inside an
// item, rows y, y + gridDim.y * 8, ... of that item, a warp each.  Its loads are three round trips: the places, the parts' m
// and l together with the first parts' sums, the rest.
constexpr int PAGED_JOIN_WARPS = 8;
template <bool BF16, int ROWS, int G>
__global__ void __launch_bounds__(PAGED_JOIN_WARPS * 32)
paged_join_kernel(const PagedArgs A) {
  __shared__ float s_w[PAGED_JOIN_WARPS][G];
  __shared__ uint8_t s_some[G + 1];                          // [0] the CTA in front of the cut
  const int c = blockIdx.x + 1, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  wait_for_previous_kernel();
  const int4 at = A.place[2 * c], item = A.place[2 * c + 1], prev = A.place[2 * c - 2];
  int4 a = A.place[2 * min(c + tid, G)], b = A.place[2 * min(c + tid + 1, G)];
  if (at.y >= A.H_kv || at.w == 0 || at.w >= item.x) return;
  if (prev.x == at.x && prev.y == at.y && prev.z == at.z && prev.w > 0) return;   // an earlier cut is in this item
  // the CTAs from c on that start inside the item (a run), and which of them have tiles of it
  int n_parts = 1;
  for (int base = c;; base += PAGED_JOIN_WARPS * 32) {
    const int x = base + tid;
    const bool in = x < G && a.x == at.x && a.y == at.y && a.z == at.z && a.w > 0 && a.w < item.x;
    if (x < G) s_some[x - c + 1] = in && !(b.x == at.x && b.y == at.y && b.z == at.z && b.w == a.w);
    const int n = __syncthreads_count(in);
    n_parts += n;
    if (n < PAGED_JOIN_WARPS * 32) break;
    a = A.place[2 * min(x + PAGED_JOIN_WARPS * 32, G)]; b = A.place[2 * min(x + PAGED_JOIN_WARPS * 32 + 1, G)];
  }
  if (tid == 0) s_some[0] = 1;
  __syncthreads();
  PagedSegment s;
  s.item.tok0 = item.z; s.item.n = item.x; s.head = at.y; s.k0 = 0; s.k1 = item.x;
  // record of part x (0: the CTA in front of the cut, its last segment; others: the first segment of CTA c + x - 1)
  auto record = [&](int x, int row) {
    return A.part + ((int64_t)(x == 0 ? 2 * (c - 1) + 1 : 2 * (c + x - 1)) * ROWS + row) * RDKV_PARTIAL_STRIDE;
  };
  auto sums = [&](int x, int row) {
    return x < n_parts && s_some[x] ? *reinterpret_cast<const float4*>(record(x, row) + 4 + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
  for (int row = blockIdx.y * PAGED_JOIN_WARPS + warp; row < item.y; row += gridDim.y * PAGED_JOIN_WARPS) {
    constexpr int EARLY = 8;
    float4 p[EARLY];
#pragma unroll
    for (int e = 0; e < EARLY; ++e) p[e] = sums(e, row);
    float M = -INFINITY, L = 0.f, l0 = 0.f;
    for (int x = lane; x < n_parts; x += 32) {
      float2 ml = make_float2(-INFINITY, 0.f);
      if (s_some[x]) ml = *reinterpret_cast<const float2*>(record(x, row));
      if (x == lane) l0 = ml.y;
      s_w[warp][x] = ml.x;
      M = fmaxf(M, ml.x);
    }
    M = warp_max(M);
    for (int x = lane; x < n_parts; x += 32) {
      const float m = s_w[warp][x], w = m == -INFINITY ? 0.f : exp2_approx((m - M) * PAGED_LOG2E);
      const float l = x == lane ? l0 : s_some[x] ? record(x, row)[1] : 0.f;
      L = fmaf(l, w, L);
      s_w[warp][x] = w;
    }
    L = warp_sum(L);
    __syncwarp();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int x0 = 0; x0 < n_parts; x0 += EARLY) {
#pragma unroll
      for (int e = 0; e < EARLY; ++e) {
        const float w = x0 + e < n_parts ? s_w[warp][x0 + e] : 0.f;
        o.x = fmaf(p[e].x, w, o.x); o.y = fmaf(p[e].y, w, o.y); o.z = fmaf(p[e].z, w, o.z); o.w = fmaf(p[e].w, w, o.w);
      }
      if (x0 + EARLY < n_parts)
#pragma unroll
        for (int e = 0; e < EARLY; ++e) p[e] = sums(x0 + EARLY + e, row);
    }
    const PagedRow d = paged_row<ROWS>(A, s, row, 0);
    if (d.rec != nullptr) {
      *reinterpret_cast<float4*>(d.rec + 4 + 4 * lane) = o;
      if (lane == 0) *reinterpret_cast<float4*>(d.rec) = make_float4(M, L, 0.f, 0.f);
    } else {
      const float w = paged_over(L);
      *reinterpret_cast<uint2*>(d.out + 4 * lane) = make_uint2(paged_pack<BF16>(o.x * w, o.y * w), paged_pack<BF16>(o.z * w, o.w * w));
    }
    __syncwarp();
  }
}

// A map over pages [n_pages][H_kv][page][128] (strides in elements) whose boxes are `rows` tokens of 64 channels, laid down with the
// 128-byte swizzle.  No pages: an empty map, which no kernel uses then.
inline bool paged_map(CUtensorMap* tm, const void* base, bool bf16, int64_t page_stride, int64_t head_stride, int64_t row_stride,
                      int64_t n_pages, int64_t heads, int64_t page, int rows) {
  memset(tm, 0, sizeof(*tm));
  if (n_pages == 0) return true;
  TensorMapEncoder enc = tensor_map_encoder();
  if (enc == nullptr || (reinterpret_cast<uintptr_t>(base) & 15) != 0) return false;
  if (heads == 1) head_stride = PAGED_CHANNELS;               // (strides of dimensions of one element mean nothing)
  if (n_pages == 1) page_stride = PAGED_CHANNELS;
  const cuuint64_t dims[4] = {PAGED_CHANNELS, (cuuint64_t)page, (cuuint64_t)heads, (cuuint64_t)n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)row_stride * 2u, (cuuint64_t)head_stride * 2u, (cuuint64_t)page_stride * 2u};
  const cuuint32_t box[4] = {64u, (cuuint32_t)rows, 1u, 1u}, elem[4] = {1u, 1u, 1u, 1u};
  if (row_stride <= 0 || head_stride <= 0 || page_stride <= 0 || (row_stride & 7) || (head_stride & 7) || (page_stride & 7)) return false;
  return enc(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, box,
             elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Workspace of a launch of G CTAs whose items have up to `rows` rows.
inline int64_t paged_workspace_bytes(int G, int rows) {
  return PAGED_STATUS_WORDS * 4 + (int64_t)(G + 1) * 32 + (int64_t)2 * G * rows * RDKV_PARTIAL_STRIDE * 4;
}
inline void paged_workspace(PagedArgs* A, void* workspace, int G) {
  char* p = static_cast<char*>(workspace);
  A->status = reinterpret_cast<int*>(p); p += PAGED_STATUS_WORDS * 4;
  A->place = reinterpret_cast<int4*>(p); p += (int64_t)(G + 1) * 32;
  A->part = reinterpret_cast<float*>(p);
}

template <class Kernel>
inline int paged_launch_join(Kernel join, const PagedArgs& A, dim3 grid, cudaStream_t st) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 1;
  cfg.gridDim = grid; cfg.blockDim = dim3(PAGED_JOIN_WARPS * 32);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, join, A);
  if (e != cudaSuccess) { g_last_cuda_error = (int)e; return RDKV_ERR_LAUNCH; }
  return launch_status();
}

}  // namespace rdkv
