// Attention of chunks of new tokens over paged caches on the fifth-generation tensor cores.
//
// An item is two halves of up to 128 rows (floor(128/g) new tokens x g query heads of a KV head each); its keys come in
// tiles of 128, which a half takes 64 at a time.  Per half and 64 keys: S = Q.K^T (tcgen05.mma, both operands in shared
// memory, fp32 scores in tensor memory), softmax of S by a warpgroup with one row per thread, the weights P written over S as
// 16-bit values, O += P.V (tcgen05.mma, P from tensor memory, V as it lies in the cache: MN-major).  Tensor memory is full:
// per half two buffers of 64 scores and an accumulator of 128 columns.  The scores of step t + 2 are asked for as soon as
// the weights of step t are used up, so a warpgroup has its next scores waiting when it is done with a step (with one
// buffer of 128 scores a half had nothing to do between its weights and its next scores, 1700 cycles of 3900 a tile).
//
// 12 warps: two warpgroups of softmax (half 0, half 1), and one of helpers: one warp works out the segments and brings in Q and the tiles (tiled TMA, one box
// per page and 64-channel panel, 128-byte swizzle, four slots of 32 KB for K and V in turn), two issue the products of a
// half each, one looks after masked values: 0 x NaN is NaN, so in tiles that some row of the item does not see whole it
// sets values of keys that no row sees to zero before the product, and values that are not finite where only some rows
// see their key; the rows that do get them added in the end (paged_repair).
//
// An accumulator is rescaled by the threads that own its rows, and only when a score passes the row's reference by more
// than PagedWeights::RAISE.  Every wait is bounded; a wait that runs out ends the CTA's work and sets its status word.
//
// What bounds it (2048 tokens behind 30000, 8 x 4 heads, bf16: 0.95 to 1.07 ms over several GPUs, 0.98 to 1.09 PFLOP/s):
// long launches reach the 1000 W limit, where the clock settles at 1.5 GHz; in short ones (2048 behind 6000: 3650 cycles
// a tile, of which the products need 2570) the chain of a step inside a softmax warp, about 1700 cycles for 345 instructions:
// tensor pipe 56 % busy, issue slots 52 %, exponential units 42 %; two of the instructions reload spilled registers, none stores them.
// Measured and dropped: two warps a row with shared
// references (sixteen softmax warps; 4040 cycles), the halves' products strictly in turn (4060), the weights worked out before
// the maximum is known (4450), next scores loaded under the exponentials (does not fit the registers).
#include "paged_attn.cuh"

namespace rdkv {

constexpr int CH_KEYS = PAGED_CHUNK_KEYS, CH_ROWS = PAGED_CHUNK_ROWS, CH_SLOTS = 4, CH_SOFTMAX_WARPS = 8, CH_THREADS = CH_SOFTMAX_WARPS * 32 + 128;
constexpr int CH_STEP = 64;                       // keys of a step
constexpr int CH_PANEL = 128 * 128;               // bytes: 128 rows of 64 channels
constexpr int CH_SLOT = 2 * CH_PANEL;
constexpr int CH_STAGE = 32 * 128;                // bytes a softmax warp's results pass through on their way out
constexpr size_t CH_SMEM = (size_t)(2 + CH_SLOTS) * CH_SLOT + CH_SOFTMAX_WARPS * CH_STAGE;   // (starts on 1024 bytes)
constexpr int CH_INFO = 8;                        // tiles whose description is kept (a softmax warp is at most three behind the loads)
// Every CH_POLY-th pair of exponentials goes to the FMA units.  (2048 behind 6000, thousand cycles: every 4th 369, every 8th 396, none 385.)
constexpr int CH_POLY = 4;
constexpr int CH_WORKS = 4;                       // segments whose description is kept
// (Six requests of up to 500 tokens behind up to 3000: 95 us with a fixed cost of one tile an item, 87 with two, 91 with three; cuts that
// leave a tile or two are moved: an item's records are 135 KB.)
constexpr int CH_FIXED = 2, CH_SNAP = 3, CH_WHOLE = 8;
constexpr int CH_SOFTMAX_REGS = 208, CH_HELPER_REGS = 88, CH_LAUNCH_REGS = 168;
static_assert(CH_SOFTMAX_WARPS * 32 * CH_SOFTMAX_REGS + 128 * CH_HELPER_REGS <= CH_THREADS * CH_LAUNCH_REGS,
              "the split draws on what the block was launched with");

// Barriers: Q arrived / free; [2 half + buffer] scores done, weights written, product with the values done; [slot] tile arrived / free,
// values looked after; [half] products at an end; [segment's place] its description written / no longer needed.
enum { CH_Q_FULL = 0, CH_Q_FREE = 1, CH_S_FULL = 2, CH_P_READY = 6, CH_O_DONE = 10, CH_FULL = 14, CH_FREE = CH_FULL + CH_SLOTS,
       CH_V_OK = CH_FREE + CH_SLOTS, CH_DRAINED = CH_V_OK + CH_SLOTS, CH_W_FULL = CH_DRAINED + 2, CH_W_FREE = CH_W_FULL + CH_WORKS,
       CH_BARS = CH_W_FREE + CH_WORKS };

struct ChunkTile { int key0, there, edge; };      // first key, a bit per 16 keys whose page is there, some row does not see all of it

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Pairs of fp32 values, one instruction for both.
__device__ __forceinline__ uint64_t two(float lo, float hi) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi)); return r; }
__device__ __forceinline__ void split(uint64_t x, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// 2^x of a pair on the FMA units, x < 128: x = n + f with |f| <= 1/2 (n by adding a number whose last place is 1), 2^f by the
// polynomial of degree 4 with the least relative error there (2.7e-6 = 2^-18.5, fitted by iterated weighted least squares), and 2^n
// from its bits; below -127 exactly zero, NaN stays NaN.
__device__ __forceinline__ uint64_t exp2_poly2(uint64_t x) {
  float a, b, ra, rb;
  split(x, a, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
  constexpr float MAGIC = 12582912.f + 127.f;              // 1.5 * 2^23, and the exponent's bias
  x = two(a, b);
  const uint64_t r = add2(x, two(MAGIC, MAGIC)), f = add2(x, fma2(r, two(-1.f, -1.f), two(MAGIC, MAGIC)));
  uint64_t p = fma2(f, two(0.009570101968f, 0.009570101968f), two(0.05591786076f, 0.05591786076f));
  p = fma2(p, f, two(0.2402474483f, 0.2402474483f));
  p = fma2(p, f, two(0.6931218147f, 0.6931218147f));
  p = fma2(p, f, two(0.9999992614f, 0.9999992614f));
  split(r, ra, rb);
  return mul2(p, two(__uint_as_float(__float_as_uint(ra) << 23), __uint_as_float(__float_as_uint(rb) << 23)));
}

// Whether some row of the item does not see the whole tile.
__device__ __forceinline__ bool chunk_edge(const PagedArgs& A, const PagedItem& it, int key0, int there) {
  const int p_last = it.p0 + it.n_tok - 1;
  return key0 + CH_KEYS - 1 > it.p0 || there != 0xFF || (A.window > 0 && key0 <= p_last - A.window && key0 + CH_KEYS > A.sinks);
}

// Steps of a segment that half h takes: up to the end of what its last row sees, but under a window not the second step of the
// last tile of sinks, where they end before it, nor the first of the window's first tile, where the window begins behind it (4000 tokens
// behind 8000, window 1024 and 4 sinks: 18 steps an item for 19.5, 121.5 -> 117.6 us; four requests of 1000 tokens under a window of 256
// 46.8 -> 40.1).  Every tile in front of the end keeps a step.
template <bool WINDOW>
struct ChunkSteps {
  int n, end, skip_sinks, skip_front;             // steps taken; end of all; the two that may be left out (-1: none)
  ChunkSteps() = default;
  __device__ __forceinline__ ChunkSteps(const PagedArgs& A, const PagedSegment& s, int h, int tm) : n(0), end(0), skip_sinks(-1), skip_front(-1) {
    const int n_tok = min(tm, s.item.n_tok - h * tm);
    if (n_tok <= 0) return;
    const int p0 = s.item.p0 + h * tm, last = min(p0 + n_tok, A.cap);
    end = 2 * (s.k1 - s.k0);
    while (end > 0 && paged_tile(s.item, s.k0 + ((end - 1) >> 1)) * CH_KEYS + ((end - 1) & 1) * CH_STEP >= last) --end;
    n = end;
    if (!WINDOW) return;
    const int sinks = 2 * (s.item.t_sink - s.k0) - 1, front = sinks + 1, key0 = s.item.t_lo * CH_KEYS;
    if (sinks > 0 && sinks < end && A.sinks <= (s.item.t_sink - 1) * CH_KEYS + CH_STEP) { skip_sinks = sinks; --n; }
    if (front >= 0 && front + 1 < end && A.sinks <= key0 && p0 - A.window + 1 >= key0 + CH_STEP) { skip_front = front; --n; }
  }
  __device__ __forceinline__ int next(int t) const {         // (the two may be neighbours)
    if (!WINDOW) return t + 1;
    t += t + 1 == skip_sinks ? 2 : 1;
    return t == skip_front ? t + 1 : t;
  }
};

// A segment as the loading warp worked it out, for the other warps.  (Each of them used to walk the line of units by itself: that cost the
// softmax warps 2400 cycles a segment, most of them waits for code that is seldom run.)
template <bool WINDOW>
struct ChunkWork { PagedSegment s; ChunkSteps<WINDOW> st[2]; };   // s.k0 < 0: there are no more

// Waits for the description of segment `at`; false if there is none, or (not ok) the wait ran out.  A half without rows waits here while the
// other takes the tiles of the segment before: the limit once more for every 1024 of them (2 ms for 2 us).
template <bool WINDOW>
__device__ __forceinline__ bool chunk_work(const ChunkWork<WINDOW>* works, unsigned at, uint32_t bar, uint32_t limit, bool& ok) {
  for (int r = 0; ok && !bar_wait_warp(bar + 8 * (CH_W_FULL + at % CH_WORKS), (at / CH_WORKS) & 1, limit); ++r) {
    const PagedSegment& before = works[(at + CH_WORKS - 1) % CH_WORKS].s;
    ok = at > 0 && r < __shfl_sync(0xffffffffu, before.k1 - before.k0, 0) >> 10;
  }
  return ok && works[at % CH_WORKS].s.k0 >= 0;
}
__device__ __forceinline__ void chunk_work_done(unsigned at, uint32_t bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) bar_arrive(bar + 8 * (CH_W_FREE + at % CH_WORKS));
}

template <bool BF16, bool WINDOW>
__device__ void chunk_load(const PagedArgs& A, const CUtensorMap* tm_q, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                           PagedWalk<CH_KEYS> walk, uint32_t q32, uint32_t ring, uint32_t bar, ChunkTile* s_info, ChunkWork<WINDOW>* works, int* s_trouble) {
  const int lane = threadIdx.x & 31, tm = A.group >> 1;
  const int rows_log2 = min(A.page_log2, 7), rows = 1 << rows_log2, per_log2 = 7 - rows_log2, per_tile = 1 << per_log2, batch = 32 >> per_log2;
  const int box = lane >> 1, panel = lane & 1;               // this lane's box of a tile
  unsigned use = 0, tile = 0, segments = 0, published = 0;   // slots filled; tiles; segments that have some; all segments
  PagedSegment s;
  bool ok = true;
  auto publish = [&]() {
    const int at = published % CH_WORKS;
    if (published >= CH_WORKS) ok = ok && bar_wait_warp(bar + 8 * (CH_W_FREE + at), (published / CH_WORKS - 1) & 1, A.wait_ns);
    if (!ok) return;
    if (lane < 2) works[at].st[lane] = ChunkSteps<WINDOW>(A, s, lane, tm);
    if (lane == 0) works[at].s = s;
    __syncwarp();
    if (lane == 0) bar_arrive(bar + 8 * (CH_W_FULL + at));
    ++published;
  };
  while (ok && walk.next(A, s)) {
    if (s.k0 == s.k1) { publish(); continue; }
    const int32_t* table = A.table + s.i * A.table_stride;
    auto page_of = [&](int k) {                              // lane's entry of the batch that starts with tile k
      const int kk = k + (lane >> per_log2);
      if (kk >= s.k1) return -1;
      const int key = paged_tile(s.item, kk) * CH_KEYS + ((lane & (per_tile - 1)) << rows_log2);
      return key < s.item.hi ? table[key >> A.page_log2] : -1;
    };
    int ids = page_of(s.k0), ids_next = -1;
    const int halves = s.item.n_tok > tm ? 2 : 1;
    if (segments > 0 && !bar_wait_warp(bar + 8 * CH_Q_FREE, (segments - 1) & 1, A.wait_ns)) { ok = false; break; }
    if (lane == 0) {
      bar_arrive_tx(bar + 8 * CH_Q_FULL, (uint32_t)halves * 2u * (uint32_t)(tm * A.g) * 128u);
      for (int h = 0; h < halves; ++h)
        for (int p = 0; p < 2; ++p)
          tma_load_3d(q32 + h * CH_SLOT + p * CH_PANEL, tm_q, 64 * p, s.head * A.g, s.item.tok0 + h * tm, bar + 8 * CH_Q_FULL);
    }
    __syncwarp();
    ++segments;
    for (int k = s.k0; ok && k < s.k1; ++k, ++tile) {
      const int in_batch = (k - s.k0) & (batch - 1);
      if (in_batch == 0) {
        if (k > s.k0) ids = ids_next;
        ids_next = page_of(k + batch);
      }
      const int key0 = paged_tile(s.item, k) * CH_KEYS;
      const int id = __shfl_sync(0xffffffffu, ids, in_batch * per_tile + (box < per_tile ? box : 0));
      const bool there = box < per_tile && id >= 0 && id < A.n_pages;
      const unsigned lanes = __ballot_sync(0xffffffffu, there);
      if (lane == 0) {
        int mask = 0;
        for (int x = 0; x < 8; ++x) mask |= (int)(lanes >> (2 * (x * 16 >> rows_log2)) & 1u) << x;
        s_info[tile % CH_INFO] = {key0, mask, chunk_edge(A, s.item, key0, mask) ? 1 : 0};
      }
      const uint32_t bytes = (uint32_t)__popc(lanes) * (uint32_t)rows * 128u;
      for (int t = 0; t < 2; ++t, ++use) {                   // K, then V
        const int slot = use % CH_SLOTS;
        if (use >= CH_SLOTS && !bar_wait_warp(bar + 8 * (CH_FREE + slot), (use / CH_SLOTS - 1) & 1, A.wait_ns)) { ok = false; break; }
        if (lane == 0) {
          if (bytes > 0) bar_arrive_tx(bar + 8 * (CH_FULL + slot), bytes);
          else bar_arrive(bar + 8 * (CH_FULL + slot));
        }
        __syncwarp();
        if (there)
          tma_load_4d(ring + slot * CH_SLOT + panel * CH_PANEL + box * rows * 128, t == 0 ? tm_k : tm_v, 64 * panel, key0 & (A.page - 1),
                      s.head, id, bar + 8 * (CH_FULL + slot));
      }
      if (k == s.k0) publish();                              // (behind the first loads, which the start waits for)
    }
  }
  if (ok) { s.k0 = s.k1 = -1; s.item.n_tok = 0; publish(); }
  if (!ok) *s_trouble = 1;
  // copies that are still on their way when nobody waits for them any more must not land in the shared memory of the next CTA
  for (unsigned n = use < CH_SLOTS ? 0 : use - CH_SLOTS; n < use; ++n) bar_wait(bar + 8 * (CH_FULL + n % CH_SLOTS), (n / CH_SLOTS) & 1, WAIT_NS);
  if (segments > 0) bar_wait(bar + 8 * CH_Q_FULL, (segments - 1) & 1, WAIT_NS);
}

__device__ __forceinline__ int chunk_uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Two warps: the products of half 0, of half 1.
template <bool BF16, bool WINDOW>
__device__ void chunk_products(int h, uint32_t limit, uint32_t q32, uint32_t ring, uint32_t bar, uint32_t tmem_, const ChunkTile* s_info,
                               const ChunkWork<WINDOW>* works, int* s_trouble) {
  constexpr uint32_t QK = mma_idesc<BF16>(CH_STEP, false), PV = mma_idesc<BF16>(128, true);
  const uint32_t t_s = (uint32_t)chunk_uniform((int)tmem_ + 128 * h), t_o = t_s + 256, one = elect_one();
  const uint64_t q = desc_k_major((uint32_t)chunk_uniform((int)(q32 + h * CH_SLOT)));
  int tile = 0;                                              // tile x is in slots 2 (x & 1) and the next, their phase is x >> 1
  uint32_t segments = 0, v_ok = 0, p_phase = 0;              // a bit per V slot / buffer: parity of its next use
  bool ok = true;
  auto wait = [&](int b, uint32_t parity) { ok = ok && bar_wait_warp(bar + 8 * b, parity, limit); };
  auto wait_k = [&](int x) { wait(CH_FULL + 2 * (x & 1), x >> 1 & 1); };
  auto wait_v = [&](int x) {
    wait(CH_FULL + 2 * (x & 1) + 1, x >> 1 & 1);
    if (ok && chunk_uniform(s_info[x % CH_INFO].edge) != 0) {
      wait(CH_V_OK + 2 * (x & 1) + 1, v_ok >> (x & 1) & 1);
      v_ok ^= 1u << (x & 1);
    }
  };
  for (unsigned at = 0; chunk_uniform(chunk_work(works, at, bar, limit, ok)); ++at) {
    const ChunkWork<WINDOW>& work = works[at % CH_WORKS];
    const int n = chunk_uniform(work.s.k1 - work.s.k0);
    ChunkSteps<WINDOW> st = work.st[h];
    chunk_work_done(at, bar);
    if (n == 0) continue;
    st.skip_sinks = chunk_uniform(st.skip_sinks); st.skip_front = chunk_uniform(st.skip_front);
    const int steps = chunk_uniform(st.n), end = chunk_uniform(st.end);
    wait(CH_Q_FULL, segments++ & 1);
    int asked = st.next(-1), taken = asked, k_tile = -1, v_tile = -1;   // the next step to ask for / to take; tiles waited for
    auto scores = [&](int u) {                               // S = Q . K^T of the u-th step, into buffer u & 1
      const int t = asked, x = tile + (t >> 1);
      asked = st.next(t);
      if (WINDOW ? t >> 1 != k_tile : (t & 1) == 0) { wait_k(x); k_tile = t >> 1; }
      if (!ok) return;
      tmem_fence_after();
      const uint64_t k = desc_k_major(ring + 2 * (x & 1) * CH_SLOT + (t & 1) * (CH_STEP * 128));
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {                       // 16 channels: 32 bytes along the swizzled row, the second panel after four
        const uint64_t off = ((uint64_t)(kk >> 2) * CH_PANEL + (uint64_t)(kk & 3) * 32u) >> 4;
        mma_ss(one, t_s + CH_STEP * (u & 1), q + off, k + off, QK, kk > 0 ? 1u : 0u);
      }
      mma_commit(one, bar + 8 * (CH_S_FULL + 2 * h + (u & 1)));
      if (u == steps - 1 || (WINDOW ? asked >> 1 != t >> 1 : (t & 1) == 1)) mma_commit(one, bar + 8 * (CH_FREE + 2 * (x & 1)));
      if (u == steps - 1) mma_commit(one, bar + 8 * CH_Q_FREE);
    };
    if (steps > 0) scores(0);
    if (steps > 1) scores(1);
    for (int u = 0; ok && u < steps; ++u) {
      const int t = taken, x = tile + (t >> 1), b = u & 1;
      taken = st.next(t);
      if (WINDOW ? t >> 1 != v_tile : (t & 1) == 0) { wait_v(x); v_tile = t >> 1; }
      wait(CH_P_READY + 2 * h + b, p_phase >> b & 1);
      p_phase ^= 1u << b;
      if (!ok) break;
      tmem_fence_after();
      const uint64_t v = desc_mn_major(ring + (2 * (x & 1) + 1) * CH_SLOT + (t & 1) * (CH_STEP * 128), CH_PANEL);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)                         // 16 keys: 8 columns of P, two groups of eight rows of V
        mma_ts(one, t_o, t_s + CH_STEP * b + 8 * kk, v + kk * (2048 >> 4), PV, u > 0 || kk > 0 ? 1u : 0u);
      mma_commit(one, bar + 8 * (CH_O_DONE + 2 * h + b));
      if (u == steps - 1 || (WINDOW ? taken >> 1 != t >> 1 : (t & 1) == 1)) mma_commit(one, bar + 8 * (CH_FREE + 2 * (x & 1) + 1));
      if (u + 2 < steps) scores(u + 2);
    }
    // tiles that this half sees nothing of: their slots go back as they come
    if (steps == 0) mma_commit(one, bar + 8 * CH_Q_FREE);
    for (int x = tile + ((end + 1) >> 1); ok && x < tile + n; ++x) {
      wait_k(x);
      if (ok) mma_commit(one, bar + 8 * (CH_FREE + 2 * (x & 1)));
      wait_v(x);
      if (ok) mma_commit(one, bar + 8 * (CH_FREE + 2 * (x & 1) + 1));
    }
    tile += n;
  }
  if (!ok) *s_trouble = 1;
  // products that are still under way (the softmax warps may have given up) must not outlive the tensor memory
  mma_commit(one, bar + 8 * (CH_DRAINED + h));
  bar_wait_warp(bar + 8 * (CH_DRAINED + h), 0, WAIT_NS);
}

// One warp: values in masked places.
template <bool BF16, bool WINDOW>
__device__ void chunk_values(const PagedArgs& A, unsigned char* ring_ptr, uint32_t bar, const ChunkTile* s_info, const ChunkWork<WINDOW>* works,
                             int* s_again, int* s_trouble) {
  const int lane = threadIdx.x & 31;
  unsigned use = 0, tile = 0, segments = 0;
  bool ok = true;
  for (unsigned at = 0; chunk_work(works, at, bar, A.wait_ns, ok); ++at) {
    const PagedSegment s = works[at % CH_WORKS].s;
    chunk_work_done(at, bar);
    if (s.k0 == s.k1) continue;
    const int p_first = s.item.p0, p_last = s.item.p0 + s.item.n_tok - 1;
    for (int j = s.k0; ok && j < s.k1; ++j, ++tile) {
      for (int t = 0; t < 2; ++t, ++use) {
        const int slot = use % CH_SLOTS;
        if (!bar_wait_warp(bar + 8 * (CH_FULL + slot), (use / CH_SLOTS) & 1, A.wait_ns)) { ok = false; break; }
        const ChunkTile info = s_info[tile % CH_INFO];
        if (t == 1 && info.edge) {
          // 16 keys at a time that not every row sees: eight lanes a key, a 16-byte chunk of each panel a lane.  x * 0 added up
          // is not a number as soon as one x is not finite.
          uint32_t sum[4] = {0u, 0u, 0u, 0u};
          for (int g = 0; g < 8; ++g) {
            const int key0 = info.key0 + 16 * g;
            const bool gone = (info.there >> g & 1) == 0 || key0 >= s.item.hi;
            if (!gone && key0 + 15 <= p_first && (!WINDOW || key0 > p_last - A.window || key0 + 15 < A.sinks)) continue;
            uint4* at = reinterpret_cast<uint4*>(ring_ptr + slot * CH_SLOT + (16 * g + (lane >> 3)) * 128 + (lane & 7) * 16);
            const int mine = key0 + (lane >> 3), low = WINDOW ? p_first - A.window : -1;   // (keys up to `low`, behind the sinks: no row's)
            if (gone || key0 + 15 >= s.item.hi || (key0 <= low && key0 + 15 >= A.sinks)) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int key = mine + 4 * i;
                if (gone || key >= s.item.hi || (key <= low && key >= A.sinks)) at[i * 32] = at[i * 32 + CH_PANEL / 16] = make_uint4(0u, 0u, 0u, 0u);
              }
              if (gone) continue;
            }
            uint4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = at[(i >> 1) * 32 + (i & 1) * (CH_PANEL / 16)];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              sum[0] = paged_fma2<BF16>(v[i].x, 0u, sum[0]); sum[1] = paged_fma2<BF16>(v[i].y, 0u, sum[1]);
              sum[2] = paged_fma2<BF16>(v[i].z, 0u, sum[2]); sum[3] = paged_fma2<BF16>(v[i].w, 0u, sum[3]);
            }
          }
          const bool again = paged_not_finite<BF16>(sum[0]) || paged_not_finite<BF16>(sum[1]) || paged_not_finite<BF16>(sum[2]) ||
                             paged_not_finite<BF16>(sum[3]);
          if (__any_sync(0xffffffffu, again)) {
            if (lane == 0) s_again[segments & 3] = (int)segments + 1;
            for (int g = 0; g < 8; ++g) {
              uint4* at = reinterpret_cast<uint4*>(ring_ptr + slot * CH_SLOT + (16 * g + (lane >> 3)) * 128 + (lane & 7) * 16);
              const int mine = info.key0 + 16 * g + (lane >> 3);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int key = mine + 4 * i;
                if (key <= p_first && !(WINDOW && key >= A.sinks && key <= p_last - A.window)) continue;   // (all rows see it)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                  uint4 x = at[i * 32 + p * (CH_PANEL / 16)];
                  x.x = paged_finite<BF16>(x.x); x.y = paged_finite<BF16>(x.y); x.z = paged_finite<BF16>(x.z); x.w = paged_finite<BF16>(x.w);
                  at[i * 32 + p * (CH_PANEL / 16)] = x;
                }
              }
            }
          }
          fence_async_smem();                                // (the product reads the zeros)
          __syncwarp();
          if (lane == 0) bar_arrive(bar + 8 * (CH_V_OK + slot));
        }
        __syncwarp();
        if (lane == 0) bar_arrive(bar + 8 * (CH_FREE + slot));
      }
    }
    ++segments;
  }
  if (!ok) *s_trouble = 1;
}

template <bool BF16, bool WINDOW>
__device__ void chunk_softmax(const PagedArgs& A, uint32_t bar, uint32_t tmem, const ChunkTile* s_info, const ChunkWork<WINDOW>* works,
                              const int* s_again, int* s_trouble, int cta, unsigned char* stage) {
  constexpr float RAISE = PagedWeights<BF16>::RAISE, LIFT = PagedWeights<BF16>::LIFT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = warp >> 2, quad = warp & 3, row = quad * 32 + lane, tm = A.group >> 1;
  const uint32_t lanes = (uint32_t)(quad * 32) << 16;
  const uint32_t t_s = tmem + 128 * h + lanes, t_o = tmem + 256 + 128 * h + lanes;
  unsigned tile = 0, segments = 0;
  uint32_t s_phase = 0;                                      // a bit per buffer: parity of its next use
  // The product of buffer b's last step.  (A barrier a buffer: the one of the step before that is done when the scores that
  // came after it are, so no phase can be mistaken for another.)
  auto product_done = [&](int b) { return bar_wait_warp(bar + 8 * (CH_O_DONE + 2 * h + b), (s_phase >> b & 1) ^ 1u, A.wait_ns); };
  bool ok = true;
  for (unsigned at = 0; chunk_work(works, at, bar, A.wait_ns, ok); ++at) {
    const PagedSegment s = works[at % CH_WORKS].s;           // (a copy: with reads from shared memory in the steps they took 3 % longer)
    const ChunkSteps<WINDOW> st = works[at % CH_WORKS].st[h];
    chunk_work_done(at, bar);
    const int tok = row / A.g, n_tok = min(tm, s.item.n_tok - h * tm);      // new tokens of this half
    const bool live = tok < n_tok && row < tm * A.g;
    const int item_row = h * tm * A.g + row;
    const int n = s.k1 - s.k0;
    const int steps = st.n;
    const int pos = live ? s.item.p0 + h * tm + tok : -1;
    // the tokens of this warp's live rows, for whether a step needs masks
    const int tok_w = (quad * 32) / A.g, tok_e = min((quad * 32 + 31) / A.g, n_tok - 1);
    const int pos_w = s.item.p0 + h * tm + tok_w, pos_e = s.item.p0 + h * tm + tok_e;
    float m = -INFINITY, l = 0.f;
    for (int u = 0, t = st.next(-1); u < steps; ++u, t = st.next(t)) {
      const int b = u & 1, half = t & 1;
      ok = bar_wait_warp(bar + 8 * (CH_S_FULL + 2 * h + b), s_phase >> b & 1, A.wait_ns);
      s_phase ^= 1u << b;
      if (!ok) break;
      tmem_fence_after();
      const ChunkTile info = s_info[(tile + (t >> 1)) % CH_INFO];
      uint32_t v[64];
      tmem_ld64(t_s + CH_STEP * b, v);
      const int key0 = info.key0 + CH_STEP * half, pages = info.there >> (4 * half) & 15;
      if (key0 + CH_STEP - 1 > pos_w || pages != 15 || (WINDOW && key0 <= pos_e - A.window && key0 + CH_STEP > A.sinks)) {
        // keys the row sees: below `over`, and, under a window, from `from` on or below the sinks (relative to the step), where the
        // page is there; a bit each
        const int over = min(pos + 1, s.item.hi) - key0, from = WINDOW ? pos - A.window + 1 - key0 : -0x3fffffff, sink = A.sinks - key0;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          auto below = [&](int x) {                          // bits of keys 32 c + i < x
            const int n = min(max(x - 32 * c, 0), 32);
            return n == 0 ? 0u : 0xFFFFFFFFu >> (32 - n);
          };
          const uint32_t there = (pages >> (2 * c) & 1 ? 0xFFFFu : 0u) | (pages >> (2 * c + 1) & 1 ? 0xFFFF0000u : 0u);
          const uint32_t seen = below(over) & (~below(from) | below(sink)) & there;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if ((seen & 1u << i) == 0) v[32 * c + i] = 0xFF800000u;
        }
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < CH_STEP; i += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(v[i + 2 * e]), __uint_as_float(v[i + 2 * e + 1]));
      const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * A.scale_log2;
      // (rows that stand for no token hold what happens to be in shared memory: they have no say, or results would not repeat)
      if (__any_sync(0xffffffffu, live && high > m + RAISE)) {
        const float to = fmaxf(m, high), f = to == -INFINITY ? 1.f : exp2_approx(m - to);   // (m = -inf: 0)
        m = to; l *= f;
        if (u > 0) {                                         // the accumulator, once the product of the step before is done
          ok = product_done(b ^ 1);
          if (!ok) break;
          tmem_fence_after();
#pragma unroll 1
          for (int c = 0; c < 128; c += 32) {
            uint32_t x[32];
            tmem_ld32(t_o + c, x);
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
            tmem_st32(t_o + c, x);
          }
        }
      }
      const float base = (m == -INFINITY ? 0.f : m) - LIFT;
      const uint64_t scale2 = two(A.scale_log2, A.scale_log2), base2 = two(-base, -base);
      uint64_t sum[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < CH_STEP; i += 2) {
        uint64_t x = fma2(two(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), scale2, base2);
        float lo, hi;
        if ((i >> 1) % CH_POLY == CH_POLY - 1) {
          x = exp2_poly2(x);
          split(x, lo, hi);
        } else {
          split(x, lo, hi);
          lo = exp2_approx(lo); hi = exp2_approx(hi);
          x = two(lo, hi);
        }
        sum[(i >> 1) & 1] = add2(sum[(i >> 1) & 1], x);
        v[i >> 1] = paged_pack<BF16>(lo, hi);
      }
      tmem_st32(t_s + CH_STEP * b, v);
      tmem_wait_st();
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) bar_arrive(bar + 8 * (CH_P_READY + 2 * h + b));
      float e0, e1, e2, e3;
      split(sum[0], e0, e1); split(sum[1], e2, e3);
      l += (e0 + e1) + (e2 + e3);
    }
    if (!ok) break;
    if (n_tok <= 0) { tile += n; segments += n > 0; continue; }             // the item has one half
    if (steps > 0) {
      ok = product_done((steps - 1) & 1);
      if (!ok) break;
      tmem_fence_after();
    }
    // (a flag for a tile behind this half's last may be up already or not: none of its rows sees a key there, so nothing is added)
    const bool repair = steps > 0 && s_again[segments & 3] == (int)segments + 1;
    // a row a thread in tensor memory, a row eight lanes on the way out: 128 bytes of every row pass through shared memory, their
    // 16-byte chunks swapped about by row (32 rows of 16 bytes each would be 32 lines an instruction)
    const bool whole = s.k0 == 0 && s.k1 == s.item.n, records = A.rec != nullptr || !whole;
    const float w = steps == 0 ? 0.f : records ? 1.f : paged_over(l);
    const int64_t at_tok = s.item.tok0 + h * tm + tok, at_head = s.head * A.g + row - tok * A.g;
    uint64_t to = 0ull;
    if (live) {
      if (records) {
        float* rec = whole ? A.rec + (at_tok * A.H_q + at_head) * RDKV_PARTIAL_STRIDE
                           : A.part + ((int64_t)(2 * cta + (s.k0 > 0 ? 0 : 1)) * CH_ROWS + item_row) * RDKV_PARTIAL_STRIDE;
        *reinterpret_cast<float4*>(rec) = make_float4((m - LIFT) * PAGED_LN2, l, 0.f, 0.f);
        to = reinterpret_cast<uint64_t>(rec + 4);
      } else {
        to = reinterpret_cast<uint64_t>(A.out + at_tok * A.o_tok + at_head * A.o_head);
      }
    }
    uint4* mine = reinterpret_cast<uint4*>(stage) + lane * 8;
#pragma unroll 1
    for (int c = 0; c < (records ? 4 : 2); ++c) {
      uint4 y[8];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (records && e == 1) break;
        uint32_t x[32];
        if (steps > 0) tmem_ld32(t_o + (records ? 32 * c : 64 * c + 32 * e), x);
        else
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = 0u;          // (no step wrote the accumulator)
        if (records) {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            auto two16 = [&](int k) { return paged_pack<BF16>(__uint_as_float(x[8 * i + k]) * w, __uint_as_float(x[8 * i + k + 1]) * w); };
            y[4 * e + i] = make_uint4(two16(0), two16(2), two16(4), two16(6));
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) mine[i ^ (lane & 7)] = y[i];
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {                        // four rows at a time
        const int r = 4 * i + (lane >> 3);
        y[i] = reinterpret_cast<const uint4*>(stage)[r * 8 + ((lane & 7) ^ (r & 7))];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint64_t at = __shfl_sync(0xffffffffu, to, 4 * i + (lane >> 3));
        if (at != 0ull) store_global(at + 128 * c + 16 * (lane & 7), y[i]);
      }
      __syncwarp();
    }
    if (repair) {
      const PagedSegment copy = s;
      const int row0 = h * tm * A.g + quad * 32, row1 = min(row0 + 32, (h * tm + n_tok) * A.g);
      paged_repair<BF16, CH_KEYS, CH_ROWS>(A, copy, row0, row1, cta);
    }
    tmem_fence_before();
    tile += n;
    segments += n > 0;
  }
  if (!ok) *s_trouble = 1;
}

template <bool BF16, bool WINDOW>
__global__ void __launch_bounds__(CH_THREADS, 1)
paged_chunk_kernel(const PagedArgs A, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v) {
  extern __shared__ __align__(1024) unsigned char ch_raw[];
  __shared__ __align__(8) uint64_t s_bar[CH_BARS];
  __shared__ ChunkTile s_info[CH_INFO];
  __shared__ PagedPlaceScratch s_place;
  __shared__ uint32_t s_tmem;
  __shared__ ChunkWork<WINDOW> s_work[CH_WORKS];
  __shared__ int s_again[4];                                 // segment (its number + 1) whose rows are repaired
  __shared__ int s_trouble;
  const int tid = threadIdx.x, warp = tid >> 5, cta = blockIdx.x;
  const uint32_t q32 = smem_addr(ch_raw), ring = q32 + 2 * CH_SLOT, bar = smem_addr(s_bar);
  if (tid == 0) {
    bar_init(bar + 8 * CH_Q_FULL, 1); bar_init(bar + 8 * CH_Q_FREE, 2);
#pragma unroll
    for (int i = 0; i < 4; ++i) { bar_init(bar + 8 * (CH_S_FULL + i), 1); bar_init(bar + 8 * (CH_P_READY + i), 4); bar_init(bar + 8 * (CH_O_DONE + i), 1); }
#pragma unroll
    for (int i = 0; i < CH_WORKS; ++i) { bar_init(bar + 8 * (CH_W_FULL + i), 1); bar_init(bar + 8 * (CH_W_FREE + i), CH_SOFTMAX_WARPS + 3); }
    bar_init(bar + 8 * CH_DRAINED, 1); bar_init(bar + 8 * (CH_DRAINED + 1), 1);
#pragma unroll
    for (int i = 0; i < CH_SLOTS; ++i) {
      bar_init(bar + 8 * (CH_FULL + i), 1); bar_init(bar + 8 * (CH_FREE + i), 3); bar_init(bar + 8 * (CH_V_OK + i), 1);
    }
    bar_init_fence();
    s_trouble = 0;
  }
  if (tid < 4) s_again[tid] = 0;
  if (tid == 32) { tma_prefetch_map(&tm_q); tma_prefetch_map(&tm_k); tma_prefetch_map(&tm_v); }
  if (warp == CH_SOFTMAX_WARPS + 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  let_next_kernel_start();
  tmem_fence_before();
  PagedPlace from, to;
  const bool ordered = paged_place<CH_KEYS, CH_THREADS, CH_FIXED, CH_SNAP, CH_WHOLE, PAGED_CHUNK_CTAS>(A, cta, s_place, from, to);
  if (!ordered && tid == 0) s_trouble = 2;                   // (the barriers in there order the set-up too)
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = s_tmem;
  unsigned char* ring_ptr = ch_raw + 2 * CH_SLOT;
  if (warp >= CH_SOFTMAX_WARPS) {
    const int role = warp - CH_SOFTMAX_WARPS;
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CH_HELPER_REGS));
    if (role == 0) chunk_load<BF16, WINDOW>(A, &tm_q, &tm_k, &tm_v, PagedWalk<CH_KEYS>(A, from, to), q32, ring, bar, s_info, s_work, &s_trouble);
    else if (role < 3) chunk_products<BF16, WINDOW>(role - 1, A.wait_ns, q32, ring, bar, tmem, s_info, s_work, &s_trouble);
    else chunk_values<BF16, WINDOW>(A, ring_ptr, bar, s_info, s_work, s_again, &s_trouble);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CH_SOFTMAX_REGS));
    chunk_softmax<BF16, WINDOW>(A, bar, tmem, s_info, s_work, s_again, &s_trouble, cta, ring_ptr + CH_SLOTS * CH_SLOT + warp * CH_STAGE);
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == CH_SOFTMAX_WARPS + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  paged_zero_padding(A, CH_THREADS, s_trouble == 2);
  paged_report(A, s_trouble);
}

// A map over query rows [T][H_q][128] (strides in elements) whose boxes are 64 channels of g heads of `tokens` tokens.
static bool chunk_q_map(CUtensorMap* tm, const PagedArgs& A, bool bf16) {
  memset(tm, 0, sizeof(*tm));
  TensorMapEncoder enc = tensor_map_encoder();
  if (enc == nullptr || (reinterpret_cast<uintptr_t>(A.q) & 15) != 0) return false;
  const int64_t head = A.H_q == 1 ? 128 : A.q_head, tok = A.T == 1 ? 128 : A.q_tok;
  if (head <= 0 || tok <= 0 || (head & 7) || (tok & 7)) return false;
  const cuuint64_t dims[3] = {PAGED_CHANNELS, (cuuint64_t)A.H_q, (cuuint64_t)A.T};
  const cuuint64_t strides[2] = {(cuuint64_t)head * 2u, (cuuint64_t)tok * 2u};
  const cuuint32_t box[3] = {64u, (cuuint32_t)A.g, (cuuint32_t)(A.group >> 1)}, elem[3] = {1u, 1u, 1u};
  return enc(tm, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<uint16_t*>(A.q), dims, strides, box,
             elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF16, bool WINDOW>
static int chunk_launch(const PagedArgs& A, const CUtensorMap& tm_q, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  constexpr auto kernel = paged_chunk_kernel<BF16, WINDOW>;
  // (the register split waits for ever if the block was launched with fewer than it hands out)
  static const int regs = [] {
    cudaFuncAttributes attr;
    return cudaFuncGetAttributes(&attr, kernel) == cudaSuccess ? attr.numRegs : 0;
  }();
  const cudaError_t e = allow_dynamic_smem_once<paged_chunk_kernel<BF16, WINDOW>>(CH_SMEM);
  if (e != cudaSuccess || regs * CH_THREADS < CH_SOFTMAX_WARPS * 32 * CH_SOFTMAX_REGS + 128 * CH_HELPER_REGS) {
    g_last_cuda_error = (int)e;
    return RDKV_ERR_LAUNCH;
  }
  kernel<<<PAGED_CHUNK_CTAS, CH_THREADS, CH_SMEM, st>>>(A, tm_q, tm_k, tm_v);
  const int rc = launch_status();
  if (rc != RDKV_OK) return rc;
  return paged_launch_join(paged_join_kernel<BF16, CH_ROWS, PAGED_CHUNK_CTAS>, A, dim3(PAGED_CHUNK_CTAS - 1, 16), st);
}

int paged_chunk_launch(const PagedArgs& A, bool bf16, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  CUtensorMap tm_q;
  if (!chunk_q_map(&tm_q, A, bf16)) return RDKV_ERR_BAD_SHAPE;
  // (the window's masks and left-out steps in a kernel of their own: in one they cost the others 3 %, 2048 behind 6000 226 -> 233 us)
  if (A.window > 0) return bf16 ? chunk_launch<true, true>(A, tm_q, tm_k, tm_v, st) : chunk_launch<false, true>(A, tm_q, tm_k, tm_v, st);
  return bf16 ? chunk_launch<true, false>(A, tm_q, tm_k, tm_v, st) : chunk_launch<false, false>(A, tm_q, tm_k, tm_v, st);
}

}  // namespace rdkv
