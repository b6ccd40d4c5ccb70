// Attention of chunks of new tokens over paged caches on the fifth-generation tensor cores.
//
// An item is two halves of up to 128 rows (floor(128/g) new tokens x g query heads of a KV head each); its keys come in
// tiles of 128.  Per half and tile: S = Q.K^T (tcgen05.mma, both operands in shared memory, fp32 scores in tensor memory),
// softmax of S by a warpgroup with one row per thread, the weights P written over S as 16-bit values, O += P.V
// (tcgen05.mma, P from tensor memory, V as it lies in the cache: MN-major).  Tensor memory is full: two score tiles and two
// accumulators of 128 columns.  While one half's scores are turned into weights, the other half's products run, so
// the tensor cores and the exponential units take turns on both halves; 2 x 128 rows share every key tile in
// shared memory.
//
// 12 warps: two warpgroups of softmax (half 0, half 1), and one of helpers: warp 8 brings in Q and the tiles (tiled TMA, one
// box per page and 64-channel panel, 128-byte swizzle, four slots of 32 KB for K and V in turn), warps 9 and 10
// issue the products of a half each, warp 11 looks after masked values: 0 x NaN is NaN, so in tiles that some row of the item does
// not see whole it sets values of keys that no row sees to zero before the product, and looks for values that are not
// finite among the others; such a segment's rows are done again one by one (paged_slow_row).
//
// An accumulator is rescaled by the threads that own its rows, and only when a score passes the row's reference by more
// than PagedWeights::RAISE.  Every wait is bounded; a wait that runs out ends the CTA's work and sets its status word.
#include "paged_attn.cuh"

namespace rdkv {

constexpr int CH_KEYS = PAGED_CHUNK_KEYS, CH_ROWS = PAGED_CHUNK_ROWS, CH_SLOTS = 4, CH_THREADS = 384;
constexpr int CH_PANEL = 128 * 128;               // bytes: 128 rows of 64 channels
constexpr int CH_SLOT = 2 * CH_PANEL;
constexpr int CH_STAGE = 32 * 128;                // bytes a softmax warp's results pass through on their way out
constexpr size_t CH_SMEM = 1024 + (size_t)(2 + CH_SLOTS) * CH_SLOT + 8 * CH_STAGE;
constexpr int CH_INFO = 8;                        // tiles whose description is kept (a softmax warp is at most three behind the loads)
constexpr int CH_POLY = 4;                         // every CH_POLY-th pair of exponentials goes to the FMA units
constexpr int CH_FIXED = 1, CH_SNAP = 3, CH_WHOLE = 8;
constexpr int CH_SOFTMAX_REGS = 208, CH_HELPER_REGS = 88;
static_assert(256 * CH_SOFTMAX_REGS + 128 * CH_HELPER_REGS <= 384 * 168, "the split draws on what the block was launched with");

// Barriers.
enum { CH_Q_FULL = 0, CH_Q_FREE = 1, CH_S_FULL = 2, CH_P_READY = 4, CH_O_DONE = 8, CH_FULL = 10, CH_FREE = CH_FULL + CH_SLOTS,
       CH_V_OK = CH_FREE + CH_SLOTS, CH_DRAINED = CH_V_OK + CH_SLOTS, CH_BARS = CH_DRAINED + 2 };

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

template <bool BF16>
__device__ void chunk_load(const PagedArgs& A, const CUtensorMap* tm_q, const CUtensorMap* tm_k, const CUtensorMap* tm_v,
                           PagedWalk<CH_KEYS> walk, uint32_t q32, uint32_t ring, uint32_t bar, ChunkTile* s_info, int* s_trouble) {
  const int lane = threadIdx.x & 31, tm = A.group >> 1;
  const int rows_log2 = min(A.page_log2, 7), rows = 1 << rows_log2, per_log2 = 7 - rows_log2, per_tile = 1 << per_log2, batch = 32 >> per_log2;
  const int box = lane >> 1, panel = lane & 1;               // this lane's box of a tile
  unsigned use = 0, tile = 0, segments = 0;                  // slots filled; tiles; segments
  PagedSegment s;
  bool ok = true;
  while (ok && walk.next(A, s)) {
    if (s.k0 == s.k1) continue;
    const int32_t* table = A.table + s.i * A.table_stride;
    auto page_of = [&](int k) {                              // lane's entry of the batch that starts with tile k
      const int kk = k + (lane >> per_log2);
      if (kk >= s.k1) return -1;
      const int key = paged_tile(s.item, kk) * CH_KEYS + ((lane & (per_tile - 1)) << rows_log2);
      return key < s.item.hi ? table[key >> A.page_log2] : -1;
    };
    int ids = page_of(s.k0), ids_next = -1;
    const int halves = s.item.n_tok > tm ? 2 : 1;
    if (segments > 0 && !bar_wait_warp(bar + 8 * CH_Q_FREE, (segments - 1) & 1)) { ok = false; break; }
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
        if (use >= CH_SLOTS && !bar_wait_warp(bar + 8 * (CH_FREE + slot), (use / CH_SLOTS - 1) & 1)) { ok = false; break; }
        if (lane == 0) {
          if (bytes > 0) bar_arrive_tx(bar + 8 * (CH_FULL + slot), bytes);
          else bar_arrive(bar + 8 * (CH_FULL + slot));
        }
        __syncwarp();
        if (there)
          tma_load_4d(ring + slot * CH_SLOT + panel * CH_PANEL + box * rows * 128, t == 0 ? tm_k : tm_v, 64 * panel, key0 & (A.page - 1),
                      s.head, id, bar + 8 * (CH_FULL + slot));
      }
    }
  }
  if (!ok) {                                                 // wait (again bounded) for the copies in flight
    *s_trouble = 1;
    for (unsigned n = use < CH_SLOTS ? 0 : use - CH_SLOTS; n < use; ++n) bar_wait(bar + 8 * (CH_FULL + n % CH_SLOTS), (n / CH_SLOTS) & 1);
    if (segments > 0) bar_wait(bar + 8 * CH_Q_FULL, (segments - 1) & 1);
  }
}

__device__ __forceinline__ int chunk_uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Warps 9 and 10: the products of half 0, of half 1.  What a half's next scores wait for is short: its weights, the rest of the product
// with the values, the product with the keys; everything else is waited for before the weights are.
template <bool BF16>
__device__ void chunk_products(const PagedArgs& A, PagedWalk<CH_KEYS> walk, int h, uint32_t q32, uint32_t ring, uint32_t bar, uint32_t tmem_,
                               const ChunkTile* s_info, int* s_trouble) {
  constexpr uint32_t QK = mma_idesc<BF16>(128, false), PV = mma_idesc<BF16>(128, true);
  const int tm = A.group >> 1;
  const uint32_t t_s = (uint32_t)chunk_uniform((int)tmem_ + 128 * h), t_o = t_s + 256, one = elect_one();
  const uint64_t q = desc_k_major((uint32_t)chunk_uniform((int)(q32 + h * CH_SLOT)));
  int slot = 0, tile = 0;                                    // the next K's slot; tiles
  uint32_t phases = 0, segments = 0, v_ok = 0, p_phase = 0;  // a bit per slot: parity of its next use
  PagedSegment s;
  bool ok = true;
  auto wait = [&](int b, uint32_t parity) { ok = ok && bar_wait_warp(bar + 8 * b, parity); };
  auto wait_slot = [&](int x) { wait(CH_FULL + x, phases >> x & 1); phases ^= 1u << x; };
  auto after = [&](int x, int n) { x += n; return x >= CH_SLOTS ? x - CH_SLOTS : x; };
  auto scores = [&](int k_slot) {                            // S = Q . K^T
    const uint64_t k = desc_k_major(ring + k_slot * CH_SLOT);
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {                         // 16 channels: 32 bytes along the swizzled row, the second panel after four
      const uint64_t off = ((uint64_t)(kk >> 2) * CH_PANEL + (uint64_t)(kk & 3) * 32u) >> 4;
      mma_ss(one, t_s, q + off, k + off, QK, kk > 0 ? 1u : 0u);
    }
    mma_commit(one, bar + 8 * (CH_S_FULL + h));
  };
  while (ok && chunk_uniform(walk.next(A, s))) {
    const int n = chunk_uniform(s.k1 - s.k0);
    if (n == 0) continue;
    const bool mine = h == 0 || chunk_uniform(s.item.n_tok > tm);
    wait(CH_Q_FULL, segments++ & 1);
    wait_slot(slot);
    if (!ok) break;
    tmem_fence_after();
    if (mine) scores(slot);
    mma_commit(one, bar + 8 * (CH_FREE + slot));             // (nothing to wait for: arrives at once)
    if (n == 1) mma_commit(one, bar + 8 * CH_Q_FREE);
    for (int j = 0; j < n; ++j, ++tile) {                    // `slot`: K of tile j, then its V, then K of tile j + 1
      const int v_slot = after(slot, 1), k_slot = after(slot, 2);
      const bool more = j + 1 < n;
      wait_slot(v_slot);
      if (ok && chunk_uniform(s_info[tile % CH_INFO].edge) != 0) {
        wait(CH_V_OK + v_slot, v_ok >> v_slot & 1);
        v_ok ^= 1u << v_slot;
      }
      if (more) wait_slot(k_slot);
      if (!ok) break;
      if (mine) {
        const uint64_t v = desc_mn_major(ring + v_slot * CH_SLOT, CH_PANEL);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          wait(CH_P_READY + 2 * h + part, p_phase);
          if (!ok) break;
          tmem_fence_after();
#pragma unroll
          for (int kk = 4 * part; kk < 4 * part + 4; ++kk)   // 16 keys: 8 columns of P, two groups of eight rows of V
            mma_ts(one, t_o, t_s + 8 * kk, v + kk * (2048 >> 4), PV, j > 0 || kk > 0 ? 1u : 0u);
        }
        p_phase ^= 1u;
        if (!ok) break;
        mma_commit(one, bar + 8 * (CH_O_DONE + h));
        if (more) scores(k_slot);
      }
      mma_commit(one, bar + 8 * (CH_FREE + v_slot));
      if (more) mma_commit(one, bar + 8 * (CH_FREE + k_slot));
      if (j + 2 == n) mma_commit(one, bar + 8 * CH_Q_FREE);
      slot = k_slot;
    }
  }
  if (!ok) {                                                 // wait (again bounded) for the products in flight
    *s_trouble = 1;
    mma_commit(one, bar + 8 * (CH_DRAINED + h));
    bar_wait_warp(bar + 8 * (CH_DRAINED + h), 0);
  }
}

// Warp 11: values in masked places.
template <bool BF16>
__device__ void chunk_values(const PagedArgs& A, PagedWalk<CH_KEYS> walk, unsigned char* ring_ptr, uint32_t bar, const ChunkTile* s_info,
                             int* s_again, int* s_trouble) {
  const int lane = threadIdx.x & 31;
  unsigned use = 0, tile = 0, segments = 0;
  PagedSegment s;
  bool ok = true;
  while (ok && walk.next(A, s)) {
    if (s.k0 == s.k1) continue;
    const int p_first = s.item.p0, p_last = s.item.p0 + s.item.n_tok - 1;
    for (int j = s.k0; ok && j < s.k1; ++j, ++tile) {
      for (int t = 0; t < 2; ++t, ++use) {
        const int slot = use % CH_SLOTS;
        if (!bar_wait_warp(bar + 8 * (CH_FULL + slot), (use / CH_SLOTS) & 1)) { ok = false; break; }
        const ChunkTile info = s_info[tile % CH_INFO];
        if (t == 1 && info.edge) {
          // 16 keys at a time that not every row sees: eight lanes a key, a 16-byte chunk of each panel a lane.  x * 0 added up
          // is not a number as soon as one x is not finite.
          uint32_t sum[4] = {0u, 0u, 0u, 0u};
          for (int g = 0; g < 8; ++g) {
            const int key0 = info.key0 + 16 * g;
            const bool gone = (info.there >> g & 1) == 0 || key0 >= s.item.hi;
            if (!gone && key0 + 15 <= p_first && (A.window == 0 || key0 > p_last - A.window || key0 + 15 < A.sinks)) continue;
            uint4* at = reinterpret_cast<uint4*>(ring_ptr + slot * CH_SLOT + (16 * g + (lane >> 3)) * 128 + (lane & 7) * 16);
            const int mine = key0 + (lane >> 3), low = A.window > 0 ? p_first - A.window : -1;   // (keys up to `low`, behind the sinks: no row's)
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
          if (again) s_again[segments & 3] = (int)segments + 1;
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

template <bool BF16>
__device__ void chunk_softmax(const PagedArgs& A, PagedWalk<CH_KEYS> walk, uint32_t bar, uint32_t tmem, const ChunkTile* s_info,
                              const int* s_again, int* s_trouble, int cta, unsigned char* stage) {
  constexpr float RAISE = PagedWeights<BF16>::RAISE, LIFT = PagedWeights<BF16>::LIFT;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = warp >> 2, row = (warp & 3) * 32 + lane, tm = A.group >> 1;
  const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
  const uint32_t t_s = tmem + 128 * h + lanes, t_o = tmem + 256 + 128 * h + lanes;
  unsigned done = 0, tile = 0, segments = 0;                 // tiles of this half; tiles; segments
  PagedSegment s;
  bool ok = true;
  while (ok && walk.next(A, s)) {
    const int tok = row / A.g, n_tok = min(tm, s.item.n_tok - h * tm);      // new tokens of this half
    const bool live = tok < n_tok && row < tm * A.g;
    const int item_row = h * tm * A.g + row;
    if (s.k0 == s.k1) {                                      // an item without keys
      if (live) {
        const PagedRow d = paged_row<CH_ROWS>(A, s, item_row, cta);
        for (int c = 0; c < 32; ++c) {
          if (d.rec != nullptr) *reinterpret_cast<float4*>(d.rec + 4 + 4 * c) = make_float4(0.f, 0.f, 0.f, 0.f);
          else *reinterpret_cast<uint2*>(d.out + 4 * c) = make_uint2(0u, 0u);
        }
        if (d.rec != nullptr) *reinterpret_cast<float4*>(d.rec) = make_float4(-INFINITY, 0.f, 0.f, 0.f);
      }
      continue;
    }
    const int n = s.k1 - s.k0;
    if (n_tok <= 0) { tile += n; ++segments; continue; }     // the item has one half
    const int pos = live ? s.item.p0 + h * tm + tok : -1;
    // the tokens of this warp's live rows, for whether a tile needs masks
    const int tok_w = ((warp & 3) * 32) / A.g, tok_e = min(((warp & 3) * 32 + 31) / A.g, n_tok - 1);
    const int pos_w = s.item.p0 + h * tm + tok_w, pos_e = s.item.p0 + h * tm + tok_e;
    float m = -INFINITY, l = 0.f;
    for (int j = 0; j < n; ++j, ++tile, ++done) {
      ok = bar_wait_warp(bar + 8 * (CH_S_FULL + h), done & 1);
      if (!ok) break;
      tmem_fence_after();
      const ChunkTile info = s_info[tile % CH_INFO];
      uint32_t v[128];
      tmem_ld128(t_s, v);
      if (info.key0 + CH_KEYS - 1 > pos_w || info.there != 0xFF || (A.window > 0 && info.key0 <= pos_e - A.window && info.key0 + CH_KEYS > A.sinks)) {
        // keys the row sees: below `over`, and, under a window, from `from` on or below the sinks (relative to the tile), where the
        // page is there; a bit each
        const int over = min(pos + 1, s.item.hi) - info.key0, from = A.window > 0 ? pos - A.window + 1 - info.key0 : -0x3fffffff;
        const int sink = A.sinks - info.key0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          auto below = [&](int x) {                          // bits of keys 32 c + i < x
            const int n = min(max(x - 32 * c, 0), 32);
            return n == 0 ? 0u : 0xFFFFFFFFu >> (32 - n);
          };
          const uint32_t there = (info.there >> (2 * c) & 1 ? 0xFFFFu : 0u) | (info.there >> (2 * c + 1) & 1 ? 0xFFFF0000u : 0u);
          const uint32_t seen = below(over) & (~below(from) | below(sink)) & there;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if ((seen & 1u << i) == 0) v[32 * c + i] = 0xFF800000u;
        }
      }
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 128; i += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[e] = max3(top[e], __uint_as_float(v[i + 2 * e]), __uint_as_float(v[i + 2 * e + 1]));
      const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * A.scale_log2;
      if (__any_sync(0xffffffffu, high > m + RAISE)) {
        const float to = fmaxf(m, high), f = to == -INFINITY ? 1.f : exp2_approx(m - to);   // (m = -inf: 0)
        m = to; l *= f;
        if (j > 0) {                                         // the accumulator, once the product before is done
          ok = bar_wait_warp(bar + 8 * (CH_O_DONE + h), (done - 1) & 1);
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
      auto weights = [&](int first, int end) {
#pragma unroll
        for (int i = first; i < end; i += 2) {
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
      };
      auto ready = [&](int part) {
        tmem_wait_st();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) bar_arrive(bar + 8 * (CH_P_READY + 2 * h + part));
      };
      weights(0, 64);                                        // 64 keys: their product starts while the rest is worked out
      tmem_st32(t_s, v);
      weights(64, 80);
      ready(0);
      weights(80, 128);
      tmem_st32(t_s + 32, v + 32);
      ready(1);
      float a, b, c, d;
      split(sum[0], a, b); split(sum[1], c, d);
      l += (a + b) + (c + d);
    }
    if (!ok) break;
    ok = bar_wait_warp(bar + 8 * (CH_O_DONE + h), (done - 1) & 1);
    if (!ok) break;
    tmem_fence_after();
    if (s_again[segments & 3] == (int)segments + 1) {
      const PagedSegment copy = s;
      for (int r = 0; r < 32; ++r)
        if (__shfl_sync(0xffffffffu, live ? 1 : 0, r) != 0) paged_slow_row<BF16, CH_KEYS, CH_ROWS>(A, copy, item_row - lane + r, cta);
    } else {
      // a row a thread in tensor memory, a row eight lanes on the way out: 128 bytes of every row pass through shared memory, their
      // 16-byte chunks swapped about by row (32 rows of 16 bytes each would be 32 lines an instruction)
      PagedRow d = {nullptr, nullptr};
      if (live) d = paged_row<CH_ROWS>(A, s, item_row, cta);
      const bool records = A.rec != nullptr || s.k0 != 0 || s.k1 != s.item.n;
      const float w = records ? 1.f : paged_over(l);
      if (d.rec != nullptr) *reinterpret_cast<float4*>(d.rec) = make_float4((m - LIFT) * PAGED_LN2, l, 0.f, 0.f);
      const uint64_t to = !live ? 0ull : records ? reinterpret_cast<uint64_t>(d.rec + 4) : reinterpret_cast<uint64_t>(d.out);
      uint4* mine = reinterpret_cast<uint4*>(stage) + lane * 8;
#pragma unroll 1
      for (int c = 0; c < (records ? 4 : 2); ++c) {
        uint4 y[8];
        if (records) {
          uint32_t x[32];
          tmem_ld32(t_o + 32 * c, x);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        } else {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t x[32];
            tmem_ld32(t_o + 64 * c + 32 * e, x);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              auto pair = [&](int k) { return paged_pack<BF16>(__uint_as_float(x[8 * i + k]) * w, __uint_as_float(x[8 * i + k + 1]) * w); };
              y[4 * e + i] = make_uint4(pair(0), pair(2), pair(4), pair(6));
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[i ^ (lane & 7)] = y[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i) {                        // four rows at a time
          const int r = 4 * i + (lane >> 3);
          const uint64_t at = __shfl_sync(0xffffffffu, to, r);
          const uint4 x = reinterpret_cast<const uint4*>(stage)[r * 8 + ((lane & 7) ^ (r & 7))];
          if (at != 0ull) *reinterpret_cast<uint4*>(at + 128 * c + 16 * (lane & 7)) = x;
        }
        __syncwarp();
      }
    }
    tmem_fence_before();
    ++segments;
  }
  if (!ok) *s_trouble = 1;
}

template <bool BF16>
__global__ void __launch_bounds__(CH_THREADS, 1)
paged_chunk_kernel(const PagedArgs A, const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v) {
  extern __shared__ unsigned char ch_raw[];
  __shared__ __align__(8) uint64_t s_bar[CH_BARS];
  __shared__ ChunkTile s_info[CH_INFO];
  __shared__ PagedPlaceScratch s_place;
  __shared__ uint32_t s_tmem;
  __shared__ int s_again[4];                                 // segment (its number + 1) whose rows are done again
  __shared__ int s_trouble;
  const int tid = threadIdx.x, warp = tid >> 5, cta = blockIdx.x;
  const uint32_t q32 = (smem_addr(ch_raw) + 1023u) & ~1023u, ring = q32 + 2 * CH_SLOT, bar = smem_addr(s_bar);
  if (tid == 0) {
    bar_init(bar + 8 * CH_Q_FULL, 1); bar_init(bar + 8 * CH_Q_FREE, 2);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bar_init(bar + 8 * (CH_S_FULL + h), 1); bar_init(bar + 8 * (CH_P_READY + 2 * h), 4); bar_init(bar + 8 * (CH_P_READY + 2 * h + 1), 4); bar_init(bar + 8 * (CH_O_DONE + h), 1); bar_init(bar + 8 * (CH_DRAINED + h), 1);
    }
#pragma unroll
    for (int i = 0; i < CH_SLOTS; ++i) {
      bar_init(bar + 8 * (CH_FULL + i), 1); bar_init(bar + 8 * (CH_FREE + i), 3); bar_init(bar + 8 * (CH_V_OK + i), 1);
    }
    bar_init_fence();
    s_trouble = 0;
  }
  if (tid < 4) s_again[tid] = 0;
  if (tid == 32) { tma_prefetch_map(&tm_q); tma_prefetch_map(&tm_k); tma_prefetch_map(&tm_v); }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  let_next_kernel_start();
  tmem_fence_before();
  PagedPlace from, to;
  paged_place<CH_KEYS, CH_THREADS, CH_FIXED, CH_SNAP, CH_WHOLE>(A, cta, PAGED_CHUNK_CTAS, s_place, from, to);   // (its barriers order the set-up too)
  __syncthreads();
  tmem_fence_after();
  const uint32_t tmem = s_tmem;
  const PagedWalk<CH_KEYS> walk(A, from, to);
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(CH_HELPER_REGS));
    if (warp == 8) chunk_load<BF16>(A, &tm_q, &tm_k, &tm_v, walk, q32, ring, bar, s_info, &s_trouble);
    else if (warp < 11) chunk_products<BF16>(A, walk, warp - 9, q32, ring, bar, tmem, s_info, &s_trouble);
    else chunk_values<BF16>(A, walk, ch_raw + (ring - smem_addr(ch_raw)), bar, s_info, s_again, &s_trouble);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(CH_SOFTMAX_REGS));
    chunk_softmax<BF16>(A, walk, bar, tmem, s_info, s_again, &s_trouble, cta,
                        ch_raw + (ring - smem_addr(ch_raw)) + CH_SLOTS * CH_SLOT + warp * CH_STAGE);
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  paged_zero_padding(A, CH_THREADS);
  if (tid == 0) A.status[cta] = s_trouble;
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

int paged_chunk_launch(const PagedArgs& A, bool bf16, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  CUtensorMap tm_q;
  if (!chunk_q_map(&tm_q, A, bf16)) return RDKV_ERR_BAD_SHAPE;
  auto go = [&](auto kernel, auto join) -> int {
    cudaError_t e = allow_dynamic_smem(kernel, CH_SMEM);
    cudaFuncAttributes attr;
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&attr, kernel);
    if (e != cudaSuccess) { g_last_cuda_error = (int)e; return RDKV_ERR_LAUNCH; }
    // (the register split waits for ever if the block was launched with fewer than it hands out)
    if (attr.numRegs * CH_THREADS < 256 * CH_SOFTMAX_REGS + 128 * CH_HELPER_REGS) return RDKV_ERR_LAUNCH;
    kernel<<<PAGED_CHUNK_CTAS, CH_THREADS, CH_SMEM, st>>>(A, tm_q, tm_k, tm_v);
    const int rc = launch_status();
    if (rc != RDKV_OK) return rc;
    return paged_launch_join(join, A, dim3(PAGED_CHUNK_CTAS - 1, 16), st);
  };
  if (bf16) return go(paged_chunk_kernel<true>, paged_join_kernel<true, CH_ROWS, PAGED_CHUNK_CTAS>);
  return go(paged_chunk_kernel<false>, paged_join_kernel<false, CH_ROWS, PAGED_CHUNK_CTAS>);
}

}  // namespace rdkv
