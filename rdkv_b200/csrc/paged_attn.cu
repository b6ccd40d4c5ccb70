// Entry point of the attention over paged caches, and its kernel for few rows a KV head (single tokens).
//
// paged_decode_kernel: an item is up to 16 rows (new tokens x query heads of a KV head), which is the M of mma.sync
// m16n8k16; its keys and values are read once and are all the kernel moves, so it is bound by memory.  A CTA has four
// computing warps and one that brings in tiles of 64 keys: one tiled TMA box per page (or per 64 rows of a larger one),
// 64-channel panel and tensor, laid down with the 128-byte swizzle that ldmatrix reads without bank conflicts, three
// tiles deep, two CTAs an SM.  Page numbers are fetched 32 boxes ahead.  Each computing warp takes 16 keys of a
// tile on its own: scores (queries as A operand, keys as B), running maximum and sum, then the weights, which are
// already in A operand form, times the values (ldmatrix.trans).  The four partial results meet in the slot of the
// segment's last tile.  Why not tcgen05: its smallest M is 64 rows, of which 4 to 16 would be used, and scores would
// have to go through tensor memory between the products; the tensor pipe is 80 % idle as it is.
// 64 requests of up to 8192 tokens, 8 x 4 heads, pages of 16: 181 us, 6.2 TB/s of keys and values (96 % of a copy's rate).
//
// Few items (CLUSTER): each is cut evenly over a cluster of 8, 12 or 16 CTAs, which exchange their records through distributed
// shared memory; there is no line of units to find a place in and no second launch.
//
// Masks are applied only to 16-key blocks that reach past some row's limits.  There, values of keys that no row of
// the item sees are set to zero (0 x NaN), and so is a value that is not finite at a key that only some rows see; the rows
// that see it get it added in the end (paged_repair).
#include "paged_attn.cuh"

namespace rdkv {

constexpr int DEC_KEYS = PAGED_DECODE_KEYS, DEC_ROWS = PAGED_DECODE_ROWS, DEC_STAGES = 3;
constexpr int DEC_WARPS = 4, DEC_THREADS = DEC_WARPS * 32 + 32;
constexpr int DEC_PANEL = DEC_KEYS * 128;         // bytes of 64 keys' 64 channels
constexpr int DEC_STAGE = 4 * DEC_PANEL;          // K channels 0-63, 64-127, V channels 0-63, 64-127
constexpr size_t DEC_SMEM = 1024 + (size_t)DEC_STAGES * DEC_STAGE;
static_assert(DEC_STAGE == DEC_WARPS * DEC_ROWS * 128 * 4, "the warps' results fill a stage");
constexpr int DEC_FIXED = 2, DEC_SNAP = 1, DEC_WHOLE = 4;

template <bool BF16>
__device__ __forceinline__ void dec_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void dec_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void dec_ldmatrix_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void dec_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }   // the computing warps
__device__ __forceinline__ bool dec_barrier_any(bool x) {                                            // and whether one of their threads has x
  uint32_t any;
  asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(any) : "r"((uint32_t)x) : "memory");
  return any != 0;
}
__device__ __forceinline__ uint32_t dec_cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t dec_cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void dec_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t dec_map(uint32_t addr, uint32_t rank) {   // this shared-memory address in CTA `rank` of the cluster
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 dec_remote4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// The segments of a CTA: of the line of units, or, in a cluster, an even part of every group of the cluster's (request, head).
template <bool CLUSTER> struct DecWalk;
template <> struct DecWalk<false> : PagedWalk<DEC_KEYS> { using PagedWalk<DEC_KEYS>::PagedWalk; };
template <> struct DecWalk<true> {
  PagedRequest r;
  int i, head, group, groups, rank, size;
  __device__ __forceinline__ explicit DecWalk(const PagedArgs& A) : group(0), rank((int)dec_cluster_rank()), size((int)dec_cluster_size()) {
    const int item = blockIdx.x / size;
    i = item / A.H_kv; head = item - i * A.H_kv;
    r = paged_request(A, i);
    groups = paged_groups(A, r);
  }
  __device__ __forceinline__ bool next(const PagedArgs& A, PagedSegment& s) {
    if (group >= groups) return false;
    s.request = r; s.i = i; s.head = head; s.group = group;
    s.item = paged_item<DEC_KEYS>(A, r, group++);
    s.k0 = (int)((int64_t)s.item.n * rank / size); s.k1 = (int)((int64_t)s.item.n * (rank + 1) / size);
    return true;
  }
};

template <bool BF16, bool CLUSTER>
__global__ void __launch_bounds__(DEC_THREADS, 2)
paged_decode_kernel(const PagedArgs A, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  extern __shared__ unsigned char dec_raw[];
  __shared__ __align__(8) uint64_t s_bar[2 * DEC_STAGES];   // [slot] tile arrived, [DEC_STAGES + slot] slot free
  __shared__ int2 s_info[DEC_STAGES];                       // first key of the tile, a bit per 16 keys whose page is there
  __shared__ float2 s_ml[DEC_WARPS][DEC_ROWS];
  __shared__ int s_again[2];                                // segment (its number + 1) whose rows are repaired
  __shared__ int s_trouble;
  __shared__ PagedPlaceScratch s_place;
  __shared__ __align__(16) float s_rec[CLUSTER ? DEC_ROWS : 1][RDKV_PARTIAL_STRIDE];   // this CTA's records (m in base 2)
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  const uint32_t ring = (smem_addr(dec_raw) + 1023u) & ~1023u, bar = smem_addr(s_bar);
  unsigned char* ring_ptr = dec_raw + (ring - smem_addr(dec_raw));
  if (tid == 0) {
#pragma unroll
    for (int i = 0; i < DEC_STAGES; ++i) { bar_init(bar + 8 * i, 1); bar_init(bar + 8 * (DEC_STAGES + i), DEC_WARPS); }
    bar_init_fence();
    s_again[0] = s_again[1] = s_trouble = 0;
  }
  if (tid == 32) { tma_prefetch_map(&tm_k); tma_prefetch_map(&tm_v); }
  auto begin = [&]() {
    if constexpr (CLUSTER) {
      DecWalk<true> walk(A);
      if (__syncthreads_or(paged_falls(A, tid))) {           // (no more requests than clusters: fewer than threads)
        walk.groups = 0;
        if (tid == 0) s_trouble = 2;
      }
      return walk;
    } else {
      let_next_kernel_start();
      PagedPlace from, to;
      const bool ordered = paged_place<DEC_KEYS, DEC_THREADS, DEC_FIXED, DEC_SNAP, DEC_WHOLE, PAGED_DECODE_CTAS>(A, cta, s_place, from, to);
      if (!ordered && tid == 0) s_trouble = 2;               // (the barriers in there order the set-up too)
      return DecWalk<false>(A, from, to);
    }
  };
  auto walk = begin();
  PagedSegment s;

  if (warp == DEC_WARPS) {
    // ── the warp that brings in tiles ──
    // rows of a box, boxes of a tile, tiles of a batch of page numbers: powers of two
    const int rows_log2 = min(A.page_log2, 6), rows = 1 << rows_log2, per_log2 = 6 - rows_log2, per_tile = 1 << per_log2, batch = 32 >> per_log2;
    const int box = lane >> 2, what = lane & 3;              // this lane's box of a tile: sub-tile, (K | V) x panel
    unsigned count = 0;
    bool ok = true;
    while ((ok || CLUSTER) && walk.next(A, s)) {             // (a cluster's barriers want every CTA, whatever happened)
      if (CLUSTER && !ok) s.k1 = s.k0;
      const int32_t* table = A.table + s.i * A.table_stride;
      auto page_of = [&](int k) {                            // lane's entry of the batch that starts with tile k
        const int kk = k + (lane >> per_log2);
        if (kk >= s.k1) return -1;
        const int key = paged_tile(s.item, kk) * DEC_KEYS + ((lane & (per_tile - 1)) << rows_log2);
        return key < s.item.hi ? table[key >> A.page_log2] : -1;
      };
      int ids = page_of(s.k0), ids_next = -1;
      for (int k = s.k0; k < s.k1; ++k, ++count) {
        const int in_batch = (k - s.k0) & (batch - 1);
        if (in_batch == 0) {
          if (k > s.k0) ids = ids_next;
          ids_next = page_of(k + batch);
        }
        const int slot = count % DEC_STAGES;
        if (count >= DEC_STAGES && !bar_wait_warp(bar + 8 * (DEC_STAGES + slot), (count / DEC_STAGES - 1) & 1, A.wait_ns)) { ok = false; break; }
        const int key0 = paged_tile(s.item, k) * DEC_KEYS;
        const int id = __shfl_sync(0xffffffffu, ids, in_batch * per_tile + (box < per_tile ? box : 0));
        const bool there = box < per_tile && id >= 0 && id < A.n_pages;
        const unsigned lanes = __ballot_sync(0xffffffffu, there);
        if (lane == 0) {
          int mask = 0;
          for (int x = 0; x < 4; ++x) mask |= (int)(lanes >> (4 * (x * 16 >> rows_log2)) & 1u) << x;
          s_info[slot] = make_int2(key0, mask);
          const uint32_t bytes = (uint32_t)__popc(lanes) * (uint32_t)rows * 128u;
          if (bytes > 0) bar_arrive_tx(bar + 8 * slot, bytes);
          else bar_arrive(bar + 8 * slot);
        }
        __syncwarp();
        if (there)
          tma_load_4d(ring + slot * DEC_STAGE + what * DEC_PANEL + box * rows * 128, what < 2 ? &tm_k : &tm_v, (what & 1) * 64,
                      key0 & (A.page - 1), s.head, id, bar + 8 * slot);
      }
      if (CLUSTER) { __syncwarp(); dec_cluster_sync(); dec_cluster_sync(); }
    }
    if (!ok) s_trouble = 1;
    // copies that are still on their way when nobody waits for them any more must not land in the shared memory of the next CTA
    for (unsigned n = count < DEC_STAGES ? 0 : count - DEC_STAGES; n < count; ++n) bar_wait(bar + 8 * (n % DEC_STAGES), (n / DEC_STAGES) & 1, WAIT_NS);
  } else {
    // ── the computing warps ──
    constexpr float RAISE = PagedWeights<BF16>::RAISE, LIFT = PagedWeights<BF16>::LIFT;
    const int r0 = lane >> 2, c2 = (lane & 3) * 2;           // this thread's rows r0, r0 + 8; its pair of columns
    unsigned count = 0, segment = 0;
    bool ok = true;
    while ((ok || CLUSTER) && walk.next(A, s)) {
      const int rows = s.item.n_tok * A.g, p_first = s.item.p0, p_last = s.item.p0 + s.item.n_tok - 1;
      const bool none_mine = s.k0 == s.k1;
      if (CLUSTER && !ok) s.k1 = s.k0;
      if (!CLUSTER && none_mine) {                           // an item without keys
        for (int x = tid; x < rows * 32; x += DEC_WARPS * 32) {
          const PagedRow d = paged_row<DEC_ROWS>(A, s, x >> 5, cta);
          if (d.rec != nullptr) {
            *reinterpret_cast<float4*>(d.rec + 4 + 4 * (x & 31)) = make_float4(0.f, 0.f, 0.f, 0.f);
            if ((x & 31) == 0) *reinterpret_cast<float4*>(d.rec) = make_float4(-INFINITY, 0.f, 0.f, 0.f);
          } else {
            *reinterpret_cast<uint2*>(d.out + 4 * (x & 31)) = make_uint2(0u, 0u);
          }
        }
        continue;
      }
      // the query rows as A operand: channels 16 kk + c2, + 8 of rows r0, r0 + 8
      uint32_t qa[8][4];
      int pos[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = r0 + 8 * e, tok = row / A.g;
        pos[e] = row < rows ? s.item.p0 + tok : -1;
        const uint16_t* src = A.q + (int64_t)(s.item.tok0 + tok) * A.q_tok + (int64_t)(s.head * A.g + row - tok * A.g) * A.q_head + c2;
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          qa[kk][e] = row < rows ? *reinterpret_cast<const uint32_t*>(src + 16 * kk) : 0u;
          qa[kk][2 + e] = row < rows ? *reinterpret_cast<const uint32_t*>(src + 16 * kk + 8) : 0u;
        }
      }
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      float o[16][4];
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      for (int k = s.k0; k < s.k1; ++k, ++count) {
        const int slot = count % DEC_STAGES;
        ok = bar_wait_warp(bar + 8 * slot, (count / DEC_STAGES) & 1, A.wait_ns);
        if (!ok) break;
        const int2 info = s_info[slot];
        const int key0 = info.x + warp * 16;
        if ((info.y >> warp & 1) != 0 && key0 < s.item.hi) {
          const bool edge = key0 + 15 > p_first || key0 + 16 > s.item.hi ||
                            (A.window > 0 && key0 <= p_last - A.window && key0 + 15 >= A.sinks);
          if (edge && s.item.n_tok > 1) {
            // values of keys that some rows see and others do not: two lanes a key, a panel each
            const int at_key = lane >> 1, key = key0 + at_key;
            const bool low = A.window > 0 && key >= A.sinks;
            if (key < s.item.hi && !(low && key <= p_first - A.window) && (key > p_first || (low && key <= p_last - A.window))) {
              uint4* at = reinterpret_cast<uint4*>(ring_ptr + slot * DEC_STAGE + (2 + (lane & 1)) * DEC_PANEL + (warp * 16 + at_key) * 128);
#pragma unroll 1
              for (int i = 0; i < 8; ++i) {                  // (in an order that keeps the keys' banks apart)
                const uint4 x = at[i ^ (at_key & 7)];
                const uint4 y = {paged_finite<BF16>(x.x), paged_finite<BF16>(x.y), paged_finite<BF16>(x.z), paged_finite<BF16>(x.w)};
                if (x.x != y.x || x.y != y.y || x.z != y.z || x.w != y.w) { at[i ^ (at_key & 7)] = y; s_again[segment & 1] = (int)segment + 1; }
              }
            }
            fence_async_smem();                              // (the slot's next writer is a TMA copy)
            __syncwarp();
          }
          const uint32_t kb = ring + slot * DEC_STAGE, vb = kb + 2 * DEC_PANEL;
          // scores of 16 keys: two tiles of 8
          float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
          {
            // matrices of an ldmatrix: keys 0-7 / 8-15 (lane bit 4), channels 0-7 / 8-15 of the step (lane bit 3)
            const int row = warp * 16 + (lane & 7) + ((lane >> 4) << 3), half = lane >> 3 & 1;
#pragma unroll
            for (int kk = 0; kk < 8; ++kk) {
              uint32_t b[4];
              const int c16 = 2 * kk + half;
              dec_ldmatrix(b, kb + (c16 >> 3) * DEC_PANEL + row * 128 + (((c16 & 7) ^ (row & 7)) << 4));
              dec_mma<BF16>(sc[0], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], b[0], b[1]);
              dec_mma<BF16>(sc[1], qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3], b[2], b[3]);
            }
          }
          uint32_t live0 = 0xFFFFFFFFu, live1 = 0xFFFFFFFFu;   // this thread's keys of the V operand
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[n][e] *= A.scale_log2;
          if (edge) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              uint32_t live = 0xFFFFFFFFu;
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int key = key0 + 8 * n + c2 + e;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  const bool hidden = key > pos[r] || key >= s.item.hi || (A.window > 0 && key <= pos[r] - A.window && key >= A.sinks);
                  if (hidden) sc[n][2 * r + e] = -INFINITY;
                }
                const bool low = A.window > 0 && key >= A.sinks;
                const bool none = key >= s.item.hi || (low && key <= p_first - A.window);       // no row sees the key
                if (none) live &= e == 0 ? 0xFFFF0000u : 0x0000FFFFu;
              }
              if (n == 0) live0 = live; else live1 = live;
            }
          }
          float top[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float x = fmaxf(fmaxf(sc[0][2 * r], sc[0][2 * r + 1]), fmaxf(sc[1][2 * r], sc[1][2 * r + 1]));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            top[r] = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
          }
          if (__any_sync(0xffffffffu, top[0] > m[0] + RAISE || top[1] > m[1] + RAISE)) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float n = fmaxf(m[r], top[r]), f = n == -INFINITY ? 1.f : exp2_approx(m[r] - n);   // (m = -inf: 0)
              m[r] = n; l[r] *= f;
#pragma unroll
              for (int i = 0; i < 16; ++i) { o[i][2 * r] *= f; o[i][2 * r + 1] *= f; }
            }
          }
          uint32_t pa[4];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float base = (m[r] == -INFINITY ? 0.f : m[r]) - LIFT;
            float p[4];
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e) p[2 * n + e] = exp2_approx(sc[n][2 * r + e] - base);
            l[r] += (p[0] + p[1]) + (p[2] + p[3]);
            pa[r] = paged_pack<BF16>(p[0], p[1]); pa[2 + r] = paged_pack<BF16>(p[2], p[3]);
          }
          // values: matrices of an ldmatrix: keys 0-7 / 8-15 (lane bit 3), channels 0-7 / 8-15 of the step (lane bit 4)
          const int row = warp * 16 + (lane & 15), half = lane >> 4;
#pragma unroll
          for (int cc = 0; cc < 8; ++cc) {
            uint32_t b[4];
            const int c16 = 2 * cc + half;
            dec_ldmatrix_t(b, vb + (c16 >> 3) * DEC_PANEL + row * 128 + (((c16 & 7) ^ (row & 7)) << 4));
            if (edge) { b[0] &= live0; b[1] &= live1; b[2] &= live0; b[3] &= live1; }
            dec_mma<BF16>(o[2 * cc], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
            dec_mma<BF16>(o[2 * cc + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
          }
        }
        if (k + 1 < s.k1) {                                  // (the last tile's slot is used below)
          __syncwarp();
          if (lane == 0) bar_arrive(bar + 8 * (DEC_STAGES + slot));
        }
      }
      // the four warps' results meet in the last tile's slot
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      }
      ok = !dec_barrier_any(!ok);                            // (all four warps go on, or none does)
      if (!ok) s_trouble = 1;
      const int slot = (count + DEC_STAGES - 1) % DEC_STAGES;   // (without tiles of its own, a CTA of a cluster has only empty records)
      const bool some = !CLUSTER || s.k0 < s.k1;
      float* buf = reinterpret_cast<float*>(ring_ptr + slot * DEC_STAGE);
      if (ok && some) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = r0 + 8 * r;
          if (row < rows) {
            if ((lane & 3) == 0) s_ml[warp][row] = make_float2(m[r], l[r]);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              *reinterpret_cast<float2*>(buf + ((warp * DEC_ROWS + row) * 128 + 8 * i + c2)) = make_float2(o[i][2 * r], o[i][2 * r + 1]);
          }
        }
      }
      dec_barrier();
      if (ok) {
        for (int row = warp; row < rows; row += DEC_WARPS) {   // four channels a lane
          float M = -INFINITY, L = 0.f;
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < DEC_WARPS; ++w) if (some) M = fmaxf(M, s_ml[w][row].x);
#pragma unroll
          for (int w = 0; w < DEC_WARPS; ++w) {
            if (!some) break;
            const float2 ml = s_ml[w][row];
            const float f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - M);
            const float4 x = *reinterpret_cast<const float4*>(buf + ((w * DEC_ROWS + row) * 128 + 4 * lane));
            if (ml.x != -INFINITY || ml.y != 0.f) {        // (a warp that saw nothing of the row adds nothing)
              L = fmaf(ml.y, f, L);
              sum.x = fmaf(x.x, f, sum.x); sum.y = fmaf(x.y, f, sum.y); sum.z = fmaf(x.z, f, sum.z); sum.w = fmaf(x.w, f, sum.w);
            }
          }
          if (CLUSTER) {
            *reinterpret_cast<float4*>(&s_rec[row][4 + 4 * lane]) = sum;
            if (lane == 0) *reinterpret_cast<float4*>(&s_rec[row][0]) = make_float4(M, L, 0.f, 0.f);
            continue;
          }
          const PagedRow d = paged_row<DEC_ROWS>(A, s, row, cta);
          if (d.rec != nullptr) {
            *reinterpret_cast<float4*>(d.rec + 4 + 4 * lane) = sum;
            if (lane == 0) *reinterpret_cast<float4*>(d.rec) = make_float4((M - LIFT) * PAGED_LN2, L, 0.f, 0.f);
          } else {
            const float w = paged_over(L);
            *reinterpret_cast<uint2*>(d.out + 4 * lane) = make_uint2(paged_pack<BF16>(sum.x * w, sum.y * w), paged_pack<BF16>(sum.z * w, sum.w * w));
          }
        }
        if (!CLUSTER && s_again[segment & 1] == (int)segment + 1) {
          const PagedSegment copy = s;
          for (int row = warp; row < rows; row += DEC_WARPS) paged_repair<BF16, DEC_KEYS, DEC_ROWS>(A, copy, row, row + 1, cta);
        }
        fence_async_smem();                                  // (the slot's next writer is a TMA copy)
        __syncwarp();
        if (lane == 0 && some) bar_arrive(bar + 8 * (DEC_STAGES + slot));
      }
      if constexpr (CLUSTER) {
        // the cluster's records of a row, added up in rank order by one warp of one CTA
        const int size = walk.size, rank = walk.rank;
        const uint32_t recs = smem_addr(s_rec), flag = smem_addr(&s_again[segment & 1]);
        __syncwarp();
        dec_cluster_sync();
        bool repair = false;
        if (lane < size) {
          int x;
          asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(x) : "r"(dec_map(flag, lane)) : "memory");
          repair = x == (int)segment + 1;
        }
        repair = __any_sync(0xffffffffu, repair);
        s.k0 = 0; s.k1 = s.item.n;
        for (int row = rank + warp * size; row < rows; row += DEC_WARPS * size) {
          const uint32_t at = recs + (uint32_t)row * RDKV_PARTIAL_STRIDE * 4u;
          float4 ml = make_float4(-INFINITY, 0.f, 0.f, 0.f);
          if (lane < size) ml = dec_remote4(dec_map(at, lane));
          const float M = warp_max(ml.x), f = ml.x == -INFINITY ? 0.f : exp2_approx(ml.x - M);
          const float L = warp_sum(ml.y * f);
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int x0 = 0; x0 < size; x0 += 4) {             // (clusters are of 8, 12 or 16)
            float4 p[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) p[e] = dec_remote4(dec_map(at + 16u + 16u * lane, x0 + e));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float w = __shfl_sync(0xffffffffu, f, x0 + e);
              sum.x = fmaf(p[e].x, w, sum.x); sum.y = fmaf(p[e].y, w, sum.y); sum.z = fmaf(p[e].z, w, sum.z); sum.w = fmaf(p[e].w, w, sum.w);
            }
          }
          const PagedRow d = paged_row<DEC_ROWS>(A, s, row, cta);
          if (d.rec != nullptr) {
            *reinterpret_cast<float4*>(d.rec + 4 + 4 * lane) = sum;
            if (lane == 0) *reinterpret_cast<float4*>(d.rec) = make_float4((M - LIFT) * PAGED_LN2, L, 0.f, 0.f);
          } else {
            const float w = paged_over(L);
            *reinterpret_cast<uint2*>(d.out + 4 * lane) = make_uint2(paged_pack<BF16>(sum.x * w, sum.y * w), paged_pack<BF16>(sum.z * w, sum.w * w));
          }
          if (repair) {
            const PagedSegment copy = s;
            paged_repair<BF16, DEC_KEYS, DEC_ROWS>(A, copy, row, row + 1, cta);
          }
        }
        __syncwarp();
        dec_cluster_sync();                                  // (records stay until everybody has read them)
      }
      ++segment;
    }
  }
  __syncthreads();
  paged_zero_padding(A, DEC_THREADS, s_trouble == 2);
  paged_report(A, s_trouble);
}

// Clusters of 16 are more than every GPU promises: asked for once per device.
template <auto Kernel>
static cudaError_t allow_big_clusters_once() {
  static std::atomic<uint64_t> done{0};
  return once_per_device(done, [] { return cudaFuncSetAttribute(Kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); });
}

template <bool BF16>
static int decode_cluster(const PagedArgs& A, unsigned ctas, unsigned size, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  constexpr auto kernel = paged_decode_kernel<BF16, true>;
  cudaError_t e = allow_dynamic_smem_once<paged_decode_kernel<BF16, true>>(DEC_SMEM);
  if (e == cudaSuccess && size > 8) e = allow_big_clusters_once<paged_decode_kernel<BF16, true>>();
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 1;
  cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(DEC_THREADS); cfg.dynamicSmemBytes = DEC_SMEM;
  if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, kernel, A, tm_k, tm_v);
  if (e != cudaSuccess) { g_last_cuda_error = (int)e; return RDKV_ERR_LAUNCH; }
  return launch_status();
}

template <bool BF16>
static int decode_line(const PagedArgs& A, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  const cudaError_t e = allow_dynamic_smem_once<paged_decode_kernel<BF16, false>>(DEC_SMEM);
  if (e != cudaSuccess) { g_last_cuda_error = (int)e; return RDKV_ERR_LAUNCH; }
  paged_decode_kernel<BF16, false><<<PAGED_DECODE_CTAS, DEC_THREADS, DEC_SMEM, st>>>(A, tm_k, tm_v);
  const int rc = launch_status();
  if (rc != RDKV_OK) return rc;
  return paged_launch_join(paged_join_kernel<BF16, DEC_ROWS, PAGED_DECODE_CTAS>, A, dim3(PAGED_DECODE_CTAS - 1, DEC_ROWS / PAGED_JOIN_WARPS), st);
}

// CTAs of the cluster that an item gets where all items' clusters fit the GPU at once, two CTAs an SM (14 clusters of 16, 21 of 12, 33
// of 8: a cluster lies in one GPC); 0: too many items.  (8 KV heads, us, clusters / line of units with its second launch: one
// request of 1000 tokens 9.0 / 13.5, of 8000 15.4 / 18.0, of 32000 38 / 38; two of 1000 10.6 / 12.7, of 32000 51 / 52; four of 1000 10.2 / 13.1.
// Sixteen clusters of 16 are two waves: two requests of 1000 tokens 16.0.)
static int paged_cluster_size(int64_t n_requests, int H_kv) {
  const int64_t items = n_requests * H_kv;
  return items <= 0 || items > 33 ? 0 : items <= 14 ? 16 : items <= 21 ? 12 : 8;
}

int paged_decode_launch(const PagedArgs& A, bool bf16, const CUtensorMap& tm_k, const CUtensorMap& tm_v, cudaStream_t st) {
  const int size = paged_cluster_size(A.S, A.H_kv);
  if (size > 0) {
    const unsigned ctas = (unsigned)(A.S * A.H_kv * size);
    return bf16 ? decode_cluster<true>(A, ctas, (unsigned)size, tm_k, tm_v, st) : decode_cluster<false>(A, ctas, (unsigned)size, tm_k, tm_v, st);
  }
  return bf16 ? decode_line<true>(A, tm_k, tm_v, st) : decode_line<false>(A, tm_k, tm_v, st);
}

}  // namespace rdkv

using namespace rdkv;

// Rows of a request's longest chunk under one KV head decide the kernel: up to 16 fill one tile of the decode kernel, up to 24 (two
// tiles, which read the keys twice, the second time from L2) are still faster there unless clusters would take the two in
// turn.  (8 KV heads, us, decode kernel / chunk kernel: 16 requests x 4000 tokens, 20 rows 40 / 52; 64 x 4000, 20 rows 106 / 120 and 32 rows
// 141 / 123; 200 x 1000, 20 rows 101 / 133; one request of 30000, 32 rows 72 / 45.)
static bool paged_few_rows(int n_requests, int H_kv, int max_new, int g) {
  const int64_t rows = (int64_t)max_new * g;
  return rows <= PAGED_DECODE_ROWS || (rows <= PAGED_DECODE_ROWS + 8 && paged_cluster_size(n_requests, H_kv) == 0);
}

extern "C" int64_t rdkv_paged_attention_workspace(int n_requests, int n_tokens, int H_q, int H_kv, int max_new) {
  if (n_requests < 0 || n_tokens < 0 || H_q <= 0 || H_kv <= 0 || max_new < 0) return -1;
  if (n_tokens == 0) return 0;
  return paged_few_rows(n_requests, H_kv, max_new, H_q / H_kv) ? paged_workspace_bytes(PAGED_DECODE_CTAS, PAGED_DECODE_ROWS)
                                             : paged_workspace_bytes(PAGED_CHUNK_CTAS, PAGED_CHUNK_ROWS);
}

extern "C" int rdkv_sizeof_paged_attention_args(void) { return (int)sizeof(rdkv_paged_attention_args); }
extern "C" int rdkv_paged_attention_status_words(void) { return PAGED_STATUS_WORDS; }

extern "C" int rdkv_paged_attention(const rdkv_paged_attention_args* args, const void* q, const void* k_pages, const void* v_pages,
                                    const int32_t* block_tables, const int32_t* q_start, const int32_t* kv_lens, void* out,
                                    int64_t out_tok_stride, int64_t out_head_stride, int zero_padding, float* out_partial,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
  return rdkv_paged_attention_within(args, q, k_pages, v_pages, block_tables, q_start, kv_lens, out, out_tok_stride, out_head_stride, zero_padding,
                                     out_partial, workspace, workspace_bytes, (int)(WAIT_NS / 1000u), stream);
}

extern "C" int rdkv_paged_attention_within(const rdkv_paged_attention_args* args, const void* q, const void* k_pages, const void* v_pages,
                                           const int32_t* block_tables, const int32_t* q_start, const int32_t* kv_lens, void* out,
                                           int64_t out_tok_stride, int64_t out_head_stride, int zero_padding, float* out_partial,
                                           void* workspace, int64_t workspace_bytes, int wait_us, void* stream) {
  if (args == nullptr) return RDKV_ERR_BAD_ARG;
  const rdkv_paged_attention_args& g = *args;
  if (g.n_tokens < 0 || g.n_requests < 0 || g.H_q <= 0 || g.H_kv <= 0 || g.n_pages < 0 || g.width < 0 || g.window < 0 || g.sinks < 0 ||
      g.max_new < 0 || !(g.scale > 0.f && g.scale <= 1e30f) || wait_us < 0 || wait_us > 4000000)
    return RDKV_ERR_BAD_ARG;
  if (g.dtype != RDKV_F16 && g.dtype != RDKV_BF16) return RDKV_ERR_BAD_ARG;
  if (g.H_q % g.H_kv != 0 || g.H_q / g.H_kv > MAX_GROUP) return RDKV_ERR_BAD_SHAPE;
  if (g.page_size < 16 || g.page_size > 1024 || (g.page_size & (g.page_size - 1)) != 0) return RDKV_ERR_BAD_SHAPE;
  if (g.n_tokens == 0) return RDKV_OK;
  if (q == nullptr || q_start == nullptr || (out == nullptr) == (out_partial == nullptr)) return RDKV_ERR_BAD_ARG;
  if (g.n_requests > 0 && (kv_lens == nullptr || (g.width > 0 && block_tables == nullptr))) return RDKV_ERR_BAD_ARG;
  if (g.n_pages > 0 && (k_pages == nullptr || v_pages == nullptr)) return RDKV_ERR_BAD_ARG;
  if (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0 ||
      workspace_bytes < rdkv_paged_attention_workspace(g.n_requests, g.n_tokens, g.H_q, g.H_kv, g.max_new))
    return RDKV_ERR_BAD_ARG;
  // queries are read, results and records written, 16 bytes at a time
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) || (reinterpret_cast<uintptr_t>(out_partial) & 15))
    return RDKV_ERR_BAD_ARG;
  auto whole = [](int64_t n, int64_t stride) { return n == 1 || (stride & 7) == 0; };   // (strides of dimensions of one element mean nothing)
  if (!whole(g.n_tokens, g.q_tok_stride) || !whole(g.H_q, g.q_head_stride) ||
      (out != nullptr && (!whole(g.n_tokens, out_tok_stride) || !whole(g.H_q, out_head_stride))))
    return RDKV_ERR_BAD_SHAPE;
  PagedArgs A = {};
  A.q = (const uint16_t*)q; A.k = (const uint16_t*)k_pages; A.v = (const uint16_t*)v_pages;
  A.q_tok = g.q_tok_stride; A.q_head = g.q_head_stride;
  A.k_page = g.k_page_stride; A.k_head = g.k_head_stride; A.k_row = g.k_row_stride;
  A.v_page = g.v_page_stride; A.v_head = g.v_head_stride; A.v_row = g.v_row_stride;
  A.n_pages = g.n_pages; A.page = g.page_size; A.H_q = g.H_q; A.H_kv = g.H_kv; A.g = g.H_q / g.H_kv;
  for (A.page_log2 = 0; (1 << A.page_log2) < g.page_size; ++A.page_log2) {}
  A.table = block_tables; A.table_stride = g.table_stride; A.width = g.width;
  A.cap = (int)std::min<int64_t>((int64_t)g.width * g.page_size, 0x7fff0000);
  A.q_start = q_start; A.kv_lens = kv_lens; A.S = g.n_requests; A.T = g.n_tokens;
  A.window = std::min(g.window, 1 << 30); A.sinks = std::min(g.sinks, 1 << 30); A.scale_log2 = g.scale * PAGED_LOG2E;
  A.wait_ns = (uint32_t)wait_us * 1000u;
  A.out = (uint16_t*)out; A.o_tok = out_tok_stride; A.o_head = out_head_stride; A.zero_pad = zero_padding; A.rec = out_partial;
  const bool bf = g.dtype == RDKV_BF16, few = paged_few_rows(g.n_requests, g.H_kv, g.max_new, A.g);
  A.group = few ? PAGED_DECODE_ROWS / A.g : 2 * (128 / A.g);
  // a head's line of units has to fit 31 bits: (groups of new tokens) x (tiles of the longest request the table has room for)
  const int64_t groups = (int64_t)g.n_tokens / A.group + g.n_requests + 1, tiles = A.cap / (few ? PAGED_DECODE_KEYS : PAGED_CHUNK_KEYS) + 4;
  if (groups * tiles > 0x7fffffffLL) return RDKV_ERR_TOO_LARGE;
  paged_workspace(&A, workspace, few ? PAGED_DECODE_CTAS : PAGED_CHUNK_CTAS);
  CUtensorMap tm_k, tm_v;
  const int box = std::min(g.page_size, few ? PAGED_DECODE_KEYS : PAGED_CHUNK_KEYS);
  if (!paged_map(&tm_k, k_pages, bf, g.k_page_stride, g.k_head_stride, g.k_row_stride, g.n_pages, g.H_kv, g.page_size, box) ||
      !paged_map(&tm_v, v_pages, bf, g.v_page_stride, g.v_head_stride, g.v_row_stride, g.n_pages, g.H_kv, g.page_size, box))
    return RDKV_ERR_BAD_SHAPE;
  return few ? paged_decode_launch(A, bf, tm_k, tm_v, (cudaStream_t)stream) : paged_chunk_launch(A, bf, tm_k, tm_v, (cudaStream_t)stream);
}
