// Rotation of query and key rows by positions with several axes, alone or together with the write of the key and
// value rows to their pages: one launch.
//
// Of the 64 rotation frequencies of a head, section a (a run of them) turns with axis a of the token's position:
//   angle_j = position[axis(j)] * inv_freq[j],   (x[j], x[j+64]) -> (x[j] cos - x[j+64] sin, x[j+64] cos + x[j] sin).
// The angle is taken in turns: position * inv_freq / (2 pi) as a sum of two 64-bit numbers (the products' rounding errors are kept),
// whose whole turns are dropped, which is exact.  What is left (half a turn at most) is rounded to 32 bits, 2^-25 of a turn,
// for every position up to 2^53 (larger ones are no longer whole numbers in 64 bits).  In 32 bits a position of 10^6
// would leave an error of 2^-5 radians.  Rows are rotated in 32 bits and rounded once.
//
// A warp belongs to a token: each lane computes two of its 64 angles and the warp trades them (16 shuffles); eight lanes
// then take a row, eight pairs each, with 16-byte loads and stores, four rows at a time, and the angles serve all rows
// of the token that the warp takes.  Few tokens: their rows are dealt out to several warps.  Bound by memory traffic (rows
// once in, once out; bf16, in a replayed graph): 8192 tokens of 64 + 2 x 8 heads into pages of 16 60.5 us, 5.5 TB/s; 6007 tokens of 32 + 8
// heads with three axes 24.7 us, 5.0 TB/s.
#include <algorithm>

#include "rdkv_common.cuh"

namespace rdkv {

constexpr int AXES_THREADS = 128;
constexpr int AXES_MAX = 4;

struct AxesArgs {
  const void* q; const void* k; const void* v;   // [T][H][128]; v only with pages
  void* q_out; void* k_out;                      // k_out: rows [T][H_kv][128], or the key pages
  void* v_pages;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head, ko_tok, ko_head;   // elements; with pages ko_* are unused
  int64_t kp_page, kp_head, kp_row, vp_page, vp_head, vp_row;
  const int64_t* slots; int64_t n_slots; int page;
  const void* positions; int64_t pos_axis; int pos64;
  const float* inv_freq;
  int edge[AXES_MAX];                            // section a ends before frequency edge[a]
  int n_axes, T, H_q, H_kv, warps_per_token, aligned;
};

template <class E> struct AxesType;
template <> struct AxesType<__half> {
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};
template <> struct AxesType<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
};
template <> struct AxesType<float> {
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};

template <class E> struct alignas(16) AxesEight { E x[8]; };

template <class E>
__device__ __forceinline__ AxesEight<E> axes_load(const E* p, bool aligned) {
  AxesEight<E> r;
  if (aligned) r = *reinterpret_cast<const AxesEight<E>*>(p);
  else
#pragma unroll
    for (int e = 0; e < 8; ++e) r.x[e] = p[e];
  return r;
}
template <class E>
__device__ __forceinline__ void axes_store(E* p, const AxesEight<E>& r, bool aligned) {
  if (aligned) *reinterpret_cast<AxesEight<E>*>(p) = r;
  else
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = r.x[e];
}

template <class E, bool PAGES>
__global__ void __launch_bounds__(AXES_THREADS)
rope_axes_kernel(const AxesArgs A) {
  const int lane = threadIdx.x & 31, l8 = lane & 7, group = lane >> 3;
  const int64_t warp = (int64_t)blockIdx.x * (AXES_THREADS / 32) + (threadIdx.x >> 5);
  const int64_t t = warp / A.warps_per_token;
  if (t >= A.T) return;
  const int part = (int)(warp - t * A.warps_per_token);
  float c[8], s[8];
  if (A.n_axes > 0) {
    float cs[2], sn[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int j = 2 * lane + e;
      int axis = 0;
#pragma unroll
      for (int a = 0; a < AXES_MAX - 1; ++a) axis += (a < A.n_axes - 1 && j >= A.edge[a]) ? 1 : 0;
      const int64_t at = axis * A.pos_axis + t;
      const double pos = A.pos64 ? (double)reinterpret_cast<const int64_t*>(A.positions)[at]
                                 : (double)reinterpret_cast<const int32_t*>(A.positions)[at];
      // inv_freq / (2 pi) = w + w_lo, 1 / (2 pi) = INV + INV_LO; the position times that = x + x_lo
      constexpr double INV = 0x1.45f306dc9c883p-3, INV_LO = -0x1.6b01ec5417056p-57;
      const double f = A.inv_freq[j], w = f * INV, w_lo = fma(f, INV, -w) + f * INV_LO;
      const double x = pos * w, x_lo = fma(pos, w, -x) + pos * w_lo;
      const double turns = (x - rint(x)) + x_lo;             // (x_lo is over a turn where x has no bits below one)
      sincospif(2.f * (float)(turns - rint(turns)), &sn[e], &cs[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {                            // frequency 8*l8 + e is with lane 4*l8 + e/2
      c[e] = __shfl_sync(0xffffffffu, cs[e & 1], 4 * l8 + (e >> 1));
      s[e] = __shfl_sync(0xffffffffu, sn[e & 1], 4 * l8 + (e >> 1));
    }
  }
  int64_t page = -1, row = 0;
  if (PAGES) {
    const int64_t slot = A.slots[t];
    if (slot >= 0 && slot < A.n_slots) { page = slot / A.page; row = slot - page * A.page; }
  }
  const bool al = A.aligned != 0;
  const int rows = A.H_q + A.H_kv * (PAGES ? 2 : 1);
  for (int r = part * 4 + group; r < rows; r += A.warps_per_token * 4) {
    const E* src; E* dst;
    bool turn = A.n_axes > 0;
    if (r < A.H_q) {
      src = reinterpret_cast<const E*>(A.q) + t * A.q_tok + r * A.q_head;
      dst = reinterpret_cast<E*>(A.q_out) + t * A.qo_tok + r * A.qo_head;
    } else if (r < A.H_q + A.H_kv) {
      const int h = r - A.H_q;
      src = reinterpret_cast<const E*>(A.k) + t * A.k_tok + h * A.k_head;
      dst = reinterpret_cast<E*>(A.k_out) + (PAGES ? page * A.kp_page + h * A.kp_head + row * A.kp_row : t * A.ko_tok + h * A.ko_head);
      if (PAGES && page < 0) continue;
    } else {
      const int h = r - A.H_q - A.H_kv;
      if (page < 0) continue;
      src = reinterpret_cast<const E*>(A.v) + t * A.v_tok + h * A.v_head;
      dst = reinterpret_cast<E*>(A.v_pages) + page * A.vp_page + h * A.vp_head + row * A.vp_row;
      turn = false;
    }
    AxesEight<E> a = axes_load(src + 8 * l8, al), b = axes_load(src + 64 + 8 * l8, al);
    if (turn) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = AxesType<E>::up(a.x[e]), y = AxesType<E>::up(b.x[e]);
        a.x[e] = AxesType<E>::down(fmaf(x, c[e], -(y * s[e])));
        b.x[e] = AxesType<E>::down(fmaf(y, c[e], x * s[e]));
      }
    }
    axes_store(dst + 8 * l8, a, al);
    axes_store(dst + 64 + 8 * l8, b, al);
  }
}

// `sections` [n_axes] on the host; false if they are not 1 to 4 runs that cover the 64 frequencies.
static bool axes_sections(AxesArgs* A, const int* sections, int n_axes) {
  if (n_axes < 1 || n_axes > AXES_MAX) return false;
  int end = 0;
  for (int a = 0; a < n_axes; ++a) {
    if (sections[a] < 0 || sections[a] > 64) return false;
    end += sections[a];
    A->edge[a] = end;
  }
  A->n_axes = n_axes;
  return end == 64;
}

static int axes_launch(AxesArgs& A, int dtype, bool pages, cudaStream_t st) {
  const int rows = A.H_q + A.H_kv * (pages ? 2 : 1);
  if (A.T == 0 || rows == 0) return RDKV_OK;
  // warps a token: enough for 48 per SM, four rows each at least.  (6007 tokens of 40 heads, bf16, a call in a stream of calls: 28.2 us with a warp a token,
  // 26.1 with two, 27.4 with three; several rows a lane at a time were slower, 28.7 with two, 35.4 with four.)
  const int most = (rows + 3) / 4;
  A.warps_per_token = (int)std::min<int64_t>(most, std::max<int64_t>(1, (148 * 48 + A.T - 1) / A.T));
  const int64_t blocks = ((int64_t)A.T * A.warps_per_token + AXES_THREADS / 32 - 1) / (AXES_THREADS / 32);
  if (blocks > 0x7fffffffLL) return RDKV_ERR_TOO_LARGE;
  auto go = [&](auto kernel) { kernel<<<(unsigned)blocks, AXES_THREADS, 0, st>>>(A); };
  if (dtype == RDKV_F16) { if (pages) go(rope_axes_kernel<__half, true>); else go(rope_axes_kernel<__half, false>); }
  else if (dtype == RDKV_BF16) { if (pages) go(rope_axes_kernel<__nv_bfloat16, true>); else go(rope_axes_kernel<__nv_bfloat16, false>); }
  else { if (pages) go(rope_axes_kernel<float, true>); else go(rope_axes_kernel<float, false>); }
  return launch_status();
}

// Whether eight elements of every row lie on a boundary of their size (16 bytes; 32-bit rows: two such loads).
static bool axes_aligned(int dtype, std::initializer_list<const void*> bases, std::initializer_list<int64_t> strides) {
  const int64_t unit = dtype == RDKV_F32 ? 4 : 8;
  for (const void* p : bases) if (reinterpret_cast<uintptr_t>(p) & 15) return false;
  for (int64_t s : strides) if (s % unit) return false;
  return true;
}

}  // namespace rdkv

using namespace rdkv;

extern "C" int rdkv_sizeof_rope_axes_args(void) { return (int)sizeof(rdkv_rope_axes_args); }
extern "C" int rdkv_sizeof_paged_append_args(void) { return (int)sizeof(rdkv_paged_append_args); }

extern "C" int rdkv_rope_axes(const rdkv_rope_axes_args* args, const void* q, void* q_out, const void* k, void* k_out,
                              const void* positions, const float* inv_freq, void* stream) {
  if (args == nullptr) return RDKV_ERR_BAD_ARG;
  const rdkv_rope_axes_args& g = *args;
  if (g.n_tokens < 0 || g.H_q < 0 || g.H_kv < 0 || g.dtype < RDKV_F16 || g.dtype > RDKV_F32) return RDKV_ERR_BAD_ARG;
  if (g.n_tokens > 0 && ((g.H_q > 0 && (q == nullptr || q_out == nullptr)) || (g.H_kv > 0 && (k == nullptr || k_out == nullptr)) ||
                         positions == nullptr || inv_freq == nullptr))
    return RDKV_ERR_BAD_ARG;
  AxesArgs A = {};
  if (!axes_sections(&A, g.sections, g.n_axes)) return RDKV_ERR_BAD_SHAPE;
  A.q = q; A.k = k; A.q_out = q_out; A.k_out = k_out;
  A.q_tok = g.q_tok_stride; A.q_head = g.q_head_stride; A.k_tok = g.k_tok_stride; A.k_head = g.k_head_stride;
  A.qo_tok = g.q_out_tok_stride; A.qo_head = g.q_out_head_stride; A.ko_tok = g.k_out_tok_stride; A.ko_head = g.k_out_head_stride;
  A.positions = positions; A.pos_axis = g.axis_stride; A.pos64 = g.positions_64; A.inv_freq = inv_freq;
  A.T = g.n_tokens; A.H_q = g.H_q; A.H_kv = g.H_kv;
  A.aligned = axes_aligned(g.dtype, {q, k, q_out, k_out}, {A.q_tok, A.q_head, A.k_tok, A.k_head, A.qo_tok, A.qo_head, A.ko_tok, A.ko_head});
  return axes_launch(A, g.dtype, false, (cudaStream_t)stream);
}

extern "C" int rdkv_paged_append(const rdkv_paged_append_args* args, const void* k, const void* v, void* k_pages, void* v_pages,
                                 const int64_t* slot_map, const void* q, void* q_out, const void* positions,
                                 const float* inv_freq, void* stream) {
  if (args == nullptr) return RDKV_ERR_BAD_ARG;
  const rdkv_paged_append_args& g = *args;
  if (g.n_tokens < 0 || g.H_q < 0 || g.H_kv <= 0 || g.dtype < RDKV_F16 || g.dtype > RDKV_F32 || g.n_pages < 0 || g.page_size <= 0)
    return RDKV_ERR_BAD_ARG;
  if (g.n_tokens > 0 &&
      (k == nullptr || v == nullptr || slot_map == nullptr || (g.n_pages > 0 && (k_pages == nullptr || v_pages == nullptr)) ||
       (g.H_q > 0 && (q == nullptr || q_out == nullptr)) || (g.n_axes > 0 && (positions == nullptr || inv_freq == nullptr))))
    return RDKV_ERR_BAD_ARG;
  AxesArgs A = {};
  if (g.n_axes != 0 && !axes_sections(&A, g.sections, g.n_axes)) return RDKV_ERR_BAD_SHAPE;
  A.q = q; A.k = k; A.v = v; A.q_out = q_out; A.k_out = k_pages; A.v_pages = v_pages;
  A.q_tok = g.q_tok_stride; A.q_head = g.q_head_stride; A.k_tok = g.k_tok_stride; A.k_head = g.k_head_stride; A.v_tok = g.v_tok_stride;
  A.v_head = g.v_head_stride; A.qo_tok = g.q_out_tok_stride; A.qo_head = g.q_out_head_stride;
  A.kp_page = g.k_page_stride; A.kp_head = g.k_page_head_stride; A.kp_row = g.k_page_row_stride;
  A.vp_page = g.v_page_stride; A.vp_head = g.v_page_head_stride; A.vp_row = g.v_page_row_stride;
  A.slots = slot_map; A.n_slots = (int64_t)g.n_pages * g.page_size; A.page = g.page_size;
  A.positions = positions; A.pos_axis = g.axis_stride; A.pos64 = g.positions_64; A.inv_freq = inv_freq;
  A.T = g.n_tokens; A.H_q = g.H_q; A.H_kv = g.H_kv;
  A.aligned = axes_aligned(g.dtype, {q, k, v, q_out, k_pages, v_pages},
                           {A.q_tok, A.q_head, A.k_tok, A.k_head, A.v_tok, A.v_head, A.qo_tok, A.qo_head, A.kp_page, A.kp_head, A.kp_row,
                            A.vp_page, A.vp_head, A.vp_row});
  return axes_launch(A, g.dtype, true, (cudaStream_t)stream);
}
