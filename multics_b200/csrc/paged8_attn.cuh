// What the attention kernels over an 8-bit paged cache share: their arguments,
// the tiles of rows a call is cut into, and the exponents of its rows.
//
// out[r, h] = sum_j softmax_j(scale q[r, h] . (sk K8[j])) sv V8[j] over the keys
// that row r sees.  A tile is `kRows` consecutive (row, head of the key head's
// group) pairs of one request, row-major: rho = row * G + g.  Tile t of request
// b is number q_start[b] * G / kRows + min(b, q_start[b]) + t, so a launch needs
// no count from the device; numbers between the requests' tiles are empty.
// (Before a request with rows there are at most that many others with rows, so
// requests without any take no numbers.)
//
// The page scales never touch the codes: a page's key scale multiplies its
// scores s_j, and its value scale 2^ve is added to their exponents, so that with
//   s_j = scale log2(e) sk q.k_j,   m = max (s_j + ve),   p_j = 2^(s_j + ve - m)
// the product sum p_j V8[j] is the output's numerator times 2^-m and p_j is at
// most 1 (fp16 keeps 11 bits of it whatever the pages' scales are).  The
// denominator has a maximum of its own, n = max s_j:
//   l = sum 2^(s_j - n) = sum over pages 2^(m - ve - n) sum p_j,
// from the same exponentials.  Only a page whose p_j are below 2^-60 and whose
// s_j are not far below n (far_page: value scales far apart, such as those of a
// page of zeros) is summed by exponentials of its own: its p_j may be flushed
// though it weighs.  Results of parts of the keys are joined as outputs with the
// weights l 2^n.
#pragma once

#include <float.h>

#include "paged8.cuh"

namespace hier {

struct Paged8Args {
  const __nv_bfloat16* q;
  int64_t q_stride;
  int rows, heads;
  Divisor kv_heads, group;  // key heads, query heads of each
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  int n_pages;
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* lengths;
  const int32_t* q_start;
  int n;
  Paged8Mask mask;
  float scale_log2;
  __nv_bfloat16* out;
  int64_t out_stride;
  float* lse;       // [rows][heads] log2-sum-exp, or NULL
  int zero_rest;    // rows of no request: 1 zeros, 2 their log-sum-exp alone, 0 left
  Divisor splits;   // most parts a tile's keys are cut into
  float* part_o;    // [tile][kv head][split][kRows][128]
  float* part_nl;   // [tile][kv head][split][kRows][2]: n and l
  int cluster;      // the parts of a small tile are the blocks of a cluster
  int row_limit;    // requests of up to row_limit pairs are the small kernel's, the others the
                    // large one's (INT_MAX: all the small one's, 0: all the large one's)
  int keep;         // small kernels: whether there are blocks of no unit (keep_rows)
  Divisor direct;   // small kernel: its tile t is tile t % direct of request t / direct
  int32_t* status;
  int* err;         // bounded waits
};

constexpr int kPaged8SmallRows = 8;
constexpr int kPaged8LargeRows = 256;
constexpr int kPaged8LargeMin = 8;  // 128-key tiles of a part at least

template <int kRows>
__host__ __device__ inline int64_t paged8_tiles(int64_t rows, int group, int n) {
  return rows * group / kRows + (n < rows ? n : rows) + 1;
}

// The rows that requests can have: q_start's ends, within the row tensor.  A
// request whose rows leave them is refused, so that the rows outside are
// nobody's whatever stands between the ends.
struct RowSpan {
  int first, end;
  __device__ __forceinline__ bool holds(int row0, int row1) const { return row0 >= first && row1 <= end; }
};
__device__ __forceinline__ RowSpan row_span(int first, int end, int rows) {
  first = max(0, min(first, rows));
  return {first, max(first, min(end, rows))};
}
__device__ __forceinline__ RowSpan row_span(const Paged8Args& a) {
  return row_span(a.q_start[0], a.q_start[a.n], a.rows);
}

struct Paged8Tile {
  int b;
  Paged8Request rq;
  int rho0, pairs;  // first pair of the tile, pairs of the request
  int lo, hi;       // keys the tile's rows see between them
  int p0, np;       // their pages
  bool live;
};

// position of row i of a request; negative rows see nothing
__device__ __forceinline__ int row_pos(const Paged8Request& r, int i) { return r.held - r.n + i; }

__device__ __forceinline__ void row_keys(const Paged8Args& a, const Paged8Request& r, int i, int& lo,
                                         int& hi) {
  const int pos = row_pos(r, i);
  if (pos >= 0) {
    lo = a.mask.first(pos);
    hi = a.mask.end(pos, r.held);
  } else {  // rows beyond the held tokens see keys only where positions do not matter
    lo = 0;
    hi = a.mask.blocks == 0 && a.mask.window < 0 ? r.held : 0;
  }
}

// the keys that the tile's rows (up to kRows pairs from rho0) see between them
__device__ __forceinline__ void paged8_span(const Paged8Args& a, Paged8Tile& t, int rows) {
  const int last = min(t.pairs, t.rho0 + rows) - 1;
  int unused;
  row_keys(a, t.rq, t.rho0 / a.group, t.lo, unused);
  row_keys(a, t.rq, last / a.group, unused, t.hi);
  if (t.hi > t.lo) {
    t.p0 = t.lo / kPage;
    t.np = (t.hi + kPage - 1) / kPage - t.p0;
  }
}

// Number of a request's first tile, b and q_start[b] given.
template <int kRows>
__device__ __forceinline__ int64_t first_tile(const Paged8Args& a, int b, int row0) {
  return row0 * (int64_t)a.group.d / kRows + min(b, row0);
}

// The request (n: none) that tile `tile` is of, if row starts ascend; q: the
// lane's row start where n < 32.
template <int kRows>
__device__ __forceinline__ int tile_request(const Paged8Args& a, int64_t tile, int q) {
  const int32_t* qs = a.q_start;
  if (a.n < 32) {
    const int lane = threadIdx.x & 31;
    return 31 - __clz(__ballot_sync(0xffffffffu, lane <= a.n && first_tile<kRows>(a, lane, q) <= tile) | 1u);
  }
  return warp_find(a.n + 1, tile, [&](int i) { return first_tile<kRows>(a, i, qs[i]); });
}

// Whether every tile of request b is found to be its.  (As the first and the
// last are, so are those between: a search compares with tiles alone, and its
// outcomes ascend with the tile.)
template <int kRows>
__device__ __forceinline__ bool tiles_found(const Paged8Args& a, int b, int row0, int pairs) {
  const int q = a.q_start[min((int)(threadIdx.x & 31), a.n)];
  const int64_t first = first_tile<kRows>(a, b, row0);
  return tile_request<kRows>(a, first, q) == b && tile_request<kRows>(a, first + (pairs - 1) / kRows, q) == b;
}

template <int kRows>
__device__ __forceinline__ Paged8Tile paged8_tile(const Paged8Args& a, int64_t tile, bool report) {
  Paged8Tile t;
  const int32_t* qs = a.q_start;
  const int64_t G = a.group.d;
  t.live = false;
  t.rho0 = t.pairs = t.lo = t.hi = t.p0 = t.np = 0;
  int row0, row1, held, starts, ends;
  if (a.n < 32) {  // one read of everything
    const int lane = threadIdx.x & 31, i = min(lane, a.n);
    const int q = qs[i], len = a.n ? a.lengths[min(lane, a.n - 1)] : 0;
    t.b = tile_request<kRows>(a, tile, q);
    row0 = __shfl_sync(0xffffffffu, q, t.b);
    row1 = __shfl_sync(0xffffffffu, q, min(t.b + 1, 31));
    held = __shfl_sync(0xffffffffu, len, t.b);
    starts = __shfl_sync(0xffffffffu, q, 0);
    ends = __shfl_sync(0xffffffffu, q, a.n);
  } else {
    t.b = tile_request<kRows>(a, tile, 0);
    row0 = qs[t.b];
    row1 = t.b < a.n ? qs[t.b + 1] : 0;
    held = t.b < a.n ? a.lengths[t.b] : 0;
    starts = qs[0], ends = qs[a.n];
  }
  const int64_t first = first_tile<kRows>(a, t.b, row0);
  if (tile < first || t.b == a.n) return t;  // rows of no request
  const int64_t rho0 = (tile - first) * kRows;
  t.rq = paged8_request(row0, row1, held, a.rows, a.width, false, report ? a.status : nullptr);
  if (row1 <= row0 || !row_span(starts, ends, a.rows).holds(row0, row1) || rho0 >= t.rq.n * G) return t;
  if (!t.rq.ok) t.rq.held = 0;  // a length outside the table: the rows see nothing
  t.live = true;
  t.rho0 = (int)rho0;
  t.pairs = (int)(t.rq.n * G);
  paged8_span(a, t, kRows);
  return t;
}

// Zeros to a warp's heads, those of key head kvh, of a row, as zero_rest says.
__device__ __forceinline__ void zero_row(const Paged8Args& a, int64_t r, int kvh, int lane) {
  uint4* dst = reinterpret_cast<uint4*>(a.out + r * a.out_stride + kvh * a.group.d * 128);
  if (a.zero_rest == 1)
    for (int e = lane; e < a.group.d * 16; e += 32) dst[e] = make_uint4(0u, 0u, 0u, 0u);
  if (a.lse)
    for (int e = lane; e < a.group.d; e += 32) a.lse[r * a.heads + kvh * a.group.d + e] = -INFINITY;
}

// Zeros to the rows before the first request and behind the last one (to all
// where the only one is refused); worker i of n takes every n-th row.
__device__ __forceinline__ void zero_rest(const Paged8Args& a, int kvh, int64_t i, int64_t n, int lane) {
  const RowSpan s = row_span(a);
  const int64_t between = a.n == 1 && !s.holds(a.q_start[0], a.q_start[1]) ? 0 : s.end - s.first;
  for (int64_t j = i; j < a.rows - between; j += n)
    zero_row(a, j < s.first ? j : j + between, kvh, lane);
}

__device__ __forceinline__ float finite_or_0(float m) { return m == -INFINITY ? 0.f : m; }

// Whether a page's weights p, of maximum x and of scores up to s, are too small
// for the denominator's terms to be taken from them.
constexpr float kFarWeights = 60.f;
__device__ __forceinline__ bool far_page(float m, float x, float n, float s) {
  return m - x > kFarWeights && n - s < 48.f;
}
// 2^(m - ve - n): the denominator's terms from p.  (Beyond 2^126 only for pages
// whose terms are below 2^-48.)
__device__ __forceinline__ float sum_factor(float m, float ve, float n) {
  return ex2_approx(fminf(m - ve - n, 126.f));
}
// What brings the numerator to the output, 2^(m - n) / l: 0 where nothing was seen,
// NaN where the sum is.  In two factors, the second 1 but for outputs below 2^-90,
// so that none leaves fp32's normal numbers.
struct OutFactor {
  float a, b;
  __device__ __forceinline__ OutFactor(float m, float n, float l) : a(l), b(1.f) {
    if (!(l > 0.f)) return;
    a = __fdividef(ex2_approx(fmaxf(m - n, -96.f)), l);
    b = ex2_approx(fminf(m - n + 96.f, 0.f));
  }
};
__device__ __forceinline__ float inverse_or_0(float l) { return l > 0.f ? __fdividef(1.f, l) : l; }

// factor of a page's scores: finite and not 0, since a score may be 0 or -infinity
__device__ __forceinline__ float score_factor(float sc, float ks) {
  return fminf(fmaxf(sc * ks, FLT_MIN), FLT_MAX);
}

// log2-sum-exp of a pair from its maximum and sum: -inf where nothing was seen,
// NaN where the sum is
__device__ __forceinline__ float row_lse(float m, float l) {
  return l > 0.f ? m + log2f(l) : l == 0.f ? -INFINITY : l;
}

// parts that np pages are really cut into: at least kMin pages each
template <int kMin>
__device__ __forceinline__ int parts_of(int np, int splits) {
  return max(1, min(splits, np / kMin));
}

// power of two that brings a row's largest magnitude into [2^14, 2^15) in
// fp16: bf16 values keep all their bits there down to 2^-28 of the largest
__device__ __forceinline__ int fp16_shift(float amax) {
  const int e = (int)(__float_as_uint(amax) >> 23);  // biased; 0: zero or a bf16 subnormal
  return e >= 255 ? 0 : min(120, 14 + 127 - e);
}

__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// exponent of a power-of-two scale
__device__ __forceinline__ int scale_log2_of(float s) {
  return (int)((__float_as_uint(s) >> 23) & 0xffu) - 127;
}

int paged8_launch_large(const Paged8Args& a, int format, int64_t tiles, cudaStream_t st);

}  // namespace hier
