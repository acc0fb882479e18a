// Attention of a few rows over an 8-bit paged cache (sm_100a), the merge of
// split keys, and the entry point of all attention kernels.
//
// A warp takes 8 (row, head) pairs of one key head and walks pages of 64 keys.
// Bound by the bytes of the cache: the codes go from global memory straight to
// registers (16 bytes per lane, every line used whole), are turned into fp16
// there and fed to m16n8k16 products with the keys (or the value dimensions) as
// rows and the 8 pairs as columns:
//   S^T (keys x pairs) = K Q^T,    O^T (dimensions x pairs) += V^T P^T.
// The page layout gives a lane consecutive codes of the reduction axis; the
// order of the reduction inside a product is free as long as both operands use
// the same one, so no code is moved between lanes.  P^T goes from the layout
// of a result to that of an operand by an 8x8 transpose in the register file.
//
// Two kernels.  paged8_long_kernel, where rows can see more than kShortPages
// pages: four warps of a block share a tile's pages (joined in shared memory),
// and with few tiles the keys are also split over blocks.  Few parts are the
// blocks of a cluster, which joins them over distributed shared memory: no
// workspace and no second launch (a row of each of 4 requests over 3 000 tokens,
// 24 heads to 8: 11.9 us, with a second kernel 2.2 more; 3.3 us less of the host).
// Where twice the portable cluster's 8 blocks could share the keys, the parts go
// to a workspace and a second kernel joins them (one row over 9 240 tokens of 24
// heads: 20.0 us, as a cluster 1.4 more; over 100 000 tokens, 8 heads to one: 32.5
// against 94), and so they do beyond one wave of blocks, where clusters wait for places
// (37 rows of 4 key heads: 91 us against 103).  Parts are always joined in their
// order.
// While a page's scores are computed its values are in flight, and while its
// values are consumed the next page's keys are: the loads of one take the
// registers that the other's products have just used.  37 rows over up to 19 001
// tokens, 32 heads to 4, e4m3: 92.5 us, 5.7 TB/s, 0.87 of the measured copy rate.
// One row over 9 240 tokens: DRAM 37 % and issue slots 41 % busy, its warps with two
// pages each wait for loads.  Beyond 888 (request, key head) tiles the keys are not
// split whatever the lengths are: one long request among hundreds of short ones is
// read by a block per key head.
// paged8_short_kernel: a warp per tile, and products over 16 or 32 keys at a
// time, its loads issued together.  880 requests of 3 rows over 12 to 24 tokens, 24
// heads, int8: 51 us, 4.9 TB/s (a value's 64-byte row is read whole, which makes
// 249 MB of 126) with half of the issue slots used; more warps than the 16 of 128
// registers spill much (5 blocks per SM: 70 us; as built 4 bytes, 16 for e4m3, and 44
// in the other kernel).

#include <math.h>

#include <algorithm>

#include "paged8_attn.cuh"

namespace hier {
namespace {

constexpr int kRows = kPaged8SmallRows;
constexpr int kWarps = 4;
constexpr int kPitch = 132;  // floats: 8 x 4 lanes of one store fall into 32 banks

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// 16 codes, or zeros; volatile, so that the loads stay where they are written
// between the products and the registers they fill are those just used up
__device__ __forceinline__ uint4 ld_codes(const uint8_t* p, bool in) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((int)in));
  return v;
}

__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

__device__ __forceinline__ uint2 ld_shared2(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}

// page of the table entry, or -1 (reported) when it leaves the pool
__device__ __forceinline__ int page_at(const Paged8Args& a, const int32_t* row, int p, int lane) {
  const int page = row[p];
  if (page >= 0 && page < a.n_pages) return page;
  if (lane == 0) atomicOr(a.status, P8_BAD_PAGE);
  return -1;
}

// row of a request and head of the group of pair rho
__device__ __forceinline__ void split_pair(const Paged8Args& a, int rho, int& row, int& g) {
  row = rho / a.group;
  g = rho - row * a.group.d;
}

// The 8 pairs of tile i of request b, from pair rho0.
__device__ __forceinline__ Paged8Tile small_tile(const Paged8Args& a, int b, int rho0, bool report) {
  Paged8Tile t;
  t.b = b;
  t.rho0 = rho0;
  t.lo = t.hi = t.p0 = t.np = t.pairs = 0;
  const RowSpan span = row_span(a);
  const int row0 = a.q_start[b], row1 = a.q_start[b + 1];
  t.rq = paged8_request(row0, row1, a.lengths[b], a.rows, a.width, false, report ? a.status : nullptr);
  t.live = row1 > row0 && span.holds(row0, row1);
  if (!t.live) return t;
  t.pairs = t.rq.n * a.group;
  t.live = rho0 < t.pairs && t.pairs <= a.row_limit;
  if (!t.rq.ok) t.rq.held = 0;  // a length outside the table: the rows see nothing
  if (t.live) paged8_span(a, t, kRows);
  return t;
}

// What a lane knows of its tile's pairs.  In the products a lane's group g owns
// column g of the queries, and it holds results of columns 2t and 2t + 1.
struct Columns {
  const __nv_bfloat16* q;  // the lane's 32 query values of pair g of key head 0
  bool in;
  int lo[2], hi[2];        // keys that columns 2t, 2t + 1 see
  int all_lo, all_hi;      // keys that every pair sees
};

__device__ __forceinline__ Columns columns(const Paged8Args& a, const Paged8Tile& tl, int lane) {
  const int g = lane >> 2, t = lane & 3;
  Columns c;
  const int rho = tl.rho0 + g;
  c.in = rho < tl.pairs;
  int qi, qg, lo = INT_MAX, hi = 0;
  split_pair(a, c.in ? rho : tl.rho0, qi, qg);
  if (c.in) row_keys(a, tl.rq, qi, lo, hi);
  c.q = a.q + (tl.rq.row0 + (int64_t)qi) * a.q_stride + qg * 128 + 16 * t;
  c.all_lo = c.in ? lo : 0, c.all_hi = c.in ? hi : INT_MAX;
#pragma unroll
  for (int i = 4; i < 32; i <<= 1) {
    c.all_lo = max(c.all_lo, __shfl_xor_sync(0xffffffffu, c.all_lo, i));
    c.all_hi = min(c.all_hi, __shfl_xor_sync(0xffffffffu, c.all_hi, i));
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    c.lo[k] = __shfl_sync(0xffffffffu, lo, (2 * t + k) * 4);
    c.hi[k] = __shfl_sync(0xffffffffu, hi, (2 * t + k) * 4);
  }
  return c;
}

// The queries of a key head as fragments of the eight products over the
// dimensions, fp16 after one power of two per pair; sc: the factors of the
// scores of columns 2t, 2t + 1.
__device__ __forceinline__ void load_queries(const Paged8Args& a, const Columns& c, int kvh, int t,
                                             uint32_t (&qf)[8][2], float (&sc)[2]) {
  const __nv_bfloat16* q = c.q + (int64_t)kvh * a.group * 128;
  uint4 raw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    raw[i] = c.in ? *reinterpret_cast<const uint4*>(q + (i >> 1) * 64 + (i & 1) * 8)
                  : make_uint4(0u, 0u, 0u, 0u);
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = word(raw[i], j);
      amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(x << 16)), fabsf(__uint_as_float(x & 0xffff0000u))));
    }
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const int sh = fp16_shift(amax);
  const float f = exp2_int(sh), mine = a.scale_log2 * exp2_int(-sh);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = word(raw[i], j);
      // 8 dimensions = words of two products: (i, j) -> product 2i + j/2, register j % 2
      qf[2 * i + (j >> 1)][j & 1] =
          pack_f16x2(__uint_as_float(x << 16) * f, __uint_as_float(x & 0xffff0000u) * f);
    }
  sc[0] = __shfl_sync(0xffffffffu, mine, 8 * t);
  sc[1] = __shfl_sync(0xffffffffu, mine, 8 * t + 4);
}

// Running softmax of a lane's two columns and their output.
struct Running {
  float m[2], n[2], l[2], o[8][4];
};

__device__ __forceinline__ void start(Running& R) {
#pragma unroll
  for (int d = 0; d < 8; ++d) R.o[d][0] = R.o[d][1] = R.o[d][2] = R.o[d][3] = 0.f;
  R.m[0] = R.m[1] = R.n[0] = R.n[1] = -INFINITY;
  R.l[0] = R.l[1] = 0.f;
}

// Scores of 16 * MB keys to weights (operand fragments) and their sums.  key0:
// key of the lane's result row g of product 0; product m is + 4 m, row g + 8 + 2.
template <int MB>
__device__ __forceinline__ void weigh(Running& R, float (&s)[MB][4], const Columns& c,
                                      const float (&sc)[2], float ks, float vs, bool whole, bool have,
                                      int key0, uint32_t (&pb)[MB][2]) {
  const int ve = scale_log2_of(vs);
  const float vef = (float)ve;
  const float c_ks[2] = {score_factor(sc[0], ks), score_factor(sc[1], ks)};
  float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int k = r & 1;
      float x = fmaf(s[m][r], c_ks[k], vef);
      if (!whole) {
        const int key = key0 + 4 * m + (r & 2);
        x = have && key >= c.lo[k] && key < c.hi[k] ? x : -INFINITY;
      }
      s[m][r] = x;
      mx[k] = fmaxf(mx[k], x);
    }
#pragma unroll
  for (int i = 4; i < 32; i <<= 1) {
    mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], i));
    mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], i));
  }
  float ref[2], factor[2];
  bool grown = false, far[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float top = mx[k] - vef;
    far[k] = far_page(fmaxf(R.m[k], mx[k]), mx[k], fmaxf(R.n[k], top), top);
    grown = grown || far[k] || mx[k] > R.m[k] || top > R.n[k];
  }
  const bool any = __any_sync(0xffffffffu, grown);
  if (any) {
    float alpha[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float m_new = fmaxf(R.m[k], mx[k]), n_new = fmaxf(R.n[k], mx[k] - vef);
      alpha[k] = ex2_approx(R.m[k] - finite_or_0(m_new));
      R.l[k] *= ex2_approx(R.n[k] - finite_or_0(n_new));
      R.m[k] = m_new, R.n[k] = n_new;
    }
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) R.o[d][r] *= alpha[r & 1];
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    ref[k] = finite_or_0(R.m[k]);
    factor[k] = sum_factor(ref[k], vef, finite_or_0(R.n[k]));
  }
  if (any && __any_sync(0xffffffffu, far[0] || far[1])) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (far[k]) {
#pragma unroll
        for (int m = 0; m < MB; ++m)
          R.l[k] += ex2_approx(s[m][k] - vef - R.n[k]) + ex2_approx(s[m][k + 2] - vef - R.n[k]);
        factor[k] = 0.f;
      }
  }
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float p0 = ex2_approx(s[m][2 * e] - ref[0]), p1 = ex2_approx(s[m][2 * e + 1] - ref[1]);
      sum[0] += p0;
      sum[1] += p1;
      pb[m][e] = transpose8x8(pack_f16x2(p0, p1));
    }
  R.l[0] = fmaf(sum[0], factor[0], R.l[0]);
  R.l[1] = fmaf(sum[1], factor[1], R.l[1]);
}

// The lanes' numerators as rows of 128 floats in shared memory, with n, l and the
// factor to the outputs.
__device__ __forceinline__ void spill(Running& R, float (*so)[kPitch], float* sn, float* sl, float* sf,
                                      int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 4; i < 32; i <<= 1) {
    R.l[0] += __shfl_xor_sync(0xffffffffu, R.l[0], i);
    R.l[1] += __shfl_xor_sync(0xffffffffu, R.l[1], i);
  }
  const OutFactor f[2] = {{R.m[0], R.n[0], R.l[0]}, {R.m[1], R.n[1], R.l[1]}};
  if (__any_sync(0xffffffffu, f[0].b != 1.f || f[1].b != 1.f)) {
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) R.o[d][r] *= f[r & 1].b;
  }
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) so[2 * t + (r & 1)][16 * d + 8 * (r >> 1) + g] = R.o[d][r];
  if (g == 0) {
    sn[2 * t] = R.n[0], sn[2 * t + 1] = R.n[1];
    sl[2 * t] = R.l[0], sl[2 * t + 1] = R.l[1];
    sf[2 * t] = f[0].a, sf[2 * t + 1] = f[1].a;
  }
}

// one pair's output row: 4 dimensions per lane, and its denominator
__device__ __forceinline__ void write_pair(const Paged8Args& a, const Paged8Tile& tl, int rho, int kvh,
                                           int lane, const float (&o)[4], float N, float L) {
  int row, g;
  split_pair(a, rho, row, g);
  const int64_t r = tl.rq.row0 + (int64_t)row;
  const int h = kvh * a.group + g;
  // (written past the caches' reuse: 50.1 us for 880 requests of 3 rows, else 51.6)
  __stcs(reinterpret_cast<uint2*>(a.out + r * a.out_stride + h * 128 + 4 * lane),
         make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])));
  if (a.lse && lane == 0) a.lse[r * a.heads + h] = row_lse(N, L);
}

// The shares of up to 32 parts of a pair's keys in its output, lane s's of part s,
// from the parts' n and l; N and L those of all.
struct Shares {
  float N, L, mine;
  __device__ __forceinline__ Shares(float n, float l) : N(n) {
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) N = fmaxf(N, __shfl_xor_sync(0xffffffffu, N, i));
    mine = l * ex2_approx(n - finite_or_0(N));
    L = mine;
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) L += __shfl_xor_sync(0xffffffffu, L, i);
    mine *= inverse_or_0(L);
  }
};

constexpr int kMinPages = 2 * kWarps;  // of a part at least

// Until the kernel before this one is done, where it was launched beside it.
__device__ __forceinline__ void wait_for_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// What the blocks of no unit do (in front of the short kernel's units, behind the
// long one's): the first of them writes zeros to the rows between q_start's ends
// that no kernel writes, and all wait for the kernel before.  There are such rows
// only where row starts descend or leave the row tensor: those of refused requests
// alone, and of requests whose tiles the large kernel cannot find.  (A block of its
// own: 0.5 us of 51 for 880 requests of 3 rows, where the tiles' warps took 5.7 to do
// it for their own request; in front, since it took 30 us of 168 as the last block of
// 20 000 requests; a function of its own for the registers of the kernels.)
constexpr int kKeptWords = 128;  // 4 096 rows at a time
__device__ __noinline__ void keep_rows(const Paged8Args& a, bool first, uint32_t* covered) {
  const int32_t* qs = a.q_start;
  int bad = qs[0] < 0 || qs[a.n] > a.rows;
  if (first && a.zero_rest) {
#pragma unroll 8
    for (int i = threadIdx.x; i < a.n; i += kWarps * 32) bad |= qs[i + 1] < qs[i];
  }
  bad = __syncthreads_or(bad);
  wait_for_prior();
  if (!bad || !first || !a.zero_rest) return;
  const RowSpan s = row_span(a);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int64_t at = s.first; at < s.end; at += 32 * kKeptWords) {
    for (int i = threadIdx.x; i < kKeptWords; i += blockDim.x) covered[i] = 0u;
    __syncthreads();
    for (int b0 = 32 * warp; b0 < a.n; b0 += 32 * warps) {
      const int b = b0 + lane, row0 = b < a.n ? qs[b] : 0, row1 = b < a.n ? qs[b + 1] : 0;
      bool live = row1 > row0 && s.holds(row0, row1);
      const int pairs = live ? (row1 - row0) * a.group : 0;
      for (unsigned large = __ballot_sync(0xffffffffu, pairs > a.row_limit); large; large &= large - 1) {
        const int of = __ffs(large) - 1;
        const bool found = tiles_found<kPaged8LargeRows>(a, b0 + of, __shfl_sync(0xffffffffu, row0, of),
                                                         __shfl_sync(0xffffffffu, pairs, of));
        if (lane == of) live = found;
      }
      const int64_t from = max((int64_t)row0 - at, (int64_t)0);
      const int64_t to = min((int64_t)row1 - at, (int64_t)32 * kKeptWords);
      for (int64_t w = from / 32; live && w * 32 < to; ++w) {
        const uint32_t below = to >= w * 32 + 32 ? ~0u : (1u << (to - w * 32)) - 1u;
        atomicOr(covered + w, below & (from > w * 32 ? ~0u << (from - w * 32) : ~0u));
      }
    }
    __syncthreads();
    for (int64_t w = warp; w < kKeptWords; w += warps)
      for (uint32_t rest = ~covered[w]; rest; rest &= rest - 1) {
        const int64_t r = at + 32 * w + __ffs(rest) - 1;
        if (r < s.end)
          for (int kvh = 0; kvh < a.kv_heads; ++kvh) zero_row(a, r, kvh, lane);
      }
    __syncthreads();
  }
}

template <int FMT>
__global__ void __launch_bounds__(kWarps * 32, 3) paged8_long_kernel(const __grid_constant__ Paged8Args a) {
  __shared__ __align__(16) float so[kWarps][kRows][kPitch];
  __shared__ __align__(16) uint32_t sq[kWarps][8][32][2];
  __shared__ float sn[kWarps][kRows], sl[kWarps][kRows], sf[kWarps][kRows];
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int unit = (int)blockIdx.x / a.splits, split = (int)blockIdx.x - unit * a.splits.d;
  const int tile = unit / a.kv_heads, kvh = unit - tile * a.kv_heads.d;
  const int b = tile / a.direct, first = tile % a.direct * kRows;
  if (b >= a.n) return keep_rows(a, split == 0, reinterpret_cast<uint32_t*>(so));
  if (a.zero_rest && split == 0)
    zero_rest(a, kvh, (int64_t)tile * kWarps + w, (int64_t)a.n * a.direct * kWarps, lane);
  // Tiles beyond those the launch counted on (a request of more rows than
  // max_rows said) follow in the same block, their keys in one part.
  for (int rho0 = first;; rho0 += a.direct * kRows) {
    const Paged8Tile tl = small_tile(a, b, rho0, split == 0 && kvh == 0 && threadIdx.x == 0);
    if (!tl.live) return;
    const int parts = rho0 == first ? parts_of<kMinPages>(tl.np, a.splits) : 1;
    if (split >= parts) return;
    const int p_end = tl.p0 + tl.np * (split + 1) / parts;
    int p = tl.p0 + tl.np * split / parts + w;
    Running R;
    start(R);
    if (p < p_end) {
      const int32_t* row = a.table + tl.b * a.table_stride;
      int page = page_at(a, row, p, lane);
      int page_next = p + kWarps < p_end ? page_at(a, row, p + kWarps, lane) : -1;
      const Columns c = columns(a, tl, lane);
      const int key0 = 16 * (g >> 1) + (g & 1);  // key of row g (+ 2: row g + 8) of product m: + 4 m
      // codes of product m: [row g, g + 8][dimension half]
      const auto load_k = [&](uint4 (&kr)[2][2], int m, int pp, int pg) {
        const uint8_t* kp = a.k + ((int64_t)pg * a.kv_heads + kvh) * kPageHeadBytes + t * 16;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = key0 + 4 * m + 2 * e;
          const bool in = pg >= 0 && pp * kPage + key >= tl.lo && pp * kPage + key < tl.hi;
          kr[e][0] = ld_codes(kp + key * 64, in);
          kr[e][1] = ld_codes(kp + kPage * 64 + key * 64, in);
        }
      };
      uint4 kr[4][2][2];
#pragma unroll
      for (int m = 0; m < 4; ++m) load_k(kr[m], m, p, page);
      float sc[2];
      {  // the query fragments wait in shared memory: a lane reads back its own
        uint32_t qf[8][2];
        load_queries(a, c, kvh, t, qf, sc);
#pragma unroll
        for (int i = 0; i < 8; ++i) sq[w][i][lane][0] = qf[i][0], sq[w][i][lane][1] = qf[i][1];
      }
      const uint32_t q_at = smem_u32(&sq[w][0][lane][0]);
      for (; p < p_end; p += kWarps) {
        const int page_now = page;
        page = page_next;
        page_next = p + 2 * kWarps < p_end ? page_at(a, row, p + 2 * kWarps, lane) : -1;
        const bool have = page_now >= 0;
        const int64_t at = have ? (int64_t)page_now * a.kv_heads + kvh : 0;
        const float ks = a.k_scale[at], vs = a.v_scale[at];
        const uint8_t* vp = a.v + at * kPageHeadBytes + t * 16 + g * kPage;
        const bool v_in = have && p * kPage + 16 * t + 15 >= tl.lo && p * kPage + 16 * t < tl.hi;
        // the values' codes take the registers that the keys' leave
        uint4 vr[8][2];
        float s[4][4];
        // two products' chains alternate
#pragma unroll
        for (int m = 0; m < 4; m += 2) {
#pragma unroll
          for (int q = m; q < m + 2; ++q) s[q][0] = s[q][1] = s[q][2] = s[q][3] = 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint2 qf = ld_shared2(q_at + (4 * h + i) * 256);
#pragma unroll
              for (int q = m; q < m + 2; ++q) {
                uint32_t a0, a1, a2, a3;
                decode4<FMT>(word(kr[q][0][h], i), a0, a2);
                decode4<FMT>(word(kr[q][1][h], i), a1, a3);
                mma_f16(s[q], a0, a1, a2, a3, qf.x, qf.y);
              }
            }
#pragma unroll
          for (int d = 2 * m; d < 2 * m + 4; ++d)
#pragma unroll
            for (int e = 0; e < 2; ++e) vr[d][e] = ld_codes(vp + (16 * d + 8 * e) * kPage, v_in);
        }
        const bool whole = have && p * kPage >= c.all_lo && (p + 1) * kPage <= c.all_hi;
        uint32_t pb[4][2];
        weigh<4>(R, s, c, sc, ks, vs, whole, have, p * kPage + key0, pb);
#pragma unroll
        for (int d = 0; d < 8; d += 2) {
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int q = d; q < d + 2; ++q) {
              uint32_t a0, a1, a2, a3;
              decode4<FMT>(word(vr[q][0], m), a0, a2);
              decode4<FMT>(word(vr[q][1], m), a1, a3);
              mma_f16(R.o[q], a0, a1, a2, a3, pb[m][0], pb[m][1]);
            }
          // the next page's keys (zeros behind the last) take the values' registers
          load_k(kr[d >> 1], d >> 1, p + kWarps, page);
        }
      }
    }
    spill(R, so[w], sn[w], sl[w], sf[w], lane);
    __syncthreads();
    for (int r = w; r < kRows && tl.rho0 + r < tl.pairs; r += kWarps) {
      float N = -INFINITY;
#pragma unroll
      for (int q = 0; q < kWarps; ++q) N = fmaxf(N, sn[q][r]);
      float L = 0.f, acc[4] = {}, share[kWarps];
#pragma unroll
      for (int q = 0; q < kWarps; ++q) {
        share[q] = sl[q][r] * ex2_approx(sn[q][r] - finite_or_0(N));
        L += share[q];
      }
      const float inv = inverse_or_0(L);
#pragma unroll
      for (int q = 0; q < kWarps; ++q) {
        const float f = share[q] * inv * sf[q][r];
        const float4 v = *reinterpret_cast<const float4*>(&so[q][r][4 * lane]);
        acc[0] = fmaf(v.x, f, acc[0]), acc[1] = fmaf(v.y, f, acc[1]);
        acc[2] = fmaf(v.z, f, acc[2]), acc[3] = fmaf(v.w, f, acc[3]);
      }
      if (parts == 1) {
        write_pair(a, tl, tl.rho0 + r, kvh, lane, acc, N, L);
      } else if (!a.cluster) {
        const int64_t at = (int64_t)blockIdx.x * kRows + r;
        *reinterpret_cast<float4*>(a.part_o + at * 128 + 4 * lane) =
            make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (lane == 0) *reinterpret_cast<float2*>(a.part_nl + at * 2) = make_float2(N, L);
      } else {  // the block's result takes the place of its first warp's
        *reinterpret_cast<float4*>(&so[0][r][4 * lane]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        __syncwarp();
        if (lane == 0) sn[0][r] = N, sl[0][r] = L;
      }
    }
    if (parts == 1 || !a.cluster) {
      __syncthreads();
      continue;
    }
    // blocks of the cluster: each joins some of the rows, part by part
    cluster_sync();
    for (int r = split + w * parts; r < kRows && tl.rho0 + r < tl.pairs; r += kWarps * parts) {
      Shares sh(lane < parts ? ld_peer(peer_smem(&sn[0][r], lane)) : -INFINITY,
                lane < parts ? ld_peer(peer_smem(&sl[0][r], lane)) : 0.f);
      float acc[4] = {};
      for (int s = 0; s < parts; ++s) {
        const float f = __shfl_sync(0xffffffffu, sh.mine, s);
        const float4 v = ld_peer4(peer_smem(&so[0][r][4 * lane], s));
        acc[0] = fmaf(v.x, f, acc[0]), acc[1] = fmaf(v.y, f, acc[1]);
        acc[2] = fmaf(v.z, f, acc[2]), acc[3] = fmaf(v.w, f, acc[3]);
      }
      write_pair(a, tl, tl.rho0 + r, kvh, lane, acc, sh.N, sh.L);
    }
    cluster_sync();  // nobody leaves while its rows are read
  }
}

// Codes that no other warp reads: past the L1 cache (880 requests of 3 rows: 51.7
// us, with it 55.0).
__device__ __forceinline__ uint4 ld_once(const uint8_t* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.b32 {%0,%1,%2,%3}, [%4];"
      : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
      : "l"(p));
  return v;
}
__device__ __forceinline__ void ld_words(const uint8_t* p, uint32_t (&w)[2]) {
  asm("ld.global.nc.L1::no_allocate.v2.b32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
}
__device__ __forceinline__ void ld_words(const uint8_t* p, uint32_t (&w)[1]) {
  asm("ld.global.nc.L1::no_allocate.b32 %0, [%1];" : "=r"(w[0]) : "l"(p));
}

// 16 * MB of a page's keys from token `base` of it.  Keys outside [from, to] of
// the page read the nearest one inside: they are masked.
template <int FMT, int MB>
__device__ __forceinline__ void short_keys(const Paged8Args& a, const Columns& c, Running& R,
                                           const uint32_t (&qf)[8][2], const float (&sc)[2], int64_t at,
                                           int page_key, int base, int from, int to, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const uint8_t* kp = a.k + at * kPageHeadBytes + t * 16;
  const uint8_t* vp = a.v + at * kPageHeadBytes + g * kPage + base + 4 * MB * t;
  const float ks = a.k_scale[at], vs = a.v_scale[at];
  const int key0 = base + 4 * MB * (g >> 1) + (g & 1);
  uint4 kr[MB][2][2];
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int key = min(max(key0 + 4 * m + 2 * e, from), to);
      kr[m][e][0] = ld_once(kp + key * 64);
      kr[m][e][1] = ld_once(kp + kPage * 64 + key * 64);
    }
  uint32_t vw[8][2][MB];
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int e = 0; e < 2; ++e) ld_words(vp + (16 * d + 8 * e) * kPage, vw[d][e]);
  float s[MB][4];
#pragma unroll
  for (int m = 0; m < MB; ++m) s[m][0] = s[m][1] = s[m][2] = s[m][3] = 0.f;
  // the products of different keys are independent: they alternate
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int m = 0; m < MB; ++m) {
        uint32_t a0, a1, a2, a3;
        decode4<FMT>(word(kr[m][0][h], i), a0, a2);
        decode4<FMT>(word(kr[m][1][h], i), a1, a3);
        mma_f16(s[m], a0, a1, a2, a3, qf[4 * h + i][0], qf[4 * h + i][1]);
      }
  const bool whole = page_key + base >= c.all_lo && page_key + base + 16 * MB <= c.all_hi;
  uint32_t pb[MB][2];
  weigh<MB>(R, s, c, sc, ks, vs, whole, true, page_key + key0, pb);
#pragma unroll
  for (int m = 0; m < MB; ++m)
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      uint32_t a0, a1, a2, a3;
      decode4<FMT>(vw[d][0][m], a0, a2);
      decode4<FMT>(vw[d][1][m], a1, a3);
      mma_f16(R.o[d], a0, a1, a2, a3, pb[m][0], pb[m][1]);
    }
}

template <int FMT>
__global__ void __launch_bounds__(kWarps * 32, 4) paged8_short_kernel(const __grid_constant__ Paged8Args a, int units) {
  __shared__ __align__(16) float so[kWarps][kRows][kPitch];
  __shared__ float sn[kWarps][kRows], sl[kWarps][kRows], sf[kWarps][kRows];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if ((int)blockIdx.x < a.keep) return keep_rows(a, true, reinterpret_cast<uint32_t*>(so));
  const int unit = ((int)blockIdx.x - a.keep) * kWarps + w;
  if (unit >= units) return;
  const int tile = unit / a.kv_heads, kvh = unit - tile * a.kv_heads.d;
  const int b = tile / a.direct;
  if (a.zero_rest) zero_rest(a, kvh, tile, (int64_t)a.n * a.direct, lane);
  for (int rho0 = tile % a.direct * kRows;; rho0 += a.direct * kRows) {
    const Paged8Tile tl = small_tile(a, b, rho0, kvh == 0 && lane == 0);
    if (!tl.live) return;
    const Columns c = columns(a, tl, lane);
    const int32_t* row = a.table + tl.b * a.table_stride;
    Running R;
    start(R);
    uint32_t qf[8][2];
    float sc[2];
    load_queries(a, c, kvh, lane & 3, qf, sc);
    for (int p = tl.p0; p < tl.p0 + tl.np; ++p) {
      const int page = page_at(a, row, p, lane);
      if (page < 0) continue;
      const int64_t at = (int64_t)page * a.kv_heads + kvh;
      const int from = max(tl.lo - p * kPage, 0), to = min(tl.hi - p * kPage, kPage) - 1;
      for (int base = from & ~15; base <= to; base += 32) {
        if (to - base < 16)
          short_keys<FMT, 1>(a, c, R, qf, sc, at, p * kPage, base, from, to, lane);
        else
          short_keys<FMT, 2>(a, c, R, qf, sc, at, p * kPage, base, from, to, lane);
      }
    }
    spill(R, so[w], sn[w], sl[w], sf[w], lane);
    __syncwarp();
    for (int r = 0; r < kRows && tl.rho0 + r < tl.pairs; ++r) {
      const float4 v = *reinterpret_cast<const float4*>(&so[w][r][4 * lane]);
      const float f = sf[w][r], acc[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
      write_pair(a, tl, tl.rho0 + r, kvh, lane, acc, sn[w][r], sl[w][r]);
    }
    __syncwarp();
  }
}

// The parts of a tile's keys joined in split order; one warp per (row, head)
// pair.  The large kernel numbers its tiles from the last and counts its parts
// in 128-key tiles.  Launched to overlap the end of the kernel before it (an
// attention kernel, or the other merge), which is done after every kernel
// before it is.
template <int kTileRows>
__global__ void __launch_bounds__(256) paged8_merge_kernel(Paged8Args a, int64_t tiles) {
  constexpr bool kLarge = kTileRows == kPaged8LargeRows;
  constexpr int kGroups = kTileRows / 8;
  const int lane = threadIdx.x & 31;
  const int unit = blockIdx.x / kGroups;  // (tile, key head) as its kernel numbers them
  const int r = (int)(blockIdx.x % kGroups) * 8 + (threadIdx.x >> 5);
  const int tile = unit / a.kv_heads, kvh = unit - tile * a.kv_heads.d;
  const Paged8Tile tl = kLarge ? paged8_tile<kTileRows>(a, tiles - 1 - tile, false)
                               : small_tile(a, tile / a.direct, tile % a.direct * kRows, false);
  wait_for_prior();
  if (!tl.live || (kLarge && tl.pairs <= a.row_limit)) return;
  const int parts = kLarge ? parts_of<kPaged8LargeMin>((tl.np + 1) / 2, a.splits)
                           : parts_of<kMinPages>(tl.np, a.splits);
  const int pr = tl.rho0 + r;
  if (parts == 1 || pr >= tl.pairs) return;
  const int64_t at = (int64_t)unit * a.splits * kTileRows + r;
  float2 nl = make_float2(-INFINITY, 0.f);
  if (lane < parts) nl = *reinterpret_cast<const float2*>(a.part_nl + (at + (int64_t)lane * kTileRows) * 2);
  const Shares sh(nl.x, nl.y);
  float acc[4] = {};
#pragma unroll 8
  for (int s = 0; s < parts; ++s) {
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + (at + (int64_t)s * kTileRows) * 128 + 4 * lane);
    const float f = __shfl_sync(0xffffffffu, sh.mine, s);
    acc[0] = fmaf(v.x, f, acc[0]), acc[1] = fmaf(v.y, f, acc[1]);
    acc[2] = fmaf(v.z, f, acc[2]), acc[3] = fmaf(v.w, f, acc[3]);
  }
  write_pair(a, tl, pr, kvh, lane, acc, sh.N, sh.L);
}

// How a call is cut, from the sizes the host knows (the same for every content
// of the device tables).  Requests of up to small_pairs() (row, head) pairs per
// key head run on the small kernels, longer ones on the large one; a call that
// may hold both runs both, each leaving the other's requests.
//
// Per SM and 8 pairs the small kernels take about 0.3 us and 0.25 us a page, the
// large one 11 us and 0.67 us a page for up to 128 pairs (651 x 56 pairs over one
// page, 2 key heads: 101 us on the large kernel): the sides meet at 169 pairs for
// one page, 84 for four, 22 for hundreds.  Pages are those a table row can list.
int small_pairs(int width) { return (int)(8 * (440 + 27 * (int64_t)width) / (12 + 10 * (int64_t)width)); }
constexpr int kShortPages = 4;
constexpr int kMaxCluster = 8;

struct Shape {
  bool small, large;
  int direct, small_splits, large_splits;
  int64_t small_tiles, large_tiles;
  int64_t floats;  // workspace: the small kernel's parts, then the large one's
  int64_t small_floats;
  bool cluster;    // the small kernel's parts are a cluster's
  int limit;       // small_pairs
  bool few_pages;  // the small kernel is the short one
};

// Pages that the rows of a small tile can see between them, as far as the host
// knows: those of a table row, or of a window's frames and the rows' own block.
int reach_of(int width, int frame, int block, int window) {
  if (window < 0 || block == 0) return width;
  const int64_t tokens = ((int64_t)block + window) * frame + kRows;
  return (int)std::min<int64_t>(width, (tokens + kPage - 1) / kPage + 1);
}

int clamp_int(int64_t v, int64_t lo, int64_t hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }

Shape shape_of(int64_t rows, int group, int kv_heads, int n, int width, int max_rows) {
  Shape s = {};
  const int64_t most = max_rows > 0 && max_rows < rows ? max_rows : rows;
  const int64_t some = n < rows ? n : rows;  // requests that can have rows
  s.large_splits = 1;
  s.limit = small_pairs(width);
  // all of it on the small kernels where that takes no longer than one CTA of the
  // large one, its keys in parts of 16 pages (15 requests of 19 rows over two pages,
  // 24 heads to 3: 6.8 us against 12.9; 3 of 24 over 2 000 tokens, 16 heads to 2:
  // 16.4 against 42.6)
  const int64_t all = ((rows * group + kRows - 1) / kRows + some) * kv_heads;  // tiles at most
  if (n > 0 && all * (30 + 25 * (int64_t)width) <= 148 * (1200 + 67 * (int64_t)std::min(width, 16)))
    s.limit = INT32_MAX;
  s.small = n > 0 && (most * group <= s.limit || n > 1);
  s.large = n == 0 || most * group > s.limit;
  if (s.small) {
    // (beside the large kernel most requests may be its own: two tiles each, the
    // others in turn; and where max_rows says little, four waves of blocks' worth)
    s.direct = s.large ? 2
                       : (int)std::min<int64_t>((most * group + kRows - 1) / kRows,
                                                std::max<int64_t>(4 * 148 * 3 / ((int64_t)n * kv_heads), 2));
    s.small_tiles = (int64_t)n * s.direct;
    s.small_splits = 1;
    s.few_pages = width <= kShortPages;
    if (!s.few_pages) {
      // one wave of blocks (3 per SM) with 2 pages per warp at least, or four
      // waves, which even out unequal lengths, with 4
      constexpr int kWave = 148 * 3;
      const int64_t work = some * s.direct * kv_heads;
      const int64_t one = std::min<int64_t>(kWave / work, width / kMinPages);
      const int64_t four = std::min<int64_t>(4 * kWave / work, width / (2 * kMinPages));
      // (requests without rows have places in the workspace too: 68 MB of it at most)
      s.small_splits =
          clamp_int(std::max(one, four), 1, clamp_int((1 << 14) / (s.small_tiles * kv_heads), 1, 32));
      if (s.small_splits > 1 && s.small_splits < 2 * kMaxCluster &&
          work * std::min(s.small_splits, kMaxCluster) <= kWave) {
        s.cluster = true;
        while (s.small_splits > kMaxCluster || (s.small_splits & (s.small_splits - 1)))
          --s.small_splits;  // the power of two below, up to the portable cluster size
      }
    }
    if (s.small_splits > 1 && !s.cluster)
      s.small_floats = s.small_tiles * kv_heads * s.small_splits * kRows * 130;
  }
  if (s.large) {
    s.large_tiles = paged8_tiles<kPaged8LargeRows>(rows, group, n);
    // tiles that are likely there: every request has one
    const int64_t full = (rows * group + kPaged8LargeRows - 1) / kPaged8LargeRows;
    const int64_t work = std::max<int64_t>({full, some, 1}) * kv_heads;
    s.large_splits = clamp_int(148 / work, 1, clamp_int(width / (2 * kPaged8LargeMin), 1, 16));
  }
  s.floats = s.small_floats;
  if (s.large_splits > 1)
    s.floats += s.large_tiles * kv_heads * s.large_splits * kPaged8LargeRows * 130;
  return s;
}

template <int kTileRows>
int launch_merge(const Paged8Args& a, int64_t tiles, cudaStream_t st) {
  const int64_t blocks = tiles * a.kv_heads * (kTileRows / 8);
  if (blocks > INT32_MAX) {
    set_error(HIER_EVALUE, "too many rows, requests and heads");
    return HIER_EVALUE;
  }
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  HIER_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged8_merge_kernel<kTileRows>, a, tiles),
                  "paged8_merge_kernel launch");
  return HIER_OK;
}

// beside: on the stream after the large kernel, without waiting for it (its
// requests are others, and its blocks leave SMs idle: few of them, or the last
// wave's).  The blocks of one unit more (keep_rows) do wait for it, so that what
// follows on the stream finds both done.
int launch_small(Paged8Args a, int format, int64_t tiles, bool few_pages, bool beside,
                 cudaStream_t st) {
  const int64_t units = tiles * a.kv_heads * a.splits;
  a.keep = beside || a.zero_rest;
  if (units > INT32_MAX - 2 * kWarps * a.splits) {
    set_error(HIER_EVALUE, "too many rows, requests and heads");
    return HIER_EVALUE;
  }
  cudaLaunchAttribute attrs[2] = {};
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kWarps * 32);
  cfg.stream = st;
  cfg.attrs = attrs;
  if (beside) {
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  if (few_pages) {
    auto* kernel = format == P8_INT8 ? paged8_short_kernel<P8_INT8> : paged8_short_kernel<P8_E4M3>;
    cfg.gridDim = dim3((unsigned)((units + kWarps - 1) / kWarps + a.keep));
    HIER_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, (int)units), "paged8_short_kernel launch");
    return HIER_OK;
  }
  auto* kernel = format == P8_INT8 ? paged8_long_kernel<P8_INT8> : paged8_long_kernel<P8_E4M3>;
  if (a.cluster) {
    cudaLaunchAttribute& dim = attrs[cfg.numAttrs++];
    dim.id = cudaLaunchAttributeClusterDimension;
    dim.val.clusterDim.x = a.splits.d;
    dim.val.clusterDim.y = dim.val.clusterDim.z = 1;
  }
  cfg.gridDim = dim3((unsigned)(units + a.keep * a.splits.d));
  HIER_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kernel, a), "paged8_long_kernel launch");
  return a.splits > 1 && !a.cluster ? launch_merge<kPaged8SmallRows>(a, tiles, st) : HIER_OK;
}

}  // namespace

}  // namespace hier

using namespace hier;

namespace {

int check_paged8(int32_t rows, int32_t heads, int32_t kv_heads, int32_t n, int32_t width) {
  if (rows < 0 || heads < 1 || kv_heads < 1 || n < 0 || width < 0) {
    set_error(HIER_EVALUE, "invalid rows=%d, heads=%d, key heads=%d, requests=%d or table width=%d",
              rows, heads, kv_heads, n, width);
    return HIER_EVALUE;
  }
  if (heads % kv_heads) {
    set_error(HIER_EVALUE, "%d query heads are not a multiple of %d key heads", heads, kv_heads);
    return HIER_EVALUE;
  }
  if ((int64_t)rows * (heads / kv_heads) > INT32_MAX || (int64_t)width * kPage > INT32_MAX) {
    set_error(HIER_EVALUE, "rows x heads per key head, or tokens of a table row, pass 2^31");
    return HIER_EVALUE;
  }
  return HIER_OK;
}

}  // namespace

extern "C" int hier_paged8_attn_workspace(int32_t rows, int32_t heads, int32_t kv_heads, int32_t n,
                                          int32_t width, int32_t max_rows, int64_t* floats) {
  clear_error();
  int rc = check_paged8(rows, heads, kv_heads, n, width);
  if (rc) return rc;
  if (!floats) {
    set_error(HIER_EVALUE, "no place for the workspace size");
    return HIER_EVALUE;
  }
  *floats = rows ? shape_of(rows, heads / kv_heads, kv_heads, n, width, max_rows).floats : 0;
  return HIER_OK;
}

extern "C" int hier_paged8_attn(const void* q, int64_t q_stride, int32_t rows, int32_t heads,
                                int32_t kv_heads, int32_t D, int32_t format, const void* k_codes,
                                const void* v_codes, const float* k_scale, const float* v_scale,
                                int32_t n_pages, const int32_t* table, int64_t table_stride,
                                int32_t width, const int32_t* lengths, const int32_t* q_start,
                                int32_t n, int32_t frame, int32_t block, int32_t window,
                                float softmax_scale, int32_t max_rows, void* out,
                                int64_t out_stride, float* lse, int32_t zero_rest,
                                float* workspace, int32_t* status, int32_t* dev_err,
                                void* stream) {
  clear_error();
  int rc = check_paged8(rows, heads, kv_heads, n, width);
  if (rc) return rc;
  if (D != 128) {
    set_error(HIER_ENOTIMPL, "the 8-bit cache's attention supports head_dim=128 only; got %d", D);
    return HIER_ENOTIMPL;
  }
  if (format != P8_INT8 && format != P8_E4M3) {
    set_error(HIER_EVALUE, "cache format must be 0 (int8) or 1 (e4m3); got %d", format);
    return HIER_EVALUE;
  }
  if (n_pages < 1 || table_stride < width || frame < 1 || frame > (1 << 30) || block < 0 ||
      block > (1 << 30) || window == 0 || window > (1 << 30)) {
    set_error(HIER_EVALUE, "invalid pages=%d, table stride=%lld, frame=%d, block=%d or window=%d",
              n_pages, (long long)table_stride, frame, block, window);
    return HIER_EVALUE;
  }
  if (!(softmax_scale > 0.f) || !(softmax_scale < INFINITY)) {
    set_error(HIER_EVALUE, "softmax_scale must be positive and finite, got %g", softmax_scale);
    return HIER_EVALUE;
  }
  if ((reinterpret_cast<uintptr_t>(q) & 15) || q_stride % 8 || (reinterpret_cast<uintptr_t>(out) & 15) ||
      out_stride % 8 || (reinterpret_cast<uintptr_t>(k_codes) & 15) ||
      (reinterpret_cast<uintptr_t>(v_codes) & 15)) {
    set_error(HIER_EVALUE, "rows and codes must be 16-byte aligned with 16-byte row strides");
    return HIER_EVALUE;
  }
  if (rows == 0) return HIER_OK;
  Paged8Args a = {};
  a.q = reinterpret_cast<const __nv_bfloat16*>(q);
  a.q_stride = q_stride;
  a.rows = rows, a.heads = heads, a.kv_heads = divisor(kv_heads), a.group = divisor(heads / kv_heads);
  a.k = reinterpret_cast<const uint8_t*>(k_codes), a.v = reinterpret_cast<const uint8_t*>(v_codes);
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.n_pages = n_pages;
  a.table = table, a.table_stride = table_stride, a.width = width;
  a.lengths = lengths, a.q_start = q_start, a.n = n;
  a.mask.frame = divisor(frame), a.mask.block = divisor(block ? block : 1), a.mask.blocks = block;
  a.mask.window = window;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.out_stride = out_stride;
  a.lse = lse;
  zero_rest = zero_rest == 2 ? 2 * (lse != nullptr) : zero_rest != 0;
  a.status = status;
  a.err = dev_err;
  cudaStream_t st = (cudaStream_t)stream;
  // what the mask leaves of a table row, where that needs no more workspace (350
  // requests of 7 rows over 1 280 tokens, 4 of them seen, 24 heads to 8: 23 us;
  // by the table's 20 pages 108)
  const Shape whole = shape_of(rows, a.group, kv_heads, n, width, max_rows);
  const Shape seen = shape_of(rows, a.group, kv_heads, n, reach_of(width, frame, block, window), max_rows);
  const Shape& s = seen.floats <= whole.floats ? seen : whole;
  if (s.floats > 0 && !workspace) {
    set_error(HIER_EVALUE, "this call needs a workspace (hier_paged8_attn_workspace)");
    return HIER_EVALUE;
  }
  // both kernels: one rule for whose a request is; the rows of no request are the
  // small one's where it runs
  a.row_limit = !s.large ? INT32_MAX : s.small ? s.limit : 0;
  Paged8Args large = a;
  if (s.large) {
    large.zero_rest = s.small ? 0 : zero_rest;
    large.splits = divisor(s.large_splits);
    large.part_o = workspace + s.small_floats;
    large.part_nl = large.part_o + (s.floats - s.small_floats) / 130 * 128;
    rc = paged8_launch_large(large, format, s.large_tiles, st);
    if (rc) return rc;
  }
  if (s.small) {
    a.zero_rest = zero_rest;
    a.direct = divisor(s.direct);
    a.splits = divisor(s.small_splits);
    a.cluster = s.cluster;
    a.part_o = workspace;
    a.part_nl = workspace + s.small_floats / 130 * 128;
    rc = launch_small(a, format, s.small_tiles, s.few_pages, s.large, st);
    if (rc) return rc;
  }
  if (s.large && s.large_splits > 1) rc = launch_merge<kPaged8LargeRows>(large, s.large_tiles, st);
  return rc;
}
