// Attention of a few rows over an 8-bit paged cache (sm_100a), the merge of
// split keys, and the entry point of both attention kernels.
//
// A warp takes 8 (row, head) pairs of one key head and walks pages of 64 keys.
// Bound by the bytes of the cache: the codes go from global memory straight to
// registers (16 bytes per lane, every 128-byte line used whole), are turned
// into fp16 there and fed to m16n8k16 products with the keys (or the value
// dimensions) as rows and the 8 pairs as columns:
//   S^T (keys x pairs) = K Q^T,    O^T (dimensions x pairs) += V^T P^T.
// The page layout gives a lane 16 consecutive codes of the reduction axis; the
// order of the reduction inside a product is free as long as both operands use
// the same one, so no code is moved between lanes.  P^T goes from the layout
// of a result to that of an operand by an 8x8 transpose in the register file.
// While a page's scores are computed its values are in flight, and while its
// values are consumed the next page's keys are.
//
// With few tiles the keys of each are split over blocks (partial outputs in
// fp32 with their maximum and sum, merged in split order by a second kernel)
// and over the four warps of a block (merged in shared memory).

#include <math.h>

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

__device__ __forceinline__ uint32_t word(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

__device__ __forceinline__ uint4 ld_codes(const uint8_t* p, bool in) {
  return in ? __ldg(reinterpret_cast<const uint4*>(p)) : make_uint4(0u, 0u, 0u, 0u);
}

// page of the table entry, or -1 (reported) when it leaves the pool
__device__ __forceinline__ int page_at(const Paged8Args& a, const int32_t* row, int p, int lane) {
  const int page = row[p];
  if (page >= 0 && page < a.n_pages) return page;
  if (lane == 0) atomicOr(a.status, P8_BAD_PAGE);
  return -1;
}

template <int WPU>
constexpr int kMinPages = 2 * WPU;

template <int FMT, int WPU>
__global__ void __launch_bounds__(kWarps * 32, 2) paged8_small_kernel(Paged8Args a, int64_t units) {
  __shared__ __align__(16) float so[kWarps][kRows][kPitch];
  __shared__ float sm[kWarps][kRows], sl[kWarps][kRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int64_t unit = WPU == 1 ? (int64_t)blockIdx.x * kWarps + warp : (int64_t)blockIdx.x;
  const int w = WPU == 1 ? 0 : warp;
  if (unit >= units) return;
  const int split = (int)(unit % a.splits);
  const int kvh = (int)(unit / a.splits % a.kv_heads);
  const int64_t tile_id = unit / ((int64_t)a.splits * a.kv_heads);
  const Paged8Tile tl = paged8_tile<kRows>(a, tile_id, split == 0 && kvh == 0 && lane == 0 && w == 0);
  if (!tl.live) return;
  const int parts = parts_of<kMinPages<WPU>>(tl.np, a.splits);
  if (split >= parts) return;
  if (tl.b == a.n) {
    if (!a.zero_tail) return;
  } else if (tl.pairs > a.row_limit) {
    return;
  }
  // row of this lane's group: a column of the products
  const int rho = tl.rho0 + g;
  const bool in_row = rho < tl.pairs && tl.b < a.n;
  const int qi = rho / a.group, head = kvh * a.group + rho % a.group;
  int lo_g = INT_MAX, hi_g = 0;
  if (in_row) row_keys(a, tl.rq, qi, lo_g, hi_g);
  const int np0 = tl.np ? (int)((int64_t)tl.np * split / parts) : 0;
  const int np1 = tl.np ? (int)((int64_t)tl.np * (split + 1) / parts) : 0;
  float o[8][4] = {};
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  if (np0 < np1) {
    uint32_t qf[8][2];
    float sc_g;
    {
      const __nv_bfloat16* qp = a.q + (tl.rq.row0 + (int64_t)qi) * a.q_stride + head * 128 + 16 * t;
      uint4 raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        raw[i] = in_row ? *reinterpret_cast<const uint4*>(qp + (i >> 1) * 64 + (i & 1) * 8)
                        : make_uint4(0u, 0u, 0u, 0u);
      float amax = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = word(raw[i], j);
          amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(x << 16)),
                                   fabsf(__uint_as_float(x & 0xffff0000u))));
        }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int sh = fp16_shift(amax);
      const float f = exp2_int(sh);
      sc_g = a.scale_log2 * exp2_int(-sh);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = word(raw[i], j);
          // 8 dimensions = words of two products: (i, j) -> product 2i + j/2, register j % 2
          qf[2 * i + (j >> 1)][j & 1] =
              pack_f16x2(__uint_as_float(x << 16) * f, __uint_as_float(x & 0xffff0000u) * f);
        }
    }
    float sc[2];
    int lo[2], hi[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      sc[c] = __shfl_sync(0xffffffffu, sc_g, (2 * t + c) * 4);
      lo[c] = __shfl_sync(0xffffffffu, lo_g, (2 * t + c) * 4);
      hi[c] = __shfl_sync(0xffffffffu, hi_g, (2 * t + c) * 4);
    }
    // keys that every row of the tile sees
    int all_lo = in_row ? lo_g : 0, all_hi = in_row ? hi_g : INT_MAX;
#pragma unroll
    for (int i = 4; i < 32; i <<= 1) {
      all_lo = max(all_lo, __shfl_xor_sync(0xffffffffu, all_lo, i));
      all_hi = min(all_hi, __shfl_xor_sync(0xffffffffu, all_hi, i));
    }
    const int32_t* row = a.table + tl.b * a.table_stride;
    const int key0 = 16 * (g >> 1) + (g & 1);  // key of row g (+ 2: row g + 8) of product m: + 4 m
    uint4 kr[4][2][2];
    const auto load_k = [&](int p, int page) {
      const uint8_t* kp = a.k + ((int64_t)page * a.kv_heads + kvh) * kPageHeadBytes + t * 16;
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = key0 + 4 * m + 2 * e;
          const bool in = page >= 0 && p * kPage + key >= tl.lo && p * kPage + key < tl.hi;
          kr[m][e][0] = ld_codes(kp + key * 64, in);
          kr[m][e][1] = ld_codes(kp + kPage * 64 + key * 64, in);
        }
    };
    int p = tl.p0 + np0 + w;
    const int p_end = tl.p0 + np1;
    int page = -1, page_next = -1;
    if (p < p_end) {
      page = page_at(a, row, p, lane);
      if (p + WPU < p_end) page_next = page_at(a, row, p + WPU, lane);
      load_k(p, page);
    }
    for (; p < p_end; p += WPU) {
      const int page_now = page;
      page = page_next;
      if (p + 2 * WPU < p_end) page_next = page_at(a, row, p + 2 * WPU, lane);
      if (page_now < 0) {
        if (p + WPU < p_end) load_k(p + WPU, page);
        continue;
      }
      const int64_t at = (int64_t)page_now * a.kv_heads + kvh;
      const float ks = a.k_scale[at], vs = a.v_scale[at];
      uint4 vr[8][2];
      {
        const uint8_t* vp = a.v + at * kPageHeadBytes + t * 16;
        const bool in = p * kPage + 16 * t + 15 >= tl.lo && p * kPage + 16 * t < tl.hi;
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
          for (int e = 0; e < 2; ++e) vr[d][e] = ld_codes(vp + (16 * d + 8 * e + g) * kPage, in);
      }
      float s[4][4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        s[m][0] = s[m][1] = s[m][2] = s[m][3] = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t a0, a1, a2, a3;
            decode4<FMT>(word(kr[m][0][h], i), a0, a2);
            decode4<FMT>(word(kr[m][1][h], i), a1, a3);
            mma_f16(s[m], a0, a1, a2, a3, qf[4 * h + i][0], qf[4 * h + i][1]);
          }
      }
      if (p + WPU < p_end) load_k(p + WPU, page);
      const int ve = scale_log2_of(vs);
      const float vef = (float)ve;
      const bool whole = p * kPage >= all_lo && (p + 1) * kPage <= all_hi;
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int c = r & 1;
          float x = fmaf(s[m][r], sc[c] * ks, vef);
          if (!whole) {
            const int key = p * kPage + key0 + 4 * m + (r & 2);
            x = key >= lo[c] && key < hi[c] ? x : -INFINITY;
          }
          s[m][r] = x;
          mx[c] = fmaxf(mx[c], x);
        }
#pragma unroll
      for (int i = 4; i < 32; i <<= 1) {
        mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], i));
        mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], i));
      }
      float ref[2], alpha[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float m_new = fmaxf(m_run[c], mx[c]);
        ref[c] = m_new == -INFINITY ? 0.f : m_new;
        alpha[c] = ex2_approx(m_run[c] - ref[c]);
        m_run[c] = m_new;
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) o[d][r] *= alpha[r & 1];
        l_run[0] *= alpha[0];
        l_run[1] *= alpha[1];
      }
      const float unscale = exp2_int(max(-126, min(126, -ve)));
      float sum[2] = {0.f, 0.f};
      uint32_t pb[4][2];
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p0 = ex2_approx(s[m][2 * e] - ref[0]), p1 = ex2_approx(s[m][2 * e + 1] - ref[1]);
          sum[0] += p0;
          sum[1] += p1;
          pb[m][e] = transpose8x8(pack_f16x2(p0, p1));
        }
      l_run[0] = fmaf(sum[0], unscale, l_run[0]);
      l_run[1] = fmaf(sum[1], unscale, l_run[1]);
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          uint32_t a0, a1, a2, a3;
          decode4<FMT>(word(vr[d][0], m), a0, a2);
          decode4<FMT>(word(vr[d][1], m), a1, a3);
          mma_f16(o[d], a0, a1, a2, a3, pb[m][0], pb[m][1]);
        }
    }
#pragma unroll
    for (int i = 4; i < 32; i <<= 1) {
      l_run[0] += __shfl_xor_sync(0xffffffffu, l_run[0], i);
      l_run[1] += __shfl_xor_sync(0xffffffffu, l_run[1], i);
    }
  }
  // results: rows of 128 through shared memory
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r) so[warp][2 * t + (r & 1)][16 * d + 8 * (r >> 1) + g] = o[d][r];
  if (g == 0) {
    sm[warp][2 * t] = m_run[0], sm[warp][2 * t + 1] = m_run[1];
    sl[warp][2 * t] = l_run[0], sl[warp][2 * t + 1] = l_run[1];
  }
  if (WPU == 1)
    __syncwarp();
  else
    __syncthreads();
  // 8 rows x 32 lanes of 4 dimensions over the unit's warps
  for (int r = w; r < kRows; r += WPU) {
    const int pr = tl.rho0 + r;
    if (pr >= tl.pairs) break;
    float M = -INFINITY;
#pragma unroll
    for (int q = 0; q < WPU; ++q) M = fmaxf(M, sm[WPU == 1 ? warp : q][r]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc[4] = {};
#pragma unroll
    for (int q = 0; q < WPU; ++q) {
      const int src = WPU == 1 ? warp : q;
      const float f = ex2_approx(sm[src][r] - ref);
      L = fmaf(sl[src][r], f, L);
      const float4 v = *reinterpret_cast<const float4*>(&so[src][r][4 * lane]);
      acc[0] = fmaf(v.x, f, acc[0]), acc[1] = fmaf(v.y, f, acc[1]);
      acc[2] = fmaf(v.z, f, acc[2]), acc[3] = fmaf(v.w, f, acc[3]);
    }
    if (parts == 1) {
      const float inv = L > 0.f ? 1.f / L : 0.f;
      const int64_t orow = tl.rq.row0 + (int64_t)(pr / a.group);
      const int oh = kvh * a.group + pr % a.group;
      const uint2 v = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv),
                                 pack_bf16x2(acc[2] * inv, acc[3] * inv));
      *reinterpret_cast<uint2*>(a.out + orow * a.out_stride + oh * 128 + 4 * lane) = v;
      if (a.lse && lane == 0) a.lse[orow * a.heads + oh] = L > 0.f ? M + log2f(L) : -INFINITY;
    } else {
      const int64_t at = unit * kRows + r;
      *reinterpret_cast<float4*>(a.part_o + at * 128 + 4 * lane) =
          make_float4(acc[0], acc[1], acc[2], acc[3]);
      if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(M, L);
    }
  }
}

// The parts of a tile's keys joined in split order; one warp per (row, head)
// pair.  The large kernel numbers its tiles from the last and counts its parts
// in 128-key tiles.
template <int kTileRows>
__global__ void __launch_bounds__(256) paged8_merge_kernel(Paged8Args a, int64_t tiles) {
  constexpr bool kLarge = kTileRows == kPaged8LargeRows;
  constexpr int kGroups = kTileRows / 8;
  const int lane = threadIdx.x & 31;
  const int64_t unit = blockIdx.x / kGroups;  // (tile, key head) as its kernel numbers them
  const int r = (int)(blockIdx.x % kGroups) * 8 + (threadIdx.x >> 5);
  const int kvh = (int)(unit % a.kv_heads);
  const int64_t tile = kLarge ? tiles - 1 - unit / a.kv_heads : unit / a.kv_heads;
  const Paged8Tile tl = paged8_tile<kTileRows>(a, tile, false);
  if (!tl.live || tl.b == a.n || (tl.pairs <= a.row_limit) == kLarge) return;
  const int parts = kLarge ? parts_of<kPaged8LargeMin>((tl.np + 1) / 2, a.splits)
                           : parts_of<kMinPages<4>>(tl.np, a.splits);
  const int pr = tl.rho0 + r;
  if (parts == 1 || pr >= tl.pairs) return;
  const int64_t at = unit * a.splits * kTileRows + r;
  float M = -INFINITY;
  for (int s = 0; s < parts; ++s) M = fmaxf(M, a.part_ml[(at + (int64_t)s * kTileRows) * 2]);
  const float ref = M == -INFINITY ? 0.f : M;
  float L = 0.f, acc[4] = {};
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const int64_t ps = at + (int64_t)s * kTileRows;
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + ps * 2);
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + ps * 128 + 4 * lane);
    const float f = ex2_approx(ml.x - ref);
    L = fmaf(ml.y, f, L);
    acc[0] = fmaf(v.x, f, acc[0]), acc[1] = fmaf(v.y, f, acc[1]);
    acc[2] = fmaf(v.z, f, acc[2]), acc[3] = fmaf(v.w, f, acc[3]);
  }
  const float inv = L > 0.f ? 1.f / L : 0.f;
  const int64_t orow = tl.rq.row0 + (int64_t)(pr / a.group);
  const int oh = kvh * a.group + pr % a.group;
  *reinterpret_cast<uint2*>(a.out + orow * a.out_stride + oh * 128 + 4 * lane) = make_uint2(
      pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  if (a.lse && lane == 0) a.lse[orow * a.heads + oh] = L > 0.f ? M + log2f(L) : -INFINITY;
}

// How a call is cut, from the sizes the host knows (the same for every content
// of the device tables).  Requests of up to kSmallPairs (row, head) pairs per
// key head run on the small kernel, longer ones on the large one; a call that
// may hold both runs both, each leaving the other's requests.
constexpr int kSmallPairs = 16;

struct Shape {
  bool small, large;
  int direct, warps, small_splits, large_splits;
  int64_t small_tiles, large_tiles;
  int64_t floats;  // workspace: the small kernel's parts, then the large one's
  int64_t small_floats;
};

int clamp_int(int64_t v, int64_t lo, int64_t hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }

Shape shape_of(int64_t rows, int group, int kv_heads, int n, int width, int max_rows) {
  Shape s = {};
  const int64_t most = max_rows > 0 && max_rows < rows ? max_rows : rows;
  const int64_t some = n < rows ? n : rows;  // requests that can have rows
  s.small = most * group <= kSmallPairs || n > 1;
  s.large = most * group > kSmallPairs;
  if (s.small) {
    s.direct = s.large ? (kSmallPairs + kRows - 1) / kRows : 0;
    s.small_tiles = s.large ? (int64_t)n * s.direct : paged8_tiles<kRows>(rows, group, n);
    // tiles that are likely there, to size the splits by
    int64_t real = s.large ? some : (rows * group + kRows - 1) / kRows;
    if (real < some) real = some;
    s.warps = width > 4 ? 4 : 1;
    s.small_splits = 1;
    if (s.warps == 4) {
      const int64_t want = (148 * 2 + real * kv_heads - 1) / (real * kv_heads);
      s.small_splits = clamp_int(want, 1, clamp_int(width / kMinPages<4>, 1, 64));
    }
    if (s.small_splits > 1) s.small_floats = s.small_tiles * kv_heads * s.small_splits * kRows * 130;
  }
  if (s.large) {
    s.large_tiles = paged8_tiles<kPaged8LargeRows>(rows, group, n);
    const int64_t real = (rows * group + kPaged8LargeRows - 1) / kPaged8LargeRows;
    const int64_t work = real * kv_heads;
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
  paged8_merge_kernel<kTileRows><<<(unsigned)blocks, 256, 0, st>>>(a, tiles);
  HIER_CHECK_CUDA(cudaGetLastError(), "paged8_merge_kernel launch");
  return HIER_OK;
}

int launch_small(const Paged8Args& a, int format, int warps, int64_t tiles, cudaStream_t st) {
  const int64_t units = tiles * a.kv_heads * a.splits;
  const int64_t blocks = warps == 1 ? (units + kWarps - 1) / kWarps : units;
  if (blocks > INT32_MAX) {
    set_error(HIER_EVALUE, "too many rows, requests and heads");
    return HIER_EVALUE;
  }
  auto* kernel = warps == 1 ? (format == P8_INT8 ? paged8_small_kernel<P8_INT8, 1>
                                                 : paged8_small_kernel<P8_E4M3, 1>)
                            : (format == P8_INT8 ? paged8_small_kernel<P8_INT8, 4>
                                                 : paged8_small_kernel<P8_E4M3, 4>);
  kernel<<<(unsigned)blocks, kWarps * 32, 0, st>>>(a, units);
  HIER_CHECK_CUDA(cudaGetLastError(), "paged8_small_kernel launch");
  return a.splits > 1 ? launch_merge<kPaged8SmallRows>(a, tiles, st) : HIER_OK;
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
                                int64_t out_stride, float* lse, int32_t zero_tail,
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
  if (n_pages < 0 || table_stride < width || frame < 1 || frame > (1 << 30) || block < 0 ||
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
  a.rows = rows, a.heads = heads, a.kv_heads = kv_heads, a.group = heads / kv_heads;
  a.k = reinterpret_cast<const uint8_t*>(k_codes), a.v = reinterpret_cast<const uint8_t*>(v_codes);
  a.k_scale = k_scale, a.v_scale = v_scale;
  a.n_pages = n_pages;
  a.table = table, a.table_stride = table_stride, a.width = width;
  a.lengths = lengths, a.q_start = q_start, a.n = n;
  a.mask.frame = frame, a.mask.block = block, a.mask.window = window;
  a.scale_log2 = softmax_scale * 1.4426950408889634f;
  a.out = reinterpret_cast<__nv_bfloat16*>(out);
  a.out_stride = out_stride;
  a.lse = lse;
  a.status = status;
  a.err = dev_err;
  cudaStream_t st = (cudaStream_t)stream;
  const Shape s = shape_of(rows, a.group, kv_heads, n, width, max_rows);
  if (s.floats > 0 && !workspace) {
    set_error(HIER_EVALUE, "this call needs a workspace (hier_paged8_attn_workspace)");
    return HIER_EVALUE;
  }
  // both kernels: one rule for whose a request is, and the rows behind the last
  // request are the large one's
  a.row_limit = !s.large ? INT32_MAX : s.small ? kSmallPairs : 0;
  if (s.large) {
    a.zero_tail = zero_tail;
    a.splits = s.large_splits;
    a.part_o = workspace + s.small_floats;
    a.part_ml = a.part_o + (s.floats - s.small_floats) / 130 * 128;
    rc = paged8_launch_large(a, format, s.large_tiles, st);
    if (!rc && a.splits > 1) rc = launch_merge<kPaged8LargeRows>(a, s.large_tiles, st);
    if (rc) return rc;
  }
  if (s.small) {
    a.zero_tail = s.large ? 0 : zero_tail;
    a.direct = s.direct;
    a.splits = s.small_splits;
    a.part_o = workspace;
    a.part_ml = workspace + s.small_floats / 130 * 128;
    rc = launch_small(a, format, s.warps, s.small_tiles, st);
  }
  return rc;
}
