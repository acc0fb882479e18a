// RMSNorm of every head of q and k with the position rotation in the same
// pass, and its backward (sm_100a).
//
// Per head x of D values at position p, with the norm weight w [D] shared by
// the heads of q (or of k):
//   y = R(p) (x * rstd * w),  rstd = rsqrt(mean(x^2) + eps)
// in fp32 with one bf16 rounding at the end; R rotates the pairs (2i, 2i+1) by
// table row p.  Backward, with g the gradient of y, g' = R(p)^T g, xh = x rstd:
//   dx = rstd * (w g' - xh mean(w g' xh)),   dw = sum over rows and heads g' xh.
//
// Memory bound: 4 bytes per value forward, 8 backward.  A head is D/8 lanes of
// 8 values (16 bytes), so a warp holds 32*8/D heads at once and the sum of
// squares is a few shuffles.  A warp takes up to kUnroll such groups of one
// row's heads: their loads are all in flight together (3 KiB per warp), the
// lane's four (cos, sin) pairs are read once per row and are the same for all
// of its heads.  Results are stored past the caches' reuse (written once, 165
// against 183 us).  38 556 rows of 24 + 24 heads of 128: 150 us = 6.3 TB/s, 0.97
// of the measured copy bandwidth (8 groups per warp: 165 us, 4: 162, 2: 200).
// Backward on 9 241 rows of 24 + 8 heads: 46 us = 4.9 TB/s, and 4 us for the
// weights' sums.  DRAM is half busy and so are the issue slots: its 16 warps per SM
// wait for their loads, and then for two sums per head one after the other with no
// load in flight.

#include "common.cuh"

namespace hier {
namespace {

constexpr int kWarps = 8;
constexpr int kUnroll = 6;

struct HeadNormArgs {
  const __nv_bfloat16* x[2];  // q, k
  int64_t x_stride[2];
  int heads[2];
  const void* w[2];
  int w_f32;
  const float2* freqs;
  int64_t freqs_rows;
  const int32_t* positions;  // NULL: row r uses table row r % freqs_rows
  int64_t rows;
  float eps;
  __nv_bfloat16* y[2];
  int64_t y_stride[2];
  const int32_t* out_rows[2];  // output row of row r (NULL: r; < 0: not written)
  int64_t out_total[2];
  int zero_skipped;
  int chunks[2];  // items of a row: groups of kUnroll * heads-per-warp heads
  int* err;
  // backward
  const __nv_bfloat16* g[2];
  int64_t g_stride[2];
  float* part;  // [blocks][D]
};

// Table row of row r: < 0 skips the row.
__device__ __forceinline__ int64_t table_row(const HeadNormArgs& a, int64_t r) {
  if (!a.positions) return (uint32_t)r % (uint32_t)a.freqs_rows;
  const int p = a.positions[r];
  if (p >= a.freqs_rows) {
    if (a.err) atomicCAS(a.err, 0, DEV_BAD_INDEX);
    return -1;
  }
  return p;
}

__device__ __forceinline__ void unpack8(uint4 v, float (&f)[8]) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ void load_weight(const HeadNormArgs& a, int kind, int d, float (&w)[8]) {
  if (a.w_f32) {
    const float* p = reinterpret_cast<const float*>(a.w[kind]) + d;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = p[i];
  } else {
    const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(a.w[kind]) + d;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __bfloat162float(p[i]);
  }
}

template <int LPH>
__device__ __forceinline__ float head_sum(float v) {
#pragma unroll
  for (int o = LPH / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32) head_norm_kernel(HeadNormArgs a) {
  constexpr int LPH = D / 8, HPW = 32 / LPH;
  const int lane = threadIdx.x & 31;
  const int sub = lane / LPH, d = (lane % LPH) * 8;
  const uint32_t per_row = a.chunks[0] + a.chunks[1];
  const uint32_t item = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (item >= (uint32_t)a.rows * per_row) return;
  const int64_t r = item / per_row;
  int c = (int)(item - (uint32_t)r * per_row);
  const int kind = c >= a.chunks[0];
  if (kind) c -= a.chunks[0];
  const int h0 = c * (kUnroll * HPW) + sub, heads = a.heads[kind];
  const __nv_bfloat16* x = a.x[kind] + r * a.x_stride[kind] + d;
  uint4 v[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int h = h0 + u * HPW;
    v[u] = h < heads ? __ldcs(reinterpret_cast<const uint4*>(x + (int64_t)h * D))
                     : make_uint4(0u, 0u, 0u, 0u);
  }
  const int64_t t = table_row(a, r);
  int64_t dst = r;
  if (a.out_rows[kind]) {
    dst = a.out_rows[kind][r];
    if (dst >= a.out_total[kind]) {
      if (a.err) atomicCAS(a.err, 0, DEV_BAD_INDEX);
      dst = -1;
    }
    if (dst < 0) return;  // uniform over the warp
  }
  __nv_bfloat16* y = a.y[kind] + dst * a.y_stride[kind] + d;
  if (t < 0) {
    if (a.zero_skipped) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int h = h0 + u * HPW;
        if (h < heads) *reinterpret_cast<uint4*>(y + (int64_t)h * D) = make_uint4(0u, 0u, 0u, 0u);
      }
    }
    return;
  }
  const float4* fr = reinterpret_cast<const float4*>(a.freqs + t * (D / 2) + d / 2);
  const float4 f0 = fr[0], f1 = fr[1];
  const float cs[4] = {f0.x, f0.z, f1.x, f1.z}, sn[4] = {f0.y, f0.w, f1.y, f1.w};
  float w[8];
  load_weight(a, kind, d, w);
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int h = h0 + u * HPW;
    if (u * HPW + c * (kUnroll * HPW) >= heads) break;  // uniform over the warp
    float f[8];
    unpack8(v[u], f);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
    const float rs = rsqrtf(head_sum<LPH>(ss) * (1.f / D) + a.eps);
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = f[2 * i] * rs * w[2 * i], q = f[2 * i + 1] * rs * w[2 * i + 1];
      o[i] = pack_bf16x2(fmaf(p, cs[i], -q * sn[i]), fmaf(p, sn[i], q * cs[i]));
    }
    if (h < heads)
      __stcs(reinterpret_cast<uint4*>(y + (int64_t)h * D), make_uint4(o[0], o[1], o[2], o[3]));
  }
}

// dw: a block works on q or on k; every lane keeps the sums of its 8 channels
// over the heads it walks.  The block adds its lanes' sums in a fixed order and
// writes one partial row, which head_norm_dw_kernel adds in block order.
constexpr int kBwdUnroll = 4;

template <int D>
__global__ void __launch_bounds__(kWarps * 32, 2) head_norm_bwd_kernel(HeadNormArgs a, int q_blocks) {
  constexpr int LPH = D / 8, HPW = 32 / LPH, kU = kBwdUnroll;
  __shared__ float sums[kWarps][HPW][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / LPH, d = (lane % LPH) * 8;
  const int kind = (int)blockIdx.x >= q_blocks;
  const int block = kind ? blockIdx.x - q_blocks : blockIdx.x;
  const int blocks = kind ? gridDim.x - q_blocks : q_blocks;
  const uint32_t per_row = a.chunks[kind], items = (uint32_t)a.rows * per_row;
  const int heads = a.heads[kind];
  float w[8], acc[8] = {};
  load_weight(a, kind, d, w);
  for (uint32_t item = block * kWarps + warp; item < items; item += blocks * kWarps) {
    const int64_t r = item / per_row;
    const int c = (int)(item - (uint32_t)r * per_row);
    const int h0 = c * (kU * HPW) + sub;
    const __nv_bfloat16* x = a.x[kind] + r * a.x_stride[kind] + d;
    const __nv_bfloat16* g = a.g[kind] + r * a.g_stride[kind] + d;
    __nv_bfloat16* y = a.y[kind] + r * a.y_stride[kind] + d;
    uint4 v[kU], gv[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int h = h0 + u * HPW;
      const bool in = h < heads;
      v[u] = in ? __ldcs(reinterpret_cast<const uint4*>(x + (int64_t)h * D)) : make_uint4(0u, 0u, 0u, 0u);
      gv[u] = in ? __ldcs(reinterpret_cast<const uint4*>(g + (int64_t)h * D)) : make_uint4(0u, 0u, 0u, 0u);
    }
    const int64_t t = table_row(a, r);
    if (t < 0) {  // a row that the forward skipped: no gradient
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        const int h = h0 + u * HPW;
        if (h < heads) *reinterpret_cast<uint4*>(y + (int64_t)h * D) = make_uint4(0u, 0u, 0u, 0u);
      }
      continue;
    }
    const float4* fr = reinterpret_cast<const float4*>(a.freqs + t * (D / 2) + d / 2);
    const float4 f0 = fr[0], f1 = fr[1];
    const float cs[4] = {f0.x, f0.z, f1.x, f1.z}, sn[4] = {f0.y, f0.w, f1.y, f1.w};
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int h = h0 + u * HPW;
      if (u * HPW + c * (kU * HPW) >= heads) break;  // uniform over the warp
      float f[8], q[8];
      unpack8(v[u], f);
      unpack8(gv[u], q);
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss = fmaf(f[i], f[i], ss);
      const float rs = rsqrtf(head_sum<LPH>(ss) * (1.f / D) + a.eps);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float g0 = fmaf(q[2 * i], cs[i], q[2 * i + 1] * sn[i]);
        const float g1 = fmaf(q[2 * i + 1], cs[i], -q[2 * i] * sn[i]);
        f[2 * i] *= rs;
        f[2 * i + 1] *= rs;
        if (h < heads) {  // (lanes without a head: 0 x rsqrt(eps), eps may be 0)
          acc[2 * i] = fmaf(g0, f[2 * i], acc[2 * i]);
          acc[2 * i + 1] = fmaf(g1, f[2 * i + 1], acc[2 * i + 1]);
        }
        q[2 * i] = g0 * w[2 * i];
        q[2 * i + 1] = g1 * w[2 * i + 1];
        dot = fmaf(q[2 * i], f[2 * i], dot);
        dot = fmaf(q[2 * i + 1], f[2 * i + 1], dot);
      }
      dot = head_sum<LPH>(dot) * (1.f / D);
      uint32_t o[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o[i] = pack_bf16x2(rs * fmaf(-f[2 * i], dot, q[2 * i]),
                           rs * fmaf(-f[2 * i + 1], dot, q[2 * i + 1]));
      if (h < heads)
        __stcs(reinterpret_cast<uint4*>(y + (int64_t)h * D), make_uint4(o[0], o[1], o[2], o[3]));
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sums[warp][sub][d + i] = acc[i];
  __syncthreads();
  for (int ch = threadIdx.x; ch < D; ch += blockDim.x) {
    float s = 0.f;
    for (int q = 0; q < kWarps; ++q)
      for (int p = 0; p < HPW; ++p) s += sums[q][p][ch];
    a.part[(int64_t)blockIdx.x * D + ch] = s;
  }
}

// dw[ch] = sum over q's blocks, or over k's, of the partial rows: one warp per
// channel, lanes over the blocks, then a fixed tree.
__global__ void head_norm_dw_kernel(const float* part, int q_blocks, int blocks, int D, int f32, void* dwq,
                                    void* dwk) {
  const int e = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (e >= 2 * D) return;
  const int kind = e >= D, ch = kind ? e - D : e;
  const int from = kind ? q_blocks : 0, to = kind ? blocks : q_blocks;
  float s = 0.f;
  for (int b = from + lane; b < to; b += 32) s += part[(int64_t)b * D + ch];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane) return;
  void* out = kind ? dwk : dwq;
  if (f32)
    reinterpret_cast<float*>(out)[ch] = s;
  else
    reinterpret_cast<__nv_bfloat16*>(out)[ch] = __float2bfloat16_rn(s);
}

constexpr int kMaxBwdBlocks = 148 * 4;

// Blocks of the backward on q and on k: what their items fill, at most
// kMaxBwdBlocks together, shared out by the items.
struct BwdBlocks {
  int q, k;
};
BwdBlocks bwd_blocks(int64_t rows, int hq, int hk, int D) {
  const int per = kBwdUnroll * (256 / D);
  const int64_t iq = rows * ((hq + per - 1) / per), ik = rows * ((hk + per - 1) / per);
  const auto fill = [](int64_t items) { return items < kWarps ? 1 : (items + kWarps - 1) / kWarps; };
  int64_t bq = fill(iq), bk = fill(ik);
  if (bq + bk > kMaxBwdBlocks) {
    bq = kMaxBwdBlocks * iq / (iq + ik);
    if (bq < 1) bq = 1;
    if (bq > kMaxBwdBlocks - 1) bq = kMaxBwdBlocks - 1;
    bk = kMaxBwdBlocks - bq;
  }
  return {(int)bq, (int)bk};
}

bool aligned_rows(const void* p, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && stride % 8 == 0;
}

int check_sizes(int64_t rows, int hq, int hk, int D, int64_t freqs_rows, const void* freqs,
                const void* positions) {
  if (D != 64 && D != 128 && D != 256) {
    set_error(HIER_ENOTIMPL, "the per-head norm supports head_dim 64, 128 and 256; got %d", D);
    return HIER_ENOTIMPL;
  }
  if (rows < 0 || hq < 1 || hk < 1 || hq > 4096 || hk > 4096 || freqs_rows < 1) {
    set_error(HIER_EVALUE, "invalid rows=%lld, heads=%d, key heads=%d or table rows=%lld",
              (long long)rows, hq, hk, (long long)freqs_rows);
    return HIER_EVALUE;
  }
  if (rows * ((hq + 1) / 2 + (hk + 1) / 2) > INT32_MAX || freqs_rows > INT32_MAX) {
    set_error(HIER_EVALUE, "too many rows (%lld) or table rows (%lld)", (long long)rows,
              (long long)freqs_rows);
    return HIER_EVALUE;
  }
  if (!positions && rows % freqs_rows) {
    set_error(HIER_EVALUE, "without positions the %lld table rows must divide the %lld rows",
              (long long)freqs_rows, (long long)rows);
    return HIER_EVALUE;
  }
  if (reinterpret_cast<uintptr_t>(freqs) & 15) {
    set_error(HIER_EVALUE, "the rotation table must be 16-byte aligned");
    return HIER_EVALUE;
  }
  return HIER_OK;
}

}  // namespace
}  // namespace hier

using namespace hier;

extern "C" int hier_head_norm_rope(const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                                   int64_t rows, int32_t hq, int32_t hk, int32_t D, const void* wq,
                                   const void* wk, int32_t w_f32, const float* freqs,
                                   int64_t freqs_rows, const int32_t* positions, float eps,
                                   void* q_out, int64_t qo_stride, const int32_t* q_out_rows,
                                   int64_t q_out_total, void* k_out, int64_t ko_stride,
                                   const int32_t* k_out_rows, int64_t k_out_total,
                                   int32_t zero_skipped, int32_t* dev_err, void* stream) {
  clear_error();
  int rc = check_sizes(rows, hq, hk, D, freqs_rows, freqs, positions);
  if (rc) return rc;
  if (!aligned_rows(q, q_stride) || !aligned_rows(k, k_stride) || !aligned_rows(q_out, qo_stride) ||
      !aligned_rows(k_out, ko_stride)) {
    set_error(HIER_EVALUE, "rows must be 16-byte aligned with 16-byte row strides");
    return HIER_EVALUE;
  }
  if (rows == 0) return HIER_OK;
  HeadNormArgs a = {};
  a.x[0] = reinterpret_cast<const __nv_bfloat16*>(q), a.x[1] = reinterpret_cast<const __nv_bfloat16*>(k);
  a.x_stride[0] = q_stride, a.x_stride[1] = k_stride;
  a.heads[0] = hq, a.heads[1] = hk;
  a.w[0] = wq, a.w[1] = wk;
  a.w_f32 = w_f32;
  a.freqs = reinterpret_cast<const float2*>(freqs);
  a.freqs_rows = freqs_rows;
  a.positions = positions;
  a.rows = rows;
  a.eps = eps;
  a.y[0] = reinterpret_cast<__nv_bfloat16*>(q_out), a.y[1] = reinterpret_cast<__nv_bfloat16*>(k_out);
  a.y_stride[0] = qo_stride, a.y_stride[1] = ko_stride;
  a.out_rows[0] = q_out_rows, a.out_rows[1] = k_out_rows;
  a.out_total[0] = q_out_total, a.out_total[1] = k_out_total;
  a.zero_skipped = zero_skipped;
  a.err = dev_err;
  const int per = kUnroll * (256 / D);
  a.chunks[0] = (hq + per - 1) / per, a.chunks[1] = (hk + per - 1) / per;
  const int64_t blocks = (rows * (a.chunks[0] + a.chunks[1]) + kWarps - 1) / kWarps;
  cudaStream_t st = (cudaStream_t)stream;
  if (D == 64)
    head_norm_kernel<64><<<(unsigned)blocks, kWarps * 32, 0, st>>>(a);
  else if (D == 128)
    head_norm_kernel<128><<<(unsigned)blocks, kWarps * 32, 0, st>>>(a);
  else
    head_norm_kernel<256><<<(unsigned)blocks, kWarps * 32, 0, st>>>(a);
  HIER_CHECK_CUDA(cudaGetLastError(), "head_norm_kernel launch");
  return HIER_OK;
}

extern "C" int hier_head_norm_rope_bwd_partials(int64_t rows, int32_t hq, int32_t hk, int32_t D,
                                                int32_t* blocks) {
  clear_error();
  int rc = check_sizes(rows, hq, hk, D, 1, nullptr, nullptr);
  if (rc) return rc;
  if (!blocks) {
    set_error(HIER_EVALUE, "no place for the number of partial rows");
    return HIER_EVALUE;
  }
  const BwdBlocks b = bwd_blocks(rows, hq, hk, D);
  *blocks = b.q + b.k;
  return HIER_OK;
}

extern "C" int hier_head_norm_rope_bwd(const void* q, int64_t q_stride, const void* k,
                                       int64_t k_stride, int64_t rows, int32_t hq, int32_t hk,
                                       int32_t D, const void* wq, const void* wk, int32_t w_f32,
                                       const float* freqs, int64_t freqs_rows,
                                       const int32_t* positions, float eps, const void* gq,
                                       int64_t gq_stride, const void* gk, int64_t gk_stride,
                                       void* dq, int64_t dq_stride, void* dk, int64_t dk_stride,
                                       float* partials, int32_t blocks, void* dwq, void* dwk,
                                       int32_t* dev_err, void* stream) {
  clear_error();
  int rc = check_sizes(rows, hq, hk, D, freqs_rows, freqs, positions);
  if (rc) return rc;
  if (!aligned_rows(q, q_stride) || !aligned_rows(k, k_stride) || !aligned_rows(gq, gq_stride) ||
      !aligned_rows(gk, gk_stride) || !aligned_rows(dq, dq_stride) || !aligned_rows(dk, dk_stride)) {
    set_error(HIER_EVALUE, "rows must be 16-byte aligned with 16-byte row strides");
    return HIER_EVALUE;
  }
  const BwdBlocks b = bwd_blocks(rows, hq, hk, D);
  if (blocks != b.q + b.k) {
    set_error(HIER_EVALUE, "partials must have %d blocks; got %d", b.q + b.k, blocks);
    return HIER_EVALUE;
  }
  HeadNormArgs a = {};
  a.x[0] = reinterpret_cast<const __nv_bfloat16*>(q), a.x[1] = reinterpret_cast<const __nv_bfloat16*>(k);
  a.x_stride[0] = q_stride, a.x_stride[1] = k_stride;
  a.heads[0] = hq, a.heads[1] = hk;
  a.w[0] = wq, a.w[1] = wk;
  a.w_f32 = w_f32;
  a.freqs = reinterpret_cast<const float2*>(freqs);
  a.freqs_rows = freqs_rows;
  a.positions = positions;
  a.rows = rows;
  a.eps = eps;
  a.y[0] = reinterpret_cast<__nv_bfloat16*>(dq), a.y[1] = reinterpret_cast<__nv_bfloat16*>(dk);
  a.y_stride[0] = dq_stride, a.y_stride[1] = dk_stride;
  a.g[0] = reinterpret_cast<const __nv_bfloat16*>(gq), a.g[1] = reinterpret_cast<const __nv_bfloat16*>(gk);
  a.g_stride[0] = gq_stride, a.g_stride[1] = gk_stride;
  a.part = partials;
  a.err = dev_err;
  const int per = kBwdUnroll * (256 / D);
  a.chunks[0] = (hq + per - 1) / per, a.chunks[1] = (hk + per - 1) / per;
  cudaStream_t st = (cudaStream_t)stream;
  if (D == 64)
    head_norm_bwd_kernel<64><<<blocks, kWarps * 32, 0, st>>>(a, b.q);
  else if (D == 128)
    head_norm_bwd_kernel<128><<<blocks, kWarps * 32, 0, st>>>(a, b.q);
  else
    head_norm_bwd_kernel<256><<<blocks, kWarps * 32, 0, st>>>(a, b.q);
  HIER_CHECK_CUDA(cudaGetLastError(), "head_norm_bwd_kernel launch");
  head_norm_dw_kernel<<<(2 * D + 7) / 8, 256, 0, st>>>(partials, b.q, blocks, D, w_f32, dwq, dwk);
  HIER_CHECK_CUDA(cudaGetLastError(), "head_norm_dw_kernel launch");
  return HIER_OK;
}
