// 8-bit paged key/value cache: block tables and slot maps from request
// lengths, and the append of new keys and values (sm_100a).

#include "paged8.cuh"

namespace hier {
namespace {

// ---------------------------------------------------------------------------
// Block tables and slot maps
// ---------------------------------------------------------------------------
//
// Request b goes from lengths[b] to lengths[b] + add[b] tokens (add < 0 drops
// its last tokens; -lengths[b] ends it).  Pages it no longer needs go to the
// end of the free list in request order, pages it now needs come off the
// list's end in request order, and its max(add, 0) new tokens become the next
// rows of the call.  One block: a few thousand requests are a few loads per
// thread and one scan, and the list is a single stack anyway.  A step that
// cannot be taken whole (too few free pages or rows, a length outside the
// table) changes nothing and maps no row.

constexpr int kStepThreads = 1024;

struct StepArgs {
  const int32_t* lengths;
  const int32_t* add;
  int n;
  int32_t* table;
  int64_t table_stride;
  int width;
  int32_t* free_pages;
  int capacity;
  const int32_t* free_count;
  int rows;
  int max_add;  // < 0: no limit
  int32_t* lengths_out;
  int32_t* free_count_out;
  int32_t* q_start;
  int32_t* slots;
  int32_t* positions;
  int32_t* status;
};

enum StepStatus : int {
  STEP_NO_PAGES = 1,
  STEP_NO_ROWS = 2,
  STEP_BAD_LENGTH = 4,
  STEP_BAD_ADD = 8,
  STEP_BAD_LIST = 16,
};

struct Sum3 {
  int64_t rows, need, given;
};
__device__ __forceinline__ Sum3 operator+(Sum3 a, Sum3 b) {
  return {a.rows + b.rows, a.need + b.need, a.given + b.given};
}
__device__ __forceinline__ Sum3 shfl_up(Sum3 v, int o) {
  return {__shfl_up_sync(0xffffffffu, v.rows, o), __shfl_up_sync(0xffffffffu, v.need, o),
          __shfl_up_sync(0xffffffffu, v.given, o)};
}

__device__ __forceinline__ int pages_of(int64_t tokens) { return (int)((tokens + kPage - 1) / kPage); }

__device__ __forceinline__ Sum3 step_of(const StepArgs& a, int b, int& bad) {
  const int64_t len = a.lengths[b], add = a.add[b], to = len + add;
  if (len < 0 || len > (int64_t)a.width * kPage || to > (int64_t)a.width * kPage) {
    bad |= STEP_BAD_LENGTH;
    return {0, 0, 0};
  }
  if (to < 0 || (a.max_add >= 0 && add > a.max_add)) {
    bad |= STEP_BAD_ADD;
    return {0, 0, 0};
  }
  const int p0 = pages_of(len), p1 = pages_of(to);
  return {add > 0 ? add : 0, p1 > p0 ? p1 - p0 : 0, p0 > p1 ? p0 - p1 : 0};
}

// slot and position of row r, from the written q_start and table
__device__ __forceinline__ void map_row(const StepArgs& a, int r, int total) {
  int slot = -1, pos = -1;
  if (r < total) {
    int lo = 0, hi = a.n;  // q_start[lo] <= r < q_start[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.q_start[mid] <= r)
        lo = mid;
      else
        hi = mid;
    }
    // the new rows are the last of the request's tokens
    pos = a.lengths_out[lo] - a.q_start[lo + 1] + r;
    slot = a.table[lo * a.table_stride + pos / kPage] * kPage + pos % kPage;
  }
  a.slots[r] = slot;
  a.positions[r] = pos;
}

__global__ void __launch_bounds__(kStepThreads) page_step_kernel(StepArgs a, int map_rows) {
  __shared__ Sum3 warp_sum[32];
  __shared__ int bad_all;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) bad_all = 0;
  const int count = *a.free_count;
  const int per = (a.n + kStepThreads - 1) / kStepThreads;
  const int b0 = min(a.n, tid * per), b1 = min(a.n, b0 + per);
  int bad = 0;
  Sum3 mine = {0, 0, 0};
  for (int b = b0; b < b1; ++b) mine = mine + step_of(a, b, bad);
  Sum3 incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Sum3 up = shfl_up(incl, o);
    if (lane >= o) incl = incl + up;
  }
  if (lane == 31) warp_sum[warp] = incl;
  __syncthreads();
  if (bad) atomicOr(&bad_all, bad);
  Sum3 base = {0, 0, 0}, total = {0, 0, 0};
  for (int w = 0; w < kStepThreads / 32; ++w) {
    if (w == warp) base = total;
    total = total + warp_sum[w];
  }
  __syncthreads();
  bad = bad_all;
  if (count < 0 || count > a.capacity || count + total.given > a.capacity) bad |= STEP_BAD_LIST;
  if (total.need > count + total.given) bad |= STEP_NO_PAGES;
  if (total.rows > a.rows) bad |= STEP_NO_ROWS;
  const Sum3 before = {base.rows + incl.rows - mine.rows, base.need + incl.need - mine.need,
                       base.given + incl.given - mine.given};
  if (tid == 0) {
    *a.status = bad;
    *a.free_count_out = bad ? count : (int)(count + total.given - total.need);
    a.q_start[a.n] = bad ? 0 : (int)total.rows;
  }
  if (bad) {
    for (int b = b0; b < b1; ++b) {
      a.q_start[b] = 0;
      a.lengths_out[b] = a.lengths[b];
    }
    if (map_rows)
      for (int r = tid; r < a.rows; r += kStepThreads) a.slots[r] = a.positions[r] = -1;
    return;
  }
  // given pages first: a page may change hands within the step.  A request
  // with many pages is handled by its whole warp.
#pragma unroll
  for (int phase = 0; phase < 2; ++phase) {
    Sum3 at = before;
    for (int i = 0; i < per; ++i) {
      const int b = b0 + i;
      Sum3 s = {0, 0, 0};
      int p0 = 0, p1 = 0, dummy = 0;
      if (b < b1) {
        s = step_of(a, b, dummy);
        p0 = pages_of(a.lengths[b]);
        p1 = pages_of((int64_t)a.lengths[b] + a.add[b]);
      }
      const int n = phase == 0 ? (int)s.given : (int)s.need;
      const int from = phase == 0 ? p1 : p0;
      const int64_t list = phase == 0 ? count + at.given : count + total.given - 1 - at.need;
      constexpr int kAlone = 4;
      unsigned many = __ballot_sync(0xffffffffu, n > kAlone);
      while (many) {
        const int src = __ffs(many) - 1;
        many &= many - 1;
        const int nb = __shfl_sync(0xffffffffu, b, src), nn = __shfl_sync(0xffffffffu, n, src);
        const int nf = __shfl_sync(0xffffffffu, from, src);
        const int64_t nl = __shfl_sync(0xffffffffu, list, src);
        for (int j = lane; j < nn; j += 32) {
          int32_t* cell = a.table + nb * a.table_stride + nf + j;
          if (phase == 0)
            a.free_pages[nl + j] = *cell;
          else
            *cell = a.free_pages[nl - j];
        }
      }
      if (n <= kAlone)
        for (int j = 0; j < n; ++j) {
          int32_t* cell = a.table + b * a.table_stride + from + j;
          if (phase == 0)
            a.free_pages[list + j] = *cell;
          else
            *cell = a.free_pages[list - j];
        }
      at = at + s;
    }
    __syncthreads();
  }
  // lengths_out may be lengths itself: each thread reads its own before it writes
  Sum3 at = before;
  for (int b = b0; b < b1; ++b) {
    int dummy = 0;
    const Sum3 s = step_of(a, b, dummy);
    a.q_start[b] = (int)at.rows;
    a.lengths_out[b] = a.lengths[b] + a.add[b];
    at = at + s;
  }
  if (!map_rows) return;
  __syncthreads();
  for (int r = tid; r < a.rows; r += kStepThreads) map_row(a, r, (int)total.rows);
}

__global__ void page_rows_kernel(StepArgs a) {
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r < a.rows) map_row(a, r, a.q_start[a.n]);
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
//
// One warp per (touched page, head, key or value).  Tokens [o, e) of the page
// are new, [0, o) were held before.  Scale: the least power of two s with
// top * s >= max |x| over the new tokens, and at least the page's scale when
// it holds tokens already; codes are x / s rounded to nearest even (the
// division is exact).  When the scale grows the held codes are re-encoded
// under the new one.  Bytes of tokens from e on stay as they are.
//
// Keys: a lane has 4 dimensions of a token (8-byte loads, a row's 256 bytes
// per warp).  Values are stored with the tokens along the row: a lane takes 4
// dimensions of 16 tokens and writes 16 bytes to each of its 4 rows, merged
// with the bytes already there (the warp owns the page and head).  The second
// read of the new rows comes from the caches.

struct AppendArgs {
  const __nv_bfloat16* x[2];  // k, v
  int64_t x_stride[2];
  int rows;
  uint8_t* codes[2];
  float* scale[2];
  int n_pages, heads;
  const int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* lengths;
  const int32_t* q_start;
  int n;
  int64_t items;
  int32_t* status;
};

constexpr int kScaleMin = -100;

template <int FMT>
__device__ __forceinline__ float top_code() {
  return FMT == P8_INT8 ? 127.f : 448.f;
}

// least e >= kScaleMin with top * 2^e >= amax (amax finite, >= 0)
template <int FMT>
__device__ __forceinline__ int scale_exponent(float amax) {
  if (!(amax > 0.f)) return kScaleMin;
  int x;
  const float m = frexpf(amax, &x);  // amax = m 2^x, 0.5 <= m < 1
  const int e = FMT == P8_INT8 ? x - 7 + (m > 127.f / 128.f) : x - 9 + (m > 448.f / 512.f);
  return max(e, kScaleMin);
}

// the code of v (already divided by the scale); NaN becomes 0
template <int FMT>
__device__ __forceinline__ uint32_t encode(float v) {
  if (v != v) return 0u;
  if (FMT == P8_INT8) {
    return (uint32_t)(uint8_t)(int8_t)__float2int_rn(fminf(fmaxf(v, -127.f), 127.f));
  }
  return (uint32_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

template <int FMT>
__device__ __forceinline__ float decode1(uint32_t byte) {
  if (FMT == P8_INT8) return (float)(int8_t)byte;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

template <int FMT>
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
  uint32_t o = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) o |= encode<FMT>(decode1<FMT>((w >> (8 * i)) & 0xffu) * ratio) << (8 * i);
  return o;
}

__device__ __forceinline__ void unpack4(uint2 v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xffff0000u);
  f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xffff0000u);
}

template <int FMT>
__global__ void __launch_bounds__(256) paged8_append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= a.items) return;
  const int head = (int)(item % a.heads);
  const int kv = (int)(item / a.heads % 2);
  const int64_t vp = item / (2 * (int64_t)a.heads);  // virtual page: see paged8_append
  const int32_t* qs = a.q_start;
  const int b = warp_find(a.n, vp, [=](int i) { return (int64_t)(qs[i] >> 6) + 2 * (int64_t)i; });
  const Paged8Request rq = paged8_request(a.q_start, a.lengths, b, a.rows, a.width, true,
                                          lane == 0 && head == 0 ? a.status : nullptr);
  if (!rq.ok || rq.n == 0) return;
  const int begin = rq.held - rq.n;
  const int64_t pg64 = begin / kPage + vp - ((int64_t)(rq.row0 >> 6) + 2 * (int64_t)b);
  if (pg64 < 0 || pg64 * kPage >= rq.held) return;
  const int pg = (int)pg64;
  const int page = a.table[b * a.table_stride + pg];
  if (page < 0 || page >= a.n_pages) {
    if (lane == 0) atomicOr(a.status, P8_BAD_PAGE);
    return;
  }
  const int o = max(0, begin - pg * kPage), e = min(kPage, rq.held - pg * kPage);
  const __nv_bfloat16* x = a.x[kv] + (rq.row0 + (int64_t)(pg * kPage + o - begin)) * a.x_stride[kv] +
                           head * 128 + 4 * lane;  // token o; token t at (t - o) strides
  const int64_t xs = a.x_stride[kv];
  const int64_t at = (int64_t)page * a.heads + head;
  uint8_t* codes = a.codes[kv] + at * kPageHeadBytes;
  // largest finite magnitude of the new tokens
  float amax = 0.f;
  bool odd = false;
#pragma unroll 8
  for (int t = 0; t < e - o; ++t) {
    float f[4];
    unpack4(*reinterpret_cast<const uint2*>(x + t * xs), f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float m = fabsf(f[i]);
      const bool fin = m < INFINITY;
      odd |= !fin;
      amax = fmaxf(amax, fin ? m : 0.f);
    }
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, i));
  if (odd) atomicOr(a.status, P8_NOT_FINITE);
  const float need = exp2_int(scale_exponent<FMT>(amax));
  float* sp = a.scale[kv] + at;
  const float old = o > 0 ? *sp : 0.f;
  const float s = fmaxf(old, need);
  const float inv = 1.f / s;  // exact: s is a power of two
  const bool grown = o > 0 && s > old;
  const float ratio = grown ? old * inv : 1.f;
  __syncwarp();
  if (lane == 0) *sp = s;
  if (kv == 0) {
    if (grown)
      for (int t = lane; t < o * 8; t += 32) {  // 16-byte pieces of the held tokens
        uint4* p = reinterpret_cast<uint4*>(codes + (t & 1 ? 16 : 0) + (t & 2 ? 32 : 0) +
                                            (t & 4 ? kPage * 64 : 0) + (t >> 3) * 64);
        uint4 w = *p;
        w.x = recode4<FMT>(w.x, ratio), w.y = recode4<FMT>(w.y, ratio);
        w.z = recode4<FMT>(w.z, ratio), w.w = recode4<FMT>(w.w, ratio);
        *p = w;
      }
    uint8_t* dst = codes + (lane >> 4) * (kPage * 64) + (lane & 15) * 4;
#pragma unroll 4
    for (int t = o; t < e; ++t) {
      float f[4];
      unpack4(*reinterpret_cast<const uint2*>(x + (t - o) * xs), f);
      uint32_t w = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) w |= encode<FMT>(f[i] * inv) << (8 * i);
      *reinterpret_cast<uint32_t*>(dst + t * 64) = w;
    }
    return;
  }
  for (int t0 = grown ? 0 : (o & ~15); t0 < e; t0 += 16) {
    // bytes of 16 tokens x the lane's 4 dimensions, kept where the token is not new
    uint4 old4[4];
    const bool whole = t0 >= o && t0 + 16 <= e;
    if (!whole) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        old4[i] = *reinterpret_cast<const uint4*>(codes + (4 * lane + i) * kPage + t0);
    }
    uint32_t w[4][4] = {};  // [dimension][4 tokens]
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 v = old4[i];
          uint32_t c = q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w;
          // the tokens of the four that were held before take the new scale
          const int held = min(4, max(0, o - (t0 + 4 * q)));
          const uint32_t hm = held >= 4 ? 0xffffffffu : (1u << (8 * held)) - 1u;
          if (grown && held > 0) c = (recode4<FMT>(c, ratio) & hm) | (c & ~hm);
          w[i][q] = c;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + 4 * q + j;
        if (t < o || t >= e) continue;  // uniform over the warp
        float f[4];
        unpack4(*reinterpret_cast<const uint2*>(x + (t - o) * xs), f);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i][q] = (w[i][q] & ~(0xffu << (8 * j))) | (encode<FMT>(f[i] * inv) << (8 * j));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint4*>(codes + (4 * lane + i) * kPage + t0) =
          make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
  }
}

}  // namespace
}  // namespace hier

using namespace hier;

extern "C" int hier_page_step(const int32_t* lengths, const int32_t* add, int32_t n, int32_t* table,
                              int64_t table_stride, int32_t width, int32_t* free_pages,
                              int32_t capacity, const int32_t* free_count, int32_t rows,
                              int32_t max_add, int32_t* lengths_out, int32_t* free_count_out,
                              int32_t* q_start, int32_t* slots, int32_t* positions,
                              int32_t* status, void* stream) {
  clear_error();
  if (n < 0 || width < 0 || rows < 0 || capacity < 0 || table_stride < width) {
    set_error(HIER_EVALUE, "invalid requests=%d, table width=%d (stride %lld), rows=%d or list=%d", n,
              width, (long long)table_stride, rows, capacity);
    return HIER_EVALUE;
  }
  if ((int64_t)width * kPage > INT32_MAX || (int64_t)capacity * kPage > INT32_MAX) {
    set_error(HIER_EVALUE, "table width %d or page list %d passes 2^31 tokens", width, capacity);
    return HIER_EVALUE;
  }
  StepArgs a = {lengths,    add,  n,       table,       table_stride,   width,   free_pages, capacity,
                free_count, rows, max_add, lengths_out, free_count_out, q_start, slots,      positions,
                status};
  cudaStream_t st = (cudaStream_t)stream;
  // the rows are mapped by the same block up to 8 per thread, beyond that by a
  // grid of their own
  const int inside = rows <= 8 * kStepThreads;
  page_step_kernel<<<1, kStepThreads, 0, st>>>(a, inside);
  HIER_CHECK_CUDA(cudaGetLastError(), "page_step_kernel launch");
  if (!inside) {
    page_rows_kernel<<<(rows + 255) / 256, 256, 0, st>>>(a);
    HIER_CHECK_CUDA(cudaGetLastError(), "page_rows_kernel launch");
  }
  return HIER_OK;
}

extern "C" int hier_paged8_append(const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                                  int32_t rows, int32_t heads, int32_t format, void* k_codes,
                                  void* v_codes, float* k_scale, float* v_scale, int32_t n_pages,
                                  const int32_t* table, int64_t table_stride, int32_t width,
                                  const int32_t* lengths, const int32_t* q_start, int32_t n,
                                  int32_t* status, void* stream) {
  clear_error();
  if (format != P8_INT8 && format != P8_E4M3) {
    set_error(HIER_EVALUE, "cache format must be 0 (int8) or 1 (e4m3); got %d", format);
    return HIER_EVALUE;
  }
  if (rows < 0 || heads < 1 || n_pages < 0 || n < 0 || width < 0 || table_stride < width ||
      (int64_t)width * kPage > INT32_MAX) {
    set_error(HIER_EVALUE, "invalid rows=%d, heads=%d, pages=%d, requests=%d or table width=%d", rows,
              heads, n_pages, n, width);
    return HIER_EVALUE;
  }
  if ((reinterpret_cast<uintptr_t>(k) & 7) || (reinterpret_cast<uintptr_t>(v) & 7) || k_stride % 4 ||
      v_stride % 4 || (reinterpret_cast<uintptr_t>(k_codes) & 15) ||
      (reinterpret_cast<uintptr_t>(v_codes) & 15)) {
    set_error(HIER_EVALUE, "key and value rows must be 8-byte aligned, the codes 16-byte aligned");
    return HIER_EVALUE;
  }
  if (rows == 0 || n == 0) return HIER_OK;
  AppendArgs a = {};
  a.x[0] = reinterpret_cast<const __nv_bfloat16*>(k), a.x[1] = reinterpret_cast<const __nv_bfloat16*>(v);
  a.x_stride[0] = k_stride, a.x_stride[1] = v_stride;
  a.rows = rows;
  a.codes[0] = reinterpret_cast<uint8_t*>(k_codes), a.codes[1] = reinterpret_cast<uint8_t*>(v_codes);
  a.scale[0] = k_scale, a.scale[1] = v_scale;
  a.n_pages = n_pages, a.heads = heads;
  a.table = table, a.table_stride = table_stride, a.width = width;
  a.lengths = lengths, a.q_start = q_start, a.n = n;
  a.status = status;
  // n rows touch at most ceil(n / 64) + 1 pages, so request b's pages fit
  // between q_start[b] / 64 + 2 b and the next request's: the grid needs no
  // count from the device
  const int64_t pages = rows / kPage + 2 * (int64_t)n;
  a.items = pages * heads * 2;
  const int64_t blocks = (a.items + 7) / 8;
  if (blocks > INT32_MAX) {
    set_error(HIER_EVALUE, "too many rows, requests and heads");
    return HIER_EVALUE;
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (format == P8_INT8)
    paged8_append_kernel<P8_INT8><<<(unsigned)blocks, 256, 0, st>>>(a);
  else
    paged8_append_kernel<P8_E4M3><<<(unsigned)blocks, 256, 0, st>>>(a);
  HIER_CHECK_CUDA(cudaGetLastError(), "paged8_append_kernel launch");
  return HIER_OK;
}
