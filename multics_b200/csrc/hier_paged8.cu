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
// rows of the call.  One block, or one cluster: the list is a single stack, and
// the requests' places in it and in the rows are one scan.  A step that cannot
// be taken whole (too few free pages or rows, a length outside the table)
// changes nothing and maps no row.
//
// Bound by the launch, the chain of loads (length, list or table cell) and, for
// a kernel that runs once, the fetch of its instructions: four requests of a
// thread at a time, all their cells in flight, took 8.0 us for 4 requests
// against 6.1 (in 32 warps), and 12.2 for 3 520 against 12.4 (in one block).

constexpr int kStepThreads = 512;  // at most, of a block

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

// The last request b in [lo, hi) with q_start[b] <= r, where q_start[lo] <= r.
__device__ __forceinline__ int request_of(const int32_t* q_start, int lo, int hi, int64_t r) {
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (q_start[mid] <= r)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Slot and position of row r of request b, whose rows end at `end`; b < 0: none.
__device__ __forceinline__ void map_row(const StepArgs& a, int64_t r, int b, int end) {
  int slot = -1, pos = -1;
  if (b >= 0) {  // the new rows are the last of the request's tokens
    pos = a.lengths_out[b] - end + (int)r;
    slot = a.table[b * a.table_stride + pos / kPage] * kPage + pos % kPage;
  }
  a.slots[r] = slot;
  a.positions[r] = pos;
}

// The 32 rows from r0 on, by a warp, from the written q_start and table: one
// search for the first row's request; the others' are among the next 32, or
// further where many have no rows.
__device__ __forceinline__ void map_rows(const StepArgs& a, int64_t r0, int total) {
  const int lane = threadIdx.x & 31;
  const int64_t r = r0 + lane;
  const int32_t* qs = a.q_start;
  int b = -1, end = 0;
  if (r0 < total) {
    const int first = warp_find(a.n, r0, [=](int i) { return (int64_t)qs[i]; });
    const int next = qs[min(first + 1 + lane, a.n)];
    b = first;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const int v = __shfl_sync(0xffffffffu, next, i);
      b += v <= r;
      end = v <= r ? end : end ? end : v;
    }
    if (r >= total) {
      b = -1;
    } else if (b == first + 32) {
      b = request_of(qs, b, a.n, r);
      end = qs[b + 1];
    }
  }
  if (r < a.rows) map_row(a, r, b, end);
}

__global__ void __launch_bounds__(kStepThreads) page_step_kernel(StepArgs a, int map_here) {
  __shared__ Sum3 warp_sum[kStepThreads / 32];
  __shared__ Sum3 block_sum, sum_before, sum_all;  // this block's, those of the blocks before it, all
  __shared__ int bad_all;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) bad_all = 0;
  asm volatile("griddepcontrol.launch_dependents;");  // page_rows_kernel
  const int count = *a.free_count;
  const int threads = blockDim.x * gridDim.x, me = blockIdx.x * blockDim.x + tid;
  const int per = (a.n + threads - 1) / threads;
  const int b0 = min(a.n, me * per), b1 = min(a.n, b0 + per);
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
  for (int w = 0; w < (int)blockDim.x / 32; ++w) {
    if (w == warp) base = total;
    total = total + warp_sum[w];
  }
  if (gridDim.x == 1) {
    __syncthreads();
    bad = bad_all;
  } else {
    if (tid == 0) block_sum = total;
    cluster_sync();
    if (tid == 0) {
      Sum3 all = {0, 0, 0};
      int bits = 0;
      for (int r = 0; r < (int)gridDim.x; ++r) {
        if (r == (int)blockIdx.x) sum_before = all;
        const uint32_t at = peer_smem(&block_sum, r);
        all = all + Sum3{ld_peer64(at), ld_peer64(at + 8), ld_peer64(at + 16)};
        bits |= (int)ld_peer32(peer_smem(&bad_all, r));
      }
      sum_all = all;
      warp_sum[0].rows = bits;
    }
    cluster_sync();  // nobody leaves, or changes it, while its sum is read
    total = sum_all;
    base = base + sum_before;
    bad = (int)warp_sum[0].rows;
  }
  if (count < 0 || count > a.capacity || count + total.given > a.capacity) bad |= STEP_BAD_LIST;
  if (total.need > count + total.given) bad |= STEP_NO_PAGES;
  if (total.rows > a.rows) bad |= STEP_NO_ROWS;
  const Sum3 before = {base.rows + incl.rows - mine.rows, base.need + incl.need - mine.need,
                       base.given + incl.given - mine.given};
  if (me == 0) {
    *a.status = bad;
    *a.free_count_out = bad ? count : (int)(count + total.given - total.need);
    a.q_start[a.n] = bad ? 0 : (int)total.rows;
  }
  if (bad) {
    for (int b = b0; b < b1; ++b) {
      a.q_start[b] = 0;
      a.lengths_out[b] = a.lengths[b];
    }
    if (map_here)
      for (int r = me; r < a.rows; r += threads) a.slots[r] = a.positions[r] = -1;
    return;
  }
  const auto sync = [] {
    if (gridDim.x == 1)
      __syncthreads();
    else
      cluster_sync();
  };
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
    sync();
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
  if (!map_here) return;
  sync();
  for (int r = me; r < a.rows; r += threads) {
    const int b = r < total.rows ? request_of(a.q_start, 0, a.n, r) : -1;
    map_row(a, r, b, b < 0 ? 0 : a.q_start[b + 1]);
  }
}

__global__ void page_rows_kernel(StepArgs a) {
  const int64_t r0 = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) & ~(int64_t)31;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (r0 < a.rows) map_rows(a, r0, a.q_start[a.n]);
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
//
// One item per (touched page, head, key or value).  Tokens [o, e) of the page
// are new, [0, o) were held before.  Scale: the least power of two s with
// top * s >= max |x| over the new tokens, and at least the page's scale when
// it holds tokens already; codes are x / s rounded to nearest even (the
// division is exact).  When the scale grows the held codes are re-encoded
// under the new one.  Bytes of tokens from e on stay as they are.
//
// Reads 2 bytes a value and writes one, but is bound by the instructions of its
// conversions and the chain of lookups of a short block: 4
// requests of 660 tokens, 24 heads, e4m3 (48 MB): 13.9 us.
//
// A lane has 4 dimensions of a token (8 bytes), a warp its 128.  Keys are
// written 4 bytes per token; values are stored with the tokens along the row.
//
// Long runs of tokens (paged8_append_pages_kernel): a block per item, 16 tokens
// per warp kept in registers between the maximum and the codes (64 registers, 8
// blocks per SM; the rows are loaded before the page is known), values written
// 16 bytes to each of the lane's 4 rows, merged with the bytes already there
// (nobody else writes the page and head).  Fewer tokens per request
// (paged8_append_rows_kernel): a warp per request, head and key or value, which
// walks the request's touched pages.

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

// Codes of four numbers within the codes' range after their scale (inv: its
// inverse, exact), or infinite where `odd`.  int8: 1.5 * 2^23 added to |v| <= 127
// rounds v to nearest even and leaves it, in two's complement, in the low byte.
template <int FMT>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], float inv, bool odd) {
  if (FMT == P8_INT8) {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = fmaf(x[i], inv, 12582912.f);
    if (odd)
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = fminf(12582912.f + 127.f, fmaxf(12582912.f - 127.f, f[i]));
    const auto q = [](float v) { return __float_as_uint(v); };
    return __byte_perm(__byte_perm(q(f[0]), q(f[1]), 0x0040), __byte_perm(q(f[2]), q(f[3]), 0x0040),
                       0x5410);
  }
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[0] * inv, x[1] * inv), __NV_SATFINITE, __NV_E4M3) |
         (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x[2] * inv, x[3] * inv), __NV_SATFINITE, __NV_E4M3)
             << 16;
}

// 4 bytes of each of 4 words, transposed
__device__ __forceinline__ void transpose_bytes(const uint32_t (&c)[4], uint32_t (&w)[4]) {
  const uint32_t a = __byte_perm(c[0], c[1], 0x5140), b = __byte_perm(c[2], c[3], 0x5140);
  const uint32_t d = __byte_perm(c[0], c[1], 0x7362), e = __byte_perm(c[2], c[3], 0x7362);
  w[0] = __byte_perm(a, b, 0x5410), w[1] = __byte_perm(a, b, 0x7632);
  w[2] = __byte_perm(d, e, 0x5410), w[3] = __byte_perm(d, e, 0x7632);
}

// the bytes [0, n) of a word
__device__ __forceinline__ uint32_t low_bytes(int n) {
  return n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
}

template <int FMT>
__device__ __forceinline__ float decode1(uint32_t byte) {
  if (FMT == P8_INT8) return (float)(int8_t)byte;
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}

template <int FMT>
__device__ __forceinline__ uint32_t recode4(uint32_t w, float ratio) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // (codes that were never written may be anything)
    const float v = decode1<FMT>((w >> (8 * i)) & 0xffu);
    f[i] = v == v ? fmaxf(v, -top_code<FMT>()) : 0.f;
  }
  return encode4<FMT>(f, ratio, false);
}

template <int FMT>
__device__ __forceinline__ uint4 recode16(uint4 w, float ratio) {
  return make_uint4(recode4<FMT>(w.x, ratio), recode4<FMT>(w.y, ratio), recode4<FMT>(w.z, ratio),
                    recode4<FMT>(w.w, ratio));
}

__device__ __forceinline__ void unpack4(uint2 v, float (&f)[4]) {
  f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xffff0000u);
  f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xffff0000u);
}

struct AppendItem {
  const __nv_bfloat16* x;  // the lane's 4 dimensions of token o
  int64_t stride;
  uint8_t* codes;
  int o, e;
};

// rows of the N tokens from t0 on that are new (read once: the codes keep their
// places in the L2 cache, 13.9 us for the case above against 15.9)
template <int N>
__device__ __forceinline__ void load_tokens(const AppendItem& it, int t0, uint2 (&x)[N]) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int t = t0 + j;
    x[j] = t >= it.o && t < it.e ? __ldcs(reinterpret_cast<const uint2*>(it.x + (t - it.o) * it.stride))
                                 : make_uint2(0u, 0u);
  }
}

// largest finite magnitude; odd: something was not finite
template <int N>
__device__ __forceinline__ float largest(const uint2 (&x)[N], bool& odd) {
  // bf16 magnitudes order like their bits, pairs of them at a time
  uint32_t big = 0u;
#pragma unroll
  for (int j = 0; j < N; ++j)
    big = __vmaxu2(big, __vmaxu2(x[j].x & 0x7fff7fffu, x[j].y & 0x7fff7fffu));
  big = max(big << 16, big & 0xffff0000u);
  if (big < 0x7f800000u) return __uint_as_float(big);
  odd = true;
  float amax = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    float f[4];
    unpack4(x[j], f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float m = fabsf(f[i]);
      amax = fmaxf(amax, m < INFINITY ? m : 0.f);
    }
  }
  return amax;
}

// A NaN becomes 0.
template <int N>
__device__ __forceinline__ void drop_nan(uint2 (&x)[N]) {
  const auto word = [](uint32_t w) {
    return ((w & 0x7fffu) > 0x7f80u ? 0u : w & 0xffffu) |
           ((w & 0x7fff0000u) > 0x7f800000u ? 0u : w & 0xffff0000u);
  };
#pragma unroll
  for (int j = 0; j < N; ++j) x[j].x = word(x[j].x), x[j].y = word(x[j].y);
}

// the bytes of N tokens of the lane's 4 value dimensions, 4 or 16 at a time
template <int N>
__device__ __forceinline__ void load_old(const AppendItem& it, int t0, int lane, uint32_t (&old)[4][N / 4]) {
  static_assert(N == 4 || N == 16, "one access to each dimension");
  const bool whole = t0 >= it.o && t0 + N <= it.e;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint8_t* p = it.codes + (4 * lane + i) * kPage + t0;
    if constexpr (N == 16) {
      const uint4 v = whole ? make_uint4(0u, 0u, 0u, 0u) : *reinterpret_cast<const uint4*>(p);
      old[i][0] = v.x, old[i][1] = v.y, old[i][2] = v.z, old[i][3] = v.w;
    } else {
      old[i][0] = whole ? 0u : *reinterpret_cast<const uint32_t*>(p);
    }
  }
}

template <int FMT, int N>
__device__ __forceinline__ void store_keys(const AppendItem& it, int t0, int lane, const uint2 (&x)[N],
                                           float inv, bool odd) {
  uint8_t* dst = it.codes + (lane >> 4) * (kPage * 64) + (lane & 15) * 4;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int t = t0 + j;
    if (t >= it.o && t < it.e) {  // uniform over the warp
      float f[4];
      unpack4(x[j], f);
      *reinterpret_cast<uint32_t*>(dst + t * 64) = encode4<FMT>(f, inv, odd);
    }
  }
}

template <int FMT, int N>
__device__ __forceinline__ void store_values(const AppendItem& it, int t0, int lane, const uint2 (&x)[N],
                                             const uint32_t (&old)[4][N / 4], float inv, bool odd) {
  uint32_t w[4][N / 4];  // [dimension][4 tokens]
#pragma unroll
  for (int q = 0; q < N / 4; ++q) {
    uint32_t c[4], t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[4];
      unpack4(x[4 * q + j], f);
      c[j] = encode4<FMT>(f, inv, odd);
    }
    transpose_bytes(c, t);
    const int at = t0 + 4 * q;
    const uint32_t fresh = low_bytes(it.e - at) & ~low_bytes(it.o - at);  // the new ones of the four
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i][q] = (t[i] & fresh) | (old[i][q] & ~fresh);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint8_t* p = it.codes + (4 * lane + i) * kPage + t0;
    if constexpr (N == 16)
      *reinterpret_cast<uint4*>(p) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
    else
      *reinterpret_cast<uint32_t*>(p) = w[i][0];
  }
}

// The scale of an item: `amax` over the new tokens of the whole item.
template <int FMT>
__device__ __forceinline__ float item_scale(float old_scale, float amax) {
  return fmaxf(old_scale, exp2_int(scale_exponent<FMT>(amax)));
}

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, i));
  return v;
}

// the page of a table entry, or -1 (reported) when it leaves the pool
__device__ __forceinline__ int append_page(const AppendArgs& a, int page, int lane) {
  if (page >= 0 && page < a.n_pages) return page;
  if (lane == 0) atomicOr(a.status, P8_BAD_PAGE);
  return -1;
}

__device__ __forceinline__ AppendItem append_item(const AppendArgs& a, const Paged8Request& rq, int pg,
                                                  int page, int head, int kv, int lane) {
  const int begin = rq.held - rq.n;
  AppendItem it;
  it.o = max(0, begin - pg * kPage), it.e = min(kPage, rq.held - pg * kPage);
  it.stride = a.x_stride[kv];
  it.x = a.x[kv] + (rq.row0 + (int64_t)(pg * kPage + it.o - begin)) * it.stride + head * 128 + 4 * lane;
  it.codes = a.codes[kv] + ((int64_t)page * a.heads + head) * kPageHeadBytes;
  return it;
}

// The held codes of an item, of tokens [from, to) (multiples of 16), under a
// scale that has grown.
template <int FMT>
__device__ __forceinline__ void regrow(const AppendItem& it, int kv, int from, int to, float ratio,
                                       int lane) {
  to = min(to, it.o);
  if (kv) {  // 16 tokens of a dimension at a time; of the last few, the held ones
    for (int t0 = from; t0 < to; t0 += 16)
#pragma unroll 1
      for (int d = lane; d < 128; d += 32) {
        uint4* p = reinterpret_cast<uint4*>(it.codes + d * kPage + t0);
        const uint4 v = *p;
        uint4 w = recode16<FMT>(v, ratio);
        const auto keep = [&](uint32_t& to, uint32_t from, int q) {
          const uint32_t held = low_bytes(it.o - (t0 + 4 * q));
          to = (to & held) | (from & ~held);
        };
        keep(w.x, v.x, 0), keep(w.y, v.y, 1), keep(w.z, v.z, 2), keep(w.w, v.w, 3);
        *p = w;
      }
  } else {
#pragma unroll 1
    for (int t = from * 8 + lane; t < to * 8; t += 32) {  // 16-byte pieces of the held tokens
      uint4* p = reinterpret_cast<uint4*>(it.codes + (t & 3) * 16 + (t & 4 ? kPage * 64 : 0) +
                                          (t >> 3) * 64);
      *p = recode16<FMT>(*p, ratio);
    }
  }
}

template <int FMT>
__global__ void __launch_bounds__(128, 8) paged8_append_pages_kernel(AppendArgs a) {
  __shared__ float most[4];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int part = blockIdx.x / a.heads, head = blockIdx.x - part * a.heads;
  const int kv = part & 1;
  const int64_t vp = part >> 1;  // virtual page: see hier_paged8_append
  const int32_t* qs = a.q_start;
  const int b = warp_find(a.n, vp, [=](int i) { return (int64_t)(qs[i] >> 6) + 2 * (int64_t)i; });
  const Paged8Request rq = paged8_request(a.q_start, a.lengths, b, a.rows, a.width, true,
                                          threadIdx.x == 0 && head == 0 ? a.status : nullptr);
  if (!rq.ok || rq.n == 0) return;
  // (rows in front of the first request have virtual pages too: nobody's)
  const int64_t nth = vp - ((int64_t)(rq.row0 >> 6) + 2 * (int64_t)b);
  const int64_t pg = (rq.held - rq.n) / kPage + nth;
  if (nth < 0 || pg * kPage >= rq.held) return;
  const int entry = a.table[b * a.table_stride + pg];
  AppendItem it = append_item(a, rq, (int)pg, 0, head, kv, lane);
  const int t0 = 16 * warp;  // this warp's tokens
  const bool mine = t0 < it.e && t0 + 16 > it.o;
  uint2 x[16];
  if (mine) load_tokens(it, t0, x);  // in flight before the page is known
  const int page = append_page(a, entry, threadIdx.x);
  if (page < 0) return;
  const int64_t at = (int64_t)page * a.heads;
  it.codes += at * kPageHeadBytes;
  float* sp = a.scale[kv] + at + head;
  const float old_scale = it.o > 0 ? *sp : 0.f;
  float amax = 0.f;
  bool odd = false;
  if (mine) amax = largest(x, odd);
  amax = warp_max(amax);
  odd = __any_sync(0xffffffffu, odd);
  if (odd && lane == 0) atomicOr(a.status, P8_NOT_FINITE);
  if (lane == 0) most[warp] = amax;
  __syncthreads();  // every warp has read the old scale
  const float s = item_scale<FMT>(old_scale, fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])));
  const float inv = 1.f / s;  // exact: s is a power of two
  if (threadIdx.x == 0) *sp = s;
  if (it.o > 0 && s > old_scale) {
    regrow<FMT>(it, kv, t0, t0 + 16, old_scale * inv, lane);
    __syncwarp();  // the new codes go into words that other lanes re-encoded
  }
  if (!mine) return;
  if (odd) drop_nan(x);
  if (kv) {
    uint32_t old[4][4];
    load_old<16>(it, t0, lane, old);
    store_values<FMT, 16>(it, t0, lane, x, old, inv, odd);
  } else {
    store_keys<FMT>(it, t0, lane, x, inv, odd);
  }
}

// N tokens of a page at a time, from a multiple of N on: 1, values written byte
// by byte, or 4 or 16, merged with the bytes that are there.
template <int FMT, int N>
__global__ void __launch_bounds__(128) paged8_append_rows_kernel(AppendArgs a, int units) {
  const int lane = threadIdx.x & 31;
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (unit >= units) return;
  const int part = unit / a.heads, head = unit - part * a.heads;
  const int b = part >> 1, kv = part & 1;
  const Paged8Request rq = paged8_request(a.q_start, a.lengths, b, a.rows, a.width, true,
                                          lane == 0 && head == 0 ? a.status : nullptr);
  if (!rq.ok || rq.n == 0) return;
  for (int pg = (rq.held - rq.n) / kPage; pg * kPage < rq.held; ++pg) {
    const int entry = a.table[b * a.table_stride + pg];
    AppendItem it = append_item(a, rq, pg, 0, head, kv, lane);
    const int first = it.o & -N;
    const bool one = it.e - first <= N;  // the tokens stay in registers
    uint2 x[N];
    if (one) load_tokens(it, first, x);  // in flight before the page is known
    const int page = append_page(a, entry, lane);
    if (page < 0) continue;
    const int64_t at = (int64_t)page * a.heads;
    it.codes += at * kPageHeadBytes;
    float* sp = a.scale[kv] + at + head;
    const float old_scale = it.o > 0 ? *sp : 0.f;
    uint32_t old[4][(N + 3) / 4];
    float amax = 0.f;
    bool odd = false;
    for (int t0 = first; t0 < it.e; t0 += N) {
      if (!one) load_tokens(it, t0, x);
      if constexpr (N > 1) {
        if (kv && one) load_old<N>(it, t0, lane, old);
      }
      amax = fmaxf(amax, largest(x, odd));
    }
    amax = warp_max(amax);
    odd = __any_sync(0xffffffffu, odd);
    if (odd && lane == 0) atomicOr(a.status, P8_NOT_FINITE);
    const float s = item_scale<FMT>(old_scale, amax);
    const float inv = 1.f / s;  // exact: s is a power of two
    if (lane == 0) *sp = s;     // (the warp has read the old one)
    const bool grown = it.o > 0 && s > old_scale;
    if (grown) {
      regrow<FMT>(it, kv, 0, kPage, old_scale * inv, lane);
      __syncwarp();  // the new codes go into words that other lanes re-encoded
    }
    for (int t0 = first; t0 < it.e; t0 += N) {
      if (!one) load_tokens(it, t0, x);
      if (odd) drop_nan(x);
      if (!kv) {
        store_keys<FMT>(it, t0, lane, x, inv, odd);
      } else if constexpr (N > 1) {
        if (!one || grown) load_old<N>(it, t0, lane, old);
        store_values<FMT, N>(it, t0, lane, x, old, inv, odd);
      } else {
        float f[4];
        unpack4(x[0], f);
        const uint32_t c = encode4<FMT>(f, inv, odd);
#pragma unroll
        for (int i = 0; i < 4; ++i) it.codes[(4 * lane + i) * kPage + t0] = (uint8_t)(c >> (8 * i));
      }
    }
  }
}

__global__ void status_take_kernel(int32_t* status, int32_t* bits) { *bits = atomicExch(status, 0); }

}  // namespace
}  // namespace hier

using namespace hier;

extern "C" int hier_status_take(int32_t* status, int32_t* bits, void* stream) {
  clear_error();
  if (!status || !bits) {
    set_error(HIER_EVALUE, "no status word, or no place for its bits");
    return HIER_EVALUE;
  }
  status_take_kernel<<<1, 1, 0, (cudaStream_t)stream>>>(status, bits);
  HIER_CHECK_CUDA(cudaGetLastError(), "status_take_kernel launch");
  return HIER_OK;
}

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
  // Up to 1 024 rows are mapped by the same kernel (a thread's searches hit its L1
  // cache: 4 rows 6.1 us, 32 at a time by a warp 7.7), more by a grid of their own
  // (1 000 requests of 8 rows: 8.2 us against 15.9).  Warps cost their barriers: 4
  // requests take 2.8 us in 4 warps and 6.1 in 32, 500 5.2 in 16.  A cluster shares
  // out the requests of a long list (3 000: 9.7 us, one block 12.8; 1 000: 8.6 and
  // 6.9).
  const int inside = rows <= 1024;
  const int most = inside && rows / 2 > n ? rows / 2 : n;
  const int blocks = n > 1024 ? 8 : 1;
  cudaLaunchAttribute attr = {};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = blocks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(most <= 128 ? 128 : most <= 256 || blocks > 1 ? 256 : kStepThreads);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = blocks > 1;
  HIER_CHECK_CUDA(cudaLaunchKernelEx(&cfg, page_step_kernel, a, inside), "page_step_kernel launch");
  if (!inside) {
    attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3((unsigned)(((int64_t)rows + 255) / 256));
    cfg.blockDim = dim3(256);
    cfg.numAttrs = 1;
    HIER_CHECK_CUDA(cudaLaunchKernelEx(&cfg, page_rows_kernel, a), "page_rows_kernel launch");
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
  if (rows < 0 || heads < 1 || n_pages < 1 || n < 0 || width < 0 || table_stride < width ||
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
  cudaStream_t st = (cudaStream_t)stream;
  // (The mean decides: a prompt beside many single tokens may be walked by a warp
  // per head, its pages one after the other.)
  // A block per page and head where requests bring more than 48 tokens each, or
  // fewer and the machine has room, else a warp per request and head (in us, warps
  // and blocks, of requests x tokens x heads: 100 x 34 x 24 27.7 and 34.0, 200 x
  // 64 x 8 33.2 and 30.5; 30 x 40 x 8 8.1 and 6.4, 100 x 30 x 8 11.4 and 13.4; 20 x
  // 16 x 8 6.5 and 4.8, 12 x 12 x 24 4.2 and 4.9).  n rows touch at most
  // ceil(n / 64) + 1 pages, so request b's pages fit between q_start[b] / 64 + 2 b
  // and the next request's: the grid needs no count from the device.
  const int64_t items = (int64_t)n * heads * 2;
  const bool many = rows > 48 * (int64_t)n || (rows > 16 * (int64_t)n && items <= 148 * 8) ||
                    (rows > 4 * (int64_t)n && items <= 148 * 3);
  const int64_t units = (many ? rows / kPage + 2 * (int64_t)n : (int64_t)n) * heads * 2;
  const int64_t blocks = many ? units : (units + 3) / 4;
  if (units > INT32_MAX - 4) {
    set_error(HIER_EVALUE, "too many rows, requests and heads");
    return HIER_EVALUE;
  }
  if (many) {
    auto* kernel = format == P8_INT8 ? paged8_append_pages_kernel<P8_INT8>
                                     : paged8_append_pages_kernel<P8_E4M3>;
    kernel<<<(unsigned)blocks, 128, 0, st>>>(a);
  } else {
    // (67 requests of one token, 24 heads: 5.5 us by 1 and 6.1 by 4; 115 of 4, 27
    // heads: 7.1 by 4 and 11.4 by 16; of 6 13.3 and 11.6)
    const auto of = [&](auto* one, auto* four, auto* sixteen) {
      return rows <= (int64_t)n ? one : rows <= 4 * (int64_t)n ? four : sixteen;
    };
    auto* kernel = format == P8_INT8
                       ? of(paged8_append_rows_kernel<P8_INT8, 1>, paged8_append_rows_kernel<P8_INT8, 4>,
                            paged8_append_rows_kernel<P8_INT8, 16>)
                       : of(paged8_append_rows_kernel<P8_E4M3, 1>, paged8_append_rows_kernel<P8_E4M3, 4>,
                            paged8_append_rows_kernel<P8_E4M3, 16>);
    kernel<<<(unsigned)blocks, 128, 0, st>>>(a, (int)units);
  }
  HIER_CHECK_CUDA(cudaGetLastError(), "paged8_append launch");
  return HIER_OK;
}
