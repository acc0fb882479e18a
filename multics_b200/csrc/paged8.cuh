// Pages of an 8-bit key/value cache and the ragged rows that read and write
// them: shared by the append and attention kernels.
//
// A page holds 64 tokens of every key head.  One (page, head) is 8 KiB of keys
// and 8 KiB of values, each with one power-of-two float scale:
//   keys    [2][64][64]   dimension half, token, 64 dimensions
//   values  [128][64]     dimension, token
// so that 16 consecutive bytes are 16 dimensions of one key, or 16 tokens of
// one value dimension: the reduction axis of both attention products, which
// is what a lane's matrix fragment and a K-major shared-memory tile both want.
// Codes are int8 (-127..127) or e4m3, both exact in fp16; a power-of-two scale
// keeps every stored value exact in bf16 and makes a scale's growth a shift.
//
// Requests are ragged: request b owns rows q_start[b] .. q_start[b+1] and holds
// lengths[b] tokens, the last of which are those rows'.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace hier {

constexpr int kPage = 64;
constexpr int kPageHeadBytes = kPage * 128;  // one (page, head) of keys or of values
enum Paged8Format : int { P8_INT8 = 0, P8_E4M3 = 1 };

// bits of a cache's status word
enum Paged8Status : int {
  P8_BAD_ROWS = 1,     // row starts leave the row tensor or descend
  P8_BAD_LENGTH = 2,   // a length is below the new rows or beyond the block table
  P8_BAD_PAGE = 4,     // a block table entry leaves the page pool
  P8_NOT_FINITE = 8,   // a NaN or an infinity was to be held
};

// Largest b in [0, n) with base(b) <= i, for ascending base; base(0) <= i.
// The warp samples 32 places at a time, so 1024 requests take two rounds.
template <class F>
__device__ __forceinline__ int warp_find(int n, int64_t i, F base) {
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 31) / 32;
    const int at = lo + min((int)(threadIdx.x & 31) * step, len - 1);
    const unsigned le = __ballot_sync(0xffffffffu, base(at) <= i);
    const int k = 31 - __clz(le | 1u);
    const int from = min(k * step, len - 1);
    lo += from;
    len = min(step, len - from);
  }
  return lo;
}

// shared memory of block `rank` of the cluster, at this block's address p
__device__ __forceinline__ uint32_t peer_smem(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint32_t ld_peer32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ int64_t ld_peer64(uint32_t at) {
  int64_t v;
  asm volatile("ld.shared::cluster.s64 %0, [%1];" : "=l"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float ld_peer(uint32_t at) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_peer4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
// (blocks that have left count as arrived)
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A divisor known to the host: n / d for 0 <= n < 2^31 in three instructions.
struct Divisor {
  int d;
  uint32_t mul, shift;
  __host__ __device__ operator int() const { return d; }
};
inline Divisor divisor(int d) {
  uint32_t s = 0;
  while (s < 31 && (1u << s) < (uint32_t)d) ++s;
  return {d, (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - d)) / d + 1), s};
}
__device__ __forceinline__ int operator/(int n, const Divisor& v) {
  return (int)((__umulhi((uint32_t)n, v.mul) + (uint32_t)n) >> v.shift);
}
__device__ __forceinline__ int operator%(int n, const Divisor& v) { return n - n / v * v.d; }

// What the rows of a call may see: frames of `frame` tokens in causal blocks
// of `block` frames (0: every held key), at most `window` frames back (< 0: no
// limit).  Both ends ascend with the position.
struct Paged8Mask {
  Divisor frame, block;  // (block: 1 where blocks is 0)
  int blocks, window;
  __device__ __forceinline__ int first(int pos) const {
    if (window < 0) return 0;
    const int f = pos / frame;
    return f < window ? 0 : (f - window + 1) * frame.d;
  }
  __device__ __forceinline__ int end(int pos, int held) const {
    if (blocks == 0) return held;
    const int f = pos / frame;
    return (int)min((int64_t)held, (int64_t)(f / block + 1) * block.d * frame.d);
  }
};

// One request's rows and keys, checked against the tensors they index.
struct Paged8Request {
  int row0, n;     // first row, rows
  int held;        // tokens held, the new rows' among them
  bool ok;
};

__device__ __forceinline__ Paged8Request paged8_request(int row0, int row1, int held, int rows,
                                                        int width, bool rows_are_held,
                                                        int32_t* status) {
  Paged8Request r;
  r.row0 = row0;
  r.held = held;
  r.n = row1 - row0;
  int bad = 0;
  if (row0 < 0 || row1 < row0 || row1 > rows) bad |= P8_BAD_ROWS;
  if (held < 0 || held > (int64_t)width * kPage || (rows_are_held && !bad && r.n > held))
    bad |= P8_BAD_LENGTH;
  r.ok = bad == 0;
  if (bad && status) atomicOr(status, bad);
  return r;
}

__device__ __forceinline__ Paged8Request paged8_request(const int32_t* q_start,
                                                        const int32_t* lengths, int b, int rows,
                                                        int width, bool rows_are_held,
                                                        int32_t* status) {
  return paged8_request(q_start[b], q_start[b + 1], lengths[b], rows, width, rows_are_held, status);
}

// ---- codes to fp16 pairs ----------------------------------------------------
// int8 q: the byte q + 128 under the exponent of 1024 is the fp16 number
// 1152 + q, one exact subtraction from q.
template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (FMT == P8_INT8) {
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140);
    const uint32_t b = __byte_perm(u, 0x64646464u, 0x4342);
    const uint32_t bias = 0x64806480u;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(bias));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(bias));
  } else {
    asm("{\n\t.reg .b16 x, y;\n\t"
        "mov.b32 {x, y}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, x;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, y;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float exp2_int(int e) { return __int_as_float((e + 127) << 23); }

}  // namespace hier
