// Attention of many rows over an 8-bit paged cache on the tensor cores
// (sm_100a: tcgen05, TMEM, bulk copies).
//
// One CTA per (256 (row, head) pairs of one key head, part of the keys): two
// 128-pair halves that ping-pong over one list of 128-key tiles (two pages
// each), as in the bf16 attention kernel:
//
//   S0(0) S1(0) | PV0(0) S0(1) PV1(0) S1(1) | PV0(1) S0(2) PV1(1) S1(2) | ...
//
// A tile of at most 128 pairs has no second half: both halves then take the
// same pairs and every other key tile, S0(0) S1(1) | PV0(0) S0(2) | PV1(1) S1(3)
// | ..., and are joined through shared memory at the end.
//
// What differs is the operands.  Codes are exact in fp16, so keys and values
// are turned into fp16 tiles in shared memory by a warpgroup of their own and
// both products run as kind::f16 on fp16 operands: the queries are brought
// into fp16's range by a power of two per row when they are loaded (bf16 keeps
// all its bits), the weights are rounded to fp16 (11 bits), and the page
// scales enter the exponents only (paged8_attn.cuh).  An fp8 product would
// have to round the queries and the weights to 4 bits.  Both operands of both
// products are K-major: the value pages are stored with the tokens along the
// row.
//
// Warp roles (512 threads, four warpgroups):
//   warp 0       loads pages: bulk copies of 8 KiB (page, head) blocks, one
//                16 KiB stage for keys and one for values, two of each for a
//                dual tile, which has no second query tile
//   warp 1       MMA issuer (one lane), TMEM allocator
//   warps 4-7    codes -> fp16 tiles (two stages of each)
//   warps 8-11   queries and softmax of half 0, one pair per thread
//   warps 12-15  the same of half 1
// Shared memory: Q 2 x 32 KiB, K and V 2 x 32 KiB each, codes 2 x 16 KiB.
// Tensor memory: S0 | S1 | O0 | O1, P over the first half of its S.
// Every mbarrier wait is bounded and records a timeout in dev_err.
//
// Bound by the chain of each half, scores to weights to products: no unit is busy
// for more than 53 % of the time (tensor pipe 46, tensor memory 53, issue slots
// 48), and one instruction more per pair of weights costs 5 %.  A 128-key tile of
// two halves takes about 3 870 cycles from e4m3 codes, against 3 216 for its four
// products; a tile of one half 2 500 to 2 750.  A CTA adds 11 us (finding its tile
// 2.4, queries 3.2, first scores 1, last products and output 3.4).  One sequence of
// 9 240 rows, causal by 220, 24 heads, e4m3: 556 us = 966 TFLOP/s of the pairs seen
// at 1 965 MHz, 590 us in calls for seconds, at 1 845 MHz under the power cap.  The
// code of all roles is large and runs the faster the smaller it is: one converter
// for keys and values 206 us against 222 (4 requests' chunks of 660 rows over 4 620
// keys, int8), 210 now.

#include <type_traits>

#include "paged8_attn.cuh"
#include "tile_mma.cuh"

namespace hier {
namespace {

constexpr int kRows = kPaged8LargeRows;
constexpr int kStages = 2;
constexpr int kThreads = 512;
constexpr int kSmemQ = 0;
constexpr int kSmemK = 2 * kTile;
constexpr int kSmemV = kSmemK + kStages * kTile;
constexpr int kSmemRaw = kSmemV + kStages * kTile;  // codes of a key tile, of a value tile
constexpr int kRawTile = 2 * kPageHeadBytes;
constexpr int kSmemBar = kSmemRaw + 2 * kRawTile;
constexpr int kNumBars = 1 + 4 * kStages + 8 + 8 + 1;
constexpr int kSmemBytes = kSmemBar + 256 + 1024;  // + slack for 1024-byte alignment
static_assert(kSmemBytes <= 227 * 1024, "shared memory of one CTA");
static_assert(kNumBars * 8 + 8 <= 256, "barriers and the TMEM slot");
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;

constexpr float kRescaleThreshold = 8.0f;  // log2 units
constexpr uint32_t kRegsControl = 40;
constexpr uint32_t kRegsConvert = 72;
constexpr uint32_t kRegsSoftmax = 200;
static_assert(128 * (kRegsControl + kRegsConvert) + 256 * kRegsSoftmax <= kThreads * 128,
              "register split exceeds the launch allocation");

struct Bars {
  uint64_t* q_full;
  uint64_t* k_full;
  uint64_t* k_empty;
  uint64_t* v_full;
  uint64_t* v_empty;
  uint64_t* raw_full;   // [stage][keys, values]
  uint64_t* raw_empty;
  uint64_t* s_full;     // [half]
  uint64_t* p_full;
  uint64_t* p_lo;
  uint64_t* o_final;
  uint64_t* drained;    // a failed issuer's products are over
};

// fp16 operands, fp32 accumulation, both K-major
constexpr uint32_t kIdesc = (1u << 4) | (static_cast<uint32_t>(128 >> 3) << 17) |
                            (static_cast<uint32_t>(128 >> 4) << 24);

template <int k>
__device__ __forceinline__ void s_step(uint32_t d, uint32_t qlo, uint32_t klo) {
  constexpr uint32_t off = ((k >> 2) * kHalf + (k & 3) * 32) >> 4;
  umma_ss_lo<off, off>(d, qlo, klo, kIdesc, k > 0 ? 1u : 0u);
}
__device__ __forceinline__ void issue_s_f16(uint32_t d, uint32_t qlo, uint32_t klo) {
  s_step<0>(d, qlo, klo), s_step<1>(d, qlo, klo), s_step<2>(d, qlo, klo), s_step<3>(d, qlo, klo);
  s_step<4>(d, qlo, klo), s_step<5>(d, qlo, klo), s_step<6>(d, qlo, klo), s_step<7>(d, qlo, klo);
}
template <int k>
__device__ __forceinline__ void pv_step(uint32_t o, uint32_t p, uint32_t vlo, bool acc) {
  constexpr uint32_t off = ((k >> 2) * kHalf + (k & 3) * 32) >> 4;
  umma_ts_lo<k * 8, off>(o, p, vlo, kIdesc, (acc || k > 0) ? 1u : 0u);
}
template <int H>
__device__ __forceinline__ void issue_pv_f16(uint32_t o, uint32_t p, uint32_t vlo, bool acc) {
  pv_step<4 * H>(o, p, vlo, acc), pv_step<4 * H + 1>(o, p, vlo, acc);
  pv_step<4 * H + 2>(o, p, vlo, acc), pv_step<4 * H + 3>(o, p, vlo, acc);
}

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// What every role of a CTA works from.
struct Job {
  Paged8Tile tl;
  int kvh;
  int page0, n_kv;       // first page, 128-key tiles of this part
  int page_end;          // pages from here on are not this part's
  int lo[2], hi[2];      // keys that a half's rows see between them (lo = hi: none)
  bool dual;             // one half's pairs, the key tiles shared out to both
  int raw_stages;        // stages of codes: 2 where the second query tile's place is free
  const int32_t* row;    // block table row
};

// the half works on the tile that starts at page p: its rows see some key of
// it, or the tile is the half's share
__device__ __forceinline__ bool uses(const Job& J, int h, int p) {
  if (J.dual) return (((p - J.page0) >> 1) & 1) == h;
  return p * kPage < (h ? J.hi[1] : J.hi[0]) && (p + 2) * kPage > (h ? J.lo[1] : J.lo[0]);
}

// Table entries are read ahead of their use and checked there, so that no role
// waits for one: -1 behind the part's pages.
__device__ __forceinline__ int entry(const Job& J, int p) {
  return p < J.page_end ? __ldg(J.row + p) : -1;
}
__device__ __forceinline__ uint8_t* raw_stage(uint8_t* smem, int stage, int kind) {
  return smem + (stage ? kSmemQ + kTile : kSmemRaw) + kind * kRawTile;
}
__device__ __forceinline__ bool in_pool(const Paged8Args& a, int page) {
  return page >= 0 && page < a.n_pages;
}

// Returns how many tiles of keys and of values, in turn, it has asked for.
__device__ __forceinline__ int load_role(const Paged8Args& a, const Job& J, uint8_t* smem,
                                          const Bars& B) {
  const int64_t page_bytes = (int64_t)a.kv_heads * kPageHeadBytes;
  const uint8_t* k = a.k + (int64_t)J.kvh * kPageHeadBytes;
  const uint8_t* v = a.v + (int64_t)J.kvh * kPageHeadBytes;
  int pg0 = entry(J, J.page0), pg1 = entry(J, J.page0 + 1);
  for (int j = 0; j < J.n_kv; ++j) {
    const int p = J.page0 + 2 * j;
    const int raw = j % J.raw_stages, raw_phase = ((j / J.raw_stages) - 1) & 1;
    const bool have0 = in_pool(a, pg0), have1 = in_pool(a, pg1);
    const int64_t at0 = pg0 * page_bytes, at1 = pg1 * page_bytes;
    pg0 = entry(J, p + 2), pg1 = entry(J, p + 3);
    if (!have0 || (!have1 && p + 1 < J.page_end)) atomicOr(a.status, P8_BAD_PAGE);
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      uint64_t* full = B.raw_full + 2 * raw + kind;
      if (j >= J.raw_stages && !mbar_wait(B.raw_empty + 2 * raw + kind, raw_phase, a.err, 40 + kind))
        return 2 * j + kind;
      mbar_arrive_expect_tx(full, (have0 + have1) * kPageHeadBytes);
      uint8_t* dst = raw_stage(smem, raw, kind);
      if (have0) bulk_load(dst, (kind ? v : k) + at0, kPageHeadBytes, full);
      if (have1) bulk_load(dst + kPageHeadBytes, (kind ? v : k) + at1, kPageHeadBytes, full);
    }
  }
  return 2 * J.n_kv;
}

// No copy outlives the block, whoever else gave up.
__device__ __forceinline__ void load_drain(const Paged8Args& a, const Job& J, const Bars& B, int issued) {
  for (int i = max(0, issued - 2 * J.raw_stages); i < issued; ++i) {
    const int j = i >> 1;
    mbar_wait(B.raw_full + 2 * (j % J.raw_stages) + (i & 1), (j / J.raw_stages) & 1, a.err, 52);
  }
}

__device__ __forceinline__ void mma_role(const Paged8Args& a, const Job& J, uint32_t tbase,
                                         uint8_t* smem, const Bars& B) {
  const uint32_t q_lo[2] = {sdesc_lo_kmajor(smem_u32(smem + kSmemQ)),
                            sdesc_lo_kmajor(smem_u32(smem + kSmemQ + (J.dual ? 0 : kTile)))};
  const uint32_t k_lo0 = sdesc_lo_kmajor(smem_u32(smem + kSmemK));
  const uint32_t v_lo0 = sdesc_lo_kmajor(smem_u32(smem + kSmemV));
  int cp[2] = {0, 0};  // PVs issued per half
  if (!mbar_wait(B.q_full, 0, a.err, 42)) return;
  if (J.dual) {
    // tile j is half j % 2's, and so are the stages it passes through
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (j >= J.n_kv) break;
      if (!mbar_wait(B.k_full + j, 0, a.err, 43)) return;
      tc_fence_after();
      issue_s_f16(tbase + j * kBN, q_lo[j], k_lo0 + ((j * kTile) >> 4));
      umma_commit(B.s_full + j);
      umma_commit(B.k_empty + j);
    }
    for (int j = 0; j < J.n_kv; ++j) {
      const int h = j & 1, phase = (j >> 1) & 1;
      const uint32_t o_t = tbase + kColO + h * kBN, p_t = tbase + h * kBN;
      const uint32_t v_lo = v_lo0 + ((h * kTile) >> 4);
      if (!mbar_wait(B.v_full + h, phase, a.err, 44)) return;
      if (!mbar_wait(B.p_lo + h, phase, a.err, 45)) return;
      tc_fence_after();
      issue_pv_f16<0>(o_t, p_t, v_lo, j > 1);
      if (!mbar_wait(B.p_full + h, phase, a.err, 46)) return;
      tc_fence_after();
      issue_pv_f16<1>(o_t, p_t, v_lo, true);
      umma_commit(B.v_empty + h);
      if (j + 2 < J.n_kv) {
        if (!mbar_wait(B.k_full + h, ((j + 2) / kStages) & 1, a.err, 43)) return;
        tc_fence_after();
        issue_s_f16(p_t, q_lo[h], k_lo0 + ((h * kTile) >> 4));
        umma_commit(B.s_full + h);
        umma_commit(B.k_empty + h);
      }
    }
    umma_commit(B.o_final);
    umma_commit(B.o_final + 1);
    return;
  }
  // every phase of the stage barriers is waited for, used or not
  if (!mbar_wait(B.k_full, 0, a.err, 43)) return;
  tc_fence_after();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (!uses(J, h, J.page0)) continue;
    issue_s_f16(tbase + h * kBN, q_lo[h], k_lo0);
    umma_commit(B.s_full + h);
  }
  umma_commit(B.k_empty);
  for (int j = 0; j < J.n_kv; ++j) {
    const bool more = j + 1 < J.n_kv;
    const int p = J.page0 + 2 * j;
    const int stv = j % kStages, stk = (j + 1) % kStages;
    if (!mbar_wait(B.v_full + stv, (j / kStages) & 1, a.err, 44)) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (uses(J, h, p)) {
        const uint32_t o_t = tbase + kColO + h * kBN, p_t = tbase + h * kBN;
        const uint32_t v_lo = v_lo0 + ((stv * kTile) >> 4);
        if (!mbar_wait(B.p_lo + h, cp[h] & 1, a.err, 45)) return;
        tc_fence_after();
        issue_pv_f16<0>(o_t, p_t, v_lo, cp[h] > 0);
        if (!mbar_wait(B.p_full + h, cp[h] & 1, a.err, 46)) return;
        tc_fence_after();
        issue_pv_f16<1>(o_t, p_t, v_lo, true);
        ++cp[h];
      }
      if (!more) continue;
      if (h == 0 && !mbar_wait(B.k_full + stk, ((j + 1) / kStages) & 1, a.err, 43)) return;
      if (uses(J, h, p + 2)) {
        tc_fence_after();
        issue_s_f16(tbase + h * kBN, q_lo[h], k_lo0 + ((stk * kTile) >> 4));
        umma_commit(B.s_full + h);
      }
    }
    umma_commit(B.v_empty + stv);
    if (more) umma_commit(B.k_empty + stk);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
    if (cp[h] > 0) umma_commit(B.o_final + h);
}

// A page's 128 lines of 64 codes (keys: 64 of each dimension half; values: one
// per dimension) become lines of 128 bytes in the swizzled tile.  Eight lanes
// read two lines of codes (128 bytes) and write two lines of eight different
// 16-byte columns: no bank conflicts either way.  A thread takes 16 bytes of
// lines line0, line0 + 32, .. of both pages; pages that are not there are zeros.
template <int FMT>
__device__ __forceinline__ void convert_tile(const uint8_t* raw, uint8_t* dst, bool kValues, bool have0,
                                             bool have1, int tid) {
  const int t = tid & 3, line0 = tid >> 2;
  const uint8_t* src = raw + tid * 16;
  // (the line's swizzle is that of line0: the others are multiples of 8 away)
  uint8_t* lo = dst + line0 * 128 + (((2 * t) ^ (line0 & 7)) << 4);
  uint8_t* hi = dst + line0 * 128 + (((2 * t + 1) ^ (line0 & 7)) << 4);
  // offsets of the second page's lines and, of a page, of its second 64 lines
  const int next_page = kValues ? kHalf : 64 * 128, next_half = kValues ? 64 * 128 : kHalf;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int page = i >> 2, line = 32 * (i & 3);  // + line0
    const int off = page * next_page + (line >> 6) * next_half + (line & 63) * 128;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (page ? have1 : have0)
      v = *reinterpret_cast<const uint4*>(src + page * kPageHeadBytes + line * 64);
    uint32_t o[8];
    decode4<FMT>(v.x, o[0], o[1]);
    decode4<FMT>(v.y, o[2], o[3]);
    decode4<FMT>(v.z, o[4], o[5]);
    decode4<FMT>(v.w, o[6], o[7]);
    *reinterpret_cast<uint4*>(lo + off) = make_uint4(o[0], o[1], o[2], o[3]);
    *reinterpret_cast<uint4*>(hi + off) = make_uint4(o[4], o[5], o[6], o[7]);
  }
}

// The proxy fence also ends the reads of the codes before their stage is given
// back to the copies.
template <int FMT>
__device__ __forceinline__ void convert_role(const Paged8Args& a, const Job& J, uint8_t* smem,
                                             const Bars& B, int tid) {
  int pg0 = entry(J, J.page0), pg1 = entry(J, J.page0 + 1);
  for (int j = 0; j < J.n_kv; ++j) {
    const int st = j % kStages, raw = j % J.raw_stages, raw_phase = (j / J.raw_stages) & 1;
    const bool have0 = in_pool(a, pg0), have1 = in_pool(a, pg1);
    pg0 = entry(J, J.page0 + 2 * j + 2), pg1 = entry(J, J.page0 + 2 * j + 3);
#pragma unroll 1
    for (int kind = 0; kind < 2; ++kind) {
      uint64_t* empty = (kind ? B.v_empty : B.k_empty) + st;
      if (j >= kStages && !mbar_wait(empty, ((j / kStages) - 1) & 1, a.err, 47)) return;
      if (!mbar_wait(B.raw_full + 2 * raw + kind, raw_phase, a.err, 48)) return;
      convert_tile<FMT>(raw_stage(smem, raw, kind), smem + (kind ? kSmemV : kSmemK) + st * kTile, kind,
                        have0, have1, tid);
      fence_proxy_async_smem();
      mbar_arrive((kind ? B.v_full : B.k_full) + st);
      mbar_arrive(B.raw_empty + 2 * raw + kind);
    }
  }
}

// bits [a, b) of the 32 keys that start at key k
__device__ __forceinline__ uint32_t key_bits(int lo, int hi, int k) {
  const int a = min(32, max(0, lo - k)), b = min(32, max(0, hi - k));
  const uint32_t below_a = a >= 32 ? ~0u : (1u << a) - 1u, below_b = b >= 32 ? ~0u : (1u << b) - 1u;
  return below_b & ~below_a;
}

// 32 bytes to a 32-byte aligned global address
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
               "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

__device__ __forceinline__ void tmem_ld16(uint32_t col, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(col));
  tmem_wait_ld();
}

// The denominator's terms of a tile's pages that are far_page, from the scores
// where they lie (factors c0, c1; the row sees keys lo to hi of the tile).  One
// at a time: eight took 1.5 % more of calls without such a page, for its code.
__device__ __forceinline__ float far_sum(uint32_t s_col, float c0, float c1, float n, int lo, int hi,
                                         bool far0, bool far1) {
  float sum = 0.f;
#pragma unroll 1
  for (int q = 0; q < 128; ++q) {
    uint32_t r;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(s_col + q));
    tmem_wait_ld();
    const float p = ex2_approx(fmaf(__uint_as_float(r), q < 64 ? c0 : c1, -n));
    sum += (q < 64 ? far0 : far1) && q >= lo && q < hi ? p : 0.f;
  }
  return sum;
}

__device__ __forceinline__ void rescale_o(uint32_t o_col, float alpha) {
#pragma unroll 1
  for (int q = 0; q < 16; ++q) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
                   "=r"(r[6]), "=r"(r[7])
                 : "r"(o_col + q * 8));
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                 ::"r"(o_col + q * 8), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                   "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  }
}

// The 32 query rows of a warp (its lanes' pairs) to registers, a lane column
// lane % 16 of row 2i + lane / 16: half a warp copies a row, all copies in flight
// together.  They go through the tile's place in shared memory: what is left of
// the L1 cache beside 227 KB of it could not hold 64 KB of loads in flight.
// at: element offset of the lane's row in q, < 0 for none.
__device__ __forceinline__ void read_queries(const Paged8Args& a, int64_t at, uint8_t* tile, int row0,
                                             int lane, uint4 (&v)[16]) {
  uint8_t* dst = tile + (row0 + (lane >> 4)) * 256 + (lane & 15) * 16;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t from = __shfl_sync(0xffffffffu, at, 2 * i + (lane >> 4));
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst + i * 512)),
                 "l"(a.q + (from >= 0 ? from : 0) + (lane & 15) * 8), "r"(from >= 0 ? 16 : 0)
                 : "memory");
  }
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = *reinterpret_cast<const uint4*>(dst + i * 512);
}

// Returns the factor of the lane's scores: scale * log2(e) over the power of
// two its row is multiplied by.
__device__ __forceinline__ float stage_queries(const Paged8Args& a, const uint4 (&v)[16], uint8_t* tile,
                                               int row0, int lane) {
  const int c = lane & 15;  // 16-byte column of the rows 2i + (lane >> 4)
  // the largest magnitudes as bits, pairs of 16 (NaN above infinity)
  uint32_t big[16];
#pragma unroll
  for (int i = 0; i < 16; ++i)
    big[i] = __vmaxu2(__vmaxu2(v[i].x & 0x7fff7fffu, v[i].y & 0x7fff7fffu),
                      __vmaxu2(v[i].z & 0x7fff7fffu, v[i].w & 0x7fff7fffu));
  // sixteen rows over sixteen lanes: each step halves the rows that a lane keeps,
  // and column c ends with row 2c + (lane >> 4)
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) {
    const bool up = (c & o) != 0;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const uint32_t give = up ? big[i] : big[i + o], keep = up ? big[i + o] : big[i];
      big[i] = __vmaxu2(keep, __shfl_xor_sync(0xffffffffu, give, o));
    }
  }
  const int sh = fp16_shift(__uint_as_float(max(big[0] << 16, big[0] & 0xffff0000u)));
  const float mine = exp2_int(sh), factor = a.scale_log2 * exp2_int(-sh);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float f = __shfl_sync(0xffffffffu, mine, (lane & 16) + i);
    const uint64_t f2 = f2_pack(f, f);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v[i]);
    uint32_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x, y;
      f2_unpack(f2_mul(f2_pack(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u)), f2), x, y);
      o[j] = pack_f16x2(x, y);
    }
    const int r = row0 + 2 * i + (lane >> 4);
    *reinterpret_cast<uint4*>(tile + (c >> 3) * kHalf + r * 128 + (((c & 7) ^ (r & 7)) << 4)) =
        make_uint4(o[0], o[1], o[2], o[3]);
  }
  return __shfl_sync(0xffffffffu, factor, ((lane & 1) << 4) + (lane >> 1));
}

// A page's scales as read; what is derived from them is computed at their use.
struct PageScale {
  float ks, vs;
  bool have;
};

__device__ __forceinline__ PageScale page_scale(const Paged8Args& a, const Job& J, int page) {
  PageScale s = {0.f, 1.f, in_pool(a, page)};
  if (s.have) {
    const int64_t at = (int64_t)page * a.kv_heads + J.kvh;
    s.ks = __ldg(a.k_scale + at);
    s.vs = __ldg(a.v_scale + at);
  }
  return s;
}

__device__ __forceinline__ void softmax_role(const Paged8Args& a, const Job& J, int split, int parts,
                                             uint32_t tbase, int warp, uint8_t* smem,
                                             const Bars& B) {
  const int h = (warp >> 2) - 2;
  const int row = threadIdx.x - 256 - 128 * h;
  const uint32_t lane_base = static_cast<uint32_t>(32 * (warp & 3)) << 16;
  const uint32_t s_col = tbase + lane_base + h * kBN;
  const uint32_t o_col = tbase + lane_base + kColO + h * kBN;
  const int half0 = J.tl.rho0 + (J.dual ? 0 : 128 * h);  // first pair of the half
  const int rho = half0 + row;
  const bool in_row = rho < J.tl.pairs;
  const int qi = (in_row ? rho : 0) / a.group;
  const int head = J.kvh * a.group.d + (in_row ? rho - qi * a.group.d : 0);
  const int64_t grow = J.tl.rq.row0 + (int64_t)qi;
  float m_run = -INFINITY, n_run = -INFINITY, l_run = 0.f;
  int c = 0;
  bool lost = false;  // a wait ran out: nothing more is waited for or written
  if (J.n_kv > 0) {
    uint4 qv[16];
    uint8_t* q_tile = smem + kSmemQ + (J.dual ? 0 : h * kTile);
    read_queries(a, in_row ? grow * a.q_stride + head * 128 : -1, q_tile, row & ~31,
                 lane_id(), qv);
    named_barrier(1, 256);  // every row is in registers: the tile may be written
    const float sc = stage_queries(a, qv, q_tile, row & ~31, lane_id());
    fence_proxy_async_smem();
    mbar_arrive(B.q_full);
    int lo = 0, hi = 0;
    if (in_row) row_keys(a, J.tl.rq, qi, lo, hi);
    // tiles that every row of the half sees whole need no mask
    int all_lo, all_hi, unused;
    {
      const int first = half0, last = min(first + 128, J.tl.pairs) - 1;
      all_lo = INT_MAX, all_hi = 0;
      if (first <= last) {
        row_keys(a, J.tl.rq, last / a.group, all_lo, unused);
        row_keys(a, J.tl.rq, first / a.group, unused, all_hi);
      }
    }
    PageScale n0 = page_scale(a, J, entry(J, J.page0)), n1 = page_scale(a, J, entry(J, J.page0 + 1));
    int pg0 = entry(J, J.page0 + 2), pg1 = entry(J, J.page0 + 3);
    for (int j = 0; j < J.n_kv; ++j) {
      const int p = J.page0 + 2 * j;
      // scales one tile ahead, table entries two
      const PageScale e0 = n0, e1 = n1;
      n0 = page_scale(a, J, pg0), n1 = page_scale(a, J, pg1);
      pg0 = entry(J, p + 4), pg1 = entry(J, p + 5);
      if (!uses(J, h, p)) continue;
      const bool b0 = e0.have, b1 = e1.have;
      const float c0 = score_factor(sc, e0.ks), c1 = score_factor(sc, e1.ks);
      const int ve0 = scale_log2_of(e0.vs), ve1 = scale_log2_of(e1.vs);
      const int k0 = p * kPage;
      const bool partial = !(k0 >= all_lo && k0 + 2 * kPage <= all_hi && b0 && b1);
      // S_h is committed after the half's previous PV, so once it is visible O
      // holds every earlier product and can be rescaled without another wait
      if (!mbar_wait(B.s_full + h, c & 1, a.err, 49)) {
        lost = true;
        break;
      }
      tc_fence_after();
      float sv[kBN];
      {
        uint32_t* r = reinterpret_cast<uint32_t*>(sv);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          tmem_ld32(s_col + q * 32, *reinterpret_cast<uint32_t(*)[32]>(r + 32 * q));
        tmem_wait_ld();
      }
      if (partial) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t w = (q < 2 ? b0 : b1) ? key_bits(lo, hi, k0 + 32 * q) : 0u;
#pragma unroll
          for (int i = 0; i < 32; ++i) sv[32 * q + i] = ((w >> i) & 1u) ? sv[32 * q + i] : -INFINITY;
        }
      }
      float m8[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) m8[i] = sv[i], m8[4 + i] = sv[64 + i];
#pragma unroll
      for (int i = 4; i < 64; ++i) {
        m8[i & 3] = fmaxf(m8[i & 3], sv[i]);
        m8[4 + (i & 3)] = fmaxf(m8[4 + (i & 3)], sv[64 + i]);
      }
      const float x0 = fmaf(fmaxf(fmaxf(m8[0], m8[1]), fmaxf(m8[2], m8[3])), c0, (float)ve0);
      const float x1 = fmaf(fmaxf(fmaxf(m8[4], m8[5]), fmaxf(m8[6], m8[7])), c1, (float)ve1);
      const float mx = fmaxf(x0, x1);
      const bool grow_max = mx > m_run + kRescaleThreshold;
      const bool need_rescale = grow_max && m_run != -INFINITY;
      const float m_new = grow_max ? mx : m_run, ref = finite_or_0(m_new);
      bool far0 = false, far1 = false;
      float own = 0.f;
      if (__any_sync(0xffffffffu, need_rescale || ref - fminf(x0, x1) > kFarWeights)) {
        if (__any_sync(0xffffffffu, need_rescale))
          rescale_o(o_col, need_rescale ? ex2_approx(m_run - ref) : 1.f);
        const float nref = finite_or_0(fmaxf(n_run, fmaxf(x0 - (float)ve0, x1 - (float)ve1)));
        far0 = far_page(ref, x0, nref, x0 - (float)ve0), far1 = far_page(ref, x1, nref, x1 - (float)ve1);
        if (__any_sync(0xffffffffu, far0 || far1))
          own = far_sum(s_col, c0, c1, nref, lo - k0, hi - k0, far0, far1);
      }
      m_run = m_new;
      float sums[2];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float ch = half ? c1 : c0, vh = (float)(half ? ve1 : ve0), rh = vh - ref;
        const uint64_t sc2 = f2_pack(ch, ch), ref2 = f2_pack(rh, rh);
        uint64_t acc[4] = {0ull, 0ull, 0ull, 0ull};
        uint32_t pk[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const uint64_t arg = f2_fma(f2_pack(sv[64 * half + 2 * i], sv[64 * half + 2 * i + 1]), sc2, ref2);
          float a0, a1;
          f2_unpack(arg, a0, a1);
          const float p0 = ex2_approx(a0), p1 = ex2_approx(a1);
          acc[i & 3] = f2_add(acc[i & 3], f2_pack(p0, p1));
          pk[i] = pack_f16x2(p0, p1);
        }
        tmem_st32(s_col + 32 * half, pk);
        if (half == 0) {  // keys 0-63 of P: the first half of PV can start
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(B.p_lo + h);
        }
        float s0, s1;
        f2_unpack(f2_add(f2_add(acc[0], acc[1]), f2_add(acc[2], acc[3])), s0, s1);
        sums[half] = s0 + s1;
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(B.p_full + h);
      const float top0 = x0 - (float)ve0, top1 = x1 - (float)ve1;
      const float n_new = fmaxf(n_run, fmaxf(top0, top1)), nref = finite_or_0(n_new);
      l_run = fmaf(l_run, ex2_approx(n_run - nref), own);
      if (!far0) l_run = fmaf(sums[0], sum_factor(ref, (float)ve0, nref), l_run);
      if (!far1) l_run = fmaf(sums[1], sum_factor(ref, (float)ve1, nref), l_run);
      n_run = n_new;
      ++c;
    }
  }
  if (c > 0 && !lost) {
    lost = !mbar_wait(B.o_final + h, 0, a.err, 50);
    tc_fence_after();
  }
  // The halves of a dual tile joined: the second leaves its outputs, column by
  // column, where the queries were (every product is done), the first adds them.
  float* other = reinterpret_cast<float*>(smem + kSmemQ) + row;
  float2* other_nl = reinterpret_cast<float2*>(smem + kSmemRaw) + row;
  OutFactor keep(m_run, n_run, l_run);
  float add = 0.f;
  if (J.dual && J.n_kv > 0) {
    named_barrier(1, 256);
    if (h == 1) {
      if (!lost) {
#pragma unroll 1
        for (int q = 0; q < 8; ++q) {
          uint32_t r[16];
          if (c > 0) tmem_ld16(o_col + q * 16, r);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            other[(16 * q + i) * 128] = c > 0 ? __uint_as_float(r[i]) * keep.a * keep.b : 0.f;
        }
      }
      *other_nl = make_float2(n_run, l_run);
    }
    named_barrier(1, 256);
    if (h == 1) return;
    const float2 nl = *other_nl;
    const float N = fmaxf(n_run, nl.x);
    const float mine = l_run * ex2_approx(n_run - finite_or_0(N)), theirs = nl.y * ex2_approx(nl.x - finite_or_0(N));
    n_run = N, l_run = mine + theirs;
    const float inv = inverse_or_0(l_run);
    keep.a *= mine * inv, add = theirs * inv;
  } else if (J.dual && h == 1) {
    return;
  }
  if (lost) return;
  const bool whole = parts == 1;
  __nv_bfloat16* orow = a.out + grow * a.out_stride + head * 128;
  const int64_t at = whole ? 0 : ((int64_t)blockIdx.x * kRows + (rho - J.tl.rho0));
  if (in_row) {
    if (whole) {
      if (a.lse) a.lse[grow * a.heads + head] = row_lse(n_run, l_run);
    } else {
      *reinterpret_cast<float2*>(a.part_nl + at * 2) = make_float2(n_run, l_run);
    }
  }
#pragma unroll 1
  for (int q = 0; q < 8; ++q) {
    uint32_t r[16];
    if (c > 0) {
      tmem_ld16(o_col + q * 16, r);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] = 0u;
    }
    if (!in_row) continue;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float v = __uint_as_float(r[i]) * keep.a * keep.b;
      if (J.dual && J.n_kv > 0) v = fmaf(other[(16 * q + i) * 128], add, v);
      r[i] = __float_as_uint(v);
    }
    if (whole) {
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i] = pack_bf16x2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
      if ((reinterpret_cast<uintptr_t>(orow) & 31) == 0) {
        st_global_v8(orow + q * 16, w);
      } else {
        uint4* dst = reinterpret_cast<uint4*>(orow + q * 16);
#pragma unroll
        for (int k = 0; k < 2; ++k)
          dst[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
      }
    } else {
      uint4* dst = reinterpret_cast<uint4*>(a.part_o + at * 128 + q * 16);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        dst[k] = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
    }
  }
}

template <int FMT>
__global__ void __launch_bounds__(kThreads, 1) paged8_mma_kernel(Paged8Args a, int64_t tiles) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  asm volatile("griddepcontrol.launch_dependents;");
  const int warp = warp_id(), lane = lane_id();
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kSmemBar);
  Bars B;
  B.q_full = bars;
  B.k_full = B.q_full + 1;
  B.k_empty = B.k_full + kStages;
  B.v_full = B.k_empty + kStages;
  B.v_empty = B.v_full + kStages;
  B.raw_full = B.v_empty + kStages;
  B.raw_empty = B.raw_full + 4;
  B.s_full = B.raw_empty + 4;
  B.p_full = B.s_full + 2;
  B.p_lo = B.p_full + 2;
  B.o_final = B.p_lo + 2;
  B.drained = B.o_final + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kNumBars);
  if (threadIdx.x == 0) {
    mbar_init(B.q_full, 256);
    mbar_init(B.drained, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(B.k_full + s, 128);
      mbar_init(B.k_empty + s, 1);
      mbar_init(B.v_full + s, 128);
      mbar_init(B.v_empty + s, 1);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(B.raw_full + i, 1);
      mbar_init(B.raw_empty + i, 128);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(B.s_full + i, 1);
      mbar_init(B.p_full + i, 128);
      mbar_init(B.p_lo + i, 128);
      mbar_init(B.o_final + i, 1);
    }
    fence_mbar_init();
  }
  // the last tiles of a request see the most keys: they come first
  const int unit = (int)blockIdx.x / a.splits, split = (int)blockIdx.x - unit * a.splits.d;
  const int64_t tile = tiles - 1 - unit / a.kv_heads;
  Job J;
  J.kvh = unit % a.kv_heads;
  J.tl = paged8_tile<kRows>(a, tile, threadIdx.x == 0 && split == 0 && J.kvh == 0);
  const bool rest = a.zero_rest && split == 0 && (warp & ~1) == 2;  // warps 2 and 3
  const int64_t rest0 = 2 * (int64_t)(unit / a.kv_heads) + (warp & 1);
  if (!J.tl.live || J.tl.pairs <= a.row_limit) {
    // (this kernel is by itself for one request at most, whose row starts may lie
    // behind every tile; block 0's is behind those of all requests)
    if (a.n == 1 && blockIdx.x == 0 && threadIdx.x == 0)
      paged8_request(a.q_start, a.lengths, 0, a.rows, a.width, false, a.status);
    if (rest) zero_rest(a, J.kvh, rest0, 2 * tiles, lane);
    return;
  }
  const int kv_all = (J.tl.np + 1) / 2;
  const int parts = parts_of<kPaged8LargeMin>(kv_all, a.splits);
  if (split >= parts) return;
  const int t0 = kv_all * split / parts, t1 = kv_all * (split + 1) / parts;
  J.page0 = J.tl.p0 + 2 * t0;
  J.n_kv = t1 - t0;
  J.page_end = min(J.tl.p0 + J.tl.np, J.tl.p0 + 2 * t1);
  J.dual = J.tl.pairs - J.tl.rho0 <= 128;
  J.raw_stages = J.dual ? 2 : 1;
  J.row = a.table + J.tl.b * a.table_stride;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int first = J.tl.rho0 + 128 * h, last = min(first + 128, J.tl.pairs) - 1;
    J.lo[h] = J.hi[h] = 0;
    int unused;
    if (first <= last) {
      row_keys(a, J.tl.rq, first / a.group, J.lo[h], unused);
      row_keys(a, J.tl.rq, last / a.group, unused, J.hi[h]);
      if (J.hi[h] <= J.lo[h]) J.lo[h] = J.hi[h] = 0;
    }
  }
  if (warp == 1) tmem_alloc(tmem_slot, kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  if (warp >= 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    softmax_role(a, J, split, parts, tbase, warp, smem, B);
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsConvert));
    if (J.n_kv > 0) convert_role<FMT>(a, J, smem, B, threadIdx.x - 128);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsControl));
    if (J.n_kv > 0 && lane == 0) {
      if (warp == 0) load_drain(a, J, B, load_role(a, J, smem, B));
      if (warp == 1) {
        mma_role(a, J, tbase, smem, B);
        umma_commit(B.drained);
        mbar_wait(B.drained, 0, a.err, 51);
      }
    }
    if (rest) zero_rest(a, J.kvh, rest0, 2 * tiles, lane);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tbase, kTmemCols);
  }
}

}  // namespace

int paged8_launch_large(const Paged8Args& a, int format, int64_t tiles, cudaStream_t st) {
  const int64_t blocks = tiles * a.kv_heads * a.splits;
  if (blocks > INT32_MAX) {
    set_error(HIER_EVALUE, "too many rows, requests and heads");
    return HIER_EVALUE;
  }
  auto* kernel = format == P8_INT8 ? paged8_mma_kernel<P8_INT8> : paged8_mma_kernel<P8_E4M3>;
  HIER_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kSmemBytes),
                  "cudaFuncSetAttribute(paged8_mma_kernel)");
  kernel<<<(unsigned)blocks, kThreads, kSmemBytes, st>>>(a, tiles);
  HIER_CHECK_CUDA(cudaGetLastError(), "paged8_mma_kernel launch");
  return HIER_OK;
}

}  // namespace hier
